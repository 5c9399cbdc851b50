"""The ends of what include/katamx_ops.h takes - scales, values and lengths far from the usual ones - through the kernels compiled for x86
(tests/fakehip/emulate_ops.cpp), against plain formulas in 64 bits."""
import ctypes

import pytest
import torch

import ops_ref as ref
from katago_amd import capi
from test_ops_emulated import PREC, Guarded, aligned_copy, eight, emu, ok  # noqa: F401 (emu: the fixture)


def check_linear_any(got, want, mag, k):
    """ref.check_linear where the formula's result may leave the output's type: what is beyond the type's largest number by more than the bound is
    infinite, with its sign (a sum may be off by `bound` before it is rounded: with terms that cancel, `mag` far above the result, that is many steps), what is
    below it by more than the bound is within it. Results between the two may be either."""
    t = got.dtype
    top = torch.finfo(t).max
    g = got.double()
    sums = 2 * ref.U * (k / 16 + 24) * mag
    bound = sums + ref.half(t) * (want.abs() + sums) + ref.SMALLEST[t] / 2 + (7 * 2.0 ** -13 * mag if t != torch.float32 else 0)
    over, fits = want.abs() - bound > top, want.abs() + bound < top
    assert bool((torch.isinf(g) & (g.sign() == want.sign()))[over].all())
    far = torch.where(fits, (g - want).abs(), torch.zeros_like(want))
    assert bool((far <= bound).all()), float((far / bound).max())
    assert int(fits.sum()) > want.numel() // 8


def spread_scales(rows, gen, low=-120, high=120):
    """one to a row, of any size and with every mantissa"""
    e = torch.randint(low, high + 1, (rows,), generator=gen).double()
    return (torch.exp2(e) * (1 + torch.rand(rows, generator=gen, dtype=torch.float64))).float()


def linear(emu, a, sa, w, sw, out, kind):  # noqa: F811
    (m, k), n = a.shape, w.shape[0]
    abuf, ap = aligned_copy(a, k)
    wbuf, wp = aligned_copy(w, k)
    y = Guarded(m, n, n + 5, ref.TYPES[out])
    args = capi.Linear8Args(out_type=PREC[out], scale_kind=kind, rows=m, n=n, k=k, a=ap, a_scales=sa.data_ptr(), w=wp, w_scales=sw.data_ptr(), out=y.ptr,
                            a_stride=k, w_stride=k, out_stride=n + 5)
    ok(emu, emu.kmx_linear8(0, None, ctypes.byref(args)))
    y.rest_untouched()
    return y.get()


@pytest.mark.parametrize("m,n,k,out", [(3, 40, 512, "fp32"), (3, 40, 512, "bf16"), (20, 33, 144, "fp16"), (70, 64, 512, "fp32"), (70, 130, 272, "bf16"),
                                       (128, 64, 1040, "fp16"), (2100, 130, 128, "bf16"), (2048, 128, 272, "fp16"), (2048, 128, 384, "bf16")])
def test_linear8_row_scales_of_any_size(emu, m, n, k, out):  # noqa: F811
    """Scales from 2^-120 to 2^120 on both sides: a large one must not carry a sum out of fp32 that the other brings back (few rows, tiles, short k)"""
    g = torch.Generator().manual_seed(m + k)
    (a, _), (w, _) = eight(m, k, "row", g), eight(n, k, "row", g)
    sa, sw = spread_scales(m, g), spread_scales(n, g)
    got = linear(emu, a, sa, w, sw, out, 1)
    check_linear_any(got, *ref.linear(ref.values(a, sa), ref.values(w, sw)), k)
    # one side all large, the other all small: every result is an ordinary number
    sa, sw = torch.rand(m, generator=g) * 1e35, torch.rand(n, generator=g) * 1e-37
    check_linear_any(linear(emu, a, sa, w, sw, out, 1), *ref.linear(ref.values(a, sa), ref.values(w, sw)), k)
