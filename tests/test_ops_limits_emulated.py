"""The ends of what include/katamx_ops.h takes - scales, values and lengths far from the usual ones - through the kernels compiled for x86
(tests/fakehip/emulate_ops.cpp), against plain formulas in 64 bits."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch

import ops_ref as ref
from conftest import REPO
from katago_amd import capi
from test_ops_emulated import PREC, Guarded, aligned_copy, eight, emu, ok, rotary_args  # noqa: F401 (emu: the fixture)


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


def rows_of_any_size(c, t, gen):
    """rows whose values are normal ones times a power of two each, from the type's smallest number to its largest, ordinary rows between them"""
    low, high = {torch.float16: (-22, 13), torch.bfloat16: (-131, 125), torch.float32: (-147, 125)}[t]
    e = list(range(low, high, 23 if t != torch.float16 else 5)) + [-51, -47, 62, 64, high] * (t != torch.float16)
    e = [v for x in e for v in (x, 0)]
    x = torch.randn(len(e), c, generator=gen, dtype=torch.float64).clamp(-3.9, 3.9)
    return (x * torch.exp2(torch.tensor(e).double())[:, None]).to(t)


@pytest.mark.parametrize("c", [50, 96, 384, 1000, 5000, 33000])
@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
def test_rms_norm_of_small_and_large_rows(emu, c, dtype):  # noqa: F811
    """Without eps: the squares of values below 1e-19 or beyond 1.8e19 leave fp32, their rows' norms are ordinary numbers. A row's result does not depend
    on what the others of its wave are."""
    t = ref.TYPES[dtype]
    x = rows_of_any_size(c, t, torch.Generator().manual_seed(c))
    n = x.shape[0]

    def call(x):
        y, codes, sc = torch.zeros_like(x), torch.zeros(x.shape, dtype=torch.float8_e4m3fn), torch.zeros(x.shape[0])
        a = capi.RmsNormArgs(type=PREC[dtype], scale_kind=1, rows=x.shape[0], channels=c, epsilon=0.0, x=x.data_ptr(), y=y.data_ptr(), codes=codes.data_ptr(),
                             scales=sc.data_ptr(), x_stride=c, y_stride=c, codes_stride=c)
        ok(emu, emu.kmx_rmsnorm(0, None, ctypes.byref(a)))
        return y, codes, sc

    y, codes, sc = call(x)
    some = x.abs().amax(1) > 0  # (16 bits: a row of the smallest numbers may be all zeros)
    want = ref.norm(x[some], eps=0.0)[1]
    ref.check_y(y[some], want)
    ref.check_codes(codes[some], sc[some], want, ref.norm_slack(want))
    assert bool(torch.isnan(y[~some].float()).all())  # 0 / 0
    for row in range(0, n, 7):
        assert torch.equal(call(x[row:row + 1].clone())[0][0].float().nan_to_num(7.0), y[row].float().nan_to_num(7.0))


def test_rms_norm_of_a_very_long_row(emu):  # noqa: F811
    """4 million channels of one value: 4096 squares a lane, whose sum must not collect a rounding each"""
    c = (1 << 22) + 8
    x = torch.full((1, c), 1.1)
    y = torch.zeros_like(x)
    a = capi.RmsNormArgs(type=capi.PREC_FP32, rows=1, channels=c, epsilon=0.0, x=x.data_ptr(), y=y.data_ptr(), x_stride=c, y_stride=c)
    ok(emu, emu.kmx_rmsnorm(0, None, ctypes.byref(a)))
    ref.check_y(y, ref.norm(x, eps=0.0)[1])


def rounded_quotients(v):
    """e4m3(v / (amax / 448)): the formula in 64 bits, its quotient rounded to fp32 (which restores one that lies on the border of two codes) and to e4m3"""
    v = v.double()
    return (v / (v.abs().amax(1, keepdim=True) / 448)).float().clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
def test_quantize_divides_as_the_formula(emu, dtype):  # noqa: F811
    """16-bit values lie on the border of two codes often enough that a product with the rounded reciprocal, or a quotient by the rounded scale, is told from
    the formula's quotient"""
    g, t = torch.Generator().manual_seed(3), ref.TYPES[dtype]
    for rows, c in ((400, 512), (3, 40000)):
        x = torch.randn(rows, c, generator=g).to(t)
        codes, sc = torch.zeros(rows, c, dtype=torch.uint8), torch.zeros(rows)
        ok(emu, emu.kmx_quantize(0, None, PREC[dtype], 1, rows, c, x.data_ptr(), c, codes.data_ptr(), c, sc.data_ptr()))
        assert torch.equal(sc, x.float().abs().amax(1) / 448)
        assert torch.equal(codes, rounded_quotients(x))


def small_sine_angles():
    """angles next to 0 and to quarters and halves of a turn, to either side, and between these"""
    near = torch.exp2(-torch.arange(2, 40, 0.25).double())
    places = torch.arange(-4, 5).double() / 4
    turns = (places[:, None, None] + torch.stack([near, -near])[None]).reshape(-1)
    return turns * 2 * torch.pi


def check_small_results(got, angle, magnitude=1.0):
    """(0, 1) and (1, 0) turned by `angle`: the results are the sine and the cosine themselves, each to be right relative to itself. fp32's roundings on the
    way: the reduced angle, three of the series' last steps, the magnitude, the result: 6 U, and 2 U for the steps before; the angle in turns
    is an fp64 number, off by 2^-53 of its size three times."""
    sin, cos = angle.sin() * magnitude, angle.cos() * magnitude
    for g, w in ((got[:, 0, 0], cos), (got[:, 0, 1], sin), (got[:, 1, 0], -sin), (got[:, 1, 1], cos)):
        far = (g.double() - w).abs()
        bound = 8 * ref.U * w.abs() + magnitude * 2.0 ** -50 * angle.abs()
        assert bool((far <= bound).all()), float((far / bound).max())


def test_rotary_of_small_sines(emu):  # noqa: F811
    """A sine next to 0 or to pi, a cosine next to pi / 2, in fp32"""
    angle = small_sine_angles()
    n = angle.shape[0]
    q = torch.eye(2).repeat(n, 1).reshape(1, 1, 2 * n, 2)  # two heads for each frequency
    out, pos, f = torch.empty_like(q), torch.ones(1, 1, 1, dtype=torch.int32), angle.reshape(n, 1, 1)
    ok(emu, emu.kmx_rotary(0, None, ctypes.byref(rotary_args(q, None, out, None, pos, f, "fp32", False, 1.0, False))))
    check_small_results(out.reshape(n, 2, 2), angle)


def block_scales(m, n, k, low, high, gen):
    """e8m0 codes of two matrices whose blocks of 32 are as far apart as `low` .. `high` allow and whose products are ordinary numbers"""
    e = torch.randint(low, high + 1, (k // 32,), generator=gen)
    e[:2] = torch.tensor([low, high])
    sa, sw = e.expand(m, -1), (low + high - e).expand(n, -1)
    near = torch.randint(0, 2, (n, k // 32), generator=gen)
    sw = (sw + near).clamp(max=high)
    return sa.to(torch.uint8).contiguous().view(torch.float8_e8m0fnu), sw.to(torch.uint8).contiguous().view(torch.float8_e8m0fnu)


def check_block_scales(run, m, n, k, gen):
    """run(a, sa, w, sw, out type) over the scales that each output's way takes: all of e8m0 but NaN into 16 bits, 2^-124 .. 2^119 into fp32"""
    a, w = (torch.randint(0, 256, (r, k), generator=gen).to(torch.uint8) for r in (m, n))
    for c in (a, w):
        c[c & 0x7f == 0x7f] = 0x3a
    a, w = a.view(torch.float8_e4m3fn), w.view(torch.float8_e4m3fn)
    for out, low, high in (("fp32", 3, 246), ("bf16", 0, 254)):
        sa, sw = block_scales(m, n, k, low, high, gen)
        check_linear_any(run(a, sa, w, sw, out), *ref.linear(ref.values(a, sa), ref.values(w, sw)), k)


@pytest.mark.parametrize("m,n,k", [(3, 40, 512), (20, 33, 96), (70, 64, 512), (130, 70, 288)])
def test_linear8_block_scales_at_their_ends(emu, m, n, k):  # noqa: F811
    check_block_scales(lambda a, sa, w, sw, out: linear(emu, a, sa, w, sw, out, 2), m, n, k, torch.Generator().manual_seed(m + k))


@pytest.mark.parametrize("mode", ["0", "1", "2"])
def test_linear8_large_tiles(emu, mode):  # noqa: F811
    """Tiles of 256 x 256 and of 128 x 128 with two stages and with four, which a chip of 256 CUs takes for far larger products: whole ones and partial ones,
    work-groups that go round several, k with steps between the first and the last ones. With copies into LDS that land at once (0), only when a wait requires
    it (1), or at the barrier behind that wait (2)."""
    code = r"""
import ctypes, os, sys
sys.path[:0] = [%r, %r]
import test_ops_emulated as t
lib = ctypes.CDLL(%r)
t.capi.bind_ops(lib)
lib.kmx_last_error.restype = ctypes.c_char_p
for cus, case in [("1", (768, 1024, 896, "row", "fp16", True)), ("1", (760, 1000, 672, "mx", "bf16", False)), ("1", (400, 600, 1168, "row", "fp32", True)),
                  ("1", (384, 384, 288, "mx", "fp32", False)), ("18", (384, 640, 1152, "row", "bf16", False)), ("18", (380, 600, 1184, "mx", "fp16", True))]:
    os.environ["KMX_EMU_CUS"] = cus
    print(cus, case, flush=True)
    t.test_linear8(lib, *case)
print("TILES_OK")
""" % (REPO, os.path.join(REPO, "tests"), emu._name)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, env=dict(os.environ, KMX_EMU_LATE_DMA=mode))
    assert r.returncode == 0 and "TILES_OK" in r.stdout, r.stdout[-500:] + r.stderr[-2000:]


def test_calls_on_another_device_than_the_current_one(emu):  # noqa: F811
    """A launch is made with the call's device current, and the thread's own is current again behind it, behind refusals too"""
    g = torch.Generator().manual_seed(1)
    x, codes, sc = torch.randn(70, 64, generator=g), torch.zeros(70, 64, dtype=torch.uint8), torch.zeros(70)
    y, rot = torch.zeros(70, 64), torch.zeros(1, 70, 1, 64)
    a, sa = eight(70, 64, "row", g)
    buf, p = aligned_copy(a, 64)
    out = torch.zeros(70, 70)
    norm = capi.RmsNormArgs(type=capi.PREC_FP32, rows=70, channels=64, epsilon=1e-6, x=x.data_ptr(), y=y.data_ptr(), x_stride=64, y_stride=64)
    lin = capi.Linear8Args(out_type=capi.PREC_FP32, scale_kind=1, rows=70, n=70, k=64, a=p, a_scales=sa.data_ptr(), w=p, w_scales=sa.data_ptr(), out=out.data_ptr(),
                           a_stride=64, w_stride=64, out_stride=70)
    pos, f = torch.zeros(1, 70, 1, dtype=torch.int32), torch.ones(1, 1, 32, dtype=torch.float64)
    turn = rotary_args(x.reshape(1, 70, 1, 64), None, rot, None, pos, f, "fp32", False, 1.0, False)
    calls = [lambda d: emu.kmx_rmsnorm(d, None, ctypes.byref(norm)), lambda d: emu.kmx_linear8(d, None, ctypes.byref(lin)), lambda d: emu.kmx_rotary(d, None, ctypes.byref(turn)),
             lambda d: emu.kmx_quantize(d, None, capi.PREC_FP32, 1, 70, 64, x.data_ptr(), 64, codes.data_ptr(), 64, sc.data_ptr())]
    try:
        for current in (0, 2):
            emu.emu_make_current(current)
            for device in (1, 0, 2):
                for call in calls:
                    ok(emu, call(device))
                    assert (emu.emu_launched_on(), emu.emu_current_device()) == (device, current)
            for call in calls:
                assert call(3) == capi.KMX_ERR_INVALID_ARG and emu.emu_current_device() == current
    finally:
        emu.emu_make_current(0)
    ref.check_y(y, ref.norm(x)[1])
    ref.check_linear(out, *ref.linear(ref.values(a, sa), ref.values(a, sa)), 64)
    assert torch.equal(codes, rounded_quotients(x)) and torch.equal(rot.reshape(70, 64), x)
