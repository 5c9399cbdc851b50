"""-m gpu: katago_amd.ops on the device against plain formulas in 64 bits (tests/ops_ref.py, with its tolerances): sizes around every kernel's borders, types,
strides, masks, spoilt values, long offsets, streams and graphs, refusals, and the operators in a row as a transformer block uses them."""
import gc
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import ops_ref as ref
from katago_amd import capi, ops
from katago_amd.capi import KatamxError

pytestmark = pytest.mark.gpu
REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(autouse=True)
def _no_grad():
    with torch.no_grad():
        yield


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(*shape, g, t=torch.float32, spread=1.0):
    return (torch.randn(*shape, device="cuda", generator=g) * spread).to(t)


def uneven(rows, c, t, g, spread=1.0, pad=3, lead=1):
    """rows x c whose rows start at element (not vector) alignment"""
    buf = randn(lead + rows * (c + pad), g=g, t=t, spread=spread)
    return buf[lead:].reshape(rows, c + pad)[:, :c]


# ---- norm -----------------------------------------------------------------------------------------------------------

# around the row kernel's shapes for few rows: 8 x 16 lanes; 64 lanes x 1, 2; 256, 512 and 1024 x 1; 1024 x 4; longer rows
SIZES = [1, 7, 8, 96, 127, 129, 256, 384, 512, 513, 1000, 1025, 2048, 2049, 4096, 4097, 8192, 8200, 32768, 32769, 70000]


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("c", SIZES)
def test_rms_norm_sizes(c, dtype):
    g, t = gen(c), ref.TYPES[dtype]
    for rows in (1, 37):
        x, r = uneven(rows, c, t, g, 3.0), uneven(rows, c, t, g, 1.0, pad=0)
        w, b = 1 + 0.3 * randn(c, g=g), 0.2 * randn(c, g=g) if c % 2 else None
        mask = (torch.arange(rows, device="cuda") % 3 != 1).float() if c % 3 else None
        for scales in (None, "row", "mx") if c % 32 == 0 else (None, "row"):
            n = ops.rms_norm(x, w, 1e-5, beta=b, residual=r, mask=mask, scales=scales, want_y=True)
            want_sum, want = ref.norm(x, w, 1e-5, b, r, mask)
            assert torch.equal(n.sum, want_sum)
            ref.check_y(n.y, want, b)
            if scales:
                ref.check_codes(n.codes, n.scales, want, ref.norm_slack(want, b))
            else:
                assert n.codes is None and n.scales is None
        n = ops.rms_norm(x)
        assert n.sum is None
        ref.check_y(n.y, ref.norm(x)[1])


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("rows,c", [(4097, 160), (4099, 384), (4100, 500), (1025, 1536), (1030, 2047), (513, 4096), (520, 3001), (257, 8192), (263, 5005)])
def test_rms_norm_of_more_rows_than_lanes(rows, c, dtype):
    """Rows of these lengths go on fewer lanes once there are more than 2^18 lanes' worth of them"""
    g, t = gen(c), ref.TYPES[dtype]
    x, r, w = uneven(rows, c, t, g, 3.0), uneven(rows, c, t, g, 1.0, pad=0), 1 + 0.3 * randn(c, g=g)
    mask = (torch.arange(rows, device="cuda") % 5 != 1).float()
    for scales in ("row", "mx") if c % 32 == 0 else ("row",):
        n = ops.rms_norm(x, w, residual=r, mask=mask, scales=scales, want_y=True)
        want_sum, want = ref.norm(x, w, 1e-6, None, r, mask)
        assert torch.equal(n.sum, want_sum)
        ref.check_y(n.y, want, None)
        ref.check_codes(n.codes, n.scales, want, ref.norm_slack(want, None))


def test_rms_norm_leading_dimensions_and_broadcasts():
    g = gen(1)
    x = randn(3, 5, 2, 64, g=g, t=torch.float16)
    n = ops.rms_norm(x[1], scales="mx")  # [5, 2, 64]
    want = ref.norm(x[1].reshape(-1, 64))[1]
    ref.check_codes(n.codes.reshape(-1, 64), n.scales.reshape(10, 2), want, ref.norm_slack(want))
    assert n.codes.shape == (5, 2, 64) and n.scales.shape == (5, 2, 2) and n.y is None


def test_rms_norm_collapsed_rows():
    g = gen(2)
    x = randn(3, 5, 2, 64, g=g, t=torch.bfloat16)
    n = ops.rms_norm(x, residual=x, scales="row", want_y=True)
    assert n.sum.shape == x.shape and n.scales.shape == (3, 5, 2)
    flat = x.reshape(-1, 64)
    want_sum, want = ref.norm(flat, residual=flat)
    assert torch.equal(n.sum.reshape(-1, 64), want_sum)
    ref.check_y(n.y.reshape(-1, 64), want)
    half = x[..., :32]  # rows of a wider matrix
    ref.check_y(ops.rms_norm(half).y.reshape(-1, 32), ref.norm(half.reshape(-1, 32))[1])
    one = randn(1, 64, g=g, t=torch.bfloat16).expand(7, 64)  # the same row seven times
    ref.check_y(ops.rms_norm(flat[:7], residual=one).y, ref.norm(flat[:7], residual=one)[1])
    with pytest.raises(KatamxError):
        ops.rms_norm(x[:, 1:4])


@pytest.mark.parametrize("c", [96, 100, 40000])
def test_rms_norm_in_place(c):
    g = gen(c)
    x, r = randn(19, c, g=g, t=torch.float16), randn(19, c, g=g, t=torch.float16)
    want_sum, want = ref.norm(x, residual=r)
    n = ops.rms_norm(x, residual=r, sum_out=r, y_out=x, scales="row")
    assert n.sum is r and n.y is x and torch.equal(r, want_sum)
    ref.check_y(x, want)
    ref.check_codes(n.codes, n.scales, want, ref.norm_slack(want))


def test_rows_beyond_the_last_stay_as_they_were():
    g = gen(3)
    x = randn(5, 64, g=g, t=torch.float16)
    out, total = (torch.full((9, 64), 7.0, device="cuda", dtype=torch.float16) for _ in range(2))
    ops.rms_norm(x, residual=x, y_out=out[2:7], sum_out=total[2:7])
    for t in (out, total):
        assert bool((t[:2] == 7).all()) and bool((t[7:] == 7).all()) and not bool((t[2:7] == 7).all(dim=1).any())


@pytest.mark.parametrize("c,rows", [(2, 134217712 + 4099), (8200, 2097151 + 40)])
def test_more_rows_than_a_launch_counts_threads(c, rows):
    """256 threads for 16 rows, 1024 for one: the second launch's rows are those that a call on them alone gives"""
    g = gen(41)
    x = torch.empty(rows, c, device="cuda", dtype=torch.float16)
    for at in (0, rows - 5000):
        x[at:at + 5000].normal_(generator=g)
    mask = torch.ones(rows, device="cuda")
    mask[-7] = 0
    n = ops.rms_norm(x, mask=mask, scales="row", want_y=True)
    for part in (slice(0, 5000), slice(rows - 5000, rows)):
        want = ops.rms_norm(x[part], mask=mask[part], scales="row", want_y=True)
        assert torch.equal(n.y[part], want.y) and torch.equal(n.scales[part], want.scales)
        assert torch.equal(n.codes[part].view(torch.uint8), want.codes.view(torch.uint8))
    assert bool((n.y[-7] == 0).all()) and bool((n.y[-8] != 0).any())


def test_masked_and_spoilt_rows():
    x = torch.randn(6, 64, device="cuda").bfloat16()
    x[1], x[2, 5], x[4, 40] = float("nan"), float("inf"), float("nan")
    mask = torch.tensor([1.0, 0.0, 1.0, 1.0, 1.0, 0.0], device="cuda")
    for scales in ("row", "mx"):
        n = ops.rms_norm(x, mask=mask, scales=scales, want_y=True)
        s = n.scales.float().reshape(6, -1)
        assert bool((n.y[[1, 5]] == 0).all()) and bool((n.codes[[1, 5]].float() == 0).all()) and bool((s[[1, 5]] == 1).all())
        assert bool(torch.isnan(n.y[2, 5])) and bool((n.y[2, :5] == 0).all())  # an infinite row: x / inf
        assert bool(torch.isnan(s[2, 0])) and bool(torch.isnan(s[4]).all()) and bool((n.codes[4].float() == 0).all())
        good = torch.tensor([0, 3], device="cuda")
        want = ref.norm(x[good])[1]
        ref.check_y(n.y[good], want)
        ref.check_codes(n.codes[good], n.scales[good], want, ref.norm_slack(want))
    assert bool((ops.rms_norm(x, mask=torch.zeros(6, device="cuda")).y == 0).all())
    zero = ops.rms_norm(torch.zeros(3, 64, device="cuda"), scales="row")
    assert bool((zero.codes.float() == 0).all()) and bool((zero.scales == 1).all())


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("scales", ["row", "mx"])
def test_quantize(dtype, scales):
    g, t = gen(4), ref.TYPES[dtype]
    for rows, c in ((1, 32), (50, 96), (3, 1536), (2, 33280)) + (((5, 77), (1, 1)) if scales == "row" else ()):
        x = uneven(rows, c, t, g, 5.0)
        codes, s = ops.quantize(x, scales)
        ref.check_codes(codes, s, x.double(), torch.zeros_like(x, dtype=torch.float64))


@pytest.mark.parametrize("scales", ["row", "mx"])
def test_quantize_borders(scales):
    top = [448.0, 449.0, 448.0 * 2 ** 20, 448.0 * 2.0 ** -60, 2.0 ** -130, 1e-44, 3.3e38, 1.0, 1.75, 1.7500001, 0.0]
    x = torch.stack([torch.linspace(-1, 1, 64, device="cuda", dtype=torch.float64) * v for v in top]).float()
    codes, s = ops.quantize(x, scales)
    ref.check_codes(codes, s, x.double(), torch.zeros_like(x, dtype=torch.float64))


def test_codes_do_not_depend_on_the_row_next_to_them():
    g = gen(5)
    x = randn(200, 384, g=g, t=torch.float16)
    all_, some = ops.rms_norm(x, scales="row", want_y=True), ops.rms_norm(x[57:60], scales="row", want_y=True)
    for a, b in ((all_.y, some.y), (all_.codes.view(torch.uint8), some.codes.view(torch.uint8)), (all_.scales, some.scales)):
        assert torch.equal(a[57:60], b)


# ---- the 8-bit product ----------------------------------------------------------------------------------------------

def eight(rows, k, scales, g, spread=1.0):
    return ops.quantize(randn(rows, k, g=g, spread=spread), scales)


@pytest.mark.parametrize("out", ["fp16", "bf16"])
@pytest.mark.parametrize("scales", ["row", "mx"])
@pytest.mark.parametrize("m,n,k", [(655400, 100, 288), (655360, 128, 384), (330001, 256, 128), (327000, 130, 256), (217100, 384, 352), (72500, 1152, 384), (71680, 1100, 32),
                                   (92416, 1152, 384), (10300, 8192, 256), (10240, 8065, 384), (10111, 8192, 96), (10305, 8192, 128), (72449, 1152, 256)])
def test_linear8_of_many_rows_and_short_k(m, n, k, scales, out):
    """The kernel that keeps its weights: whole tiles and partial ones, channels for one work-group to sixty-four, rows around the fewest that it takes"""
    g = gen(m + n)
    a, sa = eight(m, k, scales, g)
    w, sw = eight(n, k, scales, g)
    b = randn(n, g=g) if n % 3 else None
    buf = torch.full((m, n + 9), 7.0, device="cuda", dtype=ref.TYPES[out])
    y = ops.linear8(a, sa, w, sw, b, out=buf[:, 1:n + 1])
    for lo in range(0, m, 20000):
        part = slice(lo, min(m, lo + 20000))
        ref.check_linear(y[part], *ref.linear(ref.values(a[part], sa[part]), ref.values(w, sw), b), k)
    assert bool((buf[:, 0] == 7).all()) and bool((buf[:, n + 1:] == 7).all())


@pytest.mark.parametrize("out", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("scales", ["row", "mx"])
@pytest.mark.parametrize("m,n,k", [(1, 1, 32), (1, 4096, 4096), (2, 100, 96), (16, 1000, 512), (17, 64, 2048), (33, 33, 64), (361, 1152, 384), (64, 65, 128),
                                   (127, 129, 160), (130, 8, 1024), (500, 2000, 256), (2049, 2050, 288), (9000, 200, 96),
                                   (64, 100, 1024), (65, 70, 1040 - 16), (200, 3000, 1184), (1000, 4100, 1152), (1100, 5000, 1056), (5000, 4999, 512), (4100, 16400, 128)])
def test_linear8(m, n, k, scales, out):
    g = gen(m + n)
    (a, sa), (w, sw) = eight(m, k, scales, g, 2.0), eight(n, k, scales, g, 0.1)
    b = randn(n, g=g) if (m + n) % 2 else None
    y = ops.linear8(a, sa, w, sw, b, out_dtype=ref.TYPES[out])
    want, mag = ref.linear(ref.values(a, sa), ref.values(w, sw), b)
    ref.check_linear(y, want, mag, k)


def test_linear8_k_of_sixteens():
    g = gen(6)
    for k in (16, 48, 112, 144, 400):
        for m, n in ((3, 20), (300, 310)):
            (a, sa), (w, sw) = eight(m, k, "row", g), eight(n, k, "row", g)
            for t in ref.TYPES.values():
                ref.check_linear(ops.linear8(a, sa, w, sw, out_dtype=t), *ref.linear(ref.values(a, sa), ref.values(w, sw)), k)


@pytest.mark.parametrize("m", [3, 200])
def test_linear8_strides_and_outputs(m):
    """Codes and weights as columns of wider matrices whose other columns are NaN; the output inside a larger one"""
    g = gen(7)
    n, k = 75, 160
    (a, sa), (w, sw) = eight(m, k, "mx", g), eight(n, k, "mx", g)
    wide_a, wide_w = (torch.full((r, k + 64), 0x7f, dtype=torch.uint8, device="cuda") for r in (m, n))
    wide_a[:, 32:32 + k], wide_w[:, 16:16 + k] = a.view(torch.uint8), w.view(torch.uint8)
    for t in ref.TYPES.values():
        big = torch.full((m + 4, n + 11), 7.0, dtype=t, device="cuda")
        y = ops.linear8(wide_a.view(a.dtype)[:, 32:32 + k], sa, wide_w.view(w.dtype)[:, 16:16 + k], sw, out=big[2:2 + m, 3:3 + n])
        ref.check_linear(y, *ref.linear(ref.values(a, sa), ref.values(w, sw)), k)
        big[2:2 + m, 3:3 + n] = 7.0
        assert bool((big == 7).all())


@pytest.mark.parametrize("m", [2, 100])
def test_linear8_spoilt_rows_spoil_their_own(m):
    g = gen(8)
    n, k = 70, 256
    for scales in ("row", "mx"):
        x, w = randn(m, k, g=g), randn(n, k, g=g)
        x[1, 3], w[5, 200] = float("inf"), float("nan")
        (a, sa), (v, sv) = ops.quantize(x, scales), ops.quantize(w, scales)
        for t in ref.TYPES.values():
            y = ops.linear8(a, sa, v, sv, out_dtype=t).float()
            bad = torch.zeros(m, n, dtype=torch.bool, device="cuda")
            bad[1], bad[:, 5] = True, True
            assert torch.equal(torch.isnan(y), bad)


def test_linear8_scales_of_any_size():
    """e8m0 scales from 2^-60 to 2^60 beside one another; rows of zeros"""
    g = gen(9)
    x, w = randn(40, 128, g=g), randn(50, 128, g=g)
    x *= torch.exp2(torch.randint(-60, 61, (40, 4), device="cuda", generator=g).double()).float().repeat_interleave(32, dim=1)
    x[7] = 0
    (a, sa), (v, sv) = ops.quantize(x, "mx"), ops.quantize(w, "mx")
    want, mag = ref.linear(ref.values(a, sa), ref.values(v, sv))
    y = ops.linear8(a, sa, v, sv, out_dtype=torch.float32)
    ref.check_linear(y, want, mag, 128)
    assert bool((y[7] == 0).all())
    y = ops.linear8(a, sa, v, sv, out_dtype=torch.bfloat16)
    assert bool(((y.double() - want).abs() <= ref.half(torch.bfloat16) * want.abs() + 7 * 2.0 ** -13 * mag * 1.1).all())


# ---- rotary ---------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("batch,seq,hq,hk,dim,pairs,axes,fh,far", [
    (1, 1, 1, 1, 2, 1, 1, 1, 10), (8, 1, 32, 8, 128, 64, 1, 1, 1000000), (2, 361, 12, 6, 32, 16, 2, 6, 18), (3, 50, 9, 3, 24, 12, 1, 3, 3000000),
    (1, 77, 5, 5, 10, 3, 2, 1, 18), (2, 33, 8, 1, 192, 32, 1, 1, 131072), (1, 500, 16, 2, 21, 10, 1, 2, 100), (4, 19, 3, 3, 256, 128, 1, 1, 5000)])
def test_rotary(batch, seq, hq, hk, dim, pairs, axes, fh, far, layout, dtype):
    g, t = gen(dim * 10 + seq), ref.TYPES[dtype]
    q, k = randn(batch, seq, hq, dim, g=g, t=t), randn(batch, seq, hk, dim, g=g, t=t)
    pos = torch.randint(0, far + 1, (batch, seq, axes), device="cuda", generator=g, dtype=torch.int64 if far > 50000 else torch.int32)
    f = torch.rand(fh, axes, pairs, device="cuda", generator=g, dtype=torch.float64) * 2 - 1
    for magnitude, inverse in ((1.0, False), (1.3, True)):
        qo, ko = ops.rotary(q, k, pos, f, layout=layout, magnitude=magnitude, inverse=inverse)
        for x, y in ((q, qo), (k, ko)):
            flat = x.reshape(batch * seq, -1, dim)
            ref.check_rotary(y.reshape(flat.shape), *ref.rotary(flat, pos.reshape(-1, axes), f, layout == "half", magnitude, inverse), magnitude)
    qi, ki = q.clone(), k.clone()
    a, b = ops.rotary(qi, ki, pos, f, layout=layout, q_out=qi, k_out=ki)
    again = ops.rotary(q, k, pos, f, layout=layout)
    assert a is qi and b is ki and torch.equal(qi, again[0]) and torch.equal(ki, again[1])


def test_rotary_forms_of_its_arguments():
    g = gen(10)
    q, k = randn(6, 40, 4, 32, g=g, t=torch.float16), randn(6, 40, 2, 32, g=g, t=torch.float16)
    f = ops.rotary_frequencies(32)[0].cuda()
    seq_pos = torch.arange(40, device="cuda")
    full = ops.rotary(q, k, seq_pos.expand(6, 40), f.reshape(1, 1, 16))
    for pos in (seq_pos, seq_pos.int(), seq_pos.reshape(40, 1), seq_pos.expand(6, 40).contiguous(), torch.arange(80, device="cuda")[::2] // 2):
        got = ops.rotary(q, k, pos, f)
        assert torch.equal(got[0], full[0]) and torch.equal(got[1], full[1])
    one = ops.rotary(q[2], None, seq_pos, f)
    assert one[1] is None and torch.equal(one[0], full[0][2])
    heads_first = q.transpose(1, 2).contiguous().transpose(1, 2)  # [batch][heads][seq][dim] in memory
    out = torch.empty_like(heads_first)
    assert torch.equal(ops.rotary(heads_first, k, seq_pos, f, q_out=out)[0], full[0])
    x = randn(50, 4, 8, g=g)
    back = ops.rotary(*ops.rotary(x, x, seq_pos[:1].expand(50) + 7, f[:4]), seq_pos[:1].expand(50) + 7, f[:4], inverse=True)[0]
    assert float((back - x).abs().max()) < 40 * ref.U * float(x.abs().max())


def test_rotary_of_a_fused_projection():
    g = gen(11)
    n, S, hq, hk, d = 3, 361, 6, 3, 16
    row = (hq + 2 * hk) * d + 8
    buf = randn(n, S, row, g=g, t=torch.bfloat16)
    was = buf.clone()
    q, k = buf[..., :hq * d].unflatten(-1, (hq, d)), buf[..., hq * d:(hq + hk) * d].unflatten(-1, (hk, d))
    pos, f = ops.board_positions(19, 19).cuda(), ops.board_frequencies(d, 100.0).cuda()
    ops.rotary(q, k, pos, f, q_out=q, k_out=k)
    x = was[..., :(hq + hk) * d].reshape(n * S, hq + hk, d)
    ref.check_rotary(buf[..., :(hq + hk) * d].reshape(x.shape), *ref.rotary(x, pos.repeat(n, 1), f[None], False))
    assert torch.equal(buf[..., (hq + hk) * d:], was[..., (hq + hk) * d:])


def test_rotary_of_heads_before_tokens():
    """[batch, heads of q, k and v, seq, dim] in one buffer, q and k in place"""
    g = gen(42)
    n, S, hq, hk, d = 2, 50, 4, 2, 32
    buf = randn(n, hq + 2 * hk, S, d, g=g, t=torch.float16)
    was = buf.clone()
    q, k = buf[:, :hq].transpose(1, 2), buf[:, hq:hq + hk].transpose(1, 2)
    pos, f = torch.arange(S, device="cuda"), ops.rotary_frequencies(d)[0].cuda()
    ops.rotary(q, k, pos, f, q_out=q, k_out=k)
    x = was[:, :hq + hk].transpose(1, 2).reshape(n * S, hq + hk, d)
    ref.check_rotary(buf[:, :hq + hk].transpose(1, 2).reshape(x.shape), *ref.rotary(x, pos.repeat(n)[:, None], f[None, None], False))
    assert torch.equal(buf[:, hq + hk:], was[:, hq + hk:])


def test_rotary_inverse_is_the_gradient():
    """<R x, y> = <x, R^T y>, and R^T y against differences of <R x, y>, in fp32"""
    g = gen(12)
    x, y = randn(20, 3, 16, g=g), randn(20, 3, 16, g=g)
    pos, f = torch.randint(0, 1000, (20,), device="cuda", generator=g), ops.rotary_frequencies(12)[0].cuda()
    kw = dict(layout="half", magnitude=1.2)
    grad = ops.rotary(y, None, pos, f, inverse=True, **kw)[0].double()
    forward = lambda v: ops.rotary(v, None, pos, f, **kw)[0].double()  # noqa: E731
    # fp32 outputs: each of the 960 products is off by at most 12 U of its size
    assert abs(float((forward(x) * y).sum() - (x.double() * grad).sum())) <= 24 * ref.U * 1.2 * float((x.abs().double() * 2 * y.abs().max()).sum())
    for at in ((0, 0, 0), (7, 1, 5), (19, 2, 15), (3, 2, 11)):
        d = torch.zeros_like(x)
        d[at] = 0.5  # linear: a difference of any size is exact but for roundings
        slope = float(((forward(x + d) - forward(x - d)) * y).sum())
        assert abs(slope - float(grad[at])) <= 200 * ref.U * float(x.abs().max() * y.abs().max())


# ---- long offsets, streams, graphs ---------------------------------------------------------------------------------

def test_offsets_beyond_32_bits():
    g = gen(13)
    rows, stride = 1100, 1 << 22  # 4.6e9 elements from the first row to the last
    buf = torch.empty(rows * stride + 4096, dtype=torch.uint8, device="cuda")
    codes = torch.as_strided(buf.view(torch.float8_e4m3fn), (rows, 128), (stride, 1))
    a, sa = eight(rows, 128, "row", g)
    torch.as_strided(buf, (rows, 128), (stride, 1)).copy_(a.view(torch.uint8))
    w, sw = eight(96, 128, "row", g)
    assert torch.equal(ops.linear8(codes, sa, w, sw), ops.linear8(a, sa, w, sw))
    wide = torch.as_strided(buf.view(torch.float16), (rows // 2, 96), (stride, 1))
    y = ops.linear8(a[:rows // 2], sa[:rows // 2], w, sw, out=wide)
    assert torch.equal(y, ops.linear8(a[:rows // 2], sa[:rows // 2], w, sw))
    x = randn(rows // 2, 96, g=g, t=torch.float16)
    wide.copy_(x)
    assert torch.equal(ops.rms_norm(wide).y, ops.rms_norm(x).y)
    assert torch.equal(ops.rms_norm(x, y_out=wide).y, ops.rms_norm(x).y)
    wide.copy_(x)
    pos, f = torch.arange(rows // 2, device="cuda"), ops.rotary_frequencies(32)[0].cuda()
    heads = wide.unflatten(-1, (3, 32))
    want = ops.rotary(x.reshape(-1, 3, 32), None, pos, f)[0]
    assert torch.equal(ops.rotary(heads, None, pos, f, q_out=heads)[0], want)


def block(x, stream, w, qw, qs, bias, pos, f, hq, hk, d):
    """The front of an attention sublayer in 8 bits"""
    n = ops.rms_norm(x, w, residual=stream, scales="row")
    qkv = ops.linear8(n.codes, n.scales, qw, qs, bias, out_dtype=x.dtype)
    q, k = qkv[..., :hq * d].unflatten(-1, (hq, d)), qkv[..., hq * d:(hq + hk) * d].unflatten(-1, (hk, d))
    ops.rotary(q, k, pos, f, q_out=q, k_out=k)
    return n, qkv


def block_inputs(g, n=2, S=361, c=96, hq=6, hk=3, d=16, t=torch.float16):
    w = 1 + 0.2 * randn(c, g=g)
    m = randn((hq + 2 * hk) * d, c, g=g, spread=c ** -0.5)
    qw, qs = ops.quantize(m, "row")
    bias = 0.1 * randn(m.shape[0], g=g)
    f = torch.rand(hk, 2, d // 2, device="cuda", generator=g, dtype=torch.float64) * 1.4 - 0.7
    return dict(x=randn(n, S, c, g=g, t=t), stream=randn(n, S, c, g=g, t=t), w=w, qw=qw, qs=qs, bias=bias, pos=ops.board_positions(19, 19).cuda(), f=f,
                hq=hq, hk=hk, d=d), m


def test_calls_on_other_streams_and_threads():
    """The same calls on two streams at once, from two threads, each on data that its own stream has just made"""
    import threading

    inputs = [block_inputs(gen(20 + i))[0] for i in range(2)]
    torch.cuda.synchronize()
    want = [block(**i)[1].clone() for i in inputs]
    torch.cuda.synchronize()
    got = [None, None]

    def work(i):
        s = torch.cuda.Stream()
        with torch.no_grad(), torch.cuda.stream(s):
            for _ in range(20):
                mine = dict(inputs[i], x=inputs[i]["x"] * 1.0, stream=inputs[i]["stream"] * 1.0)
                got[i] = block(**mine)[1]
            s.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_captured_and_replayed():
    """Two graphs of the same operators alive at once, replayed with other inputs, the program's own eager work between"""
    graphs = []
    for i in range(2):
        a, _ = block_inputs(gen(30 + i))
        block(**a)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            n, qkv = block(**a)
        graphs.append((graph, a, n, qkv))
    for turn in range(4):
        for i, (graph, a, n, qkv) in enumerate(graphs):
            g = gen(100 * turn + i)
            a["x"].copy_(randn(*a["x"].shape, g=g, t=torch.float16))
            a["stream"].copy_(randn(*a["x"].shape, g=g, t=torch.float16))
        for graph, _, _, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, a, n, qkv in graphs:
            m, want = block(**a)
            assert torch.equal(qkv, want) and torch.equal(n.sum, m.sum) and torch.equal(n.scales, m.scales)


def test_the_current_device_and_stream_are_left_alone():
    before = torch.cuda.current_device(), torch.cuda.current_stream()
    ops.rms_norm(torch.ones(3, 32, device="cuda"))
    assert (torch.cuda.current_device(), torch.cuda.current_stream()) == before
    lib = capi.load_library()
    x = torch.ones(4, 32, device="cuda")
    codes, s = torch.empty(4, 32, dtype=torch.uint8, device="cuda"), torch.empty(4, device="cuda")
    call = lambda device: lib.kmx_quantize(device, None, capi.PREC_FP32, 1, 4, 32, x.data_ptr(), 32, codes.data_ptr(), 32, s.data_ptr())  # noqa: E731
    assert call(-1) == capi.KMX_ERR_INVALID_ARG and call(torch.cuda.device_count()) == capi.KMX_ERR_INVALID_ARG and call(0) == capi.KMX_OK
    torch.cuda.synchronize()


def test_the_first_call_of_a_process_may_be_captured():
    """Nothing has loaded or set up the kernels when their launches are recorded: a norm, a tile of 256 x 256, a rotation"""
    code = r"""
import sys, torch
sys.path.insert(0, %r)
from katago_amd import ops
with torch.no_grad():
    x, m = torch.randn(8192, 256, device="cuda").half(), torch.randn(1024, 256, device="cuda").half()
    pos, f = torch.arange(8192, device="cuda"), ops.rotary_frequencies(64)[0].cuda()
    def run():
        n = ops.rms_norm(x, scales="mx")
        y = ops.linear8(n.codes, n.scales, *ops.quantize(m, "mx"))
        return ops.rotary(y.unflatten(-1, (16, 64)), None, pos, f)[0]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for _ in range(3):
        x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, run())
print("FIRST_OK")
""" % REPO
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "FIRST_OK" in r.stdout, r.stdout[-1000:] + r.stderr[-3000:]


# ---- the operators in a row, and refusals ---------------------------------------------------------------------------

def test_an_attention_sublayer_in_8_bits():
    """norm + residual -> 8-bit projection -> rotary (a learned table on two axes) -> the framework's attention, on 19x19 and smaller boards, against the
    sublayer in 64 bits without 8-bit roundings. Both operands of the projection carry an e4m3 rounding: at most 2^-4 of each factor, uniform over half a step
    2^-4 / sqrt(3), in two factors and with independent signs sqrt(2) of that: 0.051 of the projection's norm."""
    g = gen(40)
    n, S, c, hq, hk, d = 3, 361, 96, 6, 3, 16
    a, m = block_inputs(g, n, S, c, hq, hk, d)
    mask = torch.zeros(n, 19, 19, device="cuda")
    for b, side in enumerate((19, 13, 9)):
        mask[b, :side, :side] = 1
    mask = mask.reshape(n, S)
    x, stream = a["x"] * mask[..., None].half(), a["stream"] * mask[..., None].half()
    nrm = ops.rms_norm(x, a["w"], residual=stream, mask=mask, scales="row")
    qkv = ops.linear8(nrm.codes, nrm.scales, a["qw"], a["qs"], a["bias"])
    raw = qkv.clone()
    q, k, v = qkv[..., :hq * d].unflatten(-1, (hq, d)), qkv[..., hq * d:(hq + hk) * d].unflatten(-1, (hk, d)), qkv[..., (hq + hk) * d:].unflatten(-1, (hk, d))
    ops.rotary(q, k, a["pos"], a["f"], q_out=q, k_out=k)
    lib = capi.load_library()
    host = [np.ascontiguousarray(t.float().cpu().numpy()) for t in (q, k, v, mask)]
    out = np.empty((n, S, hq * d), np.float32)
    P = capi._FP
    capi.check(lib.kmx_test_attention(n, 19, 19, capi.PREC_FP16, hq, hk, d, d, None, None, 1, *[h.ctypes.data_as(P) for h in host[:3]], host[3].ctypes.data_as(P),
                                      out.ctypes.data_as(P)), lib)
    # the projection
    _, y = ref.norm(x.reshape(-1, c), a["w"], 1e-6, None, stream.reshape(-1, c), mask.reshape(-1))
    exact = y @ m.double().t() + a["bias"].double()
    on = mask.reshape(-1) != 0
    assert float((raw.reshape(-1, exact.shape[1]).double() - exact)[on].norm() / exact[on].norm()) < 0.051
    # attention of the kernels' own q, k, v in 64 bits: one rounding of the probabilities and one of the output to fp16, and the attention kernel's own sums
    want = torch.zeros(n, S, hq, d, dtype=torch.float64, device="cuda")
    for b in range(n):
        keep = mask[b] != 0
        for h in range(hq):
            kk, vv = k[b, keep, h // 2].double(), v[b, keep, h // 2].double()
            want[b, keep, h] = torch.softmax(q[b, keep, h].double() @ kk.t() / d ** 0.5, dim=1) @ vv
    got = torch.from_numpy(out).cuda().reshape(n, S, hq, d).double()
    assert float((got - want).abs().max()) <= 3 * 2.0 ** -10 * max(1.0, float(want.abs().max()))
    assert bool((got[mask == 0] == 0).all())


def test_calls_keep_nothing():
    """Outputs are the caller's alone, also where a call is refused after some were allocated"""
    a = block_inputs(gen(43))[0]
    block(**a)
    torch.cuda.synchronize()
    gc.collect()  # (what earlier tests left in cycles)
    before = torch.cuda.memory_allocated(), [sys.getrefcount(a[k]) for k in ("x", "w", "qw", "f")]
    for _ in range(50):
        block(**a)
        with pytest.raises(KatamxError):
            ops.rms_norm(a["x"], eps=float("nan"))
    torch.cuda.synchronize()
    gc.collect()
    assert (torch.cuda.memory_allocated(), [sys.getrefcount(a[k]) for k in ("x", "w", "qw", "f")]) == before
    with pytest.raises(TypeError):
        ops.rms_norm(a["x"], eps="small")
    with pytest.raises(RuntimeError):
        ops.rms_norm(a["x"], want_y=torch.ones(2))  # (has no truth value)


def test_no_rows():
    e = torch.empty(0, 64, device="cuda", dtype=torch.float16)
    n = ops.rms_norm(e, residual=e, scales="mx", want_y=True)
    assert n.sum.shape == n.y.shape == n.codes.shape == (0, 64) and n.scales.shape == (0, 2)
    codes, s = ops.quantize(e)
    w, sw = ops.quantize(torch.ones(8, 64, device="cuda"))
    assert ops.linear8(codes, s, w, sw).shape == (0, 8)
    z = torch.empty(0, 2, 32, device="cuda", dtype=torch.float16)
    assert ops.rotary(z, z, torch.empty(0, device="cuda", dtype=torch.int32), torch.ones(16, device="cuda").double())[0].shape == z.shape


def test_refusals():
    x = torch.ones(8, 64, device="cuda", dtype=torch.float16)
    i32 = torch.int32
    codes, s = ops.quantize(x)
    mcodes, ms = ops.quantize(x, "mx")
    q, pos, f = torch.ones(8, 2, 32, device="cuda"), torch.zeros(8, device="cuda", dtype=i32), torch.ones(16, device="cuda").double()
    bad = [
        lambda: ops.rms_norm(torch._neg_view(x)), lambda: ops.rms_norm(x.double()), lambda: ops.rms_norm(x.t()), lambda: ops.rms_norm(x[:, ::2]), lambda: ops.rms_norm(x, torch.ones(63, device="cuda")),
        lambda: ops.rms_norm(x, torch.ones(64, device="cuda", dtype=torch.float16)), lambda: ops.rms_norm(x, torch.ones(64)), lambda: ops.rms_norm(x, residual=x[:4]),
        lambda: ops.rms_norm(x, residual=x.float()), lambda: ops.rms_norm(x, mask=torch.ones(7, device="cuda")), lambda: ops.rms_norm(x, scales="block"),
        lambda: ops.rms_norm(x[:, :40], scales="mx"), lambda: ops.rms_norm(x, sum_out=x), lambda: ops.rms_norm(x, y_out=x.float()), lambda: ops.rms_norm(x, y_out=x[:4]),
        lambda: ops.rms_norm(x[:4], y_out=x[1:5]), lambda: ops.rms_norm(x, want_y=False), lambda: ops.rms_norm(x, eps=-1.0), lambda: ops.rms_norm(x, scales="row", want_y=False, y_out=x),
        lambda: ops.rms_norm(x[:, :0]), lambda: ops.quantize(x, None), lambda: ops.quantize(x.to(torch.int8)),
        lambda: ops.linear8(codes.view(torch.uint8), s, codes, s), lambda: ops.linear8(codes, s, mcodes, ms), lambda: ops.linear8(codes, s[:7], codes, s),
        lambda: ops.linear8(codes[:, :32].contiguous(), s, codes, s), lambda: ops.linear8(codes, s, codes, s, out_dtype=torch.float64),
        lambda: ops.linear8(codes, s, codes, s, torch.ones(7, device="cuda")), lambda: ops.linear8(codes, s.cpu(), codes, s),
        lambda: ops.linear8(codes[:, 8:56], s, codes[:, 8:56], s), lambda: ops.linear8(codes, s, codes, s, out=torch.ones(8, 9, device="cuda")),
        lambda: ops.linear8(*(ops.quantize(x[:, :24])), *(ops.quantize(x[:, :24]))),
        lambda: ops.rotary(q, None, pos[:7], f), lambda: ops.rotary(q, None, pos.float(), f), lambda: ops.rotary(q, None, pos, f.float()),
        lambda: ops.rotary(q, None, pos, torch.ones(17, device="cuda").double()), lambda: ops.rotary(q, None, pos, torch.ones(2, 16, device="cuda").double()),
        lambda: ops.rotary(q, None, pos, torch.ones(3, 1, 16, device="cuda").double()), lambda: ops.rotary(q, q[:4].clone(), pos, f),
        lambda: ops.rotary(q, q.half(), pos, f), lambda: ops.rotary(q, None, pos, f, layout="split"), lambda: ops.rotary(q, None, pos, f, k_out=q),
        lambda: ops.rotary(q, None, pos, f, q_out=q.half()), lambda: ops.rotary(q, None, pos, f, magnitude=float("nan")), lambda: ops.rotary(x, None, pos, f),
        lambda: ops.rotary(q[:4], None, pos[:4], f, q_out=q[1:5]), lambda: ops.rotary(q[:, :0], None, pos, f)]
    for i, call in enumerate(bad):
        with pytest.raises(KatamxError) as e:
            call()
        assert e.value.code == capi.KMX_ERR_INVALID_ARG, i
    with torch.enable_grad():
        y = torch.ones(4, 32, device="cuda", requires_grad=True)
        with pytest.raises(KatamxError):
            ops.rms_norm(y)
        with torch.no_grad():
            ops.rms_norm(y)
