"""-m gpu: katago_amd.ops at the ends of what it takes - scales, values, lengths and tensors far from the usual ones - against plain formulas in 64 bits."""
import ctypes
import subprocess
import sys

import pytest
import torch
from torch.autograd import forward_ad

import ops_ref as ref
from conftest import REPO
from katago_amd import capi, ops
from katago_amd.capi import KatamxError
from test_gpu_ops import eight, gen
from test_ops_limits_emulated import check_block_scales, check_linear_any, check_small_results, rounded_quotients, rows_of_any_size, small_sine_angles, spread_scales

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_grad():
    with torch.no_grad():
        yield


@pytest.mark.parametrize("out", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("m,n,k", [(3, 40, 512), (30, 100, 4096), (64, 64, 272), (70, 64, 512), (361, 1152, 384), (200, 3000, 1184), (1000, 4100, 1152),
                                   (5000, 4999, 512), (72500, 1152, 384), (71681, 1100, 128)])
def test_linear8_row_scales_of_any_size(m, n, k, out):
    """Scales from 2^-120 to 2^120 on both sides: a large one must not carry a sum out of fp32 that the other brings back, in any of the kernels"""
    g, c = gen(m + n), torch.Generator().manual_seed(m + n)
    (a, _), (w, _) = eight(m, k, "row", g), eight(n, k, "row", g)
    for sa, sw in ((spread_scales(m, c), spread_scales(n, c)), (torch.rand(m, generator=c) * 1e35, torch.rand(n, generator=c) * 1e-37)):
        sa, sw = sa.cuda(), sw.cuda()
        y = ops.linear8(a, sa, w, sw, out_dtype=ref.TYPES[out])
        for lo in range(0, m, 10000):
            part = slice(lo, min(m, lo + 10000))
            check_linear_any(y[part], *ref.linear(ref.values(a[part], sa[part]), ref.values(w, sw)), k)


def test_linear8_scales_of_nothing():
    """Scales of zero, infinity and NaN give what the formula gives, beside rows that are as they always are"""
    g = gen(2)
    for m in (5, 70):
        (a, sa), (w, sw) = eight(m, 256, "row", g), eight(65, 256, "row", g)
        want = ops.linear8(a, sa, w, sw, out_dtype=torch.float32)
        sb = sa.clone()
        sb[1], sb[2], sb[3] = 0.0, float("inf"), float("nan")
        y = ops.linear8(a, sb, w, sw, out_dtype=torch.float32)
        assert bool((y[1] == 0).all()) and bool(torch.isinf(y[2]).all()) and bool(torch.isnan(y[3]).all())
        assert bool(((y - want)[[0, 4]].abs() <= 2 * ref.U * want[[0, 4]].abs()).all())


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("c", [50, 96, 384, 1000, 2000, 4096, 8000, 20000, 33000])
def test_rms_norm_of_small_and_large_rows(c, dtype):
    """Without eps: the squares of values below 1e-19 or beyond 1.8e19 leave fp32, their rows' norms are ordinary numbers; on lanes for few rows and for many"""
    x = rows_of_any_size(c, ref.TYPES[dtype], torch.Generator().manual_seed(c)).cuda()
    for again in (1, 300):
        many = x.repeat(again, 1)
        n = ops.rms_norm(many, eps=0.0, scales="row", want_y=True)
        some = many.abs().amax(1) > 0
        want = ref.norm(many[some], eps=0.0)[1]
        ref.check_y(n.y[some], want)
        ref.check_codes(n.codes[some], n.scales[some], want, ref.norm_slack(want))
        assert bool(torch.isnan(n.y[~some]).all()) and bool(torch.isnan(n.scales[~some]).all())
        for row in range(0, x.shape[0], 5):
            alone = ops.rms_norm(many[row:row + 1], eps=0.0).y[0]
            if again == 1:
                assert torch.equal(alone.nan_to_num(7.0), n.y[row].nan_to_num(7.0))


@pytest.mark.parametrize("c", [1 << 22, (1 << 26) + 3])
def test_rms_norm_of_a_very_long_row(c):
    """One value in all channels: thousands of squares a lane, whose sum must not collect a rounding each"""
    x = torch.full((1, c), 1.1, device="cuda")
    ref.check_y(ops.rms_norm(x, eps=0.0).y, ref.norm(x, eps=0.0)[1])


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
def test_codes_are_rounded_quotients(dtype):
    """16-bit values lie on the border of two codes often enough that a product with the rounded reciprocal, or a quotient by the rounded scale, is told from
    the formula's quotient; what a norm codes is its fp32 result"""
    g, t = gen(3), ref.TYPES[dtype]
    for rows, c in ((16383, 1536), (361, 384), (5, 8190), (3, 70000)):
        x = (torch.randn(rows, c, device="cuda", generator=g) * 3).to(t)
        codes, s = ops.quantize(x)
        assert torch.equal(s, (x.abs().amax(1).double() / 448).float())  # (torch multiplies a device tensor with 1 / 448)
        assert torch.equal(codes.view(torch.uint8), rounded_quotients(x))
        if dtype == "fp32":
            n = ops.rms_norm(x, scales="row", want_y=True)
            assert torch.equal(n.codes.view(torch.uint8), rounded_quotients(n.y))


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_of_small_sines(layout):
    """A sine next to 0 or to pi, a cosine next to pi / 2, in fp32: right relative to itself"""
    angle = small_sine_angles().cuda()
    n = angle.shape[0]
    for pairs in (1, 4, 8):  # pieces of one pair and of four
        q = torch.eye(2, device="cuda").repeat(n, 1).reshape(1, 2 * n, 2, 1).expand(1, 2 * n, 2, pairs)
        q = (q if layout == "half" else q.transpose(2, 3)).reshape(1, 2 * n, 2 * pairs).contiguous()
        f = angle.reshape(n, 1, 1).expand(n, 1, pairs).contiguous()
        for magnitude in (1.0, 1.375):
            y = ops.rotary(q, None, torch.ones(1, device="cuda", dtype=torch.int32), f, layout=layout, magnitude=magnitude)[0]
            y = y.reshape(n, 2, 2, pairs) if layout == "half" else y.reshape(n, 2, pairs, 2).transpose(2, 3)
            for p in range(pairs):
                check_small_results(y[..., p], angle, magnitude)


def test_forward_mode_tangents_are_refused():
    x, f, pos = torch.ones(4, 2, 32, device="cuda"), torch.ones(16, device="cuda").double(), torch.zeros(4, device="cuda", dtype=torch.int32)
    w, (codes, s) = torch.ones(32, device="cuda"), ops.quantize(torch.ones(4, 32, device="cuda"))
    ones = torch.ones(4, device="cuda")
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))
        for call in (lambda: ops.rms_norm(dual(x)), lambda: ops.rms_norm(x, dual(w)), lambda: ops.rms_norm(x, residual=dual(x)), lambda: ops.rms_norm(x, y_out=dual(x)),
                     lambda: ops.quantize(dual(x)), lambda: ops.linear8(codes, dual(s), codes, s), lambda: ops.linear8(codes, s, codes, s, dual(ones)),
                     lambda: ops.rotary(dual(x), None, pos, f), lambda: ops.rotary(x, dual(x), pos, f), lambda: ops.rotary(x, None, pos, dual(f))):
            with pytest.raises(KatamxError, match="tangent"):
                call()
            with torch.enable_grad(), pytest.raises(KatamxError, match="tangent"):
                call()
        primal = forward_ad.unpack_dual(dual(x)).primal
        ops.rms_norm(primal)


def test_written_tensors_have_a_new_version():
    """A tensor that autograd keeps for a backward pass and an operator writes over is noticed there, as with torch's own in-place operations"""
    x, pos, f = torch.ones(4, 2, 32, device="cuda"), torch.zeros(4, device="cuda", dtype=torch.int32), torch.ones(16, device="cuda").double()
    codes, s = ops.quantize(torch.ones(4, 32, device="cuda"))
    for write in (lambda t: ops.rms_norm(x, y_out=t), lambda t: ops.rms_norm(x, residual=x, sum_out=t), lambda t: ops.rms_norm(t, y_out=t),
                  lambda t: ops.rotary(x, None, pos, f, q_out=t), lambda t: ops.rotary(x, x, pos, f, k_out=t), lambda t: ops.rotary(t, None, pos, f, q_out=t),
                  lambda t: ops.linear8(codes, s, codes, s, out=t.reshape(-1)[:16].reshape(4, 4))):
        with torch.enable_grad():
            leaf, kept = torch.ones(4, 2, 32, device="cuda", requires_grad=True), torch.ones(4, 2, 32, device="cuda")
            loss = (leaf * kept).sum()
        before = kept._version
        write(kept)
        assert kept._version > before
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    before = x._version, codes._version
    ops.rms_norm(x, residual=x, scales="row")
    ops.rotary(x, x, pos, f)
    assert (x._version, codes._version) == before  # what is only read
    with pytest.raises(KatamxError):
        ops.rms_norm(x, y_out=x[:2])
    assert x._version == before[0]  # a refused call writes nothing
    with torch.inference_mode():
        t = torch.ones(4, 32, device="cuda")
        ops.rms_norm(t, y_out=t)
    ops.rms_norm(t, y_out=t)  # (a tensor without a version, outside the mode it was made in)


def test_an_error_of_an_earlier_call_is_left_where_it_is():
    """The program's own failed HIP call, whose error it has not fetched yet, is not an operator's, and is still there afterwards"""
    with open("/proc/self/maps") as f:
        hip = ctypes.CDLL(next(line.split()[-1] for line in f if "libamdhip64" in line))
    x = torch.randn(4, 64, device="cuda")
    (codes, s), (wide, ws) = ops.quantize(x), ops.quantize(torch.randn(100, 64, device="cuda"))
    pos, f = torch.zeros(4, device="cuda", dtype=torch.int32), torch.ones(16, device="cuda").double()
    y, q, out, codes_out = torch.empty_like(x), torch.empty(4, 2, 32, device="cuda"), torch.empty(4, 4, device="cuda"), torch.empty(100, 4, device="cuda")
    lib, stream = capi.load_library(), torch.cuda.current_stream().cuda_stream
    calls = [lambda: ops.rms_norm(x, y_out=y), lambda: ops.linear8(codes, s, codes, s, out=out), lambda: ops.linear8(wide, ws, codes, s, out=codes_out),
             lambda: ops.rotary(x.reshape(4, 2, 32), None, pos, f, q_out=q),
             lambda: lib.kmx_quantize(0, ctypes.c_void_p(stream), capi.PREC_FP32, 1, 4, 64, x.data_ptr(), 64, codes.data_ptr(), 64, s.data_ptr()) and pytest.fail()]
    for call in calls:
        call()
        torch.cuda.synchronize()
        try:
            left = hip.hipSetDevice(9999)
            assert left != 0
            call()
            still = hip.hipPeekAtLastError()
        finally:
            hip.hipGetLastError()
        assert still == left
    torch.cuda.synchronize()


@pytest.mark.parametrize("m,n,k", [(3, 40, 512), (30, 100, 4096), (64, 64, 288), (70, 64, 512), (361, 1152, 384), (1000, 4100, 1152), (5000, 4999, 512)])
def test_linear8_block_scales_at_their_ends(m, n, k):
    def run(a, sa, w, sw, out):
        return ops.linear8(a.cuda(), sa.cuda(), w.cuda(), sw.cuda(), out_dtype=ref.TYPES[out]).cpu()
    check_block_scales(run, m, n, k, torch.Generator().manual_seed(m + k))


@pytest.mark.parametrize("out", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("scales", ["row", "mx"])
@pytest.mark.parametrize("m,n,k", [(1000, 3900, 1152), (700, 3300, 1056), (5000, 4999, 1152), (4096, 4096, 1664), (4000, 4090, 1184), (1, 4096, 11008), (7, 70, 8224), (30, 100, 11008),
                                   (64, 130, 11008), (300, 2000, 11008), (1200, 1300, 8224)])
def test_linear8_of_long_k(m, n, k, scales, out):
    """Tiles of 128 x 128 with four stages, tiles of 256 x 256 whose k has steps between its first and its last ones, k of several rounds of the kernel for
    few rows"""
    g = gen(m + n)
    (a, sa), (w, sw) = eight(m, k, scales, g, 2.0), eight(n, k, scales, g, 0.1)
    b = torch.randn(n, device="cuda", generator=g) if (m + n) % 2 else None
    buf = torch.full((m, n + 9), 7.0, device="cuda", dtype=ref.TYPES[out])
    y = ops.linear8(a, sa, w, sw, b, out=buf[:, 1:n + 1])
    ref.check_linear(y, *ref.linear(ref.values(a, sa), ref.values(w, sw), b), k)
    assert bool((buf[:, 0] == 7).all()) and bool((buf[:, n + 1:] == 7).all())


def test_the_first_call_of_a_process_may_be_a_captured_large_tile():
    """Tiles of 256 x 256 (8192 x 4096 x 256) and of 128 x 128 (1100 rows), whose launches opt in to their LDS, with nothing loaded before they are recorded"""
    code = r"""
import sys, torch
sys.path.insert(0, %r)
from katago_amd import ops
with torch.no_grad():
    x, m, t = torch.randn(8192, 256, device="cuda").half(), torch.randn(4096, 256, device="cuda").half(), torch.randn(1100, 256, device="cuda").half()
    def run():
        (a, sa), (w, sw) = ops.quantize(x, "mx"), ops.quantize(m, "mx")
        return ops.linear8(a, sa, w, sw), ops.linear8(*ops.quantize(t, "mx"), w, sw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for _ in range(3):
        x.normal_()
        t.normal_()
        graph.replay()
        torch.cuda.synchronize()
        want = run()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        far = (got[0].double() - x.double() @ m.double().t()).norm() / got[0].double().norm()
        assert float(far) < 0.051  # an e4m3 rounding in each factor
print("FIRST_OK")
""" % REPO
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "FIRST_OK" in r.stdout, r.stdout[-1000:] + r.stderr[-3000:]


def test_rotary_of_more_threads_than_a_launch_counts():
    """700 times the same million tokens, a thread for each of their three pairs: more than 2^31 threads, in two launches"""
    g = gen(5)
    S, B = 1 << 20, 700
    x = torch.randn(1, S, 1, 6, device="cuda", generator=g).half()
    pos, f = torch.randint(0, 1000, (S,), device="cuda", generator=g), torch.rand(3, device="cuda", generator=g, dtype=torch.float64)
    out = torch.full((B + 1, S, 1, 6), 7.0, device="cuda", dtype=torch.float16)
    ops.rotary(x.expand(B, S, 1, 6), None, pos, f, q_out=out[:B])
    ref.check_rotary(out[0], *ref.rotary(x[0], pos[:, None], f[None, None], False))
    for b in range(1, B):
        assert torch.equal(out[b], out[0]), b
    assert bool((out[B] == 7).all())
