"""The kernels behind include/katamx_ops.h, compiled for x86 and executed on the CPU through their own C entry points (tests/fakehip/emulate_ops.cpp),
against plain formulas in 64 bits: indexing, tails, masks, strides, the layouts of codes and scales; outputs lie in larger buffers whose other bytes must
stay as they were. What the hardware adds is tests/test_gpu_ops.py's part."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch

import ops_ref as ref
from conftest import REPO
from katago_amd import capi

PREC = {"fp16": capi.PREC_FP16, "bf16": capi.PREC_BF16, "fp32": capi.PREC_FP32}


@pytest.fixture(scope="module")
def emu(tmp_path_factory):
    so = os.path.join(str(tmp_path_factory.mktemp("emuops")), "libemuops.so")
    cmd = ["/opt/rocm/lib/llvm/bin/clang++", "-x", "c++", "-std=c++20", "-O2", "-Wno-psabi", "-fPIC", "-shared", "-pthread",
           "-I" + os.path.join(REPO, "tests", "fakehip", "emul"), "-o", so, os.path.join(REPO, "tests", "fakehip", "emulate_ops.cpp")]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    lib = ctypes.CDLL(so)
    capi.bind_ops(lib)
    lib.kmx_last_error.restype = ctypes.c_char_p
    return lib


def ok(emu, rc):
    assert rc == capi.KMX_OK, emu.kmx_last_error()


class Guarded:
    """rows x width elements at `stride` inside a buffer of a known pattern, `lead` elements in front of them"""

    def __init__(self, rows, width, stride, dtype, lead=3):
        self.buf = torch.full((lead + rows * stride + 64,), 7, dtype=torch.uint8).to(dtype) if dtype != torch.float8_e4m3fn else \
            torch.full((lead + rows * stride + 64,), 0x55, dtype=torch.uint8).view(dtype)
        self.before = self.buf.clone()
        self.rows, self.width, self.stride, self.lead = rows, width, stride, lead
        self.ptr = self.buf.data_ptr() + lead * self.buf.element_size()

    def get(self):
        return self.buf[self.lead:self.lead + self.rows * self.stride].reshape(self.rows, self.stride)[:, :self.width].clone()

    def rest_untouched(self):
        raw = {1: torch.uint8, 2: torch.int16, 4: torch.int32}[self.buf.element_size()]
        now, was = self.buf.view(raw).clone(), self.before.view(raw).clone()
        for t in (now, was):
            t[self.lead:self.lead + self.rows * self.stride].reshape(self.rows, self.stride)[:, :self.width] = 0
        assert torch.equal(now, was)


def strided(rows, c, stride, dtype, gen, spread=1.0):
    """A view of a strided buffer that starts in the middle of it"""
    buf = (torch.randn(rows * stride + 5, generator=gen) * spread).to(dtype)
    return buf[5:].reshape(rows, stride)[:, :c]


# the row kernel's shapes for few rows (16 lanes, 64 x 1, 2 rounds, 256, 512 and 1024 x 1, 1024 x 4; the long one), tails of a piece, one channel, one row
@pytest.mark.parametrize("rows,c,dtype,scales,residual,masked,beta", [
    (1, 1, "fp32", "row", False, False, False), (33, 96, "fp16", "mx", True, True, False), (17, 130, "bf16", "row", True, False, True),
    (5, 384, "fp16", "row", True, True, True), (3, 511, "fp32", None, False, True, False), (6, 1024, "bf16", "mx", False, False, False),
    (5, 2047, "fp16", "row", True, False, False), (2, 4096, "bf16", "mx", True, False, False), (2, 8191, "fp32", "row", True, False, False),
    (1, 8224, "bf16", "mx", True, True, False), (1, 32800, "fp16", "row", True, False, True), (2, 33024, "bf16", "mx", False, False, False)])
def test_rms_norm(emu, rows, c, dtype, scales, residual, masked, beta):
    g = torch.Generator().manual_seed(c)
    t = ref.TYPES[dtype]
    x, r = strided(rows, c, c + 3, t, g, 3.0), strided(rows, c, c + 1, t, g) if residual else None
    w, b = 1 + 0.3 * torch.randn(c, generator=g), 0.2 * torch.randn(c, generator=g) if beta else None
    mask = (torch.arange(rows) % 3 != 1).float() if masked else None
    total, y = Guarded(rows, c, c + 7, t), Guarded(rows, c, c, t)
    codes = Guarded(rows, c, c + 2, torch.float8_e4m3fn)
    sc = torch.full((rows,), 9.0) if scales != "mx" else torch.full((rows, c // 32), 9, dtype=torch.uint8)
    a = capi.RmsNormArgs(type=PREC[dtype], scale_kind={None: 0, "row": 1, "mx": 2}[scales], rows=rows, channels=c, epsilon=1e-6, x=x.data_ptr(),
                         weight=w.data_ptr(), beta=b.data_ptr() if beta else None, mask=mask.data_ptr() if masked else None, y=y.ptr,
                         x_stride=c + 3, y_stride=c)
    if residual:
        a.residual, a.residual_stride, a.sum, a.sum_stride = r.data_ptr(), c + 1, total.ptr, c + 7
    if scales:
        a.codes, a.codes_stride, a.scales = codes.ptr, c + 2, sc.data_ptr()
    ok(emu, emu.kmx_rmsnorm(0, None, ctypes.byref(a)))
    want_sum, want = ref.norm(x, w, 1e-6, b, r, mask)
    if residual:
        assert torch.equal(total.get(), want_sum)
    total.rest_untouched()
    ref.check_y(y.get(), want, b)
    y.rest_untouched()
    codes.rest_untouched()
    if scales:
        sc = sc if scales == "row" else sc.view(torch.float8_e8m0fnu)
        ref.check_codes(codes.get(), sc, want, ref.norm_slack(want, b))
        if masked:
            off = mask == 0
            assert bool((codes.get().view(torch.uint8)[off] & 0x7f == 0).all()) and bool((sc.float().reshape(rows, -1)[off] == 1).all())


@pytest.mark.parametrize("scales", ["row", "mx"])
def test_quantize_borders(emu, scales):
    """Zeros, one value, exact powers of two, the border 448 * 2^k and its neighbours, subnormals, infinities and NaN"""
    c = 64
    rows = [torch.zeros(c), torch.full((c,), -0.0), torch.full((c,), 448.0), torch.full((c,), 449.0), torch.full((c,), 448.0 * 2 ** 20),
            torch.full((c,), 2.0 ** -130), torch.full((c,), 1e-44), torch.full((c,), 3e38), torch.arange(c) - 31.5, torch.ones(c), torch.ones(c)]
    rows[9] = rows[9].clone()
    rows[9][40] = float("inf")
    rows[10] = rows[10].clone()
    rows[10][3] = float("nan")
    x = torch.stack(rows)
    n = x.shape[0]
    codes = torch.zeros(n, c, dtype=torch.float8_e4m3fn)
    sc = torch.zeros(n) if scales == "row" else torch.zeros(n, c // 32, dtype=torch.uint8)
    ok(emu, emu.kmx_quantize(0, None, capi.PREC_FP32, 1 if scales == "row" else 2, n, c, x.data_ptr(), c, codes.data_ptr(), c, sc.data_ptr()))
    sc = sc if scales == "row" else sc.view(torch.float8_e8m0fnu)
    ref.check_codes(codes[:9], sc[:9], x[:9].double(), torch.zeros(9, c).double())
    assert bool(torch.isnan(sc[9].float().reshape(-1)[-1])) and bool(torch.isnan(sc[10].float().reshape(-1)[0]))
    spoilt = codes[9:].float().reshape(2, -1, 32 if scales == "mx" else c)
    assert bool((spoilt[0, -1] == 0).all()) and bool((spoilt[1, 0] == 0).all())
    if scales == "mx":  # the other blocks of a spoilt row are their own
        assert bool((ref.values(codes, sc)[9, :32] == 1).all()) and bool((ref.values(codes, sc)[10, 32:] == 1).all())


def test_rms_norm_in_place(emu):
    """sum over the residual and y over x, the two tensors that may be written where they are read"""
    for c in (100, 33000):
        g = torch.Generator().manual_seed(c)
        x, r = torch.randn(4, c, generator=g).half(), torch.randn(4, c, generator=g).half()
        want_sum, want = ref.norm(x, None, 1e-6, None, r)
        a = capi.RmsNormArgs(type=capi.PREC_FP16, rows=4, channels=c, epsilon=1e-6, x=x.data_ptr(), residual=r.data_ptr(), sum=r.data_ptr(),
                             y=x.data_ptr(), x_stride=c, residual_stride=c, sum_stride=c, y_stride=c)
        ok(emu, emu.kmx_rmsnorm(0, None, ctypes.byref(a)))
        assert torch.equal(r, want_sum)
        ref.check_y(x, want)


def test_rms_norm_of_an_empty_mask_and_spoilt_rows(emu):
    """Masked rows may hold anything; a row that holds an infinity spoils itself only"""
    x = torch.randn(4, 64).bfloat16()
    x[1] = float("nan")
    x[2, 5] = float("inf")
    mask = torch.tensor([1.0, 0.0, 1.0, 1.0])
    y, codes, sc = torch.zeros(4, 64).bfloat16(), torch.zeros(4, 64, dtype=torch.float8_e4m3fn), torch.zeros(4)
    a = capi.RmsNormArgs(type=capi.PREC_BF16, scale_kind=1, rows=4, channels=64, epsilon=1e-6, x=x.data_ptr(), mask=mask.data_ptr(), y=y.data_ptr(),
                         codes=codes.data_ptr(), scales=sc.data_ptr(), x_stride=64, y_stride=64, codes_stride=64)
    ok(emu, emu.kmx_rmsnorm(0, None, ctypes.byref(a)))
    assert bool((y[1] == 0).all()) and bool((codes[1].float() == 0).all()) and float(sc[1]) == 1
    assert bool(torch.isnan(y[2, 5])) and bool((y[2, :5] == 0).all()) and bool(torch.isnan(sc[2])) and bool((codes[2].float() == 0).all())
    good = torch.tensor([0, 3])
    want = ref.norm(x[good])[1]
    ref.check_y(y[good], want)
    ref.check_codes(codes[good], sc[good], want, ref.norm_slack(want))


def eight(rows, k, scales, gen, spread=1.0):
    """codes and scales as a user's model holds them, made by plain torch"""
    v = torch.randn(rows, k, generator=gen) * spread
    if scales == "row":
        s = v.abs().amax(1) / 448
        return (v / s[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn), s
    e = torch.ceil(torch.log2(v.reshape(rows, -1, 32).abs().amax(2) / 448))
    return (v.reshape(rows, -1, 32) / torch.exp2(e)[..., None]).reshape(rows, k).to(torch.float8_e4m3fn), (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def aligned_copy(codes, stride):
    """[rows][k] codes at a 16-byte aligned address and row stride, the gaps full of NaN codes"""
    rows, k = codes.shape
    buf = torch.full((rows * stride + 32,), 0x7f, dtype=torch.uint8)
    lead = -buf.data_ptr() % 16
    buf[lead:lead + rows * stride].reshape(rows, stride)[:, :k] = codes.view(torch.uint8)
    return buf, buf.data_ptr() + lead


@pytest.mark.parametrize("m,n,k,scales,out,bias", [
    (1, 1, 32, "mx", "fp32", False), (1, 40, 16, "row", "bf16", True), (70, 33, 144, "row", "fp16", True), (65, 72, 160, "mx", "bf16", False),
    (64, 64, 128, "row", "fp32", True), (66, 64, 128, "row", "fp32", True), (16, 17, 1168, "row", "bf16", True), (3, 16, 4128, "mx", "fp16", False),
    (20, 30, 1056, "mx", "fp32", True), (64, 20, 2064, "row", "fp16", False), (70, 20, 96, "mx", "bf16", False),
    (65, 66, 1168, "row", "fp16", True), (70, 130, 1056, "mx", "bf16", True), (300, 70, 1040, "row", "fp32", False), (9, 130, 288, "mx", "fp32", True), (130, 8, 272, "row", "fp16", False), (33, 64, 256, "mx", "fp16", True),
    # rows enough (here) for the kernel that keeps its weights: one, two, three steps of k, whole tiles and partial ones, one and two tiles of channels
    (4230, 100, 272, "row", "fp16", True), (4096, 128, 384, "mx", "bf16", True), (2100, 200, 128, "mx", "fp16", False), (2300, 256, 256, "row", "bf16", True),
    (4097, 128, 16, "row", "fp16", True), (4352, 128, 384, "row", "fp16", True)])
def test_linear8(emu, m, n, k, scales, out, bias):
    g = torch.Generator().manual_seed(m * 1000 + n)
    a, sa = eight(m, k, scales, g, 2.0)
    w, sw = eight(n, k, scales, g, 0.1)
    b = torch.randn(n, generator=g) if bias else None
    abuf, ap = aligned_copy(a, k + 16)
    wbuf, wp = aligned_copy(w, k + 48)
    y = Guarded(m, n, n + 5, ref.TYPES[out])
    args = capi.Linear8Args(out_type=PREC[out], scale_kind=1 if scales == "row" else 2, rows=m, n=n, k=k, a=ap, a_scales=sa.data_ptr(), w=wp,
                            w_scales=sw.data_ptr(), bias=b.data_ptr() if bias else None, out=y.ptr, a_stride=k + 16, w_stride=k + 48, out_stride=n + 5)
    ok(emu, emu.kmx_linear8(0, None, ctypes.byref(args)))
    want, mag = ref.linear(ref.values(a, sa), ref.values(w, sw), b)
    ref.check_linear(y.get(), want, mag, k)
    y.rest_untouched()


@pytest.mark.parametrize("mode", ["1", "2"])
def test_linear8_copies_as_late_as_the_waits_allow(emu, mode):
    """The same with every copy into LDS landing only when a wait requires it (1), or at the barrier behind that wait (2), the counted stores of a tile among the
    requests: work-groups that go round several tiles, whole ones and partial ones, two stages and four, and the kernel that keeps its weights"""
    code = r"""
import ctypes, sys
sys.path[:0] = [%r, %r]
import test_ops_emulated as t
lib = ctypes.CDLL(%r)
t.capi.bind_ops(lib)
lib.kmx_last_error.restype = ctypes.c_char_p
for case in [(384, 384, 160, "row", "fp16", True), (390, 384, 288, "mx", "bf16", False), (320, 384, 1152, "row", "bf16", False), (200, 200, 1056, "mx", "fp16", True),
             (384, 384, 256, "row", "fp32", False), (4352, 128, 384, "row", "fp16", True), (4100, 128, 256, "mx", "bf16", False), (2100, 200, 128, "row", "fp16", False)]:
    print(case, flush=True)
    t.test_linear8(lib, *case)
print("LATE_OK")
""" % (REPO, os.path.join(REPO, "tests"), emu._name)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, env=dict(os.environ, KMX_EMU_LATE_DMA=mode))
    assert r.returncode == 0 and "LATE_OK" in r.stdout, r.stdout[-500:] + r.stderr[-2000:]


def rotary_args(q, k, qo, ko, pos, f, dtype, half, magnitude, inverse):
    """contiguous [batch][seq][heads][dim] tensors"""
    def tensor(i, o):
        b, s, h, d = i.shape
        return capi.RotaryTensor(i.data_ptr(), o.data_ptr(), s * h * d, h * d, d, s * h * d, h * d, d)
    a = capi.RotaryArgs(type=PREC[dtype], half=int(half), inverse=int(inverse), magnitude=magnitude, batch=q.shape[0], seq=q.shape[1], q_heads=q.shape[2],
                        k_heads=0 if k is None else k.shape[2], head_dim=q.shape[3], pairs=f.shape[2], axes=f.shape[1], freq_heads=f.shape[0],
                        frequencies=f.data_ptr(), positions=pos.data_ptr(), positions_are_64bit=int(pos.dtype == torch.int64),
                        pos_batch_stride=pos.stride(0), pos_seq_stride=pos.stride(1), pos_axis_stride=pos.stride(2), q=tensor(q, qo))
    if k is not None:
        a.k = tensor(k, ko)
    return a


@pytest.mark.parametrize("batch,seq,hq,hk,dim,pairs,half,dtype,axes,fh,inverse,far", [
    (1, 1, 1, 0, 2, 1, False, "fp32", 1, 1, False, 5), (2, 7, 12, 4, 32, 16, False, "fp16", 2, 4, False, 18), (3, 5, 9, 3, 24, 12, True, "bf16", 1, 1, False, 1000),
    (1, 9, 5, 5, 10, 3, True, "fp32", 1, 5, True, 100000), (2, 3, 32, 8, 128, 48, True, "bf16", 1, 1, False, 1000000), (1, 4, 6, 2, 80, 40, False, "fp32", 2, 2, True, 18),
    (4, 2, 3, 1, 21, 10, False, "fp16", 1, 1, False, 4000000)])
@pytest.mark.parametrize("in_place", [False, True])
def test_rotary(emu, batch, seq, hq, hk, dim, pairs, half, dtype, axes, fh, inverse, far, in_place):
    g = torch.Generator().manual_seed(dim * 100 + pairs)
    t = ref.TYPES[dtype]
    q, k = torch.randn(batch, seq, hq, dim, generator=g).to(t), torch.randn(batch, seq, hk, dim, generator=g).to(t) if hk else None
    pos = torch.randint(0, far + 1, (batch, seq, axes), generator=g, dtype=torch.int64 if far > 1000 else torch.int32)
    f = torch.rand(fh, axes, pairs, generator=g, dtype=torch.float64) * 2 - 1
    magnitude = 1.25 if far > 1000 else 1.0
    q0, k0 = q.clone(), k.clone() if hk else None
    qo = q if in_place else torch.full_like(q, 77)
    ko = k if in_place or not hk else torch.full_like(k, 77)
    ok(emu, emu.kmx_rotary(0, None, ctypes.byref(rotary_args(q, k, qo, ko, pos, f, dtype, half, magnitude, inverse))))
    for before, after in ((q0, qo), (k0, ko)) if hk else ((q0, qo),):
        flat = before.reshape(batch * seq, -1, dim)
        want = ref.rotary(flat, pos.reshape(batch * seq, axes), f, half, magnitude, inverse)
        ref.check_rotary(after.reshape(flat.shape), *want, magnitude)


def test_rotary_of_a_fused_buffer(emu):
    """q and k turned in place inside the rows of one projection's output; v, and the rows' ends, stay"""
    g = torch.Generator().manual_seed(1)
    tokens, hq, hk, d, row = 11, 4, 2, 16, 4 * 16 + 2 * 16 + 2 * 16 + 8
    buf = torch.randn(tokens, row, generator=g).half()
    was = buf.clone()
    f = torch.rand(1, 1, 8, generator=g, dtype=torch.float64)
    pos = torch.arange(tokens, dtype=torch.int32).reshape(1, tokens, 1)
    qp, kp = buf.data_ptr(), buf.data_ptr() + 2 * hq * d
    a = capi.RotaryArgs(type=capi.PREC_FP16, magnitude=1.0, batch=1, seq=tokens, q_heads=hq, k_heads=hk, head_dim=d, pairs=8, axes=1, freq_heads=1,
                        frequencies=f.data_ptr(), positions=pos.data_ptr(), pos_seq_stride=1, q=capi.RotaryTensor(qp, qp, 0, row, d, 0, row, d),
                        k=capi.RotaryTensor(kp, kp, 0, row, d, 0, row, d))
    ok(emu, emu.kmx_rotary(0, None, ctypes.byref(a)))
    x = was[:, :(hq + hk) * d].reshape(tokens, hq + hk, d)
    ref.check_rotary(buf[:, :(hq + hk) * d].reshape(x.shape), *ref.rotary(x, pos[0], f, False))
    assert torch.equal(buf[:, (hq + hk) * d:], was[:, (hq + hk) * d:])
