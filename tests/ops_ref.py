"""Plain formulas, in 64 bits, of the operators of katago_amd.ops, and how far a right kernel may be from them. Shared by the tests that run the
kernels on the CPU (test_ops_emulated.py) and on a GPU (test_gpu_ops.py).

Tolerances count roundings. eps(t) / 2 relative is one rounding to type t (bf16 2^-8, fp16 2^-11, fp32 2^-24, e4m3 2^-4); U = 2^-24 one fp32 rounding."""
import torch

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
U = 2.0 ** -24
SMALLEST = {torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133, torch.float32: 2.0 ** -149}  # a step among the subnormals


def half(t):
    return torch.finfo(t).eps / 2


def norm(x, w=None, eps=1e-6, beta=None, residual=None, mask=None):
    """(sum or None, y) in 64 bits; x [rows][c]"""
    total = None
    h = x.double()
    if residual is not None:
        total = (x.float() + residual.float()).to(x.dtype)
        h = total.double()
    y = h / (h.square().mean(dim=1, keepdim=True) + eps).sqrt()
    if w is not None:
        y = y * w.double()
    if beta is not None:
        y = y + beta.double()
    if mask is not None:
        y = torch.where(mask.reshape(-1, 1) != 0, y, torch.zeros_like(y))
    return total, y


def norm_slack(y, beta=None):
    """How far fp32 arithmetic may bring y from y: the sum of squares adds at most 40 terms one after the other, then 10 levels of a tree (50 U, half
    of it in the root), the root and the products 3 U: under 32 U of the product, one more of the sum with beta."""
    b = 0.0 if beta is None else beta.double().abs()
    return 40 * U * (y.abs() + 2 * b)


def check_y(got, want, beta=None):
    t = got.dtype
    far = (got.double() - want).abs()
    ok = norm_slack(want, beta) + half(t) * (want.abs() + norm_slack(want, beta)) + SMALLEST[t] / 2
    assert bool((far <= ok).all()), float((far / ok).max())


def values(codes, scales):
    """What 8-bit codes stand for, in 64 bits"""
    c = codes.double()
    if scales.dtype == torch.float32:
        return c * scales.double().reshape(-1, 1)
    s = scales.view(torch.uint8).double()
    s = torch.where(s == 255, torch.full_like(s, float("nan")), torch.exp2(s - 127))
    return (c.reshape(c.shape[0], -1, 32) * s.reshape(c.shape[0], -1, 1)).reshape(c.shape)


def check_codes(codes, scales, want, slack):
    """codes and scales of finite `want`, which the kernel may see off by slack"""
    rows, c = want.shape
    blocks = want.reshape(rows, 1, c) if scales.dtype == torch.float32 else want.reshape(rows, -1, 32)
    sl = slack.reshape(blocks.shape)
    top, top_slack = blocks.abs().amax(dim=2), sl.amax(dim=2)
    if scales.dtype == torch.float32:
        s = scales.double().reshape(rows, 1)
        right = torch.where(top > 0, (top / 448).clamp_min(2.0 ** -126), torch.ones_like(top))
        assert bool(((s - right).abs() <= top_slack / 448 + 2 * U * right).all())
    else:
        e = scales.view(torch.uint8).to(torch.int64).reshape(rows, -1) - 127
        low, high = (torch.ceil(torch.log2(v / 448)).clamp_min(-127) for v in ((top - top_slack).clamp_min(2.0 ** -140), top + top_slack + 2.0 ** -140))
        s = torch.exp2(e.double())
        assert bool(((top == 0) & (e == 0) | (top > 0) & (e >= low) & (e <= high)).all())
    v = values(codes, scales).reshape(blocks.shape)
    # to the nearest: half a step of what has 4 significant bits, 2^-10 scales among the subnormals; the scale's own roundings move the codes
    ok = torch.maximum(half(torch.float8_e4m3fn) * (blocks.abs() + sl), s[..., None] * 2.0 ** -10) + sl + 4 * U * blocks.abs()
    far = (v - blocks).abs()
    assert bool((far <= ok).all()), float((far / ok).max())


def linear(a, w, bias=None):
    """(result, sum of magnitudes) in 64 bits of a [m][k], w [n][k]"""
    y, mag = a @ w.t(), a.abs() @ w.abs().t()
    return (y, mag) if bias is None else (y + bias.double(), mag + bias.double().abs())


def check_linear(got, want, mag, k):
    """fp32 results: at most k / 16 + 24 additions one after the other, each off by up to 2 U of the sum of magnitudes so far. 16-bit results: of each
    8 products on the 8-bit instructions the 7 smaller ones lose less than 2^-13 of the largest, in all below 7 * 2^-13 of the magnitudes; with random
    signs the squares add: below sqrt(7) 2^-13 of the result's norm times sqrt(max^2 / mean^2) <= sqrt(8): 2^-10, and the output's rounding."""
    t = got.dtype
    sums = 2 * U * (k / 16 + 24) * mag
    far = (got.double() - want).abs()
    ok = sums + half(t) * (want.abs() + sums) + SMALLEST[t] / 2
    if t != torch.float32:
        ok = ok + 7 * 2.0 ** -13 * mag
        if want.numel() >= 256:
            assert float(far.norm() / want.norm()) <= half(t) + 2.0 ** -10
    assert bool((far <= ok).all()), float((far / ok).max())


def rotary(x, positions, freqs, half_layout, magnitude=1.0, inverse=False):
    """x [tokens][heads][dim], positions [tokens][axes], freqs fp64 [freq_heads][axes][pairs] -> (result, |u| + |v| of each channel's pair, |angle|)"""
    pairs = freqs.shape[2]
    angle = (positions.double()[:, None, :, None] * freqs[None]).sum(2)  # [tokens][freq_heads][pairs]
    angle = angle.repeat_interleave(x.shape[1] // freqs.shape[0], dim=1)
    if inverse:
        angle = -angle
    c, s = angle.cos() * magnitude, angle.sin() * magnitude
    v = x.double()
    ia = torch.arange(pairs) if half_layout else 2 * torch.arange(pairs)
    ib = ia + (pairs if half_layout else 1)
    out, size, turn = v.clone(), torch.zeros_like(v), torch.zeros_like(v)
    out[..., ia] = v[..., ia] * c - v[..., ib] * s
    out[..., ib] = v[..., ia] * s + v[..., ib] * c
    size[..., ia] = size[..., ib] = v[..., ia].abs() + v[..., ib].abs()
    turn[..., ia] = turn[..., ib] = angle.abs()
    return out, size, turn


def check_rotary(got, want, size, turn, magnitude=1.0):
    """The turn's fraction is rounded to fp32 once (2^-25 of a turn: pi U), sine and cosine are good to 2.1 U, times the magnitude, three roundings of the
    rotation: below 10 U of the pair; the angle in fp64 is off by at most 2^-51 of itself (here and in the formula)."""
    t = got.dtype
    far = (got.double() - want).abs()
    slack = abs(magnitude) * size * (10 * U + turn * 2.0 ** -50)
    ok = slack + half(t) * (want.abs() + slack) + SMALLEST[t] / 2
    ok = torch.where(size == 0, torch.where(want == 0, ok, torch.zeros_like(ok)), ok)  # copied channels come as they are
    assert bool((far <= ok).all()), float((far / ok.clamp_min(1e-300)).max())
