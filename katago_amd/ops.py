"""Operators on device tensors (include/katamx_ops.h): what surrounds the attention of a transformer trunk when its projections run in
8 bits. torch is the container of device memory here, as in the rest of the package; the kernels are libkatamx.so's own.

    n = rms_norm(x, weight, eps, residual=stream, mask=mask, scales="row")   # n.sum, n.y, n.codes, n.scales
    wq, ws = quantize(weight_matrix, "row")                                  # once, when a model is loaded
    qkv = linear8(n.codes, n.scales, wq, ws, bias)
    q, k = rotary(q, k, positions, frequencies)

Each call runs on the current stream of its tensors' device, returns without waiting, allocates nothing but the outputs it returns, and gives the
same bits for the same inputs; it may be captured into a graph. Bad arguments raise KatamxError before anything is launched. The operators
compute no gradients: a tensor that requires one is refused outside torch.no_grad(), one with a forward-mode tangent everywhere (rotary(inverse=True) is the
transpose of rotary()).
"""
import collections
import ctypes
import math

import torch

from . import capi
from .capi import KatamxError

SCALES = {None: 0, "row": 1, "mx": 2}

Normed = collections.namedtuple("Normed", ["sum", "y", "codes", "scales"])

_native = None  # _ops.so (csrc/ops_torch.cpp): a call's checks, outputs and launch


def _load():
    global _native
    lib = capi.load_library()
    capi.bind_ops(lib)
    try:
        from . import _ops
    except ImportError as e:
        raise KatamxError(capi.KMX_ERR_INTERNAL, "%s: run `python -m katago_amd.build` (the extension is mandatory)" % e)
    _ops.bind(_stream, KatamxError, *(ctypes.cast(getattr(lib, n), ctypes.c_void_p).value
                                      for n in ("kmx_last_error", "kmx_rmsnorm", "kmx_quantize", "kmx_linear8", "kmx_rotary")))
    _native = _ops
    return _ops


def _refuse(why):
    raise KatamxError(capi.KMX_ERR_INVALID_ARG, why)


def _current_stream(index):
    return torch.cuda.current_stream(index).cuda_stream


# (the same address without a Stream object around it, which costs 2 us)
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _current_stream)


def rms_norm(x, weight=None, eps=1e-6, *, beta=None, residual=None, mask=None, scales=None, want_y=None, sum_out=None, y_out=None):
    """RMS norm of x's rows ([..., channels]), with the residual's addition in front and e4m3 codes behind:

        sum   = x + residual, in x's type; it is what is normalised (None without a residual)
        y     = sum / sqrt(mean(sum^2) + eps) * weight + beta; 0 on rows whose mask ([...], float32) is 0
        codes, scales = y in e4m3: scales="row" float32 [...], "mx" float8_e8m0fnu [..., channels / 32]; None: neither

    want_y: whether y itself is returned (by default only without scales). weight and beta: float32 [channels]. x's rows (and every other tensor's) lie at one
    stride, whatever their leading dimensions are: x[:, 1:4] of a [2, 5, channels] tensor does not and is refused. sum_out / y_out: the tensors to write, each may be
    x or residual itself. Returns Normed(sum, y, codes, scales), None for what was not asked for."""
    kind = SCALES.get(scales, -1)
    if kind < 0:
        _refuse("scales must be None, 'row' or 'mx'")
    return Normed._make((_native or _load()).rms_norm(x, weight, eps, beta, residual, mask, kind, want_y, sum_out, y_out))


def quantize(x, scales="row"):
    """(codes, scales) of x's rows ([..., channels], at one stride) in e4m3: what linear8 multiplies. scales as in rms_norm."""
    if scales != "row" and scales != "mx":
        _refuse("scales must be 'row' or 'mx'")
    return (_native or _load()).quantize(x, SCALES[scales])


def linear8(codes, scales, weight_codes, weight_scales, bias=None, *, out_dtype=torch.float16, out=None):
    """[..., n] = (codes * scales) (weight_codes * weight_scales)^T + bias: codes e4m3 [..., k], weight_codes e4m3 [n, k], scales of both as
    rms_norm / quantize return them (of one kind), bias float32 [n]. k is a multiple of 16 (mx: 32). out_dtype float16, bfloat16 or float32; float32
    is summed in fp32 throughout (mx: scales from 2^-124 to 2^119), the others on the 8-bit matrix instructions (katamx_ops.h). out: the tensor to write, in its
    own type."""
    return (_native or _load()).linear8(codes, scales, weight_codes, weight_scales, bias, out_dtype, out)


def rotary(q, k, positions, frequencies, *, layout="interleaved", magnitude=1.0, inverse=False, q_out=None, k_out=None):
    """Rotary positions of q and k ([batch, seq, heads, head_dim] or [tokens, heads, head_dim]; k may be None and have fewer heads): pair p of a
    head's channels - neighbours (2p, 2p + 1), or (p, p + pairs) with layout="half" - turned by sum_axis positions[..., axis] *
    frequencies[head, axis, p] and multiplied with magnitude; channels from 2 * pairs on are copied.

    positions: int32 or int64, [batch, seq] / [tokens] (or [seq] for every sequence of a batch), and a last dimension of axes, which may be
    left out where there is one. frequencies: float64 [pairs], [axes, pairs] or [freq_heads, axes, pairs] on the device (rotary_frequencies(),
    board_frequencies()); freq_heads divides the heads of q and of k: query heads turn as the key head they read. inverse: the turn back, and
    the transpose. float32 tensors turn with sines and cosines good to their last bits, 16-bit ones with such that are off by 2^-22 at most. q_out / k_out:
    the tensors to write, each may be q / k itself. Returns (q_out, k_out)."""
    if layout not in ("interleaved", "half"):
        _refuse("layout must be 'interleaved' or 'half'")
    return (_native or _load()).rotary(q, k, positions, frequencies, layout == "half", magnitude, inverse, q_out, k_out)


def rotary_frequencies(rotary_dim, base=10000.0, *, scaling=None, factor=1.0, original_length=None, fast=32.0, slow=1.0):
    """(frequencies, magnitude) for rotary() over one axis: float64 [rotary_dim / 2] on the CPU, base ^ (-2p / rotary_dim), for contexts `factor`
    times the length that a model was trained on:

      None      as trained
      "linear"  every frequency / factor (positions interpolated)
      "base"    the base grows by factor ^ (d / (d - 2)): the slowest pair is interpolated by factor, the fastest kept
      "parts"   pairs that turn more than `fast` times within original_length are kept, those that turn less than `slow` times are / factor, those
                between blended linearly in their turns; the magnitude is 0.1 ln(factor) + 1 (YaRN, Peng et al. 2023)"""
    if rotary_dim < 2 or rotary_dim % 2:
        _refuse("rotary_dim must be even and at least 2")
    if not base > 1.0 or not factor >= 1.0:
        _refuse("base must be above 1 and factor at least 1")
    if scaling not in (None, "linear", "base", "parts"):
        _refuse("scaling must be None, 'linear', 'base' or 'parts'")
    if scaling == "base":
        if rotary_dim < 4:
            _refuse("scaling='base' needs at least two pairs")
        base = base * factor ** (rotary_dim / (rotary_dim - 2.0))
    p = torch.arange(rotary_dim // 2, dtype=torch.float64)
    f = base ** (-2.0 * p / rotary_dim)
    if scaling == "linear":
        return f / factor, 1.0
    if scaling != "parts":
        return f, 1.0
    if original_length is None or original_length < 1 or not fast > slow > 0:
        _refuse("scaling='parts' needs original_length and fast > slow > 0")
    turns = original_length * f / (2 * math.pi)  # of each pair within the trained length
    kept = ((turns - slow) / (fast - slow)).clamp(0.0, 1.0)
    return f * kept + f / factor * (1.0 - kept), 0.1 * math.log(factor) + 1.0


def board_frequencies(head_dim, theta):
    """float64 [2, head_dim / 2] (x and y axis) of the nets' fixed RoPE: the first half of the pairs turns with y, the second with x
    (TransformerAttentionDesc::computeRopeCosSin, desc.cpp:1340-1358)."""
    if head_dim < 4 or head_dim % 4:
        _refuse("head_dim must be a multiple of 4")
    per = head_dim // 4
    f = theta ** (-2.0 * torch.arange(per, dtype=torch.float64) / (head_dim // 2))
    z = torch.zeros(per, dtype=torch.float64)
    return torch.stack([torch.cat([z, f]), torch.cat([f, z])])


def board_positions(nnXLen, nnYLen):
    """int32 [nnYLen * nnXLen, 2]: x and y of each cell of a board's buffer, in cell order"""
    c = torch.arange(nnXLen * nnYLen, dtype=torch.int32)
    return torch.stack([c % nnXLen, torch.div(c, nnXLen, rounding_mode="floor")], dim=1)
