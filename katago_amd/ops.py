"""Operators on device tensors (include/katamx_ops.h): what surrounds the attention of a transformer trunk when its projections run in
8 bits. torch is the container of device memory here, as in the rest of the package; the kernels are libkatamx.so's own.

    n = rms_norm(x, weight, eps, residual=stream, mask=mask, scales="row")   # n.sum, n.y, n.codes, n.scales
    wq, ws = quantize(weight_matrix, "row")                                  # once, when a model is loaded
    qkv = linear8(n.codes, n.scales, wq, ws, bias)
    q, k = rotary(q, k, positions, frequencies)

Each call runs on the current stream of its tensors' device, returns without waiting, allocates nothing but the outputs it returns, and gives the
same bits for the same inputs; it may be captured into a graph. Bad arguments raise KatamxError before anything is launched. The operators
compute no gradients: a tensor that requires one is refused outside torch.no_grad() (rotary(inverse=True) is the transpose of rotary()).
"""
import collections
import ctypes
import math

import torch

from . import capi
from .capi import KatamxError

SCALES = {None: 0, "row": 1, "mx": 2}
MX_BLOCK = 32
E4M3_MAX = 448.0
_TYPES = {torch.float16: capi.PREC_FP16, torch.bfloat16: capi.PREC_BF16, torch.float32: capi.PREC_FP32}
_CODES = torch.float8_e4m3fn

Normed = collections.namedtuple("Normed", ["sum", "y", "codes", "scales"])

_lib = None


def _library():
    global _lib
    if _lib is None:
        lib = capi.load_library()
        capi.bind_ops(lib)
        _lib = lib
    return _lib


def _refuse(why):
    raise KatamxError(capi.KMX_ERR_INVALID_ARG, why)


def _on_device(names, *tensors):
    """The index of the device all of them are on (None among them: not given); gradients are refused."""
    index, grad = None, torch.is_grad_enabled()
    for t in tensors:
        if t is None:
            continue
        try:
            d = t.get_device()
        except AttributeError:
            _refuse("%s must be a tensor" % _name(names, tensors, t))
        if d != index:
            if d < 0 or not t.is_cuda:
                _refuse("%s is on %s: the operators work on device tensors" % (_name(names, tensors, t), t.device))
            if index is not None:
                _refuse("%s is on device %d, the others on %d" % (_name(names, tensors, t), d, index))
            index = d
        if grad and t.requires_grad:
            _refuse("%s requires a gradient and the operators compute none: call them under torch.no_grad()" % _name(names, tensors, t))
    return index


def _name(names, tensors, t):
    return names.split()[[u is t for u in tensors].index(True)]


def _rows(name, t, channels=None):
    """(rows, channels, row stride) of a tensor whose leading dimensions step evenly"""
    if t.dim() < 1:
        _refuse("%s must have a dimension of channels" % name)
    shape, strides = t.shape, t.stride()
    c = shape[-1]
    if channels is not None and c != channels:
        _refuse("%s has %d channels, not %d" % (name, c, channels))
    if c > 1 and strides[-1] != 1:
        _refuse("%s: channels must be contiguous" % name)
    if t.dim() == 2:
        return shape[0], c, strides[0]
    rows, stride = 1, 0
    for n, s in zip(reversed(shape[:-1]), reversed(strides[:-1])):
        if n == 0:
            return 0, c, c
        if n == 1:
            continue
        if rows == 1:
            stride = s
        elif s != stride * rows:
            _refuse("%s: the rows' strides do not collapse to one" % name)
        rows *= n
    return rows, c, stride if rows > 1 else c


def _vector(name, t, length):
    if t is None:
        return None
    if t.dtype != torch.float32 or t.numel() != length or not t.is_contiguous():
        _refuse("%s must be %d contiguous float32 values" % (name, length))
    return t.data_ptr()


def _given(name, t, shape, dtype):
    if t.dtype != dtype or tuple(t.shape) != tuple(shape):
        _refuse("%s must be %s of shape %s" % (name, dtype, tuple(shape)))
    return t


def _type(name, dtype):
    typ = _TYPES.get(dtype)
    if typ is None:
        _refuse("%s is %s, not float16, bfloat16 or float32" % (name, dtype))
    return typ


def _current_stream(index):
    return torch.cuda.current_stream(index).cuda_stream


# (the same address without a Stream object around it, which costs 2 us of a call's 10)
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _current_stream)


def rms_norm(x, weight=None, eps=1e-6, *, beta=None, residual=None, mask=None, scales=None, want_y=None, sum_out=None, y_out=None):
    """RMS norm of x's rows ([..., channels]), with the residual's addition in front and e4m3 codes behind:

        sum   = x + residual, in x's type; it is what is normalised (None without a residual)
        y     = sum / sqrt(mean(sum^2) + eps) * weight + beta; 0 on rows whose mask ([...], float32) is 0
        codes, scales = y in e4m3: scales="row" float32 [...], "mx" float8_e8m0fnu [..., channels / 32]; None: neither

    want_y: whether y itself is returned (by default only without scales). weight and beta: float32 [channels]. sum_out / y_out: the tensors to write,
    each may be x or residual itself. Returns Normed(sum, y, codes, scales), None for what was not asked for."""
    device = _on_device("x weight beta residual mask sum_out y_out", x, weight, beta, residual, mask, sum_out, y_out)
    dtype = x.dtype
    a = capi.RmsNormArgs(_type("x", dtype), SCALES.get(scales, -1))
    if a.scale_kind < 0:
        _refuse("scales must be None, 'row' or 'mx'")
    if want_y is None:
        want_y = scales is None or y_out is not None
    if y_out is not None and not want_y or sum_out is not None and residual is None:
        _refuse("an output is given that is not computed")
    shape = x.shape
    rows, c, a.x_stride = _rows("x", x)
    a.rows, a.channels, a.epsilon, a.x = rows, c, eps, x.data_ptr()
    a.weight, a.beta, a.mask = _vector("weight", weight, c), _vector("beta", beta, c), _vector("mask", mask, rows)
    total = y = codes = sc = None
    if residual is not None:
        if residual.dtype != dtype or residual.shape != shape:
            _refuse("residual must be of x's type and shape")
        a.residual, a.residual_stride = residual.data_ptr(), _rows("residual", residual)[2]
        total = torch.empty_like(x) if sum_out is None else _given("sum_out", sum_out, shape, dtype)
        a.sum, a.sum_stride = total.data_ptr(), _rows("sum_out", total)[2]
    if want_y:
        y = torch.empty_like(x) if y_out is None else _given("y_out", y_out, shape, dtype)
        a.y, a.y_stride = y.data_ptr(), _rows("y_out", y)[2]
    if scales is not None:
        codes, sc = _codes_for(x, scales)
        a.codes, a.codes_stride, a.scales = codes.data_ptr(), c, sc.data_ptr()
    if rows:
        lib = _lib or _library()
        rc = lib.kmx_rmsnorm(device, _stream(device), ctypes.byref(a))
        if rc:
            capi.check(rc, lib)
    return Normed(total, y, codes, sc)


def _codes_for(x, scales):
    shape = x.shape
    if scales == "row":
        sc = x.new_empty(shape[:-1], dtype=torch.float32)
    else:
        if shape[-1] % MX_BLOCK:
            _refuse("scales for 32 channels each need a multiple of 32 channels, not %d" % shape[-1])
        sc = x.new_empty(shape[:-1] + (shape[-1] // MX_BLOCK,), dtype=torch.float8_e8m0fnu)
    return x.new_empty(shape, dtype=_CODES), sc


def quantize(x, scales="row"):
    """(codes, scales) of x's rows ([..., channels]) in e4m3: what linear8 multiplies. scales as in rms_norm."""
    device = _on_device("x", x)
    typ = _type("x", x.dtype)
    if scales not in ("row", "mx"):
        _refuse("scales must be 'row' or 'mx'")
    rows, c, xs = _rows("x", x)
    codes, sc = _codes_for(x, scales)
    if rows:
        lib = _lib or _library()
        rc = lib.kmx_quantize(device, _stream(device), typ, SCALES[scales], rows, c, x.data_ptr(), xs, codes.data_ptr(), c, sc.data_ptr())
        if rc:
            capi.check(rc, lib)
    return codes, sc


def _kind_of(name, codes, scales, rows, k):
    if codes.dtype != _CODES:
        _refuse("%s must be float8_e4m3fn" % name)
    if not scales.is_contiguous():
        _refuse("%s's scales must be contiguous" % name)
    if scales.dtype == torch.float32 and scales.numel() == rows:
        return 1
    if scales.dtype == torch.float8_e8m0fnu and k % MX_BLOCK == 0 and scales.numel() == rows * (k // MX_BLOCK):
        return 2
    _refuse("%s's scales must be float32 of one a row or float8_e8m0fnu of one for 32 channels" % name)


def linear8(codes, scales, weight_codes, weight_scales, bias=None, *, out_dtype=torch.float16, out=None):
    """[..., n] = (codes * scales) (weight_codes * weight_scales)^T + bias: codes e4m3 [..., k], weight_codes e4m3 [n, k], scales of both as
    rms_norm / quantize return them (of one kind), bias float32 [n]. k is a multiple of 16 (mx: 32). out_dtype float16, bfloat16 or float32; float32
    is summed in fp32 throughout, the others on the 8-bit matrix instructions (katamx_ops.h)."""
    device = _on_device("codes scales weight_codes weight_scales bias out", codes, scales, weight_codes, weight_scales, bias, out)
    if weight_codes.dim() != 2:
        _refuse("weight_codes must be [n, k]")
    n, k, ws = _rows("weight_codes", weight_codes)
    rows, k, cs = _rows("codes", codes, k)
    kind = _kind_of("codes", codes, scales, rows, k)
    if _kind_of("weight_codes", weight_codes, weight_scales, n, k) != kind:
        _refuse("the scales of codes and weight_codes are of different kinds")
    shape = codes.shape[:-1] + (n,)
    if out is None:
        typ = _type("out_dtype", out_dtype)
        out = codes.new_empty(shape, dtype=out_dtype)
        stride = n
    else:
        typ = _type("out", out.dtype)
        stride = _rows("out", _given("out", out, shape, out.dtype))[2]
    if rows:
        a = capi.Linear8Args(typ, kind, rows, n, k, codes.data_ptr(), scales.data_ptr(), weight_codes.data_ptr(), weight_scales.data_ptr(),
                             _vector("bias", bias, n), out.data_ptr(), cs, ws, stride)
        lib = _lib or _library()
        rc = lib.kmx_linear8(device, _stream(device), ctypes.byref(a))
        if rc:
            capi.check(rc, lib)
    return out


def _token_strides(name, t, lead):
    """(batch, seq, head) strides of [batch, seq, heads, dim] or [tokens, heads, dim]"""
    st = t.stride()
    if st[-1] != 1 and t.shape[-1] > 1:
        _refuse("%s: channels must be contiguous" % name)
    return (st[0] if lead == 2 else 0), st[lead - 1], st[lead]


def rotary(q, k, positions, frequencies, *, layout="interleaved", magnitude=1.0, inverse=False, q_out=None, k_out=None):
    """Rotary positions of q and k ([batch, seq, heads, head_dim] or [tokens, heads, head_dim]; k may be None and have fewer heads): pair p of a
    head's channels - neighbours (2p, 2p + 1), or (p, p + pairs) with layout="half" - turned by sum_axis positions[..., axis] *
    frequencies[head, axis, p] and multiplied with magnitude; channels from 2 * pairs on are copied.

    positions: int32 or int64, [batch, seq] / [tokens] (or [seq] for every sequence of a batch), and a last dimension of axes, which may be
    left out where there is one. frequencies: float64 [pairs], [axes, pairs] or [freq_heads, axes, pairs] on the device (rotary_frequencies(),
    board_frequencies()); freq_heads divides the heads of q and of k: query heads turn as the key head they read. inverse: the turn back, and
    the transpose. q_out / k_out: the tensors to write, each may be q / k itself. Returns (q_out, k_out)."""
    device = _on_device("q k positions frequencies q_out k_out", q, k, positions, frequencies, q_out, k_out)
    typ = _type("q", q.dtype)
    if layout not in ("interleaved", "half"):
        _refuse("layout must be 'interleaved' or 'half'")
    lead = q.dim() - 2
    if lead not in (1, 2):
        _refuse("q must be [batch, seq, heads, head_dim] or [tokens, heads, head_dim]")
    batch, seq = (q.shape[0], q.shape[1]) if lead == 2 else (1, q.shape[0])
    heads, dim = q.shape[lead], q.shape[lead + 1]
    if frequencies.dtype != torch.float64 or not frequencies.is_contiguous() or not 1 <= frequencies.dim() <= 3:
        _refuse("frequencies must be contiguous float64 [pairs], [axes, pairs] or [freq_heads, axes, pairs]")
    fshape = (1,) * (3 - frequencies.dim()) + tuple(frequencies.shape)
    axes = fshape[1]
    if positions.dtype not in (torch.int32, torch.int64):
        _refuse("positions must be int32 or int64")
    pshape, pst = tuple(positions.shape), positions.stride()
    wanted = ((seq,), (batch, seq))[:lead]
    pos_axis = 0
    if (axes > 1 or pshape not in wanted) and pshape and pshape[-1] == axes:
        pshape, pos_axis, pst = pshape[:-1], pst[-1], pst[:-1]
    elif axes > 1:
        _refuse("positions must have a last dimension of %d axes" % axes)
    if pshape not in wanted:
        _refuse("positions must be one for each token: %s for q's %s" % (tuple(positions.shape), tuple(q.shape)))
    pos_batch, pos_seq = pst if len(pshape) == 2 else (0, pst[0])
    k_heads = 0
    if k is not None:
        if k.dtype != q.dtype or k.dim() != lead + 2 or k.shape[:lead] != q.shape[:lead] or k.shape[-1] != dim:
            _refuse("k must have q's type, tokens and head_dim")
        k_heads = k.shape[lead]
    elif k_out is not None:
        _refuse("an output is given that is not computed")
    if not heads or (k is not None and not k_heads):
        _refuse("q and k must have heads")
    q_out = torch.empty_like(q) if q_out is None else _given("q_out", q_out, q.shape, q.dtype)
    tensors = [capi.RotaryTensor(q.data_ptr(), q_out.data_ptr(), *_token_strides("q", q, lead), *_token_strides("q_out", q_out, lead))]
    if k is not None:
        k_out = torch.empty_like(k) if k_out is None else _given("k_out", k_out, k.shape, k.dtype)
        tensors.append(capi.RotaryTensor(k.data_ptr(), k_out.data_ptr(), *_token_strides("k", k, lead), *_token_strides("k_out", k_out, lead)))
    if batch * seq:
        a = capi.RotaryArgs(typ, layout == "half", bool(inverse), magnitude, batch, seq, heads, k_heads, dim, fshape[2], axes, fshape[0],
                            frequencies.data_ptr(), positions.data_ptr(), positions.dtype == torch.int64, pos_batch, pos_seq, pos_axis, *tensors)
        lib = _lib or _library()
        rc = lib.kmx_rotary(device, _stream(device), ctypes.byref(a))
        if rc:
            capi.check(rc, lib)
    return q_out, k_out


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
