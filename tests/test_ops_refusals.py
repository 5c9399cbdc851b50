"""What include/katamx_ops.h refuses, through the shipped library and without a GPU: arguments are checked before any device is touched, so a call that
passes every check ends in KMX_ERR_DEVICE here and one that does not in KMX_ERR_INVALID_ARG with a message that names the entry point."""
import ctypes
import re

import pytest
import torch

import os

from conftest import REPO
from katago_amd import capi, ops

MB = 1 << 20  # made-up addresses, never read: the checks look at numbers only


@pytest.fixture(scope="module")
def lib():
    lib = capi.load_library()
    capi.bind_ops(lib)
    return lib


def refused(lib, rc, entry, word):
    said = lib.kmx_last_error().decode()
    assert rc == capi.KMX_ERR_INVALID_ARG and said.startswith(entry + ":") and word in said, (rc, said)


def passes(lib, rc):
    """Every check passed: the device is what is missing (on a machine with one, device 9999)"""
    assert (rc == capi.KMX_ERR_DEVICE) or (rc == capi.KMX_ERR_INVALID_ARG and b"there is no device" in lib.kmx_last_error()), (rc, lib.kmx_last_error())


def test_every_declared_symbol_is_exported_and_bound(lib):
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(REPO, "include", "katamx_ops.h")).read(), flags=re.S)
    declared = sorted(set(re.findall(r"\b(kmx_[a-z0-9_]+)\s*\(", text)))
    assert declared == sorted(capi.OPS_SIGNATURES)
    assert lib.kmx_ops_version() == int(re.search(r"#define KMX_OPS_VERSION (\d+)", text).group(1))


def test_the_structs_are_laid_out_as_the_header_says(tmp_path):
    import subprocess

    src = tmp_path / "layout.c"
    names = {"kmx_rmsnorm_args": capi.RmsNormArgs, "kmx_linear8_args": capi.Linear8Args, "kmx_rotary_tensor": capi.RotaryTensor, "kmx_rotary_args": capi.RotaryArgs}
    lines = []
    for c, py in names.items():
        lines.append('printf("%s %%zu\\n", sizeof(%s));' % (c, c))
        for f in py._fields_:
            lines.append('printf("%s.%s %%zu\\n", offsetof(%s, %s));' % (c, f[0], c, f[0].rstrip("_")))
    src.write_text('#include <stdio.h>\n#include "katamx_ops.h"\nint main(void) { %s return 0; }\n' % "\n".join(lines))
    subprocess.run(["gcc", "-I" + os.path.join(REPO, "include"), str(src), "-o", str(tmp_path / "layout")], check=True)
    said = dict(l.split() for l in subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.splitlines())
    for c, py in names.items():
        assert int(said[c]) == ctypes.sizeof(py)
        for f in py._fields_:
            assert int(said["%s.%s" % (c, f[0])]) == getattr(py, f[0]).offset, f[0]


def norm_args(**kw):
    a = capi.RmsNormArgs(type=capi.PREC_FP16, scale_kind=1, rows=8, channels=96, epsilon=1e-6, x=1 * MB, x_stride=96, y=2 * MB, y_stride=96, codes=3 * MB,
                         codes_stride=96, scales=4 * MB, weight=5 * MB)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,word", [
    (dict(type=0), "type"), (dict(rows=-1), "rows"), (dict(rows=1 << 31), "rows"), (dict(channels=0), "channels"), (dict(channels=-5), "channels"),
    (dict(scale_kind=3), "scales"), (dict(scale_kind=0), "scales"), (dict(scales=None), "scales"), (dict(codes=None), "scales"),
    (dict(scale_kind=2, channels=95), "32"), (dict(x=None), "x is null"), (dict(residual=6 * MB, residual_stride=96), "residual"),
    (dict(sum=6 * MB, sum_stride=96), "residual"), (dict(y=None, codes=None, scales=None, scale_kind=0), "wanted"), (dict(epsilon=-1.0), "epsilon"),
    (dict(epsilon=float("nan")), "epsilon"), (dict(epsilon=float("inf")), "epsilon"), (dict(x=MB + 1), "aligned"), (dict(y=2 * MB + 1), "aligned"),
    (dict(weight=5 * MB + 2), "aligned"), (dict(mask=6 * MB + 1), "aligned"), (dict(scales=4 * MB + 2), "aligned"), (dict(x_stride=-96), "x:"), (dict(y_stride=95), "y:"),
    (dict(codes_stride=95), "codes:"), (dict(x_stride=1 << 62), "range"), (dict(y=MB + 96), "overlap"), (dict(y=MB, y_stride=97), "overlap"),
    (dict(codes=2 * MB), "overlap"), (dict(codes=MB), "overlap"), (dict(scales=2 * MB + 4), "overlap"), (dict(weight=2 * MB), "overlap"),
    (dict(residual=6 * MB, residual_stride=96, sum=2 * MB, sum_stride=96), "overlap"), (dict(mask=2 * MB), "overlap")])
def test_rmsnorm_refuses(lib, kw, word):
    refused(lib, lib.kmx_rmsnorm(9999, None, ctypes.byref(norm_args(**kw))), "kmx_rmsnorm", word)


@pytest.mark.parametrize("kw", [
    {}, dict(rows=0), dict(x_stride=0), dict(y=MB), dict(residual=6 * MB, residual_stride=96, sum=6 * MB, sum_stride=96),
    dict(residual=6 * MB, residual_stride=0, sum=MB, sum_stride=96), dict(rows=1, y_stride=0), dict(scale_kind=0, codes=None, scales=None), dict(y=None),
    dict(x_stride=192, y_stride=192, y=MB + 192),  # the two halves of one matrix's rows
    dict(weight=None, scale_kind=2, codes=3 * MB + 1, codes_stride=97, scales=4 * MB + 3)])
def test_rmsnorm_takes(lib, kw):
    passes(lib, lib.kmx_rmsnorm(9999, None, ctypes.byref(norm_args(**kw))))


def test_quantize_refuses(lib):
    def call(type=capi.PREC_BF16, kind=1, rows=8, c=64, x=MB, xs=64, codes=2 * MB, cs=64, scales=3 * MB):
        return lib.kmx_quantize(9999, None, type, kind, rows, c, x, xs, codes, cs, scales)
    passes(lib, call())
    passes(lib, call(rows=0))
    for kw, word in ((dict(type=9), "type"), (dict(kind=0), "scales"), (dict(kind=2, c=48), "32"), (dict(x=None), "x is null"), (dict(codes=None), "scales"),
                     (dict(x=MB + 1), "aligned"), (dict(cs=63), "codes"), (dict(codes=MB), "overlap"), (dict(scales=2 * MB), "overlap"), (dict(rows=-2), "rows")):
        refused(lib, call(**kw), "kmx_quantize", word)


def linear_args(**kw):
    a = capi.Linear8Args(out_type=capi.PREC_BF16, scale_kind=1, rows=9, n=33, k=64, a=MB, a_scales=2 * MB, w=3 * MB, w_scales=4 * MB, out=5 * MB, a_stride=64,
                         w_stride=64, out_stride=33)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,word", [
    (dict(out_type=7), "type"), (dict(rows=-1), "rows"), (dict(n=0), "n must"), (dict(k=0), "k must"), (dict(k=63), "k must"), (dict(k=8), "k must"),
    (dict(scale_kind=2, k=48), "32"), (dict(k=1 << 23), "k must"), (dict(scale_kind=0), "scales"), (dict(a=None), "needed"), (dict(w=None), "needed"),
    (dict(a_scales=None), "needed"), (dict(w_scales=None), "needed"), (dict(out=None), "needed"), (dict(a=MB + 8), "aligned"), (dict(w=3 * MB + 1), "aligned"),
    (dict(a_scales=2 * MB + 1), "aligned"), (dict(bias=6 * MB + 2), "aligned"), (dict(out=5 * MB + 1), "aligned"), (dict(a_stride=72), "strides"),
    (dict(w_stride=-64), "strides"), (dict(a_stride=1 << 23), "strides"), (dict(out_stride=32), "out:"), (dict(out_stride=1 << 23), "out_stride"), (dict(n=1 << 23, out_stride=1 << 23), "n must"), (dict(out=MB), "overlap"), (dict(out=4 * MB), "overlap"),
    (dict(bias=5 * MB), "overlap")])
def test_linear8_refuses(lib, kw, word):
    refused(lib, lib.kmx_linear8(9999, None, ctypes.byref(linear_args(**kw))), "kmx_linear8", word)


@pytest.mark.parametrize("kw", [{}, dict(rows=0), dict(scale_kind=2, a_scales=2 * MB + 1), dict(a_stride=0), dict(w_stride=128), dict(bias=6 * MB), dict(k=16)])
def test_linear8_takes(lib, kw):
    passes(lib, lib.kmx_linear8(9999, None, ctypes.byref(linear_args(**kw))))


def rotary_args(**kw):
    a = capi.RotaryArgs(type=capi.PREC_FP16, magnitude=1.0, batch=2, seq=5, q_heads=4, k_heads=2, head_dim=16, pairs=8, axes=1, freq_heads=1,
                        frequencies=6 * MB, positions=7 * MB, pos_batch_stride=5, pos_seq_stride=1,
                        q=capi.RotaryTensor(MB, 2 * MB, 320, 64, 16, 320, 64, 16), k=capi.RotaryTensor(3 * MB, 4 * MB, 160, 32, 16, 160, 32, 16))
    for k, v in kw.items():
        setattr(a, k, v)
    return a


T = capi.RotaryTensor


@pytest.mark.parametrize("kw,word", [
    (dict(type=0), "type"), (dict(batch=-1), "batch"), (dict(batch=1 << 20, seq=1 << 11), "batch"), (dict(q_heads=0), "heads"), (dict(k_heads=-1), "heads"),
    (dict(pairs=9), "pairs"), (dict(pairs=0), "pairs"), (dict(axes=3), "axes"), (dict(axes=0), "axes"), (dict(freq_heads=3), "freq_heads"), (dict(freq_heads=4), "freq_heads"),
    (dict(freq_heads=0), "freq_heads"), (dict(frequencies=None), "frequencies"), (dict(positions=None), "positions"), (dict(frequencies=6 * MB + 4), "aligned"),
    (dict(positions=7 * MB + 2), "aligned"), (dict(positions=7 * MB + 4, positions_are_64bit=1), "aligned"), (dict(pos_seq_stride=-1), "strides"),
    (dict(magnitude=float("inf")), "magnitude"), (dict(magnitude=float("nan")), "magnitude"), (dict(q=T(None, 2 * MB, 320, 64, 16, 320, 64, 16)), "q is null"),
    (dict(k=T(3 * MB, None, 160, 32, 16, 160, 32, 16)), "k is null"), (dict(q=T(MB + 1, 2 * MB, 320, 64, 16, 320, 64, 16)), "aligned"),
    (dict(q=T(MB, 2 * MB, 320, 64, -16, 320, 64, 16)), "strides"), (dict(q=T(MB, 2 * MB, 320, 64, 16, 320, 64, 15)), "overlap"),
    (dict(q=T(MB, 2 * MB, 320, 64, 16, 320, 0, 16)), "overlap"), (dict(q=T(MB, 2 * MB, 320, 64, 16, 1 << 50, 64, 16)), "range"),
    (dict(q=T(MB, MB + 32, 320, 64, 16, 320, 64, 16)), "not in itself"), (dict(q=T(MB, MB, 320, 64, 16, 320, 16, 80)), "not in itself"),
    (dict(q=T(MB, 3 * MB, 320, 64, 16, 320, 64, 16)), "q and k overlap"), (dict(k=T(3 * MB, 2 * MB + 64, 160, 32, 16, 160, 32, 16)), "q and k overlap"),
    (dict(k=T(MB, 4 * MB, 160, 32, 16, 160, 32, 16), q=T(MB, MB, 320, 64, 16, 320, 64, 16)), "q and k overlap"),  # k read where q is written
    (dict(q=T(MB, MB, 479, 96, 16, 479, 96, 16), k=T(MB + 128, MB + 128, 479, 96, 16, 479, 96, 16)), "overlap"),  # columns, but sequences meet
    (dict(q=T(MB, MB, 480, 16, 80, 480, 16, 80), k=T(MB + 640 - 32, MB + 640 - 32, 480, 16, 80, 480, 16, 80)), "q and k overlap"),
    (dict(positions=2 * MB + 8), "positions"), (dict(frequencies=4 * MB + 64), "positions"), (dict(positions=4 * MB + 604, positions_are_64bit=0), "positions"),
    (dict(batch=1 << 20, seq=1 << 10, q=T(MB, 2 * MB, 1 << 39, 64, 16, 320, 64, 16)), "range"), (dict(pos_seq_stride=1 << 60), "range"),
    (dict(q_heads=1 << 16, head_dim=1 << 16, pairs=1, k_heads=0), "channels")])
def test_rotary_refuses(lib, kw, word):
    refused(lib, lib.kmx_rotary(9999, None, ctypes.byref(rotary_args(**kw))), "kmx_rotary", word)


@pytest.mark.parametrize("kw", [
    {}, dict(batch=0), dict(seq=0), dict(k_heads=0, k=T()), dict(freq_heads=2), dict(q=T(MB, MB, 320, 64, 16, 320, 64, 16)), dict(pos_batch_stride=0),
    dict(q=T(MB, 2 * MB, 0, 0, 0, 320, 64, 16)),  # a broadcast input
    dict(q=T(MB, 2 * MB, 320, 64, 16, 320, 16, 80)),  # heads before tokens
    dict(q=T(MB, MB, 500, 100, 16, 500, 100, 16), k=T(MB + 128, MB + 128, 500, 100, 16, 500, 100, 16)),  # columns of one projection's rows
    dict(q=T(MB, MB, 480, 16, 80, 480, 16, 80), k=T(MB + 640, MB + 640, 480, 16, 80, 480, 16, 80)),  # [batch, q's and k's heads, seq, dim], in place
    dict(q_heads=2, q=T(MB, MB, 480, 96, 48, 480, 96, 48), k=T(MB + 32, MB + 32, 480, 96, 48, 480, 96, 48)),  # q, k, v side by side in each head
    dict(q=T(MB, MB + 128, 640, 128, 16, 640, 128, 16)),  # out beside in, in the same rows
    dict(positions=2 * MB + 1280)])  # behind q's last channel
def test_rotary_takes(lib, kw):
    passes(lib, lib.kmx_rotary(9999, None, ctypes.byref(rotary_args(**kw))))


def test_null_arguments_are_refused(lib):
    for entry in ("kmx_rmsnorm", "kmx_linear8", "kmx_rotary"):
        refused(lib, getattr(lib, entry)(0, None, None), entry, "null")


def test_python_refuses_what_is_not_on_a_device():
    x = torch.zeros(4, 32)
    for call in (lambda: ops.rms_norm(x), lambda: ops.quantize(x), lambda: ops.rotary(x.reshape(4, 1, 32), None, torch.zeros(4, dtype=torch.int32), torch.zeros(16).double()),
                 lambda: ops.linear8(x.to(torch.float8_e4m3fn), torch.ones(4), x.to(torch.float8_e4m3fn), torch.ones(4)), lambda: ops.rms_norm([1.0])):
        with pytest.raises(capi.KatamxError) as e:
            call()
        assert e.value.code == capi.KMX_ERR_INVALID_ARG


def test_rotary_frequencies():
    f, m = ops.rotary_frequencies(8, 10000.0)
    assert m == 1.0 and torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001]).double(), rtol=1e-7)
    assert torch.equal(ops.rotary_frequencies(8, 10000.0, scaling="linear", factor=4.0)[0], f / 4)
    b, _ = ops.rotary_frequencies(8, 10000.0, scaling="base", factor=4.0)
    assert float(b[0]) == 1.0 and abs(float(b[-1] / f[-1]) - 0.25) < 1e-12  # the fastest pair kept, the slowest interpolated
    p, m = ops.rotary_frequencies(64, 10000.0, scaling="parts", factor=8.0, original_length=4096)
    f = ops.rotary_frequencies(64, 10000.0)[0]
    turns = 4096 * f / (2 * torch.pi)
    assert torch.equal(p[turns >= 32], f[turns >= 32]) and torch.allclose(p[turns <= 1], f[turns <= 1] / 8, rtol=1e-15)
    between = (turns > 1) & (turns < 32)
    assert between.any() and bool((p[between] < f[between]).all()) and bool((p[between] > f[between] / 8).all()) and abs(m - 1.2079441541679836) < 1e-12
    for bad in (dict(rotary_dim=7), dict(rotary_dim=8, base=1.0), dict(rotary_dim=8, factor=0.5), dict(rotary_dim=8, scaling="what"), dict(rotary_dim=2, scaling="base"),
                dict(rotary_dim=8, scaling="parts")):
        with pytest.raises(capi.KatamxError):
            ops.rotary_frequencies(**bad)


def test_board_frequencies_are_the_nets_tables():
    """desc.cpp:1340-1358: pair p < P / 2 turns with y by theta^(-2p / (D / 2)), the others with x"""
    f, pos = ops.board_frequencies(16, 100.0), ops.board_positions(5, 3)
    angle = (pos.double()[:, :, None] * f).sum(1)
    for y in range(3):
        for x in range(5):
            for p in range(8):
                want = (y if p < 4 else x) * 100.0 ** (-2.0 * (p % 4) / 8)
                assert abs(float(angle[y * 5 + x, p]) - want) < 1e-12
