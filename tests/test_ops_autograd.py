"""What katago_amd.ops tells autograd, on the CPU: refusals come before a device is asked for."""
import pytest
import torch
from torch.autograd import forward_ad

from katago_amd import capi, ops


def test_forward_mode_tangents_are_refused():
    """A dual tensor's tangent would be dropped without a word; torch.no_grad() leaves forward mode on"""
    x, f = torch.ones(4, 2, 32), torch.ones(16).double()
    pos = torch.zeros(4, dtype=torch.int32)
    codes, s = torch.zeros(4, 32).to(torch.float8_e4m3fn), torch.ones(4)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))
        calls = [lambda: ops.rms_norm(dual(x)), lambda: ops.rms_norm(x, dual(torch.ones(32))), lambda: ops.rms_norm(x, residual=dual(x)), lambda: ops.quantize(dual(x)),
                 lambda: ops.linear8(codes, dual(s), codes, s), lambda: ops.linear8(codes, s, codes, s, dual(s)), lambda: ops.rotary(dual(x), None, pos, f),
                 lambda: ops.rotary(x, dual(x), pos, f), lambda: ops.rotary(x, None, pos, dual(f)), lambda: ops.rms_norm(x, y_out=dual(x))]
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                for call in calls:
                    with pytest.raises(capi.KatamxError, match="tangent") as e:
                        call()
                    assert e.value.code == capi.KMX_ERR_INVALID_ARG
