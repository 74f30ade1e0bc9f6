"""Calls of the decoder operators that are refused before any device is asked."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwd

from quantem.cuda.core import ml

BF16, F32, E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


def _t(*shape, dtype=BF16):
    return torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize("call,match", [
    (lambda: ml.rms_norm(_t(4, 8), None), "weight"),
    (lambda: ml.rms_norm(None, _t(8)), "x"),
    (lambda: ml.add_rms_norm(_t(4, 8), _t(4, 8), None), "weight"),
    (lambda: ml.rms_norm_fp8(_t(4, 8), None), "weight"),
    (lambda: ml.add_rms_norm_fp8(_t(4, 8), _t(4, 8), None), "weight"),
    (lambda: ml.quantize_rows_fp8(None), "x"),
    (lambda: ml.linear_act(None, _t(6, 8)), "x"),
    (lambda: ml.linear_act(_t(4, 8), None), "weight"),
    (lambda: ml.linear_act_fp8(_t(4, 8), None, _t(6, 8), None), "x_scale"),
    (lambda: ml.linear_act_fp8(_t(4, 8, dtype=E4M3), None, _t(6, 8, dtype=E4M3), _t(6, dtype=F32)), "x_scale"),
    (lambda: ml.linear_act_fp8(_t(4, 8, dtype=E4M3), _t(4, dtype=F32), None, _t(6, dtype=F32)), "weight"),
    (lambda: ml.linear_act_fp8(_t(4, 8, dtype=E4M3), _t(4, dtype=F32), _t(6, 8, dtype=E4M3), None), "weight_scale"),
])
def test_missing_tensors_are_refused(call, match):
    with pytest.raises(TypeError, match=rf"\b{match}\b.*must be a tensor"):
        call()


@pytest.mark.parametrize("call", [
    lambda x, d: ml.rms_norm(x, d(_t(8))),
    lambda x, d: ml.rms_norm(d(x), _t(8)),
    lambda x, d: ml.add_rms_norm(x, d(x), _t(8)),
    lambda x, d: ml.rms_norm_fp8(d(x), _t(8)),
    lambda x, d: ml.add_rms_norm_fp8(x, d(x), _t(8)),
    lambda x, d: ml.quantize_rows_fp8(d(x)),
    lambda x, d: ml.linear_act(d(x), _t(6, 8)),
    lambda x, d: ml.linear_act(x, _t(6, 8), residual=d(_t(4, 6))),
    lambda x, d: ml.linear_act_fp8(_t(4, 8, dtype=E4M3), d(_t(4, dtype=F32)), _t(6, 8, dtype=E4M3), _t(6, dtype=F32)),
])
def test_forward_mode_derivatives_are_refused(call):
    x = _t(4, 8)
    with fwd.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(x, lambda t: fwd.make_dual(t, torch.ones_like(t)))
        with pytest.raises(ValueError, match="CUDA"):  # without tangents: the usual checks
            call(x, lambda t: t)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda t: ml.rms_norm(t, _t(8)), (x,), (x,))
