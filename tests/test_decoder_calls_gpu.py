"""How the decoder operators may be called on the device: missing tensors are
refused, forward-mode derivatives are refused, recorded graphs hold the
operators."""

from __future__ import annotations

import pytest
import torch

from quantem.cuda.core import ml

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def _inputs(rows=40, k=64, n=72):
    g = torch.Generator(device="cuda").manual_seed(5)
    x, w, nw = (torch.randn(s, generator=g, device="cuda").to(BF16) for s in ((rows, k), (n, k), (k,)))
    return x, w, nw


@pytest.mark.parametrize("call", [
    lambda x, w: ml.rms_norm(x, None),
    lambda x, w: ml.add_rms_norm(x, x, None),
    lambda x, w: ml.rms_norm_fp8(x, None),
    lambda x, w: ml.add_rms_norm_fp8(x, x, None),
    lambda x, w: ml.quantize_rows_fp8(None),
    lambda x, w: ml.linear_act(x, None),
    lambda x, w: ml.linear_act(None, w),
    lambda x, w: ml.linear_act_fp8(x, None, w, None),
    lambda x, w: ml.linear_act_fp8(*ml.quantize_rows_fp8(x.detach()), ml.quantize_rows_fp8(w)[0], None),
    lambda x, w: ml.linear_act_fp8(ml.quantize_rows_fp8(x.detach())[0], None, *ml.quantize_rows_fp8(w)),
    lambda x, w: ml.linear_act_fp8(ml.quantize_rows_fp8(x.detach())[0], None, ml.quantize_rows_fp8(w)[0], None),
])
def test_missing_tensors_are_refused(call):
    x, w, _ = _inputs()
    with pytest.raises(TypeError):
        call(x, w)
    with pytest.raises(TypeError):
        call(x.requires_grad_(), w)
