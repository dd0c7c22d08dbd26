"""CPU: the operators without a derivative refuse tensors through which one is
asked for, in reverse and in forward mode, before anything is launched."""

import pytest
import torch
from torch.autograd import forward_ad

from metal_liger_b200.ops.fused_sampling import fused_sample
from metal_liger_b200.ops.quantized_kv import (
    allocate_quantized_kv, quantized_kv_append, quantized_kv_attention)


def _calls():
    kv = allocate_quantized_kv(1, 1, 64, 64, device="cpu")
    row = torch.ones(1, 1, 1, 64, dtype=torch.bfloat16)
    start = torch.zeros(1, dtype=torch.int64)
    one = torch.full((1,), 0.5)
    yield "append k", row, lambda x: quantized_kv_append(kv, x, row, start)
    yield "append v", row, lambda x: quantized_kv_append(kv, row, x, start)
    yield "attention q", row, lambda x: quantized_kv_attention(x, kv, start)
    logits = torch.zeros(1, 8)
    yield "sample logits", logits, lambda x: fused_sample(x, one)
    yield "sample uniform", one, lambda x: fused_sample(logits, x)
    yield "sample temperature", one, lambda x: fused_sample(logits, one, temperature=x)
    yield "sample top_p", one, lambda x: fused_sample(logits, one, top_p=x)
    yield "sample min_p", one, lambda x: fused_sample(logits, one, min_p=x)


CALLS = list(_calls())


@pytest.mark.parametrize("what,x,call", CALLS, ids=[c[0] for c in CALLS])
def test_derivatives_are_refused(what, x, call):
    with pytest.raises(RuntimeError, match="backward"):
        call(x.clone().requires_grad_())
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(forward_ad.make_dual(x, torch.ones_like(x)))
        # (another tensor's being dual, or none being, is not this call's business)
        with pytest.raises(NotImplementedError):                 # there is no CPU kernel
            call(x)
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda y: call(y), (x,), (torch.ones_like(x),))
    with torch.no_grad(), pytest.raises(NotImplementedError):
        call(x.clone().requires_grad_())
