"""The values of a decode step over the 8-bit cache: captured steps, whole fused
layers and the eager loop against a decoder that is given the same tokens over
its own cache.

Bounds.  Two ways through the two bf16 layers (library GEMMs or this library's
GEMVs, attention over codes or over their values) differ by the layers'
roundings: 2e-2 of a hidden state's norm, as for the unfused step in
test_gpu_generation_quantized.py.  A K or V row that both ways quantise differs by
that share of its norm, and by one step of the codes (half a step each) per
element.  Two tokens' logits w.h can change places where they are closer than
|w - w'| times the hidden states' difference.
"""

import copy

import pytest
import torch

from metal_liger_b200.generation import (
    MetalLigerGenerator, MetalLigerQuantizedCache, _DecodeKernels, _QuantizedAttention)
from metal_liger_b200.patch import apply_metal_liger_to_qwen3vl, restore_attention_rope
from test_gpu_generation import DEV, _model

pytestmark = pytest.mark.gpu
REL = 2e-2


@pytest.fixture(params=["plain", "patched"])
def model(request):
    m = _model(seed=7)
    if request.param == "patched":
        apply_metal_liger_to_qwen3vl(m, fuse_lora=False, fuse_qk_norm=True,
                                     fuse_rope_in_attention=True)
    m.patched = request.param == "patched"
    yield m
    if m.patched:
        restore_attention_rope(m)


def _ids(B, n, seed=0):
    return torch.randint(0, 1000, (B, n), generator=torch.Generator().manual_seed(seed)).to(DEV)


def _step_of_codes(codes, scale, block):
    """The codes' largest step per position: int8 1, e4m3 2^-3 of 448 (a scale's
    largest value), times the scale."""
    step = 1.0 if codes.dtype == torch.int8 else 32.0
    return scale.repeat_interleave(block, 2) * step


def _check_rows(got, want, lo, hi):
    """Rows [lo, hi) of every layer's K and V of two caches."""
    for i, (a, b) in enumerate(zip(got.kv, want.kv)):
        for x, y, sa, sb, codes, name in (
                (*(c.dequantize()[0] for c in (a, b)), a.k_scale, b.k_scale, a.k_codes, "k"),
                (*(c.dequantize()[1] for c in (a, b)), a.v_scale, b.v_scale, a.v_codes, "v")):
            x, y = x[:, :, lo:hi].float(), y[:, :, lo:hi].float()
            step = torch.maximum(*(_step_of_codes(codes, s, a.block)[:, :, lo:hi] for s in (sa, sb)))
            err, size = (x - y).norm(dim=-1), y.norm(dim=-1)
            assert (size > 0).all()
            bound = REL * size + step * x.shape[-1] ** 0.5
            assert (err <= bound).all(), (i, name, (err / bound).max().item())


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("B", [1, 2, 3])
def test_captured_steps_against_given_tokens(model, B, fmt):
    """30 tokens on the captured step (a block border among them): the cache it
    leaves and every token it chose, against the eager unfused decoder."""
    n, new = 40, 30
    g = MetalLigerGenerator(model)
    ids = _ids(B, n)
    out = g.generate(ids, max_new_tokens=new, kv_cache_dtype=fmt, cuda_graph=True)
    (st,) = g._states.values()
    assert st.graph is not None
    cache = MetalLigerQuantizedCache(model, B, n + new, fmt)
    # the eager loop over the cache parts from the captured steps at a near-tie at most
    eager = g.generate(ids, max_new_tokens=new, kv_cache_dtype=fmt, cuda_graph=False)
    W = model.lm_head.weight.float()

    def near_best(logits, h, took):
        best = logits.argmax(-1)
        gap = (logits.gather(1, best[:, None]) - logits.gather(1, took[:, None]))[:, 0]
        # (and half a step of bf16 each, which the head rounds to)
        room = REL * (W[best] - W[took]).norm(dim=-1) * h.norm(dim=-1) + \
            2.0 ** -8 * 2 * logits.abs().amax(-1)
        return (best == took) | (gap <= room)

    with torch.no_grad():
        h = model.model(input_ids=ids, past_key_values=cache, use_cache=True).last_hidden_state
        cache.seen_tokens = n
        for t in range(n, n + new):
            h = h[:, -1].float()
            logits = h @ W.T
            assert near_best(logits, h, out[:, t]).all(), t
            together = (eager[:, :t] == out[:, :t]).all(1)
            assert (near_best(logits, h, eager[:, t]) | ~together).all(), t
            if t == n + new - 1:
                break
            with _QuantizedAttention(model.model, cache):
                h = model.model(input_ids=out[:, t:t + 1], past_key_values=cache,
                                use_cache=True).last_hidden_state
            cache.seen_tokens += 1
    _check_rows(st.cache, cache, 0, n + new - 1)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("B", [1, 2])
def test_one_fused_step_against_the_values_of_the_cache(model, B, fmt):
    """A step as it is captured: its hidden state against a DynamicCache of the
    dequantised keys and values, what it appends against the unfused step."""
    from transformers.cache_utils import DynamicCache

    n, L = 70, 80
    ids, tok = _ids(B, n), _ids(B, 1, seed=3)
    cache = MetalLigerQuantizedCache(model, B, L, fmt)
    with torch.no_grad():
        model.model(input_ids=ids, past_key_values=cache, use_cache=True)
        cache.seen_tokens = n
        ref = DynamicCache()
        for i in range(cache.num_layers):
            k, v = cache.kv[i].dequantize()
            ref.update(k[:, :, :n].contiguous(), v[:, :, :n].contiguous(), i)
        want = model.model(input_ids=tok, past_key_values=ref, use_cache=True).last_hidden_state
        plain = MetalLigerQuantizedCache(model, B, L, fmt)
        plain.kv = [copy.deepcopy(kv) for kv in cache.kv]
        plain.seen_tokens = n
        with _QuantizedAttention(model.model, plain):
            unfused = model.model(input_ids=tok, past_key_values=plain, use_cache=True).last_hidden_state
        pos = torch.tensor([n], dtype=torch.int64, device=DEV)
        mask = torch.zeros((B, 1, 1, L), dtype=torch.bool, device=DEV)
        mask[..., :n + 1] = True
        updates = []
        update = cache.update
        cache.update = lambda *a, **k: (updates.append(a[2]), update(*a, **k))[1]
        cache.graph_pos = pos
        with _DecodeKernels(model.model, pos, gemv=True, cache=cache), \
                _QuantizedAttention(model.model, cache):
            got = model.model(input_ids=tok, attention_mask=mask, past_key_values=cache,
                              use_cache=True, position_ids=pos.view(1, 1, 1).expand(3, B, 1)
                              ).last_hidden_state
    # whole patched layers append on their own, the others through update()
    assert updates == ([] if model.patched else [0, 1])
    assert (cache._rows is not None) == model.patched
    for other in (want, unfused):
        err = (got.float() - other.float()).norm(dim=-1) / other.float().norm(dim=-1)
        assert (err < REL).all(), err
    _check_rows(cache, plain, n, n + 1)
    # what was there before is there still (the open block's under its new scale)
    _check_rows(cache, plain, 0, n)
    if model.patched:
        # the rows of both layers went through one buffer: the last layer's are in it
        k_row = cache._rows[0].float()
        k = cache.kv[-1].dequantize()[0][:, :, n:n + 1].float()
        step = _step_of_codes(cache.kv[-1].k_codes, cache.kv[-1].k_scale, cache.kv[-1].block)
        assert ((k - k_row).abs() <= step[:, :, n:n + 1, None] * 0.51 + 2.0 ** -8 * k_row.abs()).all()
