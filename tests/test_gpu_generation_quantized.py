"""The generator over an 8-bit KV cache and with the fused sampler, on the GPU:
cache, attention and sampling together, as generate() runs them."""

import copy

import pytest
import torch

from metal_liger_b200.generation import (
    MetalLigerGenerator, MetalLigerQuantizedCache, _QuantizedAttention, patch_generator)
from metal_liger_b200.patch import apply_metal_liger_to_qwen3vl, restore_attention_rope
from oracle import generation as OG
from test_gpu_generation import DEV, _model, _same_or_near_tie

pytestmark = pytest.mark.gpu


def _ids(B, n, seed=0):
    return torch.randint(0, 1000, (B, n), generator=torch.Generator().manual_seed(seed)).to(DEV)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_decode_steps_over_the_quantized_cache(fmt):
    """Three decode steps through transformers' decoder over the quantised cache
    equal the same steps over a DynamicCache that holds the dequantised keys
    and values, in the decoder's bf16 (two layers, each rounding a few times:
    2e-2 of the hidden states' norm)."""
    from transformers.cache_utils import DynamicCache

    m = _model(seed=5)
    ids = _ids(2, 70)
    cache = MetalLigerQuantizedCache(m, 2, 80, fmt)
    with torch.no_grad():
        first = m.model(input_ids=ids, past_key_values=cache, use_cache=True).last_hidden_state
        plain = m.model(input_ids=ids, use_cache=False).last_hidden_state
        assert torch.equal(first, plain)            # the prompt attends to its own rows
        cache.seen_tokens += 70
        for step in range(3):
            ref = DynamicCache()
            for i in range(cache.num_layers):
                k, v = cache.kv[i].dequantize()
                n = cache.seen_tokens
                ref.update(k[:, :, :n].contiguous(), v[:, :, :n].contiguous(), i)
            tok = _ids(2, 1, seed=step)
            want = m.model(input_ids=tok, past_key_values=ref, use_cache=True).last_hidden_state
            with _QuantizedAttention(m.model, cache):
                got = m.model(input_ids=tok, past_key_values=cache, use_cache=True).last_hidden_state
            cache.seen_tokens += 1
            # the new token's own row is quantised in one and not in the other:
            # a further int8 / e4m3 half step of one of 70 positions
            err = (got.float() - want.float()).norm() / want.float().norm()
            assert err < 2e-2, (step, err.item())
    # outside the context the cache still answers update(), dequantised
    with torch.no_grad():
        ref = DynamicCache()
        for i in range(cache.num_layers):
            k, v = cache.kv[i].dequantize()
            ref.update(k[:, :, :73].contiguous(), v[:, :, :73].contiguous(), i)
        tok = _ids(2, 1, seed=9)
        want = m.model(input_ids=tok, past_key_values=ref, use_cache=True).last_hidden_state
        got = m.model(input_ids=tok, past_key_values=cache, use_cache=True).last_hidden_state
        assert (got.float() - want.float()).norm() / want.float().norm() < 2e-2


@pytest.mark.parametrize("patched", [False, True], ids=["plain", "patched"])
@pytest.mark.parametrize("B", [1, 3])
def test_generate_with_a_quantized_cache(patched, B):
    """Prompt and first token as without; a second call on the kept state gives
    what a fresh generator gives; the kept graph does not disturb the bf16
    one's."""
    m = _model(seed=7)
    if patched:  # whole decoder layers fused at batch 1
        apply_metal_liger_to_qwen3vl(m, fuse_lora=False, fuse_qk_norm=True,
                                     fuse_rope_in_attention=True)
    try:
        g = MetalLigerGenerator(m)
        ids, other = _ids(B, 40), _ids(B, 40, seed=1)
        plain = g.generate(ids, max_new_tokens=30)
        a = g.generate(ids, max_new_tokens=30, kv_cache_dtype="int8")
        assert a.shape == plain.shape and torch.equal(a[:, :41], plain[:, :41])
        b = g.generate(other, max_new_tokens=30, kv_cache_dtype="int8")
        assert len(g._states) == 2
        assert torch.equal(a, g.generate(ids, max_new_tokens=30, kv_cache_dtype="int8"))
        assert torch.equal(plain, g.generate(ids, max_new_tokens=30))
        fresh = MetalLigerGenerator(m)
        assert torch.equal(b, fresh.generate(other, max_new_tokens=30, kv_cache_dtype="int8"))
        # the eager loop over the cache, and a cache in e4m3
        e = g.generate(ids, max_new_tokens=6, kv_cache_dtype="int8", cuda_graph=False)
        assert e.shape == (B, 46) and torch.equal(e[:, :41], plain[:, :41])
        f = g.generate(ids, max_new_tokens=30, kv_cache_dtype="fp8")
        assert f.shape == plain.shape and torch.equal(f[:, :41], plain[:, :41])
        assert m.model.config._attn_implementation == "sdpa"
    finally:
        if patched:
            restore_attention_rope(m)


@pytest.mark.parametrize("kv", [None, "int8"])
@pytest.mark.parametrize("graph", [False, True])
def test_fused_sampling_in_generate(kv, graph):
    m = _model(seed=8)
    g = MetalLigerGenerator(m)
    ids = _ids(2, 12)

    def go(seed, **kw):
        gen = torch.Generator(device=DEV).manual_seed(seed)
        return g.generate(ids, max_new_tokens=20, kv_cache_dtype=kv, cuda_graph=graph,
                          generator=gen, **kw)

    a = go(1, temperature=1.5, top_p=0.95, min_p=0.01)
    assert a.shape == (2, 32) and torch.equal(a[:, :12], ids)
    assert torch.equal(a, go(1, temperature=1.5, top_p=0.95, min_p=0.01))
    assert not torch.equal(a, go(2, temperature=1.5, top_p=0.95, min_p=0.01))
    # the settings are the call's, not the captured step's
    greedy = g.generate(ids, max_new_tokens=20, kv_cache_dtype=kv, cuda_graph=graph)
    one = go(3, temperature=1.5, top_k=1)
    if kv is None:
        _same_or_near_tie(m, one, greedy)
    assert torch.equal(one[:, 12], greedy[:, 12])
    cold = go(4, temperature=1e-4, fused_sampling=True)
    if kv is None:
        _same_or_near_tie(m, cold, greedy)
    assert torch.equal(a, go(1, temperature=1.5, top_p=0.95, min_p=0.01))
    # temperature 0 stays the greedy path
    assert torch.equal(greedy, go(5, temperature=0.0, top_k=50))


def test_fused_sampling_follows_top_p_where_the_reference_rule_does_not():
    """With top_p next to 0 the fused sampler takes the largest logit at any
    temperature; the reference's rule ignores top_p once it samples."""
    m = _model(seed=9)
    ids = _ids(1, 8)
    patch_generator(m)
    ref = OG.generate(m, ids, max_new_tokens=16)
    out = m.generate(ids, max_new_tokens=16, temperature=3.0, top_p=1e-6, fused_sampling=True)
    _same_or_near_tie(m, out, ref)


def test_eos_stops_and_refusals():
    m = _model(seed=10)
    g = MetalLigerGenerator(m)
    ids = _ids(1, 9)
    full = g.generate(ids, max_new_tokens=24, kv_cache_dtype="int8")
    eos = int(full[0, 9 + 7])
    first = int((full[0, 9:] == eos).nonzero()[0]) + 9
    out = g.generate(ids, max_new_tokens=24, kv_cache_dtype="int8", eos_token_id=eos)
    assert torch.equal(out, full[:, :first + 1])
    with pytest.raises(ValueError):
        g.generate(ids, kv_cache_dtype="int4")
    for kw in (dict(top_k=-1), dict(min_p=1.5), dict(temperature=-1.0, fused_sampling=True),
               dict(top_p=1.2, fused_sampling=True)):
        with pytest.raises(ValueError):
            g.generate(ids, **kw)
    # too long for the cache
    cache = MetalLigerQuantizedCache(m, 1, 10)
    with pytest.raises(RuntimeError, match="max_seq_len"), torch.no_grad():
        m.model(input_ids=_ids(1, 11), past_key_values=cache, use_cache=True)
    # a decoder that does not attend through the interface
    m2 = copy.deepcopy(m)
    cache = MetalLigerQuantizedCache(m2, 1, 64)
    with torch.no_grad():
        m2.model(input_ids=ids, past_key_values=cache, use_cache=True)
    cache.seen_tokens = 9
    k = torch.zeros(1, 2, 1, 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError, match="attention interface"):
        with _QuantizedAttention(m2.model, cache):
            cache.update(k, k, 1)
    assert m2.model.config._attn_implementation == "sdpa"


@pytest.mark.parametrize("new", [0, 1])
def test_fused_sampling_of_no_and_one_token(new):
    g = MetalLigerGenerator(_model(seed=12))
    ids = _ids(2, 6)
    out = g.generate(ids, max_new_tokens=new, kv_cache_dtype="int8", top_k=1)
    assert torch.equal(out, g.generate(ids, max_new_tokens=new))
    padded = torch.ones_like(ids)
    assert torch.equal(out, g.generate(ids, max_new_tokens=new, kv_cache_dtype="int8", top_k=1,
                                       attention_mask=padded))
