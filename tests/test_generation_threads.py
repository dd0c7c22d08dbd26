"""CPU: several threads decode over quantised caches, each with a model of its
own, and a model that one thread decodes with is called from another.  The
caches are stand-ins that answer from the CPU; the threads are kept in step by
barriers, so every interleaving is the same each time."""

import threading

import pytest
import torch

from metal_liger_b200 import generation as G


class _Cache(G.MetalLigerQuantizedCache):
    """Answers update() as the quantised cache does and attends with a value of
    its own."""

    def __init__(self, value):
        self.value = value
        self.pending = None
        self.max_seq_len = 64
        self.served = []

    def update(self, key_states, value_states, layer_idx, cache_kwargs=None):
        self.pending.add(layer_idx)
        return key_states, value_states

    def decode_attention(self, layer_idx, query, scale):
        self.served.append(layer_idx)
        return torch.full_like(query.transpose(1, 2), self.value)


class _Attn(torch.nn.Module):
    is_causal = True
    num_key_value_groups = 1

    def __init__(self, layer_idx):
        super().__init__()
        self.layer_idx = layer_idx


class _Config:
    _attn_implementation = "sdpa"


class _Decoder:
    def __init__(self):
        self.config = _Config()


def _in_threads(*jobs):
    errors = []

    def run(job):
        try:
            job()
        except BaseException as e:  # noqa: BLE001  (handed to the test)
            errors.append(e)

    threads = [threading.Thread(target=run, args=(j,)) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not any(t.is_alive() for t in threads)
    if errors:
        raise errors[0]


def _registered(config):
    from transformers.modeling_utils import ALL_ATTENTION_FUNCTIONS

    return ALL_ATTENTION_FUNCTIONS[config._attn_implementation]


def test_two_threads_decode_over_their_own_caches():
    gate = threading.Barrier(2, timeout=30)
    caches = [_Cache(1.0), _Cache(2.0)]
    got = [None, None]
    q = torch.zeros(1, 2, 1, 8)

    def job(i):
        dec = _Decoder()
        gate.wait()
        with G._QuantizedAttention(dec, caches[i]):
            gate.wait()                            # both are inside
            out = []
            for layer in range(3):
                k, v = caches[i].update(q, q, layer)
                gate.wait()                        # both layers wait for their attention
                out.append(_registered(dec.config)(_Attn(layer), q, k, v, None, scaling=1.0)[0])
                gate.wait()
            got[i] = torch.stack(out)
        assert dec.config._attn_implementation == "sdpa"

    _in_threads(lambda: job(0), lambda: job(1))
    for i in range(2):
        assert (got[i] == caches[i].value).all() and caches[i].served == [0, 1, 2]
    assert G._KV8_CACHE[0] is None


def test_a_shared_config_comes_back_whoever_leaves_first():
    """Two threads on one model, the first in being the first out."""
    dec, gate = _Decoder(), threading.Barrier(2, timeout=30)
    q = torch.zeros(1, 2, 1, 8)
    caches = [_Cache(1.0), _Cache(2.0)]

    def first():
        with G._QuantizedAttention(dec, caches[0]):
            gate.wait()
            gate.wait()
        gate.wait()

    def second():
        gate.wait()
        with G._QuantizedAttention(dec, caches[1]):
            gate.wait()
            gate.wait()                            # the first has left
            k, v = caches[1].update(q, q, 4)
            out, _ = _registered(dec.config)(_Attn(4), q, k, v, None, scaling=1.0)
            assert (out == 2.0).all()

    _in_threads(first, second)
    assert dec.config._attn_implementation == "sdpa" and caches[1].served == [4]


def _tiny(implementation):
    from transformers import Qwen3Config, Qwen3ForCausalLM

    cfg = Qwen3Config(hidden_size=64, intermediate_size=128, num_hidden_layers=2,
                      num_attention_heads=4, num_key_value_heads=2, head_dim=16, vocab_size=50)
    cfg._attn_implementation = implementation
    torch.manual_seed(0)
    return Qwen3ForCausalLM(cfg).eval()


@pytest.mark.parametrize("implementation", ["sdpa", "eager"])
def test_a_plain_forward_while_another_thread_decodes_keeps_its_mask(implementation):
    m = _tiny(implementation)
    ids = torch.randint(0, 50, (2, 6), generator=torch.Generator().manual_seed(1))
    mask = torch.tensor([[0, 0, 1, 1, 1, 1], [1, 1, 1, 1, 1, 1]])
    with torch.no_grad():
        want = [m(ids, attention_mask=mask).logits, m(ids).logits]
    got = []
    gate = threading.Barrier(2, timeout=30)

    def decodes():
        with G._QuantizedAttention(m.model, _Cache(1.0)):
            gate.wait()
            gate.wait()

    def forwards():
        gate.wait()
        with torch.no_grad():
            got.extend([m(ids, attention_mask=mask).logits, m(ids).logits])
        gate.wait()

    _in_threads(decodes, forwards)
    assert m.config._attn_implementation == implementation
    for a, b in zip(want, got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("implementation", ["sdpa", "eager"])
def test_the_step_itself_attends_through_the_cache(implementation):
    """Through transformers' own decoder, whatever its implementation was."""
    m = _tiny(implementation)
    cache = _Cache(0.5)
    # a Cache of two layers for the decoder, answered by the stand-in
    cache.num_layers, cache.batch_size, cache.seen_tokens = 2, 1, 3
    cache.kv = [type("KV", (), {"k_codes": None, "v_codes": None})() for _ in range(2)]
    G.Cache.__init__(cache, layers=[G._QuantizedKVLayer(cache, i) for i in range(2)])
    cache.update = _Cache.update.__get__(cache)
    with torch.no_grad(), G._QuantizedAttention(m.model, cache):
        m.model(input_ids=torch.tensor([[7]]), past_key_values=cache, use_cache=True,
                position_ids=torch.tensor([[3]]))
    assert cache.served == [0, 1]
    assert m.config._attn_implementation == implementation


def test_replays_leave_the_config_alone():
    """Only the steps that run the decoder replace its attention."""
    g = G.MetalLigerGenerator.__new__(G.MetalLigerGenerator)
    seen = []

    class Decoder(torch.nn.Module):
        config = _Config()

    g.decoder = Decoder()

    class State:
        ids = torch.zeros(1, 8, dtype=torch.int64)
        pos, mask = torch.zeros(1, dtype=torch.int64), torch.zeros(1, 1, 1, 8, dtype=torch.bool)
        tok, sampling, uniform = torch.zeros(1, 1, dtype=torch.int64), None, None
        cache = _Cache(1.0)

        class graph:
            @staticmethod
            def replay():
                seen.append((Decoder.config._attn_implementation, G._KV8_CACHE[0]))

    assert g._decode_static(State, 3, 4, None, capture=True) == 7
    assert seen == [("sdpa", None)] * 4


def test_no_mask_is_made_for_the_step(monkeypatch):
    from transformers.masking_utils import ALL_MASK_ATTENTION_FUNCTIONS

    made = ALL_MASK_ATTENTION_FUNCTIONS[G._DECODE_ATTN]
    kw = dict(batch_size=2, q_length=6, kv_length=6, q_offset=0, kv_offset=0,
              attention_mask=torch.tensor([[0, 0, 1, 1, 1, 1], [1] * 6]).bool(), device="cpu",
              allow_is_causal_skip=False)
    want = ALL_MASK_ATTENTION_FUNCTIONS["sdpa"](**kw)
    assert torch.equal(made(**kw), want)
    with G._QuantizedAttention(_Decoder(), _Cache(1.0)):
        assert made(**kw) is None
        other = []
        _in_threads(lambda: other.append(made(**kw)))            # another thread's call
        assert torch.equal(other[0], want)
