"""CPU: refusals, shapes and the fp64 restatement of the 8-bit KV cache and the
sampler.  No GPU work is issued."""

import ctypes
import math

import pytest
import torch

from metal_liger_b200 import _C, generation
from metal_liger_b200.ops.fused_sampling import fused_sample
from metal_liger_b200.ops.quantized_kv import (
    allocate_quantized_kv, quantized_kv_append, quantized_kv_attention)
from oracle import decode as OD


def _cache(**over):
    c = _C.Kv8Cache(16, 16, 16, 16, 16, 16, 0, 1, 2, 2, 128, 64, 64)
    for n, v in over.items():
        setattr(c, n, v)
    return c


STRIDES = (ctypes.c_int64 * 3)(8, 8, 8)


@pytest.mark.parametrize("over,word", [
    (dict(format=2), b"format"), (dict(dtype=0), b"dtype"), (dict(head_dim=96), b"head_dim"),
    (dict(block=48), b"block"), (dict(max_len=100), b"multiple"), (dict(kv_heads=0), b"sizes"),
    (dict(batch=-1), b"sizes"), (dict(batch=70000), b"range"), (dict(k_codes=None), b"null"),
    (dict(v_codes=8), b"aligned"),
])
def test_c_entries_refuse_bad_caches(cuda_lib, over, word):
    c = _cache(**over)
    assert cuda_lib.ml_kv8_append(ctypes.byref(c), 16, STRIDES, 16, STRIDES, 1, 16, 0, None, 0,
                                  None) == 1
    assert word in cuda_lib.ml_last_error()
    assert cuda_lib.ml_kv8_attention(ctypes.byref(c), 16, STRIDES, 4, 1, 16, 0, None, 0, 1.0, 16,
                                     None, 0, None) == 1
    assert word in cuda_lib.ml_last_error()


def test_c_entries_refuse_bad_calls(cuda_lib):
    c = _cache()
    odd = (ctypes.c_int64 * 3)(8, 4, 8)
    ap = lambda **k: cuda_lib.ml_kv8_append(  # noqa: E731
        ctypes.byref(c), k.get("k", 16), k.get("st", STRIDES), 16, STRIDES, k.get("T", 1),
        k.get("start", 16), k.get("ss", 0), None, 0, None)
    at = lambda **k: cuda_lib.ml_kv8_attention(  # noqa: E731
        ctypes.byref(c), k.get("q", 16), k.get("st", STRIDES), k.get("hq", 4), k.get("T", 1),
        k.get("start", 16), k.get("ss", 0), None, 0, 1.0, k.get("out", 16), None, 0, None)
    for kw in (dict(k=None), dict(k=8), dict(st=odd), dict(T=-1), dict(start=None), dict(ss=2)):
        assert ap(**kw) == 1, kw
    for kw in (dict(q=None), dict(q=8), dict(st=odd), dict(T=-1), dict(start=None), dict(ss=2),
               dict(hq=3), dict(hq=0), dict(out=None), dict(out=8)):
        assert at(**kw) == 1, kw
    assert ap(T=0) == 0 and at(T=0) == 0                          # nothing to do
    assert cuda_lib.ml_kv8_append(None, 16, STRIDES, 16, STRIDES, 1, 16, 0, None, 0, None) == 1
    sm = lambda rows, vocab, dt=0, x=16: cuda_lib.ml_sample(  # noqa: E731
        x, vocab, dt, rows, vocab, 16, None, 1.0, None, 0, None, 1.0, None, 0.0, 16, 16, None)
    assert sm(1, 0) == 1 and sm(-1, 5) == 1 and sm(1, 5, dt=9) == 1 and sm(1, 5, x=None) == 1
    assert sm(1, (1 << 20) + 1) == 1 and b"vocabulary" in cuda_lib.ml_last_error()
    assert sm(0, 5) == 0


def test_python_refusals_without_a_gpu():
    x, u = torch.zeros(2, 8), torch.zeros(2)
    for kw in (dict(temperature=-1.0), dict(temperature=math.nan), dict(temperature=math.inf),
               dict(top_k=-1), dict(top_p=1.5), dict(top_p=-0.1), dict(min_p=2.0),
               dict(min_p=math.nan)):
        with pytest.raises(ValueError):
            fused_sample(x, u, **kw)
    with pytest.raises(NotImplementedError):                      # no CPU kernel, no fallback
        fused_sample(x, u)
    for kw in (dict(cache_dtype="int4"), dict(dtype=torch.float32), dict(block=16)):
        with pytest.raises(ValueError):
            allocate_quantized_kv(1, 1, 10, 64, device="cpu", **kw)
    with pytest.raises(ValueError):
        allocate_quantized_kv(1, 1, 10, 80, device="cpu")
    with pytest.raises(ValueError):
        allocate_quantized_kv(0, 1, 10, 64, device="cpu")
    kv = allocate_quantized_kv(1, 1, 10, 64, device="cpu")
    assert kv.max_len == 64 and kv.block == 64
    k = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(NotImplementedError):
        quantized_kv_append(kv, k, k, torch.zeros(1, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="backward"):
        quantized_kv_attention(k.clone().requires_grad_(), kv, torch.zeros(1, dtype=torch.int64))


def test_fakes_on_meta():
    kv = allocate_quantized_kv(2, 3, 100, 128, "fp8", device="meta")
    assert kv.k_codes.shape == (2, 3, 128, 128) and kv.v_scale.shape == (2, 3, 2)
    q = torch.empty(2, 6, 5, 128, dtype=torch.bfloat16, device="meta")
    st = torch.empty(1, dtype=torch.int64, device="meta")
    assert quantized_kv_attention(q, kv, st).shape == (2, 5, 6, 128)
    assert quantized_kv_append(kv, q[:, :3], q[:, :3], st) is None
    ids, logp = fused_sample(torch.empty(4, 9, device="meta"), torch.empty(4, device="meta"))
    assert ids.shape == logp.shape == (4,) and ids.dtype == torch.int64


def test_dequantize_on_the_cpu():
    kv = allocate_quantized_kv(1, 1, 64, 64, "int8", device="cpu")
    kv.k_codes[0, 0, 3, 7] = -100
    kv.k_scale[0, 0, 0] = 0.5
    k, v = kv.dequantize()
    assert k.dtype == torch.bfloat16 and k[0, 0, 3, 7] == -50.0 and torch.count_nonzero(v) == 0


def test_oracle_e4m3_matches_torch():
    # fp32 values: torch's conversion starts from fp32, so anything longer is rounded twice
    x = torch.linspace(-448, 448, 40001)
    x = torch.cat([x, x * 1e-3, x * 1e-5, torch.tensor([17.0, 18.0, 19.0, 2.0 ** -10, 3 * 2.0 ** -10])])
    x = x.double()
    assert torch.equal(OD.e4m3(x), x.float().to(torch.float8_e4m3fn).double())


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_oracle_history_is_independent_of_the_pieces(fmt):
    g = torch.Generator().manual_seed(0)
    x = torch.randn(1, 2, 90, 64, generator=g)
    whole, parts = (OD.History(1, 2, 96, 64, 32, fmt) for _ in range(2))
    whole.append(x, [0], [90])
    for lo, hi in ((0, 1), (1, 33), (33, 64), (64, 90)):
        parts.append(x[:, :, lo:hi], [lo], [hi - lo])
    assert torch.equal(whole.codes, parts.codes) and torch.equal(whole.scale, parts.scale)


def test_oracle_sampler_on_known_rows():
    x = torch.log(torch.tensor([0.1, 0.4, 0.2, 0.3]))
    assert OD.sample_row(x, 0.05, 1.0, 0, 1.0, 0.0)[0] == 0
    assert OD.sample_row(x, 0.49, 1.0, 0, 1.0, 0.0)[0] == 1
    assert OD.sample_row(x, 0.51, 1.0, 0, 1.0, 0.0)[0] == 2
    assert OD.sample_row(x, 0.999, 1.0, 0, 1.0, 0.0)[0] == 3
    assert OD.sample_row(x, 0.5, 1.0, 2, 1.0, 0.0)[2] == [1, 3]
    assert OD.sample_row(x, 0.5, 1.0, 0, 0.5, 0.0)[2] == [1, 3]
    assert OD.sample_row(x, 0.5, 1.0, 0, 1.0, 0.45)[2] == [1, 2, 3]
    assert OD.sample_row(x, 0.5, 0.0, 0, 1.0, 0.0)[:2] == (1, 0.0)


def test_generate_refuses_hidden_positions():
    g = generation.MetalLigerGenerator.__new__(generation.MetalLigerGenerator)
    ids = torch.zeros(2, 4, dtype=torch.int64)
    padded = torch.tensor([[0, 1, 1, 1], [1, 1, 1, 1]])
    for mask in (padded, torch.zeros(2, 1, 4, 4)):
        with pytest.raises(ValueError, match="mask"):
            g.generate(ids, kv_cache_dtype="int8", attention_mask=mask)


@pytest.mark.parametrize("extra,refused", [
    (dict(sliding_window=31), True), (dict(softcap=30.0), True), (dict(s_aux=torch.zeros(2)), True),
    (dict(sliding_window=32, softcap=None), False), (dict(sliding_window=None), False)])
def test_attention_over_the_codes_refuses_what_it_lacks(monkeypatch, extra, refused):
    class Cache:
        pending, max_seq_len = {3}, 32

        def decode_attention(self, layer, query, scale):
            return layer, scale

    class Module:
        layer_idx = 3

    monkeypatch.setattr(generation, "_KV8_CACHE", [Cache()])
    q = torch.zeros(1, 2, 1, 64)
    if refused:
        with pytest.raises(RuntimeError, match=next(iter(extra))):
            generation._kv8_attention_forward(Module(), q, q, q, None, scaling=0.5, **extra)
    else:
        Cache.pending = {3}
        out, _ = generation._kv8_attention_forward(Module(), q, q, q, None, scaling=0.5, **extra)
        assert out == (3, 0.5)
