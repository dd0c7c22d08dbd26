"""CPU: the record of which block each tail slot of the 8-bit cache has, as it
goes with a cache and into the call.  No GPU work is issued."""

import copy
import ctypes
import pickle

import pytest
import torch

from metal_liger_b200 import _C
from metal_liger_b200.ops.quantized_kv import QuantizedKV, allocate_quantized_kv, quantized_kv_append

NAMES = ("k_codes", "k_scale", "k_tail", "v_codes", "v_scale", "v_tail")


def test_held_goes_with_the_cache_and_not_with_its_buffers():
    kv = allocate_quantized_kv(2, 3, 100, 64, device="cpu")
    assert kv.held.shape == (2, 2, 3, 2) and kv.held.dtype == torch.int32
    assert (kv.held == -1).all()
    assert kv._fields == NAMES and tuple(kv._asdict()) == NAMES and len(kv) == 6
    kv.held[1, 0, 2, 1] = 5
    for twin in (copy.deepcopy(kv), pickle.loads(pickle.dumps(kv))):
        assert torch.equal(twin.held, kv.held) and twin.held is not kv.held
        assert type(twin) is QuantizedKV and twin.block == 64
    assert copy.copy(kv).held is kv.held
    for loose in (QuantizedKV(*kv), QuantizedKV(**kv._asdict()), kv._replace(k_tail=kv.k_tail.clone())):
        assert loose.held is None and loose.max_len == 128


def test_append_passes_held_on(monkeypatch):
    from metal_liger_b200.ops import quantized_kv as mod

    seen = []
    monkeypatch.setattr(mod, "_eager", lambda t: True)
    monkeypatch.setattr(mod._tl, "kv8_append_cuda", lambda *a: seen.append(a[-1]))
    kv = allocate_quantized_kv(1, 1, 64, 64, device="cpu")
    k, st = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int64)
    quantized_kv_append(kv, k, k, st)
    quantized_kv_append(QuantizedKV(*kv), k, k, st)
    assert seen[0] is kv.held and seen[1] is None


def test_append_on_meta():
    kv = allocate_quantized_kv(2, 3, 100, 128, "fp8", device="meta")
    k = torch.empty(2, 3, 5, 128, dtype=torch.bfloat16, device="meta")
    assert quantized_kv_append(kv, k, k, torch.empty(1, dtype=torch.int64, device="meta")) is None


@pytest.mark.parametrize("k_held,v_held", [(16, None), (None, 16), (16, 20), (20, 16)])
def test_c_entry_refuses_half_or_misaligned_records(cuda_lib, k_held, v_held):
    strides = (ctypes.c_int64 * 3)(8, 8, 8)
    c = _C.Kv8Cache(16, 16, 16, 16, 16, 16, 0, 1, 2, 2, 128, 64, 64, k_held, v_held)
    assert cuda_lib.ml_kv8_append(ctypes.byref(c), 16, strides, 16, strides, 1, 16, 0, None, 0,
                                  None) == 1
    assert b"held" in cuda_lib.ml_last_error()
