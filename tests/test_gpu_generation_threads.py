"""Two threads generate over 8-bit KV caches at the same time, each with its own
model, and get what they get alone."""

import threading

import pytest
import torch

from metal_liger_b200.generation import MetalLigerGenerator
from test_gpu_generation import DEV, _model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("graph", [False, True], ids=["eager", "cuda_graph"])
def test_two_threads_generate_what_each_does_alone(graph):
    ids = torch.randint(0, 1000, (2, 24), generator=torch.Generator().manual_seed(0)).to(DEV)
    kinds = ("int8", "fp8")
    gens = [MetalLigerGenerator(_model(seed=21 + i)) for i in range(2)]
    gen = lambda i: gens[i].generate(ids, max_new_tokens=24, kv_cache_dtype=kinds[i],  # noqa: E731
                                     cuda_graph=graph)
    alone = [gen(i) for i in range(2)]            # captured here, one after the other
    torch.cuda.synchronize()
    assert not torch.equal(alone[0], alone[1])
    gate = threading.Barrier(2, timeout=60)
    got, errors = [[], []], []

    def run(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(4):
                    gate.wait()
                    got[i].append(gen(i))
                torch.cuda.current_stream().synchronize()
        except BaseException as e:  # noqa: BLE001
            errors.append(e)
            gate.abort()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    assert not any(t.is_alive() for t in threads)
    if errors:
        raise errors[0]
    for i in range(2):
        assert len(got[i]) == 4
        for out in got[i]:
            assert torch.equal(out, alone[i])
        assert gens[i].decoder.config._attn_implementation == "sdpa"
