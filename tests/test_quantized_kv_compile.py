"""CPU: torch.compile traces the 8-bit cache's operators as one graph, and the
append takes the record of the tail's blocks along.  In a process of its own: the
suite runs with dynamo off.  Only traced, not run."""

import os
import subprocess
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent

PROGRAM = """
import torch
from metal_liger_b200 import (QuantizedKV, allocate_quantized_kv, quantized_kv_append,
                              quantized_kv_attention)

kv = allocate_quantized_kv(1, 1, 64, 64, device="cpu")
k, start = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int64)


def step(kv, k, start):
    quantized_kv_append(kv, k, k, start)
    return quantized_kv_attention(k, kv, start)


def closed_over(k, start):
    return step(kv, k, start)


def from_buffers(buffers, k, start):
    return step(QuantizedKV(**buffers), k, start)


def replaced(kv, k, start):
    return step(kv._replace(k_tail=kv.k_tail + 0), k, start)


class Traced(Exception):
    pass


def backend(graph, inputs):
    calls = {str(n.target): n for n in graph.graph.nodes if n.op == "call_function"}
    append = calls["metal_liger.kv8_append"]
    print(len(append.all_input_nodes), "metal_liger.kv8_attention" in calls)

    def run(*args):
        raise Traced

    return run


for f, args in ((step, (kv, k, start)), (closed_over, (k, start)),
                (from_buffers, (kv._asdict(), k, start)), (replaced, (kv, k, start))):
    try:
        torch.compile(f, backend=backend, fullgraph=True)(*args)
    except Traced:
        pass
"""


def test_compile_traces_append_and_attention():
    env = dict(os.environ, TORCHDYNAMO_DISABLE="0", PYTHONPATH=str(ROOT))
    r = subprocess.run([sys.executable, "-c", PROGRAM], env=env, capture_output=True, text=True,
                       timeout=600)
    assert r.returncode == 0, r.stderr[-2000:]
    # k (for v too), start, six buffers and, where there is one, the record
    assert r.stdout.split() == ["9", "True"] * 2 + ["8", "True"] * 2, r.stdout
