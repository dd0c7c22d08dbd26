"""Sampling with temperature, top-k, top-p and min-p from given uniform numbers.

One call from the logits to the token: no softmax, sort or filtered copy of
the logits is formed.  The reference's generator divides by the temperature
and draws with torch.multinomial, its ``top_p`` only choosing between greedy
and sampling (generation.py:118-123); this is the sampler that honours it.
"""

import math
from typing import Union

import torch
from torch import Tensor

from metal_liger_b200 import _torch_library as _tl
from metal_liger_b200.ops.quantized_kv import refuse_derivatives


def _split(name: str, x, ok):
    """(tensor, value) of a parameter given as either."""
    if isinstance(x, Tensor):
        return x, 0
    if not ok(x):
        raise ValueError(f"fused_sample: {name}={x!r}")
    return None, x


def fused_sample(logits: Tensor, uniform: Tensor, temperature: Union[float, Tensor] = 1.0,
                 top_k: Union[int, Tensor] = 0, top_p: Union[float, Tensor] = 1.0,
                 min_p: Union[float, Tensor] = 0.0):
    """(ids int64 [B], logprobs fp32 [B]) of one token per row of logits [B, V].

    ``uniform`` [B] in [0, 1) is the randomness: the same numbers give the same
    tokens, whatever the batch.  Tokens are ordered by logit, largest first,
    equal logits by index.  Of the first ``top_k`` (0: all), the shortest prefix
    that holds ``top_p`` of their probability is kept, and of that the tokens
    with at least ``min_p`` times the largest probability, never fewer than one;
    the token is the first in vocabulary order at which the running probability
    exceeds ``uniform``, and its logprob is taken in the kept, renormalised
    distribution.  ``temperature`` 0 takes the largest logit (logprob 0).

    Each parameter is a number or a [B] tensor of one per row (there, a
    temperature <= 0 or NaN is greedy, top_k <= 0, top_p >= 1 and min_p <= 0
    are off).  Logits are bf16, fp16 or fp32 with up to 2^20 tokens; NaN and
    -inf are never taken, and a row of nothing else gives id -1, logprob
    -inf."""
    t, tv = _split("temperature", temperature, lambda x: 0.0 <= x < math.inf)
    k, kv = _split("top_k", top_k, lambda x: 0 <= x < 2 ** 63)  # an int64
    p, pv = _split("top_p", top_p, lambda x: 0.0 <= x <= 1.0)
    m, mv = _split("min_p", min_p, lambda x: 0.0 <= x <= 1.0)
    refuse_derivatives("fused_sample", logits, uniform, t, k, p, m)
    eager = logits.is_cuda and type(logits) is Tensor and not torch.compiler.is_compiling()
    op = _tl.sample_cuda if eager else torch.ops.metal_liger.sample
    return op(logits, uniform, t, tv, k, kv, p, pv, m, mv)
