"""A KV cache held in 8 bits: its buffers, the append and the attention over it.

No counterpart in the reference, whose static cache keeps the model's dtype
(generation.py:18-66).  One layer's cache is a ``QuantizedKV`` of six device
buffers: int8 or e4m3 codes for K and V, one fp32 scale for each block of
positions and kv head, and the unquantised rows of the last two blocks (the
"tail"), so that a block that is written on is quantised from its values
themselves:

    a = max |x| over the block,   scale = a / qmax,   code = round(x * qmax / a)

with qmax 127 (int8) or 448 (e4m3), rounded half to even.  It halves the bytes
a decode step reads per position and the memory per sequence.

    kv = allocate_quantized_kv(batch, kv_heads, max_len, head_dim, "int8")
    quantized_kv_append(kv, k, v, start)              # in place, start on the device
    out = quantized_kv_attention(q, kv, start)        # [B, T, Hq, D]

``start`` (int64, one value or one per sequence) is the number of positions a
sequence held before the step, the same for the append and the attention;
neither advances it.  It stays on the device, so a captured CUDA graph of the
step follows it.
"""

from typing import NamedTuple, Optional

import torch
from torch import Tensor
from torch.autograd import forward_ad

from metal_liger_b200 import _torch_library as _tl

CACHE_DTYPES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
DEFAULT_BLOCK = 64


class _Buffers(NamedTuple):
    k_codes: Tensor   # [B, Hkv, L, D] int8 or float8_e4m3fn
    k_scale: Tensor   # [B, Hkv, L / block] float32
    k_tail: Tensor    # [B, Hkv, 2, block, D] bf16 or fp16
    v_codes: Tensor
    v_scale: Tensor
    v_tail: Tensor


class QuantizedKV(_Buffers):
    """One layer's cache buffers.

    ``held`` (int32 [2, B, Hkv, 2]; K, V): which block each slot of the tails
    has, negative where that is not known.  ``allocate_quantized_kv`` makes it; a
    cache put together from buffers (``_replace`` among them) has none, and its
    appends take the tails for the rows of whatever block they continue.  Whoever
    copies buffers into a cache that was in use copies ``held`` too, or fills it with
    -1."""

    held: Optional[Tensor]

    def __new__(cls, *args, **kwargs):
        self = super().__new__(cls, *args, **kwargs)
        self.held = None  # (an attribute of each instance, as torch.compile guards it)
        return self

    @classmethod
    def _make(cls, iterable):
        return cls(*iterable)

    @property
    def max_len(self) -> int:
        return self.k_codes.shape[2]

    @property
    def block(self) -> int:
        return self.k_tail.shape[3]

    def dequantize(self):
        """(K, V) [B, Hkv, L, D] in the tails' dtype: code * scale, rounded once."""
        return tuple(
            (c.float().view(*s.shape, -1) * s[..., None]).view(c.shape).to(t.dtype)
            for c, s, t in ((self.k_codes, self.k_scale, self.k_tail),
                            (self.v_codes, self.v_scale, self.v_tail)))


def allocate_quantized_kv(batch: int, kv_heads: int, max_len: int, head_dim: int,
                          cache_dtype: str = "int8", dtype: torch.dtype = torch.bfloat16,
                          block: int = DEFAULT_BLOCK, device="cuda") -> QuantizedKV:
    """Zeroed buffers for ``max_len`` positions (rounded up to whole blocks).

    ``cache_dtype`` "int8" or "fp8" (e4m3), ``dtype`` (bf16 or fp16) that of the
    rows appended and of the queries, ``head_dim`` 64, 128 or 256, ``block`` 32,
    64 or 128 positions per scale."""
    if cache_dtype not in CACHE_DTYPES:
        raise ValueError(f"cache_dtype {cache_dtype!r}: one of {sorted(CACHE_DTYPES)}")
    if dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"dtype {dtype}: bfloat16 or float16")
    if head_dim not in (64, 128, 256) or block not in (32, 64, 128):
        raise ValueError(f"head_dim {head_dim} (64, 128 or 256), block {block} (32, 64 or 128)")
    if batch < 1 or kv_heads < 1 or max_len < 1:
        raise ValueError("batch, kv_heads and max_len are at least 1")
    length = -(-max_len // block) * block
    shape = (batch, kv_heads)

    def half():
        return (torch.zeros((*shape, length, head_dim), dtype=torch.int8,
                            device=device).view(CACHE_DTYPES[cache_dtype]),
                torch.zeros((*shape, length // block), dtype=torch.float32, device=device),
                torch.zeros((*shape, 2, block, head_dim), dtype=dtype, device=device))

    kv = QuantizedKV(*half(), *half())
    kv.held = torch.full((2, *shape, 2), -1, dtype=torch.int32, device=device)
    return kv


def refuse_derivatives(name: str, *tensors: Optional[Tensor]) -> None:
    """Raises where a derivative through ``tensors`` is asked for, in reverse mode
    (one requires grad) or forward mode (one is a dual tensor): it would be
    dropped without a word."""
    # (outside any forward-mode level, -1, there are no dual tensors to look for)
    forward = getattr(forward_ad, "_current_level", 0) >= 0
    reverse = torch.is_grad_enabled()
    for t in tensors:
        if t is None:
            continue
        if reverse and t.requires_grad:
            raise RuntimeError(f"{name} has no backward: call it under torch.no_grad()")
        if forward and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{name} has no forward-mode derivative: call it on the primals")


def _eager(t: Tensor) -> bool:
    return t.is_cuda and type(t) is Tensor and not torch.compiler.is_compiling()


def quantized_kv_append(kv: QuantizedKV, k: Tensor, v: Tensor, start: Tensor,
                        counts: Optional[Tensor] = None) -> None:
    """Write k, v [B, Hkv, T, D] (any strides) at positions ``start`` + t, in place.

    ``counts`` (int64): how many of the T rows are real in each sequence, the
    others being padding.  Blocks that get a row are requantised whole; rows
    past ``max_len`` are dropped, as are those of a sequence whose start is
    negative; the codes of positions past the last new one stay as they were.

    ``start`` may go back (a drafted continuation rejected, a new prompt at 0).
    From a block border, and inside a block whose unquantised rows the tail
    still has, the cache is that of one call with all the rows.  The tail has
    the last two blocks of each append, odd and even ones in a slot of their own:
    a sequence that only goes forward, or goes back once into the block it ended
    in or the one before, always finds its rows there.  After a further step
    back the slot may have a later block: then the older rows are what their
    codes stand for, rounded to the rows' dtype, which leaves their codes as they
    are while the block's largest value stands.  (A cache without ``kv.held``
    cannot tell, and needs ``start`` to be one of the others.)"""
    refuse_derivatives("quantized_kv_append", k, v)
    op = _tl.kv8_append_cuda if _eager(k) else torch.ops.metal_liger.kv8_append
    op(k, v, start, counts, kv.k_codes, kv.v_codes, kv.k_scale, kv.v_scale, kv.k_tail, kv.v_tail,
       kv.held)


def quantized_kv_attention(q: Tensor, kv: QuantizedKV, start: Tensor,
                           counts: Optional[Tensor] = None,
                           scale: Optional[float] = None) -> Tensor:
    """softmax(scale * q k^T) v of q [B, Hq, T, D] over the cache, [B, T, Hq, D].

    Query t of a sequence sees positions j <= ``start`` + t, so the call follows
    the append of the same tokens; Hq is a multiple of the cache's kv heads.
    Rows t >= ``counts`` and rows that see nothing are zeros.  ``scale``
    defaults to D ** -0.5."""
    refuse_derivatives("quantized_kv_attention", q)
    op = _tl.kv8_attention_cuda if _eager(q) else torch.ops.metal_liger.kv8_attention
    return op(q, start, counts, kv.k_codes, kv.v_codes, kv.k_scale, kv.v_scale, kv.k_tail,
              kv.v_tail, q.shape[-1] ** -0.5 if scale is None else scale)
