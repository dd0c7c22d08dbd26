"""Attention over the 8-bit cache where one position takes nearly all the weight
and has no value to speak of (an attention sink): the output is what the many
small weights bring.

The bound per output element is the one of test_gpu_quantized_kv.py, but for
the weights below fp16's normal range.  The weights enter the second product
in fp16 with the largest at 2^15, as w 2^(15) with w <= 1 the weight against
the row's largest p_j * (V block's scale), so

  w >= 2^-29   half a step, 2^-11 of itself (in the 2^-11 A term), and
  w <  2^-29   half of fp16's smallest step, 2^-25 2^-15 = 2^-40, absolute:
               n 2^-40 max|v| over n positions.

Held with the largest at 1, the last term would be n 2^-25 max|v|, and the tails
below would come out as zero or short by several per cent.
"""

import pytest
import torch

from metal_liger_b200.ops.quantized_kv import (
    allocate_quantized_kv, quantized_kv_append, quantized_kv_attention)
from oracle import decode as OD

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _bound(out, mag, dots, vmax, n, D, dtype):
    u = torch.finfo(dtype).eps / 2
    return (u * out.abs() + 2.0 ** -11 * mag + n * 2.0 ** -40 * vmax
            + 2 * (D + 16) * 2.0 ** -24 * dots[..., None] * mag + (n + 64) * 2.0 ** -23 * mag)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("n,share,B,Hq,Hkv,D,block,T,dtype,sink", [
    (300, 0.9999, 1, 4, 2, 64, 64, 1, torch.float16, 0),      # a CTA to a segment
    (300, 0.9999, 2, 4, 2, 128, 32, 1, torch.bfloat16, 299),
    (16384, 0.9999, 8, 8, 8, 64, 64, 1, torch.bfloat16, 0),   # many tiles to a warp
    (8192, 0.9999, 1, 8, 2, 128, 64, 1, torch.float16, 0),    # joined across CTAs
    (8192, 0.9999, 3, 2, 2, 256, 128, 2, torch.bfloat16, 4100),
    (2400, 0.9999, 16, 128, 8, 64, 64, 1, torch.float16, 0),  # sixteen query rows to a tile
])
def test_attention_with_a_sink(fmt, n, share, B, Hq, Hkv, D, block, T, dtype, sink):
    gen = torch.Generator().manual_seed(n + D + sink)
    kv = allocate_quantized_kv(B, Hkv, n, D, fmt, dtype, block)
    # key 0 of the sink against query 0 gives the score that makes its share; the
    # other keys are noise in the other dimensions, of which quantisation leaves
    # what it leaves: the oracle works on the codes
    gap = torch.log(torch.tensor(share / (1 - share) * (n - 1), dtype=torch.float64)).item()
    amp = (gap * D ** 0.5) ** 0.5
    k = torch.randn((B, Hkv, n, D), generator=gen) * 0.3
    k[..., 0] = 0
    k[:, :, sink] = 0
    k[:, :, sink, 0] = amp
    v = torch.rand((B, Hkv, n, D), generator=gen) + 0.5       # of one sign
    v[:, :, sink] = 0
    q = torch.randn((B, Hq, T, D), generator=gen) * 0.3
    q[..., 0] = amp
    k, v, q = (x.to(dtype) for x in (k, v, q))
    quantized_kv_append(kv, k.to(DEV), v.to(DEV), torch.zeros(1, dtype=torch.int64, device=DEV))
    start = n - T
    st = torch.tensor([start], dtype=torch.int64, device=DEV)
    out = quantized_kv_attention(q.to(DEV), kv, st)
    ref, mag, dots = OD.attention(q, kv.k_codes.cpu().double(), kv.k_scale.cpu(),
                                  kv.v_codes.cpu().double(), kv.v_scale.cpu(), block, [start] * B,
                                  [T] * B, D ** -0.5)
    assert ref.abs().max() < 0.02 and (ref > 0).all()         # the sink has the weight
    vmax = kv.v_scale.amax().item() * OD.QMAX[fmt]
    err = (out.cpu().double() - ref).abs()
    tol = _bound(ref, mag, dots, vmax, n, D, dtype)
    assert (err <= tol).all(), f"worst {(err / tol).max().item():.2f} x the bound, " \
                               f"{(err / ref).max().item():.1e} of the output"
