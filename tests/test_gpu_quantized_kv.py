"""The KV cache held in 8 bits on the GPU: append and attention against the
fp64 restatement (oracle/decode.py).

The append is exact: each code is the formula's in exact arithmetic, the scale
one fp32 division, the tails copies, so everything is compared bit for bit.

The attention's bound per output element (derived, u = half a step of the
output type, A = sum_j p_j |v_j|, S = the largest sum_d |q_d k_d| scale):
  u |o|                      the output's rounding
  2^-11 A                    a probability held in fp16 (half a step, relative)
  n 2^-25 max|v|             a probability below fp16's normal range (absolute)
  2 (D + 16) 2^-24 S A       fp32 scores summed in any order, scale and exponent
                             products, entering numerator and denominator
  (n + 64) 2^-23 A           fp32 sums of numerator and denominator, exp (2 ulp)
"""

import pytest
import torch

import metal_liger_b200 as ml
from metal_liger_b200.ops.quantized_kv import (
    CACHE_DTYPES, allocate_quantized_kv, quantized_kv_append, quantized_kv_attention)
from oracle import decode as OD

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _rows(gen, *shape, dtype):
    x = torch.randn(shape, generator=gen)
    return (x * torch.where(torch.rand(shape[-1], generator=gen) < 0.1, 5.0, 1.0)).to(dtype)


def _check_cache(kv, hist_k, hist_v, written):
    """Codes and scales of the positions [0, written[b]) bit for bit."""
    for codes, scale, hist in ((kv.k_codes, kv.k_scale, hist_k), (kv.v_codes, kv.v_scale, hist_v)):
        c, s = codes.cpu().double(), scale.cpu()
        for b, n in enumerate(written):
            assert torch.equal(c[b, :, :n], hist.codes[b, :, :n])
            nb = -(-n // hist.block)
            want = hist.scale[b, :, :nb].float()
            got = s[b, :, :nb]
            same = (got == want) | (got.isnan() & want.isnan())
            # the fp64 quotient rounded to fp32 is the fp32 quotient, as its operands are short
            assert same.all()
            assert torch.count_nonzero(c[b, :, n:]) == 0, "positions past the last row changed"


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,H,L,D,block,steps", [
    (1, 1, 64, 64, 64, [(0, 1), (1, 1), (2, 3)]),
    (2, 3, 256, 128, 64, [(0, 63), (63, 1), (64, 1), (65, 130), (195, 61)]),
    (3, 2, 200, 64, 32, [(0, 31), (31, 2), (33, 100), (133, 1), (134, 90)]),   # runs past max_len
    (2, 2, 640, 256, 128, [(0, 200), (200, 440)]),
    (1, 8, 1024, 128, 32, [(0, 7), (7, 1000), (1007, 17)]),
])
def test_append_in_pieces_equals_the_definition(fmt, dtype, B, H, L, D, block, steps):
    gen = torch.Generator().manual_seed(L * 3 + D + block)
    kv = allocate_quantized_kv(B, H, L, D, fmt, dtype, block)
    Lr = kv.max_len
    hk = OD.History(B, H, Lr, D, block, fmt)
    hv = OD.History(B, H, Lr, D, block, fmt)
    for start, T in steps:
        k = _rows(gen, B, H, T, D, dtype=dtype)
        v = _rows(gen, B, T, H, D, dtype=dtype).transpose(1, 2)
        st = torch.full((1,), start, dtype=torch.int64, device=DEV)
        # v as a projection leaves it: strided [B, T, H, D]
        quantized_kv_append(kv, k.to(DEV), v.transpose(1, 2).to(DEV).transpose(1, 2), st)
        hk.append(k, [start] * B, [T] * B)
        hv.append(v, [start] * B, [T] * B)
        _check_cache(kv, hk, hv, [min(Lr, start + T)] * B)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_append_ragged_starts_counts_and_rows_left_alone(fmt):
    gen = torch.Generator().manual_seed(5)
    B, H, L, D, block, T = 7, 2, 256, 128, 64, 70
    kv = allocate_quantized_kv(B, H, L, D, fmt, torch.bfloat16, block)
    first = [0, 5, 64, 127, 200, 256, 31]
    hk, hv = (OD.History(B, H, L, D, block, fmt) for _ in range(2))
    k0, v0 = (_rows(gen, B, H, L, D, dtype=torch.bfloat16) for _ in range(2))
    n0 = torch.tensor(first, device=DEV)
    quantized_kv_append(kv, k0.to(DEV), v0.to(DEV), torch.zeros(B, dtype=torch.int64, device=DEV), n0)
    hk.append(k0, [0] * B, first)
    hv.append(v0, [0] * B, first)
    _check_cache(kv, hk, hv, first)
    # sequence 2 has no row, 3 is started at a negative position, 5 is full
    counts = [70, 1, 0, 9, 70, 3, 64]
    starts = [0, 5, 64, -1, 200, 256, 31]
    k1, v1 = (_rows(gen, B, H, T, D, dtype=torch.bfloat16) for _ in range(2))
    quantized_kv_append(kv, k1.to(DEV), v1.to(DEV), torch.tensor(starts, device=DEV),
                        torch.tensor(counts, device=DEV))
    hk.append(k1, starts, counts)
    hv.append(v1, starts, counts)
    end = [max(f, min(L, s + c)) for f, s, c in zip(first, starts, counts)]
    _check_cache(kv, hk, hv, end)


def test_append_taken_back_and_appended_again():
    """A drafted continuation is rejected: the same positions get other rows,
    across a block border, twice."""
    gen = torch.Generator().manual_seed(6)
    B, H, L, D, block = 2, 2, 256, 64, 64
    kv = allocate_quantized_kv(B, H, L, D, "int8", torch.float16, block)
    hk, hv = (OD.History(B, H, L, D, block, "int8") for _ in range(2))
    end = 0
    for start, T in [(0, 60), (60, 8), (61, 8), (63, 1), (64, 5), (66, 62), (125, 9), (130, 3)]:
        k, v = (_rows(gen, B, H, T, D, dtype=torch.float16) for _ in range(2))
        quantized_kv_append(kv, k.to(DEV), v.to(DEV), torch.tensor([start], device=DEV))
        hk.append(k, [start] * B, [T] * B)
        hv.append(v, [start] * B, [T] * B)
        end = start + T
        c = kv.k_codes.cpu().double()
        assert torch.equal(c[:, :, :end], hk.codes[:, :, :end])
        assert torch.equal(kv.v_codes.cpu().double()[:, :, :end], hv.codes[:, :, :end])
        nb = -(-end // block)
        assert torch.equal(kv.k_scale.cpu()[:, :, :nb], hk.scale[:, :, :nb].float())


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_append_special_values(fmt, dtype):
    """Zero blocks, the type's largest and smallest values, ties, inf and NaN."""
    B, H, D, block = 1, 1, 64, 32
    top = torch.finfo(dtype).max
    x = torch.zeros((B, H, 8 * block, D), dtype=dtype)
    x[0, 0, 1 * block:2 * block] = torch.randn(block, D).to(dtype) * 1e-3
    x[0, 0, 1 * block, 0] = top                                   # one value dwarfs a block
    x[0, 0, 2 * block:3 * block] = torch.linspace(-127, 127, block * D).view(block, D).to(dtype)
    x[0, 0, 3 * block:4 * block] = (torch.arange(block * D).view(block, D) % 255 - 127).to(dtype) / 2
    x[0, 0, 4 * block + 3, 5] = float("inf")
    x[0, 0, 5 * block + 9, 63] = float("nan")
    x[0, 0, 5 * block + 10, 3] = float("inf")
    x[0, 0, 6 * block:7 * block] = torch.finfo(dtype).tiny * torch.arange(block * D).view(block, D)
    x[0, 0, 7 * block:8 * block] = -top
    kv = allocate_quantized_kv(B, H, 8 * block, D, fmt, dtype, block)
    quantized_kv_append(kv, x.to(DEV), x.to(DEV), torch.zeros(1, dtype=torch.int64, device=DEV))
    hist = OD.History(B, H, 8 * block, D, block, fmt)
    hist.append(x, [0], [8 * block])
    _check_cache(kv, hist, hist, [8 * block])
    k, v = kv.dequantize()
    assert torch.equal(torch.isnan(k[0, 0]).all(1).view(8, block).all(1).cpu(),
                       torch.tensor([False] * 4 + [True, True, False, False]))


def _tolerance(out, mag, dots, vmax, n, D, dtype):
    u = torch.finfo(dtype).eps / 2
    return (u * out.abs() + 2.0 ** -11 * mag + n * 2.0 ** -25 * vmax
            + 2 * (D + 16) * 2.0 ** -24 * dots[..., None] * mag + (n + 64) * 2.0 ** -23 * mag)


def _filled(gen, B, H, L, D, block, fmt, dtype):
    kv = allocate_quantized_kv(B, H, L, D, fmt, dtype, block)
    k, v = (_rows(gen, B, H, kv.max_len, D, dtype=dtype) for _ in range(2))
    # scales that differ between blocks by orders of magnitude
    gain = torch.exp2(torch.randint(-6, 7, (kv.max_len // block,), generator=gen).float())
    v = (v.float().view(B, H, -1, block, D) * gain[:, None, None]).view_as(v).to(dtype)
    quantized_kv_append(kv, k.to(DEV), v.to(DEV), torch.zeros(1, dtype=torch.int64, device=DEV))
    return kv


def _check_attention(kv, q, starts, counts, scale=None, out=None):
    D = q.shape[-1]
    sc = D ** -0.5 if scale is None else scale
    st = torch.tensor(starts, dtype=torch.int64, device=DEV)
    ct = None if counts is None else torch.tensor(counts, dtype=torch.int64, device=DEV)
    if out is None:
        out = quantized_kv_attention(q.to(DEV), kv, st, ct, scale)
    B, Hq, T, _ = q.shape
    s = list(starts) * (B if len(starts) == 1 else 1)
    c = [T] * B if counts is None else list(counts) * (B if len(counts) == 1 else 1)
    ref, mag, dots = OD.attention(q, kv.k_codes.cpu().double(), kv.k_scale.cpu(),
                                  kv.v_codes.cpu().double(), kv.v_scale.cpu(), kv.block, s, c, sc)
    vmax = (kv.v_scale.amax().item() * OD.QMAX["int8" if kv.v_codes.dtype == torch.int8 else "fp8"])
    tol = _tolerance(ref, mag, dots, vmax, kv.max_len, D, q.dtype)
    assert out.shape == (B, T, Hq, D) and out.dtype == q.dtype
    err = (out.cpu().double() - ref).abs()
    assert (err <= tol).all(), f"worst {(err / tol.clamp(min=1e-30)).max().item():.2f} x tolerance"
    for b in range(B):  # queries that see nothing
        for t in range(T):
            if t >= c[b] or s[b] + t < 0:
                assert torch.count_nonzero(out[b, t]) == 0
    return out


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("B,Hq,Hkv,L,D,block,T,dtype,starts,counts", [
    (1, 16, 8, 320, 128, 64, 1, torch.bfloat16, [299], None),
    (1, 8, 8, 64, 64, 64, 1, torch.bfloat16, [0], None),              # one position
    (2, 4, 1, 128, 128, 32, 1, torch.float16, [-1, 127], None),       # an empty and a full cache
    (4, 32, 8, 2048, 128, 64, 1, torch.bfloat16, [0, 63, 64, 2047], None),
    (3, 21, 3, 777, 64, 32, 3, torch.float16, [0, 500, 774], [3, 0, 2]),
    (2, 32, 2, 512, 128, 128, 5, torch.bfloat16, [-3, 507], None),    # queries before position 0
    (2, 8, 2, 640, 256, 64, 2, torch.bfloat16, [100, 638], None),
    (1, 2, 2, 300, 256, 32, 17, torch.float16, [283], None),
    (1, 16, 1, 256, 64, 64, 40, torch.bfloat16, [100], [37]),         # many query rows
    (5, 5, 5, 96, 128, 32, 1, torch.bfloat16, [95, 94, 32, 31, 30], None),
    (2, 4, 2, 128, 64, 64, 4, torch.bfloat16, [500], None),           # start past max_len
])
def test_attention_against_the_definition(fmt, B, Hq, Hkv, L, D, block, T, dtype, starts, counts):
    gen = torch.Generator().manual_seed(B * 31 + Hq + L + T)
    kv = _filled(gen, B, Hkv, L, D, block, fmt, dtype)
    q = _rows(gen, B, Hq, T, D, dtype=dtype)
    _check_attention(kv, q, starts, counts)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("B,Hq,Hkv,L,D,block,T,dtype,starts,counts", [
    # more than 128 tiles of eight rows to an SM: sixteen query rows at a time
    (2, 16, 2, 256, 128, 64, 1251, torch.bfloat16, [-3, 200], [1251, 700]),
    (1, 21, 3, 777, 64, 32, 300, torch.float16, [500], None),
    (2, 32, 8, 20000, 128, 64, 3, torch.bfloat16, [19990, 12345], [3, 2]),
    # a short cache with more segments than one wave holds, and just fewer
    (20, 8, 8, 300, 128, 64, 1, torch.bfloat16, [299] * 10 + [0, 1, 31, 32, 63, 64, 65, 200, -1, 298],
     None),
    (18, 8, 8, 1000, 64, 64, 1, torch.float16, [999], None),
])
def test_attention_of_many_rows_and_segments(fmt, B, Hq, Hkv, L, D, block, T, dtype, starts, counts):
    gen = torch.Generator().manual_seed(B * 37 + Hq + L + T)
    kv = _filled(gen, B, Hkv, L, D, block, fmt, dtype)
    q = _rows(gen, B, Hq, T, D, dtype=dtype)
    out = _check_attention(kv, q, starts, counts)
    st = torch.tensor(starts, device=DEV)
    ct = None if counts is None else torch.tensor(counts, device=DEV)
    assert torch.equal(out, quantized_kv_attention(q.to(DEV), kv, st, ct))


def test_attention_strided_queries_scale_and_large_scores():
    gen = torch.Generator().manual_seed(8)
    kv = _filled(gen, 2, 2, 512, 128, 64, "int8", torch.bfloat16)
    base = _rows(gen, 2, 3, 8, 128, dtype=torch.bfloat16)
    q = base.transpose(1, 2)                                   # [2, 8, 3, 128], strided
    st = torch.tensor([400, 17], device=DEV)
    out = quantized_kv_attention(base.to(DEV).transpose(1, 2), kv, st, scale=0.3)
    _check_attention(kv, q, [400, 17], None, 0.3, out)
    # odd strides are read through a copy
    odd = torch.zeros(2, 8, 3, 131, dtype=torch.bfloat16, device=DEV)
    odd[..., 1:129] = q.to(DEV)
    assert torch.equal(out, quantized_kv_attention(odd[..., 1:129], kv, st, scale=0.3))
    # scores of several thousand: one position takes all the weight
    big = (q.float() * 300).to(torch.bfloat16)
    _check_attention(kv, big, [400, 17], None, 1.0)
    # queries near the type's largest value stay finite (their scores are, in fp32)
    huge = torch.full((2, 8, 1, 128), 1e30, dtype=torch.bfloat16)
    assert torch.isfinite(quantized_kv_attention(huge.to(DEV), kv, st, scale=1e-30)).all()
    zero = torch.zeros((2, 8, 1, 128), dtype=torch.bfloat16)
    _check_attention(kv, zero, [400, 17], None, 1.0)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_attention_ignores_what_lies_past_a_querys_position(fmt):
    """Codes of every pattern and NaN / inf scales past the visible positions,
    in the same block and in later ones, change nothing."""
    gen = torch.Generator().manual_seed(9)
    B, Hq, Hkv, L, D, block, T = 2, 8, 2, 512, 128, 64, 3
    kv = _filled(gen, B, Hkv, L, D, block, fmt, torch.bfloat16)
    q = _rows(gen, B, Hq, T, D, dtype=torch.bfloat16).to(DEV)
    st = torch.tensor([100, 255], device=DEV)
    want = quantized_kv_attention(q, kv, st)
    junk = torch.arange(256, dtype=torch.uint8, device=DEV).repeat(D)[:D * 2].view(2, D)
    for b, n in ((0, 103), (1, 258)):
        for c in (kv.k_codes, kv.v_codes):
            raw = c.view(torch.uint8)
            raw[b, :, n:] = junk.repeat((L - n + 1) // 2 + 1, 1)[:L - n] | 0x7f  # e4m3 NaN among them
        for s, bad in ((kv.k_scale, float("nan")), (kv.v_scale, float("inf"))):
            s[b, :, -(-n // block):] = bad
    assert torch.equal(want, quantized_kv_attention(q, kv, st))


def test_attention_of_a_block_that_reads_as_nan():
    """A non-finite row makes the queries that see its block NaN and no other."""
    gen = torch.Generator().manual_seed(10)
    B, H, L, D, block = 1, 2, 256, 64, 64
    kv = allocate_quantized_kv(B, H, L, D, "int8", torch.bfloat16, block)
    k, v = (_rows(gen, B, H, 200, D, dtype=torch.bfloat16) for _ in range(2))
    v[0, 1, 130, 3] = float("nan")
    quantized_kv_append(kv, k.to(DEV), v.to(DEV), torch.zeros(1, dtype=torch.int64, device=DEV))
    q = _rows(gen, B, 4, 2, D, dtype=torch.bfloat16).to(DEV)
    out = quantized_kv_attention(q, kv, torch.tensor([126], device=DEV))      # sees 127, 128
    assert torch.isfinite(out).all()
    out = quantized_kv_attention(q, kv, torch.tensor([127], device=DEV))      # sees 128, 129
    assert torch.isfinite(out[0, 0]).all() and torch.isfinite(out[0, 1, :2]).all()
    assert torch.isnan(out[0, 1, 2:]).all()
    # the poisoned block alone, seen by one warp, and by several CTAs
    for L2, n in ((64, 30), (4096, 4000)):
        one = allocate_quantized_kv(1, 1, L2, D, "fp8", torch.bfloat16, 32)
        rows = torch.zeros(1, 1, n, D, dtype=torch.bfloat16)
        rows[..., n - 1, 5] = float("inf")
        quantized_kv_append(one, torch.zeros_like(rows).to(DEV), rows.to(DEV),
                            torch.zeros(1, dtype=torch.int64, device=DEV))
        out = quantized_kv_attention(q[:, :1, :1], one, torch.tensor([n - 1], device=DEV))
        assert torch.isnan(out).all()
    k[0, 0, 199, 0] = float("inf")
    quantized_kv_append(kv, k.to(DEV), v.to(DEV), torch.zeros(1, dtype=torch.int64, device=DEV))
    out = quantized_kv_attention(q, kv, torch.tensor([199], device=DEV))
    assert torch.isnan(out).all()


@pytest.mark.parametrize("Hq,Hkv,T", [(32, 8, 1), (8, 8, 1), (16, 2, 9)])
def test_attention_long_context_is_deterministic(Hq, Hkv, T):
    """Work split over many CTAs: against the fp64 definition, and the same
    bits every time."""
    gen = torch.Generator().manual_seed(11)
    L, D = 20000, 128
    kv = _filled(gen, 1, Hkv, L, D, 64, "fp8", torch.bfloat16)
    q = _rows(gen, 1, Hq, T, D, dtype=torch.bfloat16)
    out = _check_attention(kv, q, [19990], None)
    st = torch.tensor([19990], device=DEV)
    for _ in range(5):
        assert torch.equal(out, quantized_kv_attention(q.to(DEV), kv, st))


def test_offsets_past_32_bits():
    """A cache whose buffers pass 2^32 bytes: the last sequence is read and
    written where it is."""
    B, H, L, D = 33, 8, 131072, 128                             # 4.6e9 codes each for K and V
    free = torch.cuda.mem_get_info()[0]
    if free < 14 << 30:
        pytest.skip("needs 14 GB of free device memory")
    kv = allocate_quantized_kv(B, H, L, D, "int8", torch.bfloat16, 64)
    gen = torch.Generator().manual_seed(12)
    k, v = (_rows(gen, 1, H, 96, D, dtype=torch.bfloat16).expand(B, H, 96, D) for _ in range(2))
    start = torch.full((B,), L - 96, dtype=torch.int64, device=DEV)
    quantized_kv_append(kv, k.to(DEV), v.to(DEV), start - start % 64)   # a block border
    last = kv.k_codes[B - 1, H - 1, -128:-32].cpu().double()
    hist = OD.History(1, H, 128, D, 64, "int8")
    hist.append(k[:1], [0], [96])
    assert torch.equal(last, hist.codes[0, H - 1, :96])
    # zero keys before: every earlier position scores 0, the last ones their own
    q = _rows(gen, 1, H, 1, D, dtype=torch.bfloat16).expand(B, H, 1, D).to(DEV)
    out = quantized_kv_attention(q, kv, torch.full((B,), L - 33, dtype=torch.int64, device=DEV))
    assert torch.equal(out[0], out[B - 1])
    kk = torch.zeros((1, 1, L - 32, D), dtype=torch.float64)
    vv = torch.zeros_like(kk)
    kk[0, 0, -96:] = hist.codes[0, 0, :96] * hist.scale[0, 0][torch.arange(96) // 64, None]
    vs = kv.v_scale[0, 0, -2:].cpu().double()
    vv[0, 0, -96:] = kv.v_codes[0, 0, -128:-32].cpu().double() * vs[torch.arange(96) // 64, None]
    p = torch.softmax((kk[0, 0] @ q[0, 0, 0].cpu().double()) * D ** -0.5, 0)
    ref = p @ vv[0, 0]
    err = (out[0, 0, 0].cpu().double() - ref).abs()
    # the values' sum is small against n: bound by the sums' fp32 error and fp16 probabilities
    A = p @ vv[0, 0].abs()
    assert (err <= 2.0 ** -9 * ref.abs() + 2.0 ** -10 * A + (L * 2.0 ** -23) * A + 1e-30).all()


def test_append_and_attend_in_a_captured_graph_with_moving_start():
    """One captured step (append, attention, start + 1) replayed gives what the
    same eager steps give; a second graph of the same cache shape does not
    disturb the first."""
    gen = torch.Generator().manual_seed(13)
    B, Hq, Hkv, L, D = 3, 8, 2, 384, 128

    def build():
        kv = _filled(torch.Generator().manual_seed(14), B, Hkv, 320, D, 64, "int8", torch.bfloat16)
        big = allocate_quantized_kv(B, Hkv, L, D, "int8", torch.bfloat16, 64)
        big.k_codes[:, :, :320].copy_(kv.k_codes)
        big.v_codes[:, :, :320].copy_(kv.v_codes)
        big.k_scale[:, :, :5].copy_(kv.k_scale)
        big.v_scale[:, :, :5].copy_(kv.v_scale)
        return big, torch.tensor([320, 319, 128], dtype=torch.int64, device=DEV)

    steps = 8
    rows = [_rows(gen, steps, B, h, 1, D, dtype=torch.bfloat16).to(DEV) for h in (Hkv, Hkv, Hq)]

    def step(kv, start, k, v, q):
        quantized_kv_append(kv, k, v, start)
        out = quantized_kv_attention(q, kv, start)
        start.add_(1)
        return out

    kv, start = build()
    start[1] = 320
    eager = [step(kv, start, *(r[i] for r in rows)).clone() for i in range(steps)]
    graphs = []
    for _ in range(2):
        kv2, s2 = build()
        s2[1] = 320
        k, v, q = (r[0].clone() for r in rows)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(kv2, s2, k, v, q)
        torch.cuda.current_stream().wait_stream(side)
        s2.sub_(1)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(kv2, s2, k, v, q)
        graphs.append((g, k, v, q, out, kv2, s2))  # a graph does not keep its buffers alive
    for i in range(steps):
        for g, k, v, q, out, _, _ in graphs:
            k.copy_(rows[0][i])
            v.copy_(rows[1][i])
            q.copy_(rows[2][i])
            g.replay()
        for g, k, v, q, out, _, _ in graphs:
            assert torch.equal(out, eager[i]), i


def test_on_another_stream_and_empty_calls():
    gen = torch.Generator().manual_seed(15)
    kv = _filled(gen, 2, 2, 256, 64, 64, "fp8", torch.bfloat16)
    q = _rows(gen, 2, 4, 1, 64, dtype=torch.bfloat16).to(DEV)
    st = torch.tensor([255], device=DEV)
    want = quantized_kv_attention(q, kv, st)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = quantized_kv_attention(q, kv, st)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(want, got)
    e = torch.empty((2, 2, 0, 64), dtype=torch.bfloat16, device=DEV)
    quantized_kv_append(kv, e, e, st)
    assert quantized_kv_attention(q[:, :, :0], kv, st).shape == (2, 0, 4, 64)


def test_registered_ops_and_refusals_on_the_gpu():
    gen = torch.Generator().manual_seed(16)
    kv = _filled(gen, 2, 2, 128, 64, 64, "int8", torch.bfloat16)
    q = _rows(gen, 2, 4, 1, 64, dtype=torch.bfloat16).to(DEV)
    st = torch.tensor([100, 3], device=DEV)
    bufs = (kv.k_codes, kv.v_codes, kv.k_scale, kv.v_scale, kv.k_tail, kv.v_tail)
    out = torch.ops.metal_liger.kv8_attention(q, st, None, *bufs, 64 ** -0.5)
    assert torch.equal(out, quantized_kv_attention(q, kv, st))
    assert torch.equal(out, ml.quantized_kv_attention(q, kv, st))
    k = torch.zeros((2, 2, 1, 64), dtype=torch.bfloat16, device=DEV)
    bad = [
        lambda: quantized_kv_attention(q.float(), kv, st),
        lambda: quantized_kv_attention(q.half(), kv, st),
        lambda: quantized_kv_attention(q[:, :3], kv, st),
        lambda: quantized_kv_attention(q[:1], kv, st),
        lambda: quantized_kv_attention(q[..., :32], kv, st),
        lambda: quantized_kv_attention(q, kv, st.int()),
        lambda: quantized_kv_attention(q, kv, st.cpu()),
        lambda: quantized_kv_attention(q, kv, torch.zeros(3, dtype=torch.int64, device=DEV)),
        lambda: quantized_kv_attention(q, kv._replace(v_scale=kv.v_scale.double()), st),
        lambda: quantized_kv_attention(q, kv._replace(v_codes=kv.v_codes.view(torch.float8_e4m3fn)), st),
        lambda: quantized_kv_attention(q, kv._replace(k_codes=kv.k_codes[:, :, :64]), st),
        lambda: quantized_kv_attention(q.clone().requires_grad_(), kv, st),
        lambda: quantized_kv_append(kv, k, k[:, :1], st),
        lambda: quantized_kv_append(kv, k.half(), k.half(), st),
        lambda: quantized_kv_append(kv, k, k, st, torch.zeros(3, dtype=torch.int64, device=DEV)),
        lambda: quantized_kv_append(kv._replace(k_codes=kv.k_codes.transpose(0, 1)), k, k, st),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {i} was not refused")
    assert sorted(CACHE_DTYPES) == ["fp8", "int8"]
