"""Appends to the 8-bit cache that go back, and back again: into blocks whose
unquantised rows the tail still has and into blocks whose rows it has lost."""

import copy

import pytest
import torch

from metal_liger_b200.ops.quantized_kv import allocate_quantized_kv, quantized_kv_append
from oracle import decode as OD

pytestmark = pytest.mark.gpu
DEV = "cuda"


class _Model:
    """What the cache should hold: the oracle's rows, but a block that is
    continued after its rows left the tail starts from what its codes stand
    for, rounded to the rows' type.  The tail has the last two blocks of each
    append, block i in slot i % 2."""

    def __init__(self, B, H, L, D, block, fmt, dtype):
        self.hist = OD.History(B, H, L, D, block, fmt)
        self.block, self.dtype = block, dtype
        self.held = [[-1, -1] for _ in range(B)]

    def append(self, x, starts, counts):
        h, blk = self.hist, self.block
        for b, (s, n) in enumerate(zip(starts, counts)):
            e = min(h.shape[2], s + n)
            first, last = s // blk, (e - 1) // blk
            if e <= s:
                continue
            if s % blk and self.held[b][first % 2] != first:
                lo = first * blk
                was = h.codes[b, :, lo:s] * h.scale[b, :, first, None, None].float().double()
                h.rows[b, :, lo:s] = was.float().to(self.dtype).double()
            for i in range(max(first, last - 1), last + 1):
                self.held[b][i % 2] = i
        h.append(x, starts, counts)


def _same(kv, models, ends):
    for codes, scale, m in ((kv.k_codes, kv.k_scale, models[0]), (kv.v_codes, kv.v_scale, models[1])):
        c, s, h = codes.cpu().double(), scale.cpu(), m.hist
        for b, n in enumerate(ends):
            nb = -(-n // h.block)
            want, got = h.scale[b, :, :nb].float(), s[b, :, :nb]
            assert ((got == want) | (got.isnan() & want.isnan())).all(), (b, n)
            assert torch.equal(c[b, :, :n], h.codes[b, :, :n]), (b, n)


def _run(steps, B=2, H=2, L=768, D=64, block=64, fmt="int8", dtype=torch.bfloat16, seed=0, rows=None):
    gen = torch.Generator().manual_seed(seed)
    kv = allocate_quantized_kv(B, H, L, D, fmt, dtype, block)
    models = [_Model(B, H, L, D, block, fmt, dtype) for _ in range(2)]
    for i, (start, T) in enumerate(steps):
        starts = list(start) if isinstance(start, tuple) else [start] * B
        k, v = ((torch.randn((B, H, T, D), generator=gen) * 2).to(dtype) for _ in range(2))
        if rows is not None:
            k, v = rows(i, k, v)
        quantized_kv_append(kv, k.to(DEV), v.to(DEV), torch.tensor(starts, device=DEV))
        for m, x in zip(models, (k, v)):
            m.append(x, starts, [T] * B)
        _same(kv, models, [min(L, s + T) for s in starts])
    return kv


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,block", [(64, 64), (128, 32), (256, 128)])
@pytest.mark.parametrize("steps", [
    # two steps back, the second into the block before the one the first ended in
    [(0, 200), (190, 1), (125, 3)],
    # to an earlier border, then into the block before it
    [(0, 650), (128, 3), (100, 4)],
    # into blocks of either parity that have left the tail, and on from there
    [(0, 500), (70, 1), (71, 1), (72, 200), (10, 1), (11, 60), (300, 4)],
    # a long append that begins in a lost block and ends in its slot
    [(0, 640), (65, 300), (140, 400), (5, 2), (7, 600)],
    # sequences that go back each to a place of its own
    [(0, 600), ((3, 599), 2), ((5, 130), 130), ((134, 129), 1), ((64, 1), 700)],
], ids=["twice", "border", "parities", "long", "ragged"])
def test_append_taken_back_twice(steps, D, block, dtype, fmt):
    _run(steps, D=D, block=block, dtype=dtype, fmt=fmt, seed=len(steps))


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_lost_rows_keep_their_codes_while_the_maximum_stands(fmt, dtype):
    """Codes that are quantised again from what they stand for do not move
    (127 of the largest code, rounded to bf16, is off by 127 / 257 of a step, less
    than a half; e4m3's steps are 2^-3 and fp16's roundings smaller), so only the
    first quantisation counts."""
    gen = torch.Generator().manual_seed(4)
    B, H, L, D, block = 1, 2, 256, 64, 64
    kv = allocate_quantized_kv(B, H, L, D, fmt, dtype, block)
    k, v = (torch.randn((B, H, 256, D), generator=gen).to(dtype) for _ in range(2))
    for x in (k, v):
        x[:, :, ::64, 0] = 8.0                                 # each block's largest value
    at = lambda s: torch.tensor([s], device=DEV)  # noqa: E731
    quantized_kv_append(kv, k.to(DEV), v.to(DEV), at(0))
    codes, scale = kv.k_codes.clone(), kv.v_scale.clone()
    for start in (50, 40, 100, 30):
        new = k[:, :, start:start + 1].to(DEV)
        quantized_kv_append(kv, new, v[:, :, start:start + 1].to(DEV), at(start))
        lo = start // 64 * 64
        assert torch.equal(codes[:, :, lo:start + 1].view(torch.uint8),
                           kv.k_codes[:, :, lo:start + 1].view(torch.uint8))
        assert torch.equal(scale, kv.v_scale)


def test_a_lost_block_that_reads_as_nan_stays_so():
    """Its codes are not its values, and there is nothing else to go by."""
    def rows(i, k, v):
        if i == 0:
            k[:, 0, 70, 3] = float("nan")
            v[:, 1, 90, 5] = float("inf")
        return k, v

    kv = _run([(0, 600), (100, 2), (102, 1)], rows=rows)
    assert kv.k_scale[:, 0, 1].isnan().all() and not kv.v_scale[:, 1, 1].isfinite().any()
    assert kv.k_scale[:, 1, 1].isfinite().all()


def test_what_a_cache_made_of_buffers_trusts():
    """Which block a slot holds is known to the caches that allocate_quantized_kv
    made (and their deep copies).  One put together from buffers takes the tail
    at its word."""
    from metal_liger_b200.ops.quantized_kv import QuantizedKV

    kv = _run([(0, 300)])
    twin = copy.deepcopy(kv)
    loose = QuantizedKV(*(t.clone() for t in kv))
    gen = torch.Generator().manual_seed(9)
    k, v = (torch.randn((2, 2, 1, 64), generator=gen).to(torch.bfloat16).to(DEV) for _ in range(2))
    for c in (kv, twin, loose):
        quantized_kv_append(c, k, v, torch.tensor([80], device=DEV))
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(kv, twin))
    # (80 lies in block 1, whose slot has block 3)
    hist = OD.History(2, 2, 768, 64, 64, "int8")
    rows = torch.cat([loose.k_tail[:, :, 1, :16], k], 2)
    hist.append(rows.cpu(), [64, 64], [17, 17])
    assert torch.equal(loose.k_codes[:, :, 64:81].cpu().double(), hist.codes[:, :, 64:81])
    assert not torch.equal(loose.k_codes[:, :, 64:81], kv.k_codes[:, :, 64:81])


def test_records_that_do_not_fit_are_refused():
    kv = allocate_quantized_kv(2, 2, 128, 64)
    k = torch.zeros((2, 2, 1, 64), dtype=torch.bfloat16, device=DEV)
    st = torch.zeros(1, dtype=torch.int64, device=DEV)
    held = kv.held
    for bad in (held.long(), held[:, :1], held.transpose(1, 3), held.cpu(), held.view(-1)):
        kv.held = bad
        with pytest.raises(RuntimeError):
            quantized_kv_append(kv, k, k, st)
    kv.held = held
    quantized_kv_append(kv, k, k, st)
    assert (kv.held[..., 0] == 0).all() and (kv.held[..., 1] == -1).all()
