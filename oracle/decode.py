"""The 8-bit KV cache and the sampler, restated in fp64 one sequence at a time.

Independent of the library: every loop is over sequences and blocks, values
are fp64, and what a position holds is derived from the definition (a block is
quantised from all its unquantised rows; a query sees the positions up to its
own; a token is drawn from a prefix of the logit order).
"""

import math

import torch

QMAX = {"int8": 127.0, "fp8": 448.0}


def e4m3(x: torch.Tensor) -> torch.Tensor:
    """fp64 values rounded half to even to e4m3 (3 fraction bits, smallest
    exponent -6), |x| <= 448."""
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(e - 3)
    return torch.round(x / step) * step


def quantise(rows: torch.Tensor, fmt: str):
    """(codes as fp64, scale) of one block's live rows [n, D] (fp64)."""
    a = float(rows.abs().max()) if rows.numel() else 0.0
    if not torch.isfinite(rows).all():
        a = math.nan if torch.isnan(rows).any() else math.inf
    scale = torch.tensor(a, dtype=torch.float64) / QMAX[fmt]
    if a == 0.0 or not math.isfinite(a):
        return torch.zeros_like(rows), scale
    q = rows * QMAX[fmt] / a
    return (torch.round(q) if fmt == "int8" else e4m3(q)), scale


class History:
    """What a cache should hold, kept as the rows themselves: per (sequence,
    head) a list of unquantised rows; ``append`` mirrors one call."""

    def __init__(self, batch, heads, max_len, dim, block, fmt):
        self.shape = (batch, heads, max_len, dim)
        self.block, self.fmt = block, fmt
        self.rows = torch.zeros(self.shape, dtype=torch.float64)
        self.codes = torch.zeros(self.shape, dtype=torch.float64)
        self.scale = torch.zeros((batch, heads, max_len // block), dtype=torch.float64)

    def append(self, x, starts, counts):
        """x [B, H, T, D]; starts / counts lists of ints."""
        B, H, L, _ = self.shape
        for b in range(B):
            s = starts[b]
            n = max(0, min(counts[b], x.shape[2]))
            if s < 0 or s >= L:
                continue
            e = min(L, s + n)
            if e <= s:
                continue
            self.rows[b, :, s:e] = x[b, :, :e - s].double()
            for blk in range(s // self.block, (e - 1) // self.block + 1):
                lo, hi = blk * self.block, min(e, (blk + 1) * self.block)
                for h in range(H):
                    q, sc = quantise(self.rows[b, h, lo:hi], self.fmt)
                    self.codes[b, h, lo:hi] = q
                    self.scale[b, h, blk] = sc


def attention(q, codes_k, scale_k, codes_v, scale_v, block, starts, counts, scale):
    """q [B, Hq, T, D] (any dtype) against codes (fp64 values) and scales;
    returns (out, weighted |v|, sum |q k| scale) in fp64: [B, T, Hq, D], [B, T,
    Hq, D] and [B, T, Hq] (the largest over the visible positions)."""
    B, Hq, T, D = q.shape
    H, L = codes_k.shape[1], codes_k.shape[2]
    out = torch.zeros((B, T, Hq, D), dtype=torch.float64)
    mag = torch.zeros_like(out)
    dots = torch.zeros((B, T, Hq), dtype=torch.float64)
    for b in range(B):
        for t in range(min(T, counts[b])):
            n = max(0, min(L, starts[b] + t + 1))
            if n == 0:
                continue
            at = torch.arange(n) // block
            for h in range(Hq):
                g = h // (Hq // H)
                k = codes_k[b, g, :n].double() * scale_k[b, g].double()[at, None]
                v = codes_v[b, g, :n].double() * scale_v[b, g].double()[at, None]
                x = q[b, h, t].double()
                p = torch.softmax((k @ x) * scale, 0)
                out[b, t, h] = p @ v
                mag[b, t, h] = p @ v.abs()
                dots[b, t, h] = (k.abs() @ x.abs()).max() * scale
    return out, mag, dots


def _running(values):
    """Running sums of floats, each exact to fp64 (Neumaier's compensated sum)."""
    total, low = 0.0, 0.0
    for v in values:
        t = total + v
        low += (total - t) + v if total >= v else (v - t) + total
        total = t
        yield total + low


def sample_row(x, u, temperature, top_k, top_p, min_p):
    """(id, logprob, kept ids) of one row of logits by the definition."""
    x = x.double().tolist()
    order = sorted((i for i in range(len(x)) if x[i] > -math.inf), key=lambda i: (-x[i], i))
    if not order:
        return -1, -math.inf, []
    if not temperature > 0:
        return order[0], 0.0, order[:1]
    top = x[order[0]]

    def w(i):
        if top == math.inf:
            return 1.0 if x[i] == math.inf else 0.0
        return math.exp((x[i] - top) / temperature)

    kept = order[:top_k] if top_k > 0 else order
    if top_p < 1:
        total = math.fsum(w(i) for i in kept)
        n = 0
        for run in _running(w(i) for i in kept):
            n += 1
            if run >= top_p * total:
                break
        kept = kept[:n]
    kept = kept[:1] + [i for i in kept[1:] if w(i) >= min_p and min_p <= 1]
    ids = sorted(kept)
    total = math.fsum(w(i) for i in ids)
    u = min(max(u, 0.0), 1.0)
    pick = None
    for i, run in zip(ids, _running(w(i) for i in ids)):
        if w(i) > 0:
            if run > u * total:
                pick = i
                break
            last = i
    if pick is None:
        pick = last
    z = 0.0 if top == math.inf else (x[pick] - top) / temperature
    return pick, z - math.log(total), ids
