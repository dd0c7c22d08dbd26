"""The decode-side operators measured against their plain forms.

Three operators of the generator's answering path:

* ``append``  — new tokens' K and V written into a KV cache held in 8 bits
  (int8 or e4m3) with one fp32 scale per block of positions and kv head;
* ``attend``  — attention of one or a few query tokens per sequence over that
  cache;
* ``sample``  — temperature / top-k / top-p / min-p sampling of a row of
  logits from a given uniform number.

``own = False`` computes them with elementary torch operations in 32 bits (64
where a border decides), ``own = True`` calls ``metal_liger_b200``.
"""

import math

import torch

own = False

DEV = "cuda"
QMAX = {"int8": 127.0, "fp8": 448.0}
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CODES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------

def listed():
    a = dict(op="append", block=64, type="bf16")
    t = dict(op="attend", block=64, type="bf16")
    s = dict(op="sample", type="bf16")
    return [
        # one decode step of a served batch: a token per sequence, ragged positions
        dict(a, name="append 1 token x 64", cache="int8", batch=64, kv_heads=8, dim=128,
             tokens=1, context=4096, ragged=True),
        # prompts of a training-length batch going into the cache after their prefill
        dict(a, name="append prompts 8 x 4096", cache="fp8", batch=8, kv_heads=8, dim=128,
             tokens=4096, context=4096, ragged=False),
        # a padded chunk of prompt appended at odd positions (continuing a conversation)
        dict(a, name="append 3 x 137 padded", cache="int8", batch=3, kv_heads=4, dim=64,
             tokens=137, context=1000, ragged=True, type="fp16", block=32),
        # one sequence just after a short prompt: latency
        dict(t, name="attend 1 x 300", cache="int8", batch=1, kv_heads=8, group=2, dim=128,
             tokens=1, context=300, ragged=False),
        # one sequence with a long context
        dict(t, name="attend 1 x 65536", cache="int8", batch=1, kv_heads=8, group=4, dim=128,
             tokens=1, context=65536, ragged=False),
        # a served batch of ragged contexts
        dict(t, name="attend 64 x 8192 ragged", cache="fp8", batch=64, kv_heads=8, group=4, dim=128,
             tokens=1, context=8192, ragged=True),
        # several query tokens per sequence (a drafted continuation being checked)
        dict(t, name="attend 4 x 8 of 4000", cache="fp8", batch=4, kv_heads=8, group=4, dim=128,
             tokens=8, context=4000, ragged=True),
        # another head shape, fp16, odd group, short blocks
        dict(t, name="attend 5 x 777 d64 g7", cache="int8", batch=5, kv_heads=3, group=7, dim=64,
             tokens=3, context=777, ragged=True, type="fp16", block=32),
        # one sequence's next token with the usual filters: latency
        dict(s, name="sample 1 x 151936", batch=1, vocab=151936, temperature=0.7, top_k=50,
             top_p=0.9, min_p=0.0, mixed=False),
        # a served batch, nucleus and min-p
        dict(s, name="sample 64 x 151936", batch=64, vocab=151936, temperature=1.0, top_k=0,
             top_p=0.95, min_p=0.02, mixed=False),
        # rollouts for training: fp32 logits, nothing filtered
        dict(s, name="sample 256 x 151936 open", batch=256, vocab=151936, temperature=1.0, top_k=0,
             top_p=1.0, min_p=0.0, mixed=False, type="fp32"),
        # every row its own settings, a flat distribution with a wide nucleus
        dict(s, name="sample 37 x 32003 mixed", batch=37, vocab=32003, temperature=1.3, top_k=400,
             top_p=0.98, min_p=0.01, mixed=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "sample"])
    if op == "sample":
        batch = _log(rng, 1, 256)
        vocab = _log(rng, 50, 152000)
        return dict(op=op, batch=batch, vocab=vocab, type=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                    temperature=round(rng.uniform(0.3, 1.5), 3),
                    top_k=rng.choice([0, 0, 1, 20, 50, _log(rng, 2, vocab)]),
                    top_p=rng.choice([1.0, 0.5, 0.8, 0.9, 0.95, 0.99]),
                    min_p=rng.choice([0.0, 0.0, 0.01, 0.05, 0.2]), mixed=rng.random() < 0.3)
    c = dict(op=op, cache=rng.choice(["int8", "fp8"]), type=rng.choice(["bf16", "bf16", "fp16"]),
             block=rng.choice([32, 64, 64, 128]), dim=rng.choice([64, 128, 128, 256]),
             batch=_log(rng, 1, 64), kv_heads=rng.choice([1, 2, 3, 4, 8, 8]),
             ragged=rng.random() < 0.7)
    if op == "append":
        c["tokens"] = rng.choice([1, 1, _log(rng, 2, 4096)])
        per = c["batch"] * c["kv_heads"] * c["dim"]
        c["tokens"] = max(1, min(c["tokens"], 8 * 8 * 128 * 4096 // per))
        c["context"] = c["tokens"] + _log(rng, 1, 4096)
        c["context"] = max(c["tokens"], min(c["context"], (1 << 30) // per))
    else:
        c["group"] = rng.choice([1, 2, 4, 4, 7, 8, 16])
        c["tokens"] = rng.choice([1, 1, 1, _log(rng, 2, 16)])
        top = (64 * 8 * 8192 * 128) // (c["batch"] * c["kv_heads"] * c["dim"])
        top = min(top, (1 << 27) // (c["batch"] * c["kv_heads"] * c["group"] * c["tokens"]))
        # the arithmetic of several query rows counts too
        top = min(top, 64 * 8 * 8192 * 128 * 4 // (c["batch"] * c["kv_heads"] * c["group"]
                                                   * c["tokens"] * c["dim"]))
        c["context"] = max(c["tokens"], _log(rng, 1, max(2, min(65536, top))))
    return c


def _capacity(c):
    return -(-c["context"] // c["block"]) * c["block"]


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _kv(gen, shape, dtype):
    """Keys / values of a head: unit variance, a few channels several times larger."""
    x = torch.randn(shape, generator=gen, device=DEV)
    gain = torch.where(torch.rand(shape[-1], generator=gen, device=DEV) < 0.05, 4.0, 1.0)
    return (x * gain).to(dtype)


def _starts(c, gen):
    """Positions filled before the call, so that the call ends at most at `context`."""
    most = c["context"] - c["tokens"]
    if not c["ragged"]:
        return torch.full((c["batch"],), most, dtype=torch.int64, device=DEV)
    u = torch.rand(c["batch"], generator=gen, device=DEV, dtype=torch.float64)
    s = (u * (most + 1)).to(torch.int64).clamp_(max=most)
    s[0] = most
    return s


def _counts(c, gen):
    """How many of the `tokens` rows are real; None where nothing is padded."""
    if not c["ragged"] or c["tokens"] == 1:
        return None
    u = torch.rand(c["batch"], generator=gen, device=DEV, dtype=torch.float64)
    n = 1 + (u * c["tokens"]).to(torch.int64)
    n = n.clamp_(max=c["tokens"])
    n[0] = c["tokens"]
    return n


def _cache(c, gen):
    """A filled cache: codes with the spread that quantised unit-variance blocks have."""
    B, H, L, D = c["batch"], c["kv_heads"], _capacity(c), c["dim"]
    out = {}
    for n in ("k", "v"):
        codes = torch.empty((B, H, L, D), dtype=CODES[c["cache"]], device=DEV)
        for b in range(B):
            x = torch.randn((H, L, D), generator=gen, device=DEV)
            x = (x * (QMAX[c["cache"]] / 4)).clamp_(-QMAX[c["cache"]], QMAX[c["cache"]])
            codes[b] = (x.round_() if c["cache"] == "int8" else x).to(codes.dtype)
        scale = torch.rand((B, H, L // c["block"]), generator=gen, device=DEV) * 0.5 + 0.75
        out[n + "_codes"] = codes
        out[n + "_scale"] = scale * (4 / QMAX[c["cache"]])
        out[n + "_tail"] = torch.zeros((B, H, 2, c["block"], D), dtype=TYPES[c["type"]], device=DEV)
    return out


def prepare(case, seed):
    c = case
    gen = torch.Generator(device=DEV).manual_seed(seed * 7919 + 13)
    if c["op"] == "sample":
        B, V = c["batch"], c["vocab"]
        x = torch.randn((B, V), generator=gen, device=DEV) * 2.2
        # a few hundred candidates stand out, as a language model's do
        peak = torch.rand((B, V), generator=gen, device=DEV)
        e = -torch.log(torch.rand((B, V), generator=gen, device=DEV).clamp_(min=1e-9))
        x = torch.where(peak < min(0.3, 200.0 / V), x + 3.0 * e, x).to(TYPES[c["type"]])
        st = dict(op="sample", logits=x, uniform=torch.rand(B, generator=gen, device=DEV))
        names = ("temperature", "top_k", "top_p", "min_p")
        if not c["mixed"]:
            st.update({n: c[n] for n in names})
            return st
        r = torch.rand((4, B), generator=gen, device=DEV)
        st["temperature"] = c["temperature"] * (0.5 + r[0])
        st["temperature"][0] = 0.0  # a greedy row among them
        st["top_k"] = torch.where(r[1] < 0.4, 0, (r[1] * max(c["top_k"], 3)).long() + 1)
        st["top_p"] = torch.where(r[2] < 0.3, 1.0, c["top_p"] * (0.4 + 0.6 * r[2]))
        st["min_p"] = torch.where(r[3] < 0.5, 0.0, c["min_p"] * r[3])
        return st
    B, H, T, D = c["batch"], c["kv_heads"], c["tokens"], c["dim"]
    dt = TYPES[c["type"]]
    st = dict(op=c["op"], cache=c["cache"], block=c["block"], start=_starts(c, gen),
              counts=_counts(c, gen), kv=_cache(c, gen))
    if c["op"] == "append":
        # k and v as the projections leave them: [B, T, H, D] seen as [B, H, T, D]
        st["k"] = _kv(gen, (B, T, H, D), dt).transpose(1, 2)
        st["v"] = _kv(gen, (B, T, H, D), dt).transpose(1, 2)
        for n in ("k", "v"):
            st["kv"][n + "_tail"] = _kv(gen, (B, H, 2, c["block"], D), dt)
    else:
        st["q"] = torch.randn((B, T, H * c["group"], D), generator=gen, device=DEV).mul_(1.5).to(dt) \
            .transpose(1, 2)
    return st


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------

def _append(st):
    kv, block, qmax = st["kv"], st["block"], QMAX[st["cache"]]
    B, H, T, D = st["k"].shape
    L = kv["k_codes"].shape[2]
    start = st["start"]
    count = st["counts"] if st["counts"] is not None else torch.full_like(start, T)
    end = torch.minimum(start + count, torch.full_like(start, L))
    nb = (T + block - 2) // block + 1
    blk = torch.div(start, block, rounding_mode="floor")[:, None] + torch.arange(nb, device=DEV)
    pos = blk[:, :, None] * block + torch.arange(block, device=DEV)   # [B, nb, block]
    new = (pos >= start[:, None, None]) & (pos < end[:, None, None])
    touched = new.any(2)
    live = (pos < end[:, None, None]) & touched[:, :, None]
    last = torch.div(end - 1, block, rounding_mode="floor")
    keep = new & (blk >= last[:, None] - 1)[:, :, None]
    row = (pos - start[:, None, None]).clamp(0, T - 1)
    b3 = torch.arange(B, device=DEV)[:, None, None].expand_as(pos)
    bi, ji, ti = live.nonzero(as_tuple=True)
    bk, jk, tk = keep.nonzero(as_tuple=True)
    bs, js = touched.nonzero(as_tuple=True)
    out = {}
    for n in ("k", "v"):
        x = st[n].transpose(1, 2)[b3, row]                             # [B, nb, block, H, D]
        old = kv[n + "_tail"].permute(0, 2, 3, 1, 4)[b3, (blk % 2)[:, :, None].expand_as(pos),
                                                     pos % block]
        f = torch.where(new[..., None, None], x, old).float()
        f = torch.where(live[..., None, None], f, 0.0)
        top = f.abs().amax(dim=(2, 4), keepdim=True)                   # [B, nb, 1, H, 1]
        q = torch.where(top > 0, f * qmax / top, 0.0)
        q = (q.round() if st["cache"] == "int8" else q).to(kv[n + "_codes"].dtype)
        codes = kv[n + "_codes"].view(torch.uint8).permute(0, 2, 1, 3)
        codes[bi, pos[bi, ji, ti]] = q.view(torch.uint8)[bi, ji, ti]
        kv[n + "_scale"].permute(0, 2, 1)[bs, blk[bs, js]] = (top / qmax)[:, :, 0, :, 0][bs, js]
        kv[n + "_tail"].permute(0, 2, 3, 1, 4)[bk, blk[bk, jk] % 2, pos[bk, jk, tk] % block] = \
            x[bk, jk, tk]
        for m in ("_codes", "_scale", "_tail"):
            out[n + m] = kv[n + m]
    return out


def _attend(st):
    kv, block = st["kv"], st["block"]
    B, Hq, T, D = st["q"].shape
    H, L = kv["k_codes"].shape[1], kv["k_codes"].shape[2]
    k, v = ((kv[n + "_codes"].float().view(B, H, L // block, block * D)
             * kv[n + "_scale"][..., None]).view(B, H, L, D) for n in ("k", "v"))
    q = st["q"].float().reshape(B, H, (Hq // H) * T, D)
    s = torch.matmul(q, k.transpose(2, 3)) * D ** -0.5
    seen = st["start"][:, None] + 1 + torch.arange(T, device=DEV)      # [B, T]
    if st["counts"] is not None:
        seen = torch.where(torch.arange(T, device=DEV) < st["counts"][:, None], seen, 0)
    mask = torch.arange(L, device=DEV) < seen[..., None]               # [B, T, L]
    s = s.view(B, H, Hq // H, T, L).masked_fill_(~mask[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(top), 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    o = torch.matmul(p.view(B, H, (Hq // H) * T, L), v).view(B, Hq, T, D)
    return o.transpose(1, 2).to(st["q"].dtype).contiguous()


def _sample(st):
    B, V = st["logits"].shape
    col = lambda x: (x if torch.is_tensor(x) else torch.tensor(x, device=DEV).expand(B))[:, None]  # noqa: E731
    temp, k = col(st["temperature"]).float().double(), col(st["top_k"])
    p, least = col(st["top_p"]).float().double(), col(st["min_p"]).float().double()
    x, order = torch.sort(st["logits"], dim=1, descending=True, stable=True)
    x = x.double()
    greedy = temp <= 0
    z = (x - x[:, :1]) / torch.where(greedy, 1.0, temp)
    w = torch.exp(z)
    rank = torch.arange(V, device=DEV)[None]
    w = torch.where((k <= 0) | (rank < k), w, 0.0)
    before = torch.cumsum(w, 1)
    total = before[:, -1:]
    before = before - w
    keep = (w >= least) & ((p >= 1) | (before < p * total)) & ~greedy
    keep[:, 0] = True
    w = torch.where(keep, w, 0.0)
    kept = torch.zeros_like(w).scatter_(1, order, w)
    run_ = torch.cumsum(kept, 1)
    hit = (run_ > st["uniform"].double()[:, None] * run_[:, -1:]) & (kept > 0)
    last = V - 1 - (kept > 0).flip(1).to(torch.uint8).argmax(1)
    ids = torch.where(hit.any(1), hit.to(torch.uint8).argmax(1), last)
    logp = torch.log(kept.gather(1, ids[:, None]) / run_[:, -1:])[:, 0]
    return {"ids": ids, "logprobs": logp.float()}


def run(state):
    if own:
        from metal_liger_b200.ops.fused_sampling import fused_sample
        from metal_liger_b200.ops.quantized_kv import (
            QuantizedKV, quantized_kv_append, quantized_kv_attention)

        if state["op"] == "sample":
            ids, logp = fused_sample(state["logits"], state["uniform"],
                                     temperature=state["temperature"], top_k=state["top_k"],
                                     top_p=state["top_p"], min_p=state["min_p"])
            return {"ids": ids, "logprobs": logp}
        kv = QuantizedKV(**state["kv"])
        if state["op"] == "append":
            quantized_kv_append(kv, state["k"], state["v"], state["start"], state["counts"])
            return kv._asdict()
        return quantized_kv_attention(state["q"], kv, state["start"], state["counts"])
    return {"append": _append, "attend": _attend, "sample": _sample}[state["op"]](state)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    c = case
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[c["type"]]
    if c["op"] == "sample":
        n = c["batch"] * c["vocab"]
        return {"bytes": n * size + c["batch"] * 16, "flops": 4 * n}
    part = 0.5 if c["ragged"] else 1.0   # ragged lengths are uniform over the range
    if c["op"] == "append":
        rows = c["batch"] * c["kv_heads"] * c["tokens"] * (part if c["tokens"] > 1 else 1.0)
        kept = c["batch"] * c["kv_heads"] * min(c["tokens"], 2 * c["block"])
        return {"bytes": 2 * c["dim"] * (rows * (size + 1) + kept * size), "flops": 8 * rows * c["dim"]}
    seen = c["batch"] * c["kv_heads"] * c["context"] * part
    rows = c["batch"] * c["kv_heads"] * c["group"] * c["tokens"]
    return {"bytes": seen * 2 * (c["dim"] + 4 / c["block"]) + rows * c["dim"] * 2 * size,
            "flops": 4 * seen * c["group"] * c["tokens"] * c["dim"]}


# ---------------------------------------------------------------------------
# The definitions in 64 bits, one sequence at a time
# ---------------------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "sample": _exact_sample}[case["op"]](
        case, st)


def _exact_append(c, st):
    block, qmax, L = c["block"], QMAX[c["cache"]], _capacity(c)
    starts = st["start"].tolist()
    counts = st["counts"].tolist() if st["counts"] is not None else [c["tokens"]] * c["batch"]
    out = {}
    for n in ("k", "v"):
        codes, scale, tail = (st["kv"][n + m].double() for m in ("_codes", "_scale", "_tail"))
        for b, (s, m) in enumerate(zip(starts, counts)):
            e, first = min(s + m, L), s // block * block
            held = tail[b, :, (s // block) % 2, :s - first]
            x = torch.cat([held, st[n][b, :, :e - s].double()], 1)    # positions [first, e)
            for lo in range(0, e - first, block):
                y, at = x[:, lo:lo + block], first + lo
                top = y.abs().amax((1, 2))
                q = torch.div(y * qmax, top[:, None, None])
                if c["cache"] == "int8":
                    q = torch.round(q)
                else:  # e4m3: 3 bits below the leading one, steps of 2^-9 at the bottom
                    step = torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6))) - 3)
                    q = torch.round(q / step) * step
                codes[b, :, at:at + y.shape[1]] = q
                scale[b, :, at // block] = top / qmax
                if at // block >= (e - 1) // block - 1:
                    i = max(s - at, 0)
                    tail[b, :, at // block % 2, i:y.shape[1]] = y[:, i:]
        out[n + "_codes"] = codes if c["cache"] == "fp8" else None
        out[n + "_scale"], out[n + "_tail"] = scale, tail
    return out


def _exact_attend(c, st):
    B, T, G, D, block = c["batch"], c["tokens"], c["group"], c["dim"], c["block"]
    out = torch.zeros((B, T, c["kv_heads"] * G, D), dtype=torch.float64, device=DEV)
    starts = st["start"].tolist()
    counts = st["counts"].tolist() if st["counts"] is not None else [T] * B
    kv = st["kv"]
    for b in range(B):
        for i in range(counts[b]):
            n = min(starts[b] + i + 1, _capacity(c))
            if n <= 0:
                continue
            at = torch.arange(n, device=DEV) // block
            k, v = (kv[m + "_codes"][b, :, :n].double() * kv[m + "_scale"][b].double()[:, at, None]
                    for m in ("k", "v"))
            q = st["q"][b, :, i].double().view(-1, G, D)
            s = torch.einsum("hgd,hnd->hgn", q, k) / math.sqrt(D)
            out[b, i] = torch.einsum("hgn,hnd->hgd", torch.softmax(s, -1), v).reshape(-1, D)
    return out


def _exact_sample(c, st):
    B, V = st["logits"].shape
    at = lambda n, b: float(st[n][b]) if torch.is_tensor(st[n]) else st[n]  # noqa: E731
    f32 = lambda x: float(torch.tensor(x, dtype=torch.float32))  # noqa: E731
    logp = torch.zeros(B, dtype=torch.float64, device=DEV)
    for b in range(B):
        x = st["logits"][b].double()
        temp, k, p, least = (f32(at(n, b)) for n in ("temperature", "top_k", "top_p", "min_p"))
        if temp <= 0:
            continue                                                   # one token, log 1 = 0
        w = torch.softmax(x / temp, 0)
        order = torch.argsort(x, descending=True, stable=True)
        n = V if k <= 0 else min(int(k), V)
        w_sorted = w[order[:n]] / w[order[:n]].sum()
        if p < 1:
            n = min(n, int((torch.cumsum(w_sorted, 0) < p).sum()) + 1)
        n = max(1, min(n, int((w_sorted[:n] >= least * w_sorted[0]).sum())))
        ids = order[:n].sort()[0]
        kept = w[ids] / w[ids].sum()
        i = int((torch.cumsum(kept, 0) <= float(st["uniform"][b])).sum())
        logp[b] = torch.log(kept[min(i, n - 1)])
    return {"ids": None, "logprobs": logp}
