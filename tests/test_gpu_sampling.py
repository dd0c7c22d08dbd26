"""fused_sample on the GPU against the fp64 definition (oracle/decode.py).

Ids are compared exactly.  The kernel's weights are exact to 2^-44 of the
largest one, so an id can only differ where u * total lies within about
V 2^-44 of a running sum: for these sizes under 1e-7 per row, and the inputs
are fixed.  A logprob is one fp32 rounding (half a step, 2^-24 relative) of a
value known to V 2^-43.
"""

import math

import pytest
import torch

import metal_liger_b200 as ml
from metal_liger_b200.ops.fused_sampling import fused_sample
from oracle import decode as OD

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _logits(gen, B, V, dtype, spread=3.0):
    return (torch.randn(B, V, generator=gen) * spread).to(dtype)


def _check(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """x, u on the CPU; parameters numbers or CPU tensors."""
    dev = lambda p: p.to(DEV) if torch.is_tensor(p) else p  # noqa: E731
    ids, logp = fused_sample(x.to(DEV), u.to(DEV), dev(temperature), dev(top_k), dev(top_p),
                             dev(min_p))
    assert ids.dtype == torch.int64 and logp.dtype == torch.float32
    f32 = lambda p: float(torch.tensor(p, dtype=torch.float32))  # noqa: E731
    at = lambda p, b: p[b].item() if torch.is_tensor(p) else p  # noqa: E731
    for b in range(x.shape[0]):
        want, lp, kept = OD.sample_row(x[b], u[b].item(), f32(at(temperature, b)),
                                       int(at(top_k, b)), f32(at(top_p, b)), f32(at(min_p, b)))
        assert ids[b].item() == want, (b, ids[b].item(), want, len(kept))
        if math.isinf(lp):
            assert logp[b].item() == lp
        else:
            assert abs(logp[b].item() - lp) <= 2.0 ** -24 * abs(lp) + x.shape[1] * 2.0 ** -43 + 1e-12
    return ids


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,V", [(1, 1), (3, 2), (5, 31), (4, 1000), (3, 32003), (2, 151936)])
@pytest.mark.parametrize("params", [
    dict(),
    dict(temperature=0.7, top_k=50, top_p=0.9),
    dict(top_p=0.95, min_p=0.02),
    dict(temperature=1.7, top_k=1),
    dict(temperature=0.3, min_p=0.3),
    dict(top_k=7, top_p=0.5, min_p=0.1),
    dict(temperature=0.0),
], ids=["open", "k_p", "p_minp", "k1", "minp", "all", "greedy"])
def test_sample_against_the_definition(dtype, B, V, params):
    gen = torch.Generator().manual_seed(V * 5 + B + len(params))
    x = _logits(gen, B, V, dtype)
    u = torch.rand(B, generator=gen)
    _check(x, u, **params)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_flat_logits_wide_nucleus(dtype):
    """Nearly equal weights: thousands of tokens kept, ties in bf16."""
    gen = torch.Generator().manual_seed(3)
    x = _logits(gen, 6, 20011, dtype, spread=0.05)
    u = torch.rand(6, generator=gen)
    _check(x, u, top_p=0.9)
    _check(x, u, top_k=9000, top_p=0.8)
    _check(x, u, min_p=0.95)
    _check(x, u, temperature=0.05, top_p=0.99)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("spread", [0.05, 1.0, 2.5, 12.0])
@pytest.mark.parametrize("top_k", [0, 3000])
def test_min_p_around_the_end_of_top_p(dtype, spread, top_k):
    """min-p ends at, just before, just after and far from the token that top-p
    ends at."""
    gen = torch.Generator().manual_seed(int(spread * 100) + top_k)
    x = _logits(gen, 1, 20011, dtype, spread)
    top_p = 0.9
    _, _, kept = OD.sample_row(x[0], 0.5, 1.0, top_k, float(torch.tensor(top_p)), 0.0)
    w = (x[0].double() - x[0].max().double()).exp()
    end = w[torch.as_tensor(list(kept))].min().item()
    least = torch.tensor([end * f for f in (1e-3, 0.5, 0.97, 0.999, 1.001, 1.03, 2.0, 30.0)])
    least = least.clamp(max=0.999)
    n = least.numel()
    u = torch.rand(n, generator=gen)
    _check(x.expand(n, -1).contiguous(), u, top_p=top_p, top_k=top_k, min_p=least)


def test_equal_logits_keep_the_lowest_indices():
    x = torch.full((4, 1000), 2.5)
    u = torch.tensor([0.0, 0.25, 0.5, 0.999])
    ids = _check(x, u, top_k=10)
    assert ids.max() < 10
    # 0.5 of 1000 equal weights is 500 tokens exactly
    ids = _check(x, u, top_p=0.5)
    assert ids.tolist() == [0, 125, 250, 499]
    x = torch.zeros((2, 300))
    x[:, 100:200] = 1.0                                          # 100 equal largest ones
    _check(x, torch.tensor([0.1, 0.9]), top_k=130)
    _check(x, torch.tensor([0.1, 0.9]), top_k=60, top_p=0.7, min_p=1.0)
    x[:, 5] = -0.0                                               # equal to 0
    _check(x, torch.tensor([0.3, 0.7]), top_k=106)


def test_uniform_at_the_ends_and_outside():
    gen = torch.Generator().manual_seed(4)
    x = _logits(gen, 6, 500, torch.float32)
    x[:, -3:] = -math.inf
    x[:, 0] = -math.inf
    u = torch.tensor([0.0, 1.0, 1.5, -0.5, 1.0 - 2.0 ** -24, 0.5])
    _check(x, u)
    _check(x, u, top_p=0.9)
    _check(x, u, top_k=3)


def test_masked_infinite_and_nan_logits():
    gen = torch.Generator().manual_seed(5)
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        low = torch.finfo(dtype).min
        x = _logits(gen, 8, 700, dtype)
        x[0] = -math.inf                                         # nothing left
        x[1] = math.nan                                          # nothing left
        x[2, ::2] = -math.inf
        x[3, 1::3] = math.nan
        x[4] = low                                               # the lowest finite value everywhere
        x[5, 10:] = low
        x[6, [3, 400, 650]] = math.inf                           # these share all weight
        x[7, 5:] = -math.inf
        x[7, 2] = math.nan
        u = torch.rand(8, generator=gen)
        ids = _check(x, u)
        assert ids[0] == -1 and ids[1] == -1
        _check(x, u, temperature=0.5, top_k=4, top_p=0.8, min_p=0.1)
        _check(x, u, top_k=600)
        _check(x, u, temperature=0.0)


def test_parameters_per_row():
    gen = torch.Generator().manual_seed(6)
    B, V = 12, 5003
    x = _logits(gen, B, V, torch.bfloat16)
    u = torch.rand(B, generator=gen)
    t = torch.tensor([1.0, 0.0, -1.0, math.nan, 0.5, 2.0, 1.0, 1.0, 1.0, 1.0, 0.9, 1e-3])
    k = torch.tensor([0, 5, 0, 0, 3, -2, V, V + 10, 1, 100, 0, 40])
    p = torch.tensor([1.0, 0.9, 0.5, 0.5, 0.0, 0.8, -1.0, 1.5, 0.9, 1e-9, 0.6, 0.99])
    m = torch.tensor([0.0, 0.1, 0.0, 0.0, 0.0, 0.0, 0.0, -0.5, 0.0, 0.0, 1.5, 0.0])
    _check(x, u, t, k, p, m)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_temperatures_and_logits_of_every_size(dtype):
    """Weights from one token's to all equal, tops far from and at zero."""
    gen = torch.Generator().manual_seed(10)
    B, V = 5, 4099
    for scale in (0.0, 1e-6, 1.0, 300.0, 6e4):
        x = _logits(gen, B, V, torch.float32, scale)
        x[1] -= 7.0
        x[2] = -x[2].abs()                                       # the top at or next to zero
        x[3] += torch.where(torch.arange(V) % 2 == 0, 0.0, -1.0) * scale
        x = x.clamp(-6.5e4, 6.5e4).to(dtype)
        u = torch.rand(B, generator=gen)
        for t in (1e-38, 1e-30, 1e-9, 1e-4, 0.02, 30.0, 1e9, 1e35):
            _check(x, u, t)
            _check(x, u, t, top_p=0.7)
            _check(x, u, t, top_k=100, top_p=0.9, min_p=0.3)


def test_a_rows_token_does_not_depend_on_the_batch():
    gen = torch.Generator().manual_seed(7)
    x = _logits(gen, 200, 40000, torch.bfloat16, 1.0).to(DEV)
    u = torch.rand(200, generator=gen).to(DEV)
    ids, logp = fused_sample(x, u, 0.8, 0, 0.95)
    for lo, hi in ((0, 1), (10, 13), (50, 150), (199, 200)):
        i, l = fused_sample(x[lo:hi], u[lo:hi], 0.8, 0, 0.95)
        assert torch.equal(i, ids[lo:hi]) and torch.equal(l, logp[lo:hi])


def test_strided_rows_graph_stream_and_empty_batch():
    gen = torch.Generator().manual_seed(8)
    x = _logits(gen, 5, 3001, torch.bfloat16).to(DEV)
    u = torch.rand(5, generator=gen).to(DEV)
    want = fused_sample(x, u, 0.7, 20, 0.9, 0.01)
    wide = torch.zeros(5, 3011, dtype=torch.bfloat16, device=DEV)
    wide[:, 3:3004] = x
    got = fused_sample(wide[:, 3:3004], u, 0.7, 20, 0.9, 0.01)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    got = fused_sample(x.t().contiguous().t(), u, 0.7, 20, 0.9, 0.01)
    assert torch.equal(want[0], got[0])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = fused_sample(x, u, 0.7, 20, 0.9, 0.01)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(want[0], got[0])
    # two graphs over the same inputs, replayed in turn on changed inputs
    outs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = fused_sample(x, u, 0.7, 20, 0.9, 0.01)
        outs.append((g, o))
    x.copy_(_logits(gen, 5, 3001, torch.bfloat16))
    u.copy_(torch.rand(5, generator=gen))
    for g, _ in outs:
        g.replay()
    want = fused_sample(x, u, 0.7, 20, 0.9, 0.01)
    for _, o in outs:
        assert torch.equal(want[0], o[0]) and torch.equal(want[1], o[1])
    ids, logp = fused_sample(x[:0], u[:0])
    assert ids.shape == (0,) and logp.shape == (0,)


def test_frequencies_follow_the_distribution():
    """Evenly spaced uniforms reproduce the kept probabilities to one draw."""
    gen = torch.Generator().manual_seed(9)
    x = _logits(gen, 1, 50, torch.float32, 1.5)
    n = 4096
    u = (torch.arange(n) + 0.5) / n
    ids, _ = fused_sample(x.expand(n, 50).to(DEV), u.to(DEV), top_p=0.9)
    _, _, kept = OD.sample_row(x[0], 0.5, 1.0, 0, float(torch.tensor(0.9)), 0.0)
    w = torch.zeros(50, dtype=torch.float64)
    w[kept] = torch.exp(x[0, kept].double())
    w /= w.sum()
    count = torch.bincount(ids.cpu(), minlength=50).double()
    assert ((count - n * w).abs() <= 1.0 + 1e-6).all()


def test_registered_op_and_refusals():
    x = torch.randn(3, 100, device=DEV)
    u = torch.rand(3, device=DEV)
    a = torch.ops.metal_liger.sample(x, u, None, 1.0, None, 5, None, 0.9, None, 0.0)
    b = ml.fused_sample(x, u, top_k=5, top_p=0.9)
    assert torch.equal(a[0], b[0])
    for call in (
        lambda: fused_sample(x, u[:2]),
        lambda: fused_sample(x[0], u),
        lambda: fused_sample(x.int(), u),
        lambda: fused_sample(x, u.cpu()),
        lambda: fused_sample(x, u, temperature=torch.ones(2, device=DEV)),
        lambda: fused_sample(x[:, :0], u),
        lambda: fused_sample(x.clone().requires_grad_(), u),
        lambda: fused_sample(torch.zeros(1, (1 << 20) + 1, device=DEV), u[:1]),
    ):
        with pytest.raises(RuntimeError):
            call()
