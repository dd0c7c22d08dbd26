"""CPU: which decoding rule generate()'s settings select.  The fused head and
sampler are CUDA kernels; here torch stands in for the head, and the sampler's
calls are counted."""

import pytest
import torch

from metal_liger_b200.generation import MetalLigerGenerator
from test_generation import _model


class _Gen(MetalLigerGenerator):
    drawn = 0

    def _greedy(self, h):
        return torch.argmax(self.head(h), dim=-1)

    def _logits(self, h):
        return self.head(h)

    def _sample(self, h, uniform, sampling):
        self.drawn += 1
        self.sampling = sampling
        return torch.argmin(self.head(h), dim=-1)


def _go(**kw):
    g = _Gen(_model())
    ids = torch.randint(0, 300, (2, 5), generator=torch.Generator().manual_seed(0))
    torch.manual_seed(7)
    return g, g.generate(ids, max_new_tokens=6, **kw)


@pytest.mark.parametrize("off", [dict(top_k=0), dict(min_p=0.0), dict(top_k=0, min_p=0)])
@pytest.mark.parametrize("rule", [dict(), dict(temperature=0.0), dict(temperature=0.7),
                                  dict(temperature=1.0, top_p=0.9)])
def test_settings_that_filter_nothing_leave_the_rule(off, rule):
    g, out = _go(**rule, **off)
    _, want = _go(**rule)
    assert g.drawn == 0 and torch.equal(out, want)


@pytest.mark.parametrize("on", [dict(top_k=3), dict(min_p=0.1), dict(fused_sampling=True),
                                dict(top_k=0, fused_sampling=True), dict(top_k=0, min_p=0.2)])
def test_settings_that_filter_select_the_sampler(on):
    g, _ = _go(**on)
    assert g.drawn == 6
    assert g.sampling["top_k"] == on.get("top_k", 0) and g.sampling["min_p"] == on.get("min_p", 0.0)
    assert _go(temperature=0.0, **on)[0].drawn == 0          # temperature 0 stays greedy


@pytest.mark.parametrize("bad", [dict(top_k=-1), dict(min_p=-0.1), dict(min_p=1.5),
                                 dict(min_p=float("nan"))])
@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_settings_out_of_range_are_refused_under_every_rule(bad, temperature):
    with pytest.raises(ValueError):
        _go(temperature=temperature, **bad)
