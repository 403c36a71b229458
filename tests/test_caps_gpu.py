"""Caps of every size that is accepted: far above the scores (a cap that changes nothing), and so far below them that every score lies at it.

The bounds are those of test_masked_gpu.py and test_cache_gpu.py: the capped score is off by 8 u of the score beside what the distance is off by, u = 2^-24.
"""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_cache_gpu import _attend, _mod, _places, _random_cache  # noqa: E402
from test_masked_gpu import BF16, F16, F32, _compare, _inputs, _op  # noqa: E402

CAPS = [1e-30, 1e-9, 1e-3, 50.0, 1e3, 1e6, 1e9, 1e30]


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("cap", CAPS)
def test_masked(cap, dt):
    _compare(*_inputs(1, 130, 2, 1, 64, 64, dt, seed=1), {}, dict(softcap=cap))


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("cap", CAPS)
def test_attend(cap, dt):
    lens = [(300, 2), (20, 1)]
    cache = _random_cache(8, 2, 64, 64, 64, seed=1)
    q = torch.randn(3, 4, 64, generator=torch.Generator().manual_seed(2)).to(dt).cuda()
    _attend(q, cache, _places(lens, 64, 8), softcap=cap)


@pytest.mark.parametrize("dt", [F16, BF16])
def test_a_cap_beyond_all_scores_changes_nothing(dt):
    """Scores differ by 2^-21 of themselves: with scores to -16 weights by 2^-16 (two of them), far below a step of the outputs."""
    q, k, v, dvo = _inputs(1, 200, 2, 1, 64, 64, dt, seed=2)
    none, capped = ([vo.detach()] + list(torch.autograd.grad(vo, (q, k, v), dvo)) for vo in (_op(softcap=c)(q, k, v) for c in (0.0, 1e30)))
    for a, b in zip(none, capped):
        assert float((a.double() - b.double()).norm() / a.double().norm()) <= torch.finfo(dt).eps


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("cap", [1e-30, 1e-9, 1e-7])
def test_queries_that_lie_on_keys(dt, cap):
    """A distance of zero may come out on either side of it by a rounding, which is many caps: the score is still a bounded number."""
    page, w = 64, 128
    cache = _random_cache(4, 1, page, w, w, seed=5)
    places = _places([(192, 64)], page, 4)
    cache[0].copy_(cache[0].abs())  # (sums of one sign: the largest roundings)
    rows = places[0][0, :4].long()
    keys = (cache[0][rows, 0].float() * cache[2][rows, 0][:, None, None]).flatten(0, 1)
    q = keys[192:256, None].to(dt)
    got = _mod().attend(q, *cache, *places, softcap=cap)
    assert torch.isfinite(got).all()
    _attend(q, cache, places, softcap=cap)
    k = (10 * torch.randn(1, 256, 1, w, generator=torch.Generator().manual_seed(3))).abs().to(dt).cuda()
    vo = _op(softcap=cap)(k, k, k)
    mean = k[0, :, 0].double().cumsum(0) / torch.arange(1, 257, device="cuda")[:, None]  # every score is 0 but for the cap
    assert float((vo[0, :, 0].double() - mean).abs().max()) <= 2 * math.exp(2 * cap) * torch.finfo(dt).eps * float(mean.max())
