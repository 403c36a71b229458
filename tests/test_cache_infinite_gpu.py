"""Infinite queries beside pages out of range: what is not seen must not show, whatever the query holds."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_cache_gpu import BF16, F16, F32, _mod, _random_cache  # noqa: E402

SIZES = [(32, 32), (130, 40)]


def _call(dt, w, wv, table, **options):
    cache = _random_cache(8, 2, 16, w, wv, seed=1)
    at = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    q = torch.randn(2, 4, w, generator=torch.Generator().manual_seed(2)).to(dt).cuda()
    q[1, 2, 5] = math.inf
    return cache, _mod().attend(q, *cache, at(*table).view(1, 3), at(40), at(0, 2), **options)


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("w,wv", SIZES)
def test_bad_pages(w, wv, dt):
    """An infinite query is infinitely far from every key that it sees: zeros, with a bad page among them or without."""
    for table in ((3, 1, 0), (3, 99, 0), (-1, 1, 0)):
        _, vo = _call(dt, w, wv, table)
        assert torch.isfinite(vo).all() and not vo[1, 2].any() and vo[1, 3].any() and vo[0, 2].any()


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("w,wv", SIZES)
def test_caps(w, wv, dt):
    """A cap bounds infinite distances too: every key scores -cap, so the row is the mean of the values -- of those that it sees."""
    table = (3, 99, 0)
    for cap in (1e-3, 5.0, 1000.0):
        cache, vo = _call(dt, w, wv, table, softcap=cap)
        v = (cache[1].double() * cache[3].double()[..., None, None])[[3, 0], 1]
        mean = torch.cat([v[0], v[1, :10]]).mean(0)  # positions 0 to 15 and 32 to 41; the page between is out of range
        step = torch.finfo(dt).eps / 2
        # weights are alike, rounded to 11 bits in 16 bits; the sum of 26 in float32; the output once
        tol = (2.0 ** -11 if dt != F32 else 0.0) * v.abs().amax() + 32 * 2.0 ** -24 * v.abs().amax() + step * mean.abs()
        assert torch.isfinite(vo).all() and ((vo[1, 2].double() - mean).abs() <= tol).all()
