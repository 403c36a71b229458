"""Pages whose value scales differ by many orders of magnitude, whichever of them hold a row's weight.

Weights times the page's value scale are rounded to 11 bits (float16: and their rest), or to 2^-29 of the row's largest weight, each relative to its own page's scale as
long as no scale is 2^58 times another; with what test_cache_gpu.py's bounds take in, a row's output is as exact as with equal scales.
"""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_cache_gpu import BF16, F16, F32, _attend, _mod, _places, _random_cache  # noqa: E402


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("ratio", [1e-9, 1e-3, 1e2, 1e4, 1e6, 1e9, 1e15])
@pytest.mark.parametrize("order", ["first", "last", "between"])
@pytest.mark.parametrize("page,h,w,wv", [(16, 4, 64, 64), (64, 24, 128, 128)])
def test_far_pages_of_other_scales(page, h, w, wv, order, ratio, dt):
    """Half of the pages are so far from the queries that their weights are below 2^-24 of the others', and their value scales `ratio` times as large."""
    n = 12
    lens = [(n * page - 1, 1), (3 * page, 2)]
    cache = _random_cache(20, 2, page, w, wv, seed=8)
    places = _places(lens, page, 20, seed=4)
    slots = {"first": range(n // 2), "last": range(n // 2, n - 1), "between": range(1, n, 2)}[order]
    far = places[0][0, list(slots)].long()
    cache[2][far] *= 60  # keys of norm 60 times as large: scores below -400 (64 wide: -380)
    cache[3][far] *= ratio
    if dt == F16:  # (outputs of about 100: what is lost would show)
        cache[3].mul_(1000)
    q = torch.randn(3, h, w, generator=torch.Generator().manual_seed(2)).to(dt).cuda()
    _attend(q, cache, places)


@pytest.mark.parametrize("dt", [F16, BF16])
def test_scales_up_and_down(dt):
    """Value scales over sixteen orders of magnitude in any order, all pages alike in weight."""
    lens = [(500, 3), (30, 1)]
    cache = _random_cache(40, 2, 16, 64, 64, seed=3)
    places = _places(lens, 16, 40, seed=5)
    order = torch.randperm(40, generator=torch.Generator().manual_seed(6)).cuda()
    cache[3].mul_(torch.logspace(-14, 2, 40, device="cuda")[order][:, None])
    cache[3][4] = 0
    _attend(torch.randn(4, 6, 64, generator=torch.Generator().manual_seed(7)).to(dt).cuda(), cache, places)


@pytest.mark.parametrize("dt", [F16, BF16])
def test_smallest_and_largest_scales(dt):
    """Scales at both ends of float32: nothing becomes infinite or NaN on the way."""
    cache = _random_cache(8, 1, 16, 64, 64, seed=3)
    places = _places([(127, 1)], 16, 8, seed=5)
    for scales in ([1e-38, 1e30, 1e-38, 1e-44, 1e36, 1e-30, 1.0, 0.0], [1e36, 1e-44, 1e-44, 1e-38, 1e-44, 1e-38, 1e-44, 1e-44]):
        cache[3].copy_(torch.tensor(scales, device="cuda")[:, None])
        for far in (False, True):
            cache[2].fill_(0.03)
            if far:
                cache[2][cache[3] > 1] = 3.0
            vo = _mod().attend(torch.randn(1, 2, 64, generator=torch.Generator().manual_seed(7)).to(dt).cuda(), *cache, *places)
            assert not vo.isnan().any() and (torch.isfinite(vo).all() or not far)
