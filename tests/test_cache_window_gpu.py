"""Pages that lie wholly before a window may have been given away: attention does not look their ids up."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_cache_gpu import BF16, F16, F32, _mod, _places, _random_cache  # noqa: E402


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("page,w", [(16, 64), (32, 64), (64, 64), (16, 140)])
@pytest.mark.parametrize("window", [1, 17, 40, 100])
@pytest.mark.parametrize("max_len", [None, 4000])
def test_pages_before_the_window(window, max_len, page, w, dt):
    lens = [(500, 1), (333, 3), (64, 1)]
    cache = _random_cache(100, 2, page, w, w, seed=2)
    table, start, cu = _places(lens, page, 100)
    q = torch.randn(5, 4, w, generator=torch.Generator().manual_seed(1)).to(dt).cuda()
    want = _mod().attend(q, *cache, table, start, cu, window=window, max_len=max_len)
    for i, (a, _) in enumerate(lens):
        table[i, :max(0, a - window + 1) // page] = -1
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = _mod().attend(q, *cache, table, start, cu, window=window, max_len=max_len, status=status)
    assert int(status) == 0 and torch.equal(got, want)
