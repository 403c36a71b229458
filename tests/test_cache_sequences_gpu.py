"""Calls of thousands of sequences, more than a warp looks at in one step or two: every row finds its own, empty ones and refused ones among them."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_cache_gpu import BF16, F32, _append_reference, _attend, _mod, _random_cache, _same  # noqa: E402


def _dev(x):
    return torch.tensor(np.asarray(x, np.int32), device="cuda")


def _call(count, page, seed):
    """Starts and counts of one page each at most, a third of the sequences empty; (table, start, cu)."""
    rng = np.random.RandomState(seed)
    start = rng.randint(0, page - 3, count)
    new = rng.choice([0, 1, 1, 2, 3, 0], count)
    new[:40] = 0  # (a run of empty ones where the first probe falls)
    return _dev(rng.permutation(count + 3)[:count, None]), _dev(start), _dev(np.concatenate([[0], np.cumsum(new)]))


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("count", [64, 65, 96, 1000, 2048, 2049, 5000])
def test_every_row_finds_its_sequence(count, dt):
    page, hk, h, w, wv = 16, 2, 4, 16, 24
    cache = _random_cache(count + 3, hk, page, w, wv, seed=count)
    places = _call(count, page, count)
    rows = int(places[2][-1])
    g = torch.Generator().manual_seed(count)
    mk = lambda heads, x: torch.randn(rows + 3, heads, x, generator=g).to(dt).cuda()  # noqa: E731
    k, v = mk(hk, w), mk(hk, wv)
    want = _append_reference(cache, k, v, *places)
    _mod().append(k, v, *cache, *places)
    _same(cache, want)
    kv = [torch.full((rows + 3, hk, x), 7.0, dtype=dt, device="cuda") for x in (w, wv)]
    _mod().gather(*cache, *places, rows + 3, dtype=dt, out=kv)
    table, start, cu = (x.cpu().numpy() for x in places)
    seq = np.repeat(np.arange(count), np.diff(cu))
    at, pos = table[seq, 0], start[seq] + np.arange(rows) - cu[seq]
    for x, codes, scale in zip(kv, want[:2], want[2:]):
        value = torch.tensor(codes[at, :, pos].astype(np.float32) * scale[at][..., None]).to(dt)
        assert torch.equal(x[:rows].cpu(), value) and (x[rows:] == 7).all()
    _attend(mk(h, w), cache, places)


@pytest.mark.parametrize("count", [300, 3000])
def test_refused_ones_among_them(count):
    """Starts that are out of range: these rows are zeros, all others what they were."""
    cache = _random_cache(count + 3, 2, 16, 16, 16, seed=1)
    table, start, cu = _call(count, 16, 5)
    rows = int(cu[-1])
    bad = torch.rand(count, generator=torch.Generator().manual_seed(2)).cuda() < 0.2
    seq = torch.repeat_interleave(torch.arange(count, device="cuda"), cu.diff())
    k, v = _mod().gather(*cache, table, start, cu, rows)
    status = _dev([0])
    k2, v2 = _mod().gather(*cache, table, torch.where(bad, -3, start).to(torch.int32), cu, rows, status=status)
    assert int(status) != 0
    for a, b in ((k, k2), (v, v2)):
        assert torch.equal(torch.where(bad[seq][:, None, None], 0.0, a), b)
