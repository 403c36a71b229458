"""The 8-bit cache on the GPU with many sequences at once and with long ones; references and tolerances are test_cache_gpu's."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_cache_gpu import (BF16, F16, F32, U, _append_reference, _attend, _empty, _mod, _places, _random_cache, _same)  # noqa: E402


def _many(count):
    return [((7 * i) % 90, (0, 1, 1, 2, 33, 0, 1)[i % 7]) for i in range(count)]


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("count", [33, 64, 200])
@pytest.mark.parametrize("page,h,hk,w,wv", [(16, 4, 2, 32, 48), (64, 3, 3, 40, 7)])
def test_many_sequences(count, page, h, hk, w, wv, dt):
    """More sequences than a warp has lanes, some without rows; rows of padding behind them stay as they were."""
    lens = _many(count)
    n_pages = sum(-(-(a + c) // page) for a, c in lens) + 2
    places = _places(lens, page, n_pages, seed=count)
    rows = int(places[2][-1])
    g = torch.Generator().manual_seed(count)
    mk = lambda heads, x: torch.randn(rows + 5, heads, x, generator=g).to(dt).cuda()  # noqa: E731
    cache = _random_cache(n_pages, hk, page, w, wv, seed=1)
    k, v = mk(hk, w), mk(hk, wv)
    want = _append_reference(cache, k, v, *places)
    _mod().append(k, v, *cache, *places)
    _same(cache, want)
    out = torch.full((rows + 5, h, wv), 7.0, dtype=dt, device="cuda")
    q = mk(h, w)
    got = _attend(q, cache, places)
    _mod().attend(q, *cache, *places, out=out)
    assert torch.equal(out[:rows], got[:rows]) and (out[rows:] == 7).all()
    kv = [torch.full((rows + 5, hk, x), 7.0, dtype=dt, device="cuda") for x in (w, wv)]
    _mod().gather(*cache, *places, rows + 5, dtype=dt, out=kv)
    table, start, cu = (x.cpu().numpy() for x in places)
    for x, codes, scale in zip(kv, want[:2], want[2:]):
        assert (x[rows:] == 7).all()
        for i in range(count):
            for r in range(cu[i], cu[i + 1]):
                p = start[i] + r - cu[i]
                at = table[i, p // page]
                value = torch.tensor(codes[at, :, p % page].astype(np.float32) * scale[at][:, None]).to(dt)
                assert torch.equal(x[r].cpu(), value)


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("lens,window", [([(70000, 1)], 0), ([(69999, 1)], 5000), ([(40000, 3), (0, 0), (12, 1), (65000, 1)], 0), ([(20000, 40)], 0), ([(20000, 40)], 700)])
@pytest.mark.parametrize("mode", ["softmax", "softmax_plus_one"])
def test_long_sequences(lens, window, mode, dt):
    """Sequences that many CTAs share, whole ones and windows of them; near keys among far ones, so that every part of the axis counts."""
    page, h, hk, w, wv = 64, 4, 2, 32, 32
    n_pages = sum(-(-(a + c) // page) for a, c in lens) + 1
    cache = _random_cache(n_pages, hk, page, w, wv, seed=5)
    q = (1.5 * torch.randn(sum(c for _, c in lens), h, w, generator=torch.Generator().manual_seed(9))).to(dt).cuda()
    places = _places(lens, page, n_pages)
    got = _attend(q, cache, places, window=window, mode=mode)
    assert torch.equal(got, _mod().attend(q, *cache, *places, window=window, mode=mode))  # the same bits again


@pytest.mark.parametrize("dt", [F16, BF16])
def test_flat_rows_keep_their_small_weights(dt):
    """One near key, and 65535 far ones of weight about 2^-25.5 each, which alone carry values.  Weights are rounded to 11 bits, or to 2^-31 of the largest
    where that is more."""
    n, w, page = 65536, 64, 256
    cache = _empty(n // page, 1, page, w, w)
    cache[2].fill_(25.5 * math.log(2.0) / math.sqrt(w) / 100)
    cache[3].fill_(1.0 / 100)
    for x in cache[:2]:
        x.fill_(100)
        x[0, 0, 0] = 0
    places = (torch.arange(n // page, dtype=torch.int32, device="cuda")[None], torch.tensor([n - 1], dtype=torch.int32, device="cuda"),
              torch.tensor([0, 1], dtype=torch.int32, device="cuda"))
    vo = _mod().attend(torch.zeros(1, 1, w, dtype=dt, device="cuda"), *cache, *places)
    x, one = -math.sqrt(w) * 100 * float(cache[2][0, 0]), 100 * float(cache[3][0, 0])
    far = (n - 1) * math.exp(x)
    want = far / (1 + far) * one
    e = 4 * U * (math.sqrt(w) + 8) * abs(x) + 8 * U * abs(x)
    tol = (n - 1) * 2.0 ** -31 * one + (2.0 ** -11 + torch.finfo(dt).eps / 2 + 4 * e + 16 * U + 4 * U * math.sqrt(n)) * want
    assert tol < 0.05 * want
    assert ((vo.double() - want).abs() <= tol).all()


def test_two_calls_at_once():
    """Calls of two streams on one cache, each with its own places, and two captured calls replayed in turn."""
    lens = [(5000, 1)] * 5
    cache = _random_cache(400, 2, 64, 64, 64)
    places = _places(lens, 64, 400)
    qs = [torch.randn(5, 8, 64, generator=torch.Generator().manual_seed(i)).to(BF16).cuda() for i in range(2)]
    m = _mod()
    want = [m.attend(q, *cache, *places).clone() for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    got = []
    for _ in range(10):
        for s, q in zip(streams, qs):
            with torch.cuda.stream(s):
                got.append(m.attend(q, *cache, *places))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i % 2]) for i, x in enumerate(got))
    graphs, held = [torch.cuda.CUDAGraph() for _ in qs], []
    for graph, q in zip(graphs, qs):
        with torch.cuda.graph(graph):
            held.append(m.attend(q, *cache, *places))
    for _ in range(3):
        for graph in graphs:
            graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(held, want))
