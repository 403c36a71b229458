"""The 8-bit cache on the GPU against its definition in float64.

append: scales and codes are equal to the definition's, bit for bit (exact quotients, ties to even).  gather: one product, one rounding.
attend, elementwise, u = 2^-24, half = torch.finfo(t).eps / 2:
  float32  scores off by e = 4 u (sqrt(w) + 8) scale sum(|q| + |k|) + 8 u |x|, weights by 2 e + 16 u of themselves, sums of n keys by 4 u sqrt(n)
  16 bits  also: q / (page's scale) is rounded to float16, clipped to +-128 with the rest kept apart: each term is off by a uniform error of at most
           2^-11 |q|, 6 standard deviations of their sum 6 scale 2^-11 sqrt(sum q^2 / 3); weights are rounded to 11 bits; the output by half of itself
"""
import math
import random

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = 2.0 ** -24


def _mod():
    import l1attn_cache_cuda
    return l1attn_cache_cuda


def _empty(n_pages, hk, page, w, wv, fill=0):
    mk = lambda x: torch.full((n_pages, hk, page, x), fill, dtype=torch.int8, device="cuda")  # noqa: E731
    return mk(w), mk(wv), torch.zeros(n_pages, hk, device="cuda"), torch.zeros(n_pages, hk, device="cuda")


def _places(lens, page, n_pages, seed=0, spare=1):
    """Random distinct pages for sequences of (start, count); (table, start, cu) on the device."""
    ids = random.Random(seed).sample(range(n_pages), sum(-(-(a + c) // page) for a, c in lens))
    width = max(1, max(-(-(a + c) // page) for a, c in lens)) + spare
    table = np.full((len(lens), width), -7, np.int32)  # (never looked at past the last page)
    for i, (a, c) in enumerate(lens):
        m = -(-(a + c) // page)
        table[i, :m], ids = ids[:m], ids[m:]
    dev = lambda x: torch.tensor(np.asarray(x, np.int32), device="cuda")  # noqa: E731
    return dev(table), dev([a for a, _ in lens]), dev(np.cumsum([0] + [c for _, c in lens]))


def _append_reference(cache, k, v, table, start, cu):
    """Codes and scales after an append, page by page and head by head in float64."""
    out = [x.cpu().numpy().copy() for x in cache]
    table, start, cu = (x.cpu().numpy() for x in (table, start, cu))
    page = out[0].shape[2]
    for which, x in enumerate((k, v)):
        x = x.detach().double().cpu().numpy()
        codes, scales = out[which], out[2 + which]
        for i in range(len(start)):
            a, c = int(start[i]), int(cu[i + 1] - cu[i])
            for p in range(a // page, -(-(a + c) // page)):
                lo, hi = max(a, p * page), min(a + c, (p + 1) * page)
                if lo >= hi:
                    continue
                at, held = table[i, p], lo - p * page
                new = x[cu[i] + lo - a:cu[i] + hi - a]  # [tokens, hk, w]
                for h in range(codes.shape[1]):
                    y = new[:, h]
                    fin = np.abs(y[np.isfinite(y)])
                    old = scales[at, h] if held else np.float32(0)
                    now = max(np.float32((fin.max() if fin.size else 0.0) / 127.0), old)
                    if held and now > old:
                        codes[at, h, :held] = np.rint(codes[at, h, :held].astype(np.float64) * float(old) / float(now))
                    with np.errstate(invalid="ignore"):
                        z = np.zeros_like(y) if now == 0 else np.clip(np.nan_to_num(np.rint(y / float(now)), nan=0.0, posinf=127, neginf=-127), -127, 127)
                    codes[at, h, held:hi - p * page] = z
                    scales[at, h] = now
    return out


def _same(cache, want):
    for x, r in zip(cache, want):
        assert np.array_equal(x.cpu().numpy(), r)


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("page,hk,w,wv,lens", [
    (16, 2, 64, 64, [(0, 1), (5, 1), (16, 1), (31, 2)]), (64, 3, 65, 7, [(0, 64), (63, 2), (10, 0), (100, 150)]), (32, 1, 1, 3, [(0, 33)]),
    (128, 2, 128, 128, [(0, 300), (127, 1), (128, 129)]), (256, 1, 256, 200, [(3, 600)]), (16, 4, 40, 80, [(i, 17 - i) for i in range(17)])])
def test_append(page, hk, w, wv, lens, dt):
    n_pages = sum(-(-(a + c) // page) for a, c in lens) + 3
    cache = _empty(n_pages, hk, page, w, wv, fill=77)
    places = _places(lens, page, n_pages)
    for t in (cache[2], cache[3]):
        t.copy_(torch.linspace(0.01, 0.05, t.numel()).view(t.shape))  # (some scales grow, some stay)
    g = torch.Generator().manual_seed(w)
    rows = sum(c for _, c in lens)
    k, v = (torch.randn(rows, hk, x, generator=g).to(dt).cuda() for x in (w, wv))
    want = _append_reference(cache, k, v, *places)
    _mod().append(k, v, *cache, *places)
    _same(cache, want)
    _mod().append(k, v, *cache, *places)  # the same tokens again: nothing changes
    _same(cache, want)


@pytest.mark.parametrize("dt", [F32, F16, BF16])
def test_append_values_off_the_usual(dt):
    """Quotients at exactly one half, all zeros, one value alone, tiny and huge values, NaN and infinities."""
    page, w = 16, 32
    rows = []
    tie = torch.arange(w).float() - 15.5
    tie[0] = 127.0  # scale 1: quotients n + 1/2
    rows += [tie, torch.zeros(w), torch.eye(w)[3] * 5, torch.linspace(-3, 3, w)]
    tiny = float(torch.finfo(dt).smallest_normal)
    rows += [torch.linspace(-1, 1, w) * tiny, torch.linspace(-1, 1, w) * float(torch.finfo(dt).max)]
    bad = torch.linspace(-2, 2, w)
    bad[4], bad[5], bad[6] = math.nan, math.inf, -math.inf
    rows += [bad, torch.full((w,), math.nan), torch.full((w,), math.inf)]
    x = torch.stack(rows).to(dt).cuda()[:, None]
    lens = [(0, 1)] * len(rows)
    cache = _empty(len(rows), 1, page, w, w)
    places = _places(lens, page, len(rows))
    want = _append_reference(cache, x, x, *places)
    _mod().append(x, x, *cache, *places)
    _same(cache, want)


def test_append_one_token_at_a_time():
    """Scales grow token by token and the codes that are there follow, each time by the definition."""
    g = torch.Generator().manual_seed(3)
    cache = _empty(4, 2, 16, 24, 24)
    x = torch.randn(40, 2, 24, generator=g) * torch.linspace(0.2, 3, 40)[:, None, None]
    places = _places([(0, 40)], 16, 4)
    for t in range(40):
        now = (places[0], torch.tensor([t], dtype=torch.int32, device="cuda"), torch.tensor([0, 1], dtype=torch.int32, device="cuda"))
        k, v = x[t:t + 1].to(BF16).cuda(), (-x[t:t + 1]).to(BF16).cuda()
        want = _append_reference(cache, k, v, *now)
        _mod().append(k, v, *cache, *now)
        _same(cache, want)


@pytest.mark.parametrize("dt", [F32, F16, BF16])
def test_gather_and_strided_append(dt):
    lens = [(0, 70), (0, 0), (3, 20), (0, 1)]
    page, hk, w, wv = 32, 2, 48, 33
    cache = _empty(9, hk, page, w, wv)
    places = _places(lens, page, 9)
    rows, g = 91, torch.Generator().manual_seed(1)
    kv = torch.randn(rows + 4, hk, w + wv, generator=g).to(dt).cuda()  # k and v are slices; four rows belong to nobody
    want = _append_reference(cache, kv[..., :w], kv[..., w:], *places)
    _mod().append(kv[..., :w], kv[..., w:], *cache, *places)
    _same(cache, want)
    out = tuple(torch.full((rows + 4, hk, x), 9.0, dtype=dt, device="cuda") for x in (w, wv))
    _mod().gather(*cache, *places, rows + 4, dtype=dt, out=out)
    assert (out[0][rows:] == 9).all() and (out[1][rows:] == 9).all()
    r = 0
    for i, (a, c) in enumerate(lens):
        for j in range(c):
            at, pos = int(places[0][i, (a + j) // page]), (a + j) % page
            for t, codes, scale in ((out[0], cache[0], cache[2]), (out[1], cache[1], cache[3])):
                assert torch.equal(t[r], (codes[at, :, pos].float() * scale[at][:, None]).to(dt))
            r += 1


def _random_cache(n_pages, hk, page, w, wv, seed=0):
    g = torch.Generator().manual_seed(seed)
    mk = lambda x: torch.randn(n_pages, hk, page, x, generator=g).mul_(32).round_().clamp_(-127, 127).to(torch.int8).cuda()  # noqa: E731
    sc = lambda: ((0.5 + torch.rand(n_pages, hk, generator=g)) * 4 / 127).cuda()  # noqa: E731
    return mk(w), mk(wv), sc(), sc()


def attend_reference(q, cache, table, start, cu, mode="softmax", window=0, softcap=0.0, slopes=None):
    k_codes, v_codes, k_scale, v_scale = cache
    rows, h, w = q.shape
    hk, page = k_codes.shape[1:3]
    half, low = torch.finfo(q.dtype).eps / 2, q.dtype != F32
    want = torch.zeros(rows, h, v_codes.shape[3], dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(want)
    scale = 1 / math.sqrt(w)
    for i in range(len(start)):
        a, r0, r1 = int(start[i]), int(cu[i]), int(cu[i + 1])
        n = a + r1 - r0
        if r0 == r1:
            continue
        ids = table[i, :-(-n // page)].long()
        t, s = torch.arange(a, n, device="cuda")[:, None], torch.arange(n, device="cuda")[None]
        ok = s <= t
        if window:
            ok &= t - s < window
        for j in range(hk):
            k, v = ((c[ids, j].double() * sc[ids, j].double()[:, None, None]).flatten(0, 1)[:n] for c, sc in ((k_codes, k_scale), (v_codes, v_scale)))
            for i_h in range(j * h // hk, (j + 1) * h // hk):
                x64 = q[r0:r1, i_h].double()
                x = -torch.cdist(x64, k, p=1.0) * scale
                e = 4 * U * (math.sqrt(w) + 8) * scale * (x64.abs().sum(1)[:, None] + k.abs().sum(1)[None]) + 8 * U * x.abs()
                if low:
                    e = e + 6 * scale * 2.0 ** -11 * (x64.square().sum(1) / 3).sqrt()[:, None]
                if softcap:
                    x = softcap * torch.tanh(x / softcap)
                if slopes is not None:
                    x = x - slopes[i_h].double() * (t - s)
                    e = e + 8 * U * x.abs()
                x = x.masked_fill(~ok, -math.inf)
                if mode == "exp":
                    p = torch.exp(x)
                else:
                    extra = torch.full_like(x[:, :1], 0.0 if mode == "softmax_plus_one" else -math.inf)
                    p = torch.softmax(torch.cat([x, extra], 1), 1)[:, :-1]
                o, mass = p @ v, p @ v.abs()
                # errors of the weights: common ones cancel in the normalised forms at worst they add
                rel = 2 * e.amax(1, keepdim=True) + 16 * U + (2.0 ** -11 if low else 0.0) + 4 * U * math.sqrt(n)
                want[r0:r1, i_h] = o
                tol[r0:r1, i_h] = rel * mass + half * o.abs() + 1e-30 + (2.0 ** -25 if q.dtype == F16 else 0.0)
    return want, tol


def _attend(q, cache, places, rows=None, **options):
    got = _mod().attend(q, *cache, *places, **options)
    options.pop("max_len", None)
    want, tol = attend_reference(q, cache, *places, **options)
    rows = int(places[2][-1])
    err = (got.double() - want).abs()[:rows]
    assert torch.isfinite(got[:rows]).all() and (err <= tol[:rows]).all(), "worst %.3g of the bound" % float((err / tol[:rows]).max())
    return got


LENS = [[(0, 1)], [(499, 1)], [(0, 5), (16, 1), (63, 2), (7, 0), (200, 130)], [(i * 37, 1) for i in range(20)], [(3000, 1), (1, 1)], [(100, 33), (0, 64), (65, 1)]]


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("page,h,hk,w,wv", [(16, 8, 8, 64, 64), (64, 8, 2, 128, 128), (32, 3, 1, 96, 40), (128, 32, 2, 64, 128), (64, 2, 1, 33, 65), (256, 12, 2, 80, 16)])
def test_attend(page, h, hk, w, wv, lens, dt):
    n_pages = sum(-(-(a + c) // page) for a, c in lens) + 2
    cache = _random_cache(n_pages, hk, page, w, wv, seed=w)
    g = torch.Generator().manual_seed(len(lens))
    q = torch.randn(sum(c for _, c in lens), h, w, generator=g).to(dt).cuda()
    _attend(q, cache, _places(lens, page, n_pages, seed=1))


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("w,wv", [(256, 256), (129, 200), (1, 1), (8, 3), (200, 16)])
def test_attend_widths(w, wv, dt):
    lens = [(150, 3), (0, 20)]
    cache = _random_cache(20, 2, 16, w, wv)
    q = torch.randn(23, 6, w, generator=torch.Generator().manual_seed(1)).to(dt).cuda()
    _attend(q, cache, _places(lens, 16, 20))


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("mode", ["softmax", "softmax_plus_one", "exp"])
@pytest.mark.parametrize("window,softcap,bias", [(0, 0.0, False), (1, 0.0, False), (100, 5.0, True), (0, 2.0, False), (700, 0.0, True)])
@pytest.mark.parametrize("max_len", [None, 0, 64, 100000])
def test_attend_options(mode, window, softcap, bias, dt, max_len):
    """Windows, caps, biases and modes, with the launch shaped for any length."""
    lens = [(1500, 1), (40, 3), (700, 40)]
    cache = _random_cache(60, 2, 64, 64, 64, seed=2)
    q = (0.7 * torch.randn(44, 8, 64, generator=torch.Generator().manual_seed(5))).to(dt).cuda()
    slopes = torch.linspace(0.5, -0.0005, 8, device="cuda") if bias else None
    _attend(q, cache, _places(lens, 64, 60), mode=mode, window=window, softcap=softcap, slopes=slopes, max_len=max_len)


@pytest.mark.parametrize("dt", [F16, BF16])
def test_attend_queries_far_from_the_codes(dt):
    """Queries much larger than what the page's scale reaches, and pages of very different scales, down to zero."""
    lens = [(250, 2), (30, 1)]
    cache = _random_cache(30, 2, 16, 64, 64, seed=8)
    cache[2].mul_(torch.logspace(-6, 1, 30, device="cuda")[:, None])
    cache[2][5] = 0
    places = _places(lens, 16, 30, seed=4)
    q = torch.randn(3, 4, 64, generator=torch.Generator().manual_seed(2)).cuda()
    q[0] *= 30
    q[:, :, 7] = 100.0
    _attend((q * 0.3).to(dt), cache, places)


def test_attend_views_streams_and_graphs():
    lens = [(300, 2), (70, 1)]
    cache = _random_cache(12, 2, 64, 64, 64, seed=3)
    places = _places(lens, 64, 12)
    g = torch.Generator().manual_seed(9)
    wide = torch.randn(5, 12, 64, generator=g).to(BF16).cuda()
    q = wide[:, :8]  # two rows belong to no sequence
    out = torch.full((5, 8, 64), 3.0, dtype=BF16, device="cuda")
    m = _mod()
    first = m.attend(q, *cache, *places, out=out)
    assert first is out and (out[3:] == 3).all()
    assert torch.equal(_attend(q.contiguous(), cache, places)[:3], out[:3])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = m.attend(q, *cache, *places)
    side.synchronize()
    assert torch.equal(other[:3], out[:3])
    k, v = (torch.randn(3, 2, 64, generator=g).to(BF16).cuda() for _ in range(2))
    graph = torch.cuda.CUDAGraph()
    keep = [x.clone() for x in cache]
    with torch.cuda.graph(graph):
        m.append(k, v, *cache, *places)
        held = m.attend(q, *cache, *places)
        values = m.gather(*cache, *places, 3)
    for x, y in zip(cache, keep):
        x.copy_(y)
    places[1].copy_(torch.tensor([200, 71], dtype=torch.int32))
    k.copy_(k.roll(1, 0))
    graph.replay()
    torch.cuda.synchronize()
    got = [x.clone() for x in (held[:3],) + values]
    for x, y in zip(cache, keep):
        x.copy_(y)
    m.append(k, v, *cache, *places)
    assert torch.equal(m.attend(q, *cache, *places)[:3], got[0])
    assert all(torch.equal(a, b) for a, b in zip(m.gather(*cache, *places, 3), got[1:]))


def test_copy_pages():
    m = _mod()
    for layers, shape in ((None, (11, 3, 16, 40)), (3, (3, 11, 2, 64, 128))):
        g = torch.Generator().manual_seed(1)
        codes = [torch.randint(-127, 128, shape[:-1] + (x,), generator=g, dtype=torch.int8).cuda() for x in (shape[-1], 33)]
        scales = [torch.rand(shape[:-2], generator=g).cuda() for _ in range(2)]
        cache = codes + scales
        want = [x.clone() for x in cache]
        src, dst = [4, 4, 0, 10], [1, 2, 3, 9]
        for x in want:
            y = x if layers else x[None]
            y[:, dst] = y[:, src].clone()
        m.copy_pages(*cache, src, dst)
        assert all(torch.equal(a, b) for a, b in zip(cache, want))
        m.copy_pages(*cache, torch.tensor([1], dtype=torch.int32, device="cuda"), torch.tensor([0], dtype=torch.int32, device="cuda"))
        for x in want:
            y = x if layers else x[None]
            y[:, 0] = y[:, 1]
        assert all(torch.equal(a, b) for a, b in zip(cache, want))
        for bad in (([1], [1]), ([1, 2], [3, 3]), ([11], [0]), ([0], [-1]), ([0, 1], [2]), ([0, 1], [1, 2])):
            with pytest.raises(ValueError):
                m.copy_pages(*cache, *bad)
        m.copy_pages(*cache, [], [])


def test_a_long_cache():
    """Codes past 2^31 bytes, and positions whose page lies there."""
    page, hk, w = 256, 2, 128
    n_pages = (1 << 31) // (page * hk * w) + 40
    cache = [torch.zeros(n_pages, hk, page, x, dtype=torch.int8, device="cuda") for x in (w, w)] + [torch.zeros(n_pages, hk, device="cuda") for _ in range(2)]
    last = list(range(n_pages - 5, n_pages))
    table = torch.tensor([last], dtype=torch.int32, device="cuda")
    at = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    g = torch.Generator().manual_seed(2)
    k, v = (torch.randn(1200, hk, w, generator=g).to(BF16).cuda() for _ in range(2))
    m = _mod()
    m.append(k, v, *cache, table, at(0), at(0, 1200))
    small = [x[n_pages - 5:].clone() for x in cache]
    near = torch.arange(5, dtype=torch.int32, device="cuda")[None]
    q = torch.randn(2, 4, w, generator=g).to(BF16).cuda()
    a = m.attend(q, *cache, table, at(1198), at(0, 2))
    assert torch.equal(a, m.attend(q, *small, near, at(1198), at(0, 2)))
    _attend(q, small, (near, at(1198), at(0, 2)))
    m.copy_pages(*cache, [n_pages - 1], [n_pages - 7])
    assert all(torch.equal(x[n_pages - 7], x[n_pages - 1]) for x in cache)


def test_bad_places_are_left_out():
    """(Host tests show that these are resolved within range.)  The rest of the call is right, and the status tells."""
    m = _mod()
    cache = _random_cache(8, 2, 16, 32, 32)
    at = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    q = torch.randn(4, 2, 32, device="cuda").to(BF16)
    status = at(0)
    good = m.attend(q, *cache, at(3, 1, 3, 1).view(2, 2), at(20, 18), at(0, 2, 4), status=status)
    assert int(status) == 0
    out = torch.zeros_like(good)
    m.attend(q, *cache, at(3, 1, 3, 1).view(2, 2), at(20, -5), at(0, 2, 4), status=status, out=out)
    assert int(status) != 0 and torch.equal(out[:2], good[:2]) and not out[2:].any()
    for table in (at(3, 99, 3, 1).view(2, 2), at(3, -1, 3, 1).view(2, 2)):
        status.zero_()
        got = m.attend(q, *cache, table, at(20, 18), at(0, 2, 4), status=status)
        assert int(status) != 0 and torch.isfinite(got).all() and torch.equal(got[2:], good[2:])
        before = [x.clone() for x in cache]
        status.zero_()
        m.append(q, q, *cache, table, at(16, 0), at(0, 4, 4), status=status)
        assert int(status) != 0 and all(torch.equal(x, y) for x, y in zip(before, cache))
        k, v = m.gather(*cache, table, at(16, 0), at(0, 4, 4), 4)
        assert not k.any() and not v.any()
    status.zero_()
    m.copy_pages(*cache, at(1, 77), at(0, 2), status=status)
    assert int(status) != 0


def test_serving_with_forks_and_compaction():
    """A run of everything together: prompts in pieces, tokens one by one, forks that write on, truncation, closing, compaction, two layers -- against
    attention over what `gather` says the cache holds, and against a replay of every sequence in a cache of its own."""
    m = _mod()
    rng = random.Random(7)
    hk, h, w, layers = 2, 6, 64, 2
    cache = m.L1Cache(40, hk, w, n_layers=layers, page=16)
    g = torch.Generator().manual_seed(11)
    history = {}  # id -> list of (length before, tokens appended, per layer k and v)
    token = lambda n: [torch.randn(n, 2 * hk, w, generator=g).to(BF16).cuda() for _ in range(layers)]  # noqa: E731

    def step(ids, counts):
        plan = cache.extend(ids, counts)
        kv = token(plan.rows)
        for layer in range(layers):
            k, v = kv[layer].split([hk, hk], 1)
            cache.append(plan, k, v, layer)
            q = torch.randn(plan.rows, h, w, generator=g).to(BF16).cuda()
            got = cache.attend(plan, q, layer, softcap=20.0)
            want, tol = attend_reference(q, cache.layer(layer), plan.table, plan.start, plan.cu, softcap=20.0)
            assert ((got.double() - want).abs() <= tol).all()
        at = 0
        for i, c in zip(ids, counts):
            history[i] = history[i] + [(cache.length(i) - c, [x[at:at + c] for x in kv])]
            at += c

    def opened():
        i = cache.open()
        history[i] = []
        return i

    for _ in range(3):
        opened()
    for n in range(40):
        ids = list(history)
        what = rng.choice(["step", "step", "step", "fork", "close", "truncate", "compact", "open"])
        if what == "open" or not ids:
            opened()
        elif what == "step":
            some = rng.sample(ids, rng.randint(1, len(ids)))
            try:
                step(some, [rng.choice([0, 1, 1, 1, 20]) for _ in some])
            except RuntimeError as e:
                assert "full" in str(e)
                victim = rng.choice(ids)
                cache.close(victim)
                del history[victim]
        elif what == "fork":
            i = rng.choice(ids)
            history[cache.fork(i)] = list(history[i])
        elif what == "close":
            i = rng.choice(ids)
            cache.close(i)
            del history[i]
        elif what == "truncate":
            i = rng.choice(ids)
            n = rng.randint(0, cache.length(i))
            cache.truncate(i, n)
            history[i] = history[i] + [(n, None)]
        else:
            cache.compact()
    assert cache.compact() >= 0 and history
    cache.check()
    for i, events in history.items():
        if not cache.length(i):
            continue
        alone = m.L1Cache(40, hk, w, n_layers=layers, page=16)
        s = alone.open()
        for at, kv in events:
            alone.truncate(s, at)
            if kv is not None and kv[0].shape[0]:
                plan = alone.extend([s], [kv[0].shape[0]])
                for layer in range(layers):
                    alone.append(plan, *kv[layer].split([hk, hk], 1), layer)
        for layer in range(layers):
            for a, b in zip(cache.gather([i], layer), alone.gather([s], layer)):
                assert torch.equal(torch.as_tensor(a), torch.as_tensor(b))


def test_plans():
    """A refreshed plan keeps its addresses and serves a captured step; an old one is refused."""
    m = _mod()
    cache = m.L1Cache(20, 2, 64, page=16)
    a, b = cache.open(), cache.open()
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(30, 2, 64, generator=g).to(BF16).cuda() for _ in range(2))
    plan = cache.extend([a, b], [20, 10], room=3)
    cache.append(plan, k, v)
    step = cache.extend([a, b], [1, 1], room=4)
    with pytest.raises(RuntimeError, match="no longer good"):
        cache.append(plan, k, v)
    with pytest.raises(RuntimeError, match="rows"):
        cache.append(step, k[:1], v[:1])
    q1, k1, v1 = (torch.randn(2, x, 64, generator=g).to(BF16).cuda() for x in (4, 2, 2))
    cache.append(step, k1, v1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.append(step, k1, v1)
        held = cache.attend(step, q1, max_len=96)
    for _ in range(25):
        address = step.table.data_ptr()
        cache.extend([a, b], [1, 1], into=step)
        assert step.table.data_ptr() == address
        for x in (q1, k1, v1):
            x.copy_(torch.randn(x.shape, generator=g))
        graph.replay()
        want, tol = attend_reference(q1, cache.layer(0), step.table, step.start, step.cu)
        assert ((held.double() - want).abs() <= tol).all()
    with pytest.raises(ValueError):
        cache.extend([a], [1], into=step)
    for bad in (([a, a], [1, 1]), ([a], [-1]), ([], []), ([a], [1, 2])):
        with pytest.raises(ValueError):
            cache.extend(*bad)
    with pytest.raises(ValueError):
        cache.extend([99], [1])
    before, free = cache.length(a), cache.free_pages
    with pytest.raises(RuntimeError, match="full"):
        cache.extend([a], [1000])
    assert cache.length(a) == before and cache.free_pages == free
    cache.check()


def test_serves_what_training_trained():
    """Prompt and tokens through the cache give what masked attention gives on the values that the cache holds."""
    from l1attn_masked_cuda import L1AttnMasked
    m = _mod()
    n, h, hk, w = 90, 4, 2, 64
    g = torch.Generator().manual_seed(21)
    q, k, v = (torch.randn(n, x, w, generator=g).cuda() for x in (h, hk, hk))
    slopes = torch.tensor([0.2, 0.1, 0.05, 0.0], device="cuda")
    cache = m.L1Cache(8, hk, w, page=16)
    s = cache.open()
    got = []
    for a, c in ((0, 64), (64, 16), (80, 1), (81, 1), (82, 8)):
        plan = cache.extend([s], [c])
        cache.append(plan, k[a:a + c], v[a:a + c])
        got.append((a, c, cache.attend(plan, q[a:a + c], window=50, softcap=10.0, slopes=slopes)))
    for a, c, vo in got[-1:]:  # (codes of a page that fills up may still change: the last call's keys are what gather says)
        kk, vv, _ = cache.gather([s])
        full = L1AttnMasked(window=50, softcap=10.0)(q[None], kk[None], vv[None], slopes=slopes)[0]
        assert float((vo - full[a:a + c]).abs().max()) <= 2e-5 * float(full.abs().max())


def test_refusals():
    m = _mod()
    cache = _random_cache(4, 2, 16, 32, 24)
    at = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    ok = (at(0, 1).view(1, 2), at(0), at(0, 3))
    k, v, q = (torch.zeros(3, i, x, device="cuda") for i, x in ((2, 32), (2, 24), (4, 32)))
    assert m.attend(q, *cache, *ok).shape == (3, 4, 24)
    for bad in ((k[:, :1], v), (k[..., :5], v), (k.half(), v), (k.double(), v.double()), (k.cpu(), v), (k, v[:2])):
        with pytest.raises(RuntimeError):
            m.append(*bad, *cache, *ok)
    for bad in (q[:, :3], q[..., :7], q.double(), q.cpu(), q[:, :0]):
        with pytest.raises(RuntimeError):
            m.attend(bad, *cache, *ok)
    for i in range(4):
        for change in (lambda t: t.cpu(), lambda t: t.double(), lambda t: t[..., :1, :] if t.dim() > 2 else t[:, :1], lambda t: t.transpose(0, 1)):
            x = list(cache)
            x[i] = change(x[i])
            with pytest.raises(RuntimeError):
                m.attend(q, *x, *ok)
    for i, change in ((0, at(0, 1)), (1, at(0, 0)), (2, at(0)), (0, ok[0].long()), (1, ok[1].cpu()), (2, ok[2].float())):
        x = list(ok)
        x[i] = change
        with pytest.raises(RuntimeError):
            m.attend(q, *cache, *x)
        with pytest.raises(RuntimeError):
            m.append(k, v, *cache, *x)
        with pytest.raises(RuntimeError):
            m.gather(*cache, *x, 3)
    with pytest.raises(RuntimeError):
        m.attend(q, *cache, *ok, out=torch.zeros(3, 4, 32, device="cuda"))
    with pytest.raises(RuntimeError):
        m.attend(q, *cache, *ok, slopes=torch.zeros(3, device="cuda"))
    with pytest.raises(ValueError):
        m.attend(q, *cache, *ok, mode="none")
    with pytest.raises(RuntimeError):
        m.gather(*cache, *ok, 3, dtype=torch.float64)
    with pytest.raises(RuntimeError):
        m.copy_pages(*cache, at(0).long(), at(1))
    assert m.attend(q[:0], *cache, *ok).shape == (0, 4, 24)
    c = m.L1Cache(4, 2, 32, n_layers=2)
    for layer in (-1, 2, True):
        with pytest.raises(ValueError):
            c.layer(layer)
    with pytest.raises(ValueError):
        c.gather([])
