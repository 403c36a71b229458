"""Rows of sequences whose places are out of range: zeros in everything that is read at them, never what the memory held before."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_cache_gpu import BF16, F16, F32, _mod, _random_cache  # noqa: E402


def _at(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# (table rows of two pages of 16, starts, offsets, which rows of the call have a place): seven rows of three sequences, an eighth behind them
PLACES = [([20, -5, 3], [0, 2, 5, 7], [0, 1, 5, 6]), ([30, 0, 31], [0, 4, 4, 7], [0, 1, 4]), ([2147483647, 40, 0], [0, 3, 6, 7], [6]),
          ([0, 0, 0], [-2, 3, 5, 7], [3, 4, 5, 6]), ([-1, -1, -1], [0, 2, 2, 7], [])]


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("start,cu,placed", PLACES)
@pytest.mark.parametrize("w,wv,max_len", [(32, 32, None), (40, 24, None), (32, 32, 5000), (200, 130, None), (200, 130, 5000)])
def test_rows_without_a_place_are_zeros(w, wv, max_len, start, cu, placed, dt):
    m = _mod()
    cache = _random_cache(8, 2, 16, w, wv, seed=1)
    table, start, cu = _at(3, 1, 0, 2, 7, 5).view(3, 2), _at(*start), _at(*cu)
    g = torch.Generator().manual_seed(2)
    q = torch.randn(8, 6, w, generator=g).to(dt).cuda()
    status = _at(0)
    out = torch.full((8, 6, wv), math.nan, dtype=dt, device="cuda")
    m.attend(q, *cache, table, start, cu, out=out, status=status, max_len=max_len)
    assert int(status) != 0
    kv = tuple(torch.full((8, 2, x), math.nan, dtype=dt, device="cuda") for x in (w, wv))
    status.zero_()
    m.gather(*cache, table, start, cu, 8, dtype=dt, out=kv, status=status)
    assert int(status) != 0
    without = [r for r in range(7) if r not in placed]
    for x in (out,) + kv:
        assert x[7].isnan().all() and not x[without].any() and not x[:7].isnan().any()
        assert all(x[r].any() for r in placed)


def test_many_sequences_some_without_a_place():
    """More sequences than a warp has lanes; what has a place is what a call without the others gives."""
    m = _mod()
    cache = _random_cache(100, 2, 16, 64, 64, seed=3)
    n = 90
    table = torch.arange(n, dtype=torch.int32, device="cuda")[:, None].contiguous()
    start, cu = torch.zeros(n, dtype=torch.int32, device="cuda"), 3 * torch.arange(n + 1, dtype=torch.int32, device="cuda")
    bad = torch.arange(n, device="cuda") % 7 == 3
    for dt in (F32, BF16):
        q = torch.randn(3 * n, 4, 64, generator=torch.Generator().manual_seed(1)).to(dt).cuda()
        want = m.attend(q, *cache, table, start, cu)
        out = torch.full_like(want, math.nan)
        m.attend(q, *cache, table, torch.where(bad, -1, start).to(torch.int32), cu, out=out)
        rows = bad.repeat_interleave(3)
        assert not out[rows].any()
        assert torch.equal(out[~rows], want[~rows]) or float((out[~rows].double() - want[~rows].double()).abs().max()) <= torch.finfo(dt).eps * float(want.abs().max())


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("cu,zero", [([0, 9, 3, 7], [0, 1, 2]), ([0, 3, 3, 9], [3, 4, 5, 6]), ([0, 2, -1, 7], [2, 3, 4, 5, 6]), ([0, 3, 9, 7], [3, 4, 5, 6])])
def test_offsets_out_of_range(cu, zero, dt):
    """One offset beyond the rows or below zero: the sequences that it is no end of stay right, gathered rows hold values or zeros."""
    m = _mod()
    cache = _random_cache(8, 2, 16, 32, 32, seed=1)
    table, start = _at(3, 1, 0, 2, 7, 5).view(3, 2), _at(1, 5, 2)
    good = [i for i in range(3) if 0 <= cu[i] <= cu[i + 1] <= 7]
    q = torch.randn(7, 4, 32, generator=torch.Generator().manual_seed(2)).to(dt).cuda()
    status = _at(0)
    out = torch.full((7, 4, 32), math.nan, dtype=dt, device="cuda")
    m.attend(q, *cache, table, start, _at(*cu), out=out, status=status)
    assert int(status) != 0
    kv = tuple(torch.full((7, 2, 32), math.nan, dtype=dt, device="cuda") for _ in range(2))
    status.zero_()
    m.gather(*cache, table, start, _at(*cu), 7, dtype=dt, out=kv, status=status)
    assert int(status) != 0 and not any(x.isnan().any() for x in kv)
    if dt != F32:  # (the 16-bit kernel looks at every sequence for itself)
        assert not out[zero].any()
        for i in good:
            rows = slice(cu[i], cu[i + 1])
            alone = m.attend(q[rows].contiguous(), *cache, table[i:i + 1], start[i:i + 1], _at(0, cu[i + 1] - cu[i]))
            assert ((out[rows].double() - alone.double()).abs() <= 2 * torch.finfo(dt).eps * (1 + alone.double().abs())).all()
