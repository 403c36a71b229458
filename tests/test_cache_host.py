"""The host side of the 8-bit cache: who holds which pages, what is refused, and how the kernels resolve places that may be wrong."""
import ctypes
import random

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import l1attn_cabi  # noqa: E402
from l1attn_cache_cuda import L1Cache, PageBook, copy_pages  # noqa: E402


def _check_book(b):
    held = [0] * len(b.refs)
    for s in b.seqs.values():
        assert len(s.pages) == -(-s.length // b.page) and len(set(s.pages)) == len(s.pages)
        for p in s.pages:
            held[p] += 1
    assert held == b.refs and sorted(b.free) == [p for p, r in enumerate(b.refs) if r == 0]


def test_book_shares_copies_and_frees():
    b = PageBook(6, 16)
    a = b.open()
    assert b.extend([a], [20]) == [] and b.seq(a).pages == [0, 1]
    f, g = b.fork(a), b.fork(a)
    assert b.extend([a, f, g], [1, 1, 1]) == [(1, 2), (1, 3)]  # the last holder keeps the page
    assert [b.seq(x).pages for x in (a, f, g)] == [[0, 2], [0, 3], [0, 1]]
    b.close(a)
    assert b.compact() == [(3, 2)] and [b.seq(x).pages for x in (f, g)] == [[0, 2], [0, 1]]
    with pytest.raises(RuntimeError, match="full"):
        b.extend([f, g], [40, 60])
    _check_book(b)
    assert b.seq(f).length == 21
    b.truncate(f, 16)
    assert b.seq(f).pages == [0] and b.extend([f], [1]) == []  # a whole shared page is not written
    for bad in (-1, 18, True, 1.5):
        with pytest.raises(ValueError):
            b.truncate(f, bad)
    with pytest.raises(ValueError):
        b.close(a)


def test_book_under_random_use():
    """Every page's contents followed as a dict: forks keep what they held, whatever the others do."""
    rng = random.Random(4)
    b, page = PageBook(40, 16), 16
    store, truth = {}, {}
    for step in range(3000):
        what = rng.choice(["open", "extend", "extend", "extend", "fork", "close", "truncate", "compact"])
        ids = list(truth)
        try:
            if what == "open":
                truth[b.open()] = []
            elif what == "extend" and ids:
                some = rng.sample(ids, rng.randint(1, min(4, len(ids))))
                counts = [rng.randint(0, 30) for _ in some]
                for old, new in b.extend(some, counts):
                    assert (old, new) != (new, old)
                    store[new] = dict(store[old])
                for s, c in zip(some, counts):
                    for _ in range(c):
                        token, pos = rng.random(), len(truth[s])
                        truth[s].append(token)
                        assert b.refs[b.seq(s).pages[pos // page]] == 1  # never into a shared page
                        store.setdefault(b.seq(s).pages[pos // page], {})[pos % page] = token
            elif what == "fork" and ids:
                s = rng.choice(ids)
                truth[b.fork(s)] = list(truth[s])
            elif what == "close" and ids:
                s = rng.choice(ids)
                b.close(s)
                del truth[s]
            elif what == "truncate" and ids:
                s = rng.choice(ids)
                n = rng.randint(0, len(truth[s]))
                b.truncate(s, n)
                del truth[s][n:]
            elif what == "compact":
                moves = b.compact()
                assert not {x for x, _ in moves} & {y for _, y in moves}
                for old, new in moves:
                    store[new] = store.pop(old)
                used = sum(r > 0 for r in b.refs)
                assert all(b.refs[:used]) and not any(b.refs[used:])
        except RuntimeError as e:
            assert "full" in str(e)
        _check_book(b)
        for s, tokens in truth.items():
            assert [store[b.seq(s).pages[i // page]][i % page] for i in range(len(tokens))] == tokens


def _places(table, start, cu, n_pages=10, page=16):
    buf = (ctypes.c_double * 64)()
    p = ctypes.addressof(buf) // 16 * 16 + 16
    t, s, u, status = (np.ascontiguousarray(x, np.int32) for x in (table, start, cu, [0]))
    c = l1attn_cabi.Cache.__new__(l1attn_cabi.Cache)
    ctypes.Structure.__init__(c, p, p, p, p, n_pages, page, 2, 4, 4, t.ctypes.data, s.ctypes.data, u.ctypes.data, t.shape[0], t.shape[1], status.ctypes.data)
    return c, status, (buf, t, s, u)


def _unit(c, rows, unit, num, den, extra, slot=0):
    out = np.zeros(6, np.int32)
    assert l1attn_cabi.lib().l1attn_test_cache_unit(ctypes.byref(c), rows, unit, num, den, extra, slot, out.ctypes.data) == 0
    return out.tolist()


@pytest.mark.parametrize("num,den,extra", [(1, 16, 2), (4, 16, 1), (3, 16, 1), (1, 1, 0), (24, 16, 1)])
def test_units_cover_every_sequence(num, den, extra):
    """Each sequence gets the units it needs, in order, and none belongs to two; empty sequences among them."""
    rng = random.Random(num * den)
    for _ in range(30):
        counts = [rng.choice([0, 1, 2, 5, 16, 17, 40]) for _ in range(rng.randint(1, 12))]
        cu = np.cumsum([0] + counts)
        rows = int(cu[-1])
        if rows == 0:
            continue
        c, status, keep = _places([[0] * 4] * len(counts), [0] * len(counts), cu)
        got = {}
        for u in range(rows * num // den + extra * len(counts)):
            seq, row, count, start, mine, _ = _unit(c, rows, u, num, den, extra)
            assert row == cu[seq] and count == counts[seq] and mine >= 0
            got.setdefault(seq, []).append(mine)
        for i, n in enumerate(counts):
            need = -(-n * num // den) + (extra - 1 if den > 1 and num == 1 and n else 0)  # (a page more when the first is not entered at its start)
            assert got.get(i, [])[:need] == list(range(need)), (counts, i)
        assert status[0] == 0


@pytest.mark.parametrize("table,start,cu,rows", [
    ([[0]], [0], [0, 5], 4), ([[0]], [0], [-1, 3], 4), ([[0]], [0], [3, 1], 4), ([[0]], [-1], [0, 4], 4), ([[0]], [14], [0, 4], 4), ([[0]], [100], [0, 4], 4),
    ([[0]], [2147483647], [0, 4], 4), ([[0], [0]], [0, 0], [0, 4, 2], 4), ([[0], [0]], [0, 0], [0, 2147483647, 4], 4), ([[0], [0]], [0, 0], [2, -2147483648, 9], 4)])
def test_bad_places_stay_in_range(table, start, cu, rows):
    """Whatever the offsets say, rows stay in the token tensors and positions in the table, and the status tells."""
    c, status, keep = _places(table, start, cu)
    for num, den, extra in ((1, 16, 2), (4, 16, 1), (1, 1, 0)):
        for u in range(rows * num // den + extra * len(table) + 1):
            seq, row, count, first, mine, page = _unit(c, rows, u, num, den, extra)
            assert 0 <= seq < len(table) and 0 <= row and count >= 0 and row + count <= rows and first >= 0 and (count == 0 or first + count <= 16)
    assert status[0] == -4


@pytest.mark.parametrize("page", [-1, 10, 2147483647, -2147483648])
def test_bad_pages_are_not_followed(page):
    c, status, keep = _places([[3, page]], [0], [0, 20])
    assert _unit(c, 20, 0, 1, 16, 2, slot=0)[5] == 3 and status[0] == 0
    assert _unit(c, 20, 0, 1, 16, 2, slot=1)[5] == -1 and status[0] == -4


def _abi(what, **change):
    lib = l1attn_cabi.lib()
    c, status, keep = _places([[0]], [0], [0, 2])
    p = c.k_codes
    mask = l1attn_cabi.Mask()
    for x in ("causal", "window", "mode", "softcap", "doc", "prefix"):
        if x in change:
            setattr(mask, x, change.pop(x))
    a = dict(q=p, k=p, v=p, vo=p, strides=(ctypes.c_int64 * 4)(8, 4, 8, 4), rows=2, heads=2, max_len=100, dtype=l1attn_cabi.F16, layers=1, src=p, dst=p, n=1, work=p)
    for x in list(change):
        if x in dict(c._fields_):
            setattr(c, x, change.pop(x))
    a.update(change)
    ref = None if a.get("no_cache") else ctypes.byref(c)
    if what == "append":
        return lib.l1attn_cache_append(ref, a["k"], a["v"], a["strides"], a["rows"], a["dtype"], None)
    if what == "gather":
        return lib.l1attn_cache_gather(ref, a["k"], a["v"], a["rows"], a["dtype"], None)
    if what == "copy":
        return lib.l1attn_cache_copy_pages(ref, a["layers"], a["src"], a["dst"], a["n"], None)
    return lib.l1attn_cache_attend(ref, a["q"], a["strides"], a["vo"], a["work"], a["rows"], a["heads"], a["max_len"], None if a.get("no_mask") else ctypes.byref(mask),
                                   a["dtype"], None)


@pytest.mark.parametrize("what", ["append", "gather", "attend"])
@pytest.mark.parametrize("change,code", [
    (dict(no_cache=True), -1), (dict(rows=-1), -1), (dict(dtype=l1attn_cabi.F64), -1), (dict(page=8), -1), (dict(page=48), -1), (dict(page=512), -1), (dict(width=0), -1),
    (dict(width=257), -2), (dict(v_width=300), -2), (dict(n_kv_heads=0), -1), (dict(n_kv_heads=65536), -2), (dict(n_pages=-1), -1), (dict(n_seqs=-1), -1),
    (dict(max_pages=-1), -1), (dict(max_pages=1 << 28), -2), (dict(table=None), -1), (dict(start=None), -1), (dict(cu=None), -1), (dict(k_codes=None), -1),
    (dict(v_scale=None), -1), (dict(k_codes=8), -6), (dict(k_scale=2), -6), (dict(status=3), -6), (dict(table=2), -6)])
def test_abi_refusals(what, change, code):
    assert _abi(what, **dict(change)) == code


def test_abi_refusals_of_one_call():
    for change in (dict(no_mask=True), dict(causal=0), dict(doc=16), dict(prefix=16), dict(window=-1), dict(mode=3), dict(softcap=float("nan")), dict(heads=3), dict(heads=0),
                   dict(q=None), dict(vo=None), dict(strides=None)):
        assert _abi("attend", **change) == -1, change
    assert _abi("attend", q=3) == -6 and _abi("append", k=3) == -6 and _abi("gather", v=3) == -6
    assert _abi("append", k=None) == -1 and _abi("append", strides=None) == -1 and _abi("gather", v=None) == -1
    assert _abi("copy", src=None) == -1 and _abi("copy", n=-1) == -1 and _abi("copy", layers=-1) == -1 and _abi("copy", dst=6) == -6 and _abi("copy", n=0) == 0
    for what in ("append", "gather", "attend"):
        assert _abi(what, rows=0) == 0 and _abi(what, n_seqs=0) == 0


@pytest.mark.parametrize("what", ["append", "gather", "attend"])
def test_abi_refuses_what_no_kernel_covers(what):
    """A cache without pages (bad ids fall back on the first), and positions whose tiles would end past int."""
    assert _abi(what, n_pages=0) == -1
    assert _abi(what, max_pages=(1 << 26) + 1) == -2
    assert what != "attend" or _abi(what, rows=1 << 30, heads=4) == -2


def test_extend_refuses_before_it_changes_anything():
    cache = L1Cache.__new__(L1Cache)
    cache.page, cache._book, cache._epoch = 16, PageBook(4, 16), 0
    s = cache._book.open()
    for change in (dict(room=-1), dict(room=1.5), dict(room=True), dict(counts=[1 << 31])):
        with pytest.raises(ValueError):
            cache.extend([s], **dict(dict(counts=[1]), **change))
    assert cache.length(s) == 0 and len(cache._book.free) == 4


def test_module_refusals():
    for bad in (dict(n_pages=0), dict(width=0), dict(width=257), dict(v_width=1.5), dict(n_layers=0), dict(page=24), dict(n_kv_heads=True)):
        with pytest.raises(ValueError):
            L1Cache(**dict(dict(n_pages=4, n_kv_heads=2, width=8), **bad))
    with pytest.raises(RuntimeError, match="CUDA"):
        L1Cache(4, 2, 8, device="cpu")
    codes, scale = torch.zeros(4, 2, 16, 8, dtype=torch.int8), torch.zeros(4, 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        copy_pages(codes, codes, scale, scale, [0], [1])
