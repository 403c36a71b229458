"""L1 attention from a paged cache in 8 bits: the serving side of `l1attn_masked_cuda.L1AttnMasked` (an ADDITIONAL set of operators).

A page holds `page` tokens of one sequence for all heads; tokens of a page share one float scale per head, for keys and for values
(value = scale * code, codes -127 .. 127).  The cache of one layer is four tensors:

    k_codes int8 [n_pages, hk, page, w]    v_codes int8 [n_pages, hk, page, wv]    k_scale, v_scale float32 [n_pages, hk]

The functions take them with the places of this call's tokens, all on the device (so a captured call replays with new contents):

    table int32 [n_seqs, max_pages]   page of a sequence's position p: table[i, p // page]
    start int32 [n_seqs]              position of the sequence's first row
    cu    int32 [n_seqs + 1]          its rows of the token tensors: cu[i] .. cu[i + 1]

    append(k, v, *cache, table, start, cu)                quantise new tokens into their pages
    vo = attend(q, *cache, table, start, cu, ...)         every row attends to its sequence up to its own position
    k, v = gather(*cache, table, start, cu, rows)         what the cache holds, as floating values
    copy_pages(*cache, src, dst)                          pages to other places

`L1Cache` owns the tensors of all layers and the bookkeeping: sequences, pages that forks share, copies on write, compaction.

    cache = L1Cache(n_pages, hk, w, n_layers=2)
    s = cache.open()
    plan = cache.extend([s], [prompt_len])                # room for the tokens
    for layer in range(2):
        cache.append(plan, k, v, layer)
        vo = cache.attend(plan, q, layer)
    t = cache.fork(s); cache.truncate(s, 10); cache.close(t); cache.compact()

Rows behind cu[n_seqs] (a padded batch) are neither read nor written.  Page ids, starts and offsets out of range are never followed: their
tokens are left out (keys are not seen, gathered rows and the outputs of queries without a place are zeros), and `status` (int32 [1], optional; `L1Cache.check()`) becomes non-zero.  float32, float16 and bfloat16 tokens, float32 sums.
No gradients (a cache answers, it does not train) and no CPU path.
"""
import torch

import l1attn_cache_cuda_drv  # torch must be imported first: the driver links against libtorch
from l1attn_masked_cuda import _options, _tensors

PAGES = (16, 32, 64, 128, 256)


def append(k, v, k_codes, v_codes, k_scale, v_scale, table, start, cu, status=None):
    """Quantises k [rows, hk, w], v [rows, hk, wv] (strided views will do) into the pages of their positions.

    Per page and head the scale is max |x| / 127 over the page's new tokens, or stays where it is larger and the page holds earlier tokens of the
    sequence; code = x / scale to the nearest (ties to even); when a scale grows the earlier codes follow it.  No two sequences of a call may write
    the same page.  NaN is stored as 0, infinities as the largest code."""
    l1attn_cache_cuda_drv.append(k, v, (k_codes, v_codes, k_scale, v_scale), table, start, cu, status)


def gather(k_codes, v_codes, k_scale, v_scale, table, start, cu, rows, dtype=torch.float32, out=None, status=None):
    """(k [rows, hk, w], v [rows, hk, wv]): the values that the cache holds at the given positions, rounded to dtype.  rows: cu[-1], or more
    (rows behind it are left as they were in `out`, and undefined without).  out: a pair of contiguous tensors to write."""
    k_out, v_out = (None, None) if out is None else out
    return tuple(l1attn_cache_cuda_drv.gather((k_codes, v_codes, k_scale, v_scale), table, start, cu, rows, dtype, k_out, v_out, status))


def attend(q, k_codes, v_codes, k_scale, v_scale, table, start, cu, mode="softmax", window=0, softcap=0.0, slopes=None, max_len=None, out=None, status=None):
    """vo [rows, h, wv] of q [rows, h, w] (h a multiple of hk; strided views will do): the weights of `L1AttnMasked` with causal=True over the keys at
    the row's own and earlier positions of its sequence.  Append a step's keys before its queries attend.

    max_len: the longest start + count, where the program knows it (default: what the table has room for); it shapes the launch alone.
    out: a contiguous tensor to write, not q itself; rows behind cu[-1] are left as they were in it, and undefined without it.

    16-bit q: query / scale is rounded to float16 next to codes that it holds exactly, weights to 11 bits (float16: 22) or 2^-29 of the
    row's largest, whatever the scales of its pages' values, up to 2^58 times one another; float32 q: float32 throughout."""
    mode, _, window, softcap = _options(mode, True, window, softcap)
    return l1attn_cache_cuda_drv.attend(q, (k_codes, v_codes, k_scale, v_scale), table, start, cu, mode, window, softcap, slopes, -1 if max_len is None else max(0, int(max_len)),
                                        out, status)


def copy_pages(k_codes, v_codes, k_scale, v_scale, src, dst, status=None):
    """Page src[i] -> page dst[i], codes and scales of all heads; with a leading layer dimension, of all layers.  src, dst: int32 tensors on the device
    (they are not checked beyond their range), or lists, which are: a page may be copied to several places, but no destination may occur twice or
    be a source."""
    _tensors(k_codes=k_codes, v_codes=v_codes, k_scale=k_scale, v_scale=v_scale)
    if not isinstance(src, torch.Tensor) or not isinstance(dst, torch.Tensor):
        if not k_codes.is_cuda:
            raise RuntimeError("k_codes must be a CUDA tensor")
        src, dst = [int(i) for i in src], [int(i) for i in dst]
        if len(src) != len(dst) or len(set(dst)) != len(dst) or set(src) & set(dst) or any(not 0 <= i < k_codes.shape[-4] for i in src + dst):
            raise ValueError("pages must be in range, and no destination may occur twice or be a source")
        if not src:
            return
        src, dst = _upload(src + dst, k_codes.device).view(2, -1)
    l1attn_cache_cuda_drv.copy_pages((k_codes, v_codes, k_scale, v_scale), src, dst, status)


def _upload(values, device):
    """Host integers to the device without waiting for it."""
    with torch.cuda.device(device):
        return torch.tensor(values, dtype=torch.int32).pin_memory().to(device, non_blocking=True)


class Plan:
    """Where one call's new tokens go: `table`, `start`, `cu` on the device, `rows` tokens in all, `max_len` the longest sequence behind it.
    Good until the cache next extends, forks, truncates, closes or compacts."""

    def __init__(self, flat, n, max_pages):
        self.flat, self.n, self.max_pages = flat, n, max_pages
        self.table = flat[:n * max_pages].view(n, max_pages)
        self.start = flat[n * max_pages:n * max_pages + n]
        self.cu = flat[n * max_pages + n:]


class _Sequence:
    __slots__ = ("pages", "length")

    def __init__(self, pages=(), length=0):
        self.pages, self.length = list(pages), length


class L1Cache:
    """Pages of `n_layers` layers and who holds them.  The bookkeeping is on the host; device work is enqueued on the current stream, so calls on one cache
    belong on one stream (or streams that wait for one another)."""

    def __init__(self, n_pages, n_kv_heads, width, v_width=None, n_layers=1, page=64, device="cuda"):
        v_width = width if v_width is None else v_width
        for name, x, lo, hi in (("n_pages", n_pages, 1, 0x7fffffff), ("n_kv_heads", n_kv_heads, 1, 65535), ("width", width, 1, 256), ("v_width", v_width, 1, 256),
                                ("n_layers", n_layers, 1, 32767)):
            if isinstance(x, bool) or int(x) != x or not lo <= x <= hi:
                raise ValueError("%s must be a whole number from %d to %d" % (name, lo, hi))
        if page not in PAGES:
            raise ValueError("page must be one of %s" % (PAGES,))
        if torch.device(device).type != "cuda":
            raise RuntimeError("the cache needs a CUDA device: there is no CPU path")
        self.n_pages, self.page, self.n_layers = int(n_pages), int(page), int(n_layers)
        mk = lambda *s, dt: torch.zeros(n_layers, n_pages, n_kv_heads, *s, dtype=dt, device=device)  # noqa: E731
        self.k_codes, self.v_codes = mk(page, width, dt=torch.int8), mk(page, v_width, dt=torch.int8)
        self.k_scale, self.v_scale = mk(dt=torch.float32), mk(dt=torch.float32)
        self.status = torch.zeros(1, dtype=torch.int32, device=self.k_codes.device)
        self._book = PageBook(n_pages, page)
        self._epoch = 0

    # -- sequences

    def open(self):
        """A new, empty sequence; its id."""
        return self._book.open()

    def length(self, seq):
        return self._book.seq(seq).length

    def pages(self, seq):
        """The ids of a sequence's pages, in order."""
        return list(self._book.seq(seq).pages)

    @property
    def free_pages(self):
        return len(self._book.free)

    def close(self, seq):
        """Gives a sequence up; pages that no fork shares become free."""
        self._book.close(seq)
        self._epoch += 1

    def fork(self, seq):
        """A new sequence with the same tokens.  Nothing is copied: the two share their pages until one of them writes into a shared one."""
        self._epoch += 1
        return self._book.fork(seq)

    def truncate(self, seq, length):
        """Keeps a sequence's first `length` tokens."""
        self._book.truncate(seq, length)
        self._epoch += 1

    def extend(self, seqs, counts, into=None, room=0):
        """Room for counts[i] more tokens of seqs[i] (ids, each once) -> the Plan of the call.  A last page that a fork shares is copied first.
        Raises RuntimeError, and changes nothing, when the pages do not suffice.
        room: columns of the plan's table beyond need, for a plan that later calls refresh in place (`into`: a plan of as many sequences;
        its tensors keep their addresses, as a captured step needs)."""
        seqs, counts = [int(s) for s in seqs], [int(c) for c in counts]
        if len(seqs) != len(counts) or not seqs or min(counts) < 0 or len(set(seqs)) != len(seqs):
            raise ValueError("extend takes sequences, each once, and a count of 0 or more for each")
        if isinstance(room, bool) or int(room) != room or room < 0:
            raise ValueError("room must be a whole number of columns")
        if sum(counts) > 0x7fffffff:
            raise ValueError("a call's tokens must fit int32")
        need = max(max(-(-(self.length(s) + c) // self.page) for s, c in zip(seqs, counts)), 1)
        if into is not None and (into.n != len(seqs) or into.max_pages < need):
            raise ValueError("the plan to refresh has room for %d sequences of %d pages, not %d of %d" % (into.n, into.max_pages, len(seqs), need))
        starts = [self.length(s) for s in seqs]
        copies = self._book.extend(seqs, counts)
        width = need + int(room) if into is None else into.max_pages
        flat, total = [], 0
        for s in seqs:
            p = self._book.seq(s).pages
            flat += p + [0] * (width - len(p))
        flat += starts + [0]
        for c in counts:
            total += c
            flat.append(total)
        if copies:
            copy_pages(self.k_codes, self.v_codes, self.k_scale, self.v_scale, *zip(*copies))
        if into is None:
            plan = Plan(_upload(flat, self.k_codes.device), len(seqs), width)
        else:
            plan = into
            with torch.cuda.device(self.k_codes.device):
                plan.flat.copy_(torch.tensor(flat, dtype=torch.int32).pin_memory(), non_blocking=True)
        self._epoch += 1
        plan.rows, plan.max_len, plan.epoch, plan.cache = total, max(a + c for a, c in zip(starts, counts)), self._epoch, self
        return plan

    def compact(self):
        """Moves the pages in use to the front; returns how many moved.  Free pages then follow each other at the end."""
        moves = self._book.compact()
        if moves:
            copy_pages(self.k_codes, self.v_codes, self.k_scale, self.v_scale, *zip(*moves))
        self._epoch += 1
        return len(moves)

    # -- the operators

    def layer(self, layer):
        """The four tensors of one layer, as the functions of this module take them."""
        if isinstance(layer, bool) or not 0 <= layer < self.n_layers:
            raise ValueError("layer must be 0 to %d" % (self.n_layers - 1))
        return self.k_codes[layer], self.v_codes[layer], self.k_scale[layer], self.v_scale[layer]

    def _places(self, plan):
        if plan.cache is not self or plan.epoch != self._epoch:
            raise RuntimeError("this plan is no longer good: the cache has been extended, forked, truncated, closed or compacted since")
        return plan.table, plan.start, plan.cu

    def append(self, plan, k, v, layer=0):
        """Quantises the plan's tokens, k [rows, hk, w] and v [rows, hk, wv], into a layer."""
        places = self._places(plan)
        if k.shape[0] < plan.rows:
            raise RuntimeError("k and v must have the plan's %d rows" % plan.rows)
        append(k, v, *self.layer(layer), *places, status=self.status)

    def attend(self, plan, q, layer=0, mode="softmax", window=0, softcap=0.0, slopes=None, out=None, max_len=None):
        """vo [rows, h, wv] of the plan's queries q [rows, h, w]; see `attend`.  max_len: for a step that is captured, the longest that its replays will see."""
        places = self._places(plan)
        if q.shape[0] < plan.rows:
            raise RuntimeError("q must have the plan's %d rows" % plan.rows)
        return attend(q, *self.layer(layer), *places, mode=mode, window=window, softcap=softcap, slopes=slopes, max_len=plan.max_len if max_len is None else max_len,
                      out=out, status=self.status)

    def gather(self, seqs, layer=0, dtype=torch.float32):
        """(k, v, cu) of whole sequences: their values one behind the other, and where each begins."""
        seqs = [self._book.seq(s) for s in seqs]
        if not seqs:
            raise ValueError("gather takes one sequence or more")
        width = max(max(len(s.pages) for s in seqs), 1)
        cu = [0]
        for s in seqs:
            cu.append(cu[-1] + s.length)
        flat = _upload([p for s in seqs for p in s.pages + [0] * (width - len(s.pages))] + [0] * len(seqs) + cu, self.k_codes.device)
        at = Plan(flat, len(seqs), width)
        return gather(*self.layer(layer), at.table, at.start, at.cu, cu[-1], dtype=dtype, status=self.status) + (cu,)

    def check(self):
        """Waits for the device; raises if a call on this cache met a page id, a start or an offset out of range."""
        code = int(self.status.item())
        if code:
            self.status.zero_()
            raise RuntimeError("a call on this cache met a page id, a start or an offset out of range (code %d): its tokens were left out" % code)


class PageBook:
    """Which sequence holds which pages (host only).  Low ids are handed out first."""

    def __init__(self, n_pages, page):
        self.page = page
        self.refs = [0] * n_pages
        self.free = list(range(n_pages - 1, -1, -1))  # the last is the next
        self.seqs, self.next_id = {}, 0

    def seq(self, i):
        if i not in self.seqs:
            raise ValueError("no open sequence %r" % (i,))
        return self.seqs[i]

    def _new(self, s):
        i = self.next_id
        self.next_id += 1
        self.seqs[i] = s
        return i

    def open(self):
        return self._new(_Sequence())

    def fork(self, i):
        s = self.seq(i)
        for p in s.pages:
            self.refs[p] += 1
        return self._new(_Sequence(s.pages, s.length))

    def _drop(self, pages):
        for p in reversed(pages):
            self.refs[p] -= 1
            if self.refs[p] == 0:
                self.free.append(p)

    def close(self, i):
        self._drop(self.seq(i).pages)
        del self.seqs[i]

    def truncate(self, i, length):
        s = self.seq(i)
        if isinstance(length, bool) or int(length) != length or not 0 <= length <= s.length:
            raise ValueError("a sequence of %d tokens cannot be cut to %r" % (s.length, length))
        keep = -(-int(length) // self.page)
        self._drop(s.pages[keep:])
        del s.pages[keep:]
        s.length = int(length)

    def extend(self, ids, counts):
        """Pages for the new tokens; the pairs (from, to) of last pages to copy because a fork shares them."""
        seqs = [self.seq(i) for i in ids]
        shared = [s.pages[-1] if c and s.length % self.page and self.refs[s.pages[-1]] > 1 else None for s, c in zip(seqs, counts)]
        # of several that write into one shared page, as many copy as leave its holders one each
        left, copy = {}, []
        for p in shared:
            if p is not None:
                left[p] = left.get(p, self.refs[p]) - 1
            copy.append(p is not None and left[p] >= 1)
        need = sum(copy) + sum(-(-(s.length + c) // self.page) - len(s.pages) for s, c in zip(seqs, counts))
        if need > len(self.free):
            raise RuntimeError("the cache is full: %d pages needed, %d free" % (need, len(self.free)))
        pairs = []
        for s, c, cp in zip(seqs, counts, copy):
            if cp:
                old, new = s.pages[-1], self.free.pop()
                self.refs[old] -= 1
                self.refs[new] = 1
                s.pages[-1] = new
                pairs.append((old, new))
            s.length += c
            while len(s.pages) * self.page < s.length:
                p = self.free.pop()
                self.refs[p] = 1
                s.pages.append(p)
        return pairs

    def compact(self):
        used = len(self.refs) - len(self.free)
        holes = [p for p in range(used) if self.refs[p] == 0]
        moves = dict(zip((p for p in range(used, len(self.refs)) if self.refs[p]), holes))
        for old, new in moves.items():
            self.refs[new], self.refs[old] = self.refs[old], 0
        for s in self.seqs.values():
            s.pages = [moves.get(p, p) for p in s.pages]
        self.free = list(range(len(self.refs) - 1, used - 1, -1))
        return list(moves.items())
