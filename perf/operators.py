"""Performance cases of the operators for language models: masked attention for training and prompts, and a cache of keys and values in 8 bits.

`kind` says which operator a case drives:

  train    l1attn_masked_cuda.L1AttnMasked, output and gradients
  prefill  the same, output alone
  attend   l1attn_cache_cuda.attend: new tokens attend to what a paged 8-bit cache holds of their sequences
  append   l1attn_cache_cuda.append: new tokens are quantised into the pages; then l1attn_cache_cuda.gather reads the sequences back
  move     l1attn_cache_cuda.copy_pages: pages copied to other places (forks, compaction)

Where `own` is false, `run` computes the same in elementary torch operations.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ELEMENT = {"f32": 4, "f16": 2, "bf16": 2}
CHUNK = 1 << 30  # elements of the largest intermediate of a plain form


def _masked(kind, b, n, h, hk, w, wv, dtype, mode="softmax", causal=True, window=0, softcap=0.0, bias=False, docs=0, prefix=False, packed=False):
    return dict(kind=kind, b=b, n=n, h=h, hk=hk, w=w, wv=wv, dtype=dtype, mode=mode, causal=causal, window=window, softcap=softcap, bias=bias, docs=docs,
                prefix=prefix, packed=packed)


def _attend(seqs, ctx, new, h, hk, w, wv, page, dtype, mode="softmax", window=0, softcap=0.0, bias=False, ragged=True):
    return dict(kind="attend", seqs=seqs, ctx=ctx, new=new, h=h, hk=hk, w=w, wv=wv, page=page, dtype=dtype, mode=mode, window=window, softcap=softcap, bias=bias,
                ragged=ragged)


def _append(seqs, ctx, new, hk, w, wv, page, dtype, ragged=True):
    return dict(kind="append", seqs=seqs, ctx=ctx, new=new, hk=hk, w=w, wv=wv, page=page, dtype=dtype, ragged=ragged)


def _move(pages, moved, hk, w, wv, page):
    return dict(kind="move", pages=pages, moved=moved, hk=hk, w=w, wv=wv, page=page)


def listed():
    return [
        # one training step of a small layer: short kernels, latency counts
        dict(_masked("train", 4, 128, 8, 8, 64, 64, "bf16"), name="train_small"),
        # a causal layer of ordinary size, heads of keys and values shared by four, scores capped; q, k, v are views of one projection
        dict(_masked("train", 2, 2048, 8, 2, 128, 128, "bf16", softcap=30.0, packed=True), name="train_causal"),
        # sizes off every multiple in float32: odd token count and width, a prefix that all tokens see, one more all-zero source row
        dict(_masked("train", 3, 501, 6, 3, 65, 40, "f32", mode="softmax_plus_one", prefix=True), name="train_odd_f32"),
        # a long prompt of packed documents with padding behind them, scores that fall with the distance
        dict(_masked("prefill", 1, 8192, 8, 2, 64, 64, "f16", bias=True, docs=5), name="prefill_documents"),
        # one token of one short sequence: latency
        dict(_attend(1, 500, 1, 8, 8, 64, 64, 16, "bf16", ragged=False), name="decode_one"),
        # a serving step: many sequences of all lengths, one new token each
        dict(_attend(64, 8192, 1, 32, 8, 128, 128, 64, "bf16"), name="decode_batch"),
        # two long sequences: a few rows against a long axis, with a bias and a cap
        dict(_attend(2, 100001, 1, 16, 2, 128, 128, 32, "f16", softcap=20.0, bias=True, ragged=False), name="decode_long"),
        # a piece of a prompt per sequence against what the cache holds already
        dict(_attend(4, 3001, 256, 8, 4, 64, 64, 64, "bf16", mode="softmax_plus_one"), name="chunk_prefill"),
        # the new token of every sequence of a serving step
        dict(_append(64, 200, 1, 8, 128, 128, 64, "bf16"), name="append_step"),
        # prompts of all lengths
        dict(_append(16, 100, 1501, 8, 128, 128, 64, "bf16"), name="append_prompts"),
        # copy on write: the last page of a few forked sequences
        dict(_move(512, 16, 4, 64, 64, 16), name="move_few"),
        # compaction: half of a cache moves
        dict(_move(8192, 4096, 8, 128, 128, 64), name="move_many"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    """One more case: sizes over their logarithm, heads shared or not, every type, odd widths now and then; no larger than the largest listed one."""
    kind = rng.choice(["train", "train", "prefill", "attend", "attend", "attend", "append", "move"])
    w = rng.choice([64, 128, 128, 64, 96, 80, 32, rng.randint(1, 128)])
    wv = w if rng.random() < 0.7 else rng.choice([64, 128, 32, rng.randint(1, 128)])
    hk = rng.choice([1, 2, 4, 8])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    mode = rng.choice(["softmax", "softmax", "softmax_plus_one"])
    softcap = rng.choice([0.0, 0.0, 20.0, 50.0])
    bias = rng.random() < 0.3
    if kind in ("train", "prefill"):
        h = hk * rng.choice([1, 1, 2, 4])
        b, n = _log(rng, 1, 8), _log(rng, 16, 4096)
        most = 4.0e9 if dtype != "f32" else 1.0e9
        while b * n * n * h * max(w, wv) > most:
            if b > 1:
                b = (b + 1) // 2
            else:
                n = n * 3 // 4
        causal = rng.random() < 0.8
        return _masked(kind, b, n, h, hk, w, wv, dtype, mode, causal, rng.choice([0, 0, max(1, n // 3)]), softcap, bias, rng.choice([0, 0, 3]),
                       causal and rng.random() < 0.2, w == wv and rng.random() < 0.5)
    page = rng.choice([16, 32, 64, 128])
    if kind == "attend":
        h = hk * rng.choice([1, 2, 4, 8, 3])
        seqs, ctx, new = _log(rng, 1, 64), _log(rng, 1, 30000), rng.choice([1, 1, 1, 4, _log(rng, 2, 300)])
        while seqs * ctx * hk * (w + wv) > 2.5e8 or seqs * new * ctx * h * w > 4e9:
            if seqs > 1:
                seqs //= 2
            else:
                new, ctx = (new + 1) // 2, ctx * 3 // 4
        return _attend(seqs, ctx, new, h, hk, w, wv, page, dtype, mode, rng.choice([0, 0, 1 + ctx // 2]), softcap, bias, rng.random() < 0.8)
    if kind == "append":
        seqs, ctx, new = _log(rng, 1, 64), _log(rng, 1, 400), rng.choice([1, _log(rng, 2, 1500)])
        while seqs * (ctx + new) * hk * (w + wv) > 4e7:
            seqs = max(1, seqs // 2)
            new = (new + 1) // 2
        return _append(seqs, ctx, new, hk, w, wv, page, dtype)
    pages = _log(rng, 64, 8192)
    while pages * page * hk * (w + wv) > 1.0e9:
        pages //= 2
    return _move(pages, max(1, int(pages * rng.uniform(0.01, 0.5))), hk, w, wv, page)


# ---------------------------------------------------------------------------------------------- what a case means

def _documents(case):
    """[b][n] document of every token, -1 for padding: unequal lengths, in another order in every row of the batch."""
    n, d = case["n"], case["docs"]
    doc = np.full((case["b"], n), -1, np.int32)
    used = n - n // 16
    for b in range(case["b"]):
        weights = [1 + (i + b) % d for i in range(d)]
        cuts = [used * sum(weights[:i]) // sum(weights) for i in range(d + 1)]
        for i in range(d):
            doc[b, cuts[i]:cuts[i + 1]] = i
    return doc


def _prefixes(case):
    return np.array([case["n"] * (b + 1) // (2 * case["b"] + 2) for b in range(case["b"])], np.int32)


def _pairs(case):
    """Pairs of query and key of a masked case that the masks leave, summed over the batch."""
    n, t, total = case["n"], np.arange(case["n"]), 0
    doc = _documents(case) if case["docs"] else None
    pre = _prefixes(case) if case["prefix"] else None
    for b in range(case["b"]):
        for t0 in range(0, n, 1024):
            tt, ss = t[t0:t0 + 1024, None], t[None, :]
            ok = np.ones((tt.shape[0], n), bool)
            if case["causal"]:
                ok &= ss <= tt
            if case["window"]:
                ok &= np.abs(tt - ss) < case["window"]
            if pre is not None:
                ok |= ss < pre[b]
            if doc is not None:
                ok &= (doc[b][t0:t0 + 1024, None] == doc[b][None, :]) & (doc[b][None, :] >= 0)
            total += int(ok.sum())
        if doc is None and pre is None:
            return total * case["b"]
    return total


def _lengths(case):
    """(tokens in the cache before the call, new tokens) of every sequence."""
    out = []
    for i in range(case["seqs"]):
        f = ((i + 1) * 0.6180339887498949) % 1.0 if case["ragged"] else 1.0
        g = ((i + 1) * 0.7548776662466927) % 1.0 if case["ragged"] else 1.0
        out.append((int(case["ctx"] * f), max(1, int(round(case["new"] * g)))))
    return out


def work(case):
    kind = case["kind"]
    if kind == "move":
        per = case["page"] * case["hk"] * (case["w"] + case["wv"]) + 8 * case["hk"]
        return {"bytes": 2 * case["moved"] * per, "flops": 0}
    w, wv, hk = case["w"], case["wv"], case["hk"]
    e = ELEMENT[case["dtype"]]
    if kind in ("train", "prefill"):
        rows, pairs = case["b"] * case["n"], _pairs(case) * case["h"]
        q, k, v, o = rows * case["h"] * w, rows * hk * w, rows * hk * wv, rows * case["h"] * wv
        if kind == "prefill":
            return {"bytes": e * (q + k + v + o), "flops": pairs * (2 * w + 2 * wv)}
        # forward 2 per term (difference, sum), backward 4 (difference, sign, two sums); value products 2, 2 + 2
        return {"bytes": e * (2 * (q + k + v) + 2 * o), "flops": pairs * (6 * w + 6 * wv)}
    old, new = sum(a for a, _ in _lengths(case)), sum(c for _, c in _lengths(case))
    if kind == "append":
        held = sum((a % case["page"]) for a, _ in _lengths(case))
        return {"bytes": hk * (w + wv) * (new * (e + 1) + held * 2 + (old + new) * (1 + 4)), "flops": hk * (w + wv) * (3 * new + old + new)}
    pairs = keys = 0
    for a, c in _lengths(case):
        reach = min(case["window"], a + c) if case["window"] else a + c
        keys += min(a + c, reach + c)
        pairs += sum(min(a + i + 1, reach) for i in range(c))
    return {"bytes": keys * hk * (w + wv + 8 / case["page"]) + new * case["h"] * (w + wv) * e, "flops": pairs * case["h"] * (2 * w + 2 * wv)}


# ---------------------------------------------------------------------------------------------- inputs

def _slopes(h):
    return 2.0 ** (-8.0 * np.arange(1, h + 1) / h)


def _cache(case, n_pages, g):
    """Pages as a running server holds them: values of about unit size, a scale for each page and head."""
    hk, page, dev = case["hk"], case["page"], g.device
    out = {}
    for name, width in (("k", case["w"]), ("v", case["wv"])):
        codes = torch.empty(n_pages, hk, page, width, dtype=torch.int8, device=dev)
        step = max(1, (1 << 28) // (hk * page * width))
        for i in range(0, n_pages, step):
            x = torch.empty(codes[i:i + step].shape, dtype=torch.float16, device=dev).normal_(0.0, 127.0 / 4.0, generator=g)
            codes[i:i + step] = x.clamp_(-127, 127).round_().to(torch.int8)
        out[name + "_codes"] = codes
        out[name + "_scale"] = (4.0 / 127.0) * (0.75 + 0.5 * torch.rand(n_pages, hk, device=dev, generator=g))
    return out


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    s = dict(case=case)
    kind, hk, w, wv = case["kind"], case["hk"], case["w"], case["wv"]
    if kind == "move":
        s.update(_cache(case, case["pages"], g))
        ids = torch.randperm(case["pages"], device=dev, generator=g)
        s["src"], s["dst"] = ids[:case["moved"]].to(torch.int32), ids[case["moved"]:2 * case["moved"]].to(torch.int32)
        return s
    dt = DTYPES[case["dtype"]]
    new = lambda *shape: torch.randn(*shape, device=dev, generator=g).to(dt)  # noqa: E731
    if kind in ("train", "prefill"):
        b, n, h = case["b"], case["n"], case["h"]
        if case["packed"]:
            s["q"], s["k"], s["v"] = new(b, n, h + 2 * hk, w).split([h, hk, hk], 2)
        else:
            s["q"], s["k"], s["v"] = new(b, n, h, w), new(b, n, hk, w), new(b, n, hk, wv)
        if kind == "train":
            for x in "qkv":
                s[x] = s[x].detach().requires_grad_(True)
            s["dvo"] = new(b, n, h, wv)
        s["slopes"] = torch.tensor(_slopes(h), dtype=torch.float32, device=dev) if case["bias"] else None
        s["doc"] = torch.tensor(_documents(case), device=dev) if case["docs"] else None
        s["prefix"] = torch.tensor(_prefixes(case), device=dev) if case["prefix"] else None
        return s
    lens = _lengths(case)
    need = [-(-(a + c) // case["page"]) for a, c in lens]
    table = np.zeros((len(lens), max(need)), np.int32)
    ids = np.random.RandomState(seed % (1 << 31)).permutation(sum(need) + 3)
    for i, m in enumerate(need):
        table[i, :m] = ids[sum(need[:i]):sum(need[:i]) + m]
    s.update(_cache(case, len(ids), g))
    s["table"] = torch.tensor(table, device=dev)
    s["start"] = torch.tensor([a for a, _ in lens], dtype=torch.int32, device=dev)
    s["cu"] = torch.tensor(np.cumsum([0] + [c for _, c in lens]), dtype=torch.int32, device=dev)
    s["end"], s["cu_all"] = s["start"] + s["cu"].diff(), torch.tensor(np.cumsum([0] + [a + c for a, c in lens]), dtype=torch.int32, device=dev)
    s["zero"] = torch.zeros_like(s["start"])
    total = sum(c for _, c in lens)
    s["max_new"], s["total_all"] = max(c for _, c in lens), sum(a + c for a, c in lens)
    if kind == "attend":
        s["q"] = new(total, case["h"], w)
        s["slopes"] = torch.tensor(_slopes(case["h"]), dtype=torch.float32, device=dev) if case["bias"] else None
    else:
        s["k"], s["v"] = 1.3 * new(total, hk, w), 0.9 * new(total, hk, wv)
    return s


# ---------------------------------------------------------------------------------------------- plain forms

def _weights(x, allowed, slope_distance, case):
    """Scores -> (weights, d(score)/d(uncapped score)); rows that the mask leaves empty have weights of zero."""
    dcap = None
    if case["softcap"]:
        th = torch.tanh(x / case["softcap"])
        x, dcap = case["softcap"] * th, 1 - th * th
    if slope_distance is not None:
        x = x - slope_distance
    x = x.masked_fill(~allowed, -math.inf)
    m = x.amax(-1, keepdim=True)
    m = m.clamp(min=0.0) if case["mode"] == "softmax_plus_one" else m.masked_fill(m == -math.inf, 0.0)
    p = torch.exp(x - m)
    l = p.sum(-1, keepdim=True)
    l = l + torch.exp(-m) if case["mode"] == "softmax_plus_one" else l.masked_fill(l == 0, 1.0)
    return p / l, dcap


def _plain_masked(s):
    case = s["case"]
    b, n, h, hk, w, wv = (case[x] for x in ("b", "n", "h", "hk", "w", "wv"))
    train, rep = case["kind"] == "train", h // hk
    heads = lambda x: x.detach().float().permute(0, 2, 1, 3)  # noqa: E731
    q, k, v = heads(s["q"]), heads(s["k"]).repeat_interleave(rep, 1), heads(s["v"]).repeat_interleave(rep, 1)
    vo = torch.empty(b, h, n, wv, device=q.device)
    if train:
        dvo = heads(s["dvo"])
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    step = max(1, CHUNK // (b * h * n * w))
    pos = torch.arange(n, device=q.device)
    for t0 in range(0, n, step):
        t1 = min(n, t0 + step)
        hi = t1 if case["causal"] and not case["prefix"] else n
        dist = (pos[t0:t1, None] - pos[None, :hi]).abs()
        ok = torch.ones_like(dist, dtype=torch.bool)
        if case["causal"]:
            ok = ok & (pos[None, :hi] <= pos[t0:t1, None])
        if case["window"]:
            ok = ok & (dist < case["window"])
        ok = ok[None, None]
        if s["prefix"] is not None:
            ok = ok | (pos[None, None, None, :hi] < s["prefix"][:, None, None, None])
        if s["doc"] is not None:
            ok = ok & (s["doc"][:, None, t0:t1, None] == s["doc"][:, None, None, :hi]) & (s["doc"][:, None, None, :hi] >= 0)
        d = q[:, :, t0:t1, None] - k[:, :, None, :hi]
        x = d.abs().sum(-1) * (-1.0 / math.sqrt(w))
        p, dcap = _weights(x, ok, None if s["slopes"] is None else s["slopes"][None, :, None, None] * dist, case)
        vo[:, :, t0:t1] = p @ v[:, :, :hi]
        if train:
            go = dvo[:, :, t0:t1]
            dv[:, :, :hi] += p.transpose(2, 3) @ go
            dx = p * (go @ v[:, :, :hi].transpose(2, 3) - (go * vo[:, :, t0:t1]).sum(-1, keepdim=True))
            if dcap is not None:
                dx = dx * dcap
            d = d.sign_().mul_((dx * (-1.0 / math.sqrt(w)))[..., None])
            dq[:, :, t0:t1] = d.sum(3)
            dk[:, :, :hi] -= d.sum(2)
    dt = DTYPES[case["dtype"]]
    back = lambda x: x.permute(0, 2, 1, 3).to(dt).contiguous()  # noqa: E731
    if not train:
        return back(vo)
    return {"vo": back(vo), "dq": back(dq), "dk": back(dk.reshape(b, hk, rep, n, w).sum(2)), "dv": back(dv.reshape(b, hk, rep, n, wv).sum(2))}


def _plain_attend(s):
    case = s["case"]
    h, hk, w, wv, page, seqs = (case[x] for x in ("h", "hk", "w", "wv", "page", "seqs"))
    rep, most = h // hk, s["table"].shape[1] * case["page"]
    dev, dt = s["q"].device, DTYPES[case["dtype"]]
    vo = torch.empty(s["q"].shape[0], h, wv, dtype=dt, device=dev)
    count = s["cu"].diff()
    new = s["max_new"]
    step = max(1, CHUNK // (new * h * most * max(w, wv)))
    pos = torch.arange(most, device=dev)
    row = torch.arange(new, device=dev)
    for i0 in range(0, seqs, step):
        sl = slice(i0, min(seqs, i0 + step))
        tab = s["table"][sl].long()
        values = lambda x: (s[x + "_codes"][tab].float() * s[x + "_scale"][tab][..., None, None]).transpose(1, 2).flatten(2, 3)  # noqa: E731, B023
        k, v = values("k"), values("v")  # [seqs, hk, most, width]
        at = (s["cu"][sl, None] + row).clamp(max=s["q"].shape[0] - 1).long()
        q = s["q"][at].float().reshape(-1, new, hk, rep, w).permute(0, 2, 1, 3, 4).reshape(-1, hk, new * rep, w)
        x = (q[:, :, :, None] - k[:, :, None]).abs().sum(-1) * (-1.0 / math.sqrt(w))
        t = (s["start"][sl, None] + row).repeat_interleave(rep, 1)[:, None, :, None]  # position of every row
        dist = t - pos
        ok = (dist >= 0) & ((dist < case["window"]) if case["window"] else True)
        slope = None if s["slopes"] is None else s["slopes"].reshape(1, hk, 1, rep).expand(1, hk, new, rep).reshape(1, hk, new * rep, 1) * dist
        p, _ = _weights(x, ok, slope, case)
        o = (p @ v).reshape(-1, hk, new, rep, wv).permute(0, 2, 1, 3, 4).reshape(-1, new, h, wv)
        real = row < count[sl, None]
        vo[at[real]] = o[real].to(dt)
    return vo


def _plain_append(s):
    """Quantises the new tokens page by page; a page that already holds tokens keeps the larger scale, its codes follow."""
    case = s["case"]
    page, dev = case["page"], s["k"].device
    count = s["cu"].diff()
    pages = (s["max_new"] + 2 * page - 2) // page  # that one sequence's new tokens may touch
    first = s["start"] // page
    token = first[:, None] * page + torch.arange(pages * page, device=dev)  # [seqs, pages * page] positions
    fresh = (token >= s["start"][:, None]) & (token < s["end"][:, None])
    held = token < s["start"][:, None]
    row = (s["cu"][:-1, None] + token - s["start"][:, None]).clamp(0, s["k"].shape[0] - 1).long()
    slot = (first[:, None] + torch.arange(pages, device=dev)).clamp(max=s["table"].shape[1] - 1).long()
    ids = s["table"].gather(1, slot).long()  # [seqs, pages]
    touched = fresh.reshape(len(first), pages, page).any(-1)
    out = []
    for name in "kv":
        codes, scale = s[name + "_codes"], s[name + "_scale"]
        x = s[name][row].float().masked_fill(~fresh[..., None, None], 0.0)
        x = x.reshape(len(first), pages, page, *x.shape[2:]).transpose(2, 3)  # [seqs, pages, hk, page, width]
        old = torch.where(held.reshape(len(first), pages, page)[:, :, :1], scale[ids], 0.0)
        now = torch.maximum((x.abs().amax((-1, -2)).double() / 127.0).float(), old)
        by = torch.where(now > 0, now, 1.0)[..., None, None].double()  # quotients next to a half: 64 bits
        kept = torch.round(codes[ids].double() * old[..., None, None] / by)
        put = torch.round(x / by).clamp(-127, 127)
        is_fresh, is_held = (m.reshape(len(first), pages, 1, page, 1) for m in (fresh, held))
        res = torch.where(is_fresh, put, torch.where(is_held, kept, codes[ids].double())).to(torch.int8)
        codes[ids[touched]] = res[touched]
        scale[ids[touched]] = now[touched]
        at = torch.repeat_interleave(torch.arange(len(first), device=dev), s["end"], output_size=s["total_all"])
        t = torch.arange(s["total_all"], device=dev) - s["cu_all"][at]
        page_of = s["table"][at, (t // page).long()].long()
        out.append(codes[page_of, :, (t % page).long()].float() * scale[page_of][..., None])
    return {"k": out[0], "v": out[1], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _plain_move(s):
    src, dst = s["src"].long(), s["dst"].long()
    for name in ("k_codes", "v_codes", "k_scale", "v_scale"):
        s[name][dst] = s[name][src]
    return {name: s[name] for name in ("k_codes", "v_codes", "k_scale", "v_scale")}


# ---------------------------------------------------------------------------------------------- one pass

def _package():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "l1-attention_b200")
    if at not in sys.path:
        sys.path.insert(0, at)


def run(s):
    case = s["case"]
    kind = case["kind"]
    if not own:
        return {"train": _plain_masked, "prefill": _plain_masked, "attend": _plain_attend, "append": _plain_append, "move": _plain_move}[kind](s)
    _package()
    if kind in ("train", "prefill"):
        from l1attn_masked_cuda import L1AttnMasked
        m = L1AttnMasked(case["mode"], causal=case["causal"], window=case["window"], softcap=case["softcap"])
        vo = m(s["q"], s["k"], s["v"], slopes=s["slopes"], doc=s["doc"], prefix=s["prefix"])
        if kind == "prefill":
            return vo
        dq, dk, dv = torch.autograd.grad(vo, (s["q"], s["k"], s["v"]), s["dvo"])
        return {"vo": vo.detach(), "dq": dq, "dk": dk, "dv": dv}
    import l1attn_cache_cuda as c
    cache = (s["k_codes"], s["v_codes"], s["k_scale"], s["v_scale"])
    if kind == "attend":
        return c.attend(s["q"], *cache, s["table"], s["start"], s["cu"], mode=case["mode"], window=case["window"], softcap=case["softcap"], slopes=s["slopes"])
    if kind == "append":
        c.append(s["k"], s["v"], *cache, s["table"], s["start"], s["cu"])
        k, v = c.gather(*cache, s["table"], s["zero"], s["cu_all"], s["total_all"])
        return {"k": k, "v": v, "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    c.copy_pages(*cache, s["src"], s["dst"])
    return {name: s[name] for name in ("k_codes", "v_codes", "k_scale", "v_scale")}


# ---------------------------------------------------------------------------------------------- 64 bits

def _row_softmax64(x, plus_one):
    """x: [rows, keys] with -inf where a key is not seen."""
    if plus_one:
        return torch.softmax(torch.cat([x, torch.zeros_like(x[:, :1])], 1), 1)[:, :-1]
    return torch.softmax(x, 1).nan_to_num(0.0)


def _exact_masked(case, s):
    b, n, h, rep, w = case["b"], case["n"], case["h"], case["h"] // case["hk"], case["w"]
    t = torch.arange(n, device=s["q"].device)
    out = {x: torch.zeros(s[y].shape, dtype=torch.float64, device=t.device) for x, y in (("dq", "q"), ("dk", "k"), ("dv", "v"))}
    out["vo"] = torch.zeros(b, n, h, case["wv"], dtype=torch.float64, device=t.device)
    rows = max(1, min(n, (1 << 25) // n))
    for i in range(b):
        for j in range(h):
            q, k, v = s["q"].detach()[i, :, j].double(), s["k"].detach()[i, :, j // rep].double(), s["v"].detach()[i, :, j // rep].double()
            for r in range(0, n, rows):
                tr = t[r:r + rows, None]
                seen = torch.ones(tr.shape[0], n, dtype=torch.bool, device=t.device)
                if case["causal"]:
                    seen &= tr >= t
                if case["window"]:
                    seen &= (tr - t).abs() < case["window"]
                if case["prefix"]:
                    seen |= t < int(s["prefix"][i])
                if case["docs"]:
                    seen &= (s["doc"][i, r:r + rows, None] == s["doc"][i]) & (s["doc"][i] >= 0)
                x = -torch.cdist(q[r:r + rows], k, p=1.0) / w ** 0.5
                slope = 1.0
                if case["softcap"]:
                    c = case["softcap"]
                    x = c * torch.tanh(x / c)
                    slope = 1.0 - (x / c) ** 2
                if case["bias"]:
                    x = x - s["slopes"][j].double() * (tr - t).abs()
                p = _row_softmax64(x.masked_fill(~seen, -math.inf), case["mode"] == "softmax_plus_one")
                o = p @ v
                out["vo"][i, r:r + rows, j] = o
                if case["kind"] == "train":
                    go = s["dvo"][i, r:r + rows, j].double()
                    out["dv"][i, :, j // rep] += p.T @ go
                    gx = p * (go @ v.T - (go * o).sum(1, keepdim=True)) * slope / w ** 0.5
                    for c in range(w):
                        signed = torch.sign(k[:, c] - q[r:r + rows, c, None]) * gx
                        out["dq"][i, r:r + rows, j, c] = signed.sum(1)
                        out["dk"][i, :, j // rep, c] -= signed.sum(0)
    return out if case["kind"] == "train" else out["vo"]


def _exact_attend(case, s):
    h, hk, page = case["h"], case["hk"], case["page"]
    out = torch.zeros(s["q"].shape[0], h, case["wv"], dtype=torch.float64, device=s["q"].device)
    row = 0
    for i, (a, c) in enumerate(_lengths(case)):
        ids = s["table"][i, :-(-(a + c) // page)].long()
        t, keys = a + torch.arange(c, device=out.device)[:, None], torch.arange(a + c, device=out.device)
        seen = keys <= t
        if case["window"]:
            seen &= t - keys < case["window"]
        for j in range(hk):
            k, v = ((s[x + "_codes"][ids, j].double() * s[x + "_scale"][ids, j].double()[:, None, None]).flatten(0, 1)[:a + c] for x in "kv")
            for r in range(j * h // hk, (j + 1) * h // hk):
                x = -torch.cdist(s["q"][row:row + c, r].double(), k, p=1.0) / case["w"] ** 0.5
                if case["softcap"]:
                    x = case["softcap"] * torch.tanh(x / case["softcap"])
                if case["bias"]:
                    x = x - s["slopes"][r].double() * (t - keys)
                out[row:row + c, r] = _row_softmax64(x.masked_fill(~seen, -math.inf), case["mode"] == "softmax_plus_one") @ v
        row += c
    return out


def _exact_append(case, s):
    page, out, row = case["page"], {}, 0
    host = {x: s[x].double().cpu().numpy() for x in ("k", "v", "k_codes", "v_codes", "k_scale", "v_scale")}
    table = s["table"].cpu().numpy()
    for x in "kv":
        got, row, scales = [], 0, host[x + "_scale"].copy()
        for i, (a, c) in enumerate(_lengths(case)):
            fresh = host[x][row:row + c]
            row += c
            for p in range(-(-(a + c) // page)):
                lo, hi, at = p * page, min((p + 1) * page, a + c), table[i, p]
                there = host[x + "_codes"][at, :, :max(0, min(hi, a) - lo)].transpose(1, 0, 2)
                come = fresh[max(lo, a) - a:max(hi, a) - a]
                old = host[x + "_scale"][at]
                if len(come):
                    most = (np.abs(come).max((0, 2)) / 127.0).astype(np.float32)  # the scale is held in 32 bits
                    scales[at] = np.maximum(most, old) if len(there) else most
                    there = np.rint(there * (old / scales[at])[:, None])
                    come = np.clip(np.rint(come / scales[at][:, None]), -127, 127)
                got.append(np.concatenate([there, come]) * scales[at][:, None])
        out[x], out[x + "_scale"] = np.concatenate(got), scales
    return {x: torch.from_numpy(out[x]) for x in ("k", "v", "k_scale", "v_scale")}


def exact(case, seed):
    kind = case["kind"]
    if kind in ("train", "prefill") and case["b"] * case["h"] * case["n"] ** 2 * case["w"] > (1.2e10 if kind == "train" else 4e10):
        return None
    s = prepare(case, seed)
    if kind == "move":
        place = np.arange(case["pages"])
        place[s["dst"].cpu().numpy()] = s["src"].cpu().numpy()
        return {"k_codes": None, "v_codes": None, "k_scale": s["k_scale"].cpu()[place].double(), "v_scale": s["v_scale"].cpu()[place].double()}
    return {"train": _exact_masked, "prefill": _exact_masked, "attend": _exact_attend, "append": _exact_append}[kind](case, s)


if __name__ == "__main__":
    for one in listed() + [draw(random.Random(i)) for i in range(8)]:
        print(one, work(one))
