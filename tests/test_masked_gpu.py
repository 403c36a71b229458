"""Masked L1 attention on the GPU against its formulas in float64.

Tolerances are elementwise and follow from the arithmetic (u = 2^-24; half a step of the outputs' type: `torch.finfo(t).eps / 2`):

  scores    sums of width terms of at most |q| + |k| (the 16-bit kernels sum max(q, k), q and k apart) and the exponential:
            |dx| <= e = 4 u (sqrt(width) + 8) scale sum(|q| + |k|) + 8 u |x|, so weights are off by 2 e + 16 u of themselves (numerator, normaliser)
  vo        weights are rounded to the type before the value product (16 bits): (half + 2 e + 16 u) sum p |v|, and half |vo|
  gradients dP is a sum of v_width products: 4 u (sqrt(v_width) + 4) sum |dvo| |v|; delta is made of the rounded output: half sum |dvo| |vo|;
            score gradients are rounded to 11 bits relative to themselves or 2^-25 of their row's largest (16 bits); the rest as above
"""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = 2.0 ** -24


def _op(**options):
    from l1attn_masked_cuda import L1AttnMasked
    return L1AttnMasked(**options)


def _allowed(n, causal, window, doc, prefix, b, dev):
    t = torch.arange(n, device=dev)
    d = t[:, None] - t[None, :]
    ok = torch.ones(n, n, dtype=torch.bool, device=dev)
    if causal:
        ok &= d >= 0
    if window:
        ok &= d.abs() < window
    if prefix is not None:
        ok |= t[None, :] < prefix[b]
    if doc is not None:
        ok &= (doc[b][:, None] == doc[b][None, :]) & (doc[b][None, :] >= 0)
    return ok, d.abs().double()


def reference(q, k, v, dvo, mode="softmax", causal=True, window=0, softcap=0.0, slopes=None, doc=None, prefix=None):
    """(vo, dq, dk, dv) in float64 and the bound of each element's error; item by item, head by head."""
    dt, dev = q.dtype, q.device
    half = torch.finfo(dt).eps / 2
    low = dt != F32  # 16 bits: weights and score gradients are rounded on their way to the products
    q, k, v, dvo = (x.detach().double() for x in (q, k, v, dvo))
    bs, n, h, w = q.shape
    hk, wv = v.shape[2:]
    rep, scale = h // hk, 1.0 / math.sqrt(w)
    out = [torch.zeros_like(x) for x in (dvo, q, k, v)]
    tol = [torch.zeros_like(x) for x in (dvo, q, k, v)]
    for b in range(bs):
        ok, dist = _allowed(n, causal, window, doc, prefix, b, dev)
        for i in range(h):
            j = i // rep
            qq, kk, vv, go = q[b, :, i], k[b, :, j], v[b, :, j], dvo[b, :, i]
            d = qq[:, None] - kk[None]
            x = -scale * d.abs().sum(-1)
            e = 4 * U * (math.sqrt(w) + 8) * scale * (qq.abs().sum(-1)[:, None] + kk.abs().sum(-1)[None]) + 8 * U * x.abs()
            slant = torch.ones_like(x)
            if softcap:
                x = softcap * torch.tanh(x / softcap)
                slant = 1 - (x / softcap) ** 2
            if slopes is not None:
                x = x - slopes[i].double() * dist
                e = e + 8 * U * x.abs()
            x = x.masked_fill(~ok, -math.inf)
            if mode == "exp":
                p = torch.exp(x)
            else:
                extra = torch.zeros(n, 1, dtype=x.dtype, device=dev) if mode == "softmax_plus_one" else torch.full((n, 1), -math.inf, dtype=x.dtype, device=dev)
                p = torch.softmax(torch.cat([x, extra], 1), 1)[:, :-1].nan_to_num(0.0)
            pv = torch.where((p == 0).all(0)[:, None], 0.0, vv)  # a key that nobody weighs contributes nothing
            vo = p @ pv
            e = torch.where(p == 0, 0.0, e)
            rel = 2 * (e + e.amax(1, keepdim=True)) + 16 * U
            gop = torch.where((p == 0).all(1)[:, None], 0.0, go)
            dP = gop @ pv.T
            delta = 0.0 if mode == "exp" else (gop * vo).sum(-1, keepdim=True)
            dx = torch.where(p == 0, 0.0, p * (dP - delta) * slant)
            vabs = p @ pv.abs()
            t_vo = ((half if low else 0) + rel.amax(1, keepdim=True)) * vabs + half * vo.abs()
            sens = gop.abs() @ pv.abs().T
            d_dx = p * slant * (4 * U * (math.sqrt(wv) + 4) * sens + (0.0 if mode == "exp" else (gop.abs() * (t_vo + half * vo.abs())).sum(-1, keepdim=True)))
            d_dx = d_dx + rel * dx.abs() + 16 * U * p * sens + (2.0 * e * p * sens if softcap else 0.0)
            if low:
                d_dx = d_dx + 2.0 ** -11 * dx.abs() + 2.0 ** -25 * torch.maximum(dx.abs().amax(1, keepdim=True), dx.abs().amax(0, keepdim=True))
            sg = torch.sign(torch.where((p == 0)[..., None], 0.0, d))
            g = scale * dx
            out[0][b, :, i] = vo
            out[1][b, :, i] = -(sg * g[..., None]).sum(1)
            out[2][b, :, j] += (sg * g[..., None]).sum(0)
            out[3][b, :, j] += p.T @ gop
            su = 4 * U * math.sqrt(n)  # sums over the keys (queries) in float32
            tol[0][b, :, i] = t_vo + su * vabs
            tol[1][b, :, i] = (scale * d_dx + su * g.abs()).sum(1, keepdim=True)
            tol[2][b, :, j] += (scale * d_dx + su * g.abs()).sum(0)[:, None]
            tol[3][b, :, j] += (p * ((half if low else 0) + rel + su)).T @ gop.abs()
    for a, b in zip(tol[1:], out[1:]):
        a += half * b.abs()
    return out, [t + 1e-30 + (2.0 ** -25 if dt == F16 else 0.0) for t in tol]  # (float16: half of the smallest subnormal step)


def _inputs(bs, n, h, hk, w, wv, dt, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    mk = lambda *s: (spread * torch.randn(*s, generator=g)).to(dt).cuda()  # noqa: E731
    return mk(bs, n, h, w).requires_grad_(), mk(bs, n, hk, w).requires_grad_(), mk(bs, n, hk, wv).requires_grad_(), mk(bs, n, h, wv)


def _compare(q, k, v, dvo, side, options, what=""):
    vo = _op(**options)(q, k, v, **side)
    got = [vo] + list(torch.autograd.grad(vo, (q, k, v), dvo))
    want, tol = reference(q, k, v, dvo, **options, **side)
    for name, a, r, t in zip(("vo", "dq", "dk", "dv"), got, want, tol):
        assert a.dtype == q.dtype and a.shape == r.shape and a.is_contiguous()
        bad = ~((a.double() - r).abs() <= t)
        assert not bad.any(), "%s %s: %d of %d elements off, worst %.3g of the bound" % (
            what, name, int(bad.sum()), bad.numel(), float(((a.double() - r).abs() / t).nan_to_num(math.inf).max()))
    return got


SIZES = [(1, 1, 1, 1, 1, 1), (2, 2, 2, 1, 8, 8), (1, 63, 2, 2, 7, 5), (2, 64, 4, 2, 64, 64), (1, 65, 3, 3, 65, 40), (1, 130, 6, 2, 33, 128), (2, 200, 2, 1, 128, 128),
         (1, 129, 8, 1, 96, 80), (1, 100, 2, 2, 40, 24), (1, 70, 1, 1, 129, 64), (1, 70, 2, 1, 64, 256), (1, 40, 1, 1, 256, 200)]


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("size", SIZES)
def test_causal(size, dt):
    _compare(*_inputs(*size, dt, seed=sum(size)), {}, {})


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("mode", ["softmax", "softmax_plus_one", "exp"])
@pytest.mark.parametrize("causal,window,softcap,bias,docs,prefix", [
    (False, 0, 0.0, False, False, False), (False, 17, 0.0, True, False, False), (True, 1, 0.0, False, False, False), (True, 70, 3.0, True, False, False),
    (True, 0, 0.5, False, True, False), (True, 40, 0.0, True, True, True), (True, 0, 0.0, False, False, True), (False, 64, 10.0, True, True, True)])
def test_masks(mode, causal, window, softcap, bias, docs, prefix, dt):
    bs, n, h, hk, w, wv = 2, 197, 4, 2, 48, 32
    q, k, v, dvo = _inputs(bs, n, h, hk, w, wv, dt, seed=n, spread=0.5)
    side = {}
    if bias:
        side["slopes"] = torch.tensor([0.5, 0.1, 0.02, -0.01], device="cuda")
    if docs:  # documents of all lengths, in any order, padding inside and behind
        g = torch.Generator().manual_seed(1)
        doc = torch.randint(0, 4, (bs, 20), generator=g).repeat_interleave(10, 1)[:, :n]
        doc[:, 30:37] = -1
        doc[0, 150:] = -5
        side["doc"] = doc.to(torch.int32).cuda()
    if prefix:
        side["prefix"] = torch.tensor([75, 0], dtype=torch.int32, device="cuda")
    _compare(q, k, v, dvo, side, dict(mode=mode, causal=causal, window=window, softcap=softcap))


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("n,window", [(1500, 0), (1500, 200)])
def test_many_tiles(n, window, dt):
    """Several tiles of keys per row, most of them whole; documents that end inside tiles, and whole tiles of padding."""
    q, k, v, dvo = _inputs(1, n, 2, 1, 64, 64, dt, seed=3)
    doc = torch.zeros(1, n, dtype=torch.int32)
    doc[:, 500:] = 3
    doc[:, 900:1100] = -1
    _compare(q, k, v, dvo, dict(doc=doc.cuda()), dict(window=window, softcap=20.0))
    _compare(q, k, v, dvo, dict(prefix=torch.tensor([700], dtype=torch.int32, device="cuda")), dict(window=window))


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("mode", ["softmax", "softmax_plus_one"])
def test_padding_holds_anything(dt, mode):
    """NaN and infinities in padded rows of every input reach nothing; empty rows give zeros and take no gradient."""
    bs, n, h, hk, w, wv = 2, 150, 4, 2, 64, 64
    q, k, v, dvo = _inputs(bs, n, h, hk, w, wv, dt, seed=9)
    doc = torch.zeros(bs, n, dtype=torch.int32)
    doc[0, 40:60] = -1
    doc[0, 140:] = -1
    doc[1, :] = -1
    pad = (doc < 0).cuda()
    with torch.no_grad():
        for x, bad in ((q, math.nan), (k, math.inf), (v, math.nan), (dvo, -math.inf)):
            x[pad] = bad
        k[0, 45] = math.nan
        v[0, 44] = -math.inf
    vo = _op(mode=mode)(q, k, v, doc=doc.cuda())
    got = [vo] + list(torch.autograd.grad(vo, (q, k, v), dvo))
    for x in got:
        assert torch.isfinite(x).all() and not x[pad].any()
    with torch.no_grad():
        clean = [torch.where(pad[..., None, None], 0.0, x).to(dt) for x in (q, k, v, dvo)]
    want, tol = reference(*clean, mode=mode, doc=doc.cuda())
    for a, r, t in zip(got, want, tol):
        assert ((a.double() - r).abs() <= t).all()


@pytest.mark.parametrize("dt", [F32, F16, BF16])
def test_values_that_are_not_finite_and_seen(dt):
    """An infinitely far key has no weight (its own value is not looked at); a NaN in a query stays in its row; keys later than a NaN value are not
    reached by it."""
    n = 100
    q, k, v, dvo = _inputs(1, n, 2, 1, 64, 64, dt, seed=4)
    with torch.no_grad():
        k[0, 20, 0, 5] = math.inf
        k[0, 21, 0, 6] = -math.inf
        v[0, 20, 0, 3] = math.nan
        q[0, 50, 1, 0] = math.nan
        v[0, 70, 0, 7] = math.inf
    vo = _op()(q, k, v).detach()
    rows = torch.arange(n, device="cuda")
    assert torch.isnan(vo[0, 50, 1]).all()
    seen = vo[0].clone()
    seen[50, 1] = 0
    assert torch.isfinite(seen[:70]).all()
    assert torch.isinf(seen[70:, :, 7]).all() and torch.isfinite(seen[70:][..., torch.arange(64) != 7]).all()
    with torch.no_grad():
        k2, v2, q2 = k.clone(), v.clone(), q.clone()
        k2[0, 20:22] = 60.0  # so far that the weight is zero in float32 too
        v2[0, 20, 0, 3] = 0
        v2[0, 70, 0, 7] = 0
        q2[0, 50, 1, 0] = 0
    want = _op()(q2, k2, v2).detach()
    keep = (rows != 50)[:, None, None] & (torch.arange(64, device="cuda") != 7)
    ok = (seen.double() - want[0].double()).abs() <= 2 * torch.finfo(dt).eps * (1 + want[0].double().abs())
    assert (ok | ~keep).all()


@pytest.mark.parametrize("dt", [F16, BF16, F32])
def test_views(dt):
    """Slices of one projection, repeated keys and values, rows that start off any boundary."""
    bs, n, h, hk, w = 2, 90, 4, 2, 64
    g = torch.Generator().manual_seed(2)
    qkv = torch.randn(bs, n, h + 2 * hk, w, generator=g).to(dt).cuda().requires_grad_()
    dvo = torch.randn(bs, n, h, w, generator=g).to(dt).cuda()
    q, k, v = qkv.split([h, hk, hk], 2)
    _compare(q, k, v, dvo, {}, {})
    flat = torch.randn(bs * n * 3 * 67 + 1, generator=g).to(dt).cuda()[1:]
    odd = flat.view(bs, n, 3, 67)
    q, k, v = odd[..., 2:66].clone().requires_grad_(), odd[..., :1, 3:67].detach().requires_grad_(), odd[..., 1:2, 1:65].detach().requires_grad_()
    _compare(q.detach().requires_grad_(), k, v, torch.randn(bs, n, 3, 64, generator=g).to(dt).cuda(), {}, {})
    k1 = torch.randn(1, n, 1, w, generator=g).to(dt).cuda().requires_grad_()  # one key row for all items and heads
    q = torch.randn(bs, n, h, w, generator=g).to(dt).cuda().requires_grad_()
    vo = _op()(q, k1.expand(bs, n, hk, w), k1.expand(bs, n, hk, w))
    got, = torch.autograd.grad(vo, (k1,), dvo)
    want, tol = reference(q, k1.expand(bs, n, hk, w), k1.expand(bs, n, hk, w), dvo)
    err = (got.double() - (want[2] + want[3]).sum((0, 2), keepdim=True)).abs()
    parts = (want[2].abs() + want[3].abs()).sum((0, 2), keepdim=True)
    assert (err <= (tol[2] + tol[3]).sum((0, 2), keepdim=True) + 4 * torch.finfo(dt).eps * parts).all()  # (torch sums the parts in their type)
    t = torch.randn(bs, h, w, n, generator=g).to(dt).cuda().permute(0, 3, 1, 2)  # rows that are not contiguous are copied
    assert torch.equal(_op()(t, t, t), _op()(t.contiguous(), t.contiguous(), t.contiguous()))


@pytest.mark.parametrize("mode", ["softmax", "softmax_plus_one", "exp"])
def test_gradient_against_differences(mode):
    """The gradient along random directions against differences of the float64 formula."""
    side = dict(slopes=torch.tensor([0.3, 0.05], device="cuda"), prefix=torch.tensor([9], dtype=torch.int32, device="cuda"))
    options = dict(mode=mode, window=31, softcap=4.0)
    q, k, v, dvo = _inputs(1, 80, 2, 1, 24, 16, F32, seed=6, spread=0.4)
    grads = torch.autograd.grad(_op(**options)(q, k, v, **side), (q, k, v), dvo)
    g = torch.Generator().manual_seed(8)
    h = 1e-7  # (below the distance of any two values in a column here, with few exceptions: each moves the result by its own share only)
    for i in range(3):
        d = torch.randn(grads[i].shape, generator=g).double().cuda()
        loss = []
        for s in (h, -h):
            x = [t.detach().double() for t in (q, k, v)]
            x[i] = x[i] + s * d
            loss.append(float((_loss64(*x, **options, **side) * dvo.double()).sum()))
        want = (loss[0] - loss[1]) / (2 * h)
        got = float((grads[i].double() * d).sum())
        assert abs(got - want) <= 2e-5 * float((grads[i].double().abs() * d.abs()).sum())


def _loss64(q, k, v, mode, window, softcap, slopes, prefix):
    ok, dist = _allowed(q.shape[1], True, window, None, prefix, 0, q.device)
    out = []
    for i in range(q.shape[2]):
        j = i // (q.shape[2] // k.shape[2])
        x = -(q[0, :, None, i] - k[0, None, :, j]).abs().sum(-1) / math.sqrt(q.shape[3])
        x = (softcap * torch.tanh(x / softcap) - slopes[i].double() * dist).masked_fill(~ok, -math.inf)
        p = torch.exp(x)
        l = {"softmax": p.sum(1, keepdim=True), "softmax_plus_one": 1 + p.sum(1, keepdim=True), "exp": 1.0}[mode]
        out.append(p / l @ v[0, :, j])
    return torch.stack(out, 1)[None]


@pytest.mark.parametrize("dt", [F32, F16, BF16])
def test_ties(dt):
    """Values on a coarse grid, and q == k: sign(0) = 0 in every gradient."""
    g = torch.Generator().manual_seed(5)
    x = torch.randint(-2, 3, (1, 140, 2, 64), generator=g).to(dt).cuda()
    q, k = x.clone().requires_grad_(), x[:, :, :1].clone().requires_grad_()
    v, dvo = (torch.randn(1, 140, i, 64, generator=g).to(dt).cuda().requires_grad_() for i in (1, 2))
    _compare(q, k, v, dvo.detach(), {}, {})


def test_small_differences_keep_their_sign():
    """float16 and bfloat16 subnormals, and neighbours of large values."""
    for dt in (F16, BF16):
        tiny = float(torch.finfo(dt).smallest_normal) / 4
        g = torch.Generator().manual_seed(7)
        q = (torch.randint(-3, 4, (1, 70, 1, 64), generator=g) * tiny).to(dt)
        q[:, :, :, 32:] = 1000.0 + 8.0 * torch.randint(0, 3, (1, 70, 1, 32), generator=g)
        k = q.flip(1).cuda().requires_grad_()
        q = q.cuda().requires_grad_()
        v, dvo = (torch.randn(1, 70, 1, 64, generator=g).to(dt).cuda().requires_grad_() for _ in range(2))
        _compare(q, k, v, dvo.detach(), {}, {})


def test_gradients_of_all_sizes():
    """Score gradients over many orders of magnitude in one call: rows of small gradients are as exact as rows of large ones."""
    for dt in (BF16, F16):
        q, k, v, dvo = _inputs(1, 160, 2, 1, 64, 64, dt, seed=12)
        dvo = (dvo.double() * 10.0 ** torch.linspace(-6, 3 if dt == F16 else 9, 160, dtype=torch.float64, device="cuda")[None, :, None, None]).to(dt)
        vo = _op()(q, k, v)
        dq, = torch.autograd.grad(vo, (q,), dvo)
        want, tol = reference(q, k, v, dvo)
        assert ((dq.double() - want[1]).abs() <= tol[1]).all()


def test_streams_graphs_and_repeats():
    """Another stream, a captured and replayed forward and backward with new inputs, and bit-equal repeats."""
    torch.cuda.synchronize()
    q, k, v, dvo = _inputs(2, 300, 4, 2, 64, 64, BF16, seed=20)
    doc = torch.randint(0, 3, (2, 300), generator=torch.Generator().manual_seed(1)).to(torch.int32).cuda()
    m = _op(window=100, softcap=10.0)

    def step():
        vo = m(q, k, v, doc=doc)
        return (vo.detach(),) + torch.autograd.grad(vo, (q, k, v), dvo)  # (detached: a graph that lives on holds its leaves to its stream)

    first = [x.clone() for x in step()]
    assert all(torch.equal(a, b) for a, b in zip(first, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    with torch.no_grad():
        for x in (q, k, v, dvo):
            x.copy_(x.roll(1, 1))
        doc.copy_(doc.roll(7, 1))
    graph.replay()
    torch.cuda.synchronize()
    held = [x.clone() for x in held]
    assert all(torch.equal(a, b) for a, b in zip(step(), held))
    assert not torch.equal(held[0], first[0])


def test_offsets_past_32_bits():
    """Items that lie 2^32 bytes and more apart."""
    n, h, w, far = 66, 2, 64, (1 << 31) + 1024
    buf = torch.zeros(far + 3 * n * h * w, dtype=BF16, device="cuda")
    q, k, v = (buf.as_strided((2, n, h, w), (far, h * w, w, 1), i * n * h * w) for i in range(3))
    g = torch.Generator().manual_seed(3)
    for x in (q, k, v):
        x.copy_(torch.randn(2, n, h, w, generator=g))
    a = _op()(q, k, v)
    assert torch.equal(a, _op()(q.contiguous(), k.contiguous(), v.contiguous()))


def test_empty_calls():
    for bs, n in ((0, 5), (3, 0)):
        q, k, v, dvo = (torch.zeros(bs, n, i, 8, device="cuda", dtype=BF16).requires_grad_() for i in (2, 1, 1, 2))
        vo = _op()(q, k, v)
        assert vo.shape == (bs, n, 2, 8)
        for g, x in zip(torch.autograd.grad(vo, (q, k, v), dvo.detach()), (q, k, v)):
            assert g.shape == x.shape
