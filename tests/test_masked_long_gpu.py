"""Masked L1 attention on the GPU where lengths change its course, and where operands of the backward are not finite.

The reference and its tolerances are test_masked_gpu's, taken over the part of a long row of tokens that the compared rows and keys can see.
"""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_masked_gpu import BF16, F16, F32, U, _compare, _inputs, _op, reference  # noqa: E402


def _grads(q, k, v, dvo, side, **options):
    vo = _op(**options)(q, k, v, **side)
    return [vo.detach()] + list(torch.autograd.grad(vo, (q, k, v), dvo))


def _compare_part(got, want, tol, at, rows, what):
    for name, a, r, t in zip(("vo", "dq", "dk", "dv"), got, want, tol):
        err = (a[:, at].double() - r[:, rows]).abs()
        assert (err <= t[:, rows]).all(), "%s %s: worst %.3g of the bound" % (what, name, float((err / t[:, rows]).max()))


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("bs,n,h,hk,w,wv", [(1, 16450, 2, 1, 32, 16), (2, 4100, 20, 10, 24, 40), (1, 16384, 3, 3, 100, 64)])
def test_more_pairs_than_are_kept(bs, n, h, hk, w, wv, dt):
    """Gradients of the distances of more than a gigabyte in all (several rounds of heads), and too many to keep any."""
    q, k, v, dvo = _inputs(bs, n, h, hk, w, wv, dt, seed=n)
    window = 48
    got = _grads(q, k, v, dvo, {}, window=window)
    for lo in (0, n // 2, n - 230):
        hi = lo + 230
        want, tol = reference(*(x[:, lo:hi] for x in (q, k, v, dvo)), window=window)
        rows = slice(0 if lo == 0 else window, 230 if hi == n else 230 - window)
        _compare_part(got, want, tol, slice(lo + rows.start, lo + rows.stop), rows, lo)
    doc = (torch.arange(n) // 211 * 7 % 53).to(torch.int32)[None].repeat(bs, 1)  # (no two neighbours alike; the same numbers come back far away)
    doc[:, 211:250] = -1
    first = doc[0, 0].item()
    again = [i for i in range(0, n, 211) if doc[0, i] == first][:2]
    side = dict(doc=doc.cuda(), slopes=torch.linspace(0.02, 0.3, h, device="cuda"))
    got = _grads(q, k, v, dvo, side, softcap=4.0, causal=False, window=600)
    for lo in again[:1]:
        want, tol = reference(*(x[:, lo:lo + 211] for x in (q, k, v, dvo)), softcap=4.0, causal=False, slopes=side["slopes"])
        _compare_part(got, want, tol, slice(lo, lo + 211), slice(0, 211), "documents")
    assert not any(x[:, 211:250].any() for x in got)


def test_flat_rows_keep_their_small_weights():
    """float16: one near key, and 32767 far ones of weight 2^-25.5 each, which alone carry values.  Weights are rounded to 11 bits, or to 2^-31 of the
    largest where that is more."""
    n, w = 32768, 64
    q, k, v = (torch.zeros(1, n, 1, w, dtype=F16, device="cuda") for _ in range(3))
    k[0, 1:] = 25.5 * math.log(2.0) / math.sqrt(w)
    v[0, 1:] = 1.0
    vo = _op(causal=False)(q, k, v)
    x = -math.sqrt(w) * float(k[0, 1, 0, 0])
    want = (n - 1) * math.exp(x) / (1 + (n - 1) * math.exp(x))
    e = 4 * U * (math.sqrt(w) + 8) * abs(x) + 8 * U * abs(x)
    tol = (n - 1) * 2.0 ** -31 + (2.0 ** -10 + 4 * e + 16 * U + 4 * U * math.sqrt(n)) * want
    assert tol < 0.05 * want
    assert ((vo.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("size", [(1, 140, 2, 1, 128, 64), (1, 100, 2, 2, 96, 40), (2, 70, 4, 1, 33, 128)])
def test_values_beyond_the_codes(size):
    """bfloat16: values below 2^-63 among ordinary ones, in some tiles; their differences keep their signs."""
    q, k, v, dvo = _inputs(*size, BF16, seed=3)
    g = torch.Generator().manual_seed(8)
    with torch.no_grad():
        for x in (q, k):
            part = x[:, 40:]
            small = (torch.rand(part.shape, generator=g) < 0.3).cuda()
            part.copy_(torch.where(small, part * 2.0 ** -75, part))
    _compare(q, k, v, dvo, {}, {})


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("h,hk", [(2, 2), (4, 1)])
def test_infinitely_far_rows_take_no_gradient(dt, h, hk):
    """An infinite key or query: weights of zero, and all other gradients as they are without it."""
    q, k, v, dvo = _inputs(1, 130, h, hk, 64, 48, dt, seed=11)
    with torch.no_grad():
        k[0, 30, 0, 5] = math.inf
        k[0, 31, -1, 6] = -math.inf
        q[0, 77, 1, 0] = math.inf
    _compare(q, k, v, dvo, {}, {})
    _compare(q, k, v, dvo, {}, dict(mode="softmax_plus_one", causal=False))


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_gradients_that_are_not_finite_reach_no_further(dt, bad):
    """A non-finite upstream gradient at one row reaches that row's query and the keys it sees; a non-finite value of a key the rows that see it."""
    q, k, v, dvo = _inputs(1, 150, 2, 1, 64, 64, dt, seed=13)
    r = 71
    spoiled = dvo.clone()
    spoiled[0, r, 1, 9] = bad
    clean = dvo.clone()
    clean[0, r, 1] = 0
    got = _grads(q, k, v, spoiled, {})
    want, tol = reference(q, k, v, clean)
    assert not torch.isfinite(got[1][0, r, 1]).any() and torch.isfinite(got[1][0, r, 0]).all()
    tie = k[0, :r, 0] == q[0, r, 1]  # (sign(0) = 0: such an element takes nothing of that row's, whatever it is)
    assert not torch.isfinite(got[3][0, :r + 1, 0, 9]).any() and not (torch.isfinite(got[2][0, :r, 0]) & ~tie).any()
    for name, a, x, t in zip(("dq", "dk", "dv"), got[1:], want[1:], tol[1:]):
        ok = (a.double() - x).abs() <= t
        if name == "dq":
            ok[0, r] = True
        else:
            ok[0, :r + 1, 0, 9 if name == "dv" else slice(None)] = True
            if name == "dv":  # (the clean row's share is missing in the reference)
                ok[0, :r + 1] = True
        assert ok.all(), name
    with torch.no_grad():
        v2 = v.clone()
        v2[0, r] = 0
        spoiled_v = v.clone()
        spoiled_v[0, r, 0, 3] = bad
    got = _grads(q, k, spoiled_v.requires_grad_(), dvo, {})
    want, tol = reference(q, k, v2, dvo)
    assert not torch.isfinite(got[1][0, r:]).all(-1).any()  # (some elements may: ties)
    assert ((got[1][0, :r].double() - want[1][0, :r]).abs() <= tol[1][0, :r]).all()
    assert ((got[3].double() - want[3]).abs() <= tol[3]).all()


@pytest.mark.parametrize("dt", [F32, BF16])
def test_repeated_inputs(dt):
    """Tensors that repeat one row of heads or one batch item (strides of zero): their gradients are the sums over the repeats."""
    q, k, v, dvo = _inputs(2, 90, 4, 2, 64, 64, dt, seed=6)
    one_q, one_k, one_v = (x[:1, :, :1].detach().clone().requires_grad_() for x in (q, k, v))
    views = one_q.expand(2, 90, 4, 64), one_k.expand(2, 90, 2, 64), one_v.expand(2, 90, 2, 64)
    got = torch.autograd.grad(_op()(*views), (one_q, one_k, one_v), dvo)
    want, tol = reference(*views, dvo)
    half = torch.finfo(dt).eps / 2
    for a, r, t in zip(got, want[1:], tol[1:]):
        parts = r.shape[0] * r.shape[2]
        r, t = r.sum((0, 2), keepdim=True), t.sum((0, 2), keepdim=True) + half * parts * r.abs().sum((0, 2), keepdim=True)  # (the sum is rounded as it goes)
        assert ((a.double() - r).abs() <= t).all()
