"""Weights far below 1 in every mode: float16 must not lose them among its subnormals.

Without a normaliser, or with the key of score 0 in it, weights are as small as exp(score): 1e-9 where scores are -20.  Values (gradients) of thousands make
outputs of them that float16 holds well.  Bounds: test_masked_gpu.py's.
"""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_masked_gpu import BF16, F16, F32, _inputs, _op, reference  # noqa: E402


def _case(dt, w, spread, large, n=300):
    q, k, v, dvo = _inputs(1, n, 2, 1, w, 64, dt, seed=2, spread=spread)
    with torch.no_grad():
        v.mul_(large)
        dvo.mul_(large)
    return q, k, v, dvo


def _check(names, got, want, tol):
    """(float16: what is 65520 or more -- 65504, its largest, and half a step of 32 -- rounds to infinity, so elements that may be are only held to be large.)"""
    for name, a, r, t in zip(("vo", "dq", "dk", "dv"), got, want, tol):
        if name in names:
            over = (r.abs() + t >= 65520) if a.dtype == F16 else torch.zeros_like(r, dtype=torch.bool)
            err = torch.where(over, 0.0, (a.double() - r).abs() / t).max()
            assert float(err) <= 1, "%s: worst %.3g of the bound" % (name, float(err))
            assert (a[over].double().abs() >= (r.abs() - t)[over].clamp(max=65504)).all()


WIDTHS = [(64, 1.0), (128, 1.0), (128, 1.2), (128, 1.6), (100, 2.0)]


@pytest.mark.parametrize("dt", [F16, BF16, F32])
@pytest.mark.parametrize("mode", ["softmax", "softmax_plus_one", "exp"])
@pytest.mark.parametrize("w,spread", WIDTHS)
def test_forward(w, spread, mode, dt):
    q, k, v, dvo = _case(dt, w, spread, 1000.0)
    want, tol = reference(q, k, v, dvo, mode=mode)
    _check(("vo",), [_op(mode=mode)(q, k, v).detach()], want, tol)


@pytest.mark.parametrize("dt", [F16, BF16, F32])
@pytest.mark.parametrize("mode", ["softmax", "softmax_plus_one", "exp"])
@pytest.mark.parametrize("w,spread", WIDTHS)
def test_gradients(w, spread, mode, dt):
    q, k, v, dvo = _case(dt, w, spread, 100.0)
    vo = _op(mode=mode)(q, k, v)
    got = [vo.detach()] + list(torch.autograd.grad(vo, (q, k, v), dvo))
    want, tol = reference(q, k, v, dvo, mode=mode)
    _check(("dq", "dk", "dv"), got, want, tol)


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("mode", ["softmax", "exp"])
def test_keys_of_all_weights(mode, dt):
    """Keys from heavy ones to ones that nobody weighs much, and a bias that grows with the distance: weights above 1 in the exp form."""
    q, k, v, dvo = _case(dt, 64, 1.0, 10.0)
    with torch.no_grad():
        k += torch.linspace(0, 2.0, 300, device="cuda")[None, torch.randperm(300, generator=torch.Generator().manual_seed(1)).cuda(), None, None].to(dt)
    side = dict(slopes=torch.tensor([-0.03, 0.01], device="cuda"))
    vo = _op(mode=mode, causal=False)(q, k, v, **side)
    got = [vo.detach()] + list(torch.autograd.grad(vo, (q, k, v), dvo))
    want, tol = reference(q, k, v, dvo, mode=mode, causal=False, **side)
    _check(("vo", "dq", "dk", "dv"), got, want, tol)
