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
    for name, a, r, t in zip(("vo", "dq", "dk", "dv"), got, want, tol):
        if name in names:
            err = ((a.double() - r).abs() / t).max()
            assert float(err) <= 1, "%s: worst %.3g of the bound" % (name, float(err))


WIDTHS = [(64, 1.0), (128, 1.0), (128, 1.2), (128, 1.6), (100, 2.0)]


@pytest.mark.parametrize("dt", [F16, BF16, F32])
@pytest.mark.parametrize("mode", ["softmax", "softmax_plus_one", "exp"])
@pytest.mark.parametrize("w,spread", WIDTHS)
def test_forward(w, spread, mode, dt):
    q, k, v, dvo = _case(dt, w, spread, 1000.0)
    want, tol = reference(q, k, v, dvo, mode=mode)
    _check(("vo",), [_op(mode=mode)(q, k, v).detach()], want, tol)
