"""16-bit outputs and gradients are about as far from 64 bits as the exact ones rounded once to the type.

What lies between, relative to a step of the output h (2^-8 bfloat16, 2^-11 float16) and as independent roundings: weights and their rests carry 16 and 22 bits,
score gradients 11 bits next to bfloat16 outputs (h / 8) and 22 next to float16 ones, sums are float32: (1/8)^2 of the square at most, 1 % of the error.  Sums that cancel
enlarge what went in before them by sum |term| / |sum|, about sqrt(keys) for random signs, but roundings of the terms add up as randomly: the ratio stays.
Held to 1.1.
"""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_masked_gpu import BF16, F16, _inputs, _op, reference  # noqa: E402


def _ratio(got, want):
    return float((got.double() - want).norm() / (want.to(got.dtype).double() - want).norm())


def _ratios(dt, mode, n, h, hk, w, wv):
    q, k, v, dvo = _inputs(1, n, h, hk, w, wv, dt, seed=n + w)
    vo = _op(mode=mode)(q, k, v)
    got = [vo.detach()] + list(torch.autograd.grad(vo, (q, k, v), dvo))
    return {name: _ratio(a, r) for name, a, r in zip(("vo", "dq", "dk", "dv"), got, reference(q, k, v, dvo, mode=mode)[0])}


SIZES = [(1024, 1, 1, 64, 64), (600, 2, 2, 128, 128), (500, 4, 2, 96, 40)]


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("mode", ["softmax", "softmax_plus_one", "exp"])
@pytest.mark.parametrize("size", SIZES)
def test_values(size, mode, dt):
    assert _ratios(dt, mode, *size)["dv"] <= 1.1


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("mode", ["softmax", "exp"])
@pytest.mark.parametrize("size", SIZES)
def test_all(size, mode, dt):
    ratios = _ratios(dt, mode, *size)
    assert max(ratios.values()) <= 1.1, ratios
