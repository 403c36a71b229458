"""What masked attention and the cache make of tensors that carry forward-mode tangents, and of slopes that are a model's parameters."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import torch.autograd.forward_ad as fw  # noqa: E402

from test_cache_gpu import BF16, F32, _mod, _places, _random_cache  # noqa: E402
from test_masked_gpu import _inputs, _op  # noqa: E402


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("grad", [True, False])
def test_tangents_are_refused(dt, grad):
    """As by the dense operator: never dropped without a word."""
    q, k, v, _ = _inputs(1, 20, 2, 1, 16, 16, dt)
    q, k, v = (x.detach().requires_grad_(grad) for x in (q, k, v))
    slopes = torch.tensor([0.1, 0.2], device="cuda")
    with fw.dual_level():
        for i in range(4):
            x = [q, k, v, slopes]
            x[i] = fw.make_dual(x[i].detach(), torch.ones_like(x[i]))
            with pytest.raises(NotImplementedError):
                _op()(x[0], x[1], x[2], slopes=x[3])
    assert _op()(q, k, v, slopes=slopes).shape == q.shape


def test_tangents_are_refused_by_the_cache():
    m = _mod()
    cache = _random_cache(4, 2, 16, 32, 32)
    places = _places([(20, 2)], 16, 4)
    q, k, v = (torch.randn(2, i, 32, device="cuda") for i in (4, 2, 2))
    slopes = torch.zeros(4, device="cuda")
    dual = lambda x: fw.make_dual(x, torch.ones_like(x))  # noqa: E731
    with fw.dual_level():
        for call in (lambda: m.attend(dual(q), *cache, *places), lambda: m.attend(q, *cache, *places, slopes=dual(slopes)), lambda: m.append(dual(k), v, *cache, *places),
                     lambda: m.append(k, dual(v), *cache, *places)):
            with pytest.raises(NotImplementedError):
                call()
    assert torch.isfinite(m.attend(q, *cache, *places, slopes=slopes)).all()


def test_slopes_of_a_model():
    """Parameters: refused where their gradient would be wanted, taken where none is."""
    q, k, v, dvo = _inputs(1, 40, 2, 1, 16, 16, F32)
    slopes = torch.nn.Parameter(torch.tensor([0.1, 0.2], device="cuda"))
    want = _op()(q, k, v, slopes=slopes.detach()).detach()
    for x in ((q, k, v), (q.detach(), k.detach(), v.detach())):
        with pytest.raises(RuntimeError, match="constant"):
            _op()(*x, slopes=slopes)
        with torch.no_grad():
            assert torch.equal(_op()(*x, slopes=slopes), want)
        with torch.inference_mode():
            assert torch.equal(_op()(*x, slopes=slopes), want)
    vo = _op()(q, k, v, slopes=slopes.detach())
    assert all(torch.isfinite(x).all() for x in torch.autograd.grad(vo, (q, k, v), dvo))
    m = _mod()
    cache, places = _random_cache(4, 1, 16, 16, 16), _places([(20, 2)], 16, 4)
    with pytest.raises(RuntimeError, match="constant"):
        m.attend(q[0, :2].detach(), *cache, *places, slopes=slopes)
    with torch.no_grad():
        assert torch.equal(m.attend(q[0, :2], *cache, *places, slopes=slopes), m.attend(q[0, :2].detach(), *cache, *places, slopes=slopes.detach()))
