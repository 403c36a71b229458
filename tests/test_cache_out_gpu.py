"""Outputs that lie over the queries are refused; ones beside them in the same buffer are not."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_cache_gpu import BF16, F32, _mod, _places, _random_cache  # noqa: E402


@pytest.mark.parametrize("dt", [F32, BF16])
def test_out_over_q(dt):
    m = _mod()
    cache = _random_cache(4, 2, 16, 32, 32)
    places = _places([(20, 3)], 16, 4)
    size = 3 * 4 * 32
    buf = torch.randn(2 * size + 8, device="cuda").to(dt)
    q = buf[:size].view(3, 4, 32)
    want = m.attend(q, *cache, *places)
    for at in (0, 8, size - 8):
        with pytest.raises(RuntimeError, match="overlap"):
            m.attend(q, *cache, *places, out=buf[at:at + size].view(3, 4, 32))
    with pytest.raises(RuntimeError, match="overlap"):
        m.attend(buf[size:2 * size].view(3, 4, 32), *cache, *places, out=buf[8:8 + size].view(3, 4, 32))
    assert torch.equal(m.attend(q, *cache, *places, out=buf[size:2 * size].view(3, 4, 32)), want)
    assert m.attend(q[:0], *cache, *places, out=buf[:0].view(0, 4, 32)).shape == (0, 4, 32)
