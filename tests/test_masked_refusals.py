"""What masked attention refuses, before anything reaches a GPU."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

import l1attn_cabi  # noqa: E402


def _call(back=False, **change):
    lib = l1attn_cabi.lib()
    buf = (ctypes.c_double * 64)()
    p = ctypes.addressof(buf)
    a = dict(q=p, k=p, v=p, strides=(ctypes.c_int64 * 9)(*[8] * 9), vo=p, rest=p, dvo=p, lse=p, dq=p, dk=p, dv=p, work=p, bs=1, n=2, h=2, hk=1, w=4, wv=4, dtype=l1attn_cabi.BF16)
    m = dict(mode="softmax", causal=True, window=0, softcap=0.0)
    m.update({x: change.pop(x) for x in list(change) if x in m})
    mask = l1attn_cabi.Mask(**m)
    if "raw_mode" in change:
        mask.mode = change.pop("raw_mode")
    mask.doc = change.pop("doc", None)
    a.update(change)
    sizes = [a[x] for x in ("bs", "n", "h", "hk", "w", "wv")]
    tail = sizes + [None if a.get("no_mask") else ctypes.byref(mask), a["dtype"], None]
    if back:
        return lib.l1attn_masked_bwd(a["q"], a["k"], a["v"], a["strides"], a["vo"], a["rest"], a["dvo"], a["lse"], a["dq"], a["dk"], a["dv"], a["work"], *tail)
    return lib.l1attn_masked_fwd(a["q"], a["k"], a["v"], a["strides"], a["vo"], a["rest"], a["lse"], a["work"], *tail)


@pytest.mark.parametrize("change,code", [
    (dict(q=None), -1), (dict(k=None), -1), (dict(v=None), -1), (dict(vo=None), -1), (dict(strides=None), -1), (dict(no_mask=True), -1), (dict(bs=-1), -1),
    (dict(w=0), -1), (dict(wv=0), -1), (dict(w=257), -2), (dict(wv=257), -2), (dict(h=3, hk=2), -1), (dict(hk=0), -1), (dict(dtype=l1attn_cabi.F64), -1),
    (dict(dtype=9), -1), (dict(window=-1), -1), (dict(softcap=-1.0), -1), (dict(softcap=float("nan")), -1), (dict(softcap=float("inf")), -1), (dict(raw_mode=3), -1),
    (dict(doc=4096, work=None), -1), (dict(strides=(ctypes.c_int64 * 9)(*[-8] * 9)), -1)])
def test_abi_refusals(change, code):
    assert _call(**dict(change)) == code
    assert _call(back=True, **dict(change)) == code


def test_abi_alignment_and_empty():
    buf = (ctypes.c_double * 8)()
    p = ctypes.addressof(buf)
    assert _call(rest=p + 1) == -6 and _call(back=True, rest=p + 1) == -6 and _call(q=p + 1) == -6 and _call(vo=p + 1) == -6 and _call(lse=p + 2) == -6 and _call(back=True, dk=p + 1) == -6
    assert _call(dtype=l1attn_cabi.F32, k=p + 2) == -6
    assert _call(back=True, work=None) == -1 and _call(back=True, lse=None) == -1
    assert _call(bs=0) == 0 and _call(n=0) == 0 and _call(back=True, bs=0) == 0


def test_work_bytes():
    f = l1attn_cabi.lib().l1attn_masked_work_bytes
    f32, bf16 = l1attn_cabi.F32, l1attn_cabi.BF16
    assert f(2, 65, 3, 3, 64, 64, bf16, 0) == 256 and f(2, 1024, 3, 3, 64, 64, bf16, 0) == 2 * 16 * 16 and f(0, 0, 0, 0, 0, 0, bf16, 1) == 256
    rows = 2 * 1024 * 4 * 4
    assert f(2, 1024, 4, 4, 64, 64, f32, 1) == f(2, 1024, 4, 4, 129, 64, bf16, 1) == 512 + rows  # ranges, delta
    assert f(2, 1024, 4, 2, 64, 64, f32, 1) == 512 + rows + rows * 128 and f(2, 1024, 4, 2, 129, 64, bf16, 1) == 512 + rows + rows * 193  # shares of shared heads
    assert f(2, 1024, 4, 4, 64, 32, bf16, 1) == 512 + rows + 8 * 1024 * 1024 * 4  # and a float per pair
    assert f(2, 1024, 4, 2, 64, 32, bf16, 1) == 512 + rows + rows * 96 + 8 * 1024 * 1024 * 4  # and shares of shared heads
    assert f(8, 8192, 8, 8, 64, 64, bf16, 1) == 8 * 128 * 16 + 8 * 8192 * 8 * 4 + (1 << 30)  # never more than a gigabyte of pairs
    assert f(1, 16385, 2, 2, 64, 64, bf16, 1) == 257 * 16 // 256 * 256 + 256 + (16385 * 2 * 4 + 255) // 256 * 256


def test_module_refusals():
    from l1attn_masked_cuda import L1AttnMasked
    for bad in (dict(mode="soft"), dict(window=-1), dict(window=1.5), dict(window=True), dict(softcap=-1.0), dict(softcap=float("nan")), dict(softcap=float("inf"))):
        with pytest.raises(ValueError):
            L1AttnMasked(**bad)
    x = torch.zeros(1, 2, 2, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        L1AttnMasked()(x, x, x)


def test_abi_refuses_what_no_kernel_covers():
    """Keys without query heads (their gradients would be left unwritten), and positions whose tiles would end past int."""
    for back in (False, True):
        assert _call(back=back, h=0) == -1 and _call(back=back, h=0, hk=0) == 0
        assert _call(back=back, n=(1 << 30) + 1) == -2
        assert _call(back=back, softcap=1e-40) == _call(back=back, softcap=1e31) == -1  # (a reciprocal that is no float32)


def test_caps_without_a_reciprocal_are_refused():
    from l1attn_cache_cuda import attend
    from l1attn_masked_cuda import L1AttnMasked
    x = torch.zeros(1)
    for cap in (1e-50, 1e-40, 1e31, 1e300):
        with pytest.raises(ValueError):
            L1AttnMasked(softcap=cap)
        with pytest.raises(ValueError):
            attend(x, x, x, x, x, x, x, x, softcap=cap)


@pytest.mark.gpu
def test_module_refuses_keys_without_queries():
    from l1attn_masked_cuda import L1AttnMasked
    z = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    with pytest.raises(RuntimeError, match="multiple"):
        L1AttnMasked()(z(2, 5, 0, 8), z(2, 5, 2, 8), z(2, 5, 2, 8))
    assert L1AttnMasked()(z(2, 5, 0, 8), z(2, 5, 0, 8), z(2, 5, 0, 6)).shape == (2, 5, 0, 6)


@pytest.mark.gpu
def test_module_refusals_of_tensors():
    from l1attn_masked_cuda import L1AttnMasked
    m = L1AttnMasked()
    z = lambda *s, **o: torch.zeros(*s, device="cuda", **o)  # noqa: E731
    q, k, v = z(2, 5, 4, 8), z(2, 5, 2, 8), z(2, 5, 2, 6)
    assert m(q, k, v).shape == (2, 5, 4, 6)
    for bad in ((z(2, 5, 4), k, v), (q, z(2, 6, 2, 8), v), (q, z(2, 5, 2, 7), v), (q, k, z(2, 5, 1, 6)), (q, z(2, 5, 3, 8), z(2, 5, 3, 6)), (q.half(), k, v),
                (q.double(), k.double(), v.double()), (z(2, 5, 4, 257), z(2, 5, 2, 257), v), (q, k, v.cpu()), (q, z(2, 5, 0, 8), z(2, 5, 0, 6))):
        with pytest.raises(RuntimeError):
            m(*bad)
    for bad in (dict(slopes=z(3)), dict(slopes=z(4).half()), dict(slopes=z(4).cpu()), dict(slopes=z(4, requires_grad=True)), dict(doc=z(2, 5)),
                dict(doc=z(2, 4, dtype=torch.int32)), dict(prefix=z(2)), dict(prefix=z(3, dtype=torch.int32)), dict(doc=[[0] * 5] * 2)):
        with pytest.raises(RuntimeError):
            m(q, k, v, **bad)
