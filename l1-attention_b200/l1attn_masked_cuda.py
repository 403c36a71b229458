"""Masked L1 attention for language models: an ADDITIONAL operator beside `l1attn_fused_cuda.L1AttnSoftmaxV`.

    m = L1AttnMasked(mode="softmax", causal=True, window=0, softcap=0.0)
    vo = m(q, k, v, slopes=None, doc=None, prefix=None)      # q [bs, n, h, w], k [bs, n, hk, w], v [bs, n, hk, wv] -> [bs, n, h, wv]

Scores are the framework's: x[t, s] = -(1/sqrt(w)) * sum_w |q_t - k_s|.  Then, each where it is asked for,

    x = softcap * tanh(x / softcap)                           a bound on the scores (they lie in (-softcap, 0])
    x = x - slopes[h] * |t - s|                               a bias that grows with the distance; slopes float32 [h], constants
    causal, window                                            t sees s <= t; |t - s| < window
    prefix   int32 [bs]                                       keys s < prefix[b] are seen by every query of the item
    doc      int32 [bs, n]                                    t sees s of its own document only; negative: padding, sees nothing, unseen

and softmax over the keys that a query sees (`mode`: also "softmax_plus_one", "exp", as in L1AttnSoftmaxV).  A query that sees nothing gets
zeros, and gradients of zero.  A key whose weight is zero contributes nothing, whatever its value row holds (NaN in padding).

Heads of queries may share heads of keys and values (h a multiple of hk).  float32, float16 and bfloat16; widths up to 256.  q, k, v may
be strided views (of one projection, say) with contiguous rows; others are copied.  The output and the gradients are contiguous.
Differentiable in q, k and v (sign(0) = 0); the backward is deterministic and keeps one float per query and head beside its inputs.
Everything runs on the tensors' device and the current stream.  No CPU path.
"""
import torch
from torch.autograd.function import once_differentiable

import l1attn_cabi as _c

MODES = tuple(_c.SV_MODES)
TYPES = (torch.float32, torch.float16, torch.bfloat16)
MAX_WIDTH = 256


def _rows(t):
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _options(mode, causal, window, softcap):
    if mode not in _c.SV_MODES:
        raise ValueError("mode must be one of %s" % (MODES,))
    if isinstance(window, bool) or int(window) != window or not 0 <= window < 1 << 31:
        raise ValueError("window must be a whole number, 0 for none")
    if not 0.0 <= float(softcap) < float("inf"):
        raise ValueError("softcap must be finite and not negative, 0 for none")
    return mode, bool(causal), int(window), float(softcap)


def _side(t, name, shape, dtype, like):
    """A small tensor beside q, k, v: its shape, type and device; contiguous."""
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or tuple(t.shape) != tuple(shape) or t.device != like.device:
        raise RuntimeError("%s must be a %s tensor of shape %s on the device of q" % (name, str(dtype).replace("torch.", ""), tuple(shape)))
    if t.requires_grad:
        raise RuntimeError("%s is a constant: it must not require a gradient" % name)
    return t.contiguous()


def _check(q, k, v):
    for name, t in (("q", q), ("k", k), ("v", v)):
        if not t.is_cuda:
            raise RuntimeError("%s must be a CUDA tensor" % name)
        if t.dim() != 4:
            raise RuntimeError("q must be [bs, n, h, w], k [bs, n, hk, w], v [bs, n, hk, wv]")
    if k.shape[:2] != q.shape[:2] or k.shape[3] != q.shape[3] or v.shape[:3] != k.shape[:3]:
        raise RuntimeError("q must be [bs, n, h, w], k [bs, n, hk, w], v [bs, n, hk, wv]")
    if (q.shape[2] % k.shape[2] if k.shape[2] else q.shape[2]):
        raise RuntimeError("the heads of q must be a multiple of those of k and v")
    if q.dtype not in TYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise RuntimeError("q, k, v must share dtype float32, float16 or bfloat16")
    if k.device != q.device or v.device != q.device:
        raise RuntimeError("q, k, v must be on one device")
    if not 1 <= q.shape[3] <= MAX_WIDTH or not 1 <= v.shape[3] <= MAX_WIDTH:
        raise RuntimeError("widths must be 1 to %d" % MAX_WIDTH)


class L1AttnMaskedFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, slopes=None, doc=None, prefix=None, mode="softmax", causal=True, window=0, softcap=0.0):
        options = _options(mode, causal, window, softcap)
        _check(q, k, v)
        slopes = _side(slopes, "slopes", q.shape[2:3], torch.float32, q)
        doc = _side(doc, "doc", q.shape[:2], torch.int32, q)
        prefix = _side(prefix, "prefix", q.shape[:1], torch.int32, q)
        q, k, v = _rows(q), _rows(k), _rows(v)
        with torch.cuda.device(q.device):
            vo, lse = _c.masked_fwd(q, k, v, _c.Mask(*options, slopes, doc, prefix))
        ctx.save_for_backward(q, k, v, vo, lse, slopes, doc, prefix)
        ctx.options = options
        return vo

    @staticmethod
    @once_differentiable
    def backward(ctx, dvo):
        q, k, v, vo, lse, slopes, doc, prefix = ctx.saved_tensors
        with torch.cuda.device(q.device):
            dq, dk, dv = _c.masked_bwd(q, k, v, vo, dvo.contiguous(), lse, _c.Mask(*ctx.options, slopes, doc, prefix))
        return (dq, dk, dv) + (None,) * 7


class L1AttnMasked(torch.nn.Module):
    """vo[b, t, h, :] = sum of weight(t, s) * v[b, s, h // (heads / kv heads), :] over the keys that t sees; see the module docstring."""

    def __init__(self, mode="softmax", causal=True, window=0, softcap=0.0):
        super().__init__()
        self.mode, self.causal, self.window, self.softcap = _options(mode, causal, window, softcap)

    def forward(self, q, k, v, slopes=None, doc=None, prefix=None):
        return L1AttnMaskedFn.apply(q, k, v, slopes, doc, prefix, self.mode, self.causal, self.window, self.softcap)
