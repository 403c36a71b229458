"""Masked L1 attention for language models: an ADDITIONAL operator beside `l1attn_fused_cuda.L1AttnSoftmaxV`.

    m = L1AttnMasked(mode="softmax", causal=True, window=0, softcap=0.0)
    vo = m(q, k, v, slopes=None, doc=None, prefix=None)      # q [bs, n, h, w], k [bs, n, hk, w], v [bs, n, hk, wv] -> [bs, n, h, wv]

Scores are the framework's: x[t, s] = -(1/sqrt(w)) * sum_w |q_t - k_s|.  Then, each where it is asked for,

    x = softcap * tanh(x / softcap)                           a bound on the scores (they lie in (-softcap, 0])
    x = x - slopes[h] * |t - s|                               a bias that grows with the distance; slopes float32 [h], constants: refused with
                                                              a gradient of their own unless gradients are off
    causal, window                                            t sees s <= t; |t - s| < window
    prefix   int32 [bs]                                       keys s < prefix[b] are seen by every query of the item
    doc      int32 [bs, n]                                    t sees s of its own document only; negative: padding, sees nothing, unseen

and softmax over the keys that a query sees (`mode`: also "softmax_plus_one", "exp", as in L1AttnSoftmaxV).  A query that sees nothing gets
zeros, and gradients of zero.  A key whose weight is zero contributes nothing, whatever its value row holds (NaN in padding).

Heads of queries may share heads of keys and values (h a multiple of hk).  float32, float16 and bfloat16; widths up to 256.  q, k, v may
be strided views (of one projection, say) with contiguous rows; others are copied.  The output and the gradients are contiguous.
Differentiable in q, k and v (sign(0) = 0; backward mode, forward-mode tangents are refused); the backward is deterministic and keeps one float per query and head beside its inputs, and in 16 bits what rounding
left of the output; while it runs it takes up to a gigabyte in 16 bits (a float per pair), and a float per query head and element of k and v where heads are shared.
In 16 bits, weights are rounded for the value products and for dv (to 22 bits, or 2^-31 of the row's largest, in float16; to 16 in bfloat16)
and score gradients to 11 bits or 2^-25 of their row's largest (float16: 22, 2^-35); scores, normalisers and all sums are float32.
The 16-bit distance (widths to 128) is sum q + sum k - 2 sum min(q, k): exact minima, but its error goes with |q| + |k|, not with |q - k| (up to 3e-5 in
a score of width 128 where q and k share a channel at 1000, 7e-4 at 10000).
Everything runs on the tensors' device and the current stream.  No CPU path.  A backward that is captured into a CUDA graph must not share its leaves with an
eager graph that is still alive: autograd ties a leaf to the stream of its first use (detach or drop the eager outputs before the capture).
"""
import torch
from torch.autograd.function import once_differentiable

import l1attn_masked_cuda_drv  # torch must be imported first: the driver links against libtorch
from l1attn_cabi import SV_MODES

MODES = tuple(SV_MODES)


def _options(mode, causal, window, softcap):
    if mode not in SV_MODES:
        raise ValueError("mode must be one of %s" % (MODES,))
    if isinstance(window, bool) or int(window) != window or not 0 <= window < 1 << 31:
        raise ValueError("window must be a whole number, 0 for none")
    if float(softcap) != 0.0 and not 1e-30 <= float(softcap) <= 1e30:
        raise ValueError("softcap must be 0 (none) or from 1e-30 to 1e30")
    return SV_MODES[mode], bool(causal), int(window), float(softcap)


def _tensors(**given):
    for name, t in given.items():
        if t is not None and not isinstance(t, torch.Tensor):
            raise RuntimeError("%s must be a tensor" % name)


class L1AttnMaskedFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, slopes=None, doc=None, prefix=None, mode="softmax", causal=True, window=0, softcap=0.0):
        ctx.options = _options(mode, causal, window, softcap)
        _tensors(q=q, k=k, v=v, slopes=slopes, doc=doc, prefix=prefix)
        vo, rest, lse, *used = l1attn_masked_cuda_drv.forward(q, k, v, slopes, doc, prefix, *ctx.options, True)
        ctx.save_for_backward(*used, vo, rest, lse)
        return vo

    @staticmethod
    @once_differentiable
    def backward(ctx, dvo):
        *used, vo, rest, lse = ctx.saved_tensors
        return (*l1attn_masked_cuda_drv.backward(*used, *ctx.options, vo, rest, lse, dvo),) + (None,) * 7


class L1AttnMasked(torch.nn.Module):
    """vo[b, t, h, :] = sum of weight(t, s) * v[b, s, h // (heads / kv heads), :] over the keys that t sees; see the module docstring."""

    def __init__(self, mode="softmax", causal=True, window=0, softcap=0.0):
        super().__init__()
        self.options = _options(mode, causal, window, softcap)
        self.mode, self.causal, self.window, self.softcap = (mode,) + self.options[1:]

    def forward(self, q, k, v, slopes=None, doc=None, prefix=None):
        _tensors(q=q, k=k, v=v, slopes=slopes, doc=doc, prefix=prefix)
        if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
            return L1AttnMaskedFn.apply(q, k, v, slopes, doc, prefix, self.mode, self.causal, self.window, self.softcap)
        return l1attn_masked_cuda_drv.forward(q, k, v, slopes, doc, prefix, *self.options, False)[0]
