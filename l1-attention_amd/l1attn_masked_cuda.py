"""Masked L1 attention with autograd, computed by the gfx950 HIP library: what a language model needs around the L1 score.
No counterpart in the reference, whose model code composes an unmasked form from L1Attn, softmax and einsum
(example-setfind/setfind.py:120-136).

    o = L1AttnMasked(causal=True, softcap=0.0, slopes=None)(q, k, v, doc=None, prefix=None)

    a[t,s] = -1/sqrt(W) * sum_w |q[b,t,h,w] - k[b,s,h',w]|          h' = h // (H / Hk)
    c = softcap * tanh(a / softcap) if softcap > 0 else a            x = c - slopes[h] * |i - s|,  i = S - T + t
    p = exp(x) / (1 + sum_s exp(x)) over the visible s               o[b,t,h,:] = sum_s p[t,s] * v[b,s,h',:]

q [B,T,H,W], k [B,S,Hk,W], v [B,S,Hk,Wv] of one type (float32, float16, bfloat16), T <= S, H a multiple of Hk, widths up to
128: the queries are the last T of the S tokens (T < S: a prompt worked off in chunks).  Token s is visible to token i where
causal is off, or s <= i, or s < prefix[b] (int32 [B]: a prefix that sees all of itself; without causal it changes nothing),
and, with doc (int32 [B,S]), where both are of one document: equal numbers >= 0; a negative number is padding, which sees
nothing and is seen by nothing.  A row that sees nothing is zero, as are its gradients.  The 1 in the denominator is the framework's no-op logit.

For its backward a forward keeps the inputs, o and 4 bytes for each row and head, and for 16-bit types what the rounding of o left
out, as large as o.

slopes: H numbers from 0 to 3e38 (constants, no gradient).  softcap from 0 to 3e38, 0 for none.  Calls on several streams and in graph capture
are fine: a call keeps nothing.  As with any operator, a backward pass is captured with no eager graph of the same leaves alive.
"""
from torch import nn
from torch.autograd import Function
from torch.autograd.function import once_differentiable

import _l1attn_lm_hip as _drv


class L1AttnMaskedFn(Function):
    @staticmethod
    def forward(ctx, q, k, v, doc=None, prefix=None, causal=True, softcap=0.0, slopes=None):
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
        slopes = None if slopes is None else _drv.slopes_of(slopes)  # as numbers: the backward's are the forward's
        o, kept = _drv.masked_forward(q, k, v, doc, prefix, causal, softcap, slopes, any(ctx.needs_input_grad[:3]))
        ctx.save_for_backward(q, k, v, o, kept, doc, prefix)
        ctx.rule = (causal, softcap, slopes)
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, d_o):
        q, k, v, o, kept, doc, prefix = ctx.saved_tensors
        dq, dk, dv = _drv.masked_backward(d_o.contiguous(), q, k, v, o, kept, doc, prefix, *ctx.rule)
        return dq, dk, dv, None, None, None, None, None


class L1AttnMasked(nn.Module):
    def __init__(self, causal=True, softcap=0.0, slopes=None):
        super(L1AttnMasked, self).__init__()
        self.causal, self.softcap = bool(causal), float(softcap)
        self.slopes = None if slopes is None else _drv.slopes_of(slopes)

    def forward(self, q, k, v, doc=None, prefix=None):
        return L1AttnMaskedFn.apply(q, k, v, doc, prefix, self.causal, self.softcap, self.slopes)
