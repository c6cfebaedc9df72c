"""Gaussians that attend to one another before the splat: norms of queries and keys with the rotation by their
positions.  No counterpart in the reference, whose features arrive finished; the kernels live in libg2v_hip.so and are
reached through ``_C`` on the caller's current stream.
"""
import math

import torch
import torch.autograd.forward_ad as forward_ad
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _C

__all__ = ["qk_norm_rotary", "rotary_frequencies", "gaussian_attention", "PyGaussianAttention"]


def _tangents(*tensors):
    """Whether one of these carries a forward-mode derivative (which has no requires_grad, and flows under no_grad too).  None
    does outside of a dual level, which is looked at first: unpacking three tensors takes 3 us of a call's 12."""
    return getattr(forward_ad, "_current_level", 0) >= 0 and any(
        isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _differentiated(*tensors):
    """Whether a derivative in either mode is asked for: the call then goes through its autograd.Function, which has the
    backward and refuses tangents.  Others save its bookkeeping."""
    return (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)) or _tangents(*tensors)


class _QkNormRotaryFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, freqs, q_weight, k_weight, k_positions, eps):
        inputs, ctx.call = _C._qk_norm_inputs(q, k, positions, freqs, q_weight, k_weight, k_positions, eps)
        ctx.save_for_backward(*inputs)
        ctx.set_materialize_grads(False)
        return _C._qk_norm_forward(inputs, ctx.call)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_q_out, grad_k_out):
        inputs = ctx.saved_tensors
        q, k = inputs[:2]
        if grad_q_out is None and grad_k_out is None:
            return (None,) * 8
        if grad_q_out is None:
            grad_q_out = torch.zeros_like(q)
        if grad_k_out is None and k is not None:
            grad_k_out = torch.zeros_like(k)
        need = ctx.needs_input_grad
        grad_q_out = _C._heads_input(grad_q_out, "grad_q_out", q)
        if k is not None:
            grad_k_out = _C._heads_input(grad_k_out, "grad_k_out", q)
        dq, dk, dqw, dkw, dpos, dkpos = _C._qk_norm_backward(grad_q_out, grad_k_out, inputs, ctx.call,
                                                             (need[4], need[5]), (need[2], need[6]))
        return dq, dk, dpos, None, dqw, dkw, dkpos, None


def qk_norm_rotary(q, k, positions, freqs, q_weight=None, k_weight=None, *, k_positions=None, eps=1e-6):
    """Norms of queries and keys for each head and their rotation by the tokens' positions, in one pass.

    q (B, Nq, Hq, D) and k (B, Nk, Hk, D; None: queries alone) are float32 or bfloat16 in any layout with unit stride
    along D (views of a fused projection are read in place).  positions (B, Nq, A) float32 are coordinates of any kind
    (the Gaussians' means in metres, pixels, time); k_positions (B, Nk, A) those of the keys, None when queries and
    keys are the same tokens.  freqs (A, P) float32, 2 P <= D: pair (2 i, 2 i + 1) of a head turns by the angle
    sum_a positions[..., a] freqs[a, i], what is left of D stays (rotary_frequencies makes the usual table).
    q_weight and k_weight (D,) scale the normed rows.  Returns (q', k') of q's type, contiguous.

    Gradients flow to q, k, the weights and the positions (once: their own gradients, and forward-mode derivatives, are
    refused); freqs is a constant."""
    if isinstance(freqs, torch.Tensor) and (freqs.requires_grad or _tangents(freqs)):
        raise RuntimeError("freqs is a constant of qk_norm_rotary: it gets no gradient")
    if q_weight is not None and q_weight.dtype == torch.bfloat16:
        q_weight = q_weight.float()
    if k_weight is not None and k_weight.dtype == torch.bfloat16:
        k_weight = k_weight.float()
    if _differentiated(q, k, positions, q_weight, k_weight, k_positions):
        return _QkNormRotaryFunction.apply(q, k, positions, freqs, q_weight, k_weight, k_positions, eps)
    return _C.qk_norm_rotary_forward(q, k, positions, freqs, q_weight, k_weight, k_positions, eps)


def rotary_frequencies(head_dim, axes=3, wavelengths=(0.8, 160.0), device="cuda"):
    """(axes, P) float32 table of qk_norm_rotary: each axis turns an equal share of the head's pairs, with wavelengths
    (in the positions' unit) spread geometrically over the given range; pairs that do not divide stay unrotated.  The
    default range is two voxels of 0.4 m to twice a scene of 80 m."""
    each = head_dim // 2 // axes
    lo, hi = float(wavelengths[0]), float(wavelengths[1])
    if each < 1 or not 0.0 < lo <= hi:
        raise RuntimeError(f"rotary_frequencies: {head_dim} values hold no pair for each of {axes} axes, or bad "
                           f"wavelengths {wavelengths}")
    table = torch.zeros(axes, axes * each, dtype=torch.float32)
    step = torch.arange(each, dtype=torch.float64) / max(1, each - 1)
    for a in range(axes):
        table[a, a * each:(a + 1) * each] = (2.0 * math.pi / (lo * (hi / lo) ** step)).float()
    return table.to(device)


class _GaussianAttentionFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, key_mask, scale):
        inputs, ctx.call = _C._attention_inputs(q, k, v, key_mask, scale)
        out, rest, lse, key_list = _C._attention_forward(inputs, ctx.call, True)
        ctx.save_for_backward(*inputs[:3], out, rest, lse, key_list)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        saved, need = ctx.saved_tensors, ctx.needs_input_grad
        grad_out = _C._heads_input(grad_out, "grad_out", saved[0])
        return _C._attention_backward(grad_out, *saved, ctx.call, need[0], need[1] or need[2]) + (None, None)


def gaussian_attention(q, k, v, key_mask=None, scale=None):
    """softmax(scale q k^T over the valid keys) v, without an order among queries or keys.

    q (B, Nq, Hq, D) and k, v (B, Nk, Hkv, D) are float32 or bfloat16 in any layout with unit stride along D; Hq is a
    multiple of Hkv (consecutive query heads share a key head), D at most 128.  key_mask (B, Nk) bool is False at keys
    that are not attended to (padding of a batch, pruned Gaussians): what their rows hold, NaN included, reaches no result
    and they get zero gradients; a query without any key gives zeros.  float32 values of valid rows have to be finite (an
    infinity gives NaN, as they are split into three bfloat16 planes), and sums within float32's range (include/g2v.h says which).  scale None: D^-1/2.  Returns (B, Nq, Hq, D) of
    q's type, contiguous.  Any number of queries and keys, zero and one included: a single query that pools a scene has its
    keys split over the GPU.

    Scores and sums are float32.  With bfloat16 inputs the probabilities are rounded to bfloat16 before their product with v, and
    the backward's factors likewise (as two such planes where keys or queries are few): outputs and gradients are off by 1.7e-3 to
    2.4e-3 of their norm, where rounding exact ones would put them 1.7e-3 off.  float32 keeps 24 bits throughout.

    Gradients flow to q, k and v; the backward recomputes the probabilities and gives the same bits on every run.  Gradients
    of gradients and forward-mode derivatives are refused."""
    if _differentiated(q, k, v):
        return _GaussianAttentionFunction.apply(q, k, v, key_mask, scale)
    return _C.attention_forward(q, k, v, key_mask, scale)[0]


class PyGaussianAttention(nn.Module):
    """Multi-head attention of Gaussians to one another, or to other tokens at positions, with normed and rotated queries and
    keys: the layer that makes the features that PyCudaGaussianVoxelizer splats.

        q = rotate(norm(x Wq)),  k = rotate(norm(c Wk)),  v = c Wv,  y = attention(q, k, v) Wo

    with c = x (self-attention) or the given context.  num_kv_heads key heads are shared by num_heads / num_kv_heads
    query heads each.  ``wavelengths`` is the range over which the rotations turn, in the positions' unit (metres).  A conversion
    (``layer.bfloat16()``) takes the weights along and leaves the table of angles, ``freqs``, in float32."""

    def __init__(self, embed_dim, num_heads, num_kv_heads=None, *, head_dim=None, axes=3, wavelengths=(0.8, 160.0), eps=1e-6,
                 device="cuda", dtype=torch.float32):
        super().__init__()
        num_kv_heads = num_heads if num_kv_heads is None else num_kv_heads
        if head_dim is None:
            if embed_dim % num_heads:
                raise RuntimeError(f"embed_dim {embed_dim} is no multiple of num_heads {num_heads}: give head_dim")
            head_dim = embed_dim // num_heads
        if num_heads % num_kv_heads:
            raise RuntimeError(f"num_heads {num_heads} is no multiple of num_kv_heads {num_kv_heads}")
        self.heads, self.kv_heads, self.head_dim, self.eps = num_heads, num_kv_heads, head_dim, eps
        kw = dict(bias=False, device=device, dtype=dtype)
        self.to_q = nn.Linear(embed_dim, num_heads * head_dim, **kw)
        self.to_kv = nn.Linear(embed_dim, 2 * num_kv_heads * head_dim, **kw)
        self.to_out = nn.Linear(num_heads * head_dim, embed_dim, **kw)
        self.q_weight = nn.Parameter(torch.ones(head_dim, device=device))
        self.k_weight = nn.Parameter(torch.ones(head_dim, device=device))
        self.register_buffer("freqs", rotary_frequencies(head_dim, axes, wavelengths, device), persistent=False)

    def _apply(self, fn, recurse=True):
        """Moves and conversions of a module's tensors.  The table of angles only moves: at 40 m from the origin one rounded to
        8 bits would turn by tenths of a radian less or more."""
        table = self.freqs
        super()._apply(fn, recurse)
        if self.freqs.dtype != table.dtype:
            self.freqs = table.to(self.freqs.device)
        return self

    def forward(self, x, positions, key_mask=None, *, context=None, context_positions=None):
        """x (B, N, embed_dim) at positions (B, N, axes) float32; context (B, M, embed_dim) at context_positions (B, M, axes),
        both or neither.  key_mask (B, N) or (B, M) bool, False at tokens that are not attended to.  Returns
        (B, N, embed_dim); gradients flow to x, context, the weights and the positions."""
        if (context is None) != (context_positions is None):
            raise RuntimeError("context and context_positions go together")
        c = x if context is None else context
        q = self.to_q(x).unflatten(-1, (self.heads, self.head_dim))
        k, v = self.to_kv(c).unflatten(-1, (2 * self.kv_heads, self.head_dim)).split(self.kv_heads, 2)
        q, k = qk_norm_rotary(q, k, positions, self.freqs, self.q_weight, self.k_weight,
                              k_positions=context_positions, eps=self.eps)
        return self.to_out(gaussian_attention(q, k, v, key_mask).flatten(2))
