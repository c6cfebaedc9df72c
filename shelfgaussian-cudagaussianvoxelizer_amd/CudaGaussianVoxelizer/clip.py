"""The norm of a training step's gradients and their clipping.  No counterpart in the reference, which leaves training to its
caller; the kernels live in libg2v_hip.so and are reached through ``_C`` on the caller's current stream.
"""
import torch

from . import _C

__all__ = ["clip_grad_norm_"]

_TYPES = {torch.Tensor, torch.nn.Parameter}


def _gradient(t):
    """The gradient that t stands for, None for a parameter without one.  A parameter is one whether it is trained or frozen: its
    values are never taken for a gradient."""
    if t.requires_grad and not (t.is_leaf or t.retains_grad):
        raise RuntimeError("a tensor that has a graph (a gradient made with create_graph) is neither a parameter nor a plain gradient: "
                           "pass it detached")
    return t.grad if t.requires_grad or t.grad is not None or isinstance(t, torch.nn.Parameter) else t


@torch.no_grad()
def clip_grad_norm_(tensors, max_norm, *, out=None):
    """Scales gradients by min(1, max_norm / (norm + 1e-6)), norm the 2-norm of all of them taken together, and returns the norm, a
    0-dim float32 GPU tensor (nothing waits for it).

    tensors: parameters (a module's ``parameters()``, frozen ones among them), whose .grad is clipped and which are skipped where they
    have none, or gradients themselves: tensors that are no torch.nn.Parameter, require no gradient and have none (one made with
    create_graph is refused as such and clipped as a parameter's .grad).  float32 and bfloat16 may be mixed, on one GPU; one tensor
    may come alone.  In place, of any strides; with ``out``, a list of as many float32 or bfloat16 tensors of the same shapes, the
    scaled gradients go there and the gradients stay (the float32 gradients of an optimizer's main weights from a bfloat16 layer's).
    What is written must not be there twice, nor share memory with another tensor but its own gradient as it lies (refused).  Squares
    are summed in 64 bits: the norm is finite where float32 holds it.  NaN or infinite gradients give a norm that is, and outputs as
    the formula says: nothing is skipped.  Two launches for up to 120 tensors, two more for every 120; they may be captured into a
    graph, which keeps the tensors' addresses."""
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    if not set(map(type, tensors)) <= _TYPES and not all(isinstance(t, torch.Tensor) for t in tensors):
        raise RuntimeError("tensors must be parameters or gradients")
    if not float(max_norm) >= 0.0:
        raise RuntimeError(f"max_norm must not be negative, got {max_norm}")
    if out is not None:
        out = [out] if isinstance(out, torch.Tensor) else list(out)
        if len(out) != len(tensors) or not (set(map(type, out)) <= _TYPES or all(isinstance(t, torch.Tensor) for t in out)):
            raise RuntimeError(f"out must hold {len(tensors)} tensors")
    # (the exact type first: isinstance takes ten times as long for a torch.nn.Parameter's class)
    plain = torch.Tensor
    grads = [t if type(t) is plain and not t.requires_grad and t.grad is None else _gradient(t) for t in tensors]
    if any(g is None for g in grads):
        if out is not None:
            out = [o for o, g in zip(out, grads) if g is not None]
        grads = [g for g in grads if g is not None]
    if not grads:    # nothing to clip
        return torch.zeros((), device=tensors[0].device if tensors else "cuda")
    return _C.clip_gradients(grads, max_norm, out)
