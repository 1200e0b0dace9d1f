"""Sequence operators next to the 2-D scan: linear attention with a decay per head (the scan's relative in one dimension,
with a matrix for a state), group normalisation with an activation on the channels-last tensors that all of this
package works on, and clipping of gradients by their global norm.

  linear_attention(q, k, v, log_decay, ...)         whole sequences, forward and backward
  linear_attention_step(q, k, v, log_decay, state)  one token of every sequence, the state updated in place
  group_norm(x, groups, weight, bias, ...)          x (N, ..., C)
  clip_norm_(tensors, max_norm)                     global norm of many tensors, all scaled in place
  clip_grad_norm_(parameters, max_norm)             of parameters' gradients: what ``refmodel.train_step`` calls

Like the scan they run on the current stream, take float32 and bfloat16 tensors, compute and carry state in float32, and
have no CPU or PyTorch path: tensors elsewhere, of another type or shape raise ``RuntimeError``; an option out of range
raises ``ValueError``.  The kernels are behind the C ABI in ``include/m2d_seq.h``.
"""
import torch

from . import _lib

__all__ = ["linear_attention", "linear_attention_step", "group_norm", "clip_norm_", "clip_grad_norm_"]

_ACTS = {None: 0, "silu": 1, "gelu": 2}


def linear_attention(q, k, v, log_decay, *, scale=None, initial_state=None, lengths=None, return_state=False):
    """``S_t = exp(log_decay_t) S_{t-1} + k_t v_t^T``, ``o_t = scale q_t^T S_t`` for every sequence and head.

    Args:
        q, k: (B, T, G, K); G divides H, each of their heads is shared by H / G neighbouring heads of v.
        v: (B, T, H, V).  Any strides (a last dimension that is not dense is copied); K and V up to 256.
        log_decay: (H,), a decay per head, or (B, T, H), one per token; used in float32.  At most 0: a positive value
            grows the state and is not checked for.  -inf forgets all earlier tokens (if they are finite).  Its
            gradient takes those of bfloat16 q and k out of the fast form (16384 tokens of 16 heads of 128: 2690 us
            for 300): where it is fixed, let it require none.
        scale: default ``K ** -0.5``.
        initial_state: (B, H, K, V) float32, or None for zero.
        lengths: (B,) integers on the device, tokens of each sequence (clamped to 0 ... T), or None for T.  Rows
            behind them are not read; outputs and gradients there are zero.
        return_state: also return the state after each sequence's last token, (B, H, K, V) float32.
    Returns:
        o (B, T, H, V) in ``v.dtype``, or ``(o, state)``.
    Differentiable in q, k, v, log_decay and initial_state, through o and the state.  A token that is not finite
    may spoil the outputs of up to 127 tokens before it, besides all later ones of its sequence and head.  Gradients of
    gradients (``create_graph``) raise; those of q, k and v are computed together, whichever is wanted.
    Outputs of bfloat16 tensors are off by a further 1.6e-3 or so beside their own rounding, their states by 3e-6; values
    (times q or k) below 1e-17 or above 1e17 may lose more where decays sum to some -65 in 128 tokens.
    """
    o, state = _lib.entry().linear_attention(q, k, v, log_decay, scale, initial_state, lengths, return_state)
    return (o, state) if return_state else o


def linear_attention_step(q, k, v, log_decay, state, *, scale=None):
    """One token of every sequence: ``state`` becomes ``exp(log_decay) state + k v^T`` in place, and the result is
    ``scale q^T state``.

    Args:
        q, k: (B, G, K); v: (B, H, V); log_decay: (H,) or (B, H); as ``linear_attention`` takes them.
        state: (B, H, K, V) float32 with dense (K, V); sequences and heads may lie apart (a layer's slice of a
            cache) but must not overlap.
    No gradients: it raises where one is wanted.
    """
    if state is None:
        raise RuntimeError("linear_attention_step: there is no state")
    return _lib.entry().linear_attention_step(q, k, v, log_decay, state, scale)


def group_norm(x, groups, weight=None, bias=None, *, eps=1e-5, act=None):
    """``act((x - mean) / sqrt(var + eps) * weight + bias)``, channels last.

    Args:
        x: (N, ..., C).  Mean and (biased) variance are taken over everything between the first and the last
            dimension and the C / groups channels of a group.  For a norm over the heads of each token pass
            (tokens, heads * size) with ``groups = heads``.
        weight, bias: (C,) or None; float32, or both of x's type.
        act: None, "silu" or "gelu" (erf form, as the block's ``act2``, models/mamba2d.py:169); at an infinity its
            value and slope are their limits.
    Differentiable in x, weight and bias, once (``create_graph`` raises).  x of any strides is copied where it is not
    contiguous.  Rows that are not whole 16-byte pieces, groups of a token (x (N, C)) of more than 512 bytes and maps of more
    than 4 KB a pixel take a slower form (100352 x 320 with one group: 310 us, 13 % of a copy's rate in float32).
    """
    if act not in _ACTS:
        raise ValueError(f"Unknown activation, got {act}...")
    if not isinstance(groups, int):
        raise ValueError(f"group_norm: groups must be an integer, got {groups}")
    return _lib.entry().group_norm(x, groups, weight, bias, eps, _ACTS[act])


def clip_norm_(tensors, max_norm, error_if_nonfinite=False):
    """Scale tensors in place so that their global 2-norm is at most ``max_norm``; returns the norm before (float32, on
    the device).

    The factor is ``max_norm / (norm + 1e-6)``, at most 1; an infinite norm makes finite values zero and infinite ones
    NaN, a NaN spoils everything.  Two launches for up to 512 tensors; nothing is written where the factor is 1.  The sum
    is taken in an order that does not change, in float64 beyond a thread's share of 32 KB (squares in float32: a value
    beyond 1.8e19 makes the norm infinite).

    Args:
        tensors: one or several; float32 or bfloat16, on one device, without gaps; they share no memory.
        max_norm: not negative; ``inf`` only measures.
        error_if_nonfinite: raise where the norm is infinite or NaN, before anything is scaled (waits for the GPU).
    """
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError(f"clip_norm_: max_norm must not be negative, got {max_norm}")
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    if not tensors:
        return torch.tensor(0.0)
    entry = _lib.entry()
    if error_if_nonfinite:
        total = entry.clip_grad_norm(tensors, float("inf"))
        if not bool(torch.isfinite(total)):
            raise RuntimeError(f"clip_norm_: the norm is {float(total)}; the tensors are left as they were")
    return entry.clip_grad_norm(tensors, max_norm)


def clip_grad_norm_(parameters, max_norm, error_if_nonfinite=False):
    """``clip_norm_`` of the parameters' gradients, as ``torch.nn.utils.clip_grad_norm_``: parameters (one or several)
    without a gradient are skipped."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    with torch.no_grad():
        return clip_norm_([p.grad for p in parameters if p.grad is not None], max_norm, error_if_nonfinite)
