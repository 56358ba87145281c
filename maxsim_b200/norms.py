"""Normalising token rows on their way from an encoder into the operators.

The scores are defined on rows an encoder has normalised: a layer norm at the
end of the encoder, unit length after the projection to the scoring width.  The
reference leaves both to its callers.  Here each is one pass over the rows,
and the forms with ``pack_`` in their name do the packing of
:func:`maxsim_b200.pack_padded` on the same pass, so padding is neither read nor
written:

* :func:`layer_norm` / :func:`pack_layer_norm` -- ``(x - mean) / sqrt(var +
  eps) * weight + bias``;
* :func:`unit_norm` / :func:`pack_unit_norm` -- ``x / max(|x|, eps)``.

All four are differentiable once.  Statistics and sums are fp32 whatever the
rows' type, every result is rounded once, and equal calls give equal bits.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _ops
from . import _validate as _v
from .layout import packed_offsets

__all__ = ["layer_norm", "pack_layer_norm", "unit_norm", "pack_unit_norm"]

_eager = torch.compiler.disable


def _two_strides(t: torch.Tensor):
    """``t [..., dim]`` as ``(tensor, (n, L), (stride_n, stride_L))``: rows the
    kernels can walk with two strides; copied only when it takes more than two."""
    dim = t.shape[-1]
    if t.stride(-1) == 1 or dim == 1:
        if t.dim() == 2:
            return t, (1, t.shape[0]), (0, t.stride(0))
        if t.dim() == 3:
            return t, (t.shape[0], t.shape[1]), (t.stride(0), t.stride(1))
    t = t.contiguous()
    return t, (1, t.numel() // dim if dim else 0), (0, dim)


def _forward(kind, tokens, weight, bias, offsets, total, eps, want_stats):
    """``offsets`` None: rows in, rows out.  Returns the result and what the
    backward pass needs."""
    if offsets is None:
        src, (n, L), strides = _two_strides(tokens)
        total = n * L
    else:
        src = tokens if tokens.stride(2) == 1 else tokens.contiguous()
        n, L = src.shape[:2]
        strides = (src.stride(0), src.stride(1))
    call = (strides, (n, L, tokens.shape[-1]), offsets, total)
    w = weight.contiguous() if weight is not None else None
    b = bias.contiguous() if bias is not None else None
    out, stats = _ops.norm_rows(kind, src, *call, w, b, eps, want_stats)
    return out if offsets is not None else out.view(tokens.shape), src, w, stats, call


class _NormFn(torch.autograd.Function):
    """The statistics of a layer norm are saved for the backward pass; a unit
    row's length is taken again from the row."""

    @staticmethod
    def forward(ctx, kind, tokens, weight, bias, offsets, total, eps):
        out, src, w, stats, call = _forward(kind, tokens, weight, bias, offsets, total, eps, kind == _ops.NORM_LAYER)
        ctx.save_for_backward(src, w, stats, offsets)
        ctx.call = (kind, call[0], call[1], call[3], eps, tokens.shape)
        return out

    @staticmethod
    def backward(ctx, grad):
        if torch.is_grad_enabled():  # create_graph: what comes out cannot be differentiated again
            return _backward_once(ctx, grad)
        return _backward(ctx, grad)


def _backward(ctx, grad):
    src, w, stats, offsets = ctx.saved_tensors
    kind, strides, shape, total, eps, token_shape = ctx.call
    needs = ctx.needs_input_grad
    dx, dw, db = _ops.norm_rows_backward(kind, grad.contiguous(), src, strides, shape, offsets, total, w, stats, eps,
                                         needs[1], needs[2], needs[3])
    return None, dx.view(token_shape) if dx is not None else None, dw, db, None, None, None


_backward_once = once_differentiable(_backward)


def _apply(kind, tokens, weight, bias, offsets, total, eps):
    if torch.is_grad_enabled() and (tokens.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return _NormFn.apply(kind, tokens, weight, bias, offsets, total, eps)
    return _forward(kind, tokens, weight, bias, offsets, total, eps, False)[0]


def _check(name: str, tokens, weight, bias, eps) -> None:
    if tokens.dim() < 1:
        raise ValueError(f"{name} must be at least 1-D; got shape {tuple(tokens.shape)}")
    _v.require_float(name, tokens)
    dim = tokens.shape[-1]
    if dim == 0:
        raise ValueError(f"{name} must have rows of at least one element; got shape {tuple(tokens.shape)}")
    if bias is not None and weight is None:
        raise ValueError("bias needs a weight")
    for what, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if tuple(t.shape) != (dim,):
            raise ValueError(f"{what} must have shape [dim={dim}]; got {tuple(t.shape)}")
        if t.dtype not in (tokens.dtype, torch.float32):
            raise TypeError(f"{what} must be float32 or {tokens.dtype} like {name}; got {t.dtype}")
        if t.dtype != weight.dtype:
            raise TypeError(f"weight and bias must have the same dtype; got {weight.dtype} and {t.dtype}")
    if not 1e-30 <= eps < float("inf"):
        raise ValueError(f"eps must be at least 1e-30 and finite; got {eps}")
    if tokens.device.type != "cuda":
        raise RuntimeError(f"{name} must be a CUDA tensor (maxsim_b200 has no CPU path); got device {tokens.device}")
    if weight is not None:
        _v.require_same_device({name: tokens, "weight": weight, "bias": weight if bias is None else bias})
    if tokens.numel() // dim > 2 ** 31 - 4096:
        raise ValueError(f"{name} may have at most 2^31 - 4096 rows; got shape {tuple(tokens.shape)}")


def _packed(kind, padded, lengths, weight, bias, eps, total_tokens):
    if padded.dim() != 3:
        raise ValueError(f"padded must be 3-D [N, L_max, D]; got shape {tuple(padded.shape)}")
    _check("padded", padded, weight, bias, eps)
    offsets, total = packed_offsets(padded, lengths, total_tokens)
    return _apply(kind, padded, weight, bias, offsets, total, float(eps)), offsets


@_eager
def layer_norm(tokens: torch.Tensor, weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None, *, eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension
    of ``tokens [..., D]`` (CUDA, float32 / float16 / bfloat16), in the tokens' type.

    ``weight [D]`` and ``bias [D]`` are optional (a bias needs a weight), both
    of the tokens' type or both float32.  Differentiable with respect to all
    three; the gradients of ``weight`` and ``bias`` are summed in fp32 and have
    their type.  Raises ``ValueError`` / ``TypeError`` for shapes and types
    outside this, ``RuntimeError`` for tensors that are not on one CUDA device."""
    _check("tokens", tokens, weight, bias, eps)
    return _apply(_ops.NORM_LAYER, tokens, weight, bias, None, 0, float(eps))


@_eager
def pack_layer_norm(padded: torch.Tensor, lengths: torch.Tensor, weight: Optional[torch.Tensor] = None,
                    bias: Optional[torch.Tensor] = None, *, eps: float = 1e-5,
                    total_tokens: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """:func:`layer_norm` of the first ``lengths[n]`` rows of every segment of
    ``padded [N, L_max, D]``, packed: ``(packed [T, D], offsets [N+1] int32)`` as
    :func:`maxsim_b200.pack_padded` gives them, in one pass.  ``lengths`` and
    ``total_tokens`` are those of ``pack_padded``.  Padding rows are never read
    (they may hold NaN) and get a zero gradient."""
    return _packed(_ops.NORM_LAYER, padded, lengths, weight, bias, eps, total_tokens)


@_eager
def unit_norm(tokens: torch.Tensor, *, eps: float = 1e-12) -> torch.Tensor:
    """``x / max(|x|, eps)`` over the last dimension of ``tokens [..., D]`` (CUDA,
    float32 / float16 / bfloat16): unit rows, the vectors late interaction is
    defined on.  Differentiable; a row no longer than ``eps`` is scaled by a
    constant and has the gradient of that."""
    _check("tokens", tokens, None, None, eps)
    return _apply(_ops.NORM_UNIT, tokens, None, None, None, 0, float(eps))


@_eager
def pack_unit_norm(padded: torch.Tensor, lengths: torch.Tensor, *, eps: float = 1e-12,
                   total_tokens: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """:func:`unit_norm` of the valid rows of ``padded [N, L_max, D]``, packed;
    see :func:`pack_layer_norm`."""
    return _packed(_ops.NORM_UNIT, padded, lengths, None, None, eps, total_tokens)
