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

All four are differentiable once, in reverse mode (a forward-mode tangent raises
``NotImplementedError``).  Statistics and sums are fp32 whatever the
rows' type, every result is rounded once, and equal calls give equal bits.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _ops
from . import _validate as _v
from .layout import packed_offsets

__all__ = ["layer_norm", "pack_layer_norm", "unit_norm", "pack_unit_norm"]

_eager = torch.compiler.disable


def _rows(tokens: torch.Tensor):
    """``tokens [..., dim]`` as ``(tensor, (stride, stride, n, L, dim, n * L))``: rows
    the kernels can walk with two strides; copied only when it takes more than two."""
    shape, dim = tokens.shape, tokens.shape[-1]
    if len(shape) in (2, 3) and (dim == 1 or tokens.stride(-1) == 1):
        if len(shape) == 2:
            return tokens, (0, tokens.stride(0), 1, shape[0], dim, shape[0])
        return tokens, (tokens.stride(0), tokens.stride(1), shape[0], shape[1], dim, shape[0] * shape[1])
    tokens = tokens.detach().contiguous()
    rows = tokens.numel() // dim
    return tokens, (0, dim, 1, rows, dim, rows)


class _NormFn(torch.autograd.Function):
    """``call`` is ``(kind, source rows, their strides and sizes, offsets, eps,
    shape of the result, lengths the offsets are to be written from or None)``.  The
    statistics of a layer norm are saved for the backward pass; a unit row's length
    is taken again from the row."""

    @staticmethod
    def forward(ctx, tokens, weight, bias, call):
        kind, src, rows, offsets, eps, out_shape, lengths = call
        out, stats = _ops.norm_rows(kind, src, rows, offsets, weight, bias, eps, out_shape, kind == _ops.NORM_LAYER,
                                    lengths)
        ctx.save_for_backward(src, weight, stats, offsets)
        ctx.call = (kind, rows, eps, tokens.shape)
        return out

    @staticmethod
    def backward(ctx, grad):
        if torch.is_grad_enabled():  # create_graph: what comes out cannot be differentiated again
            return _backward_once(ctx, grad)
        return _backward(ctx, grad)


def _backward(ctx, grad):
    src, weight, stats, offsets = ctx.saved_tensors
    kind, rows, eps, token_shape = ctx.call
    want_tokens, want_weight, want_bias, _ = ctx.needs_input_grad
    return *_ops.norm_rows_backward(kind, grad.contiguous(), src, rows, offsets, weight, stats, eps,
                                    token_shape if want_tokens else None, want_weight, want_bias), None


_backward_once = once_differentiable(_backward)


def _has_tangent(*tensors) -> bool:
    """Whether one of them carries a forward-mode tangent (which needs no gradient mode)."""
    if getattr(forward_ad, "_current_level", 0) < 0:  # outside of any such differentiation
        return False
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _apply(kind, tokens, weight, bias, offsets, total, eps, lengths=None):
    """``offsets`` None: rows in, rows out."""
    if offsets is None:
        src, rows = _rows(tokens)
        out_shape = tokens.shape
    else:
        src = tokens if tokens.stride(2) == 1 else tokens.detach().contiguous()
        n, L, dim = src.shape
        rows, out_shape = (src.stride(0), src.stride(1), n, L, dim, total), (total, dim)
    weight = weight if weight is None else weight.contiguous()
    bias = bias if bias is None else bias.contiguous()
    if (torch.is_grad_enabled() and (tokens.requires_grad or (weight is not None and weight.requires_grad)
                                     or (bias is not None and bias.requires_grad))
            or _has_tangent(tokens, weight, bias)):  # refused there: there is no forward derivative
        return _NormFn.apply(tokens, weight, bias, (kind, src, rows, offsets, eps, out_shape, lengths))
    return _ops.norm_rows(kind, src, rows, offsets, weight, bias, eps, out_shape, False, lengths)[0]


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
    if (total_tokens is not None and lengths.dtype == torch.int32 and lengths.device == padded.device
            and lengths.dim() == 1 and lengths.shape[0] == padded.shape[0] and lengths.is_contiguous()):
        # nothing to look at on the host: offsets and rows in one call of the library
        offsets = lengths.new_empty((lengths.shape[0] + 1,))
        return _apply(kind, padded, weight, bias, offsets, int(total_tokens), float(eps), lengths), offsets
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
    their type.  The variance is an fp32 number: rows whose squared deviations
    from their mean add up past 3.4e38 come out as the bias, with a gradient of
    zero.  Raises ``ValueError`` / ``TypeError`` for shapes and types
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
