"""The steps either side of the operators: packing encoder outputs, unpacking
packed rows, ranking rerank scores.

The reference has no kernels for these.  Its callers pack with a Python loop of
slices and ``torch.cat`` (``README.md:185-192``) or a boolean-mask gather
(``torch-ext/maxsim/__init__.py:516-620``), both of which synchronise with the
host, and rank with ``scores.argsort(dim=1, descending=True)``
(``README.md:270-274``).  Here each is one kernel behind the C ABI:

* :func:`pack_padded` -- ``[N, L_max, D]`` + lengths -> packed ``[T, D]`` +
  int32 offsets; differentiable (the gradient is the reverse copy);
* :func:`unpack_packed` -- packed rows back to ``[N, L_max, D]`` with zero
  padding; differentiable;
* :func:`rerank_topk` -- the ``k`` best candidates of every row of a score
  matrix, best first, equal scores by ascending candidate index;
* :func:`sample_candidates` -- candidates drawn from every row by temperature,
  top-k, top-p and min-p (hard negatives), from given random numbers;
* :func:`score_candidates_padded_from_host` -- rerank a padded batch that
  lives in pinned host memory: a kernel reads only the valid token rows over
  PCIe (a padded batch is about one third padding), the scores go back to the
  host.
"""

from __future__ import annotations

from operator import index
from typing import Optional, Tuple

import torch

from . import _ops
from . import _validate as _v

__all__ = ["pack_padded", "unpack_packed", "rerank_topk", "rerank_order", "sample_candidates",
           "score_candidates_padded_from_host"]

_eager = torch.compiler.disable


class _PackFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, padded, offsets, total):
        ctx.save_for_backward(offsets)
        ctx.L_max = padded.shape[1]
        return _ops.pack_rows(padded, offsets, total)

    @staticmethod
    def backward(ctx, grad_packed):
        (offsets,) = ctx.saved_tensors
        return _ops.unpack_rows(grad_packed, offsets, ctx.L_max), None, None


class _UnpackFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, packed, offsets, L_max):
        ctx.save_for_backward(offsets)
        ctx.rows = packed.shape[0]
        return _ops.unpack_rows(packed, offsets, L_max)

    @staticmethod
    def backward(ctx, grad_padded):
        (offsets,) = ctx.saved_tensors
        return _ops.pack_rows(grad_padded, offsets, ctx.rows), None, None


def packed_offsets(padded: torch.Tensor, lengths: torch.Tensor, total_tokens: Optional[int]):
    """``(offsets [N+1] int32, T)`` of the rows ``padded[n, :lengths[n]]`` packed
    back to back; the checks and the synchronisation are those :func:`pack_padded`
    describes."""
    if padded.device.type != "cuda":
        raise RuntimeError(f"padded must be a CUDA tensor (maxsim_b200 has no CPU path); got device {padded.device}")
    N, L_max = padded.shape[0], padded.shape[1]
    if tuple(lengths.shape) != (N,):
        raise ValueError(f"lengths must have shape [N={N}]; got {tuple(lengths.shape)}")
    if lengths.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"lengths must be int32 or int64; got {lengths.dtype}")
    if lengths.device.type != "cpu" and lengths.device != padded.device:
        raise RuntimeError(f"lengths must be on the host or on padded's device {padded.device}; got {lengths.device}")
    if lengths.device.type == "cpu":
        if N and (int(lengths.min()) <= 0 or int(lengths.max()) > L_max):
            raise ValueError(f"lengths must be in (0, L_max={L_max}]")
        host = torch.zeros(N + 1, dtype=torch.int64)
        torch.cumsum(lengths, 0, out=host[1:])
        total = int(host[-1])
        if total >= 2 ** 31:
            raise ValueError("packed token count must fit int32 offsets")
        offsets = host.to(torch.int32).to(padded.device, non_blocking=True)
    else:
        offsets, total_dev = _ops.offsets_from_lengths(lengths, L_max, total_tokens is None)
        if total_tokens is None:
            total = int(total_dev.item())
            if total >= 2 ** 31:
                raise ValueError("packed token count must fit int32 offsets")
        else:
            total = int(total_tokens)
    if total_tokens is not None and int(total_tokens) != total:
        raise ValueError(f"total_tokens={int(total_tokens)} does not match lengths.sum()={total}")
    return offsets, total


@_eager
def pack_padded(padded: torch.Tensor, lengths: torch.Tensor, *,
                total_tokens: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Pack ``padded [N, L_max, D]`` (CUDA, any dtype) by prefix ``lengths [N]``.

    Returns ``(packed [T, D], offsets [N+1] int32)`` ready for
    ``score_contrastive*`` (documents) or ``score_pairs_packed*``.

    ``lengths`` may live on the host or on the device.  On the host the offsets
    are built there and nothing synchronises.  On the device a scan kernel
    builds them; ``T`` is then read back (one synchronisation) unless the
    caller passes ``total_tokens``, in which case nothing synchronises and the
    value is trusted to equal ``lengths.sum()`` (rows beyond it are dropped,
    never written out of bounds).

    Raises ``ValueError`` for a shape mismatch or, when the lengths are visible
    to the host, a length outside ``(0, L_max]``.
    """
    if padded.dim() < 2:
        raise ValueError(f"padded must be at least 2-D [N, L_max, ...]; got shape {tuple(padded.shape)}")
    offsets, total = packed_offsets(padded, lengths, total_tokens)
    return _PackFn.apply(padded, offsets, total), offsets


@_eager
def unpack_packed(packed: torch.Tensor, offsets: torch.Tensor, L_max: int) -> torch.Tensor:
    """``packed [T, D]`` + ``offsets [N+1]`` -> ``[N, L_max, D]``, zero beyond
    each segment (segments longer than ``L_max`` are truncated)."""
    if packed.dim() < 1 or offsets.dim() != 1 or offsets.numel() < 1:
        raise ValueError("packed must be [T, ...] and offsets [N+1]")
    if int(L_max) < 0:
        raise ValueError("L_max must be >= 0")
    return _UnpackFn.apply(packed, offsets, int(L_max))


@_eager
def rerank_topk(scores: torch.Tensor, k: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """The ``k`` best candidates per row of ``scores [B, C]``: returns
    ``(values [B, k] fp32, indices [B, k] int64)``, best first; equal scores
    are ordered by ascending candidate index; NaN ranks above ``+inf`` (the
    convention of ``torch.sort``).  ``C`` may be at most 16384."""
    if scores.dim() != 2:
        raise ValueError(f"scores must be 2-D [B, C]; got shape {tuple(scores.shape)}")
    if not 0 <= int(k) <= scores.shape[1]:
        raise ValueError(f"k must be in [0, C={scores.shape[1]}]; got {k}")
    return _ops.topk_rows(scores.detach(), int(k))


@_eager
def rerank_order(scores: torch.Tensor) -> torch.Tensor:
    """Full ranking: what ``scores.argsort(dim=1, descending=True)`` gives,
    with ties by ascending index."""
    return rerank_topk(scores, scores.shape[1])[1]


def _per_row(name: str, value, rows: int, dtype, device, least: float, most: float):
    """A sampling parameter: a number in ``(least, most]``, or a ``[rows]`` tensor
    whose values the kernel looks at."""
    if isinstance(value, torch.Tensor):
        if tuple(value.shape) != (rows,):
            raise ValueError(f"{name} must be a number or have shape [B={rows}]; got shape {tuple(value.shape)}")
        if value.device != device:
            raise RuntimeError(f"{name} must be on the scores' device {device}; got {value.device}")
        if value.is_floating_point() != (dtype == torch.float32) or value.dtype == torch.bool:
            raise TypeError(f"{name} must hold {'floats' if dtype == torch.float32 else 'integers'}; got {value.dtype}")
        value = value.detach()
        if value.dtype == torch.int64:  # anything past 32 bits keeps all
            value = value.clamp(min=0, max=2 ** 31 - 1)
        return value.to(dtype).contiguous()
    if not least < value <= most:
        raise ValueError(f"{name} must be in ({least}, {most}]; got {value}")
    return value


@_eager
def sample_candidates(scores: torch.Tensor, uniforms: torch.Tensor, n: int, *, temperature=1.0,
                      top_k=None, top_p=None, min_p=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Draw ``n`` different candidates from every row of ``scores [B, C]``, each in
    proportion to ``exp(score / temperature)`` among those not drawn yet.

    ``uniforms [B, C]`` fp32 are the random numbers, one per candidate, uniform
    in ``[0, 1)`` (``torch.rand_like``): the same ones give the same draws.
    Returns ``(indices [B, n] int64, probabilities [B, n] fp32)`` in the order
    drawn; ``probabilities`` is the candidate's share of the weight the filters
    keep.  Where a row has fewer candidates left the index is -1 and the
    probability 0.

    A score that is NaN or ``-inf`` (a masked positive) is no candidate, nor is
    one more than ``700 * temperature`` below the row's best; of ``+inf`` scores
    each weighs the same and everything else nothing.  The filters apply in this order, to the
    candidates best first (equal scores by ascending index):

    * ``top_k`` keeps that many;
    * ``top_p`` keeps, of those, the ones before which less than ``top_p`` of
      their weight lies (always the best one).  Weights count here in steps
      of ``2^-51`` of the best for ``C`` up to 2048, doubling with ``C`` to
      ``2^-42``;
    * ``min_p`` keeps the ones that weigh at least ``min_p`` times the best.

    Each parameter is a number or a ``[B]`` tensor on the scores' device, one
    value per row, which is not checked: a row whose temperature is not
    positive draws nothing, and ``top_k <= 0``, ``top_p`` outside ``(0, 1)`` or
    ``min_p`` outside ``(0, 1]`` switch that row's filter off.  ``C`` may be at
    most 2^20 and ``n`` at most 1024."""
    if scores.dim() != 2:
        raise ValueError(f"scores must be 2-D [B, C]; got shape {tuple(scores.shape)}")
    _v.require_float("scores", scores)
    if uniforms.shape != scores.shape:
        raise ValueError(f"uniforms must have the scores' shape {tuple(scores.shape)}; got {tuple(uniforms.shape)}")
    if uniforms.dtype != torch.float32:
        raise TypeError(f"uniforms must be float32; got {uniforms.dtype}")
    B, C = scores.shape
    n = index(n)
    if not 0 <= n <= min(C, 1024):
        raise ValueError(f"n must be in [0, min(C={C}, 1024)]; got {n}")
    if C > 2 ** 20:
        raise ValueError(f"scores may have at most 2^20 candidates per row; got {C}")
    if top_k is None:
        top_k = 0
    else:
        top_k = _per_row("top_k", top_k, B, torch.int32, scores.device, 0, float("inf"))
        top_k = top_k if isinstance(top_k, torch.Tensor) else min(index(top_k), C)
    params = [_per_row("temperature", temperature, B, torch.float32, scores.device, 0, float("inf")), top_k,
              1.0 if top_p is None else _per_row("top_p", top_p, B, torch.float32, scores.device, 0, 1),
              0.0 if min_p is None or (not isinstance(min_p, torch.Tensor) and min_p == 0)
              else _per_row("min_p", min_p, B, torch.float32, scores.device, 0, 1)]
    if scores.dtype != torch.float32:
        scores = scores.detach().to(torch.float32)
    if C > 1 and scores.stride(1) != 1:
        scores = scores.contiguous()
    if C > 1 and uniforms.stride(1) != 1:
        uniforms = uniforms.contiguous()
    return _ops.sample_rows(scores, uniforms, n, *params)


_STAGING = {}


def _staging_for(documents: torch.Tensor, device: torch.device) -> torch.Tensor:
    key = (tuple(documents.shape), documents.dtype, str(device))
    buf = _STAGING.get(key)
    if buf is None:
        _STAGING.clear()  # one batch shape at a time: these buffers are large
        buf = torch.empty(documents.shape, dtype=documents.dtype, device=device)
        _STAGING[key] = buf
    return buf


@_eager
def score_candidates_padded_from_host(queries: torch.Tensor, documents: torch.Tensor,
                                      query_lengths: torch.Tensor, doc_lengths: torch.Tensor, *,
                                      device, staging: Optional[torch.Tensor] = None,
                                      out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """:func:`maxsim_b200.score_candidates_padded` for a batch in host memory.

    ``queries [B, Lq, D]``, ``documents [B, C, Ld, D]`` and the two length
    tensors are CPU tensors.  When ``documents`` is pinned, a kernel on
    ``device`` reads each candidate's first ``doc_lengths[b, c]`` rows straight
    from it, so padding rows never cross PCIe; a pageable ``documents`` is
    copied whole.  ``staging`` is the device-side ``[B, C, Ld, D]`` landing
    buffer (one is kept per batch shape when not given; its padding rows hold
    whatever they held before, and no kernel reads them).  The kept buffer is
    shared by every call of that shape and is ordered only by the stream the
    calls run on: callers that use several streams pass their own ``staging``.

    Returns the ``[B, C]`` fp32 scores on the host.  With a pinned ``out`` the
    copy back is asynchronous on the current stream of ``device`` and ``out``
    is returned: synchronise that stream (or the device) before reading it.
    """
    for name, t in (("queries", queries), ("documents", documents),
                    ("query_lengths", query_lengths), ("doc_lengths", doc_lengths)):
        if t.device.type != "cpu":
            raise RuntimeError(f"{name} must be a CPU tensor; got device {t.device}")
    B, C, Lq, Ld, D = _v.check_padded(queries, documents, query_lengths, doc_lengths)
    device = torch.device(device)
    if device.type != "cuda":
        raise RuntimeError(f"device must be a CUDA device (maxsim_b200 has no CPU path); got {device}")
    if device.index is None:  # "cuda" means the current device; tensors report an index
        device = torch.device("cuda", torch.cuda.current_device())
    documents = documents.contiguous()
    with torch.cuda.device(device):
        q = queries.contiguous().to(device, non_blocking=True)
        qlen = query_lengths.contiguous().to(device, non_blocking=True).to(torch.int32)
        dlen = doc_lengths.contiguous().to(device, non_blocking=True).to(torch.int32)
        if staging is None:
            staging = _staging_for(documents, device)
        elif (staging.shape != documents.shape or staging.dtype != documents.dtype
              or staging.device != device or not staging.is_contiguous()):
            raise ValueError("staging must be a contiguous tensor on `device` shaped and typed like documents")
        if documents.is_pinned():
            _ops.copy_valid_rows(documents.view(B * C, Ld, D), dlen.view(-1), staging.view(B * C, Ld, D))
        else:
            staging.copy_(documents)
        scores = _ops.ops.maxsim_padded_forward(q.view(B * Lq, D), qlen, staging.view(B * C * Ld, D),
                                                dlen.view(-1), int(Lq), int(Ld), int(C)).view(B, C)
        if out is not None:
            if tuple(out.shape) != (B, C) or out.dtype != torch.float32 or out.device.type != "cpu":
                raise ValueError(f"out must be a CPU float32 tensor of shape [B={B}, C={C}]")
            out.copy_(scores, non_blocking=True)
            return out
        return scores.cpu()
