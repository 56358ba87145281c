"""Cases of the normalisation and sampling operators either side of the scores.

``layer_norm`` / ``pack_layer_norm`` and ``unit_norm`` / ``pack_unit_norm``
normalise token rows on their way from an encoder into the scoring operators;
``sample_candidates`` draws candidates (hard negatives) from a score matrix.
A case says which operator, how large, which element types and whether the pass
is the forward alone or a training pass with its gradients.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

_TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"fp32": 4, "fp16": 2, "bf16": 2, "none": 0}


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------

def _norm(op, segments, longest, shortest, dim, dtype, *, packed=False, train=False,
          weight="none", bias=False):
    """``segments`` sequences padded to ``longest`` tokens, their lengths spread
    evenly from ``shortest`` to ``longest``.  ``packed``: the valid rows are
    written back to back; otherwise every row counts."""
    return {"op": op, "segments": segments, "longest": longest, "shortest": shortest, "dim": dim,
            "dtype": dtype, "packed": packed, "train": train, "weight": weight, "bias": bias}


def _sample(rows, cols, n, *, temperature, top_k=0, top_p=1.0, min_p=0.0, masked="none", per_row=False):
    """``n`` candidates out of each of ``rows`` score rows of ``cols``; ``top_k``
    0, ``top_p`` 1 and ``min_p`` 0 switch a filter off.  ``per_row``: temperature
    and top-p come as one value per row."""
    return {"op": "sample", "rows": rows, "cols": cols, "n": n, "temperature": temperature,
            "top_k": top_k, "top_p": top_p, "min_p": min_p, "masked": masked, "per_row": per_row}


def listed():
    return [
        # one query of 32 tokens on its way through a serving encoder: latency alone
        _norm("layer", 1, 32, 32, 768, "fp16", weight="fp16", bias=True)
        | {"name": "layer_query_fp16"},
        # the 1000 candidates of one query, padded to 300 tokens, encoded for reranking
        _norm("layer", 1000, 300, 16, 1024, "bf16", packed=True, weight="bf16", bias=True)
        | {"name": "layer_candidates_bf16"},
        # a small contrastive batch (64 documents of 32 to 256 tokens) in mixed precision
        _norm("layer", 64, 256, 32, 768, "bf16", packed=True, train=True, weight="fp32", bias=True)
        | {"name": "layer_train_small_bf16"},
        # a large contrastive batch (1024 documents of 64 to 512 tokens)
        _norm("layer", 1024, 512, 64, 768, "bf16", packed=True, train=True, weight="bf16", bias=True)
        | {"name": "layer_train_large_bf16"},
        # full precision, a width that no vector load divides, no bias, a rectangular batch
        _norm("layer", 37, 211, 211, 333, "fp32", train=True, weight="fp32")
        | {"name": "layer_train_odd_fp32"},
        # one query's projected tokens: latency alone
        _norm("unit", 1, 32, 32, 128, "fp16") | {"name": "unit_query_fp16"},
        # the documents of the large contrastive batch after the projection to 128
        _norm("unit", 1024, 512, 64, 128, "bf16", packed=True, train=True)
        | {"name": "unit_train_large_bf16"},
        # a collection of some 20000 documents, packed back to back already, 96 wide
        _norm("unit", 1, 2_400_007, 2_400_007, 96, "fp16", train=True)
        | {"name": "unit_collection_fp16"},
        # one query explores its candidate list: latency alone
        _sample(1, 1000, 1, temperature=0.5, top_k=50, top_p=0.9) | {"name": "sample_one_query"},
        # hard negatives for 256 queries out of their 1000 reranked candidates
        _sample(256, 1000, 8, temperature=0.7, top_k=100) | {"name": "sample_reranked"},
        # negatives out of the in-batch score matrix, the positives masked with -inf
        _sample(1024, 1024, 16, temperature=0.2, top_p=0.95, min_p=0.001, masked="diagonal", per_row=True)
        | {"name": "sample_in_batch"},
        # negatives out of a collection's 20000 documents
        _sample(512, 20000, 32, temperature=0.4, top_p=0.98) | {"name": "sample_collection"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["layer", "unit", "sample", "sample"])
    if op == "sample":
        cols = _log_int(rng, 8, 40000)
        return _sample(min(_log_int(rng, 1, 1024), max(1, 10_000_000 // cols)), cols,
                       min(cols, _log_int(rng, 1, 64)),
                       temperature=round(math.exp(rng.uniform(math.log(0.05), math.log(3.0))), 4),
                       top_k=rng.choice([0, _log_int(rng, 1, cols)]),
                       top_p=rng.choice([1.0, round(rng.uniform(0.3, 0.999), 4)]),
                       min_p=rng.choice([0.0, round(math.exp(rng.uniform(math.log(1e-4), math.log(0.3))), 5)]),
                       masked=rng.choice(["none", "diagonal", "some"]), per_row=rng.random() < 0.4)
    dim = _log_int(rng, 64, 1536) if op == "layer" else _log_int(rng, 16, 384)
    if rng.random() < 0.6:
        dim = dim // 16 * 16
    packed = rng.random() < 0.6
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    longest = _log_int(rng, 1, 512)
    weight = rng.choice(["none", dtype, dtype, "fp32"]) if op == "layer" else "none"
    return _norm(op, min(_log_int(rng, 1, 1024), max(1, 100_000_000 // (longest * dim))), longest,
                 rng.randint(1, longest) if packed else longest, dim, dtype, packed=packed,
                 train=rng.random() < 0.6, weight=weight, bias=weight != "none" and rng.random() < 0.7)


def _lengths(case):
    n, lo, hi = case["segments"], case["shortest"], case["longest"]
    return [hi if n == 1 else lo + round(i * (hi - lo) / (n - 1)) for i in range(n)]


def _eps(case):
    return 1e-5 if case["op"] == "layer" else 1e-12


def work(case):
    if case["op"] == "sample":
        cells, drawn = case["rows"] * case["cols"], case["rows"] * case["n"]
        return {"bytes": 8 * cells + 12 * drawn, "flops": 8 * cells}
    size, dim = _SIZE[case["dtype"]], case["dim"]
    rows = sum(_lengths(case))
    affine = (1 if case["weight"] != "none" else 0) + (1 if case["bias"] else 0)
    wide = affine * dim * _SIZE[case["weight"]]
    moved, flops = 2 * rows * dim * size + wide, 8 * rows * dim
    if case["packed"]:
        moved += 8 * case["segments"] + 4
    if case["train"]:  # the input again, the gradient in, the gradient of every padded row out
        moved += (2 * rows + case["segments"] * case["longest"]) * dim * size + 2 * wide
        flops += 14 * rows * dim
    return {"bytes": moved, "flops": flops}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *shape: torch.rand(shape, generator=g, device="cuda")  # noqa: E731
    randn = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    state = dict(case)
    if case["op"] == "sample":
        B, C = case["rows"], case["cols"]
        # sums of 32 maxima of cosines, a few relevant documents among them
        scores = 9.5 + 0.6 * randn(B, C) + 6.0 * rand(B, C) * (rand(B, C) < 0.01)
        if case["masked"] == "diagonal":
            scores[torch.arange(B, device="cuda"), torch.arange(B, device="cuda") % C] = -math.inf
        elif case["masked"] == "some":
            hole = rand(B, C)
            scores[hole < 0.2] = -math.inf
            scores[hole > 0.9] = torch.finfo(torch.float32).min
        state.update(scores=scores, uniforms=rand(B, C))
        if case["per_row"]:
            state["temperature"] = case["temperature"] * (0.5 + rand(B))
            state["top_p"] = case["top_p"] * (0.9 + 0.1 * rand(B))
        return state
    dtype, dim = _TYPES[case["dtype"]], case["dim"]
    lengths = torch.tensor(_lengths(case))
    state["total"] = int(lengths.sum())
    order = torch.randperm(len(lengths), generator=torch.Generator().manual_seed(seed))
    state["lengths"] = lengths[order].to(torch.int32).cuda()
    # hidden states: every channel with a scale and an offset of its own, a few of them large
    scale = 0.3 + rand(dim) + 8.0 * (rand(dim) < 0.01)
    x = torch.empty((case["segments"], case["longest"], dim), device="cuda", dtype=dtype)
    x.normal_(generator=g)
    state["tokens"] = x.mul_(scale.to(dtype)).add_((0.3 * randn(dim)).to(dtype))
    state["weight"] = state["bias"] = None
    if case["weight"] != "none":
        state["weight"] = (1.0 + 0.2 * randn(dim)).to(_TYPES[case["weight"]])
        if case["bias"]:
            state["bias"] = (0.1 * randn(dim)).to(_TYPES[case["weight"]])
    if not case["packed"]:
        state["tokens"] = state["tokens"].flatten(0, 1)
    if case["train"]:
        state["grad"] = torch.empty((state["total"], dim), device="cuda", dtype=dtype).normal_(generator=g).mul_(0.1)
        for name in ("tokens", "weight", "bias"):
            if state[name] is not None:
                state[name].requires_grad_(True)
    return state


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------

def _valid_rows(state):
    """Offsets of the packed rows, and the padded row that each one comes from."""
    lengths = state["lengths"].to(torch.int64)
    ends = torch.cumsum(lengths, 0)
    starts = ends - lengths
    shift = torch.arange(len(lengths), device="cuda") * state["longest"] - starts
    rows = torch.arange(state["total"], device="cuda")
    rows = rows + torch.repeat_interleave(shift, lengths, output_size=state["total"])
    return torch.cat([torch.zeros_like(ends[:1]), ends]).to(torch.int32), rows


def _plain_norm(state):
    tokens, dim, eps = state["tokens"].detach(), state["dim"], _eps(state)
    out, rows = {}, None
    if state["packed"]:
        out["offsets"], rows = _valid_rows(state)
        x = tokens.flatten(0, 1)[rows].float()
    else:
        x = tokens.float()
    w = None if state["weight"] is None else state["weight"].detach().float()
    if state["op"] == "layer":
        x = x - x.mean(dim=1, keepdim=True)
        inv = torch.rsqrt((x * x).mean(dim=1, keepdim=True) + eps)
    else:
        norm = torch.sqrt((x * x).sum(dim=1, keepdim=True))
        inv = 1.0 / norm.clamp(min=eps)
    h = x * inv
    y = h if w is None else h * w
    if state["bias"] is not None:
        y = y + state["bias"].detach().float()
    out["rows"] = y.to(tokens.dtype)
    if not state["train"]:
        return out
    g = state["grad"].float()
    u = g if w is None else g * w
    if state["op"] == "layer":
        dx = inv * (u - u.mean(dim=1, keepdim=True) - h * (u * h).mean(dim=1, keepdim=True))
        if w is not None:
            out["grad_weight"] = (g * h).sum(dim=0).to(state["weight"].dtype)
        if state["bias"] is not None:
            out["grad_bias"] = g.sum(dim=0).to(state["bias"].dtype)
    else:
        along = (u * h).sum(dim=1, keepdim=True) * (norm > eps)
        dx = inv * (u - h * along)
    if rows is None:
        out["grad_tokens"] = dx.to(tokens.dtype)
    else:
        full = torch.zeros((state["segments"] * state["longest"], dim), device="cuda", dtype=tokens.dtype)
        full[rows] = dx.to(tokens.dtype)
        out["grad_tokens"] = full.view(tokens.shape)
    return out


def _plain_sample(state):
    """In 64 bits: what is drawn hangs on comparisons of sums and logarithms."""
    s, C = state["scores"].double(), state["cols"]
    column = lambda v: v.double()[:, None] if isinstance(v, torch.Tensor) else v  # noqa: E731
    s = torch.where(torch.isnan(s), -math.inf, s)
    ranked, order = torch.sort(s, dim=1, descending=True, stable=True)
    best = ranked[:, :1]
    a = torch.where(ranked == best, 0.0, (ranked - best) / column(state["temperature"]))
    kept = (ranked > -math.inf) & (a >= -700.0)  # below, a weight counts as none
    if state["top_k"]:
        kept = kept & (torch.arange(C, device="cuda") < state["top_k"])
    w = torch.where(kept, torch.exp(a), 0.0)
    upto, p = torch.cumsum(w, dim=1), column(state["top_p"])
    p = torch.where(torch.as_tensor(p) >= 1.0, math.inf, p)  # 1 keeps all, whatever the last bits of a sum
    kept = kept & (upto - w < p * upto[:, -1:]) & (w >= state["min_p"])
    w = torch.where(kept, w, 0.0)
    share = w / w.sum(dim=1, keepdim=True)
    race = a - torch.log(-torch.log(torch.gather(state["uniforms"].double(), 1, order)))
    race = torch.where(kept, race.clamp(min=-1e300), -math.inf)  # a uniform of 0 comes last, but comes
    back = lambda v: torch.zeros_like(v).scatter_(1, order, v)  # noqa: E731
    first = torch.sort(back(race), dim=1, descending=True, stable=True).indices[:, : state["n"]]
    there = torch.gather(back(kept), 1, first)
    return {"indices": torch.where(there, first, -1),
            "probabilities": torch.where(there, torch.gather(back(share), 1, first), 0.0).float()}


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def _own_norm(state):
    import maxsim_b200 as maxsim

    x, w, b, out = state["tokens"], state["weight"], state["bias"], {}
    if state["op"] == "layer":
        if state["packed"]:
            y, out["offsets"] = maxsim.pack_layer_norm(x, state["lengths"], w, b, total_tokens=state["total"])
        else:
            y = maxsim.layer_norm(x, w, b)
    elif state["packed"]:
        y, out["offsets"] = maxsim.pack_unit_norm(x, state["lengths"], total_tokens=state["total"])
    else:
        y = maxsim.unit_norm(x)
    out["rows"] = y
    if state["train"]:
        leaves = {k: t for k, t in (("grad_tokens", x), ("grad_weight", w), ("grad_bias", b)) if t is not None}
        out.update(zip(leaves, torch.autograd.grad(y, list(leaves.values()), state["grad"])))
        out["rows"] = y.detach()
    return out


def _own_sample(state):
    import maxsim_b200 as maxsim

    indices, probabilities = maxsim.sample_candidates(
        state["scores"], state["uniforms"], state["n"], temperature=state["temperature"],
        top_k=state["top_k"] or None, top_p=state["top_p"], min_p=state["min_p"])
    return {"indices": indices, "probabilities": probabilities}


def run(state):
    if own:
        return _own_sample(state) if state["op"] == "sample" else _own_norm(state)
    return _plain_sample(state) if state["op"] == "sample" else _plain_norm(state)


# ---------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------

def _exact_rows(case, x, w, b):
    if case["op"] == "unit":
        return x / torch.linalg.vector_norm(x, dim=-1, keepdim=True).clamp_min(_eps(case))
    var, mean = torch.var_mean(x, dim=-1, correction=0, keepdim=True)
    y = (x - mean) / torch.sqrt(var + _eps(case))
    y = y if w is None else y * w
    return y if b is None else y + b


def _exact_norm(case, seed):
    """Sequence by sequence, the gradients by differentiation of the forward."""
    state = prepare(case, seed)
    x, dim = state["tokens"].detach(), case["dim"]
    wide = lambda t: None if t is None else t.detach().double().requires_grad_(True)  # noqa: E731
    w, b = wide(state["weight"]), wide(state["bias"])
    lengths = state["lengths"].tolist() if case["packed"] else [case["longest"]] * case["segments"]
    x = x.view(case["segments"], case["longest"], dim)
    y = torch.empty((sum(lengths), dim), device="cuda", dtype=torch.float64)
    dx = torch.zeros(x.shape, device="cuda", dtype=torch.float64) if case["train"] else None
    at = 0
    for i, n in enumerate(lengths):
        part = x[i, :n].double().requires_grad_(True)
        rows = _exact_rows(case, part, w, b)
        y[at:at + n] = rows.detach()
        if case["train"]:
            rows.backward(state["grad"][at:at + n].double())
            dx[i, :n] = part.grad
        at += n
    out = {"rows": y, "offsets": None} if case["packed"] else {"rows": y}
    if case["train"]:
        out["grad_tokens"] = dx if case["packed"] else dx.flatten(0, 1)
        if w is not None:
            out["grad_weight"] = w.grad
        if b is not None:
            out["grad_bias"] = b.grad
    return out


def _exact_sample(case, seed):
    """Row by row on the host: candidates in order, cut where a filter ends, raced."""
    state = prepare(case, seed)
    host = lambda v, i: float(v[i]) if isinstance(v, np.ndarray) else v  # noqa: E731
    scores = state["scores"].cpu().numpy().astype(np.float64)
    uniforms = state["uniforms"].cpu().numpy().astype(np.float64)
    params = {k: state[k].cpu().numpy() if isinstance(state[k], torch.Tensor) else state[k]
              for k in ("temperature", "top_p")}
    B, n = case["rows"], case["n"]
    indices, share = np.full((B, n), -1, dtype=np.int64), np.zeros((B, n))
    for i in range(B):
        T, p = (host(params[k], i) for k in ("temperature", "top_p"))
        there = np.flatnonzero(scores[i] > -np.inf)
        there = there[scores[i, there] - scores[i].max() >= -700.0 * T]
        if not len(there):
            continue
        there = there[np.lexsort((there, -scores[i, there]))]
        if case["top_k"]:
            there = there[: case["top_k"]]
        z = scores[i, there] / T
        w = np.exp(z - z[0])
        before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
        size = len(w) if p >= 1.0 else int(np.sum(before < p * w.sum()))
        size = min(size, int(np.sum(w >= case["min_p"])))
        there, w = there[:size], w[:size]
        with np.errstate(divide="ignore"):
            arrival = np.log(-np.log(uniforms[i, there])) - np.log(w)  # of exponential clocks with rates w
        first = np.lexsort((there, arrival))[:n]
        indices[i, : len(first)] = there[first]
        share[i, : len(first)] = w[first] / w.sum()
    return {"indices": indices, "probabilities": share}


def exact(case, seed):
    return _exact_sample(case, seed) if case["op"] == "sample" else _exact_norm(case, seed)
