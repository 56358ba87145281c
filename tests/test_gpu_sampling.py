"""Drawing candidates on the GPU against the 64-bit oracle: the indices have to
be equal, the probabilities are one fp32 rounding (and a mass rounded to whole
numbers, below 1e-9) from the oracle's."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import maxsim_b200 as maxsim
from maxsim_b200 import _ops
from oracle import maxsim_oracle as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
INF = float("inf")


def scores_of(B, C, seed, spread=0.6):
    g = torch.Generator().manual_seed(seed)
    return (9.5 + spread * torch.randn(B, C, generator=g)), torch.rand(B, C, generator=g)


def as_params(kw):
    return {k: (v.cpu().numpy() if isinstance(v, torch.Tensor) else v) for k, v in kw.items() if v is not None}


def check(s, u, n, **kw):
    got, share = maxsim.sample_candidates(s.to(DEV), u.to(DEV), n, **{
        k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in kw.items()})
    assert got.dtype == torch.int64 and share.dtype == torch.float32 and got.shape == share.shape == (s.shape[0], n)
    want, wshare = oracle.sample_candidates(s.float().numpy(), u.numpy(), n, **as_params(kw))
    np.testing.assert_array_equal(got.cpu().numpy(), want)
    np.testing.assert_allclose(share.cpu().numpy(), wshare, rtol=2.0 ** -23, atol=2.0 ** -126)
    return got, share


FILTERS = [dict(), dict(top_k=1), dict(top_k=7), dict(top_p=0.5), dict(top_p=0.999), dict(min_p=0.2), dict(min_p=1.0),
           dict(top_k=20, top_p=0.8), dict(top_k=13, top_p=0.9, min_p=0.05), dict(top_p=0.97, min_p=0.001)]


@pytest.mark.parametrize("C", [1, 2, 3, 31, 32, 33, 255, 256, 257, 1000, 1024, 1025])
@pytest.mark.parametrize("kw", FILTERS, ids=str)
def test_filters(C, kw):
    s, u = scores_of(5, C, C)
    check(s, u, min(C, 9), temperature=0.3, **kw)


@pytest.mark.parametrize("T", [1e-310, 1e-3, 0.05, 1.0, 30.0, 1e300, INF])
def test_temperatures(T):
    s, u = scores_of(6, 300, 1)
    check(s, u, 20, temperature=T, top_p=0.9)
    check(s, u, 300, temperature=T)


@pytest.mark.parametrize("B,C,n", [(1, 4096, 64), (3, 20000, 32), (2, 5001, 1024), (1, 70000, 16), (300, 64, 64),
                                   (2, 12289, 300), (2, 40000, 5)])
def test_long_rows(B, C, n):
    s, u = scores_of(B, C, C)
    check(s, u, n, temperature=0.5)
    check(s, u, n, temperature=0.5, top_k=C // 3, top_p=0.9)
    check(s, u, n, temperature=0.2, top_p=0.99, min_p=1e-4)


@pytest.mark.parametrize("B,C,n", [
    (1, 16383, 5), (1, 16384, 40), (2, 16385, 3), (27, 16387, 4), (28, 16388, 4), (74, 16390, 2), (75, 16389, 2),
    (1, 32768, 7), (13, 32771, 4), (14, 32769, 1), (1, 99999, 33), (40, 90113, 1), (1, 327680, 5), (1, 327683, 16),
    (6, 327681, 2), (7, 327682, 2), (1, 655361, 9), (1, 2 ** 20, 1024), (1, 2 ** 20, 1)])
def test_rows_shared_by_a_cluster(B, C, n):
    """Few long rows are split over the CTAs of a cluster: at and around every size where
    the split changes, equal to the same rows drawn one CTA each, among copies of them."""
    s, u = scores_of(B, C, C)
    s[:, C // 2::977] = s[:, :1]  # equal scores in every slice
    s, u = s.to(DEV), u.to(DEV)
    copies = 75 if C <= 100000 else 3
    for kw in (dict(temperature=0.5), dict(temperature=0.3, top_p=0.9), dict(temperature=1.0, top_k=C // 3, min_p=1e-3),
               dict(temperature=0.2, top_k=50, top_p=0.97)):
        got, share = maxsim.sample_candidates(s, u, n, **kw)
        if C <= 100000:
            want, wshare = maxsim.sample_candidates(s[:1].expand(copies, C), u[:1].expand(copies, C), n, **kw)
            assert torch.equal(got[0], want[0]) and torch.equal(want, want[:1].expand_as(want))
            torch.testing.assert_close(share[0], wshare[0], rtol=2.0 ** -22, atol=0)
        check_by_sorting(s[0], u[0], got[0], share[0], **kw)
        if B > 1:
            check_by_sorting(s[-1], u[-1], got[-1], share[-1], **kw)


def check_by_sorting(s, u, got, share, temperature, top_k=None, top_p=None, min_p=None):
    """One row against the definition in 64-bit torch operations, for rows too long for
    the oracle's loops."""
    best, order = torch.sort(s.double(), descending=True, stable=True)
    a = (best - best[0]) / temperature
    keep = torch.arange(len(a), device=a.device) < (top_k or len(a))
    w = torch.where(keep, a.exp(), 0.0)
    if top_p:
        keep &= w.cumsum(0) - w < top_p * w.sum()
    if min_p:
        keep &= a >= float(np.log(min_p))
    race = torch.where(keep, a - torch.log(-torch.log(u.double()[order])), -INF)
    race, place = torch.sort(race, descending=True, stable=True)
    n = min(len(got), int(keep.sum()))
    assert torch.equal(got[:n], order[place[:n]]) and (got[n:] == -1).all()
    want = (a.exp() / torch.where(keep, a.exp(), 0.0).sum())[place[:n]]
    torch.testing.assert_close(share[:n].double(), want, rtol=2.0 ** -23, atol=2.0 ** -126)


def test_clusters_meet_every_kind_of_row():
    """Empty rows, +inf, equal scores, uniforms at their ends, more draws than
    candidates: the paths of a row, in a cluster."""
    C = 16500
    s, u = scores_of(8, C, 3)
    s[0] = -INF
    s[1] = float("nan")
    s[2, 5:] = -INF
    s[3, ::41] = INF
    s[4] = 2.0
    s[5] = (s[5] * 4).round() / 4
    u[6, ::2] = 0.0
    u[6, 1::4] = 1.0
    u[7, ::3] = 1e-40
    for kw in (dict(), dict(top_p=0.6), dict(top_k=700, temperature=0.1), dict(min_p=0.3, temperature=5.0)):
        check(s, u, 12, **kw)
    check(s[:5], u[:5], 600, top_p=0.9)


def test_masked_rows():
    """-inf, NaN, the type's lowest value, +inf, and rows with nothing left."""
    s, u = scores_of(9, 70, 3)
    s[0, ::2] = -INF
    s[1, 5:60] = float("nan")
    s[2, 10:] = torch.finfo(torch.float32).min
    s[3] = -INF
    s[4] = float("nan")
    s[5, [3, 40, 41]] = INF
    s[6] = torch.finfo(torch.float32).min  # all of them the best: uniform
    s[7, :69] = -INF
    s[8, 7] = torch.finfo(torch.float32).max
    s[8, 8] = -torch.finfo(torch.float32).max
    for kw in FILTERS:
        got, share = check(s, u, 12, temperature=0.7, **kw)
        assert (got[3] == -1).all() and not share[3].any() and (got[4] == -1).all()
        assert set(got[5].tolist()) <= {3, 40, 41, -1}
        assert got[7].tolist() == [69] + [-1] * 11
    half = s.half()
    check(half, u, 12, temperature=0.7, top_p=0.9)
    check(s.bfloat16(), u, 12, temperature=0.7, top_k=9)


def test_ties_go_to_the_lowest_index():
    u = torch.full((3, 40), 0.5)
    s = torch.zeros(3, 40)
    s[1, 20:] = 1.0
    s[2, ::3] = -0.0  # equal to +0
    for kw in FILTERS:
        check(s, u, 15, **kw)
    got, _ = check(s, u, 15, top_k=10)
    assert got[0].tolist() == list(range(10)) + [-1] * 5
    assert got[1].tolist() == list(range(20, 30)) + [-1] * 5
    got, _ = check(s, u, 15, top_p=0.5)  # twenty before which less than half lies
    assert got[0].tolist() == list(range(15))
    coarse, v = scores_of(8, 600, 4)
    check(coarse.round(decimals=1), v, 40, top_k=100, temperature=0.4)
    check(coarse.round(decimals=1), v, 40, top_p=0.77, temperature=0.4)
    check(coarse.round(decimals=1), (v * 8).floor() / 8, 40, top_p=0.77, temperature=0.4)


def test_uniforms_at_and_outside_their_ends():
    s, u = scores_of(4, 50, 5)
    u[0, 10:20] = 0.0      # last of the kept, but drawn
    u[1, 7], u[1, 30] = 1.0, 1.0  # first
    u[2, 5:9] = float("nan")      # left out, as are values outside [0, 1]
    u[2, 9], u[2, 10] = -0.5, 1.5
    u[3] = 0.0
    got, _ = check(s, u, 50)
    assert set(got[0, -10:].tolist()) == set(range(10, 20))
    assert got[1, 0] == 7 and got[1, 1] == 30
    assert (got[2] == -1).sum() == 6
    assert got[3].tolist() == list(range(50))
    check(s, u, 20, top_k=30, top_p=0.9)


def test_many_equal_values():
    """More equal scores or race values than the kernels list."""
    C = 5000
    u = torch.rand(4, C, generator=torch.Generator().manual_seed(0))
    s = torch.zeros(4, C)
    s[1, ::2] = -1.0
    s[2, :100] = 5.0
    s[3, 4000:] = 2.0
    for kw in (dict(), dict(top_k=700), dict(top_k=3000, top_p=0.9), dict(top_p=0.37), dict(min_p=0.5), dict(top_p=0.999)):
        check(s, u, 30, **kw)
    check(s, torch.full((4, C), 0.25), 30)          # all race values of equal scores equal
    check(s, torch.full((4, C), 0.25), 1000, top_k=2500)
    check(s, (u * 4).floor() / 4 + 0.125, 60)
    got, _ = check(s, torch.full((4, C), 0.25), 5, top_k=700)
    assert got[0].tolist() == [0, 1, 2, 3, 4] and got[3].tolist() == [4000, 4001, 4002, 4003, 4004]


def test_scores_at_every_scale():
    """Clusters that a linear map of the whole range cannot tell apart, outliers on both
    sides, values next to zero and at both ends of the type."""
    g = torch.Generator().manual_seed(1)
    C = 4096
    u = torch.rand(8, C, generator=g)
    s = torch.randn(8, C, generator=g)
    s[0] = 1.0 + s[0] * 1e-6
    s[0, 17] = 3e38
    s[0, 18] = -3e38
    s[1] = 2.0 ** torch.randint(-140, 120, (C,), generator=g).float()
    s[2] = s[2] * 1e-40                      # subnormal
    s[3] = -(2.0 ** torch.randint(-140, 120, (C,), generator=g).float())
    s[4, ::3] = 0.0
    s[4, 1::3] = -0.0
    s[5] = torch.linspace(-3.4e38, 3.4e38, C)
    s[6] = (s[6] * 3).round()
    s[7] = 1e9 + (s[7] * 10).round() * 64
    for T in (1e-38, 1e-3, 0.01, 1.0, 1e30, INF):
        for kw in (dict(), dict(top_k=300), dict(top_k=1500, top_p=0.7), dict(top_p=0.6), dict(min_p=1.0), dict(min_p=1e-30)):
            check(s, u, 20, temperature=T, **kw)
    check(torch.tensor([[7.0, 0.0, 1e-30, -1e-30, 3.5]]), torch.tensor([[0.5, 0.6, 0.7, 0.8, 0.9]]), 5, temperature=0.01)
    check(torch.zeros(1, 400), torch.rand(1, 400, generator=g), 9, min_p=1.0)
    infinite = s.clone()
    infinite[:, ::5] = INF
    for T in (1e-310, 1.0, INF):
        for kw in (dict(), dict(top_k=300), dict(top_p=0.6), dict(min_p=0.5)):
            check(infinite, u, 20, temperature=T, **kw)


def test_uniforms_below_the_normal_range():
    s, u = scores_of(3, 400, 12)
    u[0, ::2] = 1e-40
    u[1, 5] = 1e-45
    check(s, u, 250)
    check(s, u, 20, top_k=100)


def test_rows_around_the_choices_of_a_launch():
    """Row counts and widths on both sides of where another number of threads is taken."""
    for B, C, n in ((593, 40, 5), (800, 300, 130), (600, 2048, 128), (592, 100, 20), (3, 2049, 40), (296, 8192, 9), (297, 8192, 9), (297, 8193, 9), (2, 24576, 40),
                    (2, 24577, 40), (2, 40960, 40), (2, 40961, 40), (1, 300_001, 9)):
        s, u = scores_of(B, C, B + C)
        some = torch.randperm(B, generator=torch.Generator().manual_seed(0))[:3]
        got, share = maxsim.sample_candidates(s.to(DEV), u.to(DEV), n, temperature=0.6, top_k=C // 2 + 1, top_p=0.95)
        want, wshare = oracle.sample_candidates(s[some].numpy(), u[some].numpy(), n, 0.6, C // 2 + 1, 0.95)
        np.testing.assert_array_equal(got[some].cpu().numpy(), want)
        np.testing.assert_allclose(share[some].cpu().numpy(), wshare, rtol=2.0 ** -23)


def test_two_streams_at_once():
    parts = [tuple(t.to(DEV) for t in scores_of(300, 1500, i)) for i in range(2)]
    want = [maxsim.sample_candidates(s, u, 10, temperature=0.4, top_p=0.9) for s, u in parts]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in parts]
    got = [[], []]
    for _ in range(5):
        for i, (s, u) in enumerate(parts):
            with torch.cuda.stream(streams[i]):
                got[i].append(maxsim.sample_candidates(s, u, 10, temperature=0.4, top_p=0.9))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for run in got[i] for a, b in zip(run, want[i]))


def test_one_value_per_row():
    B = 12
    s, u = scores_of(B, 200, 6)
    T = torch.linspace(0.1, 2.0, B)
    T[3], T[4], T[5] = 0.0, -1.0, float("nan")  # rows that draw nothing
    k = torch.tensor([0, 1, 2, 3, 4, 5, -7, 50, 199, 200, 201, 2 ** 31 - 1], dtype=torch.int32)
    p = torch.linspace(0.05, 1.1, B)
    p[7], p[8] = -0.1, float("nan")
    m = torch.linspace(-0.1, 1.1, B) ** 3
    check(s, u, 9, temperature=T)
    check(s, u, 9, top_k=k)
    check(s, u, 9, top_k=k.long(), temperature=0.4)
    check(s, u, 9, top_k=k.long() + 2 ** 33, temperature=0.4)
    check(s, u, 9, top_p=p)
    check(s, u, 9, min_p=m)
    got, _ = check(s, u, 9, temperature=T, top_k=k, top_p=p, min_p=m)
    assert (got[3:6] == -1).all()


def test_strided_rows():
    s, u = scores_of(6, 500, 7)
    S, U = s.to(DEV), u.to(DEV)
    want = maxsim.sample_candidates(S[:, 3:300].contiguous(), U[:, 100:397].contiguous(), 8, top_p=0.8)
    got = maxsim.sample_candidates(S[:, 3:300], U[:, 100:397], 8, top_p=0.8)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = maxsim.sample_candidates(S[:, 3:300].T.contiguous().T, U[:, 100:397], 8, top_p=0.8)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    one = maxsim.sample_candidates(S[:1].expand(4, 500), U[:1].expand(4, 500), 8)
    assert torch.equal(one[0][0], one[0][3])
    unaligned = S.flatten()[1:].view(-1)[: 5 * 499].view(5, 499)
    check(unaligned.cpu(), u[:5, :499], 8, top_k=40)


def test_nothing_to_draw():
    s, u = scores_of(3, 20, 8)
    got, share = maxsim.sample_candidates(s.to(DEV), u.to(DEV), 0)
    assert got.shape == share.shape == (3, 0)
    got, _ = maxsim.sample_candidates(torch.empty(0, 20, device=DEV), torch.empty(0, 20, device=DEV), 5)
    assert got.shape == (0, 5)
    got, _ = maxsim.sample_candidates(torch.empty(4, 0, device=DEV), torch.empty(4, 0, device=DEV), 0)
    assert got.shape == (4, 0)
    with pytest.raises(RuntimeError, match="scores' device"):
        maxsim.sample_candidates(s.to(DEV), u.to(DEV), 2, temperature=torch.ones(3))


def test_draws_follow_the_weights():
    """Counts of the first draw over 40000 rows of the same scores, within five
    standard deviations of the filtered softmax."""
    row = torch.tensor([1.0, 0.2, 2.0, -INF, 0.7, 1.5, 1.4, -3.0])
    B, T = 40000, 0.8
    u = torch.rand(B, 8, generator=torch.Generator().manual_seed(0)).to(DEV)
    got, share = maxsim.sample_candidates(row.to(DEV).expand(B, 8), u, 3, temperature=T, top_k=5)
    p = torch.exp(row / T) * (row >= 0.99)
    p[4] = torch.exp(row[4] / T)
    p = (p / p.sum()).double().numpy()
    counts = torch.bincount(got[:, 0], minlength=8).cpu().numpy()
    assert np.all(np.abs(counts - B * p) <= 5 * np.sqrt(B * p * (1 - p)))
    srt = got.sort(dim=1).values
    assert (srt[:, 1:] != srt[:, :-1]).all()
    np.testing.assert_allclose(share.cpu().numpy(), p[got.cpu().numpy()], rtol=1e-6)


def test_replays_from_a_graph_and_repeats_its_bits():
    s, u = (t.to(DEV) for t in scores_of(64, 3000, 9))
    T = torch.full((64,), 0.5, device=DEV)
    call = lambda: maxsim.sample_candidates(s, u, 16, temperature=T, top_k=500, top_p=0.9)  # noqa: E731
    first = call()
    assert all(torch.equal(a, b) for a, b in zip(first, call()))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    s2, u2 = scores_of(64, 3000, 10)
    s.copy_(s2)
    u.copy_(u2)
    T.fill_(0.3)
    graph.replay()
    torch.cuda.synchronize()
    want = call()
    assert all(torch.equal(a, b) for a, b in zip(out, want)) and not torch.equal(out[0], first[0])


def test_hard_negatives_for_a_training_step():
    """Scores of a contrastive batch -> negatives drawn with the positive masked ->
    the candidates gathered -> the padded training operator and its gradients."""
    torch.manual_seed(0)
    Nq, Lq, D, L, n = 10, 16, 64, 24, 4
    q = maxsim.unit_norm(torch.randn(Nq, Lq, D, device=DEV)).half()
    enc = torch.randn(Nq, L, D, device=DEV)
    lengths = torch.randint(3, L + 1, (Nq,), dtype=torch.int32)
    docs, off = maxsim.pack_unit_norm(enc.half(), lengths)
    scores = maxsim.score_contrastive(q, docs, off)
    masked = scores.clone().fill_diagonal_(-INF)
    u = torch.rand(masked.shape, device=DEV)
    neg, _ = check(masked.cpu(), u.cpu(), n, temperature=0.5, top_k=6)
    assert (neg >= 0).all() and (neg != torch.arange(Nq, device=DEV)[:, None]).all()
    chosen = torch.cat([torch.arange(Nq, device=DEV)[:, None], neg], 1)
    cand = maxsim.unpack_packed(docs, off, L)[chosen].detach().requires_grad_(True)
    qa = q.clone().requires_grad_(True)
    s = maxsim.score_candidates_padded_train(qa, cand, torch.full((Nq,), Lq, dtype=torch.int32, device=DEV),
                                             lengths.to(DEV)[chosen])
    torch.testing.assert_close(s.detach(), torch.gather(scores, 1, chosen), rtol=2e-2, atol=1e-2)
    loss = torch.nn.functional.cross_entropy(s / 0.5, torch.zeros(Nq, dtype=torch.long, device=DEV))
    gq, gd = torch.autograd.grad(loss, (qa, cand))
    assert torch.isfinite(gq).all() and torch.isfinite(gd).all() and gq.abs().sum() > 0
    assert _ops.device_status() == 0


def tiny_scores(B, C, T, seed):
    """Scores a few subnormal temperatures apart, a tenth of them masked."""
    g = torch.Generator().manual_seed(seed)
    s = (torch.randn(B, C, generator=g, dtype=torch.float64) * (5 * T)).float()
    u = torch.rand(B, C, generator=g)
    s[torch.rand(B, C, generator=g) < 0.1] = -INF
    s[:, 0] = 0.0
    return s, u


@pytest.mark.parametrize("T", [1e-38, 2e-39, 1e-39, 3e-40, 1e-42, 1e-44, 1.4e-45])
@pytest.mark.parametrize("C", [30, 257, 1023, 4093])
def test_subnormal_temperatures(T, C):
    """1 / T is past the 32-bit range; what is masked, and what lies behind a row whose length is no
    multiple of four, is never drawn."""
    s, u = tiny_scores(5, C, T, C)
    s[1, 2::5] = float("nan")
    s[2, 5:] = -INF
    s[3, C // 2:] = 1.0  # far above everything else
    for kw in (dict(), dict(top_k=11), dict(top_k=C // 2), dict(top_p=0.9), dict(min_p=0.1), dict(top_k=C // 2, top_p=0.7)):
        check(s, u, min(C, 25), temperature=T, **kw)
    check(s, u, 9, temperature=torch.full((5,), T, dtype=torch.float64).float(), top_k=20)
    pair = torch.tensor([[1e-38, 0.0]])
    check(pair, torch.tensor([[0.5, 0.5]]), 1, temperature=T)
    check(pair, torch.tensor([[0.5, 0.99]]), 2, temperature=T)


@pytest.mark.parametrize("B,C", [(2, 16501), (1, 330001), (75, 41001)])
def test_subnormal_temperatures_in_long_rows(B, C):
    """In a cluster, and in rows that are read again instead of kept."""
    s, u = (t.to(DEV) for t in tiny_scores(B, C, 1e-40, C))
    for kw in (dict(), dict(top_k=C // 3), dict(top_p=0.9)):
        got, share = maxsim.sample_candidates(s, u, 33, temperature=1e-40, **kw)
        for row in (0, B - 1):
            check_by_sorting(s[row], u[row], got[row], share[row], temperature=1e-40, **kw)


def ramp(C, dtype=torch.float64):
    """From the lowest value of the type to the largest.  In 32 bits torch's own steps overflow:
    +inf, -inf and NaN."""
    top = torch.finfo(torch.float32).max
    return torch.linspace(-top, top, C, dtype=dtype).float()


@pytest.mark.parametrize("T", [1e35, 1e36, 3e37, 1e38, 3e38, 1e39, 1e40, 1e42, 1e45, 1e300])
def test_scores_further_apart_than_the_type_reaches(T):
    """Differences that are no 32-bit numbers, at temperatures that leave all scores a chance."""
    g = torch.Generator().manual_seed(5)
    for B, C, n in ((12, 1022, 20), (4, 4096, 60), (2, 16501, 20)):
        for dtype in (torch.float64, torch.float32):
            s = ramp(C, dtype).expand(B, C).clone()
            s[1] = s[1][torch.randperm(C, generator=g)]
            s[1, ::7] = -INF
            u = torch.rand(B, C, generator=g)
            for kw in (dict(), dict(top_k=C - 5), dict(top_p=0.95), dict(min_p=1e-9)):
                check(s, u, n, temperature=T, **kw)


def test_long_rows_further_apart_than_the_type_reaches():
    """In a cluster, and in rows that are read again instead of kept."""
    for B, C in ((1, 330001), (75, 41001)):
        u = torch.rand(B, C, generator=torch.Generator(device=DEV).manual_seed(B), device=DEV)
        s = ramp(C).to(DEV).expand(B, C)
        assert torch.isfinite(s).all()
        for kw in (dict(temperature=1e38), dict(temperature=1e39, top_k=C // 2), dict(temperature=1e38, top_p=0.9)):
            got, share = maxsim.sample_candidates(s, u, 33, **kw)
            for row in (0, B - 1):
                check_by_sorting(s[row], u[row], got[row], share[row], **kw)
        check(ramp(C, torch.float32)[None], u[:1].cpu(), 33, temperature=1e38)


@pytest.mark.parametrize("T,step,p", [(1e-46, 1, 1 - 1e-7), (2e-45, 38, 1 - 1e-9), (1e-45, 15, 1 - 1e-9)])
def test_masses_at_temperatures_between_the_smallest_floats(T, step, p):
    """One best score and others `step` of the smallest float below it: the mass that top-p
    leaves to them depends on the temperature as it was given, which is no float."""
    g = torch.Generator().manual_seed(step)
    s = torch.full((4, 2000), -step * 2.0 ** -149)
    s[0, 700] = s[1, 0] = s[2, 1999] = s[3, 5] = 0.0
    s[3, ::11] = -INF
    u = torch.rand(4, 2000, generator=g)
    got, _ = check(s, u, 50, temperature=T, top_p=p)
    assert (got >= 0).all()
    check(s, u, 50, temperature=T, top_p=p, top_k=1500)
