"""CPU checks of row normalisation and sampling: the oracle against plain torch,
its gradients against differences, its draws against the distribution they
stand for, and the refusals of the public functions."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import maxsim_b200 as maxsim
from maxsim_b200 import _ops
from oracle import maxsim_oracle as oracle


def test_oracle_matches_torch_in_64_bits():
    rng = np.random.default_rng(0)
    x, w, b = rng.standard_normal((7, 33)), rng.standard_normal(33), rng.standard_normal(33)
    want = torch.nn.functional.layer_norm(torch.from_numpy(x), (33,), torch.from_numpy(w), torch.from_numpy(b), 1e-5)
    np.testing.assert_allclose(oracle.layer_norm(x, w, b), want.numpy(), rtol=1e-12, atol=1e-12)
    np.testing.assert_allclose(oracle.unit_norm(x), torch.nn.functional.normalize(torch.from_numpy(x), dim=-1).numpy(),
                               rtol=1e-13)


def test_oracle_gradients_match_differences():
    rng = np.random.default_rng(1)
    x, w, b, g = (rng.standard_normal(s) for s in ((3, 9), 9, 9, (3, 9)))
    step = 1e-6  # truncation ~ step^2, rounding ~ 2^-53 / step: both below 1e-9

    def slope(f, v):
        out = np.zeros_like(v)
        for i in np.ndindex(v.shape):
            up, down = v.copy(), v.copy()
            up[i] += step
            down[i] -= step
            out[i] = (f(up) - f(down)) / (2 * step)
        return out

    dx, dw, db = oracle.layer_norm_backward(g, x, w)
    np.testing.assert_allclose(dx, slope(lambda v: (g * oracle.layer_norm(v, w, b)).sum(), x), atol=1e-8)
    np.testing.assert_allclose(dw, slope(lambda v: (g * oracle.layer_norm(x, v, b)).sum(), w), atol=1e-8)
    np.testing.assert_allclose(db, slope(lambda v: (g * oracle.layer_norm(x, w, v)).sum(), b), atol=1e-8)
    np.testing.assert_allclose(oracle.unit_norm_backward(g, x), slope(lambda v: (g * oracle.unit_norm(v)).sum(), x),
                               atol=1e-8)
    short = x * 1e-3  # shorter than eps: a constant factor
    np.testing.assert_allclose(oracle.unit_norm_backward(g, short, eps=1.0), g)


def test_oracle_draws_follow_the_weights():
    """First draws over 20000 rows of the same scores: counts within five standard
    deviations of the filtered softmax; second draws are never the first again."""
    rng = np.random.default_rng(2)
    row = np.array([1.0, 0.2, 2.0, -np.inf, 0.7, 1.5])
    B, T = 20000, 0.8
    got, share = oracle.sample_candidates(np.tile(row, (B, 1)), rng.random((B, 6)), 2, T, top_k=4)
    p = np.exp(row / T) * (row >= 0.7)
    p /= p.sum()
    counts = np.bincount(got[:, 0], minlength=6)
    assert np.all(np.abs(counts - B * p) <= 5 * np.sqrt(B * p * (1 - p)))
    assert np.all(got[:, 0] != got[:, 1])
    # second draw given the first: proportional to what is left
    rest = got[got[:, 0] == 2, 1]
    q = p.copy()
    q[2] = 0
    q /= q.sum()
    counts = np.bincount(rest, minlength=6)
    assert np.all(np.abs(counts - len(rest) * q) <= 5 * np.sqrt(len(rest) * q * (1 - q)))
    np.testing.assert_allclose(share, p[got])


def test_oracle_filters():
    u = np.full((1, 5), 0.5)
    s = np.log([[0.4, 0.1, 0.3, 0.15, 0.05]])
    draw = lambda **kw: oracle.sample_candidates(s, u, 5, **kw)[0][0].tolist()  # noqa: E731
    assert draw() == [0, 2, 3, 1, 4]  # equal uniforms: by weight
    assert draw(top_k=2) == [0, 2, -1, -1, -1]
    assert draw(top_p=0.72) == [0, 2, 3, -1, -1]   # 0.7 lies before the third
    assert draw(top_p=0.01) == [0, -1, -1, -1, -1]
    assert draw(min_p=0.3) == [0, 2, 3, -1, -1]    # 0.15 >= 0.3 * 0.4
    assert draw(top_k=4, top_p=0.9) == [0, 2, 3, 1, -1]  # 0.85 lies before the fourth, the limit is 0.9 * 0.95 = 0.855
    assert draw(top_p=0.84) == [0, 2, 3, -1, -1]  # of all five: 0.85 >= 0.84
    tied = np.zeros((1, 5))
    assert oracle.sample_candidates(tied, u, 5, top_k=2)[0][0].tolist() == [0, 1, -1, -1, -1]


def test_norm_refusals():
    x = torch.zeros(4, 8, 16)
    for call in (maxsim.layer_norm, maxsim.unit_norm):
        with pytest.raises(RuntimeError, match="CUDA"):
            call(x)
        with pytest.raises(TypeError, match="float32, float16, or bfloat16"):
            call(x.to(torch.int32))
        with pytest.raises(TypeError, match="float32, float16, or bfloat16"):
            call(x.double())
        with pytest.raises(ValueError, match="at least one element"):
            call(x[..., :0])
        with pytest.raises(ValueError, match="at least 1-D"):
            call(torch.zeros(()))
        for eps in (0.0, -1.0, float("nan"), float("inf"), 1e-31):
            with pytest.raises(ValueError, match="eps"):
                call(x, eps=eps)
    w = torch.ones(16)
    with pytest.raises(ValueError, match="weight must have shape"):
        maxsim.layer_norm(x, torch.ones(8))
    with pytest.raises(ValueError, match="bias must have shape"):
        maxsim.layer_norm(x, w, torch.ones(1, 16))
    with pytest.raises(ValueError, match="bias needs a weight"):
        maxsim.layer_norm(x, None, w)
    with pytest.raises(TypeError, match="weight must be float32"):
        maxsim.layer_norm(x, w.half())
    with pytest.raises(TypeError, match="weight must be float32"):
        maxsim.layer_norm(x.half(), w.bfloat16())
    with pytest.raises(TypeError, match="same dtype"):
        maxsim.layer_norm(x.half(), w.half(), w)
    lengths = torch.tensor([1, 2, 3, 8])
    with pytest.raises(RuntimeError, match="CUDA"):
        maxsim.pack_layer_norm(x, lengths)
    with pytest.raises(ValueError, match="3-D"):
        maxsim.pack_layer_norm(x[0], lengths)
    with pytest.raises(ValueError, match="3-D"):
        maxsim.pack_unit_norm(x[None], lengths)


def test_sampling_refusals():
    s, u = torch.zeros(3, 10), torch.rand(3, 10)
    with pytest.raises(RuntimeError, match="CUDA"):
        maxsim.sample_candidates(s, u, 2)
    with pytest.raises(ValueError, match="2-D"):
        maxsim.sample_candidates(s[0], u[0], 2)
    with pytest.raises(TypeError, match="float32, float16, or bfloat16"):
        maxsim.sample_candidates(s.long(), u, 2)
    with pytest.raises(ValueError, match="scores' shape"):
        maxsim.sample_candidates(s, u[:, :9], 2)
    with pytest.raises(TypeError, match="uniforms must be float32"):
        maxsim.sample_candidates(s, u.double(), 2)
    for n in (-1, 11):
        with pytest.raises(ValueError, match="n must be"):
            maxsim.sample_candidates(s, u, n)
    with pytest.raises(ValueError, match="n must be"):
        maxsim.sample_candidates(torch.zeros(1, 2000), torch.zeros(1, 2000), 1025)
    with pytest.raises(ValueError, match="candidates per row"):
        maxsim.sample_candidates(torch.zeros(1, 2 ** 20 + 1), torch.zeros(1, 2 ** 20 + 1), 1)
    for name, bad in (("temperature", (0.0, -1.0, float("nan"))), ("top_k", (0, -2)),
                      ("top_p", (0.0, 1.5, float("nan"))), ("min_p", (-0.1, 1.5, float("nan")))):
        for v in bad:
            with pytest.raises(ValueError, match=name):
                maxsim.sample_candidates(s, u, 2, **{name: v})
        with pytest.raises(ValueError, match=name):
            maxsim.sample_candidates(s, u, 2, **{name: torch.ones(4)})
    with pytest.raises(TypeError, match="top_k must hold integers"):
        maxsim.sample_candidates(s, u, 2, top_k=torch.ones(3))
    with pytest.raises(TypeError, match="temperature must hold floats"):
        maxsim.sample_candidates(s, u, 2, temperature=torch.ones(3, dtype=torch.int32))
    with pytest.raises(TypeError):
        maxsim.sample_candidates(s, u, 2, top_k=2.5)
    with pytest.raises(TypeError):
        maxsim.sample_candidates(s, u, 2.5)


def test_c_entries_refuse_without_touching_a_device():
    """Status and message for calls no pointer of which is looked at."""
    lib = _ops.load_library()
    error = lambda: lib.maxsim_b200_last_error().decode()  # noqa: E731
    norm = lambda kind=0, n=1, L=4, dim=8, packed=4, eps=1e-5, dt=0, wdt=0, strides=(32, 8): (  # noqa: E731
        lib.maxsim_b200_norm_rows(kind, 0, *strides, 0, 0, 0, 0, 0, 0, n, L, dim, packed, eps, dt, wdt, 0))
    assert norm() == -1 and "null" in error()
    assert norm(kind=2) == -1 and "norm code" in error()
    assert norm(dim=0) == -1 and norm(n=-1) == -1 and norm(packed=-1) == -1 and norm(strides=(-1, 8)) == -1
    assert norm(eps=0.0) == -1 and norm(eps=float("nan")) == -1 and "eps" in error()
    assert norm(n=2 ** 20, L=2 ** 20) == -2 and "rows" in error()
    assert norm(n=2 ** 40, L=2 ** 40) == -2
    assert norm(n=0) == 0 and norm(L=0) == 0
    odd = lambda at, dt: lib.maxsim_b200_norm_rows(0, at, 32, 8, 0, 0, 0, 16, 0, 0, 1, 4, 8, 4, 1e-5, dt, dt, 0)  # noqa: E731
    assert odd(18, 0) == -1 and "element size" in error() and odd(17, 1) == -1
    assert norm(dt=0, wdt=1) == -2 and norm(dt=7) == -1 and "dtype" in error()
    pack = lambda off=8, dim=8, n=1: lib.maxsim_b200_pack_norm_rows(  # noqa: E731
        0, 16, 32, dim, 0, off, 0, 0, 16, 0, 0, n, 4, dim, 4, 1e-5, 0, 0, 0)
    assert pack(off=0) == -1 and pack() == -1 and "null" in error()  # no lengths
    assert pack(dim=0) == -1 and pack(n=2 ** 40) == -2
    assert lib.maxsim_b200_norm_rows_workspace(0, 4, 8) == 0
    back = lambda dw=0, ws=0, nbytes=0, kind=0: lib.maxsim_b200_norm_rows_backward(  # noqa: E731
        kind, 8, 8, 32, 8, 0, 0, 8, 8, 0, dw, 0, ws, nbytes, 1, 4, 8, 4, 1e-5, 0, 0, 0)
    assert back(dw=8) == -4 and "workspace" in error()
    assert back(dw=8, ws=8, nbytes=1) == -4
    assert back(kind=1, dw=8) == -1 and "no weights" in error()
    draw = lambda rows=1, cols=4, n=2, T=1.0, stride=4: lib.maxsim_b200_sample_rows(  # noqa: E731
        0, stride, 0, 4, rows, cols, n, T, 0, 0, 0, 1.0, 0, 0.0, 0, 0, 0, 0)
    assert draw() == -1 and "null" in error()
    assert draw(n=5) == -1 and draw(rows=-1) == -1 and draw(T=0.0) == -1 and draw(stride=-1) == -1
    assert draw(cols=2 ** 20 + 1) == -2 and draw(cols=2000, n=1025) == -2
    assert draw(rows=0) == 0 and draw(n=0) == 0


def test_workspace_has_a_row_for_every_cta():
    """The widest grid of a layer norm's backward kernel is six CTAs on each SM (fp32 rows of 385 to
    1024 elements that no 16-byte load divides); every CTA writes a row of sums for each of two gradients."""
    workspace = _ops.load_library().maxsim_b200_norm_rows_workspace
    sms = torch.cuda.get_device_properties(0).multi_processor_count if torch.cuda.is_available() else 148
    assert workspace(1, 10000, 770) >= 6 * sms * 770 * 2 * 4
    assert workspace(1, 600, 770) >= 600 * 770 * 2 * 4  # a CTA has a row at least
    assert workspace(15, 4000, 777) >= 6 * sms * 777 * 2 * 4


def test_forward_tangents_are_refused_not_lost(monkeypatch):
    """A tensor with a forward-mode tangent does not require a gradient; the operators have no forward
    derivative, and a result without a tangent would be one of zero."""
    from torch.autograd import forward_ad

    from maxsim_b200 import norms

    monkeypatch.setattr(_ops, "norm_rows", lambda kind, tokens, *rest: (tokens.clone(), None))
    x, w, b = torch.randn(3, 8), torch.ones(8), torch.zeros(8)
    lengths = torch.tensor([2, 1], dtype=torch.int32)
    offsets = torch.tensor([0, 2, 3], dtype=torch.int32)
    rows = lambda x, w, b: norms._apply(_ops.NORM_LAYER, x, w, b, None, 0, 1e-5)  # noqa: E731
    packed = lambda x, w, b: norms._apply(_ops.NORM_UNIT, x.view(1, 3, 8).expand(2, 3, 8), None, None, offsets, 3,  # noqa: E731
                                          1e-5, lengths)
    with forward_ad.dual_level():
        for i, t in enumerate((x, w, b)):
            dual = forward_ad.make_dual(t, torch.ones_like(t))
            args = [dual if j == i else other for j, other in enumerate((x, w, b))]
            for call in (rows, packed) if i == 0 else (rows,):
                with pytest.raises(NotImplementedError, match="jvp|forward"):
                    call(*args)
                with torch.no_grad(), pytest.raises(NotImplementedError, match="jvp|forward"):
                    call(*args)
                needs = [a if a is dual else a.clone().requires_grad_(True) for a in args]
                with pytest.raises(NotImplementedError, match="jvp|forward"):
                    call(*needs)
        assert forward_ad.unpack_dual(rows(x, w, b)).tangent is None  # none came in
    assert not rows(x, w, b).requires_grad


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("total", [None, 3])
def test_lengths_on_another_gpu_are_refused(dtype, total):
    """Offsets made there would be an address on the wrong device: refused before any kernel."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():  # tensors that have a device and no memory
        padded = torch.empty(3, 4, 8, device="cuda:0")
        lengths = torch.ones(3, dtype=dtype, device="cuda:1")
        for call in (maxsim.pack_layer_norm, maxsim.pack_unit_norm, maxsim.pack_padded):
            with pytest.raises(RuntimeError, match="padded's device cuda:0; got cuda:1"):
                call(padded, lengths, total_tokens=total)


def test_a_workspace_off_its_element_is_refused():
    lib = _ops.load_library()
    size = lib.maxsim_b200_norm_rows_workspace(1, 4, 8)
    for off in (1, 2, 3):
        rc = lib.maxsim_b200_norm_rows_backward(0, 8, 8, 32, 8, 0, 0, 8, 8, 0, 8, 0, 64 + off, size, 1, 4, 8, 4, 1e-5, 0, 0, 0)
        assert rc == -1 and "multiple of 4" in lib.maxsim_b200_last_error().decode()
