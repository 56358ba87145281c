"""Layer norm and unit rows on the GPU, plain and packed, forward and backward,
against the 64-bit oracle.

Tolerances.  u = 2^-24 is half a step of fp32, u_T that of the rows' type.  A
sum of D terms taken in any order is off by at most (D - 1) u times the sum of
their magnitudes; the kernels and anything else that is right take it in chains
far shorter than D, so K = D / 8 + 16 steps is what these tests grant a sum.
Every result is rounded once to its type: u_T of its size.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

import maxsim_b200 as maxsim
from maxsim_b200 import _ops
from oracle import maxsim_oracle as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
UT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}  # half a subnormal step, or flushed


def f64(t):
    return t.detach().cpu().double().numpy()


def steps(dim):
    return dim / 8 + 16


def close(got, want, dtype, slack, what):
    """|got - want| <= u_T |want| (1 + small) + slack; not finite where want is not."""
    got = f64(got)
    assert got.shape == want.shape, what
    fin = np.isfinite(want)
    assert np.array_equal(np.isfinite(got), fin), what
    err = np.abs(got - want)[fin]
    bound = (1.01 * UT[dtype] * np.abs(want) + slack + TINY[dtype])[fin]
    bad = err > bound
    assert not bad.any(), (what, int(bad.sum()), float((err - bound).max()), float(err.max()))


def layer_slack(x, w, eps=1e-5):
    """What fp32 arithmetic may add to a layer norm's rows: the mean is off by
    K u mean|x|, the variance and the products by K u of themselves."""
    d = x - x.mean(-1, keepdims=True)
    r = 1 / np.sqrt((d * d).mean(-1, keepdims=True) + eps)
    k = steps(x.shape[-1]) * U
    size = r * np.abs(x).mean(-1, keepdims=True) + np.abs(d * r) + 1
    return k * size * (1 if w is None else np.abs(w)), k * size


def check_layer(x, w, b, g, y, grads, eps=1e-5):
    """``x``, ``g`` the rows that count as tensors, ``grads`` (dx, dw, db) or None."""
    dt = x.dtype
    X, W, B = f64(x), None if w is None else f64(w), None if b is None else f64(b)
    slack, h_off = layer_slack(X, W, eps)
    close(y, oracle.layer_norm(X, W, B, eps), dt, slack + (0 if B is None else 4 * U * np.abs(B)), "rows")
    if grads is None:
        return
    G = f64(g)
    want, dw, db = oracle.layer_norm_backward(G, X, W, eps)
    u = G if W is None else G * W
    d = X - X.mean(-1, keepdims=True)
    r = 1 / np.sqrt((d * d).mean(-1, keepdims=True) + eps)
    h = np.abs(d * r)
    mean = lambda v: v.mean(-1, keepdims=True)  # noqa: E731
    k = steps(X.shape[-1]) * U
    # the two means by K u of their terms, h by h_off wherever it enters, the factor r by K u
    slack = r * (2 * k * (np.abs(u) + mean(np.abs(u)) + h * mean(np.abs(u) * h))
                 + h_off * mean(np.abs(u) * h) + h * mean(np.abs(u) * h_off))
    if grads[0] is not None:
        close(grads[0], want, dt, slack, "grad_tokens")
    rows = X.reshape(-1, X.shape[-1]).shape[0]
    sums = (rows / 8 + 64) * U
    flat = lambda v: np.broadcast_to(v, X.shape).reshape(-1, X.shape[-1])  # noqa: E731
    if grads[1] is not None:
        close(grads[1], dw, grads[1].dtype, (sums * np.abs(flat(G * h)) + np.abs(flat(G)) * flat(h_off)).sum(0), "grad_weight")
    if grads[2] is not None:
        close(grads[2], db, grads[2].dtype, sums * np.abs(flat(G)).sum(0), "grad_bias")


def check_unit(x, g, y, dx, eps=1e-12):
    dt, X = x.dtype, f64(x)
    k = steps(X.shape[-1]) * U
    want = oracle.unit_norm(X, eps)
    close(y, want, dt, k * np.abs(want), "rows")
    if dx is None:
        return
    G = f64(g)
    m = np.maximum(np.sqrt((X * X).sum(-1, keepdims=True)), eps)
    slack = 2 * k / m * (np.abs(G) + np.abs(want) * np.abs(want * G).sum(-1, keepdims=True))
    close(dx, oracle.unit_norm_backward(G, X, eps), dt, slack, "grad_tokens")


def rows_of(shape, dtype, seed, scale=1.0, shift=0.5):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=gen) * scale + shift).to(dtype).to(DEV)


# widths: one element, below / at / above every tile, odd ones, wide rows
WIDTHS = [1, 2, 7, 8, 31, 32, 40, 64, 96, 128, 129, 250, 256, 333, 512, 768, 1000, 1024, 1025, 1032, 1536, 2048, 4096,
          5000, 8192, 8200, 12345]
MIXES = [(torch.float32, torch.float32), (torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16),
         (torch.float16, torch.float32), (torch.bfloat16, torch.float32)]


@pytest.mark.parametrize("dim", WIDTHS)
@pytest.mark.parametrize("dtype,wtype", MIXES)
def test_layer_norm_and_gradients(dim, dtype, wtype):
    rows = 37 if dim < 4096 else 5
    x = rows_of((rows, dim), dtype, dim).requires_grad_(True)
    w = rows_of((dim,), wtype, dim + 1, 0.3, 1.0).requires_grad_(True)
    b = rows_of((dim,), wtype, dim + 2, 0.3, 0.0).requires_grad_(True)
    g = rows_of((rows, dim), dtype, dim + 3, 1.0, 0.1)
    y = maxsim.layer_norm(x, w, b)
    assert y.dtype == dtype and y.shape == x.shape
    grads = torch.autograd.grad(y, (x, w, b), g)
    assert [t.dtype for t in grads] == [dtype, wtype, wtype]
    check_layer(x, w, b, g, y, grads)


@pytest.mark.parametrize("dim", WIDTHS)
@pytest.mark.parametrize("dtype", list(UT))
def test_unit_norm_and_gradient(dim, dtype):
    rows = 41 if dim < 4096 else 5
    x = rows_of((rows, dim), dtype, dim).requires_grad_(True)
    g = rows_of((rows, dim), dtype, dim + 3, 1.0, 0.1)
    y = maxsim.unit_norm(x)
    (dx,) = torch.autograd.grad(y, x, g)
    check_unit(x, g, y, dx)


@pytest.mark.parametrize("rows", [1, 2, 31, 1000, 4097, 70001])
def test_row_counts(rows):
    x = rows_of((rows, 72), torch.bfloat16, rows).requires_grad_(True)
    w = rows_of((72,), torch.float32, 1, 0.3, 1.0).requires_grad_(True)
    b = rows_of((72,), torch.float32, 2).requires_grad_(True)
    g = rows_of((rows, 72), torch.bfloat16, 3)
    y = maxsim.layer_norm(x, w, b)
    check_layer(x, w, b, g, y, torch.autograd.grad(y, (x, w, b), g))
    y = maxsim.unit_norm(x)
    check_unit(x, g, y, torch.autograd.grad(y, x, g)[0])


@pytest.mark.parametrize("dim,dtype,wtype", [(768, torch.bfloat16, torch.float32), (128, torch.float16, torch.float16),
                                             (33, torch.float32, torch.float32), (1500, torch.bfloat16, torch.bfloat16),
                                             (96, torch.bfloat16, torch.bfloat16), (9000, torch.float16, torch.float32)])
@pytest.mark.parametrize("where", ["host", "device", "device_total"])
def test_packed_forms(dim, dtype, wtype, where):
    N, L = 23, 29
    lengths = torch.randint(1, L + 1, (N,), generator=torch.Generator().manual_seed(dim), dtype=torch.int32)
    lengths[0], lengths[1] = L, 1
    x = rows_of((N, L, dim), dtype, dim)
    valid = torch.arange(L)[None, :] < lengths[:, None]
    x[~valid.to(DEV)] = float("nan")  # padding is never read
    x.requires_grad_(True)
    w = rows_of((dim,), wtype, 1, 0.3, 1.0).requires_grad_(True)
    b = rows_of((dim,), wtype, 2).requires_grad_(True)
    T = int(lengths.sum())
    g = rows_of((T, dim), dtype, 3)
    ln = lengths if where == "host" else lengths.to(DEV)
    kw = {"total_tokens": T} if where == "device_total" else {}
    kept = x.detach()[valid.to(DEV)]
    want_offsets = np.concatenate([[0], np.cumsum(lengths.numpy())])

    y, off = maxsim.pack_layer_norm(x, ln, w, b, **kw)
    assert off.dtype == torch.int32 and off.cpu().tolist() == want_offsets.tolist()
    dx, dw, db = torch.autograd.grad(y, (x, w, b), g)
    assert dx.shape == x.shape and not dx[~valid.to(DEV)].any()
    check_layer(kept, w, b, g, y, (dx[valid.to(DEV)], dw, db))

    y, off = maxsim.pack_unit_norm(x, ln, **kw)
    assert off.cpu().tolist() == want_offsets.tolist()
    (dx,) = torch.autograd.grad(y, x, g)
    assert not dx[~valid.to(DEV)].any()
    check_unit(kept, g, y, dx[valid.to(DEV)])


def test_packed_form_equals_pack_then_norm_bit_for_bit():
    x = rows_of((17, 40, 256), torch.bfloat16, 5)
    lengths = torch.randint(1, 41, (17,), generator=torch.Generator().manual_seed(1))
    w = rows_of((256,), torch.float32, 1)
    packed, off = maxsim.pack_padded(x, lengths)
    y, off2 = maxsim.pack_layer_norm(x, lengths, w)
    assert torch.equal(off, off2) and torch.equal(y, maxsim.layer_norm(packed, w))
    y, _ = maxsim.pack_unit_norm(x, lengths)
    assert torch.equal(y, maxsim.unit_norm(packed))


@pytest.mark.parametrize("dim", [64, 100, 768, 1100])
def test_strided_and_unaligned_rows(dim):
    """Slices of a larger batch: skipped leading tokens, a narrower last
    dimension at an odd offset, transposed leading dimensions, expanded rows.
    (Not bit for bit the result on a contiguous copy: the width of the loads, and
    with it the order of a row's sum, follows the alignment.)"""
    base = rows_of((6, 12, dim + 24), torch.bfloat16, dim)
    w = rows_of((dim,), torch.bfloat16, 1)
    g = torch.Generator().manual_seed(0)
    lengths = torch.randint(1, 11, (6,), generator=g)
    for view in (base[:, 2:, 8:8 + dim], base[:, 2:, 3:3 + dim], base[1:, :10, 24:], base[..., :dim].transpose(0, 1)[:6, :],
                 base[:1, :10, :dim].expand(6, 10, dim), base[:, 1:11, :2 * (dim // 2):2]):
        wv = w[: view.shape[-1]]
        x = view.detach().requires_grad_(True)
        gy = rows_of(view.shape, torch.bfloat16, 2)
        y = maxsim.layer_norm(x, wv)
        dx, = torch.autograd.grad(y, x, gy)
        check_layer(view, wv, None, gy, y, (dx, None, None))
        ln = lengths[: view.shape[0]].clamp(max=view.shape[1])
        p, _ = maxsim.pack_unit_norm(view, ln)
        rows = view[(torch.arange(view.shape[1])[None, :] < ln[:, None]).to(DEV)]
        check_unit(rows, None, p, None)
    unaligned = rows_of((37 * dim + 1,), torch.bfloat16, 7)[1:].view(37, dim)
    check_layer(unaligned, w, None, None, maxsim.layer_norm(unaligned, w), None)
    w_off = rows_of((dim + 1,), torch.bfloat16, 8)[1:]
    check_layer(unaligned, w_off, w_off, None, maxsim.layer_norm(unaligned, w_off, w_off), None)
    many = rows_of((2, 3, 4, dim), torch.float32, 9)
    assert torch.equal(maxsim.unit_norm(many).view(24, dim), maxsim.unit_norm(many.view(24, dim)))
    one = rows_of((dim,), torch.float32, 10)
    assert torch.equal(maxsim.unit_norm(one), maxsim.unit_norm(one[None])[0])
    # gradients that arrive expanded (from a sum) or transposed
    x = rows_of((8, dim), torch.float32, 11).requires_grad_(True)
    (dx,) = torch.autograd.grad(maxsim.unit_norm(x).sum(), x)
    check_unit(x, torch.ones(8, dim), maxsim.unit_norm(x), dx)


def test_parts_of_the_gradient():
    x = rows_of((50, 200), torch.float16, 0)
    w = rows_of((200,), torch.float32, 1)
    b = rows_of((200,), torch.float32, 2)
    g = rows_of((50, 200), torch.float16, 3)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    full = torch.autograd.grad(maxsim.layer_norm(*leaves), leaves, g)
    for only in range(3):
        args = [t.clone().requires_grad_(i == only) for i, t in enumerate((x, w, b))]
        (got,) = torch.autograd.grad(maxsim.layer_norm(*args), args[only], g)
        assert torch.equal(got, full[only])
    # no bias, no weight, nothing to differentiate
    xa, wa = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    y = maxsim.layer_norm(xa, wa)
    check_layer(x, w, None, g, y, (*torch.autograd.grad(y, (xa, wa), g), None))
    y = maxsim.layer_norm(xa)
    check_layer(x, None, None, g, y, (torch.autograd.grad(y, xa, g)[0], None, None))
    assert not maxsim.layer_norm(x, w, b).requires_grad
    # the same tensor as weight and bias: its gradient is the sum of both
    y = maxsim.layer_norm(x, wa, wa)
    (dw,) = torch.autograd.grad(y, wa, g)
    torch.testing.assert_close(dw, full[1] + full[2], rtol=1e-6, atol=1e-6)
    with pytest.raises(RuntimeError, match="once_differentiable|does not require grad|twice"):
        first = torch.autograd.grad(maxsim.unit_norm(xa).sum(), xa, create_graph=True)[0]
        torch.autograd.grad(first.sum(), xa)


def test_gradient_against_differences():
    """Central differences of the kernel's own forward along a direction, summed in
    64 bits.  fp32 rows are off by about K u each; over sqrt(n) of them that is
    2e-5 / step, and the truncation of a step of 2^-6 is its square."""
    gen = torch.Generator().manual_seed(4)
    x, v, g = (torch.randn(64, 96, generator=gen).to(DEV) for _ in range(3))
    w, vw, b, vb = (torch.randn(96, generator=gen).to(DEV) for _ in range(4))
    h = 2.0 ** -6
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = maxsim.layer_norm(*leaves)
    dx, dw, db = torch.autograd.grad(y, leaves, g)
    along = float((dx.double() * v).sum() + (dw.double() * vw).sum() + (db.double() * vb).sum())
    at = lambda s: float((maxsim.layer_norm(x + s * v, w + s * vw, b + s * vb).double() * g).sum())  # noqa: E731
    size = float(g.double().norm() * y.double().norm())
    assert abs((at(h) - at(-h)) / (2 * h) - along) <= size * (h * h + 2e-5 / h)
    xa = x.clone().requires_grad_(True)
    (dx,) = torch.autograd.grad(maxsim.unit_norm(xa), xa, g)
    along = float((dx.double() * v).sum())
    at = lambda s: float((maxsim.unit_norm(x + s * v).double() * g).sum())  # noqa: E731
    size = float(g.double().norm() * 8)
    assert abs((at(h) - at(-h)) / (2 * h) - along) <= size * (h * h + 2e-5 / h)


@pytest.mark.parametrize("dtype", list(UT))
@pytest.mark.parametrize("dim", [24, 33, 768, 1300, 9000])
def test_extreme_rows(dim, dtype):
    """Zero rows, constant rows, rows at both ends of the type's range, and rows
    with an infinity or a NaN; a bad row changes no other."""
    lim = torch.finfo(dtype)
    x = rows_of((9, dim), dtype, dim, 1.0, 0.0)
    x[1] = 0
    x[2] = 3.0
    x[3] *= lim.max / 8
    x[4] *= lim.tiny * 4
    x[5, dim // 2] = float("inf")
    x[6, dim // 3] = float("nan")
    x[7] = lim.max
    g = rows_of((9, dim), dtype, 1, 1.0, 0.0)
    xa = x.clone().requires_grad_(True)
    with np.errstate(all="ignore"):
        y = maxsim.unit_norm(xa)
        (dx,) = torch.autograd.grad(y, xa, g)
        fine = [0, 1, 2, 3, 4, 7, 8]
        check_unit(x[fine], g[fine], y[fine], None)
        in_range = [0, 2, 8] if dtype != torch.float16 else [0, 2, 3, 7, 8]
        check_unit(x[in_range], g[in_range], y[in_range], dx[in_range])
        assert torch.isfinite(y[fine]).all() and y[1].eq(0).all()
        # |x| = inf: the infinite entry is inf / inf, the others 0
        assert torch.isnan(y[5, dim // 2]) and y[5].nan_to_num(0).eq(0).all()
        assert torch.isnan(y[6]).all()
        w = rows_of((dim,), torch.float32, 2)
        y = maxsim.layer_norm(x, w, w)
        check_layer(x[[0, 1, 2, 8]], w, w, None, y[[0, 1, 2, 8]], None)
        torch.testing.assert_close(y[1], w.to(dtype))  # a zero row: the bias
        assert torch.isnan(y[5]).all() and torch.isnan(y[6]).all()


def test_small_rows_are_scaled_by_eps():
    x = rows_of((5, 48), torch.float32, 0) * 1e-4
    g = rows_of((5, 48), torch.float32, 1)
    xa = x.clone().requires_grad_(True)
    y = maxsim.unit_norm(xa, eps=0.5)
    (dx,) = torch.autograd.grad(y, xa, g)
    check_unit(x, g, y, dx, eps=0.5)
    torch.testing.assert_close(dx, g * 2)
    y = maxsim.layer_norm(x, eps=1e-3)
    check_layer(x, None, None, None, y, None, eps=1e-3)


def test_large_offset_rows_keep_their_variance():
    """A mean a thousand times the spread: the variance is taken from the deviations."""
    x = rows_of((20, 640), torch.float32, 0, 1.0, 1000.0)
    check_layer(x, None, None, None, maxsim.layer_norm(x), None)


@pytest.mark.parametrize("dim", [4097, 4098, 4104, 6000, 20001])
@pytest.mark.parametrize("dtype,wtype", [(torch.bfloat16, torch.float32), (torch.float16, torch.float16),
                                         (torch.float32, torch.float32)])
@pytest.mark.parametrize("segments", [3, 160])
def test_rows_that_take_a_cta(dim, dtype, wtype, segments):
    """Wider than the rows that are kept on chip, few and many of them, packed, with a
    row of zeros and rows near both ends of the type's range."""
    L = 3
    lengths = torch.arange(segments, dtype=torch.int32, device=DEV) % L + 1
    x = rows_of((segments, L, dim), dtype, dim)
    x[0, 0] = 0
    x[1, 0] *= 2.0 ** 100 if dtype != torch.float16 else 2.0 ** 12
    x[2, 0] *= 2.0 ** -100 if dtype != torch.float16 else 2.0 ** -16
    x.requires_grad_(True)
    w = rows_of((dim,), wtype, 1, 0.3, 1.0).requires_grad_(True)
    b = rows_of((dim,), wtype, 2).requires_grad_(True)
    T = int(lengths.sum())
    g = rows_of((T, dim), dtype, 3)
    valid = torch.arange(L, device=DEV)[None, :] < lengths[:, None]
    plain = torch.ones(T, dtype=torch.bool, device=DEV)
    plain[lengths[:1].sum()] = plain[lengths[:2].sum()] = plain[0] = False  # the three rows above
    y, _ = maxsim.pack_unit_norm(x, lengths, total_tokens=T)
    (dx,) = torch.autograd.grad(y, x, g)
    assert not dx[~valid].any()
    kept = x.detach()[valid]
    check_unit(kept[plain], g[plain], y[plain], dx[valid][plain])
    check_unit(kept, g, y, None)
    with torch.no_grad():
        x[1, 0] = x[2, 0] = x[0, 1]
    kept = x.detach()[valid]
    y, _ = maxsim.pack_layer_norm(x, lengths, w, b, total_tokens=T)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), g)
    assert not dx[~valid].any()
    check_layer(kept, w, b, g, y, (dx[valid], dw, db))


def test_empty_batches():
    for shape in ((0, 16), (3, 0, 16), (0, 4, 16)):
        x = torch.empty(shape, device=DEV, requires_grad=True)
        w = torch.ones(16, device=DEV, requires_grad=True)
        y = maxsim.layer_norm(x, w, w)
        assert y.shape == x.shape
        dx, dw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
        assert dx.shape == x.shape and not dw.any()
        assert maxsim.unit_norm(x).shape == x.shape
    x = torch.empty(0, 4, 16, device=DEV)
    y, off = maxsim.pack_layer_norm(x, torch.empty(0, dtype=torch.int32))
    assert y.shape == (0, 16) and off.tolist() == [0]


def test_empty_segments_and_short_rows_in_much_padding():
    """Lengths on the device may be zero; one packed row among thousands of padded ones."""
    for lens, L in (([0, 3, 0, 0, 5, 0], 7), ([0, 0, 0], 4), ([1] + [0] * 40, 200), ([0] * 33 + [9], 9)):
        x = rows_of((len(lens), L, 64), torch.bfloat16, L).requires_grad_(True)
        w = rows_of((64,), torch.float32, 1).requires_grad_(True)
        T = sum(lens)
        ln = torch.tensor(lens, device=DEV)
        y, off = maxsim.pack_layer_norm(x, ln, w, w, total_tokens=T)
        assert off.tolist() == [0] + np.cumsum(lens).tolist() and y.shape == (T, 64)
        g = rows_of((T, 64), torch.bfloat16, 2)
        dx, dw = torch.autograd.grad(y, (x, w), g)
        valid = torch.arange(L, device=DEV)[None, :] < ln[:, None]
        assert not dx[~valid].any()
        if T:
            check_layer(x.detach()[valid], w, w, None, y, None)
            assert dx[valid].abs().sum() > 0 and dw.abs().sum() > 0
        else:
            assert not dw.any()
        y, _ = maxsim.pack_unit_norm(x, ln, total_tokens=T)
        (dx,) = torch.autograd.grad(y, x, g)
        assert not dx[~valid].any()
        if T:
            check_unit(x.detach()[valid], g, y, dx[valid])


@pytest.mark.parametrize("dim", [1, 3, 65, 333, 777])
@pytest.mark.parametrize("offset", [0, 1, 2, 3])
def test_odd_rows_at_every_offset(dim, offset):
    """16-bit rows of odd width that start on any element: neighbouring rows share 4-byte
    words, the first and the last row have words that reach past the tensor."""
    N, L = 5, 6
    base = rows_of((N * L * dim + 8,), torch.bfloat16, dim)
    base[:offset] = float("nan")           # what lies outside is not used
    base[offset + N * L * dim:] = float("nan")
    x = base[offset: offset + N * L * dim].view(N, L, dim).detach().requires_grad_(True)
    w = rows_of((dim,), torch.bfloat16, 1).requires_grad_(True)
    g = rows_of((N * L * dim + 1,), torch.bfloat16, 2)[1 - offset % 2:][: N * L * dim].view(N, L, dim)
    y = maxsim.layer_norm(x, w, w)
    dx, dw = torch.autograd.grad(y, (x, w), g)
    check_layer(x, w, w, g, y, (dx, None, None))
    assert torch.isfinite(dw).all()
    y = maxsim.unit_norm(x)
    check_unit(x, g, y, torch.autograd.grad(y, x, g)[0])
    ln = torch.tensor([6, 1, 3, 2, 6])
    valid = (torch.arange(L)[None, :] < ln[:, None]).to(DEV)
    y, _ = maxsim.pack_unit_norm(x, ln)
    gp = rows_of((18, dim), torch.bfloat16, 3)
    (dx,) = torch.autograd.grad(y, x, gp)
    check_unit(x.detach()[valid], gp, y, dx[valid])
    assert not dx[~valid].any()


def test_offsets_past_32_bits():
    """More than 2^31 elements: the rows at both ends and around element 2^31."""
    D, rows = 2048, 1_100_000
    x = torch.empty((rows, D), device=DEV, dtype=torch.bfloat16)
    x.normal_(generator=torch.Generator(device=DEV).manual_seed(0))
    x.requires_grad_(True)
    w = rows_of((D,), torch.float32, 1, 0.3, 1.0)
    g = torch.empty_like(x, requires_grad=False).normal_(generator=torch.Generator(device=DEV).manual_seed(1))
    some = torch.tensor([0, 1, 2 ** 20 - 1, 2 ** 20, 2 ** 20 + 1, rows - 2, rows - 1], device=DEV)
    y = maxsim.layer_norm(x, w)
    (dx,) = torch.autograd.grad(y, x, g)
    check_layer(x.detach()[some], w, None, g[some], y.detach()[some], (dx[some], None, None))
    del y, dx
    L = 11
    lens = torch.full((rows // L,), 10)
    y, off = maxsim.pack_unit_norm(x.view(rows // L, L, D), lens)
    check_unit(x.detach().view(-1, L, D)[-1, :10], None, y[-10:], None)
    assert int(off[-1]) == y.shape[0] == rows // L * 10


def test_gradients_under_create_graph_and_autocast():
    x = rows_of((6, 32), torch.float32, 0).requires_grad_(True)
    y = maxsim.unit_norm(x)
    (dx,) = torch.autograd.grad(y.sum() + (x ** 3).sum(), x, create_graph=True)  # allowed: only x ** 3 is used twice
    assert dx.shape == x.shape
    with torch.autocast("cuda", dtype=torch.bfloat16):
        w = torch.ones(32, device=DEV)
        assert maxsim.layer_norm(x.detach().bfloat16(), w).dtype == torch.bfloat16
        assert maxsim.layer_norm(x.detach(), w).dtype == torch.float32
    with torch.no_grad():
        assert not maxsim.layer_norm(x).requires_grad
    x2 = rows_of((6, 32), torch.float32, 0).requires_grad_(True)
    y = maxsim.unit_norm(x2 * 1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        z = x2 * 1
        y = maxsim.unit_norm(z)
        z.add_(1)
        y.sum().backward()


def test_packed_refusals():
    x = torch.zeros(4, 8, 16, device=DEV)
    with pytest.raises(ValueError, match="lengths must be in"):
        maxsim.pack_layer_norm(x, torch.tensor([1, 2, 9, 3]))
    with pytest.raises(ValueError, match="lengths must have shape"):
        maxsim.pack_layer_norm(x, torch.tensor([1, 2, 3]))
    with pytest.raises(TypeError, match="int32 or int64"):
        maxsim.pack_unit_norm(x, torch.ones(4))
    with pytest.raises(ValueError, match="total_tokens"):
        maxsim.pack_unit_norm(x, torch.tensor([1, 2, 3, 3]), total_tokens=8)
    with pytest.raises(RuntimeError, match="same device"):
        maxsim.layer_norm(x, torch.ones(16))


def test_a_short_total_drops_rows_and_writes_no_others():
    """A device total smaller than the lengths' sum: the rows behind it are
    dropped (as pack_padded does), their gradient is zero, nothing else is written."""
    x = rows_of((3, 4, 32), torch.float32, 0).requires_grad_(True)
    w = rows_of((32,), torch.float32, 1).requires_grad_(True)
    y, off = maxsim.pack_layer_norm(x, torch.tensor([4, 3, 4], device=DEV), w, total_tokens=9)
    assert y.shape == (9, 32) and off.tolist() == [0, 4, 7, 11]
    g = rows_of((9, 32), torch.float32, 2)
    dx, dw = torch.autograd.grad(y, (x, w), g)
    kept = torch.cat([x.detach()[0], x.detach()[1, :3], x.detach()[2, :2]])
    assert not dx[1, 3].any() and not dx[2, 2:].any()
    check_layer(kept, w, None, g, y, (torch.cat([dx[0], dx[1, :3], dx[2, :2]]), dw, None))


@pytest.mark.parametrize("lens,total", [([3, 0, 7, 5], 15), ([9, -2, 3, 1], 11), ([1, 2, 3, 4], 12), ([7] * 4, 20),
                                        ([0, 0, 0, 0], 0), ([], 0)])
def test_both_ways_of_writing_the_offsets(lens, total):
    """int32 lengths on the device with a total take one call of the library, int64
    ones two: lengths outside [0, L_max] and totals off the sum give the same."""
    L = 7
    x = rows_of((len(lens), L, 40), torch.float16, 0).requires_grad_(True)
    w = rows_of((40,), torch.float32, 1).requires_grad_(True)
    g = rows_of((total, 40), torch.float16, 2)
    used = min(total, sum(min(max(n, 0), L) for n in lens))
    got = []
    for dtype in (torch.int32, torch.int64):
        y, off = maxsim.pack_layer_norm(x, torch.tensor(lens, dtype=dtype, device=DEV), w, w, total_tokens=total)
        assert y.shape == (total, 40)
        dx, dw = torch.autograd.grad(y, (x, w), g)
        u, off_u = maxsim.pack_unit_norm(x.detach(), torch.tensor(lens, dtype=dtype, device=DEV), total_tokens=total)
        got.append((y.detach()[:used], off, dx, dw, u[:used], off_u))
    for a, b in zip(*got):
        assert torch.equal(a, b)
    valid = torch.arange(L)[None, :] < torch.tensor(lens, dtype=torch.int64).reshape(-1, 1)
    kept = x.detach()[valid.to(DEV)][:used]
    if used:
        check_layer(kept, w, w, None, got[0][0], None)


@pytest.mark.parametrize("dim,dtype", [(768, torch.bfloat16), (333, torch.float32), (5000, torch.float16)])
def test_equal_calls_give_equal_bits(dim, dtype):
    x = rows_of((3000, dim), dtype, 0).requires_grad_(True)
    w = rows_of((dim,), torch.float32, 1).requires_grad_(True)
    g = rows_of((3000, dim), dtype, 2)
    runs = []
    for _ in range(3):
        y = maxsim.layer_norm(x, w, w)
        runs.append((y.detach(), *torch.autograd.grad(y, (x, w), g)))
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


def test_two_streams_at_once():
    """Calls on two streams share nothing: results as on one."""
    xs = [rows_of((4000, 512), torch.bfloat16, i).requires_grad_(True) for i in range(2)]
    w = rows_of((512,), torch.float32, 9).requires_grad_(True)
    g = rows_of((4000, 512), torch.bfloat16, 10)

    def call(x):
        y = maxsim.layer_norm(x, w, w)
        return (y.detach(), *torch.autograd.grad(y, (x, w), g))

    want = [call(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, (x, st) in enumerate(zip(xs, streams)):
            with torch.cuda.stream(st):
                got[i].append(call(x))
    torch.cuda.synchronize()
    for i in range(2):
        for run in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(run, want[i]))


def test_training_pass_replays_from_a_graph():
    N, L, D = 8, 20, 256
    x = rows_of((N, L, D), torch.bfloat16, 0).requires_grad_(True)
    w = rows_of((D,), torch.float32, 1).requires_grad_(True)
    lengths = torch.full((N,), 10, dtype=torch.int32, device=DEV)
    g = rows_of((N * 10, D), torch.bfloat16, 2)

    def step():
        y, off = maxsim.pack_layer_norm(x, lengths, w, w, total_tokens=N * 10)
        return (y.detach(), off, *torch.autograd.grad(y, (x, w), g))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(stream)
    graphs = []
    for _ in range(2):  # two graphs over the same leaves, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    with torch.no_grad():
        x.copy_(rows_of((N, L, D), torch.bfloat16, 3))
        lengths.copy_(torch.tensor([1, 19, 20, 5, 15, 2, 17, 1], dtype=torch.int32))  # the same total
    for graph, _ in graphs + graphs:
        graph.replay()
    torch.cuda.synchronize()
    want = step()
    for _, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_the_steps_together():
    """Encoder rows -> layer norm, packed -> projection -> unit rows -> contrastive
    loss, and back: the gradients against the same chain in torch's own
    operators in fp32."""
    torch.manual_seed(0)
    N, L, H, D, Lq = 6, 30, 192, 64, 16
    enc = torch.randn(N, L, H, device=DEV)
    qe = torch.randn(N, Lq, H, device=DEV)
    lengths = torch.tensor([30, 4, 17, 1, 22, 9])
    w = (1 + 0.1 * torch.randn(H, device=DEV))
    b = 0.1 * torch.randn(H, device=DEV)
    proj = torch.randn(D, H, device=DEV) / H ** 0.5

    def run(kernels):
        leaves = [t.clone().requires_grad_(True) for t in (enc, qe, w, b, proj)]
        e, q, ww, bb, pp = leaves
        if kernels:
            rows, off = maxsim.pack_layer_norm(e, lengths, ww, bb)
            docs = maxsim.unit_norm(rows @ pp.T)
            queries = maxsim.unit_norm(maxsim.layer_norm(q, ww, bb) @ pp.T)
            loss = maxsim.contrastive_loss(queries, docs, off, temperature=0.5)
        else:
            norm = lambda t: torch.nn.functional.layer_norm(t, (H,), ww, bb)  # noqa: E731
            unit = lambda t: torch.nn.functional.normalize(t, dim=-1)  # noqa: E731
            docs, queries = unit(norm(e) @ pp.T), unit(norm(q) @ pp.T)
            sim = torch.einsum("qid,njd->qnij", queries, docs)
            mask = torch.arange(L)[None, :] >= lengths[:, None]
            s = sim.masked_fill(mask.to(DEV)[None, :, None, :], float("-inf")).amax(-1).sum(-1)
            loss = torch.nn.functional.cross_entropy(s / 0.5, torch.arange(N, device=DEV))
        return [loss.detach(), *torch.autograd.grad(loss, leaves)]

    for name, a, want in zip(("loss", "encoder", "queries", "weight", "bias", "projection"), run(True), run(False)):
        # both sides fp32: matrix products of 192 terms, K u of the largest entry
        torch.testing.assert_close(a, want, rtol=1e-4, atol=2e-5 * float(want.abs().max()) + 1e-7, msg=lambda m: name + m)
    assert _ops.device_status() == 0


def backward_beside_guards(x, w, g, offsets=None, guard=4 << 20):
    """The C backward pass with a workspace of exactly the stated size between two guards:
    ``(dx, dw, db)`` of ``x [N, L, dim]``, and whether the guards are untouched."""
    lib, (N, L, dim) = _ops.load_library(), x.shape
    rows = g.shape[0]
    call = (L * dim, dim, N, L, dim, rows)
    _, stats = _ops.norm_rows(_ops.NORM_LAYER, x, call, offsets, w, w, 1e-5, (rows, dim), True)
    size = lib.maxsim_b200_norm_rows_workspace(N, L, dim)
    memory = torch.full((2 * guard + size,), 0xA5, dtype=torch.uint8, device=DEV)
    dx, dw, db = torch.empty_like(x), torch.empty(dim, dtype=w.dtype, device=DEV), torch.empty(dim, dtype=w.dtype, device=DEV)
    rc = lib.maxsim_b200_norm_rows_backward(
        _ops.NORM_LAYER, g.data_ptr(), x.data_ptr(), L * dim, dim, 0 if offsets is None else offsets.data_ptr(),
        w.data_ptr(), stats[0].data_ptr(), stats[1].data_ptr(), dx.data_ptr(), dw.data_ptr(), db.data_ptr(),
        memory.data_ptr() + guard, size, N, L, dim, rows, 1e-5, _ops._code(x), _ops._code(w),
        torch.cuda.current_stream().cuda_stream)
    assert rc == 0, lib.maxsim_b200_last_error()
    untouched = bool((memory[:guard] == 0xA5).all()) and bool((memory[guard + size:] == 0xA5).all())
    return dx, dw, db, untouched


def weights_of(dim, wtype, off):
    return rows_of((dim + off,), wtype, 1, 0.3, 1.0)[off:]


@pytest.mark.parametrize("dim,off", [(385, 0), (390, 0), (513, 0), (770, 0), (777, 0), (1023, 0), (768, 1)])
@pytest.mark.parametrize("rows", [593, 888, 1185, 3000, 10000])
def test_weight_gradients_stay_in_their_workspace(dim, off, rows):
    """fp32 rows that no wide load divides, by their width or because the weight starts off 16
    bytes, with more rows than the SMs hold CTAs."""
    w = weights_of(dim, torch.float32, off)
    x = rows_of((1, rows, dim), torch.float32, dim)
    g = rows_of((rows, dim), torch.float32, 3)
    dx, dw, db, untouched = backward_beside_guards(x, w, g)
    assert untouched
    check_layer(x[0], w, None, g, maxsim.layer_norm(x[0], w), (dx[0], dw, db))


@pytest.mark.parametrize("dim,off", [(385, 0), (390, 0), (513, 0), (770, 0), (777, 0), (1023, 0), (768, 1)])
def test_weight_gradients_stay_in_their_workspace_in_much_padding(dim, off):
    """Few packed rows among 60000: the grid is widened for the zeros of the padding to as
    many CTAs as the SMs hold, each with a row of partial sums."""
    N, L = 15, 4000
    w = weights_of(dim, torch.float32, off)
    lengths = torch.arange(1, N + 1)
    valid = (torch.arange(L)[None, :] < lengths[:, None]).to(DEV)
    T = int(lengths.sum())
    x = torch.full((N, L, dim), float("nan"), device=DEV)
    kept = x[valid] = rows_of((T, dim), torch.float32, dim)
    g = rows_of((T, dim), torch.float32, 3)
    offsets = torch.cat([torch.zeros(1), lengths.cumsum(0)]).to(torch.int32).to(DEV)
    dx, dw, db, untouched = backward_beside_guards(x, w, g, offsets)
    assert untouched and not dx[~valid].any()
    check_layer(kept, w, None, g, maxsim.layer_norm(kept, w), (dx[valid], dw, db))


# a width for every team of threads and number of packs, for each width of a load
PER_TEAM = {
    torch.float32: [(32, 0), (64, 0), (128, 0), (256, 0), (512, 0), (764, 0), (1020, 0), (2044, 0), (4092, 0), (4100, 0),
                    (31, 0), (62, 0), (95, 0), (126, 0), (255, 0), (382, 0), (1022, 0), (1025, 0), (4095, 0), (4097, 0),
                    (128, 1), (1024, 1), (4096, 3)],
    torch.bfloat16: [(64, 0), (128, 0), (256, 0), (512, 0), (760, 0), (1016, 0), (2040, 0), (4088, 0), (4104, 0),
                     (30, 0), (62, 0), (126, 0), (254, 0), (382, 0), (1022, 0), (1534, 0), (4094, 0), (4098, 0),
                     (31, 0), (63, 0), (95, 0), (127, 0), (255, 0), (383, 0), (1023, 0), (1025, 0), (4095, 0), (4097, 0),
                     (768, 1), (768, 2), (2048, 1)],
}


@pytest.mark.parametrize("dtype,dim,off", [(t, *c) for t, cases in PER_TEAM.items() for c in cases])
def test_every_team_on_a_full_gpu(dtype, dim, off):
    """More rows than any kernel has CTAs at once (six an SM), so that CTAs and teams take several each:
    every gradient against the oracle, weights that start off the loads' width too."""
    rows = 1201
    w = weights_of(dim, dtype, off)
    x = rows_of((1, rows, dim), dtype, dim)
    g = rows_of((rows, dim), dtype, 3)
    dx, dw, db, untouched = backward_beside_guards(x, w, g)
    assert untouched
    check_layer(x[0], w, None, g, maxsim.layer_norm(x[0], w), (dx[0], dw, db))


def test_a_workspace_that_is_too_small_is_refused():
    x = rows_of((2000, 770), torch.float32, 0)
    lib = _ops.load_library()
    size = lib.maxsim_b200_norm_rows_workspace(1, 2000, 770)
    assert size >= 6 * torch.cuda.get_device_properties(0).multi_processor_count * 770 * 8
    args = lambda nbytes: (_ops.NORM_LAYER, x.data_ptr(), x.data_ptr(), 0, 770, 0, x.data_ptr(), x.data_ptr(),  # noqa: E731
                           x.data_ptr(), 0, x.data_ptr(), 0, x.data_ptr(), nbytes, 1, 2000, 770, 2000, 1e-5, 0, 0, 0)
    assert lib.maxsim_b200_norm_rows_backward(*args(size - 1)) == -4
    assert "workspace" in lib.maxsim_b200_last_error().decode()


@pytest.mark.parametrize("dtype,dim,off", [(t, *c) for t, cases in PER_TEAM.items() for c in cases])
def test_every_team_on_a_full_gpu_packed(dtype, dim, off):
    """The same out of a padded batch with empty segments, padding that is NaN, and a gradient for
    every padded row."""
    N, L = 301, 8
    lengths = torch.randint(0, L + 1, (N,), generator=torch.Generator().manual_seed(dim + off))
    valid = (torch.arange(L)[None, :] < lengths[:, None]).to(DEV)
    T = int(lengths.sum())
    w = weights_of(dim, dtype, off)
    x = torch.full((N, L, dim), float("nan"), device=DEV, dtype=dtype)
    kept = x[valid] = rows_of((T, dim), dtype, dim)
    g = rows_of((T, dim), dtype, 3)
    offsets = torch.cat([torch.zeros(1), lengths.cumsum(0)]).to(torch.int32).to(DEV)
    dx, dw, db, untouched = backward_beside_guards(x, w, g, offsets)
    assert untouched and not dx[~valid].any()
    y, _ = maxsim.pack_layer_norm(x, lengths.to(DEV), w, total_tokens=T)
    check_layer(kept, w, None, g, y, (dx[valid], dw, db))
    xa = x.requires_grad_(True)
    y, _ = maxsim.pack_unit_norm(xa, lengths.to(DEV), total_tokens=T)
    (dx,) = torch.autograd.grad(y, xa, g)
    assert not dx[~valid].any()
    check_unit(kept, g, y, dx[valid])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [1, 3, 65, 333, 777, 1025])
@pytest.mark.parametrize("offset", [0, 1, 2, 3])
def test_weight_gradients_of_odd_rows_at_every_offset(dtype, dim, offset):
    """16-bit rows of odd width whose first and last words reach past the tensor, into NaN: all three
    gradients, rows as they lie and packed."""
    N, L = 5, 6
    base = rows_of((N * L * dim + 8,), dtype, dim)
    base[:offset] = float("nan")
    base[offset + N * L * dim:] = float("nan")
    x = base[offset: offset + N * L * dim].view(N, L, dim).detach().requires_grad_(True)
    w = rows_of((dim,), dtype, 1, 0.3, 1.0).requires_grad_(True)
    b = rows_of((dim,), dtype, 2, 0.3, 0.0).requires_grad_(True)
    outer = rows_of((N * L * dim + 8,), dtype, 3)
    outer[: 1 - offset % 2] = float("nan")
    outer[1 - offset % 2 + N * L * dim:] = float("nan")
    g = outer[1 - offset % 2:][: N * L * dim].view(N, L, dim)
    y = maxsim.layer_norm(x, w, b)
    check_layer(x, w, b, g, y, torch.autograd.grad(y, (x, w, b), g))
    lengths = torch.tensor([6, 1, 3, 2, 6])
    valid = (torch.arange(L)[None, :] < lengths[:, None]).to(DEV)
    gp = rows_of((18, dim), dtype, 4)
    y, _ = maxsim.pack_layer_norm(x, lengths, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), gp)
    assert not dx[~valid].any()
    check_layer(x.detach()[valid], w, b, gp, y, (dx[valid], dw, db))


@pytest.mark.parametrize("dim,dtype", [(64, torch.bfloat16), (33, torch.float16), (770, torch.float32), (4100, torch.float32)])
@pytest.mark.parametrize("lens,L", [([0, 3, 0, 0, 5, 0], 7), ([1] + [0] * 40, 200), ([0] * 33 + [9], 9), ([0, 0, 0], 4)])
def test_gradients_of_empty_segments_and_much_padding(dim, dtype, lens, L):
    x = rows_of((len(lens), L, dim), dtype, L).requires_grad_(True)
    w = rows_of((dim,), torch.float32, 1, 0.3, 1.0).requires_grad_(True)
    b = rows_of((dim,), torch.float32, 2, 0.3, 0.0).requires_grad_(True)
    T, ln = sum(lens), torch.tensor(lens, device=DEV)
    valid = torch.arange(L, device=DEV)[None, :] < ln[:, None]
    g = rows_of((T, dim), dtype, 3)
    y, _ = maxsim.pack_layer_norm(x, ln, w, b, total_tokens=T)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), g)
    assert not dx[~valid].any()
    if T:
        check_layer(x.detach()[valid], w, b, g, y, (dx[valid], dw, db))
    else:
        assert not dw.any() and not db.any()


def test_rows_past_the_fp32_variance():
    """Deviations whose squares overflow: the bias and a gradient of zero, as documented, and no other row changes."""
    for dim in (64, 333, 768, 1500, 5000):
        x = rows_of((5, dim), torch.float32, dim)
        w, b = rows_of((dim,), torch.float32, 1, 0.3, 1.0), rows_of((dim,), torch.float32, 2)
        g = rows_of((5, dim), torch.float32, 3)
        want = maxsim.layer_norm(x, w, b)
        x[2] = rows_of((dim,), torch.float32, 4, 1e20, 0.0)
        x.requires_grad_(True)
        y = maxsim.layer_norm(x, w, b)
        (dx,) = torch.autograd.grad(y, x, g)
        others = [0, 1, 3, 4]
        assert torch.equal(y[2], b) and not dx[2].any() and torch.equal(y[others], want[others])
        check_layer(x.detach()[others], w, b, g[others], y[others], (dx[others], None, None))


def test_forward_tangents_are_refused():
    from torch.autograd import forward_ad

    x, w = rows_of((6, 32), torch.float32, 0), rows_of((32,), torch.float32, 1)
    with forward_ad.dual_level():
        dual, dual_w = forward_ad.make_dual(x, torch.ones_like(x)), forward_ad.make_dual(w, torch.ones_like(w))
        for call in (lambda: maxsim.unit_norm(dual), lambda: maxsim.layer_norm(dual), lambda: maxsim.layer_norm(x, dual_w),
                     lambda: maxsim.pack_unit_norm(dual.view(2, 3, 32), torch.tensor([1, 3]))):
            with pytest.raises(NotImplementedError):
                call()
        assert torch.equal(maxsim.layer_norm(x, w), maxsim.layer_norm(x.clone(), w))
