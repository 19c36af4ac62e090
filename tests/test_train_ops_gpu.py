"""Dropout, LayerNorm and their fusion on the GPU against 64-bit arithmetic, forward and backward.

Tolerances are bounds, not measurements.  u is half a step of fp32 (2^-24) and half a step of the output type is added relative to the
value.  A sum of n terms in some order is off by at most (longest chain of additions) * u * sum of magnitudes: 32 columns a thread, five
exchanges in a warp and sixteen warps, 53 in all, taken as CHAIN = 64 with the products' own roundings.
"""
import numpy as np
import pytest
import torch

from oracle import train_oracle as orc
from turbodeberta_b200.ops.dropout import dropout
from turbodeberta_b200.ops.layer_norm import dropout_add_layer_norm, layer_norm

pytestmark = pytest.mark.gpu
F, B = torch.float32, torch.bfloat16
U, CHAIN = 2.0 ** -24, 64
HALF = {F: 2.0 ** -24, B: 2.0 ** -8}
TINY = 1e-37                                         # results below the normal numbers


def f64(t):
    return t.detach().double().cpu().numpy()


def near(got, want, tol, what):
    got = f64(got)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = np.abs(got - want) - tol
    assert np.isfinite(got).all() and off.max(initial=-1) <= 0, f"{what}: beyond the bound by {off.max():.3e} (bound there {np.broadcast_to(tol, off.shape).flat[off.argmax()]:.3e})"


def rounding(want, dtype):
    return np.abs(want) * HALF[dtype] + TINY


# ------------------------------------------------------------------------------------------------------------------ dropout
@pytest.mark.parametrize("dtype", [F, B])
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (3, 5), (33, 1000), (2, 3, 257), (1000, 4099)])
@pytest.mark.parametrize("p,offset", [(0.1, 0), (0.5, (1 << 40) + 3)])
def test_dropout_and_its_gradient(dtype, shape, p, offset):
    g = torch.Generator("cuda").manual_seed(1)
    x = torch.randn(shape, device="cuda", generator=g).to(dtype).requires_grad_()
    dy = torch.randn(shape, device="cuda", generator=g).to(dtype)
    y = dropout(x, p, -12345678901234567, offset)
    dx, = torch.autograd.grad(y, x, dy)
    want, keep, scale = orc.dropout(f64(x), p, -12345678901234567, offset)
    assert np.array_equal(f64(y) != 0, keep & (f64(x) != 0))
    near(y, want, rounding(want, dtype) + 2 * U * np.abs(want), "y")
    want = np.where(keep, f64(dy), 0) * scale
    near(dx, want, rounding(want, dtype) + 2 * U * np.abs(want), "dx")


def test_dropout_share_and_extremes():
    x = torch.ones(1 << 22, device="cuda")
    for p in (0.1, 0.25, 0.9):
        y = dropout(x, p, 3)
        n = x.numel()
        assert abs((y == 0).sum().item() - p * n) < 6 * (p * (1 - p) * n) ** 0.5 + n / 65536
        assert abs(y.double().mean().item() - 1) < 6 * (p / (1 - p) / n) ** 0.5
    assert torch.equal(dropout(x, 0.0, 3), x)
    assert not dropout(x, 1.0, 3).any()
    a, b, c = dropout(x, 0.5, 3), dropout(x, 0.5, 4), dropout(x, 0.5, 3, 1)
    assert torch.equal(a, dropout(x, 0.5, 3)) and not torch.equal(a, b) and not torch.equal(a, c)


@pytest.mark.parametrize("dtype", [F, B])
def test_dropped_elements_may_hold_anything(dtype):
    keep = torch.from_numpy(orc.stays((40, 64), 0.5, 9, 2)).cuda()
    x = torch.full((40, 64), float("nan"), device="cuda", dtype=dtype)
    x[::2] = float("inf")
    x = torch.where(keep, torch.ones_like(x), x).requires_grad_()
    y = dropout(x, 0.5, 9, 2)
    assert torch.equal(y, keep.to(dtype) * 2)
    w, b = torch.ones(64, device="cuda", dtype=dtype), torch.zeros(64, device="cuda", dtype=dtype)
    z = dropout_add_layer_norm(x, torch.zeros_like(x), w, b, 1e-7, 0.5, 9, 2)
    dx, = torch.autograd.grad(z, x, torch.randn_like(z))
    assert torch.isfinite(z).all() and torch.isfinite(dx).all() and not dx[~keep].any()


def test_dropout_takes_any_layout():
    base = torch.randn(70, 130, device="cuda")
    for x in (base.t(), base[:, 1:], base[::2, 3:100], base[:1].expand(9, 130), base.reshape(-1)[1:]):
        want, _, _ = orc.dropout(f64(x), 0.3, 5)
        near(dropout(x, 0.3, 5), want, rounding(want, F) + 2 * U * np.abs(want), "y")
    assert dropout(base[:0], 0.3, 5).shape == (0, 130)


def test_seed_tensor_is_read_by_the_kernel_and_by_graph_replays():
    x = torch.randn(64, 256, device="cuda", requires_grad=True)
    seed = torch.tensor([77], device="cuda")
    assert torch.equal(dropout(x, 0.2, seed), dropout(x, 0.2, 77))
    dy = torch.randn_like(x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.autograd.grad(dropout(x, 0.2, seed), x, dy)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = dropout(x, 0.2, seed)
        dx, = torch.autograd.grad(y, x, dy)
    for value in (1, 2):
        seed.fill_(value)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, dropout(x, 0.2, value)) and torch.equal(dx, dropout(dy, 0.2, value))


def test_a_seed_changed_before_the_backward_pass_is_reported():
    x = torch.randn(64, device="cuda", requires_grad=True)
    seed = torch.tensor([77], device="cuda")
    y = dropout(x, 0.2, seed)
    seed.fill_(3)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


# ---------------------------------------------------------------------------------------------------------------- LayerNorm
def norm_case(rows, cols, dtype, wt, join, seed=0, mean=0.0):
    g = torch.Generator("cuda").manual_seed(seed)
    r = lambda *s, m=0.0, k=1.0, t=dtype: (torch.randn(*s, device="cuda", generator=g) * k + m).to(t)  # noqa: E731
    x, dy = r(rows, cols, m=mean), r(rows, cols)
    w, b = r(cols, m=1.0, k=0.3, t=wt), r(cols, k=0.3, t=wt)
    return x, (r(rows, cols) if join else None), w, b, dy


def bounds(z, parts, w, b, eps, dy):
    """Bounds for y, dz, dw, db without the final rounding; `parts`: the magnitudes that were added to make z."""
    d = z - z.mean(-1, keepdims=True)
    inv = 1 / np.sqrt((d * d).mean(-1, keepdims=True) + eps)
    h = d * inv
    ez = 3 * U * parts
    ed = ez + (CHAIN * U) * np.abs(z).mean(-1, keepdims=True) + ez.mean(-1, keepdims=True) + U * np.abs(d)
    # relative error of the variance: twice that of d in the mean, weighted by d, and the sum's own
    ev = (2 * (np.abs(d) * ed).mean(-1, keepdims=True) + (ed * ed).mean(-1, keepdims=True)) * inv ** 2 + CHAIN * U
    eh = ed * inv + np.abs(h) * (ev + 4 * U)
    ey = eh * np.abs(w) + 2 * U * (np.abs(h * w) + np.abs(b))
    g = dy * w
    eg = U * np.abs(g)
    c1, c2 = np.abs(g).mean(-1, keepdims=True), np.abs(g * h).mean(-1, keepdims=True)
    e1, e2 = CHAIN * U * c1, CHAIN * U * c2 + (np.abs(g) * eh).mean(-1, keepdims=True)
    inner = np.abs(g) + c1 + np.abs(h) * c2
    edz = inv * (eg + e1 + np.abs(h) * e2 + eh * (c2 + e2) + 3 * U * inner + inner * (ev + 4 * U))
    rows = z.reshape(-1, z.shape[-1]).shape[0]
    edw = (np.abs(dy) * eh).sum(0) + (rows + CHAIN) * U * np.abs(dy * h).sum(0)
    edb = (rows + CHAIN) * U * np.abs(dy).sum(0)
    return ey, edz, edw, edb


SHAPES = [(1, 1), (1, 8), (3, 16), (2, 7), (5, 257), (48, 768), (33, 1000), (700, 264), (1300, 1024), (9, 1032), (4, 4096), (3, 4100), (6, 8192), (2, 16384), (2, 16383)]


@pytest.mark.parametrize("dtype,wt", [(F, F), (B, B), (B, F)])
@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("form", ["alone", "join", "drop"])
def test_norm_and_its_gradients(rows, cols, dtype, wt, form):
    eps, p = 1e-5, 0.3 if form == "drop" else 0.0
    x, res, w, b, dy = norm_case(rows, cols, dtype, wt, form != "alone", seed=rows + cols)
    leaves = [t.requires_grad_() for t in (x, res, w, b) if t is not None]
    y = layer_norm(x, w, b, eps) if form == "alone" else dropout_add_layer_norm(x, res, w, b, eps, p, 11, 4)
    grads = dict(zip(["x"] + (["res"] if res is not None else []) + ["w", "b"], torch.autograd.grad(y, leaves, dy)))
    xs, keep, scale = orc.dropout(f64(x), p, 11, 4)
    z = xs if res is None else xs + f64(res)
    parts = np.abs(xs) + (0 if res is None else np.abs(f64(res)))
    ey, edz, edw, edb = bounds(z, parts, f64(w), f64(b), eps, f64(dy))
    want = orc.layer_norm(z, f64(w), f64(b), eps)
    near(y, want, ey + (np.abs(want) + ey) * HALF[dtype] + TINY, "y")
    dz, dw, db = orc.layer_norm_backward(z, f64(w), eps, f64(dy))
    last = (np.abs(dz) + edz) * HALF[dtype] + TINY
    near(grads["x"], np.where(keep, dz, 0) * scale, (edz + last) * scale * (1 + 4 * U) if p else edz + last, "dx")
    if res is not None:
        near(grads["res"], dz, edz + last, "dres")
    near(grads["w"], dw, edw + (np.abs(dw) + edw) * HALF[wt] + TINY, "dw")
    near(grads["b"], db, edb + (np.abs(db) + edb) * HALF[wt] + TINY, "db")


@pytest.mark.parametrize("dtype", [F, B])
def test_gradients_against_differences(dtype):
    """The kernels' gradients along a direction, against differences of the 64-bit function."""
    rows, cols, eps, p = 37, 136, 1e-5, 0.25
    x, res, w, b, dy = norm_case(rows, cols, dtype, dtype, True)
    leaves = [t.requires_grad_() for t in (x, res, w, b)]
    grads = torch.autograd.grad(dropout_add_layer_norm(*leaves, eps, p, 5, 6), leaves, dy)
    r = np.random.RandomState(3)

    def value(x, res, w, b):
        return (orc.layer_norm(orc.dropout(x, p, 5, 6)[0] + res, w, b, eps) * f64(dy)).sum()

    at = [f64(t) for t in leaves]
    for i, g in enumerate(grads):
        v = r.randn(*at[i].shape)
        up, down = list(at), list(at)
        up[i], down[i] = at[i] + 1e-5 * v, at[i] - 1e-5 * v
        diff = (value(*up) - value(*down)) / 2e-5
        # roundings of the elements, each at most half a step, in any direction; 1e-6 for the differences' own error
        bound = (np.abs(f64(g) * v)).sum() * (HALF[dtype] + 2000 * U) + 1e-6 * np.abs(f64(g) * v).sum() + 1e-6
        assert abs((f64(g) * v).sum() - diff) <= bound, i


def test_rows_far_from_zero_keep_their_variance():
    x = (torch.randn(8, 1024, device="cuda") + 4000).requires_grad_()
    w, b = torch.ones(1024, device="cuda"), torch.zeros(1024, device="cuda")
    z = f64(x)
    ey = bounds(z, np.zeros_like(z), f64(w), f64(b), 1e-7, np.zeros_like(z))[0]
    want = orc.layer_norm(z, 1.0, 0.0, 1e-7)
    near(layer_norm(x, w, b, 1e-7), want, ey + rounding(want, F), "y")
    # The bound says something here: the mean is off by at most CHAIN u 4000 = 0.0153, the variance by 2 * 0.0153 * mean|d| (0.8) = 0.0245 of
    # itself, so h by 0.0153 + 0.0245 |h|, and |h| < 5: 0.138.  A variance from sums of squares would be off by CHAIN u 4000^2 = 61.
    assert ey.max() < 0.138


@pytest.mark.parametrize("dtype", [F, B])
def test_layouts_and_alignment(dtype):
    """Views of wider tensors, odd offsets, transposed and expanded rows: the bits of the contiguous call."""
    g = torch.Generator("cuda").manual_seed(5)
    wide = torch.randn(50, 3 * 128 + 5, device="cuda", generator=g).to(dtype)
    w, b = (torch.randn(2 * 128 + 1, device="cuda", generator=g).to(dtype)[i:i + 128] for i in (1, 129))
    views = [wide[:, 128:256], wide[:, 1:129], wide[::3, 8:136], wide[:1, :128].expand(40, 128), wide[:, :256].t()[:128, :40].t(),
             wide[:40, :256].unflatten(1, (2, 128)), wide[:40, :384].unflatten(1, (3, 128))[:, ::2]]
    for x in views:
        res = torch.randn(x.shape, device="cuda", generator=g).to(dtype)
        dy = torch.randn(x.shape, device="cuda", generator=g).to(dtype)
        outs = []
        for a, d in ((x, dy), (x.contiguous(), dy), (x, dy.transpose(0, -2).contiguous().transpose(0, -2))):
            a = a.detach().requires_grad_()
            y = dropout_add_layer_norm(a, res, w, b, 1e-6, 0.2, 8)
            outs.append((y, torch.autograd.grad(y, a, d)[0]))
        for y, dx in outs[1:]:
            assert torch.equal(y, outs[0][0])
            # alignment decides between vector and single loads, and so the order of the row's sums
            assert (dx.float() - outs[0][1].float()).abs().max() <= (2 * HALF[dtype] + 256 * U) * outs[0][1].float().abs().max()


def test_empty_rows_and_missing_gradients():
    w, b = torch.ones(64, device="cuda", requires_grad=True), torch.zeros(64, device="cuda", requires_grad=True)
    x = torch.zeros(0, 5, 64, device="cuda", requires_grad=True)
    y = layer_norm(x, w, b)
    assert y.shape == x.shape
    y.sum().backward()
    assert x.grad.shape == x.shape and not w.grad.any() and not b.grad.any()
    x, res = torch.randn(20, 64, device="cuda"), torch.randn(20, 64, device="cuda")
    dy = torch.randn(20, 64, device="cuda")
    every = (x, res, w.detach(), b.detach())
    leaves = [t.clone().requires_grad_() for t in every]
    for p in (0.0, 0.4):
        want = torch.autograd.grad(dropout_add_layer_norm(*leaves, 1e-6, p, 2), leaves, dy)
        for k in range(4):                           # one input at a time
            one = [t.clone().requires_grad_(i == k) for i, t in enumerate(every)]
            got, = torch.autograd.grad(dropout_add_layer_norm(*one, 1e-6, p, 2), one[k], dy)
            assert torch.equal(got, want[k]), (p, k)


def test_two_runs_give_the_same_bits():
    x, res, w, b, dy = norm_case(3000, 1024, B, F, True)
    leaves = [t.requires_grad_() for t in (x, res, w, b)]
    runs = [torch.autograd.grad(dropout_add_layer_norm(*leaves, 1e-7, 0.1, 3), leaves, dy) for _ in range(2)]
    assert all(torch.equal(a, c) for a, c in zip(*runs))


def test_second_derivative_is_refused():
    x = torch.randn(4, 64, device="cuda", requires_grad=True)
    w, b = torch.ones(64, device="cuda"), torch.zeros(64, device="cuda")
    for y in (dropout(x, 0.5, 1), layer_norm(x, w, b)):
        with pytest.raises(RuntimeError, match="no second derivative"):
            torch.autograd.grad(y.sum(), x, create_graph=True)


def test_inputs_on_two_streams_and_a_captured_step():
    """A forward and backward pass captured once and replayed with new inputs, while an eager pass of the same sizes runs elsewhere."""
    x, res, w, b, dy = norm_case(257, 768, B, F, True)
    x.requires_grad_()
    seed = torch.tensor([5], device="cuda")
    side = torch.cuda.Stream()

    def step(x):
        y = dropout_add_layer_norm(x, res, w, b, 1e-7, 0.1, seed)
        return y.detach(), torch.autograd.grad(y, x, dy)[0]

    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, dx = step(x)
    new = torch.randn(257, 768, device="cuda").to(B)
    with torch.no_grad():
        x.copy_(new)
    seed.fill_(6)
    side.wait_stream(torch.cuda.current_stream())
    graph.replay()
    with torch.cuda.stream(side):
        other = new.clone().requires_grad_()
        y2, dx2 = step(other)
    torch.cuda.synchronize()
    assert torch.equal(y, y2) and torch.equal(dx, dx2)


@pytest.mark.parametrize("p", [0.0, 0.3])
def test_one_tensor_as_both_summands(p):
    """x and residual the same tensor: its gradient is the sum of both."""
    x, _, w, b, dy = norm_case(40, 264, F, F, False)
    both = x.clone().requires_grad_()
    got, = torch.autograd.grad(dropout_add_layer_norm(both, both, w, b, 1e-6, p, 3), both, dy)
    one, two = x.clone().requires_grad_(), x.clone().requires_grad_()
    parts = torch.autograd.grad(dropout_add_layer_norm(one, two, w, b, 1e-6, p, 3), (one, two), dy)
    assert torch.equal(got, parts[0] + parts[1])
