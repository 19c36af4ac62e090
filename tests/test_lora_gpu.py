"""Projections with adapters on the GPU against 64-bit arithmetic, forward and backward.

Bounds: u = 2^-24.  A sum of n products in fp32, in any order and with accumulators that may cut instead of round, is off by at most
2 n u times the sum of the products' magnitudes.  The inner values of the adapters may be held as two bf16 numbers, whose sum is off by at most
2^-16 of the value (half a step of the second, which is at most half a step of the first).  The result is rounded once, half a step of its type.
"""
import numpy as np
import pytest
import torch

from oracle import train_oracle as orc
from turbodeberta_b200.ops.lora import lora_linear

pytestmark = pytest.mark.gpu
F, B = torch.float32, torch.bfloat16
U, SPLIT = 2.0 ** -24, 2.0 ** -16
HALF = {F: 2.0 ** -24, B: 2.0 ** -8}


def f64(t):
    return t.detach().double().cpu().numpy()


def near(got, want, err, dtype, what):
    got = f64(got)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    tol = err + (np.abs(want) + err) * HALF[dtype] + 1e-37
    off = np.abs(got - want)
    assert np.isfinite(got).all(), what
    worst = np.argmax(off - tol) if off.size else 0
    assert not off.size or off.flat[worst] <= tol.flat[worst], f"{what}: off by {off.flat[worst]:.3e} at {worst}, bound {tol.flat[worst]:.3e}"


def problem(rows, cols, features, rank, n, dtype, ids, seed=0, bias=True):
    g = torch.Generator("cuda").manual_seed(seed)
    r = lambda *s, k=1.0: (torch.randn(*s, device="cuda", generator=g) * k).to(dtype)  # noqa: E731
    p = dict(x=r(rows, cols), w=r(features, cols, k=cols ** -0.5), bias=r(features) if bias else None, a=r(n, rank, cols, k=cols ** -0.5),
             b=r(n, features, rank, k=rank ** -0.5), s=torch.rand(n, device="cuda", generator=g) + 0.5, dy=r(rows, features))
    rs = np.random.RandomState(seed)
    if ids == "texts":                               # requests of ragged lengths
        v = np.repeat(rs.randint(-1, n, rows), rs.randint(1, 40, rows))[:rows]
    elif ids == "mixed":
        v = rs.randint(-1, n + 1, rows)              # n: not an adapter
    elif ids == "one":
        v = np.full(rows, n - 1)
    else:
        v = np.full(rows, -1)
    p["ids"] = torch.from_numpy(v.astype(np.int32)).cuda()
    return p


def exact(p):
    """Results in 64 bits and their bounds, row by row of the oracle and once more with magnitudes."""
    x, w, a, b, s, dy = (f64(p[k]) for k in ("x", "w", "a", "b", "s", "dy"))
    ids = p["ids"].cpu().numpy()
    bias = None if p["bias"] is None else f64(p["bias"])
    K, N, R, T = w.shape[1], w.shape[0], a.shape[1], len(x)
    y = orc.lora_linear(x, w, bias, a, b, s, ids)
    dx, da, db = orc.lora_linear_backward(x, w, a, b, s, ids, dy)
    ax, aw, aa, ab, ad = (np.abs(t) for t in (x, w, a, b, dy))
    ey = 2 * K * U * (ax @ aw.T) + 4 * U * (np.abs(y) + (0 if bias is None else np.abs(bias)))
    edx = 2 * N * U * (ad @ aw) + 4 * U * np.abs(dx)
    eda, edb = np.zeros_like(a), np.zeros_like(b)
    for i in range(len(a)):
        at = np.nonzero(ids == i)[0]
        if not len(at):
            continue
        mh, mu = s[i] * (ax[at] @ aa[i].T), s[i] * (ad[at] @ ab[i])               # magnitudes of h and u, products added up
        eh, eu = mh * (2 * K * U + SPLIT + 4 * U), mu * (2 * N * U + SPLIT + 4 * U)
        ey[at] += (eh + 2 * (R + K) * U * mh) @ ab[i].T
        edx[at] += (eu + 2 * (R + N) * U * mu) @ aa[i]
        eda[i] = (eu + 2 * T * U * mu).T @ ax[at]
        edb[i] = ad[at].T @ (eh + 2 * T * U * mh)
    return dict(y=(y, ey), dx=(dx, edx), da=(da, eda), db=(db, edb))


def run(p, **more):
    leaves = [p[k].detach().clone().requires_grad_() for k in ("x", "a", "b")]
    y = lora_linear(leaves[0], p["w"], p["bias"], leaves[1], leaves[2], p["s"], p["ids"], **more)
    return dict(zip(("y", "dx", "da", "db"), (y.detach(), *torch.autograd.grad(y, leaves, p["dy"]))))


SIZES = [(1, 64, 64, 8, 1), (1, 1024, 128, 16, 4), (2, 63, 65, 3, 2), (16, 1024, 256, 8, 16), (17, 128, 512, 64, 3), (33, 771, 773, 5, 3), (40, 8, 8, 1, 2),
         (64, 512, 320, 33, 5), (127, 72, 200, 16, 8), (129, 264, 128, 20, 4), (200, 1024, 1000, 16, 8), (300, 256, 264, 128, 2), (257, 640, 640, 100, 3),
         (700, 200, 136, 4, 32), (513, 1, 3, 2, 2), (150, 128, 192, 256, 2), (400, 64, 72, 2, 4095)]


@pytest.mark.parametrize("dtype", [F, B])
@pytest.mark.parametrize("rows,cols,features,rank,n", SIZES)
@pytest.mark.parametrize("ids", ["texts", "mixed", "one", "none"])
def test_forward_and_gradients(rows, cols, features, rank, n, dtype, ids):
    p = problem(rows, cols, features, rank, n, dtype, ids, seed=rows + rank, bias=rows % 2 == 0)
    want, got = exact(p), run(p)
    for k in ("y", "dx", "da", "db"):
        near(got[k], *want[k], dtype, k)
    with torch.no_grad():                            # nothing kept: the same result
        assert torch.equal(got["y"], lora_linear(p["x"], p["w"], p["bias"], p["a"], p["b"], p["s"], p["ids"]))


@pytest.mark.parametrize("dtype", [F, B])
@pytest.mark.parametrize("rows", [5, 190])
def test_an_adapter_with_nan_reaches_its_own_rows_only(rows, dtype):
    """Rows of several adapters share tiles; so do rows that hold anything."""
    p = problem(rows, 256, 192, 12, 3, dtype, "mixed", seed=4)
    clean = run(p)
    for name, bad in (("a", float("nan")), ("b", float("inf")), ("x", float("nan")), ("dy", float("-inf"))):
        q = dict(p)
        q[name] = p[name].clone()
        hurt = p["ids"] == 1
        if name in "ab":
            q[name][1, 3, 5] = bad
        else:
            q[name][hurt] = bad
        got = run(q)
        for k in ("y", "dx"):
            assert torch.equal(got[k][~hurt], clean[k][~hurt]), (name, k)
        for k in ("da", "db"):
            assert torch.equal(got[k][[0, 2]], clean[k][[0, 2]]), (name, k)
        if name == "b":                              # infinite where the row's inner value is not zero, and in that column only
            assert torch.equal(got["y"][hurt][:, 4:], clean["y"][hurt][:, 4:]) and not torch.isfinite(got["y"][hurt][:, 3]).any()
        if name == "a":
            assert torch.isnan(got["y"][hurt]).all()


@pytest.mark.parametrize("dtype", [F, B])
def test_forms_of_ids_scaling_and_x(dtype):
    p = problem(120, 256, 320, 16, 3, dtype, "texts", seed=9)
    call = lambda x, ids, s=p["s"]: lora_linear(x, p["w"], p["bias"], p["a"], p["b"], s, ids)  # noqa: E731
    want = call(p["x"], p["ids"])
    assert torch.equal(want, call(p["x"], p["ids"].long()))
    assert torch.equal(want, call(p["x"].view(4, 30, 256), p["ids"].view(4, 30)).view(120, 320))
    per = torch.tensor([2, -1, 0, 2], device="cuda")
    assert torch.equal(call(p["x"].view(4, 30, 256), per).view(120, 320), call(p["x"], per.repeat_interleave(30)))
    assert torch.equal(call(p["x"], p["ids"], torch.full((3,), 0.75, device="cuda")), call(p["x"], p["ids"], 0.75))
    one = lora_linear(p["x"], p["w"], p["bias"], p["a"][:1], p["b"][:1], 2.0)
    assert torch.equal(one, lora_linear(p["x"], p["w"], p["bias"], p["a"][:1], p["b"][:1], 2.0, torch.zeros(120, dtype=torch.int32, device="cuda")))
    wide = torch.zeros(120, 600, device="cuda", dtype=dtype)
    for at in (8, 1):                                # aligned and not
        wide[:, at:at + 256] = p["x"]
        got = call(wide[:, at:at + 256], p["ids"])
        assert (got.float() - want.float()).abs().max() <= 2 * HALF[dtype] * want.float().abs().max() + 2e-4
    assert call(p["x"][:0], p["ids"][:0]).shape == (0, 320)
    assert call(p["x"][0], p["ids"][0]).shape == (320,)


def test_empty_batch_has_zero_gradients():
    p = problem(4, 64, 64, 8, 2, B, "one")
    p["x"], p["ids"], p["dy"] = p["x"][:0], p["ids"][:0], p["dy"][:0]
    got = run(p)
    assert got["dx"].shape == (0, 64) and not got["da"].any() and not got["db"].any() and got["da"].shape == p["a"].shape


def test_single_gradients_and_frozen_parts():
    p = problem(70, 128, 192, 8, 2, B, "texts", seed=1)
    full = run(p)
    for k, name in (("x", "dx"), ("a", "da"), ("b", "db")):
        q = {n: p[n].clone().requires_grad_(n == k) for n in ("x", "a", "b")}
        y = lora_linear(q["x"], p["w"], p["bias"], q["a"], q["b"], p["s"], p["ids"])
        assert torch.equal(torch.autograd.grad(y, q[k], p["dy"])[0], full[name])
    for name in ("w", "bias", "s"):
        q = {n: (t.clone().requires_grad_(n == name) if t.is_floating_point() else t) for n, t in p.items()}
        with pytest.raises(RuntimeError, match="frozen"):
            lora_linear(q["x"], q["w"], q["bias"], q["a"], q["b"], q["s"], q["ids"])
    x = p["x"].clone().requires_grad_()
    y = lora_linear(x, p["w"], p["bias"], p["a"], p["b"], p["s"], p["ids"])
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(y.sum(), x, create_graph=True)


@pytest.mark.parametrize("dtype", [F, B])
def test_two_runs_streams_and_a_captured_step(dtype):
    p = problem(300, 512, 512, 16, 4, dtype, "texts", seed=2)
    first = run(p)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run(p)
    here = run(p)
    torch.cuda.synchronize()
    for k in first:
        assert torch.equal(first[k], second[k]) and torch.equal(first[k], here[k]), k
    leaves = [p[k].clone().requires_grad_() for k in ("x", "a", "b")]
    ids = p["ids"].clone()

    def step():
        y = lora_linear(leaves[0], p["w"], p["bias"], leaves[1], leaves[2], p["s"], ids)
        return (y.detach(), *torch.autograd.grad(y, leaves, p["dy"]))

    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    ids.copy_(p["ids"].flip(0))
    graph.replay()
    torch.cuda.synchronize()
    p["ids"] = p["ids"].flip(0)
    again = run(p)
    for got, k in zip(out, ("y", "dx", "da", "db")):
        assert torch.equal(got, again[k]), k


@pytest.mark.parametrize("rows,cols,features,rank,n,spread", [(2600, 64, 4096, 16, 128, 1), (20000, 128, 1024, 8, 3, 400), (9000, 576, 2048, 40, 9, 100),
                                                              (1500, 2048, 320, 64, 200, 1)])
def test_many_tiles_and_many_adapters_to_a_tile(rows, cols, features, rank, n, spread):
    """Blocks that take several tiles in turn, with fewer and more steps than there are stages, and from no adapter to 128 in a tile."""
    p = problem(rows, cols, features, rank, n, B, "none", seed=rows)
    rs = np.random.RandomState(rows)
    ids = np.repeat(rs.randint(-1, n, rows // spread + 1), spread)[:rows]
    ids[rows // 2:rows // 2 + 300] = -1
    p["ids"] = torch.from_numpy(ids.astype(np.int32)).cuda()
    got = run(p)
    flag = {k: t.double() for k, t in p.items() if t.is_floating_point()}
    own = torch.from_numpy(ids >= 0).cuda()
    a, b, s = flag["a"], flag["b"], flag["s"]
    y, dx = flag["x"] @ flag["w"].T + flag["bias"], flag["dy"] @ flag["w"]
    da, db = torch.zeros_like(a), torch.zeros_like(b)
    for i in range(n):
        at = (p["ids"] == i).nonzero()[:, 0]
        h, u = s[i] * (flag["x"][at] @ a[i].T), s[i] * (flag["dy"][at] @ b[i])
        y[at] += h @ b[i].T
        dx[at] += u @ a[i]
        da[i], db[i] = u.T @ flag["x"][at], flag["dy"][at].T @ h
    assert own.any() and not own.all()
    # Sums of up to 4096 random products: the worst-case bound of the other tests is far above what wrong rows or steps would do to a sum of
    # squares, so here the whole is held against half a step for every element, doubled for the sums' own error.
    for k, want in (("y", y), ("dx", dx), ("da", da), ("db", db)):
        assert (got[k].double() - want).norm() <= 2 * HALF[B] * want.norm(), k
        assert torch.isfinite(got[k]).all()
    from turbodeberta_b200.ops.flash_attention import check_pending_status
    check_pending_status()


FRESH = """
import torch
from turbodeberta_b200.ops.flash_attention import check_pending_status
from turbodeberta_b200.ops.lora import lora_linear
g = torch.Generator("cuda").manual_seed(0)
r = lambda *s: torch.randn(*s, device="cuda", generator=g).bfloat16()
x, w, a, b = r(300, 128), r(192, 128), r(2, 8, 128), r(2, 192, 8)
ids = torch.randint(-1, 2, (300,), device="cuda", generator=g)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = lora_linear(x, w, None, a, b, 0.5, ids)
graph.replay()
want = lora_linear(x, w, None, a, b, 0.5, ids)
torch.cuda.synchronize()
assert torch.equal(y, want) and torch.isfinite(y).all()
check_pending_status()
print("fine")
"""


def test_the_first_call_of_a_process_may_be_captured():
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FRESH], cwd=root, capture_output=True, text=True, timeout=240)
    assert r.returncode == 0 and "fine" in r.stdout, r.stderr[-2000:]


def test_calls_from_several_threads_and_streams():
    """Each thread with a stream of its own, at once: the results of calls one after the other."""
    import threading
    problems = [problem(400, 256, 320, 16, 5, B, "texts", seed=i) for i in range(4)]
    want = [run(p) for p in problems]
    torch.cuda.synchronize()
    got, errors = [None] * 4, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    got[i] = run(problems[i])
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for w, g in zip(want, got):
        assert all(torch.equal(w[k], g[k]) for k in w)
