"""Each form of the projection with adapters, element by element against 64-bit arithmetic, at sizes that no tile, stage or vector divides.

Bounds as in test_lora_gpu.py: u = 2^-24; a sum of n products is off by at most 2 n u times the sum of their magnitudes, inner values kept as two bf16 numbers
by 2^-16 of themselves, the result by half a step of its type.
"""
import pytest
import torch

from turbodeberta_b200 import _cabi as cabi
from turbodeberta_b200.ops.lora import lora_linear

pytestmark = pytest.mark.gpu
F, B = torch.float32, torch.bfloat16
U, SPLIT = 2.0 ** -24, 2.0 ** -16
HALF = {F: 2.0 ** -24, B: 2.0 ** -8}
PAIR, WIDE, NARROW = (256, 2), (128, 1), (64, 1)


def problem(rows, cols, features, rank, n, dtype, text, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    r = lambda *s, k=1.0: (torch.randn(*s, device="cuda", generator=g) * k).to(dtype)  # noqa: E731
    ids = torch.randint(-1, n, (rows // text + 1,), device="cuda", generator=g, dtype=torch.int32).repeat_interleave(text)[:rows]
    return dict(x=r(rows, cols), w=r(features, cols, k=cols ** -0.5), bias=r(features), a=r(n, rank, cols, k=cols ** -0.5), b=r(n, features, rank, k=rank ** -0.5),
                s=torch.rand(n, device="cuda", generator=g) + 0.5, dy=r(rows, features), ids=ids)


def exact(p):
    """Results and bounds without the last rounding."""
    x, w, a, b, s, dy, bias = (p[k].double() for k in ("x", "w", "a", "b", "s", "dy", "bias"))
    ids, (N, K), R, T = p["ids"], w.shape, a.shape[1], len(x)
    ax, aw, aa, ab, ad = (t.abs() for t in (x, w, a, b, dy))
    y, dx = x @ w.T + bias, dy @ w
    ey, edx = 2 * K * U * (ax @ aw.T) + 4 * U * bias.abs(), 2 * N * U * (ad @ aw)
    da, db, eda, edb = (torch.zeros_like(t) for t in (a, b, a, b))
    for i in range(len(a)):
        at = (ids == i).nonzero()[:, 0]
        h, u = s[i] * (x[at] @ a[i].T), s[i] * (dy[at] @ b[i])
        mh, mu = s[i] * (ax[at] @ aa[i].T), s[i] * (ad[at] @ ab[i])
        eh, eu = mh * (2 * K * U + SPLIT + 4 * U), mu * (2 * N * U + SPLIT + 4 * U)
        y[at] += h @ b[i].T
        dx[at] += u @ a[i]
        ey[at] += (eh + 2 * (R + K) * U * mh) @ ab[i].T
        edx[at] += (eu + 2 * (R + N) * U * mu) @ aa[i]
        da[i], db[i] = u.T @ x[at], dy[at].T @ h
        eda[i], edb[i] = (eu + 2 * T * U * mu).T @ ax[at], ad[at].T @ (eh + 2 * T * U * mh)
    return dict(y=(y, ey + 4 * U * y.abs()), dx=(dx, edx + 4 * U * dx.abs()), da=(da, eda), db=(db, edb))


def run(p):
    leaves = [p[k].clone().requires_grad_() for k in "xab"]
    y = lora_linear(leaves[0], p["w"], p["bias"], leaves[1], leaves[2], p["s"], p["ids"])
    return dict(zip(("y", "dx", "da", "db"), (y.detach(), *torch.autograd.grad(y, leaves, p["dy"]))))


def check(p, dtype):
    got = run(p)
    for k, (want, err) in exact(p).items():
        assert torch.isfinite(got[k]).all(), k
        over = (got[k].double() - want).abs() - (err + (want.abs() + err) * HALF[dtype] + 1e-37)
        worst = int(over.argmax())
        assert over.flatten()[worst] <= 0, (k, worst, float(over.flatten()[worst]), float(want.flatten()[worst]))
    with torch.no_grad():
        assert torch.equal(got["y"], lora_linear(p["x"], p["w"], p["bias"], p["a"], p["b"], p["s"], p["ids"]))


TENSOR_CORES = [  # rows, cols, features, rank, adapters, rows to a text, form going forward, form coming back
    (500, 1016, 4088, 5, 4, 30, WIDE, NARROW), (1301, 2040, 1000, 12, 7, 40, WIDE, PAIR), (2603, 584, 4088, 33, 5, 100, PAIR, WIDE),
    (2603, 4088, 200, 12, 40, 1, NARROW, PAIR), (3001, 1032, 776, 33, 3, 7, PAIR, PAIR), (2001, 776, 1544, 5, 3, 300, PAIR, WIDE),
    (2603, 520, 1032, 64, 6, 50, PAIR, WIDE), (1301, 1000, 2040, 8, 30, 1, PAIR, WIDE), (9001, 72, 2056, 20, 9, 100, PAIR, NARROW),
    (19999, 136, 1016, 8, 3, 400, PAIR, PAIR), (6001, 1288, 72, 7, 130, 3, NARROW, PAIR), (1500, 2056, 328, 100, 60, 2, NARROW, PAIR)]


@pytest.mark.parametrize("rows,cols,features,rank,n,text,forward,back", TENSOR_CORES)
def test_each_form_on_the_tensor_cores(rows, cols, features, rank, n, text, forward, back):
    assert cabi.host.lora_form(rows, features) == forward and cabi.host.lora_form(rows, cols) == back
    check(problem(rows, cols, features, rank, n, B, text, seed=rows + rank), B)


def test_the_forms_are_all_covered():
    seen = {(way, form, rank % 8 == 0) for _, _, _, rank, _, _, f, b in TENSOR_CORES for way, form in (("forward", f), ("back", b))}
    assert {s[:2] for s in seen} == {(w, f) for w in ("forward", "back") for f in (PAIR, WIDE)} | {("forward", NARROW), ("back", NARROW)}
    assert {s for s in seen if s[1] == PAIR} == {(w, PAIR, v) for w in ("forward", "back") for v in (False, True)}


@pytest.mark.parametrize("dtype,rows,cols,features,rank,n,text", [(F, 2000, 771, 773, 5, 3, 60), (F, 3001, 264, 520, 20, 40, 1), (F, 1025, 1024, 1024, 16, 2, 500),
                                                                  (F, 4100, 64, 96, 64, 8, 33), (B, 2000, 771, 773, 5, 3, 60), (B, 3001, 263, 129, 17, 40, 1)])
def test_the_form_for_other_types_and_sizes_with_many_rows(dtype, rows, cols, features, rank, n, text):
    check(problem(rows, cols, features, rank, n, dtype, text, seed=rows), dtype)


@pytest.mark.parametrize("rows,cols,features,rank", [(2603, 584, 4088, 12), (2603, 4088, 200, 12), (3001, 1032, 776, 16)])
@pytest.mark.parametrize("text", [1, 200])
def test_an_adapter_that_is_not_finite_in_tiles_that_two_share(rows, cols, features, rank, text):
    p = problem(rows, cols, features, rank, 3, B, text, seed=2)
    assert PAIR in (cabi.host.lora_form(rows, features), cabi.host.lora_form(rows, cols))
    clean, hurt = run(p), p["ids"] == 1
    for name, bad in (("a", float("nan")), ("a", float("inf")), ("b", float("inf")), ("b", float("nan"))):
        q = dict(p)
        q[name] = p[name].clone()
        q[name][1, 3, 5] = bad
        got = run(q)
        for k in ("y", "dx"):
            assert torch.equal(got[k][~hurt], clean[k][~hurt]), (name, k)
        for k in ("da", "db"):
            assert torch.equal(got[k][[0, 2]], clean[k][[0, 2]]), (name, k)
        if name == "b":                              # one column of the result
            others = torch.arange(features, device="cuda") != 3
            assert torch.equal(got["y"][hurt][:, others], clean["y"][hurt][:, others]) and not torch.isfinite(got["y"][hurt][:, 3]).any()
            assert not torch.isfinite(got["dx"][hurt]).any()
        else:                                        # one column of dx
            others = torch.arange(cols, device="cuda") != 5
            assert torch.equal(got["dx"][hurt][:, others], clean["dx"][hurt][:, others]) and not torch.isfinite(got["dx"][hurt][:, 5]).any()
            assert not torch.isfinite(got["y"][hurt]).any()


@pytest.mark.parametrize("dtype,cols,features", [(B, 584, 4088), (B, 4088, 200), (F, 264, 130), (B, 65, 66)])
def test_ids_of_sequences_are_ids_of_their_rows(dtype, cols, features):
    """Gradients too, with as many rows as are sorted by adapter; 64-bit ids, and ids that lie apart in memory."""
    p = problem(2600, cols, features, 12, 5, dtype, 1, seed=3)
    per = torch.tensor([3, -1, 0, 4, 4, 1 << 20, 2, 0], device="cuda", dtype=torch.int32)
    p["ids"] = per.repeat_interleave(325)
    want = run(p)
    apart = torch.stack([per.long(), torch.zeros(8, dtype=torch.int64, device="cuda")], 1)[:, 0]
    for ids in (per, per.long(), apart, torch.where(per < 0, per.long() - (1 << 40), per.long() + (per > 4) * (1 << 40))):
        q = dict(p, x=p["x"].view(8, 325, cols), dy=p["dy"].view(8, 325, features), ids=ids)
        got = run(q)
        assert all(torch.equal(got[k].reshape(want[k].shape), want[k]) for k in want)
    p["a"], p["b"], p["s"] = p["a"][:1], p["b"][:1], p["s"][:1]
    p["ids"] = torch.zeros(2600, dtype=torch.int32, device="cuda")
    want = run(p)
    p["ids"] = None                                  # one adapter for all
    got = run(p)
    assert all(torch.equal(got[k], want[k]) for k in want)
