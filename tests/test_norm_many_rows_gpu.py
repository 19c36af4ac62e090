"""LayerNorm and the joined end of a sublayer at row counts from which blocks hold eight rows (16 to an SM) and a thread of the backward pass several, against
64-bit arithmetic; the bounds are those of test_train_ops_gpu.py."""
import numpy as np
import pytest
import torch

from oracle import train_oracle as orc
from tests.test_train_ops_gpu import B, F, HALF, TINY, U, bounds, f64, near, norm_case
from turbodeberta_b200.ops.layer_norm import dropout_add_layer_norm, layer_norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,wt", [(F, F), (B, B), (B, F)])
@pytest.mark.parametrize("rows,cols", [(2367, 64), (2368, 64), (2375, 768), (2401, 1024), (3001, 1000), (2600, 771), (2500, 257), (5003, 16), (4000, 7), (2500, 520), (2369, 1032),
                                       (9216, 1024)])
@pytest.mark.parametrize("form", ["alone", "join", "drop"])
def test_many_rows(rows, cols, dtype, wt, form):
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
    with torch.no_grad():                            # the form without statistics
        again = layer_norm(x, w, b, eps) if form == "alone" else dropout_add_layer_norm(x, res, w, b, eps, p, 11, 4)
    assert torch.equal(again, y)
