"""What the projection with adapters refuses, and the oracle's gradients against differences; no GPU needed."""
import numpy as np
import pytest
import torch

from oracle import train_oracle as orc
from turbodeberta_b200.ops.lora import lora_linear

B = torch.bfloat16
Z = torch.zeros


@pytest.mark.parametrize("x,w,bias,a,b,scaling,ids,message", [
    (Z(3, 4), Z(5, 3), None, Z(1, 2, 4), Z(1, 5, 2), 1.0, None, "do not fit"),
    (Z(3, 4), Z(5, 4, 1), None, Z(1, 2, 4), Z(1, 5, 2), 1.0, None, "do not fit"),
    (Z(()), Z(5, 4), None, Z(1, 2, 4), Z(1, 5, 2), 1.0, None, "do not fit"),
    (Z(3, 0), Z(5, 0), None, Z(1, 2, 0), Z(1, 5, 2), 1.0, None, "must not be empty"),
    (Z(3, 4), Z(5, 4), None, Z(1, 2, 5), Z(1, 5, 2), 1.0, None, "lora_a must be"),
    (Z(3, 4), Z(5, 4), None, Z(2, 2, 4), Z(1, 5, 2), 1.0, None, "lora_a must be"),
    (Z(3, 4), Z(5, 4), None, Z(1, 2, 4), Z(1, 5, 3), 1.0, None, "lora_a must be"),
    (Z(3, 4), Z(5, 4), None, Z(0, 2, 4), Z(0, 5, 2), 1.0, None, "lora_a must be"),
    (Z(3, 4), Z(5, 4), None, Z(1, 257, 4), Z(1, 5, 257), 1.0, None, "up to 256"),
    (Z(3, 4), Z(5, 4), None, Z(4096, 1, 4), Z(4096, 5, 1), 1.0, Z(3, dtype=torch.int32), "up to 4095"),
    (Z(3, 4), Z(5, 4), Z(4), Z(1, 2, 4), Z(1, 5, 2), 1.0, None, "bias must be"),
    (Z(3, 4), Z(5, 4), None, Z(1, 2, 4, dtype=B), Z(1, 5, 2, dtype=B), 1.0, None, "share a dtype"),
    (Z(3, 4, dtype=torch.float16), Z(5, 4), None, Z(1, 2, 4), Z(1, 5, 2), 1.0, None, "float32 or bfloat16"),
    (Z(3, 4), Z(5, 4), None, Z(1, 2, 4), Z(1, 5, 2), Z(2), None, "scaling must be"),
    (Z(3, 4), Z(5, 4), None, Z(1, 2, 4), Z(1, 5, 2), Z(1, dtype=torch.float64), None, "scaling must be"),
    (Z(3, 4), Z(5, 4), None, Z(2, 2, 4), Z(2, 5, 2), 1.0, None, "single adapter"),
    (Z(3, 4), Z(5, 4), None, Z(2, 2, 4), Z(2, 5, 2), 1.0, Z(3), "int32 or int64"),
    (Z(3, 4), Z(5, 4), None, Z(2, 2, 4), Z(2, 5, 2), 1.0, Z(2, dtype=torch.int32), "shape of x"),
    (Z(3, 4), Z(5, 4), None, Z(2, 2, 4), Z(2, 5, 2), 1.0, Z(1, 3, dtype=torch.int32), "shape of x"),
    (Z(2, 3, 4), Z(5, 4), None, Z(2, 2, 4), Z(2, 5, 2), 1.0, Z(3, dtype=torch.int64), "shape of x"),
])
def test_refusals(x, w, bias, a, b, scaling, ids, message):
    with pytest.raises(ValueError, match=message):
        lora_linear(x, w, bias, a, b, scaling, ids)


def test_refuses_the_cpu():
    with pytest.raises(RuntimeError, match="no CPU path"):
        lora_linear(Z(3, 4), Z(5, 4), None, Z(1, 2, 4), Z(1, 5, 2))


def test_oracle_gradients_against_differences():
    r = np.random.RandomState(0)
    x, w, a, b, dy = r.randn(6, 5), r.randn(4, 5), r.randn(3, 2, 5), r.randn(3, 4, 2), r.randn(6, 4)
    s, ids = r.rand(3) + 0.5, np.array([0, 2, -1, 2, 7, 0])
    grads = orc.lora_linear_backward(x, w, a, b, s, ids, dy)
    at = [x, a, b]
    for i, g in enumerate(grads):
        v = r.randn(*at[i].shape)
        ends = []
        for k in (1e-5, -1e-5):
            p = [t + k * v if j == i else t for j, t in enumerate(at)]
            ends.append((orc.lora_linear(p[0], w, None, p[1], p[2], s, ids) * dy).sum())
        assert abs((g * v).sum() - (ends[0] - ends[1]) / 2e-5) < 1e-7
