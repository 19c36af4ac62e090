"""What the training path's operators refuse, and the oracle's random numbers against the paper's vectors; no GPU needed."""
import numpy as np
import pytest
import torch

from oracle import train_oracle as orc
from turbodeberta_b200.ops.dropout import dropout, signed64
from turbodeberta_b200.ops.layer_norm import dropout_add_layer_norm, layer_norm

F, B = torch.float32, torch.bfloat16


def test_philox_known_answers():
    """The test vectors published with the generator."""
    pi = [0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344]
    assert orc.philox4x32([0] * 4, [0] * 2) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert orc.philox4x32([orc.LOW] * 4, [orc.LOW] * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert orc.philox4x32(pi, [0xA4093822, 0x299F31D0]) == [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]


@pytest.mark.parametrize("seed,offset,first", [(0, 0, 0), (-1, 5, 3), (1 << 40, (1 << 33) + 1, (1 << 35) + 5)])
def test_oracle_numbers_are_the_blocks_halves(seed, offset, first):
    got = orc.numbers(first, 21, seed, offset)
    for i in range(21):
        e = first + i
        w = orc.philox4x32([e // 8 & orc.LOW, e // 8 >> 32, offset & orc.LOW, offset >> 32 & orc.LOW], [seed & orc.LOW, seed >> 32 & orc.LOW])
        assert got[i] == w[e % 8 // 2] >> 16 * (e % 2) & 0xFFFF


def test_seeds_are_64_bits():
    assert signed64(-1, "seed") == -1 and signed64((1 << 64) - 1, "seed") == -1 and signed64(1 << 62, "seed") == 1 << 62
    for bad in (1 << 64, -(1 << 63) - 1):
        with pytest.raises(ValueError, match="64 bits"):
            signed64(bad, "seed")


@pytest.mark.parametrize("p", [-0.1, 1.1, float("nan")])
def test_dropout_refuses_probabilities(p):
    with pytest.raises(ValueError, match="between 0 and 1"):
        dropout(torch.zeros(4), p, 1)


def test_dropout_refuses_types_seeds_and_the_cpu():
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        dropout(torch.zeros(4, dtype=torch.float16), 0.1, 1)
    for seed in (torch.zeros(2, dtype=torch.int64), torch.zeros(1, dtype=torch.int32)):
        with pytest.raises(ValueError, match="int64 tensor of one element"):
            dropout(torch.zeros(4), 0.1, seed)
    with pytest.raises(RuntimeError, match="no CPU path"):
        dropout(torch.zeros(4), 0.1, 1)


@pytest.mark.parametrize("x,w,b,eps,message", [
    (torch.zeros(()), torch.zeros(1), torch.zeros(1), 0.0, "at least one dimension"),
    (torch.zeros(2, 0), torch.zeros(0), torch.zeros(0), 0.0, "between 1 and 16384"),
    (torch.zeros(1, 16385), torch.zeros(16385), torch.zeros(16385), 0.0, "between 1 and 16384"),
    (torch.zeros(2, 4), torch.zeros(5), torch.zeros(5), 0.0, "vectors of the last dimension"),
    (torch.zeros(2, 4), torch.zeros(4), torch.zeros(1, 4), 0.0, "vectors of the last dimension"),
    (torch.zeros(2, 4), torch.zeros(4, dtype=B), torch.zeros(4, dtype=B), 0.0, "share a dtype"),
    (torch.zeros(2, 4, dtype=B), torch.zeros(4, dtype=B), torch.zeros(4), 0.0, "share a dtype"),
    (torch.zeros(2, 4, dtype=torch.float64), torch.zeros(4), torch.zeros(4), 0.0, "float32 or bfloat16"),
    (torch.zeros(2, 4), torch.zeros(4), torch.zeros(4), -1.0, "eps"),
    (torch.zeros(2, 4), torch.zeros(4), torch.zeros(4), float("nan"), "eps"),
])
def test_layer_norm_refuses(x, w, b, eps, message):
    with pytest.raises(ValueError, match=message):
        layer_norm(x, w, b, eps)


def test_dropout_add_layer_norm_refuses():
    x, w = torch.zeros(2, 4), torch.zeros(4)
    for res in (torch.zeros(1, 4), torch.zeros(2, 4, dtype=B)):
        with pytest.raises(ValueError, match="shape and the dtype"):
            dropout_add_layer_norm(x, res, w, w)
    with pytest.raises(ValueError, match="residual is missing"):
        dropout_add_layer_norm(x, None, w, w)
    with pytest.raises(ValueError, match="needs a seed"):
        dropout_add_layer_norm(x, x, w, w, p=0.1)
    with pytest.raises(ValueError, match="between 0 and 1"):
        dropout_add_layer_norm(x, x, w, w, p=2.0, seed=1)
    with pytest.raises(RuntimeError, match="no CPU path"):
        dropout_add_layer_norm(x, x, w, w, p=0.1, seed=1)


def test_oracle_gradient_against_differences():
    r = np.random.RandomState(0)
    z, w, b, dy, v = r.randn(3, 7), r.randn(7), r.randn(7), r.randn(3, 7), r.randn(3, 7)
    step = 1e-5
    want = ((orc.layer_norm(z + step * v, w, b, 1e-7) - orc.layer_norm(z - step * v, w, b, 1e-7)) * dy).sum() / (2 * step)
    assert abs((orc.layer_norm_backward(z, w, 1e-7, dy)[0] * v).sum() - want) < 1e-8
