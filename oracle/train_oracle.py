"""The training path's operators in numpy, 64 bits: dropout, LayerNorm with its gradients, projections with low-rank adapters."""
import numpy as np

ROUNDS, M0, M1, W0, W1, LOW = 10, 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85, 0xFFFFFFFF


def philox4x32(counter, key):
    """One block for whole-number counter (4 words) and key (2 words), word by word as the paper has it."""
    c, k = list(counter), list(key)
    for _ in range(ROUNDS):
        a, b = M0 * c[0], M1 * c[2]
        c = [(b >> 32) ^ c[1] ^ k[0], b & LOW, (a >> 32) ^ c[3] ^ k[1], a & LOW]
        k = [(k[0] + W0) & LOW, (k[1] + W1) & LOW]
    return c


def dropped(p):
    """Of 65536 numbers."""
    return int(np.floor(p * 65536 + 0.5))


def numbers(first, count, seed, offset):
    """The 16-bit numbers of elements first .. first + count - 1."""
    group = np.arange(first // 8, (first + count + 7) // 8, dtype=np.uint64)
    low, half = np.uint64(LOW), np.uint64(32)
    c = [group & low, group >> half, np.full_like(group, offset & LOW), np.full_like(group, (offset >> 32) & LOW)]
    k0, k1 = seed & LOW, (seed >> 32) & LOW
    for _ in range(ROUNDS):
        a, b = c[0] * np.uint64(M0), c[2] * np.uint64(M1)
        c = [(b >> half) ^ c[1] ^ np.uint64(k0), b & low, (a >> half) ^ c[3] ^ np.uint64(k1), a & low]
        k0, k1 = (k0 + W0) & LOW, (k1 + W1) & LOW
    words = np.stack(c, 1)
    both = np.stack([words & np.uint64(0xFFFF), words >> np.uint64(16)], 2).reshape(-1)
    return both[first % 8:first % 8 + count].astype(np.int64)


def stays(shape, p, seed, offset=0):
    return (numbers(0, int(np.prod(shape)), seed, offset) >= dropped(p)).reshape(shape)


def dropout(x, p, seed, offset=0):
    """(y, mask, scale)"""
    keep = stays(x.shape, p, seed, offset)
    scale = 65536 / (65536 - dropped(p)) if dropped(p) < 65536 else 0.0
    return np.where(keep, x, 0) * scale, keep, scale


def layer_norm(z, w, b, eps):
    d = z - z.mean(-1, keepdims=True)
    return d / np.sqrt((d * d).mean(-1, keepdims=True) + eps) * w + b


def layer_norm_backward(z, w, eps, dy):
    """(dz, dw, db); rows are all leading dimensions."""
    d = z - z.mean(-1, keepdims=True)
    inv = 1 / np.sqrt((d * d).mean(-1, keepdims=True) + eps)
    h, g = d * inv, dy * w
    dz = (g - g.mean(-1, keepdims=True) - h * (g * h).mean(-1, keepdims=True)) * inv
    lead = tuple(range(z.ndim - 1))
    return dz, (dy * h).sum(lead), dy.sum(lead)


def lora_linear(x, w, b, lora_a, lora_b, scaling, ids):
    """x [T, in], ids [T] (a row whose id is not an adapter's has none)."""
    y = x @ w.T
    if b is not None:
        y = y + b
    for t in range(len(x)):
        i = int(ids[t])
        if 0 <= i < len(lora_a):
            y[t] += scaling[i] * (lora_b[i] @ (lora_a[i] @ x[t]))
    return y


def lora_linear_backward(x, w, lora_a, lora_b, scaling, ids, dy):
    """(dx, dlora_a, dlora_b); w is frozen."""
    dx, da, db = dy @ w, np.zeros_like(lora_a), np.zeros_like(lora_b)
    for t in range(len(x)):
        i = int(ids[t])
        if 0 <= i < len(lora_a):
            u = scaling[i] * (dy[t] @ lora_b[i])
            dx[t] += u @ lora_a[i]
            da[i] += np.outer(u, x[t])
            db[i] += np.outer(dy[t], scaling[i] * (lora_a[i] @ x[t]))
    return dx, da, db
