"""Operators of the training path and of serving many fine-tunings at once: what is measured of them, and in which form.

* ``dropout``                 counter-based dropout (Philox4x32-10; Salmon, Moraes, Dror and Shaw, 2011): the mask is a function
                              of seed, offset and element index, so the backward pass makes it again
* ``layer_norm``              LayerNorm, forward and backward with the gradients of weight and bias
* ``dropout_add_layer_norm``  ``LayerNorm(dropout(x) + residual)``, the end of both halves of an encoder layer, as one operator
* ``lora_linear``             a shared projection with the low-rank adapter of each row's own request beside it

``run`` computes a pass in elementary torch operations (``own`` false) or through the package's operators (``own`` true).
The mask: elements are counted in row-major order; eight of them share the Philox block of counter (index // 8, offset) under the
key ``seed``, whose four words are taken as eight 16-bit numbers, low half first; an element stays when its number is at least
``round(65536 p)``, and is divided by the share that stays.  A dropped element is zero whatever it held.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-7
MOST_ELEMENTS = 16384 * 1024


def _dropout(name, rows, cols, way="train", dtype="bf16", p=0.1, offset=0):
    c = dict(op="dropout", rows=rows, cols=cols, way=way, dtype=dtype, p=p, offset=offset)
    return dict(c, name=name) if name else c


def _norm(name, rows, cols, way="train", dtype="bf16", weights="same"):
    """weights: "same" type as the rows, or "f32" beside bf16 rows (master weights)."""
    c = dict(op="layer_norm", rows=rows, cols=cols, way=way, dtype=dtype, weights=weights)
    return dict(c, name=name) if name else c


def _join(name, rows, cols, way="train", dtype="bf16", weights="same", p=0.1, offset=0):
    c = dict(op="dropout_add_layer_norm", rows=rows, cols=cols, way=way, dtype=dtype, weights=weights, p=p, offset=offset)
    return dict(c, name=name) if name else c


def _lora(name, rows, cols, features, rank, adapters, text, way="serve", dtype="bf16", bias=True):
    """rows in requests of about `text` rows each (one: single tokens), every request with an adapter of `adapters`, about one in
    sixteen with none."""
    c = dict(op="lora_linear", rows=rows, cols=cols, features=features, rank=rank, adapters=adapters, text=text, way=way,
             dtype=dtype, bias=bias)
    return dict(c, name=name) if name else c


def listed():
    return [
        # the embeddings of one short text in training: a launch each way
        _dropout("dropout_one_text", 32, 1024),
        # the embeddings of a batch of 32 x 512 tokens of the large model
        _dropout("dropout_batch", 16384, 1024),
        # a classifier's pooled vectors in fp32, forward only, a width that no vector load divides
        _norm("norm_odd_f32", 1000, 771, way="forward", dtype="f32"),
        # a whole batch through one LayerNorm, its weights kept in fp32
        _norm("norm_batch_master", 16384, 1024, weights="f32"),
        # a short text through the end of a sublayer: latency
        _join("join_one_text", 48, 768),
        # the tokens of a ragged batch (the packed stream of 32 texts) through the end of a sublayer of the large model
        _join("join_batch", 9216, 1024),
        # the same end in fp32, a wide model, where a row no longer fits one warp's registers
        _join("join_wide_f32", 2000, 4096, dtype="f32", p=0.25, offset=7),
        # the last token of sixteen requests, each with an adapter of its own: bound by reading the shared weights
        _lora("lora_single_tokens", 16, 1024, 1024, 8, 16, text=1),
        # a handful of short texts from eight customers, up-projection of the large model
        _lora("lora_short_texts", 200, 1024, 4096, 16, 8, text=25),
        # a full ragged batch of 32 texts and as many adapters
        _lora("lora_batch", 9216, 1024, 4096, 16, 32, text=288),
        # a training step of four adapters on the down-projection
        _lora("lora_train", 8192, 4096, 1024, 32, 4, text=512, way="train"),
        # exact training in fp32: odd sizes, odd rank
        _lora("lora_train_f32", 700, 771, 773, 5, 3, text=60, way="train", dtype="f32"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["dropout", "layer_norm", "dropout_add_layer_norm", "lora_linear", "lora_linear"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op == "lora_linear":
        way = rng.choice(["serve", "serve", "train"])
        widest = 4096 if dtype == "bf16" else 2048
        cols, features = _log(rng, 64, widest), _log(rng, 64, widest)
        if rng.random() < 0.7:                      # models' widths are multiples of 64
            cols, features = max(64, cols // 64 * 64), max(64, features // 64 * 64)
        rows = _log(rng, 1, 8192 if dtype == "bf16" else 2048)
        return _lora(None, rows, cols, features, rng.choice([4, 8, 16, 16, 32, 64, rng.randint(1, 64)]), _log(rng, 1, 32),
                     text=rng.choice([1, _log(rng, 1, 512)]), way=way, dtype=dtype, bias=rng.random() < 0.8)
    cols = _log(rng, 16, 4096)
    if rng.random() < 0.7:
        cols = max(16, cols // 16 * 16)
    rows = _log(rng, 1, min(16384, MOST_ELEMENTS // cols))
    way = rng.choice(["train", "train", "forward"])
    weights = rng.choice(["same", "f32"])
    p = rng.choice([0.1, 0.1, 0.0, 0.5, rng.uniform(0.01, 0.9)])
    offset = rng.choice([0, rng.randint(1, 100), rng.randint(1 << 32, 1 << 40)])
    if op == "dropout":
        return _dropout(None, rows, cols, way, dtype, p or 0.1, offset)
    if op == "layer_norm":
        return _norm(None, rows, cols, way, dtype, weights)
    return _join(None, rows, cols, way, dtype, weights, p, offset)


def _row_adapters(case, seed):
    """The adapter of every row, -1 for none: requests of ragged lengths."""
    r = np.random.RandomState(seed % (1 << 31))
    rows, text = case["rows"], case["text"]
    out, at = np.empty(rows, np.int32), 0
    while at < rows:
        n = 1 if text == 1 else int(r.randint(max(1, text // 2), text + text // 2 + 1))
        out[at:at + n] = -1 if r.rand() < 1 / 16 else r.randint(case["adapters"])
        at += n
    return out


def prepare(case, seed):
    dev, dtype = "cuda", DTYPES[case["dtype"]]
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def normal(*shape, scale=1.0, mean=0.0, dt=dtype):
        return (torch.randn(*shape, generator=g, device=dev) * scale + mean).to(dt)

    rows, cols = case["rows"], case["cols"]
    train = case["way"] == "train"
    s = {"case": case}
    if case["op"] == "lora_linear":
        n, r, f = case["adapters"], case["rank"], case["features"]
        s["x"] = normal(rows, cols).requires_grad_(train)
        s["weight"] = normal(f, cols, scale=cols ** -0.5)
        s["bias"] = normal(f, scale=0.1) if case["bias"] else None
        s["lora_a"] = normal(n, r, cols, scale=cols ** -0.5).requires_grad_(train)
        s["lora_b"] = normal(n, f, r, scale=0.4 * r ** -0.5).requires_grad_(train)
        s["scaling"] = torch.rand(n, generator=g, device=dev) * 1.5 + 0.5
        s["ids"] = torch.from_numpy(_row_adapters(case, seed)).to(dev)
        s["dy"] = normal(rows, f)
        return s
    s["x"] = normal(rows, cols).requires_grad_(train)
    s["dy"] = normal(rows, cols)
    if case["op"] != "layer_norm":
        s["seed"] = torch.randint(-(1 << 62), 1 << 62, (1,), generator=g, device=dev)
    if case["op"] != "dropout":
        wt = torch.float32 if case["weights"] == "f32" else dtype
        s["weight"] = normal(cols, scale=0.2, mean=1.0, dt=wt).requires_grad_(train)
        s["bias"] = normal(cols, scale=0.2, dt=wt).requires_grad_(train)
    if case["op"] == "dropout_add_layer_norm":
        s["residual"] = normal(rows, cols).requires_grad_(train)
    return s


# ------------------------------------------------------------------------------------------------ the package's operators
def _run_own(s):
    from turbodeberta_b200.ops.dropout import dropout
    from turbodeberta_b200.ops.layer_norm import dropout_add_layer_norm, layer_norm
    from turbodeberta_b200.ops.lora import lora_linear
    c = s["case"]
    if c["op"] == "dropout":
        y, leaves = dropout(s["x"], c["p"], s["seed"], c["offset"]), ("x",)
    elif c["op"] == "layer_norm":
        y, leaves = layer_norm(s["x"], s["weight"], s["bias"], EPS), ("x", "weight", "bias")
    elif c["op"] == "dropout_add_layer_norm":
        y = dropout_add_layer_norm(s["x"], s["residual"], s["weight"], s["bias"], EPS, c["p"], s["seed"], c["offset"])
        leaves = ("x", "residual", "weight", "bias")
    else:
        y = lora_linear(s["x"], s["weight"], s["bias"], s["lora_a"], s["lora_b"], s["scaling"], s["ids"])
        leaves = ("x", "lora_a", "lora_b")
    if c["way"] != "train":
        return {"y": y}
    grads = torch.autograd.grad(y, [s[k] for k in leaves], s["dy"])
    return {"y": y.detach(), **{"d" + k: g for k, g in zip(leaves, grads)}}


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_stays(shape, p, seed, offset):
    """The mask, in 64-bit whole numbers that hold 32-bit words."""
    low = 0xFFFFFFFF
    n = shape[0] * shape[1]
    group = torch.arange((n + 7) // 8, device=seed.device)
    c0, c1 = group & low, group >> 32
    c2, c3 = torch.full_like(group, offset & low), torch.full_like(group, (offset >> 32) & low)
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):                             # the rounds of the generator
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57     # modulo 2^64
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack([c0, c1, c2, c3], 1)
    numbers = torch.stack([words & 0xFFFF, words >> 16], 2).reshape(-1)[:n]
    return (numbers >= _dropped(p)).view(shape)


def _dropped(p):
    return int(math.floor(p * 65536 + 0.5))


def _plain_drop(x, stays, p):
    return torch.where(stays, x * (65536 / (65536 - _dropped(p))), 0.0)


@torch.no_grad()
def _run_plain(s):
    c = s["case"]
    train = c["way"] == "train"
    x, dy = s["x"].float(), s["dy"].float()
    to = s["x"].dtype
    if c["op"] == "dropout":
        stays = _plain_stays(x.shape, c["p"], s["seed"], c["offset"])
        y = _plain_drop(x, stays, c["p"]).to(to)
        return {"y": y, "dx": _plain_drop(dy, stays, c["p"]).to(to)} if train else {"y": y}
    if c["op"] == "lora_linear":
        return _plain_lora(s, x, dy, to, train)
    w, b = s["weight"].float(), s["bias"].float()
    stays = None
    if c["op"] == "dropout_add_layer_norm":
        if c["p"] > 0:
            stays = _plain_stays(x.shape, c["p"], s["seed"], c["offset"])
            x = _plain_drop(x, stays, c["p"])
        x = x + s["residual"].float()
    d = x - x.mean(1, keepdim=True)
    inv = torch.rsqrt((d * d).mean(1, keepdim=True) + EPS)
    hat = d * inv
    y = (hat * w + b).to(to)
    if not train:
        return {"y": y}
    g = dy * w
    dx = (g - g.mean(1, keepdim=True) - hat * (g * hat).mean(1, keepdim=True)) * inv
    out = {"y": y, "dx": dx if stays is None else _plain_drop(dx, stays, c["p"]), "dweight": (dy * hat).sum(0), "dbias": dy.sum(0)}
    if c["op"] == "dropout_add_layer_norm":
        out["dresidual"] = dx.to(to)
    out["dx"] = out["dx"].to(to)
    out["dweight"], out["dbias"] = out["dweight"].to(s["weight"].dtype), out["dbias"].to(s["weight"].dtype)
    return out


def _plain_lora(s, x, dy, to, train):
    """Every row against every adapter, with zeros where the adapter is not the row's."""
    c = s["case"]
    n, r = c["adapters"], c["rank"]
    w, a, b = s["weight"].float(), s["lora_a"].float(), s["lora_b"].float()
    share = (s["ids"][:, None] == torch.arange(n, device=x.device)).float() * s["scaling"]          # [rows, n]
    share = share.repeat_interleave(r, 1)
    a2, b2 = a.reshape(n * r, -1), b.transpose(1, 2).reshape(n * r, -1)
    h = (x @ a2.t()) * share
    y = x @ w.t() + h @ b2
    if s["bias"] is not None:
        y = y + s["bias"].float()
    y = y.to(to)
    if not train:
        return {"y": y}
    u = (dy @ b2.t()) * share
    return {"y": y, "dx": (dy @ w + u @ a2).to(to), "dlora_a": (u.t() @ x).view_as(a).to(to),
            "dlora_b": (h.t() @ dy).view(n, r, -1).transpose(1, 2).contiguous().to(to)}


def run(s):
    return _run_own(s) if own else _run_plain(s)


# ------------------------------------------------------------------------------------------------ cost and the exact result
def work(case):
    rows, cols = case["rows"], case["cols"]
    e = 2 if case["dtype"] == "bf16" else 4
    train = case["way"] == "train"
    if case["op"] == "lora_linear":
        f, n, r = case["features"], min(case["adapters"], rows), case["rank"]
        shared, pair = f * cols * e, n * r * (cols + f) * e
        flops = 2 * rows * f * cols + 2 * rows * r * (cols + f)
        moved = rows * (cols + f) * e + shared + pair
        if train:
            flops += 2 * rows * f * cols + 4 * rows * r * (cols + f)
            moved += rows * (cols + f) * e + pair          # dy in, dx out, the adapters' gradients out
        return {"bytes": moved, "flops": flops}
    n = rows * cols
    if case["op"] == "dropout":
        return {"bytes": n * e * (4 if train else 2), "flops": n * (2 if train else 1)}
    we = 4 if case["weights"] == "f32" else e
    joined = case["op"] == "dropout_add_layer_norm"
    rowlike = (3 if joined else 2) + ((3 if joined else 2) if train else 0)      # x, residual, y; dy, dx, dresidual
    return {"bytes": n * e * rowlike + cols * we * (4 if train else 2), "flops": n * (8 + (14 if train else 0))}


def _exact_stays(shape, p, seed, offset):
    n = int(np.prod(shape))
    m = np.uint64(0xFFFFFFFF)
    sh = np.uint64(32)
    ctr = np.zeros((4, -(-n // 8)), np.uint64)
    index = np.arange(ctr.shape[1], dtype=np.uint64)
    ctr[0], ctr[1] = index & m, index >> sh
    ctr[2], ctr[3] = np.uint64(offset & 0xFFFFFFFF), np.uint64(offset >> 32 & 0xFFFFFFFF)
    key = [seed & 0xFFFFFFFF, seed >> 32 & 0xFFFFFFFF]
    for _ in range(10):
        p0, p1 = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
        ctr = np.stack([(p1 >> sh) ^ ctr[1] ^ np.uint64(key[0]), p1 & m, (p0 >> sh) ^ ctr[3] ^ np.uint64(key[1]), p0 & m])
        key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    halves = np.ascontiguousarray(ctr.T.astype("<u4")).view("<u2").reshape(-1)[:n].reshape(shape)
    return torch.from_numpy(halves >= np.uint32(int(math.floor(p * 65536 + 0.5))))


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    train = case["way"] == "train"
    d = {k: v.detach().double() for k, v in s.items() if torch.is_tensor(v) and v.is_floating_point()}
    x, dy = d["x"], d["dy"]
    if case["op"] == "lora_linear":
        y = x @ d["weight"].T
        if "bias" in d:
            y += d["bias"]
        dx, da, db = (dy @ d["weight"], torch.zeros_like(d["lora_a"]), torch.zeros_like(d["lora_b"])) if train else (None,) * 3
        for i in range(case["adapters"]):
            at = (s["ids"] == i).nonzero()[:, 0]
            if not len(at):
                continue
            a, b, k = d["lora_a"][i], d["lora_b"][i], d["scaling"][i]
            h = k * (x[at] @ a.T)
            y[at] += h @ b.T
            if train:
                u = k * (dy[at] @ b)
                dx[at] += u @ a
                da[i] = u.T @ x[at]
                db[i] = dy[at].T @ h
        return {"y": y, "dx": dx, "dlora_a": da, "dlora_b": db} if train else {"y": y}
    if case["op"] != "layer_norm":
        stays = _exact_stays(tuple(x.shape), case["p"], int(s["seed"][0]), case["offset"]).to(x.device)
        k = 65536 / int(65536 - math.floor(case["p"] * 65536 + 0.5))
        x = x.masked_fill(~stays, 0) * k
    if case["op"] == "dropout":
        return {"y": x, "dx": dy.masked_fill(~stays, 0) * k} if train else {"y": x}
    if case["op"] == "dropout_add_layer_norm":
        x = x + d["residual"]
    mean, var = x.mean(1, keepdim=True), x.var(1, unbiased=False, keepdim=True)
    hat = (x - mean) / (var + EPS).sqrt()
    out = {"y": hat * d["weight"] + d["bias"]}
    if train:
        g = dy * d["weight"]
        dz = (g - g.mean(1, keepdim=True) - hat * (g * hat).mean(1, keepdim=True)) / (var + EPS).sqrt()
        out |= {"dx": dz, "dweight": (dy * hat).sum(0), "dbias": dy.sum(0)}
        if case["op"] == "dropout_add_layer_norm":
            out["dresidual"] = dz
            out["dx"] = dz.masked_fill(~stays, 0) * k
    return out
