"""The row-wise operators of a GCN layer that is trained, as measurable cases: layer norm, ReLU and dropout between one
sparse product and the next transform, and their gradients.

A case is a dict of plain values.  `op` says what one pass computes, on [rows, cols] features of type `dtype`:

    norm            y = dropout(relu(layer_norm(x) * weight + bias)), and with `train` the rows' mean and 1 / deviation
    norm_backward   from dy, x and those two: dx, dweight, dbias
    dropout         y = dropout(relu(x))
    dropout_backward  from dy (and x, where there is a relu): dx

`relu` and `p` > 0 say whether the activation and the dropout are there.  The mask is made from a counter, forward and
backward: element i = (row0 + row) * cols + col is kept if word i % 4 of Philox4x32-10 (Salmon et al., "Parallel random
numbers: as easy as 1, 2, 3", 2011) with the 64-bit counters i // 4 and `offset` and the key `seed` is at least
floor(p * 2^32).  `row0` is where a row block of a sharded graph begins.  `pad` > 0: the rows are a column slice of a matrix
that is that much wider.

Sizes are those of the benchmark configurations and of the tests (2 048 to 2 400 000 nodes, widths of 16 to 128), and
generic ones for wide rows and short calls.
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
EPS = 1e-5


def listed():
    f32, b16, f16 = "float32", "bfloat16", "float16"
    return [
        # The layer's tail on a graph of a few thousand nodes, the narrowest width: launch and latency.
        dict(name="norm_tiny", op="norm", rows=2_048, cols=16, dtype=f32, relu=True, p=0.5, train=True, row0=0, pad=0),
        # Inference on a citation-sized graph, a width that fills no power of two.
        dict(name="norm_infer_small", op="norm", rows=16_384, cols=60, dtype=f32, relu=True, p=0.0, train=False, row0=0, pad=0),
        # Rows that are not 16-byte aligned.
        dict(name="norm_odd", op="norm", rows=500_000, cols=61, dtype=f32, relu=True, p=0.5, train=True, row0=0, pad=0),
        # Full-batch training on millions of nodes at the full width: bound by HBM.
        dict(name="norm_large", op="norm", rows=2_400_000, cols=128, dtype=f32, relu=True, p=0.5, train=True, row0=0, pad=0),
        # Wide rows in 16 bits, no activation, no dropout: a transformer block's norm.
        dict(name="norm_wide", op="norm", rows=16_384, cols=4_096, dtype=b16, relu=False, p=0.0, train=True, row0=0, pad=0),
        # The same four of the backward pass.
        dict(name="norm_backward_tiny", op="norm_backward", rows=2_048, cols=16, dtype=f32, relu=True, p=0.5, train=True, row0=0, pad=0),
        dict(name="norm_backward_odd", op="norm_backward", rows=500_000, cols=61, dtype=f32, relu=True, p=0.5, train=True, row0=0, pad=0),
        dict(name="norm_backward_large", op="norm_backward", rows=2_400_000, cols=128, dtype=f32, relu=True, p=0.5, train=True, row0=0, pad=0),
        dict(name="norm_backward_wide", op="norm_backward", rows=16_384, cols=4_096, dtype=b16, relu=False, p=0.0, train=True, row0=0, pad=0),
        # Dropout of a small graph's features behind a product whose ReLU is fused already.
        dict(name="dropout_small", op="dropout", rows=16_384, cols=60, dtype=f32, relu=False, p=0.5, train=True, row0=0, pad=0),
        # ReLU and dropout over a large graph: bound by HBM.
        dict(name="dropout_large", op="dropout", rows=2_400_000, cols=64, dtype=f32, relu=True, p=0.2, train=True, row0=0, pad=0),
        # Their gradient in 16 bits on a row block of a sharded graph, columns of a wider matrix.
        dict(name="dropout_backward_half", op="dropout_backward", rows=1_000_000, cols=100, dtype=f16, relu=True, p=0.5, train=True,
             row0=1_000_000, pad=28),
    ]


def _between(rng, lo, hi):
    """An integer of [lo, hi], spread over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "norm_backward", "norm_backward", "dropout", "dropout_backward"])
    kind = rng.random()
    if kind < 0.5:                 # a graph's features: as often a multiple of 4 as any width
        cols = 4 * rng.randint(4, 32) if rng.random() < 0.5 else rng.randint(16, 128)
        rows = _between(rng, 2_048, 2_400_000)
    elif kind < 0.8:               # wide rows
        cols = _between(rng, 129, 8_192)
        rows = _between(rng, 16, min(65_536, 134_217_728 // cols))
    else:                          # anything, from one row and one column on
        cols = _between(rng, 1, 2_000)
        rows = _between(rng, 1, 100_000)
    dtype = rng.choice(["float32", "float32", "float32", "bfloat16", "float16"])
    p = rng.choice([0.0, 0.1, 0.5, round(rng.uniform(0.05, 0.9), 3)])
    if op.startswith("dropout") and p == 0.0:
        p = 0.5
    return dict(op=op, rows=rows, cols=cols, dtype=dtype, relu=rng.random() < 0.6, p=p, train=rng.random() < 0.7,
                row0=rng.choice([0, 0, rng.randint(1, 1 << 33)]), pad=rng.choice([0, 0, rng.randint(1, 64)]))


def prepare(case, seed):
    rows, cols, t = case["rows"], case["cols"], DTYPES[case["dtype"]]
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def buffer():
        return torch.empty((rows, cols + case["pad"]), dtype=t, device="cuda")[:, :cols]

    def normal(shape, scale, mean):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale + mean

    # features behind a sparse product: every row has a size and a mean of its own
    x = buffer()
    x.copy_(normal((rows, cols), torch.exp(normal((rows, 1), 0.5, 0.0)), normal((rows, 1), 0.5, 0.0)))
    s = dict(case)
    s.update(x=x, seed=seed * 2_654_435_761 % (1 << 62), offset=seed % 1_000)
    if case["op"].startswith("norm"):
        s.update(weight=normal((cols,), 0.1, 1.0), bias=normal((cols,), 0.1, 0.0))
    if case["op"] == "norm":
        s.update(y=buffer(), stats=torch.empty((rows, 2), device="cuda") if case["train"] else None)
    if case["op"] == "norm_backward":
        # what the forward pass has kept
        mean = x.double().mean(1)
        var = x.double().sub_(mean[:, None]).square_().mean(1)
        s["stats"] = torch.stack((mean, 1.0 / torch.sqrt(var + EPS)), 1).float()
        s.update(dweight=torch.empty(cols, device="cuda"), dbias=torch.empty(cols, device="cuda"))
    if case["op"].endswith("backward"):
        s["dy"] = buffer()
        s["dy"].copy_(normal((rows, cols), 1.0, 0.0))
        s["dx"] = buffer()
    if case["op"] == "dropout":
        s["y"] = buffer()
    return s


# ---- the plain forms --------------------------------------------------------------------------------------------------

LOW = 0xFFFFFFFF


def _kept(s):
    """The mask as truth values [rows, cols]."""
    rows, cols = s["rows"], s["cols"]
    first = s["row0"] * cols
    b0, b1 = first // 4, (first + rows * cols + 3) // 4
    block = torch.arange(b0, b1, dtype=torch.int64, device="cuda")
    offset = torch.full_like(block, s["offset"])
    c0, c1, c2, c3 = block & LOW, block >> 32, offset & LOW, offset >> 32
    k0, k1 = s["seed"] & LOW, s["seed"] >> 32
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57          # their 64 bits, whatever the sign
        c0, c1, c2, c3 = ((b >> 32) & LOW) ^ c1 ^ k0, b & LOW, ((a >> 32) & LOW) ^ c3 ^ k1, a & LOW
        k0, k1 = (k0 + 0x9E3779B9) & LOW, (k1 + 0xBB67AE85) & LOW
    words = torch.stack((c0, c1, c2, c3), 1).reshape(-1)[first - 4 * b0:][: rows * cols]
    return (words >= math.floor(s["p"] * 2.0 ** 32)).reshape(rows, cols)


def _plain_norm(s):
    x = s["x"].float()
    mean = x.mean(1, keepdim=True)
    d = x - mean
    rstd = 1.0 / torch.sqrt((d * d).mean(1, keepdim=True) + EPS)
    y = d * rstd * s["weight"] + s["bias"]
    if s["relu"]:
        y = torch.where(y < 0, 0.0, y)
    if s["p"] > 0:
        y = torch.where(_kept(s), y * (1.0 / (1.0 - s["p"])), 0.0)
    y = y.to(s["x"].dtype)
    return {"y": y, "stats": torch.cat((mean, rstd), 1)} if s["train"] else {"y": y}


def _plain_norm_backward(s):
    mean, rstd = s["stats"][:, :1], s["stats"][:, 1:]
    dz = s["dy"].float()
    if s["p"] > 0:
        dz = torch.where(_kept(s), dz * (1.0 / (1.0 - s["p"])), 0.0)
    if s["relu"]:
        # next to zero the sign needs 64 bits
        z = (s["x"].double() - mean.double()) * rstd.double() * s["weight"].double() + s["bias"].double()
        dz = torch.where(z <= 0, 0.0, dz)
    xhat = (s["x"].float() - mean) * rstd
    g = dz * s["weight"]
    dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    # sums over all rows: 64 bits
    return {"dx": dx.to(s["x"].dtype), "dweight": (dz * xhat).sum(0, dtype=torch.float64).float(), "dbias": dz.sum(0, dtype=torch.float64).float()}


def _plain_dropout(s, v):
    v = torch.where(_kept(s), v.float() * (1.0 / (1.0 - s["p"])), 0.0)
    if s["relu"]:
        v = torch.where(s["x"] <= 0, 0.0, v)
    return v.to(s["x"].dtype)


def run(s):
    op = s["op"]
    if own:
        return _own(s)
    if op == "norm":
        return _plain_norm(s)
    if op == "norm_backward":
        return _plain_norm_backward(s)
    return {"y": _plain_dropout(s, s["x"])} if op == "dropout" else {"dx": _plain_dropout(s, s["dy"])}


def _own(s):
    """The framework's calls."""
    op = s["op"]
    norm, dropout = _framework()
    mask = dict(p=s["p"], seed=s["seed"], offset=s["offset"], row0=s["row0"])
    if op == "norm":
        y = norm.layer_norm(s["x"], s["weight"], s["bias"], EPS, relu=s["relu"], out=s["y"], stats=s["stats"], **mask)
        return {"y": y, "stats": s["stats"]} if s["train"] else {"y": y}
    if op == "norm_backward":
        dx, dweight, dbias = norm.layer_norm_backward(s["dy"], s["x"], s["stats"], s["weight"], s["bias"], relu=s["relu"], dx=s["dx"],
                                                      dweight=s["dweight"], dbias=s["dbias"], **mask)
        return {"dx": dx, "dweight": dweight, "dbias": dbias}
    if op == "dropout":
        return {"y": dropout.dropout(s["x"], relu=s["relu"], out=s["y"], **mask)}
    return {"dx": dropout.dropout_backward(s["dy"], x=s["x"] if s["relu"] else None, relu=s["relu"], out=s["dx"], **mask)}


_modules = None


def _framework():
    global _modules
    if _modules is None:
        import os
        import sys
        sys.path.insert(0, os.path.join(os.getcwd(), "iccad-accel-gcn_b200"))
        from accelgcn import dropout, norm
        _modules = norm, dropout
    return _modules


def work(case):
    n, size = case["rows"] * case["cols"], DTYPES[case["dtype"]].itemsize
    if case["op"] == "norm":
        return {"bytes": 2 * n * size + 8 * case["cols"] + (8 * case["rows"] if case["train"] else 0), "flops": 8 * n}
    if case["op"] == "norm_backward":
        return {"bytes": 3 * n * size + 16 * case["cols"] + 8 * case["rows"], "flops": 15 * n}
    tensors = 3 if case["op"] == "dropout_backward" and case["relu"] else 2
    return {"bytes": tensors * n * size, "flops": n}


# ---- the definitions in 64 bits, written apart ------------------------------------------------------------------------

def _times(c, m):
    """High and low 32 bits of c * m (c in int64 holding 32 bits), by halves of 16 bits."""
    low, high = (c & 0xFFFF) * m, (c >> 16) * m          # 48 bits each
    middle = (low >> 16) + (high & 0xFFFFFFFF)
    return ((high >> 32) << 16) + (middle >> 16) & 0xFFFFFFFF, ((middle & 0xFFFF) << 16) | (low & 0xFFFF)


def _exact_factor(case, seed, offset):
    """1 / (1 - p) where an element is kept, else 0, in 64 bits."""
    rows, cols, p = case["rows"], case["cols"], case["p"]
    i = torch.arange(rows * cols, dtype=torch.int64, device="cuda") + case["row0"] * cols
    first = int(i[0]) // 4
    block = torch.arange(first, int(i[-1]) // 4 + 1, dtype=torch.int64, device="cuda")
    words = [block % (1 << 32), block // (1 << 32), torch.full_like(block, offset % (1 << 32)), torch.full_like(block, offset // (1 << 32))]
    for r in range(10):
        keys = [(seed % (1 << 32) + r * 0x9E3779B9) % (1 << 32), (seed // (1 << 32) + r * 0xBB67AE85) % (1 << 32)]
        h0, l0 = _times(words[0], 0xD2511F53)
        h1, l1 = _times(words[2], 0xCD9E8D57)
        words = [h1 ^ words[1] ^ keys[0], l1, h0 ^ words[3] ^ keys[1], l0]
    word = torch.stack(words, 1).flatten()[i - 4 * first]
    return ((word.double() >= math.floor(p * 4294967296.0)).double() / (1.0 - p)).reshape(rows, cols)


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].double()
    factor = _exact_factor(case, s["seed"], s["offset"]) if case["p"] > 0 else 1.0
    if case["op"] == "dropout":
        return {"y": (x.clamp(min=0) if case["relu"] else x) * factor}
    if case["op"] == "dropout_backward":
        return {"dx": s["dy"].double() * factor * (x > 0 if case["relu"] else 1.0)}
    w, b = s["weight"].double(), s["bias"].double()
    if case["op"] == "norm":
        mean = x.sum(1) / case["cols"]
        rstd = (((x - mean[:, None]) ** 2).sum(1) / case["cols"] + EPS) ** -0.5
        z = torch.addcmul(b, (x - mean[:, None]) * rstd[:, None], w)
        y = (z.clamp(min=0) if case["relu"] else z) * factor
        return {"y": y, "stats": torch.stack((mean, rstd), 1)} if case["train"] else {"y": y}
    mean, rstd = s["stats"].double().unbind(1)
    h = (x - mean[:, None]) * rstd[:, None]
    dz = s["dy"].double() * factor
    if case["relu"]:
        dz = dz * (h * w + b > 0)
    n = case["cols"]
    # the gradient of the normalisation, whose mean and deviation depend on x
    dh = dz * w
    dx = (dh * n - dh.sum(1, keepdim=True) - h * (dh * h).sum(1, keepdim=True)) * (rstd[:, None] / n)
    return {"dx": dx, "dweight": torch.einsum("rc,rc->c", dz, h), "dbias": dz.sum(0)}
