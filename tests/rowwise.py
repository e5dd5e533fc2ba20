"""Layer norm, ReLU and dropout in 64 bits, as the formulas say, and how far fp32 kernels may be from them.

U = 2^-24 is a rounding to fp32, at most.  A sum over a row's columns has at most 16 + 5 + 20 of them behind each term
(a thread's own 16 elements, 5 exchanges in a warp, up to 17 warps), so it is off by at most 41 U times the sum of the
absolute values.
"""
import numpy as np
import torch

U = 2.0 ** -24
MASK32 = np.uint64(0xFFFFFFFF)


def philox4x32(counter, key, rounds=10):
    """Philox4x32 of counters [n, 4] and a key of two 32-bit words, in numpy."""
    c = [counter[:, k].astype(np.uint64) for k in range(4)]
    k0, k1 = np.uint64(key[0]), np.uint64(key[1])
    for _ in range(rounds):
        a, b = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(b >> np.uint64(32)) ^ c[1] ^ k0, b & MASK32, (a >> np.uint64(32)) ^ c[3] ^ k1, a & MASK32]
        k0, k1 = (k0 + np.uint64(0x9E3779B9)) & MASK32, (k1 + np.uint64(0xBB67AE85)) & MASK32
    return np.stack(c, 1)


def kept(rows, cols, p, seed, offset=0, row0=0):
    """The mask [rows, cols] as truth values, from its definition."""
    if p == 0:
        return np.ones((rows, cols), dtype=bool)
    first = row0 * cols
    block = np.arange(first // 4, (first + rows * cols + 3) // 4, dtype=np.uint64)
    off = np.full_like(block, offset)
    words = philox4x32(np.stack((block & MASK32, block >> np.uint64(32), off & MASK32, off >> np.uint64(32)), 1),
                       (seed & 0xFFFFFFFF, seed >> 32 & 0xFFFFFFFF))
    return (words.reshape(-1)[first % 4:][: rows * cols] >= int(p * 2.0 ** 32)).reshape(rows, cols)


def forward(x, w, b, eps, relu, p, keep):
    """y, mean, rstd in 64 bits, and the bound of |y - kernel's y| for results in x's type."""
    t = x.dtype
    x = x.double()
    cols = x.shape[1]
    w = torch.ones(cols, dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros(cols, dtype=torch.float64, device=x.device) if b is None else b.double()
    mean = x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt((x - mean).square().mean(1, keepdim=True) + eps)
    h = (x - mean) * rstd
    z = h * w + b
    # h: the centre is off by 42 U deviations (two sums, their differences), 1 / deviation by 24 U of itself, three more
    # roundings; z, the scale (rounded) and the product with it: 4 more
    off = 48 * U * (w.abs() * (1 + h.abs()) + b.abs())
    scale = 1.0 / (1.0 - p)
    y = torch.where(keep, (z.clamp(min=0) if relu else z) * scale, 0.0)
    off = torch.where(keep, off * scale, 0.0)
    return y, mean[:, 0], rstd[:, 0], off + rounding(y, off, t)


def rounding(v, off, t):
    """One rounding to type t of a value that is v +- off: half a step, or half the smallest number's spacing."""
    if t == torch.float32:
        return torch.zeros_like(v)              # counted among the others
    info = torch.finfo(t)
    return (v.abs() + off) * (info.eps / 2) + info.smallest_normal * info.eps / 2


def backward(dy, x, stats, w, b, relu, p, keep):
    """dx, dweight, dbias in 64 bits from the stats as stored, and the bounds of what a kernel may be off."""
    t = x.dtype
    dy, x = dy.double(), x.double()
    rows, cols = x.shape
    w = torch.ones(cols, dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros(cols, dtype=torch.float64, device=x.device) if b is None else b.double()
    mean, rstd = stats[:, :1].double(), stats[:, 1:].double()
    h = (x - mean) * rstd
    open_ = keep & ~(h * w + b <= 0) if relu else keep
    dz = torch.where(open_, dy * (1.0 / (1.0 - p)), 0.0)
    g = dz * w
    m1, m2 = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    dx = rstd * (g - m1 - h * m2)
    # g: 3 roundings, h: 2; the means 41 of a sum and up to 6 before it; 4 at the end
    off = 56 * U * rstd * (g.abs() + g.abs().mean(1, keepdim=True) + h.abs() * (g * h).abs().mean(1, keepdim=True))
    # a column: a thread's rows in turn (fewer than 512 in these tests), up to 128 groups of a thread block, the blocks by
    # 32nds (up to 148 in turn) and 5 exchanges of those, and 5 before the sum
    deep = min(rows, 512) + 128 + 148 + 5 + 5
    return {"dx": (dx, off + rounding(dx, off, t)), "dweight": ((dz * h).sum(0), deep * U * (dz * h).abs().sum(0)),
            "dbias": (dz.sum(0), deep * U * dz.abs().sum(0))}


def check(what, got, want, bound):
    got = got.double()
    assert got.shape == want.shape, what
    # 1e-44: results that fp32 cannot hold normalised
    bad = ~((got - want).abs() <= bound + 1e-44)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got - want).abs() / (bound + 1e-44)).nan_to_num(nan=1e30).max()):.2f} times the bound"
