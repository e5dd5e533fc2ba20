"""Layer norm, ReLU and dropout and their gradients on the GPU against the formulas in 64 bits (rowwise.py has the bounds)."""
import ctypes
import random

import numpy as np
import pytest
import torch

import rowwise
from conftest import require_cuda

pytestmark = pytest.mark.gpu

F32, B16, F16 = torch.float32, torch.bfloat16, torch.float16


def _features(rows, cols, t, gen, pad=0, start=0):
    """[rows, cols] inside a matrix with `start` columns before and `pad` behind; the matrix and the slice."""
    whole = torch.full((rows, start + cols + pad), float("nan"), dtype=t, device="cuda")
    x = whole[:, start:start + cols]
    scale = torch.exp(0.5 * torch.randn((rows, 1), generator=gen, device="cuda"))
    x.copy_(torch.randn((rows, cols), generator=gen, device="cuda") * scale + torch.randn((rows, 1), generator=gen, device="cuda"))
    return whole, x


def _untouched(whole, x, start):
    cols = x.shape[1]
    return bool(torch.isnan(whole[:, :start]).all()) and bool(torch.isnan(whole[:, start + cols:]).all())


def _stats(x, eps):
    mean = x.double().mean(1)
    return torch.stack((mean, 1.0 / torch.sqrt((x.double() - mean[:, None]).square().mean(1) + eps)), 1).float()


def _case(rows, cols, t, relu, p, weight, bias, pads=(0, 0, 0), starts=(0, 0, 0), row0=0, seed=987654321987, offset=3, eps=1e-5):
    """Forward and backward pass of one case against the formulas."""
    from accelgcn import dropout, norm
    require_cuda()
    gen = torch.Generator(device="cuda").manual_seed(rows * 8191 + cols)
    xw, x = _features(rows, cols, t, gen, pads[0], starts[0])
    yw, y = _features(rows, cols, t, gen, pads[1], starts[1])
    gw, dy = _features(rows, cols, t, gen, pads[2], starts[2])
    w = torch.randn(cols, generator=gen, device="cuda") if weight else None
    b = torch.randn(cols, generator=gen, device="cuda") if bias else None
    keep = torch.from_numpy(rowwise.kept(rows, cols, p, seed, offset, row0)).cuda()
    mask = dict(p=p, seed=seed, offset=offset, row0=row0)
    stats = torch.full((rows, 2), float("nan"), device="cuda")
    assert norm.layer_norm(x, w, b, eps, relu=relu, out=y, stats=stats, **mask) is y
    want, mean, rstd, bound = rowwise.forward(x, w, b, eps, relu, p, keep)
    rowwise.check("y", y, want, bound)
    assert bool((y[~keep] == 0).all()) and _untouched(yw, y, starts[1]) and _untouched(xw, x, starts[0])
    spread = (x.double() - mean[:, None]).abs().mean(1)
    rowwise.check("mean", stats[:, 0], mean, rowwise.U * (44 * spread + 2 * mean.abs()))
    rowwise.check("rstd", stats[:, 1], rstd, 24 * rowwise.U * rstd)
    # the same without the stats, into rows that sit alike (others may be summed in another order)
    assert torch.equal(norm.layer_norm(x, w, b, eps, relu=relu, out=_features(rows, cols, t, gen, pads[1], starts[1])[1], **mask), y)

    stats = _stats(x, eps)
    dxw, dx = _features(rows, cols, t, gen, pads[1], starts[1])
    _dx, dw, db = norm.layer_norm_backward(dy, x, stats, w, b, relu=relu, dx=dx, **mask)
    ref = rowwise.backward(dy, x, stats, w, b, relu, p, keep)
    rowwise.check("dx", dx, *ref["dx"])
    assert _untouched(dxw, dx, starts[1])
    assert (dw is None) == (w is None) and (db is None) == (b is None)
    for name, got in (("dweight", dw), ("dbias", db)):
        if got is not None:
            rowwise.check(name, got, *ref[name])

    if p > 0:
        act = x.double().clamp(min=0) if relu else x.double()
        v = torch.where(keep, act * (1.0 / (1.0 - p)), 0.0)
        off = 2 * rowwise.U * v.abs()                                       # the scale and the product, rounded to fp32
        rowwise.check("dropout", dropout.dropout(x, relu=relu, out=y, **mask), v, off + rowwise.rounding(v, off, t))
        v = torch.where(keep & (x > 0) if relu else keep, dy.double() * (1.0 / (1.0 - p)), 0.0)
        off = 2 * rowwise.U * v.abs()
        rowwise.check("dropout backward", dropout.dropout_backward(dy, relu=relu, x=x if relu else None, out=dx, **mask), v,
                      off + rowwise.rounding(v, off, t))
        assert _untouched(yw, y, starts[1]) and _untouched(dxw, dx, starts[1])


@pytest.mark.parametrize("t", [F32, B16, F16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 8192), (3, 2), (5, 3), (7, 4), (2, 5), (33, 7), (100, 8), (129, 16), (64, 17), (1000, 31), (257, 60),
                                       (300, 61), (513, 64), (1, 128), (1000, 100), (4099, 128), (70, 129), (65, 255), (40, 256), (31, 500),
                                       (19, 512), (9, 513), (17, 1000), (6, 1024), (11, 1025), (5, 2047), (3, 4096), (9, 8191), (2, 8192)])
def test_sizes(rows, cols, t):
    _case(rows, cols, t, relu=True, p=0.4, weight=True, bias=True)


@pytest.mark.parametrize("relu,p,weight,bias", [(False, 0.0, False, False), (False, 0.0, True, False), (False, 0.0, False, True), (True, 0.0, True, True),
                                                (False, 0.5, True, True), (True, 0.9, False, False), (True, 2.0 ** -20, True, False)])
@pytest.mark.parametrize("rows,cols,t", [(700, 60, F32), (300, 61, F32), (50, 1500, F32), (200, 128, B16), (40, 3001, F16)])
def test_options(rows, cols, t, relu, p, weight, bias):
    _case(rows, cols, t, relu, p, weight, bias)


@pytest.mark.parametrize("pads,starts", [((3, 3, 3), (0, 0, 0)), ((4, 8, 12), (0, 0, 0)), ((1, 2, 3), (0, 0, 0)), ((0, 0, 0), (1, 1, 1)), ((7, 7, 7), (1, 5, 9)),
                                         ((7, 6, 5), (1, 2, 3)), ((2, 2, 2), (3, 3, 3)), ((0, 0, 0), (2, 4, 6))])
@pytest.mark.parametrize("rows,cols,t", [(400, 60, F32), (333, 61, F32), (257, 100, B16), (111, 37, F16), (37, 1001, F32), (20, 2050, B16), (5, 8192, F32),
                                         (5, 8192, B16), (3, 8189, F32)])
def test_strides_and_alignments(rows, cols, t, pads, starts):
    _case(rows, cols, t, relu=True, p=0.3, weight=True, bias=True, pads=pads, starts=starts)


@pytest.mark.parametrize("cols,t,row0", [(61, F32, 1), (61, B16, 3), (60, F32, 12345), (7, F16, (1 << 33) + 5), (1001, F32, 1 << 40), (128, B16, (1 << 45) + 1)])
def test_row_blocks_of_a_sharded_step(cols, t, row0):
    _case(83, cols, t, relu=True, p=0.5, weight=True, bias=True, row0=row0, seed=(1 << 62) + 12345, offset=(1 << 40) + 7)


@pytest.mark.parametrize("rows,cols,t", [(300_000, 16, F32), (200_003, 61, F32), (150_000, 128, F32), (100_001, 100, B16), (20_000, 1000, F32), (3_000, 5_000, B16)])
def test_many_rows(rows, cols, t):
    _case(rows, cols, t, relu=True, p=0.5, weight=True, bias=True)


@pytest.mark.parametrize("rows,cols,t", [(1, 16, F32), (2, 4096, F32), (5, 3000, B16), (127, 16, F32), (129, 16, F32), (8192, 16, F32), (8193, 16, F32),
                                         (2048, 60, F32), (2049, 60, F32), (2048, 61, F32), (1024, 128, F32), (1025, 128, F32), (2048, 128, B16), (2049, 128, B16),
                                         (512, 255, F32), (64, 1000, F32), (65, 1000, F32), (64, 8192, B16), (65, 8191, F16), (8, 777, F32), (9, 777, F32)])
def test_few_rows_whose_columns_one_cluster_adds_up(rows, cols, t):
    _case(rows, cols, t, relu=True, p=0.25, weight=True, bias=True)


@pytest.mark.parametrize("t", [F32, B16])
def test_every_form_of_every_width(t):
    # each number of lanes and chunks that a width can take, rows on and off 16-byte boundaries
    from accelgcn import norm
    require_cuda()
    gen = torch.Generator(device="cuda").manual_seed(18)
    for cols in [*range(1, 260), *range(260, 1100, 7), *range(1100, 8193, 131), 8185, 8186, 8191, 8192]:
        x = torch.randn((9, cols + 3), generator=gen, device="cuda").to(t)[:, cols % 3:][:, :cols]
        w, b = torch.randn(cols, generator=gen, device="cuda"), torch.randn(cols, generator=gen, device="cuda")
        keep = torch.ones_like(x, dtype=torch.bool)
        want, _, _, bound = rowwise.forward(x, w, b, 1e-5, True, 0.0, keep)
        stats = torch.empty((9, 2), device="cuda")
        out = torch.empty((9, cols + 3), dtype=t, device="cuda")[:, cols % 3:][:, :cols]
        rowwise.check(f"y {cols}", norm.layer_norm(x, w, b, relu=True, stats=stats, out=out), want, bound)
        dx, dw, db = norm.layer_norm_backward(x, x, stats, w, b, relu=True, dx=out)
        ref = rowwise.backward(x, x, stats, w, b, True, 0.0, keep)
        for name, got in (("dx", dx), ("dweight", dw), ("dbias", db)):
            rowwise.check(f"{name} {cols}", got, *ref[name])


@pytest.mark.parametrize("t,shift,row0", [(F32, 0, 1), (F32, 1, 0), (F32, 3, 2), (B16, 0, 3), (B16, 5, 1), (F16, 1, (1 << 35) + 1)])
def test_large_arrays_that_begin_inside_a_block(t, shift, row0):
    # long enough for several rounds of every warp: its chunks begin inside the generator's blocks, and in front of the array
    from accelgcn import dropout, norm
    require_cuda()
    gen = torch.Generator(device="cuda").manual_seed(19)
    rows, cols, mask = 90_001, 61, dict(p=0.35, seed=21, offset=4, row0=row0)

    def make(fill=True):
        whole = torch.full((rows * cols + 16,), float("nan"), dtype=t, device="cuda")
        x = whole[shift:shift + rows * cols].view(rows, cols)
        if fill:
            x.copy_(torch.randn((rows, cols), generator=gen, device="cuda"))
        return whole, x

    (_, x), (_, dy), (whole, out) = make(), make(), make(False)
    keep = torch.from_numpy(rowwise.kept(rows, cols, 0.35, 21, 4, row0)).cuda()
    scale = 1.0 / (1.0 - 0.35)
    for got, v in ((lambda: dropout.dropout(x, relu=True, out=out, **mask), torch.where(keep, x.double().clamp(min=0) * scale, 0.0)),
                   (lambda: dropout.dropout_backward(dy, relu=True, x=x, out=out, **mask), torch.where(keep & (x > 0), dy.double() * scale, 0.0))):
        off = 2 * rowwise.U * v.abs()
        rowwise.check("dropout", got(), v, off + rowwise.rounding(v, off, t))
        assert bool(torch.isnan(whole[:shift]).all()) and bool(torch.isnan(whole[shift + rows * cols:]).all())
    want, _, _, bound = rowwise.forward(x, None, None, 1e-5, True, 0.35, keep)
    rowwise.check("y", norm.layer_norm(x, relu=True, out=out, **mask), want, bound)


def test_drawn_cases():
    rng = random.Random(20260)
    for _ in range(40):
        cols = rng.choice([rng.randint(1, 40), rng.randint(1, 200), rng.randint(1, 8192)])
        rows = rng.randint(1, max(1, min(3000, 400_000 // cols)))
        pads, starts = [tuple(rng.randint(0, 9) for _ in range(3)) if rng.random() < 0.4 else (0, 0, 0) for _ in range(2)]
        _case(rows, cols, rng.choice([F32, B16, F16]), rng.random() < 0.5, rng.choice([0.0, 0.1, 0.75]), rng.random() < 0.7, rng.random() < 0.7, pads, starts,
              row0=rng.choice([0, rng.randint(0, 1 << 34)]), seed=rng.getrandbits(63), offset=rng.getrandbits(rng.choice([5, 63])))


def test_means_far_from_zero():
    # 1e4 deviations away: what is lost is what the inputs' own spacing loses, not its square
    from accelgcn import norm
    require_cuda()
    gen = torch.Generator(device="cuda").manual_seed(5)
    for cols in (16, 128, 3001):
        x = torch.randn((200, cols), generator=gen, device="cuda") + 1e4
        x[:, 0] += 3e5                          # and one far-off value first
        keep = torch.ones_like(x, dtype=torch.bool)
        want, mean, rstd, bound = rowwise.forward(x, None, None, 1e-5, False, 0.0, keep)
        # the first mean is rounded at |mean|; differences from it are exact to U of themselves
        rowwise.check("y", norm.layer_norm(x), want, bound + 48 * rowwise.U * 2)


@pytest.mark.parametrize("cols", [1, 6, 128, 2000])
def test_constant_rows(cols):
    from accelgcn import norm
    require_cuda()
    x = torch.full((9, cols), 0.3, device="cuda")
    x[3] = 0.0
    b = torch.linspace(-1, 1, cols, device="cuda")
    stats = torch.empty((9, 2), device="cuda")
    y = norm.layer_norm(x, None, b, relu=True, stats=stats)
    # the mean is off by its rounding (2 U of 0.3) and the deviation is 1 / sqrt(eps) then
    assert float((y - b.clamp(min=0)).abs().max()) <= 4 * rowwise.U * 0.3 / 1e-5 ** 0.5
    assert torch.equal(y[3], b.clamp(min=0))
    dy = torch.ones_like(x)
    dx, _dw, db = norm.layer_norm_backward(dy, x, stats, None, b, relu=True)
    keep = torch.ones_like(x, dtype=torch.bool)
    ref = rowwise.backward(dy, x, stats, None, b, True, 0.0, keep)
    rowwise.check("dx", dx, *ref["dx"])
    rowwise.check("dbias", db, *ref["dbias"])


def test_signs_next_to_zero_are_those_of_the_formula():
    # z = h w + b where the two terms cancel to the last bits: the gradient passes where 64 bits say so
    from accelgcn import norm
    require_cuda()
    gen = torch.Generator(device="cuda").manual_seed(6)
    rows, cols = 4000, 64
    x = torch.randn((rows, cols), generator=gen, device="cuda")
    stats = _stats(x, 1e-5)
    w = torch.randn(cols, generator=gen, device="cuda")
    h = (x - stats[:, :1]) * stats[:, 1:]
    b = -(h[0] * w)
    x[::7] = x[0]                                # rows whose every z is a rounding
    stats = _stats(x, 1e-5)
    dy = torch.randn((rows, cols), generator=gen, device="cuda")
    dx, dw, db = norm.layer_norm_backward(dy, x, stats, w, b, relu=True)
    ref = rowwise.backward(dy, x, stats, w, b, True, 0.0, torch.ones_like(x, dtype=torch.bool))
    for name, got in (("dx", dx), ("dweight", dw), ("dbias", db)):
        rowwise.check(name, got, *ref[name])


@pytest.mark.parametrize("t", [F32, B16])
@pytest.mark.parametrize("cols", [24, 61, 700])
def test_nan_and_infinity_stay_where_they_are(t, cols):
    from accelgcn import dropout, norm
    require_cuda()
    gen = torch.Generator(device="cuda").manual_seed(8)
    rows, mask = 200, dict(p=0.5, seed=77, offset=1)
    keep = torch.from_numpy(rowwise.kept(rows, cols, 0.5, 77, 1)).cuda()
    _, x = _features(rows, cols, t, gen)
    bad = x.clone()
    bad[5, 3], bad[9, 1], bad[11, 2], bad[50] = float("nan"), float("inf"), float("-inf"), float("nan")
    rows_ok = torch.ones(rows, dtype=torch.bool, device="cuda")
    rows_ok[[5, 9, 11, 50]] = False
    w = torch.randn(cols, generator=gen, device="cuda")
    y, z = norm.layer_norm(x, w, None, relu=True, **mask), norm.layer_norm(bad, w, None, relu=True, **mask)
    assert torch.equal(y[rows_ok], z[rows_ok])
    assert bool(torch.isnan(z[~rows_ok][keep[~rows_ok]]).all()) and bool((z[~keep] == 0).all())
    # dropout: dropped values are 0 whatever they were, relu lets NaN and infinity through
    z = dropout.dropout(bad, relu=True, **mask)
    assert bool((z[~keep] == 0).all())
    act = torch.where(bad < 0, torch.zeros_like(bad), bad)
    assert torch.equal(torch.isnan(z), torch.isnan(act) & keep) and torch.equal(torch.isinf(z), torch.isinf(act) & keep)
    # the backward pass: dy that is dropped does not count, x that is <= 0 blocks
    dy = x.clone()
    dy[~keep] = float("nan")
    stats = _stats(x, 1e-5)
    dx, dw, _ = norm.layer_norm_backward(dy, x, stats, w, None, relu=True, **mask)
    ref = rowwise.backward(torch.nan_to_num(dy), x, stats, w, None, True, 0.5, keep)
    rowwise.check("dx", dx, *ref["dx"])
    rowwise.check("dweight", dw, *ref["dweight"])
    dx = dropout.dropout_backward(dy, relu=True, x=bad, **mask)
    assert torch.equal(torch.isnan(dx), torch.zeros_like(keep)) and bool((dx[(bad <= 0) | ~keep] == 0).all())


def test_everything_dropped_leaves_zero_gradients():
    from accelgcn import norm
    require_cuda()
    gen = torch.Generator(device="cuda").manual_seed(9)
    _, x = _features(64, 96, F32, gen)
    w, b = torch.ones(96, device="cuda"), torch.full((96,), -1e3, device="cuda")
    stats = torch.empty((64, 2), device="cuda")
    assert bool((norm.layer_norm(x, w, b, relu=True, stats=stats) == 0).all())
    for g in norm.layer_norm_backward(torch.full_like(x, float("inf")), x, stats, w, b, relu=True):
        assert bool((g == 0).all())


@pytest.mark.parametrize("rows,cols,t", [(500, 64, F32), (300, 61, F32), (40, 2000, B16)])
def test_outputs_in_place(rows, cols, t):
    from accelgcn import dropout, norm
    require_cuda()
    gen = torch.Generator(device="cuda").manual_seed(10)
    _, x = _features(rows, cols, t, gen)
    _, dy = _features(rows, cols, t, gen)
    w, b = torch.randn(cols, generator=gen, device="cuda"), torch.randn(cols, generator=gen, device="cuda")
    mask = dict(p=0.25, seed=4, offset=4)
    stats = torch.empty((rows, 2), device="cuda")
    y = norm.layer_norm(x, w, b, relu=True, stats=stats, **mask)
    v = x.clone()
    assert norm.layer_norm(v, w, b, relu=True, out=v, **mask) is v and torch.equal(v, y)
    dx, dw, db = norm.layer_norm_backward(dy, x, stats, w, b, relu=True, **mask)
    for into in (dy.clone(), x.clone()):
        a, c = (into, x) if torch.equal(into, dy) else (dy, into)
        got = norm.layer_norm_backward(a, c, stats, w, b, relu=True, dx=into, **mask)
        assert torch.equal(got[0], dx) and torch.equal(got[1], dw) and torch.equal(got[2], db)
    y = dropout.dropout(x, relu=True, **mask)
    v = x.clone()
    assert torch.equal(dropout.dropout(v, relu=True, out=v, **mask), y)
    dx = dropout.dropout_backward(dy, relu=True, x=x, **mask)
    v = dy.clone()
    assert torch.equal(dropout.dropout_backward(v, relu=True, x=x, out=v, **mask), dx)
    v = x.clone()
    assert torch.equal(dropout.dropout_backward(dy, relu=True, x=v, out=v, **mask), dx)


def test_no_rows():
    from accelgcn import dropout, norm
    require_cuda()
    x = torch.empty((0, 24), device="cuda")
    w = torch.ones(24, device="cuda")
    assert norm.layer_norm(x, w, stats=torch.empty((0, 2), device="cuda")).shape == (0, 24)
    dw, db = torch.full((24,), 5.0, device="cuda"), torch.full((24,), 5.0, device="cuda")
    dx, _, _ = norm.layer_norm_backward(x, x, torch.empty((0, 2), device="cuda"), w, w, dweight=dw, dbias=db)
    assert dx.shape == (0, 24) and bool((dw == 0).all()) and bool((db == 0).all())
    assert dropout.dropout(x, 0.5, 1).shape == (0, 24) and dropout.dropout_backward(x, 0.5, 1).shape == (0, 24)


def test_same_bits_from_run_to_run():
    from accelgcn import norm
    require_cuda()
    gen = torch.Generator(device="cuda").manual_seed(12)
    for rows, cols, t in ((100_000, 61, F32), (5_000, 1500, B16), (200_000, 16, F32)):
        _, x = _features(rows, cols, t, gen)
        _, dy = _features(rows, cols, t, gen)
        w, b, stats = torch.randn(cols, generator=gen, device="cuda"), torch.randn(cols, generator=gen, device="cuda"), _stats(x, 1e-5)
        first = norm.layer_norm_backward(dy, x, stats, w, b, relu=True, p=0.5, seed=1)
        for _ in range(3):
            for a, c in zip(first, norm.layer_norm_backward(dy, x, stats, w, b, relu=True, p=0.5, seed=1)):
                assert torch.equal(a, c)


@pytest.mark.parametrize("rows", [3000, 9000])           # one cluster, without a workspace; thread blocks of their own, with one
def test_column_sums_alone_and_left_out(rows):
    from accelgcn import _lib, norm
    require_cuda()
    gen = torch.Generator(device="cuda").manual_seed(13)
    _, x = _features(rows, 48, F32, gen)
    _, dy = _features(rows, 48, F32, gen)
    w, b, stats = torch.randn(48, generator=gen, device="cuda"), torch.randn(48, generator=gen, device="cuda"), _stats(x, 1e-5)
    dx, dw, db = norm.layer_norm_backward(dy, x, stats, w, b)
    # without a weight, the gradient that it would have had; none wanted
    got = norm.layer_norm_backward(dy, x, stats, None, b, dweight=torch.empty(48, device="cuda"))
    assert torch.equal(got[1], dw) and torch.equal(got[2], db)
    lib, dev = _lib.load(), torch.cuda.current_stream().cuda_stream
    n = ctypes.c_int64()
    _lib.check(lib.agcn_layer_norm_backward_work(rows, 48, 0, ctypes.byref(n)))
    assert (n.value > 0) == (rows == 9000)
    out = torch.empty_like(dx)
    for pw, pb in ((None, None), (torch.empty(48, device="cuda"), None), (None, torch.empty(48, device="cuda"))):
        work = torch.full((n.value // 4 + 1,), float("nan"), device="cuda")
        none = pw is None and pb is None
        _lib.check(lib.agcn_layer_norm_backward(dy.data_ptr(), 48, x.data_ptr(), 48, stats.data_ptr(), w.data_ptr(), b.data_ptr(), out.data_ptr(), 48,
                                                pw.data_ptr() if pw is not None else None, pb.data_ptr() if pb is not None else None,
                                                None if none else work.data_ptr(), 0 if none else n.value, rows, 48, 0, 0, 0.0, 0, 0, None, 0, dev))
        assert torch.equal(out, dx) and (pw is None or torch.equal(pw, dw)) and (pb is None or torch.equal(pb, db))
        assert bool(torch.isnan(work[-1]))
    if n.value:
        # a workspace that is too small is refused, and nothing is written
        out.fill_(float("nan"))
        rc = lib.agcn_layer_norm_backward(dy.data_ptr(), 48, x.data_ptr(), 48, stats.data_ptr(), w.data_ptr(), b.data_ptr(), out.data_ptr(), 48, dw.data_ptr(),
                                          db.data_ptr(), work.data_ptr(), n.value - 4, rows, 48, 0, 0, 0.0, 0, 0, None, 0, dev)
        assert rc == _lib.ERR_INVALID and b"workspace" in lib.agcn_last_error() and bool(torch.isnan(out).all())


def test_captured_steps_have_masks_of_their_own():
    from accelgcn import dropout, norm
    require_cuda()
    gen = torch.Generator(device="cuda").manual_seed(14)
    rows, cols = 3000, 60
    _, x = _features(rows, cols, F32, gen)
    _, dy = _features(rows, cols, F32, gen)
    w, b = torch.randn(cols, generator=gen, device="cuda"), torch.randn(cols, generator=gen, device="cuda")
    count = torch.zeros(1, dtype=torch.int64, device="cuda")
    stats = torch.empty((rows, 2), device="cuda")

    def step():
        mask = dict(p=0.5, seed=9, offset=100, step=count)
        h = norm.layer_norm(x, w, b, relu=True, stats=stats, **mask)
        return (h, *norm.layer_norm_backward(dy, x, stats, w, b, relu=True, **mask), dropout.dropout(x, **mask), dropout.dropout_backward(dy, **mask))

    step()
    side = torch.cuda.Stream()
    graphs = []
    for _ in range(2):                           # two graphs of the same step: workspaces of their own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs = step()
        graphs.append((g, outs))
    for k in range(3):
        count.fill_(k)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for (g, outs), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                for o in outs:
                    o.fill_(float("nan"))
                g.replay()
        torch.cuda.synchronize()
        mask = dict(p=0.5, seed=9, offset=100 + k)
        want = (norm.layer_norm(x, w, b, relu=True, **mask), *norm.layer_norm_backward(dy, x, stats, w, b, relu=True, **mask), dropout.dropout(x, **mask),
                dropout.dropout_backward(dy, **mask))
        for _, outs in graphs:
            for a, c in zip(outs, want):
                assert torch.equal(a, c)
        keep = torch.from_numpy(rowwise.kept(rows, cols, 0.5, 9, 100 + k)).cuda()
        assert torch.equal(want[4] != 0, keep & (x != 0))


def test_calls_on_another_stream():
    from accelgcn import norm
    require_cuda()
    gen = torch.Generator(device="cuda").manual_seed(15)
    _, x = _features(20_000, 100, F32, gen)
    _, dy = _features(20_000, 100, F32, gen)
    w, stats = torch.randn(100, generator=gen, device="cuda"), torch.empty((20_000, 2), device="cuda")
    y = norm.layer_norm(x, w, stats=stats)
    want = norm.layer_norm_backward(dy, x, stats, w, None)
    torch.cuda.synchronize()
    s, busy = torch.cuda.Stream(), torch.ones(1 << 26, device="cuda")
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(s):
            for _ in range(20):
                busy.mul_(1.0)                   # what is enqueued behind this is not there yet when the call returns
            late = x * 1.0
        late.record_stream(s)
        y2 = norm.layer_norm(late, w, stream=s)
        got = norm.layer_norm_backward(dy, late, stats, w, None, stream=s)
        s.synchronize()
        assert torch.equal(y2, y)
        for a, c in zip(got[:2], want[:2]):
            assert torch.equal(a, c)
        del y2, got, late


def test_calls_behind_an_event_of_another_stream():
    # launched early behind what is before them on their own stream, but not ahead of the event that the stream waits for
    from accelgcn import dropout, norm
    require_cuda()
    gen = torch.Generator(device="cuda").manual_seed(17)
    _, x = _features(5_000, 64, F32, gen)
    w, mask = torch.randn(64, generator=gen, device="cuda"), dict(p=0.5, seed=1)
    y, d = norm.layer_norm(x, w, relu=True, **mask), dropout.dropout(x, **mask)
    one, two, busy = torch.cuda.Stream(), torch.cuda.Stream(), torch.ones(1 << 26, device="cuda")
    small = torch.zeros((16, 64), device="cuda")
    late = torch.zeros_like(x)
    for _ in range(5):
        late.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(one):
            for _ in range(10):
                busy.mul_(1.0)
            late.copy_(x)
            ready = torch.cuda.Event()
            ready.record()
        with torch.cuda.stream(two):
            dropout.dropout(small, p=0.5, seed=1, out=small)        # a launch in front of the wait
            two.wait_event(ready)
            a = norm.layer_norm(late, w, relu=True, **mask)
            b = dropout.dropout(late, **mask)
        torch.cuda.synchronize()
        assert torch.equal(a, y) and torch.equal(b, d)


def test_elements_beyond_32_bits():
    from accelgcn import dropout, norm
    require_cuda()
    rows, cols = 17_000_000, 128                 # 2.2e9 elements, 4.4 GB
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    x = torch.empty((rows, cols), dtype=B16, device="cuda").normal_()
    w, b, stats = torch.randn(cols, device="cuda"), torch.randn(cols, device="cuda"), torch.empty((rows, 2), device="cuda")
    mask = dict(p=0.5, seed=3, offset=2)
    y = norm.layer_norm(x, w, b, relu=True, stats=stats, **mask)
    dx, dw, db = norm.layer_norm_backward(y, x, stats, w, b, relu=True, **mask)
    d = dropout.dropout(x, **mask)
    for r in (0, 16_777_215, rows - 100):        # the second: element 2^31 - 128 and after
        n = 100
        part = slice(r, r + n)
        keep = torch.from_numpy(rowwise.kept(n, cols, 0.5, 3, 2, r)).cuda()
        want, _, _, bound = rowwise.forward(x[part], w, b, 1e-5, True, 0.5, keep)
        rowwise.check("y", y[part], want, bound)
        rowwise.check("dx", dx[part], *rowwise.backward(y[part], x[part], stats[part], w, b, True, 0.5, keep)["dx"])
        assert torch.equal(d[part], torch.where(keep, x[part] * 2, 0))
    # the columns' sums, from the parts' (each exact to its own bound; 17 000 000 rows: 14 400 in turn per thread at most)
    dw64, db64, aw, ab = (torch.zeros(cols, dtype=torch.float64, device="cuda") for _ in range(4))
    for r in range(0, rows, 1_000_000):
        part = slice(r, min(rows, r + 1_000_000))
        h = (x[part].double() - stats[part, :1].double()) * stats[part, 1:].double()
        dz = torch.where(y[part] > 0, y[part].double() * 2, 0.0)
        dw64 += (dz * h).sum(0); db64 += dz.sum(0); aw += (dz * h).abs().sum(0); ab += dz.abs().sum(0)
    deep = 14_400 + 128 + 148 + 5 + 5
    # (an output that rounds to 0 in 16 bits though z > 0 has dy = 0 and adds nothing)
    rowwise.check("dweight", dw, dw64, deep * rowwise.U * aw)
    rowwise.check("dbias", db, db64, deep * rowwise.U * ab)


def test_gradients_are_those_of_differences():
    # directional derivatives of sum(c * y) by central differences of the kernel's own forward pass
    from accelgcn import norm
    require_cuda()
    gen = torch.Generator(device="cuda").manual_seed(16)
    rows, cols, eps, step = 60, 40, 1e-3, 2.0 ** -7
    x = torch.randn((rows, cols), generator=gen, device="cuda")
    w, b = torch.randn(cols, generator=gen, device="cuda"), torch.randn(cols, generator=gen, device="cuda")
    c = torch.randn((rows, cols), generator=gen, device="cuda")
    mask = dict(p=0.25, seed=6, offset=6)
    keep = torch.from_numpy(rowwise.kept(rows, cols, 0.25, 6, 6)).cuda()
    stats = torch.empty((rows, 2), device="cuda")
    norm.layer_norm(x, w, b, eps, stats=stats, **mask)
    dx, dw, db = norm.layer_norm_backward(c, x, stats, w, b, **mask)
    ref = rowwise.backward(c, x, stats, w, b, False, 0.25, keep)

    def value(x, w, b):
        y = norm.layer_norm(x, w, b, eps, **mask).double()
        want, _, _, bound = rowwise.forward(x, w, b, eps, False, 0.25, keep)
        return float((c * y).sum()), float((c * want).sum()), float((c.abs() * bound).sum())

    for which, grad, name in ((0, dx, "dx"), (1, dw, "dweight"), (2, db, "dbias")):
        at = [x, w, b]
        v = torch.randn(at[which].shape, generator=gen, device="cuda")
        # steps that fp32 holds exactly next to the point are what the difference is divided by
        up, down = at[which] + step * v, at[which] - step * v
        moved = (up.double() - down.double()) / 2
        plus, minus = (value(*(u if k == which else a for k, a in enumerate(at))) for u in (up, down))
        mid = (up.double() + down.double()) / 2
        slope = float((grad.double() * moved).sum())
        # the kernel's difference is off by its bound; the quotient of exact values by the curvature, taken from 64 bits, and by
        # the point in the middle not being the point (a rounding)
        exact_slope = float((ref[name][0] * moved).sum())
        curved = abs((plus[1] - minus[1]) / 2 - exact_slope)
        tol = (plus[2] + minus[2]) / 2 + curved + float((ref[name][1] * moved.abs()).sum())
        assert abs((plus[0] - minus[0]) / 2 - slope) <= tol, (name, slope, tol)
        assert curved <= 0.02 * abs(exact_slope) + 0.02 and float((mid - at[which].double()).abs().max()) < 1e-6


def test_tail_of_gcn_layers_in_training():
    # two layers as they are trained: transform, product, norm + ReLU + dropout; transform, product, dropout; and back.  Every
    # step is checked against the formula on what it was given.
    from accelgcn import degree_sort, dropout, gemm, norm, partition, spmm, synth
    import scipy.sparse as sp
    dev = require_cuda()
    g = synth.make_config(1, dev, 0.25)
    _, ip, ix, v = degree_sort.degree_sort_device(g.indptr, g.indices, g.vals)
    n = g.n
    a = sp.csr_matrix((v.cpu().numpy().astype(np.float64), ix.cpu().numpy(), ip.cpu().numpy()), shape=(n, n))
    plan = spmm.SpmmPlan(partition.block_level_partition_device(ip), ix, n, n)
    x, w1, w2 = synth.features(n, 128, 3, dev), synth.glorot(128, 128, 5, 8, dev), synth.glorot(128, 128, 5, 9, dev)
    weight = 1 + 0.1 * synth.features(1, 128, 4, dev)[0].contiguous()
    bias = 0.1 * synth.features(1, 128, 5, dev)[0].contiguous()

    def product(z):
        y = torch.empty_like(z)
        plan.run(ix, v, z, y)
        want = torch.from_numpy(a @ z.double().cpu().numpy()).to(dev)
        assert bool(((y - want).abs() <= 1e-4 * want.abs() + 1e-5).all())
        return y

    def transform(h, w):
        z = gemm.gemm_tf32(h, w)
        assert bool(((z - h.double() @ w.double()).abs() <= 2e-3 * (h.double().abs() @ w.double().abs()) + 1e-6).all())
        return z

    one, two = dict(p=0.5, seed=11, offset=0), dict(p=0.2, seed=11, offset=1)
    keep1, keep2 = (torch.from_numpy(rowwise.kept(n, 128, m["p"], 11, m["offset"])).to(dev) for m in (one, two))
    y1 = product(transform(x, w1))
    stats = torch.empty((n, 2), device=dev)
    h1 = norm.layer_norm(y1, weight, bias, relu=True, stats=stats, **one)
    want, _, _, bound = rowwise.forward(y1, weight, bias, 1e-5, True, 0.5, keep1)
    rowwise.check("h1", h1, want, bound)
    y2 = product(transform(h1, w2))
    o = dropout.dropout(y2, relu=True, **two)
    assert torch.equal(o != 0, keep2 & (y2 > 0))

    d_o = synth.features(n, 128, 6, dev)
    dy2 = dropout.dropout_backward(d_o, relu=True, x=y2, **two)
    assert torch.equal(dy2 != 0, keep2 & (y2 > 0) & (d_o != 0))
    dz2 = product(dy2)                            # A is symmetric
    dh1 = transform(dz2, w2.t().contiguous())
    dy1, dweight, dbias = norm.layer_norm_backward(dh1, y1, stats, weight, bias, relu=True, **one)
    ref = rowwise.backward(dh1, y1, stats, weight, bias, True, 0.5, keep1)
    for name, got in (("dx", dy1), ("dweight", dweight), ("dbias", dbias)):
        rowwise.check(name, got, *ref[name])
    product(dy1)
    plan.close()


def test_python_refusals():
    from accelgcn import AccelGcnError, dropout, norm
    require_cuda()
    x = torch.zeros((6, 8), device="cuda")
    s = torch.zeros((6, 2), device="cuda")
    w = torch.ones(8, device="cuda")
    for call, error in ((lambda: norm.layer_norm(x.double()), TypeError), (lambda: norm.layer_norm(x[0]), ValueError),
                        (lambda: norm.layer_norm(x.t()), ValueError), (lambda: norm.layer_norm(x[:1].expand(6, 8)), ValueError),
                        (lambda: norm.layer_norm(x, w.half()), TypeError), (lambda: norm.layer_norm(x, w[:7]), ValueError),
                        (lambda: norm.layer_norm(x, w.cpu()), TypeError), (lambda: norm.layer_norm(x, out=x[:5]), ValueError),
                        (lambda: norm.layer_norm(x, out=x.half()), ValueError), (lambda: norm.layer_norm(x, stats=s.t()), ValueError), (lambda: norm.layer_norm(x, stats=s.view(2, 6)), ValueError),
                        (lambda: norm.layer_norm(x, stats=s.half()), TypeError), (lambda: norm.layer_norm(x, p=1.0), AccelGcnError),
                        (lambda: norm.layer_norm(x, eps=0), AccelGcnError), (lambda: norm.layer_norm(x, p=0.5, seed=1.0), TypeError),
                        (lambda: norm.layer_norm(x, step=torch.zeros(1, device="cuda")), TypeError),
                        (lambda: norm.layer_norm(torch.zeros((2, 8193), device="cuda")), AccelGcnError),
                        (lambda: norm.layer_norm_backward(x, x, None), TypeError), (lambda: norm.layer_norm_backward(x, x[:5], s), ValueError),
                        (lambda: norm.layer_norm_backward(x, x, s[:5]), ValueError), (lambda: norm.layer_norm_backward(x, x, s, dweight=w[:4]), ValueError),
                        (lambda: dropout.dropout(x, 1.5, 1), AccelGcnError), (lambda: dropout.dropout(x, 0.5, 1, row0=-1), AccelGcnError),
                        (lambda: dropout.dropout_backward(x, 0.5, 1, relu=True), TypeError),
                        (lambda: dropout.dropout_backward(x, 0.5, 1, relu=True, x=x.half()), ValueError)):
        with pytest.raises(error):
            call()
