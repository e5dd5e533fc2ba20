"""Column sums of the layer norm's backward pass: which calls need a workspace, sums that must be exact, rows off 16-byte boundaries
over many turns."""
import ctypes

import pytest
import torch

from conftest import require_cuda
from test_norm_gpu import _case

pytestmark = pytest.mark.gpu

F32, B16, F16 = torch.float32, torch.bfloat16, torch.float16
CODES = {F32: 0, B16: 1, F16: 2}


def _work(rows, cols, t):
    from accelgcn import _lib
    n = ctypes.c_int64()
    _lib.check(_lib.load().agcn_layer_norm_backward_work(rows, cols, CODES[t], ctypes.byref(n)))
    return n.value


@pytest.mark.parametrize("rows,cols,t", [(512, 510, F32), (17, 511, F32), (512, 507, B16), (100, 511, F16)])
def test_few_rows_of_a_thread_block_each_are_not_one_cluster(rows, cols, t):
    # the widest rows that a warp has, where they begin behind a 16-byte boundary: a thread block has one, and a cluster would have up to
    # 64 of them in turn.  (Once one, on 8 of the SMs, without a workspace.)
    require_cuda()
    assert _work(rows, cols, t) > 0 and _work(16, cols, t) == 0
    _case(rows, cols, t, relu=True, p=0.25, weight=True, bias=True)
    _case(16, cols, t, relu=True, p=0.25, weight=True, bias=True)


@pytest.mark.parametrize("start,needed", [(0, False), (1, True)])
def test_the_workspace_is_needed_where_the_rows_sit(start, needed):
    # 512 columns on a boundary are a warp's: a cluster adds up 512 rows of them, as ever, and needs no workspace
    from accelgcn import _lib
    require_cuda()
    gen = torch.Generator(device="cuda").manual_seed(31)
    rows, cols = 300, 512
    x, dy, dx = (torch.randn((rows, cols + 4), generator=gen, device="cuda")[:, start:start + cols] for _ in range(3))
    stats = torch.ones((rows, 2), device="cuda")
    dw, db = torch.full((cols,), 7.0, device="cuda"), torch.empty(cols, device="cuda")
    rc = _lib.load().agcn_layer_norm_backward(dy.data_ptr(), cols + 4, x.data_ptr(), cols + 4, stats.data_ptr(), None, None, dx.data_ptr(), cols + 4,
                                              dw.data_ptr(), db.data_ptr(), None, 0, rows, cols, 0, 0, 0.0, 0, 0, None, 0,
                                              torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    if needed:
        assert rc == _lib.ERR_INVALID and b"workspace" in _lib.load().agcn_last_error() and bool((dw == 7.0).all())
    else:
        assert rc == _lib.OK
        assert bool(((db - dy.double().sum(0)).abs() <= 300 * 2.0 ** -24 * dy.double().abs().sum(0)).all())


def test_a_term_of_few_rows_has_few_roundings_behind_it():
    # 2 048 rows of 16: two rows per group of a thread block of 128, 8 thread blocks.  Behind a term are at most 1 addition in its thread, 15 + 3
    # among the groups and 3 among the thread blocks.  One large term in each thread block, on which a 1 is a tie that is rounded away each
    # time: 127 in turn would be off by 127 U.
    from accelgcn import norm
    require_cuda()
    dy = torch.ones((2048, 16), device="cuda")
    dy[1024:] = 0.0
    dy[:1024:128] = 2.0 ** 24
    x = torch.ones_like(dy)
    stats = torch.tensor([[0.0, 1.0]], device="cuda").repeat(2048, 1)
    w = torch.ones(16, device="cuda")
    _dx, dw, db = norm.layer_norm_backward(dy, x, stats, w, w)
    want = dy.double().sum(0)
    for got in (dw, db):                          # h = 1: the two sums are the same
        assert bool(((got - want).abs() <= 22 * 2.0 ** -24 * want).all()), float(((got - want).abs() / want).max() * 2.0 ** 24)


def _signs(shape, t, gen):
    return torch.randint(0, 2, shape, generator=gen, device="cuda", dtype=torch.int8).mul_(2).sub_(1).to(t)


@pytest.mark.parametrize("p", [0.0, 0.5])
@pytest.mark.parametrize("cols,t,rows_per_block", [(16, F32, 128), (61, F32, 32), (128, F32, 16), (100, B16, 16), (128, F16, 16), (500, F32, 8), (701, F32, 1),
                                                   (1001, F32, 1), (1003, B16, 1)])
def test_no_row_is_lost(cols, t, rows_per_block, p):
    # terms of +1 and -1 (+2 and -2 with a mask): every sum on the way is a whole number below 2^24, so the result is exact, whatever
    # the order.  The rows end before, with and behind a whole turn of all groups, for each number of thread blocks per SM.
    import rowwise
    from accelgcn import norm
    require_cuda()
    gen = torch.Generator(device="cuda").manual_seed(cols)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    most = 5 * (4 * sms // 8 * 8) * rows_per_block + 1
    xs, dys = _signs((most, cols), t, gen), _signs((most, cols), t, gen)
    kept = torch.from_numpy(rowwise.kept(most, cols, p, 5, 0)).cuda()
    stats = torch.tensor([[0.0, 1.0]], device="cuda").repeat(most, 1)
    w, dx = torch.ones(cols, device="cuda"), torch.empty_like(xs)
    for per_sm in (1, 2, 3, 4):
        for more in (-1, 0, 1):
            rows = 5 * (per_sm * sms // 8 * 8) * rows_per_block + more
            x, dy = xs[:rows], dys[:rows]
            _dx, dw, db = norm.layer_norm_backward(dy, x, stats[:rows], w, w, p=p, seed=5, dx=dx[:rows])
            dz = torch.where(kept[:rows], dy.double(), 0.0) * (1.0 / (1.0 - p))
            assert torch.equal(db.double(), dz.sum(0)) and torch.equal(dw.double(), (dz * x.double()).sum(0)), rows


def test_no_row_is_lost_beyond_32_bits():
    from accelgcn import norm
    require_cuda()
    rows, cols = 17_000_000, 128                 # 2.2e9 elements, 4.4 GB
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    gen = torch.Generator(device="cuda").manual_seed(33)
    x, dy = _signs((rows, cols), B16, gen), _signs((rows, cols), B16, gen)
    stats = torch.tensor([[0.0, 1.0]], device="cuda").repeat(rows, 1)
    w = torch.ones(cols, device="cuda")
    _dx, dw, db = norm.layer_norm_backward(dy, x, stats, w, w)
    dw64, db64 = torch.zeros(cols, dtype=torch.float64, device="cuda"), torch.zeros(cols, dtype=torch.float64, device="cuda")
    for r in range(0, rows, 1_000_000):
        part = slice(r, min(rows, r + 1_000_000))
        db64 += dy[part].double().sum(0)
        dw64 += (dy[part].double() * x[part].double()).sum(0)
    assert torch.equal(db.double(), db64) and torch.equal(dw.double(), dw64)


@pytest.mark.parametrize("rows,cols,t,row0", [(20_000, 1001, F32, 1), (20_003, 1003, B16, 0), (20_000, 701, F32, 3), (20_001, 511, F32, 0), (12_000, 2046, F16, 1)])
def test_many_rows_of_a_thread_block_each_off_the_boundary(rows, cols, t, row0):
    # 17 and more rows in turn per thread block: the ring is filled anew by chunks that the row does not fill, and the mask's words
    # go from lane to lane, row after row
    _case(rows, cols, t, relu=True, p=0.5, weight=True, bias=True, row0=row0)
