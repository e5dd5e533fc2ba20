"""Layer norm and dropout without a GPU: the generator's known answers, the refusals, the native caller's doubles."""
import ctypes

import numpy as np
import pytest
import torch

import rowwise


def test_generator_known_answers():
    # the published answers of Philox4x32-10 (Random123's kat_vectors)
    zero = np.zeros((1, 4), dtype=np.uint64)
    ones = np.full((1, 4), 0xFFFFFFFF, dtype=np.uint64)
    pi = np.array([[0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344]], dtype=np.uint64)
    for counter, key, want in ((zero, (0, 0), "6627e8d5 e169c58d bc57ac4c 9b00dbd8"),
                               (ones, (0xFFFFFFFF, 0xFFFFFFFF), "408f276d 41c83b0e a20bc7c6 6d5451fd"),
                               (pi, (0xA4093822, 0x299F31D0), "d16cfe09 94fdcceb 5001e420 24126ea1")):
        assert " ".join(f"{int(w):08x}" for w in rowwise.philox4x32(counter, key)[0]) == want


def test_mask_of_row_blocks_is_that_of_the_whole():
    whole = rowwise.kept(50, 7, 0.3, 123456789012, offset=5)
    for r in (1, 13, 49):
        assert np.array_equal(rowwise.kept(50 - r, 7, 0.3, 123456789012, offset=5, row0=r), whole[r:])


def _c_args():
    # addresses that are never followed: every call here is refused before anything is launched
    a = 1 << 20
    norm = dict(x=a, ldx=64, weight=a, bias=a, eps=1e-5, y=a, ldy=64, stats=a, rows=10, cols=64, dtype=0, act=1, p=0.5, seed=1, offset=0, step=None,
                row0=0, stream=None)
    back = dict(dy=a, lddy=64, x=a, ldx=64, stats=a, weight=a, bias=a, dx=a, lddx=64, dweight=a, dbias=a, work=a, work_bytes=1 << 40, rows=10, cols=64,
                dtype=0, act=1, p=0.5, seed=1, offset=0, step=None, row0=0, stream=None)
    drop = dict(x=a, ldx=64, y=a, ldy=64, rows=10, cols=64, dtype=0, act=1, p=0.5, seed=1, offset=0, step=None, row0=0, stream=None)
    dropback = dict(dy=a, lddy=64, x=a, ldx=64, dx=a, lddx=64, rows=10, cols=64, dtype=0, act=1, p=0.5, seed=1, offset=0, step=None, row0=0, stream=None)
    return {"agcn_layer_norm": norm, "agcn_layer_norm_backward": back, "agcn_dropout": drop, "agcn_dropout_backward": dropback}


BAD = [(f, k, v, word) for f in ("agcn_layer_norm", "agcn_layer_norm_backward", "agcn_dropout", "agcn_dropout_backward")
       for k, v, word in (("dtype", 3, "element type"), ("dtype", -1, "element type"), ("act", 2, "activation"), ("rows", -1, "row count"),
                          ("rows", 1 << 61, "row count"), ("cols", 0, "columns"), ("cols", -5, "columns"), ("p", 1.0, "probability"),
                          ("p", -0.1, "probability"), ("p", float("nan"), "probability"), ("row0", -1, "row0"), ("row0", 1 << 60, "row0"),
                          ("step", (1 << 20) + 4, "step"), ("x", None, "x is null"), ("x", (1 << 20) + 2, "aligned"), ("ldx", 63, "apart"),
                          ("ldx", -64, "apart"), ("ldx", 1 << 62, "stride"), ("ldx", (1 << 40) + 1, "stride"))]
BAD += [(f, "cols", 8193, "8192") for f in ("agcn_layer_norm", "agcn_layer_norm_backward")]
BAD += [("agcn_layer_norm", k, v, word) for k, v, word in (("eps", 0.0, "eps"), ("eps", -1.0, "eps"), ("eps", float("nan"), "eps"), ("eps", 1e-40, "eps"),
                                                            ("eps", float("inf"), "eps"), ("y", None, "y is null"), ("ldy", 1, "apart"),
                                                            ("weight", (1 << 20) + 1, "aligned"), ("stats", (1 << 20) + 4, "aligned"))]
BAD += [("agcn_layer_norm_backward", k, v, word) for k, v, word in (("stats", None, "stats"), ("stats", (1 << 20) + 4, "aligned"), ("dy", None, "dy is null"),
                                                                     ("dx", None, "dx is null"), ("lddx", 9, "apart"), ("dbias", (1 << 20) + 2, "aligned"))]
BAD += [("agcn_dropout", "y", None, "y is null"), ("agcn_dropout_backward", "dy", None, "dy is null"), ("agcn_dropout_backward", "dx", None, "dx is null")]


@pytest.mark.parametrize("function,key,value,word", BAD)
def test_the_library_refuses(function, key, value, word):
    from accelgcn import _lib
    args = _c_args()[function]
    args[key] = value
    assert getattr(_lib.load(), function)(*args.values()) == _lib.ERR_INVALID
    assert word in _lib.load().agcn_last_error().decode()


def test_no_rows_are_no_work():
    from accelgcn import _lib
    for function in ("agcn_layer_norm", "agcn_dropout", "agcn_dropout_backward"):
        args = _c_args()[function]
        args["rows"] = 0
        assert getattr(_lib.load(), function)(*args.values()) == _lib.OK


def test_work_size_refuses():
    from accelgcn import _lib
    n = ctypes.c_int64()
    lib = _lib.load()
    assert lib.agcn_layer_norm_backward_work(10, 64, 0, None) == _lib.ERR_INVALID
    assert lib.agcn_layer_norm_backward_work(10, 8193, 0, ctypes.byref(n)) == _lib.ERR_INVALID
    assert lib.agcn_layer_norm_backward_work(10, 64, 7, ctypes.byref(n)) == _lib.ERR_INVALID


def test_python_refuses_host_tensors():
    from accelgcn import dropout, norm
    x, stats = torch.zeros((4, 8)), torch.zeros((4, 2))
    for call in (lambda: norm.layer_norm(x), lambda: norm.layer_norm_backward(x, x, stats), lambda: dropout.dropout(x, 0.5, 1),
                 lambda: dropout.dropout_backward(x, 0.5, 1)):
        with pytest.raises(TypeError, match="CUDA"):
            call()


def test_native_caller_passes_doubles_and_many_integers():
    from accelgcn import _lib
    seen = []
    i64, f64 = ctypes.c_int64, ctypes.c_double
    # doubles among the integers, more of both than fit the registers that integers have
    kinds = [i64] * 4 + [f64] + [i64] * 9 + [f64] + [i64] * 11 + [f64, f64]
    cb = ctypes.CFUNCTYPE(ctypes.c_int, *kinds)(lambda *a: (seen.append(a), 7)[1])
    address = ctypes.cast(cb, ctypes.c_void_p).value
    args = [float(k) + 0.25 if kinds[k] is f64 else (k << 33) - 50 for k in range(len(kinds))]
    assert _lib.call()(address, *args) == 7 and list(seen[0]) == args
    few = ctypes.CFUNCTYPE(ctypes.c_int, *[i64] * 14)(lambda *a: (seen.append(a), -3)[1])
    assert _lib.call()(ctypes.cast(few, ctypes.c_void_p).value, *range(14)) == -3 and list(seen[1]) == list(range(14))
    for wrong in ([1] * 25, [1.0] * 5, [1] * 30):
        with pytest.raises(TypeError):
            _lib.call()(address, *wrong)
