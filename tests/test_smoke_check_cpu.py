"""The check that smoke() makes of the layer norm's gradient sees what it should see (mistakes planted in numpy)."""
import numpy as np
import pytest

from __graft_entry__ import norm_gradient_off


def _gradient(wrong=None):
    rng = np.random.default_rng(3)
    rows, cols, p = 64, 32, 0.5
    x, dy = np.maximum(rng.standard_normal((rows, cols)), 0), rng.standard_normal((rows, cols))     # features behind a ReLU
    x[7] = 0.0                                                                                      # and a node without any
    kept = rng.random((rows, cols)) >= p
    stats = np.stack((x.mean(1), 1 / np.sqrt(x.var(1) + 1e-5)), 1).astype(np.float32)
    mean, rstd = stats[:, :1].astype(np.float64), stats[:, 1:].astype(np.float64)
    h = (x - mean) * rstd
    gate = np.ones_like(kept) if wrong == "gate" else h > 0
    mask = np.roll(kept, 1, axis=1) if wrong == "mask" else kept
    g = np.where(mask & gate, dy / (1 if wrong == "scale" else 1 - p), 0.0)
    dx = rstd * (g - (0 if wrong == "mean" else g.mean(1, keepdims=True)) - (0 if wrong == "h term" else h * (g * h).mean(1, keepdims=True)))
    if wrong == "zeros":
        dx = np.zeros_like(dx)
    if wrong == "nan":
        dx[3, 3] = np.nan
    return norm_gradient_off(dx.astype(np.float32), dy.astype(np.float32), x, stats, kept, p)


def test_the_formula_passes():
    # dy and dx are rounded to fp32: 2^-24 of themselves each, through three terms
    assert _gradient() <= 6 * 2.0 ** -24


@pytest.mark.parametrize("wrong", ["zeros", "h term", "mean", "mask", "gate", "scale", "nan"])
def test_mistakes_do_not(wrong):
    assert not _gradient(wrong) <= 1e-2
