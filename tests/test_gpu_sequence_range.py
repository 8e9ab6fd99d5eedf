"""The sequence-head operators on the GPU where their numbers end: terms that need every bit, gradients that differ by orders of magnitude from row to row,
gates and states that leave f32's range, outputs that overlap inputs, recomputation.  Tolerances follow from the arithmetic stated at each test; where
every product and every sum is exact the results are equal."""
import numpy as np
import pytest

from helpers import ROOT  # noqa: F401  (puts oracle/ on the path)

import sequence as oseq

pytestmark = pytest.mark.gpu

KINDS = ["f32", "bf16", "f16"]


@pytest.fixture(scope="module")
def T():
    import torch

    import gfnerf_amd  # noqa: F401
    from gfnerf_amd import _lib

    _lib.require_device()
    return torch


@pytest.fixture(scope="module")
def ops(T):
    from gfnerf_amd import ops as _ops

    return _ops


def dt(T, kind):
    return {"f32": T.float32, "bf16": T.bfloat16, "f16": T.float16}[kind]


def held(T, kind, v):
    """v as a tensor of the type on the device, which has to hold it exactly."""
    t = T.from_numpy(np.ascontiguousarray(v)).to(dt(T, kind)).cuda()
    assert np.array_equal(t.double().cpu().numpy(), v)
    return t


# ---- gated layer, backward --------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,k,h", [(40, 8, 16), (70, 8, 40), (33, 7, 96), (40, 40, 16), (150, 72, 8), (40, 100, 128)])
def test_gated_gradients_of_exact_terms_are_exact(T, ops, kind, n, k, h):
    """relu, and inputs on grids: 8 inputs of a row are used (multiples of 2^-3 in [-1, 1]), Wg is +-1/2, Wu multiples of 2^-6 in [-1, 1], dh of 2^-8 and zero but for some 20 rows
    of a feature.  g and u are then exact (grids 2^-4 and 2^-9), du = dh g and dg = dh u as well (17 to 19 bits: more than two operands of bf16 hold), and every
    product's sum stays on a grid of 2^-20 below 2^4: 24 bits.  So nothing rounds but the results, once."""
    rng = np.random.default_rng(5)
    grid = lambda q, *s: np.round(rng.uniform(-1, 1, s) * q) / q  # noqa: E731
    x, wu, dh = grid(8, n, k), grid(64, h, k), np.round(rng.uniform(-1, 1, (n, h)) * 255) / 256
    x[:, 8:] = 0
    dh *= rng.random((n, h)) < 20 / n
    wg = np.where(rng.random((h, k)) < 0.5, 0.5, -0.5)
    bg, bu = grid(8, h), grid(8, h)
    g, u = x @ wg.T + bg, x @ wu.T + bu
    dg, du = dh * u * (g > 0), dh * np.maximum(g, 0)
    want = {"dx": dg @ wg + du @ wu, "dwg": dg.T @ x, "dwu": du.T @ x, "dbg": dg.sum(0), "dbu": du.sum(0)}
    most = {"dx": np.abs(dg) @ np.abs(wg) + np.abs(du) @ np.abs(wu), "dwg": np.abs(dg).T @ np.abs(x), "dwu": np.abs(du).T @ np.abs(x), "dbg": np.abs(dg).sum(0), "dbu": np.abs(du).sum(0)}
    unit = {"dx": 2.0 ** -18, "dwg": 2.0 ** -20, "dwu": 2.0 ** -20, "dbg": 2.0 ** -17, "dbu": 2.0 ** -17}
    for name, v in want.items():  # what the equality below rests on
        assert (v / unit[name] == np.round(v / unit[name])).all() and most[name].max() < 2.0 ** 24 * unit[name], name
    t = [held(T, kind, v) for v in (x, wg, wu, dh, bg, bu)]
    for name, got in zip(want, ops.gated_bwd(*t, act="relu")):
        rounded = T.from_numpy(want[name]).to(got.dtype)
        differ = got.cpu() != rounded
        assert not bool(differ.any()), (name, int(differ.sum()), differ.numel())
