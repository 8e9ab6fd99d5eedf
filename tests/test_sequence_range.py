"""The sequence-head operators without a GPU, where their numbers end: what the oracle's bounds let through."""
import numpy as np
import pytest

from helpers import ROOT  # noqa: F401  (puts oracle/ on the path)

import sequence as oseq


def operands_under(dz, e):
    """dz as two numbers of f16 under 2^e (an array for each row, or one number), back in 64 bits."""
    v = np.ldexp(dz, e)
    hi = v.astype(np.float16).astype(np.float64)
    return np.ldexp(hi + (v - hi).astype(np.float16).astype(np.float64), -e)


@pytest.mark.parametrize("low,seen", [(0, False), (10, True), (12, True), (16, True)])
def test_the_f16_bound_sees_what_a_power_from_dh_loses(low, seen):
    """dz under one power of two a tile, taken from its largest |dh|, against a power of each sample's own largest |dz|: the bound accepts the second at
    every ratio of the rows' gradients, and not the first where it cuts off bits that the result has."""
    rng = np.random.default_rng(low)
    n, k, h = 64, 64, 64
    f16 = lambda v: v.astype(np.float16).astype(np.float64)  # noqa: E731
    x, wg, wu, dh = f16(rng.standard_normal((n, k))), f16(rng.standard_normal((h, k)) / 8), f16(rng.standard_normal((h, k)) / 8), rng.standard_normal((n, h))
    dh[1:] *= 2.0 ** -low
    dh = f16(dh)
    value, bound = oseq.gated_bwd(x, wg, wu, dh, None, None, "silu", "f16")["dx"]
    g, u = x @ wg.T, x @ wu.T
    a, da, _ = oseq.act(g, "silu")
    dz = np.stack([dh * u * da, dh * a])

    def outside(e):
        dx = f16(operands_under(dz[0], e) @ wg + operands_under(dz[1], e) @ wu)
        return int((np.abs(dx - value) > bound).sum())

    from_dh = -4 * ((int(np.frexp(np.abs(dh).max())[1])) // 4) - 4
    own = (15 - np.frexp(np.abs(dz).max((0, 2)))[1]) // 8 * 8
    assert (outside(from_dh) > 0) == seen and outside(own[:, None]) == 0
