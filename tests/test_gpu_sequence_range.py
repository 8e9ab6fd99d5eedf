"""The sequence-head operators on the GPU where their numbers end: terms that need every bit, gradients that differ by orders of magnitude from row to row,
gates and states that leave f32's range, outputs that overlap inputs, recomputation.  Tolerances follow from the arithmetic stated at each test; where
every product and every sum is exact the results are equal."""
import numpy as np
import pytest

from helpers import ROOT  # noqa: F401  (puts oracle/ on the path)

import sequence as oseq
from test_gpu_sequence import KINDS, close, dt, gated_inputs

pytestmark = pytest.mark.gpu

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


NAMES = ("dx", "dwg", "dwu", "dbg", "dbu")


def on_device_of(like, v):
    import torch

    return torch.from_numpy(v).to(like.device)


def backward_is_exact(ops, kind, act, x, wg, wu, bg, bu, dh):
    """Every gradient within the oracle's bound, infinite where its value is past the type's largest number (f16: 65504 and half a step, 16); x, .. are
    (tensor, its 64-bit values)."""
    want = oseq.gated_bwd(x[1], wg[1], wu[1], dh[1], bg[1], bu[1], act, kind)
    got = dict(zip(NAMES, ops.gated_bwd(x[0], wg[0], wu[0], dh[0], bg[0], bu[0], act)))
    for name, (value, bound) in want.items():
        v = got[name].double().cpu().numpy()
        over = (np.abs(value) + bound >= 65520) & np.isinf(v) & (np.sign(v) == np.sign(value)) if kind == "f16" else np.zeros(v.shape, bool)
        rest = got[name].masked_fill(on_device_of(got[name], over), 0.0)
        close(rest, (np.where(over, 0.0, value), bound), name)
    return got, want


def scaled(T, kind, v, by):
    t = (v[0].double() * T.from_numpy(np.ascontiguousarray(np.broadcast_to(by, v[1].shape))).cuda()).to(dt(T, kind))
    return t, t.double().cpu().numpy()


@pytest.mark.parametrize("k,h", [(64, 64), (128, 128), (20, 160)])
@pytest.mark.parametrize("top", [0, 10])
@pytest.mark.parametrize("low", [8, 12, 14, 16])
def test_gated_f16_rows_of_small_gradient_beside_large_ones(T, ops, k, h, top, low):
    """One row of every 64 has gradients 2^low times those of the others.  dx's rows and dW, each within what the operands and one rounding may do to
    them: a row's own gradient decides what is cut off of it, and of dW's terms only what is far below the tile's largest."""
    n = 300
    x, wg, wu, bg, bu, dh = gated_inputs(T, "f16", n, k, h, True, "silu", seed=low)
    by = np.full((n, 1), 2.0 ** (top - low))
    by[7::64] = 2.0 ** top
    dh = scaled(T, "f16", dh, by)
    backward_is_exact(ops, "f16", "silu", x, wg, wu, bg, bu, dh)
    # the large rows alone decide dW's entries; those of features that only small rows reach are seen where the large ones are taken out of x and dh
    alone = dh[0].clone()
    alone[7::64] = 0
    got = ops.gated_bwd(x[0], wg[0], wu[0], alone, bg[0], bu[0])[0]
    both = ops.gated_bwd(x[0], wg[0], wu[0], dh[0], bg[0], bu[0])[0]
    keep = T.arange(n, device="cuda") % 64 != 7
    assert T.equal(got[keep], both[keep])  # a sample's gradient does not depend on its neighbours


@pytest.mark.parametrize("act", ["silu", "sigmoid", "gelu"])
@pytest.mark.parametrize("size", [1e-2, 1e-3, 1e-4])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_gated_gradients_of_small_activations(T, ops, kind, act, size):
    """Inputs of the size of freshly initialised hash features, without biases: u and act(g) are small, and dz far below dh."""
    x, wg, wu, _, _, dh = gated_inputs(T, kind, 400, 32, 64, False, act, seed=1)
    backward_is_exact(ops, kind, act, scaled(T, kind, x, size), wg, wu, (None, None), (None, None), dh)


@pytest.mark.parametrize("scale", [2.0 ** -18, 1.0, 2.0 ** 10])
def test_gated_f16_gradients_above_the_types_range(T, ops, scale):
    """act(g) = 1e5 and u = 0.1: h = 1e4 is finite and so are its gradients where dh and the weights leave them finite, although dz passes f16's largest
    number.  Ordinary rows beside them keep theirs."""
    rng = np.random.default_rng(4)
    n, k, h = 130, 16, 32
    x, wg, wu = rng.standard_normal((n, k)), rng.standard_normal((h, k)), rng.standard_normal((h, k)) * 0.1
    x[[3, 70]], wg[:, 0] = 0, 500.0
    x[[3, 70], 0] = 200.0
    wu[:, 0] = 0.1 / 200
    dh = rng.standard_normal((n, h)) * min(scale, 1.0)
    dh[[3, 70]] = 0
    dh[3, 5], dh[70, 9] = 0.99 * min(scale, 1.0), -0.5 * min(scale, 1.0)
    made = lambda v: (lambda t: (t.cuda(), t.double().numpy()))(T.from_numpy(v).to(T.float16))  # noqa: E731
    got, want = backward_is_exact(ops, "f16", "relu", made(x), made(wg), made(wu), (None, None), (None, None), made(dh * max(scale, 1.0)))
    if scale == 1.0:
        assert np.abs(want["dx"][0][3]).max() < 65504 and bool(T.isfinite(got["dx"][3]).all())


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_gated_gradients_that_are_not_finite_stay_in_their_rows(T, ops, kind, bad):
    """An infinite or undefined dh of one sample reaches that sample's dx only, and of dW the rows of its features."""
    x, wg, wu, bg, bu, dh = gated_inputs(T, kind, 200, 24, 48, True, "silu", seed=3)
    clean = ops.gated_bwd(x[0], wg[0], wu[0], dh[0], bg[0], bu[0])
    d = dh[0].clone()
    d[70, 11] = bad
    got = ops.gated_bwd(x[0], wg[0], wu[0], d, bg[0], bu[0])
    keep = T.arange(200, device="cuda") != 70
    assert T.equal(got[0][keep], clean[0][keep]) and not bool(T.isfinite(got[0][70]).any())
    rows = T.arange(48, device="cuda") != 11
    want = oseq.gated_bwd(x[1], wg[1], wu[1], np.where(np.arange(200)[:, None] == 70, np.where(np.arange(48) == 11, 0.0, dh[1]), dh[1]), bg[1], bu[1], "silu", kind)
    for name, g in zip(NAMES[1:], got[1:]):
        assert not bool(T.isfinite(g[11]).any())
        value, bound = want[name]
        off = (g.double().cpu().numpy() - value)[rows.cpu().numpy()]
        assert (np.abs(off) <= bound[rows.cpu().numpy()]).all(), name
    if bad == float("inf"):  # an infinity stays one
        assert bool(T.isinf(got[3][11])) and bool(T.isinf(got[4][11]))


@pytest.mark.parametrize("k,h", [(20, 128), (64, 128), (90, 100), (128, 128), (33, 200)])
@pytest.mark.parametrize("first", [0, -20, 20])
def test_gated_f16_features_and_rows_of_very_different_gradients(T, ops, k, h, first):
    """Features of one block of 32 far below or above those of the next, blocks of 16 rows without any gradient, one block of features without any:
    every power is met and changed, up and down, from tile to tile."""
    n = 500
    x, wg, wu, bg, bu, dh = gated_inputs(T, "f16", n, k, h, True, "gelu", seed=2)
    by = np.ones((n, h))
    by[:, :32] *= 2.0 ** min(first, 0)
    by[:, 32:64] *= 2.0 ** -max(first, 0)
    by[:, 64:96] = 0
    by[100:170] *= 2.0 ** -3
    by[250:400] *= 2.0 ** 9
    by[16:32], by[48:64], by[448:] = 0, 0, 0
    backward_is_exact(ops, "f16", "gelu", x, wg, wu, bg, bu, scaled(T, "f16", dh, by))


# ---- recurrence, walked in runs of rows -------------------------------------------------------------------------------------------------------
LONG = [4096, 3000, 5000]  # few and long: every ray is many runs of 32 rows


def gates(T, kind, gate, n, g, seed):
    rng = np.random.default_rng(seed)
    v = rng.standard_normal((n, g))
    return T.from_numpy(np.exp(v * 1.5 - 2) if gate == "decay" else 1 / (1 + np.exp(-v - 1)) if gate == "linear" else v + 1).to(dt(T, kind)).cuda()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("gate", ["linear", "sigmoid", "decay"])
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("bad", ["nan", "large"])
@pytest.mark.parametrize("g", [8, 1])
def test_gates_of_one_ray_do_not_reach_the_next_in_runs(T, ops, kind, gate, reverse, bad, g):
    """Undefined gates in the middle of a ray, and gates whose product passes f32's range: the other rays' states, outputs and gradients are those of a
    call without them, bit for bit."""
    off = T.tensor(np.concatenate([[0], np.cumsum(LONG)]), dtype=T.int32, device="cuda")
    n, d = sum(LONG), 8
    rng = np.random.default_rng(1)
    made = lambda *s: T.from_numpy(rng.standard_normal(s))  # noqa: E731
    f, c, dh = gates(T, kind, gate, n, g, 0), made(n, d).to(dt(T, kind)).cuda(), made(n, d).to(dt(T, kind)).cuda()
    h0, ds = made(3, d).float().cuda(), made(3, d).float().cuda()

    def call(f):
        r = ops.ray_scan_fwd(off, f, c, gate, reverse, h0, save=True)
        b = ops.ray_scan_bwd(off, f, c, dh, r["saved"], gate, reverse, h0, ds)
        return [r["h"], b["df"], b["dc"]], [r["state"], b["dh0"]]

    clean_rows, clean_rays = call(f)
    for ray in range(3):
        s, e = sum(LONG[:ray]), sum(LONG[:ray + 1])
        other = f.clone()
        if bad == "nan":
            other[s + 700:s + 703] = float("nan")
        else:
            other[s + 100:e - 100] = {"linear": 20.0, "sigmoid": 80.0, "decay": -3.0}[gate]
        rows, rays = call(other)
        keep = T.ones(n, dtype=T.bool, device="cuda")
        keep[s:e] = False
        for a, b in zip(rows, clean_rows):
            assert T.equal(a[keep], b[keep]), ray
        others = [r for r in range(3) if r != ray]
        for a, b in zip(rays, clean_rays):
            assert T.equal(a[others], b[others]), ray


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_what_is_not_finite_stays_to_the_end_of_its_ray_in_runs(T, ops, kind, reverse, value):
    """An input that is undefined or infinite early in a ray whose gates multiply to nothing within a run (exp(-10) a row): the definition keeps it to the
    ray's end, in its channel."""
    off = T.tensor(np.concatenate([[0], np.cumsum(LONG)]), dtype=T.int32, device="cuda")
    n, d = sum(LONG), 8
    f = T.full((n, d), 10.0, dtype=dt(T, kind), device="cuda")
    c = T.ones(n, d, dtype=dt(T, kind), device="cuda")
    at = 4096 + (2900 if reverse else 100)
    c[at, 3] = value
    r = ops.ray_scan_fwd(off, f, c, "decay", reverse, save=True)
    want = T.zeros(n, d, dtype=T.bool, device="cuda")
    if reverse:
        want[4096:at + 1, 3] = True
    else:
        want[at:7096, 3] = True
    same = T.isnan if value != value else T.isinf
    assert T.equal(same(r["h"]), want) and T.equal(T.isfinite(r["h"]), ~want)
    assert T.equal(same(r["state"]), T.tensor([[False] * 8, [False] * 3 + [True] + [False] * 4, [False] * 8], device="cuda"))
    dh = T.ones(n, d, dtype=dt(T, kind), device="cuda")
    dh[at, 3] = value
    ok = ops.ray_scan_fwd(off, f, T.ones_like(c), "decay", reverse, save=True)
    b = ops.ray_scan_bwd(off, f, T.ones_like(c), dh, ok["saved"], "decay", reverse)
    want = T.zeros(n, d, dtype=T.bool, device="cuda")
    if reverse:
        want[at:7096, 3] = True
    else:
        want[4096:at + 1, 3] = True
    assert T.equal(~T.isfinite(b["dc"]), want)
    assert T.equal(~T.isfinite(b["dh0"]), T.tensor([[False] * 8, [False] * 3 + [True] + [False] * 4, [False] * 8], device="cuda"))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("first,start", [(2.0 ** -5, 2.0 ** 100), (2.0 ** 5, 2.0 ** -100)])
def test_a_state_in_f32s_range_survives_gates_whose_product_leaves_it(T, ops, kind, reverse, first, start):
    """32 rows of 2^-5 (2^5) and 32 of its reciprocal, over and over in the recurrence's order, from 2^100 (2^-100): every state is a power of two between
    2^-60 and 2^100 (2^-100 and 2^60), although the product of a run's gates is 2^-160 (2^160).  The adjoint meets the reciprocals first and starts from
    the reciprocal."""
    off = T.tensor([0, 4096, 6144], dtype=T.int32, device="cuda")
    n, d = 6144, 8
    f = np.where((np.arange(n) % 64 < 32) != reverse, first, 1 / first)[:, None] * np.ones((1, d))
    zero = np.zeros((n, d))
    h0, ds = np.full((2, d), start), np.full((2, d), 1 / start)
    want = oseq.ray_scan(off.cpu().numpy(), f, zero, "linear", reverse, "f32", h0, zero, ds)
    assert all(2.0 ** -100 <= v.min() and v.max() <= 2.0 ** 100 for v in (want["h"][0], want["dc"][0]))
    t = lambda v, k=kind: T.from_numpy(v).to(dt(T, k)).cuda()  # noqa: E731
    r = ops.ray_scan_fwd(off, t(f), t(zero), "linear", reverse, t(h0, "f32"), save=True)
    assert np.array_equal(r["h"].double().cpu().numpy(), want["h"][0]) and np.array_equal(r["state"].double().cpu().numpy(), want["state"][0]), lens
    b = ops.ray_scan_bwd(off, t(f), t(zero), t(zero), r["saved"], "linear", reverse, t(h0, "f32"), t(ds, "f32"))
    assert np.array_equal(b["dc"].double().cpu().numpy(), want["dc"][0]) and np.array_equal(b["dh0"].double().cpu().numpy(), want["dh0"][0])


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("reverse", [False, True])
def test_runs_pass_over_long_stretches_of_rays_without_rows(T, ops, kind, reverse):
    """Stretches of rays that miss the scene, in front of, between and behind the rays with rows, in the middle of a run and on its border: values, and
    a time that is not theirs.  (Taken one after the other they cost a walk a microsecond or two each, seven hundred several times the whole call.)"""
    lens = np.zeros(1500, np.int64)
    lens[[70, 700, 701, 750, 1450]] = (32 * 6000, 7, 32 * 1000 - 7, 96000, 90005)
    rays, n, d = len(lens), int(lens.sum()), 8
    assert n // rays >= 96 and rays < 6 * (n // rays)  # few enough and long enough on average to be walked in runs
    rng = np.random.default_rng(2)
    made = lambda *s: (lambda t: (t.cuda(), t.double().numpy()))(T.from_numpy(rng.standard_normal(s)).to(dt(T, kind)))  # noqa: E731
    f, c, dh = made(n, d), made(n, d), made(n, d)
    h0 = T.from_numpy(rng.standard_normal((rays, d))).float().cuda()
    full = np.flatnonzero(lens)
    offsets = lambda l: T.tensor(np.concatenate([[0], np.cumsum(l)]), dtype=T.int32, device="cuda")  # noqa: E731

    def call(off, h0):
        r = ops.ray_scan_fwd(off, f[0], c[0], "sigmoid", reverse, h0, save=True)
        return r, ops.ray_scan_bwd(off, f[0], c[0], dh[0], r["saved"], "sigmoid", reverse, h0, h0)

    off, few = offsets(lens), offsets(lens[full])
    at = T.from_numpy(full).cuda()
    r, b = call(off, h0)
    rf, bf = call(few, h0[at].contiguous())
    for got, want in ((r["h"], rf["h"]), (b["df"], bf["df"]), (b["dc"], bf["dc"]), (r["state"][at], rf["state"]), (b["dh0"][at], bf["dh0"])):
        assert T.equal(got, want)
    none = T.from_numpy(lens == 0).cuda()
    assert T.equal(r["state"][none], h0[none]) and T.equal(b["dh0"][none], h0[none])

    def best(*args):
        t = []
        for _ in range(5):
            a, z = T.cuda.Event(enable_timing=True), T.cuda.Event(enable_timing=True)
            a.record()
            call(*args)
            z.record()
            z.synchronize()
            t.append(a.elapsed_time(z))
        return min(t)

    few_h0 = h0[at].contiguous()
    best(few, few_h0)
    assert best(off, h0) <= 4 * best(few, few_h0)


# ---- outputs beside and over inputs ---------------------------------------------------------------------------------------------------------------
def test_outputs_beside_inputs_in_one_buffer(T, ops):
    """Columns of one buffer, input and output beside each other, are taken; one column in common is refused, and nothing is written."""
    from gfnerf_amd import _lib

    x, wg, wu, bg, bu, _ = gated_inputs(T, "f32", 500, 31, 40, True, "silu")
    want = ops.gated_fwd(x[0], wg[0], wu[0], bg[0], bu[0])
    buf = T.zeros(500, 80, device="cuda")
    for first, out in ((0, 31), (45, 0), (45, 5)):
        buf[:, first:first + 31] = x[0]
        ops.gated_fwd(buf[:, first:first + 31], wg[0], wu[0], bg[0], bu[0], out=buf[:, out:out + 40])
        assert T.equal(buf[:, out:out + 40], want)
    before = buf.clone()
    off = T.tensor([0, 250, 500], dtype=T.int32, device="cuda")
    f = T.zeros(500, 8, device="cuda")
    state = T.zeros(500, 8, device="cuda")
    call = T.zeros(1, dtype=T.int64, device="cuda")
    for bad in (lambda: ops.gated_fwd(buf[:, 0:31], wg[0], wu[0], bg[0], bu[0], out=buf[:, 30:70]), lambda: ops.gated_fwd(buf[:, 45:76], wg[0], wu[0], bg[0], bu[0], out=buf[:, 6:46]),
                lambda: ops.gated_fwd(buf[:400, 0:31], wg[0], wu[0], bg[0], bu[0], out=buf.view(-1)[7:7 + 400 * 60].view(400, 60)[:, :40]),
                lambda: ops.ray_scan_fwd(off, f, buf[:, 0:8], out=buf[:, 7:15]), lambda: ops.ray_scan_step(f, buf[:, 0:8], state, out=buf[:, 1:9]),
                lambda: ops.dropout(buf[:, 0:8], 0.5, 1, call, out=buf[:, 7:15]), lambda: ops.dropout(buf[1:, :8], 0.5, 1, call, out=buf[:-1, :8])):
        with pytest.raises(_lib.GfnError, match="overlaps"):
            bad()
    T.cuda.synchronize()
    assert T.equal(buf, before) and not bool(state.any())
    h = ops.ray_scan_fwd(off, f, buf[:, 0:8], out=buf[:, 8:16])["h"]
    assert T.equal(h, ops.ray_scan_fwd(off, f, before[:, 0:8])["h"])
    c = before[:, 0:8].contiguous()
    s = state.clone()
    want = ops.ray_scan_step(f, c, s)
    assert T.equal(ops.ray_scan_step(f, c, state, out=c), want) and T.equal(state, s)  # h may be c


# ---- captures beside eager graphs -----------------------------------------------------------------------------------------------------------------
def frozen(module):
    for p in module.parameters():
        p.requires_grad_(False)
    return module


def leaf_cases(T):
    """A forward for each entry point whose leaves other operations (a product, a reshape, a cast) stand in front of, or of which the last layer alone is
    trained: (name, forward)."""
    from gfnerf_amd.gfnerf.mlp import Dropout, GatedMLPNetwork, gated_linear
    from gfnerf_amd.gfnerf.ray_scan import RayRecurrence, ray_scan, render_features

    off = T.tensor([0, 5, 9], dtype=T.int32, device="cuda")
    leaf = lambda *s: T.rand(*s, device="cuda", requires_grad=True)  # noqa: E731
    spec = {"activation": "SwiGLU", "output_activation": "None", "n_neurons": 16, "n_hidden_layers": 1}
    net, last, rec = frozen(GatedMLPNetwork(8, 4, spec).cuda()), frozen(GatedMLPNetwork(8, 4, spec).cuda()), frozen(RayRecurrence(8, 16).cuda())
    last.layers[-1].weight.requires_grad_(True)
    drop = Dropout(0.5).cuda()
    sigma, dt_, x, x3, h0, w = leaf(9), leaf(9), leaf(9, 8), leaf(3, 3, 8), leaf(2, 8), leaf(16, 8)
    const = lambda *s: T.rand(*s, device="cuda")  # noqa: E731
    f, c, plain = const(9, 1), const(9, 8), const(9, 8)
    return [("render_features sigma", lambda: render_features(off, sigma, f.view(-1), c)), ("render_features dt", lambda: render_features(off, f.view(-1), dt_, c)),
            ("render_features features", lambda: render_features(off, f.view(-1), f.view(-1), x)), ("network input", lambda: net(x)),
            ("network input of three dimensions", lambda: net(x3)), ("last layer", lambda: last(plain)), ("recurrence input", lambda: rec(x, off)[0]),
            ("recurrence state", lambda: ray_scan(off, f, c, h0=h0)[1]), ("gated layer", lambda: gated_linear(plain, w, w)), ("dropout", lambda: drop(x))]


@pytest.mark.parametrize("i", range(10))
def test_a_capture_beside_a_live_eager_graph_of_any_leaf_is_refused(T, i):
    from gfnerf_amd import _lib

    name, forward = leaf_cases(T)[i]
    out = forward()
    assert out.requires_grad, name
    with pytest.raises(_lib.GfnError, match="eager autograd graph"):
        with T.cuda.graph(T.cuda.CUDAGraph()):
            forward()
    T.cuda.synchronize()
    del out
    with T.cuda.graph(T.cuda.CUDAGraph()):  # without it the capture is taken
        out = forward()
    T.cuda.synchronize()


# ---- dropout modules ------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("reentrant", [False, True])
def test_a_recomputed_dropout_is_refused(T, reentrant):
    from torch.utils.checkpoint import checkpoint

    from gfnerf_amd import _lib
    from gfnerf_amd.gfnerf.mlp import Dropout, gated_linear

    drop = Dropout(0.5, seed=1).cuda()
    x, w = T.randn(64, 16, device="cuda", requires_grad=True), T.randn(32, 16, device="cuda", requires_grad=True)
    y = checkpoint(lambda v: gated_linear(drop(v), w, w), x, use_reentrant=reentrant)
    with pytest.raises(_lib.GfnError, match="recomputed inside a backward pass"):
        y.sum().backward()
    # outside of the recomputed part it has one mask: the gradients are those without recomputation
    def grads(layer):
        x.grad = w.grad = None
        drop.counter.fill_(5)
        drop(layer(x)).square().sum().backward()
        return x.grad.clone(), w.grad.clone()

    got = grads(lambda v: checkpoint(gated_linear, v, w, w, use_reentrant=reentrant))
    assert all(T.equal(a, b) for a, b in zip(got, grads(lambda v: gated_linear(v, w, w)))) and int(drop.counter) == 6


def test_default_dropout_modules_draw_masks_of_their_own(T):
    """Two layers of one width, each in its first call: 64,000 pairs of fair coins agree in half, within five standard deviations."""
    from gfnerf_amd.gfnerf.mlp import Dropout

    x = T.ones(1000, 64, device="cuda")
    a, b = Dropout(0.5).cuda(), Dropout(0.5).cuda()
    masks = [m(x) != 0 for m in (a, b, a)]
    for p, q in ((0, 1), (0, 2), (1, 2)):
        assert abs(float((masks[p] == masks[q]).double().mean()) - 0.5) < 5 * 0.5 / 64000 ** 0.5


# ---- arguments of the autograd functions ------------------------------------------------------------------------------------------------------
def test_gated_linear_takes_parameters_of_any_strides(T):
    from gfnerf_amd.gfnerf.mlp import gated_linear

    x = T.randn(70, 24, device="cuda", requires_grad=True)
    wide = T.randn(24, 40, 2, device="cuda", requires_grad=True)
    flat = T.randn(40, 4, device="cuda", requires_grad=True)
    params = lambda: [wide[:, :, 0].t(), wide[:, :, 1].t(), flat[:, 1], flat[:, 3]]  # noqa: E731
    got = gated_linear(x, *params())
    want = gated_linear(x, *(p.contiguous() for p in params()))
    assert T.equal(got, want)
    g = T.randn(70, 40, device="cuda")
    for a, b in zip(T.autograd.grad(got, (x, wide, flat), g), T.autograd.grad(want, (x, wide, flat), g)):
        assert T.equal(a, b)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("act", ["silu", "gelu", "relu", "sigmoid"])
def test_an_undefined_gate_makes_its_features_gradients_undefined(T, ops, kind, act):
    """g of one feature is NaN: h, the gradients of that feature's weights and biases, and dx (a sum over all features) are; the other features' are not."""
    x, wg, wu, bg, bu, dh = gated_inputs(T, kind, 90, 20, 40, True, act)
    bad = bg[0].clone()
    bad[7] = float("nan")
    want = ops.gated_bwd(x[0], wg[0], wu[0], dh[0], bg[0], bu[0], act)
    dx, dwg, dwu, dbg, dbu = ops.gated_bwd(x[0], wg[0], wu[0], dh[0], bad, bu[0], act)
    h = ops.gated_fwd(x[0], wg[0], wu[0], bad, bu[0], act)
    rest = T.arange(40, device="cuda") != 7
    assert bool(T.isnan(h[:, 7]).all()) and bool(T.isfinite(h[:, rest]).all()) and bool(T.isnan(dx).all())
    for got, clean in zip((dwg, dwu, dbg, dbu), want[1:]):
        assert bool(T.isnan(got[7]).all()) and T.equal(got[rest], clean[rest])


@pytest.mark.parametrize("kind", KINDS)
def test_render_features_weighs_in_f32_whatever_the_features_type(T, kind):
    """The composite of 16-bit features is that of their f32 values: within the oracle's f32 bound of the 64-bit one, gradients of sigma and dt too."""
    from gfnerf_amd.gfnerf.ray_scan import render_features

    rng = np.random.default_rng(6)
    lens = rng.integers(0, 120, 40)
    off = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    n = int(off[-1])
    leaf = lambda v, k="f32": T.from_numpy(v).to(dt(T, k)).cuda().requires_grad_(True)  # noqa: E731
    sigma, delta, feats = leaf(rng.exponential(0.5, n)), leaf(rng.uniform(0.01, 0.2, n)), leaf(rng.standard_normal((n, 12)), kind)
    out = render_features(T.from_numpy(off).cuda(), sigma, delta, feats)
    g = T.from_numpy(rng.standard_normal((40, 12))).float().cuda()
    ds, dd, df = T.autograd.grad(out, (sigma, delta, feats), g)
    thick = sigma.detach() * delta.detach()  # the same f32 product
    wide = lambda t: t.detach().double().cpu().numpy()  # noqa: E731
    want = oseq.ray_scan(off, wide(thick)[:, None], wide(feats), "decay", True, "f32", None, np.zeros((n, 12)), wide(g))
    close(out.detach(), want["state"], "state")
    dthick, bound = (v[:, 0] for v in want["df"])
    for got, other, what in ((ds, delta, "sigma"), (dd, sigma, "dt")):
        o = wide(other)
        close(got, (dthick * o, bound * o + np.abs(dthick * o) * oseq.U), what)
    assert df.dtype == feats.dtype
    close(df, (want["dc"][0], oseq.rounded(want["dc"][0], want["dc"][1], kind)), "features")


def test_gated_f16_tiles_of_very_different_size_in_one_workgroups_run(T, ops):
    """dz of 2^35 in some tiles, whose dW passes f16 in column 0 and is nothing elsewhere, and of 2^-16 in the tiles that the same workgroups take before
    and behind them (more tiles than workgroups): the other columns are sums of the small tiles alone, and keep f16's precision."""
    n, k, h = 66000, 8, 32
    rng = np.random.default_rng(8)
    big = np.isin(np.arange(n) // 64, np.r_[0:256, 768:1032])
    x = np.where(big[:, None], np.eye(1, k) * 6e4, rng.standard_normal((n, k)) * 1e-2)
    x[~big, 0] = 0
    wg, wu, dh = rng.standard_normal((h, k)), rng.standard_normal((h, k)), rng.standard_normal((n, h)) * np.where(big, 1024.0, 2.0 ** -10)[:, None]
    wg[:, 0], wu[:, 0] = 600, 600
    x, wg, wu, dh = ((lambda t: (t.cuda(), t.double().numpy()))(T.from_numpy(v).to(T.float16)) for v in (x, wg, wu, dh))
    want = oseq.gated_bwd(x[1], wg[1], wu[1], dh[1], None, None, "relu", "f16")
    got = dict(zip(NAMES, ops.gated_bwd(x[0], wg[0], wu[0], dh[0], act="relu")))
    small = T.from_numpy(~big).cuda()
    close(got["dx"][small], tuple(v[~big] for v in want["dx"]), "dx")
    for name in ("dwg", "dwu"):
        value, bound = want[name]
        assert bool((~T.isfinite(got[name][:, 0])).any())
        v = got[name][:, 1:].double().cpu().numpy()
        # (the oracle's bound on dW holds the large tiles' share of the grid against the small ones' sums only where x is not zero)
        assert (np.abs(v - value[:, 1:]) <= bound[:, 1:]).all(), name
        assert np.linalg.norm(v - value[:, 1:]) <= 2.0 ** -11 * np.linalg.norm(value[:, 1:]) + 2.0 ** -25 * np.sqrt(v.size), name
