"""The sequence-head operators on the GPU -- the gated feed-forward layer, the gated recurrence along rays, dropout -- against their definitions in
64 bits (oracle/sequence.py).  A tolerance is the oracle's elementwise bound: what the kernels' roundings (f32 sums, operands of 16 bits, one
rounding of the result) can add, derived there; nothing is tuned."""
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


class Made:
    """Seeded tensors of one type, and the values they hold in 64 bits."""

    def __init__(self, T, kind, seed):
        self.T, self.kind, self.rng = T, kind, np.random.default_rng(seed)

    def normal(self, *shape, scale=1.0, grid=None, kind=None):
        v = self.rng.standard_normal(shape) * scale
        if grid:
            v = np.round(v * grid) / grid
        t = self.T.from_numpy(v).to(dt(self.T, kind or self.kind)).cuda()
        return t, t.double().cpu().numpy()


def close(got, want, what):
    value, bound = want
    g = got.double().cpu().numpy()
    assert g.shape == value.shape, what
    off = np.abs(g - value)
    bad = ~(off <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.size} values, worst {float((off / np.maximum(bound, 1e-300))[bad].max()):.3g} times the bound, at {np.argwhere(bad)[0]}"


def gated_inputs(T, kind, n, k, h, bias, act, seed=0):
    m = Made(T, kind, seed)
    grid = 8 if act == "relu" else None  # relu's kink: projections are exact multiples of 1/64, so 64 and 32 bits agree on their sign
    x, wg, wu = m.normal(n, k, grid=grid), m.normal(h, k, scale=1 if grid else k ** -0.5, grid=grid), m.normal(h, k, scale=1 if grid else k ** -0.5, grid=grid)
    bg, bu = (m.normal(h, grid=grid), m.normal(h, grid=grid)) if bias else ((None, None), (None, None))
    return x, wg, wu, bg, bu, m.normal(n, h)


GATED = [(1, 1, 1, True, "silu"), (2, 3, 5, False, "gelu"), (7, 63, 128, True, "silu"), (64, 128, 128, True, "gelu"), (129, 5, 33, True, "sigmoid"), (300, 17, 300, False, "relu"),
         (257, 128, 65, False, "silu"), (1000, 32, 64, True, "relu"), (515, 64, 256, True, "sigmoid"), (90, 97, 1000, True, "silu"), (4099, 33, 128, True, "gelu")]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,k,h,bias,act", GATED)
def test_gated_forward(T, ops, kind, n, k, h, bias, act):
    x, wg, wu, bg, bu, _ = gated_inputs(T, kind, n, k, h, bias, act)
    got = ops.gated_fwd(x[0], wg[0], wu[0], bg[0], bu[0], act)
    assert got.dtype == dt(T, kind)
    close(got, oseq.gated_fwd(x[1], wg[1], wu[1], bg[1], bu[1], act, kind), "h")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("k,h", [(63, 128), (128, 64), (8, 40)])
def test_gated_forward_of_many_samples(T, ops, kind, k, h):
    """The form for large batches (several sample groups a wave), with a ragged last tile; a strided sample of rows is compared."""
    n = 70001
    x, wg, wu, bg, bu, _ = gated_inputs(T, kind, n, k, h, True, "silu")
    got = ops.gated_fwd(x[0], wg[0], wu[0], bg[0], bu[0])
    rows = np.unique(np.concatenate([np.arange(0, n, 97), np.arange(n - 300, n)]))
    close(got[T.from_numpy(rows).cuda()], oseq.gated_fwd(x[1][rows], wg[1], wu[1], bg[1], bu[1], "silu", kind), "h")
    assert bool((got == ops.gated_fwd(x[0], wg[0], wu[0], bg[0], bu[0])).all())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,k,h,bias,act", GATED)
def test_gated_backward(T, ops, kind, n, k, h, bias, act):
    x, wg, wu, bg, bu, dh = gated_inputs(T, kind, n, k, h, bias, act)
    want = oseq.gated_bwd(x[1], wg[1], wu[1], dh[1], bg[1], bu[1], act, kind)
    got = dict(zip(("dx", "dwg", "dwu", "dbg", "dbu"), ops.gated_bwd(x[0], wg[0], wu[0], dh[0], bg[0], bu[0], act)))
    for name, w in want.items():
        close(got[name], w, name)
    assert bias or (got["dbg"] is None and got["dbu"] is None)
    again = ops.gated_bwd(x[0], wg[0], wu[0], dh[0], bg[0], bu[0], act)  # fixed order of every sum: the same bits
    assert all(a is None or bool((a == b).all()) for a, b in zip(again, got.values()))
    only = ops.gated_bwd(x[0], wg[0], wu[0], dh[0], bg[0], bu[0], act, need_dw=False)
    assert bool((only[0] == got["dx"]).all()) and only[1:] == (None,) * 4
    only = ops.gated_bwd(x[0], wg[0], wu[0], dh[0], bg[0], bu[0], act, need_dx=False)
    assert only[0] is None and all(a is None or bool((a == b).all()) for a, b in zip(only[1:], list(got.values())[1:]))


@pytest.mark.parametrize("kind", KINDS)
def test_gated_backward_of_many_samples(T, ops, kind):
    """More tiles than workgroups: every workgroup accumulates several.  The weights' gradients against a 64-bit product on the device."""
    n, k, h = 150007, 63, 128
    x, wg, wu, bg, bu, dh = gated_inputs(T, kind, n, k, h, True, "silu")
    got = ops.gated_bwd(x[0], wg[0], wu[0], dh[0], bg[0], bu[0])
    leaves = [t.double().requires_grad_(True) for t in (x[0], wg[0], wu[0], bg[0], bu[0])]
    g, u = T.nn.functional.linear(leaves[0], leaves[1], leaves[3]), T.nn.functional.linear(leaves[0], leaves[2], leaves[4])
    want = T.autograd.grad(T.nn.functional.silu(g) * u, leaves, dh[0].double())
    for name, a, b in zip(("dx", "dwg", "dwu", "dbg", "dbu"), got, want):
        # two independent roundings of half a step each (dz, the result) in the 2-norm: at most sqrt(2) half steps; f32: sums of 150007 products
        # in runs of a few hundred and 512 partials, at most 1e-6 of the norm
        rel = float((a.double() - b).norm() / b.norm())
        assert rel <= (1e-6 if kind == "f32" else 2 ** 0.5 * oseq.HALF[kind]), (name, rel)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("k", [8, 16, 31, 32, 33, 48, 64, 65, 80, 96, 100, 127, 128])
def test_gated_layer_of_every_width(T, ops, kind, k):
    """Each number of 64-byte units a row can have, whole and cut, with each number of feature blocks a workgroup keeps, whole and cut."""
    for n, h, bias, act in ((333, 32, True, "silu"), (130, 40, True, "gelu"), (333, 64, False, "sigmoid"), (200, 96, True, "silu"), (333, 128, True, "relu"), (150, 200, True, "silu")):
        x, wg, wu, bg, bu, dh = gated_inputs(T, kind, n, k, h, bias, act)
        close(ops.gated_fwd(x[0], wg[0], wu[0], bg[0], bu[0], act), oseq.gated_fwd(x[1], wg[1], wu[1], bg[1], bu[1], act, kind), "h")
        want = oseq.gated_bwd(x[1], wg[1], wu[1], dh[1], bg[1], bu[1], act, kind)
        for name, got in zip(("dx", "dwg", "dwu", "dbg", "dbu"), ops.gated_bwd(x[0], wg[0], wu[0], dh[0], bg[0], bu[0], act)):
            if name in want:
                close(got, want[name], (name, n, k, h))


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_gated_backward_loses_nothing_but_the_results_rounding(T, ops, kind):
    """The 16-bit gradients are their 64-bit values rounded, but for a few that lie next to the middle between two numbers.  What the products lose
    is at most half a step of dz's second operand: 2^-8 2^-8 = 2^-16 of a term in bf16; in f16, whose tile scale leaves terms of an ordinary size
    at 2^-9 and more, half a subnormal step, 2^-25 / 2^-9 = 2^-16 as well.  The terms' errors add up to A times that of the sum, A = norm of the
    terms over the sum: about 1 for terms of random sign, below 4 here.  A value within d of a middle may round the other way: of values spread
    evenly over a step (at least 2^-8, f16 2^-11 of the value) a share of 2 A d / step: 2 4 2^-16 / 2^-8 = 3.1 %, f16 25 %.  (With dz rounded
    to one operand, d is half a step and two values in five differ.)"""
    n, k, h = 3000, 40, 72
    x, wg, wu, bg, bu, dh = gated_inputs(T, kind, n, k, h, True, "silu")
    want = oseq.gated_bwd(x[1], wg[1], wu[1], dh[1], bg[1], bu[1], "silu", kind)
    for name, got in zip(("dx", "dwg", "dwu"), ops.gated_bwd(x[0], wg[0], wu[0], dh[0], bg[0], bu[0])):
        exact = T.from_numpy(np.ascontiguousarray(want[name][0])).to(got.dtype)  # rounded once
        differ = float((exact != got.cpu()).double().mean())
        assert differ <= (0.031 if kind == "bf16" else 0.25), (name, differ)


@pytest.mark.parametrize("scale", [2.0 ** -20, 2.0 ** 12])
def test_gated_backward_f16_follows_the_gradient_scale(T, ops, scale):
    """f16 gradients far from 1: what the two projections' gradients are rounded to follows the tile's largest |dh|, so the weights' gradients keep
    f16's precision where they are representable at all."""
    x, wg, wu, bg, bu, dh = gated_inputs(T, "f16", 3000, 32, 64, True, "silu")
    d = (dh[0] * scale).contiguous()
    want = oseq.gated_bwd(x[1], wg[1], wu[1], d.double().cpu().numpy(), bg[1], bu[1], "silu", "f16")
    for name, got in zip(("dx", "dwg", "dwu", "dbg", "dbu"), ops.gated_bwd(x[0], wg[0], wu[0], d, bg[0], bu[0])):
        v = got.double().cpu().numpy()
        if scale > 1 and not np.isfinite(want[name][0].astype(np.float16)).all():
            continue  # the result itself leaves f16
        close(got, want[name], name)
        assert np.linalg.norm(v - want[name][0]) <= 2 ** 0.5 * 2.0 ** -11 * np.linalg.norm(want[name][0]) + 2.0 ** -25 * np.sqrt(v.size)
    mixed = dh[0].clone()
    mixed[: 3000 // 2] *= 2.0 ** -12  # small tiles and large ones in one workgroup's run
    want = oseq.gated_bwd(x[1], wg[1], wu[1], mixed.double().cpu().numpy(), bg[1], bu[1], "silu", "f16")
    for name, got in zip(("dx", "dwg", "dwu", "dbg", "dbu"), ops.gated_bwd(x[0], wg[0], wu[0], mixed, bg[0], bu[0])):
        close(got, want[name], name)


@pytest.mark.parametrize("kind", KINDS)
def test_gated_rows_of_wider_buffers_and_live_counts(T, ops, kind):
    """x, dh and out as column ranges of wider buffers that hold NaN around them; rows behind the live count hold NaN and are not touched."""
    n, live, k, h = 300, 211, 31, 72
    x, wg, wu, bg, bu, dh = gated_inputs(T, kind, n, k, h, True, "gelu")
    xb, db = T.full((n, k + 9), float("nan"), dtype=x[0].dtype, device="cuda"), T.full((n, h + 5), float("nan"), dtype=x[0].dtype, device="cuda")
    xb[:live, 3:3 + k], db[:live, 1:1 + h] = x[0][:live], dh[0][:live]
    out = T.full((n, h + 7), 7.0, dtype=x[0].dtype, device="cuda")
    n_dev = T.tensor([live], dtype=T.int32, device="cuda")
    ops.gated_fwd(xb[:, 3:3 + k], wg[0], wu[0], bg[0], bu[0], "gelu", out=out[:, 2:2 + h], n_dev=n_dev)
    close(out[:live, 2:2 + h], oseq.gated_fwd(x[1][:live], wg[1], wu[1], bg[1], bu[1], "gelu", kind), "h")
    rest = out.clone()
    rest[:live, 2:2 + h] = 7.0
    assert bool((rest == 7.0).all())
    want = oseq.gated_bwd(x[1][:live], wg[1], wu[1], dh[1][:live], bg[1], bu[1], "gelu", kind)
    got = ops.gated_bwd(xb[:, 3:3 + k], wg[0], wu[0], db[:, 1:1 + h], bg[0], bu[0], "gelu", n_dev=n_dev)
    close(got[0][:live], want["dx"], "dx")
    for name, g in zip(("dwg", "dwu", "dbg", "dbu"), got[1:]):
        close(g, want[name], name)


def test_gated_empty_batch_and_refusals(T, ops):
    from gfnerf_amd import _lib

    z = lambda *s, d=T.float32: T.zeros(s, dtype=d, device="cuda")  # noqa: E731
    assert ops.gated_fwd(z(0, 8), z(16, 8), z(16, 8)).shape == (0, 16)
    w = T.ones(16, 8, device="cuda")
    dx, dwg, dwu, dbg, dbu = ops.gated_bwd(z(0, 8), w, w, z(0, 16), w[:, 0].contiguous(), w[:, 0].contiguous())
    assert dx.shape == (0, 8) and all(float(t.abs().max()) == 0 for t in (dwg, dwu, dbg, dbu))
    x, d = z(4, 8), z(4, 16)
    for bad in (lambda: ops.gated_fwd(x, w, w.half()), lambda: ops.gated_fwd(x, w, w[:8]), lambda: ops.gated_fwd(x, w.t().contiguous(), w), lambda: ops.gated_fwd(x, w, w, act="tanh"),
                lambda: ops.gated_fwd(x.double(), w.double(), w.double()), lambda: ops.gated_fwd(x, w, w, z(16)), lambda: ops.gated_fwd(x, w, w, out=z(4, 15)),
                lambda: ops.gated_fwd(x, w, w, z(16), z(15)), lambda: ops.gated_bwd(x, w, w, d[:3]), lambda: ops.gated_bwd(x, w, w, z(1, 16).expand(4, 16)),
                lambda: ops.gated_fwd(z(4, 129), z(16, 129), z(16, 129)), lambda: ops.gated_fwd(x.t(), z(16, 4), z(16, 4)), lambda: ops.gated_fwd(x[0], w, w),
                lambda: ops.gated_fwd(x, w, w, n_dev=T.zeros(1, dtype=T.int64, device="cuda")), lambda: ops.gated_fwd(z(8, 8), T.ones(8, 8, device="cuda"), w[:8], out=w[:8])):
        with pytest.raises(_lib.GfnError):
            bad()


def test_gated_values_that_are_not_finite_stay_in_their_rows(T, ops):
    """A NaN, an infinity or an overflowing value in one sample reaches that sample's outputs only; large negative gates give zeros, not NaN."""
    x, wg, wu, bg, bu, dh = gated_inputs(T, "f32", 200, 16, 48, True, "silu")
    clean = ops.gated_fwd(x[0], wg[0], wu[0], bg[0], bu[0])
    bad = x[0].clone()
    bad[17, 3], bad[18, 0], bad[19] = float("nan"), float("inf"), 1e38
    got = ops.gated_fwd(bad, wg[0], wu[0], bg[0], bu[0])
    keep = T.ones(200, dtype=T.bool, device="cuda")
    keep[17:20] = False
    assert bool((got[keep] == clean[keep]).all()) and bool(T.isnan(got[17]).all())
    dx = ops.gated_bwd(bad, wg[0], wu[0], dh[0], bg[0], bu[0], need_dw=False)[0]
    assert bool((dx[keep] == ops.gated_bwd(x[0], wg[0], wu[0], dh[0], bg[0], bu[0], need_dw=False)[0][keep]).all())
    for act in ("silu", "gelu", "relu", "sigmoid"):
        for kind in KINDS:
            one = T.ones(40, 1, dtype=dt(T, kind), device="cuda")
            far = one * T.tensor(-3e4, dtype=dt(T, kind), device="cuda")
            assert bool((ops.gated_fwd(far, one[:32], one[:32] * 0.5, act=act) == 0).all())
            assert bool((ops.gated_bwd(far, one[:32], one[:32] * 0.5, one.expand(40, 32).contiguous(), act=act)[0] == 0).all())


# ---- recurrence -------------------------------------------------------------------------------------------------------------------------------
SCANS = [([1], 1, 1), ([0], 5, 5), ([0, 0, 3, 0], 2, 1), ([1, 1, 1, 1, 1], 7, 7), ([16, 16, 32], 8, 8), ([1024, 1, 0, 17, 15, 16, 33, 255], 6, 3), ([300] * 5, 32, 1), ([5, 0, 700, 2], 64, 64),
         ([40, 41, 42], 130, 130), ([100, 3], 128, 2), ([9] * 70, 3, 1), ([2500], 4, 2), ([33, 64], 256, 1)]


def scan_inputs(T, kind, lens, d, g, gate, tail=3, seed=0):
    m = Made(T, kind, seed)
    off = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    n = int(off[-1]) + tail
    f = m.normal(n, g)
    if gate == "decay":
        t = (f[0].float() * 1.5 - 2).exp().to(f[0].dtype)
    elif gate == "linear":
        t = T.sigmoid(f[0].float() + 1).to(f[0].dtype)
    else:
        t = (f[0].float() + 1).to(f[0].dtype)
    f = (t, t.double().cpu().numpy())
    return T.from_numpy(off).cuda(), off, f, m.normal(n, d), m.normal(n, d), m.normal(len(lens), d, kind="f32"), m.normal(len(lens), d, kind="f32")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("gate", ["linear", "sigmoid", "decay"])
@pytest.mark.parametrize("lens,d,g", SCANS)
def test_ray_scan_forward_and_backward(T, ops, kind, gate, lens, d, g):
    offt, off, f, c, dh, h0, ds = scan_inputs(T, kind, lens, d, g, gate)
    for reverse in (False, True):
        for with_state in (False, True):
            a0, a1 = (h0, ds) if with_state else ((None, None), (None, None))
            want = oseq.ray_scan(off, f[1], c[1], gate, reverse, kind, a0[1], dh[1], a1[1])
            r = ops.ray_scan_fwd(offt, f[0], c[0], gate, reverse, a0[0], save=True)
            close(r["h"], want["h"], "h")
            close(r["state"], want["state"], "state")
            b = ops.ray_scan_bwd(offt, f[0], c[0], dh[0], r["saved"], gate, reverse, a0[0], a1[0])
            for name in ("df", "dc", "dh0"):
                close(b[name], want[name], name)
            assert bool((ops.ray_scan_fwd(offt, f[0], c[0], gate, reverse, a0[0])["h"] == r["h"]).all())  # saving changes nothing


@pytest.mark.parametrize("kind", KINDS)
def test_ray_scan_rows_of_wider_buffers_and_rows_behind_the_last_ray(T, ops, kind):
    lens, d, g = [13, 0, 50, 7], 12, 4
    offt, off, f, c, dh, h0, ds = scan_inputs(T, kind, lens, d, g, "sigmoid", tail=0)
    n = int(off[-1])
    nan = lambda w: T.full((n + 20, w), float("nan"), dtype=c[0].dtype, device="cuda")  # noqa: E731
    fb, cb, db, ob = nan(g + 3), nan(d + 1), nan(d + 5), nan(d + 2)
    fb[:n, 1:1 + g], cb[:n, :d], db[:n, 4:4 + d] = f[0], c[0], dh[0]
    ob.fill_(7.0)
    want = oseq.ray_scan(off, f[1], c[1], "sigmoid", False, kind, h0[1], dh[1], ds[1])
    r = ops.ray_scan_fwd(offt, fb[:, 1:1 + g], cb[:, :d], h0=h0[0], out=ob[:, 1:1 + d], save=True)
    close(ob[:n, 1:1 + d], want["h"], "h")
    ob[:n, 1:1 + d] = 7.0
    assert bool((ob == 7.0).all())  # the caller's rows behind the last ray and columns around are left alone
    b = ops.ray_scan_bwd(offt, fb[:, 1:1 + g], cb[:, :d], db[:, 4:4 + d], r["saved"], h0=h0[0], d_state=ds[0])
    for name in ("df", "dc"):
        close(b[name][:n], want[name], name)
        assert bool((b[name][n:] == 0).all())
    assert bool((ops.ray_scan_fwd(offt, fb[:, 1:1 + g], cb[:, :d])["h"][n:] == 0).all())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d,g", [(96, 96), (32, 1)])
def test_ray_scan_of_a_batch_of_rays(T, ops, kind, d, g):
    """2,000 ragged rays, compared on the device with the recurrence in 64 bits taken over all rays at once, row by row."""
    rng = np.random.default_rng(3)
    lens = rng.integers(0, 260, 2000)
    lens[::16] = 0
    lens[7] = 1024
    offt, off, f, c, dh, h0, ds = scan_inputs(T, kind, lens, d, g, "sigmoid")
    F, Cc, D = (T.from_numpy(v[1]).cuda() for v in (f, c, dh))
    A, R = T.sigmoid(F).repeat_interleave(d // g, 1), T.sigmoid(-F).repeat_interleave(d // g, 1)
    start, length = T.from_numpy(off[:-1].astype(np.int64)).cuda(), T.from_numpy(lens).cuda()
    s, h, before = h0[0].double().clone(), T.zeros_like(Cc), T.zeros_like(Cc)
    for i in range(int(lens.max())):
        at = (start + i)[length > i]
        before[at] = s[length > i]
        s[length > i] = A[at] * s[length > i] + R[at] * Cc[at]
        h[at] = s[length > i]
    lam, df, dc = ds[0].double().clone(), T.zeros_like(Cc), T.zeros_like(Cc)
    for i in reversed(range(int(lens.max()))):
        live = length > i
        at = (start + i)[live]
        lt = lam[live] + D[at]
        dc[at], df[at], lam[live] = lt * R[at], lt * (before[at] - Cc[at]) * A[at] * R[at], A[at] * lt
    r = ops.ray_scan_fwd(offt, f[0], c[0], h0=h0[0], save=True)
    b = ops.ray_scan_bwd(offt, f[0], c[0], dh[0], r["saved"], h0=h0[0], d_state=ds[0])
    for name, got, want in (("h", r["h"], h), ("state", r["state"], s), ("df", b["df"], df.view(-1, g, d // g).sum(2)), ("dc", b["dc"], dc), ("dh0", b["dh0"], lam)):
        # one rounding of half a step; f32: the errors of a chain that forgets with sigmoid(1 +- 1) add up to a few units, times 8 for the gate's own
        rel = float((got.double() - want).norm() / want.norm())
        assert rel <= (2e-6 if got.dtype == T.float32 else oseq.HALF[kind]), (name, rel)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d,g", [(96, 96), (32, 1), (10, 5), (256, 2)])
@pytest.mark.parametrize("reverse", [False, True])
def test_ray_scan_in_runs_with_many_rays_in_each(T, ops, kind, d, g, reverse):
    """Rays too few to fill the chip and long on average, but most of them short: runs of rows that several rays begin and end in, rays without
    rows among, before and behind them."""
    rng = np.random.default_rng(11)
    lens = np.where(rng.random(90) < 0.7, rng.integers(0, 9, 90), rng.integers(200, 700, 90))
    lens[:3], lens[-2:], lens[40:44] = 0, 0, (1, 0, 0, 8)
    assert lens.sum() > 100 * len(lens)
    offt, off, f, c, dh, h0, ds = scan_inputs(T, kind, lens, d, g, "sigmoid")
    want = oseq.ray_scan(off, f[1], c[1], "sigmoid", reverse, kind, h0[1], dh[1], ds[1])
    r = ops.ray_scan_fwd(offt, f[0], c[0], reverse=reverse, h0=h0[0], save=True)
    close(r["h"], want["h"], "h")
    close(r["state"], want["state"], "state")
    b = ops.ray_scan_bwd(offt, f[0], c[0], dh[0], r["saved"], reverse=reverse, h0=h0[0], d_state=ds[0])
    for name in ("df", "dc", "dh0"):
        close(b[name], want[name], name)


def test_ray_scan_composites_like_the_renderer(T, ops):
    """Back to front with the density's gate the recurrence is the framework's own compositing: three channels against gfn_composite_fwd / _bwd."""
    rng = np.random.default_rng(5)
    lens = rng.integers(0, 200, 300)
    off = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    n = int(off[-1])
    t = lambda a: T.from_numpy(a.astype(np.float32)).cuda()  # noqa: E731
    sigma, dtv, rgb, tt = t(rng.exponential(0.5, n)), t(rng.uniform(0.01, 0.2, n)), t(rng.random((n, 3))), t(np.arange(n) * 0.01)
    offt = T.from_numpy(off).cuda()
    want = ops.composite_fwd(offt, sigma, dtv, tt, rgb)["rgb"]
    from gfnerf_amd.gfnerf.ray_scan import render_features

    s, c = sigma.clone().requires_grad_(True), rgb.clone().requires_grad_(True)
    got = render_features(offt, s, dtv, c)
    # both are f32 sums of at most 200 terms of magnitude <= 1 with weights summing to <= 1; each weight is a product of up to 200 factors: 200 u 4
    assert float((got - want).abs().max()) <= 800 * 2.0 ** -24
    g = t(rng.standard_normal((300, 3)))
    got.backward(g)
    d_sigma, d_rgb = ops.composite_bwd(offt, sigma, dtv, rgb, g)
    assert float((c.grad - d_rgb).norm() / d_rgb.norm()) <= 1e-5 and float((s.grad - d_sigma).norm() / d_sigma.norm()) <= 1e-5


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("gate", ["linear", "sigmoid", "decay"])
@pytest.mark.parametrize("n,d,g", [(1, 1, 1), (5, 6, 3), (1000, 128, 128), (33, 96, 1)])
def test_ray_scan_step(T, ops, kind, gate, n, d, g):
    offt, off, f, c, _, h0, _ = scan_inputs(T, kind, [1] * n, d, g, gate, tail=0)
    want = oseq.ray_scan(off, f[1], c[1], gate, False, kind, h0[1])
    state = h0[0].clone()
    h = ops.ray_scan_step(f[0], c[0], state, gate)
    close(h, want["h"], "h")
    close(state, want["state"], "state")
    buf = T.full((n, d + 2), 7.0, dtype=c[0].dtype, device="cuda")
    state = h0[0].clone()
    ops.ray_scan_step(f[0], c[0], state, gate, out=buf[:, 1:1 + d])
    assert bool((buf[:, 1:1 + d] == h).all()) and bool((buf[:, 0] == 7).all()) and bool((buf[:, -1] == 7).all())


def test_ray_scan_carried_over_parts_is_the_whole(T, ops):
    """A ray taken in parts (its state carried) is the ray taken at once, bit for bit where the parts end on saved rows' borders."""
    offt, off, f, c, *_ = scan_inputs(T, "f32", [200, 200], 16, 16, "sigmoid", tail=0)
    whole = ops.ray_scan_fwd(offt, f[0], c[0])
    state, parts = None, []
    pick = lambda t, a, b: T.cat([t[a:b], t[200 + a:200 + b]]).contiguous()  # noqa: E731
    for a, b in ((0, 96), (96, 97), (97, 200)):
        o = T.tensor([0, b - a, 2 * (b - a)], dtype=T.int32, device="cuda")
        r = ops.ray_scan_fwd(o, pick(f[0], a, b), pick(c[0], a, b), h0=state)
        state = r["state"]
        parts.append(r["h"].view(2, b - a, 16))
    # |h| < 5; the parts' states are the same f32 numbers up to the order of a chain's multiply-adds: 200 steps of 2 u that fade
    assert float((T.cat(parts, 1).reshape(400, 16) - whole["h"]).abs().max()) <= 100 * 2.0 ** -24 * 5
    assert float((state - whole["state"]).abs().max()) <= 100 * 2.0 ** -24 * 5


def test_ray_scan_gates_at_their_ends(T, ops):
    """Gates that are exactly 0 or 1, infinite logits and opaque samples: nothing is divided, nothing becomes NaN; a NaN stays in its ray and channel."""
    off = T.tensor([0, 6, 12], dtype=T.int32, device="cuda")
    c = T.ones(12, 4, device="cuda")
    for gate, vals in (("sigmoid", [float("inf"), float("-inf"), 0.0, 100.0, -100.0, 1.0]), ("decay", [0.0, float("inf"), 1e-30, 100.0, 1e30, 0.5]), ("linear", [0.0, 1.0, 1.0, 0.0, 2.0, -1.0])):
        f = T.tensor(vals * 2, device="cuda")[:, None].expand(12, 4).contiguous()
        for reverse in (False, True):
            r = ops.ray_scan_fwd(off, f, c, gate, reverse, save=True)
            b = ops.ray_scan_bwd(off, f, c, c, r["saved"], gate, reverse)
            assert all(bool(T.isfinite(v).all()) for v in (r["h"], r["state"], b["df"], b["dc"], b["dh0"])), gate
    cn = c.clone()
    cn[2, 1] = float("nan")
    f = T.zeros(12, 4, device="cuda")
    r = ops.ray_scan_fwd(off, f, cn)
    hit = T.isnan(r["h"])
    assert bool(hit[2:6, 1].all()) and int(hit.sum()) == 4


def test_ray_scan_refusals(T, ops):
    from gfnerf_amd import _lib

    off = T.tensor([0, 4, 8], dtype=T.int32, device="cuda")
    f, c = T.zeros(8, 4, device="cuda"), T.zeros(8, 8, device="cuda")
    s = ops.ray_scan_fwd(off, f, c, save=True)["saved"]
    z = T.zeros(2, 8, device="cuda")
    for bad in (lambda: ops.ray_scan_fwd(off.long(), f, c), lambda: ops.ray_scan_fwd(off, f[:7], c), lambda: ops.ray_scan_fwd(off, f.half(), c), lambda: ops.ray_scan_fwd(off, f[:, :3], c),
                lambda: ops.ray_scan_fwd(off, f, c, gate="tanh"), lambda: ops.ray_scan_fwd(off, f, c, h0=z[:1]), lambda: ops.ray_scan_fwd(off, f, c, h0=z.half()),
                lambda: ops.ray_scan_fwd(off, f, c, out=c), lambda: ops.ray_scan_fwd(off, f, c, out=c.half()), lambda: ops.ray_scan_bwd(off, f, c, c, None),
                lambda: ops.ray_scan_bwd(off, f, c, c, s[:0]), lambda: ops.ray_scan_bwd(off, f, c, c[:, :4], s), lambda: ops.ray_scan_bwd(off, f, c, c, s, d_state=z[0]),
                lambda: ops.ray_scan_step(f, c, z), lambda: ops.ray_scan_step(f[:2], c[:2], z.half()), lambda: ops.ray_scan_step(f[:2], c[:2], None),
                lambda: ops.ray_scan_fwd(off, f[:, :1].expand(8, 4), c)):
        with pytest.raises(_lib.GfnError):
            bad()
    empty = ops.ray_scan_fwd(T.zeros(1, dtype=T.int32, device="cuda"), f[:0], c[:0], save=True)
    assert empty["h"].shape == (0, 8) and empty["state"].shape == (0, 8)


# ---- dropout ------------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,d,p", [(1, 1, 0.5), (3, 8, 0.1), (1000, 63, 0.5), (257, 128, 0.9), (40, 1024, 0.3), (5, 17, 0.0), (5, 16, 1.0), (70, 9, 1e-6)])
def test_dropout_is_the_published_generator(T, ops, kind, n, d, p):
    x, v = Made(T, kind, 1).normal(n, d)
    seed, call = 0x1234567890ABCDEF, T.tensor([(5 << 32) + 77], dtype=T.int64, device="cuda")
    keep, factor = oseq.dropout_mask(n, d, p, seed, (5 << 32) + 77)
    want = T.where(T.from_numpy(keep), x.float().cpu() * float(factor), T.zeros(())).to(dt(T, kind))
    got = ops.dropout(x, p, seed, call)
    assert T.equal(got.cpu(), want)
    wide = T.full((n, d + 3), 7.0, dtype=x.dtype, device="cuda")
    wide[:, 1:1 + d] = x
    ops.dropout(wide[:, 1:1 + d], p, seed, call, out=wide[:, 1:1 + d])  # in place, rows at another stride and alignment: the same elements
    assert T.equal(wide[:, 1:1 + d].cpu(), want) and bool((wide[:, 0] == 7).all()) and bool((wide[:, 1 + d:] == 7).all())
    bad = x.clone()
    bad[~T.from_numpy(keep).cuda()] = float("nan")  # dropped elements are zeros, not products
    assert T.equal(ops.dropout(bad, p, seed, call).cpu(), want)


def test_dropout_calls_count_on_the_device(T, ops):
    from gfnerf_amd import _lib

    counter = T.zeros(1, dtype=T.int64, device="cuda")
    assert [int(ops.dropout_call(counter)) for _ in range(3)] == [0, 1, 2] and int(counter) == 3
    x = T.ones(1000, 64, device="cuda")
    masks = [ops.dropout(x, 0.5, 1, ops.dropout_call(counter)) != 0 for _ in range(2)]
    assert 0.45 < float((masks[0] == masks[1]).float().mean()) < 0.55
    for bad in (lambda: ops.dropout(x, 1.5, 1, counter), lambda: ops.dropout(x, 0.5, 1, counter.int()), lambda: ops.dropout(x, 0.5, 1, None), lambda: ops.dropout_call(counter.float()),
                lambda: ops.dropout(x.double(), 0.5, 1, counter), lambda: ops.dropout(x, 0.5, 1, counter, out=x[:5])):
        with pytest.raises(_lib.GfnError):
            bad()
    assert ops.dropout(x[:0], 0.5, 1, counter).shape == (0, 64)


# ---- together -------------------------------------------------------------------------------------------------------------------------------------
def head(T, seed=0, dropout=0.25, dim=24):
    from gfnerf_amd.gfnerf.mlp import GatedMLPNetwork
    from gfnerf_amd.gfnerf.ray_scan import RayRecurrence

    T.manual_seed(seed)
    net = GatedMLPNetwork(31, 20, {"activation": "SwiGLU", "output_activation": "None", "n_neurons": 48, "n_hidden_layers": 2, "dropout": dropout}).cuda()
    return net, RayRecurrence(20, dim).cuda()


def rays_batch(T, seed=0):
    rng = np.random.default_rng(seed)
    lens = rng.integers(0, 90, 60)
    off = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    return T.from_numpy(off).cuda(), T.from_numpy(rng.standard_normal((int(off[-1]), 31)).astype(np.float32)).cuda()


def plain_head(T, net, rec, off, x, calls):
    """The same head in 64-bit torch: linear layers, silu, the published mask, the recurrence ray by ray."""
    v, lin = x.double(), lambda l, a: T.nn.functional.linear(a, l.weight.double(), l.bias.double())  # noqa: E731
    for i in range(net.n_hidden_layers):
        layer = net.layers[i]
        v = T.nn.functional.silu(lin(layer.gate, v)) * lin(layer.up, v)
        keep, factor = oseq.dropout_mask(v.shape[0], v.shape[1], net.dropout[i].p, net.dropout[i].seed, calls)
        v = v * T.from_numpy(keep).cuda() * float(factor)
    v = lin(net.layers[-1], v)
    a, c = T.sigmoid(lin(rec.gate, v)), lin(rec.input, v)
    rows = []
    o = off.cpu().tolist()
    for s, e in zip(o, o[1:]):
        h = T.zeros(c.shape[1], dtype=T.float64, device="cuda")
        for t in range(s, e):
            h = a[t] * h + (1 - a[t]) * c[t]
            rows.append(h)
    return T.stack(rows)


def test_head_along_rays_trains_like_its_definition(T):
    """Gated layers, dropout and the recurrence together: values and every parameter's gradient against 64-bit torch."""
    net, rec = head(T)
    off, x = rays_batch(T)
    x.requires_grad_(True)
    h, _ = rec(net(x), off)
    w = T.randn(h.shape, generator=T.Generator().manual_seed(1)).cuda()
    params = [x] + list(net.parameters()) + list(rec.parameters())
    got = T.autograd.grad((h * w).sum(), params)
    want_h = plain_head(T, net, rec, off, x, calls=0)
    want = T.autograd.grad((want_h * w.double()).sum(), params)
    # five f32 layers in a row, each within a few units of its sums of at most 90 products: 1e-5 of the norm is 170 units
    assert float((h.double() - want_h).norm() / want_h.norm()) <= 1e-5
    for i, (a, b) in enumerate(zip(got, want)):
        assert float((a.double() - b.double()).norm() / b.double().norm()) <= 1e-5, i
    assert int(net.dropout[0].counter) == 1
    net.eval()
    assert T.equal(net(x.detach()), net(x.detach())) and int(net.dropout[0].counter) == 1


def test_head_steps_sample_by_sample_like_the_whole_ray(T):
    net, rec = head(T, dropout=0.0)
    x = T.randn(50 * 7, 31, generator=T.Generator().manual_seed(2)).cuda()  # 50 rays of 7 samples
    off = T.arange(0, 351, 7, dtype=T.int32, device="cuda")
    with T.no_grad():
        h, state = rec(net(x), off)
        s = T.zeros(50, 24, device="cuda")
        for i in range(7):
            step = rec.step(net(x.view(50, 7, 31)[:, i]), s)
            assert float((step - h.view(50, 7, 24)[:, i]).abs().max()) <= 1e-5  # |h| of a few, f32 products in another order: some 20 units
    assert float((s - state).abs().max()) <= 1e-5


def test_head_captured_and_replayed(T):
    """A training step of the head (forward, backward) captured once and replayed: fresh masks each time, and every replay is the eager step of the
    same call number bit for bit; eager work of the same modules runs between the replays."""
    net, rec = head(T)
    off, x = rays_batch(T)
    params = list(net.parameters()) + list(rec.parameters())
    w = T.randn(x.shape[0], 24, generator=T.Generator().manual_seed(1)).cuda()

    linear = {id(p) for m in (net.layers[-1], rec) for p in m.parameters()}

    def step():
        h, _ = rec(net(x), off)
        return [h] + list(T.autograd.grad(h, params, w))

    def same(p, a, b):
        # gfn_linear_bwd adds its workgroups' f32 partial sums of dW with atomics, in any order: ceil(n / 64) < 64 of them, each addition within u of
        # the partial sum, whose norm is at most the sum of the partials' norms -- below 64 u = 4e-6 of that sum, itself within a small factor of
        # the result's norm for the random signs here: 1e-4 of it is far beyond.  Everything else of the step repeats its bits
        return float((a - b).norm() / b.norm()) <= 1e-4 if id(p) in linear else T.equal(a, b)

    def at(call):
        for m in net.dropout:
            m.counter.fill_(call)

    side = T.cuda.Stream()
    side.wait_stream(T.cuda.current_stream())
    with T.cuda.stream(side):
        step()
    T.cuda.current_stream().wait_stream(side)
    T.cuda.synchronize()
    eager = []
    for call in range(4):
        at(call)
        eager.append([t.detach().clone() for t in step()])
    at(0)
    g = T.cuda.CUDAGraph()
    with T.cuda.graph(g):
        out = step()
    at(0)
    for call in range(4):
        g.replay()
        T.cuda.synchronize()
        assert all(same(p, a, b) for p, a, b in zip([None] + params, out, eager[call])), call
        keep = [m.counter.clone() for m in net.dropout]
        at(9)
        step()  # eager work between the replays
        T.cuda.synchronize()
        for m, k in zip(net.dropout, keep):
            m.counter.copy_(k)
    assert not T.equal(eager[0][0], eager[1][0])


def test_a_capture_beside_a_live_eager_graph_is_refused(T):
    """The leaves' gradient accumulators belong to the eager graph's stream: a backward captured now would end the process.  The forward raises."""
    from gfnerf_amd import _lib

    net, rec = head(T)
    off, x = rays_batch(T)
    h, _ = rec(net(x), off)
    with pytest.raises(_lib.GfnError, match="eager autograd graph"):
        with T.cuda.graph(T.cuda.CUDAGraph()):
            net(x)
    T.cuda.synchronize()
    del h
    with T.no_grad():  # inference has no accumulators
        h = net(x)
        with T.cuda.graph(T.cuda.CUDAGraph()):
            net(x)


def test_a_capture_of_a_recurrence_beside_its_live_eager_graph_is_refused(T):
    """The same for a recurrence on its own: its projections' parameters are the leaves."""
    from gfnerf_amd import _lib
    from gfnerf_amd.gfnerf.ray_scan import RayRecurrence

    rec = RayRecurrence(8, 16).cuda()
    off = T.tensor([0, 5, 9], dtype=T.int32, device="cuda")
    x = T.ones(9, 8, device="cuda")
    h, state = rec(x, off)
    with pytest.raises(_lib.GfnError, match="eager autograd graph"):
        with T.cuda.graph(T.cuda.CUDAGraph()):
            rec(x, off)
    T.cuda.synchronize()
    del h
    with pytest.raises(_lib.GfnError, match="eager autograd graph"):  # the state is an output as well
        with T.cuda.graph(T.cuda.CUDAGraph()):
            rec(x, off)
    T.cuda.synchronize()
    del state
    with T.cuda.graph(T.cuda.CUDAGraph()):
        rec(x, off)
    T.cuda.synchronize()


def test_operators_on_a_stream_of_their_own(T, ops):
    """Two streams at once, each with its own calls and workspaces: the results are the default stream's."""
    ins = [gated_inputs(T, "bf16", 20000, 63, 128, True, "silu", seed=s) for s in (0, 1)]
    want = [ops.gated_bwd(i[0][0], i[1][0], i[2][0], i[5][0], i[3][0], i[4][0]) for i in ins]
    T.cuda.synchronize()
    streams = [T.cuda.Stream(), T.cuda.Stream()]
    got = []
    for s, i in zip(streams, ins):
        with T.cuda.stream(s):
            got.append(ops.gated_bwd(i[0][0], i[1][0], i[2][0], i[5][0], i[3][0], i[4][0]))
    T.cuda.synchronize()
    assert all(T.equal(a, b) for x, y in zip(got, want) for a, b in zip(x, y))


def test_offsets_past_32_bits(T, ops):
    """More than 2^31 elements in one tensor: the last rows come out as in a small call."""
    n, d = 2_200_000, 1000
    x = T.empty(n, d, dtype=T.bfloat16, device="cuda")
    x[-300:] = T.randn(300, d, device="cuda").bfloat16()
    x[:-300] = 0
    call = T.tensor([3], dtype=T.int64, device="cuda")
    y = ops.dropout(x, 0.5, 11, call)
    keep, factor = oseq.dropout_mask(300, d, 0.5, 11, 3, first_row=n - 300)
    assert T.equal(y[-300:].cpu(), T.where(T.from_numpy(keep), x[-300:].float().cpu() * float(factor), T.zeros(())).bfloat16())
    del y
    off = T.tensor([0, n - 200, n], dtype=T.int32, device="cuda")
    f = T.full((n, 20), 0.5, dtype=T.bfloat16, device="cuda")  # 50 channels a gate
    small = ops.ray_scan_fwd(T.tensor([0, 200], dtype=T.int32, device="cuda"), f[-200:], x[-200:], save=True)
    r = ops.ray_scan_fwd(off, f, x, save=True)
    # the rows meet other tiles' borders in the two calls: f32 states a few units apart, of which a few round to the next bf16 number (2^-7 away)
    near = lambda p, q: float((p.float() - q.float()).norm() / q.float().norm()) <= oseq.HALF["bf16"]  # noqa: E731
    assert near(r["h"][-200:], small["h"]) and float((r["state"][1:] - small["state"]).norm() / small["state"].norm()) <= 1e-6
    want = ops.ray_scan_bwd(T.tensor([0, 200], dtype=T.int32, device="cuda"), f[-200:], x[-200:], x[-200:], small["saved"])
    b = ops.ray_scan_bwd(off, f, x, x, r["saved"])
    assert near(b["df"][-200:], want["df"]) and near(b["dc"][-200:], want["dc"])
    del r, b, x, f
    w = T.randn(1000, 8, device="cuda").bfloat16()
    z = T.randn(n, 8, device="cuda").bfloat16()
    h = ops.gated_fwd(z, w, w)
    assert T.equal(h[-64:], ops.gated_fwd(z[-64:], w, w))
    dx, dwg, _, _, _ = ops.gated_bwd(z, w, w, h)
    assert T.equal(dx[-64:], ops.gated_bwd(z[-64:], w, w, h[-64:], need_dw=False)[0]) and bool(T.isfinite(dwg).all())
