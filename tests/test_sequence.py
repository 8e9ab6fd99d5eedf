"""The sequence-head operators without a GPU: their refusals (through the tensor front-end and through the C ABI), the modules' arguments, and the
oracle the GPU tests compare with (oracle/sequence.py) against published values and finite differences."""
import ctypes as C

import numpy as np
import pytest

from helpers import ROOT  # noqa: F401  (puts oracle/ on the path)

import sequence as oseq


@pytest.fixture(scope="module")
def lib():
    import gfnerf_amd  # noqa: F401
    from gfnerf_amd import _lib

    return _lib


P = C.c_void_p(4096)  # a pointer no call below gets as far as using


def refused(lib, name, *args, match):
    rc = getattr(lib.lib(), name)(*args)
    assert rc == -1, (name, rc)
    text = lib.lib().gfn_last_error().decode()
    assert match in text, text


def gated_fwd_args(**k):
    a = dict(x=P, ldx=63, wg=P, wu=P, bg=P, bu=P, n=100, n_dev=None, k=63, h=128, dtype=1, act=0, out=P, ldo=128, st=None)
    return list({**a, **k}.values())


@pytest.mark.parametrize("change,match", [
    (dict(k=0), "dims"), (dict(k=129, ldx=129), "dims"), (dict(h=0), "dims"), (dict(h=1025, ldo=1025), "dims"), (dict(n=-1), "n_max"), (dict(n=1 << 31), "n_max"),
    (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(act=4), "act"), (dict(act=-1), "act"), (dict(x=None), "null"), (dict(wg=None), "null"), (dict(wu=None), "null"),
    (dict(out=None), "null"), (dict(bg=None), "one bias"), (dict(bu=None), "one bias"), (dict(ldx=62), "row strides"), (dict(ldo=127), "row strides")])
def test_gated_fwd_refuses(lib, change, match):
    refused(lib, "gfn_gated_fwd", *gated_fwd_args(**change), match=match)


def gated_bwd_args(**k):
    a = dict(x=P, ldx=63, wg=P, wu=P, bg=P, bu=P, dh=P, lddh=128, n=100, n_dev=None, k=63, h=128, dtype=1, act=0, dx=P, lddx=63, dwg=P, dwu=P, dbg=P, dbu=P, ws=P,
             size=1 << 40, st=None)
    return list({**a, **k}.values())


@pytest.mark.parametrize("change,match", [
    (dict(k=129, ldx=129), "dims"), (dict(h=1025), "dims"), (dict(x=None), "null"), (dict(dh=None), "null"), (dict(bg=None), "one bias"), (dict(dwg=None), "one weight"),
    (dict(dbg=None), "biases' gradients"), (dict(bg=None, bu=None), "biases' gradients"), (dict(dwg=None, dwu=None), "biases' gradients"), (dict(lddh=127), "row stride"),
    (dict(lddx=62), "row stride"), (dict(size=16), "workspace of 16"), (dict(ws=None), "workspace"), (dict(dtype=7), "dtype")])
def test_gated_bwd_refuses(lib, change, match):
    refused(lib, "gfn_gated_bwd", *gated_bwd_args(**change), match=match)


def test_gated_workspace_is_a_function_of_the_sizes(lib):
    f = lib.lib().gfn_gated_bwd_workspace
    assert f(1000, 63, 128, 1, 1, 1, 0) == 0                       # one feature block: dx needs none
    assert f(1000, 63, 1000, 1, 1, 1, 0) == 1000 * 63 * 4          # several: the partial sums of dx
    assert f(0, 63, 128, 1, 1, 1, 1) > 0 and f(1 << 20, 63, 128, 1, 1, 1, 1) == f(1 << 21, 63, 128, 1, 1, 1, 1)  # dW: by workgroup, not by sample
    assert f(100, 0, 128, 1, 1, 1, 1) == -1


def scan_args(**k):
    a = dict(off=P, rays=10, f=P, ldf=8, c=P, ldc=32, n=100, d=32, g=8, dtype=0, gate=1, rev=0, h0=None, h=P, ldh=32, state=P, saved=None, tail=0, ws=None, size=0, st=None)
    return list({**a, **k}.values())


@pytest.mark.parametrize("change,match", [
    (dict(d=0), "gates for"), (dict(d=4097, ldc=4097), "gates for"), (dict(g=0), "gates for"), (dict(g=5), "gates for"), (dict(g=64, ldf=64), "gates for"),
    (dict(rays=-1), "rays"), (dict(n=1 << 31), "n_max"), (dict(dtype=3), "dtype"), (dict(gate=3), "gate 3"),
    (dict(off=None), "null"), (dict(f=None), "null"), (dict(c=None), "null"), (dict(h=None), "null"), (dict(ldf=7), "row stride"), (dict(ldc=31), "row stride"),
    (dict(ldh=31), "row stride")])
def test_ray_scan_fwd_refuses(lib, change, match):
    refused(lib, "gfn_ray_scan_fwd", *scan_args(**change), match=match)


def scan_bwd_args(**k):
    a = dict(off=P, rays=10, f=P, ldf=8, c=P, ldc=32, dh=P, lddh=32, n=100, d=32, g=8, dtype=0, gate=1, rev=0, h0=None, ds=None, saved=P, df=P, lddf=8, dc=P, lddc=32, dh0=None,
             tail=0, ws=None, size=0, st=None)
    return list({**a, **k}.values())


@pytest.mark.parametrize("change,match", [(dict(saved=None), "null"), (dict(df=None), "null"), (dict(dc=None), "null"), (dict(lddf=7), "row stride"),
                                          (dict(lddc=31), "row stride"), (dict(lddh=31), "row stride"), (dict(g=3), "gates for")])
def test_ray_scan_bwd_refuses(lib, change, match):
    refused(lib, "gfn_ray_scan_bwd", *scan_bwd_args(**change), match=match)


def test_ray_scan_workspace(lib):
    f = lib.lib().gfn_ray_scan_workspace
    assert f(10, 100, 32, 8) == 0 and f(10, 0, 32, 8) == 0            # short rays need none
    assert f(10, 100000, 32, 8) > 0 and f(1, 1 << 20, 128, 128) > 0
    assert f(10, 100, 0, 1) == -1 and f(10, 100, 32, 5) == -1
    refused(lib, "gfn_ray_scan_fwd", *scan_args(rays=10, n=100000), match="workspace of 0")
    refused(lib, "gfn_ray_scan_bwd", *scan_bwd_args(rays=10, n=100000, ws=P, size=64), match="workspace of 64")


def test_ray_scan_step_and_dropout_refuse(lib):
    refused(lib, "gfn_ray_scan_step", P, 8, P, 32, 10, 32, 8, 0, 1, None, P, 32, None, match="null")
    refused(lib, "gfn_ray_scan_step", P, 8, P, 32, 10, 32, 7, 0, 1, P, P, 32, None, match="gates for")
    refused(lib, "gfn_ray_scan_step", P, 8, P, 32, 10, 32, 8, 0, 1, P, P, 31, None, match="row stride")
    for p in (-0.1, 1.1, float("nan")):
        refused(lib, "gfn_dropout", P, 8, 4, 8, 0, p, 1, P, P, 8, None, match="not in [0, 1]")
    refused(lib, "gfn_dropout", P, 8, 4, 8, 0, 0.5, 1, None, P, 8, None, match="null")
    refused(lib, "gfn_dropout", P, 7, 4, 8, 0, 0.5, 1, P, P, 8, None, match="row stride")
    refused(lib, "gfn_dropout", P, 8, -1, 8, 0, 0.5, 1, P, P, 8, None, match="rows")
    refused(lib, "gfn_dropout", P, 8, 4, 8, 5, 0.5, 1, P, P, 8, None, match="dtype")
    refused(lib, "gfn_dropout_call", None, P, None, match="null")


def test_nothing_to_do_is_not_an_error(lib):
    assert lib.lib().gfn_gated_fwd(*gated_fwd_args(n=0, x=None, out=None)) == 0
    assert lib.lib().gfn_gated_bwd(*gated_bwd_args(dx=None, dwg=None, dwu=None, dbg=None, dbu=None, bg=None, bu=None)) == 0
    assert lib.lib().gfn_gated_bwd(*gated_bwd_args(n=0, dwg=None, dwu=None, dbg=None, dbu=None, bg=None, bu=None)) == 0
    assert lib.lib().gfn_ray_scan_fwd(*scan_args(rays=0, n=0, f=None, c=None, h=None)) == 0
    assert lib.lib().gfn_dropout(None, 0, 0, 8, 0, 0.5, 1, None, None, 0, None) == 0


def test_the_front_end_refuses_cpu_tensors_and_wrong_arguments(lib):
    import torch

    from gfnerf_amd import ops
    from gfnerf_amd.gfnerf.mlp import Dropout, GatedMLPNetwork
    from gfnerf_amd.gfnerf.ray_scan import RayRecurrence

    x, w = torch.zeros(4, 8), torch.zeros(16, 8)
    off = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(lib.GfnError, match="CUDA"):
        ops.gated_fwd(x, w, w)
    with pytest.raises(lib.GfnError, match="CUDA"):
        ops.gated_bwd(x, w, w, torch.zeros(4, 16))
    with pytest.raises(lib.GfnError, match="CUDA"):
        ops.ray_scan_fwd(off, x, x)
    with pytest.raises(lib.GfnError, match="CUDA"):
        ops.ray_scan_bwd(off, x, x, x, x)
    with pytest.raises(lib.GfnError, match="CUDA"):
        ops.ray_scan_step(x, x, x)
    with pytest.raises(lib.GfnError, match="CUDA"):
        ops.dropout(x, 0.5, 1, torch.zeros(1, dtype=torch.int64))
    with pytest.raises(lib.GfnError, match="CUDA"):
        ops.dropout_call(torch.zeros(1, dtype=torch.int64))
    with pytest.raises(ValueError, match="activation"):
        GatedMLPNetwork(32, 3, {"activation": "ReLU", "output_activation": "None", "n_neurons": 64, "n_hidden_layers": 1})
    with pytest.raises(ValueError, match="not in"):
        Dropout(1.5)
    with pytest.raises(ValueError, match="no next sample"):
        RayRecurrence(8, 16, reverse=True).step(x, torch.zeros(4, 16))
    net = GatedMLPNetwork(63, 3, {"activation": "SwiGLU", "output_activation": "Sigmoid", "n_neurons": 128, "n_hidden_layers": 2, "dropout": 0.1})
    assert sum(p.numel() for p in net.parameters()) == 2 * (63 * 128 + 128) + 2 * (128 * 128 + 128) + 128 * 3 + 3
    assert Dropout(0.5).eval()(x) is x and Dropout(0.0)(x) is x  # nothing to draw


# ---- the oracle itself --------------------------------------------------------------------------------------------------------------------
def test_oracle_philox_known_answers():
    """Published known answers of Philox4x32-10 (Random123's test vectors)."""
    for ctr, key, want in (((0, 0, 0, 0), (0, 0), "6627e8d5 e169c58d bc57ac4c 9b00dbd8"),
                           ((0xffffffff,) * 4, (0xffffffff,) * 2, "408f276d 41c83b0e a20bc7c6 6d5451fd"),
                           ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0), "d16cfe09 94fdcceb 5001e420 24126ea1")):
        got = oseq.philox(np.array(ctr, np.uint32), key)
        assert " ".join("%08x" % v for v in got) == want
    keep, factor = oseq.dropout_mask(2000, 100, 0.25, seed=9, call=4)
    assert factor == np.float32(4 / 3) and abs(keep.mean() - 0.75) < 5 * np.sqrt(0.25 * 0.75 / keep.size)


def difference(fn, v, g, eps=1e-6):
    """sum(g * d fn / d v[i]) for every i by central differences."""
    out = np.zeros_like(v)
    for i in np.ndindex(v.shape):
        a, b = v.copy(), v.copy()
        a[i] += eps
        b[i] -= eps
        out[i] = ((fn(a) - fn(b)) * g).sum() / (2 * eps)
    return out


@pytest.mark.parametrize("kind", ["silu", "gelu", "relu", "sigmoid"])
def test_oracle_gated_gradient_against_differences(kind):
    rng = np.random.default_rng(0)
    x, wg, wu, bg, bu, dh = (rng.standard_normal(s) for s in ((4, 3), (5, 3), (5, 3), (5,), (5,), (4, 5)))
    got = oseq.gated_bwd(x, wg, wu, dh, bg, bu, kind, "f32")
    f = lambda **k: oseq.gated_fwd(**{**dict(x=x, wg=wg, wu=wu, bg=bg, bu=bu, kind=kind, dtype="f32"), **k})[0]  # noqa: E731
    for name, v in (("x", x), ("wg", wg), ("wu", wu), ("bg", bg), ("bu", bu)):
        np.testing.assert_allclose(got["d" + name][0], difference(lambda a: f(**{name: a}), v, dh), rtol=1e-6, atol=1e-8)


@pytest.mark.parametrize("kind", ["linear", "sigmoid", "decay"])
@pytest.mark.parametrize("reverse", [False, True])
def test_oracle_recurrence_gradient_against_differences(kind, reverse):
    rng = np.random.default_rng(1)
    off = [0, 3, 3, 4, 9]
    f, c, dh = rng.standard_normal((9, 2)), rng.standard_normal((9, 4)), rng.standard_normal((9, 4))
    h0, ds = rng.standard_normal((4, 4)), rng.standard_normal((4, 4))
    if kind == "decay":
        f = np.abs(f)
    got = oseq.ray_scan(off, f, c, kind, reverse, "f32", h0, dh, ds)

    def fn(f=f, c=c, h0=h0):
        r = oseq.ray_scan(off, f, c, kind, reverse, "f32", h0)
        return np.concatenate([r["h"][0].ravel(), r["state"][0].ravel()])

    g = np.concatenate([dh.ravel(), ds.ravel()])
    for name, v in (("f", f), ("c", c), ("h0", h0)):
        np.testing.assert_allclose(got["d" + name][0], difference(lambda a: fn(**{name: a}), v, g), rtol=1e-6, atol=1e-8)
