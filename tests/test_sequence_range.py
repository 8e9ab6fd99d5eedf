"""The sequence-head operators without a GPU, where their numbers end: what the oracle's bounds let through, and calls whose outputs
overlap their inputs, the first call of two threads at once, and the dropout module's masks."""
import ctypes as C
import os
import subprocess

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


# ---- outputs that overlap inputs: refused before anything is launched ------------------------------------------------------------------------
def at(byte):
    return C.c_void_p((1 << 40) + byte)


FAR = {name: at((i + 1) << 30) for i, name in enumerate(("x", "wg", "wu", "bg", "bu", "dh", "f", "c", "h0", "off", "saved", "out"))}


def refused(name, *args, match):
    import gfnerf_amd  # noqa: F401
    from gfnerf_amd import _lib

    assert getattr(_lib.lib(), name)(*args) == -1
    assert match in _lib.lib().gfn_last_error().decode(), _lib.lib().gfn_last_error().decode()


@pytest.mark.parametrize("x,ldx,out,ldo,match", [
    (at(0), 63, at(100 * 63 * 4 - 4), 128, "out overlaps x"),         # its last element
    (at(128 * 99 * 4 + 127 * 4), 63, at(0), 128, "out overlaps x"),    # out's last element is x's first
    (at(0), 200, at(62 * 4), 200, "out overlaps x"),                  # columns 0 .. 62 and 62 .. 189 of one buffer
    (at(0), 200, at(100 * 4), 200, "out overlaps x"),                 # columns 100 .. 227: the next row's first
    (at(0), 200, at(63 * 4 + 200 * 4 * 50), 201, "out overlaps x"),   # another stride inside the same extent
    (FAR["x"], 63, at((2 << 30) + 8), 128, "out overlaps wg"), (FAR["x"], 63, at((3 << 30) - 128 * 4 * 100 + 4), 128, "out overlaps wu"),
    (FAR["x"], 63, at((4 << 30) + 127 * 4), 128, "out overlaps bg"), (FAR["x"], 63, at(5 << 30), 128, "out overlaps bu")])
def test_gated_fwd_refuses_overlap(x, ldx, out, ldo, match):
    refused("gfn_gated_fwd", x, ldx, FAR["wg"], FAR["wu"], FAR["bg"], FAR["bu"], 100, None, 63, 128, 0, 0, out, ldo, None, match=match)


@pytest.mark.parametrize("change,match", [(dict(dx=FAR["x"]), "dx overlaps x"), (dict(dx=at((6 << 30) + 4)), "dx overlaps dh"), (dict(dwg=FAR["wg"]), "dwg overlaps wg"),
                                          (dict(dwu=at((20 << 30) + 4)), "dwu overlaps dwg"), (dict(dbu=at(22 << 30)), "dbu overlaps dbg"),
                                          (dict(ws=at(6 << 30)), "the workspace overlaps dh")])
def test_gated_bwd_refuses_overlap(change, match):
    a = dict(dx=FAR["out"], dwg=at(20 << 30), dwu=at(21 << 30), dbg=at(22 << 30), dbu=at(23 << 30), ws=at(24 << 30))
    a.update(change)
    refused("gfn_gated_bwd", FAR["x"], 63, FAR["wg"], FAR["wu"], FAR["bg"], FAR["bu"], FAR["dh"], 128, 100, None, 63, 128, 0, 0, a["dx"], 63, a["dwg"], a["dwu"], a["dbg"],
            a["dbu"], a["ws"], 1 << 29, None, match=match)


@pytest.mark.parametrize("change,match", [(dict(h=at((8 << 30) + 4)), "h overlaps c"), (dict(h=FAR["f"]), "h overlaps f"), (dict(state=FAR["h0"]), "state overlaps h0"),
                                          (dict(saved=at((9 << 30) + 12)), "saved overlaps h0"), (dict(state=FAR["off"]), "state overlaps pts_offsets"),
                                          (dict(saved=at((30 << 30) + 8)), "saved overlaps state")])
def test_ray_scan_fwd_refuses_overlap(change, match):
    a = dict(h=FAR["out"], state=at(30 << 30), saved=at(31 << 30))
    a.update(change)
    refused("gfn_ray_scan_fwd", FAR["off"], 10, FAR["f"], 8, FAR["c"], 32, 100, 32, 8, 0, 1, 0, FAR["h0"], a["h"], 32, a["state"], a["saved"], 0, None, 0, None, match=match)


@pytest.mark.parametrize("change,match", [(dict(df=FAR["f"]), "df overlaps f"), (dict(dc=FAR["dh"]), "dc overlaps dh"), (dict(dc=at((8 << 30) + 64)), "dc overlaps c"),
                                          (dict(dh0=FAR["h0"]), "dh0 overlaps h0"), (dict(dc=FAR["saved"]), "dc overlaps saved"), (dict(dc=at((30 << 30) + 4)), "dc overlaps df")])
def test_ray_scan_bwd_refuses_overlap(change, match):
    a = dict(df=at(30 << 30), dc=at(31 << 30), dh0=at(32 << 30))
    a.update(change)
    refused("gfn_ray_scan_bwd", FAR["off"], 10, FAR["f"], 8, FAR["c"], 32, FAR["dh"], 32, 100, 32, 8, 0, 1, 0, FAR["h0"], None, FAR["saved"], a["df"], 8, a["dc"], 32, a["dh0"], 0,
            None, 0, None, match=match)


def test_ray_scan_step_and_dropout_refuse_overlap():
    step = lambda f, c, state, h, ldh=32: ("gfn_ray_scan_step", f, 8, c, 32, 10, 32, 8, 0, 1, state, h, ldh, None)  # noqa: E731
    refused(*step(FAR["f"], FAR["c"], FAR["h0"], at((8 << 30) + 4)), match="h overlaps c")
    refused(*step(FAR["f"], FAR["c"], FAR["h0"], FAR["c"], 33), match="h overlaps c")
    refused(*step(FAR["f"], FAR["c"], FAR["h0"], FAR["f"]), match="h overlaps f")
    refused(*step(FAR["f"], FAR["c"], FAR["h0"], FAR["h0"]), match="state overlaps h")
    refused(*step(FAR["f"], FAR["c"], at((8 << 30) + 128), FAR["out"]), match="state overlaps c")
    refused(*step(FAR["f"], FAR["c"], FAR["f"], FAR["out"]), match="state overlaps f")
    drop = lambda x, ldx, y, ldy, call=FAR["off"]: ("gfn_dropout", x, ldx, 100, 64, 0, 0.5, 1, call, y, ldy, None)  # noqa: E731
    refused(*drop(FAR["x"], 64, at((1 << 30) + 4), 64), match="y overlaps x")
    refused(*drop(FAR["x"], 64, FAR["x"], 65), match="y overlaps x")
    refused(*drop(FAR["x"], 100, at((1 << 30) + 40 * 4), 100), match="y overlaps x")
    refused(*drop(FAR["x"], 64, FAR["out"], 64, at((12 << 30) + 8)), match="y overlaps call")
    refused("gfn_dropout_call", FAR["x"], FAR["x"], None, match="call overlaps counter")


ONCE = r"""
#include <atomic>
#include <cstdio>
#include <thread>
#include "gfn_once.h"
static unsigned long long seen = 0, other = 0;
int main() {
  std::atomic<int> step{0};
  bool a1, a2, b1, b2, c1;
  std::thread a([&] { a1 = gfn_first_call(seen, 3); step = 1; while (step != 2) std::this_thread::yield(); a2 = gfn_first_call(seen, 3); });
  std::thread b([&] { while (step != 1) std::this_thread::yield(); b1 = gfn_first_call(seen, 3); step = 2; });  // while a's set-up is under way
  a.join(); b.join();
  std::thread c([&] { c1 = gfn_first_call(seen, 3); b2 = gfn_first_call(seen, 4); });
  c.join();
  bool d = true;  // a thread that meets more call sites than it remembers runs their set-up again rather than go without
  static unsigned long long sites[1000];
  for (auto& s : sites) d = d && gfn_first_call(s, 0);
  for (int i = 900; i < 1000; i++) d = d && gfn_first_call(sites[i], 0);
  std::printf("%d %d %d %d %d %d %d", a1, a2, b1, c1, b2, gfn_first_call(other, 0), d);
}
"""


def test_two_threads_in_a_first_call_both_run_its_set_up(tmp_path):
    """The set-up in front of a launch (a kernel's LDS limit) is complete for every thread that gets past it, not only for the one that came first."""
    (tmp_path / "once.cpp").write_text(ONCE)
    exe = str(tmp_path / "once")
    subprocess.check_call(["g++", "-O2", "-std=c++17", "-pthread", "-I", os.path.join(ROOT, "gf-nerf_amd", "csrc"), str(tmp_path / "once.cpp"), "-o", exe])
    assert subprocess.check_output([exe], text=True, timeout=60) == "1 0 1 0 1 1 1"


# ---- dropout's masks ----------------------------------------------------------------------------------------------------------------------------
def test_a_dropout_inside_a_backward_pass_is_refused():
    """Recomputation (torch.utils.checkpoint) runs a forward again inside the backward pass.  In eval mode and with p = 0 there is no mask to differ."""
    import torch

    from gfnerf_amd import _lib
    from gfnerf_amd.gfnerf.mlp import Dropout

    class Again(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, module):
            ctx.module = module
            return x * 2

        @staticmethod
        def backward(ctx, g):
            return ctx.module(g), None

    x = torch.ones(4, 8, requires_grad=True)
    with pytest.raises(_lib.GfnError, match="recomputed inside a backward pass"):
        Again.apply(x, Dropout(0.5)).sum().backward()
    Again.apply(x, Dropout(0.5).eval()).sum().backward()
    Again.apply(x, Dropout(0.0)).sum().backward()


def test_dropout_modules_and_ranks_have_masks_of_their_own(monkeypatch):
    import torch

    from gfnerf_amd import dist
    from gfnerf_amd.gfnerf.mlp import Dropout, GatedMLPNetwork

    spec = {"activation": "SwiGLU", "output_activation": "None", "n_neurons": 16, "n_hidden_layers": 3, "dropout": 0.1}
    seeds = [m.seed for net in (GatedMLPNetwork(8, 4, spec), GatedMLPNetwork(8, 4, spec)) for m in net.dropout] + [Dropout().seed, Dropout().seed]
    assert len(set(seeds)) == 8
    torch.manual_seed(3)
    first = [Dropout().seed, Dropout().seed]
    torch.manual_seed(3)
    assert [Dropout().seed, Dropout().seed] == first
    assert Dropout(0.5, 7).seed == 7 and [m.seed for m in GatedMLPNetwork(8, 4, spec, seed=1337).dropout] == [1337, 1338, 1339]
    module, keys = Dropout(0.5, 7), []
    assert module.key() == 7  # without a process group
    for rank in range(8):
        monkeypatch.setattr(dist, "rank", lambda group=None: rank)
        keys += [module.key(), Dropout(0.5, 8).key()]
    assert len(set(keys)) == 16 and all(0 <= k < 1 << 64 for k in keys) and keys[0] == 7
    kept = [oseq.dropout_mask(200, 64, 0.5, k, 0)[0] for k in keys[::2]]
    for i in range(1, 8):  # 12,800 pairs of fair coins: half of them agree, within five standard deviations
        assert abs((kept[0] == kept[i]).mean() - 0.5) < 5 * 0.5 / np.sqrt(12800)


def test_dropout_of_rows_without_columns_is_the_rows():
    import torch

    from gfnerf_amd.gfnerf.mlp import Dropout

    for shape in ((4, 0), (2, 3, 0), (0, 0)):
        x = torch.zeros(shape)
        assert Dropout(0.5)(x) is x
