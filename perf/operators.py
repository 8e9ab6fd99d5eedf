"""Measured cases of the sequence-head operators: the gated feed-forward layer, the gated linear recurrence along packed rays, and dropout.

A case is a dict of plain values; `prepare` makes its inputs on the GPU, `run` makes one pass (the plain torch form, or with `own` the framework's
kernels), `work` says what the pass cannot do without, and `exact` gives the result in 64 bits from the definitions.

Sizes are the framework's own: 32 hash features, the colour head's 63 inputs and its 128-wide hidden layers, 4,096 rays of about 192 (focal stage) or
128 (global stage) samples, full-frame tiles of many short rays; and ranges around them down to one sample."""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # the field queried at a handful of points (a probe of the density, one ray): latency
        dict(name="gated fwd 128 f32", op="gated_fwd", n=128, k=63, h=128, dtype="f32", act="silu", bias=True),
        # the colour head's first layer over a focal-stage batch, 4,096 rays x 192 samples
        dict(name="gated fwd focal bf16", op="gated_fwd", n=786432, k=63, h=128, dtype="bf16", act="silu", bias=True),
        # the base network's first layer on the hash features, full precision, a ragged number of samples
        dict(name="gated fwd hash f32", op="gated_fwd", n=262145, k=32, h=128, dtype="f32", act="gelu", bias=True),
        # training: the colour head's layer over a global-stage batch, 4,096 rays x 128 samples
        dict(name="gated bwd global bf16", op="gated_bwd", n=524288, k=63, h=128, dtype="bf16", act="silu", bias=True),
        # training: a hidden layer, 128 -> 128, without biases
        dict(name="gated bwd hidden f16", op="gated_bwd", n=100003, k=128, h=128, dtype="f16", act="gelu", bias=False),
        # training in full precision: a narrow layer on the hash features
        dict(name="gated bwd narrow f32", op="gated_bwd", n=49999, k=32, h=64, dtype="f32", act="sigmoid", bias=True),
        # training: a 128-channel state along the rays of a focal-stage batch
        dict(name="scan train focal bf16", op="scan_train", rays=4096, mean=192, d=128, g=128, dtype="bf16", gate="sigmoid", reverse=False, h0=False),
        # rendering 32 feature channels of an image tile: one optical thickness per sample, back to front
        dict(name="scan fwd features f32", op="scan_fwd", rays=16384, mean=128, d=32, g=1, dtype="f32", gate="decay", reverse=True, h0=False),
        # training on few, very long sequences (whole camera paths), carried in from an earlier part
        dict(name="scan train long f16", op="scan_train", rays=2, mean=131072, d=64, g=64, dtype="f16", gate="sigmoid", reverse=False, h0=True),
        # one more sample for every ray of a batch: the state is carried by the caller
        dict(name="scan step bf16", op="scan_step", rays=4096, d=128, g=128, dtype="bf16", gate="sigmoid"),
        # dropout of a focal-stage batch's hidden features, and of its gradient
        dict(name="dropout focal bf16", op="dropout", n=786432, d=128, dtype="bf16", p=0.1),
        # dropout of a few rows of odd width: latency
        dict(name="dropout rows f32", op="dropout", n=1000, d=63, dtype="f32", p=0.5),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["gated_fwd", "gated_bwd", "scan_train", "scan_fwd", "scan_step", "dropout"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op in ("gated_fwd", "gated_bwd"):
        k, h = _log(rng, 1, 128), _log(rng, 1, 256)
        most = int(min(786432, 786432 * 191 // (k + h), 786432 * 63 * 128 // (k * h)))  # no larger than the focal batch's layer
        if op == "gated_bwd":
            most = int(min(most, 524288 * 191 // (k + h), 524288 * 63 * 128 // (k * h)))
        return dict(op=op, n=_log(rng, 1, max(most, 1)), k=k, h=h, dtype=dtype, act=rng.choice(["silu", "gelu", "sigmoid"]), bias=rng.random() < 0.5)
    if op == "dropout":
        d = _log(rng, 1, 1024)
        return dict(op=op, n=_log(rng, 1, 786432 * 128 // d // (2 if dtype == "f32" else 1)), d=d, dtype=dtype, p=round(rng.uniform(0.0, 0.9), 3))
    g = _log(rng, 1, 256)
    d = g * rng.choice([1, 1, 2, 4, 8, 16, 32])
    while d > 256:
        d //= 2
    g = min(g, d) if d % min(g, d) == 0 else 1
    gate = rng.choice(["linear", "sigmoid", "decay"])
    if op == "scan_step":
        return dict(op=op, rays=_log(rng, 1, 65536), d=d, g=g, dtype=dtype, gate=gate)
    rays = _log(rng, 1, 16384)
    rows = max(rays, _log(rng, rays, max(rays, min(2097152, 50000000 // d))))
    mean = max(1, rows // rays)
    return dict(op=op, rays=rays, mean=mean, d=d, g=g, dtype=dtype, gate=gate, reverse=rng.random() < 0.5, h0=rng.random() < 0.5)


def _lengths(case):
    """Samples per ray: spread evenly from none to twice the mean, every 16th ray missing the scene. The same numbers for every seed."""
    s, mean = case["rays"], case["mean"]
    if s == 1:
        return np.array([mean], dtype=np.int64)
    lens = np.floor(2.0 * mean * (np.arange(s) + 0.5) / s + 0.5).astype(np.int64)
    if s >= 16:
        lens[5::16] = 0
    return lens


def _rows(case):
    return int(_lengths(case).sum())


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) % (1 << 31))

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, device="cuda", generator=gen) * scale

    def uniform(*shape, scale=1.0):
        return (torch.rand(*shape, device="cuda", generator=gen) * 2 - 1) * scale

    t = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"].startswith("gated"):
        n, k, h = case["n"], case["k"], case["h"]
        s["x"] = normal(n, k).to(t)
        s["wg"], s["wu"] = uniform(h, k, scale=k ** -0.5).to(t), uniform(h, k, scale=k ** -0.5).to(t)
        s["bg"] = uniform(h, scale=k ** -0.5).to(t) if case["bias"] else None
        s["bu"] = uniform(h, scale=k ** -0.5).to(t) if case["bias"] else None
        if case["op"] == "gated_bwd":
            s["dh"] = normal(n, h).to(t)
        return s
    if case["op"] == "dropout":
        s["x"], s["dy"] = normal(case["n"], case["d"]).to(t), normal(case["n"], case["d"]).to(t)
        s["seed"] = int(seed)
        s["call"] = torch.tensor([3 + int(seed) % 1000], dtype=torch.int64, device="cuda")
        return s
    d, g = case["d"], case["g"]
    if case["op"] == "scan_step":
        n = case["rays"]
        s["state"] = normal(n, d)
    else:
        lens = _lengths(case)
        lens = lens[np.random.RandomState(int(seed) % (1 << 31)).permutation(len(lens))]
        offsets = np.zeros(len(lens) + 1, dtype=np.int64)
        np.cumsum(lens, out=offsets[1:])
        n = int(offsets[-1])
        s["offsets"] = torch.from_numpy(offsets.astype(np.int32)).cuda()
        s["levels"] = max(1, math.ceil(math.log2(max(2, int(lens.max())))))
        s["h0"] = normal(len(lens), d) if case["h0"] else None
    if case["gate"] == "decay":  # optical thickness of a sample: mostly thin, some opaque
        s["f"] = normal(n, g).mul_(1.5).sub_(2.0).exp_().to(t)
    elif case["gate"] == "sigmoid":  # gates that remember for about ten samples
        s["f"] = (normal(n, g) + 2.0).to(t)
    else:
        s["f"] = torch.sigmoid(normal(n, g) + 2.0).to(t)
    s["c"] = normal(n, d).to(t)
    if case["op"] == "scan_train":
        s["dh"] = normal(n, d).to(t)
        s["d_state"] = normal(case["rays"], d)
    return s


# ---- the plain forms: elementary torch operations in 32 bits, rounded once at the end -------------------------------------------------------------
def _act(z, act):
    """act(z) and its derivative."""
    if act == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    sig = 1.0 / (1.0 + torch.exp(-z))
    if act == "silu":
        return z * sig, sig * (1.0 + z * (1.0 - sig))
    return sig, sig * (1.0 - sig)


def _gated(s):
    x, wg, wu = s["x"].float(), s["wg"].float(), s["wu"].float()
    g, u = x @ wg.t(), x @ wu.t()
    if s["bg"] is not None:
        g, u = g + s["bg"].float(), u + s["bu"].float()
    return x, wg, wu, g, u


def _gated_fwd(s):
    *_, g, u = _gated(s)
    return (_act(g, s["case"]["act"])[0] * u).to(s["x"].dtype)


def _gated_bwd(s):
    t = s["x"].dtype
    x, wg, wu, g, u = _gated(s)
    a, da = _act(g, s["case"]["act"])
    dh = s["dh"].float()
    dg, du = dh * u * da, dh * a
    dx = dg @ wg + du @ wu
    out = {"dx": dx.to(t), "dwg": _over_rows(dg, x).to(t), "dwu": _over_rows(du, x).to(t)}
    if s["bg"] is not None:
        out["dbg"], out["dbu"] = dg.sum(0).to(t), du.sum(0).to(t)
    return out


def _over_rows(dz, x):
    """dz^T x, a sum over up to half a million rows: parts of 4,096 rows in 32 bits, joined in 64."""
    n = dz.shape[0]
    full = n - n % 4096
    total = (dz[full:].t() @ x[full:]).double()
    if full:
        parts = torch.bmm(dz[:full].view(-1, 4096, dz.shape[1]).transpose(1, 2), x[:full].view(-1, 4096, x.shape[1]))
        total = total + parts.sum(0, dtype=torch.float64)
    return total


def _gate(f, c, gate):
    """a, b of h_t = a_t h_{t-1} + b_t, one column per channel."""
    f = f.float().repeat_interleave(c.shape[1] // f.shape[1], dim=1)
    c = c.float()
    if gate == "linear":
        return f, c
    if gate == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-f)), c / (1.0 + torch.exp(f))
    return torch.exp(-f), -torch.expm1(-f) * c


def _doubled(a, b, levels):
    """All prefixes of h_t = a_t h_{t-1} + b_t at once: after level i each row stands for the 2^(i+1) rows up to it."""
    step = 1
    for _ in range(levels):  # the logarithm of the longest ray, not its samples
        if step >= a.shape[0]:
            break
        b = torch.cat([b[:step], torch.addcmul(b[step:], a[step:], b[:-step])])
        a = torch.cat([a[:step], a[step:] * a[:-step]])
        step *= 2
    return b


def _segments(s, n):
    """Each row's ray, and whether it is the ray's first / last row in the order the recurrence takes."""
    off = s["offsets"].long()
    rows = torch.arange(n, device=off.device)
    ray = torch.searchsorted(off[1:].contiguous(), rows, right=True)
    low, high = rows == off[ray], rows == off[ray + 1] - 1
    return off, ray, (high, low) if s["case"]["reverse"] else (low, high)


def _scan(s):
    rev = s["case"]["reverse"]
    a, b = _gate(s["f"], s["c"], s["case"]["gate"])
    off, ray, (first, last) = _segments(s, a.shape[0])
    h0 = s["h0"] if s["h0"] is not None else torch.zeros(off.numel() - 1, a.shape[1], device=a.device)
    start = first[:, None]
    bs = torch.where(start, b + a * h0[ray], b)
    keep = torch.where(start, torch.zeros_like(a), a)  # nothing comes over from the ray before
    h = _doubled(keep.flip(0), bs.flip(0), s["levels"]).flip(0) if rev else _doubled(keep, bs, s["levels"])
    empty = (off[1:] == off[:-1])[:, None]
    end = (off[:-1] if rev else off[1:] - 1).clamp(0, a.shape[0] - 1)
    state = torch.where(empty, h0, h[end])
    return a, h, h0, state, off, ray, start, last[:, None], empty


def _scan_fwd(s):
    _, h, _, state, *_ = _scan(s)
    return {"h": h.to(s["c"].dtype), "state": state}


def _shift(v, rev):
    """v of the row before, in the recurrence's order (the first row's is never used)."""
    return torch.cat([v[1:], v[:1]]) if rev else torch.cat([v[-1:], v[:-1]])


def _scan_train(s):
    case, t = s["case"], s["c"].dtype
    rev, d, g = case["reverse"], case["d"], case["g"]
    a, h, h0, state, off, ray, start, last, empty = _scan(s)
    dl = torch.where(last, s["dh"].float() + s["d_state"][ray], s["dh"].float())
    nxt = torch.where(last, torch.zeros_like(a), _shift(a, not rev))  # the gate of the row behind
    lam = _doubled(nxt, dl, s["levels"]) if rev else _doubled(nxt.flip(0), dl.flip(0), s["levels"]).flip(0)
    before = torch.where(start, h0[ray], _shift(h, rev))
    c = s["c"].float()
    f = s["f"].float().repeat_interleave(d // g, dim=1)
    if case["gate"] == "linear":
        df, dc = lam * before, lam
    elif case["gate"] == "sigmoid":
        rest = 1.0 / (1.0 + torch.exp(f))
        df, dc = lam * (before - c) * a * rest, lam * rest
    else:
        df, dc = lam * (c - before) * a, -torch.expm1(-f) * lam
    begin = (off[1:] - 1 if rev else off[:-1]).clamp(0, a.shape[0] - 1)
    out = {"h": h.to(t), "state": state, "df": df.view(-1, g, d // g).sum(2).to(t), "dc": dc.to(t)}
    if s["h0"] is not None:
        out["dh0"] = torch.where(empty, s["d_state"], a[begin] * lam[begin])
    return out


def _scan_step(s):
    a, b = _gate(s["f"], s["c"], s["case"]["gate"])
    s["state"].copy_(a * s["state"] + b)
    return {"h": s["state"].to(s["c"].dtype), "state": s["state"]}


def _words(seed, call, n, blocks):
    """Philox4x32-10 (Salmon et al. 2011) of the counters (block, row, call): four 32-bit words each, in 64-bit integers."""
    low = 0xFFFFFFFF
    c0 = torch.arange(blocks, device="cuda").expand(n, blocks)
    c1 = torch.arange(n, device="cuda")[:, None].expand(n, blocks)
    c2, c3 = (call & low).expand(n, blocks), ((call >> 32) & low).expand(n, blocks)
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):  # the generator's rounds
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((p1 >> 32) & low) ^ c1 ^ k0, p1 & low, ((p0 >> 32) & low) ^ c3 ^ k1, p0 & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([c0, c1, c2, c3], dim=2)


def _dropout(s):
    n, d, p = s["case"]["n"], s["case"]["d"], s["case"]["p"]
    below = int(p * 65536 + 0.5)
    w = _words(s["seed"], s["call"], n, (d + 7) // 8)
    u = torch.stack([w & 0xFFFF, w >> 16], dim=3).reshape(n, -1)[:, :d]
    scale = 65536.0 / (65536 - below) if below < 65536 else 0.0
    zero = torch.zeros((), device="cuda")
    return {"y": torch.where(u >= below, s["x"].float() * scale, zero).to(s["x"].dtype),
            "dx": torch.where(u >= below, s["dy"].float() * scale, zero).to(s["x"].dtype)}


# ---- the framework's own operators, as a training loop or a renderer calls them ---------------------------------------------------------------------
def _own(s):
    from gfnerf_amd import ops

    case = s["case"]
    if case["op"] == "gated_fwd":
        return ops.gated_fwd(s["x"], s["wg"], s["wu"], s["bg"], s["bu"], act=case["act"])
    if case["op"] == "gated_bwd":
        dx, dwg, dwu, dbg, dbu = ops.gated_bwd(s["x"], s["wg"], s["wu"], s["dh"], s["bg"], s["bu"], act=case["act"])
        return {"dx": dx, "dwg": dwg, "dwu": dwu} | ({"dbg": dbg, "dbu": dbu} if case["bias"] else {})
    if case["op"] == "dropout":
        return {"y": ops.dropout(s["x"], case["p"], s["seed"], s["call"]), "dx": ops.dropout(s["dy"], case["p"], s["seed"], s["call"])}
    if case["op"] == "scan_step":
        return {"h": ops.ray_scan_step(s["f"], s["c"], s["state"], gate=case["gate"]), "state": s["state"]}
    train = case["op"] == "scan_train"
    r = ops.ray_scan_fwd(s["offsets"], s["f"], s["c"], gate=case["gate"], reverse=case["reverse"], h0=s["h0"], save=train)
    out = {"h": r["h"], "state": r["state"]}
    if train:
        b = ops.ray_scan_bwd(s["offsets"], s["f"], s["c"], s["dh"], r["saved"], gate=case["gate"], reverse=case["reverse"], h0=s["h0"], d_state=s["d_state"])
        out["df"], out["dc"] = b["df"], b["dc"]
        if s["h0"] is not None:
            out["dh0"] = b["dh0"]
    return out


def run(state):
    if own:
        return _own(state)
    return {"gated_fwd": _gated_fwd, "gated_bwd": _gated_bwd, "scan_train": _scan_train, "scan_fwd": _scan_fwd, "scan_step": _scan_step,
            "dropout": _dropout}[state["case"]["op"]](state)


def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "gated_fwd":
        n, k, h = case["n"], case["k"], case["h"]
        return {"bytes": e * (n * (k + h) + 2 * h * k), "flops": 4.0 * n * k * h}
    if case["op"] == "gated_bwd":  # both projections again, the input's gradient, the weights' gradients
        n, k, h = case["n"], case["k"], case["h"]
        return {"bytes": e * (n * (2 * k + h) + 4 * h * k), "flops": 12.0 * n * k * h}
    if case["op"] == "dropout":
        return {"bytes": 4.0 * e * case["n"] * case["d"], "flops": 2.0 * case["n"] * case["d"]}
    d, g = case["d"], case["g"]
    if case["op"] == "scan_step":
        return {"bytes": case["rays"] * (e * (g + 2 * d) + 8 * d), "flops": 4.0 * case["rays"] * d}
    n, state = _rows(case), 4 * case["rays"] * d
    if case["op"] == "scan_fwd":
        return {"bytes": e * n * (g + 2 * d) + state * (2 if case["h0"] else 1), "flops": 4.0 * n * d}
    return {"bytes": e * n * (2 * g + 4 * d) + state * (4 if case["h0"] else 2), "flops": 12.0 * n * d}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------------------------------------
def _exact_gated(s):
    leaves = {k: s[k].double().requires_grad_(True) for k in ("x", "wg", "wu", "bg", "bu") if s[k] is not None}
    lin = torch.nn.functional.linear
    g, u = lin(leaves["x"], leaves["wg"], leaves.get("bg")), lin(leaves["x"], leaves["wu"], leaves.get("bu"))
    act = {"silu": lambda z: z * torch.special.expit(z), "gelu": lambda z: z * torch.special.ndtr(z), "sigmoid": torch.special.expit}[s["case"]["act"]]
    if "dh" not in s:
        return (act(g) * u).detach()
    grads = torch.autograd.grad(act(g) * u, list(leaves.values()), s["dh"].double())
    names = {"x": "dx", "wg": "dwg", "wu": "dwu", "bg": "dbg", "bu": "dbu"}
    return {names[k]: v for k, v in zip(leaves, grads)}


def _exact_recurrence(a, b):
    """h_t = a_t h_{t-1} + b_t over all rows, h_{-1} = 0: each of about sqrt(n) blocks row by row, then from block to block."""
    n, d = a.shape
    size = max(1, math.isqrt(n))
    blocks = -(-n // size)
    pad = blocks * size - n
    a = torch.cat([a, a.new_zeros(pad, d)]).view(blocks, size, d)
    h = torch.cat([b, b.new_zeros(pad, d)]).view(blocks, size, d).clone()
    p = a.clone()
    for i in range(1, size):
        h[:, i] += a[:, i] * h[:, i - 1]
        p[:, i] *= p[:, i - 1]
    carry = torch.zeros(blocks, d, dtype=a.dtype, device=a.device)
    for j in range(1, blocks):
        carry[j] = h[j - 1, -1] + p[j - 1, -1] * carry[j - 1]
    return (h + p * carry[:, None]).view(-1, d)[:n]


def _exact_scan(s):
    case = s["case"]
    off = s["offsets"].cpu().numpy().astype(np.int64)
    n, d, g, rays = s["c"].shape[0], case["d"], case["g"], case["rays"]
    order = np.arange(n)[::-1] if case["reverse"] else np.arange(n)  # the recurrence's order of rows
    ray = np.repeat(np.arange(rays), np.diff(off))[order]
    begin = np.flatnonzero(np.diff(ray, prepend=-1))  # first row of each ray that has any
    end = np.flatnonzero(np.diff(ray, append=-1))
    order, of, begin, end = (torch.from_numpy(np.ascontiguousarray(v)).cuda() for v in (order, ray[begin], begin, end))
    f = s["f"].double()[order][:, torch.arange(d, device="cuda") // (d // g)]
    c = s["c"].double()[order]
    if case["gate"] == "linear":
        a, rest, slope = f, None, None
    elif case["gate"] == "sigmoid":
        a, rest = torch.special.expit(f), torch.special.expit(-f)
        slope = a * rest
    else:
        a, rest = torch.exp(-f), -torch.special.expm1(-f)
        slope = -a
    b = c if rest is None else rest * c
    h0 = s["h0"].double() if s["h0"] is not None else torch.zeros(rays, d, dtype=torch.float64, device="cuda")
    inner, first = a.clone(), b.clone()
    inner[begin] = 0
    first[begin] += a[begin] * h0[of]
    h = _exact_recurrence(inner, first)
    state = h0.clone()
    state[of] = h[end]
    out = {"h": torch.empty_like(h).index_copy_(0, order, h), "state": state}
    if case["op"] == "scan_fwd":
        return out
    dl = s["dh"].double()[order]
    dl[end] += s["d_state"].double()[of]
    inner = torch.cat([a[1:], a[:1]])
    inner[end] = 0
    lam = _exact_recurrence(inner.flip(0), dl.flip(0)).flip(0)
    before = torch.cat([h[-1:], h[:-1]])
    before[begin] = h0[of]
    df = lam * before if rest is None else lam * (before - c) * slope
    dc = lam if rest is None else lam * rest
    df = torch.zeros(n, g, dtype=torch.float64, device="cuda").index_add_(1, torch.arange(d, device="cuda") // (d // g), df)
    out["df"], out["dc"] = torch.empty_like(df).index_copy_(0, order, df), torch.empty_like(dc).index_copy_(0, order, dc)
    if s["h0"] is not None:
        out["dh0"] = s["d_state"].double()
        out["dh0"][of] = a[begin] * lam[begin]
    return out


def _exact_step(s):
    f = s["f"].double()[:, torch.arange(s["case"]["d"], device="cuda") // (s["case"]["d"] // s["case"]["g"])]
    c, h = s["c"].double(), s["state"].double()
    if s["case"]["gate"] == "linear":
        h = f * h + c
    elif s["case"]["gate"] == "sigmoid":
        h = torch.special.expit(f) * h + torch.special.expit(-f) * c
    else:
        h = torch.exp(-f) * h - torch.special.expm1(-f) * c
    return {"h": h, "state": h}


def _exact_dropout(s):
    n, d, p = s["case"]["n"], s["case"]["d"], s["case"]["p"]
    below, blocks, call = int(math.floor(p * 65536 + 0.5)), -(-d // 8), int(s["call"].item())
    u = np.empty((n, blocks, 8), dtype=np.uint16)
    part = max(1, (1 << 18) // blocks)
    for i in range(0, n, part):
        m = min(part, n - i)
        ctr = [np.tile(np.arange(blocks, dtype=np.uint64), m), np.repeat(np.arange(i, i + m, dtype=np.uint64), blocks),
               np.full(m * blocks, call & 0xFFFFFFFF, np.uint64), np.full(m * blocks, call >> 32, np.uint64)]
        key = [s["seed"] & 0xFFFFFFFF, s["seed"] >> 32 & 0xFFFFFFFF]
        for _ in range(10):
            a, b = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
            low = np.uint64(0xFFFFFFFF)
            ctr = [(b >> np.uint64(32)) ^ ctr[1] ^ np.uint64(key[0]), b & low, (a >> np.uint64(32)) ^ ctr[3] ^ np.uint64(key[1]), a & low]
            key = [(key[0] + 0x9E3779B9) & 0xFFFFFFFF, (key[1] + 0xBB67AE85) & 0xFFFFFFFF]
        u[i:i + m] = np.stack(ctr, axis=1).astype("<u4").view("<u2").reshape(m, blocks, 8)
    keep = torch.from_numpy(u.reshape(n, -1)[:, :d] >= below).cuda()
    scale = 65536.0 / (65536 - below) if below < 65536 else 0.0
    return {"y": s["x"].double() * keep * scale, "dx": s["dy"].double() * keep * scale}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"].startswith("gated"):
        return _exact_gated(s)
    if case["op"] == "dropout":
        return _exact_dropout(s)
    return _exact_step(s) if case["op"] == "scan_step" else _exact_scan(s)
