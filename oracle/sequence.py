"""CPU restatement, in 64 bits, of the sequence-head operators (gfn_gated_*, gfn_ray_scan_*, gfn_dropout), with bounds on what their kernels'
roundings may add -- test infrastructure only.  Every function returns (value, bound): |kernel - value| <= bound elementwise follows from the
arithmetic stated at it; `half(dtype)` is the unit roundoff of a type, u = 2^-24 that of f32."""
import numpy as np
from scipy import special

U = 2.0 ** -24
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
TINY = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -25}  # half a step of the smallest numbers (subnormals)


def rounded(v, err, dtype):
    """The bound after one rounding of a value within `err` of v to `dtype`."""
    return err + (np.abs(v) + err) * HALF[dtype] + TINY[dtype]


# ---- gated feed-forward ---------------------------------------------------------------------------------------------------------------
def act(z, kind):
    """act(z), act'(z), and a bound on |act''|."""
    if kind == "relu":
        return np.maximum(z, 0.0), (z > 0).astype(np.float64), 0.0
    if kind == "gelu":
        cdf, pdf = special.ndtr(z), np.exp(-0.5 * z * z) / np.sqrt(2 * np.pi)
        return z * cdf, cdf + z * pdf, 0.8  # |pdf (2 - z^2)| <= 2 / sqrt(2 pi)
    s = special.expit(z)
    if kind == "silu":
        return z * s, s * (1 + z * (1 - s)), 0.5
    return s, s * (1 - s), 0.1


def _act_error(z, kind):
    """What evaluating act and act' in f32 adds for an exact z: the argument of exp2 is rounded twice (|z| 2^-23 relative in the result),
    exp2 and the reciprocal are good to a few units; gelu's polynomial to 1.5e-7 plus the reciprocal's and the fma chain's rounding (4e-7)."""
    if kind == "relu":
        return np.zeros_like(z)
    if kind == "gelu":
        return (np.abs(z) + 1) * 6e-7
    rel = (np.abs(z) + 8) * 2 * U
    s = special.expit(z)
    base = np.abs(z) * s if kind == "silu" else s
    return rel * (base + s) + 4 * U


def _project(x, w, b):
    """z = x w^T + b and the bound of an f32 sum of k + 1 products in any order: (k + 2) u sum |x w| + |b|."""
    z, mag = x @ w.T, np.abs(x) @ np.abs(w).T
    if b is not None:
        z, mag = z + b, mag + np.abs(b)
    return z, (x.shape[1] + 2) * U * mag


def gated_fwd(x, wg, wu, bg, bu, kind, dtype):
    g, eg = _project(x, wg, bg)
    u, eu = _project(x, wu, bu)
    a, _, _ = act(g, kind)
    ea = 1.13 * eg + _act_error(g, kind)  # |act'| <= 1.13
    h = a * u
    return h, rounded(h, (np.abs(u) + eu) * ea + np.abs(a) * eu + 2 * U * np.abs(h), dtype)


def gated_bwd(x, wg, wu, dh, bg, bu, kind, dtype):
    """dg = dh u act'(g), du = dh act(g) in f32, which the matrix units of the 16-bit types take as several operands: bf16 three of 8 bits, which are
    dz itself down to 2^-126; f16 two, each within 2^-11 of what it stands for, under powers of two that leave the sample's largest |dz| (for dx) and
    the tile's (for dW; 64 or 128 rows: the bound takes 128) at 2^7 or above.  Half a step of f16's grid is 2^-25; a pair of operands meets it when it
    is formed, and twice when it is brought to a lower power: below 2^-30 of that largest in all.  Sums over 2 h (dx) and n (dW) products of each operand in f32: (count + 2) u of their magnitudes; the result rounded once."""
    g, eg = _project(x, wg, bg)
    u, eu = _project(x, wu, bu)
    a, da, dda = act(g, kind)
    ea = _act_error(g, kind)
    dg, du = dh * u * da, dh * a
    edg = np.abs(dh) * (eu * np.abs(da) + (np.abs(u) + eu) * (dda * eg + 3 * ea)) + 4 * U * np.abs(dg)
    edu = np.abs(dh) * (1.13 * eg + ea) + 2 * U * np.abs(du)
    n, h = dg.shape
    ops = {"f32": 1, "bf16": 3, "f16": 2}[dtype]

    def fed(v, e, floor):  # what the operands add
        return e + (np.abs(v) + e) * 2.0 ** -22 + floor if dtype == "f16" else e + (2.0 ** -126 if dtype == "bf16" else 0.0)

    row = np.maximum(np.abs(dg), np.abs(du)).max(1, initial=0.0)[:, None]
    tile = np.concatenate([np.full((len(r), 1), r.max()) for r in np.split(row, range(128, n, 128))]) if n else row

    def total(parts, count):
        v = sum(p @ q for p, e, q in parts)
        err = sum(e @ np.abs(q) + (ops * count + 2) * U * ((np.abs(p) + e) @ np.abs(q)) for p, e, q in parts)
        return v, rounded(v, err, dtype)

    xdg, xdu, wdg, wdu = (fed(v, e, f) for f in (row * 2.0 ** -30, tile * 2.0 ** -30) for v, e in ((dg, edg), (du, edu)))
    ones = np.ones((n, 1))
    out = {"dx": total([(dg, xdg, wg), (du, xdu, wu)], 2 * h), "dwg": total([(dg.T, wdg.T, x)], n), "dwu": total([(du.T, wdu.T, x)], n)}
    if bg is not None:
        out["dbg"], out["dbu"] = ((v[:, 0], e[:, 0]) for v, e in (total([(dg.T, wdg.T, ones)], n), total([(du.T, wdu.T, ones)], n)))
    return out


# ---- gated recurrence -------------------------------------------------------------------------------------------------------------------
def gate(f, kind):
    """a, 1 - a (linear: 1), da/df, and the relative errors of evaluating a and 1 - a in f32: |f| 2^-23 from the argument of exp2 and a few
    units from exp2, the reciprocal and the products."""
    rel = (np.abs(f) + 8) * 2 * U
    if kind == "linear":
        return f, np.ones_like(f), np.ones_like(f), 0.0 * f, 0.0 * f
    if kind == "sigmoid":
        a, rest = special.expit(f), special.expit(-f)
        return a, rest, a * rest, rel, rel
    a, rest = np.exp(-f), -np.expm1(-f)
    # 1 - a by the series below 1/4 (5e-8 of its value cut off), by subtraction above: a's error over 1 - a >= 0.22
    return a, rest, -a, rel, rel + 1e-7 + rel * a / np.maximum(np.abs(rest), 1e-30) * (np.abs(f) >= 0.25)


def ray_scan(offsets, f, c, kind, reverse, dtype, h0=None, dh=None, d_state=None):
    """Row by row.  Bounds by the same recurrences: E_t = |a| E_{t-1} + |a h_{t-1}| ea + |b| (eb + u) + 2 u |h_t| forward, the same with l
    for the adjoint; products add their factors' relative errors."""
    n, d = c.shape
    rep = d // f.shape[1]
    a, rest, slope, ea, er = (np.repeat(v, rep, axis=1) for v in gate(f, kind))
    b = rest * c
    h, eh = np.zeros((n, d)), np.zeros((n, d))
    rays = len(offsets) - 1
    state = np.zeros((rays, d)) if h0 is None else h0.copy()
    es = np.zeros((rays, d))
    before, ebefore = np.zeros((n, d)), np.zeros((n, d))
    for r in range(rays):
        rows = range(offsets[r], offsets[r + 1])
        for t in reversed(rows) if reverse else rows:
            before[t], ebefore[t] = state[r], es[r]
            h[t] = a[t] * state[r] + b[t]
            eh[t] = np.abs(a[t]) * (1 + ea[t]) * es[r] + np.abs(a[t] * state[r]) * ea[t] + np.abs(b[t]) * (er[t] + U) + 2 * U * (np.abs(h[t]) + np.abs(b[t]))
            state[r], es[r] = h[t], eh[t]
    live = np.zeros((n, 1))
    live[offsets[0]:offsets[-1]] = 1
    out = {"h": (h, rounded(h, eh, dtype) * live), "state": (state, es + TINY["f32"])}
    if dh is None:
        return out
    df, edf, dc, edc = (np.zeros((n, d)) for _ in range(4))
    l = np.zeros((rays, d)) if d_state is None else d_state.copy()
    el = np.zeros((rays, d))
    for r in range(rays):
        rows = range(offsets[r], offsets[r + 1])
        for t in rows if reverse else reversed(rows):
            lam = l[r] + dh[t]
            elam = el[r] + U * np.abs(lam)
            dc[t] = lam * rest[t]
            edc[t] = elam * np.abs(rest[t]) + np.abs(dc[t]) * (er[t] + 2 * U)
            diff = before[t] if kind == "linear" else before[t] - c[t]
            ediff = ebefore[t] + U * np.abs(diff)
            df[t] = lam * diff * slope[t]
            edf[t] = np.abs(slope[t]) * (elam * (np.abs(diff) + ediff) + np.abs(lam) * ediff) + np.abs(df[t]) * (ea[t] + er[t] + 4 * U)
            l[r], el[r] = a[t] * lam, np.abs(a[t]) * (1 + ea[t]) * elam + np.abs(a[t] * lam) * (ea[t] + U)
    g = f.shape[1]
    dfs = df.reshape(n, g, rep).sum(2)
    edfs = edf.reshape(n, g, rep).sum(2) + rep * U * np.abs(df).reshape(n, g, rep).sum(2)
    out["df"], out["dc"] = (dfs, rounded(dfs, edfs, dtype) * live), (dc, rounded(dc, edc, dtype) * live)
    out["dh0"] = (l, el + TINY["f32"])
    return out


# ---- dropout ------------------------------------------------------------------------------------------------------------------------------
def philox(counter, key):
    """Philox4x32-10 (Salmon et al., SC'11): counter u32 [..., 4], key (k0, k1) -> u32 [..., 4]."""
    c = [counter[..., i].astype(np.uint64) for i in range(4)]
    k, low, hi = [int(key[0]), int(key[1])], np.uint64(0xFFFFFFFF), np.uint64(32)
    for _ in range(10):
        p, q = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(q >> hi) ^ c[1] ^ np.uint64(k[0]), q & low, (p >> hi) ^ c[3] ^ np.uint64(k[1]), p & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, axis=-1).astype(np.uint32)


def dropout_mask(rows, cols, p, seed, call, first_row=0):
    """keep (bool [rows, cols]) and the kept elements' factor."""
    blocks = -(-cols // 8)
    ctr = np.zeros((rows, blocks, 4), np.uint32)
    ctr[..., 0] = np.arange(blocks)
    ctr[..., 1] = (first_row + np.arange(rows))[:, None]
    ctr[..., 2], ctr[..., 3] = call & 0xFFFFFFFF, call >> 32
    w = philox(ctr, (seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF))
    bits = np.stack([w & 0xFFFF, w >> 16], axis=-1).reshape(rows, blocks * 8)[:, :cols]
    below = int(p * 65536 + 0.5)
    return bits >= below, np.float32(65536.0 / (65536 - below)) if below < 65536 else np.float32(0)
