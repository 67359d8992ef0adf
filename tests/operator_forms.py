"""The operators of laed_amd.ops in 64-bit numpy, from their definitions, with running error bounds where outputs are rounded.

Unit of a bound: E = 2^-24, half a step of fp32 relative to the value (the largest error of one rounding)."""
import numpy as np

E = 2.0 ** -24
HALF_STEP = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}


def sigmoid(f):
    return np.where(f >= 0, 1.0 / (1.0 + np.exp(-np.abs(f))), np.exp(-np.abs(f)) / (1.0 + np.exp(-np.abs(f))))


def gated_scan(gi, h0=None, lengths=None, reverse=False, dout=None, dhT=None):
    """gi [T,B,2H] float64 -> dict of out, hT (and dgi, dh0) with a bound of the fp32 kernel's error beside each ("out_err"...).

    Bounds.  A gate comes from 2^(f log2 e): the argument carries (1 + 1/2) E relative, so the exponential carries 1.5 |f| E plus
    one ulp (2 E) of the instruction, the reciprocal one ulp, the sum and the product one rounding each: k E with
    k = 6 + 1.5 |f| for the smaller gate, and no more for the larger one (1 - smaller).  A step h' = z h + u x then adds
    (k z |h| + (k + 1) u |x| + |h'|) E to z times the error before it.  Steps grouped in blocks (the state in front of a
    block times the block's product of z, plus the block's own sum) round each of those three quantities once more per
    level of grouping: a factor of 4 covers three levels.
    Backwards g' = z (g + d): a block of steps computes A g + q with q = z d, each product rounded before the sum, so its
    error goes by z |g| + z |d| also where g and d cancel (z = 1/2, g = 1, d = -1 + 2^-20: the products 1/2 and -1/2 + 2^-21
    are off by up to k E / 2 each, the exact result is 2^-21): (k + 1) E z (|g| + |d|) + E |g'|, not k E |g'|."""
    T, B, H2 = gi.shape
    H = H2 // 2
    f, x = gi[:, :, :H], gi[:, :, H:]
    z, u = sigmoid(f), sigmoid(-f)
    k = 6 + 1.5 * np.abs(np.where(np.isfinite(f), f, 0))
    mask = np.ones((T, B, 1), bool) if lengths is None else (np.arange(T)[:, None] < np.asarray(lengths)[None, :])[:, :, None]
    h = np.zeros((B, H)) if h0 is None else h0.astype(np.float64).copy()
    eh = np.zeros((B, H))
    out, before, e_out, e_before = np.zeros((T, B, H)), np.zeros((T, B, H)), np.zeros((T, B, H)), np.zeros((T, B, H))
    order = range(T - 1, -1, -1) if reverse else range(T)
    for t in order:
        before[t], e_before[t] = h, eh
        ux = np.where(mask[t], u[t] * np.where(mask[t], x[t], 0), 0)
        new = z[t] * h + ux
        e = z[t] * eh + E * (k[t] * z[t] * np.abs(h) + (k[t] + 1) * np.abs(ux) + np.abs(new))
        h, eh = np.where(mask[t], new, h), np.where(mask[t], e, eh)
        out[t], e_out[t] = np.where(mask[t], h, 0), np.where(mask[t], eh, 0)
    got = {"out": out, "hT": h, "out_err": 4 * e_out, "hT_err": 4 * eh}
    if dout is None and dhT is None:
        return got
    dout = np.zeros((T, B, H)) if dout is None else dout
    g = np.zeros((B, H)) if dhT is None else dhT.astype(np.float64).copy()
    eg = np.zeros((B, H))
    dgi, e_dgi = np.zeros((T, B, H2)), np.zeros((T, B, H2))
    for t in reversed(list(order)):
        at = g + np.where(mask[t], dout[t], 0)
        e_at = eg + E * np.abs(at)
        xs, zu = np.where(mask[t], x[t], 0), z[t] * u[t]
        d = before[t] - xs
        dx, df, back = u[t] * at, at * d * zu, z[t] * at
        e_dx = u[t] * e_at + (k[t] + 1) * E * np.abs(dx)
        e_df = np.abs(d) * zu * e_at + np.abs(at) * zu * (e_before[t] + E * np.abs(d)) + (2 * k[t] + 3) * E * np.abs(df)
        e_back = z[t] * eg + E * ((k[t] + 1) * z[t] * (np.abs(g) + np.abs(at - g)) + np.abs(back))
        dgi[t, :, :H], dgi[t, :, H:] = np.where(mask[t], df, 0), np.where(mask[t], dx, 0)
        e_dgi[t, :, :H], e_dgi[t, :, H:] = np.where(mask[t], e_df, 0), np.where(mask[t], e_dx, 0)
        g, eg = np.where(mask[t], back, g), np.where(mask[t], e_back, eg)
    got.update(dgi=dgi, dh0=g, dgi_err=4 * e_dgi, dh0_err=4 * eg)
    return got


def keep_draws(seed, offset, n):
    """The counter generator's 24-bit draws [n]; the uniform number is draw / 2^24."""
    def mix(v):
        v = v + np.uint64(0x9E3779B97F4A7C15)
        v = (v ^ (v >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
        v = (v ^ (v >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
        return v ^ (v >> np.uint64(31))

    with np.errstate(over="ignore"):
        key = mix(np.array([seed & 0xFFFFFFFFFFFFFFFF], dtype=np.uint64))
        index = np.arange(n, dtype=np.uint64) + np.uint64(offset & 0xFFFFFFFFFFFFFFFF)
        return (mix((index * np.uint64(0xD6E8FEB86659FD93)) ^ key) >> np.uint64(40)).astype(np.int64)


def dropout(x, p, seed, offset, residual=None):
    """x float64, row-major -> (y, bound of the fp32 arithmetic's error): the factor 1/(1-p) and its product are rounded once
    each, the sum with the residual once."""
    keep = (keep_draws(seed, offset, x.size) / 2.0 ** 24 >= np.float64(np.float32(p))).reshape(x.shape)
    xs = np.where(keep, x / (1 - p) if p < 1 else 0.0, 0.0)
    y = xs if residual is None else xs + residual
    return y, E * (2 * np.abs(xs) + (0 if residual is None else np.abs(y))) * 1.001, keep


def sample_row(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One row (float64 array of the stored values) -> (token, log-probability)."""
    l = np.where(np.isnan(logits), -np.inf, logits) + 0.0
    V = len(l)
    m = l.max()
    if m == -np.inf:
        return -1, -np.inf
    if not temperature > 0:
        return int(np.argmax(l)), 0.0
    with np.errstate(invalid="ignore", over="ignore"):
        y = np.where(l == m, 0.0, (l - m) / temperature)
    w = np.exp(y)
    order = np.lexsort((np.arange(V), -l))                          # by value descending, then by index
    kept = l > -np.inf
    if 0 < top_k < V:
        chosen = np.zeros(V, bool)
        chosen[order[:top_k]] = True
        kept &= chosen
    if top_p < 1:
        ws = np.where(kept, w, 0.0)[order]
        mass = np.cumsum(ws)
        inside = mass - ws < max(top_p, 0.0) * mass[-1]
        inside[0] = True
        chosen = np.zeros(V, bool)
        chosen[order[inside]] = True
        kept &= chosen
    if min_p > 0:
        kept &= y >= np.log(min(min_p, 1.0))
    line = np.cumsum(np.where(kept, w, 0.0))
    u = 0.0 if not u > 0 else min(float(u), 1.0 - 2.0 ** -24)
    token = int(np.argmax(line > u * line[-1]))
    return token, float(y[token] - np.log(line[-1]))
