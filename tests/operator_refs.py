"""The operators around the layer from their definitions, in 64 bits (numpy), with bounds on the error of
a computation in 32 bits.

Each bound is a sum of worst cases: a rounding to f32 is off by at most u = 2^-24 of the value, one to
bf16 by 2^-8; a sum of n terms in chains of at most k additions by k u of the sum of magnitudes."""
import numpy as np

from gyro_moe import synth

U32 = 2.0 ** -24
HALF_STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8}
Q4_0, Q4_1 = 2, 3
BLOCK = {Q4_0: 18, Q4_1: 20}


def q4_matrix(seed, kind, rows, cols, negative=True):
    """Packed bytes [rows, cols/32 * 18|20] and the exact weights [rows, cols] they stand for."""
    rng = np.random.default_rng(seed)
    g = cols // 32
    q = rng.integers(0, 16, (rows, g, 32), dtype=np.uint8)
    d = (np.exp(rng.normal(0, 0.5, (rows, g, 1))) / 8).astype(np.float16)
    if negative:
        d = d * rng.choice(np.array([-1, 1], np.float16), d.shape)
    d[rng.random(d.shape) < 0.05] = 0.0
    m = (rng.normal(0, 0.5, (rows, g, 1))).astype(np.float16)
    packed = [d.view(np.uint8)] + ([m.view(np.uint8)] if kind == Q4_1 else []) + [q[..., :16] | (q[..., 16:] << 4)]
    packed = np.concatenate(packed, axis=2).reshape(rows, -1)
    w, mag = q4_weights(packed, kind, cols)
    return packed, w, mag


def q4_weights(packed, kind, cols):
    """Exact weights, and the magnitudes |d| q + |d| 8 (or |d| q + |m|) that a product may be summed from."""
    b = packed.reshape(packed.shape[0], cols // 32, BLOCK[kind])
    half = np.ascontiguousarray(b[..., :-16]).view(np.float16).astype(np.float64)
    q = np.concatenate([b[..., -16:] & 15, b[..., -16:] >> 4], axis=2).astype(np.float64)
    d = half[..., :1]
    off = -8.0 * d if kind == Q4_0 else half[..., 1:]
    shape = (packed.shape[0], cols)
    return (d * q + off).reshape(shape), (np.abs(d) * q + np.abs(off)).reshape(shape)


def linear(x, w, mag, y_kind):
    """y and its bound. A group of 32 columns is summed in at most two matrix products of 17 terms with
    f32 accumulators that may truncate (34 * 2 u), the groups in a chain of up to cols / 32 additions,
    and an activation keeps 22 bits of its token's largest value or better (2^-23 of it). More tokens are
    summed in steps of 16 terms whose truncations may point alike, cols / 8 * 2 u at worst; they are held to
    the same bound."""
    x = x.astype(np.float64)
    y = x @ w.T
    s = np.abs(x) @ mag.T
    big = np.abs(x).max(1, keepdims=True) * mag.sum(1)[None]
    cols = x.shape[1]
    bound = s * (68 * U32 + (cols / 32 + 8) * U32 + 2.0 ** -23) + big * 2.0 ** -38
    return y, bound + HALF_STEP[y_kind] * (np.abs(y) + bound)


def norm_rel(width):
    """Relative bound of x / sqrt(mean x^2 + eps) * w: the sum of squares in chains of at most
    width / 32 + 32 additions, halved by the root, and 8 more roundings."""
    return (0.5 * (width / 32 + 32) + 8) * U32


def norm(x, weight, eps, kind, gate_w=None):
    x = x.astype(np.float64)
    w = np.ones(x.shape[1]) if weight is None else weight.astype(np.float64)
    y = x / np.sqrt((x * x).mean(1, keepdims=True) + eps) * w
    rel = norm_rel(x.shape[1])
    out = [(y, np.abs(y) * (rel + HALF_STEP[kind] * (1 + rel)))]
    if gate_w is not None:
        out.append(dot(y, np.abs(y) * rel, gate_w))
    return out


def dot(h, dh, gate_w):
    g = gate_w.astype(np.float64)
    return h @ g, (np.abs(h) @ np.abs(g)) * (h.shape[1] / 32 + 32) * U32 + dh @ np.abs(g)


def sigmoid(v):
    return 1.0 / (1.0 + np.exp(-v.astype(np.float64)))


def residual(y, res, post, post_norm, eps, a, b, gate, next_w, has_out, kinds, gate_w=None):
    """[(res_out, bound), (out, bound), (next_gate, bound)]; kinds: encodings of res and out."""
    y, res = y.astype(np.float64), res.astype(np.float64)
    width, rel = y.shape[1], 0.0
    v = y
    if post_norm:
        v = y / np.sqrt((y * y).mean(1, keepdims=True) + eps)
        v = v * (1.0 if post is None else post.astype(np.float64))
        rel = norm_rel(width)
    if gate is not None:
        g = sigmoid(gate if gate.ndim == 2 else gate[:, None])
        v = v * g
        # expf is off by at most 2 units in the last place (4 u), 1 + e, the quotient and the product by u
        rel += 8 * U32
    # block_scale * gate * v and its sum with res_scale * res: four more roundings
    r = a * res + b * v
    dr = np.abs(b * v) * (rel + 3 * U32) + np.abs(a * res) * U32 + 2 * U32 * (np.abs(a * res) + np.abs(b * v))
    out = [(r, dr + HALF_STEP[kinds[0]] * (np.abs(r) + dr))]
    if has_out:
        scale = 1.0 / np.sqrt((r * r).mean(1, keepdims=True) + eps)
        w = np.ones(width) if next_w is None else next_w.astype(np.float64)
        h = r * scale * w
        # the root mean square moves by at most the norm of the errors over the norm of the row
        size = np.sqrt((r * r).sum(1, keepdims=True) + width * eps)
        shift = np.sqrt((dr * dr).sum(1, keepdims=True)) / size
        dh = dr * scale * np.abs(w) * (1 + shift) + np.abs(h) * (norm_rel(width) + 2 * shift)
        out.append((h, dh + HALF_STEP[kinds[1]] * (np.abs(h) + dh)))
        if gate_w is not None:
            out.append(dot(h, dh, gate_w))
    return out


def logprobs(x, tokens, n_top, scale):
    """dict of outputs, and of bounds for the floating ones. x is one row set [n, V] (f32 values)."""
    x = x.astype(np.float64)
    n, V = x.shape
    scale = float(np.float32(scale))
    bad = np.isnan(x).any(1) | (x == np.inf).any(1)
    # NaN orders below -Inf
    key = np.where(np.isnan(x), -np.inf, x) + 0.0
    order = np.lexsort((np.broadcast_to(np.arange(V), x.shape), np.isnan(x), -key), axis=1)
    top = order[:, :n_top]
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        m = x.max(1, keepdims=True)
        empty = (m == -np.inf)
        t = np.where(empty, 0.0, (x - m) * scale)
        e = np.exp(t)
        s = e.sum(1, keepdims=True)
        lp = t - np.log(s)
        et = np.where(e > 0, e * t, 0.0).sum(1) / s[:, 0]
        ent = np.log(s[:, 0]) - et
        lp[bad], ent[bad] = np.nan, np.nan
        # (x - m) * scale is off by 2 u |t|, e^t by that and 4 u more; the sums run in chains of at most
        # V / 128 + 64 additions; the terms below 2^-126 that may be dropped add V 2^-100
        chain = V / 128 + 64
        absum = np.where(e > 0, e * np.abs(t), 0.0).sum(1) / s[:, 0]
        sq = np.where(e > 0, e * t * t, 0.0).sum(1) / s[:, 0]
        ds = (2 * absum + 4 + chain) * U32 + V * 2.0 ** -100
        dls = ds + 2 * U32 * (1 + np.log(s[:, 0]))
        dent = dls + (2 * sq + (4 + chain) * absum + 2 * absum) * U32 + absum * ds + 4 * U32 * (absum + np.abs(ent))
        dlp = lambda v: np.where(np.isfinite(v), (2 * np.abs(np.where(np.isfinite(v), v, 0.0)) + 2) * U32 * 2, 0.0)  # noqa: E731
    rows = np.arange(n)
    tok = np.minimum(tokens.astype(np.int64), V - 1)
    given = (tokens < V)
    xt = x[rows, tok][:, None]
    above = np.where(np.isnan(xt), ~np.isnan(x), x > xt).sum(1)
    # an f32 result past the largest f32 by more than half its step is an infinity (round to nearest)
    far = np.isfinite(lp) & (np.abs(lp) >= 2.0 ** 128 - 2.0 ** 103)
    lp = np.where(far, np.where(lp < 0, -np.inf, np.inf), lp)
    logprob = np.where(given, lp[rows, tok], np.where(tokens == 0xFFFFFFFF, 0.0, np.nan))
    top_lp = np.take_along_axis(lp, top, 1)
    values = {"logprob": logprob, "entropy": ent, "rank": np.where(given, above + 1, 0), "top_ids": top,
              "top_logprobs": top_lp}
    bounds = {"logprob": dlp(logprob) + dls, "entropy": dent, "top_logprobs": dlp(top_lp) + dls[:, None]}
    return values, bounds


def to_kind(a, kind):
    """f32 values that the encoding holds exactly."""
    a = np.asarray(a, np.float32)
    return synth.bf16_round(a) if kind == "bf16" else a
