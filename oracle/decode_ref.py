"""float64 numpy statements of the decode operators and of how far a result may be from them.
TEST INFRASTRUCTURE ONLY: nothing in the product may import it.

Every function that returns a reference returns a bound with it where the result is computed in f32: the bound
counts the roundings (U = 2^-24 each, 2^-23 for a step of a tensor-core accumulation, which may cut instead of
round) times the magnitudes that are added up, and half a step of the result's type at the end.
"""
import numpy as np

BLOCK = 64
U = 2.0 ** -24
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}   # of a normal number, relative
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -133}     # half a step of a denormal one (f32: a whole one)


def round_to(x, kind):
    """x (any float array) rounded once to the type; the values, as float32 (bf16 has no numpy type)."""
    if kind == "f16":
        with np.errstate(over="ignore"):
            return np.asarray(x).astype(np.float16).astype(np.float32)
    x = np.asarray(x).astype(np.float32)
    if kind == "f32":
        return x
    u = x.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint32) << 16
    return np.where(np.isnan(x), np.float32(np.nan), r.astype(np.uint32).view(np.float32))


def store(x, kind):
    """Values of the type as the array the binding takes: f32, f16, or bf16 as uint16 bits."""
    if kind == "bf16":
        return (np.ascontiguousarray(x, np.float32).view(np.uint32) >> 16).astype(np.uint16)
    return np.asarray(x).astype(np.float16 if kind == "f16" else np.float32)


def load(a, kind):
    return (a.astype(np.uint32) << 16).view(np.float32) if kind == "bf16" else np.asarray(a).astype(np.float32)


def rounding(ref, kind):
    return np.abs(ref) * HALF_STEP[kind] + TINY[kind]


# ---- norm and rotation ------------------------------------------------------------------------------------------------
def norm_rope(x, w, cos, sin, eps, positions):
    """x [..., tokens, D], positions [..., tokens] or [tokens]; returns (reference, bound on the f32 part)."""
    x = np.asarray(x, np.float64)
    d = x.shape[-1]
    r = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + float(np.float32(eps)))
    y = x * r * np.asarray(w, np.float64)
    c, s = np.asarray(cos, np.float64)[positions], np.asarray(sin, np.float64)[positions]
    lo, hi = y[..., : d // 2], y[..., d // 2:]
    ref = np.concatenate([lo * c - hi * s, hi * c + lo * s], -1)
    size = np.concatenate([np.abs(lo * c) + np.abs(hi * s), np.abs(hi * c) + np.abs(lo * s)], -1)
    # the sum of squares: at most d additions and a product each, halved by the root; then the root, the quotient, two
    # products, a product and a sum
    return ref, size * (d / 2 + 8) * U


# ---- the cache ----------------------------------------------------------------------------------------------------------
def codes(x):
    """x [tokens, D] of one head (values of the type): (codes int, scale per block, f32)."""
    n = -(-x.shape[0] // BLOCK)
    out, scales = np.zeros(x.shape, np.int64), np.zeros(n, np.float32)
    for b in range(n):
        part = np.asarray(x[b * BLOCK: (b + 1) * BLOCK], np.float64)
        if not np.isfinite(part).all():
            scales[b] = np.nan
            continue
        top = max(np.abs(part).max(), 2.0 ** -100)
        out[b * BLOCK: (b + 1) * BLOCK] = np.rint(127.0 * part / top)
        scales[b] = min(np.float32(top) / np.float32(127), np.float32(float.fromhex("0x1.020406p+121")))     # 127 times it is finite
    return out, scales


def stands_for(x):
    """The f32 values of the codes of x [tokens, D]."""
    c, s = codes(x)
    return c.astype(np.float32) * np.repeat(s, BLOCK)[: x.shape[0], None]


def attention(q, k, v, scale, count=None, kind="f32"):
    """One sequence: q [heads, t, D], k and v [kv_heads, tokens, D] (values the codes stand for); the first `count` queries
    stand at the last positions.  Returns (reference, bound)."""
    heads, t, d = q.shape
    kv, n, _ = k.shape
    count = t if count is None else count
    ref, bound = np.zeros((heads, t, d)), np.zeros((heads, t, d))
    scale = float(np.float32(scale))
    for h in range(heads):
        kk, vv = np.asarray(k[h * kv // heads], np.float64), np.asarray(v[h * kv // heads], np.float64)
        for i in range(count):
            m = max(n - count + i + 1, 0)
            if m == 0:
                continue
            qq = np.asarray(q[h, i], np.float64)
            s = kk[:m] @ qq * scale
            # scores: the query keeps 22 bits; two accumulations of d / 16 steps; scale, block scale and log2(e)
            ds = np.abs(scale) * (np.abs(kk[:m]) @ np.abs(qq)) * (2 * (d / 16 + 2) * 2.0 ** -23 + 2.0 ** -21 + 4 * U) + np.abs(s) * 4 * U
            p = np.exp(s - s.max())
            total = p.sum()
            ref[h, i] = p @ vv[:m] / total
            # probabilities: two scores' errors each way, the exponential, the rescalings of the running maximum
            # (one a block and two joins), the sums of m / 16 steps; of a small probability 2^-40 of the largest may be lost
            rel = 2 * ds.max() * 1.01 + (m / 16 + m / BLOCK + 40) * 2.0 ** -23
            bound[h, i] = 2 * rel * (p @ np.abs(vv[:m])) / total + 2.0 ** -39 * np.abs(vv[:m]).sum(0) / total
    return ref, bound + rounding(ref, kind)


# ---- 4-bit weights --------------------------------------------------------------------------------------------------------
def q4_quantize(w, group, kind):
    """w [n, k] values of the type: (codes -8..7, scales [n, groups] values of the type)."""
    n, k = w.shape
    pad = np.concatenate([w, np.zeros((n, -k % group), np.float32)], 1).reshape(n, -1, group)
    top = np.abs(pad).max(-1)
    with np.errstate(invalid="ignore", divide="ignore"):
        scales = round_to(top.astype(np.float32) * np.float32(1 / 7), kind)
        x = np.rint(pad.astype(np.float64) / np.where(scales > 0, scales, 1).astype(np.float64)[..., None])
    x = np.where((scales > 0)[..., None], x, 0)
    return np.clip(x, -8, 7).astype(np.int64).reshape(n, -1)[:, :k], scales


def q4_values(c, scales, group):
    """The values the codes stand for, exactly (a product of 4 and at most 24 bits)."""
    return c.astype(np.float64) * np.repeat(scales.astype(np.float64), group, 1)[:, : c.shape[1]]


def q4_product(x, values, kind, through=None):
    """x [m, k] times values [n, k] transposed; `through`: the type that the weights are rounded to on the way, if they are."""
    x = np.asarray(x, np.float64)
    ref = x @ values.T
    size = np.abs(x) @ np.abs(values).T
    k = x.shape[1]
    bound = size * (k / 16 + k / 32 + 24) * 2.0 ** -23
    if through:
        bound = size * (k + 8) * 2.0 ** -23 + size * HALF_STEP[through]
    return ref, bound + rounding(ref, kind)
