"""Plain statement of the 4-bit cache and the attention over it (NumPy, float64)."""
import numpy as np

GROUP = 32


def quantise(x):
    """Rows [..., dim] -> (codes, steps, smallest values), the last two per group of 32 columns and rounded to float16.  A code is the
    nearest to (x - m) / s, the even one of two as near; magnitudes end at 65504, NaN counts for neither bound and has code 0."""
    x = np.clip(np.asarray(x, dtype=np.float64), -65504, 65504).reshape(*np.shape(x)[:-1], -1, GROUP)
    nothing = np.isnan(x).all(-1)
    low = np.where(nothing, 0.0, np.where(np.isnan(x), np.inf, x).min(-1))
    high = np.where(nothing, 0.0, np.where(np.isnan(x), -np.inf, x).max(-1))
    m = low.astype(np.float32).astype(np.float16)
    s = ((high - low) / 15).astype(np.float32).astype(np.float16)
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.rint((x - m.astype(np.float64)[..., None]) / s.astype(np.float64)[..., None])
    q = np.where((s[..., None] > 0) & ~np.isnan(q), np.clip(q, 0, 15), 0)
    return q.reshape(*x.shape[:-2], -1), s, m


def values(codes, s, m):
    """What codes stand for."""
    q = codes.reshape(*codes.shape[:-1], -1, GROUP)
    return (m.astype(np.float64)[..., None] + s.astype(np.float64)[..., None] * q).reshape(codes.shape)


def held(x):
    """What a cache holds of rows [..., dim]."""
    return values(*quantise(x))


def coded(x):
    """The part s code of what is held."""
    q, s, _ = quantise(x)
    return values(q, s, np.zeros_like(s))


def attend(q, k, v, past, scale, window=0, sinks=None, parts=0.0):
    """q [batch, seq, heads, dim] at positions past[b] + i over held rows k, v [batch, kv_heads, positions, dim].  Returns the outputs, the
    weighted sums of |v| and of `parts` (like v, not negative), and for each query the largest sum of |q| |k| over its positions: what
    rounding scales with."""
    parts = np.broadcast_to(parts, np.shape(v))
    q, k, v = (np.asarray(t, dtype=np.float64) for t in (q, k, v))
    batch, seq, heads, dim = q.shape
    each = heads // k.shape[1]
    out, size, reach = np.zeros(q.shape), np.zeros(q.shape), np.zeros((batch, seq, heads))
    for b in range(batch):
        for i in range(seq):
            at = int(past[b]) + i
            first, last = max(0, at - window + 1) if window else 0, min(at, k.shape[2] - 1)
            if first > last:
                continue
            for h in range(heads):
                keys, vals = k[b, h // each, first:last + 1], v[b, h // each, first:last + 1]
                x = keys @ q[b, i, h] * scale
                sink = -np.inf if sinks is None else float(sinks[h])
                top = max(x.max(), sink)
                e = np.exp(x - top)
                p = e / (e.sum() + np.exp(sink - top))
                out[b, i, h], size[b, i, h] = p @ vals, p @ (np.abs(vals) + parts[b, h // each, first:last + 1])
                reach[b, i, h] = (np.abs(keys) @ np.abs(q[b, i, h])).max() * abs(scale)
    return out, size, reach
