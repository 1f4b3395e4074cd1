"""The 4-bit key/value cache and the attention over it, in numpy: decisions (scale, minimum, code) in the float32
steps of their definition, everything else in float64."""
import numpy as np

TOP = np.float32(65280.0)


def held(k, v, group):
    """float32 [..., D] keys and values (exact images of 16-bit ones) -> the values the cache holds, float64."""
    bad = (np.isnan(k) | np.isnan(v)).any(-1, keepdims=True)
    out = []
    for x in (k, v):
        with np.errstate(all="ignore"):
            f = np.where(np.isnan(x), np.float32(0), np.clip(x, -TOP, TOP)).astype(np.float32)
            g = f.reshape(*f.shape[:-1], -1, group)
            m = g.min(-1, keepdims=True).astype(np.float16).astype(np.float32)
            s = ((g.max(-1, keepdims=True) - m) * (np.float32(1) / np.float32(15))).astype(np.float16).astype(np.float32)
            c = np.where(s == 0, np.float32(0), np.clip(np.rint((g - m) / np.where(s == 0, np.float32(1), s)), 0, 15))
        y = (m.astype(np.float64) + c.astype(np.float64) * s.astype(np.float64)).reshape(f.shape)
        out.append(np.where(bad, np.nan, y))
    return out


def attention(q, k, v, pos, there, scale, window=None, sinks=0):
    """q [rows, D], k / v [tokens, D] float64, pos [rows] -> (o, bound pieces): o [rows, D] and, for the error of a
    computation with 16-bit operands, sum_j p_j |v_j - o|, sum_j p_j |v_j| and the largest scale sum_d |q_d k_jd| of a row."""
    j = np.arange(k.shape[0])
    seen = (j[None, :] <= pos[:, None]) & there[None, :]
    if window:
        seen &= (j[None, :] > pos[:, None] - window) | (j[None, :] < sinks)
    o = np.zeros((q.shape[0], v.shape[1]))
    spread, size, reach = np.zeros_like(o), np.zeros_like(o), np.zeros(q.shape[0])
    for i in range(q.shape[0]):
        w = np.flatnonzero(seen[i])
        if not w.size:
            continue
        s = scale * (k[w] @ q[i])
        e = np.exp(s - s.max())
        p = e / e.sum()
        o[i] = p @ v[w]
        spread[i] = p @ np.abs(v[w] - o[i])
        size[i] = p @ np.abs(v[w])
        reach[i] = scale * (np.abs(k[w]) @ np.abs(q[i])).max()
    return o, spread, size, reach
