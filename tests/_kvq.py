"""The 4-bit cache, the attention over it and filtered sampling in 64 bits, for the tests (numpy, no library code)."""
import numpy as np

GROUP = 32


def tables(n_pos, hd, theta):
    inv = float(theta) ** (-np.arange(0, hd, 2, dtype=np.float64) / hd)
    a = np.arange(n_pos, dtype=np.float64)[:, None] * inv
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def rotate(x, pos, cos, sin, interleaved):
    """x [rows][heads][hd] (f64) at positions pos [rows]"""
    c, s = (t[pos][:, None].astype(np.float64) for t in (cos, sin))
    out = np.empty_like(x, dtype=np.float64)
    h = x.shape[-1] // 2
    a, b = (slice(0, None, 2), slice(1, None, 2)) if interleaved else (slice(0, h), slice(h, None))
    out[..., a] = x[..., a] * c - x[..., b] * s
    out[..., b] = x[..., b] * c + x[..., a] * s
    return out


def store(x):
    """what x [..., hd] stands for after quantisation, as fp16"""
    g = np.asarray(x, np.float64).reshape(-1, GROUP)
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        hi, lo = g.max(1), -g.min(1)
        big = np.maximum(hi, lo)
        d = (big / 8).astype(np.float32).astype(np.float16)
        d = np.where(hi > lo, -d, d)
        bad = ~(big <= 65504) | np.isnan(g).any(1)
        d = np.where(bad, np.float16(np.nan), d).astype(np.float16)
        step = d.astype(np.float64)[:, None]
        c = np.where((step == 0) | bad[:, None], 0.0, np.clip(np.rint(g / step), -8, 7))
        return (c * step).astype(np.float32).astype(np.float16).reshape(np.shape(x))


def attend(q, k, v, visible, scale):
    """q [rows][H][hd], k and v [T][KV][hd], visible [rows][T] -> (out, sum of p |v|, largest sum of |q k| scale)"""
    rows, H, hd = q.shape
    KV = k.shape[1]
    out, mag, smax = np.zeros((rows, H, hd)), np.zeros((rows, H, hd)), 0.0
    for h in range(H):
        kh, vh = k[:, h * KV // H].astype(np.float64), v[:, h * KV // H].astype(np.float64)
        for r in range(rows):
            at = np.nonzero(visible[r])[0]
            if not at.size:
                continue
            qr = q[r, h].astype(np.float64)
            s = kh[at] @ qr * scale
            with np.errstate(invalid="ignore"):
                smax = max(smax, float(np.max(np.abs(kh[at]) @ np.abs(qr)) * abs(scale)))
                m = s.max()
                if m == -np.inf:
                    continue
                p = np.exp(s - m)
                p = p / p.sum()
                out[r, h] = p @ vh[at]
                mag[r, h] = p @ np.abs(vh[at])
    return out, mag, smax


def sample(x, u, temperature, top_k=0, top_p=1.0, min_p=0.0):
    """(token, distribution) of one row; token -1 where there is none"""
    x = np.asarray(x, np.float32).astype(np.float64)
    V = x.size
    if np.isnan(x).any() or (x == np.inf).any() or (x == -np.inf).all():
        return -1, np.zeros(V)
    if temperature == 0:
        temperature, top_k, top_p, min_p = 1.0, 1, 1.0, 0.0
    order = np.lexsort((np.arange(V), -x))
    w = np.exp((x[order] - x[order[0]]) / float(np.float32(temperature)))
    n = int(np.count_nonzero(x > -np.inf))
    if 0 < top_k < n:
        n = top_k
    if top_p < 1.0:
        c = np.cumsum(w[:n])
        n = min(n, int(np.searchsorted(c, float(np.float32(top_p)) * c[-1], side="left")) + 1)
    keep = w[:n] >= float(np.float32(min_p))
    p = np.zeros(V)
    p[order[:n][keep]] = w[:n][keep]
    c = np.cumsum(p)
    token = int(np.searchsorted(c, float(np.float32(u)) * c[-1], side="right"))
    return token, p / c[-1]
