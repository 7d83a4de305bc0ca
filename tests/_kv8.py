"""The 8-bit cache, the attention over it with windows, its positions' weights and their eviction in 64 bits, for the
tests (numpy, no library code)."""
import numpy as np

BLOCK = 32
MOST = 448.0  # the largest 8-bit float


def nearest8(y):
    """the 8-bit float (4 exponent bits, 3 of mantissa) nearest to y, halves to even; |y| <= 448"""
    y = np.asarray(y, np.float64)
    step = np.ldexp(1.0, np.maximum(np.frexp(y)[1] - 4, -9))
    return np.rint(y / step) * step


def exponent(top):
    """the smallest E in [-15, 8] with top <= 448 * 2^E"""
    e = np.full(np.shape(top), 8)
    for k in range(7, -16, -1):
        e = np.where(np.asarray(top) <= MOST * 2.0 ** k, k, e)
    return e


def block(x):
    """what the rows x [n][heads][hd] of one block stand for; NaN rows are NaN in all channels"""
    x = np.asarray(x, np.float64)
    with np.errstate(invalid="ignore"):
        bad = ~(np.abs(x) <= 65504).all(-1)
    top = np.where(bad[..., None], 0.0, np.abs(x)).max((0, 2), initial=0.0)
    scale = np.ldexp(1.0, exponent(top))[None, :, None]
    # (what would be 2^16, beyond fp16, is the number below)
    return np.where(bad[..., None], np.nan, np.clip(nearest8(np.where(bad[..., None], 0.0, x) / scale) * scale, -61440, 61440))


def append(held, P, rows):
    """a sequence that holds `held` [T][heads][hd] after `rows` came from position P on"""
    first = P // BLOCK * BLOCK
    out = [np.asarray(held, np.float64)[:first]]
    tail = np.concatenate([np.asarray(held, np.float64)[first:P], np.asarray(rows, np.float64)])
    return np.concatenate(out + [block(tail[a:a + BLOCK]) for a in range(0, len(tail), BLOCK)]) if len(tail) else out[0]


def visible(n, T, mask=None, window=0, sinks=0):
    """[n][T]: what the last n of T positions see; mask: bool [n][n] among themselves"""
    i, j = np.arange(n)[:, None] + (T - n), np.arange(T)[None]
    seen = j <= i
    if mask is not None:
        seen = np.concatenate([np.ones((n, max(0, T - n)), bool), mask[:, max(0, n - T):]], 1)
    if window:
        seen = seen & ((j < sinks) | (j > i - window))
    return seen


def words(mask):
    """bits of a bool mask [n][n] as [n][words] uint64"""
    n = len(mask)
    out = np.zeros((n, -(-n // 64)), np.uint64)
    for i, j in np.argwhere(mask):
        out[i, j // 64] |= np.uint64(1) << np.uint64(j % 64)
    return out


class Attention:
    """Everything about the attention of q [rows][H][hd] over k, v [T][KV][hd] with `seen` [rows][T]."""

    def __init__(self, q, k, v, seen, scale):
        self.q, self.k, self.v, self.seen = (np.asarray(a, np.float64) for a in (q, k, v, seen))
        self.seen = np.asarray(seen, bool)
        self.scale, self.rep = float(scale), q.shape[1] // k.shape[1]

    def head(self, h):
        """(scores with -inf where nothing is seen, their magnitude's bound)"""
        k = self.k[:, h // self.rep]
        with np.errstate(invalid="ignore"):
            s = np.where(self.seen, self.q[:, h] @ np.where(np.isnan(k), 0, k).T * self.scale, -np.inf)
            nan = np.isnan(k).any(-1)
            s[:, nan] = np.where(self.seen[:, nan], np.nan, -np.inf)
            mag = np.abs(self.q[:, h]) @ np.abs(np.where(np.isnan(k), 0, k)).T * abs(self.scale)
        return s, float(np.nanmax(np.where(self.seen & np.isfinite(mag), mag, 0), initial=0.0))

    def check(self, out, lse=None):
        """Within the roundings: fp16 weights (half a step, 2^-11, of each, and 2^-25 where they are subnormal, of weights whose
        largest is at least 2^7), the fp16 result (2^-11), fp32 scores (hd products and sums, 2^-23 each of their magnitude)
        inside the exponential, fp32 sums and outputs (2^-24 a term) of the log-sum-exp."""
        hd, T = self.q.shape[-1], self.k.shape[0]
        for h in range(self.q.shape[1]):
            s, smax = self.head(h)
            v = self.v[:, h // self.rep]
            with np.errstate(invalid="ignore", divide="ignore"):
                top = s.max(-1, initial=-np.inf, keepdims=True)
                w = np.exp(s - np.where(top == -np.inf, 0.0, top))
                total = w.sum(-1, keepdims=True)
                p = np.where(total > 0, w / np.where(total > 0, total, 1.0), np.where(np.isnan(total), np.nan, 0.0))
                holes = np.isnan(v).any(-1)
                clean = np.where(np.isnan(v), 0, v)
                want = np.where(np.isnan(p).any(-1, keepdims=True), np.nan, p @ clean)
                want[(self.seen & holes[None]).any(-1)] = np.nan
                mag = np.nan_to_num(p) @ np.abs(clean)
                want_lse = (top + np.log(total))[:, 0]
            score = hd * 2.0 ** -23 * smax + 2.0 ** -20
            got = np.asarray(out[:, h], np.float64)
            assert np.array_equal(np.isnan(got), np.isnan(want)), ("NaN", h)
            tol = 2.0 ** -11 * (np.abs(want) + mag) * 1.01 + 2 * score * mag + T * 2.0 ** -32 * np.abs(clean).max(initial=0.0) + 2.0 ** -25
            bad = np.abs(got - want) > tol
            assert not bad.any(), (h, float(np.nanmax(np.abs(got - want) - tol)), np.argwhere(bad)[:4].tolist())
            if lse is not None:
                g, fine = np.asarray(lse[:, h], np.float64), np.isfinite(want_lse)
                assert np.array_equal(g[~fine], want_lse[~fine], equal_nan=True), (h, g[~fine], want_lse[~fine])
                tol = 2 * score + T * 2.0 ** -24 + 2.0 ** -22 * (np.abs(want_lse[fine]) + smax + 1)
                assert np.all(np.abs(g[fine] - want_lse[fine]) <= tol), (h, float(np.max(np.abs(g[fine] - want_lse[fine]) - tol)))

    def check_weights(self, lse, got, previous=0.0, decay=1.0):
        """got [KV][T] against decay previous + sums of exp(score - lse), lse as the device has it.  Each term: the score's
        error as above, the fp32 difference of score and lse and the products with log2(e) (2^-23 each, three), and n additions."""
        hd, n = self.q.shape[-1], self.q.shape[0] * self.rep
        previous = np.broadcast_to(np.asarray(previous, np.float64), got.shape) * decay
        want, tol = previous.copy(), 2.0 ** -22 * np.abs(previous) + 2.0 ** -126
        for h in range(self.q.shape[1]):
            s, smax = self.head(h)
            ls = np.asarray(lse[:, h], np.float64)[:, None]
            with np.errstate(invalid="ignore", over="ignore"):
                w = np.where(self.seen & (ls != -np.inf), np.exp(s - ls), 0.0)
            lmax = float(np.max(np.abs(ls[np.isfinite(ls)]), initial=0.0))
            want[h // self.rep] += w.sum(0)
            rel = 2 * (hd * 2.0 ** -23 * smax) + 2.0 ** -21 * (smax + lmax) + n * 2.0 ** -23 + 2.0 ** -20
            tol[h // self.rep] += w.sum(0) * rel + n * 2.0 ** -125
        assert np.array_equal(np.isnan(got), np.isnan(want))
        bad = np.abs(got - want) > tol
        assert not bad.any(), (float(np.nanmax(np.abs(got - want) - tol)), np.argwhere(bad)[:4].tolist())


def evict(score, T, budget, sinks, recent):
    """positions of one head that stay: score [>= T] fp32"""
    n = min(T, budget)
    if T <= budget:
        return np.arange(n)
    rank = np.asarray(score[:T], np.float64).copy()
    rank[np.isnan(rank)] = -np.inf
    # NaN below -inf, equal scores by position
    order = sorted(range(sinks, T - recent), key=lambda i: (np.isnan(score[i]), -rank[i], i))[:budget - sinks - recent]
    return np.array(sorted(list(range(sinks)) + order + list(range(T - recent, T))), np.int64)
