"""The 8-bit paged KV cache, the attention over it, its positions' weights and their eviction (sd_kv8_*) against a 64-bit
restatement: stored values and what stays bit for bit, attention and weights within their roundings, at the lengths,
masks, windows, strides and pages where they can go wrong."""
import numpy as np
import pytest

import _kv8
import _kvq
from _devmem import Graph, Stream, dev, full, ptr, synchronize, zeros

pytestmark = pytest.mark.gpu

MAX_POS = 6000


class Pool:
    """A pool with the sequences' pages at random places and the oracle's copy of what they hold."""

    def __init__(self, hip, seed, H, KV, hd, caps, page=64, layers=1, interleaved=True, theta=10000.0, spare=2):
        self.hip, self.H, self.KV, self.hd, self.page = hip, H, KV, hd, page
        self.inter, self.rng = interleaved, np.random.default_rng(seed)
        need = [max(1, -(-n // page)) for n in caps]
        self.n_pages = sum(need) + spare
        ids = self.rng.permutation(self.n_pages).tolist()
        self.table = np.full((len(caps), max(need)), -1, np.int32)
        for s, n in enumerate(need):
            self.table[s, :n] = [ids.pop() for _ in range(n)]
        self.free = ids
        self.pool = hip.HipKv8Pool(n_layers=layers, n_heads=H, n_kv_heads=KV, head_dim=hd, n_pages=self.n_pages, page_tokens=page,
                                   max_pos=MAX_POS, rope_theta=theta, interleaved=interleaved)
        self.cos, self.sin = _kvq.tables(MAX_POS, hd, theta)
        self.dtable = dev(self.table)
        self.held = [[np.zeros((0, KV, hd)), np.zeros((0, KV, hd))] for _ in caps]

    def rows(self, n, heads, dt=np.float16):
        return (self.rng.standard_normal((n, heads, self.hd)) * (1 + 5 * (self.rng.random((1, heads, self.hd)) > .95))).astype(dt)

    def turned(self, x, pos):
        with np.errstate(invalid="ignore"):
            return _kvq.rotate(x.astype(np.float64), np.asarray(pos), self.cos, self.sin, self.inter)

    def append(self, counts, lens, k, v, layer=0, pos=None, q=None, stream=0, max_rows=None, rows=None):
        """counts[s] rows that end at lens[s]; the oracle's copy follows for layer 0 (all rows' positions must exist)"""
        dt = self.hip.F32 if k.dtype == np.float32 else self.hip.F16
        start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        a = [dev(x) for x in (k, v, start, np.asarray(lens, np.int32))]
        dp = None if pos is None else dev(np.asarray(pos, np.int32))
        dq = None if q is None else dev(q)
        qo = None if q is None else full((len(k), self.H, self.hd), 77.0, np.float16)
        synchronize()
        self.pool.append(layer, len(k) if rows is None else rows, ptr(a[2]), ptr(a[3]), ptr(self.dtable), *self.table.shape,
                         max_rows=max(max(counts), 1) if max_rows is None else max_rows, k=ptr(a[0]), v=ptr(a[1]), dtype=dt,
                         pos=ptr(dp), q=ptr(dq), q_out=ptr(qo), stream=stream)
        synchronize()
        if layer == 0 and max_rows is None:
            for s, n in enumerate(counts):
                if n:
                    at = slice(start[s], start[s] + n)
                    P = lens[s] - n
                    where = np.arange(P, lens[s]) if pos is None else np.asarray(pos)[at]
                    for i, x in enumerate((self.turned(k[at], where), v[at].astype(np.float64))):
                        self.held[s][i] = _kv8.append(self.held[s][i], P, x)
        return None if q is None else qo.get()

    def fill(self, lens, edit=None, layer=0):
        """all positions of all sequences in one call"""
        k, v = self.rows(sum(lens), self.KV), self.rows(sum(lens), self.KV)
        if edit:
            edit(k, v)
        self.append(lens, lens, k, v, layer)

    def read(self, seq, slot, layer=0, fill=5.0, table=None):
        n = len(slot)
        ds, dl = dev(np.asarray(seq, np.int32)), dev(np.asarray(slot, np.int32))
        ko, vo = (full((n, self.KV, self.hd), fill, np.float16) for _ in range(2))
        t = self.dtable if table is None else table
        self.pool.read(layer, n, ptr(dl), ptr(t), *t.shape, ptr(ko), ptr(vo), seqs=ptr(ds))
        return ko.get(), vo.get()

    def check_held(self, layer=0, table=None):
        for s, (k, v) in enumerate(self.held):
            if len(k):
                gk, gv = self.read([s] * len(k), range(len(k)), layer, table=table)
                for g, want in ((gk.astype(np.float64), k), (gv.astype(np.float64), v)):
                    bad = ~((g == want) | (np.isnan(g) & np.isnan(want)))
                    assert not bad.any(), (s, np.argwhere(bad)[:4].tolist(), g[bad][:4], want[bad][:4])

    def call(self, q, counts, lens, mask=None, table=None, **more):
        """the arguments of a query over the sequences, and what keeps them alive"""
        rows = int(sum(counts))
        start = dev(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32))
        keep = [start, dev(np.asarray(lens, np.int32)), dev(q), None if mask is None else dev(mask)]
        table = self.dtable if table is None else table
        a = dict(q=ptr(keep[2]), row_start=ptr(start), kv_len=ptr(keep[1]), table=ptr(table), n_seqs=table.shape[0],
                 table_ld=table.shape[1], rows=rows, max_rows=max(max(counts), 1), max_len=max(lens), mask=ptr(keep[3]),
                 mask_words=0 if mask is None else mask.shape[1])
        a.update(more)
        return a, keep

    def attend(self, q, counts, lens, layer=0, lse=True, out=None, **more):
        a, keep = self.call(q, counts, lens, **more)
        rows = a["rows"]
        if out is None:
            out = full((rows, self.H, self.hd), 9.0, np.float16)
        stat = full((rows, self.H), 9.0) if lse else None
        n = self.pool.attend_workspace(rows, a["n_seqs"], a["max_rows"], a["max_len"], a.get("window", 0), a.get("sinks", 0))
        ws = full((max(n, 16),), 255, np.uint8)
        synchronize()
        self.pool.attend(layer, out=ptr(out), lse=ptr(stat), ws=ptr(ws), ws_bytes=n, **a)
        return (out.get(), stat.get()) if lse else out.get()

    def weights(self, q, lse, counts, lens, ld, previous=None, layer=0, decay=1.0, out=None, **more):
        a, keep = self.call(q, counts, lens, **more)
        dl, dp = dev(lse), None if previous is None else dev(previous)
        if out is None:
            out = full((a["n_seqs"], self.KV, ld), 3.0)
        synchronize()
        self.pool.weights(layer, lse=ptr(dl), scores=ptr(out), ld=ld, previous=ptr(dp), decay=decay, **a)
        return out.get()


# ---- append and read -------------------------------------------------------------
@pytest.mark.parametrize("hd,KV,H", [(128, 8, 32), (64, 8, 8), (128, 1, 7), (64, 3, 6)])
@pytest.mark.parametrize("dt", [np.float16, np.float32])
@pytest.mark.parametrize("inter", [True, False])
def test_append_and_read(hip, hd, KV, H, dt, inter):
    """Ragged calls one after the other: whole blocks, single rows, ends inside blocks and pages."""
    p = Pool(hip, hd + KV, H, KV, hd, [300, 40, 33, 64, 5], page=32, interleaved=inter, theta=500000.0)
    lens = [0] * 5
    for counts in ([130, 1, 33, 0, 0], [1, 1, 0, 64, 1], [0, 30, 0, 0, 1], [33, 0, 0, 0, 3], [95, 8, 0, 0, 0]):
        lens = [a + b for a, b in zip(lens, counts)]
        n = sum(counts)
        k, v, q = p.rows(n, KV, dt), p.rows(n, KV, dt), p.rows(n, H, dt)
        k[n // 2, 0] = 0.0
        v[n // 3] *= np.asarray(1e-6, dt)
        pos = p.rng.integers(0, MAX_POS, n)
        qo = p.append(counts, lens, k, v, pos=pos, q=q)
        p.check_held()
        want = p.turned(q, pos)
        # an fp16 rounding and two fp32 ones of terms up to the pair's magnitude
        assert np.all(np.abs(qo.astype(np.float64) - want) <= 2.0 ** -11 * np.abs(want) + 2.0 ** -22 * np.abs(q).max() + 2.0 ** -25)


@pytest.mark.parametrize("hd", [64, 128])
def test_scales_follow_what_a_block_holds(hip, hd):
    """Single rows of very different magnitudes into one block, a rollback, and the block's end without its largest row."""
    p = Pool(hip, hd, 2, 1, hd, [96], page=32)
    at = 0
    for mag in (1.0, 1e-4, 300.0, 1e-3, 2.0, 6e4, 1e-7, 0.0, 5.0):
        k, v = p.rows(1, 1, np.float32), p.rows(1, 1, np.float32)
        k, v = (x / np.abs(x).max() * np.float32(mag) if mag else x * 0 for x in (k, v))
        at += 1
        p.append([1], [at], k.astype(np.float32), v.astype(np.float32))
        p.check_held()
    p.append([2], [6], p.rows(2, 1), p.rows(2, 1))  # positions 4 and 5 again: what was behind is gone
    p.check_held()
    assert len(p.held[0][0]) == 6
    p.append([60], [66], p.rows(60, 1), p.rows(60, 1))
    p.check_held()


def test_append_extremes_and_ties(hip):
    """Rows at the codes' borders: halves between them, the largest values, below the least scale, not finite."""
    n = 70
    p = Pool(hip, 3, 4, 2, 64, [n], page=32)
    k, v = p.rows(n, 2, np.float32), np.zeros((n, 2, 64), np.float32)
    codes = np.array([c / 512 if c < 8 else 2.0 ** (c // 8 - 7) * (1 + c % 8 / 8) for c in range(127)])
    halves = ((codes[1:] + codes[:-1]) / 2).astype(np.float32)  # exact ties of a block whose scale is 1
    v[0, :, 0] = 448.0
    v[1, 0], v[1, 1], v[2, 0], v[2, 1] = halves[:64], -halves[:64], halves[62:], -halves[62:]
    v[3, 0] = np.nextafter(halves[:64], np.float32(1e9))
    v[3, 1] = np.nextafter(halves[:64], np.float32(-1e9))
    v[32] = 2.0 ** -27  # below everything: the least scale
    v[33, 0, 0] = 2.0 ** -6
    v[40, 0, 5], v[40, 1, 5] = 65504.0, -65504.0
    v[64, 0, 7], v[65, 1, 40], v[66, 0, 1], v[67, 1, 33] = 65505.0, np.nan, np.inf, -np.inf
    k[64, 0, 2], k[65, 1, 50] = np.nan, np.inf
    k[66] *= 1e5
    p.append([n], [n], k, v)
    p.check_held()
    gk, gv = p.read([0] * n, range(n))
    assert np.isnan(gv[64, 0]).all() and not np.isnan(gv[64, 1]).any() and np.isnan(gk[66]).all()
    p.append([1], [n + 1 - 10], p.rows(1, 2), p.rows(1, 2))  # NaN rows that are behind the end are forgotten
    p.check_held()


def test_left_out_rows_and_absent_pages(hip):
    p = Pool(hip, 4, 4, 2, 128, [64, 64], page=32, layers=2)
    p.fill([64, 64])
    before = p.read([0] * 64 + [1] * 64, list(range(64)) * 2)
    p.table[1, 1] = p.n_pages  # outside the pool
    p.dtable = dev(p.table)
    k, v, q = p.rows(12, 2), p.rows(12, 2), p.rows(12, 4)
    # sequence 0: five rows of which two may be written (max_rows), ending at 3: positions -2, -1, 0 ..: only those below max_rows
    qo = p.append([5, 4], [3, 64], k, v, q=q, max_rows=2)
    assert (qo[:5] == 77.0).all() and (qo[7:] == 77.0).all() and not (qo[5:7] == 77.0).any()  # rows 5, 6: positions 60, 61
    # nothing written: no rows, past the table, a length that no sequence has
    p.append([0, 3], [64, 70], k[:3], v[:3], max_rows=3)
    p.append([0, 3], [64, 2 ** 31 - 1], k[:3], v[:3], max_rows=3)
    p.append([3, 0], [-5, 64], k[:3], v[:3], max_rows=3)
    after = p.read([0] * 64 + [1] * 64, list(range(64)) * 2, fill=7.0)
    for x, y in zip(before, after):
        assert np.array_equal(x[:96], y[:96]) and (y[96:] == 7.0).all()
    rk, rv = p.read([-1, 2, 0, 0, 1, 0, -2147483648], [3, 3, -1, 64, 40, 2147483647, 0])
    assert (rk == 5.0).all() and (rv == 5.0).all()
    lk, lv = p.read([0] * 64, range(64), layer=1)  # the other layer holds zeros
    assert not lk.any() and not lv.any()


def test_rotation_positions_that_do_not_exist_are_nan(hip):
    p = Pool(hip, 6, 4, 2, 64, [40], page=32)
    k, v, q = p.rows(5, 2), p.rows(5, 2), p.rows(5, 4)
    pos = np.array([0, -1, MAX_POS, MAX_POS - 1, 2 ** 31 - 1], np.int32)
    qo = p.append([5], [5], k, v, pos=np.clip(pos, 0, MAX_POS - 1), q=q)  # (for the oracle's copy of the good rows)
    kept = [x.copy() for x in p.held[0]]
    bad = np.array([1, 2, 4])
    k2, v2 = k.copy(), v.copy()
    k2[bad], v2[bad] = 0, 0  # they do not count for the scale
    want = [_kv8.block(p.turned(k2, np.clip(pos, 0, MAX_POS - 1))), _kv8.block(v2)]
    qn = p.append([5], [5], k, v, pos=pos, q=q, max_rows=5)
    got = p.read([0] * 5, range(5))
    for g, w in zip(got, want):
        w[bad] = np.nan
        assert np.array_equal(g.astype(np.float64), w, equal_nan=True)
    assert np.isnan(qn[bad]).all() and np.array_equal(qn[[0, 3]], qo[[0, 3]]) and len(kept[0]) == 5


def test_strided_rows(hip):
    """q, k and v as column ranges of one product's rows, as the decoder has them."""
    p = Pool(hip, 5, 4, 2, 64, [50], page=64, interleaved=False)
    n, w = 50, 8 * 64
    x = p.rng.standard_normal((n, w)).astype(np.float32)
    dx, start, lens = dev(x), dev(np.array([0, n], np.int32)), dev(np.array([n], np.int32))
    qo = zeros((n, 4, 64), np.float16)
    synchronize()
    p.pool.append(0, n, ptr(start), ptr(lens), ptr(p.dtable), 1, 1, max_rows=n, k=ptr(dx) + 4 * 256, v=ptr(dx) + 4 * 384,
                  dtype=hip.F32, q=ptr(dx), q_out=ptr(qo), q_ld=w, k_ld=w, v_ld=w)
    p.held[0] = [_kv8.append(np.zeros((0, 2, 64)), 0, y) for y in (p.turned(x[:, 256:384].reshape(n, 2, 64), range(n)),
                                                                     x[:, 384:].reshape(n, 2, 64))]
    p.check_held()
    want = p.turned(x[:, :256].reshape(n, 4, 64), range(n))
    assert np.all(np.abs(qo.get() - want) <= 2.0 ** -11 * np.abs(want) + 2.0 ** -22 * np.abs(x).max())


def test_many_ragged_sequences_in_one_append(hip):
    """One long sequence among many short ones: its blocks are dealt round fewer workgroups."""
    counts = [1] * 40 + [2000] + [3] * 20
    p = Pool(hip, 12, 2, 2, 64, counts, page=64)
    p.fill(counts)
    p.check_held()


# ---- attention -------------------------------------------------------------------
@pytest.mark.parametrize("hd,KV,H,page", [(128, 2, 8, 64), (64, 4, 4, 32), (128, 1, 7, 128), (64, 2, 16, 256), (128, 2, 2, 32)])
@pytest.mark.parametrize("rows,T", [(1, 1), (1, 2), (1, 31), (1, 32), (1, 33), (1, 777), (1, 3000), (2, 2), (5, 5), (5, 64), (5, 1025),
                                    (17, 17), (33, 100), (70, 200), (300, 301), (129, 129)])
def test_attention_causal(hip, hd, KV, H, page, rows, T):
    p = Pool(hip, rows * 7 + T, H, KV, hd, [T], page=page)
    p.fill([T])
    q = p.rows(rows, H)
    out, lse = p.attend(q, [rows], [T])
    _kv8.Attention(q, *p.held[0], _kv8.visible(rows, T), hd ** -0.5).check(out, lse)
    assert np.array_equal(p.attend(q, [rows], [T], lse=False), out)


@pytest.mark.parametrize("hd,KV,H", [(128, 2, 8), (64, 4, 4), (128, 1, 7)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 3)])
def test_attention_ragged_batch(hip, hd, KV, H, window, sinks):
    lens = [0, 1, 700, 33, 64, 5, 2000, 31]
    counts = [0, 1, 3, 0, 64, 5, 1, 2]
    p = Pool(hip, 11, H, KV, hd, lens, page=64)
    p.fill(lens)
    q = p.rows(sum(counts), H)
    out, lse = p.attend(q, counts, lens, window=window, sinks=sinks)
    at = 0
    for s, n in enumerate(counts):
        if n:
            seen = _kv8.visible(n, lens[s], window=window, sinks=sinks)
            _kv8.Attention(q[at:at + n], *p.held[s], seen, hd ** -0.5).check(out[at:at + n], lse[at:at + n])
        at += n


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows,T", [(1, 1), (7, 7), (60, 500), (64, 96), (65, 65), (128, 1000), (100, 131)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 2)])
def test_attention_tree_masks(hip, hd, rows, T, window, sinks):
    """Random masks, among them rows that see only the prefix, or (without one) nothing at all."""
    p = Pool(hip, rows + T, 4, 2, hd, [T], page=32)
    p.fill([T])
    bits = p.rng.random((rows, rows)) < 0.2
    bits[::5] = False
    mask = _kv8.words(bits)
    mask[:, -1] |= np.uint64(1) << np.uint64(63) if rows % 64 else np.uint64(0)  # a bit past the rows means nothing
    q = p.rows(rows, 4)
    out, lse = p.attend(q, [rows], [T], mask=mask, window=window, sinks=sinks)
    _kv8.Attention(q, *p.held[0], _kv8.visible(rows, T, bits, window, sinks), hd ** -0.5).check(out, lse)
    if T == rows:
        assert not out[::5].any() and (lse[::5] == -np.inf).all()


@pytest.mark.parametrize("hd,KV,H", [(128, 2, 8), (64, 4, 4)])
@pytest.mark.parametrize("rows,T", [(1, 1), (1, 2500), (4, 600), (40, 41), (100, 1000), (700, 701)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (31, 1), (32, 33), (33, 0), (100, 64), (600, 4), (5000, 4), (1 << 40, 1 << 40)])
def test_attention_windows(hip, hd, KV, H, rows, T, window, sinks):
    p = Pool(hip, rows + T + window % 97, H, KV, hd, [T], page=64)
    p.fill([T])
    q = p.rows(rows, H)
    out, lse = p.attend(q, [rows], [T], window=window, sinks=sinks)
    _kv8.Attention(q, *p.held[0], _kv8.visible(rows, T, window=window, sinks=sinks), hd ** -0.5).check(out, lse)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows", [6, 70])
@pytest.mark.parametrize("window", [0, 40])
def test_attention_nan_rows_behind_masks(hip, hd, rows, window):
    """NaN keys and values of positions that a row does not see leave it alone; a row that sees them is NaN."""
    T = 90 + rows

    def edit(k, v):
        v[T - 3, 0, 40] = np.nan
        k[T - 4, 1, 3] = np.inf
        v[T - 1, 1, 0] = np.inf
        v[60, 1, 5], k[20, 0, 1] = np.nan, np.nan
    p = Pool(hip, 8 + rows, 4, 2, hd, [T], page=32)
    p.fill([T], edit)
    q = p.rows(rows, 4)
    bits = np.tril(np.ones((rows, rows), bool))
    bits[-2, -3] = False
    bits[-1] = False
    bits[-1, [0, rows - 1]] = True
    for mask, b in ((None, None), (_kv8.words(bits), bits)):
        out, lse = p.attend(q, [rows], [T], mask=mask, window=window, sinks=0)
        a = _kv8.Attention(q, *p.held[0], _kv8.visible(rows, T, b, window, 0), hd ** -0.5)
        a.check(out, lse)
        assert np.isnan(out).any() and (window == 0 or not np.isnan(out).all())
        w = p.weights(q, lse, [rows], [T], T, mask=mask, window=window)
        a.check_weights(lse, w[0])
    # what lies behind the end does not count
    out, lse = p.attend(q[:3], [3], [60])
    _kv8.Attention(q[:3], *[x[:60] for x in p.held[0]], _kv8.visible(3, 60), hd ** -0.5).check(out, lse)


@pytest.mark.parametrize("rows", [2, 40])
@pytest.mark.parametrize("value", [1.0, 60.0, -60.0])
def test_attention_sharp_and_flat_scores(hip, value, rows):
    """Scores of some hundreds, one above the rest by far, and all alike."""
    p = Pool(hip, 21, 4, 2, 128, [300], page=64)
    p.fill([300])
    q = (p.rows(rows, 4).astype(np.float32) * value).astype(np.float16)
    for x in (q, q * np.float16(0)):
        out, lse = p.attend(x, [rows], [300])
        _kv8.Attention(x, *p.held[0], _kv8.visible(rows, 300), 128 ** -0.5).check(out, lse)


@pytest.mark.parametrize("rows", [1, 33])
def test_attention_infinite_scores(hip, rows):
    """A query of infinities: rows whose scores are all -inf weigh nothing, +inf gives NaN as the formula does."""
    p = Pool(hip, 22, 2, 1, 64, [40], page=32)
    k, v = np.ones((40, 1, 64), np.float16), p.rows(40, 1)
    p.append([40], [40], k, v, pos=[0] * 40)
    q = np.zeros((rows, 2, 64), np.float16)
    q[:, 0, 0], q[:, 1, 0] = -np.inf, np.inf
    out, lse = p.attend(q, [rows], [40])
    assert not out[:, 0].any() and np.isnan(out[:, 1]).all()
    assert (lse[:, 0] == -np.inf).all() and np.isnan(lse[:, 1]).all()
    w = p.weights(q[:, :1].repeat(2, 1), np.full((rows, 2), -np.inf, np.float32), [rows], [40], 40)
    assert not w.any()


@pytest.mark.parametrize("rows", [3, 60])
def test_attention_huge_scores(hip, rows):
    """Scores of some 10^8, whose fp32 spacing is far above 1: still no infinities, and a maximum weighs what it should."""
    p = Pool(hip, 23, 2, 1, 64, [200], page=64)
    k = (p.rng.standard_normal((200, 1, 64)) * 1e4).astype(np.float32)
    v = p.rows(200, 1, np.float32)
    p.append([200], [200], k, v)
    q = (p.rng.standard_normal((rows, 2, 64)) * 2e3).astype(np.float16)
    out, lse = p.attend(q, [rows], [200])
    assert np.isfinite(out).all() and np.isfinite(lse).all()
    assert np.all(np.abs(out.astype(np.float64)) <= np.abs(p.held[0][1]).max() * 1.01)
    a = _kv8.Attention(q, *p.held[0], _kv8.visible(rows, 200), 64 ** -0.5)
    for h in range(2):
        s, smax = a.head(h)
        assert np.all(np.abs(lse[:, h] - s.max(-1)) <= 64 * 2.0 ** -22 * smax + 10)


def test_attention_long_tail_of_small_weights(hip):
    """One position far above 5999 others that together weigh as much."""
    T = 6000
    p = Pool(hip, 24, 1, 1, 64, [T], page=64)
    k, v = np.zeros((T, 1, 64), np.float32), np.ones((T, 1, 64), np.float32)
    k[100, 0, 0] = 1.0
    v[100] = -1.0
    p.append([T], [T], k, v, pos=[0] * T)
    q = np.zeros((1, 1, 64), np.float16)
    q[0, 0, 0] = 8.0
    scale = float(np.float32(np.log(T - 1) / 8))
    out, lse = p.attend(q, [1], [T], scale=scale)
    _kv8.Attention(q, *p.held[0], _kv8.visible(1, T), scale).check(out, lse)
    assert abs(float(out[0, 0, 0])) < 1e-3


@pytest.mark.parametrize("rows", [2, 70])
def test_attention_strides_scale_and_untouched_rows(hip, rows):
    p = Pool(hip, 31, 4, 2, 64, [200, 190], page=64)
    p.fill([200, 190])
    n = 2 * (rows + 1) + 3
    wide = np.zeros((n, 4 * 64 + 24), np.float16)
    q = p.rows(n, 4)
    wide[:, :256] = q.reshape(n, 256)
    out, stat = full((n, 4 * 64 + 12), 3.0, np.float16), full((n, 4), 3.0)
    # rows + 1 rows of each sequence, of which max_rows leaves out the last; three belong to nobody
    a, keep = p.call(wide, [rows + 1, rows + 1], [200, 190], max_rows=rows, rows=n, scale=0.3, q_ld=280, out_ld=268)
    ws = zeros(max(16, p.pool.attend_workspace(n, 2, rows, 200)), np.uint8)
    synchronize()
    p.pool.attend(0, out=ptr(out), lse=ptr(stat), ws=ptr(ws), ws_bytes=ws.nbytes, **a)
    got, lse = out.get(), stat.get()
    idle = [rows, 2 * rows + 1] + list(range(n - 3, n))
    assert (got[:, 256:] == 3.0).all() and (got[idle] == 3.0).all() and (lse[idle] == 3.0).all()
    for s, T in ((0, 200), (1, 190)):
        r = slice(s * (rows + 1), s * (rows + 1) + rows)
        seen = _kv8.visible(rows + 1, T)[:rows]
        _kv8.Attention(q[r], *p.held[s], seen, np.float32(0.3)).check(got[r, :256].reshape(rows, 4, 64), lse[r])


@pytest.mark.parametrize("rows", [1, 50])
def test_attention_absent_pages(hip, rows):
    """Page ids outside the pool and tables shorter than the length hold nothing."""
    p = Pool(hip, 33, 4, 2, 128, [320], page=64)
    p.fill([320])
    q = p.rows(rows, 4)
    t = p.table.copy()
    t[0, 1], t[0, 2] = -1, p.n_pages + 7
    seen = _kv8.visible(rows, 320)
    seen[:, 64:192] = False
    for table, hole in ((t, 320), (t[:, :1], 64), (np.full((1, 5), -1, np.int32), 0)):
        seen[:, hole:] = False
        dt = dev(np.ascontiguousarray(table))
        out, lse = p.attend(q, [rows], [320], table=dt)
        a = _kv8.Attention(q, *p.held[0], seen, 128 ** -0.5)
        a.check(out, lse)
        a.check_weights(lse, p.weights(q, lse, [rows], [320], 320, table=dt)[0])
    assert not out.any() and (lse == -np.inf).all()


@pytest.mark.parametrize("rows", [6, 40])
def test_attention_fewer_positions_than_rows(hip, rows):
    """Rows before the first position see nothing."""
    p = Pool(hip, 34, 2, 1, 64, [80], page=32)
    p.fill([80])
    q = p.rows(rows, 2)
    out, lse = p.attend(q, [rows], [2])
    assert not out[:-2].any() and (lse[:-2] == -np.inf).all()
    _kv8.Attention(q[-2:], *[x[:2] for x in p.held[0]], _kv8.visible(2, 2), 64 ** -0.5).check(out[-2:], lse[-2:])
    for T in (0, -7):
        out, lse = p.attend(q, [rows], [T], max_len=1)
        assert not out.any() and (lse == -np.inf).all()
    # a length past max_len costs time, not correctness
    out, lse = p.attend(q, [rows], [80], max_len=1)
    _kv8.Attention(q, *p.held[0], _kv8.visible(rows, 80), 64 ** -0.5).check(out, lse)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("KV,H,seqs,most", [(8, 32, 32, 20), (16, 16, 8, 300)])
def test_attention_many_rows_in_many_sequences(hip, hd, KV, H, seqs, most):
    rng = np.random.default_rng(seqs)
    counts = [most, 0, 1] + [int(v) for v in rng.integers(1, most, seqs - 3)]
    lens = [c + int(v) for c, v in zip(counts, rng.integers(0, 200, seqs))]
    p = Pool(hip, 77, H, KV, hd, lens, page=64)
    p.fill(lens)
    q = p.rows(sum(counts), H)
    out, lse = p.attend(q, counts, lens)
    at = 0
    for s, n in enumerate(counts):
        if n and s < 6:
            _kv8.Attention(q[at:at + n], *p.held[s], _kv8.visible(n, lens[s]), hd ** -0.5).check(out[at:at + n], lse[at:at + n])
        at += n


@pytest.mark.parametrize("rows,max_len", [(1, 700), (1, 100000), (40, 700), (40, 100000)])
def test_results_are_the_same_every_time(hip, rows, max_len):
    p = Pool(hip, 51, 8, 2, 128, [700], page=64)
    p.fill([700])
    q = p.rows(rows, 8)
    first = p.attend(q, [rows], [700], max_len=max_len)
    w = p.weights(q, first[1], [rows], [700], 700, max_len=max_len)
    _kv8.Attention(q, *p.held[0], _kv8.visible(rows, 700), 128 ** -0.5).check(*first)
    for _ in range(5):
        again = p.attend(q, [rows], [700], max_len=max_len)
        assert np.array_equal(first[0], again[0]) and np.array_equal(first[1], again[1])
        assert np.array_equal(w, p.weights(q, first[1], [rows], [700], 700, max_len=max_len))


# ---- weights ---------------------------------------------------------------------
@pytest.mark.parametrize("hd,KV,H", [(128, 2, 8), (64, 4, 4), (128, 1, 7), (64, 2, 16)])
@pytest.mark.parametrize("rows,T", [(1, 1), (1, 33), (1, 1500), (5, 64), (33, 100), (300, 301), (129, 2000)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 3)])
def test_weights(hip, hd, KV, H, rows, T, window, sinks):
    p = Pool(hip, rows + T, H, KV, hd, [T], page=64)
    p.fill([T])
    q = p.rows(rows, H)
    _, lse = p.attend(q, [rows], [T], window=window, sinks=sinks)
    a = _kv8.Attention(q, *p.held[0], _kv8.visible(rows, T, window=window, sinks=sinks), hd ** -0.5)
    w = p.weights(q, lse, [rows], [T], T + 5, window=window, sinks=sinks)
    assert (w[0, :, T:] == 3.0).all()
    a.check_weights(lse, w[0, :, :T])
    # what the rows give adds up to one for each query
    assert np.allclose(w[0, :, :T].sum(1), rows * H // KV, rtol=1e-3)
    before = p.rng.random((1, KV, T)).astype(np.float32)
    got = p.weights(q, lse, [rows], [T], T, previous=before, decay=0.75, window=window, sinks=sinks)
    a.check_weights(lse, got[0], before[0], 0.75)
    both = dev(before)  # in place
    ca, keep = p.call(q, [rows], [T], window=window, sinks=sinks)
    dl = dev(lse)
    synchronize()
    p.pool.weights(0, lse=ptr(dl), scores=ptr(both), ld=T, previous=ptr(both), decay=0.75, **ca)
    assert np.array_equal(both.get(), got)
    # with decay 0 what was there is not read
    got = p.weights(q, lse, [rows], [T], T, previous=np.full((1, KV, T), np.nan, np.float32), decay=0.0, window=window, sinks=sinks)
    assert np.array_equal(got, w[:, :, :T])


@pytest.mark.parametrize("hd", [64, 128])
def test_weights_of_a_ragged_batch_and_trees(hip, hd):
    lens, counts = [0, 700, 33, 64, 5, 2000, 31], [0, 3, 0, 64, 5, 1, 2]
    p = Pool(hip, 13, 8, 2, hd, lens, page=64)
    p.fill(lens)
    q = p.rows(sum(counts), 8)
    bits = np.zeros((sum(counts), 64), bool)
    for at, n in ((0, 3), (3, 64), (67, 5), (72, 1), (73, 2)):
        bits[at:at + n, :n] = np.tril(p.rng.random((n, n)) < 0.6) | np.eye(n, dtype=bool)
    mask = np.ascontiguousarray(np.concatenate([_kv8.words(bits[i:i + 1, :].repeat(64, 0))[:1] for i in range(len(bits))]))
    for m in (None, mask):
        for ld in (2000, 600):
            _, lse = p.attend(q, counts, lens, mask=m)
            w = p.weights(q, lse, counts, lens, ld, mask=m)
            at = 0
            for s, n in enumerate(counts):
                end = min(lens[s], ld)
                if n:
                    seen = _kv8.visible(n, lens[s], None if m is None else bits[at:at + n, :n])
                    a = _kv8.Attention(q[at:at + n], p.held[s][0][:end], p.held[s][1][:end], seen[:, :end], hd ** -0.5)
                    a.check_weights(lse[at:at + n], w[s, :, :end])
                assert (w[s, :, end if n else 0:] == 3.0).all()
                at += n


def test_weights_past_max_len(hip):
    p = Pool(hip, 14, 4, 2, 64, [900], page=64)
    p.fill([900])
    q = p.rows(2, 4)
    _, lse = p.attend(q, [2], [900])
    assert np.array_equal(p.weights(q, lse, [2], [900], 900), p.weights(q, lse, [2], [900], 900, max_len=1))


# ---- eviction --------------------------------------------------------------------
def scores_of(rng, shape, kind):
    x = np.exp(rng.standard_normal(shape) * 2).astype(np.float32)
    if kind == "ties":
        x = np.floor(x).astype(np.float32)  # many equal ones, most of them 0
    elif kind == "all equal":
        x[:] = 0.25
    elif kind == "odd":
        x[rng.random(shape) < 0.2] = np.nan
        x[rng.random(shape) < 0.1] = -np.inf
        x[rng.random(shape) < 0.1] = np.inf
        x[rng.random(shape) < 0.2] *= -1
        x[rng.random(shape) < 0.1] = -0.0
        x[rng.random(shape) < 0.1] = 0.0
        x[rng.random(shape) < 0.05] = 1e-42
    return x


def run_evict(p, lens, x, budget, sinks, recent, in_place, scores_out="own", ws_fill=255):
    S, KV, ld = x.shape
    ds, dl = dev(x), dev(np.asarray(lens, np.int32))
    kept, new_len = full((S, KV, budget), 99, np.int32), full((S,), 99, np.int32)
    out = {"own": full((S, KV, budget + 3), 4.0), "same": ds, "none": None}[scores_out]
    out_ld = {"own": budget + 3, "same": ld, "none": 0}[scores_out]
    table = None
    if not in_place:
        n = max(1, -(-budget // p.page))
        ids = [p.free.pop() for _ in range(S * n)]
        table = dev(np.array(ids, np.int32).reshape(S, n))
    need = p.pool.evict_workspace(S, budget) if in_place else 0
    ws = full((max(need, 16),), ws_fill, np.uint8)
    synchronize()
    p.pool.evict(0, ptr(dl), ptr(p.dtable), *p.table.shape, scores=ptr(ds), scores_ld=ld, budget=budget, kept=ptr(kept),
                 new_len=ptr(new_len), sinks=sinks, recent=recent, scores_out=ptr(out), scores_out_ld=out_ld, new_table=ptr(table),
                 new_table_ld=table.shape[1] if table else 0, ws=ptr(ws) if need else 0, ws_bytes=need)
    return kept.get(), new_len.get(), None if out is None else out.get(), table


def check_evict(p, lens, x, budget, sinks, recent, got):
    kept, new_len, out, table = got
    S, KV, _ = x.shape
    assert new_len.tolist() == [min(n, budget) for n in lens]
    for s, T in enumerate(lens):
        n = min(T, budget)
        new = [np.zeros((n, KV, p.hd)) for _ in range(2)]
        for h in range(KV):
            want = _kv8.evict(x[s, h], T, budget, sinks, recent)
            assert np.array_equal(kept[s, h, :n], want), (s, h)
            assert (kept[s, h, n:] == -1).all()
            if out is not None:
                assert np.array_equal(out[s, h, :n], x[s, h, want], equal_nan=True)
            for i in range(2):
                new[i][:, h] = p.held[s][i][want, h]
        if T > budget:
            p.held[s] = [_kv8.append(np.zeros((0, KV, p.hd)), 0, a) for a in new]
    p.check_held(table=table)


@pytest.mark.parametrize("hd,KV", [(128, 2), (64, 3)])
@pytest.mark.parametrize("kind", ["plain", "ties", "all equal", "odd"])
@pytest.mark.parametrize("budget,sinks,recent", [(100, 4, 20), (33, 0, 0), (64, 32, 32), (1, 0, 1), (500, 0, 499)])
@pytest.mark.parametrize("in_place", [True, False])
def test_evict(hip, hd, KV, kind, budget, sinks, recent, in_place):
    lens = [700, budget, budget + 1, 5, 0, 1500, 129]
    p = Pool(hip, hd + budget, 2 * KV, KV, hd, [max(n, 1) for n in lens], page=32, spare=7 * 16 + 4)

    def edit(k, v):
        k[10, 0, 3], v[sum(lens[:5]) + 60, 0, 2] = np.nan, np.inf  # NaN rows move as such
        v[20:40] *= np.float16(1e-3)
    p.fill(lens, edit)
    x = scores_of(p.rng, (len(lens), KV, 1600), kind)
    got = run_evict(p, lens, x, budget, sinks, recent, in_place, "own" if in_place else "none")
    if in_place:
        for s, n in enumerate(lens):
            assert (got[2][s, :, min(n, budget):] == 4.0).all()
    check_evict(p, lens, x, budget, sinks, recent, got)


@pytest.mark.parametrize("T,budget", [(40000, 3001), (66000, 17), (20000, 19999)])
@pytest.mark.parametrize("kind", ["plain", "ties", "all equal"])
def test_evict_of_long_sequences(hip, T, budget, kind):
    p = Pool(hip, T, 1, 1, 64, [T], page=256, spare=100)
    n = T // 2
    k, v = p.rows(T, 1), p.rows(T, 1)
    pos = np.arange(T) % MAX_POS
    p.append([n], [n], k[:n], v[:n], pos=pos[:n])
    p.append([T - n], [T], k[n:], v[n:], pos=pos[n:])
    x = scores_of(p.rng, (1, 1, T), kind)
    check_evict(p, [T], x, budget, 4, 10, run_evict(p, [T], x, budget, 4, 10, True, "same"))


def test_evict_of_nothing_and_to_nothing(hip):
    p = Pool(hip, 15, 2, 1, 64, [100], page=32, spare=8)
    p.fill([100])
    x = scores_of(p.rng, (1, 1, 100), "plain")
    # a score row shorter than the sequence: what lies past it does not exist
    got = run_evict(p, [100], x[:, :, :50].copy(), 40, 1, 1, False)
    p.held[0] = [a[:50] for a in p.held[0]]
    check_evict(p, [50], x[:, :, :50], 40, 1, 1, got)
    kept, new_len, out, _ = run_evict(p, [100], x, 0, 0, 0, True, "none")
    assert new_len[0] == 0


def test_evict_with_absent_pages(hip):
    """Positions of absent pages stand for zeros; what goes to an absent page is dropped."""
    p = Pool(hip, 16, 2, 1, 64, [192], page=64, spare=8)
    p.fill([192])
    p.table[0, 1] = -1
    p.dtable = dev(p.table)
    x = np.zeros((1, 1, 192), np.float32)
    x[0, 0, 60:130] = 1.0
    kept, new_len, _, table = run_evict(p, [192], x, 70, 0, 0, False)
    assert kept[0, 0].tolist() == list(range(60, 130)) and new_len[0] == 70
    new = [a[60:130].copy() for a in p.held[0]]
    for a in new:
        a[4:68] = 0
    got = p.read([0] * 70, range(70), table=table)
    for g, a in zip(got, new):
        assert np.array_equal(g.astype(np.float64), _kv8.append(np.zeros((0, 1, 64)), 0, a))
    t = table.get()
    before = p.read([0] * 64, range(64), table=dev(t[:, :1].copy()))
    t[0, 1] = p.n_pages
    p.free += [0]
    dl, ds, kd, nl = dev(np.array([192], np.int32)), dev(x), zeros((1, 1, 70), np.int32), zeros((1,), np.int32)
    nt = dev(t)
    synchronize()
    p.pool.evict(0, ptr(dl), ptr(p.dtable), *p.table.shape, scores=ptr(ds), scores_ld=192, budget=70, kept=ptr(kd), new_len=ptr(nl),
                 new_table=ptr(nt), new_table_ld=2)
    synchronize()
    after = p.read([0] * 64, range(64), table=nt)
    assert np.array_equal(before[0], after[0]) and np.array_equal(before[1], after[1])


# ---- together --------------------------------------------------------------------
@pytest.mark.parametrize("hd,KV,H", [(128, 2, 8), (64, 4, 4)])
def test_decoding_under_a_budget(hip, hd, KV, H):
    """A prompt is scored and cut down, then rows come, are attended to, scored, and now and then evicted by the scores."""
    budget, sinks, recent, ld = 96, 4, 16, 200
    prompt = [150, 60]
    p = Pool(hip, 91, H, KV, hd, [ld, ld], page=32)
    p.fill(prompt)
    lens, true_len, ld_scores = list(prompt), list(prompt), ld
    q = p.rows(sum(prompt), H)
    out, lse = p.attend(q, prompt, lens)
    sums = p.weights(q, lse, prompt, lens, ld_scores, out=zeros((2, KV, ld)))
    for step in range(8):
        got = run_evict(p, lens, sums, budget, sinks, recent, True, "same")
        check_evict(p, lens, sums, budget, sinks, recent, got)
        lens, sums = got[1].tolist(), got[2]
        counts = [1 + step % 3, 20 if step == 4 else 1]
        n = sum(counts)
        k, v, qr = p.rows(n, KV), p.rows(n, KV), p.rows(n, H)
        pos = np.concatenate([np.arange(a, a + c) for a, c in zip(true_len, counts)])  # rotation goes on where it was
        lens, true_len = ([a + c for a, c in zip(x, counts)] for x in (lens, true_len))
        turned = p.append(counts, lens, k, v, pos=pos, q=qr)
        p.check_held()
        out, lse = p.attend(turned, counts, lens)
        for s in range(2):
            sums[s, :, lens[s] - counts[s]:lens[s]] = 0
        new = p.weights(turned, lse, counts, lens, ld_scores, previous=sums, out=dev(sums))
        at = 0
        for s, c in enumerate(counts):
            a = _kv8.Attention(turned[at:at + c], *p.held[s], _kv8.visible(c, lens[s]), hd ** -0.5)
            a.check(out[at:at + c], lse[at:at + c])
            a.check_weights(lse[at:at + c], new[s, :, :lens[s]], sums[s, :, :lens[s]])
            at += c
        sums = new


@pytest.mark.parametrize("rows", [1, 40])
def test_captured_and_replayed(hip, rows):
    """append, attend, weights and an eviction into other pages recorded into a graph, replayed on new inputs with eager
    calls between."""
    T, budget = 500, 128
    p = Pool(hip, 41, 8, 2, 128, [T], page=64, spare=8)
    p.fill([T])
    start, lens = dev(np.array([0, rows], np.int32)), dev(np.array([T], np.int32))
    q, k, v = (zeros((rows, h, 128), np.float16) for h in (8, 2, 2))
    qo, out, lse = zeros((rows, 8, 128), np.float16), zeros((rows, 8, 128), np.float16), zeros((rows, 8))
    sums, kept, new_len = zeros((1, 2, T)), zeros((1, 2, budget), np.int32), zeros((1,), np.int32)
    table = dev(np.array([[p.free.pop(), p.free.pop()]], np.int32))
    ws = zeros(max(16, p.pool.attend_workspace(rows, 1, rows, T, 100, 4)), np.uint8)

    def step(st):
        p.pool.append(0, rows, ptr(start), ptr(lens), ptr(p.dtable), *p.table.shape, max_rows=rows, k=ptr(k), v=ptr(v), q=ptr(q),
                      q_out=ptr(qo), stream=st)
        a = dict(row_start=ptr(start), kv_len=ptr(lens), table=ptr(p.dtable), n_seqs=1, table_ld=p.table.shape[1], rows=rows,
                 max_rows=rows, max_len=T, window=100, sinks=4, stream=st)
        p.pool.attend(0, ptr(qo), ptr(out), ws=ptr(ws), ws_bytes=ws.nbytes, lse=ptr(lse), **a)
        p.pool.weights(0, ptr(qo), ptr(lse), ptr(sums), T, **a)
        p.pool.evict(0, ptr(lens), ptr(p.dtable), *p.table.shape, scores=ptr(sums), scores_ld=T, budget=budget, sinks=4, recent=30,
                     kept=ptr(kept), new_len=ptr(new_len), new_table=ptr(table), new_table_ld=2, stream=st)
    graph, side = Graph(step), Stream()
    pos = np.arange(T - rows, T)
    for i in range(4):
        nq, nk, nv = p.rows(rows, 8), p.rows(rows, 2), p.rows(rows, 2)
        for t, a in ((q, nq), (k, nk), (v, nv)):
            t.put(a)
        out.put(np.zeros(out.shape))
        graph.launch()
        p.held[0] = [_kv8.append(x, T - rows, y) for x, y in zip(p.held[0], (p.turned(nk, pos), nv))]
        p.check_held()
        got = [t.get() for t in (out, lse, sums, kept)]
        a = _kv8.Attention(qo.get(), *p.held[0], _kv8.visible(rows, T, window=100, sinks=4), 128 ** -0.5)
        a.check(got[0], got[1])
        a.check_weights(got[1], got[2][0])
        for h in range(2):
            assert np.array_equal(got[3][0, h], _kv8.evict(got[2][0, h], T, budget, 4, 30))
        out.put(np.zeros(out.shape))
        sums.put(np.zeros(sums.shape))
        step(side.handle)
        side.wait()
        for x, y in zip(got, (out, lse, sums, kept)):
            assert np.array_equal(x, y.get()), i


def test_two_streams_and_pools(hip):
    """Two pools at once on two streams, each call with its own workspace."""
    a, b = (Pool(hip, 60 + i, 8, 2, 128, [3000], page=64) for i in range(2))
    a.fill([3000])
    b.fill([3000])
    runs = []
    for p in (a, b):
        q = p.rows(5, 8)
        args, keep = p.call(q, [5], [3000])
        out, lse = full((5, 8, 128), 9.0, np.float16), full((5, 8), 9.0)
        ws = zeros(max(16, p.pool.attend_workspace(5, 1, 5, 3000)), np.uint8)
        runs.append((p, q, args, keep, out, lse, ws, Stream()))
    synchronize()
    for _ in range(10):
        for p, q, args, keep, out, lse, ws, st in runs:
            p.pool.attend(0, out=ptr(out), lse=ptr(lse), ws=ptr(ws), ws_bytes=ws.nbytes, stream=st.handle, **args)
    for p, q, args, keep, out, lse, ws, st in runs:
        st.wait()
        _kv8.Attention(q, *p.held[0], _kv8.visible(5, 3000), 128 ** -0.5).check(out.get(), lse.get())


# ---- refusals --------------------------------------------------------------------
def test_refusals(hip):
    p = Pool(hip, 71, 4, 2, 64, [100], page=32, spare=8)
    p.fill([100])
    buf, ints = zeros((1 << 16,)), zeros((64,), np.int32)
    f, i, t = ptr(buf), ptr(ints), ptr(p.dtable)
    row = 2 * 64 * 2  # bytes of a row of k or v
    A = dict(layer=0, rows=4, row_start=i, kv_len=i, table=t, n_seqs=1, table_ld=4, max_rows=4, k=f, v=f + 4 * row)
    q = dict(A, q=f + 16 * row, q_out=f + 64 * row)
    bad = hip.ArgError
    for change, err in ((dict(layer=1), bad), (dict(layer=-1), bad), (dict(row_start=0), bad), (dict(kv_len=0), bad), (dict(table=0), bad),
                        (dict(k=0), bad), (dict(v=0), bad), (dict(max_rows=0), bad), (dict(max_rows=5), bad), (dict(n_seqs=0), bad),
                        (dict(n_seqs=65536), bad), (dict(table_ld=0), bad), (dict(rows=1 << 25, max_rows=1), bad), (dict(k_ld=64), bad),
                        (dict(k=f + 8), bad), (dict(v_ld=130), bad), (dict(dtype=hip.F16 + 7), hip.UnsupportedMethod),
                        (dict(q_out=0), bad), (dict(q_out=f), bad), (dict(q_out=f + 4 * row), bad), (dict(q_out=f + 17 * row), bad),
                        (dict(q=f + 16 * row + 4), bad), (dict(q_out=f + 64 * row + 8), bad)):
        with pytest.raises(err):
            p.pool.append(**dict(q, **change))
    p.pool.append(**dict(A, rows=0))
    for change in (dict(slots=0), dict(table=0), dict(n_seqs=0), dict(table_ld=0), dict(k_out=f + 2), dict(v_out=f + row), dict(layer=3)):
        with pytest.raises(bad):
            p.pool.read(**dict(dict(layer=0, n=4, slots=i, table=t, n_seqs=1, table_ld=4, k_out=f, v_out=f + 4 * row), **change))
    B = dict(layer=0, q=f, row_start=i, kv_len=i, table=t, n_seqs=1, table_ld=4, rows=4, max_rows=4, max_len=100)
    qrow = 4 * 64 * 2
    need = p.pool.attend_workspace(4, 1, 4, 5000)
    assert need > 0 and p.pool.attend_workspace(0, 1, 1, 1) == 0 and p.pool.attend_workspace(4, 1, 5, 1) == 0
    common = ((dict(layer=1), bad), (dict(q=0), bad), (dict(row_start=0), bad), (dict(kv_len=0), bad), (dict(table=0), bad),
              (dict(n_seqs=0), bad), (dict(table_ld=0), bad), (dict(mask=f), bad), (dict(scale=float("nan")), bad), (dict(scale=float("inf")), bad),
              (dict(max_rows=0), bad), (dict(max_rows=5), bad), (dict(max_len=1 << 31), bad), (dict(q=f + 2), bad), (dict(q_ld=200), bad),
              (dict(q_ld=257), bad), (dict(n_seqs=65536), bad), (dict(rows=1 << 25), bad))
    att = dict(B, out=f + 8 * qrow, lse=f + 16 * qrow, ws=f + 32 * qrow, ws_bytes=1 << 20)
    for change, err in common + ((dict(out=0), bad), (dict(out=f), bad), (dict(out=f + 2 * qrow), bad), (dict(lse=f), bad), (dict(lse=f + 8 * qrow + 4), bad),
                                 (dict(lse=f + 16 * qrow + 2), bad), (dict(out_ld=100), bad), (dict(out=f + 8 * qrow + 4), bad),
                                 (dict(max_len=5000, ws_bytes=need - 1), bad), (dict(max_len=5000, ws=0), bad),
                                 (dict(max_len=5000, ws=f + 32 * qrow + 8), bad), (dict(max_len=5000, ws=f), bad),
                                 (dict(max_len=5000, ws=f + 8 * qrow), bad), (dict(max_len=5000, ws=f + 16 * qrow), bad)):
        with pytest.raises(err):
            p.pool.attend(**dict(att, **change))
    p.pool.attend(**dict(att, rows=0, max_rows=0))
    w = dict(B, lse=f + 8 * qrow, scores=f + 16 * qrow, ld=100, previous=f + 32 * qrow)
    for change, err in common + ((dict(lse=0), bad), (dict(scores=0), bad), (dict(ld=0), bad), (dict(ld=1 << 31), bad), (dict(decay=float("nan")), bad),
                                 (dict(scores=f + 2 * qrow), bad), (dict(scores=f + 8 * qrow), bad), (dict(previous=f + 16 * qrow + 4), bad),
                                 (dict(scores=f + 16 * qrow + 2), bad), (dict(lse=f + 8 * qrow + 1), bad)):
        with pytest.raises(err):
            p.pool.weights(**dict(w, **change))
    need = p.pool.evict_workspace(1, 40)
    assert need == 2 * 2 * (64 * 64 + 16) and p.pool.evict_workspace(0, 40) == 0 and p.pool.evict_workspace(1, 1 << 31) == 0
    e = dict(layer=0, kv_len=i, table=t, n_seqs=1, table_ld=4, scores=f, scores_ld=100, budget=40, kept=f + 4096, new_len=f + 8192, sinks=4,
             recent=4, scores_out=f + 12288, ws=f + 16384, ws_bytes=1 << 17)
    for change, err in ((dict(layer=1), bad), (dict(kv_len=0), bad), (dict(table=0), bad), (dict(scores=0), bad), (dict(kept=0), bad), (dict(new_len=0), bad),
                        (dict(n_seqs=0), bad), (dict(n_seqs=65536), bad), (dict(table_ld=0), bad), (dict(new_table=t), bad), (dict(sinks=41), bad),
                        (dict(sinks=20, recent=21), bad), (dict(recent=1 << 40), bad), (dict(scores_ld=0), bad), (dict(scores_ld=1 << 31), bad),
                        (dict(scores_out_ld=39), bad), (dict(ws=0), bad), (dict(ws_bytes=need - 1), bad), (dict(ws=f + 16384 + 8), bad),
                        (dict(kept=f), bad), (dict(kept=f + 4098), bad), (dict(new_len=i), bad), (dict(new_len=f + 4096), bad), (dict(ws=f), bad),
                        (dict(scores_out=f), bad), (dict(scores_out=f + 4), bad), (dict(scores_out=f + 4096), bad), (dict(kept=t), bad),
                        (dict(budget=1 << 31), bad), (dict(budget=1 << 30, sinks=0, recent=0), hip.UnsupportedMethod)):
        with pytest.raises(err):
            p.pool.evict(**dict(e, **change))
    p.check_held()


def test_refused_calls_leave_no_error_behind(hip):
    p = Pool(hip, 72, 4, 2, 64, [40], page=32)
    with pytest.raises(hip.ArgError):
        p.pool.append(0, 1, 0, 0, 0, 1, 1, max_rows=1, k=0, v=0)
    p.fill([40])
    p.check_held()


# ---- sizes that take other paths ---------------------------------------------------
@pytest.mark.parametrize("inter", [True, False])
@pytest.mark.parametrize("hd,dt", [(128, np.float16), (64, np.float32)])
def test_append_of_many_queries(hip, hd, dt, inter):
    """Above 65536 pairs of rows and query heads these have a launch of their own."""
    counts = [2500, 3, 700]
    p = Pool(hip, hd, 32, 2, hd, [c + 45 for c in counts], page=64, interleaved=inter)
    p.append([45] * 3, [45] * 3, p.rows(135, 2), p.rows(135, 2))
    n = sum(counts)
    k, v, q = p.rows(n, 2, dt), p.rows(n, 2, dt), p.rows(n, 32, dt)
    pos = p.rng.integers(0, MAX_POS, n)
    qo = p.append(counts, [c + 45 for c in counts], k, v, pos=pos, q=q)
    p.check_held()
    want = p.turned(q, pos)
    assert np.all(np.abs(qo.astype(np.float64) - want) <= 2.0 ** -11 * np.abs(want) + 2.0 ** -22 * np.abs(q).max() + 2.0 ** -25)


@pytest.mark.parametrize("hd,window", [(128, 0), (64, 0), (128, 4800)])
def test_attention_of_many_steps_a_wave(hip, hd, window):
    """Enough rows that a key range is the whole sequence: a wave's pages and headers are asked for more than once; one page in
    between is absent."""
    T, rows = 6000, 620
    p = Pool(hip, 61, 32, 8, hd, [T], page=64)
    p.fill([T])
    q = p.rows(rows, 32)
    t = p.table.copy()
    t[0, 70] = -1
    out, lse = p.attend(q, [rows], [T], table=dev(t), window=window, sinks=3 if window else 0)
    seen = _kv8.visible(rows, T, window=window, sinks=3 if window else 0)
    seen[:, 70 * 64:71 * 64] = False
    pick = p.rng.permutation(rows)[:60]  # (the oracle takes its time)
    _kv8.Attention(q[pick], *p.held[0], seen[pick], hd ** -0.5).check(out[pick], lse[pick])


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("window,sinks,tree", [(0, 0, False), (300, 70, False), (0, 0, True), (100, 5, True)])
def test_weights_of_many_positions(hip, hd, window, sinks, tree):
    """Enough positions for 64 of them a wave, ends inside both of its blocks, NaN rows and an absent page."""
    lens = [2100, 2047, 33, 2100, 1999, 2080, 2100, 1900]
    counts = [70, 1, 33, 40, 5, 64, 3, 90]
    p = Pool(hip, hd + window, 8, 4, hd, lens, page=64)

    def edit(k, v):
        k[5, 0, 1] = np.nan  # of sequence 0
        k[sum(lens) - 10, 2, 3] = np.inf  # and of the last's own rows
    p.fill(lens, edit)
    q = p.rows(sum(counts), 8)
    bits = [np.tril(p.rng.random((n, n)) < 0.5) | np.eye(n, dtype=bool) for n in counts] if tree else [None] * len(counts)
    mask = None
    if tree:
        mask = np.zeros((sum(counts), 2), np.uint64)
        at = 0
        for n, b in zip(counts, bits):
            w = _kv8.words(b)
            mask[at:at + n, :w.shape[1]] = w
            at += n
    t = p.table.copy()
    t[3, 20] = p.n_pages + 1
    dt = dev(t)
    more = dict(table=dt, window=window, sinks=sinks)
    _, lse = p.attend(q, counts, lens, mask=mask, **more)
    before = p.rng.random((len(lens), 4, 2100)).astype(np.float32)
    w = p.weights(q, lse, counts, lens, 2100, previous=before, mask=mask, **more)
    at = 0
    for s, n in enumerate(counts):
        seen = _kv8.visible(n, lens[s], bits[s], window, sinks)
        if s == 3:
            seen[:, 20 * 64:21 * 64] = False
        a = _kv8.Attention(q[at:at + n], *p.held[s], seen, hd ** -0.5)
        a.check_weights(lse[at:at + n], w[s, :, :lens[s]], before[s, :, :lens[s]])
        assert (w[s, :, lens[s]:] == 3.0).all()
        at += n


def test_pages_past_32_bits(hip):
    """Page ids whose bytes lie past 2^33 in the pool, for every call."""
    p = Pool(hip, 81, 8, 8, 128, [600, 64], page=256, spare=17000)
    assert p.pool.page_bytes() * p.n_pages > 2 ** 33
    p.table[0, :3] = [p.n_pages - 1, 5, p.n_pages - 3]
    p.table[1, 0] = 8200  # around 2^32 bytes
    p.dtable = dev(p.table)
    p.fill([600, 64])
    p.check_held()
    q = p.rows(3, 8)
    out, lse = p.attend(q, [2, 1], [600, 64])
    w = p.weights(q, lse, [2, 1], [600, 64], 600)
    for s, (r, T) in enumerate(((slice(0, 2), 600), (slice(2, 3), 64))):
        a = _kv8.Attention(q[r], *p.held[s], _kv8.visible(r.stop - r.start, T), 128 ** -0.5)
        a.check(out[r], lse[r])
        a.check_weights(lse[r], w[s, :, :T])
    check_evict(p, [600, 64], w, 300, 4, 100, run_evict(p, [600, 64], w, 300, 4, 100, True, "same"))


def test_eviction_in_place_captured_and_replayed(hip):
    """A long sequence (its ranks need more LDS than a kernel has by default) cut down in a graph, filled again in between."""
    T, budget = 20000, 700
    p = Pool(hip, 82, 2, 2, 64, [T], page=64)
    x = scores_of(p.rng, (1, 2, T), "plain")
    ds, dl, kept, new_len = dev(x), dev(np.array([T], np.int32)), zeros((1, 2, budget), np.int32), zeros((1,), np.int32)
    ws = zeros(p.pool.evict_workspace(1, budget), np.uint8)

    def step(st):
        p.pool.evict(0, ptr(dl), ptr(p.dtable), *p.table.shape, scores=ptr(ds), scores_ld=T, budget=budget, sinks=4, recent=100,
                     kept=ptr(kept), new_len=ptr(new_len), scores_out=ptr(ds), scores_out_ld=T, ws=ptr(ws), ws_bytes=ws.nbytes, stream=st)
    graph = Graph(step)
    for i in range(3):
        p.held[0] = [np.zeros((0, 2, 64))] * 2
        for a in range(0, T, 5000):
            p.append([5000], [a + 5000], p.rows(5000, 2), p.rows(5000, 2), pos=np.arange(a, a + 5000) % MAX_POS)
        x = scores_of(p.rng, (1, 2, T), ("plain", "ties", "all equal")[i])
        ds.put(x)
        synchronize()
        graph.launch()
        check_evict(p, [T], x, budget, 4, 100, (kept.get(), new_len.get(), ds.get(), None))


def test_windows_that_no_sequence_fills(hip):
    # from 2^31 - 64 on a window is none, whatever `sinks` is; between that and 2^30 it is refused
    p = Pool(hip, 90, 4, 2, 64, [300], page=32)
    p.fill([300])
    q = p.rows(3, 4)
    want, lse = p.attend(q, [3], [300])
    for window in (1 << 30, 2 ** 31 - 64, 2 ** 31, 2 ** 63):
        for sinks in (0, 5, 2 ** 63):
            out, stat = p.attend(q, [3], [300], window=window, sinks=sinks)
            assert np.array_equal(out, want) and np.array_equal(stat, lse)
            got = p.weights(q, lse, [3], [300], 300, window=window, sinks=sinks)
            assert np.array_equal(got, p.weights(q, lse, [3], [300], 300))
    for window in (2 ** 30 + 1, 2 ** 31 - 65):
        assert p.pool.attend_workspace(3, 1, 3, 300, window) == 0
        with pytest.raises(hip.ArgError):
            p.attend(q, [3], [300], window=window)
        with pytest.raises(hip.ArgError):
            p.weights(q, lse, [3], [300], 300, window=window)


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("rows", [1, 5, 70])
def test_the_longest_sequence_through_a_window(hip, rows, tree):
    # 2^31 - 64 positions of which the first and the last page exist: what a window sees is what it sees of two pages
    page, T, short = 2048, 2 ** 31 - 64, 2 * 2048 - 64
    p = Pool(hip, 91 + rows, 8, 2, 128, [short], page=page)
    p.fill([short])
    table = np.full((1, (T - 1) // page + 1), -1, np.int32)
    table[0, 0], table[0, -1] = p.table[0, :2]
    big = dev(table)
    q, k, v = p.rows(rows, 8), p.rows(rows, 2), p.rows(rows, 2)
    pos = dev((short - rows + np.arange(rows)).astype(np.int32))
    start, lens, dk, dv = dev(np.array([0, rows], np.int32)), dev(np.array([T], np.int32)), dev(k), dev(v)
    p.pool.append(0, rows, ptr(start), ptr(lens), ptr(big), 1, table.shape[1], rows, ptr(dk), ptr(dv), pos=ptr(pos))
    for i, x in enumerate((p.turned(k, short - rows + np.arange(rows)), v.astype(np.float64))):
        p.held[0][i] = _kv8.append(p.held[0][i], short - rows, x)
    p.check_held()
    rng = np.random.default_rng(rows)
    bits = np.tril(rng.random((rows, rows)) < 0.5) | np.eye(rows, dtype=bool)
    mask = _kv8.words(bits) if tree else None
    for window, sinks in ((100, 5), (1500, 0), (1900, 40)):
        see = _kv8.visible(rows, short, bits if tree else None, window, sinks)
        out, lse = p.attend(q, [rows], [T], mask=mask, table=big, window=window, sinks=sinks)
        _kv8.Attention(q, *p.held[0], see, 128 ** -0.5).check(out, lse)
        shared = dict(mask=mask, window=window, sinks=sinks)
        assert np.array_equal(p.weights(q, lse, [rows], [T], page, table=big, **shared), p.weights(q, lse, [rows], [short], page, **shared))


def test_scales_that_base_2_cannot_hold(hip):
    p = Pool(hip, 95, 4, 2, 64, [40], page=32)
    p.fill([40])
    q = p.rows(1, 4)
    for scale in (3e38, -3e38, float("inf"), float("nan")):
        with pytest.raises(hip.ArgError):
            p.attend(q, [1], [40], scale=scale)
        with pytest.raises(hip.ArgError):
            p.weights(q, np.zeros((1, 4), np.float32), [1], [40], 40, scale=scale)


@pytest.mark.parametrize("hd,KV,page", [(128, 2, 32), (64, 3, 128)])
def test_reading_any_positions_in_any_order(hip, hd, KV, page):
    # runs that start inside a group of 8, go backwards, change their sequence or pass a page's end, positions that are not there
    p = Pool(hip, 96, KV, KV, hd, [300, 77], page=page)
    p.fill([300, 77], edit=lambda k, v: (k.__setitem__((50, 1, 3), np.nan), v.__setitem__((305, 0, 7), np.inf)))
    rng = np.random.default_rng(5)
    cases = [([0] * 300, range(300)), ([0] * 64, range(3, 67)), ([0] * 40, range(40, 80)), ([1] * 77, range(76, -1, -1)),
             ([0] * 8 + [1] * 8, [*range(8, 16)] * 2), ([0] * 12 + [1] * 12, [*range(16, 28)] * 2), ([0], [5]), ([0] * 16, [9] * 16),
             ([0, 1] * 30, rng.integers(0, 77, 60)), ([0] * 8 + [5] + [0] * 7 + [-1] * 8, [*range(24, 32), 0, *range(33, 40), *range(8)]),
             ([0] * 10 + [1] * 6, [*range(8), -1, 1 << 20, *range(8, 14)]), (rng.integers(0, 2, 3000), rng.integers(0, 77, 3000))]
    for seq, slot in cases:
        k, v = p.read(seq, slot)
        for i, (s, at) in enumerate(zip(seq, slot)):
            there = 0 <= s < 2 and 0 <= at < p.table.shape[1] * page and p.table[s, at // page] >= 0
            for got, held in ((k[i], p.held[s][0]), (v[i], p.held[s][1])) if there else ():
                assert np.array_equal(got.astype(np.float64), held[at], equal_nan=True), (s, at)
            assert there or ((k[i] == 5).all() and (v[i] == 5).all())


@pytest.mark.parametrize("hd,KV", [(128, 2), (64, 3)])
@pytest.mark.parametrize("budget,sinks,recent", [(100, 4, 20), (1, 0, 1), (1500, 3, 200)])
@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("scores_out", ["own", "same", "none"])
def test_scores_move_with_their_positions(hip, hd, KV, budget, sinks, recent, in_place, scores_out):
    """In place and into new pages, into the scores themselves and elsewhere: of sequences above and under the budget, and no
    entry past the new length is written."""
    lens = [1700, budget, budget + 1, 5, 0, 3100]
    p = Pool(hip, 3 * hd + budget, 2 * KV, KV, hd, [max(n, 1) for n in lens], page=64, spare=len(lens) * 25)
    p.fill(lens)
    x = scores_of(p.rng, (len(lens), KV, 3200), "plain")
    got = run_evict(p, lens, x, budget, sinks, recent, in_place, scores_out)
    check_evict(p, lens, x, budget, sinks, recent, got)
    if scores_out != "none":
        for s, n in enumerate(min(n, budget) for n in lens):
            past = got[2][s, :, n:]
            assert np.array_equal(past, np.full_like(past, 4.0) if scores_out == "own" else x[s, :, n:])


@pytest.mark.parametrize("hd,KV,H", [(128, 2, 8), (64, 4, 4), (128, 1, 7)])
def test_own_rows_start_anew(hip, hd, KV, H):
    """What is summed over steps of a batch, none of it cleared by hand: rows come, are scored, some of them are rolled back and
    others come in their places, sequences are cut down.  The array starts as NaN: nothing is read that no call has written."""
    budget, sinks, recent, ld, decay = 96, 4, 16, 200, 0.75
    counts, lens, true_len = [150, 60, 1], [150, 60, 1], [150, 60, 1]
    p = Pool(hip, 101 + hd, H, KV, hd, [ld] * 3, page=32)
    scores = full((3, KV, ld), np.nan)
    want = np.full((3, KV, ld), np.nan)  # what the array held before the call, with zeros where rows are new
    for step in range(10):
        n = sum(counts)
        pos = np.concatenate([np.arange(t - c, t) for t, c in zip(true_len, counts)])
        turned = p.append(counts, lens, p.rows(n, KV), p.rows(n, KV), pos=pos, q=p.rows(n, H))
        window = dict(window=50, sinks=3) if step % 3 == 2 else {}
        mask = None
        if step % 4 == 3:
            mask = np.ascontiguousarray(np.concatenate([_kv8.words(np.tril(np.ones((c, c), bool)))[:, :1] for c in counts if c]))
        _, lse = p.attend(turned, counts, lens, mask=mask, **window)
        call, keep = p.call(turned, counts, lens, mask=mask, **window)
        dl = dev(lse)
        synchronize()
        p.pool.weights(0, lse=ptr(dl), scores=ptr(scores), ld=ld, previous=ptr(scores), decay=decay, own_rows_anew=True, **call)
        new, at = scores.get(), 0
        for s, c in enumerate(counts):
            T = lens[s]
            if c:
                want[s, :, T - c:T] = 0
                a = _kv8.Attention(turned[at:at + c], *p.held[s], _kv8.visible(c, T, **window), hd ** -0.5)
                a.check_weights(lse[at:at + c], new[s, :, :T], want[s, :, :T], decay)
            assert np.array_equal(new[s, :, T if c else 0:], want[s, :, T if c else 0:].astype(np.float32), equal_nan=True)
            at += c
        # some of the last rows go again
        for s in range(3):
            back = min(counts[s], step % 3)
            lens[s], true_len[s] = lens[s] - back, true_len[s] - back
            p.held[s] = [a[:lens[s]] for a in p.held[s]]
        if step % 2 == 0:
            got = run_evict(p, lens, new, budget, sinks, recent, True, "same")
            check_evict(p, lens, new, budget, sinks, recent, got)
            lens, new = got[1].tolist(), got[2]
            scores = dev(new)
        want = new.astype(np.float64)
        counts = [1 + step % 3, 20 if step == 4 else 1, 0 if step == 5 else 5]
        lens, true_len = ([a + c for a, c in zip(x, counts)] for x in (lens, true_len))


@pytest.mark.parametrize("rows,T,most", [(1, 1, 1), (3, 40, 3), (40, 30, 40), (700, 1400, 700), (40, 300, 20)])
def test_own_rows_and_no_others_start_anew(hip, rows, T, most):
    """The sums of a call with own_rows_anew are those of one whose `in` is 0 at the rows' positions, bit for bit; more rows than
    positions, and rows past max_rows, are the sequence's own as well."""
    p = Pool(hip, rows + T, 4, 2, 64, [T], page=64)
    p.fill([T])
    q = p.rows(rows, 4)
    _, lse = p.attend(q, [rows], [T], max_rows=most)
    lse[most:] = 0
    before = p.rng.random((1, 2, T + 3)).astype(np.float32)
    cleared = before.copy()
    cleared[:, :, max(T - rows, 0):] = 0
    stale = before.copy()
    stale[:, :, max(T - rows, 0):] = np.nan
    got = p.weights(q, lse, [rows], [T], T + 3, previous=stale, decay=0.75, own_rows_anew=True, max_rows=most)
    assert np.array_equal(got, p.weights(q, lse, [rows], [T], T + 3, previous=cleared, decay=0.75, max_rows=most))
    assert np.array_equal(p.weights(q, lse, [rows], [T], T + 3, own_rows_anew=True, max_rows=most),
                          p.weights(q, lse, [rows], [T], T + 3, max_rows=most))


def test_more_queries_of_a_head_than_32_bits_number(hip):
    """2^24 rows of 4096 query heads over one KV head: 2^31 tiles of 32, refused before anything is launched."""
    pools = [kind(n_layers=1, n_heads=4096, n_kv_heads=1, head_dim=64, n_pages=1, page_tokens=32, max_pos=64)
             for kind in (hip.HipKv8Pool, hip.HipKvPool)]
    buf, ints = zeros((1 << 12,)), zeros((8,), np.int32)
    a = dict(row_start=ptr(ints), kv_len=ptr(ints), table=ptr(ints), n_seqs=1, table_ld=1, rows=1 << 24, max_rows=1 << 24, max_len=32)
    far = ptr(buf) + (1 << 44)  # (never read: a result that does not meet the queries)
    for pool in pools:
        assert pool.attend_workspace(1 << 24, 1, 1 << 24, 32) == 0
        with pytest.raises(hip.UnsupportedMethod):
            pool.attend(0, q=ptr(buf), out=far, **a)
    with pytest.raises(hip.UnsupportedMethod):
        pools[0].weights(0, q=ptr(buf), lse=ptr(buf), scores=far, ld=32, **a)
    assert pools[0].attend_workspace(1 << 10, 1, 1 << 10, 32) == pools[1].attend_workspace(1 << 10, 1, 1 << 10, 32) == 0
