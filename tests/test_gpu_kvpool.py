"""The 4-bit paged KV cache and the attention over it (sd_kvpool_*) against a
64-bit restatement: stored values bit for bit, attention within the rounding of
its fp16 weights, at the lengths, masks, strides and pages where it can go wrong."""
import numpy as np
import pytest

import _kvq
from _devmem import Graph, Stream, dev, full, ptr, synchronize, zeros

pytestmark = pytest.mark.gpu

MAX_POS = 5000


class Pool:
    """A pool with the sequences' pages at random places and the oracle's copy of what they hold."""

    def __init__(self, hip, seed, H, KV, hd, lens, page=64, layers=1, interleaved=True, theta=10000.0):
        self.hip, self.H, self.KV, self.hd, self.page, self.lens = hip, H, KV, hd, page, list(lens)
        self.inter, self.rng = interleaved, np.random.default_rng(seed)
        need = [max(1, -(-n // page)) for n in lens]
        self.n_pages = sum(need) + 2
        ids = self.rng.permutation(self.n_pages).tolist()
        self.table = np.full((len(lens), max(need)), -1, np.int32)
        for s, n in enumerate(need):
            self.table[s, :n] = [ids.pop() for _ in range(n)]
        self.pool = hip.HipKvPool(n_layers=layers, n_heads=H, n_kv_heads=KV, head_dim=hd, n_pages=self.n_pages,
                                  page_tokens=page, max_pos=MAX_POS, rope_theta=theta, interleaved=interleaved)
        self.cos, self.sin = _kvq.tables(MAX_POS, hd, theta)
        self.dtable = dev(self.table)

    def rows(self, n, heads, dt=np.float16):
        return (self.rng.standard_normal((n, heads, self.hd)) * (1 + 5 * (self.rng.random((1, heads, self.hd)) > .95))).astype(dt)

    def append(self, k, v, seq, slot, layer=0, pos=None, q=None, stream=0):
        dt = self.hip.F32 if k.dtype == np.float32 else self.hip.F16
        dk, dv, ds, dl = dev(k), dev(v), dev(np.asarray(seq, np.int32)), dev(np.asarray(slot, np.int32))
        dp = None if pos is None else dev(np.asarray(pos, np.int32))
        dq = None if q is None else dev(q)
        qo = None if q is None else full((len(k), self.H, self.hd), 77.0, np.float16)
        synchronize()
        self.pool.append(layer, len(k), ptr(dk), ptr(dv), ptr(dl), ptr(self.dtable), *self.table.shape, dtype=dt,
                         seqs=ptr(ds), pos=ptr(dp), q=ptr(dq), q_out=ptr(qo), stream=stream)
        synchronize()
        return None if q is None else qo.get()

    def read(self, seq, slot, layer=0, fill=5.0):
        n = len(slot)
        ds, dl = dev(np.asarray(seq, np.int32)), dev(np.asarray(slot, np.int32))
        ko, vo = (full((n, self.KV, self.hd), fill, np.float16) for _ in range(2))
        self.pool.read(layer, n, ptr(dl), ptr(self.dtable), *self.table.shape, ptr(ko), ptr(vo), seqs=ptr(ds))
        return ko.get(), vo.get()

    def fill(self, layer=0, edit=None):
        """all positions of all sequences; returns the values they stand for, a (k, v) pair per sequence"""
        out = []
        for s, n in enumerate(self.lens):
            k, v = self.rows(n, self.KV), self.rows(n, self.KV)
            if edit:
                edit(s, k, v)
            if n:
                self.append(k, v, [s] * n, range(n), layer)
            with np.errstate(invalid="ignore"):
                out.append((_kvq.store(_kvq.rotate(k.astype(np.float64), np.arange(n), self.cos, self.sin, self.inter)),
                            _kvq.store(v.astype(np.float64))))
        return out

    def attend(self, q, counts, lens=None, layer=0, mask=None, scale=0.0, max_len=None, out=None, q_ld=0, out_ld=0,
               max_rows=None, table=None, stream=0, ws=None):
        lens = self.lens if lens is None else lens
        rows = int(sum(counts))
        start = dev(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32))
        dl, dq, dm = dev(np.asarray(lens, np.int32)), dev(q), None if mask is None else dev(mask)
        if out is None:
            out = full((rows, self.H, self.hd), 9.0, np.float16)
        table = self.dtable if table is None else table
        max_rows = max(counts) if max_rows is None else max_rows
        max_len = max(lens) if max_len is None else max_len
        if ws is None:
            ws = zeros(self.pool.attend_workspace(rows, len(counts), max_rows, max_len), np.uint8)
        synchronize()
        self.pool.attend(layer, ptr(dq), ptr(out), ptr(start), ptr(dl), ptr(table), *table.shape, rows=rows,
                         max_rows=max_rows, max_len=max_len, ws=ptr(ws) if ws.nbytes else 0, ws_bytes=ws.nbytes,
                         mask=ptr(dm), mask_words=0 if mask is None else mask.shape[1], scale=scale, q_ld=q_ld,
                         out_ld=out_ld, stream=stream)
        return out.get()


def causal(n, T):
    return np.arange(T)[None] <= np.arange(n)[:, None] + (T - n)


def check_rows(got, q, kv, visible, scale):
    """Within the roundings: fp16 weights (2^-11 of each, and 2^-25 where they are subnormal), the fp16 result, fp32 scores
    (hd products and sums of 2^-24) inside the exponential."""
    k, v = kv
    want, mag, smax = _kvq.attend(q, k, v, visible, scale)
    hd, T = q.shape[-1], len(k)
    vmax = float(np.max(np.abs(v.astype(np.float64)))) if T else 0.0
    score = 2 * hd * 2.0 ** -24 * smax + 2.0 ** -20
    tol = 2.0 ** -11 * (np.abs(want) + mag) * 1.01 + 2 * score * mag + T * 2.0 ** -25 * vmax + 2.0 ** -25
    err = np.abs(got.astype(np.float64) - want)
    assert not np.isnan(err).any()
    bad = err > tol
    assert not bad.any(), (float(np.max(err - tol)), np.argwhere(bad)[:4].tolist())


# ---- append and read -------------------------------------------------------------
@pytest.mark.parametrize("hd,KV,H", [(128, 8, 32), (64, 8, 8), (128, 1, 7), (64, 3, 6)])
@pytest.mark.parametrize("dt", [np.float16, np.float32])
@pytest.mark.parametrize("inter", [True, False])
def test_append_and_read(hip, hd, KV, H, dt, inter):
    p = Pool(hip, hd + KV, H, KV, hd, [130, 1, 33, 64], page=32, interleaved=inter, theta=500000.0)
    seq = np.concatenate([[s] * n for s, n in enumerate(p.lens)])
    slot = np.concatenate([np.arange(n) for n in p.lens])
    order = p.rng.permutation(len(seq))  # any order
    seq, slot = seq[order], slot[order]
    pos = (slot * 13 + seq * 1000) % MAX_POS
    k, v, q = p.rows(len(seq), KV, dt), p.rows(len(seq), KV, dt), p.rows(len(seq), H, dt)
    k[3, 0, :32] = 0.0  # a group of zeros
    v[5] *= np.asarray(1e-7, dt)  # steps that are subnormal or 0
    qo = p.append(k, v, seq, slot, pos=pos, q=q)
    gk, gv = p.read(seq, slot)
    turned = _kvq.rotate(k.astype(np.float64), pos, p.cos, p.sin, inter)
    assert np.array_equal(gk, _kvq.store(turned))
    assert np.array_equal(gv, _kvq.store(v.astype(np.float64)))
    want = _kvq.rotate(q.astype(np.float64), pos, p.cos, p.sin, inter)
    # an fp16 rounding and two fp32 ones of terms up to the pair's magnitude
    assert np.all(np.abs(qo.astype(np.float64) - want) <= 2.0 ** -11 * np.abs(want) + 2.0 ** -22 * np.abs(q).max() + 2.0 ** -25)


def test_append_extremes_and_ties(hip):
    """V rows chosen at the borders: halves, +A beside -A, the fp16 maximum, values that are not finite."""
    p = Pool(hip, 3, 4, 2, 64, [40], page=32)
    n = 40
    v = np.zeros((n, 2, 64), np.float32)
    k = p.rows(n, 2, np.float32)
    for i in range(n):
        v[i] = p.rng.integers(-16, 17, (2, 64)) * 0.5 * 2.0 ** p.rng.integers(-10, 8)  # many exact halves
    v[0, 0, :32] = 0.0
    v[0, 0, 3], v[0, 0, 9] = 4.0, -4.0
    v[1, 0, 5] = 65504.0
    v[1, 1, 5] = -65504.0
    v[2, 0, 7] = 65505.0
    v[2, 1, 40] = np.nan
    v[3, 0, 1] = np.inf
    v[3, 1, 33] = -np.inf
    v[4] = 1e-30
    k[6, 0, 2] = np.nan
    k[6, 1, 50] = np.inf
    k[7] *= 1e5
    p.append(k, v, [0] * n, range(n))
    gk, gv = p.read([0] * n, range(n))
    with np.errstate(invalid="ignore"):
        wk = _kvq.store(_kvq.rotate(k.astype(np.float64), np.arange(n), p.cos, p.sin, True))
    assert np.array_equal(gv, _kvq.store(v.astype(np.float64)), equal_nan=True)
    assert np.array_equal(gk, wk, equal_nan=True)
    assert np.isnan(gv[2, 0, :32]).all() and not np.isnan(gv[2, 0, 32:]).any()


def test_padding_rows_and_bad_pages_are_left_out(hip):
    """Sequences, slots, positions and pages outside leave memory and outputs as they were."""
    p = Pool(hip, 4, 4, 2, 128, [64, 64], page=32, layers=2)
    p.table[1, 1] = p.n_pages  # outside the pool
    p.dtable = dev(p.table)
    base = p.rows(96, 2), p.rows(96, 2)
    seq, slot = [0] * 64 + [1] * 32, list(range(64)) + list(range(32))
    p.append(*base, seq, slot)
    before = p.read(seq, slot)
    bad_seq = [-1, 2, 0, 0, 1, 0, -2147483648, 0]
    bad_slot = [3, 3, -1, 64, 40, 2147483647, 0, 5]
    bad_pos = [0, 0, 0, 0, 0, 0, 0, MAX_POS]
    k, v, q = p.rows(8, 2), p.rows(8, 2), p.rows(8, 4)
    qo = p.append(k, v, bad_seq, bad_slot, pos=bad_pos, q=q)
    assert (qo == 77.0).all()
    p.append(k, v, bad_seq, bad_slot, layer=1, pos=bad_pos)
    after = p.read(seq, slot)
    assert np.array_equal(before[0], after[0]) and np.array_equal(before[1], after[1])
    rk, rv = p.read(bad_seq[:7], bad_slot[:7], fill=5.0)
    assert (rk == 5.0).all() and (rv == 5.0).all()
    lk, lv = p.read(seq, slot, layer=1)  # the other layer holds zeros
    assert not lk.any() and not lv.any()


def test_strided_rows(hip):
    """q, k and v as column ranges of one product's rows, as the decoder has them."""
    p = Pool(hip, 5, 4, 2, 64, [50], page=64, interleaved=False)
    n, w = 50, 8 * 64
    x = p.rng.standard_normal((n, w)).astype(np.float32)
    dx, ds = dev(x), dev(np.arange(n, dtype=np.int32))
    qo = zeros((n, 4, 64), np.float16)
    synchronize()
    p.pool.append(0, n, ptr(dx) + 4 * 256, ptr(dx) + 4 * 384, ptr(ds), ptr(p.dtable), 1, 1, dtype=hip.F32, q=ptr(dx),
                  q_out=ptr(qo), q_ld=w, k_ld=w, v_ld=w)
    gk, gv = p.read([0] * n, range(n))
    k = x[:, 256:384].reshape(n, 2, 64).astype(np.float64)
    assert np.array_equal(gk, _kvq.store(_kvq.rotate(k, np.arange(n), p.cos, p.sin, False)))
    assert np.array_equal(gv, _kvq.store(x[:, 384:].reshape(n, 2, 64)))
    want = _kvq.rotate(x[:, :256].reshape(n, 4, 64).astype(np.float64), np.arange(n), p.cos, p.sin, False)
    assert np.all(np.abs(qo.get() - want) <= 2.0 ** -11 * np.abs(want) + 2.0 ** -22 * np.abs(x).max())


# ---- attention -------------------------------------------------------------------
@pytest.mark.parametrize("hd,KV,H,page", [(128, 2, 8, 64), (64, 4, 4, 32), (128, 1, 7, 128), (64, 2, 16, 256), (128, 2, 2, 32)])
@pytest.mark.parametrize("rows,T", [(1, 1), (1, 2), (1, 31), (1, 32), (1, 33), (1, 777), (1, 3000), (2, 2), (5, 5), (5, 64), (5, 1025),
                                    (17, 17), (33, 100), (70, 200), (300, 301), (129, 129)])
def test_attention_causal(hip, hd, KV, H, page, rows, T):
    p = Pool(hip, rows * 7 + T, H, KV, hd, [T], page=page)
    (kv,) = p.fill()
    q = p.rows(rows, H)
    got = p.attend(q, [rows])
    check_rows(got, q, kv, causal(rows, T), hd ** -0.5)


@pytest.mark.parametrize("hd,KV,H", [(128, 2, 8), (64, 4, 4), (128, 1, 7)])
def test_attention_ragged_batch(hip, hd, KV, H):
    lens = [0, 1, 700, 33, 64, 5, 2000, 31]
    counts = [0, 1, 3, 0, 64, 5, 1, 2]
    p = Pool(hip, 11, H, KV, hd, lens, page=64)
    kvs = p.fill()
    q = p.rows(sum(counts), H)
    got = p.attend(q, counts)
    at = 0
    for s, n in enumerate(counts):
        if n:
            check_rows(got[at:at + n], q[at:at + n], kvs[s], causal(n, lens[s]), hd ** -0.5)
        at += n


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows,T", [(1, 1), (7, 7), (60, 500), (64, 96), (65, 65), (128, 1000), (100, 131)])
def test_attention_tree_masks(hip, hd, rows, T):
    """Random masks, among them rows that see only the prefix, or (without one) nothing at all."""
    p = Pool(hip, rows + T, 4, 2, hd, [T], page=32)
    (kv,) = p.fill()
    bits = p.rng.random((rows, rows)) < 0.2
    bits[::5] = False
    words = -(-rows // 64)
    mask = np.zeros((rows, words), np.uint64)
    for i, j in np.argwhere(bits):
        mask[i, j // 64] |= np.uint64(1) << np.uint64(j % 64)
    mask[:, -1] |= np.uint64(1) << np.uint64(63) if rows % 64 else np.uint64(0)  # a bit past the rows means nothing
    visible = np.concatenate([np.ones((rows, T - rows), bool), bits], 1)
    q = p.rows(rows, 4)
    got = p.attend(q, [rows], mask=mask)
    check_rows(got, q, kv, visible, hd ** -0.5)
    if T == rows:
        assert not got[::5].any()


@pytest.mark.parametrize("hd", [64, 128])
def test_attention_nan_and_inf_behind_masks(hip, hd):
    """NaN keys and values of positions that a row does not see leave it alone; a row that sees them is NaN there."""
    T, rows = 70, 6

    def edit(s, k, v):
        v[67, 0, 40] = np.nan  # the second group of KV head 0
        k[66, 1, 3] = np.inf  # a key of KV head 1
        v[69, 1, 0] = np.inf
    p = Pool(hip, 8, 4, 2, hd, [T], page=32)
    kv = p.fill(edit=edit)[0]
    q = p.rows(rows, 4)
    bits = np.tril(np.ones((rows, rows), bool))
    bits[4, 3] = False  # row 4 does not see position 67
    bits[5] = [1, 0, 0, 0, 0, 1]
    mask = np.zeros((rows, 1), np.uint64)
    for i, j in np.argwhere(bits):
        mask[i, 0] |= np.uint64(1) << np.uint64(j)
    got = p.attend(q, [rows], mask=mask)
    clean = [np.where(np.isnan(x), 0, x) for x in kv]
    visible = np.concatenate([np.ones((rows, T - rows), bool), bits], 1)
    for h in range(4):
        kvh = h // 2
        for r in range(rows):
            hole = np.zeros(hd, bool)
            for t in np.nonzero(visible[r])[0]:
                if np.isnan(kv[0][t, kvh]).any():
                    hole[:] = True
                hole |= np.isnan(kv[1][t, kvh])
            assert np.array_equal(np.isnan(got[r, h]), hole), (r, h)
            if not hole.any():
                one = [x[:, kvh:kvh + 1] for x in clean]
                check_rows(got[r:r + 1, h:h + 1], q[r:r + 1, h:h + 1], one, visible[r:r + 1], hd ** -0.5)
    # the same behind a causal mask and past the end
    got = p.attend(q[:3], [3], lens=[66 + 1])
    check_rows(got[:2], q[:2], [x[:66] for x in clean], causal(2, 66), hd ** -0.5)


@pytest.mark.parametrize("value", [1.0, 60.0, -60.0])
def test_attention_sharp_and_flat_scores(hip, value):
    """Scores of some hundreds, one above the rest by far, and all alike."""
    p = Pool(hip, 21, 4, 2, 128, [300], page=64)
    (kv,) = p.fill()
    q = (p.rows(2, 4).astype(np.float32) * value).astype(np.float16)
    check_rows(p.attend(q, [2]), q, kv, causal(2, 300), 128 ** -0.5)
    q[:] = 0
    check_rows(p.attend(q, [2]), q, kv, causal(2, 300), 128 ** -0.5)


def test_attention_infinite_scores(hip):
    """A query of infinities: rows whose scores are all -inf weigh nothing, +inf gives NaN as the formula does."""
    p = Pool(hip, 22, 2, 1, 64, [5], page=32)
    n = 5
    k, v = np.ones((n, 1, 64), np.float16), p.rows(n, 1)
    p.append(k, v, [0] * n, range(n), pos=[0] * n)
    q = np.zeros((1, 2, 64), np.float16)
    q[0, 0, 0], q[0, 1, 0] = -np.inf, np.inf
    got = p.attend(q, [1])
    assert not got[0, 0].any() and np.isnan(got[0, 1]).all()


def test_attention_strides_scale_and_untouched_rows(hip):
    p = Pool(hip, 31, 4, 2, 64, [200, 90], page=64)
    kvs = p.fill()
    wide = np.zeros((9, 4 * 64 + 24), np.float16)
    q = p.rows(9, 4)
    wide[:, :256] = q.reshape(9, 256)
    out = full((9, 4 * 64 + 12), 3.0, np.float16)
    # rows 0-2 of the first sequence, 3-5 of the second; max_rows 2 leaves each one's third; 6-8 belong to nobody
    start, lens, dq = dev(np.array([0, 3, 6], np.int32)), dev(np.array([200, 90], np.int32)), dev(wide)
    ws = zeros(max(16, p.pool.attend_workspace(9, 2, 2, 200)), np.uint8)
    synchronize()
    p.pool.attend(0, ptr(dq), ptr(out), ptr(start), ptr(lens), ptr(p.dtable), *p.table.shape, rows=9, max_rows=2, max_len=200,
                  ws=ptr(ws), ws_bytes=ws.nbytes, scale=0.3, q_ld=280, out_ld=268)
    got = out.get()
    assert (got[:, 256:] == 3.0).all() and (got[[2, 5, 6, 7, 8]] == 3.0).all()
    for s, T in ((0, 200), (1, 90)):
        vis = causal(3, T)[:2]
        check_rows(got[3 * s:3 * s + 2, :256].reshape(2, 4, 64), q[3 * s:3 * s + 2], kvs[s], vis, np.float32(0.3))


def test_attention_absent_pages(hip):
    """Page ids outside the pool and tables shorter than the length hold nothing."""
    p = Pool(hip, 33, 4, 2, 128, [256], page=64)
    (kv,) = p.fill()
    q = p.rows(1, 4)
    t = p.table.copy()
    t[0, 1], t[0, 2] = -1, p.n_pages + 7
    vis = np.ones((1, 256), bool)
    vis[:, 64:192] = False
    check_rows(p.attend(q, [1], table=dev(t)), q, kv, vis, 128 ** -0.5)
    vis[:, 192:] = False
    check_rows(p.attend(q, [1], table=dev(t[:, :1])), q, kv, vis, 128 ** -0.5)
    assert not p.attend(q, [1], table=dev(np.full((1, 4), -1, np.int32))).any()


def test_attention_fewer_positions_than_rows(hip):
    """Rows before the first position see nothing."""
    p = Pool(hip, 34, 2, 1, 64, [40], page=32)
    (kv,) = p.fill()
    q = p.rows(6, 2)
    got = p.attend(q, [6], lens=[2])
    assert not got[:4].any()
    check_rows(got[4:], q[4:], [x[:2] for x in kv], causal(2, 2), 64 ** -0.5)
    assert not p.attend(q, [6], lens=[0]).any()
    # a length past max_len costs time, not correctness
    check_rows(p.attend(q, [6], lens=[40], max_len=1), q, kv, causal(6, 40), 64 ** -0.5)


@pytest.mark.parametrize("rows", [1, 40])
def test_captured_and_replayed(hip, rows):
    """append and attend recorded into a graph, replayed on new inputs with eager calls between."""
    T = 500
    p = Pool(hip, 41, 8, 2, 128, [T], page=64)
    (kv,) = p.fill()
    ks, vs = kv[0].copy(), kv[1].copy()
    slots = dev(np.arange(T - rows, T, dtype=np.int32))
    q, k, v = (zeros((rows, h, 128), np.float16) for h in (8, 2, 2))
    qo, out = zeros((rows, 8, 128), np.float16), zeros((rows, 8, 128), np.float16)
    start, lens = dev(np.array([0, rows], np.int32)), dev(np.array([T], np.int32))
    ws = zeros(max(16, p.pool.attend_workspace(rows, 1, rows, T)), np.uint8)

    def step(st):
        p.pool.append(0, rows, ptr(k), ptr(v), ptr(slots), ptr(p.dtable), *p.table.shape, q=ptr(q), q_out=ptr(qo), stream=st)
        p.pool.attend(0, ptr(qo), ptr(out), ptr(start), ptr(lens), ptr(p.dtable), *p.table.shape, rows=rows, max_rows=rows,
                      max_len=T, ws=ptr(ws), ws_bytes=ws.nbytes, stream=st)
    graph, side = Graph(step), Stream()
    for i in range(4):
        nq, nk, nv = p.rows(rows, 8), p.rows(rows, 2), p.rows(rows, 2)
        for t, a in ((q, nq), (k, nk), (v, nv)):
            t.put(a)
        out.put(np.zeros(out.shape))
        graph.launch()
        got, turned = out.get(), qo.get()
        pos = np.arange(T - rows, T)
        ks[T - rows:] = _kvq.store(_kvq.rotate(nk.astype(np.float64), pos, p.cos, p.sin, True))
        vs[T - rows:] = _kvq.store(nv.astype(np.float64))
        check_rows(got, turned, (ks, vs), causal(rows, T), 128 ** -0.5)
        out.put(np.zeros(out.shape))
        step(side.handle)
        side.wait()
        assert np.array_equal(out.get(), got), i


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("KV,H,seqs,most", [(8, 32, 32, 20), (16, 16, 8, 300)])
def test_attention_many_rows_in_many_sequences(hip, hd, KV, H, seqs, most):
    """Enough rows for tiles of 256 queries, the sequences with from none to `most` of them."""
    rng = np.random.default_rng(seqs)
    counts = [most, 0, 1] + [int(v) for v in rng.integers(1, most, seqs - 3)]
    lens = [n + int(v) for n, v in zip(counts, rng.integers(0, 90, seqs))]
    p = Pool(hip, hd + seqs, H, KV, hd, lens, page=32)
    kvs = p.fill()
    q = p.rows(sum(counts), H)
    got = p.attend(q, counts)
    at = 0
    for s, n in enumerate(counts):
        if n:
            check_rows(got[at:at + n], q[at:at + n], kvs[s], causal(n, lens[s]), hd ** -0.5)
        at += n


@pytest.mark.parametrize("rows,H", [(1, 1), (1, 20), (40, 1), (60, 4)])
def test_attention_long_tail_of_small_weights(hip, rows, H):
    """One position 16 nats above thousands of others whose values alone are not zero: a weight is rounded by 2^-11 of itself
    or 2^-32 of the largest, so the result by 2^-11 of itself, the positions times 2^-32 of the largest value, its own fp16
    rounding, and what the fp32 scores (64 products) do to the exponentials."""
    T, hd = 4000, 64
    p = Pool(hip, 71, H, 1, hd, [T], page=256)
    k, v = np.zeros((T, 1, hd), np.float16), np.ones((T, 1, hd), np.float16)
    k[0], v[0] = 2.0, 0.0
    p.append(k, v, [0] * T, range(T), pos=[0] * T)
    q = np.ones((rows, H, hd), np.float16)  # scores 2 hd / sqrt(hd) = 16 and 0
    got = p.attend(q, [rows], mask=None).astype(np.float64)
    n = T - rows + np.arange(rows, dtype=np.float64)  # positions after the first that row i sees
    want = (n * np.exp(-16.0) / (1 + n * np.exp(-16.0)))[:, None, None]
    tol = 2.0 ** -11 * want * 2.01 + T * 2.0 ** -32 + 2.0 ** -25 + 2 * hd * 2.0 ** -24 * 16 * want
    assert np.all(np.abs(got - want) <= tol), float(np.max(np.abs(got - want) - tol))


def test_pages_past_32_bits(hip):
    """Pages that begin more than 2^32 bytes into a layer, of the second layer: appended, read and attended as the first ones."""
    hd, KV, page, n_pages, T = 128, 8, 4096, 1000, 300
    pool = hip.HipKvPool(n_layers=2, n_heads=8, n_kv_heads=KV, head_dim=hd, n_pages=n_pages, page_tokens=page, max_pos=MAX_POS)
    assert pool.page_bytes() * (n_pages - 2) > 1 << 32
    rng = np.random.default_rng(5)
    dk, dv, dq = (dev(rng.standard_normal((n, 8, hd)).astype(np.float16)) for n in (T, T, 2))
    slots, start, lens = dev(np.arange(T, dtype=np.int32)), dev(np.array([0, 2], np.int32)), dev(np.array([T], np.int32))
    ws = zeros(max(16, pool.attend_workspace(2, 1, 2, T)), np.uint8)
    seen = []
    for layer, pg in ((0, 0), (0, n_pages - 1), (1, n_pages - 2)):
        table = dev(np.array([[pg]], np.int32))
        ko, vo, out = (full((n, 8, hd), 3.0, np.float16) for n in (T, T, 2))
        synchronize()
        pool.append(layer, T, ptr(dk), ptr(dv), ptr(slots), ptr(table), 1, 1)
        pool.read(layer, T, ptr(slots), ptr(table), 1, 1, ptr(ko), ptr(vo))
        pool.attend(layer, ptr(dq), ptr(out), ptr(start), ptr(lens), ptr(table), 1, 1, rows=2, max_rows=2, max_len=T,
                    ws=ptr(ws), ws_bytes=ws.nbytes)
        seen.append((ko.get(), vo.get(), out.get()))
    assert seen[0][0].any() and seen[0][2].any()
    for other in seen[1:]:
        for a, b in zip(seen[0], other):
            assert np.array_equal(a, b)
    pool.close()


def test_two_streams_over_the_same_pages(hip):
    """Calls on two streams, each with its workspace, read the same pages and give what they give one after the other."""
    T = 3000
    p = Pool(hip, 81, 8, 2, 128, [T], page=64)
    p.fill()
    start, lens = dev(np.array([0, 5], np.int32)), dev(np.array([T], np.int32))
    qs, outs = [dev(p.rows(5, 8)) for _ in range(2)], [full((5, 8, 128), 9.0, np.float16) for _ in range(2)]
    wss = [zeros(max(16, p.pool.attend_workspace(5, 1, 5, T)), np.uint8) for _ in range(2)]

    def call(i, st):
        p.pool.attend(0, ptr(qs[i]), ptr(outs[i]), ptr(start), ptr(lens), ptr(p.dtable), *p.table.shape, rows=5, max_rows=5,
                      max_len=T, ws=ptr(wss[i]), ws_bytes=wss[i].nbytes, stream=st)
    synchronize()
    want = []
    for i in range(2):
        call(i, 0)
        want.append(outs[i].get())
    streams = [Stream(), Stream()]
    for _ in range(8):
        for i in range(2):
            call(i, streams[i].handle)
    for s in streams:
        s.wait()
    assert all(np.array_equal(outs[i].get(), want[i]) for i in range(2)) and not np.array_equal(*want)


def test_repeated_calls_agree_bit_for_bit(hip):
    p = Pool(hip, 51, 8, 2, 128, [3000, 40, 1500], page=64)
    p.fill()
    q = p.rows(9, 8)
    first = p.attend(q, [3, 3, 3])
    for _ in range(3):
        assert np.array_equal(p.attend(q, [3, 3, 3]), first)


# ---- refusals ---------------------------------------------------------------------
def test_refusals(hip):
    p = Pool(hip, 61, 4, 2, 64, [10], page=32, layers=2)
    buf = zeros(1 << 16, np.uint8)
    b, P = ptr(buf), p.pool
    ok = dict(n=1, k=b, v=b, slots=b, table=b, n_seqs=1, table_ld=1)
    for bad in (dict(k=0), dict(v=0), dict(slots=0), dict(table=0), dict(n_seqs=0), dict(table_ld=0), dict(k=b + 2),
                dict(q=b), dict(q=b, q_out=b + 8), dict(q=b, q_out=b), dict(k_ld=64), dict(v_ld=100), dict(k_ld=132), dict(n=1 << 25),
                dict(n=1 << 24)):
        with pytest.raises(hip.ArgError):
            P.append(0, **dict(ok, **bad))
    with pytest.raises(hip.UnsupportedMethod):
        P.append(0, **dict(ok, dtype=hip.Q8_0))
    for layer in (-1, 2):
        with pytest.raises(hip.ArgError):
            P.append(layer, **ok)
        with pytest.raises(hip.ArgError):
            P.read(layer, 1, b, b, 1, 1, b, b)
    with pytest.raises(hip.ArgError):
        P.read(0, 1, b, b, 1, 1, b + 2, b)
    need = P.attend_workspace(2, 1, 1, 100000)
    assert need > 0 and P.attend_workspace(2, 1, 3, 10) == 0 and P.attend_workspace(0, 1, 1, 10) == 0
    at = dict(q=b, out=b + 32768, row_start=b, kv_len=b, table=b, n_seqs=1, table_ld=1, rows=2, max_rows=1, max_len=100000, ws=b,
              ws_bytes=need)
    for bad in (dict(q=0), dict(out=0), dict(row_start=0), dict(kv_len=0), dict(table=0), dict(n_seqs=0), dict(table_ld=0),
                dict(out=b), dict(max_rows=0), dict(max_rows=3), dict(ws=0), dict(ws_bytes=need - 1), dict(ws=b + 8), dict(q=b + 8),
                dict(out=b + 32772), dict(mask=b), dict(scale=float("nan")), dict(q_ld=128), dict(out_ld=255), dict(out_ld=258),
                dict(n_seqs=70000), dict(max_len=1 << 40)):
        with pytest.raises(hip.ArgError):
            P.attend(0, **dict(at, **bad))
    P.append(0, **dict(ok, n=0))
    P.read(0, 0, b, b, 1, 1, b, b)
    P.attend(0, **dict(at, rows=0))
    assert P.page_bytes() == 2 * 36 * 64
    P.close()
    with pytest.raises(hip.ArgError):
        P.append(0, **ok)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows,H", [(1, 1), (1, 20), (5, 8), (20, 4), (60, 4), (300, 1)])
@pytest.mark.parametrize("T", [40, 1000])
def test_attention_scores_near_the_formats_end(hip, hd, rows, H, T):
    """Queries and keys of 65504 and a little less in one channel: scores of some 5e8, whose fp32 neighbours are 32 or 64 apart.
    A position that is alone at the top is the answer, positions that share it are averaged; nothing overflows."""
    T = max(T, rows)
    p = Pool(hip, hd + rows, H, 1, hd, [T], page=32)
    rng = np.random.default_rng(hd + rows + T)
    k = np.zeros((T, 1, hd), np.float16)
    k[:, 0, 3] = rng.integers(0, 3, T) * 32 + 65408  # 65408, 65440, 65472
    k[:, 0, 40] = rng.standard_normal(T)
    v = rng.integers(-7, 8, (T, 1, hd)).astype(np.float16)
    v[:, 0, 5] = 0
    v[:, 0, ::32] = 8  # steps of 1: the values are stored as they are
    top, low = T - rows, max(0, T - rows - 17)  # seen by every row
    k[top, 0, 3] = 65504
    p.append(k, v, [0] * T, range(T), pos=[0] * T)
    q = np.zeros((rows, H, hd), np.float16)
    half = 2.0 ** -11  # an fp16 rounding: of a weight, of the result
    for big in (4096.0, 60000.0, 65504.0):
        q[:, :, 3] = big
        got = p.attend(q, [rows]).astype(np.float64)
        want = v[top, 0].astype(np.float64)
        assert np.all(np.abs(got - want) <= 2.01 * half * np.abs(want)), big
    # two at the top, in blocks of their own where there is room
    k[low, 0, 3] = 65504
    k[:, 0, 40] = 0
    p.append(k, v, [0] * T, range(T), pos=[0] * T)
    got = p.attend(q, [rows]).astype(np.float64)
    both = v[[top, low], 0].astype(np.float64)
    assert np.all(np.abs(got - both.mean(0)) <= 1.01 * half * (np.abs(both.mean(0)) + np.abs(both).mean(0)))
    # all positions alike, far below zero: their mean
    k[:] = 0
    k[:, 0, 3] = 65504
    p.append(k, v, [0] * T, range(T), pos=[0] * T)
    q[:, :, 3] = -65504.0
    got = p.attend(q, [rows]).astype(np.float64)
    for r in range(rows):
        n = T - rows + r + 1
        seen = v[:n, 0].astype(np.float64)
        # besides, fp32 sums of up to n terms of up to 8, and the result below fp16's normal range
        tol = 1.01 * half * (np.abs(seen.mean(0)) + np.abs(seen).mean(0)) + n * 2.0 ** -24 * 8 + 2.0 ** -25
        assert np.all(np.abs(got[r] - seen.mean(0)) <= tol), r


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows,H", [(1, 1), (5, 8), (20, 4), (60, 4), (300, 1)])
def test_attention_a_later_score_one_fp32_step_higher(hip, hd, rows, H):
    """Products of 2^30 and 2^30 + 128: scores of some 1.9e8 and 1.4e8, whose fp32 neighbours are 16 apart, one step from each
    other.  In any rounding the second weighs 2^8 times the first or more (they are 23 and 16 apart, less half a step)."""
    T = max(200, rows + 200)
    p = Pool(hip, hd * rows, H, 1, hd, [T], page=32)
    k, v = np.zeros((T, 1, hd), np.float16), np.zeros((T, 1, hd), np.float16)
    k[[0, 130], 0, 1] = 2.0 ** 15
    k[130, 0, 33] = 8.0
    v[0, 0, 7], v[130, 0, 9] = 7.0, 5.0
    p.append(k, v, [0] * T, range(T), pos=[0] * T)
    q = np.zeros((rows, H, hd), np.float16)
    q[:, :, 1], q[:, :, 33] = 2.0 ** 15, 16.0
    got = p.attend(q, [rows]).astype(np.float64)
    assert np.all(np.abs(got[..., 9] - 5.0) <= 5.0 * (2.0 ** -8 + 2.01 * 2.0 ** -11)), float(got[..., 9].min())
    assert np.all((got[..., 7] >= 0) & (got[..., 7] <= 7.0 * 2.0 ** -8))
    got[..., [7, 9]] = 0
    assert not got.any()


def test_overlapping_rows_are_refused(hip):
    """Outputs that share a byte with an input or the workspace, at either end or between strided rows; rows that lie between
    another's are taken."""
    H, KV, hd, n, T = 4, 2, 64, 5, 2000  # (shorter ones need no workspace)
    p = Pool(hip, 91, H, KV, hd, [T], page=64)
    (kv,) = p.fill()
    P, w, kw = p.pool, 2 * H * hd, 2 * KV * hd  # bytes of a query's and of a key's row
    slots = dev(np.arange(n, dtype=np.int32))
    buf = zeros(1 << 20, np.uint8)
    at = ptr(buf) + (1 << 19)  # q; k, v and the outputs around it
    far = dict(k=at + 65536, v=at + 131072)

    def append(**k):
        P.append(0, n, **dict(dict(far, slots=ptr(slots), table=ptr(p.dtable), n_seqs=1, table_ld=p.table.shape[1], q=at), **k))
    for out in (at, at + 16, at + n * w - 16, at - n * w + 16, far["k"] + kw, far["v"] + n * kw - 16, far["k"] - n * w + 16):
        with pytest.raises(hip.ArgError):
            append(q_out=out)
    with pytest.raises(hip.ArgError):  # in the gaps of strided q, but longer than they are
        append(q_out=at + w, q_ld=H * hd + 64)
    start, lens = dev(np.array([0, n], np.int32)), dev(np.array([T], np.int32))
    need = P.attend_workspace(n, 1, n, T)
    assert need > 0

    def attend(**k):
        P.attend(0, **dict(dict(q=at, out=at + 65536, row_start=ptr(start), kv_len=ptr(lens), table=ptr(p.dtable), n_seqs=1,
                                table_ld=p.table.shape[1], rows=n, max_rows=n, max_len=T, ws=at + 131072, ws_bytes=need), **k))
    for bad in (dict(out=at), dict(out=at + 8), dict(out=at - n * w + 8), dict(out=at + n * w - 8), dict(ws=at + n * w - 16),
                dict(ws=at - need // 16 * 16 + 16), dict(ws=at + 65536 + 16), dict(out=at + w - 8, q_ld=2 * H * hd, out_ld=2 * H * hd),
                dict(out=at + w, q_ld=2 * H * hd, out_ld=3 * H * hd)):
        with pytest.raises(hip.ArgError):
            attend(**bad)
    # q and out as the halves of one buffer's rows, and one right behind the other
    q = p.rows(n, H)
    both = np.full((n, 2, H, hd), 9.0, np.float16)
    both[:, 0] = q
    d = dev(both)
    ws = zeros(need, np.uint8)
    attend(q=ptr(d), out=ptr(d) + w, q_ld=2 * H * hd, out_ld=2 * H * hd, ws=ptr(ws))
    got = d.get()
    assert np.array_equal(got[:, 0], q)
    check_rows(got[:, 1], q, kv, causal(n, T), hd ** -0.5)
    d = dev(np.concatenate([q, q]))
    attend(q=ptr(d), out=ptr(d) + n * w, ws=ptr(ws))
    assert np.array_equal(d.get(), np.concatenate([q, got[:, 1]]))


# ---- every kernel's masks, NaN groups and absent pages, in batches ---------------------
def check_but_holes(got, q, kv, visible, scale):
    """check_rows for what is a number; NaN exactly where a row sees a key of one (everywhere) or a value of one (that group)."""
    rows, H, hd = q.shape
    KV, T = kv[0].shape[1], len(kv[0])
    bad_k, bad_v = np.isnan(kv[0]).any(-1), np.isnan(kv[1])  # [T][KV], [T][KV][hd]
    hole = np.zeros((rows, H, hd), bool)
    for t in np.nonzero(bad_k.any(-1) | bad_v.any((1, 2)))[0]:
        for h in range(H):
            g = h // (H // KV)
            hole[visible[:, t], h] |= bad_k[t, g] | bad_v[t, g]
    assert np.array_equal(np.isnan(got), hole)
    k, v, q = (np.where(np.isnan(x), 0, x).astype(np.float64) for x in (*kv, q))
    want, mag, smax = np.zeros((rows, H, hd)), np.zeros((rows, H, hd)), 0.0
    for h in range(H):
        kh, vh = k[:, h // (H // KV)], v[:, h // (H // KV)]
        s = np.where(visible, q[:, h] @ kh.T * scale, -np.inf)
        smax = max(smax, float(np.max(np.abs(q[:, h]) @ np.abs(kh).T)) * scale)
        m = s.max(-1, keepdims=True)
        w = np.exp(s - np.where(m == -np.inf, 0, m))
        w /= np.where(m == -np.inf, 1, w.sum(-1, keepdims=True))
        want[:, h], mag[:, h] = w @ vh, w @ np.abs(vh)
    score = 2 * hd * 2.0 ** -24 * smax + 2.0 ** -20  # as in check_rows
    vmax = float(np.max(np.abs(v.astype(np.float64)))) if T else 0.0
    tol = 2.0 ** -11 * (np.abs(want) + mag) * 1.01 + 2 * score * mag + T * 2.0 ** -25 * vmax + 2.0 ** -25
    bad = (np.abs(got.astype(np.float64) - want) > tol) & ~hole
    assert not bad.any(), np.argwhere(bad)[:4].tolist()


def fill_long(p, edit):
    """Pool.fill with rotation positions that start again at MAX_POS."""
    out = []
    for s, n in enumerate(p.lens):
        k, v, pos = p.rows(n, p.KV), p.rows(n, p.KV), np.arange(n) % MAX_POS
        edit(s, k, v)
        p.append(k, v, [s] * n, range(n), pos=pos)
        with np.errstate(invalid="ignore"):
            out.append((_kvq.store(_kvq.rotate(k.astype(np.float64), pos, p.cos, p.sin, p.inter)), _kvq.store(v.astype(np.float64))))
    return out


# counts of rows, prefixes before them, heads, KV heads; the kernel and tile that these sizes take
BATCHES = {
    "16 queries": ([1, 0, 3, 2], [70, 9, 300, 0], 8, 4),
    "32 queries, two tiles": ([25, 7, 30], [40, 500, 3], 4, 2),
    "128 queries in two key groups, ranges": ([60, 33, 0, 41], [440, 900, 50, 7], 4, 2),
    "256 queries in one range": ([300, 1, 70, 129, 200, 5, 64, 300], [0, 90, 33, 64, 5, 200, 1, 31], 16, 16),
    "256 queries, ranges": ([150], [12350], 8, 8),
}


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("name", sorted(BATCHES))
def test_batches_with_masks_holes_and_absent_pages(hip, name, masked, hd):
    counts, before, H, KV = BATCHES[name]
    held = [n + b for n, b in zip(counts, before)]
    rng = np.random.default_rng(len(name) + hd + masked)

    def edit(s, k, v):
        """Numbers that are none: in the sequence's own rows, where masks hide them from some rows, and behind its end."""
        n, T = counts[s], held[s]
        for at in {T - n // 2, T - 1} if n > 1 else ():
            v[at, rng.integers(KV), rng.integers(hd)] = rng.choice([np.nan, np.inf, -np.inf])
        if n > 2:
            k[T - n // 3, 0, 5] = np.nan
        v[T:], k[T:] = np.nan, np.inf
    p = Pool(hip, hd + masked, H, KV, hd, [n + 3 for n in held], page=32)
    kvs = fill_long(p, edit)
    q, total, words = p.rows(sum(counts), H), sum(counts), -(-max(counts) // 64)
    mask, seen, table, at = np.zeros((total, words), np.uint64), [], p.table.copy(), 0
    for s, (n, T) in enumerate(zip(counts, held)):
        vis = causal(n, T)
        if masked:
            bits = rng.random((n, n)) < 0.3
            bits[::7] = False
            vis = np.concatenate([np.ones((n, T - n), bool), bits], 1)
            for i, j in np.argwhere(bits):
                mask[at + i, j // 64] |= np.uint64(1) << np.uint64(j % 64)
            if n % 64 and n:
                mask[at:at + n, n // 64] |= np.uint64(1) << np.uint64(63)  # past the sequence's rows: nothing
        if s % 2 == 0:  # every other sequence has pages that are not there
            for pg, bad in ((T // 64, -1), (max(0, T // 32 - 1), p.n_pages + 3)):
                table[s, pg] = bad
                vis[:, 32 * pg:32 * pg + 32] = False
        seen.append(vis)
        at += n
    got = p.attend(q, counts, lens=held, mask=mask if masked else None, table=dev(table))
    at = 0
    for s, n in enumerate(counts):
        if n:
            kv = [x[:held[s]] for x in kvs[s]]
            check_but_holes(got[at:at + n], q[at:at + n], kv, seen[s], hd ** -0.5)
        at += n
