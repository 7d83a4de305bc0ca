"""Decoders whose cache is held in 4 bits (KV_Q4), and tokens sampled on the device: the decoder's entry points run
over the 4-bit cache, against the fp16 decoder, the oracle with a 4-bit cache, and themselves."""
import numpy as np
import pytest

import _kvq
import oracle as O
from _devmem import dev, ptr, zeros
from _models import MIX_IDS, hip_cfg, oracle_cfg, rel_err

pytestmark = pytest.mark.gpu

SHAPES = {
    "llama": dict(n_layers=2, n_heads=8, n_kv_heads=2, vocab=2048, ctx_len=2600),
    "mha": dict(n_layers=2, vocab=2048, ctx_len=2600),
    "qwen": dict(arch="qwen2", n_layers=2, hidden=1024, n_heads=8, n_kv_heads=1, head_dim=128, vocab=2048, ctx_len=2600, mix="q8_0"),
}


def decoder(hip, ocfg, q4=True, max_batch=128):
    cfg = hip_cfg(hip, ocfg, max_batch)
    cfg.kv_format = hip.KV_Q4 if q4 else hip.KV_F16
    d = hip.HipQuantDecoder(cfg)
    d.synthesize(MIX_IDS[ocfg.mix], ocfg.seed, ocfg.weight_std)
    return d


def ids(seed, n, vocab):
    return [int(v) for v in np.random.default_rng(seed).integers(0, vocab, n)]


def kv(d, ocfg, layer, n, pos0=0):
    return [np.stack([d.read_kv_rows(layer, w, h, pos0, n).view(np.float16) for h in range(ocfg.n_kv_heads)], 1) for w in (0, 1)]


@pytest.mark.parametrize("shape", sorted(SHAPES))
@pytest.mark.parametrize("n", [1, 5, 16, 17, 50, 128, 300])
def test_first_layer_rows_are_the_fp16_rows_quantised(hip, shape, n):
    """The first layer's rows do not depend on the cache: each is within half a step of the fp16 decoder's."""
    ocfg = oracle_cfg(**SHAPES[shape])
    a, b, t = decoder(hip, ocfg), decoder(hip, ocfg, q4=False), ids(n, n, ocfg.vocab)
    a.observe(t)
    b.observe(t)
    for got, ref in zip(kv(a, ocfg, 0, n), kv(b, ocfg, 0, n)):
        ref = ref.astype(np.float64)
        g = ref.reshape(n, ocfg.n_kv_heads, -1, 32)
        hi, lo = g.max(-1, keepdims=True), -g.min(-1, keepdims=True)
        step = np.maximum(hi, lo) / 8
        # Half a step, and what an extreme on the end without a code lacks (up to half a step more).  Besides, of values of up
        # to 8 steps, each rounded to fp16 (2^-11 of itself): the fp16 row, 8 * 2^-11 steps; the stored value, the same; the
        # stored step in the bound 0.5 + 7.5 steps, the same; the step taken here from a rounded extreme, the same: 32 * 2^-11.
        # Above 16 rows the fp16 decoder may add K slices in another order (fp32 roundings of terms up to some 30 steps).
        # Extremes of both signs within 2 * 2^-11 of each other may be the other way round before they were rounded to fp16, and
        # then the other end is the one without a code.
        far = np.where(np.abs(hi - lo) <= 2.0 ** -10 * np.maximum(hi, lo), np.abs(g), np.where(hi > lo, -g, g))
        end = np.maximum(0.0, far - 7.5 * step)
        tol = 0.5 * step + end + step * 32 * 2.0 ** -11 + 1e-4 * step
        err = np.abs(got.astype(np.float64).reshape(g.shape) - g)
        assert np.all(err <= tol), float(np.max((err - tol) / step))


class FourBitOracle(O.OracleModel):
    """The oracle with its cache in 4 bits."""

    def forward(self, *a, **k):
        plain, O.round_f16 = O.round_f16, lambda x: _kvq.store(x).astype(np.float32)
        try:
            return super().forward(*a, **k)
        finally:
            O.round_f16 = plain


@pytest.mark.parametrize("shape", sorted(SHAPES))
def test_logits_against_the_oracle_with_a_4_bit_cache(hip, shape):
    """fp16 activations move a value by about 5e-4 of itself and so about one code in 100 by one step, where quantising
    moves every value by 0.29 steps rms: the device stays within half of what the 4-bit cache itself changes."""
    ocfg = oracle_cfg(**SHAPES[shape])
    om = O.OracleModel(ocfg)
    f16, q4 = O.OracleDecoder(om), O.OracleDecoder(FourBitOracle(ocfg, om.raw))
    d, prefix, drafts = decoder(hip, ocfg), ids(1, 100, ocfg.vocab), ids(2, 5, ocfg.vocab)
    for x in (f16, q4, d):
        x.observe(prefix)
    for rows in (lambda x: x.next_logits()[None], lambda x: np.asarray(x.batched_logits(drafts))):
        want, plain, got = (rows(x).astype(np.float64) for x in (q4, f16, d))
        change = np.linalg.norm(want - plain)
        assert np.linalg.norm(got - want) <= 0.5 * change
        assert np.linalg.norm(got - plain) >= 0.5 * change  # the cache really is in 4 bits


@pytest.mark.parametrize("shape", sorted(SHAPES))
def test_tree_verify_commit_and_rollback(hip, shape):
    ocfg = oracle_cfg(**SHAPES[shape])
    d, V = decoder(hip, ocfg), ocfg.vocab
    prefix = ids(3, 200, V)
    d.observe(prefix)
    chain = [prefix[-1]] + ids(4, 6, V)
    # a linear tree is the batched pass
    lin = d.batched_logits(chain[1:])
    d.rollback_to(200)
    tree = (chain, [0, 0, 1, 2, 3, 4, 5])
    tl, hidden = d.tree_logits_keep_kv(tree)
    assert np.array_equal(lin, tl) and np.isfinite(hidden).all()
    d.rollback_to(200)
    # a branching tree: the accepted rows move, the others go
    toks, pars = [prefix[-1]] + ids(5, 39, V), [0] + [max(0, (i - 1) // 3) for i in range(1, 40)]
    d.tree_logits_keep_kv((toks, pars))
    path = [0, 2, 8, 26]
    before = [kv(d, ocfg, l, 40, 199) for l in range(2)]
    d.commit_tree_path((toks, pars), path)
    assert d.cache_len() == 199 + len(path) and d.history() == prefix + [toks[i] for i in path[1:]]
    for l in range(2):
        for x, y in zip(before[l], kv(d, ocfg, l, len(path), 199)):
            assert np.array_equal(x[path], y)
    # and decoding goes on as on a fresh decoder over the same tokens, up to the fp16 path's own differences in rows per pass
    e = decoder(hip, ocfg)
    e.observe(d.history())
    d.observe([7])
    e.observe([7])
    assert rel_err(d.next_logits(), e.next_logits()) < 5e-2
    d.rollback_to(100)
    e.rollback_to(100)
    assert d.cache_len() == 100 and np.isfinite(d.next_logits()).all()


@pytest.mark.parametrize("shape", sorted(SHAPES))
@pytest.mark.parametrize("n", [129, 700, 2500])
def test_prompts_in_chunks(hip, shape, n):
    """A long prompt's chunks against the same prompt in passes of 16 rows."""
    ocfg = oracle_cfg(**SHAPES[shape])
    a, b, t = decoder(hip, ocfg), decoder(hip, ocfg, max_batch=16), ids(n, n, ocfg.vocab)
    a.observe(t)
    b.observe(t)
    la, lb = a.next_logits().astype(np.float64), b.next_logits().astype(np.float64)
    # fp16 K-quant weights above 16 rows, and the codes that they move
    assert np.linalg.norm(la - lb) <= 5e-2 * np.linalg.norm(lb)
    for x, y in zip(kv(a, ocfg, 0, n), kv(b, ocfg, 0, n)):
        # A value is a code times its group's step, and the step is 1/8 of an extreme that itself moves by 5e-4: most values of a
        # group whose step moved differ, by up to 8 * 5e-4 steps.  Another code is a whole step: about 8 * 2 * 5e-4 of the values
        # lie that close to a border.
        x, y = (t.astype(np.float64).reshape(n, ocfg.n_kv_heads, -1, 32) for t in (x, y))
        step = np.maximum(np.abs(x).max(-1, keepdims=True), np.abs(y).max(-1, keepdims=True)) / 8
        assert np.mean(np.abs(x - y) > 0.5 * step) < 0.05


def test_acceptance_entry_points_run_over_the_4_bit_cache(hip):
    ocfg = oracle_cfg(**SHAPES["llama"])
    d, V = decoder(hip, ocfg), ocfg.vocab
    prefix = ids(6, 64, V)
    d.observe(prefix)
    g = []
    for _ in range(4):
        g.append(int(np.argmax(d.next_logits())))
        d.observe([g[-1]])
    d.rollback_to(64)
    commits, n = d.verify_greedy_linear(g)
    am = d.last_argmax(5)
    assert commits[:n] == g[:n] and commits[n] == int(am[n])
    d.rollback_to(64)
    path, bonus, _ = d.verify_greedy_tree(([prefix[-1]] + g, [0, 0, 1, 2, 3]))
    assert len(path) == n + 1
    d.rollback_to(64)
    row0 = d.tree_logits(([prefix[-1]] + g, [0, 0, 1, 2, 3]))[0]
    assert np.array_equal(row0, d.next_logits())  # the one-token pass's row
    fin, mids = d.last_hidden_states_multi([0, 1])
    assert np.isfinite(fin).all() and all(np.isfinite(m).all() for m in mids)


def test_prime_synthetic_rows(hip):
    ocfg = oracle_cfg(**SHAPES["llama"])
    a, b, t = decoder(hip, ocfg), decoder(hip, ocfg, q4=False), ids(9, 300, ocfg.vocab)
    a.prime_synthetic(t, 77)
    b.prime_synthetic(t, 77)
    for l in range(2):
        for x, y in zip(kv(a, ocfg, l, 300), kv(b, ocfg, l, 300)):
            assert np.array_equal(x, _kvq.store(y.astype(np.float64)))
    assert np.isfinite(a.next_logits()).all()


def test_format_can_change_while_empty(hip):
    ocfg = oracle_cfg(**SHAPES["llama"])
    a, b, t = decoder(hip, ocfg), decoder(hip, ocfg, q4=False), ids(10, 40, ocfg.vocab)
    a.observe(t)
    with pytest.raises(hip.ArgError):
        a.set_kv_format(hip.KV_F16)
    four = a.next_logits()
    a.reset()
    with pytest.raises(hip.UnsupportedMethod):
        a.set_kv_format(7)
    a.set_kv_format(hip.KV_F16)
    a.observe(t)
    b.observe(t)
    assert np.array_equal(a.next_logits(), b.next_logits())
    a.reset()
    a.set_kv_format(hip.KV_Q4)
    a.observe(t)
    assert np.array_equal(a.next_logits(), four)


# ---- sampling on the decoder -------------------------------------------------------
FILTERS = [dict(), dict(temperature=0.7, top_k=40, top_p=0.95), dict(temperature=0.3, top_p=0.9), dict(min_p=0.2), dict(temperature=0.0)]


@pytest.mark.parametrize("q4", [False, True])
def test_sample_next_and_rows(hip, q4):
    ocfg = oracle_cfg(**SHAPES["llama"])
    d, V, rng = decoder(hip, ocfg, q4), ocfg.vocab, np.random.default_rng(0)
    d.observe(ids(11, 50, V))
    row = d.next_logits()
    for kw in FILTERS:
        u = float(np.float32(rng.random()))
        assert d.sample_next(u, **kw) == _kvq.sample(row, u, **dict(dict(temperature=1.0), **kw))[0]
    rows = d.batched_logits(ids(12, 4, V))
    for kw in FILTERS:
        u = rng.random(5).astype(np.float32)
        want = [_kvq.sample(r, x, **dict(dict(temperature=1.0), **kw))[0] for r, x in zip(rows, u)]
        assert d.sample_rows(u, **kw) == want
        assert d.sample_rows(u[:2], **kw) == want[:2]
    assert d.sample_rows([]) == []
    with pytest.raises(hip.ArgError):
        d.sample_rows(np.zeros(6))
    for kw in (dict(temperature=-1.0), dict(top_p=1.5), dict(top_k=-3), dict(min_p=float("nan"))):
        with pytest.raises(hip.SamplingError):
            d.sample_next(0.5, **kw)
        with pytest.raises(hip.SamplingError):
            d.sample_rows([0.5], **kw)
    # the row of a verify pass without drafts is the next-token row
    d.rollback_to(50)
    d.verify_greedy_linear([])
    assert d.sample_rows([0.4]) == [_kvq.sample(d.next_logits(), 0.4, 1.0)[0]]
    with pytest.raises(hip.SamplingError):
        decoder(hip, ocfg, q4).sample_next(0.5)


def test_sampled_decoding_over_a_4_bit_cache(hip):
    """Append, attend and sample together, as a sampled decoding loop and a speculative one use them."""
    ocfg = oracle_cfg(**SHAPES["qwen"])
    d, e, V = decoder(hip, ocfg), decoder(hip, ocfg), ocfg.vocab
    rng = np.random.default_rng(3)
    prompt = ids(13, 333, V)
    d.observe(prompt)
    e.observe(prompt)
    for _ in range(12):
        u = float(np.float32(rng.random()))
        tok = d.sample_next(u, temperature=0.8, top_k=50, top_p=0.9)
        assert tok == _kvq.sample(e.next_logits(), u, 0.8, top_k=50, top_p=0.9)[0]
        d.observe([tok])
        e.observe([tok])
    assert d.history() == e.history()
    # draft rows from the sampler, in device memory, verified against the target by rejection sampling
    k = 3
    s = hip.HipSampler(V, k)
    x, u = dev(rng.standard_normal((k, V)).astype(np.float32) * 2), dev(rng.random(k).astype(np.float32))
    tok, dq = zeros(k, np.int32), zeros((k, V))
    s.sample(ptr(x), k, ptr(u), ptr(tok), temperature=0.9, top_p=0.8, probs=ptr(dq))
    drafts, q, uni = tok.get().tolist(), dq.get(), rng.random(2 * k + 2).astype(np.float32)
    assert all(q[i, t] > 0 for i, t in enumerate(drafts))
    n0 = d.history_len()
    a = d.verify_rejection_linear_device(drafts, ptr(dq), uni, 1.0)
    d.rollback_to(n0)
    b = d.verify_rejection_linear(drafts, q, uni, 1.0)
    assert a == b


@pytest.mark.parametrize("q4", [False, True])
def test_a_verify_pass_without_drafts_is_the_last_pass(hip, q4):
    """batched_logits of no drafts gives one row, the next token's: that row is what sample_rows and last_argmax then see,
    not the first of the pass before."""
    ocfg = oracle_cfg(**SHAPES["llama"])
    d, V = decoder(hip, ocfg, q4), ocfg.vocab
    d.observe(ids(14, 50, V))
    rows = d.batched_logits(ids(15, 4, V))
    us = [0.05, 0.35, 0.65, 0.95]
    want, stale = ([_kvq.sample(rows[i], u, 1.0)[0] for u in us] for i in (4, 0))
    assert want != stale and np.argmax(rows[0]) != np.argmax(rows[4])
    assert np.array_equal(d.batched_logits([])[0], rows[4])
    assert [d.sample_rows([u])[0] for u in us] == want
    assert int(d.last_argmax(1)[0]) == int(np.argmax(rows[4]))
    for call in (lambda: d.sample_rows([0.5, 0.5]), lambda: d.last_argmax(2)):
        with pytest.raises(hip.ArgError):
            call()


@pytest.mark.parametrize("q4", [False, True])
def test_cache_rows_out_of_range_are_refused(hip, q4):
    """Positions whose end wraps around 64 bits among them."""
    ocfg = oracle_cfg(**SHAPES["llama"])
    d = decoder(hip, ocfg, q4)
    d.observe(ids(16, 40, ocfg.vocab))
    out = np.zeros((64, ocfg.head_dim), np.uint16)
    cap = (ocfg.ctx_len + 128 + 31) // 32 * 32  # positions that the cache holds
    for pos0, n in ((cap, 1), (cap - 3, 4), (2 ** 64 - 1, 2), (2 ** 64 - 64, 64), (2 ** 63, 1), (0, cap + 1), (1, 2 ** 64 - 1)):
        with pytest.raises(hip.ArgError):
            hip._check(hip._lib.sd_read_kv_rows(d._h, 0, 0, 0, pos0, n, out.ctypes.data))
    assert not out.any()
    assert d.read_kv_rows(0, 0, 0, cap - 4, 4).shape == (4, ocfg.head_dim) and d.read_kv_rows(0, 1, 0, cap, 0).size == 0


@pytest.mark.parametrize("shape", sorted(SHAPES))
@pytest.mark.parametrize("rows", [17, 33, 64, 128])
def test_many_rows_against_the_oracle_with_a_4_bit_cache(hip, shape, rows):
    """As test_logits_against_the_oracle_with_a_4_bit_cache, by the kernels that more than 16 rows take: weights in fp16 besides,
    2^-11 of each, which move a value no more than the activations do."""
    ocfg = oracle_cfg(**SHAPES[shape])
    om = O.OracleModel(ocfg)
    f16, q4 = O.OracleDecoder(om), O.OracleDecoder(FourBitOracle(ocfg, om.raw))
    d, prefix, drafts = decoder(hip, ocfg), ids(1, 90, ocfg.vocab), ids(rows, rows - 1, ocfg.vocab)
    for x in (f16, q4, d):
        x.observe(prefix)
    want, plain, got = (np.asarray(x.batched_logits(drafts)).astype(np.float64) for x in (q4, f16, d))
    change = np.linalg.norm(want - plain)
    assert np.linalg.norm(got - want) <= 0.5 * change
    assert np.linalg.norm(got - plain) >= 0.5 * change
