"""Decoders whose cache is held in 8 bits (KV_Q8): the decoder's entry points run over it, against the fp16 decoder, the
oracle with an 8-bit cache, and themselves."""
import numpy as np
import pytest

import _kv8
import _kvq
import oracle as O
from _models import MIX_IDS, hip_cfg, oracle_cfg, rel_err

pytestmark = pytest.mark.gpu

SHAPES = {
    "llama": dict(n_layers=2, n_heads=8, n_kv_heads=2, vocab=2048, ctx_len=2600),
    "mha": dict(n_layers=2, vocab=2048, ctx_len=2600),
    "qwen": dict(arch="qwen2", n_layers=2, hidden=1024, n_heads=8, n_kv_heads=1, head_dim=128, vocab=2048, ctx_len=2600, mix="q8_0"),
}


def decoder(hip, ocfg, q8=True, max_batch=128):
    cfg = hip_cfg(hip, ocfg, max_batch)
    cfg.kv_format = hip.KV_Q8 if q8 else hip.KV_F16
    d = hip.HipQuantDecoder(cfg)
    d.synthesize(MIX_IDS[ocfg.mix], ocfg.seed, ocfg.weight_std)
    return d


def ids(seed, n, vocab):
    return [int(v) for v in np.random.default_rng(seed).integers(0, vocab, n)]


def kv(d, ocfg, layer, n, pos0=0):
    return [np.stack([d.read_kv_rows(layer, w, h, pos0, n).view(np.float16) for h in range(ocfg.n_kv_heads)], 1).astype(np.float64)
            for w in (0, 1)]


def most(x):
    """the largest magnitude of each row's block, which starts at a multiple of 32 of x's rows"""
    return np.concatenate([np.broadcast_to(np.abs(x[a:a + 32]).max((0, 2))[None, :, None], x[a:a + 32].shape) for a in range(0, len(x), 32)])


@pytest.mark.parametrize("shape", sorted(SHAPES))
@pytest.mark.parametrize("n", [1, 5, 16, 17, 50, 128, 300])
def test_first_layer_rows_are_the_fp16_rows_quantised(hip, shape, n):
    """The first layer's rows do not depend on the cache: each is within half a step of the fp16 decoder's."""
    ocfg = oracle_cfg(**SHAPES[shape])
    a, b, t = decoder(hip, ocfg), decoder(hip, ocfg, q8=False), ids(n, n, ocfg.vocab)
    a.observe(t)
    b.observe(t)
    for got, ref in zip(kv(a, ocfg, 0, n), kv(b, ocfg, 0, n)):
        # Half a step of an 8-bit float, 2^-4 of the value or, below the normal ones, 2^-10 of a scale that is at most 1/224 of
        # the block's largest; the fp16 row's own rounding, 2^-11 of it; and above 16 rows K slices in another order (1e-4).
        tol = np.abs(ref) * (2.0 ** -4 + 2.0 ** -10) + most(ref) * (2.0 ** -10 / 224 + 1e-4) + 2.0 ** -25
        assert np.all(np.abs(got - ref) <= tol), float(np.max(np.abs(got - ref) - tol))
        if n > 16:
            assert np.mean(got != ref) > 0.5  # it is in 8 bits


class EightBitOracle(O.OracleModel):
    """The oracle with its cache in 8 bits; calls start at multiples of 32 positions."""

    def forward(self, *a, **k):
        def stored(x):
            x = np.asarray(x, np.float64)
            y = x.reshape(-1, self.cfg.n_kv_heads, self.cfg.head_dim)
            return _kv8.append(y[:0], 0, y).reshape(x.shape).astype(np.float32)
        plain, O.round_f16 = O.round_f16, stored
        try:
            return super().forward(*a, **k)
        finally:
            O.round_f16 = plain


@pytest.mark.parametrize("shape", sorted(SHAPES))
@pytest.mark.parametrize("rows", [1, 6, 17, 33, 64, 128])
def test_logits_against_the_oracle_with_an_8_bit_cache(hip, shape, rows):
    """fp16 activations move a value by about 5e-4 of itself, and so about one code in 60 (a step is 1/16 to 1/8 of its value)
    by a step, where quantising moves every value by 0.29 steps rms: the square root of 1/60 is below half of that.  The device
    stays within 0.6 of what the 8-bit cache itself changes (the activations' own part of the logits besides)."""
    ocfg = oracle_cfg(**SHAPES[shape])
    om = O.OracleModel(ocfg)
    f16, q8 = O.OracleDecoder(om), O.OracleDecoder(EightBitOracle(ocfg, om.raw))
    d, prefix, drafts = decoder(hip, ocfg), ids(1, 96, ocfg.vocab), ids(rows, rows, ocfg.vocab)
    for x in (f16, q8, d):
        x.observe(prefix)
        x.observe(drafts[:1])  # the row that a verify pass starts with
    rows_of = (lambda x: x.next_logits()[None]) if rows == 1 else (lambda x: np.asarray(x.batched_logits(drafts[1:])))
    want, plain, got = (rows_of(x).astype(np.float64) for x in (q8, f16, d))
    change = np.linalg.norm(want - plain)
    assert np.linalg.norm(got - want) <= 0.6 * change
    assert np.linalg.norm(got - plain) >= 0.5 * change  # the cache really is in 8 bits


@pytest.mark.parametrize("shape", sorted(SHAPES))
@pytest.mark.parametrize("at", [200, 225, 254])
def test_tree_verify_commit_and_rollback(hip, shape, at):
    ocfg = oracle_cfg(**SHAPES[shape])
    d, V = decoder(hip, ocfg), ocfg.vocab
    prefix = ids(3, at, V)
    d.observe(prefix)
    chain = [prefix[-1]] + ids(4, 6, V)
    # a linear tree is the batched pass
    lin = d.batched_logits(chain[1:])
    d.rollback_to(at)
    tl, hidden = d.tree_logits_keep_kv((chain, [0, 0, 1, 2, 3, 4, 5]))
    assert np.array_equal(lin, tl) and np.isfinite(hidden).all()
    d.rollback_to(at)
    # a branching tree: the accepted rows move, the others go
    toks, pars = [prefix[-1]] + ids(5, 39, V), [0] + [max(0, (i - 1) // 3) for i in range(1, 40)]
    d.tree_logits_keep_kv((toks, pars))
    path, P = [0, 2, 8, 26], at - 1
    b0 = P // 32 * 32
    before = [kv(d, ocfg, l, P + 40 - b0, b0) for l in range(2)]
    d.commit_tree_path((toks, pars), path)
    assert d.cache_len() == P + len(path) and d.history() == prefix + [toks[i] for i in path[1:]]
    for l in range(2):
        for x, y in zip(before[l], kv(d, ocfg, l, P + len(path) - b0, b0)):
            stay = x[:P - b0]
            assert np.array_equal(y, _kv8.append(stay, P - b0, x[[P - b0 + i for i in path]]))
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
    assert np.linalg.norm(la - lb) <= 5e-2 * np.linalg.norm(lb)
    for x, y in zip(kv(a, ocfg, 0, n), kv(b, ocfg, 0, n)):
        # values move by about 5e-4 of themselves, and so about one in 60 to the code beside: 2^-3 of it
        assert np.all(np.abs(x - y) <= np.maximum(np.abs(x), np.abs(y)) * 2.0 ** -3 + most(np.maximum(np.abs(x), np.abs(y))) * 2e-3)
        assert np.mean(x != y) < 0.1


def test_acceptance_entry_points_run_over_the_8_bit_cache(hip):
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
    u = 0.37
    assert d.sample_next(u, temperature=0.8, top_k=50) == _kvq.sample(d.next_logits(), u, 0.8, top_k=50)[0]


def test_prime_synthetic_rows(hip):
    ocfg = oracle_cfg(**SHAPES["llama"])
    a, b, t = decoder(hip, ocfg), decoder(hip, ocfg, q8=False), ids(9, 300, ocfg.vocab)
    a.prime_synthetic(t, 77)
    b.prime_synthetic(t, 77)
    for l in range(2):
        for x, y in zip(kv(a, ocfg, l, 300), kv(b, ocfg, l, 300)):
            assert np.array_equal(x, _kv8.append(y[:0], 0, y))
    assert np.isfinite(a.next_logits()).all()


def test_format_can_change_while_empty(hip):
    ocfg = oracle_cfg(**SHAPES["llama"])
    a, t = decoder(hip, ocfg), ids(10, 40, ocfg.vocab)
    a.observe(t)
    for f in (hip.KV_F16, hip.KV_Q4):
        with pytest.raises(hip.ArgError):
            a.set_kv_format(f)
    got = {hip.KV_Q8: a.next_logits()}
    with pytest.raises(hip.ArgError):
        a.set_kv_format(hip.KV_Q8)  # as with the others, not while it holds something
    for f in (hip.KV_F16, hip.KV_Q4, hip.KV_Q8, hip.KV_Q4, hip.KV_F16, hip.KV_Q8):
        a.reset()
        a.set_kv_format(f)
        a.observe(t)
        row = a.next_logits()
        assert np.array_equal(got.setdefault(f, row), row)
    assert len({v.tobytes() for v in got.values()}) == 3
