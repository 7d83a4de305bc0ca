"""Refusals of the pool's and the sampler's handles that need no GPU, and the formula of the tests' oracle."""
import ctypes

import numpy as np
import pytest

import _kvq


def test_pool_config_refusals(hip):
    ok = dict(n_layers=1, n_heads=8, n_kv_heads=2, head_dim=64, n_pages=4, page_tokens=64, max_pos=128)
    for bad, err in ((dict(n_layers=0), hip.ArgError), (dict(n_heads=0), hip.ArgError), (dict(n_kv_heads=3), hip.ArgError),
                     (dict(n_pages=-1), hip.ArgError), (dict(max_pos=0), hip.ArgError), (dict(max_pos=1 << 25), hip.ArgError),
                     (dict(head_dim=96), hip.UnsupportedMethod), (dict(page_tokens=48), hip.UnsupportedMethod),
                     (dict(page_tokens=16), hip.UnsupportedMethod), (dict(rope_theta=0.0), hip.ArgError),
                     (dict(rope_theta=float("nan")), hip.ArgError), (dict(n_heads=8192), hip.UnsupportedMethod),
                     (dict(n_pages=2 ** 31 - 1, n_layers=1000), hip.ArgError)):
        with pytest.raises(err):
            hip.HipKvPool(**dict(ok, **bad))


def test_sampler_refusals(hip):
    for bad, err in (((0, 1), hip.ArgError), ((100, 0), hip.ArgError), ((262145, 1), hip.UnsupportedMethod), ((10, 70000), hip.ArgError)):
        with pytest.raises(err):
            hip.HipSampler(*bad)


def test_null_handles(hip):
    lib = hip.load_library()
    rows, q, s = hip.KvRows(), hip.KvQuery(), hip.Sampling()
    assert lib.sd_kvpool_append(None, 0, ctypes.byref(rows), 1, 0, 0, 0, 0, 0, 0, 0, 0, 0) == hip.SD_ERR_ARG
    assert lib.sd_kvpool_read(None, 0, ctypes.byref(rows), 0, 0, 0) == hip.SD_ERR_ARG
    assert lib.sd_kvpool_attend(None, 0, ctypes.byref(q), 0, 0, 0) == hip.SD_ERR_ARG
    assert lib.sd_kvpool_attend_workspace(None, 1, 1, 1, 1) == 0 and lib.sd_kvpool_page_bytes(None) == 0
    assert lib.sd_sampler_run(None, 0, 0, 1, ctypes.byref(s), 0, 0, 0, 0) == hip.SD_ERR_ARG
    lib.sd_kvpool_destroy(None)
    lib.sd_sampler_destroy(None)


def test_oracle_store():
    x = np.zeros(32)
    x[:4] = [8.0, -4.0, 3.4, 0.5]  # the largest is positive: step -1, codes -8, 4, -3, and a half to even
    assert _kvq.store(x)[:4].tolist() == [8.0, -4.0, 3.0, 0.0]
    x[4] = -8.0  # both signs: step 1, +8 has no code
    assert _kvq.store(x)[:5].tolist() == [7.0, -4.0, 3.0, 0.0, -8.0]
    rng = np.random.default_rng(0)
    x = rng.standard_normal((100, 128))
    g = np.abs(x).reshape(100, 4, 32).max(-1, keepdims=True)
    # half a step, a whole one at the end opposite to -8; fp16 steps
    assert np.all(np.abs(_kvq.store(x) - x).reshape(100, 4, 32) <= g / 8 * 1.001)
    assert np.mean(np.abs(_kvq.store(x) - x).reshape(100, 4, 32) <= g / 16 * 1.001) > 0.95


def test_oracle_sample():
    x = np.log(np.array([0.1, 0.4, 0.2, 0.3]))
    assert [_kvq.sample(x, u, 1.0)[0] for u in (0.0, 0.05, 0.11, 0.49, 0.51, 0.71, 0.99)] == [0, 0, 1, 1, 2, 3, 3]
    assert np.allclose(_kvq.sample(x, 0, 1.0, top_k=2)[1], [0, 4 / 7, 0, 3 / 7])
    assert np.allclose(_kvq.sample(x, 0, 1.0, top_p=0.65)[1], [0, 4 / 7, 0, 3 / 7])
    assert np.allclose(_kvq.sample(x, 0, 1.0, top_k=3, top_p=0.7)[1], [0, 4 / 7, 0, 3 / 7])  # 0.7 of 0.9 is 0.63
    assert np.allclose(_kvq.sample(x, 0, 1.0, min_p=0.6)[1], [0, 4 / 7, 0, 3 / 7])
    assert _kvq.sample([1.0, 2.0, 2.0], 0.9, 0.0)[0] == 1
    assert _kvq.sample([1.0, np.nan], 0.5, 1.0)[0] == -1
