"""Refusals of the 8-bit pool's calls that need no GPU, and the formulas of the tests' oracle."""
import ctypes

import numpy as np
import pytest

import _kv8


def test_pool_config_refusals(hip):
    ok = dict(n_layers=1, n_heads=8, n_kv_heads=2, head_dim=64, n_pages=4, page_tokens=64, max_pos=128)
    for bad, err in ((dict(n_layers=0), hip.ArgError), (dict(n_heads=0), hip.ArgError), (dict(n_kv_heads=3), hip.ArgError),
                     (dict(n_pages=-1), hip.ArgError), (dict(max_pos=0), hip.ArgError), (dict(max_pos=1 << 25), hip.ArgError),
                     (dict(head_dim=96), hip.UnsupportedMethod), (dict(page_tokens=48), hip.UnsupportedMethod),
                     (dict(page_tokens=16), hip.UnsupportedMethod), (dict(rope_theta=0.0), hip.ArgError),
                     (dict(n_heads=8192), hip.UnsupportedMethod), (dict(n_pages=2 ** 31 - 1, n_layers=1000), hip.ArgError)):
        with pytest.raises(err):
            hip.HipKv8Pool(**dict(ok, **bad))


def test_null_handles(hip):
    lib = hip.load_library()
    r, s, q, w, sc, e = hip.KvRows(), hip.KvSeqs(), hip.KvQuery(), hip.KvWindow(), hip.KvScores(), hip.KvEvict()
    assert lib.sd_kv8_append(None, 0, ctypes.byref(s), 1, 0, 0, 0, 0, 0, 0, 0, 0, 0) == hip.SD_ERR_ARG
    assert lib.sd_kv8_read(None, 0, ctypes.byref(r), 0, 0, 0) == hip.SD_ERR_ARG
    assert lib.sd_kv8_attend(None, 0, ctypes.byref(q), ctypes.byref(w), 0, 0, 0, 0) == hip.SD_ERR_ARG
    assert lib.sd_kv8_weights(None, 0, ctypes.byref(q), ctypes.byref(w), 0, ctypes.byref(sc), 0) == hip.SD_ERR_ARG
    assert lib.sd_kv8_evict(None, 0, ctypes.byref(e), 0, 0, 0) == hip.SD_ERR_ARG
    assert lib.sd_kv8_attend_workspace(None, 1, 1, 1, 1, None) == 0 and lib.sd_kv8_evict_workspace(None, 1, 1) == 0
    assert lib.sd_kv8_page_bytes(None) == 0
    lib.sd_kv8_destroy(None)


def test_oracle_codes():
    # every finite code is its own nearest, and a half between two goes to the even one
    codes = [c / 512 if c < 8 else 2.0 ** (c // 8 - 7) * (1 + c % 8 / 8) for c in range(127)]
    assert codes[-1] == 448 and np.array_equal(_kv8.nearest8(codes), codes)
    for a in range(126):
        half, low = (codes[a] + codes[a + 1]) / 2, codes[a]
        assert _kv8.nearest8(half) == codes[a + a % 2] and _kv8.nearest8(-half) == -codes[a + a % 2]
        assert _kv8.nearest8(half - 1e-9) == low and _kv8.nearest8(half + 1e-9) == codes[a + 1]


def test_oracle_scales():
    assert _kv8.exponent([448.0, 448.1, 896.0, 0.0, 1e-9, 65504.0, 224.0]).tolist() == [0, 1, 1, -15, -15, 8, -1]
    x = np.zeros((3, 1, 64))
    x[0, 0, 0], x[1, 0, 1], x[2, 0, 2] = 448.0, 1.0, 2.0 ** -10  # the last is half the least step: to even, 0
    assert _kv8.block(x)[:, 0, :3].tolist() == [[448, 0, 0], [0, 1, 0], [0, 0, 0]]
    x[0, 0, 0] = 449.0  # the scale is 2: steps of 64 up there
    assert _kv8.block(x)[0, 0, 0] == 448
    x[1, 0, 5] = np.inf
    assert np.isnan(_kv8.block(x)[1]).all() and not np.isnan(_kv8.block(x)[0]).any()
    rng = np.random.default_rng(0)
    x = rng.standard_normal((32, 4, 128))
    assert np.all(np.abs(_kv8.block(x) - x) <= np.maximum(2.0 ** -4 * np.abs(x), 2.0 ** -10 * np.abs(x).max() / 224))
    # a row that comes alone joins what the block holds, in one scale; what is appended again replaces what was behind
    a = _kv8.append(np.zeros((0, 4, 128)), 0, x[:20])
    b = _kv8.append(a, 20, x[20:21] * 1000)
    assert len(b) == 21 and np.all(np.abs(b[:20] - a[:20]) <= np.abs(b[20]).max() / 224 * 2.0 ** -10)
    assert len(_kv8.append(b, 10, x[:1])) == 11


def test_oracle_evict():
    s = np.array([9, 1, 5, 5, np.nan, 0, 5, -1, 7], np.float32)
    assert _kv8.evict(s, 9, 5, 1, 1).tolist() == [0, 2, 3, 6, 8]
    assert _kv8.evict(s, 9, 4, 1, 1).tolist() == [0, 2, 3, 8]
    assert _kv8.evict(s, 9, 8, 0, 0).tolist() == [0, 1, 2, 3, 5, 6, 7, 8]
    assert _kv8.evict(s, 9, 2, 1, 1).tolist() == [0, 8] and _kv8.evict(s, 4, 4, 1, 1).tolist() == [0, 1, 2, 3]


def test_oracle_windows():
    v = _kv8.visible(2, 6, window=2, sinks=1)
    assert v.astype(int).tolist() == [[1, 0, 0, 1, 1, 0], [1, 0, 0, 0, 1, 1]]
    m = np.array([[1, 0], [0, 1]], bool)
    assert _kv8.visible(2, 4, mask=m).astype(int).tolist() == [[1, 1, 1, 0], [1, 1, 0, 1]]
    assert _kv8.visible(2, 4, mask=m, window=2).astype(int).tolist() == [[0, 1, 1, 0], [0, 0, 0, 1]]
