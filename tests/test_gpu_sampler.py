"""Filtered sampling (sd_sampler_*) against a 64-bit restatement: tokens equal, distributions to an fp32 rounding."""
import ctypes

import numpy as np
import pytest

import _kvq
from _devmem import Dev, Graph, Stream, dev, full, ptr, runtime, zeros

pytestmark = pytest.mark.gpu


def draw(hip, x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, probs=True, ld=0, sampler=None, V=None):
    x = np.ascontiguousarray(x, np.float32)
    rows, V = x.shape[0], V or x.shape[1]
    s = sampler or hip.HipSampler(V, rows)
    dx, du = dev(x), dev(np.asarray(u, np.float32))
    tok = full(rows, -7, np.int32)
    pr = full((rows, V), 5.0) if probs else None
    s.sample(ptr(dx), rows, ptr(du), ptr(tok), temperature, top_k, top_p, min_p, probs=ptr(pr), ld=ld)
    return tok.get(), pr.get() if probs else None


def check(hip, x, u, **kw):
    tok, pr = draw(hip, x, u, **kw)
    args = {k: kw.get(k, d) for k, d in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0))}
    for r in range(len(x)):
        want, p = _kvq.sample(x[r], u[r], **args)
        assert tok[r] == want, (r, tok[r], want, args)
        # an fp32 rounding of a value known to 1e-10
        assert np.all(np.abs(pr[r] - p) <= 2.0 ** -24 * p * 1.01 + 2.0 ** -150), (r, args)
        assert np.array_equal(pr[r] > 0, p.astype(np.float32) > 0) or np.abs(p[(pr[r] > 0) != (p > 0)]).max() < 2.0 ** -149


FILTERS = [dict(), dict(top_k=1), dict(top_k=40), dict(top_k=700), dict(top_p=0.9), dict(top_p=0.3), dict(min_p=0.05), dict(top_k=50, top_p=0.8),
           dict(top_k=5000, top_p=0.99, min_p=0.001), dict(top_p=0.0), dict(top_p=0.999, min_p=1.0), dict(temperature=0.0),
           dict(temperature=0.1, top_p=0.9), dict(temperature=8.0, top_p=0.95), dict(temperature=8.0, top_k=4000),
           dict(temperature=30.0), dict(temperature=1e-30, top_k=3), dict(temperature=1e30, top_p=0.5)]


@pytest.mark.parametrize("V", [1, 2, 63, 1000, 8191, 8193, 32000])
@pytest.mark.parametrize("f", range(len(FILTERS)))
def test_filters(hip, V, f):
    rng = np.random.default_rng(V * 100 + f)
    x = rng.standard_normal((4, V)) * np.array([[0.2], [1.0], [2.5], [6.0]])
    if V > 20:
        x[:, 5::17] = -np.inf
    check(hip, x.astype(np.float32), rng.random(4), **FILTERS[f])


@pytest.mark.parametrize("V", [128256, 152064, 262144])
@pytest.mark.parametrize("f", [0, 2, 3, 4, 6, 7, 8, 13])
def test_filters_large_vocabularies(hip, V, f):
    rng = np.random.default_rng(V + f)
    x = rng.standard_normal((2, V)) * np.array([[1.0], [2.5]])
    x[:, 1::1009] += 3.0
    check(hip, x.astype(np.float32), rng.random(2), **FILTERS[f])


@pytest.mark.parametrize("f", range(len(FILTERS)))
def test_ties(hip, f):
    """Few distinct values, so that every bound falls inside a run of equal ones; uniforms on exact borders; all equal."""
    rng = np.random.default_rng(f)
    V = 20011
    x = rng.integers(-3, 4, (4, V)).astype(np.float32)
    x[1] = 0.0
    x[2, ::2], x[2, 1::2] = -0.0, 0.0
    x[3, 7:] = -np.inf
    check(hip, x, [0.5, 0.25, 0.75, 0.0], **FILTERS[f])


@pytest.mark.parametrize("V", [1, 9000, 152064])
@pytest.mark.parametrize("min_p", [1.0, 0.5, 1e-3, 1e-9, 1e-30])
def test_min_p_alone(hip, V, min_p):
    """From the ties of the maximum to every entry kept: flat, ordinary and steep rows, and one of equal values."""
    rng = np.random.default_rng(V)
    x = (rng.standard_normal((4, V)) * np.array([[0.01], [1.0], [4.0], [0.0]])).astype(np.float32)
    for T in (0.3, 5.0):
        check(hip, x, rng.random(4), min_p=min_p, temperature=T)


def test_two_near_values(hip):
    """A bin full of values that differ in their last bits only."""
    rng = np.random.default_rng(1)
    x = (np.float32(3.0) + rng.integers(0, 60, (2, 30000)).astype(np.float32) * np.float32(2.0 ** -22)).astype(np.float32)
    for kw in (dict(top_k=9000), dict(top_p=0.37), dict(top_k=25000, top_p=0.5)):
        check(hip, x, rng.random(2), **kw)


def test_uniform_ends(hip):
    x = np.zeros((4, 1000), np.float32)
    u = np.array([0.0, np.nextafter(np.float32(1), np.float32(0)), 0.5, 0.999], np.float32)
    check(hip, x, u)
    check(hip, x, u, top_p=0.5)
    tok, _ = draw(hip, x, np.array([1.0, 2.0, -1.0, np.nan], np.float32))  # outside [0, 1): still a token
    assert ((tok >= 0) & (tok < 1000)).all()


def test_rows_without_a_distribution(hip):
    rng = np.random.default_rng(2)
    x = rng.standard_normal((6, 9000)).astype(np.float32)
    x[0, 8999] = np.nan
    x[1, 17] = np.inf
    x[2] = -np.inf
    x[3, :8500] = -np.inf
    x[4, 1:] = -np.inf
    for kw in (dict(), dict(top_k=10), dict(top_p=0.9), dict(min_p=0.1), dict(temperature=0.0)):
        check(hip, x, rng.random(6), **kw)


def test_stride_fewer_rows_and_untouched_outputs(hip):
    rng = np.random.default_rng(3)
    V, ld = 5000, 5013
    wide = rng.standard_normal((5, ld)).astype(np.float32)
    u = rng.random(5)
    s = hip.HipSampler(V, 9)
    tok, pr = draw(hip, wide, u, top_k=20, ld=ld, sampler=s, V=V)
    for r in range(5):
        want, p = _kvq.sample(wide[r, :V], u[r], 1.0, top_k=20)
        assert tok[r] == want and np.all(np.abs(pr[r] - p) <= 2.0 ** -24 * p * 1.01)
    # a smaller call after a larger one on the same handle
    tok, _ = draw(hip, wide[:1], u[:1], top_p=0.5, ld=ld, sampler=s, V=V, probs=False)
    assert tok[0] == _kvq.sample(wide[0, :V], u[0], 1.0, top_p=0.5)[0]


def test_distribution_of_draws(hip):
    """The draws over a grid of uniforms have the distribution's frequencies."""
    rng = np.random.default_rng(4)
    x = np.tile(rng.standard_normal(50).astype(np.float32) * 2, (4096, 1))
    u = (np.arange(4096) + 0.5) / 4096
    tok, pr = draw(hip, x, u, top_p=0.95)
    freq = np.bincount(tok, minlength=50) / 4096
    assert np.all(np.abs(freq - pr[0]) <= 1.0 / 4096 + 1e-6)  # a grid counts each interval to within one


@pytest.mark.parametrize("kw", [dict(top_k=40, top_p=0.9), dict(), dict(top_p=0.9)])
def test_captured_and_replayed(hip, kw):
    rng = np.random.default_rng(5)
    V, rows = 33333, 3
    s = hip.HipSampler(V, rows)
    x, u, tok, pr = zeros((rows, V)), zeros(rows), zeros(rows, np.int32), zeros((rows, V))

    def step(st):
        s.sample(ptr(x), rows, ptr(u), ptr(tok), probs=ptr(pr), stream=st, **kw)
    graph, side = Graph(step), Stream()
    for i in range(4):
        a, b = (rng.standard_normal((rows, V)) * 2).astype(np.float32), rng.random(rows).astype(np.float32)
        x.put(a)
        u.put(b)
        graph.launch()
        got, dist = tok.get(), pr.get()
        for r in range(rows):
            want, p = _kvq.sample(a[r], b[r], 1.0, **kw)
            assert got[r] == want and np.all(np.abs(dist[r] - p) <= 2.0 ** -24 * p * 1.01 + 2.0 ** -150)
        tok.put(np.full(rows, -9))
        step(side.handle)
        side.wait()
        assert np.array_equal(tok.get(), got)


def test_refusals(hip):
    s = hip.HipSampler(100, 4)
    buf = zeros(4096)
    b = ptr(buf)
    for kw in (dict(temperature=-1.0), dict(temperature=float("nan")), dict(temperature=float("inf")), dict(top_k=-1),
               dict(top_p=-0.1), dict(top_p=1.1), dict(top_p=float("nan")), dict(min_p=-0.1), dict(min_p=2.0)):
        with pytest.raises(hip.SamplingError):
            s.sample(b, 1, b, b, **kw)
    for args, kw in (((0, 1, b, b), {}), ((b, 1, 0, b), {}), ((b, 1, b, 0), {}), ((b, 5, b, b), {}), ((b, 1, b, b), dict(ld=99)),
                     ((b, 1 << 20, b, b), {}), ((b, 1, b, b), dict(probs=b))):
        with pytest.raises(hip.ArgError):
            s.sample(*args, **kw)
    s.sample(b, 0, b, b)
    s.close()
    with pytest.raises(hip.ArgError):
        s.sample(b, 1, b, b)


def far_rows(V, first, rest=-200.0):
    """A row whose slices but the last lie `first` below its maximum (8192 entries each), the last one's single 0 apart."""
    x = np.full((1, V), rest, np.float32)
    for s, at in enumerate(first):
        x[0, 8192 * s:8192 * (s + 1)] = at
    x[0, V - 5] = 0.0
    return x


@pytest.mark.parametrize("kw", [dict(), dict(min_p=1e-30), dict(top_k=9000), dict(top_p=1 - 2.0 ** -24), dict(temperature=0.05),
                                dict(temperature=0.05, min_p=1e-30), dict(top_k=40)])
@pytest.mark.parametrize("first", [[-32.0], [-31.5], [-31.0, -31.9], [-36.0, -31.9], [-40.0], [-40.0, -31.2, -38.5], [-300.0, -31.4]])
def test_draws_from_slices_far_below_the_maximum(hip, first, kw):
    """Small uniforms lead to slices none of whose entries weighs 2^-45 of the row's maximum: still an entry that is kept, and the
    rule's own but for what sums lose.  Each of V weights is rounded to 2^-44 of the row's maximum, half a unit: V 2^-45 of the
    sum, which is at least 1; where histograms add them up, to 2^-36 of the slice's maximum: V 2^-37.  The weights themselves
    are within 1e-11."""
    T = kw.get("temperature", 1.0)
    x = far_rows(8192 * (len(first) + 1), [a * T for a in first], -200.0 * T)
    u = np.array([0.0, 1e-14, 1e-12, 1e-11, 5e-11, 0.25], np.float32)
    tol = x.shape[1] * 2.0 ** (-45 if set(kw) <= {"temperature"} or kw.get("top_k") == 40 else -37) + 1e-11
    tok, pr = draw(hip, np.repeat(x, len(u), 0), u, **kw)
    for r in range(len(u)):
        p = _kvq.sample(x[0], u[r], **dict(dict(temperature=1.0), **kw))[1]
        c = np.cumsum(p)
        assert 0 <= tok[r] < x.shape[1], (r, tok[r])
        assert p[tok[r]] > 0 and pr[r, tok[r]] > 0
        assert c[tok[r]] - p[tok[r]] <= u[r] + tol and c[tok[r]] >= u[r] - tol, (r, tok[r])


@pytest.mark.parametrize("top_k", [11, 40, 256])
@pytest.mark.parametrize("spread", [0.0, 0.001, 3.0])
@pytest.mark.parametrize("slices", [2, 5])
def test_top_k_reaches_slices_far_below(hip, top_k, spread, slices):
    """Fewer finite entries near the maximum than top-k: the rest come, in order, from slices more than 32 nats below."""
    rng = np.random.default_rng(top_k + slices)
    x = np.full((2, 8192 * slices), -np.inf, np.float32)
    x[:, 100:110] = rng.standard_normal((2, 10))
    for s in range(1, slices):
        x[:, 8192 * s + 7:8192 * s + 307] = -40.0 - s + spread * rng.random((2, 300))
    check(hip, x, [0.3, 0.9], top_k=top_k)
    check(hip, x, [0.3, 0.9], top_k=top_k, temperature=0.5)
    check(hip, x, [0.3, 0.9], top_k=top_k, top_p=0.9)


@pytest.mark.parametrize("top_k", [1, 40, 256])
@pytest.mark.parametrize("V", [20000, 128256])
def test_top_k_of_sharp_rows(hip, top_k, V):
    """At low temperatures nearly all of a row, and all but a few of its top-k, lie more than 32 nats below its maximum."""
    rng = np.random.default_rng(top_k + V)
    x = (rng.standard_normal((3, V)) * 2).astype(np.float32)
    x[0, 17] = x[1, V - 1] = 30.0
    x[2, 9000:9300] = 7.0  # more than a slice lists in one bin
    for T in (0.05, 0.2):
        check(hip, x, rng.random(3), top_k=top_k, temperature=T)


def test_a_refused_handle_leaves_no_error_behind(hip):
    """A handle that cannot be made says so once: the runtime's last error is clear and the next launch is taken."""
    rt = runtime()
    x = np.random.default_rng(6).standard_normal((1, 500)).astype(np.float32)
    s = hip.HipSampler(500, 1)

    def refused(make):
        with pytest.raises(hip.BackendError):
            make()
        tok, _ = draw(hip, x, [0.5], sampler=s)
        assert tok[0] == _kvq.sample(x[0], 0.5, 1.0)[0]
        assert rt.hipGetLastError() == 0

    refused(lambda: hip.HipSampler(500, 1, device=9999))
    refused(lambda: hip.HipKvPool(n_layers=1, n_heads=1, n_kv_heads=1, head_dim=64, n_pages=1, device=9999))
    # memory that is not there: 60 GB where 30 are left
    free, total = ctypes.c_size_t(), ctypes.c_size_t()
    assert rt.hipMemGetInfo(ctypes.byref(free), ctypes.byref(total)) == 0
    if free.value < 80 << 30:
        pytest.skip("less than 80 GiB of GPU memory free")
    held = Dev(free.value - (30 << 30), np.uint8)
    refused(lambda: hip.HipSampler(262144, 65535))
    del held


def test_overlapping_probabilities_are_refused(hip):
    V, ld, rows = 100, 220, 3
    rng = np.random.default_rng(8)
    x = rng.standard_normal((rows, ld)).astype(np.float32)
    s = hip.HipSampler(V, rows)
    d, u, tok = dev(x), dev(np.full(rows, 0.5, np.float32)), zeros(rows, np.int32)
    end = 4 * ((rows - 1) * ld + V)
    for at in (4, 4 * (V - 1), -4 * (rows * V - 1), end - 4, 4 * V):
        with pytest.raises(hip.ArgError):
            s.sample(ptr(d), rows, ptr(u), ptr(tok), probs=ptr(d) + at, ld=ld)
    # one row's fits behind it, before the next one's logits
    s.sample(ptr(d), 1, ptr(u), ptr(tok), probs=ptr(d) + 4 * V, ld=ld)
    got = d.get()
    want, p = _kvq.sample(x[0, :V], 0.5, 1.0)
    assert tok.get()[0] == want and np.all(np.abs(got[0, V:2 * V] - p) <= 2.0 ** -24 * p * 1.01)
    got[0, V:2 * V] = x[0, V:2 * V]
    assert np.array_equal(got, x)
