"""hyq_sample_d on the GPU against the rules in 64 bits (tests/paged_ref.py):
tokens are equal, probabilities within the rounding of the kernel's weights
(2^-46 of the largest each, vocabulary of them in a sum) and of f32."""
import ctypes

import numpy as np
import pytest

import paged_ref as R

pytestmark = pytest.mark.gpu

SETTINGS = [  # temperature, top_k, top_p, min_p
    (1.0, 0, 1.0, 0.0), (0.7, 20, 0.6, 0.0), (0.7, 1, 1.0, 0.0), (1.0, 0, 0.95, 0.0),
    (1.0, 0, 0.0, 0.0), (1.0, 0, 1.0, 0.05), (1.0, 0, 1.0, 1.0), (0.0, 5, 0.5, 0.1),
    (2.5, 500, 0.9, 0.001), (0.3, 7, 0.99, 0.2), (1e-3, 0, 0.9, 0.0), (1e6, 0, 0.5, 0.0),
    (1.0, 10 ** 9, 2.0, -1.0), (-1.0, 0, 1.0, 0.0), (1.0, -4, -0.5, 7.0), (1.0, 40000, 0.999, 0.0)]


def check(hyq, ctx, logits, u, settings):
    t, k, p, m = (np.array(x) for x in zip(*settings))
    t, p, m, u = (x.astype(np.float32) for x in (t, p, m, np.asarray(u)))
    token, prob = hyq.sample(ctx, logits, u, t, k, p, m)
    for r in range(len(logits)):
        want, pw = R.sample(logits[r], t[r], int(k[r]), p[r], m[r], u[r])
        assert token[r] == want, (r, settings[r], u[r], token[r], want)
        # the sum's rounding, up to vocab * 2^-46, is relative to at least 1
        tol = 2 * R.U + logits.shape[1] * 2.0 ** -45
        assert abs(prob[r] - pw) <= tol * max(pw, 2.0 ** -20), (r, settings[r], prob[r], pw)


@pytest.mark.parametrize("vocab", [1, 2, 3, 63, 64, 65, 1000, 1025, 4099, 20011, 120818, 128167])
def test_settings(gpu_ctx, hyq, vocab):
    r = np.random.default_rng(vocab)
    n = len(SETTINGS)
    logits = r.normal(0, 2.5, (n, vocab)).astype(np.float32)
    at = r.integers(0, vocab, (n, 20))
    np.put_along_axis(logits, at, np.take_along_axis(logits, at, 1) +
                      r.uniform(0, 9, (n, 20)).astype(np.float32), 1)
    for _ in range(2):
        check(hyq, gpu_ctx, logits, r.random(n), SETTINGS)


@pytest.mark.parametrize("u", [0.0, 0.5, 1 - 2.0 ** -24, 1.0, -3.0, np.nan])
def test_random_numbers_at_the_ends(gpu_ctx, hyq, u):
    r = np.random.default_rng(7)
    logits = r.normal(0, 3, (len(SETTINGS), 777)).astype(np.float32)
    if u != u:  # (not a number: taken as 0)
        t, k, p, m = zip(*SETTINGS)
        a = hyq.sample(gpu_ctx, logits, np.float32(np.nan), t, k, p, m)
        b = hyq.sample(gpu_ctx, logits, np.float32(0), t, k, p, m)
        assert np.array_equal(a[0], b[0])
        return
    check(hyq, gpu_ctx, logits, [u] * len(SETTINGS), SETTINGS)


@pytest.mark.parametrize("vocab", [5, 300, 70001])
@pytest.mark.parametrize("step", [1.0, 0.25])
def test_ties(gpu_ctx, hyq, vocab, step):
    """Few distinct values: cuts fall among equal ones, the lower index first.
    (Sums of weights that meet a border exactly would be decided by rounding:
    the distinct weights here are irrational.)"""
    r = np.random.default_rng(vocab)
    n = len(SETTINGS)
    logits = (np.round(r.normal(0, 1, (n, vocab)) / step) * step).astype(np.float32)
    check(hyq, gpu_ctx, logits, r.random(n), SETTINGS)
    settings = [(1.0, int(k), 1.0, 0.0) for k in r.integers(1, vocab + 2, n)]
    check(hyq, gpu_ctx, logits, r.random(n), settings)
    settings = [(0.9, int(k), float(p), 0.0) for k, p in zip(r.integers(1, vocab + 2, n),
                                                            r.random(n))]
    check(hyq, gpu_ctx, logits, r.random(n), settings)


@pytest.mark.parametrize("vocab", [4, 1024, 99991])
def test_all_equal(gpu_ctx, hyq, vocab):
    """Equal weights are exact in both: borders may be met exactly."""
    logits = np.full((6, vocab), -3.25, np.float32)
    settings = [(1.0, 0, 0.5, 0.0), (1.0, vocab // 2, 1.0, 0.0), (1.0, vocab // 2, 0.5, 0.0),
                (1.0, 0, 1.0, 1.0), (1.0, 3, 0.25, 0.0), (0.0, 0, 1.0, 0.0)]
    for u in (0.0, 0.25, 0.5, 0.75):
        check(hyq, gpu_ctx, logits, [u] * 6, settings)


def test_infinities_and_nans(gpu_ctx, hyq):
    """Masked logits (-inf, the type's lowest value) and NaNs are never taken;
    plus infinity takes all; a row of nothing gives -1."""
    r = np.random.default_rng(3)
    n, vocab = len(SETTINGS), 2500
    base = r.normal(0, 2, (n, vocab)).astype(np.float32)
    for fill in (-np.inf, np.nan, np.finfo(np.float32).min):
        x = base.copy()
        x[r.random(x.shape) < 0.7] = fill
        check(hyq, gpu_ctx, x, r.random(n), SETTINGS)
        x[:] = fill
        x[:, 1234] = -55.0
        check(hyq, gpu_ctx, x, r.random(n), SETTINGS)
        x[:, 77] = np.inf
        x[:, 2000] = np.inf
        check(hyq, gpu_ctx, x, r.random(n), SETTINGS)
    for fill in (-np.inf, np.nan):
        token, prob = hyq.sample(gpu_ctx, np.full((3, 500), fill, np.float32), 0.5, [0, 1, 1],
                                 [0, 5, 0], 0.9)
        assert token.tolist() == [-1] * 3 and prob.tolist() == [0] * 3
    x = np.full((2, 300), np.nan, np.float32)
    x[:, 7] = -0.0
    x[:, 200] = 0.0
    token, _ = hyq.sample(gpu_ctx, x, 0.0, [0.0, 1.0], 1)
    assert token.tolist() == [7, 7]


def test_extreme_sizes(gpu_ctx, hyq):
    """Logits whose differences pass f32's range, and temperatures at its ends
    (below 2^-100 only equal maxima are left)."""
    r = np.random.default_rng(8)
    n, vocab = 8, 900
    x = (r.uniform(-1, 1, (n, vocab)) * 3.3e38).astype(np.float32)
    u = r.random(n)
    check(hyq, gpu_ctx, x, u, [(1e38, 0, 1.0, 0.0), (3e38, 50, 0.7, 0.0), (2e37, 0, 0.9, 0.0),
                               (3e38, 0, 1.0, 0.3), (1e38, 300, 0.99, 0.0), (1.0, 0, 1.0, 0.0),
                               (np.inf, 0, 1.0, 0.0), (np.inf, 0, 0.5, 0.0)])
    x = r.normal(0, 2, (n, vocab)).astype(np.float32)
    x[:, [5, 300, 301, 888]] = 20.0
    tiny = [(t, k, p, 0.0) for t, k, p in ((1e-38, 0, 1.0), (1e-45, 3, 1.0), (1e-31, 0, 0.6),
                                           (1e-30, 0, 1.0), (2e-29, 2, 0.9), (1e-38, 2000, 0.5),
                                           (1e-12, 0, 0.9), (1e-38, 1, 1.0))]
    check(hyq, gpu_ctx, x, u, tiny)


def test_more_rows_than_splits_serve(gpu_ctx, hyq):
    """Rows by a workgroup each (more than half of 512), by two, and on both sides
    of those whose splits find their cuts by themselves."""
    r = np.random.default_rng(9)
    for rows, vocab in ((600, 1500), (257, 4100), (256, 4100), (17, 9000), (16, 9000)):
        x = r.normal(0, 2.5, (rows, vocab)).astype(np.float32)
        check(hyq, gpu_ctx, x, r.random(rows), [SETTINGS[i % len(SETTINGS)] for i in range(rows)])


@pytest.mark.parametrize("vocab", [2049, 128167])
def test_where_lists_end(gpu_ctx, hyq, vocab):
    """A top-k around the largest whose members are listed whole, and cuts by
    top-k far behind the one by top-p."""
    r = np.random.default_rng(10)
    settings = [(1.0, k, p, 0.0) for k in (63, 64, 65, 1023, 1024, 1025, 2047, 2048, 30000)
                for p in (1.0, 0.3, 0.97)]
    n = len(settings)
    x = r.normal(0, 2.5, (n, vocab)).astype(np.float32)
    check(hyq, gpu_ctx, x, r.random(n), settings)
    flat = r.uniform(0, 0.02, (n, vocab)).astype(np.float32)  # (all in two bins)
    check(hyq, gpu_ctx, flat, r.random(n), settings)


def test_without_probabilities_and_the_argmax(gpu_ctx, hyq):
    """prob may be null; temperature 0 is hyq_argmax_d's token."""
    r = np.random.default_rng(5)
    L, ctx = hyq.lib(), gpu_ctx
    x = r.normal(0, 1, (3, 120818)).astype(np.float32)
    x[1, [50, 90000]] = 30.0
    d = ctx.array(x)
    f = [ctx.array(np.full(3, v, t)) for v, t in ((0, np.float32), (0, np.int32), (1, np.float32),
                                                 (0, np.float32), (0.3, np.float32))]
    need = L.hyq_sample_scratch_bytes(3, x.shape[1])
    scratch, token = ctx.array(np.full(need + 16, 0xFF, np.uint8)), ctx.empty(3, np.int32)
    hyq.check(L.hyq_sample_d(ctx.handle, d.ptr, 3, x.shape[1], *[a.ptr for a in f], scratch.ptr,
                             need, token.ptr, None))
    one, s = ctx.empty(1, np.int32), ctx.empty(128, np.float32)
    for row in range(3):
        hyq.check(L.hyq_argmax_d(ctx.handle, d.ptr + row * x.shape[1] * 4, x.shape[1], s.ptr,
                                 one.ptr))
        assert one.numpy()[0] == token.numpy()[row] == np.argmax(x[row])


def test_frequencies(gpu_ctx, hyq):
    """Tokens over a grid of random numbers come as often as their weights say:
    u = (i + 1/2) / n draws token t between floor and ceil of n p_t times."""
    r = np.random.default_rng(6)
    n = 400
    x = np.broadcast_to(r.normal(0, 2, 50).astype(np.float32), (n, 50))
    token, prob = hyq.sample(gpu_ctx, x, (np.arange(n) + 0.5) / n)
    p = np.exp(x[0].astype(np.float64))
    p /= p.sum()
    count = np.bincount(token, minlength=50)
    assert np.all(np.abs(count - n * p) <= 1 + 1e-3)
    assert np.all(np.diff(token) >= 0)
    assert np.allclose(prob, p[token], rtol=4 * R.U, atol=0)
