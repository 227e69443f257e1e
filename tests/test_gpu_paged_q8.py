"""The paged cache's 8-bit pool on the GPU against plain 64-bit forms
(tests/paged_q8_ref.py): quantising as it is written, reading back, attention,
and the pages' bookkeeping, with any bytes and NaN scales in unused places."""
import ctypes

import numpy as np
import pytest

import paged_q8_ref as Q
import paged_ref as R

pytestmark = pytest.mark.gpu
D = R.D
HEADS = [(2, 2), (4, 2), (6, 2), (16, 4), (8, 1), (16, 1)]


def layout(hyq, b, layers=1):
    return hyq.KvLayout(hyq.KV_Q8, layers, b.kvh, D, b.pt, b.pages, b.seqs, b.width)


def attention(hyq, ctx, b, max_rows=None):
    """hyq_paged_attention_d of a batch; rows of no slot stay at -7."""
    d = {n: ctx.array(a) for n, a in dict(pool=b.bytes, table=b.table, len=b.lens, start=b.start,
                                          q=b.q).items()}
    kl = layout(hyq, b)
    most = max_rows or max(1, int(b.news.max()))
    assert hyq.lib().hyq_kv_pool_bytes(ctypes.byref(kl)) == b.bytes.nbytes
    need = hyq.lib().hyq_paged_attention_scratch_bytes(ctypes.byref(kl), b.rows, most, b.heads)
    scratch = ctx.array(np.full(need, 0xFF, np.uint8))  # (NaNs: nothing may be read unwritten)
    out = ctx.array(np.full((b.rows, b.heads, D), -7, np.float32))
    hyq.check(hyq.lib().hyq_paged_attention_d(
        ctx.handle, ctypes.byref(kl), d["pool"].ptr, 0, d["table"].ptr, d["len"].ptr,
        d["start"].ptr, b.rows, most, b.heads, d["q"].ptr, scratch.ptr, need, out.ptr))
    return out.numpy()


def check(b, got):
    want, tol = b.attention()
    for s in range(b.seqs):
        for r in range(b.start[s], b.start[s + 1]):
            err = np.abs(got[r] - want[r]).max(-1)
            assert np.all(err <= tol[r]), (
                f"slot {s} (len {b.lens[s]}, {b.news[s]} new) row {r - b.start[s]}: "
                f"{err.max():.3e} > {tol[r][err.argmax()]:.3e}")
    assert np.all(got[b.new:] == -7), "rows behind the last slot changed"


# ---- attention ----
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("pt", [16, 64, 256])
def test_decode(gpu_ctx, hyq, heads, pt):
    """One new token per slot, lengths around tiles and pages, empty slots."""
    lens = [1, 0, 15, 16, 17, 31, 33, 64, 65, 200, 300, 1]
    news = [1, 0, 1, 1, 1, 1, 1, 1, 1, 1, 0, 1]
    b = Q.BatchQ8(lens, news, *heads, pt, seed=pt + heads[0], tail=2)
    check(b, attention(hyq, gpu_ctx, b))


@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("pt", [16, 64])
def test_mixed_rows(gpu_ctx, hyq, heads, pt):
    """Decode steps, drafts on both sides of the two forms' border, and prompts
    around a block of 128 query rows, with and without earlier tokens."""
    rep = heads[0] // heads[1]
    few, block = 16 // rep, 128 // rep
    news = [1, few, few + 1, block, 0, block + 1, 2, min(2 * block + 3, 70), 33]
    lens = [90, few, few + 40, block, 50, block + 37, 300, min(2 * block + 3, 70) + 1, 33]
    b = Q.BatchQ8(lens, news, *heads, pt, seed=pt * 3 + heads[0], tail=3)
    check(b, attention(hyq, gpu_ctx, b))


def test_long_and_short(gpu_ctx, hyq):
    """One long slot cut over many workers beside short ones; one long prompt."""
    b = Q.BatchQ8([5000, 3, 17], [1, 1, 1], 8, 2, 64, seed=5)
    check(b, attention(hyq, gpu_ctx, b))
    b = Q.BatchQ8([4100], [45], 8, 2, 64, seed=6, tail=1)
    check(b, attention(hyq, gpu_ctx, b))


@pytest.mark.parametrize("news", [1, 30])
def test_slots_that_share_pages(gpu_ctx, hyq, news):
    b = Q.BatchQ8([600, 600, 480, 600, 600, 200], [news] * 6, 8, 2, 32, seed=22)
    b.table[1, :18] = b.table[0, :18]
    b.table[2, :14] = b.table[0, :14]
    b.table[4, 7:18] = b.table[3, 7:18]
    check(b, attention(hyq, gpu_ctx, b))


@pytest.mark.parametrize("news", [1, 40])
def test_scales_of_very_different_size(gpu_ctx, hyq, news):
    """Positions whose scales differ by factors of 2^30, with new largest ones on
    the way."""
    b = Q.BatchQ8([400, 333], [news] * 2, 4, 1, 16, seed=9, spread=5.0)
    b.q *= np.float32(0.05)
    check(b, attention(hyq, gpu_ctx, b))


@pytest.mark.parametrize("news", [1, 17])
def test_equal_scores(gpu_ctx, hyq, news):
    """Queries of zeros: every weight is one, and what is left are the scales' products
    (rounded twice and split to 2^-22) and sums over few positions."""
    b = Q.BatchQ8([32] * 200, [news] * 200, 4, 4, 16, seed=17, spread=0.5)
    b.q[:] = 0
    got, (want, _) = attention(hyq, gpu_ctx, b), b.attention()
    for s in range(b.seqs):
        rows = slice(b.start[s], b.start[s + 1])
        big = np.array([np.abs(b.kv(s, h)[1]).max() for h in range(4)])
        err = np.abs(got[rows] - want[rows]).max((0, 2))
        assert np.all(err <= big * ((32 + 12) * R.U + 2.0 ** -22)), s


@pytest.mark.parametrize("news", [2, 40])
@pytest.mark.parametrize("size", [1e-30, 1e-4, 1e4, 1e30])
def test_sizes_of_queries_and_values(gpu_ctx, hyq, news, size):
    """Queries and keys whose product is of ordinary size, values of any: scores do
    not overflow on the way."""
    b = Q.BatchQ8([150, 77], [news] * 2, 4, 2, 32, seed=12)
    b.q *= np.float32(size)
    with np.errstate(invalid="ignore"):
        b.scales[:, 0] /= np.float32(size)
        b.scales[:, 1] *= np.float32(size)
    b.bytes = Q.join(b.codes, b.scales)
    check(b, attention(hyq, gpu_ctx, b))


def far(b, case):
    """Values up to the ends of f32's range. small: as many weights of 2^-21 of the largest
    as make 2^-10 of a sum, the largest one's values of the other sign; equal: equal
    weights of values whose sum is beyond f32; jump: values below 2^-90, then far ones."""
    b.codes[:, 0, ..., 1:] = 0  # (keys of one number)
    b.codes[:, 0, ..., 0] = 0
    b.scales[:, 0] = np.float32(2.0 ** -7)
    b.codes[:, 1] = np.abs(b.codes[:, 1])
    b.q[:] = 0
    with np.errstate(invalid="ignore"):
        b.scales[:, 1] = np.where(np.isnan(b.scales[:, 1]), np.nan, 2.6e36 if case == "equal" else 8e35)
    if case == "small":
        b.q[..., 0] = 21 * np.log(2.0) * np.sqrt(D) * 2.0 ** 7 / 127
    for s in range(b.seqs):
        at = np.arange(b.lens[s])
        page, place = b.table[s, at // b.pt], at % b.pt
        if case == "small":
            x = (b.lens[s] - b.news[s]) // 2
            b.codes[page[x], 0, :, place[x], 0] = 127
            b.codes[page[x], 1, :, place[x]] *= -1
        if case == "jump":
            half = at < len(at) // 2
            b.scales[page[half], 1, :, place[half]] = np.float32(2.0 ** -100)
    b.bytes = Q.join(b.codes, b.scales)


@pytest.mark.parametrize("case", ["small", "equal", "jump"])
@pytest.mark.parametrize("news", [1, 40])
def test_values_at_the_ends_of_the_range(gpu_ctx, hyq, news, case):
    """Small weights of far values count, sums of many do not leave f32 and weights of
    values before far ones stay, in slots that one worker takes and in cut ones."""
    b = Q.BatchQ8([2100, 60 if news > 1 else 30, 700], [news, news, 2], 4, 2, 32, seed=14)
    far(b, case)
    check(b, attention(hyq, gpu_ctx, b))


@pytest.mark.parametrize("news", [2, 40])
def test_far_keys_of_small_queries(gpu_ctx, hyq, news):
    """Keys of 2^116 and queries of 2^-100: scores of +-5000, so that one position has all
    the weight (the others' is 2^-14426 of it, zero) and its values are the result, to the
    roundings of their product with the scale, of the weight's two parts and of the
    normalisation."""
    b = Q.BatchQ8([150, 77], [news] * 2, 4, 2, 32, seed=16)
    b.codes[:, 0, ..., 1:] = 0
    b.codes[:, 0, ..., 0] = -127
    with np.errstate(invalid="ignore"):
        b.scales[:, 0] = np.where(np.isnan(b.scales[:, 0]), np.nan,
                                  np.float32(5000 * np.sqrt(D) / 127 * 2.0 ** 100))
    b.q[:], b.q[..., 0] = 0, np.float32(2.0 ** -100)
    for s, at in enumerate((37, 20)):
        b.codes[b.table[s, at // 32], 0, :, at % 32, 0] = 127
    b.bytes = Q.join(b.codes, b.scales)
    got, (want, _) = attention(hyq, gpu_ctx, b), b.attention()
    big = np.abs(want).max(-1, keepdims=True)
    assert np.all(np.abs(got - want) <= big * (8 * R.U + 2.0 ** -22))


@pytest.mark.parametrize("case", ["small", "jump"])
@pytest.mark.parametrize("news", [1, 40])
def test_far_values_in_one_piece(gpu_ctx, hyq, news, case):
    """The same where one wave or workgroup goes through all of a slot: in a batch that
    gives each worker more tiles than the slot has, and one of more blocks than pieces.
    (The other slots name the first one's pages, over and over.)"""
    b = Q.BatchQ8([2100], [news], 4, 2, 32, seed=15)
    far(b, case)
    want, tol = b.attention()
    seqs, pages = (21, 3600) if news == 1 else (200, b.width)
    row = np.resize(b.table[0, :2100 // 32], pages).astype(np.int32)
    b.table = np.concatenate([np.resize(b.table[0], (1, b.width))] * seqs) if news > 1 else (
        np.concatenate([np.full((1, pages), -1, np.int32)] + [row[None]] * (seqs - 1)))
    if news == 1:
        b.table[0, :66] = Q.BatchQ8([2100], [news], 4, 2, 32, seed=15).table[0, :66]
    b.seqs, b.width = seqs, pages
    b.lens = np.full(seqs, 2100 if news > 1 else pages * 32, np.int32)
    b.lens[0] = 2100
    b.news = np.full(seqs, news, np.int32)
    b.start = (np.arange(seqs + 1) * news).astype(np.int32)
    b.q, b.rows = np.concatenate([b.q] * seqs), seqs * news
    got = attention(hyq, gpu_ctx, b)
    for s in range(seqs if news > 1 else 1):
        err = np.abs(got[s * news:(s + 1) * news] - want).max(-1)
        assert np.all(err <= tol), (s, (err / tol).max())


@pytest.mark.parametrize("pt", [16, 64])
@pytest.mark.parametrize("news", [3, 50])
def test_missing_pages(gpu_ctx, hyq, news, pt):
    """Positions of entries that name no page are not attended; a slot without any
    gives zeros."""
    b = Q.BatchQ8([200, 130, 60], [news] * 3, 4, 2, pt, seed=15)
    b.table[0, 0], b.table[0, 1] = -1, b.pages + 7
    b.table[2, :] = -1
    got = attention(hyq, gpu_ctx, b)
    check(b, got)
    assert np.all(got[b.start[2]:b.start[3]] == 0)


@pytest.mark.parametrize("news", [4, 40])
def test_numbers_that_are_not_finite(gpu_ctx, hyq, news):
    """A NaN scale reaches the rows that see its position and no other: a key's and a
    value's all of a row. A query's NaN or infinity its own row and head."""
    b = Q.BatchQ8([100, 90], [news] * 2, 4, 2, 32, seed=31)
    row = b.start[1] + 1
    clean = attention(hyq, gpu_ctx, b)
    last = 100 - news + 2  # seen by the slot's new rows from the third on
    b.scales[b.table[0, last // 32], 0, 0, last % 32] = np.nan
    b.scales[b.table[0, last // 32], 1, 1, last % 32] = np.nan
    b.bytes = Q.join(b.codes, b.scales)
    b.q[row, 3, 5] = np.inf
    b.q[row, 0, 9] = np.nan
    got = attention(hyq, gpu_ctx, b)
    bad = np.zeros((b.rows, 4), bool)
    bad[2:news] = True
    bad[row, [0, 3]] = True
    assert not np.isfinite(got[bad]).any()
    assert np.array_equal(got[~bad], clean[~bad])


def test_bounds_of_slots(gpu_ctx, hyq):
    """Lengths past the table, starts that do not ascend or pass the rows, a slot of
    more rows than max_rows: no access outside, and the other slots right."""
    b = Q.BatchQ8([100, 64, 40], [1, 1, 1], 4, 2, 32, seed=41, tail=4)
    want, tol = b.attention()
    b.lens = np.array([100, 1 << 30, -5], np.int32)
    got = attention(hyq, gpu_ctx, b)
    assert np.all(np.abs(got[0] - want[0]).max(-1) <= tol[0])
    assert np.all(got[2] == 0)
    b = Q.BatchQ8([100, 64, 40], [1, 30, 1], 4, 2, 32, seed=42)
    want, tol = b.attention()
    got = attention(hyq, gpu_ctx, b, max_rows=8)
    for r in (0, 31):
        assert np.all(np.abs(got[r] - want[r]).max(-1) <= tol[r])
    assert np.all(got[1:31] == -7)
    b.start = np.array([0, 40, 2, 90], np.int32)
    attention(hyq, gpu_ctx, b, max_rows=30)


# ---- writing and reading ----
def append(hyq, ctx, b, pool, k, v, qn, kn, freq, eps, first):
    kl = layout(hyq, b)
    a = lambda x, t=np.float32: ctx.array(np.ascontiguousarray(x, t))
    out = a(np.full((b.rows, b.heads, D), -7))
    d = [a(x) for x in (b.q, k, v, qn, kn, freq)]
    pd, td, ld, sd = ctx.array(pool), ctx.array(b.table), ctx.array(b.lens), ctx.array(b.start)
    hyq.check(hyq.lib().hyq_paged_rope_norm_append_d(
        ctx.handle, ctypes.byref(kl), pd.ptr, 0, td.ptr, ld.ptr, sd.ptr, b.rows, b.heads,
        *[x.ptr for x in d], eps, first, out.ptr))
    return out.numpy(), pd.numpy()


@pytest.mark.parametrize("first", [0, 1])
@pytest.mark.parametrize("heads,pt", [((2, 2), 16), ((6, 2), 64), ((16, 4), 32), ((8, 1), 256)],
                         ids=str)
def test_append(gpu_ctx, hyq, heads, pt, first):
    """Codes and scales of the new rows' keys and values as the 64-bit form has them,
    every other byte of the pool as it was, queries as in other pools."""
    lens, news = [1, 0, 17, 300, 64, 130000], [1, 0, 5, 70, 1, 2]
    b = Q.BatchQ8([1, 0, 17, 300, 64, 50], news, *heads, pt, seed=pt + first, tail=3)
    r = np.random.default_rng(3)
    # the last slot's positions are far: only its last pages are in the table
    width = 130000 // pt + 1
    table = np.full((6, width), -1, np.int32)
    table[:, :b.width] = b.table
    table[5, 129998 // pt:129999 // pt + 1] = b.table[5, 0]
    b.table, b.width, b.lens = table, width, np.array(lens, np.int32)
    k, v = r.normal(0, 1, (2, b.rows, b.kvh, D)).astype(np.float32)
    v[1, 0], v[2, 0, 5], v[3, 0, 9] = 0, np.inf, np.nan
    v[4] *= np.float32(1e-30)
    k[5, 0, 3], k[6, 0] = np.nan, 0
    qn, kn = r.normal(1, 0.1, (2, D)).astype(np.float32)
    freq = (11158840.0 ** (-np.arange(64) / 64)).astype(np.float32)
    q_out, pool = append(hyq, gpu_ctx, b, b.bytes, k, v, qn, kn, freq, 1e-5, first)
    plain = R.Batch.__new__(R.Batch)  # (the 64-bit form, on a pool of numbers)
    plain.__dict__.update(b.__dict__, pool=np.zeros((b.pages, 2, b.kvh, pt, D)))
    want_q, formed = R.append(plain, k, v, qn, kn, freq, 1e-5, bool(first))
    assert np.allclose(q_out[:b.new], want_q[:b.new], rtol=0, atol=2e-5)
    assert np.all(q_out[b.new:] == -7)
    codes, scales = b.codes.copy(), b.scales.copy()
    for s in range(b.seqs):
        for i in range(news[s]):
            pos = lens[s] - news[s] + i
            at = (table[s, pos // pt], slice(None), slice(None), pos % pt)
            codes[at], scales[at] = Q.quantise(formed[at])
    got_codes, got_scales = Q.split(pool, b.kvh, pt)
    fine = ~np.isnan(scales)
    assert np.array_equal(fine, ~np.isnan(got_scales))
    assert np.array_equal(codes[fine], got_codes[fine])
    assert np.allclose(scales[fine], got_scales[fine], rtol=2.0 ** -23, atol=0)
    # places that nothing wrote keep their bytes
    written = np.zeros((b.pages, 2, b.kvh, pt), bool)
    for s in range(b.seqs):
        for i in range(news[s]):
            pos = lens[s] - news[s] + i
            written[table[s, pos // pt], :, :, pos % pt] = True
    n = 2 * b.kvh * pt * D
    assert np.array_equal(pool[:, :n].reshape(-1, D)[~written.reshape(-1)],
                          b.bytes[:, :n].reshape(-1, D)[~written.reshape(-1)])
    assert np.array_equal(pool[:, n:].reshape(-1, 4)[~written.reshape(-1)],
                          b.bytes[:, n:].reshape(-1, 4)[~written.reshape(-1)])


def test_append_of_halves_and_extremes(gpu_ctx, hyq):
    """Values whose quotients are halves go to the even code; the largest numbers
    that f32 holds, and those below its normal ones."""
    b = Q.BatchQ8([8], [8], 2, 1, 16, seed=1)
    v = np.zeros((8, 1, D), np.float32)
    v[0, 0] = np.arange(128) - 64 + 0.5
    v[0, 0, 0] = 127
    v[1, 0, :2] = 3.4e38, -3.4e38
    v[2, 0, :3] = 1e-40, -1e-40, 3e-41
    v[3, 0, :3] = 1.4e-45, -1.4e-45, 0
    v[4, 0, :3] = 254, 1, 3
    v[5, 0] = -1
    v[6, 0, 0] = -127.49
    v[7, 0, 127] = 2.0 ** -120
    one, freq = np.ones(D, np.float32), np.zeros(64, np.float32)
    _, pool = append(hyq, gpu_ctx, b, b.bytes, np.ones((8, 1, D), np.float32), v, one, one, freq,
                     1e-5, 0)
    codes, scales = Q.split(pool, 1, 16)
    want, ws = Q.quantise(v[:, 0])
    page = b.table[0, 0]
    assert np.array_equal(codes[page, 1, 0, :8], want) and np.array_equal(scales[page, 1, 0, :8], ws)
    assert list(want[4, :3]) == [127, 0, 2]


def test_read_back_at_the_ends_of_the_range(gpu_ctx, hyq):
    """Half a scale from what was written, and 127 * 2^-150 more where the scale is no
    normal number; never infinite. (A code's product with the scale is rounded once.)"""
    top, step = float(np.finfo(np.float32).max), 2.0 ** -149
    heads = [top, top * (1 - 2.0 ** -24), top * (1 - 2.0 ** -22), 127 * 2.0 ** -126,
             126 * 2.0 ** -126, 178 * step, 190 * step, 127 * step, 64 * step, 63 * step, step]
    n = len(heads)
    b = Q.BatchQ8([n], [n], 2, 1, 16, seed=26)
    v = np.array(heads)[:, None] * np.linspace(-1, 1, D)
    v = v.astype(np.float32).reshape(n, 1, D)
    one, freq = np.ones(D, np.float32), np.zeros(64, np.float32)
    _, pool = append(hyq, gpu_ctx, b, b.bytes, np.ones((n, 1, D), np.float32), v, one, one, freq,
                     1e-5, 0)
    scales = Q.split(pool, 1, 16)[1][b.table[0, 0], 1, 0, :n].astype(np.float64)
    kl = layout(hyq, b)
    d = [gpu_ctx.array(x) for x in (pool, b.table, b.lens, b.start)]
    k, got = (gpu_ctx.array(np.full((n, 1, D), -7, np.float32)) for _ in range(2))
    hyq.check(hyq.lib().hyq_paged_read_d(gpu_ctx.handle, ctypes.byref(kl), d[0].ptr, 0, d[1].ptr,
                                         d[2].ptr, d[3].ptr, n, k.ptr, got.ptr))
    got = got.numpy()[:, 0].astype(np.float64)
    assert np.isfinite(got).all()
    most = np.abs(v[:, 0].astype(np.float64)).max(-1)
    bound = scales / 2 + np.where(most < 127 * 2.0 ** -126, 127 * 2.0 ** -150, 0)
    err = np.abs(got - v[:, 0])
    assert np.all(err <= (bound + most * R.U)[:, None]), (err.max(-1) / bound)


DTYPES = ["F32", "F16", "Q8"]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kvh,pt", [(1, 16), (3, 64), (8, 32), (20, 16)])
def test_read(gpu_ctx, hyq, kvh, pt, dtype):
    """The rows that the starts name, as the pages hold them: the last ones of a slot
    or all, zeros without a page, rows of no slot untouched; a pool of two layers."""
    lens, news = [1, 0, 40, 130, 64], [1, 0, 3, 130, 64]
    q8 = dtype == "Q8"
    b = (Q.BatchQ8(lens, news, kvh, kvh, pt, seed=kvh, tail=2) if q8 else
         R.Batch(lens, news, kvh, kvh, pt, dtype == "F16", seed=kvh, tail=2))
    b.table[3, 1] = -1
    b.table[4, 0] = b.pages
    want = np.zeros((2, b.rows, kvh, D), np.float64)
    for s in range(b.seqs):
        for h in range(kvh):
            k, v, ok = b.kv(s, h)
            n = lens[s] - news[s]
            rows = slice(b.start[s], b.start[s + 1])
            want[0, rows, h], want[1, rows, h] = (np.where(ok[:, None], x, 0)[n:] for x in (k, v))
    pages = b.bytes if q8 else b.pool
    pool = gpu_ctx.array(np.stack([np.zeros_like(pages), pages]))
    kl = hyq.KvLayout({"F32": hyq.F32, "F16": hyq.F16, "Q8": hyq.KV_Q8}[dtype], 2, kvh, D, pt,
                      b.pages, b.seqs, b.width)
    td, ld, sd = gpu_ctx.array(b.table), gpu_ctx.array(b.lens), gpu_ctx.array(b.start)
    k, v = (gpu_ctx.array(np.full((b.rows, kvh, D), -7, np.float32)) for _ in range(2))
    hyq.check(hyq.lib().hyq_paged_read_d(gpu_ctx.handle, ctypes.byref(kl), pool.ptr, 1, td.ptr,
                                         ld.ptr, sd.ptr, b.rows, k.ptr, v.ptr))
    for got, w in zip((k.numpy(), v.numpy()), want):
        # (an 8-bit number is its scale times its code, rounded once)
        assert np.all(np.abs(got[:b.new] - w[:b.new]) <= np.abs(w[:b.new]) * R.U * q8)
        assert np.all(got[b.new:] == -7)
    hyq.check(hyq.lib().hyq_paged_read_d(gpu_ctx.handle, ctypes.byref(kl), pool.ptr, 1, td.ptr,
                                         ld.ptr, sd.ptr, 0, k.ptr, v.ptr))  # no rows: nothing


def test_cache_reads_as_many_rows_as_a_call_takes(gpu_ctx, hyq):
    """2^20 positions at once; one more are to be read in parts."""
    c = hyq.PagedCache(gpu_ctx, 1, 1, 4097, 2, 1 << 20, page_tokens=256, dtype=hyq.F16)
    page = np.random.default_rng(25).normal(0, 1, (2, 256, D)).astype(np.float16)
    c.pool.copy_from(np.resize(page.view(np.uint8), c.pool.shape))
    assert not c.extend([1 << 20, 0]).any()
    k, v = c.read(0)[0]
    for got, want in ((k, page[0]), (v, page[1])):
        assert got.shape == (1 << 20, D)
        assert np.array_equal(got[:256], want) and np.array_equal(got[-256:], want)
    assert not c.extend([0, 1]).any()
    with pytest.raises(ValueError, match="parts"):
        c.read(0)


# ---- the pages' bookkeeping ----
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layers,kvh,pt", [(2, 1, 16), (1, 3, 64), (3, 2, 256)])
def test_cache_forks_and_compacts(gpu_ctx, hyq, dtype, layers, kvh, pt):
    """Slots that are forked, extended over shared pages, written, freed and made
    dense hold what a list of each slot's tokens says, in every layer."""
    kind = {"F32": hyq.F32, "F16": hyq.F16, "Q8": hyq.KV_Q8}[dtype]
    seqs = 4
    c = hyq.PagedCache(gpu_ctx, layers, kvh, 40, seqs, 4 * pt, page_tokens=pt, dtype=kind)
    r = np.random.default_rng(8)
    one, freq = gpu_ctx.array(np.ones(D, np.float32)), gpu_ctx.array(np.zeros(64, np.float32))
    held = [[np.zeros((2, 0, kvh, D)) for _ in range(layers)] for _ in range(seqs)]
    qo = gpu_ctx.empty((seqs * 3 * pt, kvh, D), np.float32)

    def step(parent, add):
        nonlocal held
        c.fork(parent)
        held = [held[p] if p >= 0 else [np.zeros((2, 0, kvh, D)) for _ in range(layers)]
                for p in parent]
        assert not c.extend(add).any()
        start = np.concatenate([[0], np.cumsum(np.maximum(add, 0))]).astype(np.int32)
        rows, sd = int(start[-1]), gpu_ctx.array(start)
        for l in range(layers):
            q, k, v = r.normal(0, 1, (3, rows, kvh, D)).astype(np.float32)
            k /= np.sqrt((k.astype(np.float64) ** 2).mean(-1, keepdims=True))
            given = [gpu_ctx.array(x) for x in (q, k, v)]
            c.append_d(l, sd.ptr, rows, kvh, *[x.ptr for x in given], one.ptr, one.ptr, freq.ptr,
                       0.0, qo.ptr)
            gpu_ctx.sync()
            held = [[np.concatenate([held[s][x], np.stack([k, v])[:, start[s]:start[s + 1]]], 1)
                     if x == l else held[s][x] for x in range(layers)] for s in range(seqs)]
        compare()

    def compare():
        for l in range(layers):
            for s, (k, v) in enumerate(c.read(l)):
                for got, want in zip((k, v), held[s][l]):
                    got = got.reshape(-1, kvh, D)
                    assert got.shape == want.shape
                    if not want.size:
                        continue
                    # half a step of the type (a key's norm adds a few roundings)
                    step = {"F32": 0, "F16": 2.0 ** -11,
                            "Q8": np.abs(want).max(-1, keepdims=True) / 254}[dtype]
                    assert np.all(np.abs(got - want) <= step * (1 if dtype == "Q8" else
                                                                np.abs(want)) + 2e-6 + 2.0 ** -25)

    step([-1] * 4, [pt + 3, 5, 2 * pt, 0])
    step([0, 0, 0, 2], [1, 2, pt, 1])
    step([1, 1, 2, 3], [3, 0, 1, pt - 1])
    live = c.compact()
    assert live == int((c.refs.numpy() > 0).sum())
    compare()
    step([0, -1, 2, 2], [1, 7, 1, 2])
    c.compact()
    compare()
