"""The paged cache's append and attention on the GPU against plain 64-bit
forms (tests/paged_ref.py): ragged batches at the sizes where tiles, pages and
row blocks end, with every unused place of the pool a NaN."""
import ctypes

import numpy as np
import pytest

import paged_ref as R

pytestmark = pytest.mark.gpu
D = R.D


def put(ctx, b):
    return {n: ctx.array(a) for n, a in dict(pool=b.pool, table=b.table, len=b.lens, start=b.start,
                                             q=b.q).items()}


def layout(hyq, b, layers=1, pages=None):
    return hyq.KvLayout(hyq.F16 if b.f16 else hyq.F32, layers, b.kvh, D, b.pt, pages or b.pages,
                        b.seqs, b.width)


def attention(hyq, ctx, b, max_rows=None, d=None):
    """hyq_paged_attention_d of a batch; rows of no slot stay at -7."""
    d = d or put(ctx, b)
    kl = ctypes.byref(layout(hyq, b))
    most = max_rows or max(1, int(b.news.max()))
    need = hyq.lib().hyq_paged_attention_scratch_bytes(kl, b.rows, most, b.heads)
    scratch = ctx.array(np.full(need, 0xFF, np.uint8))  # (NaNs: nothing may be read unwritten)
    out = ctx.array(np.full((b.rows, b.heads, D), -7, np.float32))
    hyq.check(hyq.lib().hyq_paged_attention_d(
        ctx.handle, kl, d["pool"].ptr, 0, d["table"].ptr, d["len"].ptr, d["start"].ptr, b.rows,
        most, b.heads, d["q"].ptr, scratch.ptr, need, out.ptr))
    return out.numpy()


def check(b, got, rows=None):
    want, tol = b.attention()
    for s in range(b.seqs):
        for r in range(b.start[s], b.start[s + 1]):
            err = np.abs(got[r] - want[r]).max(-1)
            assert np.all(err <= tol[r]), (
                f"slot {s} (len {b.lens[s]}, {b.news[s]} new) row {r - b.start[s]}: "
                f"{err.max():.3e} > {tol[r][err.argmax()]:.3e}")
    assert np.all(got[b.new:] == -7), "rows behind the last slot changed"


# (heads, kv heads): 1, 2, 3, 4, 8 and 16 query heads per KV head
HEADS = [(2, 2), (4, 2), (6, 2), (16, 4), (8, 1), (16, 1)]


@pytest.mark.parametrize("f16", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("pt", [16, 64, 256])
def test_decode(gpu_ctx, hyq, heads, pt, f16):
    """One new token per slot, lengths around tiles and pages, empty slots."""
    lens = [1, 0, 15, 16, 17, 31, 33, 64, 65, 200, 300, 1]
    news = [1, 0, 1, 1, 1, 1, 1, 1, 1, 1, 0, 1]
    b = R.Batch(lens, news, *heads, pt, f16, seed=pt + heads[0], tail=2)
    check(b, attention(hyq, gpu_ctx, b))


@pytest.mark.parametrize("f16", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("pt", [16, 64])
def test_mixed_rows(gpu_ctx, hyq, heads, pt, f16):
    """Decode steps, drafts on both sides of the two forms' border, and prompts
    around a block of 128 query rows, with and without earlier tokens."""
    rep = heads[0] // heads[1]
    few, block = 16 // rep, 128 // rep
    news = [1, few, few + 1, block, 0, block + 1, 2, min(2 * block + 3, 70), 33]
    lens = [90, few, few + 40, block, 50, block + 37, 300, min(2 * block + 3, 70) + 1, 33]
    b = R.Batch(lens, news, *heads, pt, f16, seed=pt * 3 + heads[0], tail=3)
    check(b, attention(hyq, gpu_ctx, b))


@pytest.mark.parametrize("f16", [False, True], ids=["f32", "f16"])
def test_long_and_short(gpu_ctx, hyq, f16):
    """One long slot cut over many workers beside short ones; one long prompt
    cut into pieces."""
    b = R.Batch([5000, 3, 17], [1, 1, 1], 8, 2, 64, f16, seed=5)
    check(b, attention(hyq, gpu_ctx, b))
    b = R.Batch([4100], [45], 8, 2, 64, f16, seed=6, tail=1)
    check(b, attention(hyq, gpu_ctx, b))


@pytest.mark.parametrize("f16", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("news", [1, 30])
def test_slots_that_share_pages(gpu_ctx, hyq, news, f16):
    """Beams of one prompt: slots that name the same pages at the same places,
    all of them, the first ones, later ones only, and none."""
    b = R.Batch([600, 600, 480, 600, 600, 200], [news] * 6, 8, 2, 32, f16, seed=22)
    b.table[1, :18] = b.table[0, :18]
    b.table[2, :14] = b.table[0, :14]
    b.table[4, 7:18] = b.table[3, 7:18]
    check(b, attention(hyq, gpu_ctx, b))


@pytest.mark.parametrize("f16", [False, True], ids=["f32", "f16"])
def test_uneven_prompts(gpu_ctx, hyq, f16):
    """Two long prompts beside many short ones, too many blocks for the long
    ones to be cut finely by themselves: workgroups take several blocks' steps."""
    b = R.Batch([30] * 15 + [2500] + [30] * 13 + [2437], [30] * 15 + [64] + [30] * 13 + [64], 16, 8,
                64, f16, seed=20, tail=1)
    check(b, attention(hyq, gpu_ctx, b))


@pytest.mark.parametrize("f16", [False, True], ids=["f32", "f16"])
def test_more_blocks_than_the_plan_takes_at_once(gpu_ctx, hyq, f16):
    """Some 390 blocks of prompts, with decode steps and empty slots between."""
    news = np.array([5, 1, 0] * 300)
    lens = news + np.arange(900) % 97
    news[[100, 700]] = 350, 353
    lens[[100, 700]] = 900, 353
    b = R.Batch(lens, news, 16, 1, 16, f16, seed=21)
    check(b, attention(hyq, gpu_ctx, b))


@pytest.mark.parametrize("f16", [False, True], ids=["f32", "f16"])
def test_many_slots(gpu_ctx, hyq, f16):
    """More slots than a workgroup has threads, most of them empty."""
    r = np.random.default_rng(3)
    lens = np.where(r.random(1100) < 0.2, r.integers(1, 60, 1100), 0)
    news = np.minimum(lens, r.integers(0, 3, 1100))
    news[[5, 1040]], lens[[5, 1040]] = 37, 50
    b = R.Batch(lens, news, 2, 1, 16, f16, seed=4)
    check(b, attention(hyq, gpu_ctx, b))


@pytest.mark.parametrize("f16", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("news", [3, 40])
@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf], ids=str)
def test_values_that_are_not_finite_stay_unseen(gpu_ctx, hyq, f16, news, what):
    """A new token's value (and key) that is not finite reaches the rows that
    see it and no other."""
    b = R.Batch([70 + news], [news], 4, 1, 16, f16, seed=9)
    clean, tol = b.attention()
    at = 70 + news - 2  # seen by the last two rows alone
    b.pool[b.table[0, at // 16], 1, 0, at % 16, 5] = what
    got = attention(hyq, gpu_ctx, b)
    assert np.all(np.abs(got[:news - 2] - clean[:news - 2]).max(-1) <= tol[:news - 2])
    assert not np.isfinite(got[news - 2:, :, 5]).any()
    keep = np.arange(D) != 5
    err = np.abs(got - clean)[..., keep].max(-1)
    assert np.all(err <= tol)
    b.pool[b.table[0, at // 16], 0, 0, at % 16, 5] = np.nan  # and the key
    got = attention(hyq, gpu_ctx, b)
    assert np.all(np.abs(got[:news - 2] - clean[:news - 2]).max(-1) <= tol[:news - 2])


@pytest.mark.parametrize("f16", [False, True], ids=["f32", "f16"])
def test_pages_that_are_not_there(gpu_ctx, hyq, f16):
    """Entries outside the pool hold nothing; a slot of only such entries, one
    with more new tokens than positions and one of none see nothing."""
    news = [1, 1, 5, 2, 40, 40, 1]
    lens = [100, 40, 60, 0, 90, 80, 33]
    b = R.Batch(lens, news, 4, 1, 16, f16, seed=11, tail=1)
    b.table[0, [0, 3]] = [-1, b.pages]
    b.table[1, :3] = [-5, 2 ** 31 - 1, -2 ** 31]
    b.table[2, 1] = 1 << 20
    b.table[4, [1, 4]] = -1
    b.table[5, :] = b.pages
    b.lens[6] = 0  # one new token over no positions
    got = attention(hyq, gpu_ctx, b)
    check(b, got)
    assert np.all(got[b.start[1]:b.start[2]] == 0) and np.all(got[b.start[3]:b.start[4]] == 0)


def fill_unused(b, what):
    """Another content than NaN for every place of the pool that no position
    uses, page 0 (which is read where a slot has no page) among them."""
    spare = np.setdiff1d(np.arange(b.pages), b.table)[0]
    b.table[b.table == 0] = spare
    b.pool[[0, spare]] = b.pool[[spare, 0]]
    assert np.isnan(b.pool[0]).all()
    holes = np.isnan(b.pool)
    if what == "bits":
        kind = np.uint16 if b.f16 else np.uint32
        b.pool[holes] = b.rng.integers(0, np.iinfo(kind).max, holes.sum(), kind, True).view(
            b.pool.dtype)
    else:
        b.pool[holes] = what


@pytest.mark.parametrize("f16", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("what", ["bits", np.inf, -np.inf, 65504.0, 65520.0, -1e5, 3e38], ids=str)
@pytest.mark.parametrize("pt", [16, 32, 64, 256])
def test_places_that_nobody_wrote(gpu_ctx, hyq, pt, what, f16):
    """The rest of a slot's last page and a missing page's places hold anything,
    finite numbers past f16's range among them: nothing of it reaches a row."""
    if f16 and what not in ("bits", np.inf, -np.inf, 65504.0):
        what = np.float16(np.sign(what) * 65504)
    news = [1, 3, 40, 130, 33, 1]
    lens = [70, 3, 110, 140, 600, 65]
    b = R.Batch(lens, news, 8, 2, pt, f16, seed=31 + pt, tail=1)
    fill_unused(b, what)
    with np.errstate(invalid="ignore"):  # (bits that are signalling NaNs)
        check(b, attention(hyq, gpu_ctx, b))
    if pt < 256:
        b.table[2, 1], b.table[4, 2], b.table[4, -2], b.table[0, 0] = -1, b.pages, -1, -9
    b.table[5, 0] = -1
    with np.errstate(invalid="ignore"):
        check(b, attention(hyq, gpu_ctx, b))


@pytest.mark.parametrize("news", [3, 40])
@pytest.mark.parametrize("what", [65520.0, -3e38], ids=str)
def test_values_past_f16_stay_unseen(gpu_ctx, hyq, news, what):
    """A new token's finite value beyond what f16 parts hold reaches the rows
    that see it and no other."""
    b = R.Batch([70 + news], [news], 4, 1, 64, False, seed=32)
    clean, tol = b.attention()
    at = 70 + news - 2  # seen by the last two rows alone
    b.pool[b.table[0, at // 64], 1, 0, at % 64, 5] = what
    got = attention(hyq, gpu_ctx, b)
    assert np.all(np.abs(got[:news - 2] - clean[:news - 2]).max(-1) <= tol[:news - 2])
    seen = got[news - 2:, :, 5]
    assert np.all((np.abs(seen) > 1) | ~np.isfinite(seen))
    keep = np.arange(D) != 5
    assert np.all(np.abs(got - clean)[..., keep].max(-1) <= tol)


def test_starts_and_lengths_out_of_range(gpu_ctx, hyq):
    """Wrong starts and lengths make wrong rows but stay inside the buffers;
    slots that they leave right are right."""
    b = R.Batch([40, 50, 60, 70], [2, 3, 40, 1], 4, 1, 16, True, seed=12)
    d = put(gpu_ctx, b)
    want, tol = b.attention()
    d["len"] = gpu_ctx.array(np.array([40, -7, 2 ** 31 - 1, 70], np.int32))
    got = attention(hyq, gpu_ctx, b, d=d)
    for s in (0, 3):
        r = slice(b.start[s], b.start[s + 1])
        assert np.all(np.abs(got[r] - want[r]).max(-1) <= tol[r])
    assert np.all(got[2:5] == 0)
    for start in ([0, 2 ** 31 - 1, 3, -5, 10], [46, 0, 46, 0, 46], [-9, 60, 70, 80, 90]):
        d["start"] = gpu_ctx.array(np.array(start, np.int32))
        attention(hyq, gpu_ctx, b, d=d)
        attention(hyq, gpu_ctx, b, max_rows=1, d=d)


def test_rows_past_the_promise_are_left(gpu_ctx, hyq):
    """Slots of more new tokens than max_rows are not computed."""
    b = R.Batch([40, 50, 60], [1, 3, 1], 4, 1, 16, True, seed=13)
    want, tol = b.attention()
    got = attention(hyq, gpu_ctx, b, max_rows=1)
    assert np.all(got[1:4] == -7)
    for r in (0, 4):
        assert np.all(np.abs(got[r] - want[r]).max(-1) <= tol[r])


@pytest.mark.parametrize("most", [20, 33])
def test_prompts_past_the_promise_are_left(gpu_ctx, hyq, most):
    """The same where max_rows admits prompts."""
    b = R.Batch([40, 90, 60, 50], [1, 40, 20, 34], 4, 1, 16, True, seed=34, tail=2)
    want, tol = b.attention()
    got = attention(hyq, gpu_ctx, b, max_rows=most)
    for s in range(4):
        r = slice(b.start[s], b.start[s + 1])
        if b.news[s] > most:
            assert np.all(got[r] == -7)
        else:
            assert np.all(np.abs(got[r] - want[r]).max(-1) <= tol[r])
    assert np.all(got[b.new:] == -7)


@pytest.mark.parametrize("f16", [False, True], ids=["f32", "f16"])
def test_queries_of_any_size(gpu_ctx, hyq, f16):
    """Large and small queries, beyond what f16 holds: scores far apart, and
    all alike."""
    b = R.Batch([100, 60], [1, 40], 4, 1, 16, f16, seed=14)
    for scale in (2.0 ** 20, 2.0 ** -40):
        b.q = (b.q / np.abs(b.q).max() * scale).astype(np.float32)
        want, tol = b.attention()
        got = attention(hyq, gpu_ctx, b)
        assert np.isfinite(got).all()
        if scale < 1:
            assert np.all(np.abs(got - want).max(-1) <= tol)


@pytest.mark.parametrize("f16", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("power", [-99, -100, -101, -113, -115, -126, -128, -140, -149])
def test_tiny_queries(gpu_ctx, hyq, power, f16):
    """Queries down to the smallest f32, zeros among their dims: every score is
    zero, the output the mean of the values seen, in both forms."""
    b = R.Batch([100, 60, 9], [1, 40, 3], 4, 1, 16, f16, seed=33)
    b.q = np.ldexp(np.clip(np.round(b.q * 2), -4, 4) / 4, power).astype(np.float32)
    if power == -149:
        b.q[:] = np.where(b.q > 0, np.float32(2.0 ** -149), 0)
    assert (b.q != 0).any(-1).all() and (b.q == 0).any(-1).all()
    check(b, attention(hyq, gpu_ctx, b))


@pytest.mark.parametrize("scale", [2.0 ** -10, 2.0 ** -13, 2.0 ** 10])
@pytest.mark.parametrize("news", [2, 40])
def test_values_of_any_size(gpu_ctx, hyq, news, scale):
    """Small and large cached values keep their relative accuracy in an f32
    pool, in both forms (tolerance() is relative to the largest value)."""
    b = R.Batch([300, 90], [news, news], 8, 2, 32, False, seed=17)
    b.pool[:, 1] *= np.float32(scale)
    check(b, attention(hyq, gpu_ctx, b))


@pytest.mark.parametrize("scale", [2.0 ** -10, 2.0 ** 10])
@pytest.mark.parametrize("news", [2, 40])
def test_keys_of_any_size(gpu_ctx, hyq, news, scale):
    """The same of keys, with queries that bring the scores back to size: what
    tolerance() allows them is relative to the products' magnitude."""
    b = R.Batch([300, 90], [news, news], 8, 2, 32, False, seed=19)
    b.pool[:, 0] *= np.float32(scale)
    b.q *= np.float32(1 / scale)
    check(b, attention(hyq, gpu_ctx, b))


@pytest.mark.parametrize("f16", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("news", [2, 40])
def test_many_small_weights(gpu_ctx, hyq, news, f16):
    """Thousands of positions of one small weight, 194.5 * 2^-24 of the largest,
    whose values alone make the output: they are rounded alike, so that a
    weight's error does not average out. Keys are zero but for one in every 32
    positions, whose values are zero. Relative bound: the score's (tolerance()'s
    d, twice), the sums' 2 (n + 8) U, and the weight's resolution where its f16
    parts hold 2^-25 of 2^7: 2^-32 of it, 2^-15.6 of the small ones."""
    n = 2000
    b = R.Batch([n], [news], 4, 2, 64, f16, seed=18, spare=0)
    b.pool[:] = 0
    for s in range(0, n, 32):
        b.pool[b.table[0, s // 64], 0, :, s % 64, 0] = 2.0
    for i in range(n):
        if i % 32:
            b.pool[b.table[0, i // 64], 1, :, i % 64] = 1.0
    b.q[:] = 0
    b.q[..., 0] = -np.log2(194.5 * 2.0 ** -24) * np.log(2) * np.sqrt(128) / 2.0
    out = attention(hyq, gpu_ctx, b)
    want, _ = b.attention()
    score = 11.4
    d = (128 * R.U + 3 * 2.0 ** -22) * (score + 1) + 9 * R.U * score + 2 * R.U
    bound = 2 * d + 2 * (n + 8) * R.U + 2.0 ** -15.6
    assert np.all(np.abs(out / want - 1) <= bound), np.abs(out / want - 1).max()


def test_offsets_past_32_bits(gpu_ctx, hyq):
    """Pages whose byte offsets pass 2^32 (and element offsets 2^31 in f16)."""
    small = R.Batch([600, 530], [1, 40], 8, 8, 256, True, seed=15, spare=1)
    page = small.pool[0].nbytes
    n = (2 ** 32 + 2 ** 30) // page
    L = hyq.lib()
    pool = gpu_ctx.empty(n * page, np.uint8)
    high = n - small.pages
    hyq.check(L.hyq_memcpy_h2d(gpu_ctx.handle, pool.ptr + high * page, small.pool.ctypes.data,
                               small.pool.nbytes))
    want, tol = small.attention()
    d = put(gpu_ctx, small)
    d["pool"] = pool
    d["table"] = gpu_ctx.array(np.where(small.table >= 0, small.table + high, -1).astype(np.int32))
    small.pages = n
    got = attention(hyq, gpu_ctx, small, d=d)
    assert np.all(np.abs(got - want).max(-1) <= tol)
    # and an append there
    small.pages = n - high
    k = small.rng.normal(0, 1, (small.rows, 8, D)).astype(np.float32)
    kd, w = gpu_ctx.array(k), gpu_ctx.array(np.ones(D, np.float32))
    f = gpu_ctx.array(np.zeros(64, np.float32))
    q = gpu_ctx.empty(small.q.size, np.float32)
    small.pages = n
    hyq.check(L.hyq_paged_rope_norm_append_d(
        gpu_ctx.handle, ctypes.byref(layout(hyq, small)), pool.ptr, 0, d["table"].ptr,
        d["len"].ptr, d["start"].ptr, small.rows, 8, d["q"].ptr, kd.ptr, kd.ptr, w.ptr, w.ptr,
        f.ptr, ctypes.c_float(1e-5), 0, q.ptr))
    back = np.empty_like(small.pool)
    hyq.check(L.hyq_memcpy_d2h(gpu_ctx.handle, back.ctypes.data, pool.ptr + high * page,
                               back.nbytes))
    last = small.table[1, 529 // 256]
    assert np.array_equal(back[last, 1, :, 529 % 256], k[40].astype(np.float16))
    pool.free()


@pytest.mark.parametrize("f16", [False, True], ids=["f32", "f16"])
def test_the_same_bits_twice(gpu_ctx, hyq, f16):
    b = R.Batch([900, 33, 500], [1, 2, 130], 8, 2, 32, f16, seed=16)
    one, two = attention(hyq, gpu_ctx, b), attention(hyq, gpu_ctx, b)
    assert np.array_equal(one.view(np.uint32), two.view(np.uint32))


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------
def append(hyq, ctx, b, k, v, qn, kn, freq, eps, norm_first, layer=0, layers=1, in_place=False):
    d = put(ctx, b)
    x = {n: ctx.array(a) for n, a in dict(k=k, v=v, qn=qn, kn=kn, freq=freq).items()}
    pool = ctx.array(np.broadcast_to(b.pool, (layers,) + b.pool.shape).copy())
    out = d["q"] if in_place else ctx.array(np.full(b.q.shape, -7, np.float32))
    hyq.check(hyq.lib().hyq_paged_rope_norm_append_d(
        ctx.handle, ctypes.byref(layout(hyq, b, layers)), pool.ptr, layer, d["table"].ptr,
        d["len"].ptr, d["start"].ptr, b.rows, b.heads, d["q"].ptr, x["k"].ptr, x["v"].ptr,
        x["qn"].ptr, x["kn"].ptr, x["freq"].ptr, ctypes.c_float(eps), int(norm_first), out.ptr))
    return out.numpy().reshape(b.q.shape), pool.numpy()


def check_append(hyq, ctx, b, norm_first, **kw):
    """Rounding: the reduced angle (|a| <= pi) to f32, at most 2 U off, moves a
    pair by 2 U of its length; sine and cosine by 2 U more; the rotation's three
    operations 3 U of it; the mean square's 128 terms and its root and quotient
    (128 / 2 + 4) U, two products 2 U; all relative to the head's largest
    possible |value|, its pair's length."""
    r = b.rng
    k, v = (r.normal(0, 1, (b.rows, b.kvh, D)).astype(np.float32) for _ in range(2))
    qn, kn = (r.normal(1, 0.1, D).astype(np.float32) for _ in range(2))
    freq = (11158840.0 ** (-np.arange(64) / 64)).astype(np.float32)
    q_out, pool = append(hyq, ctx, b, k, v, qn, kn, freq, 1e-5, norm_first, **kw)
    want_q, want_pool = R.append(b, k, v, qn, kn, freq, 1e-5, norm_first)
    pair = lambda x: np.sqrt(x[..., :64] ** 2 + x[..., 64:] ** 2)
    wmax = max(np.abs(qn).max(), np.abs(kn).max()) / min(np.abs(qn).min(), np.abs(kn).min())
    tol = lambda x: np.concatenate([pair(x)] * 2, -1) * wmax * 80 * R.U
    new = slice(0, b.new)
    assert np.all(np.abs(q_out[new] - want_q[new]) <= tol(want_q[new]))
    layer, layers = kw.get("layer", 0), kw.get("layers", 1)
    for l in range(layers):
        if l != layer:
            assert np.array_equal(pool[l], b.pool, equal_nan=True)
    got = pool[layer].astype(np.float64)
    # keys within the tolerance and a rounding to the pool's type; the rest exact
    half = 2.0 ** -11 if b.f16 else 0.0
    kt = tol(want_pool[:, 0]) * (1 + half) + half * np.abs(want_pool[:, 0]) + 2.0 ** -25 * b.f16
    assert np.array_equal(np.isnan(got), np.isnan(want_pool))
    assert np.all(~(np.abs(got[:, 0] - want_pool[:, 0]) > kt))
    assert np.array_equal(got[:, 1], want_pool[:, 1].astype(b.pool.dtype).astype(np.float64),
                          equal_nan=True)
    return q_out


@pytest.mark.parametrize("f16", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("heads", [(2, 2), (6, 2), (16, 4), (16, 1), (5, 5)], ids=str)
@pytest.mark.parametrize("norm_first", [False, True])
def test_append(gpu_ctx, hyq, heads, f16, norm_first):
    b = R.Batch([1, 17, 0, 64, 65, 40, 9], [1, 3, 0, 1, 2, 40, 0], *heads, 16, f16, seed=20,
                tail=3)
    q = check_append(hyq, gpu_ctx, b, norm_first, layer=1, layers=3)
    assert np.all(q[b.new:] == -7)
    same = append_in_place(hyq, gpu_ctx, b, norm_first)
    assert np.array_equal(same[b.new:], b.q[b.new:])


def append_in_place(hyq, ctx, b, norm_first):
    return check_append(hyq, ctx, b, norm_first, in_place=True)


@pytest.mark.parametrize("seqs", [63, 64, 65, 200])
def test_append_many_slots(gpu_ctx, hyq, seqs):
    r = np.random.default_rng(seqs)
    news = r.integers(0, 3, seqs)
    b = R.Batch(news + r.integers(0, 40, seqs), news, 2, 1, 16, True, seed=21, tail=70)
    check_append(hyq, gpu_ctx, b, False)


def test_append_at_far_positions(gpu_ctx, hyq):
    """Positions up to 2^24 - 1: the angle keeps its accuracy (an f32 product
    would be off by a radian there)."""
    b = R.Batch([30], [2], 4, 2, 256, False, seed=22, width=65536)
    b.lens[0] = 2 ** 24
    b.table[0, -1] = 0
    check_append(hyq, gpu_ctx, b, False)


def test_append_without_a_page(gpu_ctx, hyq):
    """Rows whose table entry is missing or out of range, or whose position is
    negative or past the table, write nothing; their queries are formed."""
    b = R.Batch([20, 40, 5], [4, 3, 2], 4, 2, 16, True, seed=23)
    b.table[0, 1], b.table[1, 2] = -1, b.pages
    check_append(hyq, gpu_ctx, b, True)
    k = np.ones((b.rows, 2, D), np.float32)
    ones, freq = np.ones(D, np.float32), np.zeros(64, np.float32)
    b.lens[:] = [2, 2 ** 31 - 1, -9]
    b.table[0] = -1
    _, pool = append(hyq, gpu_ctx, b, k, k, ones, ones, freq, 1e-5, False)
    assert np.array_equal(pool[0], b.pool, equal_nan=True)


def test_append_agrees_with_the_contiguous_cache(gpu_ctx, hyq):
    """One slot whose pages lie in order against hyq_rope_norm_append_d at
    positions where both angles' products are exact: the same function."""
    heads, kvh, n = 4, 2, 3
    b = R.Batch([n], [n], heads, kvh, 16, False, seed=24)
    r = b.rng
    k, v = (r.normal(0, 1, (n, kvh, D)).astype(np.float32) for _ in range(2))
    qn, kn = (r.normal(1, 0.1, D).astype(np.float32) for _ in range(2))
    freq = (2.0 ** -np.arange(64)).astype(np.float32)
    q_out, pool = append(hyq, gpu_ctx, b, k, v, qn, kn, freq, 1e-5, False)
    kc, vc = (gpu_ctx.array(np.zeros((16, kvh, D), np.float32)) for _ in range(2))
    x = {m: gpu_ctx.array(a) for m, a in dict(qn=qn, kn=kn, freq=freq).items()}
    for i in range(n):
        q, ki, vi = gpu_ctx.array(b.q[i]), gpu_ctx.array(k[i]), gpu_ctx.array(v[i])
        pos = gpu_ctx.array(np.array([i], np.int32))
        hyq.check(hyq.lib().hyq_rope_norm_append_d(
            gpu_ctx.handle, q.ptr, ki.ptr, vi.ptr, x["qn"].ptr, x["kn"].ptr, x["freq"].ptr,
            pos.ptr, heads, kvh, D, ctypes.c_float(1e-5), kc.ptr, vc.ptr))
        # both round the angle, its functions, the rotation and the norm alone: twice 80 U
        assert np.allclose(q.numpy().reshape(heads, D), q_out[i], rtol=0, atol=160 * R.U * 4)
    page = pool[0, b.table[0, 0]]
    assert np.allclose(kc.numpy()[:n], page[0, :, :n].transpose(1, 0, 2), rtol=0,
                       atol=160 * R.U * 4)
    assert np.array_equal(vc.numpy()[:n], page[1, :, :n].transpose(1, 0, 2))
