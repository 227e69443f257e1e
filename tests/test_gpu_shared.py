"""Attention over prefixes that several slots share, on the GPU: the plan against a
plain one, the results against the 64-bit forms of tests/paged_ref.py and
tests/paged_q8_ref.py."""
import ctypes

import numpy as np
import pytest

import paged_q8_ref as Q
import paged_ref as R
from test_gpu_paged_q8 import far
from test_gpu_serving import captured, hip, ok

pytestmark = pytest.mark.gpu
D = R.D
KINDS = ["F32", "F16", "Q8"]
# (heads, kv heads): 1, 2, 3, 4, 8 and 16 query heads per KV head
HEADS = [(2, 2), (4, 2), (6, 2), (16, 4), (8, 1), (16, 1)]


def batch(kind, lens, news, heads, pt, seed, **kw):
    if kind == "Q8":
        return Q.BatchQ8(lens, news, *heads, pt, seed=seed, **kw)
    return R.Batch(lens, news, *heads, pt, kind == "F16", seed=seed, **kw)


def layout(hyq, b):
    kind = hyq.KV_Q8 if hasattr(b, "bytes") else hyq.F16 if b.f16 else hyq.F32
    return hyq.KvLayout(kind, 1, b.kvh, D, b.pt, b.pages, b.seqs, b.width)


class Call:
    """The plan and the attention of a batch, its buffers filled with NaNs."""

    def __init__(self, hyq, ctx, b, max_rows=None, group=None):
        self.hyq, self.ctx, self.b, self.L = hyq, ctx, b, hyq.lib()
        self.most = max_rows or max(1, int(b.news.max()))
        self.kl = layout(hyq, b)
        self.k = ctypes.byref(self.kl)
        self.d = {n: ctx.array(a) for n, a in dict(
            pool=getattr(b, "bytes", b.pool), table=b.table, len=b.lens, start=b.start,
            q=b.q).items()}
        self.group = None if group is None else ctx.array(np.array(group, np.int32))
        self.np = self.L.hyq_paged_shared_plan_bytes(self.k, b.rows, b.heads)
        self.ns = self.L.hyq_paged_shared_attention_scratch_bytes(self.k, b.rows, self.most, b.heads)
        assert self.np and self.ns
        self.plan = ctx.array(np.full(self.np, 0xFF, np.uint8))
        self.scratch = ctx.array(np.full(self.ns, 0xFF, np.uint8))
        self.out = ctx.array(np.full((b.rows + 1, b.heads, D), -7, np.float32))

    def make(self, least=0):
        """(least: None for the rule of the call without it)"""
        args = [self.ctx.handle, self.k, self.group.ptr if self.group else None,
                self.d["table"].ptr, self.d["len"].ptr, self.d["start"].ptr, self.b.rows,
                self.b.heads]
        if least is None:
            rc = self.L.hyq_paged_shared_plan_d(*args, self.plan.ptr, self.np)
        else:
            rc = self.L.hyq_paged_shared_plan_least_d(*args, least, self.plan.ptr, self.np)
        self.hyq.check(rc)
        return self

    def enqueue(self):
        self.hyq.check(self.L.hyq_paged_shared_attention_d(
            self.ctx.handle, self.k, self.d["pool"].ptr, 0, self.d["table"].ptr, self.d["len"].ptr,
            self.d["start"].ptr, self.b.rows, self.most, self.b.heads, self.plan.ptr, self.np,
            self.d["q"].ptr, self.scratch.ptr, self.ns, self.out.ptr))

    def result(self):
        out = self.out.numpy()
        assert np.all(out[-1] == -7), "memory behind the output changed"
        return out[:-1]

    def attend(self):
        self.enqueue()
        return self.result()

    def skips(self):
        """What the plan leaves to the slots' groups: its [seqs] ints behind the first
        256 bytes."""
        return self.plan.numpy()[256:256 + 4 * self.b.seqs].view(np.int32)


def plain_skips(b, group=None):
    few, first = 16 // (b.heads // b.kvh), {}
    run, lead = np.zeros(b.seqs, int), np.full(b.seqs, -1)
    own = np.maximum(b.lens - b.news, 0) // b.pt
    for s in range(b.seqs):
        page = b.table[s, 0]
        if not 1 <= b.news[s] <= few or own[s] < 1 or not 0 <= page < b.pages:
            continue
        key = page if group is None else group[s]
        if key < 0:
            continue
        lead[s] = first.setdefault(key, s)
        n = min(own[s], own[lead[s]])
        same = (b.table[s, :n] == b.table[lead[s], :n]) & (b.table[s, :n] >= 0)
        same &= b.table[s, :n] < b.pages
        run[s] = own[s] if lead[s] == s else (n if same.all() else same.argmin())
    skip = np.zeros(b.seqs, int)
    for l in set(lead[lead >= 0]):
        who = np.flatnonzero(lead == l)
        saves = [(int((run[who] >= run[s]).sum() - 1) * int(run[s]), int(run[s])) for s in who]
        best = max(saves)
        if best[0] > 0:
            skip[who[run[who] >= best[1]]] = best[1] * b.pt
    return skip


def check(b, got, rows=None):
    want, tol = b.attention()
    for s in range(b.seqs):
        for r in range(b.start[s], b.start[s + 1]):
            err = np.abs(got[r] - want[r]).max(-1)
            assert np.all(err <= tol[r]), (
                f"slot {s} (len {b.lens[s]}, {b.news[s]} new) row {r - b.start[s]}: "
                f"{err.max():.3e} > {tol[r][err.argmax()]:.3e}")
    assert np.all(got[b.new:] == -7), "rows behind the last slot changed"


def share(b, members, pages):
    """Slots of `members` name the pages of the first of them for their first ones."""
    for s in members[1:]:
        b.table[s, :pages] = b.table[members[0], :pages]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("pt", [16, 64, 256])
def test_a_group(gpu_ctx, hyq, heads, pt, kind):
    """Slots of one to as many new rows as the form takes behind three common pages,
    their own parts of one position up to pages, a slot beside them."""
    few = 16 // (heads[0] // heads[1])
    news = [1, few, 1, max(1, few // 2), 1, 1]
    lens = [3 * pt + x + n for x, n in zip([0, 5, pt, 70, 1, 0], news)]
    lens[5] = 40
    b = batch(kind, lens, news, heads, pt, seed=pt + heads[0], tail=2)
    share(b, [0, 1, 2, 3, 4], 3)
    c = Call(hyq, gpu_ctx, b).make()
    assert np.array_equal(c.skips(), [3 * pt] * 5 + [0])
    check(b, c.attend())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("pt", [16, 32, 64])
def test_groups_beside_others(gpu_ctx, hyq, pt, kind):
    """Several groups mixed among slots without new rows, prompts, slots of one page
    in common, slots without pages, and prefixes that are no whole steps."""
    r = np.random.default_rng(pt)
    news = r.choice([1, 1, 2, 0, 4, 30], 40)
    lens = news + 5 * pt + r.integers(0, 90, 40)
    lens[7], lens[8] = news[7], 0
    news[8] = 0
    b = batch(kind, lens, news, (8, 2), pt, seed=pt, tail=3)
    share(b, list(range(0, 40, 4)), 5)
    share(b, list(range(1, 40, 4)), 3)
    share(b, list(range(2, 40, 8)), 1)
    b.table[30, :] = -1
    c = Call(hyq, gpu_ctx, b).make()
    want = plain_skips(b)
    assert (want > 0).sum() > 10 and np.array_equal(c.skips(), want)
    check(b, c.attend())


@pytest.mark.parametrize("kind", KINDS)
def test_more_rows_than_a_block(gpu_ctx, hyq, kind):
    """A group whose rows fill several blocks, a long prefix cut into many pieces, slot
    borders inside blocks."""
    news = [3, 1, 2, 5] * 20
    b = batch(kind, [1300 + n + i for i, n in enumerate(news)], news, (3, 1), 32, seed=4, tail=1)
    share(b, list(range(80)), 40)
    c = Call(hyq, gpu_ctx, b).make()
    assert np.all(c.skips() == 40 * 32)
    check(b, c.attend())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("pt,heads", [(64, (16, 4)), (32, (6, 2))], ids=str)
def test_prefixes_of_many_tiles(gpu_ctx, hyq, pt, heads, kind):
    """Groups whose blocks of 16 rows would have more tiles than the plan gives the
    few-row form: blocks of 128 rows by the tile form, more than one and partly filled,
    one of a prefix that is no whole steps, with slots beside them."""
    r = np.random.default_rng(pt)
    kvh = heads[1]
    most = {"Q8": 12288 * 32, "F32": 6500 * 16}.get(kind, 4096 * 16)
    few = 16 // (heads[0] // heads[1])
    news = np.where(np.arange(75) % 9 == 8, 0, r.integers(1, 3, 75))
    blocks = -(-int((news[:60] > 0).sum()) // (few // 2))  # of 16 rows, of the larger group
    pages = int(1.1 * most / kvh / blocks / pt) + 1
    lens = news + pages * pt + r.integers(0, 30, 75)
    lens[60:] = news[60:] + (pages // 2) * pt + r.integers(0, 30, 15)
    b = batch(kind, lens, news, heads, pt, seed=pt, tail=1)
    share(b, list(range(60)), pages)
    share(b, [60, 61, 63, 64], pages // 2 - 1)
    c = Call(hyq, gpu_ctx, b).make()
    assert np.array_equal(c.skips(), plain_skips(b))
    head = c.plan.numpy()[:16].view(np.int32)
    assert head[0] >= 2 and head[1] > head[0] and head[3] == 0  # blocks, their pieces, not narrow
    check(b, c.attend())


def alike(b, seqs, pages, seed):
    """A batch of many slots of one new token that name the pages of b's only slot: the
    first `pages` whole, and one to 30 positions of the next."""
    r = np.random.default_rng(seed)
    b.seqs, b.table = seqs, np.repeat(b.table, seqs, 0)
    b.lens = (pages * b.pt + 1 + np.arange(seqs) % 30).astype(np.int32)
    b.news = np.ones(seqs, np.int32)
    b.start = np.arange(seqs + 1, dtype=np.int32)
    b.new = b.rows = seqs
    b.q = np.resize(b.q[0], (seqs, b.heads, D)) + r.normal(0, 0.5, (seqs, b.heads, D)).astype(
        np.float32) * (np.abs(b.q[0]).max() > 0)
    return b


# tiles over all KV heads up to which blocks are narrow, and a tile's positions
MOST_NARROW = {"F32": (6500, 16), "F16": (3500, 16), "Q8": (8192, 32)}


@pytest.mark.parametrize("over", [0, 1], ids=["narrow", "wide"])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,seqs", [((16, 4), 32), ((6, 2), 45)], ids=str)
def test_the_border_of_narrow_blocks(gpu_ctx, hyq, heads, seqs, kind, over):
    """As many tiles as blocks of 16 rows may have, and a page's more: either form's
    results."""
    most, tile = MOST_NARROW[kind]
    blocks = -(-seqs // (16 // (heads[0] // heads[1])))
    pages = most // (blocks * heads[1]) + over
    b = alike(batch(kind, [pages * tile + 30], [1], heads, tile, seed=27), seqs, pages, seed=28)
    c = Call(hyq, gpu_ctx, b).make()
    assert np.all(c.skips() == pages * tile)
    head = c.plan.numpy()[:16].view(np.int32)
    assert head[3] == 1 - over and (over or head[0] == blocks)
    check(b, c.attend())


def not_finite(kind, b, where, value):
    """Puts `value` into keys or values (where[1]) of a page's place and head: number 7,
    of an 8-bit page the scale (a NaN, whatever the value)."""
    page, x, h, place = where
    if kind == "Q8":
        b.scales[page, x, h, place] = np.nan
        b.bytes = Q.join(b.codes, b.scales)
    else:
        b.pool[page, x, h, place, 7] = value


def without(b, where):
    """The 64-bit form over all positions but that of a place."""
    seen = b.kv

    def kv(s, h):
        k, v, ok = seen(s, h)
        at = np.flatnonzero(b.table[s] == where[0])
        for page in at:
            p = page * b.pt + where[3]
            if p < len(ok):
                ok = ok.copy()
                ok[p] = False
        return k, v, ok

    b.kv = kv
    try:
        return b.attention()
    finally:
        del b.kv


@pytest.mark.parametrize("form", ["narrow", "wide"])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("pt", [16, 64])
def test_numbers_of_a_prefix_that_are_not_finite(gpu_ctx, hyq, pt, kind, form):
    """In the common pages of one of two groups, in whole steps and in a last step of
    which the prefix has a part, in narrow and in wide blocks: keys reach their head's
    whole rows of that group, values one dim of them, and no other number changes. A
    value that f32 holds and f16 does not is finite in narrow blocks and no number in
    wide ones. An infinite key's score may be minus infinity, its weight exp(-inf) = 0:
    such a row may also be as if the position were not there."""
    seqs, rep, kvh = 24, 8, 2  # (narrow blocks of two slots)
    pages = (5 if pt == 16 else 3) if form == "narrow" else (
        MOST_NARROW[kind][0] // (2 * 6) * MOST_NARROW[kind][1] // pt + 1)
    pages += pt == 16 and pages % 4 == 0  # (the last step of 64 positions in part)
    b = batch(kind, [pages * pt + 30] * 2, [1] * 2, (rep * kvh, kvh), pt, seed=29)
    table, half = b.table.copy(), seqs // 2
    b = alike(b, seqs, pages, seed=30)
    b.table = np.concatenate([np.repeat(table[:1], half, 0), np.repeat(table[1:], half, 0)])

    def attend():
        c = Call(hyq, gpu_ctx, b).make()
        assert np.all(c.skips() == pages * pt)
        assert c.plan.numpy()[:16].view(np.int32)[3] == (form == "narrow")
        return c.attend()

    clean = attend()
    n = pages * pt
    values = [np.nan] if kind == "Q8" else [np.inf, np.nan] + [1e5] * (kind == "F32")
    for value in values:
        for at in (3, n - 2):
            for x in (0, 1):
                where = (table[0, at // pt], x, 1, at % pt)
                kept = b.scales.copy() if kind == "Q8" else b.pool[where].copy()
                not_finite(kind, b, where, value)
                got = attend()
                if kind == "Q8":
                    b.scales = kept
                    b.bytes = Q.join(b.codes, b.scales)
                else:
                    b.pool[where] = kept
                bad = np.zeros(got.shape, bool)
                bad[:half, rep:] = True
                if x and kind != "Q8":
                    bad[..., :7] = bad[..., 8:] = False
                none = np.zeros(got.shape[:2], bool)
                if x == 0 and value == np.inf:
                    none = bad.all(-1) & np.isfinite(got).all(-1)
                    assert np.all(b.q[..., 7][none] < 0), (value, at)
                if none.any():
                    want, tol = without(b, where)
                    assert np.all(np.abs(got - want).max(-1)[none] <= tol[none]), (value, at)
                if value == 1e5 and form == "narrow":
                    assert np.isfinite(got).all()
                else:
                    assert not np.isfinite(got[bad & ~none[..., None]]).any(), (value, at, x)
                assert np.array_equal(got[~bad], clean[~bad]), (value, at, x)


@pytest.mark.parametrize("case", ["equal", "jump"])
@pytest.mark.parametrize("over", [0, 1], ids=["narrow", "wide"])
def test_far_values_in_a_prefix(gpu_ctx, hyq, over, case):
    """8-bit values near the end of f32's range in narrow and in wide blocks, whose parts
    are joined with the slots' own."""
    most, tile = MOST_NARROW["Q8"]
    pages = most // (15 * 2) + over  # 15 blocks of two slots, over two heads
    b = Q.BatchQ8([pages * tile + 30], [1], 16, 2, tile, seed=21)
    far(b, case)
    b = alike(b, 30, pages, seed=22)
    c = Call(hyq, gpu_ctx, b).make()
    assert np.all(c.skips() == pages * tile)
    assert c.plan.numpy()[:16].view(np.int32)[3] == 1 - over
    check(b, c.attend())


@pytest.mark.parametrize("kind", KINDS)
def test_the_prefix_that_saves_most(gpu_ctx, hyq, kind):
    """One instruction of a page before several requests' beams: beams that share more
    with the first slot are taken, if they save more; and by groups, each request's."""
    b = batch(kind, [700] * 9, [1] * 9, (4, 2), 64, seed=6)
    share(b, list(range(9)), 1)
    share(b, [0, 1, 2], 9)
    share(b, [3, 4, 5], 8)
    share(b, [6, 8], 7)
    c = Call(hyq, gpu_ctx, b).make()
    assert np.array_equal(c.skips(), [576] * 3 + [0] * 6)  # 18 pages against 8
    check(b, c.attend())
    group = [5, 5, 5, 70000, 70000, 70000, 2, -1, 2]
    c = Call(hyq, gpu_ctx, b, group=group).make()
    assert np.array_equal(c.skips(), [576] * 3 + [512] * 3 + [448, 0, 448])
    assert np.array_equal(c.skips(), plain_skips(b, group))
    check(b, c.attend())
    # a group that has nothing in common, and one of a single slot
    c = Call(hyq, gpu_ctx, b, group=[-1, -1, 1, 1, 9, 9, -3, 4, 3]).make()
    assert np.array_equal(c.skips(), plain_skips(b, [-1, -1, 1, 1, 9, 9, -3, 4, 3]))
    check(b, c.attend())


@pytest.mark.parametrize("kind,least", [(k, 25000) for k in KINDS])
def test_what_is_worth_sharing(gpu_ctx, hyq, kind, least):
    """Nothing is shared where all groups together save less than the given number, or
    the rule's; the results are the same but for rounding."""
    b = batch(kind, [150] * 8, [1] * 8, (4, 2), 16, seed=19)
    share(b, [0, 2, 4], 7)
    share(b, [1, 5, 6, 7], 5)
    skips = plain_skips(b)
    saving = (2 * 7 + 3 * 5) * 16 * 2
    for n, want in ((0, skips), (saving, skips), (saving + 1, 0), (1 << 63, 0), (None, 0)):
        c = Call(hyq, gpu_ctx, b).make(n)
        assert np.all(c.skips() == want), n
        check(b, c.attend())
    # the rule at its number: one group of 26 slots over 4 heads (the plan reads no pool)
    pages = -(-least // (25 * 4 * 16))
    for n, want in ((pages, pages * 16), (pages - 1, 0)):
        b = batch(kind, [40] * 26, [1] * 26, (4, 4), 16, seed=20)
        b.width = pages + 3
        b.table = np.arange(26 * b.width, dtype=np.int32).reshape(26, -1)
        b.pages = 26 * b.width
        b.table[:, :n] = b.table[0, :n]
        b.lens = np.full(26, n * 16 + 5, np.int32)
        assert np.all(Call(hyq, gpu_ctx, b).make(None).skips() == want)


@pytest.mark.parametrize("kind", KINDS)
def test_pages_missing_in_a_prefix(gpu_ctx, hyq, kind):
    """Entries that name no page end what slots have in common."""
    b = batch(kind, [500] * 4, [2] * 4, (4, 1), 32, seed=7)
    share(b, [0, 1, 2, 3], 15)
    b.table[:, 4] = -1
    b.table[:, 9] = b.pages + 3
    c = Call(hyq, gpu_ctx, b).make()
    assert np.all(c.skips() == 4 * 32)
    check(b, c.attend())
    b.table[:, 0] = -1
    c = Call(hyq, gpu_ctx, b).make()
    assert not c.skips().any()
    check(b, c.attend())


@pytest.mark.parametrize("kind", KINDS)
def test_far_scores(gpu_ctx, hyq, kind):
    """All weight in the prefix, and all behind it."""
    for size in (30.0, -30.0):
        b = batch(kind, [260] * 3, [1] * 3, (2, 1), 64, seed=8)
        share(b, [0, 1, 2], 3)
        b.q[:] = 0
        b.q[:, :, 0] = size
        if kind == "Q8":
            b.codes[..., 0] = 0
            b.codes[b.table[0, :3], 0, :, :, 0] = 100
            b.bytes = Q.join(b.codes, b.scales)
        else:
            used = ~np.isnan(b.pool[:, 0, :, :, 0])
            b.pool[:, 0, :, :, 0][used] = 0
            b.pool[b.table[0, :3], 0, :, :, 0] = 3
        check(b, Call(hyq, gpu_ctx, b).make().attend())


def test_numbers_that_are_not_finite(gpu_ctx, hyq):
    """A NaN in a common page reaches all its slots, one in a slot's own page that one."""
    for kind in KINDS:
        b = batch(kind, [200] * 4, [1] * 4, (4, 2), 32, seed=9)
        share(b, [0, 1, 2], 5)
        clean = Call(hyq, gpu_ctx, b).make().attend()
        for page, at, rows in ((b.table[0, 2], 3, [0, 1, 2]), (b.table[1, 6], 1, [1])):
            if kind == "Q8":
                kept = b.scales.copy()
                b.scales[page, 0, 1, at] = np.nan
                b.bytes = Q.join(b.codes, b.scales)
            else:
                kept = b.pool.copy()
                b.pool[page, 0, 1, at, 7] = np.nan
            got = Call(hyq, gpu_ctx, b).make().attend()
            bad = np.zeros((4, 4), bool)
            bad[rows, 2:] = True
            assert not np.isfinite(got[bad]).any(), kind
            assert np.array_equal(got[~bad], clean[~bad]), kind
            if kind == "Q8":
                b.scales = kept
            else:
                b.pool = kept


@pytest.mark.parametrize("kind", KINDS)
def test_fewer_rows_than_the_plan_took(gpu_ctx, hyq, kind):
    """A slot of more new rows than max_rows is left alone, grouped or not."""
    b = batch(kind, [200, 203, 201, 300], [1, 4, 2, 60], (4, 1), 32, seed=11)
    share(b, [0, 1, 2], 5)
    c = Call(hyq, gpu_ctx, b, max_rows=2).make()
    assert np.array_equal(c.skips(), [160, 160, 160, 0])
    got, (want, tol) = c.attend(), b.attention()
    for r in (0, 5, 6):
        assert np.all(np.abs(got[r] - want[r]).max(-1) <= tol[r])
    assert np.all(got[1:5] == -7) and np.all(got[7:] == -7)


def test_many_slots(gpu_ctx, hyq):
    """A table of 4096 slots: 512 groups of seven slots and one of its own."""
    seqs, pt = 4096, 16
    b = R.Batch([1] * 2, [1] * 2, 2, 2, pt, True, seed=1)
    r = np.random.default_rng(12)
    pages = 512 * 3 + seqs
    b.seqs, b.pages, b.width = seqs, pages, 5
    b.pool = r.normal(0, 1, (pages, 2, 2, pt, D)).astype(np.float16)
    b.lens = np.where(np.arange(seqs) % 8 == 7, 9, 3 * pt + 4).astype(np.int32)
    b.news = np.ones(seqs, np.int32)
    b.start = np.arange(seqs + 1, dtype=np.int32)
    b.new = b.rows = seqs
    b.q = r.normal(0, 1, (seqs, 2, D)).astype(np.float32)
    b.table = np.full((seqs, 5), -1, np.int32)
    order = r.permutation(512).repeat(8)
    for s in range(seqs):
        if s % 8 < 7:
            b.table[s, :3] = 3 * order[s] + np.arange(3)
            b.table[s, 3] = 512 * 3 + s
        else:
            b.table[s, 0] = 512 * 3 + s
    c = Call(hyq, gpu_ctx, b).make()
    assert np.array_equal(c.skips(), np.where(np.arange(seqs) % 8 == 7, 0, 3 * pt))
    got = c.attend()
    for s in list(range(0, 24)) + [2047, 2048, 4088, 4095]:
        for h in range(2):
            k, v, _ = b.kv(s, h)
            sc = k @ b.q[s, h].astype(np.float64) / np.sqrt(D)
            w = np.exp(sc - sc.max())
            want = (w[:, None] * v).sum(0) / w.sum()
            tol = R.tolerance((np.abs(k) @ np.abs(b.q[s, h])).max() / np.sqrt(D), np.abs(sc).max(),
                              np.abs(v).max(), len(k))
            assert np.abs(got[s, h] - want).max() <= tol


def test_a_plan_of_another_batch(gpu_ctx, hyq):
    """A plan that is not the batch's, and one of any bytes: no access outside."""
    b = R.Batch([200] * 6, [2] * 6, 8, 2, 32, True, seed=13, tail=3)
    share(b, [0, 1, 2, 3, 4, 5], 6)
    c = Call(hyq, gpu_ctx, b).make()
    plan = c.plan.numpy()
    c.d["len"].copy_from(np.array([3, 0, 200, 1, 90, 7], np.int32))
    c.d["start"].copy_from(np.array([0, 1, 1, 9, 9, 10, 11], np.int32))
    c.attend()
    r = np.random.default_rng(14)
    for i in range(6):
        junk = r.integers(0, 256, plan.size).astype(np.uint8)
        words = junk.view(np.int32)
        if i % 2:  # (small numbers, which bounds do not cut away)
            words[:] = r.integers(-3, 40, words.size)
        words[:2] = [1, r.integers(1, 12)]  # blocks, pieces
        c.plan.copy_from(junk)
        c.attend()


class Guarded:
    """A buffer between two others that are to stay as they are."""
    ROOM = 1 << 16

    def __init__(self, ctx, nbytes):
        self.whole = ctx.array(np.full(nbytes + 2 * self.ROOM, 0xA5, np.uint8))
        self.ptr = self.whole.ptr + self.ROOM

    def intact(self):
        a = self.whole.numpy()
        return np.all(a[:self.ROOM] == 0xA5) and np.all(a[-self.ROOM:] == 0xA5)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,pt", [((8, 2), 32), ((6, 2), 64), ((16, 1), 16)], ids=str)
def test_plans_of_any_bytes(gpu_ctx, hyq, heads, pt, kind):
    """A batch's plan with some numbers exchanged, and plans of small numbers and of any
    bytes: nothing beside the scratch and the output is written, and no input."""
    few = 16 // (heads[0] // heads[1])
    b = batch(kind, [9 * pt + 3] * 6, [min(2, few)] * 6, heads, pt, seed=31, tail=3)
    share(b, [0, 1, 2, 4, 5], 8)
    c = Call(hyq, gpu_ctx, b)
    out = Guarded(gpu_ctx, b.rows * b.heads * D * 4)
    c.scratch, c.out, plan = Guarded(gpu_ctx, c.ns), out, Guarded(gpu_ctx, c.np)
    c.plan = plan
    c.make()
    held = {n: a.numpy() for n, a in c.d.items()}
    true = plan.whole.numpy()[plan.ROOM:-plan.ROOM].copy()
    r = np.random.default_rng(32)
    for i in range(24):
        junk = true.copy()
        words = junk[:junk.size // 4 * 4].view(np.int32)
        if i % 3 == 0:  # (an eighth of the numbers another one)
            at = r.random(words.size) < 0.125
            words[at] = r.integers(-3, 300, at.sum())
        elif i % 3 == 1:
            words[:] = r.integers(-3, 40, words.size)
        else:
            junk[:] = r.integers(0, 256, junk.size)
        words[:2] = r.integers(1, 12, 2)  # blocks, pieces
        words[2:4] = [r.integers(1, 3000), i // 3 % 2]  # workers, narrow
        given = np.concatenate([np.full(plan.ROOM, 0xA5, np.uint8), junk,
                                np.full(plan.ROOM, 0xA5, np.uint8)])
        plan.whole.copy_from(given)
        c.enqueue()
        assert c.scratch.intact() and out.intact(), i
        assert np.array_equal(plan.whole.numpy(), given), i
    for n, a in c.d.items():
        assert np.array_equal(a.numpy().view(np.uint8), held[n].view(np.uint8)), n


@pytest.mark.parametrize("kind", KINDS)
def test_cache(gpu_ctx, hyq, kind):
    """PagedCache: forked slots attend with and without the plan alike; a plan is
    asked for after each step's pages."""
    b = batch(kind, [90], [1], (4, 2), 16, seed=16)
    c = hyq.PagedCache(gpu_ctx, 1, 2, 64, 5, 200, page_tokens=16,
                       dtype={"F32": hyq.F32, "F16": hyq.F16, "Q8": hyq.KV_Q8}[kind])
    r = np.random.default_rng(17)
    one, freq = (gpu_ctx.array(x) for x in (np.ones(D, np.float32),
                                            (10000.0 ** (-np.arange(64) / 64)).astype(np.float32)))
    start = gpu_ctx.array(np.zeros(6, np.int32))

    def step(news):
        first = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
        start.copy_from(first)
        rows = int(first[-1])
        x = [gpu_ctx.array(r.normal(0, 1, (rows, n, D)).astype(np.float32)) for n in (4, 2, 2)]
        out = [gpu_ctx.array(np.full((rows, 4, D), -7, np.float32)) for _ in range(2)]
        assert not c.extend(news).any()
        qo = gpu_ctx.empty((rows, 4, D), np.float32)
        c.append_d(0, start.ptr, rows, 4, *[a.ptr for a in x], one.ptr, one.ptr, freq.ptr, 1e-5,
                   qo.ptr)
        with pytest.raises(ValueError, match="share_d"):
            c.attention_d(0, start.ptr, rows, max(news), 4, qo.ptr, out[0].ptr, shared=True)
        c.share_d(start.ptr, rows, 4, least=0)
        c.attention_d(0, start.ptr, rows, max(news), 4, qo.ptr, out[0].ptr, shared=True)
        c.attention_d(0, start.ptr, rows, max(news), 4, qo.ptr, out[1].ptr)
        a, b = (o.numpy() for o in out)
        assert np.abs(a - b).max() < 2e-5 and np.abs(a).max() > 0.01
        return a, b

    step([70, 0, 0, 0, 0])
    c.fork([0, 0, 0, 0, -1])
    step([1, 1, 1, 1, 33])
    a, b = step([1, 2, 1, 3, 1])
    assert not np.array_equal(a, b)  # (the prefix was summed apart)
    c.fork([3, 0, 1, 4, 4])
    step([1, 1, 1, 1, 1])


def test_captured(gpu_ctx, hyq):
    """A captured plan and attention follow the tables of each replay, with eager work
    between; two graphs with buffers of their own replayed side by side."""
    other = hyq.Context(0)
    try:
        b = R.Batch([200] * 6, [1] * 6, 8, 2, 32, True, seed=18)
        calls = [Call(hyq, gpu_ctx, b) for _ in range(2)]
        graphs = [captured(gpu_ctx, lambda: c.make().enqueue()) for c in calls]
        tables = [b.table.copy() for _ in range(4)]
        for s in range(6):
            tables[1][s, :6] = tables[1][0, :6]
            tables[2][s, :2 + s // 3] = tables[2][s // 3 * 3, :2 + s // 3]
        tables[3][1, :5] = tables[3][4, :5]
        for i in range(6):
            for j, c in enumerate(calls):
                c.d["table"].copy_from(tables[(i + j) % 4])
                c.out.copy_from(np.full(c.out.shape, -7, np.float32))
            gpu_ctx.sync()
            for (_, run), ctx in zip(graphs, (gpu_ctx, other)):
                ok(hip("hipGraphLaunch")(run, ctypes.c_void_p(ctx.stream)))
            other.sync()
            gpu_ctx.sync()
            for j, c in enumerate(calls):
                b.table = tables[(i + j) % 4]
                check(b, c.result())
                eager = Call(hyq, gpu_ctx, b).make().attend()
                assert np.array_equal(eager, c.result())
                assert np.array_equal(c.skips(), plain_skips(b))
        for graph, run in graphs:
            ok(hip("hipGraphExecDestroy")(run))
            ok(hip("hipGraphDestroy")(graph))
    finally:
        other.close()


def test_a_captured_attention_keeps_its_plan(gpu_ctx, hyq):
    """Attention captured without its plan goes by the plan that is made before each
    replay, also after one of another number of heads, whose buffer is larger."""
    c = hyq.PagedCache(gpu_ctx, 1, 2, 64, 4, 200, page_tokens=16)
    c.pool.copy_from(np.random.default_rng(19).integers(0, 40, c.pool.shape).astype(np.uint8))
    start = gpu_ctx.array(np.arange(5, dtype=np.int32))
    q = gpu_ctx.array(np.random.default_rng(20).normal(0, 1, (4, 16, D)).astype(np.float32))
    outs = [gpu_ctx.array(np.full((4, 16, D), -7, np.float32)) for _ in range(3)]
    assert not c.extend([75, 0, 0, 0]).any()
    c.fork([0, 0, 0, 0])
    assert not c.extend([1, 1, 1, 1]).any()

    def attend(out, **kw):
        c.attention_d(0, start.ptr, 4, 1, 16, q.ptr, out.ptr, **kw)

    c.share_d(start.ptr, 4, 16, least=0)
    attend(outs[0], shared=True)
    graph, run = captured(gpu_ctx, lambda: attend(outs[0], shared=True))
    c.share_d(start.ptr, 4, 2, least=0)
    for i in range(3):
        assert not c.extend([1 + 20 * i, 2, 1, 3]).any()
        c.share_d(start.ptr, 4, 16, least=0)
        ok(hip("hipGraphLaunch")(run, ctypes.c_void_p(gpu_ctx.stream)))
        attend(outs[1], shared=True)
        attend(outs[2])
        a, b, plain = (o.numpy() for o in outs)
        assert np.array_equal(a, b)
        assert np.abs(a - plain).max() <= 2e-5 * np.abs(plain).max()
    ok(hip("hipGraphExecDestroy")(run))
    ok(hip("hipGraphDestroy")(graph))


def test_plans_of_two_numbers_of_heads(gpu_ctx, hyq):
    """Each number of heads keeps its plan until the next step's pages, whichever was
    made last; a plan of other rows takes the place of the one before."""
    c = hyq.PagedCache(gpu_ctx, 1, 2, 64, 4, 200, page_tokens=16)
    c.pool.copy_from(np.random.default_rng(23).integers(0, 40, c.pool.shape).astype(np.uint8))
    start, other = (gpu_ctx.array(np.arange(5, dtype=np.int32)) for _ in range(2))
    q = gpu_ctx.array(np.random.default_rng(24).normal(0, 1, (4, 16, D)).astype(np.float32))
    outs = [gpu_ctx.array(np.full((4, 16, D), -7, np.float32)) for _ in range(2)]
    assert not c.extend([75, 0, 0, 0]).any()
    c.fork([0, 0, 0, 0])
    assert not c.extend([1, 1, 1, 1]).any()
    for heads in (16, 2):
        c.share_d(start.ptr, 4, heads, least=0)
    for heads in (16, 2, 16):
        for out, shared in zip(outs, (True, False)):
            c.attention_d(0, start.ptr, 4, 1, heads, q.ptr, out.ptr, shared=shared)
        a, b = (o.numpy().ravel()[:4 * heads * D] for o in outs)
        assert np.abs(a - b).max() <= 2e-5 * np.abs(b).max()
    c.share_d(other.ptr, 4, 16, least=0)
    attend = lambda at, heads: c.attention_d(0, at.ptr, 4, 1, heads, q.ptr, outs[0].ptr,
                                             shared=True)
    attend(other, 16)
    attend(start, 2)
    with pytest.raises(ValueError, match="share_d"):
        attend(start, 16)
    assert not c.extend([1, 1, 1, 1]).any()
    for at, heads in ((other, 16), (start, 2)):
        with pytest.raises(ValueError, match="share_d"):
            attend(at, heads)
