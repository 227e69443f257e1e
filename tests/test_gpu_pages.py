"""The pages' bookkeeping on the GPU against a step-by-step model
(tests/paged_ref.py): forks, trims, frees, extensions with copies on write,
exhausted pools and compactions, in place and into other arrays. Every result
is exact."""
import ctypes

import numpy as np
import pytest

import paged_ref as R

pytestmark = pytest.mark.gpu


class Device:
    """A pool whose every token carries one number, over layers and heads."""

    def __init__(self, hyq, ctx, pages, seqs, width, pt, layers=2, kvh=2, dtype=0):
        self.hyq, self.ctx, self.L = hyq, ctx, hyq.lib()
        self.kl = hyq.KvLayout(dtype, layers, kvh, 128, pt, pages, seqs, width)
        self.ref = ctypes.byref(self.kl)
        self.shape = (layers, pages, 2, kvh, pt, 128)
        self.type = np.float16 if dtype else np.float32
        self.table = ctx.array(np.full((seqs, width), -1, np.int32))
        self.len = ctx.array(np.zeros(seqs, np.int32))
        self.refs = ctx.array(np.zeros(pages, np.int32))
        self.status = ctx.array(np.full(seqs, -9, np.int32))
        self.live = ctx.empty(1, np.int32)
        self.need = self.L.hyq_pages_scratch_bytes(self.ref)
        self.scratch = ctx.array(np.full(self.need, 0xAB, np.uint8))
        self.pool = ctx.empty(self.shape, self.type)

    def put(self, m):
        """The model's state; data [pages][pt] spread over layers and heads."""
        self.table.copy_from(m.table)
        self.len.copy_from(m.lens)
        self.refs.copy_from(m.refs)
        self.pool.copy_from(self.spread(m.data))

    def spread(self, data):
        l, p, two, h, t, d = self.shape
        out = np.broadcast_to(data[None, :, None, None, :, None], self.shape).astype(self.type)
        out += np.arange(l).reshape(-1, 1, 1, 1, 1, 1).astype(self.type) * 128
        out[:, :, 1] += 512
        out += np.arange(h).reshape(1, 1, 1, -1, 1, 1).astype(self.type) * 64
        return out

    def other(self, a):
        return self.ctx.array(np.full(a.shape, -77, np.int32))

    def fork(self, parent, keep):
        t, n = self.other(self.table), self.other(self.len)
        p = self.ctx.array(np.asarray(parent, np.int32))
        k = None if keep is None else self.ctx.array(np.asarray(keep, np.int32))
        self.hyq.check(self.L.hyq_pages_fork_d(self.ctx.handle, self.ref, p.ptr,
                                               k.ptr if k else None, self.table.ptr, self.len.ptr,
                                               t.ptr, n.ptr, self.refs.ptr))
        self.ctx.sync()
        self.table, self.len = t, n

    def extend(self, add, in_place):
        a = self.ctx.array(np.asarray(add, np.int32))
        t, n, r = ((self.table, self.len, self.refs) if in_place else
                   tuple(self.other(x) for x in (self.table, self.len, self.refs)))
        self.hyq.check(self.L.hyq_pages_extend_d(
            self.ctx.handle, self.ref, self.pool.ptr, a.ptr, self.table.ptr, self.len.ptr,
            self.refs.ptr, t.ptr, n.ptr, r.ptr, self.status.ptr, self.scratch.ptr, self.need))
        self.ctx.sync()
        self.table, self.len, self.refs = t, n, r
        return self.status.numpy()

    def compact(self, in_place):
        t, r = (self.table, self.refs) if in_place else (self.other(self.table),
                                                         self.other(self.refs))
        self.hyq.check(self.L.hyq_pages_compact_d(
            self.ctx.handle, self.ref, self.pool.ptr, self.table.ptr, self.refs.ptr, t.ptr, r.ptr,
            self.live.ptr, self.scratch.ptr, self.need))
        self.ctx.sync()
        self.table, self.refs = t, r
        return int(self.live.numpy()[0])

    def check(self, m, pool=True):
        assert np.array_equal(self.len.numpy(), m.lens)
        assert np.array_equal(self.refs.numpy(), m.refs)
        assert np.array_equal(self.table.numpy(), m.table)
        if pool:
            assert np.array_equal(self.pool.numpy(), self.spread(m.data))


def model(pages, seqs, width, pt, seed):
    r = np.random.default_rng(seed)
    return R.Pages(np.full((seqs, width), -1, np.int32), np.zeros(seqs, np.int32), pages, pt,
                   r.integers(0, 60, (pages, pt)).astype(np.float32))


@pytest.mark.parametrize("pages,seqs,width,pt,dtype", [(40, 6, 5, 16, 0), (90, 12, 9, 32, 1),
                                                      (7, 5, 3, 16, 0), (1, 1, 1, 256, 1)])
def test_random_steps(gpu_ctx, hyq, pages, seqs, width, pt, dtype):
    """Steps in any order; what a page's unfilled rows hold is part of the
    comparison, so a copy touches the filled rows and nothing else."""
    m = model(pages, seqs, width, pt, seed=pages)
    d = Device(hyq, gpu_ctx, pages, seqs, width, pt, dtype=dtype)
    d.put(m)
    r = np.random.default_rng(pages + 1)
    seen = set()
    for step in range(60):
        kind = r.choice(["extend", "extend", "one", "fork", "beams", "trim", "compact"])
        if kind in ("extend", "one"):
            add = (np.ones(seqs, int) if kind == "one" else
                   r.choice([0, 1, 2, pt - 1, pt, pt + 1, 3 * pt, -3, 2 ** 31 - 1], seqs))
            want = m.extend(add)
            got = d.extend(add, in_place=bool(step % 2))
            assert np.array_equal(got, want), (step, add)
            seen |= set(want.tolist())
        elif kind == "compact":
            assert d.compact(in_place=bool(step % 2)) == m.compact()
        else:
            parent = np.arange(seqs)
            if kind != "trim":
                change = r.random(seqs) < (0.3 if kind == "fork" else 0.8)
                parent[change] = r.integers(-1 if kind == "fork" else 0, seqs, change.sum())
                if kind == "fork" and r.random() < 0.3:
                    parent[r.integers(0, seqs)] = r.choice([seqs, 2 ** 31 - 1, -2 ** 31])
            keep = r.integers(-2, width * pt + 5, seqs) if kind == "trim" else None
            m.fork(parent, keep)
            d.fork(parent, keep)
        d.check(m)
    assert 0 in seen and (len(seen) > 1 or pages > 60)


def test_shared_last_page(gpu_ctx, hyq):
    """Four beams of one parent extend: three copies and the first keeps. With
    one of them standing still all that extend copy. After a trim the one that
    holds most of the page keeps it."""
    m = model(30, 4, 4, 16, seed=1)
    d = Device(hyq, gpu_ctx, 30, 4, 4, 16)
    d.put(m)
    for add, parent, keep in ([(21, 0, 0, 0), None, None], [None, (0, 0, 0, 0), None],
                              [(1, 1, 1, 1), None, None], [None, (2, 2, 2, 2), None],
                              [(0, 1, 1, 1), None, None], [None, (1, 1, 1, 1), (20, 22, 18, 22)],
                              [(1, 1, 1, 1), None, None]):
        if add is None:
            m.fork(parent, keep)
            d.fork(parent, keep)
        else:
            assert np.array_equal(d.extend(add, True), m.extend(np.array(add)))
        d.check(m)
    first = m.table[:, 0]
    assert len(set(first.tolist())) == 1 and len(set(m.table[:, 1].tolist())) == 4


def test_an_exhausted_pool(gpu_ctx, hyq):
    """Slots are served in order; those that no longer fit stay as they were,
    also the sharers of a page whose keeper was served."""
    m = model(3, 4, 4, 16, seed=2)
    d = Device(hyq, gpu_ctx, 3, 4, 4, 16)
    d.put(m)
    for add in ((5, 0, 0, 0), (0, 0, 0, 0)):
        assert np.array_equal(d.extend(add, True), m.extend(np.array(add)))
    m.fork([0, 0, 0, 0], None)
    d.fork([0, 0, 0, 0], None)
    got = d.extend((1, 1, 1, 1), True)
    assert got.tolist() == [0, 0, 0, 1] and np.array_equal(got, m.extend(np.array([1, 1, 1, 1])))
    d.check(m)
    # (slots 0 and 3 still share a page; slot 0 holds more of it and goes on in it)
    got = d.extend((1, 1, 1, 12), True)
    assert got.tolist() == [0, 0, 0, 1] and np.array_equal(got, m.extend(np.array([1, 1, 1, 12])))
    d.check(m)


@pytest.mark.parametrize("in_place", [False, True])
def test_large_tables(gpu_ctx, hyq, in_place):
    """More slots and pages than one workgroup has threads."""
    pages, seqs, width, pt = 5000, 1500, 40, 16
    m = model(pages, seqs, width, pt, seed=3)
    d = Device(hyq, gpu_ctx, pages, seqs, width, pt, layers=1, kvh=1, dtype=1)
    r = np.random.default_rng(4)
    m.data[:] = r.integers(0, 60, m.data.shape)
    d.put(m)
    for step in range(3):
        add = r.integers(0, 60, seqs)
        assert np.array_equal(d.extend(add, in_place), m.extend(add))
        d.check(m, pool=False)
        parent = np.where(r.random(seqs) < 0.5, r.integers(-1, seqs, seqs), np.arange(seqs))
        m.fork(parent, None)
        d.fork(parent, None)
        d.check(m, pool=False)
        assert np.array_equal(d.extend(np.ones(seqs), in_place), m.extend(np.ones(seqs, int)))
        d.check(m)
        m.fork(np.where(r.random(seqs) < 0.4, -1, np.arange(seqs)), None)
        d.fork(np.where(m.lens > 0, np.arange(seqs), -1), None)
        d.check(m)
        assert d.compact(in_place) == m.compact()
        d.check(m)


@pytest.mark.parametrize("pages,seqs,width", [(4096, 1024, 16), (4096, 1024, 17), (4097, 1024, 16),
                                              (4096, 1025, 15), (4095, 1023, 5)])
def test_where_the_small_forms_end(gpu_ctx, hyq, pages, seqs, width):
    """Pools and tables on both sides of what one workgroup's counts hold."""
    pt = 16
    m = model(pages, seqs, width, pt, seed=6)
    d = Device(hyq, gpu_ctx, pages, seqs, width, pt, layers=1, kvh=1, dtype=1)
    r = np.random.default_rng(7)
    d.put(m)
    for step in range(2):
        add = r.integers(0, 40, seqs)
        assert np.array_equal(d.extend(add, True), m.extend(add))
        parent = np.where(r.random(seqs) < 0.6, r.integers(-1, seqs, seqs), np.arange(seqs))
        keep = None if step else r.integers(0, width * pt, seqs)
        m.fork(parent, keep)
        d.fork(parent, keep)
        d.check(m, pool=False)
        add = r.integers(0, 3, seqs)
        assert np.array_equal(d.extend(add, False), m.extend(add))
        d.check(m)


def test_wrong_entries_and_counts(gpu_ctx, hyq):
    """Ids outside the pool, negative lengths and counts that fit no table make
    no access outside the arrays, and slots beside them stay right."""
    m = model(20, 4, 4, 16, seed=5)
    d = Device(hyq, gpu_ctx, 20, 4, 4, 16)
    d.put(m)
    add = np.array([20, 17, 5, 30])
    m.extend(add)
    d.extend(add, True)
    table = m.table.copy()
    table[1, 1], table[2, 0] = 10 ** 6, -5
    d.table.copy_from(table)
    d.len.copy_from(np.array([20, 17, -4, 2 ** 31 - 1], np.int32))
    d.refs.copy_from(np.where(m.refs > 0, m.refs, 0) + (np.arange(20) == 9) * 5 -
                     (np.arange(20) == 10) * 3)
    d.fork([0, 1, 2, 3], None)
    assert d.len.numpy().tolist() == [20, 17, 0, 64]
    d.extend([1, 1, 1, 1], True)
    d.compact(True)
    d.fork([0, 0, -1, -1], [1, 40, 0, 0])
    assert d.len.numpy().tolist() == [1, 21, 0, 0]


def test_cache_class(gpu_ctx, hyq):
    """PagedCache drives the same calls."""
    c = hyq.PagedCache(gpu_ctx, layers=1, kv_heads=1, pages=8, seqs=3, context=64, page_tokens=16)
    assert c.extend([20, 0, 3]).tolist() == [0, 0, 0]
    c.fork([0, 0, 2])
    assert c.lengths().tolist() == [20, 20, 3]
    assert c.extend([1, 1, 70]).tolist() == [0, 0, 2]
    assert c.table.numpy().tolist() == [[0, 1, -1, -1], [0, 3, -1, -1], [2, -1, -1, -1]]
    c.fork([-1, 1, 2], [0, 17, 3])
    assert c.compact() == 3
    assert c.table.numpy().tolist() == [[-1] * 4, [0, 1, -1, -1], [2, -1, -1, -1]]
    with pytest.raises(ValueError):
        c.extend([1, 2])


def test_cache_class_keeps_its_scratch(gpu_ctx, hyq):
    """A larger attention call takes a larger scratch and leaves the first one,
    which a captured graph may hold, allocated; a refused call says why."""
    c = hyq.PagedCache(gpu_ctx, layers=1, kv_heads=1, pages=4, seqs=1, context=64, page_tokens=16)
    c.extend([50])
    c.pool.copy_from(np.zeros(c.pool.nbytes, np.uint8))
    q = gpu_ctx.array(np.ones((50, 2, 128), np.float32))
    out = gpu_ctx.array(np.ones((50, 2, 128), np.float32))
    for n in (1, 50, 20):
        start = gpu_ctx.array(np.array([0, n], np.int32))
        c.attention_d(0, start.ptr, n, n, 2, q.ptr, out.ptr)
        assert np.all(out.numpy()[:n] == 0)
    assert len(c._attention) == 2 and all(x.ptr for x in c._attention)
    with pytest.raises(ValueError, match="0 rows"):
        c.attention_d(0, start.ptr, 0, 1, 2, q.ptr, out.ptr)
