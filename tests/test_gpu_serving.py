"""The paged cache's operators and the sampler as a server runs them: steps of
several sequences, eagerly, captured in a HIP graph, and on two contexts at
once."""
import ctypes

import numpy as np
import pytest

import paged_ref as R

pytestmark = pytest.mark.gpu
D, HEADS, KVH, PT, PAGES, SEQS, STRIDE, VOCAB, LAYERS = 128, 4, 2, 16, 60, 5, 6, 700, 2


class Server:
    """Slots decoded one token a step: fork, extend, and for each layer append
    and attention of rows made from the last token; a token from logits that
    the last layer's output gives. All arrays stay on the device."""

    def __init__(self, hyq, ctx, seed=1, f16=True):
        self.hyq, self.ctx, self.L = hyq, ctx, hyq.lib()
        self.f16 = f16
        r = np.random.default_rng(seed)
        a = lambda x, t=np.float32: ctx.array(np.ascontiguousarray(x, t))
        kl = hyq.KvLayout(hyq.F16 if f16 else hyq.F32, LAYERS, KVH, D, PT, PAGES, SEQS, STRIDE)
        self.layout, self.kl = kl, ctypes.byref(kl)
        pool = r.normal(0, 1, (LAYERS, PAGES, 2, KVH, PT, D))
        table = np.full((SEQS, STRIDE), -1)
        lens = np.array([17, 32, 1, 0, 47])
        ids = iter(r.permutation(PAGES))
        for s in range(SEQS):
            for i in range(-(-lens[s] // PT)):
                table[s, i] = next(ids)
        refs = np.bincount(table[table >= 0], minlength=PAGES)
        self.start0 = dict(pool=pool.astype(np.float16 if f16 else np.float32),
                           table=table.astype(np.int32), len=lens.astype(np.int32),
                           refs=refs.astype(np.int32))
        self.d = {n: ctx.array(x) for n, x in self.start0.items()}
        self.table2, self.len2 = ctx.empty((SEQS, STRIDE), np.int32), ctx.empty(SEQS, np.int32)
        self.status = a(np.zeros(SEQS), np.int32)
        self.parent, self.add = a(np.arange(SEQS), np.int32), a(np.ones(SEQS), np.int32)
        self.start = a(np.arange(SEQS + 1), np.int32)
        self.q = [a(r.normal(0, 1, (SEQS, HEADS, D))) for _ in range(LAYERS)]
        self.k = [a(r.normal(0, 1, (SEQS, KVH, D))) for _ in range(LAYERS)]
        self.v = [a(r.normal(0, 1, (SEQS, KVH, D))) for _ in range(LAYERS)]
        self.norm, self.freq = a(r.normal(1, 0.1, D)), a(10000.0 ** (-np.arange(64) / 64))
        self.qo = ctx.empty((SEQS, HEADS, D), np.float32)
        self.out = a(np.zeros((LAYERS, SEQS, HEADS, D)))
        self.set = [a(np.full(SEQS, 0.8)), a([0, 20, 5, 100, 0], np.int32),
                    a([1, 0.9, 1, 0.7, 0.8]), a([0, 0, 0.1, 0, 0])]
        self.u = a(np.full(SEQS, 0.5))
        self.logits = a(r.normal(0, 3, (SEQS, VOCAB)))
        self.token, self.prob = a(np.zeros(SEQS), np.int32), a(np.zeros(SEQS))
        self.na = self.L.hyq_paged_attention_scratch_bytes(self.kl, SEQS, 1, HEADS)
        self.np = self.L.hyq_pages_scratch_bytes(self.kl)
        self.ns = self.L.hyq_sample_scratch_bytes(SEQS, VOCAB)
        self.scratch = ctx.empty(max(self.na, self.np, self.ns, 16), np.uint8)
        ctx.sync()

    def reset(self):
        for n, x in self.start0.items():
            self.d[n].copy_from(x)

    def step(self):
        L, h, kl, d, x = self.L, self.ctx.handle, self.kl, self.d, self.scratch.ptr
        rc = [L.hyq_pages_fork_d(h, kl, self.parent.ptr, None, d["table"].ptr, d["len"].ptr,
                                 self.table2.ptr, self.len2.ptr, d["refs"].ptr),
              L.hyq_pages_extend_d(h, kl, d["pool"].ptr, self.add.ptr, self.table2.ptr,
                                   self.len2.ptr, d["refs"].ptr, d["table"].ptr, d["len"].ptr,
                                   d["refs"].ptr, self.status.ptr, x, self.np)]
        size = SEQS * HEADS * D * 4
        for l in range(LAYERS):
            rc += [L.hyq_paged_rope_norm_append_d(
                       h, kl, d["pool"].ptr, l, d["table"].ptr, d["len"].ptr, self.start.ptr, SEQS,
                       HEADS, self.q[l].ptr, self.k[l].ptr, self.v[l].ptr, self.norm.ptr,
                       self.norm.ptr, self.freq.ptr, ctypes.c_float(1e-5), 0, self.qo.ptr),
                   L.hyq_paged_attention_d(
                       h, kl, d["pool"].ptr, l, d["table"].ptr, d["len"].ptr, self.start.ptr, SEQS,
                       1, HEADS, self.qo.ptr, x, self.na, self.out.ptr + l * size)]
        rc.append(L.hyq_sample_d(h, self.logits.ptr, SEQS, VOCAB, *[a.ptr for a in self.set],
                                 self.u.ptr, x, self.ns, self.token.ptr, self.prob.ptr))
        for c in rc:
            self.hyq.check(c)

    def state(self):
        self.ctx.sync()
        return [a.numpy() for a in (self.d["table"], self.d["len"], self.d["refs"],
                                    self.d["pool"], self.status, self.out, self.token,
                                    self.prob)]


INPUTS = [(np.arange(SEQS), [1, 1, 1, 0, 1]), ([0, 0, 1, 1, 4], [1, 1, 1, 1, 1]),
          ([0, 1, 2, 3, 0], [1, 1, 1, 1, 1]), ([-1, 1, 2, 2, 4], [20, 1, 1, 1, 1]),
          ([0, 1, 2, 3, 4], [1, 1, 17, 1, 60])]


def feed(server, i, logits):
    parent, add = INPUTS[i % len(INPUTS)]
    server.parent.copy_from(np.array(parent, np.int32))
    server.add.copy_from(np.array(add, np.int32))
    server.logits.copy_from(logits[i])
    server.u.copy_from(np.random.default_rng(i).random(SEQS).astype(np.float32))


def test_steps_against_the_plain_forms(gpu_ctx, hyq):
    """Every step's tables, pool, outputs and tokens against 64-bit forms run
    on the state before it."""
    s = Server(hyq, gpu_ctx, f16=False)
    logits = np.random.default_rng(2).normal(0, 3, (5, SEQS, VOCAB)).astype(np.float32)
    for i in range(5):
        feed(s, i, logits)
        table, lens, refs, pool = (x.copy() for x in s.state()[:4])
        m = R.Pages(table, lens, PAGES, PT, np.zeros((PAGES, PT)))
        names = np.arange(PAGES, dtype=np.float64)[:, None] * PT + np.arange(PT)
        m.data = names.copy()  # which old row a row of the pool now holds
        m.fork(INPUTS[i][0], None)
        status = m.extend(np.array(INPUTS[i][1]))
        s.step()
        got = s.state()
        assert np.array_equal(got[0], m.table) and np.array_equal(got[1], m.lens)
        assert np.array_equal(got[2], m.refs) and np.array_equal(got[4], status)
        src = m.data.astype(int)
        # one row per slot: at the last position of those that hold one
        news = np.ones(SEQS, int)
        for l in range(LAYERS):
            b = R.Batch(np.maximum(m.lens, 1), news, HEADS, KVH, PT, False, 0)
            b.table, b.lens, b.pages, b.width = m.table, m.lens.copy(), PAGES, STRIDE
            old = pool[l].transpose(0, 3, 1, 2, 4).reshape(PAGES * PT, 2, KVH, D)
            b.pool = old[src].transpose(0, 2, 3, 1, 4).astype(np.float32)
            b.q = s.q[l].numpy()
            k, v, w, f = s.k[l].numpy(), s.v[l].numpy(), s.norm.numpy(), s.freq.numpy()
            full = m.lens > 0
            b.news = full.astype(np.int32)  # (a slot of no positions: its row writes nothing)
            b.start = np.arange(SEQS + 1)
            q_out, want_pool = R.append(b, k, v, w, w, f, 1e-5, False)
            close = np.abs(got[3][l] - want_pool) <= 400 * R.U
            assert close.all()
            b.pool, b.q = got[3][l], np.where(full[:, None, None], q_out, 0).astype(np.float32)
            want, tol = b.attention()
            err = np.abs(got[5][l][full] - want[full]).max(-1)
            # the queries' own 80 U (twice: their rounding here too) move scores of
            # at most |q| |k| / sqrt(128) < 40 each, and an output by twice that
            assert np.all(err <= tol[full] + 2 * 160 * R.U * 40)
            assert np.all(got[5][l][~full] == 0)
        t, kk, p, mp = (x.numpy() for x in s.set)
        u = s.u.numpy()
        for r in range(SEQS):
            want, pw = R.sample(logits[i][r], t[r], kk[r], p[r], mp[r], u[r])
            assert got[6][r] == want and abs(got[7][r] - pw) <= 4 * R.U


@pytest.mark.parametrize("f16", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("pages", [3, 4200])
@pytest.mark.parametrize("chunk", [1, 7])
def test_refused_slots_write_nothing(gpu_ctx, hyq, chunk, pages, f16):
    """Beams of one prompt, and a slot at its table's end, in a pool that runs
    out: the new rows of those that extend refuses (of one of them in a page that
    a served beam goes on writing) change no cached row and attend nothing; the
    others' are as if they were alone. (4200 pages: the large form of extend,
    whose other pages a slot of its own holds.)"""
    seqs, stride = 6, max(4, pages - 3)
    c = hyq.PagedCache(gpu_ctx, 1, KVH, pages, seqs, stride * PT, PT,
                       hyq.F16 if f16 else hyq.F32)
    r = np.random.default_rng(chunk)
    f = lambda *n: r.normal(0, 1, n).astype(np.float32)
    pool0 = f(pages, 2, KVH, PT, D).astype(np.float16 if f16 else np.float32)
    c.pool.copy_from(np.frombuffer(pool0.tobytes(), np.uint8))
    hoard = (pages - 3) * PT
    assert c.extend([5, 0, 0, 0, hoard, 0]).tolist() == [0] * 6
    c.fork([0, 0, 0, 0, 4, -1])
    held = c.lengths()
    add = [chunk] * 4 + [stride * PT + 1 - hoard, 0]
    news = np.array([chunk] * 5 + [0], np.int32)
    status = c.extend(add)
    assert status.tolist() == [0, 0, 0, 1, 2, 0]
    start = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
    rows = int(start[-1])
    q, k, v = f(rows, HEADS, D), f(rows, KVH, D), f(rows, KVH, D)
    w, freq = f(D), (10000.0 ** (-np.arange(64) / 64)).astype(np.float32)
    a = [gpu_ctx.array(x) for x in (start, q, k, v, w, freq)]
    qo, out = (gpu_ctx.array(np.full((rows, HEADS, D), -7, np.float32)) for _ in range(2))
    c.append_d(0, a[0].ptr, rows, HEADS, a[1].ptr, a[2].ptr, a[3].ptr, a[4].ptr, a[4].ptr,
               a[5].ptr, 1e-5, qo.ptr)
    c.attention_d(0, a[0].ptr, rows, chunk, HEADS, qo.ptr, out.ptr)
    got = np.frombuffer(c.pool.numpy().tobytes(), pool0.dtype).reshape(pool0.shape)
    table, lens = c.table.numpy(), c.lengths()
    assert np.array_equal(lens, held + np.where(status == 0, add, 0))
    # what is written: the served slots' new positions, nothing else
    fresh = np.zeros(pool0.shape, bool)
    for s in range(3):
        for p in range(lens[s] - chunk, lens[s]):
            fresh[table[s, p // PT], :, :, p % PT] = True
    kept = pool0.copy()  # (the beams' shared positions, copied)
    for s in range(3):
        kept[table[s, 0], :, :, :5] = pool0[table[3, 0], :, :, :5]
    assert np.array_equal(got[~fresh], kept[~fresh])
    b = R.Batch([1] * seqs, [1] * seqs, HEADS, KVH, PT, f16, 0)
    b.table, b.lens, b.news, b.start = table, np.where(status == 0, lens, 0), news, start
    b.pool, b.pages, b.width, b.rows = got, pages, stride, rows
    b.q = qo.numpy()
    want, tol = b.attention()
    o = out.numpy()
    assert np.all(np.abs(o - want).max(-1) <= tol)
    assert np.all(o[3 * chunk:] == 0)


def hip(name):
    """The HIP runtime that libhyq.so uses."""
    lib = ctypes.CDLL("libamdhip64.so")
    fn = getattr(lib, name)
    fn.restype = ctypes.c_int
    return fn


def ok(rc):
    assert rc == 0, rc


def captured(ctx, work):
    P = ctypes.c_void_p
    stream, graph, run = P(ctx.stream), P(), P()
    ok(hip("hipStreamBeginCapture")(stream, 2))  # relaxed
    try:
        work()
    finally:
        rc = hip("hipStreamEndCapture")(stream, ctypes.byref(graph))
    ok(rc)
    ok(hip("hipGraphInstantiate")(ctypes.byref(run), graph, None, None, P(0)))
    return graph, run


@pytest.mark.parametrize("f16", [False, True], ids=["f32", "f16"])
def test_a_captured_step(gpu_ctx, hyq, f16):
    """A whole step in one graph, replayed with new inputs, eager work and
    waits in between: every replay gives the eager step's bits."""
    eager, graphed = Server(hyq, gpu_ctx, f16=f16), Server(hyq, gpu_ctx, f16=f16)
    logits = np.random.default_rng(3).normal(0, 3, (10, SEQS, VOCAB)).astype(np.float32)
    graph, run = captured(gpu_ctx, graphed.step)
    graphed.reset()
    for i in range(10):
        if i == 5:
            eager.reset()
            graphed.reset()
        feed(eager, i, logits)
        feed(graphed, i, logits)
        eager.step()
        want = eager.state()
        ok(hip("hipGraphLaunch")(run, ctypes.c_void_p(gpu_ctx.stream)))
        for a, b in zip(want, graphed.state()):
            assert np.array_equal(a, b, equal_nan=True), i
    ok(hip("hipGraphExecDestroy")(run))
    ok(hip("hipGraphDestroy")(graph))


@pytest.mark.parametrize("f16", [False, True], ids=["f32", "f16"])
def test_a_captured_ragged_batch(gpu_ctx, hyq, f16):
    """Append and attention of prompts, drafts and single tokens in one graph,
    replayed for other splits of the same number of rows, shorter ones among
    them: every replay gives the eager call's bits and leaves the rows behind."""
    ctx, L = gpu_ctx, hyq.lib()
    rows, most, context = 300, 200, 512
    r = np.random.default_rng(6)
    kl = hyq.KvLayout(hyq.F16 if f16 else hyq.F32, 1, KVH, D, PT, 5 * context // PT, 5,
                      context // PT)
    ref = ctypes.byref(kl)
    f = lambda *s: ctx.array(r.normal(0, 1, s).astype(np.float32))
    q, k, v, w, freq = f(rows, HEADS, D), f(rows, KVH, D), f(rows, KVH, D), f(D), f(64)
    pool0 = r.normal(0, 1, (kl.pages, 2, KVH, PT, D)).astype(np.float16 if f16 else np.float32)
    table = ctx.array(r.permutation(kl.pages).reshape(5, -1).astype(np.int32))
    lens, start = ctx.empty(5, np.int32), ctx.empty(6, np.int32)
    pool, qo, out = ctx.array(pool0), ctx.empty((rows, HEADS, D), np.float32), f(rows, HEADS, D)
    need = L.hyq_paged_attention_scratch_bytes(ref, rows, most, HEADS)
    scratch = ctx.empty(need, np.uint8)

    def work():
        hyq.check(L.hyq_paged_rope_norm_append_d(
            ctx.handle, ref, pool.ptr, 0, table.ptr, lens.ptr, start.ptr, rows, HEADS, q.ptr,
            k.ptr, v.ptr, w.ptr, w.ptr, freq.ptr, ctypes.c_float(1e-5), 0, qo.ptr))
        hyq.check(L.hyq_paged_attention_d(
            ctx.handle, ref, pool.ptr, 0, table.ptr, lens.ptr, start.ptr, rows, most, HEADS,
            qo.ptr, scratch.ptr, need, out.ptr))

    graph, run = captured(ctx, work)
    for news, held in (([1, 1, 1, 1, 1], [40, 0, 511, 3, 64]), ([200, 50, 8, 9, 33], [0, 20, 1, 0, 9]),
                       ([0, 200, 0, 100, 0], [5, 312, 0, 0, 0]), ([0, 0, 0, 0, 0], [9, 9, 9, 9, 9]),
                       ([1, 1, 1, 1, 1], [40, 0, 511, 3, 64]), ([60, 60, 60, 60, 60], [100] * 5)):
        got = []
        start.copy_from(np.cumsum([0] + news).astype(np.int32))
        lens.copy_from(np.add(news, held).astype(np.int32))
        for call in (work, lambda: ok(hip("hipGraphLaunch")(run, ctypes.c_void_p(ctx.stream)))):
            pool.copy_from(pool0)
            qo.copy_from(np.full((rows, HEADS, D), 5, np.float32))
            out.copy_from(np.full((rows, HEADS, D), -7, np.float32))
            scratch.copy_from(np.full(need, 0xFF, np.uint8))
            call()
            got.append([a.numpy() for a in (pool, qo, out)])
        n = sum(news)
        for a, b in zip(*got):
            assert np.array_equal(a, b), news
        assert np.all(got[0][2][n:] == -7) and not np.any(got[0][2][:n] == -7)
    ok(hip("hipGraphExecDestroy")(run))
    ok(hip("hipGraphDestroy")(graph))


@pytest.mark.parametrize("f16", [False, True], ids=["f32", "f16"])
def test_a_captured_step_of_the_cache_class(gpu_ctx, hyq, f16):
    """PagedCache's step of one fork, extension, append and attention in a graph,
    replayed for other forks, refused slots among them, with eager calls between:
    every replay gives the eager step's bits."""
    ctx = gpu_ctx
    r = np.random.default_rng(8)
    f = lambda *n: ctx.array(r.normal(0, 1, n).astype(np.float32))
    q, k, v, w, freq = f(SEQS, HEADS, D), f(SEQS, KVH, D), f(SEQS, KVH, D), f(D), f(64)
    start = ctx.array(np.arange(SEQS + 1, dtype=np.int32))
    parent, add = ctx.empty(SEQS, np.int32), ctx.empty(SEQS, np.int32)
    qo, out = f(SEQS, HEADS, D), f(SEQS, HEADS, D)
    pool0 = r.normal(0, 1, (30, 2, KVH, PT, D)).astype(np.float16 if f16 else np.float32)

    def cache():
        c = hyq.PagedCache(ctx, 1, KVH, 30, SEQS, STRIDE * PT, PT, hyq.F16 if f16 else hyq.F32)
        c.pool.copy_from(np.frombuffer(pool0.tobytes(), np.uint8))
        assert not c.extend([17, 32, 1, 0, 47]).any()
        return c

    def step(c):
        c.fork_d(parent.ptr)
        c.extend_d(add.ptr)
        c.append_d(0, start.ptr, SEQS, HEADS, q.ptr, k.ptr, v.ptr, w.ptr, w.ptr, freq.ptr, 1e-5,
                   qo.ptr)
        c.attention_d(0, start.ptr, SEQS, 1, HEADS, qo.ptr, out.ptr)

    eager, graphed = cache(), cache()
    parent.copy_from(np.arange(SEQS, dtype=np.int32))
    add.copy_from(np.zeros(SEQS, np.int32))
    step(graphed)  # (its attention's scratch)
    step(eager)
    for c in (eager, graphed):
        c.pool.copy_from(np.frombuffer(pool0.tobytes(), np.uint8))
    graph, run = captured(ctx, lambda: step(graphed))
    seen = set()
    long = (np.arange(SEQS), [1, STRIDE * PT + 1, 1, 1, 1])  # (no slot has that much room)
    for i, (p, a) in enumerate([INPUTS[i % len(INPUTS)] for i in range(12)] + [long, long]):
        got = []
        for c, call in ((eager, lambda: step(eager)),
                        (graphed, lambda: ok(hip("hipGraphLaunch")(run, ctypes.c_void_p(ctx.stream))))):
            if i == 6:  # (a slot freed between, by the calls that wait)
                c.fork([0, 1, -1, 3, 4])
                assert not c.extend([0, 0, 3, 0, 0]).any()
            parent.copy_from(np.array(p, np.int32))
            add.copy_from(np.array(a, np.int32))
            out.copy_from(np.full((SEQS, HEADS, D), -7, np.float32))
            call()
            got.append([x.numpy() for x in (c.table, c.len, c.refs, c.status, c.pool, qo, out)])
        for x, y in zip(*got):
            assert np.array_equal(x, y), i
        refused = got[0][3] != 0
        seen |= set(got[0][3].tolist())
        assert not got[0][6][refused].any() and (got[0][6][~refused] != -7).all()
    assert seen >= {0, 2}
    ok(hip("hipGraphExecDestroy")(run))
    ok(hip("hipGraphDestroy")(graph))


def test_two_contexts_at_once(gpu_ctx, hyq):
    """Steps enqueued on two contexts (streams) in turn, each with buffers of
    its own, give what one alone gives."""
    other = hyq.Context(0)
    try:
        alone = Server(hyq, gpu_ctx, seed=4)
        one, two = Server(hyq, gpu_ctx, seed=4), Server(hyq, other, seed=4)
        logits = np.random.default_rng(5).normal(0, 3, (5, SEQS, VOCAB)).astype(np.float32)
        for i in range(5):
            for s in (alone, one, two):
                feed(s, i, logits)
            alone.step()
            want = alone.state()
            for _ in range(3):  # (idle repeats of attention and sampling beside each other)
                one.L.hyq_sample_d(one.ctx.handle, one.logits.ptr, SEQS, VOCAB,
                                   *[a.ptr for a in one.set], one.u.ptr, one.scratch.ptr, one.ns,
                                   one.token.ptr, one.prob.ptr)
            one.step()
            two.step()
            for s in (one, two):
                for a, b in zip(want, s.state()):
                    assert np.array_equal(a, b, equal_nan=True)
        del two
    finally:
        other.close()
