"""A server's step over 8-bit pages with shared prefixes and logits rules, as they are
used together: fork, extension, plan, append and attention of every layer, penalties
and grammars, sampling; eagerly against the plain 64-bit forms, captured in a HIP
graph, and on two contexts at once."""
import ctypes

import numpy as np
import pytest

import logits_ref
import paged_q8_ref as Q
import paged_ref as R
from test_gpu_serving import captured, hip, ok

pytestmark = pytest.mark.gpu
D, HEADS, KVH, PT, PAGES, SEQS, LAYERS, VOCAB, HISTORY = 128, 8, 2, 16, 80, 6, 2, 900, 40


class Server:
    """Six slots of one prompt of four pages, a token a step. Everything that a step
    reads is on the device; `feed` sets what changes from step to step."""

    def __init__(self, hyq, ctx, seed=1):
        self.hyq, self.ctx, self.L = hyq, ctx, hyq.lib()
        r = np.random.default_rng(seed)
        a = lambda x, t=np.float32: ctx.array(np.ascontiguousarray(x, t))
        self.cache = hyq.PagedCache(ctx, LAYERS, KVH, PAGES, SEQS, 20 * PT, PT, hyq.KV_Q8)
        self.cache.pool.copy_from(np.zeros(self.cache.pool.shape, np.uint8))
        self.norm, self.freq = a(np.ones(D)), a(10000.0 ** (-np.arange(64) / 64))
        prompt = 4 * PT + 5
        assert not self.cache.extend([prompt] + [0] * (SEQS - 1)).any()
        start = a([0] + [prompt] * SEQS, np.int32)
        rows = [a(r.normal(0, 1, (prompt, n, D))) for n in (HEADS, KVH, KVH)]
        out = ctx.empty((prompt, HEADS, D), np.float32)
        for l in range(LAYERS):
            self.cache.append_d(l, start.ptr, prompt, HEADS, *[x.ptr for x in rows], self.norm.ptr,
                                self.norm.ptr, self.freq.ptr, 1e-5, out.ptr)
        self.cache.fork([0] * SEQS)
        assert not self.cache.extend([0] * SEQS).any()
        self.parent, self.add = a(np.arange(SEQS), np.int32), a(np.ones(SEQS), np.int32)
        self.start = a(np.arange(SEQS + 1), np.int32)
        self.q, self.k, self.v = ([a(r.normal(0, 1, (SEQS, n, D))) for _ in range(LAYERS)]
                                  for n in (HEADS, KVH, KVH))
        self.qo = [ctx.empty((SEQS, HEADS, D), np.float32) for _ in range(LAYERS)]
        self.out = [a(np.zeros((SEQS, HEADS, D))) for _ in range(LAYERS)]
        self.logits, self.ruled = a(np.zeros((SEQS, VOCAB))), a(np.zeros((SEQS, VOCAB)))
        self.history = a(np.zeros((SEQS, HISTORY)), np.int32)
        self.held = a(np.zeros(SEQS), np.int32)
        self.settings = dict(repetition=[1.1, 1, 1.5, 1, 2, 0], presence=[0, .5, 0, -.5, 0, 1],
                             frequency=[0, .1, .2, 0, 0, .3])
        self.masks = r.random((2, VOCAB)) < np.array([[0.5], [0.02]])
        words = np.zeros((2, -(-VOCAB // 32) * 32), bool)
        words[:, :VOCAB] = self.masks
        self.mask_row = [0, -1, 1, 0, -1, 1]
        self.kept = [a(self.settings[n]) for n in ("repetition", "presence", "frequency")] + [
            ctx.array(np.packbits(words, axis=1, bitorder="little")), a(self.mask_row, np.int32)]
        k = [x.ptr for x in self.kept]
        self.rules = hyq.LogitRules(self.history.ptr, self.held.ptr, None, HISTORY, k[0], k[1], k[2],
                                    None, None, None, 0, k[3], k[4], 2)
        self.set = [a(np.full(SEQS, 0.8)), a([0, 20, 5, 100, 0, 3], np.int32),
                    a([1, 0.9, 1, 0.7, 0.8, 1]), a([0, 0, 0.1, 0, 0, 0])]
        self.u = a(np.full(SEQS, 0.5))
        self.token, self.prob = a(np.zeros(SEQS), np.int32), a(np.zeros(SEQS))
        self.ns = self.L.hyq_sample_scratch_bytes(SEQS, VOCAB)
        self.scratch = ctx.empty(max(self.ns, 16), np.uint8)
        ctx.sync()
        self.begin = [x.numpy() for x in (self.cache.pool, self.cache.table, self.cache.len,
                                          self.cache.refs)]

    def reset(self):
        c = self.cache
        for x, v in zip((c.pool, c.table, c.len, c.refs), self.begin):
            x.copy_from(v)

    def step(self):
        c = self.cache
        c.fork_d(self.parent.ptr)
        c.extend_d(self.add.ptr)
        c.share_d(self.start.ptr, SEQS, HEADS, least=0)
        for l in range(LAYERS):
            c.append_d(l, self.start.ptr, SEQS, HEADS, self.q[l].ptr, self.k[l].ptr, self.v[l].ptr,
                       self.norm.ptr, self.norm.ptr, self.freq.ptr, 1e-5, self.qo[l].ptr)
            c.attention_d(l, self.start.ptr, SEQS, 1, HEADS, self.qo[l].ptr, self.out[l].ptr,
                          shared=True)
        h, L = self.ctx.handle, self.L
        self.hyq.check(L.hyq_logits_adjust_d(h, self.logits.ptr, SEQS, VOCAB,
                                             ctypes.byref(self.rules), self.ruled.ptr))
        self.hyq.check(L.hyq_sample_d(h, self.ruled.ptr, SEQS, VOCAB, *[x.ptr for x in self.set],
                                      self.u.ptr, self.scratch.ptr, self.ns, self.token.ptr,
                                      self.prob.ptr))

    def state(self):
        self.ctx.sync()
        c = self.cache
        return [x.numpy() for x in (c.table, c.len, c.refs, c.status, c.pool, *self.qo, *self.out,
                                    self.ruled, self.token, self.prob)]


PARENTS = [[0, 1, 2, 3, 4, 5], [0, 0, 0, 3, 4, 4], [5, 1, 1, -1, 4, 2], [0, 1, 2, 3, 4, 5],
           [4, 4, 4, 4, 4, 4], [0, 1, 2, 3, 4, 5]]


def feed(s, i, seed=0):
    r = np.random.default_rng(100 * seed + i)
    s.parent.copy_from(np.array(PARENTS[i % len(PARENTS)], np.int32))
    s.add.copy_from(np.array([1, 1, 17 if i % 3 == 2 else 1, 1, 1, 0 if i == 3 else 1], np.int32))
    s.logits.copy_from(r.normal(0, 3, (SEQS, VOCAB)).astype(np.float32))
    s.history.copy_from(r.integers(0, VOCAB, (SEQS, HISTORY)).astype(np.int32))
    s.held.copy_from(r.integers(0, HISTORY + 1, SEQS).astype(np.int32))
    s.u.copy_from(r.random(SEQS).astype(np.float32))


def test_against_the_plain_forms(gpu_ctx, hyq):
    """Each step's attention from the pages that it wrote, its logits and tokens."""
    s = Server(hyq, gpu_ctx)
    for i in range(8):
        feed(s, i)
        s.step()
        got = s.state()
        table, lens, refs, status, pool = got[:5]
        assert not status.any()
        used = np.bincount(np.concatenate([table[x, :-(-lens[x] // PT)] for x in range(SEQS)]),
                           minlength=PAGES)
        assert np.array_equal(used, refs)
        pages = pool.reshape(LAYERS, PAGES, -1)
        for l in range(LAYERS):
            b = Q.BatchQ8([1] * SEQS, [1] * SEQS, HEADS, KVH, PT, seed=0)
            b.table, b.lens, b.pages, b.width = table, lens, PAGES, table.shape[1]
            b.news = (lens > 0).astype(np.int32)
            b.start = np.arange(SEQS + 1)
            b.codes, b.scales = Q.split(pages[l], KVH, PT)
            b.q = got[5 + l]
            # (the last of a slot's new places alone was written: the others hold what
            # their pages held, zeros of a new pool among them)
            want, tol = b.attention()
            held = lens > 0
            err = np.abs(got[5 + LAYERS + l][held] - want[held]).max(-1)
            assert np.all(err <= tol[held]), (i, l)
        logits, hist, n = s.logits.numpy(), s.history.numpy(), s.held.numpy()
        x, tol = logits_ref.adjust(logits, [hist[r, :n[r]] for r in range(SEQS)], None,
                                   masks=s.masks, mask_row=s.mask_row, **s.settings)
        ruled, token, prob = got[-3:]
        fine = np.isfinite(x)
        assert np.array_equal(ruled[~fine], x[~fine])
        assert np.all(np.abs(ruled[fine] - x[fine]) <= tol[fine])
        t, k, p, m = (v.numpy() for v in s.set)
        for r in range(SEQS):
            want = R.sample(ruled[r], t[r], k[r], p[r], m[r], s.u.numpy()[r])
            assert token[r] == want[0] and abs(prob[r] - want[1]) < 1e-6
            assert s.mask_row[r] < 0 or s.masks[s.mask_row[r], token[r]]


def test_a_captured_step(gpu_ctx, hyq):
    """The whole step in one graph, replayed with new inputs and with eager calls and
    waits between: every replay gives the eager step's bits."""
    eager, graphed = Server(hyq, gpu_ctx), Server(hyq, gpu_ctx)
    for s in (eager, graphed):
        feed(s, 0)
        s.step()
        s.reset()
    graph, run = captured(gpu_ctx, graphed.step)
    for i in range(10):
        if i == 6:
            eager.reset()
            graphed.reset()
        feed(eager, i)
        feed(graphed, i)
        eager.step()
        want = eager.state()
        ok(hip("hipGraphLaunch")(run, ctypes.c_void_p(gpu_ctx.stream)))
        for a, b in zip(want, graphed.state()):
            assert np.array_equal(a, b, equal_nan=True), i
        assert sum(len(x) for x in graphed.cache.read(0)[0]) == 2 * graphed.cache.lengths()[0]
    ok(hip("hipGraphExecDestroy")(run))
    ok(hip("hipGraphDestroy")(graph))


def test_two_contexts_at_once(gpu_ctx, hyq):
    """Steps on two contexts (streams) in turn, each with buffers of its own."""
    other = hyq.Context(0)
    try:
        alone, one, two = Server(hyq, gpu_ctx, 3), Server(hyq, gpu_ctx, 3), Server(hyq, other, 3)
        for i in range(5):
            for s in (alone, one, two):
                feed(s, i, 1)
            alone.step()
            want = alone.state()
            one.step()
            two.step()
            for s in (one, two):
                for a, b in zip(want, s.state()):
                    assert np.array_equal(a, b, equal_nan=True), i
        del two
    finally:
        other.close()
