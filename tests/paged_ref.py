"""Plain 64-bit forms of the paged cache's operators and of the sampler, in
numpy, and the batches that their tests share."""
import numpy as np

D = 128
U = 2.0 ** -24  # f32 rounding: half a step


class Batch:
    """Slots of given lengths (new tokens included) and new tokens over a pool
    whose every unused place holds a NaN."""

    def __init__(self, lens, news, heads, kv_heads, page_tokens, f16, seed, spare=3, width=None,
                 tail=0, scale=1.0):
        r = np.random.default_rng(seed)
        self.lens, self.news = np.array(lens, np.int32), np.array(news, np.int32)
        self.heads, self.kvh, self.pt, self.f16 = heads, kv_heads, page_tokens, f16
        self.seqs = len(lens)
        counts = [-(-int(n) // page_tokens) for n in lens]
        self.width = width or max(counts + [1]) + 1
        self.pages = sum(counts) + spare
        ids = r.permutation(self.pages).astype(np.int32)
        self.table = np.full((self.seqs, self.width), -1, np.int32)
        self.pool = np.full((self.pages, 2, kv_heads, page_tokens, D), np.nan,
                            np.float16 if f16 else np.float32)
        at = 0
        for s, c in enumerate(counts):
            self.table[s, :c] = ids[at:at + c]
            at += c
            for i in range(c):
                n = min(page_tokens, int(lens[s]) - i * page_tokens)
                self.pool[self.table[s, i], :, :, :n] = scale * r.normal(
                    0, 1, (2, kv_heads, n, D))
        self.start = np.concatenate([[0], np.cumsum(self.news)]).astype(np.int32)
        self.new = int(self.start[-1])
        self.rows = self.new + tail
        self.q = r.normal(0, 1, (self.rows, heads, D)).astype(np.float32)
        self.rng = r

    def kv(self, s, h):
        """Keys and values [len, 128] of a slot's KV head h in 64 bits, and
        whether a page holds each position."""
        n = int(self.lens[s])
        ids = self.table[s][np.arange(n) // self.pt]
        ok = (ids >= 0) & (ids < self.pages)
        rows = self.pool[np.where(ok, ids, 0), :, h, np.arange(n) % self.pt].astype(np.float64)
        return rows[:, 0], rows[:, 1], ok

    def attention(self):
        """Outputs [rows, heads, 128] in 64 bits and, per row and head, the
        bound of the kernels' error (tolerance() below). Rows of no slot: NaN."""
        out = np.full((self.rows, self.heads, D), np.nan)
        tol = np.zeros((self.rows, self.heads))
        rep = self.heads // self.kvh
        for s in range(self.seqs):
            n, m, b = int(self.lens[s]), int(self.news[s]), int(self.start[s])
            for h in range(self.kvh):
                k, v, ok = self.kv(s, h)
                for i in range(m):
                    last = n - m + i
                    see = ok & (np.arange(n) <= last)
                    for g in range(rep):
                        head = h * rep + g
                        if not see.any():
                            out[b + i, head] = 0
                            continue
                        q = self.q[b + i, head].astype(np.float64)
                        sc = k[see] @ q / np.sqrt(D)
                        w = np.exp(sc - sc.max())
                        out[b + i, head] = (w[:, None] * v[see]).sum(0) / w.sum()
                        mag = (np.abs(k[see]) @ np.abs(q)).max() / np.sqrt(D)
                        tol[b + i, head] = tolerance(mag, np.abs(sc).max(), np.abs(v[see]).max(),
                                                     int(see.sum()))
        return out, tol


def tolerance(mag, score, vmax, n):
    """Bound of an output's error for scores of at most `score` formed from
    products that sum to `mag` in magnitude, over n positions, values up to
    vmax. A score is off by its operands' (two f16 parts each: 2 * 2^-22, the
    product of the low parts left out: 2^-22, and below 2^-3 an absolute 2^-25,
    which `mag + 1` covers for keys and queries of mean size about one) and by
    its sum's rounding (128 products added in f32: 128 U mag); its scaling, the
    difference with the maximum and the exponential's argument round by U of at
    most 2 |score| * log2(e) each, the exponential by 2 U. A weight off by a
    factor 1 + d moves numerator and denominator: 2 d vmax. Sums over n
    positions in f32 and the weights' own split: (n + 8) U + 3 * 2^-22."""
    d = (128 * U + 3 * 2.0 ** -22) * (mag + 1) + 3 * U * 3 * score + 2 * U
    return vmax * (2 * d + (n + 8) * U + 3 * 2.0 ** -22)


def append(batch, k, v, qn, kn, freq, eps, norm_first):
    """(q_out, pool) of the rotation, norms and writes in 64 bits; the pool's
    values before its own rounding."""
    pool = batch.pool.astype(np.float64)
    q_out = np.full((batch.rows, batch.heads, D), np.nan)

    def formed(x, w, pos):
        x = x.astype(np.float64)
        a = pos * freq.astype(np.float64)
        c, s = np.cos(a), np.sin(a)

        def turn(y):
            lo, hi = y[..., :64], y[..., 64:]
            return np.concatenate([lo * c - hi * s, lo * s + hi * c], -1)

        def norm(y):
            return y * w.astype(np.float64) / np.sqrt((y * y).mean(-1, keepdims=True) + eps)

        return turn(norm(x)) if norm_first else norm(turn(x))

    for s in range(batch.seqs):
        n, m, b = int(batch.lens[s]), int(batch.news[s]), int(batch.start[s])
        for i in range(m):
            pos = n - m + i
            q_out[b + i] = formed(batch.q[b + i], qn, pos)
            page = batch.table[s, pos // batch.pt]
            if 0 <= page < batch.pages:
                pool[page, 0, :, pos % batch.pt] = formed(k[b + i], kn, pos)
                pool[page, 1, :, pos % batch.pt] = v[b + i]
    return q_out, pool


class Pages:
    """The pages' bookkeeping, step by step; `data` [pages][page_tokens] stands
    for what the pages hold."""

    def __init__(self, table, lens, pages, pt, data):
        self.table, self.lens, self.pages, self.pt = table.copy(), lens.copy(), pages, pt
        self.data = data.copy()
        self.count()

    def held(self, n):
        return -(-int(n) // self.pt)

    def count(self):
        self.refs = np.zeros(self.pages, np.int32)
        for s, n in enumerate(self.lens):
            for p in self.table[s, :self.held(n)]:
                if 0 <= p < self.pages:
                    self.refs[p] += 1

    def fork(self, parent, keep):
        table, lens = self.table.copy(), self.lens.copy()
        for s, p in enumerate(parent):
            n = 0
            if 0 <= p < len(lens):
                n = int(lens[p]) if keep is None else max(0, min(int(lens[p]), int(keep[s])))
            self.table[s] = -1
            if n:
                self.table[s, :self.held(n)] = table[p, :self.held(n)]
            self.lens[s] = n
        self.count()

    def extend(self, add):
        width = self.table.shape[1]
        refs, free = self.refs.copy(), [p for p in range(self.pages) if self.refs[p] == 0]
        status = np.zeros(len(add), np.int32)
        asks = [s for s, a in enumerate(add) if a > 0 and self.lens[s] + a <= width * self.pt]
        last = {s: self.table[s, self.held(self.lens[s]) - 1] for s in asks
                if self.lens[s] % self.pt}
        copies = set()
        for s, p in last.items():
            if refs[p] > 1:
                who = [x for x in last if last[x] == p]
                fill = max(self.lens[x] % self.pt for x in who)
                keeper = min(x for x in who if self.lens[x] % self.pt == fill)
                if not (len(who) == refs[p] and s == keeper):
                    copies.add(s)
        used, before = 0, self.data.copy()
        for s in range(len(add)):
            if add[s] > 0 and s not in asks:
                status[s] = 2
            if s not in asks:
                continue
            held, wants = self.held(self.lens[s]), self.held(self.lens[s] + add[s])
            need = wants - held + (s in copies)
            used += need
            if need and used > len(free):
                status[s] = 1
                continue
            got = free[used - need:used]
            if s in copies:
                p, fill = got.pop(0), self.lens[s] % self.pt
                self.table[s, held - 1] = p
                self.data[p, :fill] = before[last[s], :fill]
                self.refs[last[s]] -= 1
                self.refs[p] = 1
            for i, p in enumerate(got):
                self.table[s, held + i] = p
                self.refs[p] = 1
            self.lens[s] += add[s]
        return status

    def compact(self):
        live = int((self.refs > 0).sum())
        src = [p for p in range(live, self.pages) if self.refs[p] > 0]
        dst = [p for p in range(live) if self.refs[p] == 0]
        to = np.arange(self.pages, dtype=np.int32)
        to[src] = dst
        self.data[dst] = self.data[src]
        ok = self.table >= 0
        self.table[ok] = to[self.table[ok]]
        self.refs[dst] = self.refs[src]
        self.refs[src] = 0
        return live


def sample(logits, temperature, top_k, top_p, min_p, random):
    """(token, probability) of one row in 64 bits."""
    x = np.where(np.isnan(logits), -np.inf, logits.astype(np.float64))
    if x.max() == -np.inf:
        return -1, 0.0
    if not temperature > 0:
        return int(np.argmax(x)), 1.0
    with np.errstate(invalid="ignore"):
        w = np.where(x == x.max(), 1.0, np.exp((x - x.max()) / np.float64(temperature)))
    w = np.where(x > -np.inf, np.nan_to_num(w), 0.0)
    order = np.argsort(-x, kind="stable")
    if top_k > 0:
        order = order[:top_k]
    ws = w[order]
    n = len(order)
    if top_p < 1:
        n = int(np.argmax(np.cumsum(ws) >= max(float(top_p), 0.0) * ws.sum())) + 1
    n = max(1, min(n, int((ws >= min(float(min_p), 1.0)).sum())))
    keep = np.sort(order[:n])
    upto = np.cumsum(w[keep])
    u = min(max(float(random), 0.0), 1.0)
    at = int(np.searchsorted(upto, u * upto[-1], side="right"))
    at = min(at, int(np.flatnonzero(w[keep] > 0)[-1]))
    return int(keep[at]), float(w[keep[at]] / upto[-1])
