"""The operators of one serving step over a paged KV cache, as measurable cases.

A server that translates for many sessions at once keeps their keys and values
in pages of one pool. Each step it forks or frees the slots of its beams and
requests and gives every slot the pages of its next tokens (``pages``), forms
the new tokens' queries and keys and writes keys and values into the pages
(``append``), attends (``attention``), and draws a token for every row of
logits (``sample``).

Pools are [layers][pages][2][kv_heads][page_tokens][128] (keys, then values),
page tables [slots][entries] of page ids, -1 where a slot holds none. Head
counts, widths and vocabularies are those of the 1.8B and 7B models that
bench.py builds, or generic.
"""
import ctypes
import importlib.util
import math
import os
import random
import sys

import torch

own = False
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "hy-mt-rs_amd")
D = 128
EPS = 1e-5
ROPE_BASE = 11158840.0
VOCAB_1P8B, VOCAB_7B = 120818, 128167


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    small = dict(heads=16, kv_heads=4)
    large = dict(heads=32, kv_heads=8)
    return [
        # one new token in each of 48 sessions
        dict(name="append_decode", kind="append", dtype="F16", page_tokens=64, slots=48, prompts=0,
             chunk=1, step=1, idle=0, context=4096, pad=0, norm_first=False, **small),
        # six prompts of some hundred tokens at once, in a padded batch
        dict(name="append_prompts", kind="append", dtype="F32", page_tokens=32, slots=6, prompts=6,
             chunk=500, step=1, idle=0, context=2500, pad=13, norm_first=True, **large),
        # the two concurrent requests that a server takes by default
        dict(name="attn_two", kind="attention", dtype="F32", page_tokens=64, slots=2, prompts=0,
             chunk=1, step=1, idle=0, context=1100, pad=0, **small),
        # 64 sessions of very different length
        dict(name="attn_decode", kind="attention", dtype="F16", page_tokens=64, slots=64,
             prompts=0, chunk=1, step=1, idle=0, context=8192, pad=0, **large),
        # a few sessions over whole books
        dict(name="attn_long", kind="attention", dtype="F32", page_tokens=128, slots=4, prompts=0,
             chunk=1, step=1, idle=0, context=60001, pad=0, **small),
        # the second part of one prompt
        dict(name="attn_prompt", kind="attention", dtype="F32", page_tokens=64, slots=1,
             prompts=1, chunk=512, step=1, idle=0, context=2012, pad=0, **small),
        # three prompts taken in beside 27 running sessions and two empty slots
        dict(name="attn_mixed", kind="attention", dtype="F16", page_tokens=64, slots=32,
             prompts=3, chunk=400, step=1, idle=2, context=4000, pad=5, **large),
        # a beam search's step: beams chosen, the next token's pages made
        dict(name="beams_8", kind="beams", dtype="F16", page_tokens=16, slots=8, layers=32,
             kv_heads=4, context=700, spare=64),
        # the same for many requests with their beams
        dict(name="beams_128", kind="beams", dtype="F16", page_tokens=64, slots=128, layers=32,
             kv_heads=4, context=1500, spare=300),
        # a pool after most of its requests have ended, made dense
        dict(name="compact", kind="compact", dtype="F16", page_tokens=64, slots=24, layers=32,
             kv_heads=4, context=1500, spare=200),
        # the next tokens of two requests, with a translation model's usual settings
        dict(name="sample_two", kind="sample", rows=2, vocab=VOCAB_1P8B, mix="usual"),
        # 64 requests with settings of their own
        dict(name="sample_batch", kind="sample", rows=64, vocab=VOCAB_7B, mix="any"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(["append", "attention", "beams", "compact", "sample"], [3, 7, 2, 1, 3])[0]
    if kind == "sample":
        vocab = rng.choice([VOCAB_1P8B, VOCAB_7B, _log_int(rng, 1000, 120000)])
        return dict(kind=kind, rows=_log_int(rng, 1, 64), vocab=vocab,
                    mix=rng.choice(["usual", "any"]))
    dtype = rng.choice(["F16", "F32"])
    page_tokens = rng.choice([16, 32, 64, 128])
    if kind in ("beams", "compact"):
        return dict(kind=kind, dtype=dtype, page_tokens=page_tokens, slots=_log_int(rng, 2, 48),
                    layers=rng.randint(1, 16), kv_heads=rng.choice([1, 2, 4]),
                    context=_log_int(rng, 2 * page_tokens, 1500), spare=_log_int(rng, 50, 200))
    heads, kv_heads = rng.choice([(16, 4), (32, 8), (8, 2), (12, 4), (8, 8), (16, 2)])
    case = dict(kind=kind, dtype=dtype, page_tokens=page_tokens, heads=heads, kv_heads=kv_heads,
                pad=rng.choice([0, _log_int(rng, 1, 60)]))
    if kind == "append":
        case["norm_first"] = rng.random() < 0.5
    form = rng.choice(["decode", "decode", "draft", "prompt", "mixed"])
    if form == "prompt":
        chunk = _log_int(rng, 2, 700)
        return dict(case, slots=rng.randint(1, 3), prompts=3, chunk=chunk, step=1, idle=0,
                    context=chunk + rng.choice([0, _log_int(rng, 1, 2000)]))
    if form == "mixed":
        chunk = _log_int(rng, 20, 300)
        return dict(case, slots=rng.randint(4, 20), prompts=rng.randint(1, 3), chunk=chunk,
                    step=1, idle=rng.randint(0, 1), context=chunk + _log_int(rng, 16, 2000))
    slots = _log_int(rng, 1, 64)
    step = 1 if form == "decode" else rng.randint(2, 6)
    return dict(case, slots=slots, prompts=0, chunk=1, step=step, idle=rng.choice([0, slots // 8]),
                context=step + _log_int(rng, 1, max(2, min(16000, 200000 // slots))))


def _batch(case):
    """Positions held (the new tokens among them) and new tokens, by slot."""
    c = case
    r = random.Random(c["slots"] * 1009 + c["context"])
    lens, news = [], []
    for s in range(c["slots"]):
        prompt = s < c["prompts"]
        if s >= c["slots"] - c["idle"]:
            news.append(0)
        elif prompt:
            news.append(c["chunk"] if s == 0 else r.randint((c["chunk"] + 1) // 2, c["chunk"]))
        else:
            news.append(c["step"])
        low = max(news[s], c["context"] // 8, 1)
        lens.append(c["context"] if s == 0 else _log_int(r, low, max(low, c["context"])))
    return lens, news


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
class Source:
    """Seeded random tensors on the GPU, in the order they are asked for."""

    def __init__(self, seed):
        self.g = torch.Generator("cuda")
        self.g.manual_seed(int(seed) * 6151 + 29)

    def normal(self, *shape, dtype=torch.float32):
        return torch.randn(shape, generator=self.g, device="cuda", dtype=dtype)

    def uniform(self, *shape):
        return torch.rand(shape, generator=self.g, device="cuda", dtype=torch.float32)

    def order(self, n):
        return torch.randperm(n, generator=self.g, device="cuda").to(torch.int32)


def _ints(values):
    return torch.tensor(values, device="cuda", dtype=torch.int32)


def _type(case):
    return torch.float16 if case["dtype"] == "F16" else torch.float32


def _pages_of(n, page_tokens):
    return -(-n // page_tokens)


def _tables(source, lens, page_tokens, spare, width):
    """A page table of the slots' own pages, scattered over a pool."""
    counts = [_pages_of(n, page_tokens) for n in lens]
    pages = sum(counts) + spare
    ids = source.order(pages)
    table = torch.full((len(lens), width), -1, device="cuda", dtype=torch.int32)
    at = 0
    for s, n in enumerate(counts):
        table[s, :n] = ids[at:at + n]
        at += n
    return table, pages


def _inputs(case, seed):
    c, src = case, Source(seed)
    if c["kind"] == "sample":
        rows, vocab = c["rows"], c["vocab"]
        logits = 2.0 * src.normal(rows, vocab)
        likely = torch.randint(0, vocab, (rows, 24), generator=src.g, device="cuda")
        logits.scatter_add_(1, likely, 12.0 * src.uniform(rows, 24))
        if c["mix"] == "usual":
            settings = [(0.7, 20, 0.6, 0.0)] * rows
        else:
            kinds = [(0.7, 20, 0.6, 0.0), (1.0, 0, 1.0, 0.0), (0.8, 0, 0.95, 0.0),
                     (1.0, 0, 1.0, 0.05), (0.0, 0, 1.0, 0.0), (1.3, 1000, 0.9, 0.001),
                     (0.6, 40, 1.0, 0.1), (1.0, 50000, 0.99, 0.0)]
            settings = [kinds[r % len(kinds)] for r in range(rows)]
        t, k, p, m = zip(*settings)
        f = dict(device="cuda", dtype=torch.float32)
        return dict(logits=logits, temperature=torch.tensor(t, **f), top_k=_ints(k),
                    top_p=torch.tensor(p, **f), min_p=torch.tensor(m, **f),
                    u=src.uniform(rows))
    pt = c["page_tokens"]
    if c["kind"] in ("beams", "compact"):
        r = random.Random(c["slots"] * 31 + c["context"])
        lens = [r.randint(pt, c["context"]) for _ in range(c["slots"])]
        width = _pages_of(c["context"], pt) + 2
        table, pages = _tables(src, lens, pt, c["spare"] + c["slots"] * 2, width)
        refs = torch.bincount(table[table >= 0].long(), minlength=pages).to(torch.int32)
        s = dict(table=table, lens=_ints(lens), refs=refs, pages=pages, width=width)
        # groups of four beams: a step keeps some, doubles some, drops some
        parent = [min(g - g % 4 + r.choice([0, 0, 1, 2, 3]), c["slots"] - 1)
                  for g in range(c["slots"])]
        if c["slots"] > 4:
            parent[-1] = -1  # a request that has ended
        s.update(parent=_ints(parent), add=_ints([1] * c["slots"]),
                 keep=_ints([width * pt] * c["slots"]))
        s["pool"] = src.normal(c["layers"], pages, 2, c["kv_heads"], pt, D, dtype=_type(c))
        return s
    lens, news = _batch(c)
    width = _pages_of(c["context"], pt) + 1
    table, pages = _tables(src, lens, pt, 5, width)
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    rows = starts[-1] + c["pad"]
    s = dict(table=table, lens=_ints(lens), starts=_ints(starts), pages=pages, width=width,
             rows=rows, new=starts[-1], most=max(news),
             pool=src.normal(1, pages, 2, c["kv_heads"], pt, D, dtype=_type(c)),
             q=src.normal(rows, c["heads"] * D))
    if c["kind"] == "append":
        j = torch.arange(D // 2, device="cuda", dtype=torch.float64)
        s.update(k=src.normal(rows, c["kv_heads"] * D), v=src.normal(rows, c["kv_heads"] * D),
                 qn=1.0 + 0.02 * src.normal(D), kn=1.0 + 0.02 * src.normal(D),
                 freq=(ROPE_BASE ** (-2.0 * j / D)).float())
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    kind = case["kind"]
    like = torch.zeros_like
    if kind == "sample":
        s.update(token=torch.zeros(case["rows"], device="cuda", dtype=torch.int32),
                 prob=torch.zeros(case["rows"], device="cuda", dtype=torch.float32))
    elif kind in ("append", "attention"):
        s["out"] = like(s["q"])
    else:
        s.update(table_a=like(s["table"]), lens_a=like(s["lens"]), refs_a=like(s["refs"]),
                 table_b=like(s["table"]), lens_b=like(s["lens"]), refs_b=like(s["refs"]),
                 status=like(s["lens"]), live=_ints([0]))
    return s


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _rows_of(s):
    """Slot and position of every new row."""
    rows = torch.arange(s["new"], device="cuda")
    slot = torch.searchsorted(s["starts"].long(), rows, right=True) - 1
    start, count = s["starts"][slot], s["starts"][slot + 1] - s["starts"][slot]
    return slot, (s["lens"][slot] - count + (rows - start)).long()


def _plain_append(s):
    c, n = s["case"], s["new"]
    slot, pos = _rows_of(s)
    angle = pos[:, None].double() * s["freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def norm(x, w):
        return x * (w / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS))

    def turn(x):
        a, b = x[..., :D // 2], x[..., D // 2:]
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)

    def both(x, w):
        x = x[:n].view(n, -1, D)
        return turn(norm(x, w)) if c["norm_first"] else norm(turn(x), w)

    s["out"][:n] = both(s["q"], s["qn"]).reshape(n, -1)
    pt, pool = c["page_tokens"], s["pool"][0]
    page, at = s["table"][slot, pos // pt].long(), pos % pt
    pool[page, 0, :, at] = both(s["k"], s["kn"]).to(pool.dtype)
    pool[page, 1, :, at] = s["v"][:n].view(n, -1, D).to(pool.dtype)
    return {"q": s["out"], "pool": s["pool"]}


def _plain_attention(s):
    c, pt = s["case"], s["case"]["page_tokens"]
    slots, kvh, heads, most = c["slots"], c["kv_heads"], c["heads"], s["most"]
    pages = s["pool"][0][s["table"].clamp(min=0).long()]      # [slots, width, 2, kvh, pt, D]
    kv = pages.permute(2, 0, 3, 1, 4, 5).reshape(2, slots, kvh, -1, D).float()
    i = torch.arange(most, device="cuda")
    count = s["starts"][1:] - s["starts"][:-1]
    given = i < count[:, None]                                 # [slots, most]
    row = torch.where(given, s["starts"][:-1, None] + i, 0).long()
    q = s["q"][row].view(slots, most, kvh, heads // kvh, D).permute(0, 2, 1, 3, 4)
    scores = torch.matmul(q.reshape(slots, kvh, -1, D) * D ** -0.5, kv[0].transpose(-1, -2))
    scores = scores.view(slots, kvh, most, heads // kvh, -1)
    last = (s["lens"] - count)[:, None] + i                    # a row's own position
    seen = torch.arange(s["width"] * pt, device="cuda") <= last[:, :, None]
    scores = scores.masked_fill(~seen[:, None, :, None], -math.inf)
    e = torch.exp(scores - scores.max(-1, keepdim=True).values)
    o = torch.matmul((e / e.sum(-1, keepdim=True)).view(slots, kvh, -1, seen.shape[-1]), kv[1])
    o = o.view(slots, kvh, most, -1, D).permute(0, 2, 1, 3, 4).reshape(slots, most, -1)
    s["out"][:s["new"]] = o[given]
    return s["out"]


def _plain_fork(s, table, lens):
    parent, width, pt = s["parent"].long(), s["width"], s["case"]["page_tokens"]
    got = torch.where(parent >= 0, torch.minimum(lens[parent.clamp(min=0)], s["keep"]), 0)
    used = torch.arange(width, device="cuda") < ((got + pt - 1) // pt)[:, None]
    entries = torch.where(used, table[parent.clamp(min=0)], -1)
    refs = torch.bincount(entries[used].long(), minlength=s["pages"])
    return entries, got.to(torch.int32), refs.to(torch.int32)


def _plain_extend(s, table, lens, refs):
    c, width, pt, n = s["case"], s["width"], s["case"]["page_tokens"], s["case"]["slots"]
    slot = torch.arange(n, device="cuda")
    add = s["add"]
    long = lens + add > width * pt
    asks = (add > 0) & ~long
    held, wants = (lens + pt - 1) // pt, (lens + add + pt - 1) // pt
    fill = lens % pt
    last = table[slot, (held - 1).clamp(min=0).long()].clamp(min=0).long()
    shared = asks & (fill > 0) & (refs[last] > 1)
    # where all who name a page extend it, the one that holds most of it (the first of those) keeps it
    askers = torch.bincount(last[shared], minlength=s["pages"])
    key = torch.where(shared, fill.long() * 65536 + 65535 - slot, -1)
    top = torch.full((s["pages"],), -1, device="cuda").scatter_reduce(0, last, key, "amax")
    copies = shared & ~((askers[last] == refs[last]) & (key == top[last]))
    need = torch.where(asks, wants - held + copies, 0)
    upto = torch.cumsum(need, 0)
    free = torch.nonzero(refs == 0)[:, 0]
    served = asks & ((need == 0) | (upto <= free.numel()))
    begin = (upto - need)[:, None]
    entry = torch.arange(width, device="cuda")[None]
    copied = (copies & served)[:, None] & (entry == held[:, None] - 1)
    fresh = served[:, None] & (entry >= held[:, None]) & (entry < wants[:, None])
    rank = torch.where(copied, begin, begin + copies[:, None] + entry - held[:, None])
    new = free[rank[copied | fresh].long()]
    table_out = table.clone()
    table_out[copied | fresh] = new.to(torch.int32)
    refs_out = refs.clone()
    refs_out[new] = 1
    who = torch.nonzero(copies & served)[:, 0]
    refs_out -= torch.bincount(last[who], minlength=s["pages"]).to(torch.int32)
    dst = table_out[who, (held - 1)[who].long()].long()
    kept = (torch.arange(pt, device="cuda") < fill[who, None])[None, :, None, None, :, None]
    pool = s["pool"]
    pool[:, dst] = torch.where(kept, pool[:, last[who]], pool[:, dst])
    status = torch.where(long & (add > 0), 2, torch.where(asks & ~served, 1, 0))
    return (table_out, torch.where(served, lens + add, lens).to(torch.int32), refs_out,
            status.to(torch.int32))


def _plain_beams(s):
    forked = _plain_fork(s, s["table"], s["lens"])
    s["table_a"], s["lens_a"], s["refs_a"] = forked
    s["table_b"], s["lens_b"], s["refs_b"], s["status"] = _plain_extend(s, *forked)


def _plain_compact(s):
    refs, pages = s["refs_a"], s["pages"]
    live = refs > 0
    ids = torch.arange(pages, device="cuda")
    count = live.sum()
    src, dst = torch.nonzero(live & (ids >= count))[:, 0], torch.nonzero(~live & (ids < count))[:, 0]
    to = ids.clone()
    to[src] = dst
    s["pool"][:, dst] = s["pool"][:, src]
    table = s["table_a"]
    s["table_b"] = torch.where(table >= 0, to[table.clamp(min=0).long()].to(torch.int32), -1)
    s["refs_b"] = torch.zeros_like(refs).scatter_add(0, to[live], refs[live])
    s["live"] = count.to(torch.int32).view(1)


def _plain_sample(s):
    logits, t = s["logits"].double(), s["temperature"].double()[:, None]
    rows, vocab = logits.shape
    logits = torch.where(torch.isnan(logits), -math.inf, logits)
    top, first = logits.max(-1, keepdim=True)
    greedy = ~(t > 0)
    w = torch.where(logits == top, 1.0, torch.exp((logits - top) / torch.where(greedy, 1.0, t)))
    order = torch.sort(logits, dim=-1, descending=True, stable=True).indices
    rank = torch.arange(vocab, device="cuda")
    k = torch.where(s["top_k"] > 0, s["top_k"], vocab)[:, None]
    ws = torch.where(rank < k, w.gather(1, order), 0.0)
    upto = torch.cumsum(ws, -1)
    before = torch.cat([torch.zeros_like(upto[:, :1]), upto[:, :-1]], -1)
    p = s["top_p"].double()[:, None]
    kept = (rank < k) & ((p >= 1) | (before < p * upto[:, -1:])) & (ws >= s["min_p"][:, None])
    kept[:, 0] = True  # the most likely token always stays
    w = torch.zeros_like(w).scatter(1, order, torch.where(kept, ws, 0.0))
    upto = torch.cumsum(w, -1)
    total = upto[:, -1:]
    drawn = (upto <= s["u"].double()[:, None] * total).sum(-1, keepdim=True)
    best = torch.where(logits == top, rank, vocab).min(-1, keepdim=True).values
    token = torch.where(greedy, best, drawn.clamp(max=vocab - 1))
    prob = torch.where(greedy, 1.0, w.gather(1, token) / total)
    s["token"], s["prob"] = token[:, 0].to(torch.int32), prob[:, 0].float()


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
_kept = {}


def _package():
    if "hy_mt_rs_amd" not in sys.modules:
        spec = importlib.util.spec_from_file_location(
            "hy_mt_rs_amd", os.path.join(PKG, "__init__.py"), submodule_search_locations=[PKG])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["hy_mt_rs_amd"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["hy_mt_rs_amd"]


def _own(s):
    """The context a host thread keeps, and a state's layout, scratch and addresses."""
    if not _kept:
        hyq = _package()
        _kept.update(hyq=hyq, lib=hyq.lib(), handle=hyq.Context(0))
    hyq, L, h = _kept["hyq"], _kept["lib"], _kept["handle"].handle
    if "layout" not in s:
        c = s["case"]
        if c["kind"] == "sample":
            s["layout"], need = None, L.hyq_sample_scratch_bytes(c["rows"], c["vocab"])
        else:
            s["layout"] = hyq.KvLayout(hyq.DTYPES[c["dtype"]], c.get("layers", 1), c["kv_heads"],
                                       D, c["page_tokens"], s["pages"], c["slots"], s["width"])
            kl = ctypes.byref(s["layout"])
            need = (L.hyq_paged_attention_scratch_bytes(kl, s["rows"], s["most"], c["heads"])
                    if c["kind"] == "attention" else L.hyq_pages_scratch_bytes(kl))
        s["nbytes"] = need
        s["scratch"] = torch.empty(max(1, need), device="cuda", dtype=torch.uint8)
        s["at"] = {k: v.data_ptr() for k, v in s.items() if isinstance(v, torch.Tensor)}
    return hyq.check, L, h, ctypes.byref(s["layout"]) if s["layout"] is not None else None, s["at"]


def run(s):
    c = s["case"]
    kind = c["kind"]
    if kind == "append":
        if not own:
            return _plain_append(s)
        ok, L, h, kl, a = _own(s)
        ok(L.hyq_paged_rope_norm_append_d(h, kl, a["pool"], 0, a["table"], a["lens"], a["starts"],
                                          s["rows"], c["heads"], a["q"], a["k"], a["v"], a["qn"],
                                          a["kn"], a["freq"], EPS, c["norm_first"], a["out"]))
        return {"q": s["out"], "pool": s["pool"]}
    if kind == "attention":
        if not own:
            return _plain_attention(s)
        ok, L, h, kl, a = _own(s)
        ok(L.hyq_paged_attention_d(h, kl, a["pool"], 0, a["table"], a["lens"], a["starts"],
                                   s["rows"], s["most"], c["heads"], a["q"], a["scratch"],
                                   s["nbytes"], a["out"]))
        return s["out"]
    if kind == "beams":
        if not own:
            _plain_beams(s)
        else:
            ok, L, h, kl, a = _own(s)
            ok(L.hyq_pages_fork_d(h, kl, a["parent"], a["keep"], a["table"], a["lens"],
                                  a["table_a"], a["lens_a"], a["refs_a"]))
            ok(L.hyq_pages_extend_d(h, kl, a["pool"], a["add"], a["table_a"], a["lens_a"],
                                    a["refs_a"], a["table_b"], a["lens_b"], a["refs_b"],
                                    a["status"], a["scratch"], s["nbytes"]))
        return {k: s[k] for k in ("table_a", "lens_a", "refs_a", "table_b", "lens_b", "refs_b",
                                  "status", "pool")}
    if kind == "compact":
        if not own:
            s["table_a"], s["lens_a"], s["refs_a"] = _plain_fork(s, s["table"], s["lens"])
            _plain_compact(s)
        else:
            ok, L, h, kl, a = _own(s)
            ok(L.hyq_pages_fork_d(h, kl, a["parent"], a["keep"], a["table"], a["lens"],
                                  a["table_a"], a["lens_a"], a["refs_a"]))
            ok(L.hyq_pages_compact_d(h, kl, a["pool"], a["table_a"], a["refs_a"], a["table_b"],
                                     a["refs_b"], a["live"], a["scratch"], s["nbytes"]))
        return {k: s[k] for k in ("table_b", "refs_b", "live", "pool")}
    if not own:
        _plain_sample(s)
    else:
        ok, L, h, _, a = _own(s)
        ok(L.hyq_sample_d(h, a["logits"], c["rows"], c["vocab"], a["temperature"], a["top_k"],
                          a["top_p"], a["min_p"], a["u"], a["scratch"], s["nbytes"], a["token"],
                          a["prob"]))
    return {"token": s["token"], "prob": s["prob"]}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    c = case
    if c["kind"] == "sample":
        return dict(bytes=4 * c["rows"] * (c["vocab"] + 7), flops=4 * c["rows"] * c["vocab"])
    size = 2 if c["dtype"] == "F16" else 4
    pt = c["page_tokens"]
    if c["kind"] in ("beams", "compact"):
        r = random.Random(c["slots"] * 31 + c["context"])
        lens = [r.randint(pt, c["context"]) for _ in range(c["slots"])]
        width = _pages_of(c["context"], pt) + 2
        pages = sum(_pages_of(n, pt) for n in lens) + c["spare"] + 2 * c["slots"]
        parent = [min(g - g % 4 + r.choice([0, 0, 1, 2, 3]), c["slots"] - 1)
                  for g in range(c["slots"])]
        if c["slots"] > 4:
            parent[-1] = -1
        entries = c["slots"] * width
        token = 2 * c["kv_heads"] * D * size * c["layers"]
        kept = [p for p in parent if p >= 0]
        if c["kind"] == "beams":
            # a parent's partly filled page is copied for all of its beams but one
            copied = sum((kept.count(p) - 1) * (lens[p] % pt) for p in set(kept))
            return dict(bytes=4 * (4 * entries + 3 * pages) + 2 * copied * token, flops=0)
        # of the live pages, the share that lies behind their own count
        live = sum(_pages_of(lens[p], pt) for p in set(kept))
        moved = int(live * (pages - live) / pages)
        return dict(bytes=4 * (4 * entries + 3 * pages) + 2 * moved * pt * token, flops=0)
    lens, news = _batch(c)
    heads, kvh, rows = c["heads"], c["kv_heads"], sum(news)
    if c["kind"] == "append":
        return dict(bytes=rows * D * (4 * (2 * heads + 2 * kvh) + 2 * kvh * size),
                    flops=rows * D * 8 * (heads + kvh))
    held = sum(n for n, m in zip(lens, news) if m)
    seen = sum(m * n - m * (m - 1) // 2 for n, m in zip(lens, news))
    return dict(bytes=2 * held * kvh * D * size + 8 * rows * heads * D,
                flops=4 * D * heads * seen)


# ---------------------------------------------------------------------------
# the definition, in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    c = case
    s = _inputs(c, seed)
    if c["kind"] in ("beams", "compact"):
        return None  # whole numbers, and cached values copied as they are
    if c["kind"] == "sample":
        return {"token": None, "prob": _exact_probabilities(s)}
    lens, starts = s["lens"].tolist(), s["starts"].tolist()
    kvh, heads, pt = c["kv_heads"], c["heads"], c["page_tokens"]
    out = torch.zeros(s["rows"], heads * D, device="cuda", dtype=torch.float64)
    if c["kind"] == "append":
        pool = s["pool"].clone() if c["dtype"] == "F16" else s["pool"].double()
    for i, n in enumerate(lens):
        a, b = starts[i], starts[i + 1]
        if a == b:
            continue
        ids = s["table"][i, :_pages_of(n, pt)].long()
        q = s["q"][a:b].double().view(b - a, heads, D)
        if c["kind"] == "attention":
            kv = s["pool"][0, ids].double()                    # [pages, 2, kvh, pt, D]
            hidden = torch.ones(b - a, n, device="cuda", dtype=torch.bool).triu(n - (b - a) + 1)
            for h in range(heads):
                k, v = (kv[:, x, h * kvh // heads].reshape(-1, D)[:n] for x in (0, 1))
                sc = (q[:, h] @ k.t().contiguous() / math.sqrt(D)).masked_fill(hidden, -math.inf)
                out[a:b, h * D:(h + 1) * D] = torch.softmax(sc, -1) @ v
            continue
        for r in range(a, b):
            pos = n - b + r
            z = torch.polar(torch.ones(D // 2, device="cuda", dtype=torch.float64),
                            pos * s["freq"].double())

            def formed(x, weight):
                x = x.double().view(-1, D)
                rms = torch.sqrt(x.square().sum(-1, keepdim=True) / D + EPS)
                if c["norm_first"]:
                    x = x / rms * weight.double()
                y = torch.complex(x[:, :D // 2].contiguous(), x[:, D // 2:].contiguous()) * z
                y = torch.cat([y.real, y.imag], -1)
                return y if c["norm_first"] else y / rms * weight.double()

            out[r] = formed(s["q"][r], s["qn"]).flatten()
            pool[0, ids[pos // pt], 0, :, pos % pt] = formed(s["k"][r], s["kn"]).to(pool.dtype)
            pool[0, ids[pos // pt], 1, :, pos % pt] = s["v"][r].view(-1, D).to(pool.dtype)
    if c["kind"] == "attention":
        return out
    return {"q": out, "pool": pool if c["dtype"] == "F32" else None}


def _exact_probabilities(s):
    import numpy as np
    probs = []
    values = {k: s[k].double().cpu().numpy() for k in ("logits", "temperature", "top_p", "min_p", "u")}
    for r, k in enumerate(s["top_k"].tolist()):
        x, t = values["logits"][r], values["temperature"][r]
        if not t > 0:
            probs.append(1.0)
            continue
        order = np.argsort(-x, kind="stable")
        order = order[:k] if k > 0 else order
        w = np.exp((x[order] - x[order[0]]) / t)
        keep = len(w)
        if values["top_p"][r] < 1:
            reached = np.cumsum(w) >= values["top_p"][r] * w.sum()
            keep = int(np.argmax(reached)) + 1
        keep = max(1, min(keep, int((w >= values["min_p"][r]).sum())))
        byindex = np.argsort(order[:keep])
        w = w[:keep][byindex]
        upto = np.cumsum(w)
        at = min(int(np.searchsorted(upto, values["u"][r] * upto[-1], side="right")), keep - 1)
        probs.append(w[at] / upto[-1])
    return torch.tensor(probs, device="cuda", dtype=torch.float64)
