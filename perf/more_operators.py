"""More operators of a serving step over a paged KV cache, as measurable cases.

Beside what perf/operators.py measures, a server may hold its cache in 8 bits
(``store``: new tokens' keys and values quantised as they are written, and read
back; ``attention8``: attention over such pages), compute the attention over a
prefix that many of its slots share once for all of them (``shared``: the plan
of a step, then every layer's attention), and change the logits by each
request's penalties, biases and grammar before it samples (``adjust``).

Pools are [layers][pages][2][kv_heads][page_tokens][128] (keys, then values);
an 8-bit page holds one byte for each number - a key's code as a signed byte,
a value's as code + 128 - and behind them one f32 scale for every 128 of them,
[2][kv_heads][page_tokens]. Page tables are [slots][entries] of page ids, -1
where a slot holds none. Head counts, widths and vocabularies are those of the
1.8B and 7B models that bench.py builds, or generic.
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
        # one new token in each of 48 sessions, into 8-bit pages and back
        dict(name="store_decode", kind="store", page_tokens=64, slots=48, prompts=0, chunk=1,
             step=1, idle=0, context=4096, pad=0, norm_first=False, **small),
        # six prompts of some hundred tokens at once, in a padded batch
        dict(name="store_prompts", kind="store", page_tokens=32, slots=6, prompts=6, chunk=500,
             step=1, idle=0, context=2500, pad=13, norm_first=True, **large),
        # the two concurrent requests that a server takes by default
        dict(name="attn8_two", kind="attention8", page_tokens=64, slots=2, prompts=0, chunk=1,
             step=1, idle=0, context=1100, pad=0, **small),
        # 64 sessions of very different length
        dict(name="attn8_decode", kind="attention8", page_tokens=64, slots=64, prompts=0, chunk=1,
             step=1, idle=0, context=8192, pad=0, **large),
        # a few sessions over whole books
        dict(name="attn8_long", kind="attention8", page_tokens=128, slots=4, prompts=0, chunk=1,
             step=1, idle=0, context=60001, pad=0, **small),
        # the second part of one prompt
        dict(name="attn8_prompt", kind="attention8", page_tokens=64, slots=1, prompts=1, chunk=512,
             step=1, idle=0, context=2012, pad=0, **small),
        # three prompts taken in beside 27 running sessions and two empty slots
        dict(name="attn8_mixed", kind="attention8", page_tokens=64, slots=32, prompts=3, chunk=400,
             step=1, idle=2, context=4000, pad=5, **large),
        # the beams of one long prompt, through a few layers
        dict(name="shared_beams", kind="shared", dtype="F32", page_tokens=32, groups=1, members=8,
             lone=0, prefix=1500, tail=60, step=1, layers=4, hint=False, **small),
        # many requests behind one long instruction with its glossary
        dict(name="shared_batch", kind="shared", dtype="F16", page_tokens=64, groups=1, members=64,
             lone=0, prefix=8200, tail=300, step=1, layers=2, hint=False, **large),
        # four instructions and some requests of their own, in 8-bit pages, drafted tokens
        dict(name="shared_groups", kind="shared", dtype="Q8", page_tokens=64, groups=4, members=24,
             lone=9, prefix=3100, tail=700, step=3, layers=2, hint=True, **large),
        # two requests with a translation model's usual penalty
        dict(name="adjust_two", kind="adjust", rows=2, vocab=VOCAB_1P8B, history=900, biases=0,
             masks=0),
        # 64 requests with penalties, biases and grammars of their own
        dict(name="adjust_batch", kind="adjust", rows=64, vocab=VOCAB_7B, history=4000,
             biases=300, masks=8),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(["store", "attention8", "shared", "adjust"], [2, 5, 4, 3])[0]
    if kind == "adjust":
        vocab = rng.choice([VOCAB_1P8B, VOCAB_7B, _log_int(rng, 1000, 120000)])
        return dict(kind=kind, rows=_log_int(rng, 1, 64), vocab=vocab,
                    history=_log_int(rng, 1, 4000), biases=rng.choice([0, _log_int(rng, 1, 400)]),
                    masks=rng.choice([0, rng.randint(1, 12)]))
    heads, kv_heads = rng.choice([(16, 4), (32, 8), (8, 2), (12, 4), (8, 8), (16, 2)])
    page_tokens = rng.choice([16, 32, 64, 128])
    case = dict(kind=kind, page_tokens=page_tokens, heads=heads, kv_heads=kv_heads)
    if kind == "shared":
        rep = heads // kv_heads
        groups = rng.choice([1, 1, rng.randint(2, 6)])
        return dict(case, dtype=rng.choice(["F32", "F16", "Q8"]), groups=groups,
                    members=_log_int(rng, 2, 64 // groups), lone=rng.choice([0, rng.randint(1, 8)]),
                    prefix=_log_int(rng, page_tokens, 8000 if groups == 1 else 3000),
                    tail=_log_int(rng, 6, 500), step=rng.choice([1, 1, min(16 // rep, 4)]),
                    layers=rng.randint(1, 2), hint=rng.random() < 0.5)
    case["pad"] = rng.choice([0, _log_int(rng, 1, 60)])
    if kind == "store":
        case["norm_first"] = rng.random() < 0.5
    form = rng.choice(["decode", "decode", "draft", "prompt", "mixed"])
    if form == "prompt":
        chunk = _log_int(rng, 2, 500)
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


def _sharing(case):
    """Slots of a ``shared`` case: the group of each (-1: its own), positions held
    and new tokens, and the pages that the slots of a group share."""
    c = case
    r = random.Random(c["members"] * 917 + c["prefix"])
    who = [g for g in range(c["groups"]) for _ in range(c["members"])] + [-1] * c["lone"]
    r.shuffle(who)
    # a prefix ends where it ends: the slots share its whole pages
    common = [max(1, (c["prefix"] - (g * c["prefix"]) // 7) // c["page_tokens"])
              for g in range(c["groups"])]
    lens = [(common[g] * c["page_tokens"] if g >= 0 else 0) + c["step"] + r.randint(0, c["tail"])
            for g in who]
    return who, lens, [c["step"]] * len(who), common


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
class Source:
    """Seeded random tensors on the GPU, in the order they are asked for."""

    def __init__(self, seed):
        self.g = torch.Generator("cuda")
        self.g.manual_seed(int(seed) * 7507 + 11)

    def normal(self, *shape, dtype=torch.float32):
        return torch.randn(shape, generator=self.g, device="cuda", dtype=dtype)

    def uniform(self, *shape):
        return torch.rand(shape, generator=self.g, device="cuda", dtype=torch.float32)

    def whole(self, lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=self.g, device="cuda", dtype=torch.int32)

    def order(self, n):
        return torch.randperm(n, generator=self.g, device="cuda").to(torch.int32)


def _ints(values):
    return torch.tensor(values, device="cuda", dtype=torch.int32)


def _pages_of(n, page_tokens):
    return -(-n // page_tokens)


def _parts(pool, case):
    """An 8-bit pool's codes (bytes) [layers][pages][2][kv_heads][page_tokens][128]
    and scales [layers][pages][2][kv_heads][page_tokens], as views of it."""
    kvh, pt = case["kv_heads"], case["page_tokens"]
    n = 2 * kvh * pt * D
    codes = pool[..., :n].unflatten(-1, (2, kvh, pt, D))
    return codes, pool[..., n:].view(torch.float32).unflatten(-1, (2, kvh, pt))


def _quantise(x):
    """Codes in -127 .. 127 and the scale of each row of 128 numbers (64 bits)."""
    scale = (x.abs().amax(-1) / 127.0).float()
    safe = torch.where(scale > 0, scale, 1.0).double()
    return torch.round(x / safe[..., None]), scale


def _pool(src, case, layers, pages):
    kvh, pt = case["kv_heads"], case["page_tokens"]
    dtype = case.get("dtype", "Q8")
    shape = (layers, pages, 2, kvh, pt, D)
    if dtype != "Q8":
        return src.normal(*shape, dtype=torch.float16 if dtype == "F16" else torch.float32)
    pool = torch.zeros(layers, pages, 2 * kvh * pt * (D + 4), device="cuda", dtype=torch.uint8)
    codes, scales = _parts(pool, case)
    for layer in range(layers):
        x = src.normal(pages, 2, kvh, pt, D)
        scale = x.abs().amax(-1) / 127.0
        code = torch.round(x / scale[..., None])
        code[:, 1] += 128.0
        codes[layer] = code.to(torch.int16).to(torch.uint8)  # (a negative key's code by its low byte)
        scales[layer] = scale
    return pool


def _adjust_inputs(c, src):
    rows, vocab = c["rows"], c["vocab"]
    logits = 2.0 * src.normal(rows, vocab)
    likely = src.whole(0, vocab, rows, 24).long()
    logits.scatter_add_(1, likely, 12.0 * src.uniform(rows, 24))
    r = random.Random(rows * 7 + c["history"])
    lens = [c["history"]] + [r.randint(0, c["history"]) for _ in range(rows - 1)]
    # a third of a text's tokens are those of few words
    history = torch.where(src.uniform(rows, c["history"]) < 0.33,
                          src.whole(0, min(vocab, 50), rows, c["history"]),
                          src.whole(0, vocab, rows, c["history"]))
    some = c["masks"] or c["biases"]  # requests with settings of their own, or the usual one
    settings = [(1.05, 0.0, 0.0)] * rows if not some else [
        [(1.05, 0.0, 0.0), (1.0, 0.5, 0.2), (1.3, 0.0, 0.0), (1.0, 0.0, 0.0),
         (1.1, -0.3, 0.7)][i % 5] for i in range(rows)]
    rep, pres, freq = zip(*settings)
    f = dict(device="cuda", dtype=torch.float32)
    s = dict(logits=logits, history=history, history_len=_ints(lens),
             prompt_len=_ints([n // 2 for n in lens]), repetition=torch.tensor(rep, **f),
             presence=torch.tensor(pres, **f), frequency=torch.tensor(freq, **f))
    if c["biases"]:
        n = min(c["biases"], vocab)
        counts = [n if i % 3 == 0 else (i * 37) % (n + 1) for i in range(rows)]
        token = src.uniform(rows, vocab).topk(n, dim=1).indices.to(torch.int32)
        value = 8.0 * src.normal(rows, n)
        given = torch.arange(n, device="cuda") < _ints(counts)[:, None]
        s.update(bias_token=token[given], bias=value[given],
                 bias_start=_ints([sum(counts[:i]) for i in range(rows + 1)]))
    if c["masks"]:
        words = -(-vocab // 32)
        # grammars that allow nearly all, half and few of the tokens
        share = torch.tensor([(0.98, 0.5, 0.03)[m % 3] for m in range(c["masks"])], **f)
        allowed = src.uniform(c["masks"], words * 32) < share[:, None]
        bits = allowed.view(c["masks"], words, 32).long() << torch.arange(32, device="cuda")
        s.update(mask=(bits.sum(-1) & 0xffffffff).to(torch.int64).where(
            bits.sum(-1) < 2 ** 31, bits.sum(-1) - 2 ** 32).to(torch.int32),
            mask_row=_ints([-1 if i % 4 == 3 else i % c["masks"] for i in range(rows)]))
    return s


def _inputs(case, seed):
    c, src = case, Source(seed)
    if c["kind"] == "adjust":
        return _adjust_inputs(c, src)
    pt = c["page_tokens"]
    if c["kind"] == "shared":
        who, lens, news, common = _sharing(c)
        layers = c["layers"]
    else:
        lens, news = _batch(c)
        who, common, layers = [-1] * len(lens), [], 1
    width = _pages_of(max(lens), pt) + 1
    counts = [_pages_of(n, pt) - (common[g] if g >= 0 else 0) for n, g in zip(lens, who)]
    pages = sum(counts) + sum(common) + 5
    ids = src.order(pages)
    table = torch.full((len(lens), width), -1, device="cuda", dtype=torch.int32)
    at = sum(common)
    for s, n in enumerate(counts):
        have = common[who[s]] if who[s] >= 0 else 0
        if have:
            first = sum(common[:who[s]])
            table[s, :have] = ids[first:first + have]
        table[s, have:have + n] = ids[at:at + n]
        at += n
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    rows = starts[-1] + c.get("pad", 0)
    s = dict(table=table, lens=_ints(lens), starts=_ints(starts), pages=pages, width=width,
             slots=len(lens), rows=rows, new=starts[-1], most=max(news), layers=layers,
             pool=_pool(src, c, layers, pages), group=_ints(who),
             q=src.normal(layers, rows, c["heads"] * D))
    if c["kind"] == "store":
        j = torch.arange(D // 2, device="cuda", dtype=torch.float64)
        s.update(q=s["q"][0], k=src.normal(rows, c["kv_heads"] * D),
                 v=src.normal(rows, c["kv_heads"] * D), qn=1.0 + 0.02 * src.normal(D),
                 kn=1.0 + 0.02 * src.normal(D), freq=(ROPE_BASE ** (-2.0 * j / D)).float())
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["kind"] == "adjust":
        s["out"] = torch.zeros_like(s["logits"])
    else:
        s["out"] = torch.zeros_like(s["q"])
    if case["kind"] == "store":
        s.update(k_back=torch.zeros_like(s["k"]), v_back=torch.zeros_like(s["v"]))
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


def _plain_store(s):
    """Rotation and norms; keys, whose codes a last bit may turn, in 64 bits."""
    c, n = s["case"], s["new"]
    slot, pos = _rows_of(s)
    angle = pos[:, None].double() * s["freq"].double()
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]

    def norm(x, w):
        return x * (w.to(x) / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS))

    def turn(x):
        a, b = x[..., :D // 2], x[..., D // 2:]
        return torch.cat([a * cos.to(x) - b * sin.to(x), a * sin.to(x) + b * cos.to(x)], -1)

    def both(x, w):
        x = x.view(n, -1, D)
        return turn(norm(x, w)) if c["norm_first"] else norm(turn(x), w)

    s["out"][:n] = both(s["q"][:n], s["qn"]).reshape(n, -1)
    codes, scales = _parts(s["pool"], c)
    codes, scales = codes[0], scales[0]
    page, at = s["table"][slot, pos // c["page_tokens"]].long(), pos % c["page_tokens"]
    kc, ks = _quantise(both(s["k"][:n].double(), s["kn"]))
    vc, vs = _quantise(s["v"][:n].double().view(n, -1, D))
    codes[page, 0, :, at] = kc.to(torch.int16).to(torch.uint8)
    codes[page, 1, :, at] = (vc + 128.0).to(torch.uint8)
    scales[page, 0, :, at], scales[page, 1, :, at] = ks, vs
    k = codes[page, 0, :, at].view(torch.int8).float() * scales[page, 0, :, at][..., None]
    v = (codes[page, 1, :, at].float() - 128.0) * scales[page, 1, :, at][..., None]
    s["k_back"][:n], s["v_back"][:n] = k.reshape(n, -1), v.reshape(n, -1)
    return {"q": s["out"], "k": s["k_back"], "v": s["v_back"]}


def _cached(s, table):
    """Keys and values [2, layers, slots, kv_heads, positions, 128] in 32 bits."""
    c, at = s["case"], table.clamp(min=0).long()
    if c.get("dtype", "Q8") == "Q8":
        codes, scales = _parts(s["pool"], c)
        codes, scales = codes[:, at], scales[:, at]
        k = codes[:, :, :, 0].view(torch.int8).float() * scales[:, :, :, 0, ..., None]
        v = (codes[:, :, :, 1].float() - 128.0) * scales[:, :, :, 1, ..., None]
        pages = torch.stack([k, v])
    else:
        pages = s["pool"][:, at].permute(3, 0, 1, 2, 4, 5, 6).float()
    pages = pages.transpose(3, 4)  # [2, layers, slots, kv_heads, width, page_tokens, 128]
    return pages.reshape(*pages.shape[:4], -1, D)


def _plain_attention(s):
    c, pt = s["case"], s["case"]["page_tokens"]
    slots, layers, kvh, heads, most = s["slots"], s["layers"], c["kv_heads"], c["heads"], s["most"]
    keys, values = _cached(s, s["table"])
    i = torch.arange(most, device="cuda")
    count = s["starts"][1:] - s["starts"][:-1]
    given = i < count[:, None]                                 # [slots, most]
    row = torch.where(given, s["starts"][:-1, None] + i, 0).long()
    q = s["q"][:, row].view(layers, slots, most, kvh, heads // kvh, D).transpose(2, 3)
    scores = torch.matmul(q.reshape(layers * slots * kvh, -1, D) * D ** -0.5,
                          keys.reshape(layers * slots * kvh, -1, D).transpose(-1, -2))
    scores = scores.view(layers, slots, kvh, most, heads // kvh, -1)
    last = (s["lens"] - count)[:, None] + i                    # a row's own position
    seen = torch.arange(s["width"] * pt, device="cuda") <= last[:, :, None]
    scores = scores.masked_fill(~seen[:, None, :, None], -math.inf)
    e = torch.exp(scores - scores.max(-1, keepdim=True).values)
    p = (e / e.sum(-1, keepdim=True)).view(layers * slots * kvh, -1, seen.shape[-1])
    o = torch.matmul(p, values.reshape(layers * slots * kvh, -1, D))
    o = o.view(layers, slots, kvh, most, -1, D).transpose(2, 3).reshape(layers, slots, most, -1)
    s["out"][:, :s["new"]] = o[:, given]
    return s["out"]


def _bits(words, tokens):
    """The bits of `tokens` in rows of 32-bit words."""
    return (words[:, tokens >> 5] >> (tokens & 31).to(torch.int32)) & 1


def _plain_adjust(s):
    c, x = s["case"], s["logits"]
    rows, vocab = x.shape
    at = torch.arange(c["history"], device="cuda")
    held = at < s["history_len"][:, None]
    token = s["history"].long()
    none = torch.zeros(rows, vocab, device="cuda", dtype=torch.int32)
    seen = none.scatter_add(1, token, held.to(torch.int32)) > 0
    count = none.scatter_add(1, token, (held & (at >= s["prompt_len"][:, None])).to(torch.int32))
    r = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - torch.where(count > 0, s["presence"][:, None] + s["frequency"][:, None] * count, 0.0)
    if c["biases"]:
        pair = torch.arange(s["bias"].numel(), device="cuda")
        row = torch.searchsorted(s["bias_start"].long(), pair, right=True) - 1
        x[row, s["bias_token"].long()] += s["bias"]
    if c["masks"]:
        allowed = _bits(s["mask"], torch.arange(vocab, device="cuda")) != 0
        of = s["mask_row"].long()
        x = torch.where((of < 0)[:, None] | allowed[of.clamp(min=0)], x, -math.inf)
    s["out"].copy_(x)
    return s["out"]


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
    if "at" not in s:
        c = s["case"]
        at = {k: v.data_ptr() for k, v in s.items() if isinstance(v, torch.Tensor)}
        if c["kind"] == "adjust":
            s["layout"] = hyq.LogitRules(
                at["history"], at["history_len"], at["prompt_len"], c["history"],
                at["repetition"], at["presence"], at["frequency"], at.get("bias_start"),
                at.get("bias_token"), at.get("bias"), s["bias"].numel() if c["biases"] else 0,
                at.get("mask"), at.get("mask_row"), c["masks"])
        else:
            dtype = {"F32": hyq.F32, "F16": hyq.F16, "Q8": hyq.KV_Q8}[c.get("dtype", "Q8")]
            s["layout"] = hyq.KvLayout(dtype, s["layers"], c["kv_heads"], D, c["page_tokens"],
                                       s["pages"], s["slots"], s["width"])
            kl, sizes = ctypes.byref(s["layout"]), {}
            if c["kind"] == "attention8":
                sizes["scratch"] = L.hyq_paged_attention_scratch_bytes(kl, s["rows"], s["most"],
                                                                       c["heads"])
            if c["kind"] == "shared":
                sizes["plan"] = L.hyq_paged_shared_plan_bytes(kl, s["rows"], c["heads"])
                sizes["scratch"] = L.hyq_paged_shared_attention_scratch_bytes(
                    kl, s["rows"], s["most"], c["heads"])
            s["sizes"] = sizes
            for name, n in sizes.items():
                s[name] = torch.empty(max(1, n), device="cuda", dtype=torch.uint8)
                at[name] = s[name].data_ptr()
        s["at"] = at
    return hyq.check, L, h, ctypes.byref(s["layout"]), s["at"]


def run(s):
    c = s["case"]
    kind = c["kind"]
    if not own:
        return {"store": _plain_store, "attention8": _plain_attention, "shared": _plain_attention,
                "adjust": _plain_adjust}[kind](s)
    ok, L, h, kl, a = _own(s)
    if kind == "adjust":
        ok(L.hyq_logits_adjust_d(h, a["logits"], c["rows"], c["vocab"], kl, a["out"]))
        return s["out"]
    if kind == "store":
        ok(L.hyq_paged_rope_norm_append_d(h, kl, a["pool"], 0, a["table"], a["lens"], a["starts"],
                                          s["rows"], c["heads"], a["q"], a["k"], a["v"], a["qn"],
                                          a["kn"], a["freq"], EPS, c["norm_first"], a["out"]))
        ok(L.hyq_paged_read_d(h, kl, a["pool"], 0, a["table"], a["lens"], a["starts"], s["rows"],
                              a["k_back"], a["v_back"]))
        return {"q": s["out"], "k": s["k_back"], "v": s["v_back"]}
    if kind == "attention8":
        ok(L.hyq_paged_attention_d(h, kl, a["pool"], 0, a["table"], a["lens"], a["starts"],
                                   s["rows"], s["most"], c["heads"], a["q"], a["scratch"],
                                   s["sizes"]["scratch"], a["out"]))
        return s["out"]
    ok(L.hyq_paged_shared_plan_d(h, kl, a["group"] if c["hint"] else None, a["table"], a["lens"],
                                 a["starts"], s["rows"], c["heads"], a["plan"],
                                 s["sizes"]["plan"]))
    size = s["rows"] * c["heads"] * D * 4
    for layer in range(s["layers"]):
        ok(L.hyq_paged_shared_attention_d(
            h, kl, a["pool"], layer, a["table"], a["lens"], a["starts"], s["rows"], s["most"],
            c["heads"], a["plan"], s["sizes"]["plan"], a["q"] + layer * size, a["scratch"],
            s["sizes"]["scratch"], a["out"] + layer * size))
    return s["out"]


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    c = case
    if c["kind"] == "adjust":
        n = c["rows"] * c["vocab"]
        return dict(bytes=8 * n + c["masks"] * c["vocab"] // 8
                    + c["rows"] * (2 * c["history"] + 4 * c["biases"]), flops=4 * n)
    kvh, heads = c["kv_heads"], c["heads"]
    cached = 2 * kvh * {"F32": 4 * D, "F16": 2 * D, "Q8": D + 4}[c.get("dtype", "Q8")]
    if c["kind"] == "shared":
        who, lens, news, common = _sharing(c)
        shared = [common[g] * c["page_tokens"] if g >= 0 else 0 for g in who]
        held = sum(lens) - sum(shared) + sum(common) * c["page_tokens"]
        layers = c["layers"]
    else:
        lens, news = _batch(c)
        held, layers = sum(n for n, m in zip(lens, news) if m), 1
    rows = sum(news)
    if c["kind"] == "store":  # (what is written is read again)
        return dict(bytes=rows * (4 * D * (2 * heads + 4 * kvh) + 2 * cached),
                    flops=rows * D * 8 * (heads + 2 * kvh))
    seen = sum(m * n - m * (m - 1) // 2 for n, m in zip(lens, news))
    return dict(bytes=layers * (held * cached + 8 * rows * heads * D),
                flops=layers * 4 * D * heads * seen)


# ---------------------------------------------------------------------------
# the definition, in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    c = case
    s = _inputs(c, seed)
    if c["kind"] == "adjust":
        return _exact_adjust(s, c)
    lens, starts = s["lens"].tolist(), s["starts"].tolist()
    kvh, heads, pt = c["kv_heads"], c["heads"], c["page_tokens"]
    if c["kind"] == "store":
        return _exact_store(s, c, lens, starts)
    out = torch.zeros(s["layers"], s["rows"], heads * D, device="cuda", dtype=torch.float64)
    for layer in range(s["layers"]):
        for i, n in enumerate(lens):
            a, b = starts[i], starts[i + 1]
            if a == b:
                continue
            ids = s["table"][i, :_pages_of(n, pt)].long()
            page = s["pool"][layer, ids]
            if page.dtype == torch.uint8:
                codes, scales = _parts(page, c)
                sign = torch.tensor([0.0, 128.0], device="cuda", dtype=torch.float64)
                kv = codes.double() - sign[:, None, None, None]
                kv[:, 0] = torch.where(kv[:, 0] > 127, kv[:, 0] - 256, kv[:, 0])
                kv = kv * scales.double()[..., None]
            else:
                kv = page.double()                              # [pages, 2, kvh, pt, D]
            q = s["q"][layer, a:b].double().view(b - a, heads, D)
            hidden = torch.ones(b - a, n, device="cuda", dtype=torch.bool).triu(n - (b - a) + 1)
            for h in range(heads):
                k, v = (kv[:, x, h * kvh // heads].reshape(-1, D)[:n] for x in (0, 1))
                sc = (q[:, h] @ k.t().contiguous() / math.sqrt(D)).masked_fill(hidden, -math.inf)
                out[layer, a:b, h * D:(h + 1) * D] = torch.softmax(sc, -1) @ v
    return out


def _exact_store(s, c, lens, starts):
    kvh = c["kv_heads"]
    outs = {n: torch.zeros(s["rows"], w * D, device="cuda", dtype=torch.float64)
            for n, w in (("q", c["heads"]), ("k", kvh), ("v", kvh))}
    for i, n in enumerate(lens):
        a, b = starts[i], starts[i + 1]
        if a == b:
            continue
        pos = torch.arange(n - (b - a), n, device="cuda", dtype=torch.float64)
        z = torch.polar(torch.ones(b - a, 1, D // 2, device="cuda", dtype=torch.float64),
                        (pos[:, None] * s["freq"].double())[:, None])

        def formed(x, weight):
            x = x[a:b].double().view(b - a, -1, D)
            rms = torch.sqrt(x.square().sum(-1, keepdim=True) / D + EPS)
            if c["norm_first"]:
                x = x / rms * weight.double()
            y = torch.complex(x[..., :D // 2].contiguous(), x[..., D // 2:].contiguous()) * z
            y = torch.cat([y.real, y.imag], -1)
            return y if c["norm_first"] else y / rms * weight.double()

        def held(x):
            step = (x.abs().max(-1, keepdim=True).values / 127.0).float().double()
            return torch.round(x / step) * step

        outs["q"][a:b] = formed(s["q"], s["qn"]).flatten(1)
        outs["k"][a:b] = held(formed(s["k"], s["kn"])).flatten(1)
        outs["v"][a:b] = held(s["v"][a:b].double().view(b - a, kvh, D)).flatten(1)
    return outs


def _exact_adjust(s, c):
    import numpy as np
    x = s["logits"].double().cpu().numpy()
    get = {k: v.cpu().numpy() for k, v in s.items() if k != "logits"}
    for r in range(c["rows"]):
        tokens = get["history"][r, :get["history_len"][r]]
        seen = np.unique(tokens)
        rep = float(get["repetition"][r])
        x[r, seen] = np.where(x[r, seen] > 0, x[r, seen] / rep, x[r, seen] * rep)
        made, count = np.unique(tokens[get["prompt_len"][r]:], return_counts=True)
        x[r, made] -= float(get["presence"][r]) + float(get["frequency"][r]) * count
        if c["biases"]:
            a, b = get["bias_start"][r], get["bias_start"][r + 1]
            x[r, get["bias_token"][a:b]] += get["bias"][a:b].astype(np.float64)
        if c["masks"] and get["mask_row"][r] >= 0:
            words = get["mask"][get["mask_row"][r]].view(np.uint32)
            bits = np.unpackbits(words.view(np.uint8), bitorder="little")[:c["vocab"]]
            x[r, bits == 0] = -np.inf
    return torch.tensor(x, device="cuda", dtype=torch.float64)
