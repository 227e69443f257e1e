"""CPU tests of the paged cache's and the sampler's entry points: layouts and
sizes, and every refusal, which is made before a device is touched (the
context given is then never read)."""
import ctypes

import pytest

GOOD = dict(dtype=1, layers=2, kv_heads=4, head_dim=128, page_tokens=64, pages=10, seqs=3, stride=8)


@pytest.fixture(scope="module")
def L(hyq):
    return hyq.lib()


@pytest.fixture(scope="module")
def ctx():
    return ctypes.create_string_buffer(1 << 16)


def layout(hyq, **kw):
    return hyq.KvLayout(*{**GOOD, **kw}.values())


def test_pool_bytes(hyq, L):
    kl = layout(hyq)
    assert L.hyq_kv_pool_bytes(ctypes.byref(kl)) == 2 * 10 * 2 * 4 * 64 * 128 * 2
    kl = layout(hyq, dtype=0)
    assert L.hyq_kv_pool_bytes(ctypes.byref(kl)) == 2 * 10 * 2 * 4 * 64 * 128 * 4
    assert L.hyq_kv_pool_bytes(None) == 0


BAD = [dict(dtype=8), dict(layers=0), dict(kv_heads=0), dict(kv_heads=257), dict(head_dim=64),
       dict(page_tokens=8), dict(page_tokens=48), dict(page_tokens=512), dict(pages=0),
       dict(pages=(1 << 24) + 1), dict(seqs=0), dict(seqs=4097), dict(stride=0),
       dict(stride=(1 << 18) + 1),
       # more bytes than a size holds (2^16 * 2^24 pages of 2^26)
       dict(dtype=0, layers=65536, pages=1 << 24, kv_heads=256, page_tokens=256)]


@pytest.mark.parametrize("bad", BAD, ids=str)
def test_layouts_are_refused(hyq, L, ctx, bad):
    kl = ctypes.byref(layout(hyq, **bad))
    code = hyq.EDTYPE if bad.get("dtype", 0) == 8 else hyq.EINVAL
    assert L.hyq_kv_pool_bytes(kl) == 0
    assert L.hyq_pages_scratch_bytes(kl) == 0
    assert L.hyq_paged_attention_scratch_bytes(kl, 1, 1, 4) == 0
    p = 4096
    assert L.hyq_paged_rope_norm_append_d(ctx, kl, p, 0, p, p, p, 1, 4, p, p, p, p, p, p, 1e-5, 0,
                                          p) == code
    assert L.hyq_paged_attention_d(ctx, kl, p, 0, p, p, p, 1, 1, 4, p, p, 1 << 40, p) == code
    assert L.hyq_pages_fork_d(ctx, kl, p, p, p, p, p + 64, p + 64, p) == code
    assert L.hyq_pages_extend_d(ctx, kl, p, p, p, p, p, p, p, p, p, p, 1 << 40) == code
    assert L.hyq_pages_compact_d(ctx, kl, p, p, p, p, p, p, p, 1 << 40) == code


def _calls(hyq, L, ctx, kl):
    """(call, good arguments, positions of its pointers, those that may be null
    and those that must be 16-byte aligned)"""
    p, big = 4096, 1 << 40
    return {
        "append": (L.hyq_paged_rope_norm_append_d,
                   [ctx, kl, p, 0, p, p, p, 5, 16, p, p, p, p, p, p, 1e-5, 0, p],
                   [2, 4, 5, 6, 9, 10, 11, 12, 13, 14, 17], [2, 9, 10, 11, 12, 13, 14, 17]),
        "attention": (L.hyq_paged_attention_d,
                      [ctx, kl, p, 0, p, p, p, 5, 2, 16, p, p, big, p],
                      [2, 4, 5, 6, 10, 11, 13], [2, 10, 11, 13]),
        "fork": (L.hyq_pages_fork_d, [ctx, kl, p, p, p, p, p + 64, p + 64, p],
                 [2, 4, 5, 6, 7, 8], []),
        "extend": (L.hyq_pages_extend_d, [ctx, kl, p, p, p, p, p, p, p, p, p, p, big],
                   [2, 3, 4, 5, 6, 7, 8, 9, 10, 11], [2, 11]),
        "compact": (L.hyq_pages_compact_d, [ctx, kl, p, p, p, p, p, p, p, big],
                    [2, 3, 4, 5, 6, 7, 8], [2, 8]),
    }


@pytest.mark.parametrize("name", ["append", "attention", "fork", "extend", "compact"])
def test_pointers_are_refused(hyq, L, ctx, name):
    layout_ = layout(hyq)
    call, good, pointers, aligned = _calls(hyq, L, ctx, ctypes.byref(layout_))[name]
    for i in [0, 1] + pointers:
        assert call(*[None if j == i else a for j, a in enumerate(good)]) == hyq.EINVAL, i
        assert b"null" in L.hyq_last_error()
    for i in aligned:
        assert call(*[a + 4 if j == i else a for j, a in enumerate(good)]) == hyq.EINVAL, i
        assert b"aligned" in L.hyq_last_error()


def test_shapes_and_scratch_are_refused(hyq, L, ctx):
    layout_ = layout(hyq)
    calls = _calls(hyq, L, ctx, ctypes.byref(layout_))

    def refused(name, word, **change):
        call, good, _, _ = calls[name]
        args = list(good)
        for i, v in change.items():
            args[int(i[1:])] = v
        assert call(*args) == hyq.EINVAL, (name, change)
        assert word in L.hyq_last_error(), (name, change, L.hyq_last_error())

    for layer in (-1, 2):
        refused("append", b"layer", _3=layer)
        refused("attention", b"layer", _3=layer)
    for heads in (0, 6, 68):  # none, not a multiple, 17 per KV head
        refused("append", b"heads", _8=heads)
        refused("attention", b"heads", _9=heads)
    refused("append", b"rows", _7=(1 << 20) + 1)
    for rows in (0, (1 << 20) + 1):
        refused("attention", b"rows", _7=rows)
    refused("attention", b"rows", _8=0)
    kl = ctypes.byref(layout_)
    need = L.hyq_paged_attention_scratch_bytes(kl, 5, 2, 16)
    assert need > 0
    refused("attention", b"scratch", _12=need - 1)
    refused("attention", b"must not be q", _12=need)  # (the output is q here)
    refused("extend", b"scratch", _12=L.hyq_pages_scratch_bytes(kl) - 1)
    refused("compact", b"scratch", _9=L.hyq_pages_scratch_bytes(kl) - 1)
    refused("fork", b"old", _6=4096)
    refused("fork", b"old", _7=4096)
    assert L.hyq_paged_attention_scratch_bytes(kl, 0, 1, 16) == 0
    assert L.hyq_paged_attention_scratch_bytes(kl, 1, 0, 16) == 0
    assert L.hyq_paged_attention_scratch_bytes(kl, 1, 1, 6) == 0


def test_served_lengths_are_refused(hyq, L, ctx):
    """hyq_pages_extend_served_d: hyq_pages_extend_d's refusals, and served
    lengths that are null or one of the other arrays."""
    layout_ = layout(hyq)
    kl, p = ctypes.byref(layout_), 4096
    good = [ctx, kl, p, p, p, p, p, p, p, p, p, p + 64, p, 1 << 40]
    call = L.hyq_pages_extend_served_d
    for i in range(13):
        assert call(*[None if j == i else a for j, a in enumerate(good)]) == hyq.EINVAL, i
        assert b"null" in L.hyq_last_error()
    for i in range(3, 11):
        assert call(*[p + 64 if j == i else a for j, a in enumerate(good)]) == hyq.EINVAL, i
        assert b"own" in L.hyq_last_error()
    for i in (2, 12):
        assert call(*[a + 4 if j == i else a for j, a in enumerate(good)]) == hyq.EINVAL, i
        assert b"aligned" in L.hyq_last_error()
    assert call(*good[:-1], L.hyq_pages_scratch_bytes(kl) - 1) == hyq.EINVAL
    bad = layout(hyq, dtype=8)
    assert call(ctx, ctypes.byref(bad), *good[2:]) == hyq.EDTYPE


def test_sample_refusals(hyq, L, ctx):
    p, big = 4096, 1 << 40
    good = [ctx, p, 2, 100, p, p, p, p, p, p, big, p, p]
    for i in (0, 1, 4, 5, 6, 7, 8, 9, 11):
        assert L.hyq_sample_d(*[None if j == i else a for j, a in enumerate(good)]) == hyq.EINVAL
        assert b"null" in L.hyq_last_error()
    for i, v in ((2, 0), (2, 65537), (3, 0), (3, (1 << 24) + 1)):
        assert L.hyq_sample_d(*[v if j == i else a for j, a in enumerate(good)]) == hyq.EINVAL
        assert b"rows" in L.hyq_last_error()
    assert L.hyq_sample_d(*[a + 4 if j == 9 else a for j, a in enumerate(good)]) == hyq.EINVAL
    assert L.hyq_sample_scratch_bytes(0, 5) == 0 and L.hyq_sample_scratch_bytes(5, 0) == 0


def test_sample_rows_of_a_grid(hyq, L, ctx):
    """A row is a workgroup's second grid index: at most 65535."""
    p = 4096
    assert L.hyq_sample_scratch_bytes(65535, 7) > 0 and L.hyq_sample_scratch_bytes(65536, 7) == 0
    assert L.hyq_sample_d(ctx, p, 65536, 7, p, p, p, p, p, p, 1 << 40, p, p) == hyq.EINVAL


def test_cache_checks_its_layout(hyq):
    with pytest.raises(ValueError, match="layout"):
        hyq.PagedCache(None, 1, 4, 10, 2, 100, page_tokens=24)
