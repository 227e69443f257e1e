"""CPU tests of the shared prefixes' entry points: refusals, made before a device is
touched."""
import ctypes

import pytest

GOOD = dict(dtype=1, layers=2, kv_heads=4, head_dim=128, page_tokens=64, pages=10, seqs=3, stride=8)


def layout(hyq, **kw):
    return hyq.KvLayout(*{**GOOD, **kw}.values())


@pytest.mark.parametrize("dtype", [0, 1, 1008])
def test_refusals(hyq, dtype):
    L, ctx, p, big = hyq.lib(), ctypes.create_string_buffer(1 << 16), 4096, 1 << 40
    kl = layout(hyq, dtype=dtype)
    k = ctypes.byref(kl)
    plan, need = (L.hyq_paged_shared_plan_bytes(k, 5, 16),
                  L.hyq_paged_shared_attention_scratch_bytes(k, 5, 2, 16))
    assert plan > 0 and need > L.hyq_paged_attention_scratch_bytes(k, 5, 2, 16)
    calls = {
        "plan": (L.hyq_paged_shared_plan_d, [ctx, k, None, p, p, p, 5, 16, p, plan], [3, 4, 5, 8],
                 [8]),
        "plan_least": (L.hyq_paged_shared_plan_least_d,
                       [ctx, k, None, p, p, p, 5, 16, 7, p, plan], [3, 4, 5, 9], [9]),
        "attention": (L.hyq_paged_shared_attention_d,
                      [ctx, k, p, 0, p, p, p, 5, 2, 16, p, plan, p, p, need, p + 64],
                      [2, 4, 5, 6, 10, 12, 13, 15], [2, 10, 12, 13, 15]),
    }

    def refused(name, word, code=hyq.EINVAL, **change):
        call, good, _, _ = calls[name]
        args = list(good)
        for i, v in change.items():
            args[int(i[1:])] = v
        assert call(*args) == code, (name, change)
        assert word in L.hyq_last_error(), (name, change, L.hyq_last_error())

    for name, (_, good, pointers, aligned) in calls.items():
        for i in [0, 1] + pointers:
            refused(name, b"null", **{f"_{i}": None})
        for i in aligned:
            refused(name, b"aligned", **{f"_{i}": good[i] + 4})
        bad = layout(hyq, dtype=8)
        refused(name, b"type", hyq.EDTYPE, _1=ctypes.byref(bad))
        bad2 = layout(hyq, page_tokens=24)
        refused(name, b"layout", _1=ctypes.byref(bad2))
    for heads in (0, 6, 68):
        refused("plan", b"heads", _7=heads)
        refused("plan_least", b"heads", _7=heads)
        refused("attention", b"heads", _9=heads)
    for rows in (0, (1 << 20) + 1):
        refused("plan", b"rows", _6=rows)
        refused("plan_least", b"rows", _6=rows)
        refused("attention", b"rows", _7=rows)
    refused("attention", b"rows", _8=0)
    for layer in (-1, 2):
        refused("attention", b"layer", _3=layer)
    refused("plan", b"needed", _9=plan - 1)
    refused("plan_least", b"needed", _10=plan - 1)
    refused("attention", b"plan", _11=plan - 1)
    refused("attention", b"scratch", _14=need - 1)
    refused("attention", b"must not be q", _15=p)
    for rows, heads in ((0, 16), (5, 6), ((1 << 20) + 1, 16)):
        assert L.hyq_paged_shared_plan_bytes(k, rows, heads) == 0
        assert L.hyq_paged_shared_attention_scratch_bytes(k, rows, 1, heads) == 0
    assert L.hyq_paged_shared_attention_scratch_bytes(k, 5, 0, 16) == 0


def test_python_refuses_a_negative_least(hyq):
    """(As a size it would be the largest there is, and nothing be shared.)"""
    cache = hyq.PagedCache.__new__(hyq.PagedCache)
    with pytest.raises(ValueError, match="least"):
        cache.share_d(0, 4, 16, least=-1)
