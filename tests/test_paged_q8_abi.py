"""CPU tests of the 8-bit pool's and the read-back's entry points: sizes and
refusals, made before a device is touched."""
import ctypes

import pytest

GOOD = dict(dtype=1008, layers=2, kv_heads=4, head_dim=128, page_tokens=64, pages=10, seqs=3,
            stride=8)


@pytest.fixture(scope="module")
def L(hyq):
    return hyq.lib()


@pytest.fixture(scope="module")
def ctx():
    return ctypes.create_string_buffer(1 << 16)


def layout(hyq, **kw):
    return hyq.KvLayout(*{**GOOD, **kw}.values())


def test_pool_bytes(hyq, L):
    assert hyq.KV_Q8 == 1008
    kl = layout(hyq)
    assert L.hyq_kv_pool_bytes(ctypes.byref(kl)) == 2 * 10 * 2 * 4 * 64 * (128 + 4)
    assert L.hyq_paged_attention_scratch_bytes(ctypes.byref(kl), 5, 2, 16) > 0


@pytest.mark.parametrize("bad", [dict(dtype=2), dict(dtype=8), dict(head_dim=64),
                                 dict(page_tokens=8), dict(kv_heads=257), dict(seqs=0)], ids=str)
def test_read_refuses_layouts(hyq, L, ctx, bad):
    kl, p = layout(hyq, **bad), 4096
    want = hyq.EDTYPE if "dtype" in bad else hyq.EINVAL
    assert L.hyq_paged_read_d(ctx, ctypes.byref(kl), p, 0, p, p, p, 1, p, p + 64) == want


@pytest.mark.parametrize("dtype", [0, 1, 1008])
def test_read_refuses_arguments(hyq, L, ctx, dtype):
    kl, p = layout(hyq, dtype=dtype), 4096
    good = [ctx, ctypes.byref(kl), p, 0, p, p, p, 5, p, p + 64]

    def refused(i, v, word):
        args = [v if j == i else a for j, a in enumerate(good)]
        assert L.hyq_paged_read_d(*args) == hyq.EINVAL, (i, v)
        assert word in L.hyq_last_error()

    for i in (0, 1, 2, 4, 5, 6, 8, 9):
        refused(i, None, b"null")
    for i in (2, 8, 9):
        refused(i, good[i] + 4, b"aligned")
    refused(3, -1, b"layer")
    refused(3, 2, b"layer")
    refused(7, (1 << 20) + 1, b"rows")
    refused(9, p, b"one place")


def test_cache_of_bytes_checks_its_layout(hyq):
    with pytest.raises(ValueError, match="layout"):
        hyq.PagedCache(None, 1, 4, 10, 2, 100, page_tokens=24, dtype=hyq.KV_Q8)
