"""CPU tests of the logits' rules: refusals, made before a device is touched."""
import ctypes

import pytest


def test_refusals(hyq):
    L, p = hyq.lib(), 4096
    ctx = ctypes.create_string_buffer(1 << 16)
    whole = dict(history=p, history_len=p, prompt_len=p, history_stride=9, repetition=p, presence=p,
                 frequency=p, bias_start=p, bias_token=p, bias=p, biases=3, mask=p, mask_row=p,
                 masks=2)

    def refused(word, rows=2, vocab=100, logits=p, out=p, where=ctx, none=False, **change):
        rules = hyq.LogitRules(**{**whole, **change})
        code = L.hyq_logits_adjust_d(where, logits, rows, vocab, None if none else
                                     ctypes.byref(rules), out)
        assert code == hyq.EINVAL and word in L.hyq_last_error(), (change, L.hyq_last_error())

    refused(b"null", where=None)
    refused(b"null", logits=None)
    refused(b"null", out=None)
    refused(b"null", none=True)
    for rows, vocab in ((0, 5), (65536, 5), (2, 0), (2, (1 << 24) + 1)):
        refused(b"rows", rows=rows, vocab=vocab)
    refused(b"lengths", history_len=None)
    for stride in (0, (1 << 24) + 1):
        refused(b"history", history_stride=stride)
    for name in ("bias_start", "bias_token", "bias"):
        refused(b"biases without", **{name: None})
    refused(b"biases", biases=(1 << 30) + 1)
    refused(b"masks", mask=None)
    refused(b"masks", mask_row=None)
    refused(b"masks", masks=(1 << 24) + 1)
    for out in (p + 4, p + 4 * 199, p - 4 * 199):
        refused(b"overlaps", out=out)


def test_python_checks(hyq):
    import numpy as np
    x = np.zeros((2, 8), np.float32)
    for bad in (dict(history=[[1]]), dict(bias=[([1], [1.0])]), dict(bias=[([1], []), ([], [])]),
                dict(masks=np.ones((1, 7), bool), mask_row=0), dict(masks=np.ones((1, 8), bool))):
        with pytest.raises(ValueError):
            hyq.adjust_logits(None, x, **bad)
