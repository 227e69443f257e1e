"""Penalties, biases and grammar masks on logits on the GPU against 64-bit forms
(tests/logits_ref.py), and with the sampler behind them."""
import ctypes

import numpy as np
import pytest

import logits_ref
import paged_ref as R

pytestmark = pytest.mark.gpu


def close(got, want):
    x, tol = want
    fine = np.isfinite(x)
    assert np.array_equal(np.isnan(x), np.isnan(got))
    assert np.array_equal(got[~fine & ~np.isnan(x)], x[~fine & ~np.isnan(x)])
    err = np.abs(got[fine].astype(np.float64) - x[fine])
    assert np.all(err <= tol[fine]), (err - tol[fine]).max()


def rules_of(r, rows, vocab, most):
    """Histories, biases and masks of every kind for rows of a vocabulary."""
    history = [r.integers(0, vocab, r.integers(0, most + 1)) if i % 4 else
               r.integers(0, min(vocab, 3), most) for i in range(rows)]
    return dict(history=history, prompt_len=[len(h) // 2 if i % 3 else 0
                                             for i, h in enumerate(history)],
                repetition=[[1.05, 1.0, 0.8, 0.0, float("nan")][i % 5] for i in range(rows)],
                presence=[[0.0, 0.5, -1.5][i % 3] for i in range(rows)],
                frequency=[[0.0, 0.25, -0.1, 3.0][i % 4] for i in range(rows)])


@pytest.mark.parametrize("vocab", [1, 2, 31, 33, 255, 2047, 2048, 2049, 5000, 120818])
@pytest.mark.parametrize("rows", [1, 3, 9])
def test_rules(gpu_ctx, hyq, rows, vocab):
    """All rules at once, at the sizes where words and workgroups end."""
    r = np.random.default_rng(vocab + rows)
    x = (5 * r.normal(0, 1, (rows, vocab))).astype(np.float32)
    rules = rules_of(r, rows, vocab, 40 if vocab < 3000 else 700)
    rules["bias"] = [(r.integers(0, vocab, n), 4 * r.normal(0, 1, n))
                     for n in (0 if i % 3 == 1 else 1 + i * 20 for i in range(rows))]
    rules["masks"] = r.random((3, vocab)) < np.array([[0.9], [0.5], [0.02]])
    rules["mask_row"] = [[-1, 0, 1, 2, 3][i % 5] for i in range(rows)]
    for drop in ([], ["bias"], ["masks", "mask_row"], ["history"], ["history", "masks", "mask_row"]):
        some = {k: v for k, v in rules.items() if k not in drop}
        close(hyq.adjust_logits(gpu_ctx, x, **some), logits_ref.adjust(x, **some))


def call(hyq, ctx, x, rows, vocab, rules, out):
    hyq.check(hyq.lib().hyq_logits_adjust_d(ctx.handle, x.ptr, rows, vocab, ctypes.byref(rules),
                                            out.ptr))


def raw_rules(hyq, ctx, table, held, prompt=None, rep=None, pres=None, freq=None):
    keep = [None if a is None else ctx.array(np.ascontiguousarray(a, t)) for a, t in
            ((table, np.int32), (held, np.int32), (prompt, np.int32), (rep, np.float32),
             (pres, np.float32), (freq, np.float32))]
    p = [None if a is None else a.ptr for a in keep]
    rules = hyq.LogitRules(p[0], p[1], p[2], np.shape(table)[1], p[3], p[4], p[5])
    return rules, keep


def test_out_of_place_is_in_place(gpu_ctx, hyq):
    """The same logits wherever they go; the input stays, and a neighbour's memory."""
    r = np.random.default_rng(1)
    rows, vocab = 5, 4099
    x = r.normal(0, 5, (rows, vocab)).astype(np.float32)
    table = r.integers(0, vocab, (rows, 300))
    rules, keep = raw_rules(hyq, gpu_ctx, table, [300, 0, 299, 1, 77], [0, 0, 500, -3, 30],
                            [1.3] * 5, [0.5] * 5, [0.125] * 5)
    d = gpu_ctx.array(x)
    out = gpu_ctx.array(np.full(rows * vocab + 64, -7, np.float32))
    call(hyq, gpu_ctx, d, rows, vocab, rules, out)
    got = out.numpy()
    assert np.array_equal(d.numpy(), x) and np.all(got[rows * vocab:] == -7)
    call(hyq, gpu_ctx, d, rows, vocab, rules, d)
    assert np.array_equal(d.numpy().ravel(), got[:rows * vocab])
    hist = [table[i, :n] for i, n in enumerate([300, 0, 299, 1, 77])]
    close(d.numpy(), logits_ref.adjust(x, hist, [0, 0, 500, -3, 30], 1.3, 0.5, 0.125))


def test_what_lies_outside_is_passed_over(gpu_ctx, hyq):
    """Tokens outside the vocabulary, lengths past the stride and below zero, pairs
    outside the list, masks that there are not."""
    r = np.random.default_rng(2)
    rows, vocab = 4, 1000
    x = r.normal(0, 5, (rows, vocab)).astype(np.float32)
    table = r.integers(-500, 1500, (rows, 64))
    table[0, :3] = 2 ** 31 - 1, -2 ** 31, vocab
    held = np.array([64, 1 << 30, -4, 5])
    rules, keep = raw_rules(hyq, gpu_ctx, table, held, None, [1.5] * rows, None, [0.5] * rows)
    start = gpu_ctx.array(np.array([-9, 3, 2, 90, 1 << 30], np.int32))
    token = gpu_ctx.array(np.array([-1, vocab, 7, 8, 9, 9], np.int32))
    value = gpu_ctx.array(np.array([1, 1, 2, 3, 4, 5], np.float32))
    rules.bias_start, rules.bias_token, rules.bias, rules.biases = (start.ptr, token.ptr, value.ptr,
                                                                    6)
    words = gpu_ctx.array(np.zeros((2, 32), np.uint32))
    which = gpu_ctx.array(np.array([2, -1, 1 << 30, -2 ** 31], np.int32))
    rules.mask, rules.mask_row, rules.masks = words.ptr, which.ptr, 2
    d = gpu_ctx.array(x)
    call(hyq, gpu_ctx, d, rows, vocab, rules, d)
    hist = [table[i, :min(max(n, 0), 64)] for i, n in enumerate(held)]
    pairs = [([7], [2]), ([], []), ([7, 8, 9, 9], [2, 3, 4, 5]), ([], [])]
    close(d.numpy(), logits_ref.adjust(x, hist, None, 1.5, 0.0, 0.5, pairs))


def test_of_several_pairs_the_last_counts(gpu_ctx, hyq):
    x = np.zeros((2, 3000), np.float32)
    tokens = np.tile([5, 2999, 5, 7], 400)
    values = np.arange(1600, dtype=np.float32)
    for _ in range(3):
        got = hyq.adjust_logits(gpu_ctx, x, bias=[(tokens, values), ([5, 5], [2.5, -1.5])])
        assert got[0, 5] == 1598 and got[0, 2999] == 1597 and got[0, 7] == 1599
        assert got[1, 5] == -1.5 and np.count_nonzero(got) == 4


def test_numbers_that_are_not_finite(gpu_ctx, hyq):
    """Infinities and NaN follow the arithmetic; masked places are minus infinity
    whatever they were."""
    x = np.tile(np.array([np.inf, -np.inf, np.nan, 3.0, -3.0, 0.0], np.float32), (2, 2))
    masks = np.ones((1, 12), bool)
    masks[0, 6:] = False
    got = hyq.adjust_logits(gpu_ctx, x, [[0, 1, 2, 3, 4, 5]] * 2, None, 2.0, 1.0, 0.0,
                            masks=masks, mask_row=[0, -1])
    want = np.array([np.inf, -np.inf, np.nan, 0.5, -7, -1])
    assert np.array_equal(got[0, :6], want, equal_nan=True)
    assert np.all(got[0, 6:] == -np.inf)
    assert np.array_equal(got[1, 6:], x[1, 6:], equal_nan=True)


def test_long_history(gpu_ctx, hyq):
    """More tokens than a workgroup reads at once, all of few words."""
    r = np.random.default_rng(4)
    x = r.normal(0, 5, (2, 9000)).astype(np.float32)
    hist = [r.integers(0, 12, 50000), r.integers(0, 9000, 30001)]
    rules = dict(prompt_len=[20000, 0], repetition=1.2, presence=0.1, frequency=1.0 / 1024)
    close(hyq.adjust_logits(gpu_ctx, x, hist, **rules), logits_ref.adjust(x, hist, **rules))


def test_with_the_sampler(gpu_ctx, hyq):
    """Rows whose grammar leaves one token, none, and all; a penalty that turns a
    greedy choice."""
    r = np.random.default_rng(5)
    x = r.normal(0, 3, (4, 500)).astype(np.float32)
    best = x.argmax(1)
    masks = np.zeros((2, 500), bool)
    masks[0, 123] = True
    y = hyq.adjust_logits(gpu_ctx, x, [[], [], [], [best[3]]], None, 50.0, masks=masks,
                          mask_row=[0, 1, -1, -1])
    token, prob = hyq.sample(gpu_ctx, y, 0.5, temperature=[0.7, 0.7, 0.0, 0.0])
    z = x[3].copy()
    z[best[3]] = -np.inf
    assert list(token) == [123, -1, best[2], z.argmax()]
    assert list(prob) == [1, 0, 1, 1]
    for i in range(4):
        want = R.sample(y[i], [0.7, 0.7, 0, 0][i], 0, 1.0, 0.0, 0.5)
        assert (token[i], pytest.approx(prob[i], abs=1e-6)) == want


def test_tokens_beyond_32_bits(gpu_ctx, hyq):
    """Tokens of 64 bits are passed over, not cut to others of the vocabulary."""
    x = np.arange(1, 17, dtype=np.float32).reshape(2, 8)
    far = [np.array([(1 << 32) + 5, 2]), [(1 << 40) + 1, -(1 << 32) + 3]]
    got = hyq.adjust_logits(gpu_ctx, x, history=far, repetition=2.0,
                            bias=[(far[0], [100.0, 1.0]), (far[1], [100.0, 100.0])])
    want = x.copy()
    want[0, 2] = want[0, 2] / 2 + 1
    assert np.array_equal(got, want)
