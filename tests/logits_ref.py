"""The rules on logits in 64 bits, row by row."""
import numpy as np


def adjust(logits, history=None, prompt_len=None, repetition=1.0, presence=0.0, frequency=0.0,
           bias=None, masks=None, mask_row=None):
    """(logits, bound of the f32 kernel's error): the penalty's product or quotient
    rounds once, the two others' sum twice, its difference once, the bias's sum once,
    each by half a step of what it has."""
    x = logits.astype(np.float64)
    rows, vocab = x.shape
    u, tol = 2.0 ** -24, np.zeros_like(x)
    each = lambda v: np.broadcast_to(np.asarray(v, np.float32), (rows,)).astype(np.float64)
    rep, pres, freq = each(repetition), each(presence), each(frequency)
    prompt = np.broadcast_to(np.asarray(0 if prompt_len is None else prompt_len), (rows,))
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        for r in range(rows):
            if history is not None:
                h = np.asarray(history[r], np.int64)
                made = h[max(int(prompt[r]), 0):]
                n = np.bincount(made[(made >= 0) & (made < vocab)], minlength=vocab)
                seen = np.zeros(vocab, bool)
                seen[h[(h >= 0) & (h < vocab)]] = True
                f = rep[r] if rep[r] > 0 else 1.0
                y = np.where(x[r] > 0, x[r] / f, x[r] * f)
                x[r] = np.where(seen, y, x[r])
                tol[r] += np.where(seen, np.abs(y) * u, 0)
                off = pres[r] + freq[r] * n
                x[r] = np.where(n > 0, x[r] - off, x[r])
                tol[r] += np.where(n > 0, (2 * (abs(pres[r]) + abs(freq[r]) * n) + np.abs(x[r])) * u,
                                   0)
            if bias is not None:
                last = {int(t): float(np.float32(v)) for t, v in zip(*bias[r]) if 0 <= t < vocab}
                for t, v in last.items():
                    x[r, t] += v
                    tol[r, t] += abs(x[r, t]) * u
            if masks is not None and 0 <= np.broadcast_to(mask_row, (rows,))[r] < len(masks):
                x[r, ~masks[np.broadcast_to(mask_row, (rows,))[r]]] = -np.inf
    return x, tol * 1.001 + 2.0 ** -149
