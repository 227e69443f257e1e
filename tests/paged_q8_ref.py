"""Batches over an 8-bit pool for the paged cache's tests, and the plain forms of
its quantisation (numpy, 64 bits)."""
import numpy as np

import paged_ref as R

D, U = R.D, R.U


def quantise(x):
    """Codes and scales of rows of 128 numbers: scale = max |x| / 127 in f32,
    code = rint(x / scale); a row that is not finite has a NaN for its scale."""
    x = np.asarray(x, np.float64)
    with np.errstate(over="ignore", invalid="ignore"):
        scale = (np.abs(x).max(-1) / 127.0).astype(np.float32)
        fine = np.isfinite(x).all(-1) & np.isfinite(scale)
        safe = np.where(fine & (scale > 0), scale, 1).astype(np.float64)
        code = np.clip(np.rint(np.where(fine[..., None], x, 0) / safe[..., None]), -127, 127)
        code = np.where((scale > 0)[..., None], code, 0)
    return code.astype(np.int64), np.where(fine, scale, np.float32(np.nan))


def split(pool, kvh, pt):
    """Codes (signed) [pages][2][kvh][pt][128] and scales of pages of bytes, as copies."""
    n = 2 * kvh * pt * D
    codes = pool[:, :n].reshape(-1, 2, kvh, pt, D).astype(np.int64)
    codes[:, 0] = np.where(codes[:, 0] > 127, codes[:, 0] - 256, codes[:, 0])
    codes[:, 1] -= 128
    scales = np.ascontiguousarray(pool[:, n:]).view(np.float32).reshape(-1, 2, kvh, pt)
    return codes, scales


def join(codes, scales):
    """Pages of bytes."""
    codes = codes.copy()
    codes[:, 1] += 128
    pages = len(codes)
    return np.concatenate([(codes & 255).astype(np.uint8).reshape(pages, -1),
                           np.ascontiguousarray(scales, np.float32).reshape(pages, -1).view(
                               np.uint8)], 1)


class BatchQ8(R.Batch):
    """A batch whose pool is of bytes: quantised normals in the places that
    positions use, any bytes and NaN scales in the others."""

    def __init__(self, lens, news, heads, kv_heads, page_tokens, seed, spread=0.0, **kw):
        super().__init__(lens, news, heads, kv_heads, page_tokens, False, seed, **kw)
        r = np.random.default_rng(seed + 1000)
        x = self.pool.astype(np.float64)
        used = ~np.isnan(x[..., 0])
        x *= 2.0 ** (spread * r.normal(0, 1, x.shape[:-1]))[..., None]
        codes, scales = quantise(np.where(used[..., None], x, 0))
        junk = r.integers(-127, 128, codes.shape)
        self.codes = np.where(used[..., None], codes, junk)
        self.scales = np.where(used, scales, np.float32(np.nan)).astype(np.float32)
        self.bytes = join(self.codes, self.scales)

    def kv(self, s, h):
        n = int(self.lens[s])
        ids = self.table[s][np.arange(n) // self.pt]
        ok = (ids >= 0) & (ids < self.pages)
        at = (np.where(ok, ids, 0), slice(None), h, np.arange(n) % self.pt)
        rows = self.codes[at].astype(np.float64) * self.scales[at].astype(np.float64)[..., None]
        return rows[:, 0], rows[:, 1], ok

    def attention(self):
        """As Batch.attention; the bound of an output's error is tolerance()'s."""
        out = np.full((self.rows, self.heads, D), np.nan)
        tol = np.zeros((self.rows, self.heads))
        rep = self.heads // self.kvh
        for s in range(self.seqs):
            n, m, b = int(self.lens[s]), int(self.news[s]), int(self.start[s])
            for h in range(self.kvh):
                k, v, ok = self.kv(s, h)
                for i in range(m):
                    see = ok & (np.arange(n) <= n - m + i)
                    for head in range(h * rep, (h + 1) * rep):
                        if not see.any():
                            out[b + i, head] = 0
                            continue
                        q = self.q[b + i, head].astype(np.float64)
                        sc = k[see] @ q / np.sqrt(D)
                        w = np.exp(sc - sc.max())
                        out[b + i, head] = (w[:, None] * v[see]).sum(0) / w.sum()
                        mag = (np.abs(k[see]) @ np.abs(q)).max() / np.sqrt(D)
                        ksum = np.abs(k[see]).sum(-1).max() * np.abs(q).max() / np.sqrt(D)
                        tol[b + i, head] = tolerance(mag, ksum, np.abs(sc).max(),
                                                     np.abs(v[see]).max(), int(see.sum()))
        return out, tol


def tolerance(mag, ksum, score, vmax, n):
    """Bound of an output's error. Codes are exact. A query's numbers are off by at
    most 2^-22 of the row's largest (its two f16 parts, or 22-bit whole numbers), so
    a score by 2^-22 ksum, ksum the sum of |k| times that largest, and twice that
    where both parts round; its sum in f32 by 128 U of the products' magnitude `mag`;
    its scales, the difference with the maximum and the exponential's argument by U
    of at most 3 |score| log2(e) each, the exponential by 2 U. A weight off by a
    factor 1 + d moves numerator and denominator: 2 d vmax. A weight times its scale
    is rounded twice more and split to 2^-22 of itself or, where it is small, to
    2^-25 of the unit in which the largest is 2^7 at least: with scales below the
    power of two that is at most twice the largest, 2^-31 vmax for each position.
    Sums over n positions in f32: (n + 8) U."""
    d = 2.0 ** -21 * ksum + 128 * U * mag + 3 * U * 3 * score + 2 * U
    return vmax * (2 * d + (n + 12) * U + 2.0 ** -22 + n * 2.0 ** -31)
