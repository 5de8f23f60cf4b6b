"""The block-scaled E4M3 format and its products in float64, for the tests."""
from __future__ import annotations

import numpy as np

BLOCK = 128


def _values():
    v = np.empty(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        v[c] = (m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)) * (-1 if c & 128 else 1)
        if c & 127 == 127:
            v[c] = np.nan
    return v


#: the value of each E4M3 code
VALUES = _values()


def nearest(v):
    """E4M3 codes of v (|v| <= 448): nearest, ties to even, by search among
    the 127 magnitudes."""
    mags = VALUES[:127]
    a = np.abs(np.asarray(v, np.float64))
    hi = np.clip(np.searchsorted(mags, a), 0, 126)
    lo = np.clip(hi - 1, 0, 126)
    dh, dl = mags[hi] - a, a - mags[lo]
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    return (code | np.where(np.signbit(v), 128, 0)).astype(np.uint8)


def exponent(amax):
    """The smallest e >= -126 with amax <= 448 * 2^e."""
    e = -126
    while amax > 448 * 2.0 ** e:
        e += 1
    return e


def block_scales(w, bn, bk):
    """Codes uint8 [N, K] and scale bytes [N/bn, K/bk] of w (float64)."""
    N, K = w.shape
    q = np.zeros((N, K), np.uint8)
    s = np.zeros((-(-N // bn), -(-K // bk)), np.uint8)
    for i in range(s.shape[0]):
        for j in range(s.shape[1]):
            at = (slice(i * bn, (i + 1) * bn), slice(j * bk, (j + 1) * bk))
            top = np.abs(w[at]).max()
            if not np.isfinite(top):
                s[i, j] = 255
                continue
            e = exponent(top)
            s[i, j] = e + 127
            q[at] = nearest(w[at] / 2.0 ** e)
    return q, s


def scale_values(s):
    """float64 scales of float32 scales or E8M0 bytes."""
    s = np.asarray(s)
    if s.dtype == np.uint8:
        return np.where(s == 255, np.nan, 2.0 ** (s.astype(np.float64) - 127))
    return s.astype(np.float64)


def spread(s, bn, bk, N, K):
    return np.repeat(np.repeat(scale_values(s), bn, 0)[:N], bk, 1)[:, :K]


def rows(x):
    """x's rows as quantized inside the products, in float64."""
    q, s = block_scales(np.asarray(x, np.float64), 1, BLOCK)
    return VALUES[q] * spread(s, 1, BLOCK, *x.shape)


def weights(q, s):
    return VALUES[q] * spread(s, BLOCK, BLOCK, *q.shape)


def product(x, q, s):
    """(y, sum of the products' magnitudes, sum over the runs of 8 inputs of
    the largest product's) of x against one weight."""
    a, b = rows(x), weights(q, s)
    m, n = np.abs(a), np.abs(b)
    cut = np.zeros((a.shape[0], b.shape[0]))
    with np.errstate(invalid="ignore"):
        for k in range(0, a.shape[1], 8):
            cut += (m[:, None, k:k + 8] * n[None, :, k:k + 8]).max(-1)
        return a @ b.T, m @ n.T, cut


def bound(y, mag, cut, K, eps):
    """How far a product may be from y: half a step of the result's type; for
    the float32 sums 2^-23 of the products' magnitudes for each addition one
    after the other (blocks of a wave, the product by the scale, 8 waves, the
    runs of a block); and what the matrix instruction drops: it lines up the 8
    products of a run with the largest's exponent E and keeps the places down
    to 2^(E - 13) (a product of 2^-14 of the largest is lost, one of 2^-13 is
    not), so each of the 8 loses less than 2^-13 of the largest: 2^-10 of it in
    all."""
    n = -(-K // BLOCK) + 24
    return eps / 2 * np.abs(y) * (1 + 1e-6) + n * 2.0 ** -23 * mag + 2.0 ** -10 * cut + 2.0 ** -25
