"""The block-scaled E4M3 format and its products in float64, for the tests."""
from __future__ import annotations

import numpy as np
import torch

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
    """The smallest e >= -126 with amax <= 448 * 2^e (448 = 0.875 * 2^9)."""
    f, x = np.frexp(amax)
    return np.where(np.asarray(amax) > 0, np.maximum(x - np.where(f <= 0.875, 9, 8), -126), -126)


def block_scales(w, bn, bk):
    """Codes uint8 [N, K] and scale bytes [N/bn, K/bk] of w (float64)."""
    N, K = w.shape
    n, k = -(-N // bn), -(-K // bk)
    p = np.zeros((n * bn, k * bk))
    p[:N, :K] = w
    top = np.abs(p).reshape(n, bn, k, bk).max((1, 3))
    bad = ~np.isfinite(top)
    e = exponent(np.where(bad, 1.0, top))
    wide = lambda v: np.repeat(np.repeat(v, bn, 0)[:N], bk, 1)[:, :K]
    with np.errstate(invalid="ignore"):
        q = np.where(wide(bad), 0, nearest(np.where(wide(bad), 0, w) / 2.0 ** wide(e)))
    return q.astype(np.uint8), np.where(bad, 255, e + 127).astype(np.uint8)


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
    m, n = torch.from_numpy(np.abs(a)), torch.from_numpy(np.abs(b))
    cut = torch.zeros(len(a), len(b), dtype=torch.float64)
    for k in range(0, a.shape[1], 8):
        cut += (m[:, None, k:k + 8] * n[None, :, k:k + 8]).amax(-1)
    with np.errstate(invalid="ignore"):
        return a @ b.T, (m @ n.T).numpy(), cut.numpy()


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
