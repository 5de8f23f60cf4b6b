"""GPU parity: block-scaled E4M3 products where the weights' scale and x's
leave float32's range together but the result does not, and E8M0 scales at
their ends and at NaN, on every route."""
import numpy as np
import pytest
import torch

import knurlogic_amd as K
from tests import fp8_ref as R
from tests.util import to_numpy

pytestmark = pytest.mark.gpu
BF, FH = torch.bfloat16, torch.float16

# rows of x that reach the stream, tiles of 64 rows (K in one part: it is short)
# and of 128; (1030, 8192) reaches tiles of 256
DENSE = [(4, 200), (16, 200), (40, 200), (2100, 2048), (1030, 8192)]
# (pairs, experts): pair by pair, the stream by the sorted list, tiles of 64 and
# 128 rows
GROUPED = [(2, 8), (40, 8), (300, 8), (400, 2)]


def _up(t, dev):
    return torch.from_numpy(np.ascontiguousarray(t)).to(dev)


def _codes(seed, shape, top=256):
    rng = np.random.default_rng(seed)
    q = rng.integers(0, top, shape, dtype=np.uint8)
    q[(q & 127) == 127] = 0x30
    return q


def _rows(seed, shape, dev, dtype=BF, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dtype).to(dev)


def _close(got, x, q, s):
    """As the products' bound, with nothing absolute but the result's and the
    sums' smallest steps (2^-133 in bfloat16, 2^-149 for each of the float32
    additions)."""
    y, mag, cut = R.product(to_numpy(x), q, s)
    n = -(-x.shape[-1] // 128) + 24
    b = torch.finfo(got.dtype).eps / 2 * np.abs(y) * (1 + 1e-6) + n * 2.0 ** -23 * mag + 2.0 ** -10 * cut + \
        2.0 ** -133 + n * 2.0 ** -149
    d = np.abs(to_numpy(got).astype(np.float64) - y)
    assert (d <= b).all(), f"{np.nanmax(d / b):.3g} of the bound; {np.isnan(to_numpy(got)).sum()} NaN"


def _loud_block(N, M, dev, dtype=BF):
    """x whose second block is around 2^60 (one input of it 2^50), and codes
    that are zero there but for the smallest one at that input: with a scale of
    2^76 the two scales' product is past 2^128, the block's term 2^117 or 0."""
    q = _codes(1, (N, 512))
    q[:, 128:256] = 0
    q[::3, 130] = 1
    s = np.full((-(-N // 128), 4), 1e-3, np.float32)
    s[:, 1] = 1.5 * 2.0 ** 76
    x = _rows(2, (M, 512), dev, dtype)
    x[:, 128:256] *= 2.0 ** 60
    x[:, 128], x[:, 130] = 2.0 ** 60, 2.0 ** 50
    return x, q, s


@pytest.mark.parametrize("M,N", DENSE)
def test_matmul_scales_whose_product_overflows(dev, M, N):
    x, q, s = _loud_block(N, M, dev)
    got = K.quantized_matmul(x, _up(q, dev).view(torch.uint32), _up(s, dev), mode="fp8")
    rows = [0, 1, M // 2, M - 1]
    _close(got[rows], x[rows], q, s)
    # a block of zero codes adds nothing, whatever its scale
    q[:, 128:256] = 0
    w = _up(q, dev).view(torch.uint32)
    got = K.quantized_matmul(x, w, _up(s, dev), mode="fp8")
    s[:, 1] = 1
    assert torch.equal(got, K.quantized_matmul(x, w, _up(s, dev), mode="fp8"))


@pytest.mark.parametrize("M,N", DENSE[:4])
@pytest.mark.parametrize("Kd", [512, 4096])
def test_matmul_scales_whose_product_underflows(dev, M, N, Kd):
    """x around 2^-118 and scales around 2^-22: the product of the two scales
    is 2^-148, of which float32 holds one bit, the result some 2^-122."""
    q = _codes(3, (N, Kd), 127) | 0x60                       # 32 to 448
    q[(q & 127) == 127] = 0x7E
    s = (np.random.default_rng(4).random((-(-N // 128), Kd // 128)) + 1).astype(np.float32) * np.float32(2.0 ** -22)
    x = ((1 + torch.rand(M, Kd, generator=torch.Generator().manual_seed(5))) * 2.0 ** -118).to(BF).to(dev)
    got = K.quantized_matmul(x, _up(q, dev).view(torch.uint32), _up(s, dev), mode="fp8")
    rows = [0, 1, M // 2, M - 1]
    _close(got[rows], x[rows], q, s)


@pytest.mark.parametrize("P,E", GROUPED)
def test_gather_scales_whose_product_overflows(dev, P, E):
    x, q, s = _loud_block(200, P, dev)
    q, s = np.stack([q] * E), np.stack([s] * E)
    rhs = torch.arange(P, device=dev) % E
    got = K.gather_qmm(x[:, None], _up(q, dev).view(torch.uint32), _up(s, dev), rhs_indices=rhs, mode="fp8")
    _close(got[:, 0], x, q[0], s[0])


@pytest.mark.parametrize("M", [4, 40, 300])
def test_both_kinds_of_scale_agree(dev, M):
    """The same powers of two as bytes and as float32, from 2^-100 to 2^100."""
    q = _codes(6, (200, 400))
    s = np.array([[27, 127, 227, 120], [60, 90, 130, 160]], np.uint8)
    x = _rows(7, (M, 400), dev)
    for b, by in enumerate((2.0 ** 100, 1.0, 2.0 ** -100, 2.0 ** 7)):
        x[:, 128 * b:128 * (b + 1)] *= by
    w = _up(q, dev).view(torch.uint32)
    a = K.quantized_matmul(x, w, _up(s, dev), mode="fp8")
    b = K.quantized_matmul(x, w, _up(R.scale_values(s).astype(np.float32), dev), mode="fp8")
    assert torch.equal(a, b) and torch.isfinite(a).all()


# (tokens, experts): pair by pair, the stream by the sorted list, tiles
BLOCK = [(1, 16), (24, 8), (300, 8)]


def _experts(seed, E, H, I):
    g, d = _codes(seed, (E, 2 * I, H)), _codes(seed + 1, (E, H, I))
    sg, sd = np.full((E, 2 * I // 128, H // 128), 0.0625, np.float32), np.full((E, H // 128, I // 128), 1e-3, np.float32)
    rng = np.random.default_rng(seed)
    return g, sg * rng.uniform(1, 2, sg.shape).astype(np.float32), d, sd * rng.uniform(1, 2, sd.shape).astype(np.float32)


def _block(dev, x, inds, scores, g, sg, d, sd):
    return K.switch_glu_fp8(x, inds, _up(g, dev).view(torch.uint32), _up(sg, dev), _up(d, dev).view(torch.uint32),
                            _up(sd, dev), scores)


@pytest.mark.parametrize("T,E", BLOCK)
@pytest.mark.parametrize("with_scores", [True, False])
def test_block_scales_whose_product_overflows(dev, T, E, with_scores):
    """Blocks of zero codes under a scale of 2^76, where x (gate and up) and the
    activations (down) are around 2^60."""
    H, I, k = 512, 256, 2
    g, sg, d, sd = _experts(8, E, H, I)
    x = _rows(9, (T, H), dev)
    x[:, 256:384] *= 2.0 ** 60
    g[:, :, 256:384] = 0
    sg[:, 3] *= 2.0 ** 60                                    # up's second block: activations of 2^60
    d[:, :, 128:] = 0
    inds = torch.stack([torch.randperm(E, generator=torch.Generator().manual_seed(t))[:k] for t in range(T)]).to(dev)
    scores = torch.full((T, k), 0.5, dtype=BF, device=dev) if with_scores else None
    want = _block(dev, x, inds, scores, g, sg, d, sd)
    sg[:, :, 2], sd[:, :, 1] = 2.0 ** 76, 2.0 ** 76
    got = _block(dev, x, inds, scores, g, sg, d, sd)
    assert torch.isfinite(want).all() and (want != 0).any() and torch.equal(got, want)


@pytest.mark.parametrize("T,E", BLOCK)
@pytest.mark.parametrize("by", [114, -100])
def test_block_scales_against_large_and_small_rows(dev, T, E, by):
    """x times 2^by against scales times 2^-by is the same block, also where a
    block's sum without the scale is past 2^128."""
    H, I, k = 512, 256, 2
    g, sg, d, sd = _experts(10, E, H, I)
    x = _rows(11, (T, H), dev, std=8.0)
    inds = torch.stack([torch.randperm(E, generator=torch.Generator().manual_seed(t))[:k] for t in range(T)]).to(dev)
    want = _block(dev, x, inds, None, g, sg, d, sd)
    got = _block(dev, (x.float() * 2.0 ** by).to(BF), inds, None, g, np.ldexp(sg, -by).astype(np.float32), d, sd)
    assert torch.isfinite(want).all() and torch.equal(got, want)


# --- E8M0 bytes at their ends, and NaN ----------------------------------------------

def _bytes(seed, shape):
    return np.random.default_rng(seed).integers(112, 120, shape).astype(np.uint8)


@pytest.mark.parametrize("M,N", DENSE)
@pytest.mark.parametrize("lo", [1, 30, 200])
def test_matmul_of_far_bytes(dev, M, N, lo):
    """One block's byte away from the others', as far as x stays in its type."""
    q = _codes(12, (N, 272))
    s = np.full((-(-N // 128), 3), lo, np.uint8)
    s[0, 1], s[-1, 2] = lo + 3, max(lo - 3, 0)
    x = _rows(13, (M, 272), dev, std=2.0 ** (119 - lo))
    got = K.quantized_matmul(x, _up(q, dev).view(torch.uint32), _up(s, dev), mode="fp8")
    rows, cols = [0, 1, M // 2, M - 1], np.r_[0:20, N - 20:N]
    sel = torch.from_numpy(cols).to(dev)
    y, mag, cut = R.product(to_numpy(x[rows]), q, s)
    d = np.abs(to_numpy(got[rows][:, sel]).astype(np.float64) - y[:, cols])
    assert (d <= R.bound(y, mag, cut, 272, torch.finfo(BF).eps)[:, cols]).all() and torch.isfinite(got).all()


@pytest.mark.parametrize("M,N,Kd", [(*d, 512) for d in DENSE] + [(40, 200, 4096)])
def test_matmul_nan_byte(dev, M, N, Kd):
    """A byte of 255 makes its own 128 rows of weights NaN and no others,
    zeros in x or not; one that kmi_quantize_fp8 wrote, too."""
    w = _rows(14, (N, Kd), dev, std=0.02)
    clean = K.quantize(w, mode="fp8")
    w[130, Kd - 1] = float("inf")
    bad = K.quantize(w, mode="fp8")
    assert int(bad[1][1, -1]) == 255
    x = _rows(15, (M, Kd), dev)
    x[M // 2, -128:] = 0
    a, b = (K.quantized_matmul(x, *t, mode="fp8") for t in (clean, bad))
    hit = slice(128, min(256, N))
    assert b[:, hit].isnan().all() and torch.isfinite(a).all()
    assert torch.equal(a[:, :128], b[:, :128]) and torch.equal(a[:, 256:], b[:, 256:])


@pytest.mark.parametrize("P,E", GROUPED)
def test_gather_far_and_nan_bytes(dev, P, E):
    q, s = _codes(16, (E, 200, 272)), _bytes(17, (E, 2, 3))
    for lo in (1, 200):
        s[0] = lo
        s[1, :, 1] = 117
        x = _rows(18, (P, 1, 272), dev)
        rhs = torch.arange(P, device=dev) % E
        x[rhs == 0] *= 2.0 ** (119 - lo)
        got = K.gather_qmm(x, _up(q, dev).view(torch.uint32), _up(s, dev), rhs_indices=rhs, mode="fp8")
        for p in (0, 1, P - 2, P - 1):
            e = p % E
            y, mag, cut = R.product(to_numpy(x[p]), q[e], s[e])
            d = np.abs(to_numpy(got[p]).astype(np.float64) - y)
            assert (d <= R.bound(y, mag, cut, 272, torch.finfo(BF).eps)).all()
        s[1, 1, 1] = 255
        bad = K.gather_qmm(x, _up(q, dev).view(torch.uint32), _up(s, dev), rhs_indices=rhs, mode="fp8")
        of = rhs == 1
        assert bad[of][:, 0, 128:].isnan().all() and torch.equal(bad[of][:, 0, :128], got[of][:, 0, :128])
        assert torch.equal(bad[~of], got[~of])


@pytest.mark.parametrize("T,E", BLOCK)
@pytest.mark.parametrize("with_scores", [True, False])
def test_block_far_and_nan_bytes(dev, T, E, with_scores):
    """Bytes 100 lower against x 2^100 times as large; then 255 in one expert's
    gate, and in one block of its down rows."""
    H, I, k = 512, 256, 2
    g, d = _codes(19, (E, 2 * I, H)), _codes(20, (E, H, I))
    sg, sd = _bytes(21, (E, 2 * I // 128, H // 128)), _bytes(22, (E, H // 128, I // 128)) - 5
    x = _rows(23, (T, H), dev)
    inds = torch.stack([torch.randperm(E, generator=torch.Generator().manual_seed(t))[:k] for t in range(T)]).to(dev)
    scores = torch.full((T, k), 0.5, dtype=BF, device=dev) if with_scores else None
    want = _block(dev, x, inds, scores, g, sg, d, sd)
    assert torch.isfinite(want).all()
    assert torch.equal(_block(dev, (x.float() * 2.0 ** 100).to(BF), inds, scores, g, sg - 100, d, sd), want)
    e = int(inds[0, 0])
    of = (inds == e).any(-1) if with_scores else inds == e
    for at in ("gate", "down"):
        a, b = sg.copy(), sd.copy()
        if at == "gate":
            a[e, 1, 2] = 255
        else:
            b[e, 2, 1] = 255
        got = _block(dev, x, inds, scores, g, a, d, b)
        cols = slice(0, H) if at == "gate" else slice(256, 384)
        assert got[of][:, cols].isnan().all() and torch.equal(got[~of], want[~of])
        if at == "down":
            assert torch.equal(got[of][:, :256], want[of][:, :256]) and torch.equal(got[of][:, 384:], want[of][:, 384:])
