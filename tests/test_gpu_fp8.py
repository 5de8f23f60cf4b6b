"""GPU parity: block-scaled E4M3 (mode "fp8") -- quantize and dequantize bit
for bit, the dense and expert-gathered products against float64 within a
bound counted from their roundings, SwitchGLU and the modules over them."""
import numpy as np
import pytest
import torch

import knurlogic_amd as K
from knurlogic_amd import checkpoint as C
from knurlogic_amd import nn
from tests import fp8_ref as R
from tests.util import MIN_COS, assert_close, cosine, to_numpy

pytestmark = pytest.mark.gpu
BF, FH, FS = torch.bfloat16, torch.float16, torch.float32


def _x(seed, shape, dtype, dev, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dtype).to(dev)


def _w(seed, shape, kind, dev):
    """Random codes (no NaN) and scales: (uint8 [..., N, K], scales) on the
    host, (packed words, scales) on the GPU."""
    rng = np.random.default_rng(seed)
    q = rng.integers(0, 256, shape, dtype=np.uint8)
    q[(q & 127) == 127] = 0x30
    sh = (*shape[:-2], -(-shape[-2] // 128), -(-shape[-1] // 128))
    s = rng.integers(110, 120, sh).astype(np.uint8) if kind == "e8m0" else \
        (rng.random(sh) * 3e-4 + 1e-5).astype(np.float32)
    return (q, s), (torch.from_numpy(q.copy()).to(dev).view(torch.uint32), torch.from_numpy(s).to(dev))


def _check(got, x, q, s, what=""):
    y, mag, cut = R.product(to_numpy(x).reshape(-1, x.shape[-1]), q, s)
    eps = torch.finfo(got.dtype).eps
    d = np.abs(to_numpy(got).reshape(y.shape).astype(np.float64) - y)
    b = R.bound(y, mag, cut, x.shape[-1], eps)
    assert (d <= b).all(), f"{what}: {np.max(d / b):.3g} of the bound at {np.unravel_index(np.argmax(d / b), d.shape)}"


# --- quantize / dequantize -----------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF, FH, FS])
@pytest.mark.parametrize("shape", [(1, 16), (3, 128), (128, 128), (129, 144), (300, 1040), (2, 3, 140, 272)])
def test_quantize_bit_exact(dev, shape, dtype):
    w = _x(sum(shape), shape, dtype, dev, 0.02)
    wq, s = K.quantize(w, mode="fp8")
    assert wq.dtype == torch.uint32 and s.dtype == torch.uint8
    flat = to_numpy(w).reshape(-1, *shape[-2:]).astype(np.float64)
    got_q = wq.view(torch.uint8).cpu().numpy().reshape(flat.shape)
    got_s = s.cpu().numpy().reshape(flat.shape[0], -1, s.shape[-1])
    for i, f in enumerate(flat):
        q, sc = R.block_scales(f, 128, 128)
        assert np.array_equal(got_s[i], sc)
        assert np.array_equal(got_q[i], q)
    d = K.dequantize(wq, s, mode="fp8", dtype=FS)
    want = np.stack([R.weights(*R.block_scales(f, 128, 128)) for f in flat]).reshape(shape)
    assert np.array_equal(to_numpy(d), want.astype(np.float32))


@pytest.mark.parametrize("dtype", [BF, FH, FS])
def test_quantize_at_the_borders(dev, dtype):
    """Blocks whose largest value is at, just under and just over a power's
    448, ties between codes, zeros, the type's smallest and largest values,
    infinities and NaN (which make their own block NaN only)."""
    fi = torch.finfo(dtype)
    top = torch.tensor([448.0, 448.0, 1.75, 1.75, 0.0, fi.max, fi.tiny, fi.smallest_normal, 1.0, 2.0 ** -10, 3.5, 7.0])
    w = torch.zeros(128, 128 * len(top))
    for i, t in enumerate(top.tolist()):
        b = w[:, 128 * i:128 * (i + 1)]
        b[0, 0] = -t
        # every midpoint between neighbouring codes under t
        mids = torch.from_numpy((R.VALUES[:126] + R.VALUES[1:127]) / 2).float() * (t / 448 if 0 < t < fi.max else 0)
        b[1, :126], b[2, :126] = mids, -mids
    w = w.to(dtype)
    w[5, 128 + 7] = torch.nextafter(torch.tensor(448.0), torch.tensor(500.0)) if dtype == FS else 450.0
    w[7, 2 * 128 + 1] = fi.tiny / 2
    w[9, 8 * 128] = float("inf")
    w[9, 9 * 128] = float("nan")
    wq, s = K.quantize(w.to(dev), mode="fp8")
    q, sc = R.block_scales(to_numpy(w).astype(np.float64), 128, 128)
    assert np.array_equal(s.cpu().numpy(), sc) and list(sc[0, 8:10]) == [255, 255]
    assert np.array_equal(wq.view(torch.uint8).cpu().numpy(), q)
    d = to_numpy(K.dequantize(wq, s, mode="fp8", dtype=FS))
    # the type's largest value in bf16 and float32, just under 2^128, is at e = 120
    # nearest to the code 256: 2^128, past float32
    rest = np.delete(d, np.r_[5 * 128:6 * 128, 8 * 128:10 * 128], 1)
    assert np.isnan(d[:, 8 * 128:10 * 128]).all() and np.isfinite(rest).all()
    assert np.isfinite(d[0, 5 * 128]) == (dtype == FH)


@pytest.mark.parametrize("out", [BF, FH, FS])
@pytest.mark.parametrize("kind", ["f32", "e8m0"])
def test_dequantize_bit_exact(dev, kind, out):
    (q, s), (wq, sc) = _w(5, (2, 130, 144), kind, dev)
    got = K.dequantize(wq, sc, mode="fp8", dtype=out)
    prod = np.stack([R.VALUES[q[i]].astype(np.float32) * R.spread(s[i], 128, 128, 130, 144).astype(np.float32)
                     for i in range(2)])
    assert torch.equal(got.cpu(), torch.from_numpy(prod).to(out))


# --- the dense product ---------------------------------------------------------------

@pytest.mark.parametrize("M", [1, 3, 16, 17, 33, 64, 65, 130, 300])
@pytest.mark.parametrize("N,Kd", [(128, 128), (100, 272), (576, 1024), (1, 16), (257, 4112)])
def test_matmul_sizes(dev, M, N, Kd):
    kind = "e8m0" if (M + N) % 2 else "f32"
    (q, s), (wq, sc) = _w(M * 7 + N, (N, Kd), kind, dev)
    x = _x(M + N + Kd, (M, Kd), BF, dev)
    got = K.quantized_matmul(x, wq, sc, mode="fp8")
    assert got.shape == (M, N) and got.dtype == BF
    _check(got, x, q, s)


@pytest.mark.parametrize("M", [1, 20, 70, 150])
@pytest.mark.parametrize("Kd", [256, 400, 1008, 2048, 4096, 8192, 8208, 16384, 16400])
def test_matmul_depths(dev, M, Kd):
    """Every way of splitting K, full and with a partial last block."""
    (q, s), (wq, sc) = _w(M + Kd, (80, Kd), "f32" if M % 4 else "e8m0", dev)
    x = _x(M, (M, Kd), BF, dev)
    _check(K.quantized_matmul(x, wq, sc, mode="fp8"), x, q, s)


@pytest.mark.parametrize("dtype", [BF, FH])
@pytest.mark.parametrize("kind", ["f32", "e8m0"])
@pytest.mark.parametrize("M", [1, 20, 50, 200, 520])
def test_matmul_types(dev, M, kind, dtype):
    (q, s), (wq, sc) = _w(M, (384, 1424), kind, dev)
    x = _x(M + 1, (M, 1424), dtype, dev)
    got = K.quantized_matmul(x, wq, sc, mode="fp8")
    assert got.dtype == dtype
    _check(got, x, q, s)


def _check_some(got, x, q, s, rows, cols, what=""):
    """The given rows, at ranges of columns that begin on a scale block."""
    got, x, rows = to_numpy(got), to_numpy(x), list(rows)
    for c0, c1 in cols:
        _check(torch.from_numpy(got[rows, c0:c1]).to(BF), torch.from_numpy(x[rows]), q[c0:c1], s[c0 // 128:], what)


@pytest.mark.parametrize("M,N,Kd", [(384, 14336, 144), (384, 14300, 8208), (900, 14332, 256), (1030, 14340, 400),
                                    (769, 14336, 8320)])
def test_matmul_of_many_tiles(dev, M, N, Kd):
    """The large tiles, their last rows and columns in part, scales in more
    than one chunk."""
    kind = "e8m0" if M % 2 else "f32"
    (q, s), (wq, sc) = _w(M, (N, Kd), kind, dev)
    x = _x(N, (M, Kd), BF, dev)
    got = K.quantized_matmul(x, wq, sc, mode="fp8")
    at = N // 128 * 128 - 128
    _check_some(got, x, q, s, [0, 63, 64, 255, 256, M - 1], [(0, 140), (at, N)])
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("dtype", [BF, FH])
@pytest.mark.parametrize("M,N,Kd", [(17, 66, 4096), (64, 127, 8208), (100, 200, 4112), (33, 4, 16384), (130, 130, 5120)])
def test_matmul_in_parts_of_k(dev, dtype, M, N, Kd):
    """Few tiles of a long K: sums of parts, the last of them shorter."""
    kind = "e8m0" if M % 2 else "f32"
    (q, s), (wq, sc) = _w(N, (N, Kd), kind, dev)
    x = _x(M + 2, (M, Kd), dtype, dev, 0.25)
    got = K.quantized_matmul(x, wq, sc, mode="fp8")
    _check(got, x, q, s)
    assert torch.equal(got, K.quantized_matmul(x, wq, sc, mode="fp8"))


@pytest.mark.parametrize("M", [2, 40, 256])
def test_matmul_row_scales_follow_each_row_and_block(dev, M):
    """Rows and blocks of very different size, zero rows, zero blocks."""
    (q, s), (wq, sc) = _w(3, (256, 640), "f32", dev)
    x = _x(9, (M, 640), BF, dev)
    x *= torch.exp2(torch.arange(M, device=dev).float() % 40 - 20)[:, None]
    x[:, 128:256] *= 1e-4
    x[:, 512:] *= 1e4
    assert x.dtype == BF
    x[1] = 0
    x[M // 2, 256:384] = 0
    got = K.quantized_matmul(x, wq, sc, mode="fp8")
    _check(got, x, q, s)
    assert (got[1] == 0).all()


@pytest.mark.parametrize("M", [5, 100, 300])
@pytest.mark.parametrize("Kd", [256, 272])
def test_matmul_nonfinite_rows_stay_alone(dev, M, Kd):
    """An infinity or a NaN makes its own row NaN and no other; a NaN code or
    scale makes its own weight rows NaN."""
    (q, s), (wq, sc) = _w(4, (200, Kd), "f32", dev)
    x = _x(2, (M, Kd), BF, dev)
    clean = K.quantized_matmul(x, wq, sc, mode="fp8")
    bad = x.clone()
    bad[1, 3], bad[4, Kd - 1] = float("inf"), float("nan")
    got = K.quantized_matmul(bad, wq, sc, mode="fp8")
    assert got[1].isnan().all() and got[4].isnan().all()
    keep = [m for m in range(M) if m not in (1, 4)]
    assert torch.equal(got[keep], clean[keep])
    # the last row's last byte; and the last row of all rows, whose
    # neighbours in memory are what partial blocks would read
    wn = wq.view(torch.uint8).clone()
    wn[7, Kd - 1] = 0x7F
    got = K.quantized_matmul(x, wn.view(torch.uint32), sc, mode="fp8")
    assert got[:, 7].isnan().all()
    cols = [n for n in range(200) if n != 7]
    assert torch.equal(got[:, cols], clean[:, cols])
    sn = sc.clone()
    sn[1, 0] = float("nan")
    got = K.quantized_matmul(x, wq, sn, mode="fp8")
    assert got[:, 128:].isnan().all() and torch.equal(got[:, :128], clean[:, :128])


def test_matmul_layouts(dev):
    """Leading dimensions, strided and unaligned x, a float8 weight, strided
    scales and weights, one-dimensional x, no rows."""
    (q, s), (wq, sc) = _w(6, (140, 256), "f32", dev)
    x = _x(3, (2, 3, 256), BF, dev)
    want = K.quantized_matmul(x.reshape(6, 256), wq, sc, mode="fp8")
    _check(want, x, q, s)
    assert torch.equal(K.quantized_matmul(x, wq, sc, mode="fp8"), want.view(2, 3, 140))
    assert torch.equal(K.quantized_matmul(x[1, 2], wq, sc, mode="fp8"), want[5])
    t = x.reshape(6, 256).t().contiguous().t()
    assert torch.equal(K.quantized_matmul(t, wq, sc, mode="fp8"), want)
    u = torch.empty(6 * 256 + 3, dtype=BF, device=dev)[3:].view(6, 256).copy_(x.reshape(6, 256))
    assert torch.equal(K.quantized_matmul(u, wq, sc, mode="fp8"), want)
    f8 = wq.view(torch.float8_e4m3fn)
    assert torch.equal(K.quantized_matmul(x.reshape(6, 256), f8, sc, mode="fp8"), want)
    wide = torch.zeros(140, 80, dtype=torch.int32, device=dev)
    wide[:, 8:72] = wq.view(torch.int32)
    assert torch.equal(K.quantized_matmul(x.reshape(6, 256), wide[:, 8:72], sc.t().contiguous().t(), mode="fp8"), want)
    assert K.quantized_matmul(x[:, :0], wq, sc, mode="fp8").shape == (2, 0, 140)


def test_matmul_large_scales_and_small(dev):
    """Scales at the ends of E8M0, and float32 ones of either sign."""
    (q, s), _ = _w(8, (256, 256), "e8m0", dev)
    for lo in (1, 30, 200):
        s = np.full((2, 2), lo, np.uint8)
        s[0, 1] += 3
        x = _x(1, (4, 256), BF, dev, 2.0 ** (127 - lo - 8))
        got = K.quantized_matmul(x, torch.from_numpy(q.copy()).to(dev).view(torch.uint32), torch.from_numpy(s).to(dev),
                                 mode="fp8")
        _check(got, x, q, s, lo)
    sf = np.array([[-0.5, 2.0], [0.0, 1e-3]], np.float32)
    x = _x(2, (4, 256), BF, dev)
    got = K.quantized_matmul(x, torch.from_numpy(q.copy()).to(dev).view(torch.uint32), torch.from_numpy(sf).to(dev),
                             mode="fp8")
    _check(got, x, q, sf)


# --- rows against their own expert -----------------------------------------------------

def _gather_check(got, x, lhs, rhs, q, s):
    """got [P, M, N] against float64; lhs and rhs lists (an index out of range:
    a zero row)."""
    for p, (l, r) in enumerate(zip(lhs, rhs)):
        if 0 <= r < q.shape[0] and 0 <= l < x.shape[0]:
            _check(got[p], x[l], q[r], s[r], f"pair {p}")
        else:
            assert (got[p] == 0).all()


@pytest.mark.parametrize("P,E,M", [(1, 1, 1), (7, 4, 1), (40, 3, 1), (90, 2, 1), (33, 64, 1), (6, 5, 9), (400, 2, 1)])
@pytest.mark.parametrize("N,Kd", [(100, 272), (256, 512)])
def test_gather_sizes(dev, P, E, M, N, Kd):
    kind = "e8m0" if P % 2 else "f32"
    (q, s), (wq, sc) = _w(P + E, (E, N, Kd), kind, dev)
    rng = np.random.default_rng(P)
    rhs = rng.integers(0, E, P)
    rhs[rng.random(P) < 0.05] = E                            # out of range
    x = _x(P, (P, M, Kd), BF, dev)
    got = K.gather_qmm(x, wq, sc, rhs_indices=torch.from_numpy(rhs).to(dev), mode="fp8")
    assert got.shape == (P, M, N)
    _gather_check(got, x, range(P), rhs, q, s)


@pytest.mark.parametrize("P,E,N,Kd", [(300, 64, 2048, 144), (700, 64, 2040, 1040), (4200, 64, 1280, 272), (300, 3, 700, 400),
                                      (9, 9, 300, 8208), (40, 16, 260, 2304), (70, 2, 260, 16400)])
def test_gather_in_groups(dev, P, E, N, Kd):
    """Several column blocks to a workgroup, units of every size, K past the
    stream's; experts without rows, rows of one expert only."""
    kind = "e8m0" if P % 3 else "f32"
    (q, s), (wq, sc) = _w(P + E, (E, N, Kd), kind, dev)
    x = _x(P, (P, 1, Kd), BF, dev)
    rng = np.random.default_rng(P)
    for rhs in (rng.integers(0, E, P), np.full(P, E - 1), rng.integers(0, E, P) // 2 * 2):
        got = K.gather_qmm(x, wq, sc, rhs_indices=torch.from_numpy(rhs).to(dev), mode="fp8")
        at = N // 128 * 128 - 128
        for p in (0, 1, P // 2, P - 1):
            if rhs[p] < E:
                _check_some(got[p], x[p], q[rhs[p]], s[rhs[p]], [0], [(0, N if N < 300 else 300), (at, N)], f"pair {p}")
            else:
                assert (got[p] == 0).all()
        assert torch.isfinite(got).all()


@pytest.mark.parametrize("dtype", [BF, FH])
@pytest.mark.parametrize("P", [5, 150])
def test_gather_types_and_lhs(dev, dtype, P):
    """x rows shared by pairs, in any order, some out of range."""
    (q, s), (wq, sc) = _w(P, (3, 140, 400), "f32", dev)
    x = _x(P, (4, 2, 400), dtype, dev)
    rng = np.random.default_rng(P)
    lhs, rhs = rng.integers(0, 4, P), rng.integers(-1, 3, P)
    lhs[2] = 9
    got = K.gather_qmm(x, wq, sc, lhs_indices=torch.from_numpy(lhs).to(dev), rhs_indices=torch.from_numpy(rhs).to(dev),
                       mode="fp8")
    assert got.shape == (P, 2, 140) and got.dtype == dtype
    _gather_check(got, x, lhs, rhs, q, s)


def test_gather_of_nothing(dev):
    _, (wq, sc) = _w(1, (3, 128, 128), "f32", dev)
    x = _x(1, (4, 1, 128), BF, dev)
    e = torch.empty(0, dtype=torch.int32, device=dev)
    assert K.gather_qmm(x, wq, sc, lhs_indices=e, rhs_indices=e, mode="fp8").shape == (0, 1, 128)


# --- the expert block --------------------------------------------------------------------

def _glu_ref(x, inds, wg, wd, scores=None):
    """float64 SwitchGLU with the bf16 roundings of its steps, and how far the
    kernels may be from it: (y [T, k, H] or [T, H], bound)."""
    bf = lambda v: torch.from_numpy(np.asarray(v, np.float32)).to(BF).double().numpy()
    (qg, sg), (qd, sd) = wg, wd
    I, H = qd.shape[2], qd.shape[1]
    out, far = np.zeros((*inds.shape, H)), np.zeros((*inds.shape, H))
    for e in np.unique(inds[(inds >= 0) & (inds < qg.shape[0])]):
        t, j = np.nonzero(inds == e)
        y, mag, cut = R.product(x[t], qg[e], sg[e])
        err = R.bound(0 * y, mag, cut, x.shape[1], 0)
        act = lambda g, u: bf(bf(g / (1 + np.exp(-g))) * u)
        half = lambda v: (v[:, :I], v[:, I:])
        h = act(*half(bf(y)))
        # gate or up may round to the other neighbour, and the activation's
        # code with it: the codes of the ends of their ranges
        off = 0
        for sg_ in (-1, 1):
            for su in (-1, 1):
                g, u = half(bf(y + err))[0] if sg_ > 0 else half(bf(y - err))[0], \
                    half(bf(y + err))[1] if su > 0 else half(bf(y - err))[1]
                off = np.maximum(off, np.abs(R.rows(act(g, u)) - R.rows(h)))
        d, mag, cut = R.product(h, qd[e], sd[e])
        out[t, j] = bf(d)
        # (what the kernel has and its neighbour may both round)
        far[t, j] = R.bound(d, mag, cut, I, 2.0 ** -7) + 2.0 ** -8 * np.abs(d) + \
            (1 + 2.0 ** -8) * off @ np.abs(R.weights(qd[e], sd[e])).T
    if scores is None:
        return out, far
    p = bf(out * scores[..., None])
    far = ((1 + 2.0 ** -7) * far * scores[..., None] + 2.0 ** -7 * np.abs(p)).sum(1)
    return bf(p.sum(1)), far + 2.0 ** -7 * np.abs(p.sum(1))


def _glu_check(got, ref):
    y, far = ref
    d = np.abs(to_numpy(got).astype(np.float64) - y)
    assert (d <= far).all(), f"{np.max(d / np.maximum(far, 1e-300)):.3g} of the bound"
    assert cosine(to_numpy(got), y) >= MIN_COS


def _experts(seed, E, H, I, kind, dev):
    """Experts whose products stay of order one."""
    g, d = _w(seed, (E, 2 * I, H), kind, dev), _w(seed + 1, (E, H, I), kind, dev)
    for (q, s), _ in (g, d):
        q &= 0xBF                                            # magnitudes below 2: sums of order one
    up = lambda h: (torch.from_numpy(h[0].copy()).to(dev).view(torch.uint32), torch.from_numpy(h[1]).to(dev))
    for (q, s), _ in (g, d):
        s[...] = (s.astype(np.float32) * 100 + 0.02).astype(np.float32) if kind == "f32" else s + 6
    return g[0], d[0], up(g[0]), up(d[0])


@pytest.mark.parametrize("T,k,E", [(1, 1, 1), (1, 8, 16), (3, 2, 4), (16, 4, 8), (50, 2, 3), (200, 2, 3), (70, 10, 12)])
@pytest.mark.parametrize("H,I", [(256, 128), (400, 384), (528, 640), (2064, 256)])
def test_switch_glu(dev, T, k, E, H, I):
    kind = "e8m0" if T % 2 == 0 else "f32"
    hg, hd, wg, wd = _experts(T + H, E, H, I, kind, dev)
    rng = np.random.default_rng(T)
    inds = np.stack([rng.choice(E, k, replace=False) if k <= E else rng.integers(0, E, k) for _ in range(T)])
    x = _x(T, (T, H), BF, dev)
    sc = torch.softmax(_x(T + 1, (T, k), FS, dev), -1).to(BF)
    ti = torch.from_numpy(inds).to(dev)
    got = K.switch_glu_fp8(x, ti, *wg, *wd)
    assert got.shape == (T, k, H)
    _glu_check(got, _glu_ref(to_numpy(x), inds, hg, hd))
    got = K.switch_glu_fp8(x, ti, *wg, *wd, sc)
    assert got.shape == (T, H)
    _glu_check(got, _glu_ref(to_numpy(x), inds, hg, hd, to_numpy(sc)))


@pytest.mark.parametrize("T,k,E,H,I", [(1, 2, 4, 256, 4224), (3, 2, 3, 8208, 128), (40, 2, 3, 8208, 128), (40, 1, 2, 128, 8320),
                                       (13, 4, 64, 144, 256), (90, 6, 65, 144, 1408)])
def test_switch_glu_long_and_wide(dev, T, k, E, H, I):
    """Scales in more than one chunk, both ways round; pairs past the combining
    kernel's depth; columns in units of every size."""
    hg, hd, wg, wd = _experts(T + I, E, H, I, "f32" if T % 2 else "e8m0", dev)
    rng = np.random.default_rng(T)
    inds = np.stack([rng.choice(E, k, replace=False) for _ in range(T)])
    x = _x(T, (T, H), BF, dev)
    sc = torch.softmax(_x(T + 1, (T, k), FS, dev), -1).to(BF)
    got = K.switch_glu_fp8(x, torch.from_numpy(inds).to(dev), *wg, *wd, sc)
    _glu_check(got, _glu_ref(to_numpy(x), inds, hg, hd, to_numpy(sc)))


def test_switch_glu_out_of_range_and_repeated_experts(dev):
    hg, hd, wg, wd = _experts(3, 4, 256, 128, "f32", dev)
    inds = np.array([[0, 0, 4], [-1, 2, 2], [7, 9, -3], [3, 1, 0]])
    x = _x(2, (4, 256), BF, dev)
    got = K.switch_glu_fp8(x, torch.from_numpy(inds).to(dev), *wg, *wd)
    _glu_check(got, _glu_ref(to_numpy(x), inds, hg, hd))
    assert (got[2] == 0).all() and torch.equal(got[0, 0], got[0, 1])
    sc = torch.full((4, 3), 0.25, dtype=BF, device=dev)
    got = K.switch_glu_fp8(x, torch.from_numpy(inds).to(dev), *wg, *wd, sc)
    _glu_check(got, _glu_ref(to_numpy(x), inds, hg, hd, np.full((4, 3), 0.25)))
    assert (got[2] == 0).all()


# Two ways of summing may round an activation, and its E4M3 code, to different
# neighbours: an eighth of one term, which for normal operands is under 16 where
# the largest sum is over 3 sqrt(144): 5.6e-2 of it.
CODE = 5.6e-2


@pytest.mark.parametrize("T", [1, 6, 40, 300])
@pytest.mark.parametrize("I", [256, 144])
def test_block_from_float_and_checkpoint(dev, T, I, tmp_path):
    """A SparseMoeBlock with a shared expert from float weights, and the same
    layers loaded from float8 tensors with block scales, agree; the block is
    its separate ops."""
    from safetensors.torch import save_file
    E, H, k = 6, 256, 3
    f = {n: _x(i, s, BF, dev, 0.05) for i, (n, s) in enumerate(
        {"gate": (E, I, H), "up": (E, I, H), "down": (E, H, I), "sg": (I, H), "su": (I, H), "sd": (H, I)}.items())}
    q = {n: K.quantize(t, mode="fp8") for n, t in f.items()}
    file = {}
    for n, (w, s) in q.items():
        file[f"{n}.weight"] = w.view(torch.float8_e4m3fn).cpu()
        file[f"{n}.weight_scale_inv"] = torch.exp2(s.float() - 127).cpu()
    save_file(file, str(tmp_path / "model.safetensors"))
    m = C.load_quantized(tmp_path, device=dev)
    assert set(m) == set(f) and all(v.mode == "fp8" and v.input_dims == f[n].shape[-1] for n, v in m.items())
    lin = lambda n: nn.QuantizedLinear.from_float(f[n], mode="fp8")
    mlp = nn.MLP(lin("sg"), lin("su"), lin("sd"))
    router, sgate = nn.Linear(_x(20, (E, H), BF, dev)), nn.Linear(_x(21, (1, H), BF, dev))
    one = nn.SparseMoeBlock(router, nn.SwitchGLU.from_float(f["gate"], f["up"], f["down"], mode="fp8"), k, mlp, sgate)
    two = nn.SparseMoeBlock(router, nn.SwitchGLU(m["gate"], m["up"], m["down"]), k,
                            nn.MLP(m["sg"], m["su"], m["sd"]), sgate)
    x = _x(30, (T, H), BF, dev)
    a = one(x)
    assert a.shape == (T, H)
    assert_close(to_numpy(two(x)), to_numpy(a), CODE, what="checkpoint")
    inds, scores = K.moe_route(router(x), k)
    sep = K.moe_combine(one.switch_mlp.gathered(x, inds), scores)
    assert_close(to_numpy(one.switch_mlp.combine(x, inds, scores)), to_numpy(sep), CODE, what="separate")
    assert (one.switch_mlp.fused is not None) == (I % 128 == 0)


# --- streams and graphs ----------------------------------------------------------------

@pytest.mark.parametrize("M", [1, 40, 300])
def test_captured_and_on_another_stream(dev, M):
    """Captured products replay with new inputs in place, beside eager calls."""
    _, (wq, sc) = _w(5, (384, 512), "f32", dev)
    hg, hd, wg, wd = _experts(3, 4, 256, 128, "f32", dev)
    x, xe = _x(1, (M, 512), BF, dev), _x(2, (M, 256), BF, dev)
    inds = torch.randint(0, 4, (M, 2), device=dev, dtype=torch.int32)
    scores = torch.full((M, 2), 0.5, dtype=BF, device=dev)
    call = lambda: (K.quantized_matmul(x, wq, sc, mode="fp8"), K.switch_glu_fp8(xe, inds, *wg, *wd, scores))
    call()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        other = call()
    torch.cuda.current_stream().wait_stream(st)
    assert all(torch.equal(a, b) for a, b in zip(other, call()))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
    for i in range(4):
        x.copy_(_x(10 + i, (M, 512), BF, dev))
        xe.copy_(_x(20 + i, (M, 256), BF, dev))
        inds.copy_(torch.randint(0, 4, (M, 2), device=dev, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, call()))
