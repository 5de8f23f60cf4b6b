"""SwitchGLU over block-scaled E4M3 experts: which calls take the one-call
kernels, and what the separate products give elsewhere."""
import numpy as np
import pytest
import torch

import knurlogic_amd as K
from knurlogic_amd import nn
from tests import fp8_ref as R
from tests.util import assert_close, to_numpy

BF = torch.bfloat16


def _layer(E, N, Kd, device):
    return nn.QuantizedSwitchLinear(torch.zeros(E, N, Kd // 4, dtype=torch.int32, device=device).view(torch.uint32),
                                    torch.ones(E, -(-N // 128), -(-Kd // 128), device=device), None, None, 128, 8, "fp8")


def test_one_call_within_its_limits():
    """64 pairs a token and 2^30 activations are the entry's limits; past them
    the block goes through the separate products."""
    glu = nn.SwitchGLU(_layer(2, 128, 272, "cpu"), _layer(2, 128, 272, "cpu"), _layer(2, 272, 128, "cpu"))
    x = torch.empty(3, 272, dtype=BF, device="meta")
    assert glu._one_call_fp8(x, 64) and not glu._one_call_fp8(x, 65)
    # a row of 272 takes 384 codes
    most = (2 ** 30 - 1) // 384
    assert glu._one_call_fp8(torch.empty(most, 272, dtype=BF, device="meta"), 1)
    assert not glu._one_call_fp8(torch.empty(7, most // 7 + 1, 272, dtype=BF, device="meta"), 1)
    assert not glu._one_call_fp8(x.half(), 2)


@pytest.mark.gpu
def test_more_pairs_than_the_one_call_takes(dev):
    g = torch.Generator().manual_seed(1)
    w = lambda *s: (torch.randn(*s, generator=g) * 0.05).to(BF).to(dev)
    glu = nn.SwitchGLU.from_float(w(70, 128, 256), w(70, 128, 256), w(70, 256, 128), mode="fp8")
    x = w(3, 256) * 20
    inds = torch.stack([torch.randperm(70, generator=g)[:65] for _ in range(3)]).to(dev)
    y = glu(x, inds)
    assert y.shape == (3, 65, 256) and torch.equal(y, glu.gathered(x, inds))
    assert torch.isfinite(y).all() and (y != 0).any()


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["affine", "mxfp8", "fp8"])
@pytest.mark.parametrize("has", ["gud", "d", "g"])
def test_biases_of_the_projections(dev, mode, has):
    """A block whose layers have biases is its layers called one by one."""
    g = torch.Generator().manual_seed(2)
    w = lambda *s: (torch.randn(*s, generator=g) * 0.05).to(BF).to(dev)
    E, H, I, T, k = 5, 256, 128, 9, 2
    layer = lambda n, N, Kd: nn.QuantizedSwitchLinear.from_float(w(E, N, Kd), w(E, N) * 20 if n in has else None, mode=mode)
    gate, up, down = layer("g", I, H), layer("u", I, H), layer("d", H, I)
    x = w(T, H) * 20
    inds = torch.randint(0, E, (T, k), generator=g).to(dev)
    scores = torch.full((T, k), 0.5, dtype=BF, device=dev)
    rows, of = x.repeat_interleave(k, 0)[:, None], inds.reshape(-1)
    want = down(K.swiglu(gate(rows, of), up(rows, of)), of).view(T, k, H)
    glu = nn.SwitchGLU(gate, up, down)
    assert_close(to_numpy(glu(x, inds)), to_numpy(want), what="pairs")
    assert_close(to_numpy(glu.combine(x, inds, scores)), to_numpy(K.moe_combine(want, scores)), what="combined")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "e8m0"])
@pytest.mark.parametrize("T,k,E,I", [(1, 8, 16, 1408), (2, 8, 40, 768), (24, 2, 8, 1024), (1, 4, 8, 4224)])
def test_few_rows_are_multiplied_exactly(dev, T, k, E, I, kind):
    """Where a block streams its weights, the down product drops nothing of the
    codes' products.  Gate and up pick one input each, so the activations are
    known exactly; a sum in float32 in some 50 steps is then 50^0.5 2^-25 = 2e-7
    from the definition's (relative, in the mean), and crosses a border of
    bfloat16, 2^-8 to 2^-7 apart, for 1 in 10^4 results.  With products lined up
    at 13 places it is 3 in 100 of such codes, spread over all of E4M3."""
    H = 2048
    rng = np.random.default_rng(I)
    pick = rng.integers(0, H, 2 * I)
    g = torch.zeros(E, 2 * I, H, dtype=torch.uint8, device=dev)
    g[:, torch.arange(2 * I), torch.from_numpy(pick).to(dev)] = 0x38                       # 1.0
    d = rng.integers(0, 256, (E, H, I), dtype=np.uint8)
    d[(d & 127) == 127] = 0x30
    one = lambda *s: torch.ones(*s, device=dev) if kind == "f32" else torch.full(s, 127, dtype=torch.uint8, device=dev)
    sd = rng.random((E, H // 128, I // 128)).astype(np.float32) + 0.5 if kind == "f32" else \
        rng.integers(124, 130, (E, H // 128, I // 128)).astype(np.uint8)
    x = torch.randn(T, H, generator=torch.Generator().manual_seed(3)).to(BF)
    inds = np.stack([rng.permutation(E)[:k] for _ in range(T)])
    scores = torch.softmax(torch.randn(T, k, generator=torch.Generator().manual_seed(4)), -1).to(BF)
    args = (x.to(dev), torch.from_numpy(inds).to(dev), g.view(torch.uint32), one(E, 2 * I // 128, H // 128),
            torch.from_numpy(d).to(dev).view(torch.uint32), torch.from_numpy(sd).to(dev))
    bf = lambda v: torch.from_numpy(np.asarray(v, np.float32)).to(BF).double().numpy()
    gu = R.rows(to_numpy(x))[:, pick]
    gate, up = gu[:, :I], gu[:, I:]
    h = R.rows(bf(bf(gate / (1 + np.exp(-gate))) * up))
    y = np.stack([np.stack([h[t] @ R.weights(d[e], sd[e]).T for e in inds[t]]) for t in range(T)])
    off = (to_numpy(K.switch_glu_fp8(*args)) != bf(y)).mean()
    assert off < 1e-3, off
    out = bf(bf(bf(y) * to_numpy(scores)[..., None]).sum(1))
    off = (to_numpy(K.switch_glu_fp8(*args, scores.to(dev))) != out).mean()
    assert off < 1e-3, off


def _separate_ref(x, inds, gate, up, down, dtype):
    """float64 SwitchGLU of separate (codes, scales) with the roundings to
    ``dtype`` of its steps, and how far separate products may be from it
    (counted as for a single product; an activation, and its code, may round to
    the neighbour)."""
    rnd = lambda v: torch.from_numpy(np.asarray(v, np.float64)).to(torch.float32).to(dtype).double().numpy()
    eps = torch.finfo(dtype).eps
    act = lambda g, u: rnd(rnd(g / (1 + np.exp(-g))) * u)
    T, k = inds.shape
    H = down[0].shape[1]
    y, far = np.zeros((T, k, H)), np.zeros((T, k, H))
    for e in np.unique(inds):
        t, j = np.nonzero(inds == e)
        (g, gm, gc), (u, um, uc) = (R.product(x[t], w[e], s[e]) for w, s in (gate, up))
        ge, ue = R.bound(0 * g, gm, gc, x.shape[1], 0), R.bound(0 * u, um, uc, x.shape[1], 0)
        h, off = act(rnd(g), rnd(u)), 0
        for a in (-1, 1):
            for b in (-1, 1):
                off = np.maximum(off, np.abs(R.rows(act(rnd(g + a * ge), rnd(u + b * ue))) - R.rows(h)))
        d, mag, cut = R.product(h, down[0][e], down[1][e])
        y[t, j] = rnd(d)
        far[t, j] = R.bound(d, mag, cut, h.shape[1], eps) + eps / 2 * np.abs(d) + \
            (1 + eps / 2) * off @ np.abs(R.weights(down[0][e], down[1][e])).T
    return y, far


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, torch.float16])
@pytest.mark.parametrize("T", [1, 20, 150])
@pytest.mark.parametrize("I", [144, 256])
def test_separate_products_against_float64(dev, dtype, T, I):
    """What SwitchGLU runs where one call does not take it: I that is not whole
    blocks, float16 rows; and gathered for what it does."""
    E, H, k = 5, 272, 2
    rng = np.random.default_rng(T + I)

    def layer(n, m):
        q = rng.integers(0, 256, (E, n, m), dtype=np.uint8) & 0xBF                     # below 2
        s = (rng.random((E, -(-n // 128), -(-m // 128))) * 0.03 + 0.02).astype(np.float32)
        up = torch.from_numpy(q.copy()).to(dev).view(torch.uint32)
        return (q, s), nn.QuantizedSwitchLinear(up, torch.from_numpy(s).to(dev), None, None, 128, 8, "fp8")
    (gate, lg), (up, lu), (down, ld) = layer(I, H), layer(I, H), layer(H, I)
    glu = nn.SwitchGLU(lg, lu, ld)
    assert (glu.fused is None) == (I == 144)
    x = torch.randn(T, H, generator=torch.Generator().manual_seed(T)).to(dtype)
    inds = np.stack([rng.permutation(E)[:k] for _ in range(T)])
    y, far = _separate_ref(to_numpy(x), inds, gate, up, down, dtype)
    ti = torch.from_numpy(inds).to(dev)
    got = glu.gathered(x.to(dev), ti)
    d = np.abs(to_numpy(got).astype(np.float64) - y)
    assert got.dtype == dtype and (d <= far).all(), f"{np.max(d / far):.3g} of the bound"
    if not glu._one_call_fp8(x, k):
        assert torch.equal(glu(x.to(dev), ti), got)
