"""Block-scaled E4M3 ops on two streams at once, and captured and replayed
beside eager calls: every route's workspace belongs to its own call."""
import pytest
import torch

import knurlogic_amd as K

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _calls(dev, seed):
    """(inputs to refill in place, a function of them) over every op: the
    stream, K in parts, tiles; pairs, sorted rows, tiles of 64 and 128; the
    block's three ways."""
    g = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=dev).to(BF)
    dense = K.quantize(r(320, 4096) * 0.02, mode="fp8")
    experts = K.quantize(r(8, 200, 528) * 0.02, mode="fp8")
    gu, down = K.quantize(r(8, 512, 528) * 0.05, mode="fp8"), K.quantize(r(8, 528, 256) * 0.05, mode="fp8")
    rows = [r(m, 4096) for m in (3, 40, 300)]
    pairs = [r(p, 1, 528) for p in (2, 40, 300, 1200)]
    tokens = [r(t, 528) for t in (1, 24, 300)]
    of = [torch.randint(0, 8, (len(p),), generator=g, device=dev, dtype=torch.int32) for p in pairs]
    inds = [torch.randint(0, 8, (len(t), 2), generator=g, device=dev, dtype=torch.int32) for t in tokens]
    scores = [torch.full((len(t), 2), 0.5, dtype=BF, device=dev) for t in tokens]
    w = r(300, 528)

    def call():
        out = [K.quantized_matmul(x, *dense, mode="fp8") for x in rows]
        out += [K.gather_qmm(x, *experts, rhs_indices=i, mode="fp8") for x, i in zip(pairs, of)]
        out += [K.switch_glu_fp8(x, i, *gu, *down, s) for x, i, s in zip(tokens, inds, scores)]
        q = K.quantize(w, mode="fp8")
        return out + [q[0].view(torch.int32), q[1], K.dequantize(*q, mode="fp8")]
    return (*rows, *pairs, *tokens, w), (*of, *inds), call


def _same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_two_streams_at_once(dev):
    calls = [_calls(dev, s)[2] for s in (1, 2)]
    want = [c() for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = [[], []]
    for _ in range(4):
        for i, (s, c) in enumerate(zip(streams, calls)):
            with torch.cuda.stream(s):
                got[i].append(c())
    torch.cuda.synchronize()
    for i in range(2):
        assert all(_same(g, want[i]) for g in got[i])


def test_two_captured_graphs_in_turn(dev):
    made = [_calls(dev, s) for s in (3, 4)]
    graphs, outs = [], []
    for _, _, call in made:
        call()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call())
        graphs.append(g)
    for turn in range(3):
        for floats, ints, _ in made:
            for t in floats:
                t.copy_(torch.randn(t.shape, device=dev))
            for t in ints:
                t.copy_(torch.randint(0, 8, t.shape, device=dev))
        for g in graphs:
            g.replay()
        want = [call() for _, _, call in made]               # (eager, beside the replays)
        torch.cuda.synchronize()
        assert all(_same(a, b) for a, b in zip(outs, want)), turn
