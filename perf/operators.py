"""Timed cases of the block-scaled 8-bit floating point operators.

Weights are E4M3 with one scale per block of 128 x 128 (float32, as checkpoints
ship them, or E8M0 bytes); activations are E4M3 with one power-of-two scale per
row and 128 inputs, quantized inside the call:

- ``quantize``: ``quantize(w, mode="fp8")``, weights into codes and scales;
- ``matmul``: ``quantized_matmul(..., mode="fp8")``, a dense projection;
- ``gather``: ``gather_qmm(..., mode="fp8")``, rows against their own expert;
- ``glu``: ``switch_glu_fp8``, an expert block's routed part (gate, up, SwiGLU,
  down and the weighted combine).

``run`` computes each in elementary torch operations in 32 bits, or, with
``own``, through this package.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK = 128
TOP = 448.0          # E4M3's largest value


def listed():
    moe = {"op": "glu", "experts": 128, "k": 8, "hidden": 2048, "inter": 768}
    return [
        # a checkpoint's bf16 projection converted at load time
        {"name": "quantize-dense", "op": "quantize", "batch": 1, "out": 14336, "in": 4096, "dtype": "bf16"},
        # a few small float32 experts whose last blocks are partial
        {"name": "quantize-ragged", "op": "quantize", "batch": 5, "out": 700, "in": 1040, "dtype": "fp32"},
        # the smallest call: one token through a square projection
        {"name": "matmul-m1", "op": "matmul", "rows": 1, "out": 4096, "in": 4096, "dtype": "bf16", "scales": "f32"},
        # 16 sequences decoded together through an up projection
        {"name": "matmul-m16", "op": "matmul", "rows": 16, "out": 14336, "in": 4096, "dtype": "bf16", "scales": "e8m0"},
        # a short odd chunk in half precision, partial blocks of both outputs and inputs
        {"name": "matmul-m77", "op": "matmul", "rows": 77, "out": 4100, "in": 2064, "dtype": "fp16", "scales": "f32"},
        # prompt chunks through an up and a down projection
        {"name": "matmul-m2048", "op": "matmul", "rows": 2048, "out": 14336, "in": 4096, "dtype": "bf16",
         "scales": "f32"},
        {"name": "matmul-m4096", "op": "matmul", "rows": 4096, "out": 4096, "in": 14336, "dtype": "bf16",
         "scales": "e8m0"},
        # the routed rows of a decode step of 16 sequences through one expert projection
        {"name": "gather-p128", "op": "gather", "rows": 128, "experts": 128, "out": 1536, "in": 2048, "dtype": "bf16",
         "scales": "f32"},
        # a chunk's rows over few experts of odd sizes
        {"name": "gather-p3001", "op": "gather", "rows": 3001, "experts": 37, "out": 1000, "in": 1424, "dtype": "bf16",
         "scales": "e8m0"},
        # the 128-expert block: one token, 16 sequences, a prompt chunk
        {"name": "glu-t1", "tokens": 1, "scales": "f32", **moe},
        {"name": "glu-t16", "tokens": 16, "scales": "f32", **moe},
        {"name": "glu-t2048", "tokens": 2048, "scales": "f32", **moe},
    ]


def _log(rng, lo, hi):
    """A whole number spread evenly over the logarithm of [lo, hi]."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["quantize", "matmul", "matmul", "matmul", "gather", "gather", "glu", "glu"])
    kind = rng.choice(["f32", "f32", "e8m0"])
    if op == "quantize":
        batch = rng.choice([1, 1, 1, 2, 7])
        K = 16 * _log(rng, 2, 896)
        N = _log(rng, 1, max(1, min(14336, 14336 * 4096 // (K * batch))))
        return {"op": op, "batch": batch, "out": N, "in": K, "dtype": rng.choice(["bf16", "fp16", "fp32"])}
    if op == "matmul":
        K = 16 * _log(rng, 8, 896)
        N = _log(rng, 64, 14336)
        M = _log(rng, 1, max(1, min(4096, 4096 * 14336 * 4096 // (K * N))))
        return {"op": op, "rows": M, "out": N, "in": K, "dtype": rng.choice(["bf16", "bf16", "fp16"]), "scales": kind}
    if op == "gather":
        return {"op": op, "rows": _log(rng, 1, 4096), "experts": _log(rng, 1, 128), "out": _log(rng, 64, 2048),
                "in": 16 * _log(rng, 8, 128), "dtype": rng.choice(["bf16", "bf16", "fp16"]), "scales": kind}
    E = _log(rng, 4, 128)
    return {"op": op, "tokens": _log(rng, 1, 2048), "experts": E, "k": min(E, rng.choice([1, 2, 4, 6, 8, 8])),
            "hidden": 16 * _log(rng, 16, 128), "inter": 128 * rng.randint(1, 6), "scales": kind}


def _weights(g, E, N, K, kind):
    """E experts of normal weights in the format: packed codes [E, N, K/4]
    (uint32) and scales [E, ceil(N/128), ceil(K/128)]."""
    nb, kb = -(-N // BLOCK), -(-K // BLOCK)
    codes = torch.empty(E, N, K, dtype=torch.float8_e4m3fn, device=DEV)
    scales = torch.empty(E, nb, kb, dtype=torch.float32, device=DEV)
    for lo in range(0, E, 16):
        n = min(16, E - lo)
        w = torch.zeros(n, nb * BLOCK, kb * BLOCK, device=DEV)
        w[:, :N, :K] = torch.randn(n, N, K, generator=g, device=DEV) * 0.02
        b = w.view(n, nb, BLOCK, kb, BLOCK)
        top = b.abs().amax((2, 4)).clamp(min=1e-6) / TOP
        s = torch.exp2(torch.ceil(torch.log2(top))) if kind == "e8m0" else top
        q = (b / s[:, :, None, :, None]).clamp(-TOP, TOP).view(n, nb * BLOCK, kb * BLOCK)
        codes[lo:lo + n] = q[:, :N, :K].to(torch.float8_e4m3fn)
        scales[lo:lo + n] = s
    if kind == "e8m0":
        scales = (torch.log2(scales).round() + 127).to(torch.uint8)
    return codes.view(torch.uint32), scales


def _activations(g, shape, dtype):
    """Normal rows with a few channels ten times as large, as hidden states have."""
    K = shape[-1]
    x = torch.randn(*shape, generator=g, device=DEV)
    loud = torch.rand(K, generator=g, device=DEV) < 0.01
    return (x * (1 + 9 * loud)).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    op = case["op"]
    if op == "quantize":
        w = torch.randn(case["batch"], case["out"], case["in"], generator=g, device=DEV) * 0.02
        return {"op": op, "w": w.to(TYPES[case["dtype"]])}
    if op == "matmul":
        w, s = _weights(g, 1, case["out"], case["in"], case["scales"])
        return {"op": op, "w": w[0], "s": s[0],
                "x": _activations(g, (case["rows"], case["in"]), TYPES[case["dtype"]])}
    if op == "gather":
        E, P = case["experts"], case["rows"]
        w, s = _weights(g, E, case["out"], case["in"], case["scales"])
        # experts differ in how often they are chosen
        odds = torch.exp(torch.randn(E, generator=g, device=DEV))
        rhs = torch.multinomial(odds, P, replacement=True, generator=g).to(torch.int32)
        return {"op": op, "w": w, "s": s, "rhs": rhs,
                "x": _activations(g, (P, 1, case["in"]), TYPES[case["dtype"]])}
    E, T, H, I, k = (case[n] for n in ("experts", "tokens", "hidden", "inter", "k"))
    wg, sg = _weights(g, E, 2 * I, H, case["scales"])
    wd, sd = _weights(g, E, H, I, case["scales"])
    odds = torch.randn(T, E, generator=g, device=DEV) + 0.5 * torch.randn(E, generator=g, device=DEV)
    p, inds = torch.topk(torch.softmax(odds, -1), k)
    scores = (p / p.sum(-1, keepdim=True)).to(torch.bfloat16)
    return {"op": op, "w_gu": wg, "s_gu": sg, "w_down": wd, "s_down": sd, "inds": inds.to(torch.int32),
            "scores": scores, "x": _activations(g, (T, H), torch.bfloat16)}


# --- the plain form ---------------------------------------------------------------

def _exponent(top):
    """The smallest e >= -126 with top <= 448 * 2^e."""
    m, e = torch.frexp(top)                                   # top = m * 2^e, m in [0.5, 1)
    return torch.clamp(e - 9 + (m > 0.875).to(e.dtype), min=-126)


def _quantized(x):
    """x's rows in E4M3 with a scale per 128 inputs, as the values they stand for."""
    K = x.shape[-1]
    kb = -(-K // BLOCK)
    b = torch.nn.functional.pad(x.float(), (0, kb * BLOCK - K)).view(*x.shape[:-1], kb, BLOCK)
    s = torch.exp2(_exponent(b.abs().amax(-1, keepdim=True)).float())
    return ((b / s).to(torch.float8_e4m3fn).float() * s).view(*x.shape[:-1], kb * BLOCK)[..., :K]


def _dense(w, s):
    """The float32 weights [..., N, K] of packed codes and block scales."""
    q = w.view(torch.float8_e4m3fn).float()
    if s.dtype == torch.uint8:
        s = torch.exp2(s.float() - 127)
    N, K = q.shape[-2:]
    return q * s.repeat_interleave(BLOCK, -2)[..., :N, :].repeat_interleave(BLOCK, -1)[..., :K]


def _by_expert(rows, inds, E):
    """Row p of ``rows`` belongs to expert inds[p]: the rows in a [E, most, K]
    block, and where each one stands in it."""
    order = torch.argsort(inds, stable=True)
    counts = torch.bincount(inds, minlength=E)
    first = torch.cumsum(counts, 0) - counts
    of = inds[order]
    most = int(counts.max())
    place = of * most + torch.arange(inds.numel(), device=inds.device) - first[of]
    block = rows.new_zeros(E * most, rows.shape[-1])
    block[place] = rows[order]
    at = torch.empty_like(place)
    at[order] = place
    return block.view(E, most, -1), at


def _products(rows, inds, w, s):
    """rows [P, K] (values), each against expert inds[p], in float32."""
    P, (E, N) = rows.shape[0], w.shape[:2]
    inds = inds.long()
    if P * 4 <= E:                                            # few rows: their experts alone
        return torch.matmul(rows[:, None], _dense(w.view(torch.int32)[inds], s[inds]).transpose(1, 2).contiguous())[:, 0]
    block, at = _by_expert(rows, inds, E)
    return torch.matmul(block, _dense(w, s).transpose(1, 2).contiguous()).view(-1, N)[at]


def run(state):
    op = state["op"]
    if own:
        import knurlogic_amd as K
        if op == "quantize":
            wq, s = K.quantize(state["w"], mode="fp8")
            return wq.view(torch.float8_e4m3fn), s
        if op == "matmul":
            return K.quantized_matmul(state["x"], state["w"], state["s"], mode="fp8")
        if op == "gather":
            return K.gather_qmm(state["x"], state["w"], state["s"], rhs_indices=state["rhs"], mode="fp8")
        return K.switch_glu_fp8(state["x"], state["inds"], state["w_gu"], state["s_gu"], state["w_down"],
                                state["s_down"], state["scores"])
    if op == "quantize":
        w = state["w"]
        E, N, K = w.shape
        nb, kb = -(-N // BLOCK), -(-K // BLOCK)
        f = torch.nn.functional.pad(w.float(), (0, kb * BLOCK - K, 0, nb * BLOCK - N))
        f = f.view(E, nb, BLOCK, kb, BLOCK)
        e = _exponent(f.abs().amax((2, 4)))
        q = f / torch.exp2(e.float())[:, :, None, :, None]
        q = q.view(E, nb * BLOCK, kb * BLOCK)[:, :N, :K].to(torch.float8_e4m3fn)
        return q, (e + 127).to(torch.uint8)
    x = state["x"]
    if op == "matmul":
        return torch.matmul(_quantized(x), _dense(state["w"], state["s"]).t()).to(x.dtype)
    if op == "gather":
        return _products(_quantized(x[:, 0]), state["rhs"], state["w"], state["s"]).to(x.dtype)[:, None]
    T, k = state["inds"].shape
    I = state["w_gu"].shape[1] // 2
    inds = state["inds"].reshape(-1)
    rows = _quantized(x).repeat_interleave(k, 0)
    gu = _products(rows, inds, state["w_gu"], state["s_gu"]).to(x.dtype).float()
    gate, up = gu[:, :I], gu[:, I:]
    h = ((gate / (1 + torch.exp(-gate))).to(x.dtype).float() * up).to(x.dtype)
    y = _products(_quantized(h), inds, state["w_down"], state["s_down"]).to(x.dtype).float().view(T, k, -1)
    return (y * state["scores"].float()[..., None]).to(x.dtype).float().sum(1).to(x.dtype)


# --- what a pass cannot do without --------------------------------------------------

def _hit(E, draws):
    """Experts that ``draws`` even choices reach, on average."""
    return E * (1 - (1 - 1 / E) ** draws)


def work(case):
    op = case["op"]
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[case.get("dtype", "bf16")]
    blocks = lambda n, k: -(-n // BLOCK) * -(-k // BLOCK)     # noqa: E731
    one = 1 if case.get("scales") == "e8m0" else 4
    if op == "quantize":
        n = case["batch"] * case["out"] * case["in"]
        return {"bytes": n * (size + 1) + case["batch"] * blocks(case["out"], case["in"]), "flops": 2 * n}
    if op in ("matmul", "gather"):
        M, N, K = case["rows"], case["out"], case["in"]
        experts = 1 if op == "matmul" else _hit(case["experts"], M)
        index = 0 if op == "matmul" else 4 * M
        return {"bytes": experts * (N * K + one * blocks(N, K)) + M * (N + K) * size + index, "flops": 2 * M * N * K}
    T, H, I, k = (case[n] for n in ("tokens", "hidden", "inter", "k"))
    weights = 3 * I * H + one * (blocks(2 * I, H) + blocks(H, I))
    # a token's k experts differ
    hit = case["experts"] * (1 - (1 - k / case["experts"]) ** T)
    return {"bytes": hit * weights + T * H * 4 + T * k * 6, "flops": 6 * T * k * I * H}


# --- the definition in 64 bits --------------------------------------------------------

def _e4m3(device):
    """The 256 values of E4M3, from its fields."""
    c = torch.arange(256, dtype=torch.float64, device=device)
    sign = torch.where(c >= 128, -1.0, 1.0).double()
    field = torch.floor(torch.remainder(c, 128) / 8)
    frac = torch.remainder(c, 8)
    v = torch.where(field == 0, frac / 8 * 2.0 ** -6, (1 + frac / 8) * torch.exp2(field - 7))
    v = torch.where(torch.remainder(c, 128) == 127, torch.full_like(v, math.nan), v)
    return sign * v


def _nearest(v):
    """v (|v| <= 448) rounded to E4M3's grid, ties to even."""
    step = torch.exp2(torch.clamp(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -30))), min=-6) - 3)
    return torch.round(v / step) * step                       # round() takes ties to even


def _power(top):
    """2^e, e the smallest with top <= 448 * 2^e (at least -126)."""
    e = torch.ceil(torch.log2(top.clamp(min=2.0 ** -160) / TOP))
    e = torch.where(top <= TOP * torch.exp2(e - 1), e - 1, e)  # log2 next to a whole number
    e = torch.where(top > TOP * torch.exp2(e), e + 1, e)
    return torch.exp2(torch.clamp(e, min=-126))


def _rows64(x):
    out = x.double().clone()
    for lo in range(0, x.shape[-1], BLOCK):
        part = out[..., lo:lo + BLOCK]
        s = _power(part.abs().amax(-1, keepdim=True))
        out[..., lo:lo + BLOCK] = _nearest(part / s) * s
    return out


def _expert64(w, s):
    """One weight [N, K] in float64."""
    v = _e4m3(w.device)[w.view(torch.uint8).long()]
    s = torch.exp2(s.double() - 127) if s.dtype == torch.uint8 else s.double()
    N, K = v.shape
    n, k = torch.arange(N, device=w.device) // BLOCK, torch.arange(K, device=w.device) // BLOCK
    return v * s[n][:, k]


def _grouped64(rows, inds, w, s):
    out = rows.new_zeros(rows.shape[0], w.shape[1])
    for e in sorted(set(inds.tolist())):
        at = torch.nonzero(inds == e)[:, 0]
        out[at] = rows[at] @ _expert64(w[e], s[e]).t()
    return out


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        w = state["w"].double()
        for n in range(0, case["out"], BLOCK):
            for k in range(0, case["in"], BLOCK):
                part = w[:, n:n + BLOCK, k:k + BLOCK]
                w[:, n:n + BLOCK, k:k + BLOCK] = _nearest(part / _power(part.abs().amax((1, 2), keepdim=True)))
        return w, None
    if op == "matmul":
        return _rows64(state["x"]) @ _expert64(state["w"], state["s"]).t()
    if op == "gather":
        return _grouped64(_rows64(state["x"][:, 0]), state["rhs"], state["w"], state["s"])[:, None]
    bf = lambda v: v.to(torch.bfloat16).double()               # noqa: E731
    T, k = state["inds"].shape
    inds = state["inds"].reshape(-1)
    gu = bf(_grouped64(_rows64(state["x"]).repeat_interleave(k, 0), inds, state["w_gu"], state["s_gu"]))
    gate, up = gu[:, :case["inter"]], gu[:, case["inter"]:]
    h = bf(bf(gate / (1 + torch.exp(-gate))) * up)
    y = bf(_grouped64(_rows64(h), inds, state["w_down"], state["s_down"])).view(T, k, -1)
    return bf(y * state["scores"].double()[..., None]).sum(1)
