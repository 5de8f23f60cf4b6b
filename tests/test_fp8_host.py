"""What the block-scaled E4M3 ops refuse, the loader's layout rules and the
reference helper itself -- no GPU needed."""
import numpy as np
import pytest
import torch

import knurlogic_amd as K
from knurlogic_amd import _abi, nn, ops
from knurlogic_amd import checkpoint as C
from tests import fp8_ref as R

BF = torch.bfloat16


def _w(N=130, Kd=272, lead=(), scales=torch.float32):
    w = torch.zeros(*lead, N, Kd // 4, dtype=torch.int32).view(torch.uint32)
    return w, torch.zeros(*lead, -(-N // 128), -(-Kd // 128), dtype=scales)


def test_reference_codes_are_torchs():
    """The helper's table and rounding against torch's float8 conversion."""
    codes = torch.arange(256, dtype=torch.int32).to(torch.uint8)
    v = codes.view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(np.nan_to_num(v, nan=9e9), np.nan_to_num(R.VALUES, nan=9e9))
    x = torch.linspace(-448, 448, 100001, dtype=torch.float32)
    x = torch.cat([x, x / 4096, x / 65536])
    assert np.array_equal(R.nearest(x.double().numpy()), x.to(torch.float8_e4m3fn).view(torch.uint8).numpy())


@pytest.mark.parametrize("top,e", [(448.0, 0), (448.0001, 1), (0.0, -126), (1.75, -8), (1.76, -7), (3.4e38, 120)])
def test_reference_exponent(top, e):
    assert R.exponent(top) == e


def test_ops_refuse_what_the_format_is_not():
    x = torch.zeros(4, 272, dtype=BF)
    w, s = _w()
    with pytest.raises(ValueError, match="GPU memory"):
        K.quantized_matmul(x, w, s, mode="fp8")
    with pytest.raises(ValueError, match="GPU memory"):
        K.quantize(torch.zeros(4, 64, dtype=BF), mode="fp8")
    with pytest.raises(ValueError, match="2-D weight with transpose=True"):
        K.quantized_matmul(x, w, s, mode="fp8", transpose=False)
    with pytest.raises(ValueError, match="2-D weight"):
        K.quantized_matmul(x, *_w(lead=(2,)), mode="fp8")
    with pytest.raises(ValueError, match="transpose=True"):
        K.gather_qmm(x[:, None], *_w(lead=(2,)), mode="fp8", transpose=False)
    with pytest.raises(ValueError, match="no biases"):
        K.quantized_matmul(x, w, s, s, mode="fp8")
    for kw in ({"group_size": 64}, {"bits": 4}):
        with pytest.raises(ValueError, match="group_size 128 and 8 bits"):
            K.quantized_matmul(x, w, s, mode="fp8", **kw)
        with pytest.raises(ValueError, match="group_size 128 and 8 bits"):
            K.quantize(x, mode="fp8", **kw)
    for bad in (s[:1], s[:, :2], s.t(), s[0]):
        with pytest.raises(ValueError, match="expected"):
            K.quantized_matmul(x, w, bad, mode="fp8")
        with pytest.raises(ValueError, match="expected"):
            K.dequantize(w, bad, mode="fp8")
    with pytest.raises(ValueError, match="float32 or uint8"):
        K.quantized_matmul(x, w, s.to(BF), mode="fp8")
    with pytest.raises(ValueError, match="packed uint32 or float8"):
        K.quantized_matmul(x, w.view(torch.uint8), s, mode="fp8")
    with pytest.raises(ValueError, match="multiples of 16"):
        K.quantized_matmul(x, torch.zeros(4, 66, dtype=torch.int32), torch.zeros(1, 3), mode="fp8")
    with pytest.raises(ValueError, match="multiples of 16"):
        K.quantized_matmul(x, torch.zeros(4, 72).to(torch.float8_e4m3fn), torch.zeros(1, 1), mode="fp8")
    with pytest.raises(ValueError, match="affine, mxfp4 and mxfp8"):
        ops.qmm_batched(x, w, s, None, mode="fp8")


def test_switch_glu_refusals():
    x, i = torch.zeros(3, 256, dtype=BF), torch.zeros(3, 2, dtype=torch.int32)
    g, d = _w(512, 256, (4,)), _w(256, 256, (4,))
    with pytest.raises(ValueError, match="GPU memory"):
        K.switch_glu_fp8(x, i, *g, *d)
    with pytest.raises(ValueError, match="bfloat16"):
        K.switch_glu_fp8(x.half(), i, *g, *d)
    with pytest.raises(ValueError, match="both weights' scales"):
        K.switch_glu_fp8(x, i, *g, *_w(256, 256, (4,), torch.uint8))


def test_c_entries_refuse_on_the_host():
    """Bad arguments come back as -1 (or -3) before anything touches the GPU:
    the pointers here are never read."""
    L = _abi.load()
    ok = dict(x=16, M=4, K=256, N=64, w=16, s=16, e8=0, dt=0, y=16, ws=None, n=0, st=None)

    def qmm(**kw):
        return L.kmi_qmm_fp8(*{**ok, **kw}.values())
    assert qmm(K=250) == -1 and b"multiple of 16" in L.kmi_last_error()
    assert qmm(K=0) == -1 and qmm(N=0) == -1 and qmm(dt=2) == -1 and qmm(M=-1) == -1
    assert qmm(K=65552) == -1 and b"65536" in L.kmi_last_error() and qmm(M=1 << 21) == -1
    assert qmm(M=64, K=65536) == -3 and qmm(M=17) == -3 and qmm(M=1, K=16400) == -3
    assert qmm(x=8) == -1 and b"16 bytes" in L.kmi_last_error()
    assert qmm(w=4) == -1 and qmm(y=None) == -1 and b"null" in L.kmi_last_error()
    assert qmm(M=0) == 0
    g = dict(x=16, X=4, M=1, K=256, w=16, s=16, e8=0, E=4, N=64, l=16, r=16, P=4, dt=0, y=16, ws=None, n=0, st=None)

    def gather(**kw):
        return L.kmi_gather_qmm_fp8(*{**g, **kw}.values())
    assert gather(P=400) == -3 and b"workspace" in L.kmi_last_error()
    assert gather(K=65552) == -1 and gather(X=1 << 20, K=4096, P=1 << 20) == -1 and b"2 GiB" in L.kmi_last_error()
    assert gather(E=5000) == -1 and gather(E=0) == -1 and gather(K=8) == -1 and gather(P=1 << 40) == -1
    assert gather(l=None) == -1 and gather(P=0) == 0
    assert L.kmi_gather_qmm_fp8_workspace_bytes(400, 4, 1, 4, 256, 64, 0) > 0
    u = dict(x=16, T=4, H=256, I=128, k=2, i=16, sc=16, wg=16, sg=16, wd=16, sd=16, e8=0, E=4, dt=0, o=16, ws=None,
             n=0, st=None)

    def glu(**kw):
        return L.kmi_switch_glu_fp8(*{**u, **kw}.values())
    assert glu() == -3 and glu(I=144) == -1 and b"blocks of 128" in L.kmi_last_error()
    assert glu(H=65552) == -1 and glu(I=65664) == -1
    assert glu(H=250) == -1 and glu(k=0) == -1 and glu(k=65) == -1 and glu(dt=1) == -1 and glu(E=0) == -1
    assert glu(wd=None) == -1 and glu(T=0) == 0 and glu(T=1 << 30, k=64) == -1
    assert L.kmi_quantize_fp8(16, 0, 1, 4, 24, 16, 16, None) == -1
    assert L.kmi_quantize_fp8(8, 0, 1, 4, 32, 16, 16, None) == -1
    assert L.kmi_quantize_fp8(16, 0, 1, 0, 32, 16, 16, None) == 0
    assert L.kmi_dequantize_fp8(16, 16, 0, 1, 4, 24, 16, 0, None) == -1
    assert L.kmi_dequantize_fp8(16, None, 0, 1, 4, 32, 16, 0, None) == -1


def test_modules_keep_the_format():
    g = nn.QuantizedSwitchLinear(*_w(256, 272, (3,)), None, None, 128, 8, "fp8")
    assert (g.input_dims, g.output_dims, g.num_experts) == (272, 256, 3)
    s = nn.SwitchGLU(g, g, nn.QuantizedSwitchLinear(*_w(272, 256, (3,)), None, None, 128, 8, "fp8"))
    assert s.fused.weight.shape == (3, 512, 68) and s.fused.scales.shape == (3, 4, 3)
    assert s.up_proj.scales.shape == (3, 2, 3) and s.up_proj.output_dims == 256
    # blocks that gate and up would share are not stacked
    p = nn.QuantizedSwitchLinear(*_w(144, 272, (3,)), None, None, 128, 8, "fp8")
    assert nn.SwitchGLU(p, p, g).fused is None


def test_loader_refuses_other_block_shapes():
    w = torch.zeros(256, 256).to(torch.float8_e4m3fn)
    m = C.build({"a.weight": w, "a.weight_scale_inv": torch.ones(2, 2, dtype=BF)}, "a", device="cpu")
    assert m.mode == "fp8" and m.scales.dtype == torch.float32 and m.input_dims == 256
    assert C.fp8_recipe({"a.weight": w}, "a") is None
    # packed words and E8M0 bytes, the mode declared by the settings
    m = C.build({"a.weight": w.view(torch.uint8).view(torch.uint32)[:, :52].contiguous(),
                 "a.scales": torch.ones(2, 2, dtype=torch.uint8)}, "a", 208, {"mode": "fp8"}, device="cpu")
    assert (m.mode, m.group_size, m.bits, m.input_dims) == ("fp8", 128, 8, 208)
    with pytest.raises(ValueError, match="128 x 128"):
        C.build({"a.weight": w, "a.weight_scale_inv": torch.ones(4, 4)}, "a", device="cpu")
    with pytest.raises(ValueError, match="not float8"):
        C.build({"a.weight": w.float(), "a.weight_scale_inv": torch.ones(2, 2)}, "a", device="cpu")
    with pytest.raises(ValueError, match="128 x 128"):
        C.build({"a.weight": w[:, :24], "a.weight_scale_inv": torch.ones(2, 1)}, "a", device="cpu")


@pytest.mark.parametrize("M,K,stream", [(1, 4096, 1), (16, 4096, 1), (17, 4096, 0), (16, 4112, 0), (9, 4112, 0), (8, 4112, 1),
                                        (8, 9216, 1), (8, 9232, 0), (2, 9232, 0), (2, 14336, 0), (16, 14336, 0),
                                        (1, 16384, 1), (1, 16400, 0)])
def test_few_rows_of_a_long_k_leave_the_stream(M, K, stream):
    """The stream quantizes x in every workgroup before its first product: with
    many inputs that costs more than the pass over x that the tiles take (which
    need a workspace for it; the stream needs none)."""
    for N in (64, 4096, 14336):
        for dtype in (0, 1):
            assert (_abi.load().kmi_qmm_fp8_workspace_bytes(M, K, N, dtype) == 0) == bool(stream)
