"""Loading block-scaled float8 layers beside what else an artifact holds."""
import json

import pytest
import torch

from knurlogic_amd import checkpoint as C

BF, F8 = torch.bfloat16, torch.float8_e4m3fn


def _float8(n, k, lead=(), blocks=True):
    w = torch.zeros(*lead, n, k).to(F8)
    s = torch.ones(*lead, -(-n // 128), -(-k // 128)) if blocks else torch.ones(1)
    return w, s


def _packed(n=64, k=128):
    """A 4-bit affine layer's tensors, groups of 64."""
    return {"weight": torch.zeros(n, k // 8, dtype=torch.int32), "scales": torch.ones(n, k // 64, dtype=BF),
            "biases": torch.zeros(n, k // 64, dtype=BF)}


def _save(tmp_path, tensors):
    from safetensors.torch import save_file
    save_file(tensors, str(tmp_path / "model.safetensors"))
    (tmp_path / "config.json").write_text(json.dumps({"quantization": {"group_size": 64, "bits": 4}}))
    return tmp_path


@pytest.mark.parametrize("bias", [torch.float32, torch.float16, BF])
@pytest.mark.parametrize("lead", [(), (3,)])
def test_a_bias_gets_a_type_of_the_products(lead, bias):
    """The products give bfloat16 or float16, and add_bias takes no other type
    with it."""
    w, s = _float8(256, 144, lead)
    m = C.build({"a.weight": w, "a.weight_scale_inv": s, "a.bias": torch.ones(*lead, 256, dtype=bias)}, "a", device="cpu")
    assert m.bias.dtype == (torch.float16 if bias == torch.float16 else BF) and m.bias.shape == (*lead, 256)


@pytest.mark.gpu
@pytest.mark.parametrize("x", [BF, torch.float16])
@pytest.mark.parametrize("bias", [torch.float32, torch.float16, BF])
@pytest.mark.parametrize("lead", [(), (3,)])
def test_a_layer_with_a_bias_runs(dev, lead, bias, x):
    """On a zero weight the layer gives its bias (1.25 in every type), the one
    of its expert."""
    w, s = _float8(256, 144, lead)
    b = torch.full((*lead, 256), 1.25, dtype=bias)
    if lead:
        b[1] = 2.5
    m = C.build({"a.weight": w, "a.weight_scale_inv": s, "a.bias": b}, "a", device=dev)
    if not lead:
        assert torch.equal(m(torch.ones(5, 144, dtype=x, device=dev)), torch.full((5, 256), 1.25, dtype=x, device=dev))
        return
    y = m(torch.ones(4, 1, 144, dtype=x, device=dev), torch.tensor([0, 1, 2, 1], device=dev))
    assert y.dtype == x and y[:, 0, 0].tolist() == [1.25, 2.5, 1.25, 2.5] and torch.equal(y, y[..., :1].expand_as(y))


@pytest.mark.parametrize("other", ["per tensor", "inputs", "not float8", "blocks of 64", "alone"])
def test_layers_of_other_forms_stay_out(tmp_path, other):
    """A float8 layer that is not in blocks of 128 x 128 is left out, as any
    layer without packed weights, and keeps nothing else from loading; build
    refuses it by name."""
    w, s = {"per tensor": _float8(128, 128, blocks=False), "inputs": _float8(128, 24),
            "not float8": (torch.zeros(128, 128, dtype=BF), torch.ones(1, 1)),
            "blocks of 64": (torch.zeros(128, 128).to(F8), torch.ones(2, 2)),
            "alone": (None, torch.ones(1, 1))}[other]
    t = {f"a.{n}": v for n, v in _packed().items()}
    t["b.weight_scale_inv"] = s
    if w is not None:
        t["b.weight"] = w
    fw, fs = _float8(128, 144)
    t["c.weight"], t["c.weight_scale_inv"] = fw, fs
    m = C.load_quantized(_save(tmp_path, t), device="cpu")
    assert set(m) == {"a", "c"} and m["a"].mode == "affine" and m["c"].mode == "fp8"
    with pytest.raises(ValueError, match="b: weight_scale_inv"):
        C.build(t, "b", device="cpu")


@pytest.mark.parametrize("shape", [(1, 2), (1,)])
def test_packed_weights_go_before_a_scale_left_beside_them(tmp_path, shape):
    t = {f"a.{n}": v for n, v in _packed().items()} | {"a.weight_scale_inv": torch.ones(shape)}
    m = C.load_quantized(_save(tmp_path, t), device="cpu")
    assert m["a"].mode == "affine"
    assert C.build(t, "a", 128, device="cpu").mode == "affine"
