"""CPU checks of the layers in the block-scaled mode: weights and outputs of
another shape than the layer's are refused before anything is launched."""

from __future__ import annotations

import pytest
import torch

from glm53flash import fp8_block, moe as moe_module
from glm53flash.contract import ContractError
from glm53flash.expert_ssd import HBMExpertBank
from glm53flash.layers import DeferredLinear, DenseMLP
from glm53flash.model_config import GLMTextConfig
from glm53flash.moe import ExpertSSDMoE


def attach(lin, n, k, dtype=torch.uint8):
    lin.weight = torch.zeros((n, k), dtype=dtype)
    lin.scales = torch.zeros((-(-n // 128), -(-k // 128)))
    lin.quantization_mode = "fp8_block"


def attached(d, I, shapes=()):
    mlp = DenseMLP(d, I, 10.0)
    for name in ("gate_proj", "up_proj", "down_proj"):
        lin = getattr(mlp, name)
        attach(lin, *dict(shapes).get(name, (lin.output_dims, lin.input_dims)))
    return mlp


@pytest.fixture
def products(monkeypatch):
    """The products as shapes alone: what they would launch is counted."""
    calls = []

    def linear(x, w, s, *, out=None):
        calls.append("linear")
        return torch.zeros((*(x.codes if isinstance(x, tuple) else x).shape[:-1], w.shape[0]), dtype=torch.bfloat16)

    def gate_up(x, g, gs, u, us, limit, *, out=None):
        calls.append("gate_up")
        shape = (*x.shape[:-1], g.shape[0])
        return fp8_block.Fp8Rows(torch.zeros(shape, dtype=torch.uint8), torch.zeros(*shape[:-1], -(-shape[-1] // 128)))

    monkeypatch.setattr(fp8_block, "linear", linear)
    monkeypatch.setattr(fp8_block, "gate_up", gate_up)
    return calls


@pytest.mark.parametrize("shape", [(16, 256), (48, 256), (32, 128), (32, 512), (256, 32)])
def test_a_linear_takes_its_own_shape_alone(products, shape):
    lin = DeferredLinear(256, 32)
    attach(lin, *shape)
    with pytest.raises(ContractError, match="the layer is"):
        lin(torch.zeros((2, shape[1])))
    assert not products
    attach(lin, 32, 256, torch.float8_e4m3fn)
    assert lin(torch.zeros((2, 256))).shape == (2, 32)


@pytest.mark.parametrize("name, shape", [("gate_proj", (32, 256)), ("up_proj", (32, 256)), ("down_proj", (128, 48)),
                                         ("down_proj", (512, 48)), ("down_proj", (256, 32))])
def test_an_mlp_takes_its_own_shapes_alone(products, name, shape):
    mlp = attached(256, 48, {name: shape})
    with pytest.raises(ContractError, match=f"{name}.weight .* the layer is"):
        mlp(torch.zeros((2, 256)))
    assert not products
    assert attached(256, 48)(torch.zeros((2, 256))).shape == (2, 256)


def test_a_conversion_takes_the_layers_own_shape(monkeypatch):
    monkeypatch.setattr(fp8_block, "quantize_weight", lambda w: pytest.fail("converted"))
    lin = DeferredLinear(32, 16)
    for shape in ((16, 24), (16, 48), (8, 32)):
        lin.weight = kept = torch.zeros(shape, dtype=torch.bfloat16)
        with pytest.raises(ContractError, match="the layer is"):
            lin.quantize_to_fp8_block()
        assert lin.weight is kept and lin.quantization_mode is None


def moe_on_the_cpu(monkeypatch):
    d = 256
    cfg = GLMTextConfig(hidden_size=d, moe_intermediate_size=128, n_routed_experts=4, num_experts_per_tok=2,
                        n_shared_experts=1, n_group=1, topk_group=1, norm_topk_prob=True, routed_scaling_factor=1.0,
                        swiglu_limit=10.0)
    layer = ExpertSSDMoE(cfg, 1, lambda i: HBMExpertBank(layer=i, num_experts=4, hidden_size=d, intermediate_size=128,
                                                         swiglu_limit=10.0, device="cpu"))
    layer.gate.weight, layer.gate.e_score_correction_bias = torch.zeros((4, d)), torch.zeros(4)
    launched = []
    monkeypatch.setattr(moe_module.N, "require_device", lambda t, name, dtypes=None: t)
    monkeypatch.setattr(moe_module.N, "stream_of", lambda t: 0)
    monkeypatch.setattr(moe_module.N, "call", lambda name, *args: launched.append(name))
    return layer, launched


@pytest.mark.parametrize("width", [128, 240, 272, 512])
def test_a_shared_expert_of_another_width_never_reaches_the_layer(monkeypatch, products, width):
    layer, launched = moe_on_the_cpu(monkeypatch)
    x = torch.zeros((3, 256), dtype=torch.bfloat16)
    # a down projection that is short or long for the layer
    layer.shared_experts = attached(256, 128, {"down_proj": (width, 128)})
    with pytest.raises(ContractError):
        layer(x)
    # the same, of an MLP that was made that way
    layer.shared_experts.down_proj.output_dims = width
    with pytest.raises(ContractError, match="shared expert output"):
        layer(x)
    assert not launched
    layer.shared_experts = attached(256, 128)
    layer(x)
    assert launched[-1] == "glm_moe_forward"


def test_other_formats_do_not_pay_for_this_one(monkeypatch):
    # a bf16 shared expert's call asks for its format once, as it did before there was a block-scaled mode
    layer, launched = moe_on_the_cpu(monkeypatch)
    for p in (layer.shared_experts.gate_proj, layer.shared_experts.up_proj, layer.shared_experts.down_proj):
        p.weight = torch.zeros((p.output_dims, p.input_dims), dtype=torch.bfloat16)
    monkeypatch.setattr(DenseMLP, "block_scaled", property(lambda self: pytest.fail("asked for")))
    x = torch.zeros((3, 256), dtype=torch.bfloat16)
    layer(x)
    assert launched[-1] == "glm_moe_forward"
    layer.shared_experts(x)
    assert launched[-1] == "glm_dense_mlp"
