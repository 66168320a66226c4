"""`LinearLoRA` as a part of a model, on the host: its scales keep their type, nothing of it is
trained, and blocks that would leave its adapters out refuse it."""
import pytest
import torch

import triton_kernels_b200 as tk
from triton_kernels_b200.flux.model import FluxDiT, FluxParams, LastLayer, MLPEmbedder
from triton_kernels_b200.modules import Modulation, SelfAttention


def lora(n_in, n_out):
    return tk.LinearLoRA(n_in, n_out, num_adapters=2, rank=4)


def test_scale_stays_fp32():
    m = lora(16, 8)
    m.lora_scale.copy_(torch.tensor([1 / 3, 0.7]))
    want = m.lora_scale.clone()
    for cast in (lambda t: t.to(torch.bfloat16), lambda t: t.half(), lambda t: t.double(), lambda t: t.float(), lambda t: torch.nn.Sequential(t).bfloat16()[0]):
        m = cast(m)
        assert m.lora_scale.dtype == torch.float32 and torch.equal(m.lora_scale, want)
    assert m.lora_a.dtype == m.lora_b.dtype == m.weight.dtype == m.bias.dtype == torch.bfloat16
    assert m.to("meta").lora_scale.is_meta and m.lora_scale.dtype == torch.float32
    assert "lora_scale" in m.state_dict()


def test_scale_is_fp32_whatever_the_default_type():
    default = torch.get_default_dtype()
    torch.set_default_dtype(torch.bfloat16)
    try:
        assert lora(16, 8).lora_scale.dtype == torch.float32
    finally:
        torch.set_default_dtype(default)


def test_a_gradient_that_would_be_lost_is_refused():
    """The operator is forward only; before it looks at anything else it refuses every argument that wants a gradient."""
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    args = [z(2, 3, 16), z(8, 16), z(8), z(1, 4, 16), z(1, 8, 4), torch.zeros(2, dtype=torch.int64), torch.ones(1)]
    for i in (0, 1, 2, 3, 4, 6):
        call = [a.clone().requires_grad_() if j == i else a for j, a in enumerate(args)]
        with pytest.raises(NotImplementedError, match="forward only"):
            tk.linear_lora(*call)
        with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA tensors only"):
            tk.linear_lora(*call)


def test_weight_and_bias_of_the_module_are_not_trained():
    m = lora(16, 8).to(torch.bfloat16)
    assert not any(p.requires_grad for p in m.parameters()) and list(m.state_dict()) == ["weight", "bias", "lora_a", "lora_b", "lora_scale"]
    x, idx = torch.zeros(2, 3, 16, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        m(x, idx)
    with pytest.raises(NotImplementedError, match="forward only"):
        m.requires_grad_()(x, idx)


C, H = 256, 2
PLACES = ["img_attn.qkv", "img_attn.proj", "txt_attn.qkv", "txt_attn.proj", "img_mlp.0", "img_mlp.2", "txt_mlp.0", "txt_mlp.2", "img_mod.lin", "txt_mod.lin"]


def put(block, place):
    old = block.get_submodule(place)
    owner, _, name = place.rpartition(".")
    setattr(block.get_submodule(owner), name, lora(old.in_features, old.out_features))
    return block.to(torch.bfloat16)


@pytest.mark.parametrize("place", PLACES)
def test_double_block_refuses_an_adapter_that_it_would_leave_out(place):
    block = put(tk.DoubleStreamBlock(C, H, 4.0, qkv_bias=True), place)
    x = torch.zeros(1, 8, C, dtype=torch.bfloat16)
    for modulation in (None, (x[:, 0].repeat(1, 6), x[:, 0].repeat(1, 6))):
        if modulation is not None and "mod" in place:
            continue  # not called then
        with pytest.raises(NotImplementedError, match="LinearLoRA"):
            block(x, x, x[:, 0], torch.zeros(1, 1, 16, C // H // 2, 2, 2), modulation=modulation)


@pytest.mark.parametrize("place", ["linear1", "linear2", "modulation.lin"])
def test_single_block_refuses_an_adapter_that_it_would_leave_out(place):
    block = put(tk.SingleStreamBlock(C, H), place)
    x = torch.zeros(1, 8, C, dtype=torch.bfloat16)
    with pytest.raises(NotImplementedError, match="LinearLoRA"):
        block(x, x[:, 0], torch.zeros(1, 1, 8, C // H // 2, 2, 2))


def test_parts_refuse_it():
    x = torch.zeros(1, 8, C, dtype=torch.bfloat16)
    for double in (False, True):
        with pytest.raises(NotImplementedError, match="LinearLoRA"):
            put(Modulation(C, double), "lin")(x[:, 0])
    with pytest.raises(NotImplementedError, match="LinearLoRA"):
        put(Modulation(C, True), "lin").packed_rows(x[:, 0], torch.empty(1, 6 * C, dtype=torch.bfloat16), True)
    for place in ("qkv", "proj"):
        with pytest.raises(NotImplementedError, match="LinearLoRA"):
            put(SelfAttention(C, H), place)(x, torch.zeros(1, 1, 8, C // H // 2, 2, 2))


def test_model_parts_refuse_it():
    p = FluxParams(in_channels=16, context_in_dim=32, hidden_size=C, num_heads=H, depth=1, depth_single_blocks=1, axes_dim=[16, 56, 56])
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    for place in ("img_in", "txt_in"):
        with pytest.raises(NotImplementedError, match="LinearLoRA"):
            put(FluxDiT(p), place)(z(1, 8, 16), z(1, 4, 32), z(1), z(1), z(1, 1, 12, 64, 2, 2))
    for place in ("in_layer", "out_layer"):
        with pytest.raises(NotImplementedError, match="LinearLoRA"):
            put(MLPEmbedder(256, C), place)(z(1, 256))
    for place in ("linear", "adaLN_modulation.1"):
        with pytest.raises(NotImplementedError, match="LinearLoRA"):
            put(LastLayer(C, 1, 16), place)(z(1, 8, C), z(1, C))
