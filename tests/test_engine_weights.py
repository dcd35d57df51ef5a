"""Int8Qwen3Weights.from_hf takes models of INT8 linears and refuses all others at once, as they were."""
import pytest
import torch

from helm_amd.kernels import Int4Linear, Int8Linear, patch_int4_linears, patch_linears
from helm_amd.runtime.decode_engine import Int8Qwen3Weights


def model():
    from transformers import Qwen3Config, Qwen3ForCausalLM
    torch.manual_seed(0)
    return Qwen3ForCausalLM(Qwen3Config(hidden_size=128, num_attention_heads=4, num_key_value_heads=2, head_dim=64,
                                        intermediate_size=256, num_hidden_layers=2, vocab_size=64)).half().eval()


def test_int8_models_are_taken_and_share_storage():
    m = model()
    patch_linears(m, exclude=("lm_head",))
    w = Int8Qwen3Weights.from_hf(m)
    assert len(w.layers) == 2 and w.layers[0]["qkv_q"].shape == (8 * 64, 128)
    assert m.model.layers[1].self_attn.q_proj.qweight.data_ptr() == w.layers[1]["qkv_q"].data_ptr()


@pytest.mark.parametrize("kind", ["int4", "fp16", "one"])
def test_other_linears_are_refused_as_they_were(kind):
    m = model()
    if kind == "int4":
        patch_int4_linears(m, 64, exclude=("lm_head",))
    elif kind == "one":                                   # the last projection alone
        down = m.model.layers[1].mlp.down_proj
        patch_linears(m, exclude=("lm_head",))
        m.model.layers[1].mlp.down_proj = Int4Linear.from_linear(down, 64)
    before = {n: (t.data_ptr(), t.shape) for n, t in m.state_dict(keep_vars=True).items()}
    name = {"int4": "layer 0's self_attn.q_proj is Int4Linear", "fp16": "layer 0's self_attn.q_proj is Linear",
            "one": "layer 1's mlp.down_proj is Int4Linear"}[kind]
    with pytest.raises(RuntimeError, match=name):
        Int8Qwen3Weights.from_hf(m)
    assert {n: (t.data_ptr(), t.shape) for n, t in m.state_dict(keep_vars=True).items()} == before
    assert kind != "one" or isinstance(m.model.layers[0].self_attn.q_proj, Int8Linear)
