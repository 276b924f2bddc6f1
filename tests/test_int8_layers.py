"""``use_int8_layers`` on the CPU: its wiring, with stand-ins for the 8-bit operators that quantize nothing.

With codes that are the values themselves and scales of 1, the converted model computes what the model did: the logits
agree to fp32 rounding (two orders of summing products of up to 1,024 terms through a handful of layers: 2^-24 * 1024 * 10
of their size is 6e-4; 1e-4 of the largest logit is asked)."""
from __future__ import annotations

import pytest
import torch

transformers = pytest.importorskip("transformers")

from test_models import tiny_qwen2  # noqa: E402
from triattention_amd import models as M  # noqa: E402
from triattention_amd.kernels import linear as Q  # noqa: E402


@pytest.fixture
def plain(monkeypatch):
    """The operators without their quantization; the calls made of them."""
    calls = []

    def quantize_rows(x):
        calls.append("rows")
        return x.float(), x.new_ones(x.shape[:-1], dtype=torch.float32)

    def rms_norm_quant(x, weight, eps, residual=None):
        calls.append("norm")
        h = x if residual is None else x + residual
        y = h * torch.rsqrt(h.pow(2).mean(-1, keepdim=True) + eps) * weight
        return y, y.new_ones(y.shape[:-1]), h

    def silu_mul_quant(gate, up):
        calls.append("silu")
        y = torch.nn.functional.silu(gate) * up
        return y, y.new_ones(y.shape[:-1])

    def int8_linear(codes, scales, weight, weight_scales, bias=None, residual=None, out_dtype=torch.bfloat16):
        calls.append("linear")
        assert (scales == 1).all() and (weight_scales == 1).all()
        y = codes @ weight.float().t()
        for extra in (bias, residual):
            y = y if extra is None else y + extra
        return y.to(out_dtype)

    for f in (quantize_rows, rms_norm_quant, silu_mul_quant, int8_linear):
        monkeypatch.setattr(Q, f.__name__, f)

    def floating(shape, dtype=None, device=None):  # (the codes' store keeps the stand-ins' floating values)
        return empty(shape, dtype=torch.float32 if dtype == torch.int8 else dtype, device=device)

    empty = torch.empty
    monkeypatch.setattr(Q.torch, "empty", floating)
    yield calls
    monkeypatch.undo()


def tiny(kind):
    if kind == "qwen2":
        return tiny_qwen2(layers=3)
    torch.manual_seed(5)
    common = dict(vocab_size=97, hidden_size=256, intermediate_size=300, num_hidden_layers=2, num_attention_heads=4,
                  num_key_value_heads=2, head_dim=64, max_position_embeddings=512, tie_word_embeddings=False)
    if kind == "llama":
        return transformers.LlamaForCausalLM(transformers.LlamaConfig(**common, attention_bias=True)).eval()
    if kind == "mistral":
        return transformers.MistralForCausalLM(transformers.MistralConfig(**common)).eval()
    return transformers.Ministral3ForCausalLM(transformers.Ministral3Config(**common)).eval()


@pytest.mark.parametrize("lm_head", [False, True])
@pytest.mark.parametrize("kind", ["qwen2", "llama", "mistral", "ministral3"])
def test_converted_layers_compute_what_the_model_did(plain, kind, lm_head):
    model = tiny(kind)
    ids = torch.randint(0, 97, (2, 19), generator=torch.Generator().manual_seed(1))
    with torch.inference_mode():
        want = model(input_ids=ids).logits
        count = M.use_int8_layers(model, lm_head=lm_head)
        plain.clear()
        got = model(input_ids=ids).logits
        steps = model(input_ids=ids[:, :7], use_cache=True)  # the model's own cache: a prompt, then token by token
        for t in range(7, 19):
            steps = model(input_ids=ids[:, t:t + 1], past_key_values=steps.past_key_values, use_cache=True)
    assert count == len(model.model.layers)
    assert plain[:7] == ["norm", "linear", "rows", "linear", "norm", "linear", "silu"]
    assert (got - want).abs().max() <= 1e-4 * want.abs().max()
    assert (steps.logits[:, -1] - want[:, -1]).abs().max() <= 1e-4 * want.abs().max()
    kept = [n for n, p in model.named_parameters()]
    assert not any("proj" in n for n in kept) and any("layernorm" in n for n in kept)
    assert ("lm_head.weight" in kept) == (not lm_head)


def test_refusals_leave_the_model_alone(plain):
    with pytest.raises(ValueError, match="no decoder layer"):
        M.use_int8_layers(torch.nn.Linear(2, 2))
    model = tiny("llama")
    with pytest.raises(ValueError, match="inference"):
        M.use_int8_layers(model.train())
    model.eval()
    with pytest.raises(ValueError, match="made from torch.nn.Linear"):
        model.model.layers[1].mlp.up_proj = torch.nn.Identity()
        M.use_int8_layers(model)
    assert type(model.model.layers[0].self_attn.q_proj) is torch.nn.Linear
    model = tiny("llama")
    model.model.layers[1].mlp.act_fn = torch.nn.GELU()
    with pytest.raises(ValueError, match="SwiGLU"):
        M.use_int8_layers(model)
    assert type(model.model.layers[0].self_attn.q_proj) is torch.nn.Linear
    model = tiny("llama")
    model.model.layers[1].mlp.down_proj.bfloat16()
    with pytest.raises(ValueError, match="one type"):
        M.use_int8_layers(model)
    assert type(model.model.layers[0].self_attn.q_proj) is torch.nn.Linear
    model = tiny("llama")
    M.use_int8_layers(model)
    with pytest.raises(ValueError, match="already"):
        M.use_int8_layers(model)
