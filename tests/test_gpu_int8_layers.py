"""8-bit decoder layers on the GPU: a layer against its operators called one by one, and generation through
``TriAttention`` on converted models."""
from __future__ import annotations

import copy

import pytest
import torch

transformers = pytest.importorskip("transformers")

from test_gpu_models import tiny_qwen2  # noqa: E402
from triattention_amd import models as M  # noqa: E402
from triattention_amd.kernels import linear as Q  # noqa: E402
from triattention_amd.maps import INF, from_bands  # noqa: E402

pytestmark = pytest.mark.gpu


def by_hand(layer, x, embeddings, attention):
    """The layer's output from the 8-bit operators and ``attention(q, k, v)`` [B, H, T, D]."""
    attn, mlp = layer.self_attn, layer.mlp
    first, second = layer.input_layernorm, layer.post_attention_layernorm
    codes, scales, _ = Q.rms_norm_quant(x, first.weight, first.variance_epsilon)
    heads = []
    for l in (attn.q_proj, attn.k_proj, attn.v_proj):
        y = Q.int8_linear(codes, scales, *Q.quantize_rows(l.weight.detach()), l.bias.detach())
        heads.append(y.view(*x.shape[:2], -1, attn.head_dim).transpose(1, 2))
    rotate = transformers.models.qwen2.modeling_qwen2.apply_rotary_pos_emb
    q, k = rotate(heads[0], heads[1], *embeddings)
    out = attention(q, k, heads[2]).transpose(1, 2).reshape(x.shape)
    out = Q.int8_linear(*Q.quantize_rows(out), *Q.quantize_rows(attn.o_proj.weight.detach()))
    codes, scales, h = Q.rms_norm_quant(out, second.weight, second.variance_epsilon, residual=x)
    gate = Q.int8_linear(codes, scales, *Q.quantize_rows(mlp.gate_proj.weight.detach()))
    up = Q.int8_linear(codes, scales, *Q.quantize_rows(mlp.up_proj.weight.detach()))
    return Q.int8_linear(*Q.silu_mul_quant(gate, up), *Q.quantize_rows(mlp.down_proj.weight.detach()), residual=h)


@pytest.mark.parametrize("batch,t", [(1, 1), (1, 70), (3, 40)])
def test_a_layer_is_its_operators(module, batch, t):
    """The fused projections give each its own product's bits (a channel's sum does not depend on the others')."""
    model = tiny_qwen2(torch.device("cuda"))
    plain = copy.deepcopy(model.model.layers[1])
    scaling = plain.self_attn.scaling
    M.use_attention(model, "exact", lambda mod, q, k, v, s: M.exact_attention(q, k, v, s))
    M.use_int8_layers(model)
    g = torch.Generator(device="cuda").manual_seed(t)
    x = torch.randn(batch, t, 512, generator=g, device="cuda").bfloat16()
    position = torch.arange(t, device="cuda")[None].expand(batch, t)
    with torch.inference_mode():
        embeddings = model.model.rotary_emb(x, position)
        want = by_hand(plain, x, embeddings, lambda q, k, v: M.exact_attention(q, k, v, scaling))
        got = model.model.layers[1](x, attention_mask=None, position_ids=position, position_embeddings=embeddings)
    assert torch.isfinite(want).all() and torch.equal(got, want)


@pytest.mark.parametrize("lm_head", [False, True])
def test_generate_eager_and_captured(module, lm_head):
    """``generate`` on a converted model: the graph gives the eager run's tokens, over prompts of several lengths."""
    bands = {"0": [[INF, INF]] * 4, "1": [[2, 4], [1, 3], [INF, INF], [INF, INF]]}
    for prompt in (1, 77, 300):
        tokens = []
        for graph in (False, True):
            model = tiny_qwen2(torch.device("cuda"))
            assert M.use_int8_layers(model, lm_head=lm_head) == 2
            tri = M.TriAttention(model, from_bands(bands, model), max_new_tokens=12, module=module)
            ids = torch.randint(256, (1, prompt), generator=torch.Generator().manual_seed(prompt)).cuda()
            tokens.append(tri.generate(ids, 12, eos=set(), graph=graph))
        assert len(tokens[0]) == 12 and tokens[0] == tokens[1]
