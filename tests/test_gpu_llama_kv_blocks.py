"""The decoder with its KV cache in Q4_0 or Q8_0 blocks: against dense math over what the blocks stand for, against itself (prefill and
decode, eager and replayed), and what the blocks of a first layer hold."""
import dataclasses

import pytest
import torch
import torch.nn.functional as F

from xn_b200 import GgmlDType

pytestmark = pytest.mark.gpu

FORMATS = [GgmlDType.Q4_0, GgmlDType.Q8_0]


def _rel(a, b):
    return float((a - b).norm() / b.norm())


def _tokens(batch, n, seed):
    g = torch.Generator(device="cpu")
    g.manual_seed(seed)
    return torch.randint(0, 512, (batch, n), generator=g).to("cuda:0")


def _model(kv_dtype, batch, max_seq=256, heads=(4, 2, 128), rows=512, **kw):
    from xn_b200.llama import LlamaConfig, QLlama
    cfg = dataclasses.replace(LlamaConfig.tiny(), n_heads=heads[0], n_kv_heads=heads[1], head_dim=heads[2])
    return QLlama(cfg, torch.device("cuda", 0), batch=batch, max_seq=max_seq, max_prefill_rows=rows, kv_dtype=kv_dtype, **kw)


def _dense_over_blocks(m, tokens):
    """The network in f32 on the dequantized weights, every layer attending to the keys and values its cache's blocks stand for."""
    c, hd = m.cfg, m.cfg.head_dim
    B, S = tokens.shape
    x = m.embed.index_select(0, tokens.reshape(-1)).view(B, S, -1).float()
    causal = torch.ones(S, S, device=m.device, dtype=torch.bool).tril()
    for L in m.layers:
        q = (m._rms(x, L.norm1) @ L.wqkv.dequantize(torch.float32).T)[..., :c.n_heads * hd]
        q = m._rope(q.view(B, S, c.n_heads, hd).transpose(1, 2), m.cos[:S], m.sin[:S])
        k, v = L.kv.load(0, S, torch.float32)
        a = F.scaled_dot_product_attention(q, k, v, attn_mask=causal, enable_gqa=True)
        x = x + a.transpose(1, 2).reshape(B, S, -1) @ L.wo.dequantize(torch.float32).T
        gate, up = (m._rms(x, L.norm2) @ L.wgu.dequantize(torch.float32).T).split(c.ffn, dim=-1)
        x = x + (F.silu(gate) * up) @ L.wdown.dequantize(torch.float32).T
    return (m._rms(x[:, -1:, :], m.norm) @ m.lm_head.dequantize(torch.float32).T).view(B, -1)


@pytest.mark.parametrize("dt", FORMATS)
@pytest.mark.parametrize("S", [1, 12, 130])
@pytest.mark.parametrize("heads", [(4, 2, 128), (8, 2, 64)])
def test_prefill_matches_dense_math_over_its_blocks(dt, S, heads):
    m = _model(dt, batch=2, heads=heads)
    prompt = _tokens(2, S, 11)
    logits = m.prefill(prompt)
    # 8-bit activation blocks and bf16 queries against f32, as for the bf16 cache: the blocks themselves are given
    assert _rel(logits, _dense_over_blocks(m, prompt)) < 3e-2


@pytest.mark.parametrize("dt,bound", [(GgmlDType.Q4_0, 0.12), (GgmlDType.Q8_0, 0.01)])
def test_a_first_layer_holds_the_keys_and_values_of_the_bf16_cache(dt, bound):
    """The largest of 32 normal values is about 2.1 sigma: a step of 2.1 / 8 (2.1 / 127), an error of that over sqrt(12): 0.076 (0.0048), and bf16's 0.0017."""
    blocks, rows = _model(dt, batch=2), _model(None, batch=2)
    prompt = _tokens(2, 40, 12)
    blocks.prefill(prompt), rows.prefill(prompt)
    k, v = blocks.layers[0].kv.load(0, 40, torch.float32)
    assert _rel(k, rows.layers[0].k_cache[:, :, :40].float()) < bound
    assert _rel(v, rows.layers[0].v_cache[:, :, :40].float()) < bound
    # 32 values in 18 bytes (34), 64 in bf16; whole tiles of 32 positions either way here
    assert blocks.layers[0].kv.nbytes * 64 == 2 * rows.layers[0].k_cache.numel() * 2 * {GgmlDType.Q4_0: 18, GgmlDType.Q8_0: 34}[dt]


# A step's keys and values may differ from the prompt's by the activations' rounding, which moves some codes by one: a step of the format
@pytest.mark.parametrize("dt,bound", [(GgmlDType.Q4_0, 5e-2), (GgmlDType.Q8_0, 2e-2)])
@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("heads", [(4, 2, 128), (8, 2, 64)])
def test_a_decode_step_is_the_prefill_of_the_longer_prompt(dt, bound, fused, heads):
    prompt = _tokens(2, 33, 13)
    m = _model(dt, batch=2, heads=heads, fused_decode=fused)
    m.prefill(prompt)
    longer = torch.cat([prompt, m.tokens[:, None]], dim=1)
    m._decode_step()
    assert _rel(m.last_logits, _model(dt, batch=2, heads=heads).prefill(longer)) < bound


@pytest.mark.parametrize("dt", FORMATS)
@pytest.mark.parametrize("batch", [1, 3])
def test_replayed_steps_generate_what_eager_steps_do(dt, batch):
    prompt = _tokens(batch, 30, 14)
    made = []
    for graph in (False, True):
        m = _model(dt, batch=batch, max_seq=64)
        m.prefill(prompt)
        if graph:
            m.capture_decode()
        made.append((m.decode(10), m.last_logits.clone(), m.layers[-1].kv.pages.clone()))
    assert all(torch.equal(a, b) for a, b in zip(*made))


def test_a_format_that_no_cache_has_is_refused():
    with pytest.raises(ValueError, match="Q4_0 or Q8_0"):
        _model(GgmlDType.Q4K, batch=1)
