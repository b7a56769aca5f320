"""Patched layers with prompt_attention="exact": prompts attend to every key, decode steps summon as before."""

from __future__ import annotations

import pytest
import torch
from transformers import LlamaConfig
from transformers.models.llama.modeling_llama import LlamaAttention

from sva_b200 import SVALayerArtifacts, SVALlamaAttention, SVALlamaServingConfig

pytestmark = pytest.mark.gpu

H, HKV, D = 9, 3, 64


def _module(prompt_attention, allow_batch=False, mode="scan"):
    cfg = LlamaConfig(hidden_size=H * D, num_attention_heads=H, num_key_value_heads=HKV, head_dim=D,
                      intermediate_size=64, num_hidden_layers=1, vocab_size=16)
    gen = torch.Generator().manual_seed(3)
    arts = SVALayerArtifacts(torch.randn(H, D, 64, generator=gen) * 0.125, torch.randn(H, D, 64, generator=gen) * 0.125,
                             torch.randn(H, generator=gen) * 0.1, torch.randn(H, 2, 64, 32, generator=gen), 0.0, 0.0, "qk")
    serving = SVALlamaServingConfig(rank_dim=64, coarse_shortlist=64, budget=16, allow_batch=allow_batch, summon_mode=mode,
                                    prompt_attention=prompt_attention)
    return SVALlamaAttention(LlamaAttention(cfg, 0), arts, serving, None).cuda().eval()


def _qkv(batch, q_len, k_len, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(batch, h, n, D, generator=gen).to(dtype).cuda() for h, n in ((H, q_len), (HKV, k_len), (HKV, k_len))]


def _full(q, k, v):
    """Attention over every key in 64 bits, causal and aligned at the end."""
    q, k, v = q.double(), k.double().repeat_interleave(H // HKV, 1), v.double().repeat_interleave(H // HKV, 1)
    rows, keys = q.shape[2], k.shape[2]
    seen = torch.arange(keys, device=q.device) <= torch.arange(rows, device=q.device)[:, None] + keys - rows
    return (q @ k.transpose(2, 3) * D ** -0.5).masked_fill(~seen, float("-inf")).softmax(-1) @ v


# a weight of 1 in all, each term rounded once for the product and the sum once for the output (2^-8 each), values below 4.5
TOL = {torch.bfloat16: 2 * 2.0 ** -8 * 4.5, torch.float32: 1e-4}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("mode", ["scan", "inverted", "inverted_static"])
def test_prompt_is_exact_and_decode_summons(mode, dtype):
    exact, summon = _module("exact", mode=mode), _module("summon", mode=mode)
    q, k, v = _qkv(1, 200, 204, dtype)
    with torch.no_grad():
        out = exact.sva_attention(q, k[:, :, :200], v[:, :, :200], None)
        assert (out.double() - _full(q, k[:, :, :200], v[:, :, :200])).abs().max() <= TOL[dtype]
        summon.sva_attention(q, k[:, :, :200], v[:, :, :200], None)
        # a second chunk of three tokens, then a single one: the catalogs agree, so the decode step does
        for a, b in ((200, 203), (203, 204)):
            got, want = (m.sva_attention(q[:, :, :b - a], k[:, :, :b], v[:, :, :b], None) for m in (exact, summon))
            if b - a > 1:
                assert (got.double() - _full(q[:, :, :b - a], k[:, :, :b], v[:, :, :b])).abs().max() <= TOL[dtype]
            else:
                assert torch.equal(got, want)


def test_batched_and_static_cache_prompts():
    q, k, v = _qkv(3, 70, 70, torch.bfloat16, seed=1)
    want = _full(q, k, v)
    m = _module("exact", allow_batch=True)
    with torch.no_grad():
        assert (m.sva_attention(q, k, v, None).double() - want).abs().max() <= TOL[torch.bfloat16]
        padded = [torch.cat([x, torch.full_like(x[:, :, :30], float("nan"))], 2) for x in (k, v)]
        pos = torch.arange(70, device="cuda")[None]
        static = _module("exact", allow_batch=True).sva_attention_static(q, *padded, pos)
        assert (static.double() - want).abs().max() <= TOL[torch.bfloat16]


def test_refusals():
    q, k, v = _qkv(1, 5, 5, torch.bfloat16)
    mask = torch.zeros(1, 1, 5, 5, device="cuda")
    with pytest.raises(ValueError, match="attention mask"):
        _module("exact").sva_attention(q, k, v, mask)
    with pytest.raises(ValueError, match="prompt_attention"):
        _module("everything").sva_attention(q, k, v, None)
    with torch.no_grad():
        _module("exact").sva_attention(q[:, :, :1], k, v, torch.zeros(1, 1, 1, 5, device="cuda"))  # a decode step may have one
