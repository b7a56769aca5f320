"""Patched models with prompt_attention="exact": prompts, further turns behind a cache, and the graphed decoder, through the
models' own calls and with the masks that the host framework makes for them."""

from __future__ import annotations

import dataclasses

import pytest
import torch
from transformers import DynamicCache, LlamaConfig, LlamaForCausalLM, StaticCache

from sva_b200 import patch_llama_attention
from sva_b200.serving import GraphedGreedyDecoder
from tests.test_gpu_model_batch import _socket_bundle

pytestmark = pytest.mark.gpu


def _model(implementation, patched=True, batch=False, layers=(0, 1), dtype=torch.float32):
    torch.manual_seed(17)
    cfg = LlamaConfig(vocab_size=256, hidden_size=576, intermediate_size=256, num_hidden_layers=2, num_attention_heads=9,
                      num_key_value_heads=3, head_dim=64, max_position_embeddings=2048, attn_implementation=implementation)
    model = LlamaForCausalLM(cfg).eval().to(dtype).cuda()
    if patched:
        patch_llama_attention(model, _socket_bundle(), layers=list(layers), allow_batch=batch, prompt_attention="exact")
    return model


def _ids(batch, n, seed=3):
    return torch.randint(0, 256, (batch, n), generator=torch.Generator().manual_seed(seed)).cuda()


# fp32 models: both sides sum the same products in fp32 in other orders, and two layers' logits are of the order of 1
TOL = dict(rtol=1e-3, atol=1e-3)


@pytest.mark.parametrize("implementation", ["eager", "sdpa"])
@pytest.mark.parametrize("batch", [1, 2])
@pytest.mark.parametrize("with_mask", [False, True])
def test_turns_behind_a_growing_cache(implementation, batch, with_mask):
    """Three turns of several tokens: the logits are those of the unpatched model."""
    plain, exact = _model(implementation, patched=False), _model(implementation, batch=batch > 1)
    ids = _ids(batch, 200)
    caches = [DynamicCache(config=plain.config) for _ in range(2)]
    with torch.no_grad():
        for a, b in ((0, 120), (120, 150), (150, 200)):
            mask = torch.ones(batch, b, dtype=torch.long, device="cuda") if with_mask else None
            want, got = (m(input_ids=ids[:, a:b], attention_mask=mask, use_cache=True, past_key_values=c).logits
                         for m, c in zip((plain, exact), caches))
            torch.testing.assert_close(got, want, **TOL)
        assert caches[1].get_seq_length(0) == 200
        exact(input_ids=ids[:, :1], use_cache=True, past_key_values=caches[1])  # and a step that summons


@pytest.mark.parametrize("implementation", ["eager", "sdpa"])
def test_turns_behind_a_static_cache(implementation):
    plain, exact = _model(implementation, patched=False), _model(implementation)
    ids = _ids(1, 200)
    caches = [StaticCache(config=plain.config, max_cache_len=256) for _ in range(2)]
    with torch.no_grad():
        for a, b in ((0, 120), (120, 200)):
            want, got = (m(input_ids=ids[:, a:b], use_cache=True, past_key_values=c).logits for m, c in zip((plain, exact), caches))
            torch.testing.assert_close(got, want, **TOL)


@pytest.mark.parametrize("implementation", ["eager", "sdpa"])
def test_prompt_without_a_cache(implementation):
    plain, exact = _model(implementation, patched=False), _model(implementation)
    with torch.no_grad():
        want, got = (m(input_ids=_ids(1, 77), use_cache=False).logits for m in (plain, exact))
        torch.testing.assert_close(got, want, **TOL)


def test_graphed_decoder_prompts():
    """The prompt's token is the unpatched model's; the graphed steps then summon."""
    plain, exact = _model("sdpa", patched=False), _model("sdpa", batch=True)
    ids = _ids(2, 90)
    with torch.no_grad():
        want = plain(input_ids=ids).logits[:, -1].argmax(-1)
    decoder = GraphedGreedyDecoder(exact, 2, 128)
    toks = decoder.generate(ids, 6)
    decoder.release()
    assert toks.shape == (2, 6) and torch.equal(toks[:, 0], want)


@pytest.mark.parametrize("implementation", ["eager", "sdpa"])
def test_masks_that_hide_keys_are_refused(implementation):
    exact = _model(implementation, batch=True)
    padded = torch.ones(2, 40, dtype=torch.long, device="cuda")
    padded[1, :7] = 0
    with torch.no_grad(), pytest.raises(ValueError, match="attention mask"):
        exact(input_ids=_ids(2, 40), attention_mask=padded, use_cache=False)


@pytest.mark.parametrize("implementation", ["eager", "sdpa"])
def test_a_refused_prompt_leaves_the_cache_as_it_was(implementation):
    plain, exact = _model(implementation, patched=False), _model(implementation, layers=(0,))
    ids = _ids(1, 60)
    hole = torch.ones(1, 50, dtype=torch.long, device="cuda")
    hole[0, 10] = 0
    cache, other = DynamicCache(config=plain.config), DynamicCache(config=plain.config)
    with torch.no_grad():
        exact(input_ids=ids[:, :30], use_cache=True, past_key_values=cache)
        with pytest.raises(ValueError, match="attention mask"):
            exact(input_ids=ids[:, 30:50], attention_mask=hole, use_cache=True, past_key_values=cache)
        assert [cache.get_seq_length(i) for i in range(2)] == [30, 30]
        got = exact(input_ids=ids[:, 30:50], use_cache=True, past_key_values=cache).logits
        plain(input_ids=ids[:, :30], use_cache=True, past_key_values=other)
        torch.testing.assert_close(got, plain(input_ids=ids[:, 30:50], use_cache=True, past_key_values=other).logits, **TOL)
        attention = exact.model.layers[0].self_attn
        attention.serving = dataclasses.replace(attention.serving, prompt_attention="everything")
        for cache in (cache, StaticCache(config=plain.config, max_cache_len=64)):
            before = int(cache.get_seq_length(0))
            with pytest.raises(ValueError, match="prompt_attention"):
                exact(input_ids=ids[:, 50:], use_cache=True, past_key_values=cache)
            assert int(cache.get_seq_length(0)) == before
