"""What a cache refuses around a draft, before anything is stored (no GPU: layers that still collect a short prompt, and stub
layers)."""
import pytest
import torch

from lrqk_b200 import DynamicLRQKCache, patch_model, tree_mask


def _cache(**kw):
    return DynamicLRQKCache(r=8, num_active_tokens=256, lite_tokens=16, num_key_value_groups=2, **kw)


def _model():
    import transformers
    cfg = transformers.LlamaConfig(vocab_size=100, hidden_size=64, intermediate_size=128, num_hidden_layers=2, num_attention_heads=4,
                                   num_key_value_heads=2, head_dim=16, max_position_embeddings=512)
    cfg._attn_implementation = "sdpa"
    torch.manual_seed(3)
    model = transformers.AutoModelForCausalLM.from_config(cfg).eval()
    patch_model(model)
    return model


def _buffers(cache):
    return {i: [x.tensor().clone() for x in (b.Q, b.K, b.V)] for i, b in cache.temp_buff_cache_qkv.items()}


@pytest.mark.parametrize("nodes", [1, 3, 216])          # (216 would fill the buffer and factorise the prompt)
def test_a_draft_on_a_layer_that_still_collects_is_refused_and_stores_nothing(nodes):
    model, cache = _model(), _cache()
    ids = torch.randint(0, 100, (1, 40), generator=torch.Generator().manual_seed(1))
    draft = torch.randint(0, 100, (1, nodes), generator=torch.Generator().manual_seed(2))
    with torch.no_grad():
        model(input_ids=ids, past_key_values=cache, use_cache=True)
        before, states = _buffers(cache), dict(cache.sequence_state)
        assert len(before) == 2 and before[0][1].shape[2] == 40
        with pytest.raises(RuntimeError, match="decoding"):
            with cache.drafting(tree_mask([-1] + [0] * (nodes - 1))):
                model(input_ids=draft, position_ids=torch.full((1, nodes), 41), past_key_values=cache, use_cache=True)
        after = _buffers(cache)
        assert all(torch.equal(a, b) for i in before for a, b in zip(before[i], after[i])) and dict(cache.sequence_state) == states
        with pytest.raises(RuntimeError, match="no drafted"):
            cache.accept([0])
        # and the context goes on as if nothing had been tried
        got = model(input_ids=draft[:, :1], past_key_values=cache, use_cache=True).logits
        other = _cache()
        model(input_ids=ids, past_key_values=other, use_cache=True)
        assert torch.equal(got, model(input_ids=draft[:, :1], past_key_values=other, use_cache=True).logits)


def test_a_draft_as_the_first_call_is_refused():
    model, cache = _model(), _cache()
    with torch.no_grad(), cache.drafting():
        with pytest.raises(RuntimeError, match="decoding"):
            model(input_ids=torch.zeros(1, 3, dtype=torch.int64), past_key_values=cache, use_cache=True)
    assert not cache.temp_buff_cache_qkv


def test_nothing_commits_a_token_while_a_draft_is_open():
    cache = _cache()
    q, k = torch.ones(1, 4, 5, 16), torch.ones(1, 2, 5, 16)
    with cache.drafting():
        for call in (lambda: cache.update(q, k, k, 0), lambda: cache.update(q, k, k, 0, torch.zeros(1, 5)), lambda: cache.attend(q[:, :, :1], k[:, :, :1], k[:, :, :1], 0),
                     lambda: cache.attend_qkv(torch.ones(1, 1, 8 * 16), q[:, 0, :1], q[:, 0, :1], 0, 4, 2)):
            with pytest.raises(RuntimeError, match="drafting"):
                call()
    assert bool((k == 1).all()) and not cache.temp_buff_cache_qkv
    cache.update(q, k, k, 0)
    assert len(cache.temp_buff_cache_qkv[0]) == 5
