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


class _Layer:
    """A decoding layer that counts."""

    def __init__(self, fails=False):
        self.taken = []

    def attend_tree(self, q, k, v, mask):
        return torch.zeros_like(q)

    def _decode(self, q, k, v, attention):
        self.taken.append(float(q.flatten()[0]))

    def close(self):
        pass


def _drafted(mask, nodes, layers=2, batch=1):
    cache = _cache()
    cache.lwattn = {i: _Layer() for i in range(layers)}
    q = torch.arange(float(nodes))[None, None, :, None].expand(batch, 1, nodes, 16)
    for i in range(layers):
        cache.sequence_state[i] = DynamicLRQKCache.State.decoding
    with cache.drafting(mask):
        for i in range(layers):
            cache.attend_tree(q, q, q, i)
    return cache


PARENTS = [-1, 0, 0, 1, 1, 2, -1, 6]
PATHS = [[], [0], [0, 1], [0, 2], [0, 1, 4], [0, 2, 5], [6], [6, 7]]
NO_PATHS = [[1], [1, 2], [4], [0, 4], [0, 1, 2], [0, 1, 3, 4], [0, 6], [6, 0], [7], [0, 0], [5]]


@pytest.mark.parametrize("form", ["bool", "uint8", "per sequence"])
def test_accept_takes_paths_of_the_tree_only(form):
    mask = tree_mask(PARENTS)
    if form == "uint8":
        mask = mask.to(torch.uint8) * 5
    if form == "per sequence":
        mask = torch.stack([mask, mask])
    cache = _drafted(mask, len(PARENTS))
    for bad in NO_PATHS + [[0, 8], [-1]]:
        with pytest.raises(ValueError):
            cache.accept(bad)
    assert not cache.lwattn[0].taken and cache._drafted                 # refused before any layer changed, and still there
    for path in PATHS:
        cache = _drafted(mask, len(PARENTS))
        cache.accept(path)
        assert cache.lwattn[0].taken == cache.lwattn[1].taken == [float(i) for i in path]


def test_accept_of_a_chain_and_of_trees_that_differ():
    for nodes, good in (([0], True), ([0, 1, 2], True), ([1], False), ([0, 2], False)):
        cache = _drafted(None, 4)
        if good:
            cache.accept(nodes)
        else:
            with pytest.raises(ValueError):
                cache.accept(nodes)
    masks = tree_mask([[-1, 0, 0], [-1, 0, 1]])
    cache = _drafted(masks, 3, batch=2)
    with pytest.raises(ValueError, match="sequence 1"):
        cache.accept([0, 2])                                            # a path of the first sequence's tree alone
    cache.accept([0, 1])
    assert cache.lwattn[0].taken == [0.0, 1.0]


def test_a_mask_that_the_caller_reuses_is_the_drafts_own():
    mask = tree_mask([-1, 0, 0])
    cache = _drafted(mask, 3)
    mask.copy_(tree_mask([-1, 0, 1]))
    with pytest.raises(ValueError):
        cache.accept([0, 1, 2])
    cache.accept([0, 2])
    assert cache.lwattn[0].taken == [0.0, 2.0]


def test_a_draft_that_reached_some_layers_only_cannot_be_accepted():
    cache = _drafted(None, 3)
    q = torch.zeros(1, 1, 3, 16)
    with cache.drafting():
        cache.attend_tree(q, q, q, 0)
        try:
            raise KeyError("an error between two layers, caught inside")
        except KeyError:
            pass
    with pytest.raises(RuntimeError, match=r"\[1\]"):
        cache.accept([0])
    assert not cache.lwattn[0].taken


def test_a_draft_made_before_a_restore_cannot_be_accepted_onto_it():
    saved = _cache()
    x = torch.ones(1, 2, 5, 16)
    saved.update(torch.ones(1, 4, 5, 16), x, x, 0)
    sd = saved.state_dict()
    cache = _drafted(None, 3, layers=1)
    cache.load_state_dict(sd, device="cpu")
    with pytest.raises(RuntimeError, match="no drafted"):
        cache.accept([0])
    assert not cache.lwattn[0].taken
    other = _cache()
    with other.drafting():
        with pytest.raises(RuntimeError, match="drafting"):
            other.load_state_dict(sd, device="cpu")
    assert not other.temp_buff_cache_qkv


def test_check_status_and_close_look_at_the_tree_attentions_word(monkeypatch):
    from lrqk_b200 import _lib, lrqk_attention
    looked = []

    def look(device):
        looked.append(device)
        raise _lib.LrqkError(_lib.ETIMEOUT, "lrqk_tree_attention", "")

    monkeypatch.setattr(lrqk_attention, "check_tree_status", look, raising=False)
    monkeypatch.setattr(_Layer, "state", None, raising=False)
    _cache().check_status()                                             # no draft: nothing to look at
    assert not looked
    cache = _drafted(None, 3)
    for call in (cache.check_status, cache.close):
        with pytest.raises(_lib.LrqkError):
            call()
    assert looked == [torch.device("cpu")] * 2
