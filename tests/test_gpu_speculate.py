"""A drafted tree through a whole (tiny, random) decoder stack: rotated at the nodes' positions, attended over the cache,
sampled at every node, accepted along a path -- the operators as they are used together."""
import math

import pytest
import torch

from lrqk_b200 import (DynamicLRQKCache, LightAttentionIndicesFactory, apply_rotary, patch_model, rotary_frequencies, run_task, sample_tokens,
                       tree_attention, tree_mask)

pytestmark = pytest.mark.gpu

PARENTS = [-1, 0, 0, 1, 1, 2, 4]
DEPTH = [0, 1, 1, 2, 2, 2, 3]


def _stack(dtype=torch.bfloat16, **scaling):
    import transformers
    cfg = transformers.LlamaConfig(vocab_size=500, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
                                   num_key_value_heads=2, head_dim=64, max_position_embeddings=4096, **scaling)
    cfg._attn_implementation = "sdpa"
    torch.manual_seed(5)
    return transformers.AutoModelForCausalLM.from_config(cfg).to(dtype).cuda().eval()


def _cache(k=256, m=64, **kw):
    return DynamicLRQKCache(r=16, num_active_tokens=k, lite_tokens=m, max_sequence_length=1024, num_key_value_groups=2, init_aq_ak_method="top", **kw)


def _path(node):
    out = []
    while node >= 0:
        out.append(node)
        node = PARENTS[node]
    return out[::-1]


@pytest.mark.parametrize("fused_rotary", [False, True])
def test_draft_verify_accept(fused_rotary):
    """With every token resident the drafted rows are full attention: fp32 logits equal the plain model's on each path,
    and decoding on from the accepted path equals decoding those tokens one by one."""
    model, S = _stack(torch.float32), 290
    ids = torch.randint(0, 500, (1, S), generator=torch.Generator().manual_seed(1)).cuda()
    draft = torch.randint(0, 500, (1, len(PARENTS)), generator=torch.Generator().manual_seed(2)).cuda()
    with torch.no_grad():
        plain = [model(input_ids=torch.cat([ids, draft[:, _path(i)]], 1), use_cache=False).logits[0, -1] for i in range(len(PARENTS))]
        plain_next = model(input_ids=torch.cat([ids, draft[:, _path(4)], draft[:, :1]], 1), use_cache=False).logits[0, -1]
        patch_model(model, fused_rotary=fused_rotary)
        cache = _cache()
        model(input_ids=ids, past_key_values=cache, use_cache=True)
        positions = torch.tensor([[S + d for d in DEPTH]], device="cuda")
        with cache.drafting(tree_mask(PARENTS, "cuda")):
            logits = model(input_ids=draft, position_ids=positions, past_key_values=cache, use_cache=True).logits
        assert cache.get_seq_length() == S                             # nothing decoded yet
        # two layers of fp32 sums of a few hundred terms in other orders (2^-24 each, on values of size one); the model's own
        # angles are fp32 (300 rad: 2^-16 off), the fused ones exact: allow for that where they differ
        tol = 2e-3 if fused_rotary else 2e-4
        for i in range(len(PARENTS)):
            assert torch.allclose(logits[0, i], plain[i], atol=tol, rtol=tol), i
        tokens, logprobs = sample_tokens(logits[0], torch.rand(len(PARENTS), generator=torch.Generator().manual_seed(3)).cuda(), temperature=0.8,
                                         top_k=50, top_p=0.9)
        assert tokens.shape == (len(PARENTS),) and bool((logprobs <= 0).all())
        kept = torch.topk(logits[0], 50).indices
        assert all(int(tokens[i]) in kept[i].tolist() for i in range(len(PARENTS)))
        cache.accept(_path(4))
        assert cache.get_seq_length() == S + 3
        step = model(input_ids=draft[:, :1], past_key_values=cache, use_cache=True).logits[0, -1]
        assert torch.allclose(step, plain_next, atol=tol, rtol=tol)
        one = _cache()
        model(input_ids=ids, past_key_values=one, use_cache=True)
        for t in _path(4):
            model(input_ids=draft[:, t:t + 1], past_key_values=one, use_cache=True)
        for a, b in zip(cache.lwattn.values(), one.lwattn.values()):
            n = S + 3
            assert torch.allclose(a.state.K_res[:, :, :n], b.state.K_res[:, :, :n], atol=tol, rtol=tol)
            assert torch.allclose(a.state.V_res[:, :, :n], b.state.V_res[:, :, :n], atol=tol, rtol=tol)
        cache.close()
        one.close()


def test_drafts_of_a_selecting_layer_attend_the_resident_rows():
    g = torch.Generator(device="cuda").manual_seed(4)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()  # noqa: E731
    fac = LightAttentionIndicesFactory(num_lite_tokens=8, attn_topk=64, num_key_value_groups=4, r=16, init_aq_ak_method="top", capacity=1024)
    q, k, v = r(2, 8, 700, 128), r(2, 2, 700, 128), r(2, 2, 700, 128)
    with pytest.raises(RuntimeError):
        fac.attend_tree(q[:, :, :3], k[:, :, :3], v[:, :, :3])
    fac.prefill(q, k, v)
    mask = tree_mask(PARENTS, "cuda")
    for step in range(3):
        tq, tk, tv = r(2, 8, 7, 128), r(2, 2, 7, 128), r(2, 2, 7, 128)
        before = [t.clone() for t in (fac.state.K_res, fac.state.V_res, fac.state.table, fac.state.A_K)]
        out = fac.attend_tree(tq, tk, tv, mask)
        K, V = fac.state.K_res.double(), fac.state.V_res.double()
        assert K.shape[2] == 72
        for h in range(8):
            kk, vv = torch.cat((K[:, h], tk[:, h // 4].double()), 1), torch.cat((V[:, h], tv[:, h // 4].double()), 1)
            s = (tq[:, h].double() @ kk.transpose(1, 2) / math.sqrt(128)).masked_fill(
                ~torch.cat((torch.ones(7, 72, dtype=torch.bool, device="cuda"), mask), 1), -math.inf)
            want = torch.softmax(s, -1) @ vv
            # one rounding to bf16 (half a step) on top of fp32 sums over 79 keys
            assert bool(((out[:, h].double() - want).abs() <= want.abs() * 2.0 ** -8 + 2.0 ** -14).all())
        assert all(torch.equal(a, b) for a, b in zip(before, (fac.state.K_res, fac.state.V_res, fac.state.table, fac.state.A_K)))
        fac.decode_attend(r(2, 8, 1, 128), r(2, 2, 1, 128), r(2, 2, 1, 128))
    fac.close()


def test_draft_protocol_is_checked():
    cache = _cache()
    x = torch.zeros(1, 4, 2, 64, device="cuda")
    with pytest.raises(RuntimeError):
        cache.attend_tree(x, x, x, 0)
    with pytest.raises(RuntimeError):
        cache.accept([0])
    with cache.drafting():
        assert cache.is_drafting
        with pytest.raises(RuntimeError):
            with cache.drafting():
                pass
        with pytest.raises(RuntimeError):
            cache.attend_tree(x, x, x, 0)                              # the layer has no prompt yet
        with pytest.raises(RuntimeError):
            cache.accept([0])
    assert not cache.is_drafting
    model = _stack()
    patch_model(model)
    ids = torch.randint(0, 500, (1, 270), generator=torch.Generator().manual_seed(1)).cuda()
    with torch.no_grad():
        model(input_ids=ids, past_key_values=cache, use_cache=True)
        with pytest.raises(NotImplementedError):
            model(input_ids=ids[:, :3], past_key_values=cache, use_cache=True)
        with cache.drafting():
            model(input_ids=ids[:, :3], past_key_values=cache, use_cache=True)
    for bad in ([3], [-1], [1, 1], [2, 0]):
        with pytest.raises(ValueError):
            cache.accept(bad)
    cache.accept([0, 1])
    with pytest.raises(RuntimeError):
        cache.accept([0])
    with torch.no_grad():
        with cache.drafting():
            model(input_ids=ids[:, :3], past_key_values=cache, use_cache=True)
        model(input_ids=ids[:, :1], past_key_values=cache, use_cache=True)   # a token decoded in between
        with pytest.raises(RuntimeError):
            cache.accept([0])
        with pytest.raises(KeyError):
            with cache.drafting():
                model(input_ids=ids[:, :3], past_key_values=cache, use_cache=True)
                raise KeyError
        with pytest.raises(RuntimeError):
            cache.accept([0])                                          # a draft that was broken off
    cache.close()


@pytest.mark.parametrize("scaling", [dict(), dict(rope_parameters={"rope_type": "yarn", "rope_theta": 1e6, "factor": 4.0, "original_max_position_embeddings": 1024}),
                                     dict(rope_parameters={"rope_type": "llama3", "rope_theta": 5e5, "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
                                                           "original_max_position_embeddings": 1024})])
def test_fused_rotary_follows_the_models_frequencies(scaling):
    model = _stack(torch.float32, **scaling)
    own = model.model.rotary_emb
    p = dict(scaling.get("rope_parameters", {}))
    inv, factor = rotary_frequencies(64, p.get("rope_theta", model.config.rope_parameters["rope_theta"]), p or None, device="cuda")
    # the module's frequencies are fp32 powers: a few units of 2^-24
    assert torch.allclose(own.inv_freq.double(), inv, rtol=2e-6, atol=0) and math.isclose(own.attention_scaling, factor, rel_tol=1e-6)
    ids = torch.randint(0, 500, (2, 300), generator=torch.Generator().manual_seed(1)).cuda()
    with torch.no_grad():
        plain = model(input_ids=ids, use_cache=False).logits
        patch_model(model, fused_rotary=True)
        cache = _cache()
        got = model(input_ids=ids, past_key_values=cache, use_cache=True).logits
        assert torch.allclose(got, plain, atol=2e-3, rtol=2e-3)
        cache.close()
        patch_model(model)                                             # and off again
        assert all(l.self_attn._lrqk_rotary is None for l in model.model.layers)


def test_throughput_driver_samples():
    model = _stack()
    for name in ("gpu_only", "lrqk_default"):
        if name != "gpu_only":
            patch_model(model)
        rec = run_task(name, model, r=16, num_active_tokens=128, lite_tokens=16, prompt_lens=(300,), max_new_tokens=4,
                       sampling=dict(temperature=0.7, top_k=40, top_p=0.95))
        assert rec["300"]["decode_tps"] > 0


def test_captured_step_of_the_operators():
    """Rotation, tree attention over a plain cache and sampling captured in one graph, replayed on new inputs and lengths."""
    g = torch.Generator(device="cuda").manual_seed(6)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()  # noqa: E731
    b, t, hq, hkv, d, cap, vocab = 2, 7, 8, 2, 128, 900, 3001
    q, k, v = r(b, t, hq, d).transpose(1, 2), r(b, t, hkv, d).transpose(1, 2), r(b, t, hkv, d).transpose(1, 2)
    ck, cv, head = r(b, hkv, cap, d), r(b, hkv, cap, d), r(hq * d, vocab) * 0.05
    lens = torch.tensor([900, 17], dtype=torch.int32, device="cuda")
    pos = lens[:, None].long() + torch.tensor(DEPTH, device="cuda")
    inv, _ = rotary_frequencies(d, 5e5, device="cuda")
    mask, u = tree_mask(PARENTS, "cuda"), torch.rand(b * t, generator=g, device="cuda")

    def step():
        q2, k2 = apply_rotary(q, k, pos, inv)
        out = tree_attention(q2, ck, cv, k2, v, mask, cache_lens=lens)
        logits = out.transpose(1, 2).reshape(b * t, hq * d) @ head
        return sample_tokens(logits, u, top_p=0.9)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tok, lp = step()
    q.copy_(r(b, hq, t, d))
    lens.copy_(torch.tensor([3, 640], dtype=torch.int32))
    pos.copy_(lens[:, None].long() + torch.tensor(DEPTH, device="cuda"))
    u.copy_(torch.rand(b * t, generator=g, device="cuda"))
    graph.replay()
    want = step()
    assert torch.equal(tok, want[0]) and torch.equal(lp, want[1])
