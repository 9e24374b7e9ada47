"""What is measured of the operators around a drafted step of a long-context model: rotary positions, attention of a tree of
drafted tokens over a cache, and the choice of tokens from logits.

``run`` computes each case in its plain form (elementary torch operations in 32 or 64 bits) where ``own`` is false, and calls
``lrqk_b200`` where it is true.  ``exact`` is the same from the definition in 64 bits.
"""
import math

import torch

own = False

HEADS = ((32, 8), (28, 4), (40, 8), (8, 2))          # (query heads, key/value heads)
VOCABS = (128256, 152064)
ROTARY_MOST = 32 * 65536 * 128                        # query elements of the largest rotary case
TREE_MOST_KEYS = 2 * 8 * 131072                       # cache rows (over sequences and heads) of the largest tree case
TREE_MOST_WORK = 2 * 32 * 64 * 131072                 # query rows times keys of the largest tree case
SAMPLE_MOST = 64 * 152064


def listed():
    return [
        # one new token of each of four sequences, far into a context stretched by frequency bands
        dict(name="rotary step", op="rotary", dtype="bf16", batch=4, length=1, q_heads=32, kv_heads=8, head_dim=128, part=128,
             interleaved=False, adjoint=False, scaling="llama3", base=500000.0, start=131071),
        # the queries and keys of a long prompt as the projections leave them ([batch, token, head, dim]), YaRN frequencies
        dict(name="rotary prompt", op="rotary", dtype="bf16", batch=1, length=65536, q_heads=32, kv_heads=8, head_dim=128, part=128,
             interleaved=False, adjoint=False, scaling="yarn", base=1000000.0, start=0),
        # the gradient of the rotation, neighbouring pairs, half of each head, an odd length in 32 bits
        dict(name="rotary gradient", op="rotary", dtype="f32", batch=2, length=1537, q_heads=28, kv_heads=4, head_dim=128, part=64,
             interleaved=True, adjoint=True, scaling="linear", base=10000.0, start=7),
        # eight drafted tokens over a short context: launch latency
        dict(name="tree short", op="tree", dtype="bf16", batch=1, q_heads=32, cache_heads=8, kv_heads=8, head_dim=128, nodes=8,
             capacity=1100, ragged=False),
        # a batch of sequences of very different lengths (an empty cache among them), an odd number of nodes
        dict(name="tree ragged", op="tree", dtype="bf16", batch=6, q_heads=28, cache_heads=4, kv_heads=4, head_dim=128, nodes=25,
             capacity=20011, ragged=True),
        # 64 nodes over two full contexts: the largest
        dict(name="tree long", op="tree", dtype="bf16", batch=2, q_heads=32, cache_heads=8, kv_heads=8, head_dim=128, nodes=64,
             capacity=131072, ragged=False),
        # the resident rows of a decoding layer: every query head keeps keys of its own, drafted keys are shared
        dict(name="tree resident", op="tree", dtype="bf16", batch=1, q_heads=32, cache_heads=32, kv_heads=8, head_dim=128, nodes=16,
             capacity=2112, ragged=False),
        # 32-bit states, a wide tree
        dict(name="tree f32", op="tree", dtype="f32", batch=1, q_heads=8, cache_heads=2, kv_heads=2, head_dim=128, nodes=33,
             capacity=4096, ragged=False),
        # one sequence, the usual filters
        dict(name="sample one", op="sample", dtype="bf16", rows=1, vocab=128256, top_k=50, top_p=0.9, min_p=0.0, temperature=0.7,
             mixed=False),
        # the nodes of one tree, a nucleus and a floor
        dict(name="sample nodes", op="sample", dtype="bf16", rows=25, vocab=128256, top_k=0, top_p=0.95, min_p=0.02, temperature=1.0,
             mixed=False),
        # a batch whose requests each have settings of their own (greedy and unfiltered ones among them), logits in 32 bits
        dict(name="sample batch", op="sample", dtype="f32", rows=64, vocab=152064, top_k=40, top_p=0.8, min_p=0.05, temperature=1.3,
             mixed=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(("rotary", "tree", "tree", "sample"))
    dtype = rng.choice(("bf16", "bf16", "f32"))
    hq, hkv = rng.choice(HEADS)
    if op == "rotary":
        d = rng.choice((64, 128))
        b = rng.choice((1, 1, 2, 3, 8))
        length = _log_int(rng, 1, max(1, ROTARY_MOST // (b * hq * d * (1 if dtype == "bf16" else 2)) - 1))
        return dict(op=op, dtype=dtype, batch=b, length=min(length, 65536), q_heads=hq, kv_heads=hkv, head_dim=d,
                    part=rng.choice((d, d, d // 2, 3 * d // 4)), interleaved=rng.random() < 0.4, adjoint=rng.random() < 0.3,
                    scaling=rng.choice(("none", "linear", "ntk", "yarn", "llama3")), base=rng.choice((10000.0, 500000.0, 1000000.0)),
                    start=_log_int(rng, 1, 1000000))
    if op == "tree":
        b = rng.choice((1, 1, 2, 4, 7))
        nodes = _log_int(rng, 1, 64)
        own_rows = rng.random() < 0.25
        hc = hq if own_rows else hkv
        most = min(TREE_MOST_KEYS // (b * hc), TREE_MOST_WORK // (b * hq * nodes), 131072)
        if dtype == "f32":
            most = max(16, most // 64)
        return dict(op=op, dtype=dtype, batch=b, q_heads=hq, cache_heads=hc, kv_heads=hkv, head_dim=rng.choice((64, 128, 128)),
                    nodes=nodes, capacity=_log_int(rng, 1, most - 1), ragged=rng.random() < 0.4)
    rows = _log_int(rng, 1, 64)
    vocab = rng.choice(VOCABS) if rng.random() < 0.5 else _log_int(rng, 1000, min(200000, SAMPLE_MOST // rows))
    return dict(op=op, dtype=dtype, rows=min(rows, SAMPLE_MOST // vocab), vocab=vocab, top_k=rng.choice((0, 0, 1, 20, 50, 1000)),
                top_p=rng.choice((1.0, 0.5, 0.9, 0.95, 0.99)), min_p=rng.choice((0.0, 0.0, 0.02, 0.1)),
                temperature=round(rng.uniform(0.3, 1.6), 3), mixed=rng.random() < 0.3)


def _type(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---- rotary positions -------------------------------------------------------------------------------------------------------
def _frequencies(case):
    """Angular frequency of each pair, in 64 bits, and the factor on cosine and sine."""
    n, base = case["part"] // 2, case["base"]
    exponent = torch.arange(n, dtype=torch.float64) / n
    freq, kind = base ** -exponent, case["scaling"]
    if kind == "linear":
        return freq / 4.0, 1.0
    if kind == "ntk":
        return (base * 8.0 ** (n / max(1, n - 1))) ** -exponent, 1.0
    if kind == "yarn":          # trained on 32768 tokens, stretched fourfold: slow pairs interpolated, fast ones left, a ramp between
        index = lambda r: n * math.log(32768 / (r * 2 * math.pi)) / math.log(base)  # noqa: E731 - the pair that turns r times
        low, high = max(math.floor(index(32.0)), 0), min(math.ceil(index(1.0)), 2 * n - 1)
        ramp = ((torch.arange(n, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0, 1)
        return freq / 4.0 * ramp + freq * (1 - ramp), 0.1 * math.log(4.0) + 1.0
    if kind == "llama3":        # trained on 8192 tokens, stretched eightfold, bands by wavelength
        turns = 8192 * freq / (2 * math.pi)
        smooth = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return freq / 8.0 * (1 - smooth) + freq * smooth, 1.0
    return freq, 1.0


def _prepare_rotary(case, g):
    b, n, d, t = case["batch"], case["length"], case["head_dim"], _type(case)
    q = torch.randn(b, n, case["q_heads"], d, generator=g, device="cuda", dtype=t).transpose(1, 2)
    k = torch.randn(b, n, case["kv_heads"], d, generator=g, device="cuda", dtype=t).transpose(1, 2)
    positions = case["start"] + torch.arange(n, device="cuda") + torch.randint(0, 64, (b, 1), generator=g, device="cuda")
    freq, factor = _frequencies(case)
    return dict(case=case, q=q, k=k, positions=positions, freq=freq.cuda(), factor=factor)


def _turned(x, cos, sin, part, interleaved):
    y = x.to(torch.float32)
    a, b = (y[..., 0:part:2], y[..., 1:part:2]) if interleaved else (y[..., :part // 2], y[..., part // 2:part])
    u, v = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((u, v), -1).flatten(-2) if interleaved else torch.cat((u, v), -1)
    return torch.cat((turned, y[..., part:]), -1).to(x.dtype)


def _run_rotary(s):
    case = s["case"]
    if own:
        from lrqk_b200 import apply_rotary
        return apply_rotary(s["q"], s["k"], s["positions"], s["freq"], factor=s["factor"], interleaved=case["interleaved"],
                            adjoint=case["adjoint"])
    angle = s["positions"].to(torch.float64)[:, None, :, None] * s["freq"]
    cos, sin = (torch.cos(angle) * s["factor"]).to(torch.float32), (torch.sin(angle) * s["factor"]).to(torch.float32)
    sin = -sin if case["adjoint"] else sin
    return _turned(s["q"], cos, sin, case["part"], case["interleaved"]), _turned(s["k"], cos, sin, case["part"], case["interleaved"])


def _exact_rotary(case, s):
    part, out = case["part"], []
    angle = s["positions"].double()[:, :, None] * s["freq"]
    wheel = torch.polar(torch.full_like(angle, s["factor"]), -angle if case["adjoint"] else angle)
    for x in (s["q"], s["k"]):
        heads = []
        for h in range(x.shape[1]):
            y = x[:, h].double()
            if case["interleaved"]:
                y[..., :part] = torch.view_as_real(torch.view_as_complex(y[..., :part].unflatten(-1, (-1, 2)).contiguous()) * wheel).flatten(-2)
            else:
                z = torch.complex(y[..., :part // 2].contiguous(), y[..., part // 2:part].contiguous()) * wheel
                y[..., :part] = torch.cat((z.real, z.imag), -1)
            heads.append(y)
        out.append(torch.stack(heads, 1))
    return tuple(out)


# ---- attention of a tree of drafted tokens -----------------------------------------------------------------------------------
def _lengths(case):
    b, s = case["batch"], case["capacity"]
    if not case["ragged"] or b == 1:
        return [s - s // 11] * b
    return [s - (s * i) // (b - 1) if i != b - 2 or b < 4 else 1 for i in range(b)]


def _prepare_tree(case, g):
    b, t, d, s, dt = case["batch"], case["nodes"], case["head_dim"], case["capacity"], _type(case)
    z = dict(generator=g, device="cuda", dtype=dt)
    q = torch.randn(b, t, case["q_heads"], d, **z).transpose(1, 2)
    cache_k, cache_v = torch.randn(b, case["cache_heads"], s, d, **z), torch.randn(b, case["cache_heads"], s, d, **z)
    tree_k = torch.randn(b, t, case["kv_heads"], d, **z).transpose(1, 2)
    tree_v = torch.randn(b, t, case["kv_heads"], d, **z).transpose(1, 2)
    # parents at random among the earlier nodes; a node sees itself and its ancestors (the path doubled until it reaches the root)
    parent = (torch.rand(b, t, generator=g, device="cuda") * torch.arange(t, device="cuda")).long()
    step = torch.nn.functional.one_hot(parent, t).float()
    step[:, 0] = 0
    mask = torch.eye(t, device="cuda") + step
    for _ in range(max(1, t.bit_length())):
        mask = (mask @ mask).clamp(max=1.0)
    return dict(case=case, q=q, cache_k=cache_k, cache_v=cache_v, tree_k=tree_k, tree_v=tree_v, mask=mask > 0,
                lengths=torch.tensor(_lengths(case), dtype=torch.int32, device="cuda"))


def _run_tree(s):
    if own:
        from lrqk_b200 import tree_attention
        return tree_attention(s["q"], s["cache_k"], s["cache_v"], s["tree_k"], s["tree_v"], s["mask"], cache_lens=s["lengths"])
    q, hc = s["q"], s["cache_k"].shape[1]
    b, hq, t, d = q.shape
    hkv, cap = s["tree_k"].shape[1], s["cache_k"].shape[2]
    q32 = q.to(torch.float32) * d ** -0.5
    near = q32.reshape(b, hkv, -1, d) @ s["tree_k"].to(torch.float32).transpose(-1, -2)
    near = near.reshape(b, hq, t, t).masked_fill(~s["mask"][:, None], float("-inf"))
    far = (q32.reshape(b, hc, -1, d) @ s["cache_k"].to(torch.float32).transpose(-1, -2)).reshape(b, hq, t, cap)
    behind = torch.arange(cap, device=q.device) >= s["lengths"][:, None, None, None]
    far.masked_fill_(behind, float("-inf"))
    top = torch.maximum(far.amax(-1, keepdim=True), near.amax(-1, keepdim=True))
    far, near = far.sub_(top).exp_(), (near - top).exp()
    total = far.sum(-1, keepdim=True) + near.sum(-1, keepdim=True)
    out = (far.reshape(b, hc, -1, cap) @ s["cache_v"].to(torch.float32)).reshape(b, hq, t, d)
    out = out + (near.reshape(b, hkv, -1, t) @ s["tree_v"].to(torch.float32)).reshape(b, hq, t, d)
    return (out / total).to(q.dtype)


def _exact_tree(case, s):
    q, d = s["q"], case["head_dim"]
    out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lengths(case)):
        for h in range(case["q_heads"]):
            hc, hk = h * case["cache_heads"] // case["q_heads"], h * case["kv_heads"] // case["q_heads"]
            k = torch.cat((s["cache_k"][b, hc, :n], s["tree_k"][b, hk])).double()
            v = torch.cat((s["cache_v"][b, hc, :n], s["tree_v"][b, hk])).double()
            seen = torch.cat((torch.ones(case["nodes"], n, dtype=torch.bool, device="cuda"), s["mask"][b]), 1)
            score = (q[b, h].double() @ k.T / math.sqrt(d)).masked_fill(~seen, -math.inf)
            out[b, h] = torch.exp(score - torch.logsumexp(score, -1, keepdim=True)) @ v
    return out


# ---- the choice of tokens ----------------------------------------------------------------------------------------------------
def _prepare_sample(case, g):
    rows, vocab = case["rows"], case["vocab"]
    # a broad body with a heavy upper tail, as a trained head gives: few likely tokens, a long remainder
    logits = torch.randn(rows, vocab, generator=g, device="cuda") * 2.0
    logits += -torch.log(torch.rand(rows, vocab, generator=g, device="cuda").clamp_min(1e-12)) * 0.9
    u = torch.rand(rows, generator=g, device="cuda", dtype=torch.float32)
    full = lambda x, t: torch.full((rows,), x, dtype=t, device="cuda")  # noqa: E731
    temperature, top_p, min_p = (full(case[n], torch.float32) for n in ("temperature", "top_p", "min_p"))
    top_k = full(case["top_k"], torch.int32)
    if case["mixed"]:
        i = torch.arange(rows, device="cuda")
        temperature[i % 8 == 3] = 0.0
        top_k[i % 2 == 1] = 0
        top_p[i % 4 >= 2] = 1.0
        min_p[i % 3 != 0] = 0.0
    return dict(case=case, logits=logits.to(_type(case)), u=u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)


def _run_sample(s):
    if own:
        from lrqk_b200 import sample_tokens
        return sample_tokens(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
    logits, vocab = s["logits"].to(torch.float64), s["logits"].shape[1]
    t = s["temperature"].to(torch.float64)[:, None]
    greedy = t == 0
    order = torch.sort(logits, dim=1, descending=True, stable=True)
    z = (order.values - order.values[:, :1]) / torch.where(greedy, 1.0, t)
    w = torch.exp(z)
    rank = torch.arange(vocab, device=logits.device)
    k = torch.where(greedy, 1, torch.where(s["top_k"][:, None] > 0, s["top_k"][:, None], vocab))
    w = torch.where(rank < k, w, 0.0)
    p = s["top_p"].to(torch.float64)[:, None]
    before = torch.cumsum(w, 1) - w
    keep = (p >= 1) | (before < p * w.sum(1, keepdim=True)) | (rank == 0)
    w = torch.where(keep & (w >= s["min_p"].to(torch.float64)[:, None]), w, 0.0)
    w = torch.zeros_like(w).scatter_(1, order.indices, w)
    mass = torch.cumsum(w, 1)
    total = mass[:, -1:]
    token = (mass <= s["u"].to(torch.float64)[:, None] * total).sum(1)
    token = torch.minimum(token, vocab - 1 - (w.flip(1) > 0).to(torch.int32).argmax(1))
    return token, torch.log(w.gather(1, token[:, None]) / total).squeeze(1).to(torch.float32)


def _exact_sample(case, s):
    tokens, logs = [], []
    for i in range(case["rows"]):
        l, u = s["logits"][i].double(), float(s["u"][i])
        t, k, p, m = float(s["temperature"][i]), int(s["top_k"][i]), float(s["top_p"][i]), float(s["min_p"][i])
        if t == 0:
            tokens.append(torch.argmax(l)), logs.append(torch.zeros((), dtype=torch.float64, device="cuda"))
            continue
        prob = torch.softmax(l / t, 0)
        by = torch.argsort(l, descending=True, stable=True)
        if k > 0:
            by = by[:k]
        if p < 1:
            inside = torch.cumsum(prob[by], 0)
            by = by[:1 + int((inside < p * inside[-1]).sum())]
        by = by[prob[by] >= m * prob[by[0]]]
        by = by.sort().values
        share = prob[by] / prob[by].sum()
        at = min(int((torch.cumsum(share, 0) <= u).sum()), len(by) - 1)
        tokens.append(by[at]), logs.append(torch.log(share[at]))
    return torch.stack(tokens), torch.stack(logs)


# ---- what the tools call -----------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = _generator(seed)
    return {"rotary": _prepare_rotary, "tree": _prepare_tree, "sample": _prepare_sample}[case["op"]](case, g)


def run(state):
    return {"rotary": _run_rotary, "tree": _run_tree, "sample": _run_sample}[state["case"]["op"]](state)


def exact(case, seed):
    state = prepare(case, seed)
    return {"rotary": _exact_rotary, "tree": _exact_tree, "sample": _exact_sample}[case["op"]](case, state)


def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "rotary":
        n = case["batch"] * case["length"] * (case["q_heads"] + case["kv_heads"])
        return {"bytes": 2 * n * case["head_dim"] * e + 8 * case["batch"] * case["length"], "flops": 3 * n * case["part"]}
    if case["op"] == "tree":
        b, t, d, keys = case["batch"], case["nodes"], case["head_dim"], sum(_lengths(case))
        return {"bytes": (2 * keys * case["cache_heads"] + 2 * b * t * (case["kv_heads"] + case["q_heads"])) * d * e + b * t * t,
                "flops": 4 * case["q_heads"] * t * d * (keys + b * t)}
    return {"bytes": case["rows"] * (case["vocab"] * e + 32), "flops": 4 * case["rows"] * case["vocab"]}
