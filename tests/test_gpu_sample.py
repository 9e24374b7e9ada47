"""The choice of tokens against the definition in 64 bits (numpy), token for token.

The kernel sums whole numbers of 2^-44: a weight is off by at most 2^-45 (plus its double exponential's few units of 2^-53),
and V = 4e5 independent roundings add up to sqrt(V / 3) 2^-45 = 1e-11 of a mass that is at least 1.  A token can differ
only where a sum lies within that of a border: rows within ten times that, 1e-10, are let off (`near`), one in fifty at most.  Log-probabilities are
fp32 of a double: 2^-24 of the value plus 1e-8."""
import numpy as np
import pytest
import torch

from lrqk_b200 import sample_tokens

pytestmark = pytest.mark.gpu


def definition(l, u, t, k, p, m):
    """(token, log-probability, near a border) of one row of float64 logits."""
    v = len(l)
    l = np.where(np.isnan(l), -np.inf, l)
    top = l.max()
    if top == -np.inf:
        return -1, np.nan, False
    if not t > 0:
        return int(np.argmax(l)), 0.0, False
    if top == np.inf:
        w = (l == np.inf).astype(np.float64)
    else:
        with np.errstate(over="ignore"):
            w = np.exp((l - top) / t)
    cand = w > 0 if top == np.inf else l > -np.inf
    order = np.argsort(-l, kind="stable")
    order = order[cand[order]]
    if 0 < k < v:
        order = order[:k]
    near = False
    if p < 1:
        total = w[order].sum()
        before = np.cumsum(w[order]) - w[order]
        inside = before < p * total
        inside[0] = True
        off = np.abs(before - p * total)[1:]                                     # (the first always stays)
        near |= bool(((off > 0) & (off < 1e-10 * total)).any())                  # (sums of ones meet a border exactly, on both sides)
        order = order[inside]
    if m > 0:
        order = order[w[order] >= min(m, 1.0)]
    kept = np.sort(order)
    c = np.cumsum(w[kept])
    off = np.abs(c - np.float64(u) * c[-1])[:-1]
    near |= bool(((off > 0) & (off < 1e-10 * c[-1])).any())
    at = min(int((c <= np.float64(u) * c[-1]).sum()), int(np.nonzero(w[kept])[0][-1]))
    return int(kept[at]), float(np.log(w[kept[at]] / c[-1])), near


def check(logits, u, t=1.0, k=0, p=1.0, m=0.0):
    tok, lp = sample_tokens(logits, u, temperature=t, top_k=k, top_p=p, min_p=m)
    assert tok.dtype == torch.int64 and lp.dtype == torch.float32 and tok.shape == lp.shape == u.shape
    l, uu = logits.double().cpu().numpy(), u.cpu().numpy()
    tok, lp = tok.cpu().tolist(), lp.cpu().tolist()
    let_off = 0
    one = lambda x, i: float(x[i]) if isinstance(x, torch.Tensor) else float(np.float32(x))  # noqa: E731 - settings are fp32
    for i in range(len(uu)):
        want, wl, near = definition(l[i], uu[i], one(t, i), int(one(k, i)), one(p, i), one(m, i))
        if near:
            let_off += 1
            continue
        assert tok[i] == want, (i, tok[i], want, l[i][tok[i]], l[i][want])
        assert (np.isnan(wl) and np.isnan(lp[i])) or abs(lp[i] - wl) <= abs(wl) * 2.0 ** -24 + 1e-8, (i, lp[i], wl)
    assert let_off * 50 <= max(50, len(uu))
    return tok


def make(rows, vocab, dtype, seed, spread=2.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    l = torch.randn(rows, vocab, generator=g, device="cuda") * spread
    l += -torch.log(torch.rand(rows, vocab, generator=g, device="cuda").clamp_min(1e-9))
    return l.to(dtype), torch.rand(rows, generator=g, device="cuda")


DT = [torch.float32, torch.bfloat16]
FILTERS = [dict(), dict(k=1), dict(k=50), dict(k=50, p=0.9), dict(p=0.9), dict(p=0.999), dict(p=0.0), dict(m=0.05), dict(p=0.95, m=0.02),
           dict(k=2000, p=0.95, m=0.001), dict(t=0.0), dict(t=0.3, p=0.7), dict(t=4.0, k=300), dict(t=50.0, p=0.5), dict(m=1.0), dict(t=1e-3)]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("vocab", [1, 2, 3, 31, 257, 1000, 8191, 8193, 50257, 128256])
def test_filters(dtype, vocab):
    logits, u = make(5, vocab, dtype, vocab)
    for f in FILTERS:
        check(logits, u, **f)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,vocab", [(1, 152064), (3, 152064), (20, 32000), (40, 32001), (80, 4096), (200, 500), (7, 262144), (2, 400000)])
def test_rows_and_vocabularies(dtype, rows, vocab):
    logits, u = make(rows, vocab, dtype, rows)
    check(logits, u, t=0.8, k=40, p=0.9, m=0.01)
    check(logits, u, p=0.97)
    check(logits, u)


@pytest.mark.parametrize("dtype", DT)
def test_settings_per_row(dtype):
    rows, vocab = 48, 20000
    logits, u = make(rows, vocab, dtype, 7)
    g = torch.Generator(device="cuda").manual_seed(8)
    r = lambda: torch.rand(rows, generator=g, device="cuda")  # noqa: E731
    t, p, m = r() * 2, r() * 1.2, r() * 0.1 - 0.02
    t[::7], p[::5] = 0.0, 1.0
    k = torch.randint(-1, 300, (rows,), generator=g, device="cuda", dtype=torch.int32)
    check(logits, u, t, k, p, m)


@pytest.mark.parametrize("dtype", DT)
def test_equal_logits_and_ties_at_the_borders(dtype):
    g = torch.Generator(device="cuda").manual_seed(3)
    u = torch.rand(12, generator=g, device="cuda")
    for vocab in (5, 3000, 70000):
        flat = torch.zeros(12, vocab, dtype=dtype, device="cuda")
        steps = torch.randint(0, 4, (12, vocab), generator=g, device="cuda").to(dtype)
        two = torch.where(torch.rand(12, vocab, generator=g, device="cuda") < 0.5, -1.5, -0.0).to(dtype)
        two[:, ::3] = two[:, ::3].abs() * (two[:, ::3] == 0) + two[:, ::3] * (two[:, ::3] != 0)    # zeros of either sign are equal
        for l in (flat, flat - 7, steps, two):
            for f in (dict(), dict(k=3), dict(k=vocab // 2), dict(k=vocab - 1), dict(p=0.31), dict(k=vocab // 3 + 1, p=0.77), dict(t=0.0), dict(m=0.9)):
                check(l, u, **f)


@pytest.mark.parametrize("dtype", DT)
def test_infinities_nan_and_extreme_ranges(dtype):
    g = torch.Generator(device="cuda").manual_seed(5)
    logits, u = make(10, 9000, dtype, 4)
    l = logits.clone()
    l[torch.rand(l.shape, generator=g, device="cuda") < 0.7] = float("-inf")
    l[1] = float("-inf")
    l[2] = float("nan")
    l[3, ::2] = float("nan")
    l[4, 17::100] = float("inf")
    l[5, 8999] = float("inf")
    l[6] = float("-inf")
    l[6, 1234] = -3.0
    l[7] = -1e4
    l[7, 5:9] = 2.0
    l[8] = torch.linspace(-3e38, 3e38, 9000, device="cuda").to(dtype)
    l[9] = (torch.arange(9000, device="cuda") % 50).to(dtype) * 1e-40
    for f in FILTERS + [dict(k=8000), dict(k=8000, p=0.5), dict(t=1e38, p=0.5)]:
        check(l, u, **f)
    tok, lp = sample_tokens(l, u)
    assert tok[1] == -1 and tok[2] == -1 and bool(torch.isnan(lp[1:3]).all()) and tok[6] == 1234 and float(lp[6]) == 0.0


@pytest.mark.parametrize("offset", [1e3, 3e4, -5e5])
def test_logits_far_from_zero(offset):
    """A spread of a few units on a large offset: fp32 logits a few hundredths apart at best, many of them equal."""
    logits, u = make(8, 20000, torch.float32, 21)
    l = logits + offset
    for f in (dict(k=50), dict(p=0.9), dict(k=3000, p=0.6), dict(m=0.01), dict(t=0.02, p=0.99), dict()):
        check(l, u, **f)


@pytest.mark.parametrize("dtype", DT)
def test_random_numbers_at_the_ends(dtype):
    logits, _ = make(6, 5000, dtype, 6)
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, 1e-30, -0.5, float("nan")], device="cuda")
    tok, lp = sample_tokens(logits, u, top_k=20)
    kept = torch.topk(logits.float(), 20).indices
    assert all(int(tok[i]) in kept[i].tolist() for i in range(6)) and bool(torch.isfinite(lp).all())
    assert int(tok[0]) == int(kept[0].min()) and int(tok[1]) == int(kept[1].max()) and int(tok[2]) == int(kept[2].max())


@pytest.mark.parametrize("dtype", DT)
def test_strided_unaligned_and_sliced_logits(dtype):
    logits, u = make(6, 3001, dtype, 9)
    ref = check(logits, u, p=0.9)
    wide = torch.zeros(6, 3100, dtype=dtype, device="cuda")
    wide[:, 7:3008] = logits
    assert check(wide[:, 7:3008], u, p=0.9) == ref
    assert check(logits.t().contiguous().t(), u, p=0.9) == ref
    assert check(logits[2:3], u[2:3], p=0.9) == ref[2:3]
    assert check(logits[:1].expand(6, 3001), u, p=0.9)[0] == ref[0]
    big = torch.empty(2 ** 31 + 4096, dtype=dtype, device="cuda")
    far = big.as_strided((2, 3001), (2 ** 31, 1))
    far.copy_(logits[:2])
    assert check(far, u[:2], p=0.9) == ref[:2]


@pytest.mark.parametrize("dtype", DT)
def test_a_row_does_not_depend_on_its_batch_and_repeats(dtype):
    logits, u = make(150, 6000, dtype, 10)
    tok, lp = sample_tokens(logits, u, top_k=100, top_p=0.9)
    for i in (0, 77, 149):
        t1, l1 = sample_tokens(logits[i:i + 1], u[i:i + 1], top_k=100, top_p=0.9)     # another cluster size
        assert int(t1) == int(tok[i]) and float(l1) == float(lp[i])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = sample_tokens(logits, u, top_k=100, top_p=0.9)
    torch.cuda.synchronize()
    assert torch.equal(again[0], tok) and torch.equal(again[1], lp)
    graph = torch.cuda.CUDAGraph()
    p = torch.full((150,), 0.9, device="cuda")
    with torch.cuda.graph(graph):
        out = sample_tokens(logits, u, top_k=100, top_p=p)
    p.fill_(0.5)
    u.copy_(u.flip(0))
    graph.replay()
    want = sample_tokens(logits, u, top_k=100, top_p=0.5)
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_frequencies_follow_the_distribution():
    n = 20000
    p = torch.tensor([0.5, 0.25, 0.125, 0.0625, 0.0625], device="cuda")
    u = (torch.arange(n, device="cuda") + 0.5) / n
    tok, lp = sample_tokens(p.log().expand(n, 5), u.float())
    count = torch.bincount(tok, minlength=5).double()
    assert bool(((count - p.double() * n).abs() <= 1).all())          # an even comb of random numbers: exact but for the ends
    assert torch.allclose(lp, p.log()[tok], atol=1e-6)


def test_refusals():
    logits, u = make(3, 100, torch.float32, 1)
    bad = [dict(logits=logits.half()), dict(logits=logits[0]), dict(logits=logits.cpu()), dict(logits=logits[:, :0]), dict(u=u.double()), dict(u=u[:2]),
           dict(u=u.cpu()), dict(temperature=-1.0), dict(temperature=float("nan")), dict(top_p=-0.1), dict(min_p=float("inf")), dict(top_k=-1),
           dict(temperature=u.double()), dict(top_k=u), dict(top_p=u[:1]), dict(min_p=u.cpu())]
    for kw in bad:
        a = dict(logits=logits, u=u)
        a.update(kw)
        with pytest.raises(ValueError):
            sample_tokens(a.pop("logits"), a.pop("u"), **a)
    assert torch.equal(sample_tokens(logits, u, top_k=2 ** 40)[0], sample_tokens(logits, u)[0])
    from lrqk_b200._lib import LrqkError
    with pytest.raises(LrqkError):
        sample_tokens(torch.zeros(1, 500000, device="cuda"), u[:1])
    assert sample_tokens(logits[:0], u[:0])[0].shape == (0,)
