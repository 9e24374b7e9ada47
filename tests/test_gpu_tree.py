"""Attention of a tree of drafted tokens against a plain implementation in 64 bits.

Tolerance of a row, from the arithmetic (A = sum_j p_j |v_j|, the size of what is summed):
* a score is a sum of d products in fp32: off by at most d 2^-23 sum_e |q_e k_e| scale, the same again for its rounding in
  base 2, so every weight by twice the largest such error (numerator and denominator) -- relative;
* exponentials and the few operations around them: 2^-20;
* the sums over n keys: n 2^-23;
* bf16: weights enter the second product as two bf16 parts (2^-16) where the rows of a cache head (query heads of the group
  times nodes) are 128 at most, and as one (half a step, 2^-8 of each weight) above; the result is rounded once (half a step)."""
import math

import pytest
import torch

from lrqk_b200 import check_tree_status, tree_attention, tree_mask

pytestmark = pytest.mark.gpu


def reference(q, ck, cv, tk, tv, mask, lens, scale):
    """(out, lse, tolerance of out, tolerance of lse) in 64 bits, one head at a time."""
    b, hq, t, d = q.shape
    cap = ck.shape[2]
    out, tol = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse, ltol = torch.full((b, hq, t), -math.inf, dtype=torch.float64, device=q.device), torch.zeros((b, hq, t), dtype=torch.float64, device=q.device)
    for i in range(b):
        n = cap if lens is None else min(max(int(lens[i]), 0), cap)
        seen = torch.ones(t, t, dtype=torch.bool, device=q.device).tril() if mask is None else (mask if mask.dim() == 2 else mask[i if mask.shape[0] > 1 else 0]).bool()
        see = torch.cat((torch.ones(t, n, dtype=torch.bool, device=q.device), seen), 1)
        for h in range(hq):
            hc, ht = h * ck.shape[1] // hq, h * tk.shape[1] // hq
            k, v = (torch.cat((c[i, hc, :n], w[i, ht])).double() for c, w in ((ck, tk), (cv, tv)))
            qq = q[i, h].double()
            s = (qq @ k.T * scale).masked_fill(~see, -math.inf)
            size = (qq.abs() @ k.abs().T * scale).masked_fill(~see, 0.0)
            m = s.amax(1, keepdim=True).masked_fill(~see.any(1, keepdim=True), 0.0)
            e = torch.exp(s - m)
            tot = e.sum(1, keepdim=True)
            w = torch.where(tot > 0, e / tot, torch.zeros_like(e))
            part = w[:, :, None] * torch.where(see[:, :, None], v[None], torch.zeros_like(v)[None]) if t * (n + t) * d < 2 ** 24 else None
            vz = torch.where(see.any(0)[:, None], v, torch.zeros_like(v))
            out[i, h] = part.sum(1) if part is not None else w @ vz
            a = part.abs().sum(1) if part is not None else w @ vz.abs()
            err = 2 * size.amax(1, keepdim=True) * d * 2.0 ** -23 + 2.0 ** -20 + (n + t) * 2.0 ** -23
            if q.dtype == torch.bfloat16:
                err = err + (2.0 ** -16 if t * hq // ck.shape[1] <= 128 else 2.0 ** -8)
            tol[i, h] = a * err
            lse[i, h] = (m + torch.log(tot)).squeeze(1)
            ltol[i, h] = (err + size.amax(1, keepdim=True) * 2.0 ** -23 + lse[i, h].abs()[:, None].nan_to_num(0, 0, 0) * 2.0 ** -22).squeeze(1)
    half = torch.finfo(q.dtype).eps / 2
    return out, lse, tol + (out.abs() + tol) * half, ltol


def check(got, q, ck, cv, tk, tv, mask=None, lens=None, scale=None):
    out, lse = got
    want, wl, tol, ltol = reference(q, ck, cv, tk, tv, mask, lens, q.shape[-1] ** -0.5 if scale is None else scale)
    assert out.dtype == q.dtype and out.shape == q.shape and out.is_contiguous() and lse.dtype == torch.float32
    bad = ~((out.double() - want).abs() <= tol)
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:3].tolist(), out[bad][:3].tolist(), want[bad][:3].tolist(), tol[bad][:3].tolist())
    empty = torch.isinf(wl)
    assert torch.equal(torch.isinf(lse), empty) and bool((lse[empty] < 0).all()) and not bool(out[empty].any())
    badl = ~((lse.double() - wl).abs() <= ltol) & ~empty
    assert not bool(badl.any()), (lse[badl][:3].tolist(), wl[badl][:3].tolist())
    check_tree_status()


def make(b, hq, hc, ht, t, cap, d, dtype, seed=0, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: (torch.randn(*s, generator=g, device="cuda") * spread).to(dtype)  # noqa: E731
    parents = [[-1 if i == 0 else int(x * i) for i, x in enumerate(torch.rand(t, generator=torch.Generator().manual_seed(seed + j)))] for j in range(b)]
    return r(b, hq, t, d), r(b, hc, cap, d), r(b, hc, cap, d), r(b, ht, t, d), r(b, ht, t, d), tree_mask(parents, "cuda")


DT = [torch.float32, torch.bfloat16]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("t", [1, 2, 7, 16, 33, 64, 65, 129, 256])
def test_nodes(dtype, d, t):
    q, ck, cv, tk, tv, mask = make(2, 4, 2, 2, t, 300, d, dtype, seed=t)
    lens = torch.tensor([300, 77], dtype=torch.int32, device="cuda")
    check(tree_attention(q, ck, cv, tk, tv, mask, cache_lens=lens, return_lse=True), q, ck, cv, tk, tv, mask, lens)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n", [0, 1, 2, 31, 63, 64, 65, 127, 128, 129, 255, 256, 257, 1000, 4099])
def test_cache_lengths(dtype, n):
    q, ck, cv, tk, tv, mask = make(1, 8, 2, 2, 9, max(n, 1) + 5, 128, dtype, seed=n)
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    ck[:, :, n:], cv[:, :, n:] = float("nan"), float("inf")          # rows behind the length may hold anything
    check(tree_attention(q, ck, cv, tk, tv, mask, cache_lens=lens, return_lse=True), q, ck, cv, tk, tv, mask, lens)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("b,hq,hc,ht,t", [(1, 32, 8, 8, 8), (3, 28, 4, 4, 13), (2, 40, 8, 8, 5), (1, 32, 32, 8, 16), (1, 4, 4, 1, 3), (2, 6, 1, 1, 70),
                                          (40, 2, 1, 1, 3), (1, 16, 1, 1, 40), (2, 8, 2, 1, 200)])
def test_heads_and_ragged_batches(dtype, b, hq, hc, ht, t):
    cap = 513
    q, ck, cv, tk, tv, mask = make(b, hq, hc, ht, t, cap, 128, dtype, seed=b * hq)
    lens = torch.tensor([[0, 1, 513, 128, 300, 129, 64][i % 7] for i in range(b)], dtype=torch.int32, device="cuda")
    check(tree_attention(q, ck, cv, tk, tv, mask, cache_lens=lens, return_lse=True), q, ck, cv, tk, tv, mask, lens)


@pytest.mark.parametrize("dtype", DT)
def test_sharp_scores_and_other_scales(dtype):
    # scores of some hundreds: the running maximum jumps from tile to tile, most weights vanish
    q, ck, cv, tk, tv, mask = make(1, 8, 2, 2, 6, 1500, 128, dtype, seed=5, spread=4.0)
    ck[:, :, 700] = 3 * q[:, ::4, 0]
    check(tree_attention(q, ck, cv, tk, tv, mask, return_lse=True), q, ck, cv, tk, tv, mask)
    check(tree_attention(q, ck, cv, tk, tv, mask, scale=0.7, return_lse=True), q, ck, cv, tk, tv, mask, scale=0.7)
    # maxima that rise by a little with every row of the cache
    ramp = torch.linspace(0.0, 1.0, 1500, device="cuda")[:, None]
    ck.copy_((q[:, ::4, :1].float() * ramp * 0.1).to(dtype))
    check(tree_attention(q, ck, cv, tk, tv, mask, return_lse=True), q, ck, cv, tk, tv, mask)


@pytest.mark.parametrize("dtype", DT)
def test_masks_that_leave_rows_empty_and_nodes_nobody_sees(dtype):
    q, ck, cv, tk, tv, mask = make(2, 4, 2, 2, 20, 40, 64, dtype, seed=7)
    lens = torch.tensor([0, 17], dtype=torch.int32, device="cuda")
    mask[:, 3] = False                      # in the empty sequence this row sees nothing
    mask[:, :, 11] = False
    mask[:, 12:15] = False
    mask[:, :, 19] = False
    mask[:, 19, 19] = False
    tk[:, :, 11], tv[:, :, 11] = float("nan"), float("nan")
    tk[:, :, 19], tv[:, :, 19] = float("inf"), float("-inf")
    check(tree_attention(q, ck, cv, tk, tv, mask, cache_lens=lens, return_lse=True), q, ck, cv, tk, tv, mask, lens)
    got = tree_attention(q, ck, cv, tk, tv, torch.zeros(20, 20, dtype=torch.bool, device="cuda"), cache_lens=torch.zeros(2, dtype=torch.int32, device="cuda"), return_lse=True)
    assert not bool(got[0].any()) and bool((got[1] == -math.inf).all())


@pytest.mark.parametrize("dtype", DT)
def test_values_out_of_range_reach_only_the_rows_that_see_them(dtype):
    """A padded node with garbage that it alone sees: the other rows are what they are without it."""
    for t in (12, 140):
        q, ck, cv, tk, tv, mask = make(1, 4, 2, 2, t, 90, 128, dtype, seed=t)
        last = t - 1
        mask[:, :, last] = False
        mask[:, last, last] = True
        clean = tree_attention(q, ck, cv, tk, tv, mask)
        for kind in (float("nan"), float("inf")):
            v = tv.clone()
            v[:, :, last, 5::7] = kind
            got = tree_attention(q, ck, cv, tk, v, mask)
            assert torch.equal(got[:, :, :last], clean[:, :, :last])
            row = got[:, :, last]
            assert bool((torch.isnan(row) if math.isnan(kind) else row == kind)[..., 5::7].all())
            keep = torch.ones(128, dtype=torch.bool)
            keep[5::7] = False
            assert torch.equal(row[..., keep], clean[:, :, last][..., keep])
            k = tk.clone()
            k[:, :, last, 3] = kind
            assert torch.equal(tree_attention(q, ck, cv, k, tv, mask)[:, :, :last], clean[:, :, :last])
        q2 = q.clone()
        q2[:, :, 1] = float("nan")
        got = tree_attention(q2, ck, cv, tk, tv, mask)
        assert bool(torch.isnan(got[:, :, 1]).all()) and torch.equal(got[:, :, 2:], clean[:, :, 2:])


@pytest.mark.parametrize("dtype", DT)
def test_strides_views_and_shared_caches(dtype):
    g = torch.Generator(device="cuda").manual_seed(9)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)  # noqa: E731
    q, tk, tv = r(3, 11, 8, 64).transpose(1, 2), r(3, 11, 2, 64).transpose(1, 2), r(3, 2, 11, 72)[..., :64]
    store_k, store_v = r(3, 2, 400, 64), r(3, 400, 2, 128).transpose(1, 2)
    ck, cv = store_k[:, :, 16:301], store_v[:, :, :285, 64:]
    check(tree_attention(q, ck, cv, tk, tv, return_lse=True), q, ck, cv, tk, tv)
    one_k, one_v = store_k[:1].expand(3, 2, 400, 64), store_v[:1, :1, :, :64].expand(3, 2, 400, 64)
    mask = tree_mask([-1] + [0] * 10, "cuda")
    for m in (mask, mask.to(torch.uint8), mask[None], mask.expand(3, 11, 11), mask.t().contiguous().t()):
        check(tree_attention(q, one_k, one_v, tk, tv, m, return_lse=True), q, one_k, one_v, tk, tv, mask)
    one = q[:, :, 4:5]
    check(tree_attention(one, ck, cv, tk[:, :, :1], tv[:, :, :1], return_lse=True), one, ck, cv, tk[:, :, :1], tv[:, :, :1])


@pytest.mark.parametrize("dtype", DT)
def test_lengths_outside_the_cache_and_an_empty_cache(dtype):
    q, ck, cv, tk, tv, mask = make(3, 4, 2, 2, 5, 70, 64, dtype, seed=3)
    lens = torch.tensor([-5, 1000, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    check(tree_attention(q, ck, cv, tk, tv, mask, cache_lens=lens, return_lse=True), q, ck, cv, tk, tv, mask, lens)
    nk = ck[:, :, :0]
    check(tree_attention(q, nk, nk, tk, tv, mask, return_lse=True), q, nk, nk, tk, tv, mask)
    assert tree_attention(q[:0], ck[:0], cv[:0], tk[:0], tv[:0]).shape == (0, 4, 5, 64)
    assert tree_attention(q[:, :, :0], ck, cv, tk[:, :, :0], tv[:, :, :0]).shape == (3, 4, 0, 64)


def test_offsets_beyond_32_bits():
    big = torch.empty((2 ** 31 + 2 ** 20) * 2, dtype=torch.bfloat16, device="cuda")       # 8.6 GB
    shape, strides = (2, 2, 300, 128), (2 ** 31 + 2 ** 19, 2 ** 31 - 2 ** 18, 128)
    ck, cv = big.as_strided(shape, strides + (1,)), big.as_strided(shape, strides + (1,), 300 * 128)
    g = torch.Generator(device="cuda").manual_seed(1)
    ck.copy_(torch.randn(shape, generator=g, device="cuda"))
    cv.copy_(torch.randn(shape, generator=g, device="cuda"))
    q, tk, tv = (torch.randn(2, h, 6, 128, generator=g, device="cuda").bfloat16() for h in (4, 2, 2))
    check(tree_attention(q, ck, cv, tk, tv, return_lse=True), q, ck, cv, tk, tv)


@pytest.mark.parametrize("dtype", DT)
def test_same_bits_again_captured_and_beside_another_call(dtype):
    q, ck, cv, tk, tv, mask = make(4, 8, 2, 2, 24, 3000, 128, dtype, seed=11)
    lens = torch.tensor([3000, 5, 1700, 0], dtype=torch.int32, device="cuda")
    ref = tree_attention(q, ck, cv, tk, tv, mask, cache_lens=lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = []
    for _ in range(4):
        outs.append(tree_attention(q, ck, cv, tk, tv, mask, cache_lens=lens))
        with torch.cuda.stream(side):
            outs.append(tree_attention(q, ck, cv, tk, tv, mask, cache_lens=lens))
    torch.cuda.synchronize()
    assert all(torch.equal(o, ref) for o in outs)
    graphs, got = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for gr in graphs:
        with torch.cuda.graph(gr):
            got.append(tree_attention(q, ck, cv, tk, tv, mask, cache_lens=lens))
    lens.copy_(torch.tensor([1, 2999, 0, 640], dtype=torch.int32))
    want = tree_attention(q, ck, cv, tk, tv, mask, cache_lens=lens)
    for gr in graphs:
        gr.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in got)
    check_tree_status()


def test_a_chain_of_single_tokens_equals_the_tree():
    """A chain of nodes gives what attending token by token over a growing cache gives."""
    q, ck, cv, tk, tv, _ = make(1, 8, 2, 2, 6, 200, 128, torch.bfloat16, seed=2)
    all_k, all_v = torch.cat((ck, tk), 2), torch.cat((cv, tv), 2)
    whole = tree_attention(q, ck, cv, tk, tv)
    for i in range(6):
        one = tree_attention(q[:, :, i:i + 1], all_k[:, :, :200 + i], all_v[:, :, :200 + i], tk[:, :, i:i + 1], tv[:, :, i:i + 1], return_lse=True)
        check(one, q[:, :, i:i + 1], all_k[:, :, :200 + i], all_v[:, :, :200 + i], tk[:, :, i:i + 1], tv[:, :, i:i + 1])
        # each is within half a step of the exact row plus its fp32 error: two roundings apart at most
        a, b = whole[:, :, i].double(), one[0][:, :, 0].double()
        assert bool(((a - b).abs() <= (a.abs() + b.abs()) * 2.0 ** -8 + 2.0 ** -12).all())


def test_refusals():
    q, ck, cv, tk, tv, mask = make(2, 4, 2, 2, 5, 30, 64, torch.bfloat16)
    lens = torch.tensor([1, 2], dtype=torch.int32, device="cuda")
    base = dict(q=q, ck=ck, cv=cv, tk=tk, tv=tv, mask=mask, cache_lens=lens)
    wide = torch.zeros(2, 2, 5, 65, dtype=torch.bfloat16, device="cuda")
    bad = [dict(q=q.half()), dict(q=q[0]), dict(q=q.cpu()), dict(ck=ck.float()), dict(ck=ck[:1]), dict(cv=cv[:, :, :29]), dict(cv=cv[:, :1]),
           dict(tk=tk[:, :, :4]), dict(tv=tv[:, :1]), dict(q=q[:, :3]), dict(tk=wide[..., :64]), dict(tk=wide[..., 1:]), dict(mask=mask.float()),
           dict(mask=mask[:, :4]), dict(mask=mask.cpu()), dict(mask=mask.repeat(2, 1, 1)), dict(cache_lens=lens.long()), dict(cache_lens=lens[:1]),
           dict(cache_lens=lens.cpu()), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan"))]
    for kw in bad:
        a = dict(base)
        a.update(kw)
        with pytest.raises(ValueError):
            tree_attention(a.pop("q"), a.pop("ck"), a.pop("cv"), a.pop("tk"), a.pop("tv"), a.pop("mask"), **a)
    with pytest.raises(ValueError):
        tree_attention(*make(1, 2, 1, 1, 257, 8, 64, torch.bfloat16)[:5])
    with pytest.raises(ValueError):
        tree_attention(*make(1, 2, 1, 1, 3, 8, 96, torch.bfloat16)[:5])
    one = ck[:, :, :1].expand(2, 2, 30, 64)                            # one row for all: a tensor copy cannot repeat it
    for a in ((q, one, cv, tk, tv), (q, ck, one, tk, tv), (q, ck, cv, tk[:, :, :1].expand(2, 2, 5, 64), tv), (q[:, :, :1].expand(2, 4, 5, 64), ck, cv, tk, tv)):
        with pytest.raises(ValueError):
            tree_attention(*a)
    grad = q.float().requires_grad_()
    with pytest.raises(ValueError):
        tree_attention(grad, ck.float(), cv.float(), tk.float(), tv.float())


@pytest.mark.parametrize("t,spoilt", [(64, 63), (30, 29), (160, 130)])
def test_values_out_of_range_in_some_of_many_short_sequences(t, spoilt):
    """A CTA meets many (sequence, head) units in a row, each with other drafted values out of range: every row that sees one has
    it, no other row has any."""
    q, ck, cv, tk, tv = make(60, 32, 8, 8, t, 40, 128, torch.bfloat16, seed=5)[:5]
    columns = [(7 * i + 3) % 128 for i in range(60)]
    for i in range(0, 60, 2):
        tv[i, :, spoilt, columns[i]] = math.inf
    for lens in (torch.zeros(60, dtype=torch.int32, device="cuda"), torch.arange(60, dtype=torch.int32, device="cuda") % 41):
        for _ in range(10):
            out = tree_attention(q, ck, cv, tk, tv, cache_lens=lens)
            want = torch.zeros(out.shape, dtype=torch.bool, device="cuda")
            for i in range(0, 60, 2):
                want[i, :, spoilt:, columns[i]] = True
            assert torch.equal(torch.isinf(out), want) and not bool(torch.isnan(out).any())
    check_tree_status()
