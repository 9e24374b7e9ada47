"""Tree attention where a CTA walks many segments of one tile each: empty and one-tile caches, and runs cut after one tile.  The
two chains of softmax warps then take turns, and the one without a tile has only its statistics to hand over: nothing else
holds it back."""
import pytest
import torch

from lrqk_b200 import check_tree_status, tree_attention
from test_gpu_tree import check, make, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("b,cap", [(60, 0), (200, 1), (300, 128), (37, 129)])
@pytest.mark.parametrize("t,hq,hc", [(3, 8, 8), (9, 8, 2), (128, 2, 2), (17, 28, 4)])
def test_segments_of_one_tile(b, cap, t, hq, hc):
    q, ck, cv, tk, tv, _ = make(1, hq, hc, hc, t, cap, 64, torch.bfloat16, seed=b + t)
    # every sequence has the same content, so each has to be the one 64-bit result (a unit cut between two CTAs is summed in
    # another order: within the tolerance, not bit for bit)
    want, wl, tol, ltol = reference(q, ck, cv, tk, tv, None, None, 64 ** -0.5)
    q, ck, cv, tk, tv = (x.expand(b, -1, -1, -1) for x in (q, ck, cv, tk, tv))
    for _ in range(5):
        out, lse = tree_attention(q, ck, cv, tk, tv, return_lse=True)
        assert bool(((out.double() - want).abs() <= tol).all()) and bool(((lse.double() - wl).abs() <= ltol).all())
    check_tree_status()


def test_ragged_batches_of_empty_and_short_caches():
    b = 150
    q, ck, cv, tk, tv, mask = make(b, 4, 2, 2, 11, 300, 128, torch.bfloat16, seed=3)
    for kind in range(3):
        lens = torch.tensor([[0, 0, 0], [0, 128, 1], [300, 0, 129]][kind], dtype=torch.int32, device="cuda").repeat(b // 3)
        first = tree_attention(q, ck, cv, tk, tv, mask, cache_lens=lens, return_lse=True)
        check(first, q, ck, cv, tk, tv, mask, lens)
        for _ in range(10):
            again = tree_attention(q, ck, cv, tk, tv, mask, cache_lens=lens, return_lse=True)
            assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])
