"""Tree attention in bf16: a row is as accurate whatever the number of rows that share its cache head.

Weights enter the product with the values as two bf16 parts: the high one leaves at most half a step (2^-8) of a weight, the low
one half a step of that (2^-16).  The rest of the tolerance is that of fp32 arithmetic (`reference` of the tree tests on the same
values in fp32: scores, exponentials, sums), then one rounding of the result (2^-8)."""
import pytest
import torch

from lrqk_b200 import check_tree_status, tree_attention
from test_gpu_tree import make, reference

pytestmark = pytest.mark.gpu


def check_two_parts(out, lse, q, ck, cv, tk, tv, mask, lens=None):
    scale = q.shape[-1] ** -0.5
    f = [x.float() for x in (q, ck, cv, tk, tv)]
    want, wl, tol, ltol = reference(*f, mask, lens, scale)
    size = reference(f[0], f[1], f[2].abs(), f[3], f[4].abs(), mask, lens, scale)[0]    # sum_j p_j |v_j|
    tol = tol + size * 2.0 ** -16
    bad = ~((out.double() - want).abs() <= tol + (want.abs() + tol) * 2.0 ** -8)
    assert not bool(bad.any()), (int(bad.sum()), out[bad][:3].tolist(), want[bad][:3].tolist(), tol[bad][:3].tolist())
    assert bool(((lse.double() - wl).abs() <= ltol + 2.0 ** -16).all())
    check_tree_status()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("t,hq,hc", [(32, 8, 2), (33, 8, 2), (64, 8, 2), (25, 14, 2), (129, 1, 1), (256, 4, 1), (7, 96, 1), (150, 2, 2)])
def test_accuracy_does_not_depend_on_the_rows_of_a_head(d, t, hq, hc):
    for cap in (3, 90, 700):
        q, ck, cv, tk, tv, mask = make(2, hq, hc, hc, t, cap, d, torch.bfloat16, seed=t + cap, spread=0.5)
        lens = torch.tensor([cap, cap // 2], dtype=torch.int32, device="cuda")
        out, lse = tree_attention(q, ck, cv, tk, tv, mask, cache_lens=lens, return_lse=True)
        check_two_parts(out, lse, q, ck, cv, tk, tv, mask, lens)


@pytest.mark.parametrize("heads", [80, 256])
def test_more_row_blocks_than_multiprocessors(heads):
    """256 nodes of 80 and 256 query heads on one cache head: 20480 and 65536 rows, the most there are."""
    q, ck, cv, tk, tv, mask = make(1, heads, 1, 1, 256, 200, 64, torch.bfloat16, seed=1, spread=0.5)
    out, lse = tree_attention(q, ck, cv, tk, tv, mask, return_lse=True)
    check_two_parts(out, lse, q, ck, cv, tk, tv, mask)
