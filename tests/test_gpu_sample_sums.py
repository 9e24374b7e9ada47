"""The choice of tokens where all roundings of the weights go one way: a peak and thousands of equal small weights.

A weight is a whole number of 2^-44 of the largest: off by 2^-45 at most, a sum over V tokens by V 2^-45 (plus the double
exponential's few units of 2^-53 each, and the one rounding of u times the sum).  So the chosen token's stretch of the cumulative
mass, computed in 64 bits, meets u within that, on either side of the comparison."""
import numpy as np
import pytest
import torch

from lrqk_b200 import sample_tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1000, 128256])
@pytest.mark.parametrize("peak", [0, 0.5, 1])
def test_a_peak_and_many_equal_small_weights(dtype, vocab, peak):
    at = min(vocab - 1, int(peak * vocab))
    for low in (-30.25, -30.5, -31.0, -31.25, -33.0, -20.0, -10.0):      # around half of 2^-44 (-31.19) and above
        logits = torch.full((12, vocab), low, device="cuda").to(dtype)
        logits[:, at] = 0.0
        l = logits[0].double().cpu().numpy()
        w = np.exp(l)
        c, total, err = np.cumsum(w), w.sum(), 2 * (vocab * (2.0 ** -45 + w.max() * 2.0 ** -52))
        small = (vocab - 1) * w[(at + 1) % vocab]
        us = [0.0, 2.0 ** -60, small / 3, small / 2, small * 0.9, small, small * 1.1, 0.25, 0.5, 1 - small, 1 - 2.0 ** -24, 1 - 2.0 ** -20]
        u = torch.tensor([min(max(x, 0.0), 1 - 2.0 ** -24) for x in us], dtype=torch.float32, device="cuda")
        p = float(np.float32(1 - 2.0 ** -24))
        for top_p in (1.0, p):
            tok, lp = sample_tokens(logits, u, top_p=top_p)
            # the kept mass: all, or down to the first small one (from the highest index) without which p of it is there
            least = total if top_p == 1.0 else p * total - err
            most = total if top_p == 1.0 else min(total, p * total + w[(at + 1) % vocab]) + err
            for x, t, q in zip(u.cpu().double().numpy(), tok.tolist(), lp.tolist()):
                # c counts the small ones that top_p dropped too: what is kept before t lacks at most what was dropped in all
                assert 0 <= t < vocab and c[t] - w[t] - (total - least) - err <= x * most and x * least <= c[t] + err
                # an fp32 rounding, and a kept mass that is off by 2^-24 of itself (top_p) and err
                assert abs(q - np.log(w[t] / total)) <= abs(q) * 2.0 ** -24 + 2.0 ** -24 + 2 * err
