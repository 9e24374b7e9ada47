"""Frequencies of the rotary positions against the formulas, evaluated one pair at a time, and the refusals that need no GPU."""
import math

import pytest
import torch

from lrqk_b200 import apply_rotary, rotary_frequencies


@pytest.mark.parametrize("dim,base", [(2, 10000.0), (64, 10000.0), (96, 500000.0), (128, 1e6)])
def test_plain_linear_and_dynamic(dim, base):
    plain, one = rotary_frequencies(dim, base)
    assert plain.dtype == torch.float64 and plain.shape == (dim // 2,) and one == 1.0
    for i in range(dim // 2):
        assert math.isclose(float(plain[i]), base ** (-2 * i / dim), rel_tol=1e-14)
    lin, one = rotary_frequencies(dim, base, {"rope_type": "linear", "factor": 8})
    assert torch.allclose(lin * 8, plain, rtol=1e-15, atol=0) and one == 1.0
    if dim >= 4:
        s = {"type": "dynamic", "factor": 4.0, "original_max_position_embeddings": 4096}
        short, _ = rotary_frequencies(dim, base, s, seq_len=1000)
        assert torch.allclose(short, plain, rtol=1e-14, atol=0)                # within the original context nothing changes
        grown, _ = rotary_frequencies(dim, base, s, seq_len=16384)
        b2 = base * (4.0 * 16384 / 4096 - 3.0) ** (dim / (dim - 2))
        for i in range(dim // 2):
            assert math.isclose(float(grown[i]), b2 ** (-2 * i / dim), rel_tol=1e-13)


def test_yarn_leaves_fast_pairs_and_divides_slow_ones():
    dim, base, f, orig = 128, 1e6, 4.0, 32768
    plain, _ = rotary_frequencies(dim, base)
    s = {"rope_type": "yarn", "factor": f, "original_max_position_embeddings": orig}
    inv, out = rotary_frequencies(dim, base, s)
    assert math.isclose(out, 0.1 * math.log(4.0) + 1.0)
    for i in range(dim // 2):
        turns = orig * float(plain[i]) / (2 * math.pi)
        ratio = float(inv[i] / plain[i])
        assert 1 / f - 1e-12 <= ratio <= 1 + 1e-12
        if turns > 40:
            assert math.isclose(ratio, 1.0, rel_tol=1e-12)
        if turns < 0.8:
            assert math.isclose(ratio, 1 / f, rel_tol=1e-12)
    assert rotary_frequencies(dim, base, dict(s, attention_factor=0.5))[1] == 0.5
    both = rotary_frequencies(dim, base, dict(s, mscale=2.0, mscale_all_dim=1.0))[1]
    assert math.isclose(both, (0.2 * math.log(4.0) + 1.0) / (0.1 * math.log(4.0) + 1.0))


def test_llama3_bands():
    dim, base, f, orig, lo, hi = 128, 500000.0, 8.0, 8192, 1.0, 4.0
    plain, _ = rotary_frequencies(dim, base)
    inv, out = rotary_frequencies(dim, base, {"rope_type": "llama3", "factor": f, "low_freq_factor": lo, "high_freq_factor": hi,
                                              "original_max_position_embeddings": orig})
    assert out == 1.0
    for i in range(dim // 2):
        w = float(plain[i])
        wavelength = 2 * math.pi / w
        if wavelength < orig / hi:
            want = w
        elif wavelength > orig / lo:
            want = w / f
        else:
            t = (orig / wavelength - lo) / (hi - lo)
            want = (1 - t) * w / f + t * w
        assert math.isclose(float(inv[i]), want, rel_tol=1e-12)


@pytest.mark.parametrize("kw", [dict(rotary_dim=0), dict(rotary_dim=7), dict(rotary_dim=64, base=0.0),
                                dict(rotary_dim=64, scaling={"rope_type": "linear"}), dict(rotary_dim=64, scaling={"rope_type": "linear", "factor": 0.5}),
                                dict(rotary_dim=64, scaling={"rope_type": "yarn", "factor": 2.0}),
                                dict(rotary_dim=64, scaling={"rope_type": "nosuch", "factor": 2.0})])
def test_refused_settings(kw):
    with pytest.raises(ValueError):
        rotary_frequencies(**kw)


def test_cpu_tensors_are_refused():
    inv, _ = rotary_frequencies(64)
    x = torch.zeros(1, 2, 3, 64)
    with pytest.raises(ValueError):
        apply_rotary(x, None, torch.arange(3), inv)


def test_dual_tensors_are_noticed():
    from torch.autograd import forward_ad
    from lrqk_b200.state import has_tangent
    x = torch.ones(3)
    assert not has_tangent(x, None)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones(3))
        assert not dual.requires_grad and has_tangent(None, dual) and has_tangent(x, dual) and not has_tangent(x, None)
        with torch.no_grad():
            assert has_tangent(dual)
