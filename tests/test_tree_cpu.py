"""Ancestor masks of drafted trees, and the refusals that need no GPU."""
import ctypes as C

import pytest
import torch

from lrqk_b200 import _lib, tree_attention, tree_mask


def test_mask_of_parents():
    m = tree_mask([-1, 0, 0, 1, -1, 4])
    want = [[1, 0, 0, 0, 0, 0], [1, 1, 0, 0, 0, 0], [1, 0, 1, 0, 0, 0], [1, 1, 0, 1, 0, 0], [0, 0, 0, 0, 1, 0], [0, 0, 0, 0, 1, 1]]
    assert m.dtype == torch.bool and m.int().tolist() == want
    two = tree_mask([[-1, 0], [-1, -1]])
    assert two.int().tolist() == [[[1, 0], [1, 1]], [[1, 0], [0, 1]]]
    assert tree_mask([]).shape == (0, 0)
    for bad in ([0], [-1, 1], [-1, -2], [-1, 2, 0]):
        with pytest.raises(ValueError):
            tree_mask(bad)


def test_cpu_tensors_are_refused():
    x = torch.zeros(1, 2, 3, 64)
    with pytest.raises(ValueError):
        tree_attention(x, x, x, x, x)


def test_workspace_of_refused_shapes_is_zero():
    lib = _lib.lib()

    def ws(**kw):
        a = _lib.TreeArgs()
        base = dict(dtype=_lib.LRQK_BF16, batch=1, nodes=8, q_heads=8, cache_heads=2, tree_heads=2, head_dim=128, capacity=100)
        base.update(kw)
        for k, v in base.items():
            setattr(a, k, v)
        return lib.lrqk_tree_attention_workspace_bytes(C.byref(a))

    assert ws() > 0 and ws(dtype=_lib.LRQK_F32) > 0 and ws(nodes=256, q_heads=64) > 0
    for bad in (dict(dtype=7), dict(batch=0), dict(nodes=0), dict(nodes=257), dict(q_heads=9), dict(tree_heads=3), dict(cache_heads=0),
                dict(head_dim=96), dict(capacity=-1), dict(capacity=1 << 31), dict(q_heads=1 << 16, cache_heads=1, tree_heads=1, nodes=256)):
        assert ws(**bad) == 0, bad
    assert lib.lrqk_tree_attention_workspace_bytes(None) == 0


def test_an_error_while_accepting_leaves_nothing_to_decode_twice():
    from lrqk_b200 import DynamicLRQKCache

    class Layer:
        def __init__(self, fails):
            self.fails, self.steps = fails, 0

        def _decode(self, q, k, v, attention):
            if self.fails:
                raise RuntimeError("full")
            self.steps += 1

        def close(self):
            pass

    cache = DynamicLRQKCache(r=8, num_active_tokens=16, lite_tokens=4, num_key_value_groups=1)
    cache.lwattn = {0: Layer(False), 1: Layer(True)}
    row = torch.zeros(1, 1, 3, 64)
    cache._drafted = {0: (row, row, row), 1: (row, row, row)}
    with pytest.raises(RuntimeError, match="full"):
        cache.accept([0, 2])
    with pytest.raises(RuntimeError, match="no drafted"):
        cache.accept([0, 2])
    assert cache.lwattn[0].steps == 2
