"""Refusals of the token choice that need no GPU."""
import ctypes as C

import pytest
import torch

from lrqk_b200 import _lib, sample_tokens


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError):
        sample_tokens(torch.zeros(2, 10), torch.zeros(2))


def test_the_entry_needs_a_device_first():
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    assert _lib.lib().lrqk_sample_tokens(C.byref(_lib.SampleArgs()), None) == _lib.ENODEVICE
