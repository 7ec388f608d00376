"""Rotary objects: on the CPU, without a device."""

from __future__ import annotations

import pytest

import onednn_flash_hip as F


@pytest.mark.parametrize("name", ["frequencies", "head_dim", "rotary_dim", "interleaved", "magnitude"])
def test_attributes_are_not_assigned(name):
    """Parameter blocks hold the frequencies' address and their number: another tensor
    in their place would be freed memory to the kernels, another number a read past it."""
    rotary = object.__new__(F.Rotary)
    with pytest.raises(AttributeError):
        setattr(rotary, name, 64)
    with pytest.raises(AttributeError):
        delattr(rotary, name)
