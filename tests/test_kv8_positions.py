"""Positions of KVCache8 calls: whole numbers or int64 device tensors."""
import numpy as np
import pytest
import torch

from fathom_b200.kv8 import _position


def test_positions_are_whole_numbers():
    cpu = torch.device("cpu")
    assert _position(5, 1, cpu, "end") == _position(np.int64(5), 1, cpu, "end") == (5, None)
    for bad in (5.5, 5.0, "5", None):
        with pytest.raises(TypeError):
            _position(bad, 1, cpu, "end")
