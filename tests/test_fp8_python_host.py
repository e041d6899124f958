"""The Python side of a cache held in 8 bits without a GPU."""
import sys
from pathlib import Path

import pytest
import torch

import qmm as Q

sys.path.insert(0, str(Path(Q.__file__).parent))


def test_rows_of_a_bfloat16_layer_are_not_read_back():
    """Its cache has no scales: refused by what it is, before anything is made."""
    from attention_layer import AttentionLayer

    layer = AttentionLayer.__new__(AttentionLayer)
    layer.eight, layer.Hkv, layer.D, layer.caches = False, 2, 64, ()
    with pytest.raises(ValueError, match="cache='e4m3'"):
        layer.read(torch.zeros(3, dtype=torch.int32), None)
