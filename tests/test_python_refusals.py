"""Arguments that the Python calls of the e4m3 blocks and the experts refuse by themselves (no GPU)."""
from types import SimpleNamespace

import pytest
import torch

import axon_b200 as ax
from axon_b200 import f8


def test_stream_of_another_device():
    """Its work would have gone to the tensors' device's current stream, in no order with the stream asked for."""
    with pytest.raises(ax.AxqError, match="stream is on cuda:1, not on cuda:0"):
        f8._on(torch.device("cuda", 0), SimpleNamespace(device_index=1))
