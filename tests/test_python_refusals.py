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


def test_number_of_choices():
    """Before anything is allocated for them: a negative number ended in torch's own error, a huge one out of memory."""
    from axon_b200 import moe

    x = torch.zeros(3, 8)
    for k in (0, -1):
        with pytest.raises(ax.AxqError, match="top_k must be positive"):
            moe._choices(x, 4, k)
    for k in (5, 1 << 40):
        with pytest.raises(ax.AxqError, match="larger than the number of experts"):
            moe._choices(x, 4, k)
    ids, weights = moe._choices(x, 4, 4)
    assert ids.shape == weights.shape == (3, 4) and ids.dtype == torch.int32 and weights.dtype == torch.float32
