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


def test_kinds_of_weights():
    from axon_b200 import moe

    q = ax.QTensor.empty(8, 32, ax.QuantFormat.Q8_0, device="cpu")
    d = ax.QTensor.empty(2 * 32, 4, ax.QuantFormat.Q8_0, device="cpu")
    for bad in (None, [1], torch.zeros(8, 32)):
        for at, name in enumerate(("w_gate", "w_up", "w_down")):
            w = [q, q, d]
            w[at] = bad
            with pytest.raises(ax.AxqError, match=f"{name} must be a QTensor or an F8Tensor"):
                moe._experts(*w, 2, 32)
    none = ax.QTensor(q.data, (8, 32), ax.QuantFormat.NONE)
    with pytest.raises(ax.AxqError, match="block format"):
        moe._experts(none, q, d, 2, 32)
