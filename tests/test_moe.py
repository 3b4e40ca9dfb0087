"""Mixture-of-experts layer without a GPU: sizes and refusals."""
import pytest
import torch

import axon_b200 as ax


def test_workspace_size():
    L = ax.lib()
    one = L.axq_moe_workspace_size(1, 8, 2048, 1408)
    assert one > 0 and one % 256 == 0
    assert L.axq_moe_workspace_size(64, 8, 2048, 1408) == L.axq_moe_workspace_size(5000, 8, 2048, 1408)  # passes share it
    assert L.axq_moe_workspace_size(1, 0, 2048, 1408) == 0 and L.axq_moe_workspace_size(-1, 1, 1, 1) == 0


def test_c_refusals():
    L, S = ax.lib(), ax.Status
    p = 4096  # never dereferenced

    def route(dtype=0, tokens=2, experts=8, top_k=2, hidden=64):
        return L.axq_moe_route(dtype, p, p, p, p, tokens, experts, top_k, hidden, 1, None)

    assert route(dtype=3) == S.ERR_UNSUPPORTED
    assert route(experts=1025) == S.ERR_UNSUPPORTED and b"experts" in L.axq_last_error()
    assert route(top_k=33, experts=64) == S.ERR_UNSUPPORTED and route(top_k=0) == S.ERR_UNSUPPORTED
    assert route(top_k=9) == S.ERR_INVALID and route(hidden=0) == S.ERR_INVALID and route(tokens=-1) == S.ERR_INVALID
    assert route(tokens=0) == 0

    def mlp(fmt=5, down=2, dtype=0, tokens=2, experts=8, top_k=2, hidden=64, ffn=64):
        return L.axq_moe_mlp(fmt, p, None, p, None, down, p, None, dtype, p, p, p, p, tokens, experts, top_k, hidden, ffn, p,
                             1 << 30, None)

    assert mlp(fmt=0) == S.ERR_UNSUPPORTED and mlp(down=8) == S.ERR_UNSUPPORTED and mlp(dtype=7) == S.ERR_UNSUPPORTED
    assert mlp(fmt=64, ffn=128) == S.ERR_UNSUPPORTED and b"multiples of 128" in L.axq_last_error()
    assert mlp(experts=0) == S.ERR_UNSUPPORTED and mlp(ffn=-1) == S.ERR_INVALID and mlp(tokens=(1 << 24) + 1) == S.ERR_INVALID
    assert mlp(tokens=0) == 0 and mlp(hidden=0) == 0


def test_python_refusals():
    with pytest.raises(ax.AxqError, match="CUDA"):
        ax.moe_route(torch.zeros(1, 64), torch.zeros(4, 64), 2)
    with pytest.raises(ax.AxqError, match="float32, float16 or bfloat16"):
        ax.moe_route(torch.zeros(1, 64, dtype=torch.float64), torch.zeros(4, 64), 2)
