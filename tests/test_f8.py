"""e4m3 blocks without a GPU: the codec's definition, sizes and refusals."""
import numpy as np
import pytest
import torch

import axon_b200 as ax
from f8_ref import e4m3_round, e4m3_values, pack, unpack


def test_codec_table_matches_torch():
    v = e4m3_values()
    t = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(v.astype(np.float32), t, equal_nan=True)
    r = np.random.default_rng(0).standard_normal(20000).astype(np.float32) * 100
    r[:512] = np.concatenate([v, (v + np.roll(v, -1)) / 2]).astype(np.float32)
    r = np.clip(np.nan_to_num(r), -448, 448)
    assert np.array_equal(e4m3_round(r), torch.from_numpy(r).to(torch.float8_e4m3fn).view(torch.uint8).numpy())


def test_packing_error_is_half_a_step():
    x = np.random.default_rng(1).standard_normal((130, 300)).astype(np.float32)
    for rows in (1, 128):
        c, s = pack(x, rows)
        big = np.repeat(np.repeat(s.astype(np.float64), rows, 0)[:130], 128, 1)[:, :300]
        # relative 2^-4 of the value, half a subnormal step (2^-10 of the scale) near zero
        assert (np.abs(unpack(c, s, rows) - x) <= np.maximum(2.0 ** -4 * np.abs(x), 2.0 ** -10 * big) * (1 + 1e-6)).all()


def test_tensor_shapes():
    q = ax.F8Tensor.empty(130, 300, 128, device="cpu")
    assert q.data.shape == (130, 304) and q.scales.shape == (2, 3)
    q = ax.F8Tensor.empty(5, 16, 1, device="cpu")
    assert q.data.shape == (5, 16) and q.scales.shape == (5, 1)
    with pytest.raises(ax.AxqError, match="block_rows"):
        ax.F8Tensor.empty(4, 4, 64, device="cpu")


def test_workspace_size():
    L = ax.lib()
    assert L.axq_linear_f8_workspace_size(3, 4096, 7) == 256
    assert L.axq_linear_f8_workspace_size(2, 300, 3) == 256 + 1024 + 256  # 3 x 304 codes, 3 x 3 scales
    assert L.axq_linear_f8_workspace_size(0, -1, 3) == 0


def test_c_refusals():
    """Every bad argument is refused before a pointer is touched."""
    L, S = ax.lib(), ax.Status
    p = 4096  # never dereferenced
    assert L.axq_quantize_f8(3, p, p, 16, p, 4, 4, 1, None) == S.ERR_UNSUPPORTED
    assert L.axq_quantize_f8(0, p, p, 16, p, 4, 4, 2, None) == S.ERR_INVALID and b"block_rows" in L.axq_last_error()
    assert L.axq_quantize_f8(0, p, p, 16, p, -4, 4, 1, None) == S.ERR_INVALID
    assert L.axq_quantize_f8(0, p, p, 16, p, 1 << 25, 1 << 20, 1, None) == S.ERR_INVALID
    assert b"too large" in L.axq_last_error()
    assert L.axq_quantize_f8(0, None, None, 0, None, 0, 4, 1, None) == 0
    assert L.axq_dequantize_f8(p, 20, p, 1, p, 4, 20, None) == S.ERR_INVALID and b"multiple of 16" in L.axq_last_error()
    assert L.axq_dequantize_f8(p, 16, p, 1, p, 4, 20, None) == S.ERR_INVALID
    args = dict(w=p, w_ld=16, ws=p, xt=0, x=p, x_ld=16, xs=None, bias=None, yt=0, y=p, M=4, K=16, N=2, ws2=p, wb=1 << 20)

    def call(**kw):
        return L.axq_linear_f8(*{**args, **kw}.values(), None)

    assert call(xt=9) == S.ERR_UNSUPPORTED and call(yt=3) == S.ERR_UNSUPPORTED
    assert call(M=-1) == S.ERR_INVALID and call(N=(1 << 24) + 1) == S.ERR_INVALID
    assert call(M=0, y=None) == 0 and call(N=0, y=None) == 0


def test_python_refusals():
    w = ax.F8Tensor.empty(128, 128, device="cpu")
    with pytest.raises(ax.AxqError, match="CUDA"):
        ax.linear_f8(torch.zeros(1, 128), w)
    with pytest.raises(ax.AxqError, match="CUDA"):
        ax.quantize_f8(w, torch.zeros(128, 128))
    with pytest.raises(ax.AxqError, match="float32, float16 or bfloat16"):
        ax.quantize_f8(w, torch.zeros(128, 128, dtype=torch.float64))
