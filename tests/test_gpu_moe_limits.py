"""Mixture-of-experts layer at the ends of its ranges: experts beyond 4 GB, magnitudes far below their neighbours'."""
import numpy as np
import pytest
import torch

import axon_b200 as ax
from moe_ref import Weights, layer
from test_gpu_moe import FORMATS, TYPES, _case, _q

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("T,E,K,hidden,ffn", [(5, 4, 2, 384, 256), (20, 2, 2, 640, 384), (2, 5, 1, 128, 512)])
def test_e4m3_experts_in_every_type(cuda, orc, T, E, K, hidden, ffn, dtype):
    """Groups of four tokens and of eight, one and two terms."""
    _case(orc, np.random.default_rng(T * hidden), "F8", "F8", T, E, K, hidden, ffn, dtype)


def _bytes(n, gen):
    """Bytes below 0x3C: as e4m3 codes and as fp16 scales no infinities or NaN, nothing above 2."""
    return torch.empty(n, dtype=torch.uint8, device="cuda").random_(0, 0x3C, generator=gen)


@pytest.mark.parametrize("fmt", ["F8", "Q8_0", "Q4_K", "Q6_K"])
def test_experts_beyond_4_gb(cuda, fmt):
    """The last expert among others, its rows past 4 GB, against the same expert by itself: the same bits."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    hidden, ffn = 16384, 49152
    if fmt == "F8":
        E, size = 6, ffn * hidden
    else:
        F = ax.QuantFormat[fmt]
        size = ax.quantized_size_2d(ffn, hidden, F)
        E = -(-(1 << 32) // size) + 1
    data = _bytes(E * size, gen)  # gate, up and down in one

    def weights(first, n):
        part = data[first * size:(first + n) * size]
        for rows, cols in ((ffn, hidden), (ffn, hidden), (hidden, ffn)):
            if fmt == "F8":
                scales = torch.full((n * rows // 128, cols // 128), 2.0 ** -6, device="cuda")
                yield ax.F8Tensor(part.view(torch.float8_e4m3fn).view(n * rows, cols), scales, (n * rows, cols))
            else:
                yield ax.QTensor(part, (n * rows, cols), F)

    for T in (1, 9):
        x = torch.randn(T, hidden, device="cuda", generator=gen) / hidden
        p = torch.rand(T, 1, device="cuda", generator=gen) / ffn
        ids = torch.full((T, 1), E - 1, dtype=torch.int32, device="cuda")
        y = ax.moe_mlp_q(x, ids, p, *weights(0, E), experts=E)
        alone = ax.moe_mlp_q(x, torch.zeros_like(ids), p, *weights(E - 1, 1), experts=1)
        assert torch.isfinite(y).all() and y.any() and torch.equal(y, alone)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", list(TYPES))
def test_far_below_the_largest(cuda, orc, fmt, dtype):
    """Elements 2^-10 to 2^-38 below the largest of their 256: held to within 2^-33 of it."""
    rng = np.random.default_rng(40)
    gate, up = (Weights(orc, fmt, 2, 16, 512, rng) for _ in range(2))
    down = Weights(orc, "Q8_0", 2, 512, 16, rng)
    T = 6
    # fp16 reaches from 2^15 down to 2^-24
    top = 2.0 ** 12 if dtype == "fp16" else 1.0
    x = np.ldexp(rng.uniform(1, 2, (T, 512)) * top, -rng.integers(10, 38, (T, 512)))
    x[np.arange(T), rng.integers(0, 256, T)] = top * 1.5
    x[:3, 256:] *= 2.0 ** -4  # the second group has a largest of its own
    xd = torch.from_numpy(x).to(TYPES[dtype]).cuda()
    ids = np.array([[0, 1]] * T, np.int32)
    p = np.full((T, 2), 1 / top ** 2 / 16, np.float32)
    got = ax.moe_mlp_q(xd, torch.from_numpy(ids).cuda(), torch.from_numpy(p).cuda(), _q(gate), _q(up), _q(down), experts=2)
    y, tol = layer(xd.double().cpu().numpy(), ids, p, gate, up, down, torch.finfo(xd.dtype).eps)
    err = np.abs(got.double().cpu().numpy() - y)
    assert np.isfinite(err).all() and (err <= tol).all(), (err / tol).max()
