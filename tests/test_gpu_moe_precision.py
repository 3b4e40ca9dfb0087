"""How many bits the mixture-of-experts layer keeps, where few terms make the rounding steps visible."""
import numpy as np
import pytest
import torch

import axon_b200 as ax
from moe_ref import Weights, layer
from test_gpu_moe import F8Weights, FORMATS, _q

pytestmark = pytest.mark.gpu


def _half_step_bf16(v):
    """Half the distance between bf16 values around v (8 significant bits)."""
    return np.ldexp(1.0, np.frexp(np.abs(v))[1] - 9)


def _one_feature(orc, fmt, rng):
    """Experts with a single hidden feature (e4m3: 128 of which one is not 0), so that y is one product."""
    if fmt != "F8":
        return [Weights(orc, fmt, 3, r, c, rng) for r, c in ((1, 256), (1, 256), (256, 1))]
    w = [F8Weights(3, r, c, rng) for r, c in ((128, 256), (128, 256), (256, 128))]
    for m in w[:2]:
        m.q.data.view(torch.uint8).view(3, 128, 256)[:, 1:] = 0
        m.value[:, 1:] = m.size[:, 1:] = 0
    return w


@pytest.mark.parametrize("fmt", FORMATS + ["F8"])
def test_bf16_result_is_rounded_once(cuda, orc, fmt):
    """y = w_down * h with one h for each token: y lies within half a bf16 step of the exact value, but for the errors of
    the fp32 sums.  A hidden activation held in 11 bits would be off by up to 2^-12 of it, several times those errors."""
    rng = np.random.default_rng(31 + len(fmt))
    gate, up, down = _one_feature(orc, fmt, rng)
    T, K = 24, 1
    x = np.zeros((T, 256))  # one element each: sums of magnitudes are the magnitudes
    x[np.arange(T), rng.integers(0, 256, T)] = 1 + rng.random(T)
    xd = torch.from_numpy(x).to(torch.bfloat16).cuda()
    ids = rng.integers(0, 3, (T, K)).astype(np.int32)
    p = np.ones((T, K), np.float32)
    w = [v.q if fmt == "F8" else _q(v) for v in (gate, up, down)]
    got = ax.moe_mlp_q(xd, torch.from_numpy(ids).cuda(), torch.from_numpy(p).cuda(), *w, experts=3)
    y, tol = layer(xd.double().cpu().numpy(), ids, p, gate, up, down, 0.0)  # no rounding of the result
    err = np.abs(got.double().cpu().numpy() - y)
    bound = tol + _half_step_bf16(np.abs(y) + tol)
    assert np.isfinite(err).all() and (err <= bound).all(), (err / bound).max()


@pytest.mark.parametrize("fmt", ["Q2_K", "Q3_K", "Q4_K", "Q5_K", "Q6_K"])
@pytest.mark.parametrize("T", [4, 24])
def test_fp32_sums(cuda, orc, fmt, T):
    """An fp32 layer as a whole (2-norms): the sums are fp32 in earnest, as a plain computation's.

    An addition of the tensor core may truncate, by up to 2^-23 of the running sum and always toward zero.  Over four in a
    row, the running sum growing as the square root, that is up to 3.1 * 2^-23 of the chain's sum and half of it on
    average.  A chain covers 64 elements (32 of Q6_K); chains have signs and errors of their own, which add as squares, so
    the sum of all is off by 1.5 * 2^-23 of itself.  Sums of codes are up to twice the size of what is left once their
    offset is taken off, and three products follow one another: 2 * sqrt(3) * 1.5 * 2^-23 = 6.2e-7; with fp32's own
    roundings beside that, less than 2^-20 (9.5e-7).  Sixteen or 32 additions in a row were off by 1.4 to 3.9e-6."""
    rng = np.random.default_rng(50 + T)
    E, K, hidden, ffn = 4, 2, 1024, 512
    gate, up = (Weights(orc, fmt, E, ffn, hidden, rng) for _ in range(2))
    down = Weights(orc, fmt, E, hidden, ffn, rng)
    x = (rng.standard_normal((T, hidden)) / np.sqrt(hidden)).astype(np.float32)
    ids = np.stack([rng.permutation(E)[:K] for _ in range(T)]).astype(np.int32)
    p = rng.random((T, K)).astype(np.float32)
    got = ax.moe_mlp_q(*(torch.from_numpy(v).cuda() for v in (x, ids, p)), _q(gate), _q(up), _q(down), experts=E)
    y, _ = layer(x.astype(np.float64), ids, p, gate, up, down, 0.0)
    assert np.linalg.norm(got.double().cpu().numpy() - y) <= 2.0 ** -20 * np.linalg.norm(y)
