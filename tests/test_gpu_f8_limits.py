"""e4m3 blocks at the ends of their ranges: K beyond one kernel's shared memory, matrices beyond 4 GB, packed x in a graph.

Codes of 0 and 1 with scales of 1, 2 and 4: every sum is an integer below 2^24, exact in fp32 in any order."""
import pytest
import torch

import axon_b200 as ax

pytestmark = pytest.mark.gpu


def _ones(rows, cols, block_rows, gen, scale_bits=3):
    """An F8Tensor of codes 0 and 1 (0x38) under scales 1, 2, .. 2^(scale_bits - 1)."""
    q = ax.F8Tensor.empty(rows, cols, block_rows)
    q.data.view(torch.uint8).random_(0, 2, generator=gen).mul_(0x38)
    q.scales.copy_(torch.randint(0, scale_bits, q.scales.shape, device="cuda", generator=gen).exp2())
    return q


def _value(q, rows):
    """float64 values of these rows (a slice)."""
    r = torch.arange(*rows.indices(q.shape[0]), device="cuda")
    s = q.scales[r // q.block_rows].double().repeat_interleave(128, 1)[:, :q.shape[1]]
    return q.data[rows, :q.shape[1]].double() * s


# 64 tokens, 8 ranks: a CTA's 700 blocks of scales leave room for two stages, 701 do not and the pair kernel takes over
@pytest.mark.parametrize("N,K", [(64, 700 * 1024), (64, 701 * 1024), (33, 701 * 1024), (40, 1 << 20), (16, 3000 * 1024)])
def test_long_k(cuda, N, K):
    gen = torch.Generator(device="cuda").manual_seed(K)
    M = 64
    x, w = _ones(N, K, 1, gen, 1), _ones(M, K, 128, gen)
    y = ax.linear_f8(x, w)
    want = _value(x, slice(None)) @ _value(w, slice(None)).t()
    assert want.max() < 2 ** 24 and torch.equal(y.double(), want)


@pytest.mark.parametrize("N", [2, 40, 130])
def test_weights_beyond_4_gb(cuda, N):
    gen = torch.Generator(device="cuda").manual_seed(N)
    M, K = 66000, 65600
    w = _ones(M, K, 128, gen, 2)
    x = _ones(N, K, 1, gen, 2)
    y = ax.linear_f8(x, w)
    for rows in (slice(0, 200), slice(M - 300, M)):
        want = _value(x, slice(None)) @ _value(w, rows).t()
        assert want.max() < 2 ** 24 and torch.equal(y[:, rows].double(), want)


def test_results_beyond_4_gb(cuda):
    gen = torch.Generator(device="cuda").manual_seed(5)
    N, M, K = 4200, 300100, 128
    x, w = _ones(N, K, 1, gen), _ones(M, K, 128, gen)
    y = ax.linear_f8(x, w)
    for t in (slice(0, 100), slice(N - 100, N)):
        for rows in (slice(0, 300), slice(M - 300, M)):
            assert torch.equal(y[t, rows].double(), _value(x, t) @ _value(w, rows).t())


@pytest.mark.parametrize("block_rows", [1, 128])
def test_packing_beyond_4_gb(cuda, block_rows):
    rows, cols, last = 290048, 16400, 256
    src = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    q = ax.quantize_f8(ax.F8Tensor.empty(rows, cols, block_rows), src)
    tail = ax.quantize_f8(ax.F8Tensor.empty(last, cols, block_rows), src[-last:].clone())
    del src
    assert torch.equal(q.data[-last:, :cols].view(torch.uint8), tail.data[:, :cols].view(torch.uint8))
    assert torch.equal(q.scales[-tail.scales.shape[0]:], tail.scales)
    back = ax.dequantize_f8(torch.empty(rows, cols, device="cuda"), q)
    assert torch.equal(back[-last:], ax.dequantize_f8(torch.empty(last, cols, device="cuda"), tail))


@pytest.mark.parametrize("N", [1, 30, 64, 100, 600])
def test_packed_x_in_a_graph(cuda, N):
    """Captured behind the packing of both operands, and replayed on other inputs in the same memory."""
    gen = torch.Generator(device="cuda").manual_seed(N)
    src = [(torch.randn(N, 700, device="cuda", generator=gen), torch.randn(300, 700, device="cuda", generator=gen)) for _ in range(3)]
    xs, ws = torch.empty_like(src[0][0]), torch.empty_like(src[0][1])
    x, w = ax.F8Tensor.empty(N, 700, 1), ax.F8Tensor.empty(300, 700)

    def step():
        return ax.linear_f8(ax.quantize_f8(x, xs), ax.quantize_f8(w, ws))

    want = []
    for a, b in src:
        xs.copy_(a), ws.copy_(b)
        want.append(step())
        torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = step()
    for _ in range(5):
        for (a, b), v in zip(src, want):
            xs.copy_(a), ws.copy_(b)
            g.replay()
            assert torch.equal(y, v)
