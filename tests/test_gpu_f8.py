"""e4m3 blocks on the GPU: packing bit by bit, the product within its bound."""
import numpy as np
import pytest
import torch

import axon_b200 as ax
from f8_ref import e4m3_values, pack, product_bound, unpack

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _rand(rng, rows, cols, kind="plain"):
    x = rng.standard_normal((rows, cols)).astype(np.float32)
    if kind == "outliers":
        x[:, rng.random(cols) < 0.02] *= 50
    if kind == "wide":  # magnitudes over the whole range of fp32
        x = np.ldexp(x, rng.integers(-140, 120, (rows, cols))).astype(np.float32)
    return x


def _same_codes(got, want):
    nan = np.isnan(e4m3_values()[want])
    assert np.array_equal(np.isnan(e4m3_values()[got]), nan)
    assert np.array_equal(got[~nan], want[~nan])


def _packed(x, block_rows):
    q = ax.F8Tensor.empty(x.shape[0], x.shape[1], block_rows)
    q.data.view(torch.uint8).fill_(0xAA)
    ax.quantize_f8(q, x)
    return q, q.data.view(torch.uint8).cpu().numpy(), q.scales.cpu().numpy()


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 127), (2, 129), (129, 256), (260, 1000), (17, 4096)])
def test_pack_bits(cuda, rows, cols, dtype, block_rows):
    rng = np.random.default_rng(rows * 1000 + cols)
    kind = "outliers" if cols > 500 else "plain"
    x = torch.from_numpy(_rand(rng, rows, cols, kind)).to(TYPES[dtype])
    q, codes, scales = _packed(x.cuda(), block_rows)
    want, s = pack(x.float().numpy(), block_rows)
    assert np.array_equal(scales, s)
    _same_codes(codes[:, :cols], want)
    assert not codes[:, cols:].any()  # the padding up to the row stride
    back = torch.empty(rows, cols, device="cuda")
    ax.dequantize_f8(back, q)
    assert np.array_equal(back.cpu().numpy(), unpack(want, s, block_rows).astype(np.float32))


@pytest.mark.parametrize("block_rows", [1, 128])
def test_pack_every_magnitude(cuda, block_rows):
    """Scales from below the smallest normal to 2^120 (the division's both paths), and quotients at the codes' ties."""
    rng = np.random.default_rng(5)
    x = _rand(rng, 256, 640, "wide")
    x[128:, :128] = np.ldexp(x[128:, :128], -60)
    # exact ties: multiples of half a code step under a scale of a power of two
    v = e4m3_values()[:127]
    x[0:128, 128:256] = 0
    x[0, 128:255] = (v + np.append(v[1:], 448)) / 2
    x[0, 255] = 448
    # a scale whose significand is all ones
    x[0:128, 256:384] = rng.standard_normal((128, 128)) * 0.1
    x[0, 256] = np.float32(448) * np.nextafter(np.float32(2), np.float32(0))
    got = _packed(torch.from_numpy(x).cuda(), block_rows)
    want, s = pack(x, block_rows)
    assert np.array_equal(got[2], s)
    _same_codes(got[1][:, :640], want)


def test_pack_special_values(cuda):
    x = np.zeros((6, 256), np.float32)
    x[0, 3], x[0, 4] = np.nan, 2.0
    x[1, :128] = -0.0
    x[2, 5], x[2, 6] = np.inf, 1.0
    x[3, 7] = np.nan  # a block of zeros and a NaN
    x[4, :] = 1e-44
    x[5, 0] = 3e38
    q, codes, scales = _packed(torch.from_numpy(x).cuda(), 1)
    with np.errstate(invalid="ignore"):
        want, s = pack(x, 1)
    assert np.array_equal(scales, s)
    _same_codes(codes, want)
    back = torch.empty(6, 256, device="cuda")
    ax.dequantize_f8(back, q)
    b = back.cpu().numpy()
    assert np.isnan(b[2, :128]).all() and np.isnan(b[0, 3]) and np.isnan(b[3, 7])
    assert b[0, 4] == 2.0 and not b[1].any() and not b[3, :7].any()


def test_unaligned_source(cuda):
    """A source that starts off a 16-byte boundary takes plain loads."""
    for dtype in TYPES.values():
        big = torch.randn(1 + 40 * 256, device="cuda").to(dtype)
        x = big[1:].view(40, 256)
        for rows in (1, 128):
            a, b = _packed(x, rows), _packed(x.clone(), rows)
            assert np.array_equal(a[1], b[1]) and np.array_equal(a[2], b[2])


def _linear_case(rng, N, M, K, dtype, bias, packed=False, out_dtype=None):
    x = torch.from_numpy(_rand(rng, N, K, "outliers")).to(TYPES[dtype]).cuda()
    w = ax.quantize_f8(ax.F8Tensor.empty(M, K), torch.from_numpy(_rand(rng, M, K) * 0.02).cuda())
    b = torch.from_numpy(rng.standard_normal(M).astype(np.float32)).cuda() if bias else None
    xq = ax.quantize_f8(ax.F8Tensor.empty(N, K, 1), x)
    # the output lies between sentinels: nothing around it may change
    want_type = TYPES[out_dtype] if out_dtype else (torch.float32 if packed else x.dtype)
    buf = torch.full((N * M + 128,), 7.0, dtype=want_type, device="cuda")
    out = buf[64:64 + N * M].view(N, M)
    got = ax.linear_f8(xq if packed else x, w, out=out, bias=b)
    assert got is out
    assert (buf[:64] == 7).all() and (buf[64 + N * M:] == 7).all()
    xv = unpack(xq.data.view(torch.uint8).cpu().numpy()[:, :K], xq.scales.cpu().numpy(), 1)
    wv = unpack(w.data.view(torch.uint8).cpu().numpy()[:, :K], w.scales.cpu().numpy(), 128)
    y = xv @ wv.T
    tol = product_bound(xv, wv, torch.finfo(want_type).eps)
    if bias:
        bv = b.double().cpu().numpy()
        y = y + bv
        tol = tol + (torch.finfo(want_type).eps / 2 + 2.0 ** -24) * (np.abs(bv) + np.abs(y))
    err = np.abs(got.double().cpu().numpy() - y)
    assert np.isfinite(err).all() and (err <= tol).all(), (err / tol).max()


@pytest.mark.parametrize("N", [1, 2, 15, 16, 17, 33, 64, 65, 128, 129, 257])
@pytest.mark.parametrize("M,K", [(1, 1), (7, 300), (128, 128), (130, 127), (384, 1000), (1000, 4096)])
def test_linear(cuda, N, M, K):
    rng = np.random.default_rng(N * 7919 + M * 31 + K)
    _linear_case(rng, N, M, K, ["fp32", "bf16", "fp16"][(N + M + K) % 3], bias=(N + M) % 2 == 0)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("N,M,K", [(3, 520, 640), (40, 300, 2000), (100, 256, 528), (700, 1100, 900), (300, 8192, 256)])
def test_linear_types_and_packed_input(cuda, N, M, K, dtype):
    rng = np.random.default_rng(N + M)
    _linear_case(rng, N, M, K, dtype, bias=True)
    _linear_case(rng, N, M, K, dtype, bias=False, packed=True)
    _linear_case(rng, N, M, K, "fp32", bias=False, out_dtype=dtype)


def test_linear_many_tiles(cuda):
    """More tiles than CTA pairs in both widths of the pair kernel, with ragged edges."""
    rng = np.random.default_rng(3)
    _linear_case(rng, 1300, 4100, 260, "bf16", bias=True)
    _linear_case(rng, 150, 20000, 130, "fp32", bias=False)


def test_linear_long_k(cuda):
    """K so long that a few tokens' scales no longer fit beside the tiles."""
    rng = np.random.default_rng(4)
    _linear_case(rng, 128, 130, 131072, "fp32", bias=False)
    _linear_case(rng, 70, 30, 400000, "fp32", bias=False)
    _linear_case(rng, 16, 64, 262144, "bf16", bias=False)


def test_linear_empty(cuda):
    w = ax.F8Tensor.empty(6, 0)
    b = torch.arange(6.0, device="cuda")
    assert torch.equal(ax.linear_f8(torch.zeros(3, 0, device="cuda"), w, bias=b), b.expand(3, 6))
    assert not ax.linear_f8(torch.zeros(3, 0, device="cuda"), w).any()
    w = ax.quantize_f8(ax.F8Tensor.empty(6, 40), torch.randn(6, 40, device="cuda"))
    assert ax.linear_f8(torch.zeros(0, 40, device="cuda"), w).shape == (0, 6)


def test_linear_non_finite(cuda):
    """A NaN or an infinity in one token leaves the others as they are."""
    for N in (5, 200):
        x = torch.randn(N, 300, device="cuda")
        w = ax.quantize_f8(ax.F8Tensor.empty(140, 300), torch.randn(140, 300, device="cuda"))
        good = ax.linear_f8(x, w)
        bad = x.clone()
        bad[2, 17], bad[4, 290] = float("nan"), float("inf")
        y = ax.linear_f8(bad, w)
        keep = [i for i in range(N) if i not in (2, 4)]
        assert torch.equal(y[keep], good[keep])
        assert torch.isnan(y[2]).all() and torch.isnan(y[4]).all()


def test_streams_and_graphs(cuda):
    """Another stream, two captured graphs at once and repeated calls give the same bits."""
    x1, x2 = torch.randn(9, 1024, device="cuda"), torch.randn(200, 1024, device="cuda")
    w = ax.quantize_f8(ax.F8Tensor.empty(700, 1024), torch.randn(700, 1024, device="cuda"))
    a, b = ax.linear_f8(x1, w), ax.linear_f8(x2, w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    c = ax.linear_f8(x1, w, stream=s)
    s.synchronize()
    assert torch.equal(a, c)
    graphs, outs = [], []
    for x in (x1, x2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ax.linear_f8(x, w))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for o in outs:
        o.zero_()
    torch.cuda.synchronize()
    for _ in range(5):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], a) and torch.equal(outs[1], b)


def test_refusals(cuda):
    w = ax.quantize_f8(ax.F8Tensor.empty(256, 256), torch.randn(256, 256, device="cuda"))
    x = torch.randn(4, 256, device="cuda")
    with pytest.raises(ax.AxqError, match=r"\[N x 256\]"):
        ax.linear_f8(x[:, :128].contiguous(), w)
    with pytest.raises(ax.AxqError, match="contiguous"):
        ax.linear_f8(torch.randn(256, 4, device="cuda").t(), w)
    with pytest.raises(ax.AxqError, match="128 x 128"):
        ax.linear_f8(x, ax.F8Tensor.empty(256, 256, 1))
    with pytest.raises(ax.AxqError, match="1 x 128"):
        ax.linear_f8(ax.F8Tensor.empty(4, 256, 128), w)
    with pytest.raises(ax.AxqError, match="scales must be"):
        ax.linear_f8(x, ax.F8Tensor(w.data, w.scales[:1], (256, 256)))
    with pytest.raises(ax.AxqError, match="bias"):
        ax.linear_f8(x, w, bias=torch.zeros(255, device="cuda"))
    with pytest.raises(ax.AxqError, match="out must be"):
        ax.linear_f8(x, w, out=torch.empty(4, 255, device="cuda"))
    L = ax.lib()
    ws = torch.empty(512, dtype=torch.uint8, device="cuda")
    y = torch.empty(4, 256, device="cuda")
    st = L.axq_linear_f8(w.data.data_ptr(), 256, w.scales.data_ptr(), 0, x.data_ptr(), 256, None, None, 0, y.data_ptr(), 256,
                         256, 4, ws.data_ptr(), 512, None)
    assert st == ax.Status.ERR_WORKSPACE
    cpu = torch.empty(4, 256)
    big = torch.empty(8192, dtype=torch.uint8, device="cuda")
    st = L.axq_linear_f8(w.data.data_ptr(), 256, w.scales.data_ptr(), 0, cpu.data_ptr(), 256, None, None, 0, y.data_ptr(), 256,
                         256, 4, big.data_ptr(), 8192, None)
    assert st == ax.Status.ERR_INVALID


def test_overlaps_are_refused(cuda):
    w = ax.quantize_f8(ax.F8Tensor.empty(256, 256), torch.randn(256, 256, device="cuda"))
    x = torch.randn(4, 256, device="cuda")
    both = torch.zeros(5, 256, device="cuda")
    for first in (0, 1):  # the same rows, and shifted by one
        with pytest.raises(ax.AxqError, match="must not overlap x"):
            ax.linear_f8(both[:4], w, out=both[first:first + 4])
    room = torch.zeros(4 * 256 * 4, dtype=torch.uint8, device="cuda")
    xq = ax.F8Tensor(room[:1024].view(torch.float8_e4m3fn).view(4, 256), torch.zeros(4, 2, device="cuda"), (4, 256), 1)
    with pytest.raises(ax.AxqError, match="must not overlap x"):
        ax.linear_f8(xq, w, out=room.view(torch.float32).view(4, 256))
    bias = torch.zeros(4 * 256, device="cuda")
    with pytest.raises(ax.AxqError, match="the bias"):
        ax.linear_f8(x, w, bias=bias[256:512], out=bias.view(4, 256))
    src = torch.zeros(64, 64, device="cuda")
    codes = ax.F8Tensor(src.view(torch.float8_e4m3fn).view(-1)[:64 * 64].view(64, 64), torch.empty(1, 1, device="cuda"), (64, 64))
    with pytest.raises(ax.AxqError, match="must not overlap"):
        ax.quantize_f8(codes, src)
    with pytest.raises(ax.AxqError, match="must not overlap"):
        ax.dequantize_f8(src, codes)
    rows = torch.zeros(8, 256, device="cuda")
    rows[:4] = x
    assert torch.equal(ax.linear_f8(rows[:4], w, out=rows[4:]), ax.linear_f8(x, w))  # neighbours do not
