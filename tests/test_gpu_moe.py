"""Mixture-of-experts layer on the GPU against its definition in 64 bits, within derived bounds."""
import numpy as np
import pytest
import torch

import axon_b200 as ax
from f8_ref import unpack
from moe_ref import Weights, layer, route

pytestmark = pytest.mark.gpu

FORMATS = ["Q8_0", "Q4_0", "Q2_K", "Q3_K", "Q4_K", "Q5_K", "Q6_K"]
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _q(w):
    e, r, c = w.shape
    return ax.QTensor(torch.from_numpy(w.packed).cuda(), (e * r, c), ax.QuantFormat[w.fmt])


class F8Weights:
    def __init__(self, experts, rows, cols, rng):
        self.shape = (experts, rows, cols)
        w = torch.from_numpy(rng.standard_normal((experts * rows, cols)).astype(np.float32)).cuda()
        self.q = ax.quantize_f8(ax.F8Tensor.empty(experts * rows, cols), w)
        v = unpack(self.q.data.view(torch.uint8).cpu().numpy(), self.q.scales.cpu().numpy(), 128)
        self.value = v.reshape(self.shape)
        self.size = np.abs(self.value)


def _case(orc, rng, fmt, fmt_down, T, E, K, hidden, ffn, dtype="fp32", ids=None):
    """Runs moe_mlp_q and checks it; returns what it ran on."""
    if fmt == "F8":
        gate, up, down = F8Weights(E, ffn, hidden, rng), F8Weights(E, ffn, hidden, rng), F8Weights(E, hidden, ffn, rng)
        q = [w.q for w in (gate, up, down)]
    else:
        gate, up = (Weights(orc, fmt, E, ffn, hidden, rng) for _ in range(2))
        down = Weights(orc, fmt_down, E, hidden, ffn, rng)
        q = [_q(w) for w in (gate, up, down)]
    # magnitudes that keep fp16 results finite
    x = torch.from_numpy((rng.standard_normal((T, hidden)) / np.sqrt(hidden)).astype(np.float32)).to(TYPES[dtype]).cuda()
    if ids is None:
        ids = np.stack([rng.permutation(E)[:K] for _ in range(T)]).astype(np.int32).reshape(T, K)
    p = rng.random((T, ids.shape[1])).astype(np.float32) / ffn
    args = (x, torch.from_numpy(ids).cuda(), torch.from_numpy(p).cuda(), *q)
    buf = torch.full((T * hidden + 128,), 7.0, dtype=x.dtype, device="cuda")
    out = buf[64:64 + T * hidden].view(T, hidden)
    got = ax.moe_mlp_q(*args, experts=E, out=out)
    assert got is out and (buf[:64] == 7).all() and (buf[64 + T * hidden:] == 7).all()
    y, tol = layer(x.double().cpu().numpy(), ids, p, gate, up, down, torch.finfo(x.dtype).eps)
    err = np.abs(got.double().cpu().numpy() - y)
    assert np.isfinite(err).all() and (err <= tol).all(), (err / tol).max()
    assert torch.equal(ax.moe_mlp_q(*args, experts=E), got)  # the same bits again
    return args


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("T,E,K,hidden,ffn", [(1, 4, 2, 512, 256), (3, 5, 3, 300, 70), (9, 2, 1, 768, 2304), (40, 3, 2, 256, 48)])
def test_formats(cuda, orc, fmt, T, E, K, hidden, ffn):
    rng = np.random.default_rng(T * 100 + hidden)
    down = FORMATS[(FORMATS.index(fmt) + 3) % 7]
    _case(orc, rng, fmt, down, T, E, K, hidden, ffn, ["fp32", "bf16", "fp16"][(T + FORMATS.index(fmt)) % 3])


@pytest.mark.parametrize("T,E,K,hidden,ffn", [(1, 3, 2, 128, 128), (5, 4, 2, 384, 256), (20, 2, 2, 2432, 640)])
def test_e4m3_experts(cuda, orc, T, E, K, hidden, ffn):
    rng = np.random.default_rng(T + hidden)
    _case(orc, rng, "F8", "F8", T, E, K, hidden, ffn, ["fp32", "bf16", "fp16"][T % 3])


@pytest.mark.parametrize("hidden,ffn", [(1, 1), (31, 33), (257, 15), (513, 600), (5000, 100), (40, 4500)])
def test_odd_sizes(cuda, orc, hidden, ffn):
    rng = np.random.default_rng(hidden + ffn)
    for fmt, down in (("Q4_K", "Q8_0"), ("Q4_0", "Q6_K"), ("Q3_K", "Q2_K")):
        _case(orc, rng, fmt, down, 2, 3, 2, hidden, ffn)


def test_token_counts(cuda, orc):
    """Around the groups' borders, one expert for all tokens, and more choices than one pass takes."""
    rng = np.random.default_rng(8)
    for T in (4, 5, 8, 12, 17):
        _case(orc, rng, "Q4_K", "Q6_K", T, 1, 1, 256, 64)
    _case(orc, rng, "Q5_K", "Q4_K", 300, 3, 2, 256, 40)
    _case(orc, rng, "Q2_K", "Q3_K", 40, 40, 32, 256, 16)


def test_absent_and_repeated_experts(cuda, orc):
    rng = np.random.default_rng(9)
    ids = np.array([[0, -1, 2], [7, 3, -5], [1, 1, 1], [-1, -1, -1], [2147483647, 0, -2147483648], [3, 0, 3]], np.int32)
    args = _case(orc, rng, "Q4_K", "Q6_K", 6, 4, 3, 512, 100, ids=ids)
    y = ax.moe_mlp_q(*args, experts=4)
    assert not y[3].any()  # a padded token


def test_ranges(cuda, orc):
    """Activations over fp32's range in one row and from row to row; a non-finite token leaves the others alone."""
    rng = np.random.default_rng(10)
    gate, up = (Weights(orc, "Q4_K", 2, 32, 512, rng) for _ in range(2))
    down = Weights(orc, "Q6_K", 2, 512, 32, rng)
    # the same kind of x at scales far apart
    x = np.abs(rng.standard_normal((5, 512))).astype(np.float32)
    x[1] *= 1e12
    x[2] *= 1e-12
    x[3, :256] *= 1e9
    x[4, ::2] = 0
    ids = np.array([[0, 1]] * 5, np.int32)
    p = np.full((5, 2), 0.5, np.float32)
    w = [_q(v) for v in (gate, up, down)]
    xd = torch.from_numpy(x).cuda()
    got = ax.moe_mlp_q(xd, torch.from_numpy(ids).cuda(), torch.from_numpy(p).cuda(), *w, experts=2)
    y, tol = layer(x.astype(np.float64), ids, p, gate, up, down, 2.0 ** -23)
    assert (np.abs(got.double().cpu().numpy() - y) <= tol).all()
    bad = xd.clone()
    bad[1, 300], bad[3, 5] = float("nan"), float("inf")
    z = ax.moe_mlp_q(bad, torch.from_numpy(ids).cuda(), torch.from_numpy(p).cuda(), *w, experts=2)
    assert torch.equal(z[[0, 2, 4]], got[[0, 2, 4]]) and not torch.isfinite(z[1]).any() and not torch.isfinite(z[3]).any()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("T,E,K,hidden", [(1, 64, 8, 2048), (3, 4, 4, 31), (9, 257, 5, 1024), (130, 8, 2, 512), (4, 1024, 32, 256),
                                          (2, 1, 1, 7)])
def test_route(cuda, T, E, K, hidden, dtype):
    rng = np.random.default_rng(T + E)
    x = torch.from_numpy(rng.standard_normal((T, hidden)).astype(np.float32)).to(TYPES[dtype]).cuda()
    w = (rng.standard_normal((E, hidden)) / np.sqrt(hidden)).astype(np.float32)
    xv = x.double().cpu().numpy()
    ids, logits, err = route(xv, w.astype(np.float64), K)
    for normalize in (True, False):
        got, p = ax.moe_route(x, torch.from_numpy(w).cuda(), K, normalize=normalize)
        got, p = got.cpu().numpy(), p.double().cpu().numpy()
        assert got.dtype == np.int32 and (np.sort(got, 1)[:, 1:] != np.sort(got, 1)[:, :-1]).all()
        l = np.take_along_axis(logits, got, 1)
        e = err.max(axis=1, keepdims=True)
        # each choice is as large as the 64-bit one at its place, up to the logits' errors
        assert (np.abs(l - np.take_along_axis(logits, ids, 1)) <= 2 * e).all()
        z = np.exp(l - logits.max(axis=1, keepdims=True))
        want = z / (z.sum(1, keepdims=True) if normalize else np.exp(logits - logits.max(1, keepdims=True)).sum(1, keepdims=True))
        # a weight moves by the errors of its logit and of the sum's; expf and the sum add a few units
        assert (np.abs(p - want) <= want * (4 * e + (K + E + 16) * 2.0 ** -24)).all()


def test_route_ties_and_nan(cuda):
    w = torch.randn(12, 256, device="cuda")
    w[3] = w[9]
    w[7] = w[9]
    x = w[9:10].clone()
    ids, p = ax.moe_route(x, w, 4)
    assert ids[0, :3].tolist() == [3, 7, 9] and p[0, 0] == p[0, 1] == p[0, 2]
    ids, _ = ax.moe_route(torch.zeros(2, 256, device="cuda"), w, 5)
    assert ids.tolist() == [[0, 1, 2, 3, 4]] * 2
    w[5, 0] = float("nan")
    ids, _ = ax.moe_route(x, w, 12)
    assert sorted(ids[0].tolist()) == list(range(12)) and ids[0, 11] == 5


def test_whole_layer_beside_linear_f8(cuda, orc):
    """A decoder step as a model would run it: projection, router, experts, projection; each op against its own bound."""
    rng = np.random.default_rng(12)
    T, hidden, ffn, E, K = 5, 512, 256, 6, 2
    gate, up = (Weights(orc, "Q4_K", E, ffn, hidden, rng, 0.05) for _ in range(2))
    down = Weights(orc, "Q6_K", E, hidden, ffn, rng, 0.5)
    wr = torch.from_numpy((rng.standard_normal((E, hidden)) / 16).astype(np.float32)).cuda()
    w1, w2 = (ax.quantize_f8(ax.F8Tensor.empty(hidden, hidden), torch.from_numpy(
        (rng.standard_normal((hidden, hidden)) * 0.05).astype(np.float32)).cuda()) for _ in range(2))
    x = torch.from_numpy(rng.standard_normal((T, hidden)).astype(np.float32)).to(torch.bfloat16).cuda()

    def step():
        a = ax.linear_f8(x, w1)
        y, ids, p = ax.moe_q(a, wr, _gate, _up, _down, K)
        return a, y, ids, p, ax.linear_f8(y, w2)

    _gate, _up, _down = _q(gate), _q(up), _q(down)
    a, y, ids, p, z = step()
    i64, logits, err = route(a.double().cpu().numpy(), wr.double().cpu().numpy(), K)
    assert (np.abs(np.take_along_axis(logits, ids.cpu().numpy(), 1) - np.take_along_axis(logits, i64, 1))
            <= 2 * err.max(1, keepdims=True)).all()
    want, tol = layer(a.double().cpu().numpy(), ids.cpu().numpy(), p.cpu().numpy(), gate, up, down, 2.0 ** -7)
    assert (np.abs(y.double().cpu().numpy() - want) <= tol).all()
    # captured and replayed on another stream, beside an eager run: the same bits
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(side):
            g.replay()
        eager = step()
    torch.cuda.synchronize()
    for one, two, three in zip((a, y, ids, p, z), captured, eager):
        assert torch.equal(one, two) and torch.equal(one, three)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    y2, _, _ = ax.moe_q(a, wr, _gate, _up, _down, K, stream=s)
    s.synchronize()
    assert torch.equal(y2, y)


@pytest.mark.parametrize("T", [1, 8, 9, 70, 300])
def test_whole_layer_is_its_parts(cuda, orc, T):
    """moe_q against moe_route and moe_mlp_q, bit by bit, for every form of the call: three kernels, one pass, several."""
    rng = np.random.default_rng(T)
    E, K, hidden, ffn = 6, 2, 300, 520
    q = [_q(Weights(orc, f, E, r, c, rng)) for f, r, c in
         (("Q5_K", ffn, hidden), ("Q5_K", ffn, hidden), ("Q4_0", hidden, ffn))]
    wr = torch.from_numpy(rng.standard_normal((E, hidden)).astype(np.float32)).cuda()
    for dtype in TYPES.values():
        x = torch.from_numpy((rng.standard_normal((T, hidden)) * 0.05).astype(np.float32)).to(dtype).cuda()
        for normalize in (True, False):
            y, ids, p = ax.moe_q(x, wr, *q, K, normalize=normalize)
            ids2, p2 = ax.moe_route(x, wr, K, normalize=normalize)
            assert torch.equal(ids, ids2) and torch.equal(p, p2)
            assert torch.equal(y, ax.moe_mlp_q(x, ids, p, *q, experts=E))


def test_first_call_inside_a_capture(cuda):
    """In a fresh process: nothing that a call looks up once may keep it from being captured."""
    import subprocess
    import sys

    code = """
import torch, axon_b200 as ax
x = torch.randn(40, 512, device='cuda'); few = torch.randn(2, 512, device='cuda'); many = torch.randn(300, 512, device='cuda')
w = ax.quantize_f8(ax.F8Tensor.empty(512, 512), torch.randn(512, 512, device='cuda'))
e = ax.quantize_f8(ax.F8Tensor.empty(4 * 512, 512), torch.randn(2048, 512, device='cuda'))
r = torch.randn(4, 512, device='cuda')
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = [ax.linear_f8(v, w) for v in (x, few, many)] + [ax.moe_q(v, r, e, e, e, 2)[0] for v in (few, x)]
g.replay()
torch.cuda.synchronize()
for a, b in zip(out, [ax.linear_f8(v, w) for v in (x, few, many)] + [ax.moe_q(v, r, e, e, e, 2)[0] for v in (few, x)]):
    assert torch.equal(a, b)
print('captured')
"""
    from conftest import ROOT
    p = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert p.returncode == 0 and "captured" in p.stdout, p.stderr[-2000:]


def test_two_streams_at_once(cuda, orc):
    """Two calls that overlap on the GPU, each on its own stream: results as alone."""
    rng = np.random.default_rng(21)
    q = [_q(Weights(orc, f, 4, r, c, rng)) for f, r, c in (("Q4_K", 512, 768), ("Q4_K", 512, 768), ("Q6_K", 768, 512))]
    wr = torch.randn(4, 768, device="cuda")
    xs = [torch.randn(n, 768, device="cuda") * 0.05 for n in (3, 20)]
    alone = [ax.moe_q(x, wr, *q, 2)[0] for x in xs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for i in range(2):
            outs[i].append(ax.moe_q(xs[i], wr, *q, 2, stream=streams[i])[0])
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, alone[i]) for o in outs[i])


def test_empty(cuda, orc):
    rng = np.random.default_rng(1)
    q = _q(Weights(orc, "Q4_K", 2, 32, 64, rng))
    d = _q(Weights(orc, "Q4_K", 2, 64, 32, rng))
    y = ax.moe_mlp_q(torch.zeros(0, 64, device="cuda"), torch.zeros(0, 2, dtype=torch.int32, device="cuda"),
                     torch.zeros(0, 2, device="cuda"), q, q, d, experts=2)
    assert y.shape == (0, 64)
    ids, p = ax.moe_route(torch.zeros(0, 64, device="cuda"), torch.zeros(2, 64, device="cuda"), 1)
    assert ids.shape == (0, 1)


def test_refusals(cuda, orc):
    rng = np.random.default_rng(2)
    q = _q(Weights(orc, "Q4_K", 2, 32, 64, rng))
    q8 = _q(Weights(orc, "Q8_0", 2, 32, 64, rng))
    d = _q(Weights(orc, "Q4_K", 2, 64, 32, rng))
    x, ids, p = torch.zeros(1, 64, device="cuda"), torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.ones(1, 1, device="cuda")
    with pytest.raises(ax.AxqError, match="same format"):
        ax.moe_mlp_q(x, ids, p, q, q8, d, experts=2)
    with pytest.raises(ax.AxqError, match="w_down must be"):
        ax.moe_mlp_q(x, ids, p, q, q, q, experts=2)
    with pytest.raises(ax.AxqError, match="int32"):
        ax.moe_mlp_q(x, ids.long(), p, q, q, d, experts=2)
    with pytest.raises(ax.AxqError, match="experts"):
        ax.moe_mlp_q(x, ids, p, q, q, d, experts=3)
    with pytest.raises(ax.AxqError, match="larger than"):
        ax.moe_route(x, torch.zeros(2, 64, device="cuda"), 3)
    f = ax.F8Tensor.empty(2 * 100, 128)
    with pytest.raises(ax.AxqError, match="multiples of 128"):
        ax.moe_mlp_q(torch.zeros(1, 128, device="cuda"), ids, p, f, f, _q(Weights(orc, "Q4_K", 2, 128, 100, rng)), experts=2)


def test_overlaps_and_no_features_are_refused(cuda, orc):
    rng = np.random.default_rng(3)
    q = _q(Weights(orc, "Q4_K", 2, 32, 64, rng))
    d = _q(Weights(orc, "Q4_K", 2, 64, 32, rng))
    both = torch.zeros(3, 64, device="cuda")
    ids, p = torch.zeros(2, 1, dtype=torch.int32, device="cuda"), torch.ones(2, 1, device="cuda")
    wr = torch.zeros(2, 64, device="cuda")
    for first in (0, 1):
        with pytest.raises(ax.AxqError, match="must not overlap"):
            ax.moe_mlp_q(both[:2], ids, p, q, q, d, experts=2, out=both[first:first + 2])
        with pytest.raises(ax.AxqError, match="must not overlap"):
            ax.moe_q(both[:2], wr, q, q, d, 1, out=both[first:first + 2])
    p = torch.ones(2, 64, device="cuda")
    with pytest.raises(ax.AxqError, match="must not overlap"):
        ax.moe_mlp_q(both[:2], torch.zeros(2, 32, dtype=torch.int32, device="cuda"), p.view(-1)[:64].view(2, 32), q, q, d,
                     experts=2, out=p)
    none = ax.QTensor(torch.empty(0, dtype=torch.uint8, device="cuda"), (2 * 32, 0), ax.QuantFormat.Q4_K)
    down = ax.QTensor(torch.empty(0, dtype=torch.uint8, device="cuda"), (0, 32), ax.QuantFormat.Q4_K)
    with pytest.raises(ax.AxqError, match="hidden must be positive"):
        ax.moe_q(torch.zeros(2, 0, device="cuda"), torch.zeros(2, 0, device="cuda"), none, none, down, 1)


@pytest.mark.parametrize("T", [2, 24])
def test_weights_packed_right_before_each_call(cuda, T):
    """The kernels of a stream start early on one another: calls without a wait between them, on weights that are packed
    anew in the same memory before each, against the same calls with a wait after every step."""
    E, K, hidden, ffn = 4, 2, 512, 1024
    g = torch.Generator(device="cuda").manual_seed(T)
    src = [[torch.randn(E * r, c, device="cuda", generator=g) * 0.05 for r, c in ((ffn, hidden), (ffn, hidden), (hidden, ffn))]
           for _ in range(3)]
    xs = [torch.randn(T, hidden, device="cuda", generator=g) for _ in range(3)]
    wr = torch.randn(E, hidden, device="cuda", generator=g)
    w = [ax.F8Tensor.empty(*s.shape) for s in src[0]]
    x = torch.empty_like(xs[0])

    def call(i, wait):
        steps = [lambda: x.copy_(xs[i])] + [lambda k=k: ax.quantize_f8(w[k], src[i][k]) for k in range(3)]
        for s in steps:
            s()
            if wait:
                torch.cuda.synchronize()
        y = ax.moe_q(x, wr, *w, K)[0]
        if wait:
            torch.cuda.synchronize()
        return y

    want = [call(i, True) for i in range(3)]
    got = [(i, call(i, False)) for _ in range(20) for i in range(3)]
    torch.cuda.synchronize()
    for i, y in got:
        assert torch.equal(y, want[i])


@pytest.mark.parametrize("T,E,K", [(4, 1000, 32), (1, 1000, 1), (4, 3, 3), (5, 1000, 32), (16, 1024, 32)])
def test_plan_of_the_router_and_of_its_own_kernel(cuda, T, E, K):
    """Many experts and choices: the layer, whose plan the router's kernel makes for up to 4 tokens, against its parts."""
    g = torch.Generator(device="cuda").manual_seed(E)
    q = []
    for r, c in ((32, 64), (32, 64), (64, 32)):
        w = ax.QTensor.empty(E * r, c, ax.QuantFormat.Q8_0)
        ax.quantize(w, torch.randn(E * r, c, device="cuda", generator=g), ax.QuantFormat.Q8_0)
        q.append(w)
    x, wr = torch.randn(T, 64, device="cuda", generator=g), torch.randn(E, 64, device="cuda", generator=g)
    y, ids, p = ax.moe_q(x, wr, *q, K)
    ids2, p2 = ax.moe_route(x, wr, K)
    assert torch.equal(ids, ids2) and torch.equal(p, p2)
    assert torch.equal(y, ax.moe_mlp_q(x, ids, p, *q, experts=E))
    # each choice by itself, weighed and added in fp32, within the rounding of K sums
    for t in range(min(T, 2)):
        parts = torch.cat([ax.moe_mlp_q(x[t:t + 1], ids[t:t + 1, j:j + 1].contiguous(), p[t:t + 1, j:j + 1].contiguous(), *q,
                                        experts=E) for j in range(K)]).double()
        assert ((y[t].double() - parts.sum(0)).abs() <= (K + 1) * 2.0 ** -23 * parts.abs().sum(0)).all()
