"""A caller's workspace in the e4m3 and mixture-of-experts calls, and the status that is read from it."""
import pytest
import torch

import axon_b200 as ax

pytestmark = pytest.mark.gpu


def _word(ws):
    """The status word: the first four bytes at the workspace's first multiple of 256."""
    buf = ws.get(0, torch.device("cuda", torch.cuda.current_device()))
    at = -buf.data_ptr() % 256
    return buf[at:at + 4].view(torch.int32)


def _calls():
    """Every path of the calls that take a workspace: (name, call)."""
    g = torch.Generator(device="cuda").manual_seed(1)

    def rand(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    w = ax.quantize_f8(ax.F8Tensor.empty(384, 512), rand(384, 512))
    gate, up, down = (ax.quantize_f8(ax.F8Tensor.empty(4 * r, c), rand(4 * r, c) * 0.05) for r, c in ((128, 512), (128, 512), (512, 128)))
    wr = rand(4, 512)
    for n in (1, 40, 300):  # packed within the product, by a kernel of its own, and for the pair kernel
        x = rand(n, 512)
        yield f"linear {n}", lambda x=x, **kw: (ax.linear_f8(x, w, **kw),)
        q = ax.quantize_f8(ax.F8Tensor.empty(n, 512, 1), x)
        yield f"linear packed {n}", lambda q=q, **kw: (ax.linear_f8(q, w, **kw),)
        yield f"layer {n}", lambda x=x, **kw: ax.moe_q(x, wr, gate, up, down, 2, **kw)
        ids, p = ax.moe_route(x, wr, 2)
        yield f"experts {n}", lambda x=x, ids=ids, p=p, **kw: (ax.moe_mlp_q(x, ids, p, gate, up, down, 4, **kw),)
    none, bias = ax.F8Tensor.empty(6, 0), rand(6)
    yield "no features", lambda **kw: (ax.linear_f8(torch.zeros(3, 0, device="cuda"), none, bias=bias, **kw),)


def test_results_and_status(cuda):
    ws = ax.Workspace()
    ws.status()  # nothing has used it
    for name, call in _calls():
        want = call()
        got = call(workspace=ws)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), name
        ws.status()
        _word(ws).fill_(1)  # as a kernel leaves it that gave up
        with pytest.raises(ax.AxqError) as e:
            ws.status()
        assert e.value.status == ax.Status.ERR_TIMEOUT, name
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        got = call(workspace=ws, stream=s)  # a call starts anew
        ws.status(s)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), name
        ws.status()


def test_empty_calls_leave_the_status(cuda):
    ws = ax.Workspace()
    w = ax.F8Tensor.empty(6, 40)
    assert ax.linear_f8(torch.zeros(0, 40, device="cuda"), w, workspace=ws).shape == (0, 6)
    none = ax.QTensor(torch.empty(0, dtype=torch.uint8, device="cuda"), (0, 64), ax.QuantFormat.Q8_0)
    down = ax.QTensor(torch.empty(0, dtype=torch.uint8, device="cuda"), (2 * 64, 0), ax.QuantFormat.Q8_0)
    y, ids, _ = ax.moe_q(torch.ones(3, 64, device="cuda"), torch.ones(2, 64, device="cuda"), none, none, down, 1, workspace=ws)
    assert not y.any() and not ids.any()  # no hidden features, equal logits
    ws.status()


def test_older_calls_too(cuda):
    """The same workspace serves the block formats' calls, whose status it reads as well."""
    ws = ax.Workspace()
    q = ax.QTensor.empty(64, 256, ax.QuantFormat.Q4_K)
    ax.quantize(q, torch.randn(64, 256, device="cuda"), ax.QuantFormat.Q4_K)
    for n in (1, 40):
        x = torch.randn(n, 256, device="cuda")
        assert torch.equal(ax.linear_q(x, q, workspace=ws), ax.linear_q(x, q))
        ws.status()
        _word(ws).fill_(1)
        with pytest.raises(ax.AxqError):
            ws.status()
