"""Mixture-of-experts layer for a few tokens on packed experts.

Beside :func:`gate_up_silu` and :func:`mlp_q`: the same gated block, with each
token's experts chosen by a router.  Expert weights are one tensor per matrix,
the experts' rows after one another: a :class:`QTensor` in any packed format or
an :class:`F8Tensor` in 128 x 128 blocks.  The reference (ruwwww/Axon) has no
router and no gated block.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from ._capi import BLOCK_BYTES, F8_BLOCK, F8_E4M3, check, lib
from .f8 import F8Tensor, _float_type, _invalid, _on, _plain, _raw_stream, _same_device, _scratch
from .ops import QTensor, Workspace, _packed_bytes


def _weights(w, rows: int, cols: int, name: str):
    """(format id, codes, address of the scales or None) of experts' weights [rows x cols]."""
    if w.shape != (rows, cols):
        raise _invalid(f"{name} must be [{rows} x {cols}] (got {tuple(w.shape)})")
    if isinstance(w, F8Tensor):
        w._check(name)
        if w.block_rows != F8_BLOCK or w.data.shape[1] != cols:
            raise _invalid(f"{name}: e4m3 experts are packed in 128 x 128 blocks, their rows without padding")
        return F8_E4M3, w.data, w.scales.data_ptr()
    if w.fmt not in BLOCK_BYTES:
        raise _invalid(f"{name} must be in a block format (got {w.fmt})")
    _plain(w.data, name, torch.uint8)
    if w.data.numel() < _packed_bytes(rows, cols, w.fmt):
        raise _invalid(f"{name} is smaller than its shape")
    return int(w.fmt), w.data, None


def _choices(x: torch.Tensor, experts: int, top_k: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """(ids, weights) of x's tokens, to be written."""
    if top_k < 1:
        raise _invalid(f"top_k must be positive (got {top_k})")
    if top_k > experts:
        raise _invalid(f"top_k is larger than the number of experts ({top_k} of {experts})")
    shape = (x.shape[0], top_k)
    return x.new_empty(shape, dtype=torch.int32), x.new_empty(shape, dtype=torch.float32)


def moe_route(x: torch.Tensor, w_router: torch.Tensor, top_k: int, normalize: bool = True,
              stream: Optional[torch.cuda.Stream] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(ids int32 [N, top_k], weights fp32 [N, top_k]) of the top_k largest of
    softmax(x . w_router^T), largest first, ties to the lowest index.

    x is fp32, fp16 or bf16 [N, hidden], w_router fp32 [experts, hidden];
    ``normalize``: a token's weights add up to 1."""
    dtype = _float_type(x, "x")
    _plain(w_router, "w_router", torch.float32)
    if x.dim() != 2 or w_router.dim() != 2 or x.shape[1] != w_router.shape[1]:
        raise _invalid("moe_route: x must be [N x hidden] and w_router [experts x hidden]")
    device = x.device
    _same_device(device, ("w_router",), w_router)
    on = _on(device, stream)
    if on is not None:
        with on:
            return moe_route(x, w_router, top_k, normalize)
    ids, weights = _choices(x, w_router.shape[0], top_k)
    check(lib().axq_moe_route(dtype, x.data_ptr(), w_router.data_ptr(), ids.data_ptr(), weights.data_ptr(), x.shape[0],
                              w_router.shape[0], top_k, x.shape[1], 1 if normalize else 0, _raw_stream(device.index)))
    return ids, weights


def _experts(w_gate, w_up, w_down, experts: int, hidden: int):
    """(ffn, their arguments of the C entry points, their tensors)."""
    for w, name in ((w_gate, "w_gate"), (w_up, "w_up"), (w_down, "w_down")):
        if not isinstance(w, (QTensor, F8Tensor)):
            raise _invalid(f"{name} must be a QTensor or an F8Tensor")
    if experts < 1 or w_gate.shape[0] % experts:
        raise _invalid("w_gate must have experts * ffn rows")
    ffn = w_gate.shape[0] // experts
    fmt, gate, gate_s = _weights(w_gate, experts * ffn, hidden, "w_gate")
    fmt_up, up, up_s = _weights(w_up, experts * ffn, hidden, "w_up")
    fmt_down, down, down_s = _weights(w_down, experts * hidden, ffn, "w_down")
    if fmt != fmt_up:
        raise _invalid("w_gate and w_up must have the same format")
    return (ffn, (fmt, gate.data_ptr(), gate_s, up.data_ptr(), up_s, fmt_down, down.data_ptr(), down_s), (gate, up, down))


def _out(x: torch.Tensor, out: Optional[torch.Tensor], dtype: int) -> torch.Tensor:
    if out is None:
        return torch.empty_like(x)
    if _float_type(out, "out") != dtype or out.shape != x.shape:
        raise _invalid("out must have x's shape and type")
    return out


def moe_mlp_q(x: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor, w_gate, w_up, w_down, experts: int,
              out: Optional[torch.Tensor] = None, stream: Optional[torch.cuda.Stream] = None,
              workspace: Optional[Workspace] = None) -> torch.Tensor:
    """y[t] = sum_j weights[t, j] * W_down[e] . (silu(W_gate[e] . x[t]) * (W_up[e] . x[t])), e = ids[t, j].

    x [N, hidden] in fp32, fp16 or bf16; ids int32 [N, top_k] (an id outside
    0 .. experts - 1 adds nothing); w_gate and w_up [experts * ffn, hidden] in one
    format, w_down [experts * hidden, ffn].  Products and sums are fp32, y has x's
    type.  ``workspace``: scratch of the caller's, whose ``status`` may be asked for."""
    dtype = _float_type(x, "x")
    _plain(ids, "ids", torch.int32)
    _plain(weights, "weights", torch.float32)
    if x.dim() != 2 or ids.dim() != 2 or ids.shape[0] != x.shape[0] or ids.shape != weights.shape:
        raise _invalid("moe_mlp_q: x must be [N x hidden], ids and weights [N x top_k]")
    (n, hidden), top_k, device = x.shape, ids.shape[1], x.device
    ffn, w, tensors = _experts(w_gate, w_up, w_down, experts, hidden)
    _same_device(device, ("ids", "weights", "out", "w_gate", "w_up", "w_down"), ids, weights, out, *tensors)
    on = _on(device, stream)
    if on is not None:
        with on:
            return moe_mlp_q(x, ids, weights, w_gate, w_up, w_down, experts, out, workspace=workspace)
    out = _out(x, out, dtype)
    L = lib()
    buf, wp, wbytes = _scratch(L.axq_moe_workspace_size(n, top_k, hidden, ffn) if n and hidden and ffn else 0, x, workspace)
    check(L.axq_moe_mlp(*w, dtype, x.data_ptr(), ids.data_ptr(), weights.data_ptr(), out.data_ptr(), n, experts, top_k, hidden,
                        ffn, wp, wbytes, _raw_stream(device.index)))
    del buf
    return out


def moe_q(x: torch.Tensor, w_router: torch.Tensor, w_gate, w_up, w_down, top_k: int, normalize: bool = True,
          out: Optional[torch.Tensor] = None, stream: Optional[torch.cuda.Stream] = None,
          workspace: Optional[Workspace] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The whole layer: what :func:`moe_route` and then :func:`moe_mlp_q` give, in
    fewer kernels.  Returns (y, ids, weights).  ``workspace`` as there."""
    dtype = _float_type(x, "x")
    _plain(w_router, "w_router", torch.float32)
    if x.dim() != 2 or w_router.dim() != 2 or x.shape[1] != w_router.shape[1]:
        raise _invalid("moe_q: x must be [N x hidden] and w_router [experts x hidden]")
    (n, hidden), experts, device = x.shape, w_router.shape[0], x.device
    ffn, w, tensors = _experts(w_gate, w_up, w_down, experts, hidden)
    _same_device(device, ("w_router", "out", "w_gate", "w_up", "w_down"), w_router, out, *tensors)
    on = _on(device, stream)
    if on is not None:
        with on:
            return moe_q(x, w_router, w_gate, w_up, w_down, top_k, normalize, out, workspace=workspace)
    out = _out(x, out, dtype)
    ids, weights = _choices(x, experts, top_k)
    L = lib()
    buf, wp, wbytes = _scratch(L.axq_moe_workspace_size(n, top_k, hidden, ffn) if n and hidden and ffn else 0, x, workspace)
    check(L.axq_moe(*w, dtype, x.data_ptr(), w_router.data_ptr(), 1 if normalize else 0, ids.data_ptr(), weights.data_ptr(),
                    out.data_ptr(), n, experts, top_k, hidden, ffn, wp, wbytes, _raw_stream(device.index)))
    del buf
    return out, ids, weights
