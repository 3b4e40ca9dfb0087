"""8-bit floating point blocks: packing and the quantized Linear.

Beside :func:`quantize`, :func:`dequantize` and :func:`linear_q` for matrices
held as e4m3 codes with one fp32 scale per 128 x 128 block (weights) or 1 x 128
block (activations).  The reference (ruwwww/Axon) has no floating-point blocks.

Scratch and outputs come from torch's caching allocator for the call's stream,
one allocation per call: nothing is shared between streams or captured graphs.
A call that is given a :class:`Workspace` takes its scratch there instead; calls
that share one must be ordered, and its ``status`` says whether a kernel gave up
a bounded wait (the call itself only enqueues work; without a workspace of the
caller's there is nowhere to read that from).
"""
from __future__ import annotations

import contextlib
from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from ._capi import DType, F8_BLOCK, AxqError, Status, check, lib
from .ops import Workspace, _aligned_ptr, _req_cuda

# element types as C ABI ids (plain ints: these run on every call)
FLOAT_TYPES = {torch.float32: int(DType.F32), torch.float16: int(DType.F16), torch.bfloat16: int(DType.BF16)}
_E4M3 = torch.float8_e4m3fn
_current_device = torch._C._cuda_getDevice
_raw_stream = torch._C._cuda_getCurrentRawStream


def _up(n: int, m: int) -> int:
    return -(-n // m)


def _invalid(msg: str) -> AxqError:
    return AxqError(Status.ERR_INVALID, msg)


def _float_type(t, name: str) -> int:
    """The element type id of a contiguous CUDA float tensor."""
    if isinstance(t, torch.Tensor):
        dtype = FLOAT_TYPES.get(t.dtype)
        if dtype is not None and t.is_cuda and t.is_contiguous():
            return dtype
        if dtype is None:
            raise _invalid(f"{name} must be float32, float16 or bfloat16 (got {t.dtype})")
        _req_cuda(t, name, t.dtype)  # says what is wrong
    raise _invalid(f"{name} must be a torch.Tensor")


def _plain(t, name: str, dtype: torch.dtype) -> None:
    """A contiguous CUDA tensor of this type."""
    if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.is_cuda and t.is_contiguous()):
        _req_cuda(t, name, dtype)


def _same_device(device: torch.device, names, *tensors) -> None:
    for k, t in enumerate(tensors):
        if t is not None and t.device != device:
            raise _invalid(f"{names[k]} is on {t.device}, not on {device}")


def _on(device: torch.device, stream: Optional[torch.cuda.Stream]):
    """None where the call's device is current and it goes to the current
    stream; else a context that makes both so (what the call allocates then
    belongs to its stream)."""
    if stream is None:
        return None if device.index == _current_device() else torch.cuda.device(device)
    if stream.device_index != device.index:
        raise _invalid(f"stream is on cuda:{stream.device_index}, not on {device}")
    both = contextlib.ExitStack()
    both.enter_context(torch.cuda.device(device))
    both.enter_context(torch.cuda.stream(stream))
    return both


def _scratch(nbytes: int, like: torch.Tensor, workspace: Optional[Workspace]):
    """(tensor on `like`'s device, 256-byte aligned address, bytes from there); nothing for 0 bytes, so that a workspace
    whose status no kernel would set is not made."""
    if not nbytes:
        return None, None, 0
    buf = like.new_empty(nbytes + 256, dtype=torch.uint8) if workspace is None else workspace.get(nbytes + 256, like.device)
    return (buf, *_aligned_ptr(buf))


@dataclass
class F8Tensor:
    """e4m3 codes of a [rows x cols] matrix, one byte each in rows of
    ``data.shape[1]`` bytes (a multiple of 16, at least cols), and their scales
    [ceil(rows / block_rows) x ceil(cols / 128)]; value = code * scale."""

    data: torch.Tensor
    scales: torch.Tensor
    shape: Tuple[int, int]
    block_rows: int = F8_BLOCK

    @staticmethod
    def empty(rows: int, cols: int, block_rows: int = F8_BLOCK, device="cuda") -> "F8Tensor":
        if block_rows not in (1, F8_BLOCK):
            raise _invalid("F8Tensor: block_rows must be 1 or 128")
        data = torch.empty(rows, _up(cols, 16) * 16, dtype=torch.float8_e4m3fn, device=device)
        scales = torch.empty(_up(rows, block_rows), _up(cols, F8_BLOCK), dtype=torch.float32, device=device)
        return F8Tensor(data, scales, (rows, cols), block_rows)

    def _check(self, name: str) -> None:
        rows, cols = self.shape
        d, s, br = self.data, self.scales, self.block_rows
        if br != 1 and br != F8_BLOCK:
            raise _invalid(f"{name}: block_rows must be 1 or 128")
        _plain(d, f"{name}.data", _E4M3)
        _plain(s, f"{name}.scales", torch.float32)
        if d.dim() != 2 or d.shape[0] != rows or d.shape[1] < cols or d.shape[1] % 16:
            raise _invalid(f"{name}: codes of a [{rows} x {cols}] matrix must be [{rows} x ld], ld a multiple of 16 of at "
                           f"least {cols} (got {tuple(d.shape)})")
        want = (_up(rows, br), _up(cols, F8_BLOCK))
        if s.shape != want:
            raise _invalid(f"{name}: scales must be {want} (got {tuple(s.shape)})")
        if s.device != d.device:
            raise _invalid(f"{name}.scales is on {s.device}, not on {d.device}")


def quantize_f8(dst: F8Tensor, src: torch.Tensor, stream: Optional[torch.cuda.Stream] = None) -> F8Tensor:
    """Pack ``src`` (fp32, fp16 or bf16, [rows, cols]) into ``dst``: per block
    scale = max|x| / 448 and code = e4m3(x / scale), rounded to nearest even
    (C ABI axq_quantize_f8, which states what zeros, NaN and infinities give)."""
    dtype = _float_type(src, "src")
    if src.dim() != 2:
        raise _invalid("quantize_f8: src must be 2-D")
    dst._check("dst")
    if src.shape != tuple(dst.shape):
        raise _invalid(f"quantize_f8: src is {tuple(src.shape)}, dst {tuple(dst.shape)}")
    device = src.device
    _same_device(device, ("dst",), dst.data)
    on = _on(device, stream)
    if on is not None:
        with on:
            return quantize_f8(dst, src)
    rows, cols = src.shape
    check(lib().axq_quantize_f8(dtype, src.data_ptr(), dst.data.data_ptr(), dst.data.shape[1], dst.scales.data_ptr(), rows,
                                cols, dst.block_rows, _raw_stream(device.index)))
    return dst


def dequantize_f8(dst: torch.Tensor, src: F8Tensor, stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """Decode ``src`` into ``dst`` (fp32, [rows, cols])."""
    src._check("src")
    _plain(dst, "dst", torch.float32)
    if dst.shape != tuple(src.shape):
        raise _invalid(f"dequantize_f8: dst is {tuple(dst.shape)}, src {tuple(src.shape)}")
    device = dst.device
    _same_device(device, ("src",), src.data)
    on = _on(device, stream)
    if on is not None:
        with on:
            return dequantize_f8(dst, src)
    rows, cols = src.shape
    check(lib().axq_dequantize_f8(src.data.data_ptr(), src.data.shape[1], src.scales.data_ptr(), src.block_rows,
                                  dst.data_ptr(), rows, cols, _raw_stream(device.index)))
    return dst


def linear_f8(x, w: F8Tensor, out: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
              stream: Optional[torch.cuda.Stream] = None, workspace: Optional[Workspace] = None) -> torch.Tensor:
    """Linear on e4m3 blocks: y[N, M] = x[N, K] . W[M, K]^T (+ bias[M], fp32).

    ``w`` is packed in 128 x 128 blocks.  ``x`` is fp32, fp16 or bf16 (packed in
    1 x 128 blocks by the call) or an :class:`F8Tensor` with ``block_rows`` 1.
    The result has ``out``'s type, else x's (fp32 for a packed x); sums are fp32.
    ``workspace``: scratch of the caller's, whose ``status`` may be asked for."""
    w._check("w")
    if w.block_rows != F8_BLOCK:
        raise _invalid("linear_f8: w must be packed in 128 x 128 blocks")
    M, K = w.shape
    if isinstance(x, F8Tensor):
        x._check("x")
        if x.block_rows != 1:
            raise _invalid("linear_f8: x must be packed in 1 x 128 blocks")
        xd, x_type, x_ld, x_scales, y_type = x.data, int(DType.F8), x.data.shape[1], x.scales.data_ptr(), torch.float32
    else:
        x_type = _float_type(x, "x")
        xd, x_ld, x_scales, y_type = x, K, None, x.dtype
        if x.dim() != 2:
            raise _invalid("linear_f8: x must be 2-D")
    N, xk = x.shape
    if xk != K:
        raise _invalid(f"linear_f8: x must be [N x {K}]")
    device = xd.device
    bias_ptr = None
    if bias is not None:
        _plain(bias, "bias", torch.float32)
        if bias.numel() != M:
            raise _invalid(f"linear_f8: bias must have {M} elements")
        bias_ptr = bias.data_ptr()
    _same_device(device, ("w", "bias", "out"), w.data, bias, out)
    on = _on(device, stream)
    if on is not None:
        with on:
            return linear_f8(x, w, out, bias, workspace=workspace)
    if out is None:
        out = xd.new_empty((N, M), dtype=y_type)
        out_type = FLOAT_TYPES[y_type]
    else:
        out_type = _float_type(out, "out")
        if out.shape != (N, M):
            raise _invalid(f"linear_f8: out must be [{N} x {M}]")
    L = lib()
    buf, wp, wbytes = _scratch(L.axq_linear_f8_workspace_size(x_type, K, N) if M and N else 0, xd, workspace)
    check(L.axq_linear_f8(w.data.data_ptr(), w.data.shape[1], w.scales.data_ptr(), x_type, xd.data_ptr(), x_ld, x_scales,
                          bias_ptr, out_type, out.data_ptr(), M, K, N, wp, wbytes, _raw_stream(device.index)))
    del buf
    return out
