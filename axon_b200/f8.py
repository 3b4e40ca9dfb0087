"""8-bit floating point blocks: packing and the quantized Linear.

Beside :func:`quantize`, :func:`dequantize` and :func:`linear_q` for matrices
held as e4m3 codes with one fp32 scale per 128 x 128 block (weights) or 1 x 128
block (activations).  The reference (ruwwww/Axon) has no floating-point blocks.

Scratch and outputs come from torch's caching allocator for the call's stream,
one allocation per call: nothing is shared between streams or captured graphs.
"""
from __future__ import annotations

import contextlib
from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from ._capi import DType, F8_BLOCK, AxqError, Status, check, lib
from .ops import _req_cuda, _stream_handle

FLOAT_TYPES = {torch.float32: DType.F32, torch.float16: DType.F16, torch.bfloat16: DType.BF16}


def _up(n: int, m: int) -> int:
    return -(-n // m)


def _invalid(msg: str) -> AxqError:
    return AxqError(Status.ERR_INVALID, msg)


def _float_type(t, name: str) -> DType:
    """The element type of a contiguous CUDA float tensor."""
    if not isinstance(t, torch.Tensor):
        raise _invalid(f"{name} must be a torch.Tensor")
    if t.dtype not in FLOAT_TYPES:
        raise _invalid(f"{name} must be float32, float16 or bfloat16 (got {t.dtype})")
    _req_cuda(t, name, t.dtype)
    return FLOAT_TYPES[t.dtype]


def _same_device(device: torch.device, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise _invalid(f"{name} is on {t.device}, not on {device}")


@contextlib.contextmanager
def _on(device: torch.device, stream: Optional[torch.cuda.Stream]):
    """The call's device and stream made current, so that what it allocates
    belongs to that stream."""
    with torch.cuda.device(device):
        if stream is None:
            yield
        else:
            with torch.cuda.stream(stream):
                yield


def _scratch(nbytes: int, device: torch.device) -> Tuple[torch.Tensor, int, int]:
    """(tensor, 256-byte aligned address, bytes from there)."""
    buf = torch.empty(nbytes + 256, dtype=torch.uint8, device=device)
    off = -buf.data_ptr() % 256
    return buf, buf.data_ptr() + off, nbytes + 256 - off


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
        if self.block_rows not in (1, F8_BLOCK):
            raise _invalid(f"{name}: block_rows must be 1 or 128")
        _req_cuda(self.data, f"{name}.data", torch.float8_e4m3fn)
        _req_cuda(self.scales, f"{name}.scales", torch.float32)
        if self.data.dim() != 2 or self.data.shape[0] != rows or self.data.shape[1] < cols or self.data.shape[1] % 16:
            raise _invalid(f"{name}: codes of a [{rows} x {cols}] matrix must be [{rows} x ld], ld a multiple of 16 of at "
                           f"least {cols} (got {tuple(self.data.shape)})")
        want = (_up(rows, self.block_rows), _up(cols, F8_BLOCK))
        if tuple(self.scales.shape) != want:
            raise _invalid(f"{name}: scales must be {want} (got {tuple(self.scales.shape)})")
        _same_device(self.data.device, **{f"{name}.scales": self.scales})


def quantize_f8(dst: F8Tensor, src: torch.Tensor, stream: Optional[torch.cuda.Stream] = None) -> F8Tensor:
    """Pack ``src`` (fp32, fp16 or bf16, [rows, cols]) into ``dst``: per block
    scale = max|x| / 448 and code = e4m3(x / scale), rounded to nearest even
    (C ABI axq_quantize_f8, which states what zeros, NaN and infinities give)."""
    dtype = _float_type(src, "src")
    if src.dim() != 2:
        raise _invalid("quantize_f8: src must be 2-D")
    dst._check("dst")
    if tuple(src.shape) != tuple(dst.shape):
        raise _invalid(f"quantize_f8: src is {tuple(src.shape)}, dst {tuple(dst.shape)}")
    _same_device(src.device, dst=dst.data)
    rows, cols = src.shape
    with _on(src.device, stream):
        check(lib().axq_quantize_f8(int(dtype), src.data_ptr(), dst.data.data_ptr(), dst.data.shape[1],
                                    dst.scales.data_ptr(), rows, cols, dst.block_rows,
                                    _stream_handle(stream, src.device)))
    return dst


def dequantize_f8(dst: torch.Tensor, src: F8Tensor, stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """Decode ``src`` into ``dst`` (fp32, [rows, cols])."""
    src._check("src")
    _req_cuda(dst, "dst", torch.float32)
    if tuple(dst.shape) != tuple(src.shape):
        raise _invalid(f"dequantize_f8: dst is {tuple(dst.shape)}, src {tuple(src.shape)}")
    _same_device(dst.device, src=src.data)
    rows, cols = src.shape
    with _on(dst.device, stream):
        check(lib().axq_dequantize_f8(src.data.data_ptr(), src.data.shape[1], src.scales.data_ptr(), src.block_rows,
                                      dst.data_ptr(), rows, cols, _stream_handle(stream, dst.device)))
    return dst


def linear_f8(x, w: F8Tensor, out: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
              stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """Linear on e4m3 blocks: y[N, M] = x[N, K] . W[M, K]^T (+ bias[M], fp32).

    ``w`` is packed in 128 x 128 blocks.  ``x`` is fp32, fp16 or bf16 (packed in
    1 x 128 blocks by the call) or an :class:`F8Tensor` with ``block_rows`` 1.
    The result has ``out``'s type, else x's (fp32 for a packed x); sums are fp32."""
    w._check("w")
    if w.block_rows != F8_BLOCK:
        raise _invalid("linear_f8: w must be packed in 128 x 128 blocks")
    M, K = w.shape
    packed = isinstance(x, F8Tensor)
    if packed:
        x._check("x")
        if x.block_rows != 1:
            raise _invalid("linear_f8: x must be packed in 1 x 128 blocks")
        xd, x_type, x_ld, x_scales, y_type = x.data, DType.F8, x.data.shape[1], x.scales, torch.float32
    else:
        x_type = _float_type(x, "x")
        xd, x_ld, x_scales, y_type = x, K, None, x.dtype
        if x.dim() != 2:
            raise _invalid("linear_f8: x must be 2-D")
    if x.shape[1] != K:
        raise _invalid(f"linear_f8: x must be [N x {K}]")
    N, device = x.shape[0], xd.device
    if bias is not None:
        _req_cuda(bias, "bias", torch.float32)
        if bias.numel() != M:
            raise _invalid(f"linear_f8: bias must have {M} elements")
    _same_device(device, w=w.data, bias=bias, out=out)
    with _on(device, stream):
        if out is None:
            out = torch.empty((N, M), dtype=y_type, device=device)
        out_type = _float_type(out, "out")
        if tuple(out.shape) != (N, M):
            raise _invalid(f"linear_f8: out must be [{N} x {M}]")
        buf, wp, wbytes = _scratch(int(lib().axq_linear_f8_workspace_size(int(x_type), K, N)), device)
        check(lib().axq_linear_f8(w.data.data_ptr(), w.data.shape[1], w.scales.data_ptr(), int(x_type), xd.data_ptr(), x_ld,
                                  None if x_scales is None else x_scales.data_ptr(),
                                  None if bias is None else bias.data_ptr(), int(out_type), out.data_ptr(), M, K, N, wp,
                                  wbytes, _stream_handle(stream, device)))
        del buf
    return out
