"""Projections in 4-bit microscaled floating point (MXFP4) on packed token rows.

    w = mxfp4.pack_weight(kernel)                          # once, when the weights are loaded: [in, out] -> 4 bits
    y = mxfp4.linear(x, w, bias=b, activation="gelu")      # x [T, in] fp16 or fp32 -> y [T, out]

    a = mxfp4.quantize(x)                                  # or step by step: rows to 4 bits,
    f = mxfp4.gemm(a, w1, bias=b1, activation="gelu", out=mxfp4.empty(T, ffn))  # a product that stays in 4 bits,
    y = mxfp4.gemm(f, w2, bias=b2, residual=x)             # and one that leaves them

32 consecutive values of a row share a power-of-two scale, each value is a 4-bit float (include/et_b200.h, et_mxfp4_*).
Every call runs on the current stream of the tensors' device and returns without waiting.  `valid_rows` is a device
int32 [1] (valid_word_num of the input op): rows past it are neither read nor written, an output passed as `out` keeps
them.  Tensors must be contiguous (x of quantize and linear: contiguous rows) and on one device.
"""
from __future__ import annotations

import ctypes as C
from typing import Dict, Optional, Union

import torch

from . import _capi

__all__ = ["MxTensor", "empty", "quantize", "dequantize", "pack_weight", "gemm", "linear", "device_status"]

_DTYPE = {torch.float16: _capi.ET_FP16, torch.float32: _capi.ET_FP32}
_EPILOGUE = {None: 1, "gelu": 2, "tanh": 3}
_status: Dict[int, torch.Tensor] = {}


class MxTensor:
    """`rows` rows of `cols` values in MXFP4; `data` is the device buffer, in the layout of the tensor core."""

    __slots__ = ("data", "rows", "cols")

    def __init__(self, data: torch.Tensor, rows: int, cols: int):
        self.data, self.rows, self.cols = data, rows, cols

    def __repr__(self) -> str:
        return f"MxTensor({self.rows} x {self.cols}, {self.data.device})"


def _require(ok: bool, message: str) -> None:
    if not ok:
        raise ValueError(message)


def _check(t: Optional[torch.Tensor], name: str, shape, dtype: torch.dtype, device: torch.device) -> None:
    if t is None:
        return
    _require(isinstance(t, torch.Tensor) and t.is_contiguous() and t.dtype == dtype and t.device == device
             and tuple(t.shape) == shape, f"{name} must be a contiguous {list(shape)} tensor of dtype {dtype} on {device}")


def _check_rows(t: torch.Tensor, name: str) -> None:
    _require(isinstance(t, torch.Tensor) and t.is_cuda and t.dtype in _DTYPE and t.dim() == 2,
             f"{name} must be a [rows, width] CUDA tensor of dtype torch.float16 or torch.float32")
    _require(t.shape[1] > 0 and t.shape[1] % 32 == 0, f"the width of {name} must be a positive multiple of 32")


def _check_count(valid_rows: Optional[torch.Tensor], device: torch.device) -> None:
    if valid_rows is None:
        return
    _require(isinstance(valid_rows, torch.Tensor) and valid_rows.dtype == torch.int32 and valid_rows.numel() == 1
             and valid_rows.device == device, "valid_rows must be one int32 on the rows' device")


def _check_mx(t: MxTensor, name: str, rows: Optional[int], cols: int, device: torch.device) -> None:
    _require(isinstance(t, MxTensor), f"{name} must be an MxTensor")
    _require(t.cols == cols and (rows is None or t.rows >= rows) and t.data.device == device,
             f"{name} must be an MxTensor of {'' if rows is None else f'at least {rows} rows of '}{cols} values on {device}")


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


class _On:
    """Makes a tensor's device current for a call (the library launches on the current device)."""

    __slots__ = ("device", "previous")

    def __init__(self, device: torch.device):
        self.device, self.previous = device.index, -1

    def __enter__(self) -> int:
        if torch.cuda.current_device() != self.device:
            self.previous = torch.cuda.current_device()
            torch.cuda.set_device(self.device)
        return torch.cuda.current_stream().cuda_stream

    def __exit__(self, *exc) -> None:
        if self.previous >= 0:
            torch.cuda.set_device(self.previous)


def _status_word(device: torch.device) -> torch.Tensor:
    word = _status.get(device.index)
    if word is None:
        _require(not torch.cuda.is_current_stream_capturing(),
                 "call mxfp4.device_status(device) once before a product is captured on this device")
        word = _status[device.index] = torch.zeros(1, dtype=torch.int32, device=device)
    return word


def device_status(device: Union[int, str, torch.device] = "cuda") -> int:
    """0, or the code of a bounded device-side wait that ran out in a product on this device since the last call
    (its results are then incomplete).  Waits for the device's current stream."""
    device = torch.device(device) if not isinstance(device, int) else torch.device("cuda", device)
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    word = _status_word(device)
    code = int(word.item())
    if code != 0:
        word.zero_()
    return code


def empty(rows: int, cols: int, device: Union[str, torch.device] = "cuda") -> MxTensor:
    """An uninitialised MXFP4 tensor (an output or workspace of the calls below)."""
    _require(rows >= 0 and cols > 0 and cols % 32 == 0, "rows must not be negative, cols a positive multiple of 32")
    size = _capi.load().et_mxfp4_bytes(rows, cols)
    return MxTensor(torch.empty(size, dtype=torch.uint8, device=device), rows, cols)


def quantize(x: torch.Tensor, valid_rows: Optional[torch.Tensor] = None, out: Optional[MxTensor] = None) -> MxTensor:
    """Rows of x [rows, width] to MXFP4 (rows may be strided, the values of a row are contiguous)."""
    _check_rows(x, "x")
    _require(x.stride(1) == 1, "the values of a row of x must be contiguous")
    _check_count(valid_rows, x.device)
    if out is None:
        out = empty(x.shape[0], x.shape[1], x.device)
    _check_mx(out, "out", x.shape[0], x.shape[1], x.device)
    with _On(x.device) as stream:
        _capi.check(_capi.load().et_mxfp4_quantize(
            _DTYPE[x.dtype], x.data_ptr(), _row_stride(x), _ptr(valid_rows), x.shape[0], x.shape[1],
            out.data.data_ptr(), stream))
    return out


def _row_stride(x: torch.Tensor) -> int:
    # (torch gives a single row any stride)
    return x.shape[1] if x.shape[0] <= 1 else x.stride(0)


def dequantize(mx: MxTensor, dtype: torch.dtype, valid_rows: Optional[torch.Tensor] = None,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The values that an MXFP4 tensor stands for, as [rows, cols] of `dtype`."""
    _require(isinstance(mx, MxTensor), "mx must be an MxTensor")
    _require(dtype in _DTYPE, "dtype must be torch.float16 or torch.float32")
    rows = mx.rows if out is None else out.shape[0]
    if out is None:
        out = torch.empty(mx.rows, mx.cols, dtype=dtype, device=mx.data.device)
    _require(rows <= mx.rows, "out has more rows than mx")
    _check(out, "out", (rows, mx.cols), dtype, mx.data.device)
    _check_count(valid_rows, mx.data.device)
    with _On(mx.data.device) as stream:
        _capi.check(_capi.load().et_mxfp4_dequantize(_DTYPE[dtype], mx.data.data_ptr(), _ptr(valid_rows), rows, mx.cols,
                                                     out.data_ptr(), stream))
    return out


def pack_weight(kernel: torch.Tensor) -> MxTensor:
    """A projection's kernel [in, out] (TF dense layout) to the MXFP4 operand of gemm and linear."""
    _require(isinstance(kernel, torch.Tensor) and kernel.is_cuda and kernel.dtype in _DTYPE and kernel.dim() == 2
             and kernel.is_contiguous(), "kernel must be a contiguous [in, out] CUDA tensor, torch.float16 or torch.float32")
    k, n = kernel.shape
    _require(k > 0 and n > 0 and k % 32 == 0 and n % 32 == 0, "in and out must be positive multiples of 32")
    w = empty(n, k, kernel.device)
    with _On(kernel.device) as stream:
        _capi.check(_capi.load().et_mxfp4_pack_weight(_DTYPE[kernel.dtype], kernel.data_ptr(), w.data.data_ptr(), k, n,
                                                      stream))
    return w


def _product(a, stride: Optional[int], workspace: Optional[MxTensor], rows: int, device: torch.device, weight: MxTensor,
             bias, activation, residual, valid_rows, out, dtype: Optional[torch.dtype]):
    _require(isinstance(weight, MxTensor) and weight.data.device == device, "weight must be an MxTensor on the rows' device")
    k, n = weight.cols, weight.rows
    _require(activation in _EPILOGUE, "activation must be None, 'gelu' or 'tanh'")
    _require(activation is None or bias is not None, "an activation needs a bias")
    to_mx = isinstance(out, MxTensor)
    if dtype is None:
        given = next((t for t in (None if to_mx else out, bias, residual) if t is not None), None)
        dtype = torch.float16 if given is None else given.dtype
    _require(dtype in _DTYPE, "dtype must be torch.float16 or torch.float32")
    if out is None:
        out = torch.empty(rows, n, dtype=dtype, device=device)
    if to_mx:
        _check_mx(out, "out", rows, n, device)
        _require(n % 64 == 0 and residual is None, "MXFP4 output needs a width that is a multiple of 64, and no residual")
    else:
        _check(out, "out", (rows, n), dtype, device)
    _check(bias, "bias", (n,), dtype, device)
    _check(residual, "residual", (rows, n), dtype, device)
    _check_count(valid_rows, device)
    epilogue = 0 if bias is None else _EPILOGUE[activation]
    c, c_mx = (None, out.data.data_ptr()) if to_mx else (out.data_ptr(), None)
    lib = _capi.load()
    with _On(device) as stream:
        word = _status_word(device).data_ptr()
        if stride is None:
            rc = lib.et_mxfp4_gemm(_DTYPE[dtype], a, weight.data.data_ptr(), _ptr(bias), _ptr(residual), c, c_mx,
                                   _ptr(valid_rows), rows, n, k, epilogue, word, stream)
        else:
            rc = lib.et_mxfp4_linear(_DTYPE[dtype], a, stride, workspace.data.data_ptr(), weight.data.data_ptr(),
                                     _ptr(bias), _ptr(residual), c, c_mx, _ptr(valid_rows), rows, n, k, epilogue, word,
                                     stream)
    _capi.check(rc)
    return out


def gemm(a: MxTensor, weight: MxTensor, bias: Optional[torch.Tensor] = None, activation: Optional[str] = None,
         residual: Optional[torch.Tensor] = None, dtype: Optional[torch.dtype] = None,
         valid_rows: Optional[torch.Tensor] = None,
         out: Union[torch.Tensor, MxTensor, None] = None) -> Union[torch.Tensor, MxTensor]:
    """act(A W + bias) (+ residual) on rows that are in MXFP4 already.  The result has the dtype of out, bias or
    residual, or `dtype` (torch.float16 where nothing says); an MxTensor as out keeps it in 4 bits.  out may be residual."""
    _require(isinstance(a, MxTensor) and isinstance(weight, MxTensor), "a and weight must be MxTensors")
    _require(a.cols == weight.cols, "a and weight must have the same inner width")
    rows = out.shape[0] if isinstance(out, torch.Tensor) else a.rows
    _require(rows <= a.rows, "out has more rows than a")
    return _product(a.data.data_ptr(), None, None, rows, a.data.device, weight, bias, activation, residual, valid_rows,
                    out, dtype)


def linear(x: torch.Tensor, weight: MxTensor, bias: Optional[torch.Tensor] = None, activation: Optional[str] = None,
           residual: Optional[torch.Tensor] = None, valid_rows: Optional[torch.Tensor] = None,
           workspace: Optional[MxTensor] = None,
           out: Union[torch.Tensor, MxTensor, None] = None) -> Union[torch.Tensor, MxTensor]:
    """gemm(quantize(x), weight, ...) in one call; the result has x's dtype.  `workspace` takes x in MXFP4 (a program
    that calls this in a loop keeps one per stream)."""
    _check_rows(x, "x")
    _require(isinstance(weight, MxTensor) and x.shape[1] == weight.cols, "weight must be an MxTensor of x's width")
    _require(x.stride(1) == 1, "the values of a row of x must be contiguous")
    if workspace is None:
        workspace = empty(x.shape[0], x.shape[1], x.device)
    _check_mx(workspace, "workspace", x.shape[0], x.shape[1], x.device)
    return _product(x.data_ptr(), _row_stride(x), workspace, x.shape[0], x.device, weight, bias, activation, residual,
                    valid_rows, out, x.dtype)
