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

There is no backward pass.  Where autograd records and a tensor requires a gradient, a new result raises in backward, as a
custom op without a formula does; a call that writes into a given buffer or into 4 bits, which could not, is refused.
pack_weight takes a copy, to which no gradient belongs.
"""
from __future__ import annotations

import threading
from typing import Dict, Optional, Union

import torch

from . import _capi

__all__ = ["MxTensor", "empty", "quantize", "dequantize", "pack_weight", "gemm", "linear", "device_status"]

_DTYPE = {torch.float16: _capi.ET_FP16, torch.float32: _capi.ET_FP32}
_EPILOGUE = {None: 1, "gelu": 2, "tanh": 3}
_status: Dict[int, tuple] = {}
_status_lock = threading.Lock()
_lib = None


class MxTensor:
    """`rows` rows of `cols` values in MXFP4; `data` is the device buffer, in the layout of the tensor core (`ptr` its
    address, `device` the index of its GPU)."""

    __slots__ = ("data", "rows", "cols", "ptr", "device")

    def __init__(self, data: torch.Tensor, rows: int, cols: int):
        _require(rows >= 0 and cols > 0 and cols % 32 == 0,
                 "rows must not be negative, cols a positive multiple of 32")
        _require(isinstance(data, torch.Tensor) and data.dtype is torch.uint8 and data.is_contiguous()
                 and data.numel() >= _capi.load().et_mxfp4_bytes(rows, cols),
                 "data must be a contiguous uint8 tensor that holds rows x cols values (empty() makes one)")
        self.data, self.rows, self.cols = data, rows, cols
        self.ptr, self.device = data.data_ptr(), data.get_device()

    def __repr__(self) -> str:
        return f"MxTensor({self.rows} x {self.cols}, {self.data.device})"


def _require(ok: bool, message: str) -> None:
    if not ok:
        raise ValueError(message)


# The checks run in front of every launch, and for few rows they are what a call costs: one comparison per property,
# and the text of an error is put together only when it is raised.  Devices are compared by index (get_device(), -1 on
# the CPU).

def _check(t: torch.Tensor, name: str, shape, dtype: torch.dtype, device: int) -> None:
    try:
        if t.dtype is dtype and t.shape == shape and t.get_device() == device and t.is_contiguous():
            return
    except AttributeError:  # not a tensor
        pass
    raise ValueError(f"{name} must be a contiguous {list(shape)} tensor of dtype {dtype} on cuda:{device}")


def _check_rows(x: torch.Tensor, name: str):
    """(rows, width, row stride, device) of a matrix whose rows may be strided."""
    if not (isinstance(x, torch.Tensor) and x.dtype in _DTYPE and x.dim() == 2 and x.is_cuda):
        raise ValueError(f"{name} must be a [rows, width] CUDA tensor of dtype torch.float16 or torch.float32")
    rows, width = x.shape
    if width <= 0 or width % 32 != 0:
        raise ValueError(f"the width of {name} must be a positive multiple of 32")
    stride, step = x.stride()
    if step != 1:
        raise ValueError(f"the values of a row of {name} must be contiguous")
    return rows, width, stride if rows > 1 else width, x.get_device()   # (torch gives a single row any stride)


def _count(valid_rows: Optional[torch.Tensor], device: int) -> Optional[int]:
    if valid_rows is None:
        return None
    try:
        if valid_rows.dtype is torch.int32 and valid_rows.numel() == 1 and valid_rows.get_device() == device:
            return valid_rows.data_ptr()
    except AttributeError:  # not a tensor
        pass
    raise ValueError("valid_rows must be one int32 on the rows' device")


def _check_mx(t: "MxTensor", name: str, rows: int, cols: int, device: int) -> None:
    if not (isinstance(t, MxTensor) and t.cols == cols and t.rows >= rows and t.device == device):
        raise ValueError(f"{name} must be an MxTensor of at least {rows} rows of {cols} values on cuda:{device}")


def _wants_gradient(*tensors: Optional[torch.Tensor]) -> bool:
    if not torch.is_grad_enabled():
        return False
    for t in tensors:
        if t is not None and t.requires_grad:
            return True
    return False


_NO_BACKWARD = "4-bit operators and gated norms have no backward pass: "


class _NoBackward(torch.autograd.Function):
    """Results (the first `count` tensors) tied to the tensors that require a gradient."""

    @staticmethod
    def forward(ctx, count: int, *tensors):
        ctx.mark_dirty(*tensors[:count])
        return tensors[:count]

    @staticmethod
    def backward(ctx, *_):
        raise NotImplementedError(_NO_BACKWARD + "call them under torch.no_grad(), or detach what goes in")


def _tie(results, *tensors):
    """New results of a call that was given tensors with a gradient."""
    return _NoBackward.apply(len(results), *results, *(t for t in tensors if t is not None and t.requires_grad))


def _refuse_gradients() -> None:
    raise ValueError(_NO_BACKWARD + "with a given buffer or an MXFP4 tensor for the result, call them under "
                     "torch.no_grad(), or detach what goes in")


def _call(device: int, name: str, *args) -> None:
    """One entry point of the library on the current stream of `device` (it launches on the current device)."""
    global _lib
    if _lib is None:
        _lib = _capi.load()
    stream = torch._C._cuda_getCurrentRawStream(device)
    if torch._C._cuda_getDevice() == device:
        rc = getattr(_lib, name)(*args, stream)
    else:
        with torch.cuda.device(device):
            rc = getattr(_lib, name)(*args, stream)
    if rc != 0:
        _capi.check(rc)


def _status_word(device: int) -> int:
    """Address of the device's status word, one for all threads: a kernel may write to it at any time."""
    word = _status.get(device)
    if word is None:
        with _status_lock, torch.cuda.device(device):
            word = _status.get(device)
            if word is None:
                _require(not torch.cuda.is_current_stream_capturing(),
                         "call mxfp4.device_status(device) once before a product is captured on this device")
                data = torch.zeros(1, dtype=torch.int32, device=torch.device("cuda", device))
                torch.cuda.current_stream(device).synchronize()  # (other streams may use it from now on)
                word = _status[device] = (data.data_ptr(), data)
    return word[0]


def device_status(device: Union[int, str, torch.device] = "cuda") -> int:
    """0, or the code of a bounded device-side wait that ran out in a product on this device since the last call
    (its results are then incomplete).  Waits for the device's current stream."""
    device = torch.device(device) if not isinstance(device, int) else torch.device("cuda", device)
    index = torch.cuda.current_device() if device.index is None else device.index
    _status_word(index)
    data = _status[index][1]
    with torch.cuda.device(index):
        code = int(data.item())
        if code != 0:
            data.zero_()
    return code


def empty(rows: int, cols: int, device: Union[str, torch.device] = "cuda") -> MxTensor:
    """An uninitialised MXFP4 tensor (an output or workspace of the calls below)."""
    _require(rows >= 0 and cols > 0 and cols % 32 == 0, "rows must not be negative, cols a positive multiple of 32")
    size = _capi.load().et_mxfp4_bytes(rows, cols)
    return MxTensor(torch.empty(size, dtype=torch.uint8, device=device), rows, cols)


def quantize(x: torch.Tensor, valid_rows: Optional[torch.Tensor] = None, out: Optional[MxTensor] = None) -> MxTensor:
    """Rows of x [rows, width] to MXFP4 (rows may be strided, the values of a row are contiguous)."""
    rows, k, stride, device = _check_rows(x, "x")
    if _wants_gradient(x):
        _refuse_gradients()
    count = _count(valid_rows, device)
    if out is None:
        out = empty(rows, k, x.device)
    _check_mx(out, "out", rows, k, device)
    _call(device, "et_mxfp4_quantize", _DTYPE[x.dtype], x.data_ptr(), stride, count, rows, k, out.ptr)
    return out


def dequantize(mx: MxTensor, dtype: torch.dtype, valid_rows: Optional[torch.Tensor] = None,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The values that an MXFP4 tensor stands for, as [rows, cols] of `dtype`."""
    _require(isinstance(mx, MxTensor) and mx.device >= 0, "mx must be an MxTensor on a GPU")
    _require(dtype in _DTYPE, "dtype must be torch.float16 or torch.float32")
    if out is None:
        out = torch.empty(mx.rows, mx.cols, dtype=dtype, device=mx.data.device)
    rows = out.shape[0]
    _require(rows <= mx.rows, "out has more rows than mx")
    _check(out, "out", (rows, mx.cols), dtype, mx.device)
    _call(mx.device, "et_mxfp4_dequantize", _DTYPE[dtype], mx.ptr, _count(valid_rows, mx.device), rows, mx.cols,
          out.data_ptr())
    return out


def pack_weight(kernel: torch.Tensor) -> MxTensor:
    """A projection's kernel [in, out] (TF dense layout) to the MXFP4 operand of gemm and linear."""
    _require(isinstance(kernel, torch.Tensor) and kernel.is_cuda and kernel.dtype in _DTYPE and kernel.dim() == 2
             and kernel.is_contiguous(), "kernel must be a contiguous [in, out] CUDA tensor, torch.float16 or torch.float32")
    k, n = kernel.shape
    _require(k > 0 and n > 0 and k % 32 == 0 and n % 32 == 0, "in and out must be positive multiples of 32")
    w = empty(n, k, kernel.device)
    _call(w.device, "et_mxfp4_pack_weight", _DTYPE[kernel.dtype], kernel.data_ptr(), w.ptr, k, n)
    return w


def _result(rows: int, device: int, weight: MxTensor, bias, activation, residual, valid_rows, out, dtype: torch.dtype):
    """(out, arguments of the entry points from the bias on) of a product of `rows` rows."""
    n = weight.rows
    epilogue = _EPILOGUE.get(activation)
    if epilogue is None:
        raise ValueError("activation must be None, 'gelu' or 'tanh'")
    c = c_mx = bias_ptr = res_ptr = None
    if isinstance(out, MxTensor):
        _check_mx(out, "out", rows, n, device)
        _require(n % 64 == 0 and residual is None, "MXFP4 output needs a width that is a multiple of 64, and no residual")
        c_mx = out.ptr
    else:
        if out is None:
            out = torch.empty(rows, n, dtype=dtype, device=torch.device("cuda", device))
        else:
            _check(out, "out", (rows, n), dtype, device)
        c = out.data_ptr()
    if bias is not None:
        _check(bias, "bias", (n,), dtype, device)
        bias_ptr = bias.data_ptr()
    elif activation is None:
        epilogue = 0
    else:
        raise ValueError("an activation needs a bias")
    if residual is not None:
        _check(residual, "residual", (rows, n), dtype, device)
        res_ptr = residual.data_ptr()
    return out, (bias_ptr, res_ptr, c, c_mx, None if valid_rows is None else _count(valid_rows, device), rows, n,
                 weight.cols, epilogue, _status_word(device))


def gemm(a: MxTensor, weight: MxTensor, bias: Optional[torch.Tensor] = None, activation: Optional[str] = None,
         residual: Optional[torch.Tensor] = None, dtype: Optional[torch.dtype] = None,
         valid_rows: Optional[torch.Tensor] = None,
         out: Union[torch.Tensor, MxTensor, None] = None) -> Union[torch.Tensor, MxTensor]:
    """act(A W + bias) (+ residual) on rows that are in MXFP4 already.  The result has the dtype of out, bias or
    residual, or `dtype` (torch.float16 where nothing says); an MxTensor as out keeps it in 4 bits.  out may be residual;
    it shares no memory with the other operands."""
    _require(isinstance(a, MxTensor) and isinstance(weight, MxTensor), "a and weight must be MxTensors")
    _require(a.cols == weight.cols and a.device == weight.device >= 0,
             "a and weight must have one inner width and be on one GPU")
    plain = isinstance(out, torch.Tensor)
    rows = out.shape[0] if plain else a.rows
    _require(rows <= a.rows, "out has more rows than a")
    if dtype is None:
        given = out if plain else bias if bias is not None else residual
        dtype = torch.float16 if given is None else given.dtype
    _require(dtype in _DTYPE, "dtype must be torch.float16 or torch.float32")
    given = out
    out, args = _result(rows, a.device, weight, bias, activation, residual, valid_rows, out, dtype)
    gradient = _wants_gradient(bias, residual)
    if gradient and given is not None:
        _refuse_gradients()
    _call(a.device, "et_mxfp4_gemm", _DTYPE[dtype], a.ptr, weight.ptr, *args)
    return _tie((out,), bias, residual)[0] if gradient else out


def linear(x: torch.Tensor, weight: MxTensor, bias: Optional[torch.Tensor] = None, activation: Optional[str] = None,
           residual: Optional[torch.Tensor] = None, valid_rows: Optional[torch.Tensor] = None,
           workspace: Optional[MxTensor] = None,
           out: Union[torch.Tensor, MxTensor, None] = None) -> Union[torch.Tensor, MxTensor]:
    """gemm(quantize(x), weight, ...) in one call; the result has x's dtype.  `workspace`: an MxTensor of x's shape that
    the call may use (a program that calls this in a loop keeps one per stream); few rows need none.  out may be x or
    residual; it shares no memory with the weight, the bias or the workspace."""
    rows, k, stride, device = _check_rows(x, "x")
    _require(isinstance(weight, MxTensor) and weight.cols == k and weight.device == device,
             "weight must be an MxTensor of x's width and device")
    if workspace is None:
        workspace = empty(rows, k, x.device)
    _check_mx(workspace, "workspace", rows, k, device)
    dtype = x.dtype
    given = out
    out, args = _result(rows, device, weight, bias, activation, residual, valid_rows, out, dtype)
    gradient = _wants_gradient(x, bias, residual)
    if gradient and given is not None:
        _refuse_gradients()
    _call(device, "et_mxfp4_linear", _DTYPE[dtype], x.data_ptr(), stride, workspace.ptr, weight.ptr, *args)
    return _tie((out,), x, bias, residual)[0] if gradient else out
