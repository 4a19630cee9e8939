"""The norms before and after a block, fused with the block's gate and residual scale.

    h, y = norms.gated_residual_norm(x, residual=h, bias=b, post_norm="layer", post_gamma=g1, post_beta=b1,
                                     gate=gate, batch_idx=batch_idx, residual_scale=alpha,
                                     pre_norm="layer", pre_gamma=g2, pre_beta=b2)

p = post(x + bias);  h = residual_scale * residual + gate * p;  y = pre(h)   (include/et_b200.h, et_gated_residual_norm)
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch

from . import _capi
from .mxfp4 import MxTensor, _call, _check, _check_mx, _count, _DTYPE, _ptr, _require

__all__ = ["gated_residual_norm"]

_KIND = {"none": 0, "layer": 1, "rms": 2}


def gated_residual_norm(x: torch.Tensor, bias: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
                        residual_scale: float = 1.0, gate: Optional[torch.Tensor] = None,
                        batch_idx: Optional[torch.Tensor] = None, post_norm: str = "none",
                        post_gamma: Optional[torch.Tensor] = None, post_beta: Optional[torch.Tensor] = None,
                        pre_norm: str = "layer", pre_gamma: Optional[torch.Tensor] = None,
                        pre_beta: Optional[torch.Tensor] = None, eps: float = 1e-6,
                        valid_rows: Optional[torch.Tensor] = None, h_out: Optional[torch.Tensor] = None,
                        y_out: Optional[torch.Tensor] = None, mx_out: Optional[MxTensor] = None
                        ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(h, y) of packed rows x [rows, width], fp16 or fp32.

    gate [width], or [sequences, width] with batch_idx int32 [rows] (of the input op; any shape with at least that many
    entries).  A row whose batch_idx is outside the gate's rows has gate 0.  post_norm / pre_norm: "none", "layer" or
    "rms"; parameters of a norm that is not used are ignored.  valid_rows: device int32 [1], rows past it are left as
    they are.  h_out / y_out: buffers for the results, either may be x or residual.  mx_out takes y in MXFP4 for the
    projection behind it; y itself is then written only where y_out is given (None is returned otherwise).  The width
    is a multiple of 16 bytes (of 32 with mx_out), at most 8192 (fp16) or 4096 (fp32)."""
    if not (isinstance(x, torch.Tensor) and x.dtype in _DTYPE and x.dim() == 2 and x.is_cuda and x.is_contiguous()):
        raise ValueError("x must be a contiguous [rows, width] CUDA tensor of dtype torch.float16 or torch.float32")
    shape, dtype, device = x.shape, x.dtype, x.get_device()
    rows, n = shape
    row = (n,)
    post, pre = _KIND.get(post_norm), _KIND.get(pre_norm)
    _require(post is not None and pre is not None, "post_norm and pre_norm must be 'none', 'layer' or 'rms'")
    if h_out is None:
        h_out = torch.empty_like(x)
    if y_out is None and mx_out is None:
        y_out = torch.empty_like(x)
    h_ptr, y_ptr = h_out.data_ptr(), _ptr(y_out)
    _require(h_ptr != y_ptr or rows == 0, "h_out and y_out must be two buffers")
    _check(residual, "residual", shape, dtype, device)
    _check(h_out, "h_out", shape, dtype, device)
    _check(y_out, "y_out", shape, dtype, device)
    if post != 0:
        _require(post_gamma is not None and (post != 1 or post_beta is not None), "post_norm needs its gamma (and beta)")
        _check(post_gamma, "post_gamma", row, dtype, device)
        if post == 1:
            _check(post_beta, "post_beta", row, dtype, device)
    if pre != 0:
        _require(pre_gamma is not None and (pre != 1 or pre_beta is not None), "pre_norm needs its gamma (and beta)")
        _check(pre_gamma, "pre_gamma", row, dtype, device)
        if pre == 1:
            _check(pre_beta, "pre_beta", row, dtype, device)
    _check(bias, "bias", row, dtype, device)
    gate_rows, idx = 0, None
    if gate is not None:
        gate_rows = 1 if gate.dim() == 1 else gate.shape[0]
        _check(gate, "gate", row if gate.dim() == 1 else (gate_rows, n), dtype, device)
        _require(gate_rows >= 1, "gate must have a row")
        if gate_rows > 1:
            _require(isinstance(batch_idx, torch.Tensor) and batch_idx.dtype is torch.int32
                     and batch_idx.is_contiguous() and batch_idx.get_device() == device and batch_idx.numel() >= rows,
                     "a gate of several rows needs batch_idx, int32, one entry per row of x")
            idx = batch_idx.data_ptr()
    if mx_out is not None:
        _check_mx(mx_out, "mx_out", rows, n, device)
    p = _capi.GatedNormParam(
        x.data_ptr(), _ptr(bias), _ptr(residual), _ptr(gate), idx, _ptr(post_gamma) if post != 0 else None,
        _ptr(post_beta) if post == 1 else None, _ptr(pre_gamma) if pre != 0 else None,
        _ptr(pre_beta) if pre == 1 else None, h_ptr, y_ptr, None if mx_out is None else mx_out.ptr,
        _count(valid_rows, device), rows, n, gate_rows, post, pre, residual_scale, eps)
    _call(device, "et_gated_residual_norm", _DTYPE[dtype], C.byref(p))
    return h_out, y_out
