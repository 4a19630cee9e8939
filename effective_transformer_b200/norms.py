"""The norms before and after a block, fused with the block's gate and residual scale.

    h, y = norms.gated_residual_norm(x, residual=h, bias=b, post_norm="layer", post_gamma=g1, post_beta=b1,
                                     gate=gate, batch_idx=batch_idx, residual_scale=alpha,
                                     pre_norm="layer", pre_gamma=g2, pre_beta=b2)

p = post(x + bias);  h = residual_scale * residual + gate * p;  y = pre(h)   (include/et_b200.h, et_gated_residual_norm)

There is no backward pass: tensors that require a gradient are taken as effective_transformer_b200.mxfp4 takes them.
"""
from __future__ import annotations

import struct
from typing import Optional, Tuple

import torch

from .mxfp4 import (MxTensor, _call, _check, _check_mx, _count, _DTYPE, _refuse_gradients, _require, _tie,
                    _wants_gradient)

__all__ = ["gated_residual_norm"]

_KIND = {"none": 0, "layer": 1, "rms": 2}
_PARAM = struct.Struct("@13P5i2f4x")  # _capi.GatedNormParam, put together in a third of the time


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

    gate [width] or [1, width], for every row; or [sequences, width] with batch_idx int32 [rows] (of the input op; any shape
    with at least that many entries), where a row whose batch_idx is outside the gate's rows has gate 0.  eps <= 0 selects
    1e-6.  post_norm / pre_norm: "none", "layer" or
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
    if post is None or pre is None:
        raise ValueError("post_norm and pre_norm must be 'none', 'layer' or 'rms'")
    fresh = h_out is None and y_out is None and mx_out is None
    bias_p = res_p = gate_p = idx_p = post_g = post_b = pre_g = pre_b = y_p = mx_p = 0
    if h_out is None:
        h_out = torch.empty_like(x)
    else:
        _check(h_out, "h_out", shape, dtype, device)
    h_p = h_out.data_ptr()
    if y_out is None and mx_out is None:
        y_out = torch.empty_like(x)
        y_p = y_out.data_ptr()
    elif y_out is not None:
        _check(y_out, "y_out", shape, dtype, device)
        y_p = y_out.data_ptr()
        if y_p == h_p and rows > 0:
            raise ValueError("h_out and y_out must be two buffers")
    if residual is not None:
        _check(residual, "residual", shape, dtype, device)
        res_p = residual.data_ptr()
    if bias is not None:
        _check(bias, "bias", row, dtype, device)
        bias_p = bias.data_ptr()
    # (a norm's missing gamma or beta fails its check)
    if post != 0:
        _check(post_gamma, "post_gamma", row, dtype, device)
        post_g = post_gamma.data_ptr()
        if post == 1:
            _check(post_beta, "post_beta", row, dtype, device)
            post_b = post_beta.data_ptr()
    if pre != 0:
        _check(pre_gamma, "pre_gamma", row, dtype, device)
        pre_g = pre_gamma.data_ptr()
        if pre == 1:
            _check(pre_beta, "pre_beta", row, dtype, device)
            pre_b = pre_beta.data_ptr()
    gate_rows = 0
    if gate is not None:
        _require(isinstance(gate, torch.Tensor) and gate.dim() in (1, 2), "gate must be [width] or [sequences, width]")
        gate_rows = 1 if gate.dim() == 1 else gate.shape[0]
        _check(gate, "gate", row if gate.dim() == 1 else (gate_rows, n), dtype, device)
        _require(gate_rows >= 1, "gate must have a row")
        gate_p = gate.data_ptr()
        if gate_rows > 1:
            _require(isinstance(batch_idx, torch.Tensor) and batch_idx.dtype is torch.int32
                     and batch_idx.is_contiguous() and batch_idx.get_device() == device and batch_idx.numel() >= rows,
                     "a gate of several rows needs batch_idx, int32, one entry per row of x")
            idx_p = batch_idx.data_ptr()
    if mx_out is not None:
        _check_mx(mx_out, "mx_out", rows, n, device)
        mx_p = mx_out.ptr
    # (what a norm does not use has been ignored above and is here)
    inputs = (x, bias, residual, gate, post_gamma if post_g else None, post_beta if post_b else None,
              pre_gamma if pre_g else None, pre_beta if pre_b else None)
    gradient = _wants_gradient(*inputs)
    if gradient and not fresh:
        _refuse_gradients()
    try:
        p = _PARAM.pack(x.data_ptr(), bias_p, res_p, gate_p, idx_p, post_g, post_b, pre_g, pre_b, h_p, y_p, mx_p,
                        0 if valid_rows is None else _count(valid_rows, device), rows, n, gate_rows, post, pre,
                        residual_scale, eps)
    except (struct.error, OverflowError) as e:
        raise ValueError("residual_scale and eps must be numbers that fp32 has, and sizes fit 32 bits") from e
    _call(device, "et_gated_residual_norm", _DTYPE[dtype], p)
    if gradient:
        return _tie((h_out, y_out), *inputs)
    return h_out, y_out
