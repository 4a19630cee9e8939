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
from .mxfp4 import MxTensor, _check, _check_count, _check_mx, _DTYPE, _On, _ptr, _require

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
    _require(isinstance(x, torch.Tensor) and x.is_cuda and x.dtype in _DTYPE and x.dim() == 2 and x.is_contiguous(),
             "x must be a contiguous [rows, width] CUDA tensor of dtype torch.float16 or torch.float32")
    rows, n = x.shape
    dtype, device = x.dtype, x.device
    _require(post_norm in _KIND and pre_norm in _KIND, "post_norm and pre_norm must be 'none', 'layer' or 'rms'")
    if h_out is None:
        h_out = torch.empty_like(x)
    if y_out is None and mx_out is None:
        y_out = torch.empty_like(x)
    for name, t in (("residual", residual), ("h_out", h_out), ("y_out", y_out)):
        _check(t, name, (rows, n), dtype, device)
    _require(y_out is None or y_out.data_ptr() != h_out.data_ptr() or rows == 0, "h_out and y_out must be two buffers")
    for name, t, kinds, kind in (("post_gamma", post_gamma, ("layer", "rms"), post_norm),
                                 ("post_beta", post_beta, ("layer",), post_norm),
                                 ("pre_gamma", pre_gamma, ("layer", "rms"), pre_norm),
                                 ("pre_beta", pre_beta, ("layer",), pre_norm)):
        if kind in kinds:
            _require(t is not None, f"{kind} norm needs {name}")
            _check(t, name, (n,), dtype, device)
    _check(bias, "bias", (n,), dtype, device)
    gate_rows = 0
    if gate is not None:
        gate_rows = 1 if gate.dim() == 1 else gate.shape[0]
        _check(gate, "gate", (n,) if gate.dim() == 1 else (gate_rows, n), dtype, device)
        _require(gate_rows >= 1, "gate must have a row")
    if gate_rows > 1:
        _require(isinstance(batch_idx, torch.Tensor) and batch_idx.dtype == torch.int32 and batch_idx.is_contiguous()
                 and batch_idx.device == device and batch_idx.numel() >= rows,
                 "a gate of several rows needs batch_idx, int32, one entry per row of x")
    _check_count(valid_rows, device)
    if mx_out is not None:
        _check_mx(mx_out, "mx_out", rows, n, device)
    p = _capi.GatedNormParam(
        x.data_ptr(), _ptr(bias), _ptr(residual), _ptr(gate), _ptr(batch_idx) if gate_rows > 1 else None,
        _ptr(post_gamma), _ptr(post_beta), _ptr(pre_gamma), _ptr(pre_beta), h_out.data_ptr(), _ptr(y_out),
        None if mx_out is None else mx_out.data.data_ptr(), _ptr(valid_rows), None, rows, n, gate_rows,
        _KIND[post_norm], _KIND[pre_norm], residual_scale, eps)
    with _On(device) as stream:
        p.stream = stream
        _capi.check(_capi.load().et_gated_residual_norm(_DTYPE[dtype], C.byref(p)))
    return h_out, y_out
