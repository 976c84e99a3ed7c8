"""Layer norm with an optional residual on the B200 kernels (csrc/layer_norm.cu).

``layer_norm(x, weight, bias, residual=r)`` is the step that follows every
sublayer of a transformer: the residual is added in fp32 inside the kernel, so
neither the sum nor its gradient makes a trip of its own through memory. The
weight's and bias's gradients are summed in a fixed order: the backward is
bitwise reproducible. There is no CPU path.
"""

from __future__ import annotations

import torch

from . import _lib
from .ops import _DTYPE_CODE, _FLOAT_DTYPES, _apply, _device_guard, _once, _raw_stream, _wants_node


def _as_rows(x: torch.Tensor) -> torch.Tensor:
    """x (..., C) as (N, C) rows of contiguous channels: a view where the
    strides allow one, else a copy."""
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    return x if x.shape[1] == 1 or x.stride(1) == 1 else x.contiguous()


def _address(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _param_code(code: int, weight, bias) -> int:
    param = weight if weight is not None else bias
    return code if param is None else _DTYPE_CODE[param.dtype]


def _forward(x, residual, weight, bias, eps, want_sum, grad):
    """(y, sum or None, rows, residual rows, statistics or None)."""
    rows = _as_rows(x)
    res = None if residual is None else _as_rows(residual)
    N, C = rows.shape
    y = x.new_empty(x.shape)
    total = x.new_empty(x.shape) if want_sum else None
    stats = mean = rstd = None
    if grad:  # means, then reciprocal deviations
        stats = torch.empty(2 * N, dtype=torch.float32, device=x.device)
        mean = stats.data_ptr()
        rstd = mean + 4 * N
    code = _DTYPE_CODE[x.dtype]
    device = x.device
    with _device_guard(device):
        rc = _lib.load().msda_layer_norm_forward(
            rows.data_ptr(), _address(res), _address(weight), _address(bias), y.data_ptr(), _address(total),
            mean, rstd, N, C, rows.stride(0), 0 if res is None else res.stride(0), eps, code,
            _param_code(code, weight, bias), _raw_stream(device))
    if rc:
        _lib.check("msda_layer_norm_forward", rc)
    return y, total, rows, res, stats


class _LayerNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps, want_sum):
        y, total, *saved = _forward(x, residual, weight, bias, eps, want_sum, True)
        ctx.save_for_backward(weight, bias, *saved)
        ctx.shape = x.shape
        ctx.set_materialize_grads(False)
        return (y, total) if want_sum else y

    @staticmethod
    @_once
    def backward(ctx, grad_y, grad_sum=None):
        weight, bias, rows, res, stats = ctx.saved_tensors
        N, C = rows.shape
        if grad_y is None:
            grad_y = rows.new_zeros(N, C)
        g = _as_rows(grad_y if grad_y.dtype == rows.dtype else grad_y.to(rows.dtype))
        gs = None if grad_sum is None else _as_rows(grad_sum.to(rows.dtype)).contiguous()
        dx = rows.new_empty(ctx.shape)
        dw = torch.empty_like(weight) if weight is not None and ctx.needs_input_grad[2] else None
        db = torch.empty_like(bias) if bias is not None and ctx.needs_input_grad[3] else None
        lib = _lib.load()
        nbytes, ws = 0, None
        if dw is not None or db is not None:
            nbytes = lib.msda_layer_norm_backward_workspace_size(N, C)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=rows.device)
        code = _DTYPE_CODE[rows.dtype]
        device = rows.device
        mean = stats.data_ptr()
        with _device_guard(device):
            rc = lib.msda_layer_norm_backward(
                rows.data_ptr(), _address(res), _address(weight), mean, mean + 4 * N, g.data_ptr(), _address(gs),
                dx.data_ptr(), _address(dw), _address(db), _address(ws), nbytes, N, C, rows.stride(0),
                0 if res is None else res.stride(0), g.stride(0), code, _param_code(code, weight, bias),
                _raw_stream(device))
        if rc:
            _lib.check("msda_layer_norm_backward", rc)
        return dx, None if res is None else dx, dw, db, None, None


def layer_norm(
    x: torch.Tensor,
    weight: torch.Tensor | None = None,
    bias: torch.Tensor | None = None,
    *,
    residual: torch.Tensor | None = None,
    eps: float = 1e-5,
    return_sum: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Layer norm over the last dimension of ``x`` (+ ``residual``).

    Args:
        x: ``(..., C)``, fp32, fp16 or bf16.
        weight, bias: ``(C,)`` in ``x.dtype`` or both in fp32; ``None`` leaves
            that step out.
        residual: of ``x``'s shape and dtype; ``x + residual`` is formed in
            fp32 and not rounded before it is normalised.
        eps: added to the variance.
        return_sum: also return ``x + residual``, rounded (a pre-norm
            layer's next residual).

    Returns:
        ``y``, or ``(y, x + residual)``, in ``x.dtype``, contiguous.
    """
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"layer_norm: x must be (..., C) with C >= 1, got {tuple(x.shape)}")
    C = x.shape[-1]
    if C > _lib.MSDA_LAYER_NORM_MAX_WIDTH:
        raise ValueError(f"layer_norm: C={C} exceeds {_lib.MSDA_LAYER_NORM_MAX_WIDTH}")
    dtype, device = x.dtype, x.device
    if dtype not in _FLOAT_DTYPES:
        raise ValueError(f"layer_norm: unsupported dtype {dtype}; use fp32, fp16 or bf16")
    for p in (weight, bias):
        if p is not None and p.shape != (C,):
            raise ValueError(f"layer_norm: weight and bias must be ({C},), got {tuple(p.shape)}")
        if p is not None and (p.dtype not in (dtype, torch.float32) or
                              (weight is not None and p.dtype != weight.dtype)):
            raise ValueError(f"layer_norm: weight and bias must both be {dtype} or fp32, got "
                             f"{'/'.join(str(q.dtype) for q in (weight, bias) if q is not None)}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != dtype):
        raise ValueError(f"layer_norm: residual must be {tuple(x.shape)} {dtype}, got "
                         f"{tuple(residual.shape)} {residual.dtype}")
    if not eps >= 0:
        raise ValueError(f"layer_norm: eps must be >= 0, got {eps}")
    if device.type != "cuda":
        raise ValueError("layer_norm requires CUDA tensors on a B200 (sm_100a) GPU")
    for t in (weight, bias, residual):
        if t is not None and t.device != device:
            raise ValueError("layer_norm: all tensors must be on the same CUDA device")
    if weight is not None:
        weight = weight.contiguous()
    if bias is not None:
        bias = bias.contiguous()
    if _wants_node(x, weight, bias, residual):
        return _apply(_LayerNormFunction, x, residual, weight, bias, float(eps), bool(return_sum))
    y, total, *_ = _forward(x, residual, weight, bias, float(eps), return_sum, False)
    return (y, total) if return_sum else y
