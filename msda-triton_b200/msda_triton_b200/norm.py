"""Layer norm with an optional residual on the B200 kernels (csrc/layer_norm.cu).

``layer_norm(x, weight, bias, residual=r)`` is the step that follows every
sublayer of a transformer: the residual is added in fp32 inside the kernel, so
neither the sum nor its gradient makes a trip of its own through memory. The
weight's and bias's gradients are summed in a fixed order: the backward is
bitwise reproducible. There is no CPU path.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .ops import _DTYPE_CODE, _FLOAT_DTYPES, _device_guard, _ptr, _stream


def _as_rows(x: torch.Tensor) -> torch.Tensor:
    """x (..., C) as (N, C) rows of contiguous channels: a view where the
    strides allow one, else a copy."""
    x = x.reshape(-1, x.shape[-1])
    return x if x.shape[1] == 1 or x.stride(1) == 1 else x.contiguous()


class _LayerNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps, want_sum):
        rows = _as_rows(x)
        res = _as_rows(residual) if residual is not None else None
        N, C = rows.shape
        y = rows.new_empty(x.shape)
        total = rows.new_empty(x.shape) if want_sum else None
        grad = any(ctx.needs_input_grad)
        stats = torch.empty(2, N, dtype=torch.float32, device=x.device) if grad else None
        param = weight if weight is not None else bias
        code = _DTYPE_CODE[x.dtype]
        lib = _lib.load()
        with _device_guard(x.device):
            rc = lib.msda_layer_norm_forward(
                _ptr(rows), _ptr(res), _ptr(weight), _ptr(bias), _ptr(y), _ptr(total),
                _ptr(stats[0] if grad else None), _ptr(stats[1] if grad else None), N, C, rows.stride(0),
                res.stride(0) if res is not None else 0, eps, code,
                _DTYPE_CODE[param.dtype] if param is not None else code, _stream(x.device))
        _lib.check("msda_layer_norm_forward", rc)
        if grad:
            ctx.save_for_backward(rows, res, weight, bias, stats)
        ctx.shape = x.shape
        ctx.set_materialize_grads(False)
        return y, total

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y, grad_sum):
        rows, res, weight, bias, stats = ctx.saved_tensors
        N, C = rows.shape
        if grad_y is None:
            grad_y = rows.new_zeros(N, C)
        g = _as_rows(grad_y.to(rows.dtype))
        gs = _as_rows(grad_sum.to(rows.dtype)).contiguous() if grad_sum is not None else None
        dx = rows.new_empty(ctx.shape)
        dw = torch.empty_like(weight) if weight is not None and ctx.needs_input_grad[2] else None
        db = torch.empty_like(bias) if bias is not None and ctx.needs_input_grad[3] else None
        lib = _lib.load()
        columns = dw is not None or db is not None
        nbytes = lib.msda_layer_norm_backward_workspace_size(N, C) if columns else 0
        ws = torch.empty(nbytes, dtype=torch.uint8, device=rows.device) if nbytes else None
        code = _DTYPE_CODE[rows.dtype]
        param = weight if weight is not None else bias
        with _device_guard(rows.device):
            rc = lib.msda_layer_norm_backward(
                _ptr(rows), _ptr(res), _ptr(weight), _ptr(stats[0]), _ptr(stats[1]), _ptr(g), _ptr(gs), _ptr(dx),
                _ptr(dw), _ptr(db), _ptr(ws), nbytes, N, C, rows.stride(0), res.stride(0) if res is not None else 0,
                g.stride(0), code, _DTYPE_CODE[param.dtype] if param is not None else code, _stream(rows.device))
        _lib.check("msda_layer_norm_backward", rc)
        return dx, dx if res is not None else None, dw, db, None, None


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
    if x.dtype not in _FLOAT_DTYPES:
        raise ValueError(f"layer_norm: unsupported dtype {x.dtype}; use fp32, fp16 or bf16")
    params = [p for p in (weight, bias) if p is not None]
    for p in params:
        if p.shape != (C,):
            raise ValueError(f"layer_norm: weight and bias must be ({C},), got {tuple(p.shape)}")
        if p.dtype != params[0].dtype or p.dtype not in (x.dtype, torch.float32):
            raise ValueError(f"layer_norm: weight and bias must both be {x.dtype} or fp32, got "
                             f"{'/'.join(str(q.dtype) for q in params)}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"layer_norm: residual must be {tuple(x.shape)} {x.dtype}, got "
                         f"{tuple(residual.shape)} {residual.dtype}")
    if not eps >= 0:
        raise ValueError(f"layer_norm: eps must be >= 0, got {eps}")
    if x.device.type != "cuda":
        raise ValueError("layer_norm requires CUDA tensors on a B200 (sm_100a) GPU")
    if any(t.device != x.device for t in params + ([residual] if residual is not None else [])):
        raise ValueError("layer_norm: all tensors must be on the same CUDA device")
    _lib.load()
    y, total = _LayerNormFunction.apply(
        x, residual, weight.contiguous() if weight is not None else None,
        bias.contiguous() if bias is not None else None, float(eps), bool(return_sum))
    return (y, total) if return_sum else y
