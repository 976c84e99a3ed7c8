"""Rotary positions over several axes on the B200 kernel (csrc/layer_rotary.cu).

A vision transformer turns its channels with height and width (and time), a
detection decoder's queries with their reference points, a text model with one
axis. :func:`rotary` turns the query and the key heads in one launch; its
gradient is the same kernel turning back. There is no CPU path.
"""

from __future__ import annotations

import ctypes
from collections.abc import Sequence

import torch

from . import _lib
from .ops import _DTYPE_CODE, _FLOAT_DTYPES, _apply, _device_guard, _once, _raw_stream, _wants_node

_LADDER = {"axis": 0, "shared": 1}
_PAIRING = {"half": 0, "interleaved": 1}
_POSITION = {torch.float32: _lib.MSDA_POSITION_F32, torch.int32: _lib.MSDA_POSITION_I32,
             torch.int64: _lib.MSDA_POSITION_I64}
_Strides = ctypes.c_int64 * 3


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x with contiguous channels: itself, or a copy."""
    return x if x.shape[-1] <= 1 or x.stride(-1) == 1 else x.contiguous()


def _turn(query, key, positions, axes, base, ladder, pairing, inverse):
    B, S, H, D = query.shape
    query = _rows(query)
    out = query.new_empty(B, S, H, D)
    key_out, key_at, key_to, key_strides, Hkv = None, None, None, None, 0
    if key is not None:
        key, Hkv = _rows(key), key.shape[2]
        key_out = key.new_empty(B, S, Hkv, D)
        key_at, key_to, key_strides = key.data_ptr(), key_out.data_ptr(), _Strides(*key.stride()[:3])
    device = query.device
    with _device_guard(device):
        rc = _lib.load().msda_rotary(
            query.data_ptr(), key_at, positions.data_ptr(), out.data_ptr(), key_to, B, S, H, Hkv, D,
            _Strides(*query.stride()[:3]), key_strides, positions.stride(0) if positions.dim() == 3 else 0,
            _POSITION[positions.dtype], len(axes), axes, base, ladder, pairing, inverse, _DTYPE_CODE[query.dtype],
            _raw_stream(device))
    if rc:
        _lib.check("msda_rotary", rc)
    return out, key_out


class _RotaryFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, key, positions, axes, base, ladder, pairing):
        ctx.save_for_backward(positions)
        ctx.cfg = (axes, base, ladder, pairing)
        ctx.set_materialize_grads(False)
        out, key_out = _turn(query, key, positions, axes, base, ladder, pairing, 0)
        return out if key is None else (out, key_out)

    @staticmethod
    @_once
    def backward(ctx, grad_query, grad_key=None):
        positions, = ctx.saved_tensors
        if grad_query is None and grad_key is None:
            return (None,) * 7
        if grad_query is None:
            return None, _turn(grad_key, None, positions, *ctx.cfg, 1)[0], None, None, None, None, None
        turned = _turn(grad_query, grad_key, positions, *ctx.cfg, 1)
        return turned[0], turned[1], None, None, None, None, None


def rotary(
    query: torch.Tensor,
    positions: torch.Tensor,
    *,
    axis_dims: Sequence[int],
    key: torch.Tensor | None = None,
    base: float = 10000.0,
    ladder: str = "axis",
    pairing: str = "half",
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Turn head channels by their tokens' positions on several axes.

    Step ``k`` of a ladder of ``n`` channels turns one pair of channels by the
    angle ``position * base ** (-2 * k / n)``, formed to about twice fp32's
    precision: long positions cost no accuracy.

    Args:
        query: ``(B, S, H, D)``, fp32, fp16 or bf16; any strides (channels
            that are not contiguous are copied).
        positions: ``(B, S, A)`` or ``(S, A)``, fp32, int32 or int64 (whole
            numbers exact below 2**24). Treated as constants: they may not
            require a gradient.
        axis_dims: ``A`` even channel counts, one for each axis; channels past
            their sum pass through.
        key: ``(B, S, Hkv, D)``, turned in the same launch.
        base: of the frequencies.
        ladder: ``"axis"``: each axis turns its own block of channels, with a
            ladder of its own; ``"shared"``: one ladder over all the turned
            channels, whose steps go to the axes in sections of
            ``axis_dims[a] / 2``.
        pairing: ``"half"``: channels ``k`` and ``k + n / 2`` of a ladder are
            a pair; ``"interleaved"``: channels ``2 k`` and ``2 k + 1``.

    Returns:
        The turned query, or ``(query, key)`` where a key is given; contiguous.
    """
    if query.dim() != 4:
        raise ValueError(f"rotary: query must be (B, S, H, D), got {tuple(query.shape)}")
    B, S, H, D = query.shape
    axis_dims = tuple(axis_dims)
    A = len(axis_dims)
    if not 1 <= A <= _lib.MSDA_ROTARY_MAX_AXES:
        raise ValueError(f"rotary: axis_dims must name 1 to {_lib.MSDA_ROTARY_MAX_AXES} axes, got {A}")
    total = 0
    for d in axis_dims:
        total = D + 1 if d < 0 or d % 2 else total + d
    if total > D:
        raise ValueError(f"rotary: axis_dims must be even and sum to at most D={D}, got {axis_dims}")
    if positions.shape != (B, S, A) and positions.shape != (S, A):
        raise ValueError(f"rotary: positions must be {(B, S, A)} or {(S, A)}, got {tuple(positions.shape)}")
    if positions.dtype not in _POSITION:
        raise ValueError(f"rotary: positions must be fp32, int32 or int64, got {positions.dtype}")
    if positions.requires_grad:
        raise ValueError("rotary: positions are constants and may not require a gradient; detach() them")
    if ladder not in _LADDER:
        raise ValueError(f"rotary: expected ladder to be 'axis' or 'shared', got '{ladder}'")
    if pairing not in _PAIRING:
        raise ValueError(f"rotary: expected pairing to be 'half' or 'interleaved', got '{pairing}'")
    if query.dtype not in _FLOAT_DTYPES:
        raise ValueError(f"rotary: unsupported dtype {query.dtype}; use fp32, fp16 or bf16")
    if key is not None:
        if key.dim() != 4 or key.shape[:2] != query.shape[:2] or key.shape[3] != D:
            raise ValueError(f"rotary: key must be ({B}, {S}, Hkv, {D}), got {tuple(key.shape)}")
        if key.dtype != query.dtype:
            raise ValueError(f"rotary: query/key dtypes must match, got {query.dtype}/{key.dtype}")
    if query.device.type != "cuda":
        raise ValueError("rotary requires CUDA tensors on a B200 (sm_100a) GPU")
    if positions.device != query.device or (key is not None and key.device != query.device):
        raise ValueError("rotary: query, key and positions must be on the same CUDA device")
    if query.numel() == 0 and (key is None or key.numel() == 0):
        return query.clone() if key is None else (query.clone(), key.clone())
    args = (query, key, positions.contiguous(), (ctypes.c_int32 * A)(*axis_dims), float(base), _LADDER[ladder],
            _PAIRING[pairing])
    if _wants_node(query, key):
        return _apply(_RotaryFunction, *args)
    out, key_out = _turn(*args, 0)
    return out if key is None else (out, key_out)
