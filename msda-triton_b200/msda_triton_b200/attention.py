"""Masked attention on the B200 kernels (csrc/layer_attention*.cu).

The dense attention that stands beside deformable attention in a transformer:
self-attention among object queries (with denoising groups), packed texts,
prefix and causal masks, capped scores and distance biases, for training; and
the form for single tokens over a cache of keys and values. The masks are
ids and lengths, never a (Sq, Sk) tensor. Forward and backward are bitwise
reproducible. There is no CPU path.
"""

from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .ops import _DTYPE_CODE, _FLOAT_DTYPES, _device_guard, _stream


def _laid_out(x: torch.Tensor) -> torch.Tensor:
    """x (B, S, H, D) with contiguous channels and, for 16-bit types whose
    heads are whole 16-byte vectors, rows that start on 16 bytes: itself where
    it is so already, else a copy. The kernels take any other strides."""
    D = x.shape[3]
    if D > 1 and x.stride(3) != 1:
        return x.contiguous()
    if x.element_size() == 2 and D % 8 == 0 and (
            x.data_ptr() % 16 or any(n > 1 and (s <= 0 or s % 8) for n, s in zip(x.shape[:3], x.stride()[:3]))):
        return x.clone(memory_format=torch.contiguous_format)
    return x


def _args(query, key, value, out, residue, lse, options) -> _lib.AttentionArgs:
    a = _lib.AttentionArgs()
    a.query, a.key, a.value, a.out = query.data_ptr(), key.data_ptr(), value.data_ptr(), out.data_ptr()
    a.out_residue = residue.data_ptr() if residue is not None else None
    a.lse = lse.data_ptr() if lse is not None else None
    a.batch, a.num_queries, a.num_heads, a.head_dim = query.shape
    a.num_keys, a.num_key_heads = key.shape[1], key.shape[2]
    a.dtype = _DTYPE_CODE[query.dtype]
    a.query_strides[:], a.key_strides[:], a.value_strides[:] = query.stride()[:3], key.stride()[:3], value.stride()[:3]
    a.scale, a.softcap, a.causal, shared, tensors = options
    a.shared_document = shared
    (a.distance_slopes, a.query_documents, a.key_documents, a.prefix_lengths,
     a.key_lengths) = (t.data_ptr() if t is not None else None for t in tensors)
    return a


def _call(fn: str, a: _lib.AttentionArgs, backward: int, device: torch.device) -> None:
    lib = _lib.load()
    nbytes = lib.msda_attention_workspace_size(ctypes.byref(a), backward)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    if ws is not None:
        a.workspace, a.workspace_bytes = ws.data_ptr(), nbytes
    with _device_guard(device):
        rc = getattr(lib, fn)(ctypes.byref(a), _stream(device))
    _lib.check(fn, rc)


class _AttentionFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, key, value, options, want_lse):
        B, Sq, H, D = query.shape
        query, key, value = _laid_out(query), _laid_out(key), _laid_out(value)
        out = query.new_empty(B, Sq, H, D)
        grad = any(ctx.needs_input_grad)
        lse = torch.empty(B, H, Sq, dtype=torch.float32, device=query.device) if grad or want_lse else None
        residue = torch.empty_like(out) if grad and out.element_size() == 2 else None
        if out.numel():
            _call("msda_attention_forward", _args(query, key, value, out, residue, lse, options), 0, query.device)
        if grad:
            ctx.save_for_backward(query, key, value, out, residue, lse, *options[4])
        ctx.options = options[:4]
        if lse is not None:
            ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out, _):
        if grad_out is None:
            return (None,) * 5
        query, key, value, out, residue, lse, *tensors = ctx.saved_tensors
        grad_out = _laid_out(grad_out.to(query.dtype))
        dq = query.new_empty(query.shape)
        dk, dv = key.new_empty(key.shape), value.new_empty(value.shape)
        a = _args(query, key, value, out, residue, lse, (*ctx.options, tensors))
        a.grad_out, a.grad_query, a.grad_key, a.grad_value = (t.data_ptr() for t in (grad_out, dq, dk, dv))
        a.grad_out_strides[:] = grad_out.stride()[:3]
        _call("msda_attention_backward", a, 1, query.device)
        return dq, dk, dv, None, None


def attention(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    *,
    scale: float | None = None,
    softcap: float = 0.0,
    distance_slopes: torch.Tensor | None = None,
    causal: bool = False,
    prefix_lengths: torch.Tensor | None = None,
    query_documents: torch.Tensor | None = None,
    key_documents: torch.Tensor | None = None,
    shared_document: int | None = None,
    key_lengths: torch.Tensor | None = None,
    return_lse: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Attention with capped scores, a distance bias and masks by ids and lengths.

    With ``length = key_lengths[b]`` (or ``Sk``), query ``i`` stands at
    ``place = length - Sq + i`` among the keys: the last query at the last key,
    as when new tokens are appended to a cache. It sees key ``j`` if
    ``j < length`` and the causal and document masks below allow it. A query
    that sees no key gives zeros and no gradient.

    Args:
        query: ``(B, Sq, H, D)``, fp32, fp16 or bf16, ``D <= 256``.
        key, value: ``(B, Sk, Hkv, D)``, ``H`` a multiple of ``Hkv``: head
            ``h`` reads key head ``h // (H // Hkv)``.
        scale: of the scores; ``D ** -0.5`` by default.
        softcap: ``c > 0`` makes a score ``c * tanh(score / c)``; 0: not.
        distance_slopes: ``(H,)`` fp32; subtracts ``slope * |place - j|``.
            A constant: may not require a gradient.
        causal: key ``j`` must lie at ``j <= place``...
        prefix_lengths: ``(B,)`` int32: ...or ``j < prefix_lengths[b]``
            (needs ``causal``).
        query_documents, key_documents: ``(B, Sq)`` and ``(B, Sk)`` int32: a
            query sees the keys of its own document; negative ids are padding,
            which sees nothing and is not seen.
        shared_document: a document whose keys every query that is no padding
            sees (the matching queries beside denoising groups).
        key_lengths: ``(B,)`` int32, visible keys of each item. What lies past
            them is never read into a result.
        return_lse: also return the log-sum-exp of the scores, ``(B, H, Sq)``
            fp32 (-inf for a row that sees no key); not differentiable.

    Returns:
        ``(B, Sq, H, D)`` in ``query.dtype``, contiguous; or ``(out, lse)``.
    """
    if query.dim() != 4:
        raise ValueError(f"attention: query must be (B, Sq, H, D), got {tuple(query.shape)}")
    B, Sq, H, D = query.shape
    if key.dim() != 4 or key.shape[0] != B or key.shape[3] != D:
        raise ValueError(f"attention: key must be ({B}, Sk, Hkv, {D}), got {tuple(key.shape)}")
    if value.shape != key.shape:
        raise ValueError(f"attention: value must be {tuple(key.shape)}, got {tuple(value.shape)}")
    Sk, Hkv = key.shape[1], key.shape[2]
    if not 1 <= D <= _lib.MSDA_ATTENTION_MAX_HEAD_DIM:
        raise ValueError(f"attention: D={D} outside [1, {_lib.MSDA_ATTENTION_MAX_HEAD_DIM}]")
    if H < 1 or Hkv < 1 or H % Hkv:
        raise ValueError(f"attention: H={H} must be a multiple of Hkv={Hkv}")
    if not query.dtype == key.dtype == value.dtype:
        raise ValueError(f"attention: query/key/value dtypes must match, got {query.dtype}/{key.dtype}/{value.dtype}")
    if query.dtype not in _FLOAT_DTYPES:
        raise ValueError(f"attention: unsupported dtype {query.dtype}; use fp32, fp16 or bf16")
    scale = D ** -0.5 if scale is None else float(scale)
    softcap = float(softcap or 0.0)
    if not math.isfinite(scale) or not 0.0 <= softcap < math.inf:
        raise ValueError(f"attention: scale must be finite and softcap finite and >= 0, got {scale} and {softcap}")
    if (query_documents is None) != (key_documents is None):
        raise ValueError("attention: query_documents and key_documents come together")
    if shared_document is not None and (key_documents is None or shared_document < 0):
        raise ValueError("attention: shared_document is an id >= 0 and needs documents")
    if prefix_lengths is not None and not causal:
        raise ValueError("attention: prefix_lengths needs causal=True")
    masks = (("distance_slopes", distance_slopes, (H,), torch.float32),
             ("query_documents", query_documents, (B, Sq), torch.int32),
             ("key_documents", key_documents, (B, Sk), torch.int32),
             ("prefix_lengths", prefix_lengths, (B,), torch.int32),
             ("key_lengths", key_lengths, (B,), torch.int32))
    for name, t, shape, dtype in masks:
        if t is not None and (tuple(t.shape) != shape or t.dtype != dtype):
            raise ValueError(f"attention: {name} must be {shape} {dtype}, got {tuple(t.shape)} {t.dtype}")
    if distance_slopes is not None and distance_slopes.requires_grad:
        raise ValueError("attention: distance_slopes are constants and may not require a gradient; detach() them")
    if query.device.type != "cuda":
        raise ValueError("attention requires CUDA tensors on a B200 (sm_100a) GPU")
    if any(t.device != query.device for t in (key, value, *(m[1] for m in masks)) if t is not None):
        raise ValueError("attention: all tensors must be on the same CUDA device")
    _lib.load()
    options = (scale, softcap, int(bool(causal)), -1 if shared_document is None else int(shared_document),
               tuple(m[1].contiguous() if m[1] is not None else None for m in masks))
    out, lse = _AttentionFunction.apply(query, key, value, options, bool(return_lse))
    return (out, lse) if return_lse else out
