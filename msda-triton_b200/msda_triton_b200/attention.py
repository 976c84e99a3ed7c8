"""Masked attention on the B200 kernels (csrc/layer_attention*.cu).

The dense attention that stands beside deformable attention in a transformer:
self-attention among object queries (with denoising groups), packed texts,
prefix and causal masks, capped scores and distance biases, for training; and
the form for single tokens over a cache of keys and values. The masks are
ids and lengths, never a (Sq, Sk) tensor. Forward and backward are bitwise
reproducible. There is no CPU path.
"""

from __future__ import annotations

import struct

import torch

from . import _lib
from .ops import _DTYPE_CODE, _FLOAT_DTYPES, _apply, _device_guard, _once, _raw_stream, _wants_node

# msda_attention_args of include/msda_layer_b200.h, packed in one call.
_ARGS = struct.Struct("@10P3q4i12q2f5P2iPN")

_FLOAT_MAX = torch.finfo(torch.float32).max
# Wider and narrower caps leave 32 bits once they are taken to base 2 or divided by.
_CAP_MIN, _CAP_MAX = 2.0**-100, 2.0**100


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


def _pack(query, key, value, out, residue, lse, grads, options, tensors, ws=0, nbytes=0) -> bytes:
    """`grads`: (grad_out, and the three gradients' buffers), or None."""
    B, Sq, H, D = query.shape
    scale, softcap, causal, shared = options
    go, dq, dk, dv = (0, 0, 0, 0) if grads is None else [t.data_ptr() for t in grads]
    gs = (0, 0, 0) if grads is None else grads[0].stride()[:3]
    return _ARGS.pack(
        query.data_ptr(), key.data_ptr(), value.data_ptr(), out.data_ptr(),
        0 if residue is None else residue.data_ptr(), 0 if lse is None else lse.data_ptr(), go, dq, dk, dv,
        B, Sq, key.shape[1], H, key.shape[2], D, _DTYPE_CODE[query.dtype],
        *query.stride()[:3], *key.stride()[:3], *value.stride()[:3], *gs, scale, softcap,
        *[0 if t is None else t.data_ptr() for t in tensors], shared, causal, ws, nbytes)


def _call(fn, name: str, args, backward: int) -> None:
    lib = _lib.load()
    packed = _pack(*args)
    device = args[0].device
    with _device_guard(device):
        nbytes = lib.msda_attention_workspace_size(packed, backward)
        if nbytes:
            ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
            packed = packed[:-16] + struct.pack("@PN", ws.data_ptr(), nbytes)
        rc = fn(packed, _raw_stream(device))
    if rc:
        _lib.check(name, rc)


def _forward(query, key, value, options, tensors, want_lse, grad):
    """(out, lse or None, query, key, value as they were read, residue or None)."""
    query, key, value = _laid_out(query), _laid_out(key), _laid_out(value)
    B, Sq, H, _ = query.shape
    out = query.new_empty(query.shape)
    lse = torch.empty(B, H, Sq, dtype=torch.float32, device=query.device) if grad or want_lse else None
    residue = torch.empty_like(out) if grad and query.element_size() == 2 else None
    if out.numel():
        _call(_lib.load().msda_attention_forward, "msda_attention_forward",
              (query, key, value, out, residue, lse, None, options, tensors), 0)
    return out, lse, query, key, value, residue


class _AttentionFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, key, value, options, tensors):
        out, lse, *saved = _forward(query, key, value, options, tensors, True, True)
        ctx.save_for_backward(out, lse, *saved, *tensors)
        ctx.options = options
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    @_once
    def backward(ctx, grad_out, _):
        if grad_out is None:
            return (None,) * 5
        out, lse, query, key, value, residue, *tensors = ctx.saved_tensors
        grad_out = _laid_out(grad_out if grad_out.dtype == query.dtype else grad_out.to(query.dtype))
        dq, dk, dv = query.new_empty(query.shape), key.new_empty(key.shape), key.new_empty(key.shape)
        _call(_lib.load().msda_attention_backward, "msda_attention_backward",
              (query, key, value, out, residue, lse, (grad_out, dq, dk, dv), ctx.options, tensors), 1)
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

    With ``Sq == Sk`` and items padded at their end, ``key_lengths`` would thus
    shift an item's places, its causal mask and its distances by its padding:
    such prompts mark their padding by negative document ids instead (all else
    id 0), and leave ``key_lengths`` out.

    Args:
        query: ``(B, Sq, H, D)``, fp32, fp16 or bf16, ``D <= 256``.
        key, value: ``(B, Sk, Hkv, D)``, ``H`` a multiple of ``Hkv``: head
            ``h`` reads key head ``h // (H // Hkv)``.
        scale: of the scores; ``D ** -0.5`` by default.
        softcap: ``c > 0`` makes a score ``c * tanh(score / c)``; 0: not.
            From ``2**-100`` to ``2**100``.
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
        key_lengths: ``(B,)`` int32, visible keys of each item, the last of
            which is the last query's own (see above). What lies past them is
            never read into a result.
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
    if not abs(scale) <= _FLOAT_MAX or not (softcap == 0.0 or _CAP_MIN <= softcap <= _CAP_MAX and abs(scale) <= _FLOAT_MAX * softcap):
        raise ValueError(f"attention: scale must be finite in 32 bits and softcap 0 or from 2**-100 to 2**100 (scale / softcap "
                         f"finite too), got {scale} and {softcap}")
    if (query_documents is None) != (key_documents is None):
        raise ValueError("attention: query_documents and key_documents come together")
    if shared_document is not None and (key_documents is None or not 0 <= shared_document < 2**31):
        raise ValueError("attention: shared_document is an int32 id >= 0 and needs documents")
    if prefix_lengths is not None and not causal:
        raise ValueError("attention: prefix_lengths needs causal=True")
    device = query.device
    tensors = (distance_slopes, query_documents, key_documents, prefix_lengths, key_lengths)
    if any(t is not None for t in tensors):
        shapes = ((H,), (B, Sq), (B, Sk), (B,), (B,))
        for name, t, shape in zip(("distance_slopes", "query_documents", "key_documents", "prefix_lengths",
                                   "key_lengths"), tensors, shapes):
            if t is None:
                continue
            dtype = torch.float32 if t is distance_slopes else torch.int32
            if t.shape != shape or t.dtype != dtype:
                raise ValueError(f"attention: {name} must be {shape} {dtype}, got {tuple(t.shape)} {t.dtype}")
            if t.device != device:
                raise ValueError("attention: all tensors must be on the same CUDA device")
        if distance_slopes is not None and distance_slopes.requires_grad:
            raise ValueError("attention: distance_slopes are constants and may not require a gradient; detach() them")
        tensors = tuple(None if t is None else t.contiguous() for t in tensors)
    if device.type != "cuda":
        raise ValueError("attention requires CUDA tensors on a B200 (sm_100a) GPU")
    if key.device != device or value.device != device:
        raise ValueError("attention: all tensors must be on the same CUDA device")
    options = (scale, softcap, 1 if causal else 0, -1 if shared_document is None else int(shared_document))
    if _wants_node(query, key, value):
        out, lse = _apply(_AttentionFunction, query, key, value, options, tensors)
    else:
        out, lse, *_ = _forward(query, key, value, options, tensors, return_lse, False)
    return (out, lse) if return_lse else out
