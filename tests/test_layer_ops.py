"""The operators that complete a transformer layer -- rotary positions, layer
norm, masked attention -- against plain 64-bit forms of their formulas
(layer_reference.py), their gradients against the formulas' and against
differences, and their refusals."""

from __future__ import annotations

import ctypes
import os
import re
import subprocess
import sys
import zlib
from pathlib import Path

import pytest
import torch

import layer_reference as ref
from hostonly import host_only
from layer_reference import close
from msda_triton_b200 import _lib, attention, layer_norm, rotary

DEV = "cuda"
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
HALF = [torch.float16, torch.bfloat16]
gpu = pytest.mark.gpu

ROUNDED = (1.5, 8)  # (norm, element) in u


def randn(*shape, seed=0, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(zlib.crc32(repr((shape, seed)).encode()))
    return (torch.randn(*shape, generator=g) * scale).to(DEV, dtype)


# ---------------------------------------------------------------------------
# Host side
# ---------------------------------------------------------------------------
def test_layer_header_matches_the_binding():
    text = (Path(__file__).resolve().parent.parent / "include" / "msda_layer_b200.h").read_text()
    names = re.findall(r"MSDA_API\s+[\w\s\*]+?\b(msda_\w+)\s*\(", text)
    lib = _lib.load()
    assert len(names) == len(set(names)) >= 7
    for n in names:
        assert hasattr(lib, n) and n in _lib.SIGNATURES
    for macro in ("MSDA_ROTARY_MAX_AXES", "MSDA_ROTARY_MAX_HEAD_DIM", "MSDA_ATTENTION_MAX_HEAD_DIM"):
        assert int(re.search(rf"#define {macro} (\d+)", text).group(1)) == getattr(_lib, macro)


def _cpu(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("call, words", [
    (lambda: rotary(_cpu(2, 3, 4), _cpu(2, 3, 1), axis_dims=[2]), "query must be"),
    (lambda: rotary(_cpu(2, 3, 1, 8), _cpu(2, 3, 2), axis_dims=[4]), "positions must be"),
    (lambda: rotary(_cpu(2, 3, 1, 8), _cpu(2, 3, 1), axis_dims=[3]), "even"),
    (lambda: rotary(_cpu(2, 3, 1, 8), _cpu(2, 3, 2), axis_dims=[6, 4]), "at most D"),
    (lambda: rotary(_cpu(2, 3, 1, 8), _cpu(2, 3, 1, dtype=torch.float64), axis_dims=[4]), "fp32, int32 or int64"),
    (lambda: rotary(_cpu(2, 3, 1, 8), _cpu(2, 3, 1).requires_grad_(), axis_dims=[4]), "require a gradient"),
    (lambda: rotary(_cpu(2, 3, 1, 8), _cpu(2, 3, 1), axis_dims=[4], ladder="both"), "ladder"),
    (lambda: rotary(_cpu(2, 3, 1, 8), _cpu(2, 3, 1), axis_dims=[4], pairing="none"), "pairing"),
    (lambda: rotary(_cpu(2, 3, 1, 8), _cpu(2, 3, 1), axis_dims=[4], key=_cpu(2, 4, 1, 8)), "key must be"),
    (lambda: rotary(_cpu(2, 3, 1, 8), _cpu(2, 3, 1), axis_dims=[4]), "CUDA"),
    (lambda: layer_norm(_cpu(2, 8), _cpu(7)), "weight and bias must be"),
    (lambda: layer_norm(_cpu(2, 8), _cpu(8, dtype=torch.float16)), "weight and bias must both"),
    (lambda: layer_norm(_cpu(2, 8), residual=_cpu(2, 7)), "residual must be"),
    (lambda: layer_norm(_cpu(2, 8), eps=-1.0), "eps"),
    (lambda: layer_norm(_cpu(2, 8, dtype=torch.float64)), "unsupported dtype"),
    (lambda: layer_norm(_cpu(2, 8)), "CUDA"),
    (lambda: attention(_cpu(1, 2, 3), _cpu(1, 2, 1, 8), _cpu(1, 2, 1, 8)), "query must be"),
    (lambda: attention(_cpu(1, 2, 3, 8), _cpu(1, 2, 2, 8), _cpu(1, 2, 2, 8)), "multiple of Hkv"),
    (lambda: attention(_cpu(1, 2, 2, 8), _cpu(1, 2, 2, 8), _cpu(1, 3, 2, 8)), "value must be"),
    (lambda: attention(_cpu(1, 2, 2, 300), _cpu(1, 2, 2, 300), _cpu(1, 2, 2, 300)), "outside"),
    (lambda: attention(*[_cpu(1, 2, 2, 8)] * 3, softcap=-1.0), "softcap"),
    (lambda: attention(*[_cpu(1, 2, 2, 8)] * 3, prefix_lengths=_cpu(1, dtype=torch.int32)), "needs causal"),
    (lambda: attention(*[_cpu(1, 2, 2, 8)] * 3, key_documents=_cpu(1, 2, dtype=torch.int32)), "come together"),
    (lambda: attention(*[_cpu(1, 2, 2, 8)] * 3, shared_document=0), "needs documents"),
    (lambda: attention(*[_cpu(1, 2, 2, 8)] * 3, key_lengths=_cpu(1)), "key_lengths must be"),
    (lambda: attention(*[_cpu(1, 2, 2, 8)] * 3, distance_slopes=_cpu(2).requires_grad_()), "constants"),
    (lambda: attention(*[_cpu(1, 2, 2, 8)] * 3), "CUDA"),
])
def test_python_refusals(call, words):
    with pytest.raises(ValueError, match=words):
        call()


@host_only
def test_c_abi_refuses_before_any_device_work():
    lib, vp = _lib.load(), ctypes.c_void_p
    strides = (ctypes.c_int64 * 3)(8, 8, 8)

    def rot(D=8, axes=(4,), heads=1, dtype=0, q=16, base=10000.0, ptype=0):
        return lib.msda_rotary(vp(q), None, vp(16), vp(16), None, 1, 1, heads, 0, D, strides, None, 0, ptype,
                               len(axes), (ctypes.c_int32 * len(axes))(*axes), base, 0, 0, 0, dtype, None)

    assert rot(dtype=9) == _lib.MSDA_ERR_UNSUPPORTED
    assert rot(D=1024) == _lib.MSDA_ERR_UNSUPPORTED
    assert rot(axes=(3,)) == _lib.MSDA_ERR_INVALID_ARGUMENT
    assert rot(axes=(8, 2)) == _lib.MSDA_ERR_INVALID_ARGUMENT
    assert rot(heads=0) == _lib.MSDA_ERR_INVALID_ARGUMENT
    assert rot(base=-1.0) == _lib.MSDA_ERR_INVALID_ARGUMENT
    assert rot(ptype=3) == _lib.MSDA_ERR_UNSUPPORTED
    assert rot(q=0) == _lib.MSDA_ERR_INVALID_ARGUMENT
    assert rot(q=18) == _lib.MSDA_ERR_INVALID_ARGUMENT

    def norm(rows=2, width=8, dtype=0, pdtype=0, x=16, eps=1e-5):
        return lib.msda_layer_norm_forward(vp(x), None, None, None, vp(16), None, None, None, rows, width, width, 0,
                                           eps, dtype, pdtype, None)

    assert norm(dtype=5) == _lib.MSDA_ERR_UNSUPPORTED
    assert norm(dtype=1, pdtype=2) == _lib.MSDA_ERR_UNSUPPORTED
    assert norm(width=0) == _lib.MSDA_ERR_UNSUPPORTED
    assert norm(width=_lib.MSDA_LAYER_NORM_MAX_WIDTH + 1) == _lib.MSDA_ERR_UNSUPPORTED
    assert norm(x=0) == _lib.MSDA_ERR_INVALID_ARGUMENT
    assert norm(x=18) == _lib.MSDA_ERR_INVALID_ARGUMENT
    assert norm(eps=-1.0) == _lib.MSDA_ERR_INVALID_ARGUMENT
    assert norm(rows=0, x=0) == _lib.MSDA_OK
    assert lib.msda_layer_norm_backward_workspace_size(5, 8) == 5 * 8 * 2 * 4
    rc = lib.msda_layer_norm_backward(vp(16), None, vp(16), vp(16), vp(16), vp(16), None, vp(16), vp(16), None, None, 0,
                                      4, 8, 8, 0, 8, 0, 0, None)
    assert rc == _lib.MSDA_ERR_INVALID_ARGUMENT and b"workspace" in lib.msda_last_error()

    def att(backward=0, **over):
        a = _lib.AttentionArgs()
        fields = dict(query=16, key=16, value=16, out=16, batch=1, num_queries=100, num_keys=100, num_heads=2,
                      num_key_heads=1, head_dim=8, scale=1.0, shared_document=-1)
        for k, v in (fields | over).items():
            setattr(a, k, v)
        fn = lib.msda_attention_backward if backward else lib.msda_attention_forward
        return fn(ctypes.byref(a), None)

    assert att(dtype=4) == _lib.MSDA_ERR_UNSUPPORTED
    assert att(head_dim=257) == _lib.MSDA_ERR_UNSUPPORTED
    assert att(num_heads=3, num_key_heads=2) == _lib.MSDA_ERR_INVALID_ARGUMENT
    assert att(num_queries=-1) == _lib.MSDA_ERR_INVALID_ARGUMENT
    assert att(query=0) == _lib.MSDA_ERR_INVALID_ARGUMENT
    assert att(key=18) == _lib.MSDA_ERR_INVALID_ARGUMENT
    assert att(softcap=-1.0) == _lib.MSDA_ERR_INVALID_ARGUMENT
    assert att(scale=float("inf")) == _lib.MSDA_ERR_INVALID_ARGUMENT
    assert att(prefix_lengths=16) == _lib.MSDA_ERR_INVALID_ARGUMENT
    assert att(key_documents=16) == _lib.MSDA_ERR_INVALID_ARGUMENT
    assert att(key_documents=16, query_documents=16) == _lib.MSDA_ERR_INVALID_ARGUMENT  # no workspace
    assert b"workspace" in lib.msda_last_error()
    assert att(backward=1) == _lib.MSDA_ERR_INVALID_ARGUMENT  # no lse, no gradients
    assert att(batch=0, query=0) == _lib.MSDA_OK
    assert lib.msda_attention_forward(None, None) == _lib.MSDA_ERR_INVALID_ARGUMENT


# ---------------------------------------------------------------------------
# Rotary positions
# ---------------------------------------------------------------------------
ROTARY = [
    dict(B=2, S=5, H=4, Hkv=2, D=64, axes=[16, 24, 24], ladder="shared", pairing="half"),
    dict(B=1, S=1, H=1, Hkv=1, D=2, axes=[2], ladder="axis", pairing="half"),
    dict(B=2, S=301, H=8, Hkv=8, D=32, axes=[16, 16], ladder="axis", pairing="interleaved"),
    dict(B=3, S=17, H=3, Hkv=1, D=38, axes=[6, 10, 2], ladder="axis", pairing="half"),       # passes through, odd vectors
    dict(B=3, S=17, H=3, Hkv=1, D=37, axes=[6, 10], ladder="shared", pairing="interleaved"),  # odd head
    dict(B=1, S=3000, H=2, Hkv=0, D=128, axes=[0, 64, 64], ladder="axis", pairing="half"),
    dict(B=1, S=9, H=40, Hkv=8, D=512, axes=[512], ladder="axis", pairing="half"),
]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("c", ROTARY, ids=lambda c: f"{c['D']}{c['ladder']}{c['pairing']}")
@pytest.mark.parametrize("whole", [False, True])
def test_rotary(c, dtype, whole, cuda_lib):
    B, S, H, Hkv, D, axes = (c[k] for k in ("B", "S", "H", "Hkv", "D", "axes"))
    how = dict(ladder=c["ladder"], pairing=c["pairing"])
    q = randn(B, S, H, D, dtype=dtype).requires_grad_()
    k = randn(B, S, Hkv, D, dtype=dtype, seed=1).requires_grad_() if Hkv else None
    pos = randn(B, S, len(axes), seed=2) * (70000 if whole else 40)
    pos = pos.long() if whole else pos
    got = rotary(q, pos, key=k, axis_dims=axes, **how)
    got = got if Hkv else (got,)
    for x, y in zip((q, k), got):
        close(y.detach(), ref.rotary(x.detach(), pos, axes, **how), dtype, *(ROUNDED if dtype != torch.float32 else (8, 64)), what="out")
        g = randn(*y.shape, dtype=dtype, seed=3)
        gx, = torch.autograd.grad(y, x, g, retain_graph=True)
        close(gx, ref.rotary(g, pos, axes, **how, inverse=True), dtype,
              *(ROUNDED if dtype != torch.float32 else (8, 64)), what="grad")


@gpu
def test_rotary_strides_and_shared_positions(cuda_lib):
    """Views of a fused projection, heads before tokens, channels not last, (S, A) positions, int32."""
    packed = randn(2, 7, 3, 4, 16, dtype=torch.bfloat16)
    q, k = packed[:, :, 0], packed[:, :, 1]
    pos = torch.arange(14, device=DEV, dtype=torch.int32).view(7, 2)
    for x, y in zip((q, k), rotary(q, pos, key=k, axis_dims=[8, 4])):
        close(y, ref.rotary(x, pos, [8, 4]), torch.bfloat16, *ROUNDED)
    odd = randn(2, 4, 7, 17).transpose(1, 2)[..., 1:]  # rows that start off 16 bytes
    close(rotary(odd, pos, axis_dims=[8, 8]), ref.rotary(odd, pos, [8, 8]), torch.float32, 8, 64)
    last = randn(2, 7, 16, 4).transpose(2, 3)
    close(rotary(last, pos, axis_dims=[8, 8]), ref.rotary(last, pos, [8, 8]), torch.float32, 8, 64)
    assert rotary(randn(0, 7, 4, 16), pos, axis_dims=[8, 8]).shape == (0, 7, 4, 16)


@gpu
def test_rotary_only_one_gradient(cuda_lib):
    q, k = randn(1, 3, 2, 8).requires_grad_(), randn(1, 3, 1, 8).requires_grad_()
    pos = torch.arange(3, device=DEV).view(3, 1)
    for i, x in enumerate((q, k)):
        y = rotary(q, pos, key=k, axis_dims=[8])[i]
        gx, other = torch.autograd.grad(y.sum(), (x, (k, q)[i]), allow_unused=True)
        assert other is None or not other.any()
        close(gx, ref.rotary(torch.ones_like(x), pos, [8], inverse=True), torch.float32, 8, 64)


# ---------------------------------------------------------------------------
# Layer norm
# ---------------------------------------------------------------------------
def _norm_u(dtype, rows=0):
    # 16 bits: rounded once. 32 bits: sums of C or `rows` terms.
    return ROUNDED if dtype != torch.float32 else (64, 1024)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (2, 5, 256), (1201, 256), (33, 1000), (5, 1025), (9, 1001),
                                   (700, 2048), (4, 5001), (3, 8192), (2, 8193), (2, 20000)], ids=str)
@pytest.mark.parametrize("residual, affine, fp32_params", [(True, True, False), (False, True, True), (True, False, False)])
def test_layer_norm(shape, dtype, residual, affine, fp32_params, cuda_lib):
    C = shape[-1]
    x = (randn(*shape, dtype=dtype) * 2 + 1).detach().requires_grad_()
    r = randn(*shape, dtype=dtype, seed=1).requires_grad_() if residual else None
    pd = torch.float32 if fp32_params else dtype
    w = (1 + 0.3 * randn(C, seed=2)).to(pd).requires_grad_() if affine else None
    b = randn(C, seed=3).to(pd).requires_grad_() if affine else None
    g = randn(*shape, dtype=dtype, seed=4)
    y = layer_norm(x, w, b, residual=r, eps=1e-5)
    want, z, rstd = ref.layer_norm(x.detach(), w, b, r, 1e-5)
    close(y.detach(), want.detach(), dtype, *_norm_u(dtype), floor=0.1, what="y")
    leaves = [t for t in (x, r, w, b) if t is not None]
    got = dict(zip([n for n, t in zip("xrwb", (x, r, w, b)) if t is not None], torch.autograd.grad(y, leaves, g)))
    dx, dw, db = (t.detach() for t in ref.layer_norm_grad(z, rstd, w, g))
    floor = 1e-3 * float(rstd.max())  # of dx, which cancels to nothing in the narrowest rows
    close(got["x"].view_as(dx), dx, dtype, *_norm_u(dtype), floor=floor, what="dx")
    if residual:
        assert torch.equal(got["r"], got["x"])
    if affine:
        close(got["w"], dw, pd, *_norm_u(pd), floor=0.1, what="dw")
        close(got["b"], db, pd, *_norm_u(pd), floor=0.1, what="db")


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C", [64, 8200])
def test_layer_norm_sum_output(dtype, C, cuda_lib):
    x, r = randn(37, C, dtype=dtype).requires_grad_(), randn(37, C, dtype=dtype, seed=1).requires_grad_()
    w, b = randn(C, dtype=dtype, seed=2), randn(C, dtype=dtype, seed=3)
    gy, gs = randn(37, C, dtype=dtype, seed=4), randn(37, C, dtype=dtype, seed=5)
    y, s = layer_norm(x, w, b, residual=r, return_sum=True)
    close(s.detach(), (x.double() + r.double()).detach(), dtype, *ROUNDED)
    _, z, rstd = ref.layer_norm(x.detach(), w, b, r.detach(), 1e-5)
    got, = torch.autograd.grad((y, s), x, (gy, gs), retain_graph=True)
    close(got, ref.layer_norm_grad(z, rstd, w, gy, gs)[0], dtype, *_norm_u(dtype))
    got, = torch.autograd.grad(s, x, gs)
    close(got, gs, dtype, *_norm_u(dtype))


@gpu
def test_layer_norm_strides_constant_rows_and_repeats(cuda_lib):
    wide = randn(50, 3, 70, dtype=torch.bfloat16)
    x = wide[:, 1, 3:67]  # strided rows off 16 bytes
    close(layer_norm(x), ref.layer_norm(x, None, None, None, 1e-5)[0], torch.bfloat16, *ROUNDED)
    t = randn(64, 30).t()  # channels not contiguous
    close(layer_norm(t), ref.layer_norm(t, None, None, None, 1e-5)[0], torch.float32, 64, 1024)
    flat = torch.full((4, 256), 3.0, device=DEV)
    assert torch.equal(layer_norm(flat), torch.zeros_like(flat))
    big = randn(8, 512) + 1000.0  # the variance about the mean, not by squares
    close(layer_norm(big), ref.layer_norm(big, None, None, None, 1e-5)[0], torch.float32, 64, 1024)
    assert layer_norm(randn(0, 16)).shape == (0, 16)
    x = randn(5000, 256, dtype=torch.float16).requires_grad_()
    w = randn(256, dtype=torch.float16).requires_grad_()
    g = randn(5000, 256, dtype=torch.float16, seed=9)
    first = torch.autograd.grad(layer_norm(x, w), (x, w), g)
    for _ in range(3):
        again = torch.autograd.grad(layer_norm(x, w), (x, w), g)
        assert all(torch.equal(a, b) for a, b in zip(first, again))
    e = randn(0, 16).requires_grad_()
    w = randn(16).requires_grad_()
    assert not torch.autograd.grad(layer_norm(e, w).sum(), w)[0].any()


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------
def _ids(B, S, n, seed, pad=0):
    g = torch.Generator().manual_seed(seed)
    cuts = (torch.rand(B, n - 1, generator=g) * S).long().sort(-1).values
    ids = (torch.arange(S)[None, :, None] >= cuts[:, None]).sum(-1)
    if pad:
        ids[::2, S - pad:] = -1
    return ids.int().to(DEV)


def _masks(kind, B, Sq, Sk):
    ints = lambda *v: torch.tensor([v[i % len(v)] for i in range(B)], dtype=torch.int32, device=DEV)  # noqa: E731
    if kind == "none":
        return {}
    if kind == "causal":
        return dict(causal=True)
    if kind == "prefix":
        return dict(causal=True, prefix_lengths=ints(Sk // 3, 0, Sk + 5))
    if kind == "lengths":
        return dict(key_lengths=ints(Sk - 1, 0, Sk + 9, Sk // 2))
    if kind == "causal_lengths":  # some queries stand before the first key: empty rows
        return dict(causal=True, key_lengths=ints(max(0, Sk - 3), Sq // 2, Sk))
    ids = _ids(B, Sk, 5, 3, pad=Sk // 7)
    if kind == "documents":
        return dict(query_documents=ids, key_documents=ids)
    if kind == "packed":
        return dict(query_documents=ids, key_documents=ids, causal=True)
    if kind == "shared":
        return dict(query_documents=ids, key_documents=ids, shared_document=2)
    if kind == "scattered":  # ids in no order, a document without keys
        g = torch.Generator().manual_seed(5)
        q = torch.randint(-1, 4, (B, Sq), generator=g, dtype=torch.int32).to(DEV)
        k = torch.randint(-1, 3, (B, Sk), generator=g, dtype=torch.int32).to(DEV)
        return dict(query_documents=q, key_documents=k, key_lengths=ints(Sk, Sk - 2))
    raise AssertionError(kind)


MASKS = ["none", "causal", "prefix", "lengths", "causal_lengths", "documents", "packed", "shared", "scattered"]


def _check(q, k, v, dtype, train=True, size=64, **how):
    """`size`: of the scores, where it is above 64."""
    q, k, v = (t.detach().requires_grad_(train) for t in (q, k, v))
    g = randn(*q.shape, dtype=dtype, seed=11) if train else None
    with torch.no_grad():
        want, lse, grads = ref.attention(q, k, v, g, **how)
    out, got_lse = attention(q, k, v, return_lse=True, **how)
    tol = (3, 12) if dtype != torch.float32 else (size, 16 * size)
    close(out.detach(), want, dtype, *tol, floor=0.02, what="out")
    assert not out.detach()[want == 0].any()  # rows that see no key
    close(got_lse, lse, torch.float32, size, 16 * size, floor=1.0, what="lse")
    if train:
        got = torch.autograd.grad(out, (q, k, v), g)
        for n, a, b in zip(("dq", "dk", "dv"), got, grads):
            close(a, b, dtype, *tol, floor=0.02, what=n)
        return out.detach(), got
    return out.detach(), None


def _check_by_terms(q, k, v, dtype, **how):
    """As _check with gradients, in 16 bits with each element held to its terms."""
    if dtype == torch.float32:
        return _check(q, k, v, dtype, **how)
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    g = randn(*q.shape, dtype=dtype, seed=11)
    with torch.no_grad():
        want, _, grads, terms = ref.attention(q, k, v, g, terms=2.0**-14 if dtype == torch.float16 else 0.0, **how)
    out = attention(q, k, v, **how)
    got = (out, *torch.autograd.grad(out, (q, k, v), g))
    u = ref.U[dtype]
    for n, a, b, size in zip(("out", "dq", "dk", "dv"), got, (want, *grads), terms):
        off = (a.detach().double() - b).abs()
        assert off.norm() <= 3 * u * b.norm(), n
        assert (off <= 1.25 * u * (size + b.abs()) + 1e-5 * b.square().mean().sqrt()).all(), n


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", MASKS)
@pytest.mark.parametrize("D, Hkv", [(32, 4), (64, 2)])
def test_attention_masks(kind, D, Hkv, dtype, cuda_lib):
    B, S = 3, 301
    q, k, v = randn(B, S, 4, D, dtype=dtype), randn(B, S, Hkv, D, dtype=dtype, seed=1), randn(B, S, Hkv, D, dtype=dtype, seed=2)
    _check(q, k, v, dtype, **_masks(kind, B, S, S))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("softcap, slopes", [(20.0, False), (1.5, False), (0.0, True), (4.0, True)])
@pytest.mark.parametrize("kind", ["none", "packed", "causal_lengths"])
def test_attention_scores(softcap, slopes, kind, dtype, cuda_lib):
    B, S, H, D = 2, 200, 4, 64
    q, k, v = (randn(B, S, h, D, dtype=dtype, seed=i) for i, h in enumerate((H, 2, 2)))
    s = torch.tensor([0.5, 0.1, 0.02, -0.01], device=DEV) if slopes else None
    _check(q * 2, k, v, dtype, softcap=softcap, distance_slopes=s, **_masks(kind, B, S, S))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Sq, Sk", [(1, 1), (1, 7), (2, 3), (65, 64), (127, 129), (128, 128), (129, 700), (300, 1), (513, 77), (256, 384)])
@pytest.mark.parametrize("D", [8, 128])
def test_attention_sizes(Sq, Sk, D, dtype, cuda_lib):
    q, k, v = randn(2, Sq, 2, D, dtype=dtype), randn(2, Sk, 2, D, dtype=dtype, seed=1), randn(2, Sk, 2, D, dtype=dtype, seed=2)
    for kind in ("none", "causal", "lengths"):
        _check(q, k, v, dtype, **_masks(kind, 2, Sq, Sk))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B, S, H, Hkv, D", [(1, 70, 24, 2, 32), (1, 260, 8, 1, 128), (30, 130, 12, 4, 32), (20, 130, 24, 4, 40),
                                             (70, 130, 8, 4, 24)])
def test_attention_shared_heads(B, S, H, Hkv, D, dtype, cuda_lib):
    """Key gradients whose query heads share CTAs wholly, in parts or not at all."""
    q, k, v = randn(B, S, H, D, dtype=dtype), randn(B, S, Hkv, D, dtype=dtype, seed=1), randn(B, S, Hkv, D, dtype=dtype, seed=2)
    for kind in ("causal", "shared"):
        _check_by_terms(q, k, v, dtype, **_masks(kind, B, S, S))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B, Sq, Sk, H, Hkv, D", [(1, 100, 2000, 4, 4, 64), (1, 61, 3000, 8, 2, 128), (2, 250, 900, 2, 1, 32),
                                                  (9, 130, 600, 8, 8, 40)])
def test_attention_some_queries_over_more_keys(B, Sq, Sk, H, Hkv, D, dtype, cuda_lib):
    q, k, v = randn(B, Sq, H, D, dtype=dtype), randn(B, Sk, Hkv, D, dtype=dtype, seed=1), randn(B, Sk, Hkv, D, dtype=dtype, seed=2)
    s = 0.01 * torch.arange(H, device=DEV, dtype=torch.float32)
    for kind in ("none", "prefix", "causal_lengths", "scattered"):
        _check_by_terms(q, k, v, dtype, distance_slopes=s, **_masks(kind, B, Sq, Sk))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [1, 3, 20, 40, 72, 96, 104, 136, 250])
def test_attention_head_sizes(D, dtype, cuda_lib):
    q, k, v = (randn(2, 150, h, D, dtype=dtype, seed=i) for i, h in enumerate((6, 3, 3)))
    _check(q, k, v, dtype, causal=True)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Sq, Sk, H, Hkv, D", [(1, 1, 4, 4, 32), (1, 900, 8, 8, 32), (1, 1000, 16, 2, 64), (1, 3001, 32, 2, 128),
                                               (2, 515, 24, 1, 104), (4, 2000, 8, 8, 64), (1, 5000, 8, 1, 128), (3, 333, 5, 5, 40),
                                               (1, 777, 2, 1, 33), (1, 600, 4, 2, 200)])
def test_attention_tokens(Sq, Sk, H, Hkv, D, dtype, cuda_lib):
    """A few queries over a cache whose tail holds whatever memory held."""
    B = 3
    q, k, v = randn(B, Sq, H, D, dtype=dtype), randn(B, Sk, Hkv, D, dtype=dtype, seed=1), randn(B, Sk, Hkv, D, dtype=dtype, seed=2)
    lengths = torch.tensor([Sk, max(1, Sk // 2), 0], dtype=torch.int32, device=DEV)
    past = torch.arange(Sk, device=DEV)[None] >= lengths[:, None]
    k[past], v[past] = float("nan"), float("inf")
    s = 0.01 * torch.arange(H, device=DEV, dtype=torch.float32)
    for how in (dict(), dict(causal=True), dict(causal=True, softcap=10.0, distance_slopes=s),
                dict(query_documents=_ids(B, Sq, 2, 1), key_documents=_ids(B, Sk, 3, 2, pad=Sk // 9), shared_document=1)):
        _check(q, k, v, dtype, train=False, key_lengths=lengths, **how)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [40, 64, 128])
def test_attention_ignores_what_padding_holds(D, dtype, cuda_lib):
    """Not-a-numbers past the lengths, in padded keys and in padded queries' rows of the gradient."""
    B, S = 2, 300
    q, k, v = (randn(B, S, 2, D, dtype=dtype, seed=i) for i in range(3))
    ids = _ids(B, S, 3, 4, pad=45)
    ids[:, 130:140] = -1
    lengths = torch.tensor([S, 211], dtype=torch.int32, device=DEV)
    pad = (ids < 0) | (torch.arange(S, device=DEV)[None] >= lengths[:, None])
    g = randn(B, S, 2, D, dtype=dtype, seed=5)
    how = dict(query_documents=ids, key_documents=ids, key_lengths=lengths)
    want, _, grads = ref.attention(q, k, v, g.masked_fill((ids < 0)[:, :, None, None], 0), **how)
    k[pad], v[pad], q[ids < 0], g[ids < 0] = float("nan"), float("inf"), float("nan"), float("inf")
    q, k, v = (t.requires_grad_() for t in (q, k, v))
    out = attention(q, k, v, **how)
    tol = (3, 12) if dtype != torch.float32 else (64, 1024)
    close(out.detach(), want, dtype, *tol, floor=0.02)
    for a, b in zip(torch.autograd.grad(out, (q, k, v), g), grads):
        close(a, b, dtype, *tol, floor=0.02)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_strides(dtype, cuda_lib):
    """One fused projection's views, heads before tokens, rows off 16 bytes, broadcast keys and gradients."""
    B, S, H, D = 2, 190, 3, 32
    packed = randn(B, S, 3, H, D, dtype=dtype)
    q, k, v = packed.unbind(2)
    want, _, _ = ref.attention(q, k, v)
    tol = (3, 12) if dtype != torch.float32 else (64, 1024)
    close(attention(q, k, v), want, dtype, *tol)
    qt, kt, vt = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v))
    close(attention(qt, kt, vt), want, dtype, *tol)
    odd = randn(B, S, H, D + 5, dtype=dtype)[..., 3:3 + D]
    _check(odd, kt, v, dtype)
    one = randn(1, S, 1, D, dtype=dtype, seed=4).expand(B, S, H, D)
    _check(q, one, v, dtype)
    a, b, c = (t.detach().clone().requires_grad_() for t in (q, k, v))
    gs = torch.autograd.grad(attention(a, b, c).sum(), (a, b, c))
    _, _, grads = ref.attention(q, k, v, torch.ones_like(q))
    for x, y in zip(gs, grads):
        close(x, y, dtype, *tol, floor=0.02)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_large_scores_and_empty(dtype, cuda_lib):
    q, k, v = (randn(1, 260, 2, 64, dtype=dtype, seed=i) for i in range(3))
    # Scores of several hundred, growing along the keys: the running maximum moves.
    ramp = torch.linspace(-6, 6, 260, device=DEV).view(1, 260, 1, 1)
    _check(q * 0 + 4, (ramp * 2 + 0 * k).to(dtype), v, dtype, train=False, size=384)
    _check(q * 0 + 4, (-ramp * 2 + 0 * k).to(dtype), v, dtype, train=False, size=384)
    _check(q, k, v, dtype, scale=-1.0, train=False)
    e = attention(q[:, :0], k, v)
    assert e.shape == (1, 0, 2, 64)
    assert not attention(q, k[:, :0], v[:, :0]).any()
    out, lse = attention(q[:, :1], k[:, :0], v[:, :0], return_lse=True)
    assert not out.any() and (lse == float("-inf")).all()
    leaves = [t.detach().clone().requires_grad_() for t in (q, k[:, :0], v[:, :0])]
    assert not torch.autograd.grad(attention(*leaves).sum(), leaves[0])[0].any()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_repeats_bitwise_and_on_other_streams(dtype, cuda_lib):
    B, S = 2, 400
    q, k, v = (randn(B, S, h, 64, dtype=dtype, seed=i).requires_grad_() for i, h in enumerate((8, 2, 2)))
    g = randn(B, S, 8, 64, dtype=dtype, seed=7)
    how = dict(causal=True, softcap=9.0, query_documents=_ids(B, S, 3, 1), key_documents=_ids(B, S, 3, 1))

    def step():
        out = attention(q, k, v, **how)
        return (out.detach(), *torch.autograd.grad(out, (q, k, v), g))

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [step() for _ in range(3)]
    side.synchronize()
    for a in again:
        assert all(torch.equal(x, y) for x, y in zip(first, a))


@gpu
def test_attention_backward_as_a_threads_first_cuda_call(cuda_lib):
    """A fresh process whose backward takes its memory from the allocator's cache:
    autograd's thread has made no CUDA call before it asks for tensor maps."""
    code = """
import torch
from msda_triton_b200 import attention
q = torch.randn(1, 300, 2, 64, device="cuda", dtype=torch.bfloat16).requires_grad_()
cached = [torch.empty(n, device="cuda", dtype=torch.bfloat16) for n in (1 << 16, 1 << 20, 1 << 24) for _ in range(4)]
g = torch.randn_like(q)
del cached
out = attention(q, q, q, causal=True)
grad, = torch.autograd.grad(out, q, g)
assert bool(torch.isfinite(grad).all()) and bool(grad.any())
"""
    path = os.pathsep.join([str(Path(_lib.__file__).resolve().parent.parent), os.environ.get("PYTHONPATH", "")])
    done = subprocess.run([sys.executable, "-c", code], env={**os.environ, "PYTHONPATH": path}, capture_output=True, text=True,
                          timeout=300)
    assert done.returncode == 0, done.stderr


@gpu
def test_attention_gradient_against_differences(cuda_lib):
    """Central differences of a weighted sum of the outputs, in 32 bits: step
    1e-2 leaves about 1e-4 of third-order and 1e-5 of rounding error."""
    q, k, v = (randn(1, 40, h, 16, seed=i).requires_grad_() for i, h in enumerate((2, 1, 1)))
    g = randn(1, 40, 2, 16, seed=5)
    how = dict(causal=True, softcap=3.0, distance_slopes=torch.tensor([0.1, 0.05], device=DEV))
    grads = torch.autograd.grad(attention(q, k, v, **how), (q, k, v), g)
    for i, (x, gx) in enumerate(zip((q, k, v), grads)):
        d = randn(*x.shape, seed=20 + i)
        d = d / d.norm()
        ends = []
        for sign in (1, -1):
            args = [t.detach() + (sign * 1e-2 * d if j == i else 0) for j, t in enumerate((q, k, v))]
            ends.append((attention(*args, **how).double() * g.double()).sum())
        assert abs(float((ends[0] - ends[1]) / 2e-2) - float((gx.double() * d.double()).sum())) < 2e-3
