"""The layer operators at their edges: what padding and empty rows hold, hand-overs
between the tensor-core kernels' roles, caps, offsets and sizes at their limits."""

from __future__ import annotations

import ctypes

import pytest
import torch
from torch.autograd import forward_ad

import layer_reference as ref
from hostonly import host_only
from layer_reference import close
from msda_triton_b200 import _lib, attention, layer_norm, rotary
from msda_triton_b200.attention import _pack
from test_layer_ops import DEV, DTYPES, HALF, _ids, randn

gpu = pytest.mark.gpu


def tolerance(dtype):
    return (3, 12) if dtype != torch.float32 else (64, 1024)


def waits_given_up():
    n = ctypes.c_int32(-1)
    _lib.check("msda_attention_gave_up", _lib.load().msda_attention_gave_up(ctypes.byref(n)))
    return n.value


@gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("D", [32, 64, 128])
def test_padding_in_every_tile(D, dtype, cuda_lib):
    """Scattered padding: each tile of keys, and of queries in the key gradient, is
    cleared before its products, in calls of one tile to many."""
    before = waits_given_up()
    for B, S in ((1, 100), (3, 250), (2, 1300), (40, 700)):
        q, k, v, g = (randn(B, S, 2, D, dtype=dtype, seed=i) for i in range(4))
        ids = (torch.arange(S, device=DEV) // 400).int().expand(B, S).clone()
        pad = torch.arange(S, device=DEV)[None] * 7 % (13 + torch.arange(B, device=DEV)[:, None]) == 0
        ids[pad] = -1
        how = dict(query_documents=ids, key_documents=ids)
        want, _, grads = ref.attention(q, k, v, g.masked_fill(pad[:, :, None, None], 0), **how)
        k[pad], v[pad], q[pad], g[pad] = float("nan"), float("inf"), float("nan"), float("inf")
        q, k, v = (t.requires_grad_() for t in (q, k, v))
        for _ in range(4):
            out = attention(q, k, v, **how)
            close(out.detach(), want, dtype, *tolerance(dtype), floor=0.02, what="out")
            for n, a, b in zip(("dq", "dk", "dv"), torch.autograd.grad(out, (q, k, v), g), grads):
                close(a, b, dtype, *tolerance(dtype), floor=0.02, what=n)
    assert waits_given_up() == before


@gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("D", [32, 64, 128])
def test_query_gradient_of_many_steps(D, dtype, cuda_lib):
    """Odd and even numbers of steps, of whole tiles and halves; the same each time."""
    before = waits_given_up()
    for Sk in (60, 128, 190, 300, 449, 2050):
        q, k, v, g = (randn(2, 130 if i in (0, 3) else Sk, 2, D, dtype=dtype, seed=i) for i in range(4))
        _, _, grads = ref.attention(q, k, v, g)
        q, k, v = (t.requires_grad_() for t in (q, k, v))
        out = attention(q, k, v)
        first = None
        for _ in range(20):
            dq, = torch.autograd.grad(out, q, g, retain_graph=True)
            first = dq if first is None else first
            assert torch.equal(dq, first)
        close(first, grads[0], dtype, *tolerance(dtype), floor=0.02, what="dq")
    assert waits_given_up() == before


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [40, 64, 128])
@pytest.mark.parametrize("softcap, documents", [(20.0, False), (20.0, True), (1.0, True), (0.0, False)])
def test_capped_scores_ignore_what_padding_holds(softcap, documents, D, dtype, cuda_lib):
    """Not-a-numbers past the lengths, in padded keys and in padded queries' rows."""
    B, S = 2, 300
    q, k, v, g = (randn(B, S, 2, D, dtype=dtype, seed=i) for i in range(4))
    lengths = torch.tensor([S - 1, 211], dtype=torch.int32, device=DEV)
    how = dict(key_lengths=lengths, softcap=softcap)
    pad = torch.arange(S, device=DEV)[None] >= lengths[:, None]
    idle = torch.zeros_like(pad)
    if documents:
        ids = _ids(B, S, 3, 4, pad=45)
        ids[:, 130:140] = -1
        how.update(query_documents=ids, key_documents=ids)
        idle = ids < 0
        pad = pad | idle
    want, _, grads = ref.attention(q, k, v, g.masked_fill(idle[:, :, None, None], 0), **how)
    k[pad], v[pad], q[idle], g[idle] = float("nan"), float("inf"), float("nan"), float("inf")
    q, k, v = (t.requires_grad_() for t in (q, k, v))
    out = attention(q, k, v, **how)
    close(out.detach(), want, dtype, *tolerance(dtype), floor=0.02, what="out")
    for n, a, b in zip(("dq", "dk", "dv"), torch.autograd.grad(out, (q, k, v), g), grads):
        close(a, b, dtype, *tolerance(dtype), floor=0.02, what=n)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [20, 64, 128])
@pytest.mark.parametrize("kind", ["before the first key", "document without keys", "both"])
def test_queries_that_see_no_key_have_no_gradient(kind, D, dtype, cuda_lib):
    """Whatever their rows of the query and of the output's gradient hold."""
    B, S = 2, 300
    q, k, v, g = (randn(B, S, 4 if i in (0, 3) else 2, D, dtype=dtype, seed=i) for i in range(4))
    how, idle = {}, torch.zeros(B, S, dtype=torch.bool, device=DEV)
    if kind != "document without keys":
        lengths = torch.tensor([S, 120], dtype=torch.int32, device=DEV)
        how.update(causal=True, key_lengths=lengths)
        idle |= torch.arange(S, device=DEV)[None] < S - lengths[:, None]
    if kind != "before the first key":
        ids = _ids(B, S, 3, 4)
        theirs = ids.clone()
        theirs[:, 5::7] = 9
        how.update(query_documents=theirs, key_documents=ids)
        seen, _ = ref.visible(B, S, S, DEV, **how)
        idle = ~seen.any(-1)
    want, _, grads = ref.attention(q, k, v, g.masked_fill(idle[:, :, None, None], 0), **how)
    q[idle], g[idle] = float("nan"), float("inf")
    q, k, v = (t.requires_grad_() for t in (q, k, v))
    out = attention(q, k, v, **how)
    close(out.detach(), want, dtype, *tolerance(dtype), floor=0.02, what="out")
    for n, a, b in zip(("dq", "dk", "dv"), torch.autograd.grad(out, (q, k, v), g), grads):
        close(a, b, dtype, *tolerance(dtype), floor=0.02, what=n)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale, softcap", [(1 / 128, 500.0), (0.01, 1000.0), (0.125, 5000.0), (64.0, 30.0), (1e-4, 0.01)])
@pytest.mark.parametrize("Sq, H", [(1, 2), (300, 2), (300, 16)])
@pytest.mark.parametrize("share", [0.15, 0.6, 0.74, 1.5])
def test_scores_at_a_share_of_the_cap(share, Sq, H, scale, softcap, dtype, cuda_lib):
    """Scores of about `share` of the cap, before it, with wide and narrow caps. A score
    may be off by 16 u (32 bits) of itself, which its probability is off by too."""
    S, D, u = 300, 64, ref.U[torch.float32]
    size = (share * softcap / scale / D) ** 0.5
    g = torch.Generator(DEV).manual_seed(1)
    q = torch.full((1, Sq, H, D), size, device=DEV).to(dtype)
    k = (size * (1 - 0.02 * torch.rand(1, S, H, D, device=DEV, generator=g))).to(dtype)
    v, grad = randn(1, S, H, D, dtype=dtype, seed=2), randn(1, Sq, H, D, dtype=dtype, seed=3)
    how = dict(scale=scale, softcap=softcap)
    want, want_lse, grads = ref.attention(q, k, v, grad, **how)
    v.requires_grad_()
    out, lse = attention(q, k, v, return_lse=True, **how)
    top = float(want_lse.abs().max())
    assert float((lse.double() - want_lse).abs().max()) <= 16 * u * softcap + 4 * u * top
    more = 16 * u * softcap / ref.U[dtype]
    norm, element = tolerance(dtype)
    close(out.detach(), want, dtype, norm + more, element + 4 * more, floor=0.02, what="out")
    close(torch.autograd.grad(out, v, grad)[0], grads[2], dtype, norm + more, element + 4 * more, floor=0.02, what="dv")


def _offset_case(C, residual):
    grid = lambda t: (t * 4096).round() / 4096  # noqa: E731  (sums without a rounding)
    x = grid(randn(37, C) + 1000.0)
    r = grid(randn(37, C, seed=1) - 300.0) if residual else None
    w = 1 + 0.3 * randn(C, seed=2)
    return x, r, w, randn(37, C, seed=4)


@gpu
@pytest.mark.parametrize("C", [7, 256, 511, 1000, 2047, 5001, 8192, 8200])
@pytest.mark.parametrize("residual", [False, True])
def test_layer_norm_gradient_far_from_zero(C, residual, cuda_lib):
    """Rows a thousand deviations from zero: the gradients take the rows that made y."""
    x, r, w, g = _offset_case(C, residual)
    leaves = [t.requires_grad_() for t in (x, r, w) if t is not None]
    y = layer_norm(x, w, None, residual=r)
    want, z, rstd = ref.layer_norm(x.detach(), w.detach(), None, None if r is None else r.detach(), 1e-5)
    dx, dw, _ = ref.layer_norm_grad(z, rstd, w.detach(), g)
    got = torch.autograd.grad(y, leaves, g)
    close(y.detach(), want, torch.float32, 64, 1024, what="y")
    close(got[0], dx, torch.float32, 64, 1024, what="dx")
    close(got[-1], dw, torch.float32, 64, 1024, what="dw")


@gpu
@pytest.mark.parametrize("C", [3, 7, 100, 1000, 5001, 8192, 8200])
def test_layer_norm_of_constant_rows(C, cuda_lib):
    """Far from zero their variance is what rounding left: sums of up to 26 terms in a row
    leave 28 u of the row and, of that, 28 u again, by at most 1 / sqrt(eps)."""
    at = torch.tensor([0.1, 1e4, 1e8, -3.3e9, 514228608.0, 2063394304.0, 33778102272.0, 15217946624.0], device=DEV)
    x = at[:, None].expand(8, C).contiguous().requires_grad_()
    y = layer_norm(x)
    off = (28 * ref.U[torch.float32]) ** 2 * at.abs() / 1e-5 ** 0.5
    assert (y.abs() <= off[:, None]).all()
    gx, = torch.autograd.grad(y, x, randn(8, C))
    assert torch.isfinite(gx).all()


def _attention_args(**over):
    a = _lib.AttentionArgs()
    names = ("query", "key", "value", "out", "lse", "grad_out", "grad_query", "grad_key", "grad_value")
    fields = dict.fromkeys(names, 16) | dict(batch=1, num_queries=100, num_keys=100, num_heads=2, num_key_heads=1, head_dim=8,
                                             scale=1.0, shared_document=-1)
    for n, v in (fields | over).items():
        setattr(a, n, v)
    for n in ("query_strides", "key_strides", "value_strides", "grad_out_strides"):
        getattr(a, n)[:] = (8, 8, 8)
    return ctypes.byref(a)


REFUSED = [dict(batch=65536), dict(num_heads=4097), dict(num_queries=2**22 + 1), dict(num_queries=65535 * 64 + 1),
           dict(num_queries=65535 * 64 + 1, head_dim=136, dtype=1), dict(num_keys=2**30 + 1), dict(head_dim=257), dict(dtype=3),
           dict(num_heads=3, num_key_heads=2), dict(num_queries=-1)]
REFUSED_BACKWARD = [dict(num_keys=65535 * 64 + 1), dict(num_keys=2**22 + 1, dtype=2)]


@host_only
def test_attention_refuses_sizes_that_no_grid_holds():
    """The launches and the workspace's size by the same limits; one less or another layout passes them
    (the launches then ask for a workspace)."""
    lib = _lib.load()
    for over in REFUSED:
        assert lib.msda_attention_forward(_attention_args(**over), None) in (_lib.MSDA_ERR_UNSUPPORTED, _lib.MSDA_ERR_INVALID_ARGUMENT)
        assert b"workspace" not in lib.msda_last_error()
    for over in REFUSED + REFUSED_BACKWARD:
        assert lib.msda_attention_workspace_size(_attention_args(**over), 1) == 0
        assert lib.msda_attention_backward(_attention_args(**over), None) in (_lib.MSDA_ERR_UNSUPPORTED, _lib.MSDA_ERR_INVALID_ARGUMENT)
        assert b"workspace" not in lib.msda_last_error()
    for over in (dict(batch=65535), dict(num_queries=65535 * 64), dict(num_queries=2**22, dtype=1), dict(num_keys=65535 * 64),
                 dict(num_keys=2**22, dtype=2)):
        assert lib.msda_attention_workspace_size(_attention_args(**over), 1) > 0
        assert lib.msda_attention_backward(_attention_args(**over), None) == _lib.MSDA_ERR_INVALID_ARGUMENT
        assert b"workspace" in lib.msda_last_error()
    assert lib.msda_attention_workspace_size(None, 0) == 0


@gpu
@pytest.mark.parametrize("recorded", [True, False])
def test_forward_mode_is_refused(recorded, cuda_lib):
    """A tangent is not dropped: the operators have no forward-mode derivative."""
    x, q = randn(3, 8), randn(1, 3, 2, 8)
    w = randn(8)
    pos = torch.arange(3, device=DEV).view(3, 1)
    plain = layer_norm(x), rotary(q, pos, axis_dims=[8]), attention(q, q, q)
    with forward_ad.dual_level(), torch.set_grad_enabled(recorded):
        dx, dw, dq = (forward_ad.make_dual(t, t.clone()) for t in (x, w, q))
        for call in (lambda: layer_norm(dx), lambda: layer_norm(x, dw), lambda: layer_norm(x, w, dw), lambda: layer_norm(x, residual=dx),
                     lambda: rotary(dq, pos, axis_dims=[8]), lambda: rotary(q, pos, key=dq, axis_dims=[8]),
                     lambda: attention(dq, q, q), lambda: attention(q, dq, q), lambda: attention(q, q, dq)):
            with pytest.raises(RuntimeError, match="forward mode AD"):
                call()
        for a, b in zip(plain, (layer_norm(x), rotary(q, pos, axis_dims=[8]), attention(q, q, q))):
            assert torch.equal(a, b)
    with pytest.raises(RuntimeError):
        torch.func.jvp(layer_norm, (x,), (x,))


def test_attention_arguments_are_packed_as_the_header_lays_them_out():
    """The one-call packing against the structure by its fields."""
    tensors = [torch.empty(2, 3 + i % 2, 4, 8).transpose(1, 2).contiguous().transpose(1, 2) for i in range(8)]
    lse, slopes = torch.empty(2, 4, 3), torch.empty(4)
    ints = [torch.empty(n, dtype=torch.int32) for n in (6, 8, 2, 2)]
    q, k, v, out, residue, dq, dk, dv = tensors
    packed = _pack(q, k, v, out, residue, lse, (q, dq, dk, dv), (0.5, 20.0, 1, 7), (slopes, *ints), 4096, 12345)
    a = _lib.AttentionArgs()
    pointers = dict(query=q, key=k, value=v, out=out, out_residue=residue, lse=lse, grad_out=q, grad_query=dq, grad_key=dk, grad_value=dv,
                    distance_slopes=slopes, query_documents=ints[0], key_documents=ints[1], prefix_lengths=ints[2], key_lengths=ints[3])
    for n, t in pointers.items():
        setattr(a, n, t.data_ptr())
    for n, value in dict(batch=2, num_queries=3, num_keys=4, num_heads=4, num_key_heads=4, head_dim=8, dtype=0, scale=0.5, softcap=20.0,
                         shared_document=7, causal=1, workspace=4096, workspace_bytes=12345).items():
        setattr(a, n, value)
    for n, t in dict(query_strides=q, key_strides=k, value_strides=v, grad_out_strides=q).items():
        getattr(a, n)[:] = t.stride()[:3]
    assert packed == bytes(a)


@gpu
def test_offsets_past_32_bits(cuda_lib):
    """Tensors of more than 2^32 bytes and 2^31 elements, of which the last rows count."""
    dtype, D, heads, near = torch.bfloat16, 128, 8, 200
    n = 2**31 // (heads * D) + near  # rows of heads x D
    x = torch.zeros(1, n, heads, D, dtype=dtype, device=DEV)
    end = x[:, -near:]
    end.copy_(randn(1, near, heads, D, dtype=dtype))
    value = torch.zeros_like(x)
    value[:, -near:] = randn(1, near, heads, D, dtype=dtype, seed=1)
    ids = torch.full((1, n), -1, dtype=torch.int32, device=DEV)
    ids[:, -near:] = 0
    for Sq in (1, 130):
        q, g = randn(1, Sq, heads, D, dtype=dtype, seed=2), randn(1, Sq, heads, D, dtype=dtype, seed=3)
        want, _, grads = ref.attention(q, end, value[:, -near:], g)
        leaves = [t.detach().requires_grad_() for t in (q, x, value)]
        out = attention(*leaves, query_documents=ids[:, -Sq:].contiguous(), key_documents=ids)
        close(out.detach(), want, dtype, *tolerance(dtype), floor=0.02, what="out")
        dq, dk, dv = torch.autograd.grad(out, leaves, g)
        for what, a, b in zip(("dq", "dk", "dv"), (dq, dk[:, -near:], dv[:, -near:]), grads):
            close(a, b, dtype, *tolerance(dtype), floor=0.02, what=what)
        assert not dk[:, :-near].any() and not dv[:, :-near].any()
        del leaves, out, dq, dk, dv
    del value, ids
    rows, g = x.view(n * heads, D), torch.zeros_like(x).view(n * heads, D)
    g[-near:] = randn(near, D, dtype=dtype, seed=5)
    rows = rows.requires_grad_()
    y = layer_norm(rows)
    want, z, rstd = ref.layer_norm(rows.detach()[-near:], None, None, None, 1e-5)
    close(y.detach()[-near:], want, dtype, 1.5, 8, floor=0.1, what="y")
    close(torch.autograd.grad(y, rows, g)[0][-near:], ref.layer_norm_grad(z, rstd, None, g[-near:])[0], dtype, 1.5, 8, floor=0.1, what="dx")
    del y, g, rows
    at = torch.arange(n, device=DEV)[:, None]
    y = rotary(x.detach(), at, axis_dims=[D])
    close(y[:, -near:], ref.rotary(x.detach()[:, -near:], at[-near:], [D]), dtype, 1.5, 8, what="rotary")


@pytest.mark.parametrize("how, words", [(dict(shared_document=2**31), "shared_document"), (dict(shared_document=-1), "shared_document"),
                                        (dict(scale=1e39), "scale"), (dict(scale=float("-inf")), "scale"), (dict(softcap=1e39), "softcap"),
                                        (dict(softcap=float("nan")), "softcap"), (dict(softcap=3e38), "softcap"),
                                        (dict(softcap=1e-40), "softcap"), (dict(softcap=1e-29, scale=1e10), "scale")])
def test_attention_refuses_numbers_that_32_bits_do_not_hold(how, words):
    x, ids = torch.zeros(1, 2, 2, 8), torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match=words):
        attention(x, x, x, query_documents=ids, key_documents=ids, **how)


@host_only
def test_c_abi_refuses_caps_that_leave_32_bits():
    lib = _lib.load()
    for over in (dict(softcap=3e38), dict(softcap=1e-40), dict(softcap=1e-29, scale=1e10)):
        assert lib.msda_attention_forward(_attention_args(**over), None) == _lib.MSDA_ERR_INVALID_ARGUMENT
        assert b"softcap" in lib.msda_last_error()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("softcap", [2.0**100, 2.0**-100])
@pytest.mark.parametrize("Sq, H", [(1, 2), (300, 16)])
def test_caps_at_their_limits(Sq, H, softcap, dtype, cuda_lib):
    """The widest changes nothing, the narrowest leaves equal scores."""
    q, k, v, g = (randn(1, Sq if i in (0, 3) else 300, H, 64, dtype=dtype, seed=i) for i in range(4))
    want, _, grads = ref.attention(q, k, v, g, softcap=softcap)
    q, k, v = (t.requires_grad_() for t in (q, k, v))
    out = attention(q, k, v, softcap=softcap)
    close(out.detach(), want, dtype, *tolerance(dtype), floor=0.02, what="out")
    for n, a, b in zip(("dq", "dk", "dv"), torch.autograd.grad(out, (q, k, v), g), grads):
        close(a, b, dtype, *tolerance(dtype), floor=0.02, what=n)
