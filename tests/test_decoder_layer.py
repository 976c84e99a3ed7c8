"""DeformableDecoderLayer: the operators together, as a detection decoder runs
them -- against the same composition in 64 bits (the cross-attention's own part by
its module, which test_layers.py pins), with denoising groups, its gradients
against differences, and step by step over a cache."""

from __future__ import annotations

import pytest
import torch

import layer_reference as ref
from msda_triton_b200 import DeformableDecoderLayer

SHAPES = [(12, 16), (6, 8)]


def test_refuses_heads_that_do_not_split_in_two_axes():
    with pytest.raises(ValueError, match="multiple of 4"):
        DeformableDecoderLayer(36, 6, 2, 4)


def _inputs(B, Q, C, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    S = sum(h * w for h, w in SHAPES)
    rand = lambda *s: torch.randn(*s, generator=g).to("cuda", dtype)  # noqa: E731
    points = torch.rand(B, Q, 2, generator=g).to("cuda", dtype)
    return rand(B, Q, C), points, rand(B, S, C), torch.tensor(SHAPES, device="cuda")


def _layer(C=64, M=4, dtype=torch.float32, seed=1):
    torch.manual_seed(seed)
    layer = DeformableDecoderLayer(C, M, len(SHAPES), 4, ffn_dim=96).to("cuda", dtype)
    for n in (layer.norm1, layer.norm2, layer.norm3):
        torch.nn.init.normal_(n.weight, 1.0, 0.2)
        torch.nn.init.normal_(n.bias, 0.0, 0.2)
    return layer


def _reference(layer, query, points, value, shapes, **masks):
    """The layer in 64 bits, but for the cross-attention."""
    lin = lambda m, x: x @ m.weight.double().T + m.bias.double()  # noqa: E731
    B, Q, C = query.shape
    q, k, v = lin(layer.in_proj, query.double()).view(B, Q, 3, layer.num_heads, -1).unbind(2)
    at, half = points.double() * layer.position_scale, [layer.head_dim // 2] * 2
    x, _, _ = ref.attention(ref.rotary(q, at, half), ref.rotary(k, at, half), v, **masks)
    norm = lambda n, x, r: ref.layer_norm(x, n.weight, n.bias, r, n.eps)[0]  # noqa: E731
    x = norm(layer.norm1, lin(layer.self_out_proj, x.flatten(2)), query)
    cross = layer.cross_attn(x.to(query.dtype), points, value, shapes).double()
    x = norm(layer.norm2, cross, x)
    return norm(layer.norm3, lin(layer.linear2, lin(layer.linear1, x).relu()), x)


@pytest.mark.gpu
@pytest.mark.parametrize("grouped", [False, True])
def test_forward_and_gradient(grouped, cuda_lib):
    """fp32, matrix products of torch included: sums of up to 96 terms and three
    norms in a row; 1e-5 of outputs near 1 leaves them a factor of ten."""
    B, Q, C = 2, 150, 64
    layer = _layer()
    query, points, value, shapes = _inputs(B, Q, C, torch.float32)
    masks = {}
    if grouped:
        ids = (torch.arange(Q, device="cuda") // 30).int().expand(B, Q).contiguous()
        masks = dict(groups=ids, shared_group=0)
    kinds = dict(query_documents=ids, key_documents=ids, shared_document=0) if grouped else {}
    with torch.no_grad():
        got = layer(query, points, value, shapes, **masks)
        want = _reference(layer, query, points, value, shapes, **kinds)
    assert float((got.double() - want).abs().max()) < 1e-5 * max(1.0, float(want.abs().max()))
    # The derivative along a random direction, against central differences
    # (step 1e-3: third-order and rounding errors of about 1e-3 of it).
    g = torch.randn_like(query)
    d = torch.randn_like(query)
    d /= d.norm()
    x = query.clone().requires_grad_()
    loss = (layer(x, points, value, shapes, **masks) * g).sum()
    params = [p for p in layer.parameters()]
    grads = torch.autograd.grad(loss, [x, *params])
    assert all(torch.isfinite(t).all() for t in grads)
    with torch.no_grad():
        ends = [(_reference(layer, (query.double() + s * 1e-3 * d.double()).float(), points, value, shapes, **kinds)
                 * g.double()).sum() for s in (1, -1)]
    slope = float(ends[0] - ends[1]) / 2e-3
    assert abs(slope - float((grads[0] * d).sum())) < 2e-2 * max(1.0, abs(slope))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_steps_over_a_cache_give_the_causal_layer(dtype, cuda_lib):
    """bf16: four layers' worth of roundings of 2^-8 each on outputs near 1."""
    B, Q, C, M = 3, 9, 64, 4
    layer = _layer(dtype=dtype)
    query, points, value, shapes = _inputs(B, Q, C, dtype)
    keys = torch.full((B, Q + 3, M, C // M), float("nan"), device="cuda", dtype=dtype)
    values = keys.clone()
    with torch.no_grad():
        whole = layer(query, points, value, shapes, causal=True)
        for i in range(Q):
            lengths = torch.full((B,), i + 1, dtype=torch.int32, device="cuda")
            one = layer.step(query[:, i:i + 1], points[:, i:i + 1], value, shapes, None, keys, values, lengths)
            off = (one[:, 0].double() - whole[:, i].double()).abs().max()
            assert float(off) < (1e-4 if dtype == torch.float32 else 16 * 2.0 ** -8)
