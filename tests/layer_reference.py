"""Plain 64-bit forms of the layer operators (rotary positions, layer norm,
masked attention), each from its formula, and the tolerances of their tests.

Tolerances. u is the unit roundoff of the output's type (2^-11 fp16, 2^-8
bf16, 2^-24 fp32). The error is measured in the 2-norm, relative to the
result's, and for single elements relative to the larger of the element and
the result's root mean square.

* An output rounded once from 32 bits is at most u off; ROUNDED allows 1.5 u.
* Attention in 16 bits also rounds the probabilities (or their derivative) to
  the inputs' type before the second product: two errors of at most u each,
  and 3 u leaves room for the sums; a single element meets them at full size
  and may be smaller than its terms: 12 u.
* Where early keys meet many terms far above the result's root mean square (long
  causal calls), an element is held to its own terms instead: each is rounded
  once, by at most u, and their sum once more; the sum over g . out that enters
  each ds has its own terms rounded; a quarter above that is for the sums in 32
  bits. What lies below fp16's normal numbers, 2^-14, is rounded as they are.
* In 32 bits the sums dominate: n terms in order are off by at most n u, near
  sqrt(n) u for signs at random; n is at most a few thousand here, and scores
  of size s turn an error of s u into one of the exponential's: 64 u in the
  norm and 1024 u for single elements while scores stay below 64, and in
  proportion above.
"""

from __future__ import annotations

import math

import torch

U = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.float16, torch.bfloat16)}


def off(got: torch.Tensor, want: torch.Tensor, floor: float = 0.0) -> tuple[float, float]:
    """(error in the norm, largest element's error), relative as above;
    `floor`: the least root mean square to measure against."""
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    assert torch.equal(torch.isfinite(got), torch.isfinite(want))
    assert torch.equal(got[~torch.isfinite(want)], want[~torch.isfinite(want)])
    got, want = got[torch.isfinite(want)], want[torch.isfinite(want)]
    d = (got - want).abs()
    if not d.numel():
        return 0.0, 0.0
    rms = max(float(want.square().mean().sqrt()), floor, 1e-30)
    return float(d.square().mean().sqrt()) / rms, float((d / want.abs().clamp_min(rms)).max())


def close(got, want, dtype, norm_u, element_u, floor=0.0, what=""):
    u = U[dtype]
    norm, element = off(got, want, floor)
    assert norm <= norm_u * u and element <= element_u * u, (
        f"{what}: {norm / u:.2f} u in the norm (at most {norm_u}), {element / u:.2f} u at an element (at most {element_u})")


def rotary(x, positions, axis_dims, ladder="axis", pairing="half", base=10000.0, inverse=False):
    y = x.double().clone()
    p = positions.double()
    if p.dim() == 2:
        p = p[None]
    start, total = 0, sum(axis_dims)
    for a, d in enumerate(axis_dims):
        for i in range(d // 2):
            n, k, at = (d, i, start) if ladder == "axis" else (total, start // 2 + i, 0)
            c0, c1 = (at + k, at + k + n // 2) if pairing == "half" else (at + 2 * k, at + 2 * k + 1)
            t = p[..., a, None] * base ** (-2.0 * k / n) * (-1 if inverse else 1)
            u, v = x[..., c0].double(), x[..., c1].double()
            y[..., c0] = u * t.cos() - v * t.sin()
            y[..., c1] = u * t.sin() + v * t.cos()
        start += d
    return y


def layer_norm(x, weight, bias, residual, eps):
    h = x.double() if residual is None else x.double() + residual.double()
    h = h.reshape(-1, h.shape[-1])
    c = h - h.mean(-1, keepdim=True)
    r = 1 / (c.square().mean(-1, keepdim=True) + eps).sqrt()
    z = c * r
    y = z * (weight.double() if weight is not None else 1) + (bias.double() if bias is not None else 0)
    return y.reshape(x.shape), z, r


def layer_norm_grad(z, r, weight, g, grad_sum=None):
    g = g.double().reshape(z.shape)
    gw = g * (weight.double() if weight is not None else 1)
    dx = r * (gw - gw.mean(-1, keepdim=True) - z * (gw * z).mean(-1, keepdim=True))
    if grad_sum is not None:
        dx = dx + grad_sum.double().reshape(z.shape)
    return dx, (g * z).sum(0), g.sum(0)


def visible(B, Sq, Sk, device, causal=False, prefix_lengths=None, query_documents=None, key_documents=None,
            shared_document=None, key_lengths=None):
    """(B, Sq, Sk) truth values and (B, Sq) places, one item at a time."""
    seen, places = [], []
    j = torch.arange(Sk, device=device)
    for b in range(B):
        n = Sk if key_lengths is None else min(max(int(key_lengths[b]), 0), Sk)
        place = n - Sq + torch.arange(Sq, device=device)
        s = (j < n).expand(Sq, Sk).clone()
        if causal:
            c = j[None] <= place[:, None]
            if prefix_lengths is not None:
                c = c | (j < int(prefix_lengths[b]))[None]
            s &= c
        if key_documents is not None:
            q, k = query_documents[b][:, None], key_documents[b][None]
            d = q == k
            if shared_document is not None:
                d = d | (k == shared_document)
            s &= d & (q >= 0) & (k >= 0)
        seen.append(s)
        places.append(place)
    return torch.stack(seen), torch.stack(places)


def attention(q, k, v, g=None, scale=None, softcap=0.0, distance_slopes=None, terms=None, **masks):
    """out, lse and, for an output gradient g, (dq, dk, dv); with `terms` also the
    sums of the sizes of out's, dq's, dk's and dv's terms, of which the rounded
    factor counts for `terms` at least."""
    B, Sq, H, D = q.shape
    Sk, Hkv = k.shape[1:3]
    scale = D ** -0.5 if scale is None else scale
    seen, place = visible(B, Sq, Sk, q.device, **masks)
    # What no query of the item sees counts for nothing, whatever it holds.
    kill = ~seen.any(1)[:, :, None, None]
    q, k, v = q.double(), k.double().masked_fill(kill, 0), v.double().masked_fill(kill, 0)
    G = H // Hkv
    kk, vv = k.repeat_interleave(G, 2), v.repeat_interleave(G, 2)
    s = torch.einsum("bihd,bjhd->bhij", q, kk) * scale
    t = torch.zeros_like(s)
    if softcap:
        t = torch.tanh(s / softcap)
        s = softcap * t
    if distance_slopes is not None:
        far = (place[:, :, None] - torch.arange(Sk, device=q.device)).abs().double()
        s = s - distance_slopes.double()[None, :, None, None] * far[:, None]
    s = s.masked_fill(~seen[:, None], -math.inf)
    lse = torch.logsumexp(s, -1) if Sk else torch.full(s.shape[:3], -math.inf, dtype=s.dtype, device=s.device)
    p = torch.exp(s - lse.masked_fill(lse == -math.inf, 0)[..., None])
    out = torch.einsum("bhij,bjhd->bihd", p, vv)
    if g is None:
        return out, lse, None
    g = g.double()
    dp = torch.einsum("bihd,bjhd->bhij", g, vv)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * (1 - t * t) * scale
    fold = lambda x: x.reshape(B, Sk, Hkv, G, D).sum(3)  # noqa: E731
    grads = (torch.einsum("bhij,bjhd->bihd", ds, kk), fold(torch.einsum("bhij,bihd->bjhd", ds, q)),
             fold(torch.einsum("bhij,bihd->bjhd", p, g)))
    if terms is None:
        return out, lse, grads
    # The output's rounded probabilities reach every ds of a row by sum(g . out).
    ds = ds.abs() + p * (p * dp.abs()).sum(-1, keepdim=True) * (1 - t * t) * scale
    ds = (ds / scale).clamp_min(terms).masked_fill(~seen[:, None], 0) * scale
    p = p.clamp_min(terms).masked_fill(~seen[:, None], 0)
    return out, lse, grads, (torch.einsum("bhij,bjhd->bihd", p, vv.abs()), torch.einsum("bhij,bjhd->bihd", ds, kk.abs()),
                             fold(torch.einsum("bhij,bihd->bjhd", ds, q.abs())), fold(torch.einsum("bhij,bihd->bjhd", p, g.abs())))
