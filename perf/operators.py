"""The transformer operators beside deformable attention, as cases that can be
timed and compared: rotary positions over several axes, (residual and) layer
norm, and attention with a tanh cap, a distance bias and document, prefix and
length masks, for training and for single tokens.

``run`` computes a case either in its plain form (elementary torch operations
in 32 bits) or, where ``own`` is true, by the calls that a user makes of this
repository's package. ``exact`` computes the same outputs from the operators'
definitions in 64 bits.

Layouts: query (B, Sq, H, D), key and value (B, Sk, Hkv, D) with H a multiple
of Hkv, rotary positions (B, S, A), layer norm rows (N, C).
"""

import math
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}

# The visual configurations of this repository: 300 object queries of a
# detection decoder, 22 223 pixels of an encoder's pyramid (800 x 1333, strides
# 8 to 64), 8 heads of 32 channels, batches of 4.
ROTARY = dict(op="rotary", dtype="bf16", B=4, S=300, H=8, Hkv=8, D=32, axes="16,16", ladder="axis",
              pairing="half", train=True, whole=False, reach=100.0)
NORM = dict(op="norm", dtype="bf16", N=1200, C=256, residual=True, train=True)
ATTENTION = dict(op="attention", dtype="bf16", B=4, Sq=300, Sk=300, H=8, Hkv=8, D=32, train=True, softcap=0.0,
                 slopes=False, causal=False, prefix=False, documents=0, shared=False, lengths=False)


def listed():
    return [
        # One new token in each of 8 streams of a decoder over images and
        # text (time, height, width): query and key heads in one call.
        ROTARY | dict(name="rotary_token", B=8, S=1, Hkv=2, D=64, axes="16,24,24", ladder="shared", train=False,
                      whole=True, reach=30000.0),
        # A detection decoder's object queries, rotated by their reference points.
        ROTARY | dict(name="rotary_queries", dtype="f32"),
        # An encoder's pixels, height and width, a training step.
        ROTARY | dict(name="rotary_pixels", S=22223, pairing="interleaved"),
        # The norm after a decoder's sublayer, with its residual, a training step.
        NORM | dict(name="norm_queries"),
        # The same after an encoder's sublayer.
        NORM | dict(name="norm_pixels", N=4 * 22223),
        # A wide model's norm without a residual; an odd width in 32 bits.
        NORM | dict(name="norm_wide", dtype="f32", N=4095, C=5001, residual=False),
        # Self-attention among object queries with denoising groups: each group
        # sees itself and the matching queries, which see themselves only.
        ATTENTION | dict(name="attention_denoising", Sq=500, Sk=500, documents=5, shared=True),
        # A long causal training step with capped scores and shared key heads.
        ATTENTION | dict(name="attention_capped", B=1, Sq=8192, Sk=8192, H=16, Hkv=4, D=128, softcap=30.0, causal=True),
        # A packed batch of texts of different lengths, distance bias, forward only.
        ATTENTION | dict(name="attention_packed", dtype="f16", B=2, Sq=4097, Sk=4097, H=16, Hkv=16, D=64, causal=True,
                         slopes=True, documents=6, train=False),
        # A captioner's prefix mask in 32 bits, a training step.
        ATTENTION | dict(name="attention_prefix", dtype="f32", B=2, Sq=1201, Sk=1201, causal=True, prefix=True),
        # One new token of one short stream: latency.
        ATTENTION | dict(name="token_short", dtype="f16", B=1, Sq=1, Sk=900, causal=True, lengths=True, train=False),
        # One new token in each of 32 long streams of different lengths.
        ATTENTION | dict(name="token_long", B=32, Sq=1, Sk=16384, H=32, Hkv=8, D=128, softcap=30.0, causal=True,
                         lengths=True, train=False),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, uniform in its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5)))))))


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    op = rng.choice(["rotary", "norm", "attention", "attention", "token"])
    if op == "rotary":
        D = 2 * rng.randint(4, 64)
        cuts = sorted(rng.randint(1, D // 2) for _ in range(rng.randint(1, 3)))
        axes = [2 * (b - a) for a, b in zip([0] + cuts, cuts)]
        Hkv = rng.choice([1, 2, 4, 8])
        H = Hkv * rng.choice([1, 2, 4])
        B = rng.randint(1, 8)
        # The elements of the largest listed case: 4 x 22223 x 16 x 32.
        S = _spread(rng, 1, max(1, min(30000, 45_000_000 // (B * (H + Hkv) * D))))
        return ROTARY | dict(dtype=dtype, B=B, S=S, H=H, Hkv=Hkv, D=D, axes=",".join(str(a) for a in axes if a),
                             ladder=rng.choice(["axis", "shared"]), pairing=rng.choice(["half", "interleaved"]),
                             train=rng.random() < 0.6, whole=rng.random() < 0.5, reach=rng.choice([1.0, 100.0, 30000.0]))
    if op == "norm":
        C = _spread(rng, 1, 8192)
        N = _spread(rng, 1, min(90000, 20_000_000 // C))
        return NORM | dict(dtype=dtype, N=N, C=C, residual=rng.random() < 0.5, train=rng.random() < 0.6)
    Hkv = rng.choice([1, 2, 3, 4, 8])
    H = Hkv * rng.choice([1, 2, 4, 8])
    more = dict(dtype=dtype, H=H, Hkv=Hkv, softcap=rng.choice([0.0, 0.0, 15.0, 50.0]), slopes=rng.random() < 0.3)
    if op == "token":
        D = rng.choice([32, 64, 64, 128, 128, 8 * rng.randint(1, 16)])
        B = _spread(rng, 1, 32)
        Sk = _spread(rng, 1, max(1, min(16384, (32 * 16384 * 8 * 128) // (B * Hkv * D * (2 if dtype == "f32" else 1)))))
        Sq = min(Sk, rng.choice([1, 1, 1, 2, 4]))
        return ATTENTION | more | dict(B=B, Sq=Sq, Sk=Sk, D=D, causal=True, lengths=True, train=False)
    D = rng.choice([32, 32, 64, 64, 128, 8 * rng.randint(1, 16)])
    train = rng.random() < 0.6
    B = rng.randint(1, 4)
    # At most an eighth of the largest listed case's scores: its masks leave half.
    most = 16 * 8192 * 8192 / (32 if dtype == "f32" else 8)
    Sq = _spread(rng, 1, int(min(8192, math.sqrt(most / (B * H)))))
    mask = rng.choice(["none", "causal", "prefix", "documents", "packed", "shared", "lengths"])
    Sk = Sq if mask != "none" else _spread(rng, 1, int(min(8192, most / (B * H * Sq))))
    return ATTENTION | more | dict(B=B, Sq=Sq, Sk=Sk, D=D, train=train, causal=mask in ("causal", "prefix", "packed"),
                                   prefix=mask == "prefix", lengths=mask == "lengths", shared=mask == "shared",
                                   documents=rng.randint(2, 8) if mask in ("documents", "packed", "shared") else 0)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda").to(dtype)

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device="cuda")

    if case["op"] == "rotary":
        B, S, H, Hkv, D = (case[k] for k in ("B", "S", "H", "Hkv", "D"))
        axes = [int(a) for a in case["axes"].split(",")]
        positions = uniform(B, S, len(axes)) * case["reach"]
        state = dict(query=normal(B, S, H, D), key=normal(B, S, Hkv, D), axes=axes,
                     positions=positions.long() if case["whole"] else positions)
        if case["train"]:
            state |= dict(grad_query=normal(B, S, H, D), grad_key=normal(B, S, Hkv, D))
        wants = ("query", "key")
    elif case["op"] == "norm":
        N, C = case["N"], case["C"]
        state = dict(x=normal(N, C) * 1.5 + 0.25, weight=1 + 0.1 * normal(C), bias=0.1 * normal(C))
        if case["residual"]:
            state["residual"] = normal(N, C)
        if case["train"]:
            state["grad"] = normal(N, C)
        wants = ("x", "weight", "bias", "residual")
    else:
        B, Sq, Sk, H, Hkv, D = (case[k] for k in ("B", "Sq", "Sk", "H", "Hkv", "D"))
        state = dict(query=normal(B, Sq, H, D), key=normal(B, Sk, Hkv, D), value=normal(B, Sk, Hkv, D), options={})
        options = state["options"]
        if case["softcap"]:
            options["softcap"] = case["softcap"]
        if case["slopes"]:  # slopes halve from head to head over eight octaves
            options["distance_slopes"] = 2.0 ** (-8.0 / H * torch.arange(1, H + 1, device="cuda"))
        if case["causal"]:
            options["causal"] = True
        if case["prefix"]:
            options["prefix_lengths"] = (uniform(B) * (Sk + 1)).int()
        if case["lengths"]:  # between a quarter of the cache and all of it
            options["key_lengths"] = (Sk * (0.25 + 0.75 * uniform(B))).ceil().int().clamp(Sq, Sk)
        if case["documents"]:
            # Random cuts; the last twentieth of every other row is padding.
            # With a shared document the first group is the one all see.
            cuts = (uniform(B, case["documents"] - 1) * Sk).int()
            token = torch.arange(Sk, device="cuda")
            ids = (token[None, :, None] >= cuts[:, None, :]).sum(-1).int()
            ids[1::2, Sk - Sk // 20:] = -1
            options["query_documents"] = options["key_documents"] = ids
            if case["shared"]:
                options["shared_document"] = 0
        if case["train"]:
            state["grad"] = normal(B, Sq, H, D)
        wants = ("query", "key", "value")
    if case["train"]:
        for k in wants:
            if k in state:
                state[k] = state[k].detach().requires_grad_(True)
    state["case"] = dict(case)
    return state


def run(state):
    step = {"rotary": (_plain_rotary, _own_rotary), "norm": (_plain_norm, _own_norm),
            "attention": (_plain_attention, _own_attention)}[state["case"]["op"]]
    if own:
        return step[1](state)
    with torch.no_grad():
        return step[0](state)


# The package's calls ---------------------------------------------------------
def _package():
    path = str(Path(__file__).resolve().parent.parent / "msda-triton_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import msda_triton_b200

    return msda_triton_b200


def _own_rotary(s):
    case = s["case"]
    q, k = _package().rotary(s["query"], s["positions"], key=s["key"], axis_dims=s["axes"], base=10000.0,
                             ladder=case["ladder"], pairing=case["pairing"])
    if not case["train"]:
        return {"query": q, "key": k}
    gq, gk = torch.autograd.grad((q, k), (s["query"], s["key"]), (s["grad_query"], s["grad_key"]))
    return {"query": q, "key": k, "grad_query": gq, "grad_key": gk}


def _own_norm(s):
    case = s["case"]
    y = _package().layer_norm(s["x"], s["weight"], s["bias"], residual=s.get("residual"), eps=1e-5)
    if not case["train"]:
        return {"y": y}
    wants = ["x", "weight", "bias"] + (["residual"] if case["residual"] else [])
    grads = torch.autograd.grad(y, [s[w] for w in wants], s["grad"])
    return {"y": y} | {"grad_" + w: g for w, g in zip(wants, grads)}


def _own_attention(s):
    out = _package().attention(s["query"], s["key"], s["value"], **s["options"])
    if not s["case"]["train"]:
        return {"out": out}
    wants = ("query", "key", "value")
    grads = torch.autograd.grad(out, [s[w] for w in wants], s["grad"])
    return {"out": out} | {"grad_" + w: g for w, g in zip(wants, grads)}


# The plain forms -------------------------------------------------------------
def _pairs(axes, ladder, pairing, base=10000.0):
    """For each rotated pair: its two channels, its axis and its frequency in
    turns per unit of position (64-bit numbers)."""
    first, second, axis, turns, start, total = [], [], [], [], 0, sum(axes)
    for a, d in enumerate(axes):
        for i in range(d // 2):
            offset, n, k = (start, d, i) if ladder == "axis" else (0, total, start // 2 + i)
            first.append(offset + (k if pairing == "half" else 2 * k))
            second.append(offset + (k + n // 2 if pairing == "half" else 2 * k + 1))
            axis.append(a)
            turns.append(base ** (-2.0 * k / n) / (2 * math.pi))
        start += d
    return first, second, axis, turns


def _halves(x):
    """x as the sum of two numbers of twelve bits each."""
    c = x * 4097.0
    high = c - (c - x)
    return high, x - high


def _plain_rotary(s):
    case = s["case"]
    first, second, axis, turns = _pairs(s["axes"], case["ladder"], case["pairing"])
    exact_turns = torch.tensor(turns, dtype=torch.float64)
    f = exact_turns.float()
    rest = (exact_turns - f.double()).float().cuda()
    f = f.cuda()
    p = s["positions"].float()[..., torch.tensor(axis, device="cuda")]
    # position * frequency to twice 32 bits, less its whole turns.
    t = p * f
    (ph, pl), (fh, fl) = _halves(p), _halves(f)
    error = ((ph * fh - t) + ph * fl + pl * fh) + pl * fl
    angle = ((t - t.round()) + (error + p * rest)) * (2 * math.pi)
    cos, sin = angle.cos()[:, :, None, :], angle.sin()[:, :, None, :]
    first, second = torch.tensor(first, device="cuda"), torch.tensor(second, device="cuda")

    def turn(x, sin):
        x32 = x.float()
        a, b, y = x32[..., first], x32[..., second], x32.clone()
        y[..., first] = a * cos - b * sin
        y[..., second] = a * sin + b * cos
        return y.to(x.dtype)

    out = {"query": turn(s["query"], sin), "key": turn(s["key"], sin)}
    if case["train"]:
        out |= {"grad_query": turn(s["grad_query"], -sin), "grad_key": turn(s["grad_key"], -sin)}
    return out


def _plain_norm(s):
    case, dtype = s["case"], s["x"].dtype
    x, w, b = s["x"].float(), s["weight"].float(), s["bias"].float()
    if case["residual"]:
        x = x + s["residual"].float()
    x = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-5)
    hat = x * r
    out = {"y": (hat * w + b).to(dtype)}
    if case["train"]:
        g = s["grad"].float()
        gw = g * w
        gx = (r * (gw - gw.mean(-1, keepdim=True) - hat * (gw * hat).mean(-1, keepdim=True))).to(dtype)
        out |= {"grad_x": gx, "grad_weight": (g * hat).sum(0).to(dtype), "grad_bias": g.sum(0).to(dtype)}
        if case["residual"]:
            out["grad_residual"] = gx
    return out


def _visible(case, options, Sq, Sk):
    """Which keys each query sees, (B or 1, Sq, Sk), and each query's place among the keys."""
    j = torch.arange(Sk, device="cuda")
    length = options.get("key_lengths")
    length = torch.full((1,), Sk, device="cuda") if length is None else length.long()
    place = length[:, None] - Sq + torch.arange(Sq, device="cuda")
    seen = (j < length[:, None])[:, None, :].expand(-1, Sq, -1)
    if options.get("causal"):
        earlier = j <= place[..., None]
        if "prefix_lengths" in options:
            earlier = earlier | (j < options["prefix_lengths"][:, None, None])
        seen = seen & earlier
    if "key_documents" in options:
        qd, kd = options["query_documents"][:, :, None], options["key_documents"][:, None, :]
        same = qd == kd
        if "shared_document" in options:
            same = same | (kd == options["shared_document"])
        seen = seen & same & (qd >= 0) & (kd >= 0)
    return seen, place


def _plain_attention(s):
    case, o, dtype = s["case"], s["options"], s["query"].dtype
    B, Sq, Sk, H, Hkv, D = (case[k] for k in ("B", "Sq", "Sk", "H", "Hkv", "D"))
    G, scale, cap = H // Hkv, 1 / math.sqrt(D), case["softcap"]

    def rows(x):  # (B, Sq, H, D) -> (B, Hkv, G * Sq, D)
        return x.float().view(B, Sq, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * Sq, D)

    def back(x):
        return x.view(B, Hkv, G, Sq, D).permute(0, 3, 1, 2, 4).reshape(B, Sq, H, D).to(dtype)

    q, k, v = rows(s["query"]), s["key"].float().transpose(1, 2), s["value"].float().transpose(1, 2)
    seen, place = _visible(case, o, Sq, Sk)
    score = (q @ k.transpose(-1, -2)).mul_(scale)
    if cap:
        score.div_(cap).tanh_()
        slope = 1 - score * score if case["train"] else None  # of the cap, for the gradient
        score.mul_(cap)
    score = score.view(B, Hkv, G, Sq, Sk)
    if case["slopes"]:
        far = (place[..., None] - torch.arange(Sk, device="cuda")).abs().float()
        score -= o["distance_slopes"].view(1, Hkv, G, 1, 1) * far[:, None, None]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    top.masked_fill_(top == -math.inf, 0.0)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(total.masked_fill_(total == 0, 1.0))
    p = p.view(B, Hkv, G * Sq, Sk)
    out = {"out": back(p @ v)}
    if case["train"]:
        g = rows(s["grad"])
        ds = g @ v.transpose(-1, -2)
        ds.sub_((p * ds).sum(-1, keepdim=True)).mul_(p)
        if cap:
            ds.mul_(slope)
        ds.mul_(scale)
        out |= {"grad_query": back(ds @ k), "grad_key": (ds.transpose(-1, -2) @ q).transpose(1, 2).to(dtype),
                "grad_value": (p.transpose(-1, -2) @ g).transpose(1, 2).to(dtype)}
    return out


# In 64 bits ------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"rotary": _exact_rotary, "norm": _exact_norm, "attention": _exact_attention}[case["op"]](case, s)


def _exact_rotary(case, s):
    """Axis by axis: channel pairs as complex numbers times exp(i * position * frequency)."""
    axes, total = s["axes"], sum(s["axes"])

    def turn(x, sign):
        y, start = x.detach().double(), 0
        for a, d in enumerate(axes):
            i = torch.arange(d // 2, device="cuda", dtype=torch.float64)
            if case["ladder"] == "axis":
                block, freq, at, apart = y[..., start:start + d], 10000.0 ** (-2 * i / d), 0, d // 2
            else:
                block, freq, at, apart = y[..., :total], 10000.0 ** (-2 * (i + start // 2) / total), start // 2, total // 2
            angle = s["positions"][..., a, None].double() * freq * sign
            factor = torch.complex(angle.cos(), angle.sin())[:, :, None]
            if case["pairing"] == "half":
                one, two = block[..., at:at + d // 2], block[..., apart + at:apart + at + d // 2]
            else:
                one, two = block[..., 2 * at:2 * at + d:2], block[..., 2 * at + 1:2 * at + d:2]
            z = torch.complex(one, two) * factor
            one.copy_(z.real), two.copy_(z.imag)
            start += d
        return y

    out = {n: turn(s[n], 1.0) for n in ("query", "key")}
    if case["train"]:
        out |= {n: turn(s[n], -1.0) for n in ("grad_query", "grad_key")}
    return out


def _exact_norm(case, s):
    x = s["x"].double() + (s["residual"].double() if case["residual"] else 0.0)
    C = case["C"]
    mean = x.sum(1) / C
    var = ((x - mean[:, None]) ** 2).sum(1) / C
    hat = (x - mean[:, None]) / (var + 1e-5).sqrt()[:, None]
    w = s["weight"].double()
    out = {"y": hat * w + s["bias"].double()}
    if case["train"]:
        g = s["grad"].double()
        h = g * w
        inner = torch.einsum("nc,nc->n", h, hat) / C
        gx = (h - (h.sum(1) / C)[:, None] - inner[:, None] * hat) / (var + 1e-5).sqrt()[:, None]
        out |= {"grad_x": gx, "grad_weight": torch.einsum("nc,nc->c", g, hat), "grad_bias": g.sum(0)}
        if case["residual"]:
            out["grad_residual"] = gx
    return out


def _exact_attention(case, s):
    """One batch item and head at a time, by the derivative of the log-sum-exp."""
    B, Sq, Sk, H, Hkv, D = (case[k] for k in ("B", "Sq", "Sk", "H", "Hkv", "D"))
    if B * H * Sq * Sk * D > 2e11:
        return None
    o, cap = s["options"], case["softcap"]
    q, k, v = (s[n].detach().double() for n in ("query", "key", "value"))
    out = {"out": torch.zeros_like(q)}
    if case["train"]:
        out |= {"grad_query": torch.zeros_like(q), "grad_key": torch.zeros_like(k), "grad_value": torch.zeros_like(v)}
    i, j = torch.arange(Sq, device="cuda")[:, None], torch.arange(Sk, device="cuda")[None]
    for b in range(B):
        length = int(o["key_lengths"][b]) if case["lengths"] else Sk
        far = length - Sq + i - j  # how far back of the query the key lies
        hidden = j >= length
        if case["causal"]:
            hidden = hidden | ((far < 0) & (j >= int(o["prefix_lengths"][b]) if case["prefix"] else far < 0))
        if case["documents"]:
            qd, kd = o["query_documents"][b][:, None], o["key_documents"][b][None]
            other = (qd != kd) & (kd != 0) if case["shared"] else qd != kd
            hidden = hidden | other | (qd < 0) | (kd < 0)
        mask, far = ~hidden.expand(Sq, Sk), far.abs().double()
        for h in range(H):
            kv = h // (H // Hkv)
            x = torch.einsum("id,jd->ij", q[b, :, h], k[b, :, kv]) / math.sqrt(D)
            t = torch.tanh(x / cap) if cap else None
            x = cap * t if cap else x
            if case["slopes"]:
                x = x - o["distance_slopes"][h].double() * far
            x = torch.where(mask, x, -math.inf)
            p = torch.exp(x - torch.logsumexp(x, 1, keepdim=True))
            p = torch.where(mask, p, 0.0)
            out["out"][b, :, h] = p @ v[b, :, kv]
            if case["train"]:
                g = s["grad"][b, :, h].double()
                ds = p * (torch.einsum("id,jd->ij", g, v[b, :, kv]) - (g * out["out"][b, :, h]).sum(1, keepdim=True))
                ds = ds * ((1 - t * t) if cap else 1.0) / math.sqrt(D)
                out["grad_query"][b, :, h] = ds @ k[b, :, kv]
                out["grad_key"][b, :, kv] += ds.T @ q[b, :, h]
                out["grad_value"][b, :, kv] += p.T @ g
    return out


def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "rotary":
        elements = case["B"] * case["S"] * (case["H"] + case["Hkv"]) * case["D"] * (2 if case["train"] else 1)
        axes = len(case["axes"].split(","))
        return {"bytes": 2 * es * elements + case["B"] * case["S"] * axes * (8 if case["whole"] else 4), "flops": 3 * elements}
    if case["op"] == "norm":
        # Forward: rows in, rows out; backward: rows and their gradient in, one gradient out.
        rows = case["N"] * case["C"]
        passes = 2 + case["residual"] + (2 if case["train"] else 0)
        return {"bytes": es * (rows * passes + 4 * case["C"]), "flops": rows * (8 + (10 if case["train"] else 0))}
    B, Sq, Sk, H, Hkv, D = (case[k] for k in ("B", "Sq", "Sk", "H", "Hkv", "D"))
    # Pairs that the masks leave, in expectation over the inputs.
    keys = Sk * (0.625 if case["lengths"] else 1.0)
    pairs = Sq * keys
    if case["documents"]:  # uniform cuts into n documents: sum of squares 2 / (n + 1)
        n = case["documents"]
        share = 2 / (n + 1)
        pairs *= min(1.0, share + (1 / n if case["shared"] else 0.0))
    if case["causal"] and Sq > 1:
        pairs *= 0.75 if case["prefix"] else 0.5 if Sq == Sk else 1.0
    size = 2 * B * Sq * H * D + 2 * B * keys * Hkv * D  # query, output; key, value
    if case["train"]:
        size += 2 * B * Sq * H * D + 2 * B * Sk * Hkv * D  # output gradient, query gradient; key, value gradients
    return {"bytes": es * size, "flops": (14 if case["train"] else 4) * B * H * D * pairs}
