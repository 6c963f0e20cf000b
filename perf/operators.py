"""Measured cases of the transformer feed-forward operators.

Four operators, each in a plain form (`own` false: elementary torch operations
in 32 or 64 bits) and as the library's calls (`own` true):

  linear / linear_backward   C = act(alpha * A.B^T + bias) + residual, and its gradients
  route                      experts, top-k and weights of every token from router logits (and the logits' gradient)
  experts                    a whole mixture-of-experts layer on routed tokens: plan, gate/up product, down product, combine
  product / product_backward one product of every expert with its own tokens, and its gradients

A case is a dict of plain values; `listed()` holds the fixed ones, `draw(rng)`
makes another of the same ranges.
"""

import math

import torch

own = False

FP4_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn}
BITS = {"bf16": 16, "f16": 16, "e4m3": 8, "nvfp4": 4, "mxfp8": 8}
SCALE_BLOCK = {"nvfp4": 16, "mxfp8": 32}


# ------------------------------------------------------------------ the cases


def listed():
    return [
        # one token through a wide projection: the weight is read once, nothing else counts
        dict(name="linear one token", op="linear", fmt="bf16", m=1, n=8192, k=8192, out="bf16", activation="silu", bias=True, residual=True, save=False),
        # a short odd batch in half precision that keeps its pre-activation for training: launch latency
        dict(name="linear ragged f16", op="linear", fmt="f16", m=301, n=520, k=768, out="f16", activation="gelu", bias=True, residual=True, save=True),
        # an fp8 projection of a prompt with per-tensor scales folded into alpha
        dict(name="linear e4m3 prompt", op="linear", fmt="e4m3", m=4096, n=4096, k=4096, out="bf16", activation="gelu_tanh", bias=True, residual=True, save=False),
        # an fp4 projection of a prompt, block-scaled operands
        dict(name="linear nvfp4 prompt", op="linear", fmt="nvfp4", m=2048, n=14336, k=4096, out="bf16", activation="relu", bias=False, residual=True, save=False),
        # gradients of a small ragged layer: launches count
        dict(name="gradients ragged", op="linear_backward", fmt="f16", m=1001, n=520, k=768, activation="gelu", bias=True),
        # gradients of a training step's layer
        dict(name="gradients training", op="linear_backward", fmt="bf16", m=4096, n=8192, k=4096, activation="gelu_tanh", bias=True),
        # one token's choice among many experts in limited groups: latency
        dict(name="route one token", op="route", fmt="f32", tokens=1, experts=256, top_k=8, scores="sigmoid", bias=True, groups=8, top_groups=4, group_top=2, renormalise=True, scale=2.5, masked=False, backward=False),
        # a training batch's routing and the gradient of its logits, padding rows included
        dict(name="route training", op="route", fmt="bf16", tokens=16384, experts=128, top_k=8, scores="softmax", bias=False, groups=1, top_groups=1, group_top=1, renormalise=True, scale=1.0, masked=True, backward=True),
        # decoding a small batch: every expert's weights are read for a row or two
        dict(name="experts decode", op="experts", fmt="bf16", tokens=16, experts=64, top_k=8, hidden=2048, inner=1024, activation="swiglu", dropped=False),
        # a prompt through a few wide experts, padding tokens included
        dict(name="experts prompt", op="experts", fmt="bf16", tokens=4096, experts=8, top_k=2, hidden=4096, inner=2048, activation="swiglu", dropped=True),
        # fp8 experts with a dequantisation factor of their own, odd counts
        dict(name="product e4m3", op="product", fmt="e4m3", tokens=1111, experts=32, top_k=4, k=1024, n=1536, activation="swiglu", save=False),
        # a training step's gradients of the gate/up product
        dict(name="product gradients", op="product_backward", fmt="bf16", tokens=2048, experts=8, top_k=2, k=2048, n=2048, activation="swiglu"),
    ]


def _size(rng, low, high, step=1):
    """Log-uniform in [low, high], a multiple of `step`."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high))) / step)) * step
    return min(max(v, step if low <= step else low), high)


def draw(rng):
    op = rng.choice(["linear", "linear", "linear_backward", "route", "experts", "product", "product_backward"])
    act = rng.choice(["relu", "gelu", "gelu_tanh", "silu"])
    if op == "linear":
        fmt = rng.choice(["bf16", "f16", "e4m3", "nvfp4", "mxfp8"])
        step = {"bf16": 8, "f16": 8, "e4m3": 16, "nvfp4": 32, "mxfp8": 32}[fmt]
        while True:
            m, n, k = _size(rng, 1, 8192), _size(rng, 16, 14336, 1 if fmt in ("bf16", "f16", "e4m3") else 8), _size(rng, 64, 8192, step)
            if m * n * k < 2**36:
                break
        wide = fmt in ("bf16", "f16", "e4m3")
        return dict(op=op, fmt=fmt, m=m, n=n, k=k, out=rng.choice(["bf16", "f16", "f32"]) if wide else "bf16", activation=rng.choice([act, act, "none"]), bias=rng.random() < 0.7,
                    residual=rng.random() < 0.7, save=rng.random() < 0.3)
    if op == "linear_backward":
        while True:
            m, n, k = _size(rng, 8, 8192), _size(rng, 64, 8192, 8), _size(rng, 64, 8192, 8)
            if m * n * k < 2**35:
                break
        return dict(op=op, fmt=rng.choice(["bf16", "f16"]), m=m, n=n, k=k, activation=rng.choice([act, act, "none"]), bias=rng.random() < 0.7)
    if op == "route":
        groups, each = rng.choice([(1, rng.randint(4, 300)), (4, 16), (8, 32), (8, 20), (2, 5)])
        top_groups = rng.randint(1, groups)
        tokens, top_k = _size(rng, 1, 16384), rng.randint(1, min(8, top_groups * each))
        return dict(op=op, fmt=rng.choice(["bf16", "f32"]), tokens=tokens, experts=groups * each, top_k=top_k,
                    scores=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5, groups=groups, top_groups=top_groups, group_top=rng.randint(1, 2),
                    renormalise=top_k > 1 and rng.random() < 0.7, scale=rng.choice([1.0, 2.5]), masked=tokens > 64 and rng.random() < 0.4, backward=rng.random() < 0.5)
    experts = rng.choice([4, 8, 16, 60, 64])
    top_k = rng.randint(1, min(8, experts))
    gated = rng.choice(["swiglu", "geglu", act])
    while True:
        tokens, k, n = _size(rng, 1, 8192), _size(rng, 128, 4096, 16), _size(rng, 64, 4096, 16)
        if tokens * top_k * k * n < 2**35 and experts * k * n < 2**29 and tokens * top_k * max(k, n) < 2**27:
            break
    if op == "experts":
        return dict(op=op, fmt=rng.choice(["bf16", "f16"]), tokens=tokens, experts=experts, top_k=top_k, hidden=k, inner=n // 2 // 8 * 8, activation=gated, dropped=rng.random() < 0.4)
    if op == "product":
        return dict(op=op, fmt=rng.choice(["bf16", "f16", "e4m3"]), tokens=tokens, experts=experts, top_k=top_k, k=k, n=n, activation=rng.choice([gated, "none"]), save=rng.random() < 0.3)
    return dict(op=op, fmt=rng.choice(["bf16", "f16"]), tokens=tokens, experts=experts, top_k=top_k, k=k, n=n, activation=rng.choice([gated, "none"]))


# ------------------------------------------------------------------ the inputs


def _values(g, shape, fmt, spread=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * spread).to(TYPES[fmt])


def _blocked(scales):
    """[rows, groups] scale bytes -> the 128x4 blocked layout that block-scaled products read."""
    rows, cols = scales.shape
    rb, cb = -(-rows // 128), -(-cols // 4)
    padded = torch.zeros((rb * 128, cb * 4), dtype=torch.uint8, device=scales.device)
    padded[:rows, :cols] = scales
    return padded.view(rb, 4, 32, cb, 4).permute(0, 3, 2, 1, 4).reshape(-1).contiguous()


def _block_scaled(g, rows, k, fmt, spread):
    """Random codes and scales of a block-scaled operand: (operand, blocked scales, row-major scales)."""
    groups = k // SCALE_BLOCK[fmt]
    if fmt == "nvfp4":
        codes = torch.randint(0, 256, (rows, k // 2), generator=g, device="cuda", dtype=torch.uint8)
        scales = ((0.5 + torch.rand((rows, groups), generator=g, device="cuda")) * spread / 3).to(torch.float8_e4m3fn)
        return codes.view(torch.float4_e2m1fn_x2), _blocked(scales.view(torch.uint8)).view(torch.float8_e4m3fn), scales
    codes = torch.randn((rows, k), generator=g, device="cuda").to(torch.float8_e4m3fn)
    exponents = torch.randint(-1, 2, (rows, groups), generator=g, device="cuda") + int(round(math.log2(spread)))
    scales = (exponents + 127).to(torch.uint8)
    return codes, _blocked(scales).view(torch.float8_e8m0fnu), scales


def _routed(g, tokens, experts, top_k, dropped):
    """Experts of every token, some chosen more often than others; with `dropped`, padding tokens go nowhere."""
    liking = torch.randn((1, experts), generator=g, device="cuda") * 0.7
    scores = torch.randn((tokens, experts), generator=g, device="cuda") + liking
    weights, indices = torch.softmax(scores, -1).topk(top_k, dim=-1)
    weights, indices = (weights / weights.sum(-1, keepdim=True)).contiguous(), indices.to(torch.int32)
    if dropped:
        gone = torch.rand((tokens, 1), generator=g, device="cuda") < 0.06
        weights, indices = torch.where(gone, 0.0, weights), torch.where(gone, -1, indices)
    return weights, indices.contiguous()


def _router_logits(g, c):
    """Router logits and balancing bias.  Rows whose order would hang on the last bits of a score
    (two scores or two groups nearer than 1e-6 of the row's largest) are replaced by a row that is clear."""
    t, e = c["tokens"], c["experts"]
    rows = t + 64
    logits = (torch.randn((rows, e), generator=g, device="cuda") * 1.5).to(TYPES[c["fmt"]])
    # biases move in steps of 1/1024, as balancing by fixed updates leaves them
    bias = torch.randint(-64, 65, (e,), generator=g, device="cuda").float() / 1024 if c["bias"] else None
    x = logits.double()
    s = torch.softmax(x, -1) if c["scores"] == "softmax" else torch.sigmoid(x)
    choice = s if bias is None else s + bias.double()
    ordered = choice.sort(-1).values
    near = lambda v: (v.diff(dim=-1) < 1e-6 * v.abs().amax(-1, keepdim=True)).any(-1) if v.size(-1) > 1 else torch.zeros(v.size(0), dtype=torch.bool, device="cuda")  # noqa: E731
    unclear = near(ordered)
    if c["fmt"] == "bf16" and bias is None:  # equal bf16 logits are equal scores, which the lowest index settles
        equal = x.sort(-1).values
        unclear = ((ordered.diff(dim=-1) < 1e-6 * ordered.abs().amax(-1, keepdim=True)) & (equal.diff(dim=-1) != 0)).any(-1) if e > 1 else unclear
    if c["groups"] > 1:
        best = choice.view(rows, c["groups"], -1).topk(min(c["group_top"], e // c["groups"]), -1).values.sum(-1)
        unclear |= near(best.sort(-1).values)
    clear = (~unclear).nonzero().flatten()
    if clear.numel():
        pick = clear[torch.arange(rows, device="cuda") % clear.numel()]
        logits = torch.where(unclear[:, None], logits[pick], logits)
    logits = logits[:t].clone()
    if c["masked"]:  # padding rows have no expert at all; some experts are switched off
        logits[torch.rand((t,), generator=g, device="cuda") < 0.05] = -math.inf
        off = torch.rand((e,), generator=g, device="cuda") < 0.1
        off[: max(c["top_k"], 1)] = False
        logits[:, off] = -math.inf
    return logits, bias


def prepare(case, seed):
    c, g = dict(case), torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": c}
    if c["op"] == "linear":
        m, n, k = c["m"], c["n"], c["k"]
        s["alpha"] = None
        if c["fmt"] in SCALE_BLOCK:
            s["a"], s["sfa"], s["raw_sfa"] = _block_scaled(g, m, k, c["fmt"], 1.0)
            s["b"], s["sfb"], s["raw_sfb"] = _block_scaled(g, n, k, c["fmt"], 1 / math.sqrt(k) if c["fmt"] == "mxfp8" else 0.25)
            if c["fmt"] == "nvfp4":
                s["alpha"] = 4 / math.sqrt(k)
        elif c["fmt"] == "e4m3":
            s["a"], s["b"] = _values(g, (m, k), "e4m3", 16.0), _values(g, (n, k), "e4m3", 16.0)
            s["alpha"] = 1 / (256 * math.sqrt(k))
        else:
            s["a"], s["b"] = _values(g, (m, k), c["fmt"]), _values(g, (n, k), c["fmt"], 1 / math.sqrt(k))
        s["bias"] = torch.randn((n,), generator=g, device="cuda") if c["bias"] else None
        s["residual"] = _values(g, (m, n), c["out"]) if c["residual"] else None
    elif c["op"] == "linear_backward":
        m, n, k = c["m"], c["n"], c["k"]
        s["a"], s["b"] = _values(g, (m, k), c["fmt"]), _values(g, (n, k), c["fmt"], 1 / math.sqrt(k))
        s["grad"] = _values(g, (m, n), c["fmt"])
        s["z"] = _values(g, (m, n), c["fmt"]) if c["activation"] != "none" else None
    elif c["op"] == "route":
        s["logits"], s["bias"] = _router_logits(g, c)
        s["grad"] = torch.randn((c["tokens"], c["top_k"]), generator=g, device="cuda") if c["backward"] else None
    elif c["op"] == "experts":
        h, f = c["hidden"], c["inner"]
        f1 = 2 * f if c["activation"].endswith("glu") else f
        s["x"] = _values(g, (c["tokens"], h), c["fmt"])
        s["w1"] = _values(g, (c["experts"], f1, h), c["fmt"], 1 / math.sqrt(h))
        s["w2"] = _values(g, (c["experts"], h, f), c["fmt"], 1 / math.sqrt(f))
        s["weights"], s["indices"] = _routed(g, c["tokens"], c["experts"], c["top_k"], c["dropped"])
        s["residual"] = _values(g, (c["tokens"], h), c["fmt"])
    else:
        e, k, n = c["experts"], c["k"], c["n"]
        spread = 16.0 if c["fmt"] == "e4m3" else 1.0
        s["x"] = _values(g, (c["tokens"], k), c["fmt"], spread)
        s["w"] = _values(g, (e, n, k), c["fmt"], spread if c["fmt"] == "e4m3" else 1 / math.sqrt(k))
        s["alpha"] = (0.5 + torch.rand((e,), generator=g, device="cuda")) / (256 * math.sqrt(k)) if c["fmt"] == "e4m3" else None
        _, s["indices"] = _routed(g, c["tokens"], e, c["top_k"], False)
        if c["op"] == "product_backward":
            rows = c["tokens"] * c["top_k"]
            s["grad"] = _values(g, (rows, n // 2 if c["activation"].endswith("glu") else n), c["fmt"])
            s["z"] = _values(g, (rows, n), c["fmt"]) if c["activation"] != "none" else None
    return s


# ------------------------------------------------------------ the plain forms


def _act(name, z):
    """The activation of `z`; a gated one takes the gate from the first half of the columns."""
    if name == "swiglu" or name == "geglu":
        gate, up = z.chunk(2, -1)
        return _act("silu" if name == "swiglu" else "gelu", gate) * up
    if name == "relu":
        return z.clamp(min=0)
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z / math.sqrt(2)))
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    return z * torch.sigmoid(z) if name == "silu" else z


def _act_gradient(name, z, g):
    """d act(z) / dz times `g`."""
    if name == "swiglu" or name == "geglu":
        inner = "silu" if name == "swiglu" else "gelu"
        gate, up = z.chunk(2, -1)
        return torch.cat([_act_gradient(inner, gate, g * up), g * _act(inner, gate)], -1)
    if name == "relu":
        return torch.where(z > 0, g, 0)
    if name == "gelu":
        return g * (0.5 * (1 + torch.erf(z / math.sqrt(2))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi))
    if name == "gelu_tanh":
        t = torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z))
        return g * (0.5 * (1 + t) + 0.5 * z * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z))
    if name == "silu":
        p = torch.sigmoid(z)
        return g * p * (1 + z * (1 - p))
    return g


def _dequantised(operand, scales, fmt):
    """A block-scaled operand's values in 32 bits, which hold them exactly."""
    if fmt == "nvfp4":
        codes = operand.view(torch.uint8)
        codes = torch.stack([codes & 15, codes >> 4], -1).flatten(1)
        values = torch.tensor(FP4_VALUES, device=codes.device)[codes.long()]
        steps = scales.float()
    else:
        values, steps = operand.float(), torch.exp2(scales.float() - 127)
    return values * steps.repeat_interleave(SCALE_BLOCK[fmt], -1)


def _plain_route(c, logits, bias):
    """(scores, weights, indices) in 64 bits: the order of near scores is decided there."""
    x = logits.double()
    off = x == -math.inf
    if c["scores"] == "softmax":
        e = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-1e300))
        s = e / e.sum(-1, keepdim=True).clamp(min=1e-300)
    else:
        s = 1 / (1 + torch.exp(-x))
    s = torch.where(off, 0, s)
    choice = torch.where(off, -math.inf, s if bias is None else s + bias.double())
    t, e, groups = x.size(0), x.size(1), c["groups"]
    if groups > 1:
        best = choice.view(t, groups, -1).sort(-1, descending=True).values[..., : c["group_top"]].sum(-1)
        order = best.sort(dim=-1, descending=True, stable=True).indices[:, : c["top_groups"]]
        open_ = torch.zeros((t, groups), dtype=torch.bool, device=x.device).scatter_(1, order, True)
        choice = torch.where(open_.repeat_interleave(e // groups, -1), choice, -math.inf)
    best, order = choice.sort(dim=-1, descending=True, stable=True)
    best, order = best[:, : c["top_k"]], order[:, : c["top_k"]]
    none = best == -math.inf
    w = torch.where(none, 0, s.gather(1, order))
    if c["renormalise"]:
        w = w / w.sum(-1, keepdim=True).clamp(min=1e-300)
    return s, w * c["scale"], torch.where(none, -1, order)


def _plain_route_gradient(c, s, indices, grad):
    none = indices < 0
    at = indices.clamp(min=0).long()
    q, g = torch.where(none, 0, s.gather(1, at)), torch.where(none, 0, grad.double() * c["scale"])
    if c["renormalise"]:
        total = q.sum(-1, keepdim=True).clamp(min=1e-300)
        g = torch.where(none, 0, (g - (g * q).sum(-1, keepdim=True) / total) / total)
    ds = torch.zeros_like(s).scatter_add_(1, at, g)
    return s * (ds - (ds * s).sum(-1, keepdim=True)) if c["scores"] == "softmax" else ds * s * (1 - s)


def _plain_plan(indices, experts):
    """The (token, choice) pairs in order of their expert, in the order of the tokens inside one."""
    flat = indices.flatten().long()
    key = torch.where(flat < 0, experts, flat)
    expert, order = key.sort(stable=True)
    counts = torch.bincount(key, minlength=experts + 1)
    offsets = torch.cat([torch.zeros(1, dtype=torch.long, device=flat.device), counts.cumsum(0)])
    position = torch.empty_like(order)
    position[order] = torch.arange(order.numel(), device=flat.device)
    return {"expert": expert, "order": order, "offsets": offsets[: experts + 1], "slot": torch.arange(order.numel(), device=flat.device) - offsets[expert],
            "positions": torch.where(flat < 0, -1, position).view(indices.shape), "most": max(1, int(counts[:experts].max()))}


def _by_expert(rows, plan, experts):
    """Rows in sorted order -> [experts, most, columns], zeros behind each expert's last row."""
    padded = torch.zeros((experts + 1, max(plan["most"], int((plan["slot"]).max()) + 1), rows.size(1)), dtype=rows.dtype, device=rows.device)
    padded[plan["expert"], plan["slot"]] = rows
    return padded[:experts]


def _plain_product(rows, w, plan):
    """Every sorted row times its own expert's weights, in 32 bits."""
    experts = w.size(0)
    y = torch.bmm(_by_expert(rows, plan, experts), w.float().transpose(1, 2))
    y = torch.cat([y, torch.zeros_like(y[:1])])
    return y[plan["expert"], plan["slot"]]


def _plain(s):
    c = s["case"]
    if c["op"] == "linear":
        if c["fmt"] in SCALE_BLOCK:
            a, b = _dequantised(s["a"], s["raw_sfa"], c["fmt"]), _dequantised(s["b"], s["raw_sfb"], c["fmt"])
        else:
            a, b = s["a"].float(), s["b"].float()
        z = a @ b.T
        z = z if s["alpha"] is None else z * s["alpha"]
        z = z if s["bias"] is None else z + s["bias"]
        y = _act(c["activation"], z)
        y = y if s["residual"] is None else y + s["residual"].float()
        return {"c": y.to(TYPES[c["out"]]), **({"z": z.to(TYPES[c["out"]])} if c["save"] else {})}
    if c["op"] == "linear_backward":
        dz = s["grad"].float()
        if s["z"] is not None:
            dz = _act_gradient(c["activation"], s["z"].float(), dz)
        t = TYPES[c["fmt"]]
        return {"a": (dz @ s["b"].float()).to(t), "b": (dz.T @ s["a"].float()).to(t), **({"bias": dz.sum(0)} if c["bias"] else {})}
    if c["op"] == "route":
        scores, weights, indices = _plain_route(c, s["logits"], s["bias"])
        r = {"weights": weights.float(), "indices": indices.to(torch.int32)}
        if c["backward"]:
            r["logits"] = _plain_route_gradient(c, scores, indices, s["grad"]).to(s["logits"].dtype)
        return r
    plan = _plain_plan(s["indices"], c["experts"])
    tokens = plan["order"] // c["top_k"]
    rows = s["x"].float()[tokens]
    if c["op"] == "experts":
        y = _plain_product(_act(c["activation"], _plain_product(rows, s["w1"], plan)), s["w2"], plan)
        y = y * s["weights"].flatten()[plan["order"]][:, None]
        return {"y": s["residual"].float().index_add(0, tokens, y).to(TYPES[c["fmt"]]), "offsets": plan["offsets"].to(torch.int32), "positions": plan["positions"].to(torch.int32)}
    if c["op"] == "product":
        z = _plain_product(rows, s["w"], plan)
        z = z if s["alpha"] is None else z * s["alpha"][plan["expert"]][:, None]
        t = torch.bfloat16 if c["fmt"] == "e4m3" else TYPES[c["fmt"]]
        return {"y": _act(c["activation"], z).to(t), **({"z": z.to(t)} if c["save"] else {})}
    dz = s["grad"].float()
    if s["z"] is not None:
        dz = _act_gradient(c["activation"], s["z"].float(), dz)
    t = TYPES[c["fmt"]]
    dx = _plain_product(dz, s["w"].float().transpose(1, 2), plan)
    dw = torch.bmm(_by_expert(dz, plan, c["experts"]).transpose(1, 2), _by_expert(rows, plan, c["experts"]))
    return {"x": torch.zeros_like(s["x"], dtype=torch.float32).index_add(0, tokens, dx).to(t), "w": dw.to(t)}


# ------------------------------------------------------- the library's calls


def _own(s):
    import opengemm_b200 as og

    c = s["case"]
    act = c.get("activation")
    act = None if act == "none" else act
    if c["op"] == "linear":
        t = TYPES[c["out"]]
        z = torch.empty((c["m"], c["n"]), dtype=t, device="cuda") if c["save"] else None
        scales = (s["sfa"], s["sfb"]) if c["fmt"] in SCALE_BLOCK else ()
        y = og.gemm(s["a"], s["b"], *scales, out_dtype=t, alpha=s["alpha"], bias=s["bias"], activation=act, residual=s["residual"], preactivation=z)
        return {"c": y, **({"z": z} if c["save"] else {})}
    if c["op"] == "linear_backward":
        want = ("a", "b", "bias") if c["bias"] else ("a", "b")
        da, db, dbias = og.gemm_backward(s["grad"], s["a"], s["b"], activation=act, preactivation=s["z"], want=want)
        return {"a": da, "b": db, **({"bias": dbias} if c["bias"] else {})}
    if c["op"] == "route":
        how = dict(scores=c["scores"], renormalise=c["renormalise"], scale=c["scale"])
        weights, indices = og.route(s["logits"], c["top_k"], bias=s["bias"], groups=c["groups"], top_groups=c["top_groups"], group_top=c["group_top"], **how)
        r = {"weights": weights, "indices": indices}
        if c["backward"]:
            r["logits"] = og.route_backward(s["grad"], s["logits"], indices, **how)
        return r
    plan = og.expert_plan(s["indices"], c["experts"])
    if c["op"] == "experts":
        h = og.expert_gemm(s["x"], s["w1"], plan, gather=True, activation=act)
        y = og.expert_gemm(h, s["w2"], plan)
        return {"y": og.expert_combine(y, s["weights"], plan, residual=s["residual"]), "offsets": plan.offsets, "positions": plan.positions}
    if c["op"] == "product":
        z = torch.empty((c["tokens"] * c["top_k"], c["n"]), dtype=torch.bfloat16 if c["fmt"] == "e4m3" else TYPES[c["fmt"]], device="cuda") if c["save"] else None
        y = og.expert_gemm(s["x"], s["w"], plan, gather=True, activation=act, alpha=s["alpha"], preactivation=z)
        return {"y": y, **({"z": z} if c["save"] else {})}
    dx, dw = og.expert_gemm_backward(s["grad"], s["x"], s["w"], plan, gather=True, activation=act, preactivation=s["z"])
    return {"x": dx, "w": dw}


def run(state):
    if own:
        return _own(state)
    return _plain(state)


# ------------------------------------------------------------------- the work


def work(case):
    c = case
    if c["op"].startswith("linear"):
        m, n, k = c["m"], c["n"], c["k"]
        size = BITS[c["fmt"]] / 8
        if c["op"] == "linear":
            size += 1 / SCALE_BLOCK[c["fmt"]] if c["fmt"] in SCALE_BLOCK else 0
            out = 4 if c["out"] == "f32" else 2
            return {"bytes": (m + n) * k * size + m * n * out * (1 + c["residual"] + c["save"]) + 4 * n * c["bias"], "flops": 2 * m * n * k}
        return {"bytes": 2 * (2 * (m + n) * k + m * n * (1 + (c["activation"] != "none"))) + 4 * n * c["bias"], "flops": 4 * m * n * k}
    if c["op"] == "route":
        size = 4 if c["fmt"] == "f32" else 2
        t, e, k = c["tokens"], c["experts"], c["top_k"]
        return {"bytes": t * e * size * (1 + c["backward"]) + t * k * (8 + 4 * c["backward"]) + 4 * e * c["bias"], "flops": t * e * (8 + 8 * c["backward"])}
    pairs, e = c["tokens"] * c["top_k"], c["experts"]
    busy = e * (1 - (1 - 1 / e) ** pairs)
    if c["op"] == "experts":
        h, f = c["hidden"], c["inner"]
        f1 = 2 * f if c["activation"].endswith("glu") else f
        return {"bytes": 2 * (busy * h * (f1 + f) + 3 * c["tokens"] * h) + 12 * pairs, "flops": 2 * pairs * h * (f1 + f)}
    k, n, size = c["k"], c["n"], BITS[c["fmt"]] / 8
    width = n // 2 if c["activation"].endswith("glu") else n
    if c["op"] == "product":
        return {"bytes": size * (busy * n * k + c["tokens"] * k) + 2 * pairs * (width + n * c["save"]) + 4 * pairs, "flops": 2 * pairs * n * k}
    return {"bytes": 2 * ((busy + e) * n * k + 2 * c["tokens"] * k + pairs * (width + n * (c["activation"] != "none"))) + 4 * pairs, "flops": 4 * pairs * n * k}


# ------------------------------------------------- the definitions in 64 bits


def _exact_act(name, z):
    """(activation, derivative) of one value, elementwise in 64 bits."""
    if name == "relu":
        return torch.relu(z), (z > 0).double()
    if name == "gelu":
        cdf = 0.5 * torch.special.erfc(-z / 2**0.5)
        return z * cdf, cdf + z * torch.exp(-z.square() / 2) / (2 * torch.pi) ** 0.5
    if name == "gelu_tanh":
        u = (2 / torch.pi) ** 0.5 * (z + 0.044715 * z**3)
        p = 1 / (1 + torch.exp(-2 * u))  # (1 + tanh u) / 2
        return z * p, p + 2 * z * p * (1 - p) * (2 / torch.pi) ** 0.5 * (1 + 0.134145 * z**2)
    if name == "silu":
        p = 1 / (1 + torch.exp(-z))
        return z * p, p + z * p * (1 - p)
    return z, torch.ones_like(z)


def _exact_forward(name, z):
    if name.endswith("glu"):
        f = z.size(1) // 2
        return _exact_act("silu" if name == "swiglu" else "gelu", z[:, :f])[0] * z[:, f:]
    return _exact_act(name, z)[0]


def _exact_backward(name, z, g):
    if z is None:
        return g
    if name.endswith("glu"):
        f = z.size(1) // 2
        value, slope = _exact_act("silu" if name == "swiglu" else "gelu", z[:, :f])
        return torch.cat((g * z[:, f:] * slope, g * value), 1)
    return g * _exact_act(name, z)[1]


def _exact_operand(codes, scales, fmt):
    if fmt not in SCALE_BLOCK:
        return codes.double()
    if fmt == "mxfp8":
        return (codes.double().unflatten(1, (-1, 32)) * torch.pow(2.0, scales.double() - 127)[..., None]).flatten(1)
    raw = codes.view(torch.uint8).int()
    both = torch.stack((raw % 16, raw // 16), 2).flatten(1)
    e, f = both // 2 % 4, (both % 2).double()
    value = torch.where(e > 0, (1 + f / 2) * 2.0 ** (e.double() - 1), f / 2) * (1 - 2 * (both // 8)).double()
    return (value.unflatten(1, (-1, 16)) * scales.double()[..., None]).flatten(1)


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "linear":
        z = _exact_operand(s["a"], s.get("raw_sfa"), c["fmt"]).matmul(_exact_operand(s["b"], s.get("raw_sfb"), c["fmt"]).t())
        z = z * (1.0 if s["alpha"] is None else s["alpha"]) + (0.0 if s["bias"] is None else s["bias"].double())
        y = _exact_forward(c["activation"], z) + (0.0 if s["residual"] is None else s["residual"].double())
        return {"c": y, **({"z": z} if c["save"] else {})}
    if c["op"] == "linear_backward":
        dz = _exact_backward(c["activation"], None if s["z"] is None else s["z"].double(), s["grad"].double())
        return {"a": dz.matmul(s["b"].double()), "b": dz.t().matmul(s["a"].double()), **({"bias": dz.t().sum(1)} if c["bias"] else {})}
    if c["op"] == "route":
        x = s["logits"].double()
        p = torch.softmax(x, 1) if c["scores"] == "softmax" else torch.special.expit(x)
        p = torch.nan_to_num(p, nan=0.0).masked_fill(x.isinf(), 0.0).requires_grad_()
        score = (p.detach() + (0.0 if s["bias"] is None else s["bias"].double())).masked_fill(x.isinf(), -torch.inf)
        n, each = c["groups"], c["experts"] // c["groups"]
        group = score.unflatten(1, (n, each)).topk(min(c["group_top"], each), 2).values.sum(2)
        kept = group >= group.topk(c["top_groups"], 1).values[:, -1:]
        score = score.masked_fill(~kept.repeat_interleave(each, 1), -torch.inf)
        _, at = score.sort(dim=1, descending=True, stable=True)
        at = at[:, : c["top_k"]]
        here = ~score.gather(1, at).isinf()
        w = p.gather(1, at) * here
        if c["renormalise"]:
            total = w.sum(1, keepdim=True)
            w = w / torch.where(total > 0, total, 1.0)
        w = w * c["scale"]
        r = {"weights": w.detach(), "indices": None}
        if c["backward"]:
            dp, = torch.autograd.grad((w * s["grad"].double()).sum(), p)
            q = p.detach()
            r["logits"] = q * (dp - (q * dp).sum(1, keepdim=True)) if c["scores"] == "softmax" else dp * q * (1 - q)
        return r
    k, top = s["x"].size(1), c["top_k"]
    chosen = s["indices"].long()
    flat = chosen.flatten()
    start = 0
    if c["op"] == "experts":
        y = s["residual"].double()
        for e in range(c["experts"]):
            pair = (flat == e).nonzero().flatten()
            h = _exact_forward(c["activation"], s["x"][pair // top].double().matmul(s["w1"][e].double().t()))
            y.index_add_(0, pair // top, h.matmul(s["w2"][e].double().t()) * s["weights"].flatten()[pair].double()[:, None])
        return {"y": y, "offsets": None, "positions": None}
    if c["op"] == "product":
        z = torch.zeros((flat.numel(), c["n"]), dtype=torch.float64, device="cuda")
        for e in range(c["experts"]):
            pair = (flat == e).nonzero().flatten()
            z[start : start + pair.numel()] = s["x"][pair // top].double().matmul(s["w"][e].double().t()) * (1.0 if s["alpha"] is None else s["alpha"][e].double())
            start += pair.numel()
        return {"y": _exact_forward(c["activation"], z), **({"z": z} if c["save"] else {})}
    dx = torch.zeros((c["tokens"], k), dtype=torch.float64, device="cuda")
    dw = torch.zeros(s["w"].shape, dtype=torch.float64, device="cuda")
    for e in range(c["experts"]):
        pair = (flat == e).nonzero().flatten()
        rows = slice(start, start + pair.numel())
        dz = _exact_backward(c["activation"], None if s["z"] is None else s["z"][rows].double(), s["grad"][rows].double())
        dx.index_add_(0, pair // top, dz.matmul(s["w"][e].double()))
        dw[e] = dz.t().matmul(s["x"][pair // top].double())
        start += pair.numel()
    return {"x": dx, "w": dw}
