"""Operators of the MXFP4 path beside its decode products: rounding to MXFP4 and back,
the MXFP4 linear layer, the experts of a mixture over a prompt, and the router that
chooses them. Each case is one call as a program that serves such a model makes it, through
`linnet_amd.torch.kernels` and `linnet_amd.torch.quantized`; beside it stands the same in
elementary torch operations.

MXFP4 (the OCP microscaling format): 32 values share a scale 2^(s - 127), s = the exponent
of the largest magnitude less 2 (E2M1's own largest exponent), and are rounded to E2M1
(0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), ties to the even code, past 6 to 6.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]
FEW_ROWS = 32  # rows up to which the layers multiply x unrounded


def listed():
    return [
        # A decode batch's activations rounded and read back: latency.
        dict(name="round_batch", kind="round", rows=40, k=4096, dtype="bf16"),
        # A long prompt's MLP activations.
        dict(name="round_prompt", kind="round", rows=8192, k=14336, dtype="bf16"),
        # A layer's weight as a checkpoint tool rounds it, from f32.
        dict(name="round_weight", kind="round", rows=14336, k=4096, dtype="f32"),
        # One token through an attention output projection.
        dict(name="linear_one_token", kind="linear", rows=1, k=4096, n=4096, dtype="bf16", bias=False),
        # A decode batch through an up projection, with a bias.
        dict(name="linear_batch16", kind="linear", rows=16, k=4096, n=14336, dtype="f16", bias=True),
        # A short prompt through a layer of a 2880-wide model, ragged in its rows and in 128s of its inputs.
        dict(name="linear_short_prompt", kind="linear", rows=777, k=2880, n=5760, dtype="bf16", bias=True),
        # A long prompt through a wide layer.
        dict(name="linear_prompt", kind="linear", rows=4096, k=8192, n=28672, dtype="bf16", bias=False),
        # A mixture's gate|up experts for a batch of 100 tokens: about 12 pairs an expert.
        dict(name="experts_batch100", kind="experts", form="shared", rows=100, top=4, experts=32, k=2880, n=5760, dtype="bf16"),
        # The same for a prompt of 4096 tokens.
        dict(name="experts_prompt", kind="experts", form="shared", rows=4096, top=4, experts=32, k=2880, n=5760, dtype="bf16"),
        # The down experts of a prompt of 1000 tokens: every (token, choice) pair has a row of its own.
        dict(name="experts_down", kind="experts", form="pairs", rows=1000, top=4, experts=32, k=2880, n=2880, dtype="f16"),
        # One token's router of 32 experts, a softmax over the chosen four.
        dict(name="route_one_token", kind="route", rows=1, experts=32, top=4, score="softmax", bias=False, groups=1,
             group_top=1, group_best=1, renormalize=True, scale=1.0, dtype="bf16"),
        # A prompt's router of 256 experts in 8 groups, sigmoid scores with a balancing bias.
        dict(name="route_prompt", kind="route", rows=8192, experts=256, top=8, score="sigmoid", bias=True, groups=8,
             group_top=4, group_best=2, renormalize=True, scale=2.5, dtype="f32"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["round", "linear", "linear", "linear", "experts", "experts", "route", "route"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if kind == "round":
        k = 32 * _log(rng, 1, 448)
        rows = min(_log(rng, 1, 14336), (8192 * 14336) // k)
        return dict(kind="round", rows=rows, k=k, dtype=rng.choice(["bf16", "f16", "f32"]))
    if kind == "linear":
        k = 32 * _log(rng, 8, 448)
        n = _log(rng, 64, 28672)
        n = n // 64 * 64 if rng.random() < 0.6 else n
        rows = _log(rng, 1, 64) if rng.random() < 0.4 else _log(rng, 33, 4096)
        return dict(kind="linear", rows=max(1, min(rows, int(9.6e11 / k / n))), k=k, n=n, dtype=dtype, bias=rng.random() < 0.4)
    if kind == "experts":
        experts = rng.choice([8, 16, 32, 64, 128])
        k, n = 32 * _log(rng, 16, 128), _log(rng, 256, 5760)
        n = n // 32 * 32 if rng.random() < 0.7 else n
        most = 17e9 / experts / n  # experts' weights of about the listed size
        k = max(32, min(k, int(most) // 32 * 32))
        top = rng.choice([1, 2, 4, 8])
        rows = _log(rng, 33, 4096)
        rows = max(33, min(rows, int(2.7e11 / k / n / top)))
        return dict(kind="experts", form=rng.choice(["shared", "pairs"]), rows=rows, top=top, experts=experts, k=k, n=n, dtype=dtype)
    experts = rng.choice([8, 16, 32, 60, 64, 96, 128, 160, 256, 384])
    groups = rng.choice([1, 1, 4, 8]) if experts % 8 == 0 else 1
    group_top = rng.randint(1, groups)
    best = rng.choice([1, 2]) if groups > 1 and experts // groups > 1 else 1
    top = max(1, min(_log(rng, 1, 12), group_top * (experts // groups)))
    return dict(kind="route", rows=_log(rng, 1, 8192), experts=experts, top=top, score=rng.choice(["softmax", "sigmoid"]),
                bias=rng.random() < 0.6, groups=groups, group_top=group_top, group_best=best,
                renormalize=rng.random() < 0.7, scale=rng.choice([1.0, 2.5]), dtype=rng.choice(["bf16", "f16", "f32"]))


# ------------------------------------------------------------------ inputs


def _generator(seed, salt):
    return torch.Generator(device="cuda").manual_seed(1000003 * int(seed) + salt)


def _activations(g, rows, k, dtype):
    """N(0, 1) with a few larger channels, as norm outputs have."""
    x = torch.randn(rows, k, generator=g, device="cuda")
    wide = torch.randint(0, k, (max(1, k // 512),), generator=g, device="cuda")
    x[:, wide] *= 6.0
    return x.to(dtype)


def _stored(g, count, n, k):
    """`count` weights N(0, 0.02) as a checkpoint stores them: blocks [count, n, k/32, 16], scales [count, n, k/32]."""
    blocks = torch.empty(count, n, k // 32, 16, dtype=torch.uint8, device="cuda")
    scales = torch.empty(count, n, k // 32, dtype=torch.uint8, device="cuda")
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device="cuda")
    for i in range(count):
        w = torch.randn(n, k // 32, 32, generator=g, device="cuda").mul_(0.02)
        byte = ((w.abs().amax(-1).view(torch.int32) >> 23) - 2).clamp(min=1)
        w = w * ((254 - byte) << 23).view(torch.float32)[..., None]
        q = torch.bucketize(w.abs(), edges).to(torch.uint8) | ((w < 0).to(torch.uint8) << 3)
        blocks[i] = q[..., 0::2] | (q[..., 1::2] << 4)
        scales[i] = byte.to(torch.uint8)
    return blocks, scales


def _round_inputs(case, seed):
    g = _generator(seed, 1)
    if case["dtype"] == "f32":
        return torch.randn(case["rows"], case["k"], generator=g, device="cuda").mul_(0.02)
    return _activations(g, case["rows"], case["k"], DTYPES[case["dtype"]])


def _linear_inputs(case, seed):
    g = _generator(seed, 2)
    dtype = DTYPES[case["dtype"]]
    blocks, scales = _stored(g, 1, case["n"], case["k"])
    bias = torch.randn(case["n"], generator=g, device="cuda").to(dtype) if case["bias"] else None
    return _activations(g, case["rows"], case["k"], dtype), blocks[0], scales[0], bias


def _experts_inputs(case, seed):
    g = _generator(seed, 3)
    rows, top, count, k = case["rows"], case["top"], case["experts"], case["k"]
    blocks, scales = _stored(g, count, case["n"], k)
    # A router's choice: some experts are chosen more often than others.
    logits = torch.randn(rows, count, generator=g, device="cuda") + 0.5 * torch.randn(count, generator=g, device="cuda")
    experts = logits.topk(top, dim=-1).indices
    shared = case["form"] == "shared"
    x = _activations(g, rows if shared else rows * top, k, DTYPES[case["dtype"]])
    return x if shared else x.view(rows, top, k), blocks, scales, experts


def _route_inputs(case, seed):
    g = _generator(seed, 4)
    rows, count = case["rows"], case["experts"]
    logits = (torch.randn(rows, count, generator=g, device="cuda") + 0.5 * torch.randn(count, generator=g, device="cuda"))
    bias = torch.randn(count, generator=g, device="cuda").mul_(0.05) if case["bias"] else None
    return logits.to(DTYPES[case["dtype"]]), bias


def prepare(case, seed):
    kind = case["kind"]
    if kind == "round":
        return dict(kind=kind, x=_round_inputs(case, seed))
    if kind == "route":
        logits, bias = _route_inputs(case, seed)
        return dict(kind=kind, logits=logits, bias=bias, case=case)
    if kind == "linear":
        x, blocks, scales, bias = _linear_inputs(case, seed)
        state = dict(kind=kind, x=x, blocks=blocks, scales=scales, bias=bias)
    else:
        x, blocks, scales, experts = _experts_inputs(case, seed)
        state = dict(kind=kind, x=x, blocks=blocks, scales=scales, experts=experts)
    if own:
        # The layer's operands, which a program makes once as it loads the weights.
        from linnet_amd.torch import quantized

        make = quantized.mxfp4_operands if kind == "linear" else quantized.mxfp4_experts_operands
        state["operands"] = make(blocks, scales, 1)
    return state


# ------------------------------------------------------------------ the plain form


def _power(byte):
    """2^(byte - 127) for bytes 1 .. 254."""
    return (byte << 23).view(torch.float32)


def _round_plain(x):
    """x's values rounded to MXFP4, in 32 bits (every step but the rounding is exact)."""
    v = x.float().unflatten(-1, (-1, 32))
    byte = ((v.abs().amax(-1, keepdim=True).view(torch.int32) >> 23) - 2).clamp(min=1)
    v = v * _power(254 - byte)
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = (torch.round(a / step) * step).clamp(max=6.0)
    return (torch.copysign(a, v) * _power(byte)).flatten(-2)


def _weight_plain(blocks, scales):
    codes = torch.stack([blocks & 15, blocks >> 4], dim=-1).flatten(-2)
    values = torch.tensor(E2M1, device=blocks.device)[codes.int()]
    return (values * _power(scales.int())[..., None]).flatten(-2)


def _linear_plain(x, blocks, scales, bias):
    v = _round_plain(x) if x.shape[0] > FEW_ROWS else x.float()
    y = v @ _weight_plain(blocks, scales).t()
    return (y if bias is None else y + bias.float()).to(x.dtype)


def _experts_plain(x, blocks, scales, experts):
    """The (row, choice) pairs sorted by expert into [experts, most pairs of one, k], one batched product, and back."""
    rows, top = experts.shape
    count = blocks.shape[0]
    ids = experts.flatten()
    order = torch.argsort(ids, stable=True)
    numbers = torch.bincount(ids, minlength=count)
    place = torch.arange(rows * top, device=x.device) - (numbers.cumsum(0) - numbers)[ids[order]]
    v = _round_plain(x) if rows > FEW_ROWS else x.float()
    v = v[order // top] if x.dim() == 2 else v.flatten(0, 1)[order]
    grouped = torch.zeros(count, int(numbers.max()), x.shape[-1], device=x.device)
    grouped[ids[order], place] = v
    y = torch.bmm(grouped, _weight_plain(blocks, scales).transpose(1, 2).contiguous())
    out = torch.empty(rows * top, y.shape[-1], device=x.device)
    out[order] = y[ids[order], place]
    return out.view(rows, top, -1).to(x.dtype)


def _route_plain(logits, bias, case):
    """Scores in 64 bits: a choice between two experts next to each other goes by their last bits."""
    v = logits.double()
    if case["score"] == "softmax":
        p = torch.exp(v - v.amax(-1, keepdim=True))
        s = p / p.sum(-1, keepdim=True)
    else:
        s = 1 / (1 + torch.exp(-v))
    c = s if bias is None else s + bias.double()
    if case["groups"] > 1:
        g = c.unflatten(-1, (case["groups"], -1))
        best = torch.sort(g, dim=-1, descending=True, stable=True).values[..., : case["group_best"]].sum(-1)
        kept = torch.sort(best, dim=-1, descending=True, stable=True).indices[..., : case["group_top"]]
        keep = torch.zeros_like(best, dtype=torch.bool).scatter(-1, kept, True)
        c = torch.where(keep[..., None], g, -torch.inf).flatten(-2)
    experts = torch.sort(c, dim=-1, descending=True, stable=True).indices[..., : case["top"]]
    w = s.gather(-1, experts)
    if case["renormalize"]:
        w = w / w.sum(-1, keepdim=True)
    return dict(experts=experts, weights=(w * case["scale"]).float())


# ------------------------------------------------------------------ a pass


def run(state):
    kind = state["kind"]
    if own:
        from linnet_amd.torch import kernels, quantized

        if kind == "round":
            blocks, scales = kernels.mxfp4_quantize(state["x"])
            return kernels.mxfp4_dequantize(blocks, scales, state["x"].dtype)
        if kind == "linear":
            return quantized.mxfp4_linear(state["x"], state["operands"], state["bias"])
        if kind == "experts":
            return quantized.mxfp4_experts_linear(state["x"], state["operands"], state["experts"])
        case = state["case"]
        experts, weights = kernels.expert_route(
            state["logits"], case["top"], bias=state["bias"], score=case["score"], groups=case["groups"],
            group_top=case["group_top"], group_best=case["group_best"], renormalize=case["renormalize"], scale=case["scale"])
        return dict(experts=experts, weights=weights)
    if kind == "round":
        return _round_plain(state["x"]).to(state["x"].dtype)
    if kind == "linear":
        return _linear_plain(state["x"], state["blocks"], state["scales"], state["bias"])
    if kind == "experts":
        return _experts_plain(state["x"], state["blocks"], state["scales"], state["experts"])
    return _route_plain(state["logits"], state["bias"], state["case"])


def work(case):
    kind, rows = case["kind"], case["rows"]
    if kind == "route":
        size = 4 if case["dtype"] == "f32" else 2
        return {"bytes": rows * (case["experts"] * size + case["top"] * 12) + (4 * case["experts"] if case["bias"] else 0),
                "flops": rows * case["experts"] * 4}
    k = case["k"]
    if kind == "round":
        size = 4 if case["dtype"] == "f32" else 2
        return {"bytes": rows * k * (2 * size + 2 * 17 / 32), "flops": rows * k * 4}
    n = case["n"]
    if kind == "linear":
        return {"bytes": n * k * 17 / 32 + rows * (k + n) * 2 + (2 * n if case["bias"] else 0), "flops": 2 * rows * n * k}
    pairs = rows * case["top"]
    named = case["experts"] * (1 - (1 - case["top"] / case["experts"]) ** rows)
    x = rows if case["form"] == "shared" else pairs
    return {"bytes": named * n * k * 17 / 32 + (x * k + pairs * n) * 2 + pairs * 8, "flops": 2 * pairs * n * k}


# ------------------------------------------------------------------ the same in 64 bits


def _nearest(x):
    """x rounded to MXFP4 in 64 bits, by counting the midpoints below each magnitude; a midpoint itself goes to the
    even of its two codes, so every second one counts where it is met."""
    v = x.double().unflatten(-1, (-1, 32))
    top = v.abs().amax(-1, keepdim=True)
    unit = torch.exp2((torch.frexp(top).exponent - 3).clamp(min=-127).double())
    a = v.abs() / unit
    code = torch.zeros_like(a, dtype=torch.int64)
    for i, middle in enumerate([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]):
        code += (a >= middle) if i % 2 else (a > middle)
    values = torch.tensor(E2M1[:8], dtype=torch.float64, device=x.device)
    return (values[code] * v.sign() * unit).flatten(-2)


def _weight64(blocks, scales):
    values = torch.tensor(E2M1, dtype=torch.float64, device=blocks.device)
    pairs = torch.stack([values[(blocks & 15).int()], values[(blocks >> 4).int()]], dim=-1)
    return (pairs.flatten(-2) * torch.exp2(scales.double() - 127)[..., None]).flatten(-2)


def _route64(logits, bias, case):
    v = logits.double()
    s = torch.softmax(v, -1) if case["score"] == "softmax" else torch.sigmoid(v)
    c = s.clone() if bias is None else s + bias.double()
    rows, count = c.shape
    at = torch.arange(rows, device=c.device)
    if case["groups"] > 1:
        size = count // case["groups"]
        g = c.view(rows, case["groups"], size)
        total = g.amax(-1)
        if case["group_best"] == 2:
            g = g.scatter(-1, g.argmax(-1, keepdim=True), -math.inf)
            total = total + g.amax(-1)
        keep = torch.zeros_like(c, dtype=torch.bool)
        for _ in range(case["group_top"]):
            first = (total == total.amax(-1, keepdim=True)).int().argmax(-1)
            keep.view(rows, case["groups"], size)[at, first] = True
            total[at, first] = -math.inf
        c[~keep] = -math.inf
    weights = torch.empty(rows, case["top"], dtype=torch.float64, device=c.device)
    for i in range(case["top"]):
        first = (c == c.amax(-1, keepdim=True)).int().argmax(-1)
        weights[:, i] = s[at, first]
        c[at, first] = -math.inf
    if case["renormalize"]:
        weights = weights / weights.sum(-1, keepdim=True)
    return dict(experts=None, weights=weights * case["scale"])


def exact(case, seed):
    kind = case["kind"]
    if kind == "round":
        return _nearest(_round_inputs(case, seed))
    if kind == "route":
        logits, bias = _route_inputs(case, seed)
        return _route64(logits, bias, case)
    if kind == "linear":
        x, blocks, scales, bias = _linear_inputs(case, seed)
        y = (_nearest(x) if case["rows"] > FEW_ROWS else x.double()) @ _weight64(blocks, scales).t()
        return y if bias is None else y + bias.double()
    x, blocks, scales, experts = _experts_inputs(case, seed)
    rows, top = experts.shape
    v = _nearest(x) if rows > FEW_ROWS else x.double()
    y = torch.zeros(rows, top, case["n"], dtype=torch.float64, device=x.device)
    for e in range(case["experts"]):
        r, j = (experts == e).nonzero(as_tuple=True)
        if r.numel():
            y[r, j] = (v[r] if x.dim() == 2 else v[r, j]) @ _weight64(blocks[e], scales[e]).t()
    return y
