"""The operators on 4-bit weights with a scale and a bias for each group of columns, as they are measured.

A weight is w[r, c] = code[r, c] * scale[r, c // group] + bias[r, c // group], with codes of 4 bits (0 .. 15), eight
of them in a 32-bit word (weight 8 j + i in bits 4 i of word j) and float16 scales and biases:

    quantize    floats to codes, scales and biases, and back to the floats that they stand for
    linear      y = x W^T for one to many tokens (a layer, an output head, a draft head's projections)
    moe         a whole mixture-of-experts block for a few tokens: router, choice, softmax over the chosen, the
                experts' SwiGLU feed-forwards, the gated shared expert, the weighted sum

With `own` false `run` computes them from elementary torch operations in 32 bits; with `own` true it calls
strata_mlx_b200.
"""

import math

import torch

own = False

_TYPES = {"f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # a draft head's expert matrix made 4-bit when its float16 file is loaded
        {"name": "quantize_640x2560_f16", "op": "quantize", "rows": 640, "cols": 2560, "group": 64, "dtype": "f16"},
        # a stack of experts in float32, the finest groups
        {"name": "quantize_stack_f32", "op": "quantize", "rows": 16 * 1536, "cols": 4096, "group": 32, "dtype": "f32"},
        # the smallest call: one token through one small projection, where latency counts
        {"name": "linear_1x640x2560", "op": "linear", "tokens": 1, "rows": 640, "cols": 2560, "group": 64, "dtype": "f16"},
        # one token through a shared expert's projection
        {"name": "linear_1x4096x4096", "op": "linear", "tokens": 1, "rows": 4096, "cols": 4096, "group": 64, "dtype": "f16"},
        # a verify window (1 accepted and 4 drafted tokens) through an output head with an odd number of rows
        {"name": "linear_5x64007x2560", "op": "linear", "tokens": 5, "rows": 64007, "cols": 2560, "group": 128, "dtype": "f16"},
        # a decode batch in float32
        {"name": "linear_24x1536x4096_f32", "op": "linear", "tokens": 24, "rows": 1536, "cols": 4096, "group": 32, "dtype": "f32"},
        # a prompt's chunk through the shared expert's projection
        {"name": "linear_1180x4096x4096", "op": "linear", "tokens": 1180, "rows": 4096, "cols": 4096, "group": 64, "dtype": "f16"},
        # a decode step of a model with many small experts
        {"name": "moe_1_e512", "op": "moe", "tokens": 1, "experts": 512, "top_k": 10, "hidden": 2560, "ffn": 640,
         "shared": 640, "group": 64, "dtype": "f16"},
        # a decode step of a layer of larger experts beside a wide shared expert
        {"name": "moe_1_e256", "op": "moe", "tokens": 1, "experts": 256, "top_k": 8, "hidden": 4096, "ffn": 1536,
         "shared": 4096, "group": 64, "dtype": "f16"},
        # the verify window of the same layer
        {"name": "moe_5_e256", "op": "moe", "tokens": 5, "experts": 256, "top_k": 8, "hidden": 4096, "ffn": 1536,
         "shared": 4096, "group": 64, "dtype": "f16"},
        # a decode batch: most experts chosen, several tokens in some of them
        {"name": "moe_32_e512", "op": "moe", "tokens": 32, "experts": 512, "top_k": 10, "hidden": 2560, "ffn": 640,
         "shared": 640, "group": 128, "dtype": "f16"},
        # a small float32 layer with odd widths
        {"name": "moe_3_e24_f32", "op": "moe", "tokens": 3, "experts": 24, "top_k": 4, "hidden": 1056, "ffn": 352,
         "shared": 544, "group": 32, "dtype": "f32"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["quantize", "linear", "linear", "moe", "moe"])
    group = rng.choice([32, 64, 128])
    dtype = rng.choice(["f16", "f16", "f32"])
    if op == "quantize":
        cols = group * _log_int(rng, 1, 8192 // group)
        rows = _log_int(rng, 1, min(40000, 16 * 1536 * 4096 // cols))
        return {"op": op, "rows": rows, "cols": cols, "group": group, "dtype": dtype}
    if op == "linear":
        tokens = _log_int(rng, 1, 1180)
        cols = group * _log_int(rng, 2, 8192 // group)
        most = min(1180 * 4096 * 4096 // (tokens * cols), 64007 * 2560 // cols)
        if dtype == "f32":
            most = min(most, max(64, 24 * 1536 * 4096 // (tokens * cols)))
        return {"op": op, "tokens": tokens, "rows": _log_int(rng, 16, max(16, most)), "cols": cols, "group": group, "dtype": dtype}
    experts = _log_int(rng, 4, 512)
    top_k = rng.randint(1, min(experts, 12))
    hidden = group * _log_int(rng, max(1, 256 // group), 4096 // group)
    ffn = group * _log_int(rng, max(1, 128 // group), 2048 // group)
    shared = group * _log_int(rng, max(1, 128 // group), 4096 // group)
    while experts * ffn * hidden > 256 * 1536 * 4096:
        experts = max(top_k, experts // 2)
        ffn = max(group, ffn // 2 // group * group)
    most = max(1, min(64, 40 * 1536 * 4096 // (top_k * ffn * hidden)))
    if dtype == "f32":
        most = min(most, 16)
    return {"op": op, "tokens": _log_int(rng, 1, most), "experts": experts, "top_k": top_k, "hidden": hidden, "ffn": ffn,
            "shared": shared, "group": group, "dtype": dtype}


# ---- inputs


def _weights(gen, lead, rows, cols, group, std):
    """Codes (..., rows, cols / 8) of bell-shaped values, float16 scales and biases: weights of about `std`."""
    a = torch.randint(-(2**31), 2**31, (*lead, rows, cols // 8), dtype=torch.int32, device="cuda", generator=gen)
    b = torch.randint(-(2**31), 2**31, a.shape, dtype=torch.int32, device="cuda", generator=gen)
    codes = (a & b) + (((a ^ b) >> 1) & 0x77777777)  # the mean of two uniform codes, nibble by nibble
    del a, b
    shape = (*lead, rows, cols // group)
    scales = (std / 3.3) * (0.5 + torch.rand(shape, device="cuda", generator=gen))
    biases = -7.25 * scales * (1 + 0.1 * torch.randn(shape, device="cuda", generator=gen))
    return codes, scales.to(torch.float16), biases.to(torch.float16)


def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype, group = _TYPES[case["dtype"]], case["group"]
    if case["op"] == "quantize":
        return {"w": (0.02 * torch.randn(case["rows"], case["cols"], device="cuda", generator=gen)).to(dtype)}
    if case["op"] == "linear":
        return {"x": torch.randn(case["tokens"], case["cols"], device="cuda", generator=gen).to(dtype),
                "w": _weights(gen, (), case["rows"], case["cols"], group, case["cols"] ** -0.5)}
    e, h, f, s = case["experts"], case["hidden"], case["ffn"], case["shared"]
    return {"x": torch.randn(case["tokens"], h, device="cuda", generator=gen).to(dtype),
            "router": (h**-0.5 * torch.randn(e, h, device="cuda", generator=gen)).to(torch.float16),
            "shared_gate": (h**-0.5 * torch.randn(1, h, device="cuda", generator=gen)).to(torch.float16),
            "gate": _weights(gen, (e,), f, h, group, h**-0.5), "up": _weights(gen, (e,), f, h, group, h**-0.5),
            "down": _weights(gen, (e,), h, f, group, f**-0.5), "sgate": _weights(gen, (), s, h, group, h**-0.5),
            "sup": _weights(gen, (), s, h, group, h**-0.5), "sdown": _weights(gen, (), h, s, group, s**-0.5)}


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if own:
        # the layer that a user's program holds (for a decode step captured once, as it keeps it); the floats' codes
        # are not needed any more once the layer has them
        from strata_mlx_b200 import affine, fused

        group = case["group"]
        if case["op"] == "linear":
            state["layer"] = affine.QuantizedLinear(*state.pop("w"), group_size=group)
        elif case["op"] == "moe":
            glu = affine.QuantizedSwitchGLU(*(affine.QuantizedSwitchLinear(*state.pop(n), group_size=group)
                                              for n in ("gate", "up", "down")))
            mlp = affine.QuantizedMLP(*(affine.QuantizedLinear(*state.pop(n), group_size=group)
                                        for n in ("sgate", "sup", "sdown")))
            block = fused.SparseMoeBlock(state.pop("router"), glu, mlp, state.pop("shared_gate"), case["top_k"])
            state["step"] = fused.GraphedBlock(block, case["tokens"], case["hidden"], _TYPES[case["dtype"]])
    return state


# ---- the calls


def run(state):
    if own:
        return _own(state)
    case = state["case"]
    if case["op"] == "quantize":
        return _quantize(state["w"], case["group"])
    if case["op"] == "linear":
        return _linear(state["x"].float(), _floats(*state["w"])).to(state["x"].dtype)
    return _moe(state, case["top_k"])


def _own(state):
    case = state["case"]
    if case["op"] == "quantize":
        from strata_mlx_b200 import affine

        codes, scales, biases = affine.quantize(state["w"], case["group"])
        return {"values": affine.dequantize(codes, scales, biases, case["group"], dtype=torch.float32), "scales": scales,
                "biases": biases}
    if case["op"] == "linear":
        return state["layer"](state["x"])
    return state["step"](state["x"])


# ---- the plain forms


def _quantize(w, group):
    """scale = (max - min) / 15 and bias = min of each group, both rounded to float16; code = the nearest of 0 .. 15 to
    (w - bias) / scale (0 where the scale is 0)."""
    g = w.float().reshape(w.shape[0], -1, group)
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    # (by a tensor of fifteens: a tensor over a Python number is multiplied by the number's rounded reciprocal)
    scales, biases = ((hi - lo) / torch.full_like(hi, 15)).to(torch.float16), lo.to(torch.float16)
    s, b = scales.float(), biases.float()
    q = torch.where(s > 0, ((g - b) / s).round().clamp(0, 15), torch.zeros_like(g))
    return {"values": (q * s + b).reshape(w.shape), "scales": scales.squeeze(-1), "biases": biases.squeeze(-1)}


def _floats(codes, scales, biases):
    """The weights in float32: (..., rows, cols)."""
    shifts = torch.arange(0, 32, 4, dtype=torch.int32, device=codes.device)
    q = ((codes.unsqueeze(-1) >> shifts) & 15).float()
    q = q.reshape(*scales.shape, -1)
    return (q * scales.float().unsqueeze(-1) + biases.float().unsqueeze(-1)).flatten(-2)


def _linear(x, w):
    return x @ w.transpose(-1, -2)


def _silu(x):
    return x / (1 + torch.exp(-x))


def _moe(state, k):
    x = state["x"].float()
    # (the choice goes by values that may lie close together: their sums in 64 bits)
    logits = _linear(x.double(), state["router"].double())
    order = torch.argsort(logits, dim=-1, descending=True, stable=True)[:, :k]
    w = torch.softmax(torch.gather(logits, 1, order), -1).float()
    gate, up, down = (_floats(*(t[order] for t in state[n])) for n in ("gate", "up", "down"))  # (tokens, k, out, in)
    xk = x[:, None, None, :]
    h = _silu(_linear(xk, gate)) * _linear(xk, up)  # (tokens, k, 1, ffn)
    y = (_linear(h, down).squeeze(2) * w[:, :, None]).sum(1)
    sgate, sup, sdown = (_floats(*state[n]) for n in ("sgate", "sup", "sdown"))
    shared = _linear(_silu(_linear(x, sgate)) * _linear(x, sup), sdown)
    g = 1 / (1 + torch.exp(-_linear(x, state["shared_gate"].float())))
    return (y + g * shared).to(state["x"].dtype)


# ---- what a pass cannot do without


def work(case):
    item = 2 if case["dtype"] == "f16" else 4
    per = 0.5 + 4 / case["group"]  # bytes of a weight with its share of scale and bias
    if case["op"] == "quantize":
        n = case["rows"] * case["cols"]
        # read the floats once, write codes, scales and biases, write the floats they stand for
        return {"bytes": int(n * (item + per + 4)), "flops": 6 * n}
    t = case["tokens"]
    if case["op"] == "linear":
        n = case["rows"] * case["cols"]
        return {"bytes": int(n * per + t * (case["rows"] + case["cols"]) * item), "flops": 2 * t * n}
    e, k, h, f, s = case["experts"], case["top_k"], case["hidden"], case["ffn"], case["shared"]
    chosen = e * (1 - (1 - k / e) ** t)  # distinct experts of t tokens that choose evenly
    return {"bytes": int(3 * h * (chosen * f + s) * per + (e + 1) * h * 2 + 2 * t * h * item),
            "flops": int(2 * t * h * (3 * k * f + 3 * s + e + 1))}


# ---- the definition in 64 bits


def _exact_weights(codes, scales, biases):
    pairs = codes.contiguous().view(torch.uint8)  # byte j of a row: weight 2 j in the low bits, 2 j + 1 in the high ones
    w = torch.stack((pairs % 16, pairs // 16), -1).flatten(-2).to(torch.float64)
    each = w.shape[-1] // scales.shape[-1]
    return torch.addcmul(biases.double().repeat_interleave(each, -1), w, scales.double().repeat_interleave(each, -1))


def exact(case, seed):
    data = _inputs(case, seed)
    if case["op"] == "quantize":
        g = data["w"].double().unflatten(-1, (-1, case["group"]))
        least = g.min(-1).values
        # (which code a value on the border between two takes is the float32 quotient's choice: no value in 64 bits)
        return {"values": None, "scales": (g.max(-1).values - least) / 15.0, "biases": least}
    x = data["x"].double()
    if case["op"] == "linear":
        return torch.einsum("tc,rc->tr", x, _exact_weights(*data["w"]))
    logits = torch.einsum("th,eh->te", x, data["router"].double())
    top = torch.topk(logits, case["top_k"], dim=-1)
    share = torch.exp(top.values - torch.logsumexp(top.values, -1, keepdim=True))
    chosen = {n: tuple(t[: case["experts"]] for t in data[n]) for n in ("gate", "up", "down")}
    out = torch.zeros_like(x)
    for e in torch.unique(top.indices).tolist():
        token, place = torch.nonzero(top.indices == e, as_tuple=True)
        g, u, d = (_exact_weights(*(t[e] for t in chosen[n])) for n in ("gate", "up", "down"))
        a, b = x[token] @ g.mT, x[token] @ u.mT
        out.index_add_(0, token, share[token, place, None] * ((a * torch.sigmoid(a) * b) @ d.mT))
    g, u, d = (_exact_weights(*data[n]) for n in ("sgate", "sup", "sdown"))
    a, b = x @ g.mT, x @ u.mT
    return out + torch.sigmoid(x @ data["shared_gate"].double().mT) * ((a * torch.sigmoid(a) * b) @ d.mT)
