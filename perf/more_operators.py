"""Cases of the operators that close the feed-forward half of a transformer layer, dense or by experts: routing to experts with the
plan that the grouped linears read, the weighted return of the experts' rows to their tokens, the norms around a block with gate,
residual scale and modulation, and the linear with activation and residual in its epilogue.

`own` false: the operators in their plain form, elementary torch operations in 32 bits (routing decides in 64 bits, where two scores
may lie next to each other).  `own` true: the calls of `ac4k_kernel_amd.ops`.  Sizes are those of this repository's benchmark and tests
(widths of 4096, 5120, 8192 and 14336, decode, 8192-token prefill, the 75600-token tensors, ragged relatives of them)."""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZES = {"none": 0, "bf16": 2, "fp16": 2, "fp32": 4}
_NVFP4_MAX = 448.0 * 6.0
_EPS = 1e-6


# ---------------------------------------------------------------------------------------------------------------- cases
def _route(tokens, experts, topk, **kw):
    """scoring of all experts of a token, groups of them by their `best` highest keys; the last `padding` of the tokens have no expert."""
    return dict({"op": "route", "tokens": tokens, "experts": experts, "topk": topk, "scoring": "softmax", "bias": False, "groups": 1,
                 "top_groups": 1, "best": 1, "renormalize": True, "scale": 1.0, "dtype": "bf16", "padding": 0.0}, **kw)


def _combine(tokens, topk, cols, **kw):
    """Rows of the experts in their order back to tokens; `dropped`: share of the tokens without an expert."""
    return dict({"op": "combine", "tokens": tokens, "topk": topk, "cols": cols, "dtype": "bf16", "residual": False, "dropped": 0.0}, **kw)


def _norm(batch, tokens, cols, precision, **kw):
    """Norm of residual_scale * residual + gate * (norm of) y, modulated.  gate: none, vector (one for all tokens) or batch."""
    return dict({"op": "block_norm", "batch": batch, "tokens": tokens, "cols": cols, "precision": precision, "kind": "rms", "dtype": "bf16",
                 "weights": "bf16", "weight": True, "residual": True, "post": False, "gate": "none", "alpha": 1.0, "modulate": False}, **kw)


def _linear(m, n, k, **kw):
    return dict({"op": "linear", "m": m, "n": n, "k": k, "activation": "none", "bias": "bf16", "residual": False, "out": "bf16"}, **kw)


def listed():
    return [
        # decode: 16 tokens choose 8 of 64 experts; launch latency counts
        dict(_route(16, 64, 8), name="route_16_e64_k8"),
        # ragged prefill behind a sigmoid router with a balancing bias and groups, logits in fp32, padding at the end
        dict(_route(4001, 256, 8, scoring="sigmoid", bias=True, groups=8, top_groups=4, best=2, scale=2.5, dtype="fp32", padding=0.05),
             name="route_4001_e256_k8_groups"),
        # prefill of 16384 tokens, 4 of 128 experts by softmax
        dict(_route(16384, 128, 4), name="route_16384_e128_k4"),
        # the same decode step on its way back
        dict(_combine(16, 8, 4096), name="combine_16x8_4096"),
        # prefill of 8192 tokens, 8 experts each, added to the residual stream
        dict(_combine(8192, 8, 4096, residual=True), name="combine_8192x8_4096"),
        # one decoded token between two blocks that norm their output as well, 8-bit output with its scale
        dict(_norm(1, 1, 8192, "fp8e4m3", post=True), name="norm_fp8_1x8192_post"),
        # prefill of 8192 tokens with a gate per channel, in front of an NVFP4 linear
        dict(_norm(1, 8192, 4096, "nvfp4", gate="vector", post=True), name="norm_nvfp4_8192x4096_post"),
        # ragged: two sequences, scaled residual, layer norm with int8 output and modulation in fp32
        dict(_norm(2, 2001, 5003, "int8", kind="layer", weights="fp32", weight=False, gate="batch", alpha=0.75, modulate=True),
             name="norm_int8_2x2001x5003_layer"),
        # video tokens: gated residual, layer norm without weights, shifted and scaled per sequence (the largest norm)
        dict(_norm(1, 75600, 5120, "none", kind="layer", weight=False, gate="batch", modulate=True), name="norm_bf16_75600x5120_layer"),
        # one decoded token through the first linear of a feed-forward block
        dict(_linear(1, 14336, 4096, activation="silu", bias="none"), name="linear_1x14336x4096_silu"),
        # ragged: sizes that are multiples of nothing, activation and residual, fp32 output
        dict(_linear(1001, 5003, 2880, activation="relu", bias="fp32", residual=True, out="fp32"), name="linear_1001x5003x2880_relu_residual"),
        # prefill: 8192 tokens through the first linear of a feed-forward block (the largest product)
        dict(_linear(8192, 14336, 4096, activation="gelu"), name="linear_8192x14336x4096_gelu"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi, least=1):
    """A feature dim: mostly a multiple of 128, sometimes of 64 or 8, sometimes odd."""
    w = _log_int(rng, lo, hi)
    step = max(least, rng.choice([128, 128, 128, 128, 64, 8, 1]))
    return max(lo, w // step * step)


def draw(rng):
    op = rng.choice(["route", "combine", "block_norm", "block_norm", "linear", "linear"])
    if op == "route":
        experts = rng.choice([8, 16, 60, 64, 97, 128, 160, 256, 384, 512])
        groups = rng.choice([1, 1] + [g for g in (2, 4, 8) if experts % g == 0])
        top_groups = rng.randint(1, groups)
        topk = min(rng.choice([1, 2, 4, 6, 8]), experts // groups * top_groups)
        tokens = _log_int(rng, 1, min(16384, 16384 * 128 // experts))
        return _route(tokens, experts, topk, scoring=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5, groups=groups,
                      top_groups=top_groups, best=rng.choice([1, 2]), renormalize=rng.random() < 0.7, scale=rng.choice([1.0, 2.5]),
                      dtype=rng.choice(["bf16", "fp16", "fp32"]), padding=rng.choice([0.0, 0.0, 0.1]))
    if op == "combine":
        topk, cols = rng.choice([1, 2, 4, 6, 8]), _width(rng, 256, 8192)
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        tokens = _log_int(rng, 1, min(16384, 260_000_000 // (topk * cols) // (2 if dtype == "fp32" else 1)))
        return _combine(tokens, topk, cols, dtype=dtype, residual=rng.random() < 0.5, dropped=rng.choice([0.0, 0.0, 0.1]))
    if op == "block_norm":
        cols = _width(rng, 64, 16384)
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
        batch = rng.choice([1, 1, 2, 7])
        tokens = _log_int(rng, 1, min(75600, 380_000_000 // (cols * batch) // (2 if dtype == "fp32" else 1)))
        residual = rng.random() < 0.8
        return _norm(batch, tokens, cols, rng.choice(["none", "none", "nvfp4", "nvfp4", "fp8e4m3", "int8"]), kind=rng.choice(["rms", "layer"]),
                     dtype=dtype, weights=rng.choice([dtype, "fp32"]), weight=rng.random() < 0.6, residual=residual,
                     post=residual and rng.random() < 0.4, gate=rng.choice(["none", "vector", "batch"]) if residual else "none",
                     alpha=rng.choice([1.0, 1.0, 0.75]) if residual else 1.0, modulate=rng.random() < 0.5)
    k = _width(rng, 256, 14336, 64)
    n = _width(rng, 256, 14336)
    m = _log_int(rng, 1, min(16384, 480_000_000_000 // (n * k)))
    return _linear(m, n, k, activation=rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]), bias=rng.choice(["none", "bf16", "fp32"]),
                   residual=rng.random() < 0.5, out=rng.choice(["bf16", "bf16", "fp16", "fp32"]))


# --------------------------------------------------------------------------------------------------------------- inputs
def _up(a, b):
    return (a + b - 1) // b * b


def _normal(shape, gen, std=1.0):
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0.0, std, generator=gen)


def _activation(shape, gen):
    """N(0, 1) with 0.1 % outliers of twenty times the size, as transformer activations have."""
    x = _normal(shape, gen)
    mask = torch.empty(shape, dtype=torch.float32, device="cuda").uniform_(generator=gen) < 1e-3
    return torch.where(mask, x * 20.0, x)


def _packed(codes):
    """e2m1 values [.., K] -> bytes [.., K/2], the even element in the low nibble."""
    a = codes.abs()
    index = (2 * a - (a > 2) * (a - 2) - (a > 4).to(a.dtype)).to(torch.uint8)  # 0 .. 4 are halves, 3 is 5, 4 is 6, 6 is 7
    index = index | (torch.signbit(codes).to(torch.uint8) << 3)
    return index[..., 0::2] | (index[..., 1::2] << 4)


def _scale_layout(sf, rows):
    """e4m3 scales [R, K/16] -> [K/64, R up to 16, 4], zeros behind the last row."""
    sf = torch.nn.functional.pad(sf.float(), (0, 0, 0, _up(rows, 16) - rows))
    return sf.reshape(sf.shape[0], -1, 4).transpose(0, 1).contiguous().to(torch.float8_e4m3fn)


def _scores_of(tokens, experts, gen):
    """Router logits: some experts are more popular than others."""
    return _normal((tokens, experts), gen, 1.5) + _normal((experts,), gen, 0.5)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    if case["op"] == "route":
        t, e = case["tokens"], case["experts"]
        logits = _scores_of(t, e, gen)
        logits[t - int(t * case["padding"]):] = -math.inf
        state["logits"] = logits.to(_DTYPES[case["dtype"]])
        state["bias"] = _normal((e,), gen, 0.1) if case["bias"] else None
    elif case["op"] == "combine":
        t, k, n, dtype = case["tokens"], case["topk"], case["cols"], _DTYPES[case["dtype"]]
        chosen = _scores_of(t, max(64, k), gen).topk(k, dim=1)
        dropped = torch.empty((t, 1), device="cuda").uniform_(generator=gen) < case["dropped"]
        expert = torch.where(dropped, max(64, k), chosen.indices).reshape(-1)
        places = expert.sort(stable=True).indices.argsort().reshape(t, k)
        state["places"] = torch.where(dropped, -1, places).to(torch.int32)
        state["weights"] = torch.where(dropped, 0.0, chosen.values.softmax(dim=1))
        state["y"] = _activation((t * k, n), gen).to(dtype)
        state["residual"] = _normal((t, n), gen, 3.0).to(dtype) if case["residual"] else None
    elif case["op"] == "block_norm":
        b, n, k, dtype, wtype = case["batch"], case["tokens"], case["cols"], _DTYPES[case["dtype"]], _DTYPES[case["weights"]]
        state["y"] = _activation((b, n, k), gen).to(dtype)
        state["residual"] = _normal((b, n, k), gen, 3.0).to(dtype) if case["residual"] else None
        state["weight"] = (1.0 + _normal((k,), gen, 0.2)).to(wtype) if case["weight"] else None
        state["post_weight"] = (1.0 + _normal((k,), gen, 0.2)).to(wtype) if case["post"] else None
        # what a sequence's conditioning gives: shift, scale and gate of the feed-forward half, one behind the other
        condition = _normal((b, 3, k), gen, 0.5).to(wtype)
        state["shift"], state["scale"] = (condition[:, 0:1], condition[:, 1:2]) if case["modulate"] else (None, None)
        state["gate"] = {"none": None, "vector": condition[0, 2], "batch": condition[:, 2:3]}[case["gate"]]
    else:
        m, n, k = case["m"], case["n"], case["k"]
        q, state["x_sf"], state["x_gs"] = _quantized(_activation((m, k), gen).to(torch.bfloat16).float())
        state["x"] = _packed(q)
        q, state["w_sf"], state["w_gs"] = _quantized(_normal((n, k), gen, 0.02).to(torch.bfloat16).float())
        state["w"] = _packed(q)
        state["bias"] = None if case["bias"] == "none" else _normal((n,), gen, 0.5).to(_DTYPES[case["bias"]])
        state["residual"] = _normal((m, n), gen, 3.0).to(_DTYPES[case["out"]]) if case["residual"] else None
    return state


# ----------------------------------------------------------------------------------------------------------- plain form
def _round_e2m1(v):
    """To the nearest of 0, 0.5, 1, 1.5, 2, 3, 4 and 6, the even code of two, the sign kept."""
    a = v.abs()
    r = 0.5 * ((a > 0.25).to(v.dtype) + (a >= 0.75) + (a > 1.25) + (a >= 1.75)) + (a > 2.5) + (a >= 3.5) + 2.0 * (a > 5.0)
    return torch.copysign(r, v)


def _quantized(y):
    """[R, K] -> (e2m1 values [R, K up to 64], scales in their layout, scale of the whole tensor).  A maximum under 2^-100 counts as zero."""
    rows, cols = y.shape
    blocks = torch.nn.functional.pad(y, (0, _up(cols, 64) - cols)).reshape(rows, -1, 16)
    m = blocks.abs().amax(-1)
    gs = m.amax()
    gs = torch.where(gs < 2.0 ** -100, 0.0, gs) / _NVFP4_MAX
    alpha = torch.where(gs == 0, 0.0, 1.0 / gs)
    sf = (alpha * (m * float(torch.tensor(1.0 / 6.0, dtype=torch.float32)))).clamp(max=448.0).to(torch.float8_e4m3fn)
    s = sf.float()
    inverse = torch.where(s != 0, alpha * (1.0 / s), 0.0)
    return _round_e2m1(blocks * inverse.unsqueeze(-1)).reshape(rows, -1), _scale_layout(sf, rows), gs


def _plain_values(q, sf, gs):
    """e2m1 values [R, K] times the scale of their block of 16 (exact in 32 bits), then times the tensor's."""
    rows = q.shape[0]
    s = sf.float().transpose(0, 1)[:rows].reshape(rows, -1, 1)
    return (q.reshape(rows, -1, 16) * s).reshape(q.shape) * gs


def _unpacked(packed):
    values = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device="cuda")
    return values[torch.stack((packed & 15, packed >> 4), dim=-1).reshape(packed.shape[0], -1).int()]


def _plain_route(state):
    """Scores in 64 bits; a stable sort of the keys takes equal ones in the order of their index."""
    case = state["case"]
    t, e, k, g = case["tokens"], case["experts"], case["topk"], case["groups"]
    logits = state["logits"].double()
    allowed = logits > -math.inf
    if case["scoring"] == "sigmoid":
        score = 1.0 / (1.0 + torch.exp(-logits))
    else:
        p = torch.where(allowed, torch.exp(logits - logits.amax(-1, keepdim=True)), 0.0)
        score = p / p.sum(-1, keepdim=True)
    key = score if state["bias"] is None else score + state["bias"].double()
    key = torch.where(allowed, key, -math.inf)
    if g > 1:
        best = key.reshape(t, g, -1).sort(dim=-1, descending=True).values[..., :case["best"]]
        total = torch.where(best > -math.inf, best, 0.0).sum(-1)
        total = torch.where(best[..., 0] > -math.inf, total, -math.inf)
        order = total.sort(dim=-1, descending=True, stable=True).indices
        kept = torch.zeros((t, g), dtype=torch.bool, device="cuda").scatter(1, order[:, :case["top_groups"]], True)
        key = torch.where(kept.repeat_interleave(e // g, dim=1), key, -math.inf)
    top = key.sort(dim=-1, descending=True, stable=True)
    met = top.values[:, :k] > -math.inf
    expert = torch.where(met, top.indices[:, :k], -1)
    weight = torch.where(met, score.gather(1, top.indices[:, :k]), 0.0)
    if case["renormalize"]:
        total = weight.sum(-1, keepdim=True)
        weight = torch.where(total > 0, weight / total, 0.0)
    # the plan of the grouped linears: rows in the order of expert, then token
    flat = torch.where(met, expert, e).reshape(-1)
    order = flat.sort(stable=True).indices
    offsets = torch.nn.functional.pad(torch.bincount(flat, minlength=e + 1)[:e].cumsum(0), (1, 0))
    rows = torch.where(torch.arange(t * k, device="cuda") < offsets[e], order // k, -1)
    places = torch.empty_like(order).scatter(0, order, torch.arange(t * k, device="cuda")).reshape(t, k)
    places = torch.where(met, places, -1)
    return {"weights": (weight * case["scale"]).float(), "experts": expert.int(), "offsets": offsets.int(), "rows": rows.int(), "places": places.int()}


def _plain_combine(state):
    places, weights = state["places"].long(), state["weights"]
    here = places >= 0
    out = 0.0 if state["residual"] is None else state["residual"].float()
    for s in range(places.shape[1]):
        y = state["y"][places[:, s].clamp(min=0)].float()
        out = out + torch.where(here[:, s, None], y * weights[:, s, None], 0.0)
    return out.to(state["y"].dtype)


def _plain_normed(case, h):
    if case["kind"] == "layer":
        h = h - h.mean(-1, keepdim=True)
    return h * (1.0 / (h.square().mean(-1, keepdim=True) + _EPS).sqrt())


def _plain_block_norm(state):
    case = state["case"]
    h = state["y"].float()
    more = {}
    if state["residual"] is not None:
        if state["post_weight"] is not None:
            h = _plain_normed(case, h) * state["post_weight"].float()
        if state["gate"] is not None:
            h = h * state["gate"].float()
        h = (state["residual"].float() * case["alpha"] + h).to(state["y"].dtype)
        more, h = {"residual": h}, h.float()
    z = _plain_normed(case, h)
    if state["weight"] is not None:
        z = z * state["weight"].float()
    if case["modulate"]:
        z = z * (1.0 + state["scale"].float()) + state["shift"].float()
    if case["precision"] == "none":
        return {"z": z.to(state["y"].dtype), **more}
    z = z.reshape(-1, case["cols"])
    rows, cols = z.shape
    if case["precision"] == "nvfp4":
        q, sf, gs = _quantized(z)
        return {"z": _plain_values(q, sf, gs).to(torch.bfloat16), "sf": sf, "gs": gs, **more}
    most = 127.0 if case["precision"] == "int8" else 448.0
    m = z.abs().amax(-1)
    m = torch.where(m < 2.0 ** -100, 0.0, m)
    q = torch.nn.functional.pad(z * torch.where(m == 0, 0.0, most / m)[:, None], (0, _up(cols, 16) - cols)).clamp(-most, most)
    sf = torch.nn.functional.pad(m / most, (0, _up(rows, 16) - rows))
    q = (q.round() if case["precision"] == "int8" else q.to(torch.float8_e4m3fn).float())
    return {"z": (q * sf[:rows, None]).to(torch.bfloat16), "sf": sf, **more}


def _plain_activation(kind, v):
    if kind == "relu":
        return torch.where(v < 0, 0.0, v)
    if kind == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    if kind == "gelu_tanh":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    return v / (1.0 + torch.exp(-v)) if kind == "silu" else v


def _plain_linear(state):
    case = state["case"]
    y = _plain_values(_unpacked(state["x"]), state["x_sf"], state["x_gs"]) @ _plain_values(_unpacked(state["w"]), state["w_sf"], state["w_gs"]).t()
    if state["bias"] is not None:
        y = y + state["bias"].float()
    y = _plain_activation(case["activation"], y)
    if state["residual"] is not None:
        y = y + state["residual"].float()
    return y.to(_DTYPES[case["out"]])


# ------------------------------------------------------------------------------------------------------- the operators
def _own_block_norm(state, ops):
    case = state["case"]
    precision = None if case["precision"] == "none" else case["precision"]
    got = ops.block_norm(state["y"], state["residual"], state["weight"], gate=state["gate"], residual_scale=case["alpha"],
                         post_weight=state["post_weight"], scale=state["scale"], shift=state["shift"], kind=case["kind"], eps=_EPS,
                         precision=precision)
    got = got if isinstance(got, tuple) else (got,)
    more = {} if state["residual"] is None else {"residual": got[-1]}
    if precision is None:
        return {"z": got[0], **more}
    if precision == "nvfp4":
        return {"z": ops.dequantize(*got[:3]), "sf": got[1], "gs": got[2], **more}
    return {"z": ops.dequantize(*got[:2]), "sf": got[1], **more}


def run(state):
    case = state["case"]
    if own:
        from ac4k_kernel_amd import ops
        if case["op"] == "route":
            got = ops.route_experts(state["logits"], case["topk"], scoring=case["scoring"], bias=state["bias"], groups=case["groups"],
                                    top_groups=case["top_groups"], group_best=case["best"], renormalize=case["renormalize"], scale=case["scale"])
            return dict(zip(("weights", "experts", "offsets", "rows", "places"), got))
        if case["op"] == "combine":
            return ops.combine_experts(state["y"], state["weights"], state["places"], residual=state["residual"])
        if case["op"] == "block_norm":
            return _own_block_norm(state, ops)
        out = None if case["out"] == "bf16" else torch.empty((case["m"], case["n"]), dtype=_DTYPES[case["out"]], device="cuda")
        return ops.linear(state["x"], state["x_sf"], state["x_gs"], state["w"], state["w_sf"], state["w_gs"], bias=state["bias"], out=out,
                          activation=None if case["activation"] == "none" else case["activation"], residual=state["residual"])
    return {"route": _plain_route, "combine": _plain_combine, "block_norm": _plain_block_norm, "linear": _plain_linear}[case["op"]](state)


# -------------------------------------------------------------------------------------------------- what has to be done
def _nvfp4_bytes(rows, k):
    return rows * _up(k, 64) // 2 + _up(k, 64) // 16 * _up(rows, 16)


def work(case):
    if case["op"] == "route":
        t, e, k = case["tokens"], case["experts"], case["topk"]
        return {"bytes": t * e * _SIZES[case["dtype"]] + (4 * e if case["bias"] else 0) + t * k * 16 + 4 * (e + 1), "flops": 4 * t * e}
    if case["op"] == "combine":
        t, k, n, size = case["tokens"], case["topk"], case["cols"], _SIZES[case["dtype"]]
        return {"bytes": t * (k * (1.0 - case["dropped"]) + 1 + case["residual"]) * n * size + 8 * t * k, "flops": 2 * t * k * n}
    if case["op"] == "block_norm":
        rows, k, size, wsize = case["batch"] * case["tokens"], case["cols"], _SIZES[case["dtype"]], _SIZES[case["weights"]]
        n = rows * k
        out = {"none": n * size, "nvfp4": _nvfp4_bytes(rows, k)}.get(case["precision"], rows * _up(k, 16) + 4 * _up(rows, 16))
        vectors = case["weight"] + case["post"] + case["batch"] * 2 * case["modulate"] + {"none": 0, "vector": 1, "batch": case["batch"]}[case["gate"]]
        return {"bytes": n * size * (3 if case["residual"] else 1) + out + vectors * k * wsize, "flops": n * (10 if case["post"] else 6)}
    m, n, k = case["m"], case["n"], case["k"]
    return {"bytes": _nvfp4_bytes(m, k) + _nvfp4_bytes(n, k) + _SIZES[case["bias"]] * n + m * n * _SIZES[case["out"]] * (1 + case["residual"]),
            "flops": 2 * m * n * k}


# ------------------------------------------------------------------------------------------------------------ in 64 bits
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _nearest_e2m1(v):
    """By the middles between neighbours; the even code of two that are as near."""
    middles = torch.tensor([(a + b) / 2 for a, b in zip(_E2M1, _E2M1[1:])], dtype=torch.float64, device=v.device)
    a = v.abs()
    low, high = torch.searchsorted(middles, a, right=False), torch.searchsorted(middles, a, right=True)
    code = torch.where((low != high) & (low % 2 == 1), high, low)
    return torch.tensor(_E2M1, dtype=torch.float64, device=v.device)[code] * torch.sign(v)


def _exact_first(key):
    """Largest of the last dim and the lowest index that has it."""
    m = key.amax(-1)
    index = torch.arange(key.shape[-1], device=key.device)
    return m, torch.where(key == m[..., None], index, key.shape[-1]).amin(-1)


def _exact_taken(key, count):
    """`count` times the largest that is left: its index, or -1 where nothing above -inf is left."""
    key, index, taken = key.clone(), torch.arange(key.shape[-1], device=key.device), []
    for _ in range(count):
        m, at = _exact_first(key)
        taken.append(torch.where(m > -math.inf, at, -1))
        key = torch.where(index == at[..., None], -math.inf, key)
    return torch.stack(taken, dim=-1)


def _exact_route(case, state):
    t, e, k, g = case["tokens"], case["experts"], case["topk"], case["groups"]
    x = state["logits"].double()
    if case["scoring"] == "sigmoid":
        score = torch.where(x >= 0, 1.0 / (1.0 + torch.exp(-x)), torch.exp(x) / (1.0 + torch.exp(x)))
    else:
        score = torch.exp(x - torch.logsumexp(x, dim=1, keepdim=True)).nan_to_num(0.0)
    key = score + (0.0 if state["bias"] is None else state["bias"].double())
    key = torch.where(x == -math.inf, -math.inf, key)
    if g > 1:
        grouped = key.view(t, g, e // g)
        at = _exact_taken(grouped, min(case["best"], e // g))
        total = torch.where(at >= 0, grouped.gather(2, at.clamp(min=0)), 0.0).sum(2)
        total = torch.where(at[..., 0] >= 0, total, -math.inf)
        chosen = _exact_taken(total, case["top_groups"])
        kept = (chosen[:, None, :] == torch.arange(g, device=x.device)[None, :, None]).any(2)
        key = torch.where(kept[:, :, None], grouped, -math.inf).view(t, e)
    expert = _exact_taken(key, k)
    weight = torch.where(expert >= 0, score.gather(1, expert.clamp(min=0)), 0.0)
    if case["renormalize"]:
        weight = weight / weight.sum(1, keepdim=True).clamp(min=1e-300)
    hit = torch.zeros((t, e + 1), dtype=torch.int32, device=x.device).scatter_(1, torch.where(expert >= 0, expert, e), 1)[:, :e]
    counts = hit.sum(0)
    first = counts.cumsum(0) - counts
    place = torch.where(expert >= 0, (first + hit.cumsum(0) - 1).gather(1, expert.clamp(min=0)), -1)
    rows = torch.full((t * k + 1,), -1, dtype=torch.int32, device=x.device)
    token = torch.arange(t, dtype=torch.int32, device=x.device)[:, None].expand(t, k)
    rows[torch.where(place >= 0, place, t * k)] = torch.where(place >= 0, token, -1)
    offsets = torch.cat((first, counts.sum().view(1)))
    return {"weights": weight * case["scale"], "experts": expert.int(), "offsets": offsets.int(), "rows": rows[:t * k], "places": place.int()}


def _exact_normed(case, h):
    if case["kind"] == "layer":
        return (h - h.mean(2, keepdim=True)) / torch.sqrt(h.var(2, unbiased=False, keepdim=True) + _EPS)
    return h / torch.sqrt(torch.mean(h * h, dim=2, keepdim=True) + _EPS)


def _exact_block_norm(case, state):
    h, more = state["y"].double(), {}
    if state["residual"] is not None:
        if state["post_weight"] is not None:
            h = _exact_normed(case, h) * state["post_weight"].double()
        h = case["alpha"] * state["residual"].double() + (h if state["gate"] is None else h * state["gate"].double())
        more = {"residual": h}
        h = h.to(state["y"].dtype).double()  # the norm is that of the sum that is kept
    z = _exact_normed(case, h)
    if state["weight"] is not None:
        z = z * state["weight"].double()
    if case["modulate"]:
        z = z + z * state["scale"].double() + state["shift"].double()
    if case["precision"] == "none":
        return {"z": z, **more}
    z = z.flatten(0, 1)
    rows, cols = z.shape
    if case["precision"] == "nvfp4":
        gs = z.abs().max() / _NVFP4_MAX
        blocks = torch.nn.functional.pad(z, (0, -cols % 64)).view(rows, -1, 16)
        sf = (blocks.abs().amax(2) / 6.0 / gs).clamp(max=448.0).float().to(torch.float8_e4m3fn).double()
        step = (sf * gs)[:, :, None]
        codes = torch.where(step > 0, _nearest_e2m1(blocks / step.clamp(min=1e-300)), 0.0)
        laid = torch.zeros((sf.shape[1] // 4, _up(rows, 16), 4), dtype=torch.float64, device=z.device)
        laid[:, :rows] = sf.view(rows, -1, 4).permute(1, 0, 2)
        return {"z": (codes * step).view(rows, -1), "sf": laid, "gs": gs, **more}
    most = 127.0 if case["precision"] == "int8" else 448.0
    sf = z.abs().amax(1) / most
    scaled = torch.nn.functional.pad(z / sf[:, None], (0, -cols % 16))
    q = torch.round(scaled) if case["precision"] == "int8" else scaled.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).double()
    return {"z": q * sf[:, None], "sf": torch.nn.functional.pad(sf, (0, -rows % 16)), **more}


def _exact_values(packed, sf):
    """e2m1 times the scale of the block, [R, K] from one matrix's bytes [R, K/2] and scales [K/64, R up to 16, 4]."""
    lut = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), dtype=torch.float64, device=packed.device)
    rows = packed.shape[0]
    v = torch.empty((rows, packed.shape[1] * 2), dtype=torch.float64, device=packed.device)
    v[:, 0::2], v[:, 1::2] = lut[(packed % 16).int()], lut[(packed // 16).int()]
    return v * sf.permute(1, 0, 2)[:rows].reshape(rows, -1).double().repeat_interleave(16, dim=1)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "route":
        return _exact_route(case, state)
    if case["op"] == "combine":
        places = state["places"].long()
        out = torch.zeros((case["tokens"], case["cols"]), dtype=torch.float64, device="cuda")
        for s in range(case["topk"]):
            here = places[:, s] >= 0
            out[here] += state["weights"][here, s, None].double() * state["y"][places[here, s]].double()
        return out if state["residual"] is None else out + state["residual"].double()
    if case["op"] == "block_norm":
        return _exact_block_norm(case, state)
    y = _exact_values(state["x"], state["x_sf"]) @ _exact_values(state["w"], state["w_sf"]).t() * (state["x_gs"].double() * state["w_gs"].double())
    if state["bias"] is not None:
        y = y + state["bias"].double()
    kind = case["activation"]
    if kind == "relu":
        y = y.clamp(min=0.0)
    elif kind == "gelu":
        y = y * torch.special.ndtr(y)
    elif kind == "gelu_tanh":
        y = y * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (y + 0.044715 * y ** 3))
    elif kind == "silu":
        y = y * torch.sigmoid(y)
    return y if state["residual"] is None else y + state["residual"].double()
