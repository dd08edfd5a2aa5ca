"""Cases of the operators around the quantized linears and the attention of a transformer layer: the root-mean-square norm with
the residual's addition and a quantized output, its inverse (`dequantize`), rotary positions with several axes, and linears
grouped by expert.

`own` false: the operators in their plain form, elementary torch operations in 32 bits.  `own` true: the calls of
`ac4k_kernel_amd.ops`.  Sizes are those of this repository's benchmark and tests (widths of 4096, 5120, 8192 and 14336, decode,
8192-token prefill, the 75600-token tensors with 40 heads of 128, ragged relatives of them)."""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZES = {"none": 0, "bf16": 2, "fp16": 2, "fp32": 4}
_NVFP4_MAX = 448.0 * 6.0
_EPS = 1e-6


# ---------------------------------------------------------------------------------------------------------------- cases
def _norm(rows, cols, precision, **kw):
    """y = rms_norm(x [+ residual]) * weight, rows of x `pad` elements apart from each other."""
    return dict({"op": "rms_norm", "rows": rows, "cols": cols, "precision": precision, "dtype": "bf16", "weight": "bf16", "residual": False,
                 "pad": 0}, **kw)


def _dequantize(rows, cols, precision, **kw):
    return dict({"op": "dequantize", "rows": rows, "cols": cols, "precision": precision, "out": "bf16"}, **kw)


def _rope(batch, tokens, q_heads, k_heads, dim, **kw):
    """q and k rotated in one call.  where: "grid" (time, height, width of the tokens; those behind the last one are padding and stay)
    or "positions" (one index a token and axis, -1 on padding)."""
    return dict({"op": "rope", "batch": batch, "tokens": tokens, "q_heads": q_heads, "k_heads": k_heads, "dim": dim, "layout": "BNHD",
                 "dtype": "bf16", "where": "positions", "axes": 1, "length": 4096, "t": 1, "h": 1, "w": 1, "interleaved": True,
                 "inverse": False}, **kw)


def _grouped(tokens, topk, experts, n, k, **kw):
    """Every token goes to `topk` experts; gather: the rows are read through their token's index, otherwise they lie in order."""
    return dict({"op": "grouped_linear", "tokens": tokens, "topk": topk, "experts": experts, "n": n, "k": k, "gather": True, "skew": 0.5,
                 "bias": "none", "out": "bf16"}, **kw)


def listed():
    return [
        # one decoded token: residual added, norm, 8-bit output with its scale; launch latency counts
        dict(_norm(1, 8192, "fp8e4m3", residual=True), name="norm_fp8_1x8192"),
        # prefill of 8192 tokens in front of an NVFP4 linear: the scale of the whole tensor is found in the call
        dict(_norm(8192, 4096, "nvfp4", residual=True), name="norm_nvfp4_8192x4096"),
        # ragged: rows and columns that are multiples of nothing, rows cut out of a wider tensor, weights in fp32
        dict(_norm(4001, 5003, "int8", pad=13, weight="fp32"), name="norm_int8_4001x5003"),
        # q or k of a 75600-token sequence, normalized over all heads, no quantization (the largest norm)
        dict(_norm(75600, 5120, "none"), name="norm_bf16_75600x5120"),
        # an NVFP4 activation read back as bf16
        dict(_dequantize(8192, 4096, "nvfp4"), name="dequantize_nvfp4_8192x4096"),
        # ragged int8 read back as fp32
        dict(_dequantize(4001, 5003, "int8", out="fp32"), name="dequantize_int8_4001x5003"),
        # decode: 32 requests of one token each at far positions, grouped heads, halves rotated against each other
        dict(_rope(32, 1, 40, 8, 128, length=131072, interleaved=False), name="rope_decode_32x48x128"),
        # self-attention of a video: 21 x 45 x 80 tokens, 40 heads (the largest rotation)
        dict(_rope(1, 75600, 40, 40, 128, where="grid", axes=3, t=21, h=45, w=80, length=1024), name="rope_video_75600x40x128"),
        # gradient of the rotation, fp32, heads in front of the tokens, ragged lengths with padding behind them
        dict(_rope(2, 4001, 12, 12, 64, axes=3, layout="BHND", dtype="fp32", inverse=True), name="rope_inverse_2x4001x12x64"),
        # a decode batch: 16 tokens to 8 of 64 experts each, weights streamed from memory
        dict(_grouped(16, 8, 64, 2048, 4096), name="experts_16x8_e64_n2048_k4096"),
        # ragged: sizes that are multiples of nothing, experts with few rows or none, fp32 output with bias
        dict(_grouped(1001, 4, 32, 1003, 2880, gather=False, skew=1.5, bias="fp32", out="fp32"), name="experts_1001x4_e32_n1003_k2880"),
        # prefill: 8192 tokens to 2 of 8 experts each (the largest product)
        dict(_grouped(8192, 2, 8, 14336, 4096), name="experts_8192x2_e8_n14336_k4096"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi, least=1):
    """A feature dim: mostly a multiple of 128, sometimes of 64 or 8, sometimes odd."""
    w = _log_int(rng, lo, hi)
    step = max(least, rng.choice([128, 128, 128, 128, 64, 8, 1]))
    return max(lo, w // step * step)


def draw(rng):
    op = rng.choice(["rms_norm", "rms_norm", "dequantize", "rope", "rope", "grouped_linear", "grouped_linear"])
    if op == "rms_norm":
        cols = _width(rng, 64, 16384)
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
        rows = _log_int(rng, 1, min(75600, 380_000_000 // cols // (2 if dtype == "fp32" else 1)))
        residual = rng.random() < 0.5
        return _norm(rows if not residual else (rows + 1) // 2, cols, rng.choice(["none", "nvfp4", "nvfp4", "fp8e4m3", "int8"]), dtype=dtype,
                     weight=rng.choice([dtype, "fp32"]), residual=residual, pad=rng.choice([0, 0, 0, 64, 7]))
    if op == "dequantize":
        cols = _width(rng, 64, 16384)
        return _dequantize(_log_int(rng, 64, min(75600, 200_000_000 // cols)), cols, rng.choice(["nvfp4", "nvfp4", "fp8e4m3", "int8"]),
                           out=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    if op == "rope":
        dim, batch = rng.choice([64, 96, 128, 128, 128, 40, 256]), rng.choice([1, 1, 2, 7, 32])
        q_heads = rng.choice([1, 8, 12, 24, 40])
        k_heads = rng.choice([h for h in (1, 4, 8, 12, 24, 40) if q_heads % h == 0])
        tokens = _log_int(rng, 1, min(75600, 380_000_000 // (batch * (q_heads + k_heads) * dim)))
        kw = {"layout": rng.choice(["BNHD", "BHND"]), "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
              "interleaved": rng.random() < 0.5, "inverse": rng.random() < 0.2}
        if rng.random() < 0.4:
            w = max(1, _log_int(rng, 1, min(256, tokens)))
            h = max(1, _log_int(rng, 1, min(256, max(1, tokens // w))))
            return _rope(batch, tokens, q_heads, k_heads, dim, where="grid", axes=3, t=max(1, tokens // (w * h)), h=h, w=w, length=75601, **kw)
        return _rope(batch, tokens, q_heads, k_heads, dim, axes=rng.choice([1, 1, 2, 3]), length=rng.choice([1024, 32768, 131072]), **kw)
    experts = rng.choice([4, 8, 16, 32, 64, 128])
    k = _width(rng, 256, 14336, 64)
    n = _width(rng, 256, min(14336, max(257, 470_000_000 // (experts * k))))
    topk = rng.choice([1, 2, 4, 8])
    topk = min(topk, experts)
    skew = rng.choice([0.0, 0.5, 1.5])
    most = 960_000_000_000 if skew < 1 else 120_000_000_000  # the fullest of many experts gets several times its share
    tokens = _log_int(rng, 1, min(16384, max(2, min(most // n, 400_000_000) // (k * topk))))
    return _grouped(tokens, topk, experts, n, k, gather=rng.random() < 0.6, skew=skew,
                    bias=rng.choice(["none", "none", "bf16", "fp32"]), out=rng.choice(["bf16", "bf16", "fp16", "fp32"]))


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
    """e4m3 scales [.., R, K/16] -> [.., K/64, R up to 16, 4], zeros behind the last row."""
    sf = torch.nn.functional.pad(sf.float(), (0, 0, 0, _up(rows, 16) - rows))
    sf = sf.reshape(*sf.shape[:-1], -1, 4).transpose(-3, -2).contiguous()
    return sf.to(torch.float8_e4m3fn)


def _sections(case):
    """Pairs of elements of each axis: time takes what height and width leave."""
    pairs, axes = case["dim"] // 2, case["axes"]
    each = pairs // axes
    return (pairs - each * (axes - 1),) + (each,) * (axes - 1)


def _frequencies(case):
    """theta ** (-j / n) for pair j of the n pairs of an axis, in 64 bits."""
    return torch.cat([10000.0 ** (-torch.arange(n, dtype=torch.float64, device="cuda") / n) for n in _sections(case)])


def _angles(case):
    return torch.arange(case["length"], dtype=torch.float64, device="cuda")[:, None] * _frequencies(case)


def _heads_shape(case, heads):
    b, n, d = case["batch"], case["tokens"], case["dim"]
    return (b, n, heads, d) if case["layout"] == "BNHD" else (b, heads, n, d)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    if case["op"] == "rms_norm":
        rows, cols, dtype = case["rows"], case["cols"], _DTYPES[case["dtype"]]
        state["x"] = _activation((rows, cols + case["pad"]), gen).to(dtype)[:, :cols]
        state["residual"] = _normal((rows, cols), gen, 3.0).to(dtype) if case["residual"] else None
        state["weight"] = (1.0 + _normal((cols,), gen, 0.2)).to(_DTYPES[case["weight"]])
    elif case["op"] == "dequantize":
        rows, cols = case["rows"], case["cols"]
        y = _activation((rows, cols), gen)
        q, sf, gs = _quantized(y, case["precision"])
        state["q"] = _packed(q) if case["precision"] == "nvfp4" else q.to(torch.int8) if case["precision"] == "int8" else q.to(torch.float8_e4m3fn)
        state["sf"], state["gs"] = sf, gs
    elif case["op"] == "rope":
        dtype, b, n = _DTYPES[case["dtype"]], case["batch"], case["tokens"]
        state["q"] = _normal(_heads_shape(case, case["q_heads"]), gen).to(dtype)
        state["k"] = _normal(_heads_shape(case, case["k_heads"]), gen).to(dtype)
        state["table"] = torch.stack((_angles(case).cos(), _angles(case).sin()), dim=-1).float()
        state["sections"] = _sections(case)
        if case["where"] == "positions":
            at = torch.randint(0, case["length"], (case["axes"], b, n), device="cuda", generator=gen)
            pad = torch.randint(0, n // 8 + 1, (b, 1), device="cuda", generator=gen)  # the last tokens of a batch are padding
            state["positions"] = torch.where(torch.arange(n, device="cuda") >= n - pad, -1, at).to(torch.int32)
    else:
        t, e, n, k = case["tokens"], case["experts"], case["n"], case["k"]
        popular = torch.empty((e,), device="cuda").exponential_(generator=gen).log() * case["skew"]
        gumbel = -torch.empty((t, e), device="cuda").exponential_(generator=gen).log()
        expert = (popular + gumbel).topk(case["topk"], dim=1).indices.reshape(-1)
        order = expert.sort(stable=True).indices
        counts = torch.bincount(expert, minlength=e)
        state["offsets"] = torch.nn.functional.pad(counts.cumsum(0), (1, 0)).to(torch.int32)
        state["capacity"] = int(counts.max())
        state["rows"] = (order // case["topk"]).to(torch.int32) if case["gather"] else None
        x = _activation((t if case["gather"] else t * case["topk"], k), gen)
        q, state["x_sf"], state["x_gs"] = _quantized(x.to(torch.bfloat16).float(), "nvfp4")
        state["x"] = _packed(q)
        q, state["w_sf"], state["w_gs"] = _quantized(_normal((e, n, k), gen, 0.02).to(torch.bfloat16).float(), "nvfp4")
        state["w"] = _packed(q)
        state["bias"] = None if case["bias"] == "none" else _normal((e, n), gen, 0.5).to(_DTYPES[case["bias"]])
    return state


# ----------------------------------------------------------------------------------------------------------- plain form
def _round_e2m1(v):
    """To the nearest of 0, 0.5, 1, 1.5, 2, 3, 4 and 6, the even code of two, the sign kept."""
    a = v.abs()
    r = 0.5 * ((a > 0.25).to(v.dtype) + (a >= 0.75) + (a > 1.25) + (a >= 1.75)) + (a > 2.5) + (a >= 3.5) + 2.0 * (a > 5.0)
    return torch.copysign(r, v)


def _quantized(y, precision):
    """-> (values of the codes, padded to whole pieces; scales in their layout; scale of the whole tensor or None), in y's type.
    nvfp4: [.., R, K up to 64], 8 bits: [R, K up to 16].  A maximum under 2^-100 counts as zero."""
    rows, cols = y.shape[-2:]
    if precision == "nvfp4":
        y = torch.nn.functional.pad(y, (0, _up(cols, 64) - cols))
        blocks = y.reshape(*y.shape[:-1], -1, 16)
        m = blocks.abs().amax(-1)
        gs = m.reshape(y.shape[0], -1).amax(-1) if y.dim() == 3 else m.amax()
        gs = torch.where(gs < 2.0 ** -100, 0.0, gs) / _NVFP4_MAX
        alpha = torch.where(gs == 0, 0.0, 1.0 / gs)
        alpha = alpha[:, None, None] if y.dim() == 3 else alpha
        sixth = 1.0 / 6.0 if y.dtype == torch.float64 else float(torch.tensor(1.0 / 6.0, dtype=torch.float32))
        sf = (alpha * (m * sixth)).clamp(max=448.0).to(torch.float8_e4m3fn)
        s = sf.to(y.dtype)
        inverse = torch.where(s != 0, alpha * (1.0 / s), 0.0)
        return _round_e2m1(blocks * inverse.unsqueeze(-1)).reshape(y.shape), _scale_layout(sf, rows), gs
    most = 127.0 if precision == "int8" else 448.0
    m = y.abs().amax(-1)
    m = torch.where(m < 2.0 ** -100, 0.0, m)
    factor = torch.where(m == 0, 0.0, most / m)
    q = torch.nn.functional.pad(y * factor[:, None], (0, _up(cols, 16) - cols)).clamp(-most, most)
    q = q.round() if precision == "int8" else q.to(torch.float8_e4m3fn).to(y.dtype)
    return q, torch.nn.functional.pad(m / most, (0, _up(rows, 16) - rows)), None


def _plain_norm(state):
    case = state["case"]
    h = state["x"]
    if state["residual"] is not None:
        h = (h.float() + state["residual"].float()).to(h.dtype)
    # the sum of squares in 64 bits: the last place of the factor decides codes next to a border
    r = (1.0 / (h.double().square().mean(-1, keepdim=True) + _EPS).sqrt()).float()
    y = (h.float() * r) * state["weight"].float()
    more = {} if state["residual"] is None else {"residual": h}
    if case["precision"] == "none":
        return {"y": y.to(h.dtype), **more}
    q, sf, gs = _quantized(y, case["precision"])
    if case["precision"] == "nvfp4":
        return {"y": _plain_dequantized(q, sf, gs, case["rows"]).to(torch.bfloat16), "sf": sf, "gs": gs, **more}
    if case["precision"] == "int8":
        return {"y": (q * sf[: case["rows"], None]).to(torch.bfloat16), "sf": sf, **more}
    return {"y": q.to(torch.float8_e4m3fn), "sf": sf, **more}


def _blocks_of(sf, rows):
    """Scales [.., K/64, R up to 16, 4] -> [.., R, K/16, 1]."""
    return sf.float().transpose(-3, -2)[..., :rows, :, :].reshape(*sf.shape[:-3], rows, -1, 1)


def _plain_dequantized(q, sf, gs, rows):
    """e2m1 values [.., R, K] times the scale of their block of 16 (exact in 32 bits), then times the tensor's."""
    s = _blocks_of(sf, rows).to(q.dtype)
    gs = gs.to(q.dtype)
    v = (q.reshape(*q.shape[:-1], -1, 16) * s).reshape(q.shape)
    return v * (gs[:, None, None] if gs.dim() else gs)


def _unpacked(packed, dtype):
    values = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device="cuda", dtype=dtype)
    return values[torch.stack((packed & 15, packed >> 4), dim=-1).reshape(*packed.shape[:-1], -1).int()]


def _plain_dequantize(state):
    case = state["case"]
    if case["precision"] == "nvfp4":
        v = _plain_dequantized(_unpacked(state["q"], torch.float32), state["sf"], state["gs"], case["rows"])
    else:
        v = state["q"].float() * state["sf"][: case["rows"], None]
    return v.to(_DTYPES[case["out"]])


def _coordinates(state):
    """Index of every token along every axis, [axes, B, N], -1 where it is padding."""
    case = state["case"]
    if case["where"] == "positions":
        return state["positions"].long()
    i = torch.arange(case["tokens"], device="cuda")
    at = torch.stack((i // (case["h"] * case["w"]), i // case["w"] % case["h"], i % case["w"]))
    return torch.where(i < case["t"] * case["h"] * case["w"], at, -1)[:, None].expand(3, case["batch"], -1)


def _rotated(state, x, c, s):
    """c, s [B, N, pairs] in 32 or 64 bits."""
    case = state["case"]
    heads = 2 if case["layout"] == "BNHD" else 1
    c, s = c.unsqueeze(heads), s.unsqueeze(heads)
    s = -s if case["inverse"] else s
    x = x.to(c.dtype)
    if case["interleaved"]:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * c - b * s, b * c + a * s), dim=-1).reshape(x.shape)
    a, b = x.chunk(2, dim=-1)
    return torch.cat((a * c - b * s, b * c + a * s), dim=-1)


def _axis_of_pair(state):
    return torch.repeat_interleave(torch.arange(len(state["sections"]), device="cuda"), torch.tensor(state["sections"], device="cuda"),
                                   output_size=sum(state["sections"]))


def _plain_rope(state):
    at = _coordinates(state)[_axis_of_pair(state)].permute(1, 2, 0)  # [B, N, pairs]
    pair = torch.arange(at.shape[-1], device="cuda")
    stay = at < 0
    cs = state["table"][at.clamp(min=0), pair]
    c, s = torch.where(stay, 1.0, cs[..., 0]), torch.where(stay, 0.0, cs[..., 1])
    return [_rotated(state, state[n], c, s).to(state[n].dtype) for n in ("q", "k")]


def _expert_of_row(state):
    """Expert of each row, and its place among the rows of that expert."""
    case = state["case"]
    i = torch.arange(case["tokens"] * case["topk"], device="cuda")
    expert = torch.searchsorted(state["offsets"], i.to(torch.int32), right=True) - 1
    return expert, i - state["offsets"].long()[expert]


def _plain_grouped(state):
    """Rows laid out per expert in as many places as the fullest has, one batched product, the rows taken back."""
    case = state["case"]
    x = _plain_dequantized(_unpacked(state["x"], torch.float32), state["x_sf"], state["x_gs"], state["x"].shape[0])
    w = _plain_dequantized(_unpacked(state["w"], torch.float32), state["w_sf"], state["w_gs"], case["n"])
    if state["rows"] is not None:
        x = x[state["rows"].long()]
    expert, place = _expert_of_row(state)
    laid = x.new_zeros((case["experts"], state["capacity"], x.shape[1]))
    laid[expert, place] = x
    y = torch.bmm(laid, w.transpose(1, 2).contiguous())[expert, place]
    if state["bias"] is not None:
        y = y + state["bias"].float()[expert]
    return y.to(_DTYPES[case["out"]])


# ------------------------------------------------------------------------------------------------------- the operators
def _own_norm(state, ops):
    case = state["case"]
    precision = None if case["precision"] == "none" else case["precision"]
    got = ops.rms_norm(state["x"], state["weight"], eps=_EPS, residual=state["residual"], precision=precision)
    got = got if isinstance(got, tuple) else (got,)
    more = {} if state["residual"] is None else {"residual": got[-1]}
    if precision is None:
        return {"y": got[0], **more}
    if precision == "nvfp4":
        return {"y": ops.dequantize(*got[:3]), "sf": got[1], "gs": got[2], **more}
    if precision == "int8":
        return {"y": ops.dequantize(*got[:2]), "sf": got[1], **more}
    return {"y": got[0], "sf": got[1], **more}


def run(state):
    case = state["case"]
    if own:
        from ac4k_kernel_amd import ops
        if case["op"] == "rms_norm":
            return _own_norm(state, ops)
        if case["op"] == "dequantize":
            return ops.dequantize(state["q"], state["sf"], state["gs"], dtype=_DTYPES[case["out"]])
        if case["op"] == "rope":
            where = {"positions": state["positions"]} if case["where"] == "positions" else {"grid": (case["t"], case["h"], case["w"])}
            return list(ops.rope((state["q"], state["k"]), state["table"], sections=state["sections"], layout=case["layout"],
                                 interleaved=case["interleaved"], inverse=case["inverse"], **where))
        m = case["tokens"] * case["topk"]
        out = None if case["out"] == "bf16" else torch.empty((m, case["n"]), dtype=_DTYPES[case["out"]], device="cuda")
        return ops.grouped_linear(state["x"], state["x_sf"], state["x_gs"], state["w"], state["w_sf"], state["w_gs"], state["offsets"],
                                  rows=state["rows"], bias=state["bias"], out=out)
    if case["op"] == "rms_norm":
        return _plain_norm(state)
    if case["op"] == "dequantize":
        return _plain_dequantize(state)
    if case["op"] == "rope":
        return _plain_rope(state)
    return _plain_grouped(state)


# -------------------------------------------------------------------------------------------------- what has to be done
def _nvfp4_bytes(rows, k):
    return rows * _up(k, 64) // 2 + _up(k, 64) // 16 * _up(rows, 16)


def _quantized_bytes(rows, cols, precision):
    return _nvfp4_bytes(rows, cols) if precision == "nvfp4" else rows * _up(cols, 16) + 4 * _up(rows, 16)


def work(case):
    if case["op"] == "rms_norm":
        n, size = case["rows"] * case["cols"], _SIZES[case["dtype"]]
        out = n * size if case["precision"] == "none" else _quantized_bytes(case["rows"], case["cols"], case["precision"])
        return {"bytes": n * size * (3 if case["residual"] else 1) + out + _SIZES[case["weight"]] * case["cols"], "flops": 4 * n}
    if case["op"] == "dequantize":
        width = _up(case["cols"], 64 if case["precision"] == "nvfp4" else 16)
        return {"bytes": _quantized_bytes(case["rows"], case["cols"], case["precision"]) + case["rows"] * width * _SIZES[case["out"]], "flops": 0}
    if case["op"] == "rope":
        n = case["batch"] * case["tokens"] * (case["q_heads"] + case["k_heads"]) * case["dim"]
        at = 4 * case["axes"] * case["batch"] * case["tokens"] if case["where"] == "positions" else 0
        rows = min(case["length"], case["batch"] * case["tokens"])  # of the table
        return {"bytes": 2 * n * _SIZES[case["dtype"]] + at + 4 * rows * case["dim"], "flops": 3 * n}
    m, e, n, k = case["tokens"] * case["topk"], case["experts"], case["n"], case["k"]
    met = e * (1.0 - (1.0 - 1.0 / e) ** m)  # experts that get a row, if all are alike
    x = _nvfp4_bytes(case["tokens"] if case["gather"] else m, k)
    return {"bytes": x + met * (_nvfp4_bytes(n, k) + _SIZES[case["bias"]] * n) + m * n * _SIZES[case["out"]] + (4 * m if case["gather"] else 0),
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


def _exact_norm(case, state):
    h = state["x"].double()
    more = {}
    if state["residual"] is not None:
        h = h + state["residual"].double()
        more = {"residual": h}
        h = h.to(state["x"].dtype).double()  # the norm is that of the sum that is kept
    y = h / torch.sqrt(torch.mean(h * h, dim=1, keepdim=True) + _EPS) * state["weight"].double()
    if case["precision"] == "none":
        return {"y": y, **more}
    rows, cols = y.shape
    if case["precision"] == "nvfp4":
        gs = y.abs().max() / _NVFP4_MAX
        blocks = torch.nn.functional.pad(y, (0, -cols % 64)).view(rows, -1, 16)
        sf = (blocks.abs().amax(2) / 6.0 / gs).clamp(max=448.0).float().to(torch.float8_e4m3fn).double()
        step = sf * gs
        codes = torch.where(step[:, :, None] > 0, _nearest_e2m1(blocks / step.clamp(min=1e-300)[:, :, None]), 0.0)
        laid = torch.zeros((sf.shape[1] // 4, _up(rows, 16), 4), dtype=torch.float64, device=y.device)
        laid[:, :rows] = sf.view(rows, -1, 4).permute(1, 0, 2)
        return {"y": (codes * step[:, :, None]).view(rows, -1), "sf": laid, "gs": gs, **more}
    most = 127.0 if case["precision"] == "int8" else 448.0
    sf = y.abs().amax(1) / most
    scaled = torch.nn.functional.pad(y / sf[:, None], (0, -cols % 16))
    all_sf = torch.nn.functional.pad(sf, (0, -rows % 16))
    if case["precision"] == "int8":
        return {"y": torch.round(scaled) * sf[:, None], "sf": all_sf, **more}
    return {"y": scaled.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).double(), "sf": all_sf, **more}


def _exact_values(packed, sf):
    """e2m1 times the scale of the block, [R, K] from one matrix's bytes [R, K/2] and scales [K/64, R up to 16, 4]."""
    lut = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), dtype=torch.float64, device=packed.device)
    rows = packed.shape[0]
    v = torch.empty((rows, packed.shape[1] * 2), dtype=torch.float64, device=packed.device)
    v[:, 0::2], v[:, 1::2] = lut[(packed % 16).int()], lut[(packed // 16).int()]
    return v * sf.permute(1, 0, 2)[:rows].reshape(rows, -1).double().repeat_interleave(16, dim=1)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "rms_norm":
        return _exact_norm(case, state)
    if case["op"] == "dequantize":
        if case["precision"] == "nvfp4":
            return _exact_values(state["q"], state["sf"]) * state["gs"].double()
        return state["q"].float().double() * state["sf"].double()[: case["rows"], None]
    if case["op"] == "rope":
        at = _coordinates(state)
        place = at[[a for a, n in enumerate(state["sections"]) for _ in range(n)]].permute(1, 2, 0)
        angle = torch.where(place < 0, 0.0, place.double() * _frequencies(case))
        angle = -angle if case["inverse"] else angle
        turn = torch.polar(torch.ones_like(angle), angle).unsqueeze(2 if case["layout"] == "BNHD" else 1)
        outs = []
        for x in (state["q"].double(), state["k"].double()):
            half = x.shape[-1] // 2
            z = torch.view_as_complex(x.unflatten(-1, (half, 2)).contiguous()) if case["interleaved"] else torch.complex(x[..., :half], x[..., half:])
            z = z * turn
            outs.append(torch.view_as_real(z).flatten(-2) if case["interleaved"] else torch.cat((z.real, z.imag), dim=-1))
        return outs
    ends = state["offsets"].tolist()
    x = _exact_values(state["x"], state["x_sf"])
    y = torch.empty((case["tokens"] * case["topk"], case["n"]), dtype=torch.float64, device="cuda")
    for e in range(case["experts"]):
        a, b = ends[e], ends[e + 1]
        if a == b:
            continue
        rows = x[a:b] if state["rows"] is None else x[state["rows"][a:b].long()]
        y[a:b] = rows @ _exact_values(state["w"][e], state["w_sf"][e]).t() * (state["x_gs"].double() * state["w_gs"][e].double())
        if state["bias"] is not None:
            y[a:b] += state["bias"][e].double()
    return y
