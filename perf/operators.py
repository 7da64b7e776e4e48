"""Cases of the MXFP products with an epilogue and of the products grouped by expert.

Two operators on the same operands: an activation ``x`` that is quantised to MXFP (blocks of 32 along its last
dimension, one power-of-two scale each) within the call, and weights that a program holds as MXFP codes and scales.

* ``linear``:   y = act(Q(x) W^T + bias) * multiplier + residual, one weight ``[N, K]``;
* ``grouped``:  the rows of ``x`` (or those that ``row_index`` names) lie expert after expert, expert ``e`` has the rows
  ``offsets[e] .. offsets[e + 1]`` and its own weight ``[N, K]`` of a ``[E, N, K]`` tensor and its own bias; the same
  epilogue; rows behind the last expert's keep what the output held.
"""

import math

import torch

own = False

FORMATS = {"e4m3": (4, 3), "e5m2": (5, 2), "e2m3": (2, 3), "e3m2": (3, 2), "e2m1": (2, 1)}
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
MOST_FLOPS = 2 * 16384 * 4096 * 14336


def _linear(name, M, K, N, dtype, x, w, bias=False, act="none", extra="none"):
    return {"name": name, "op": "linear", "M": M, "K": K, "N": N, "dtype": dtype, "x": x, "w": w, "bias": bias, "act": act, "extra": extra}


def _grouped(name, T, E, K, N, dtype, x, w, top=0, pad=0, bias=False, act="none", extra="none"):
    return {"name": name, "op": "grouped", "T": T, "E": E, "K": K, "N": N, "dtype": dtype, "x": x, "w": w, "top": top, "pad": pad,
            "bias": bias, "act": act, "extra": extra}


def listed():
    return [
        # one token through a gated projection (the up projection's result is the multiplier): a read of the weight
        _linear("token_gate", 1, 4096, 14336, "bfloat16", "e4m3", "e4m3", act="silu", extra="multiplier"),
        # a few tokens back to the model width, added to the residual stream: a long axis, few outputs
        _linear("tokens_down", 5, 14336, 4096, "bfloat16", "e4m3", "e3m2", extra="residual"),
        # a batch of sequences that each decode one token
        _linear("batch_gelu", 192, 4096, 4096, "float16", "e5m2", "e4m3", bias=True, act="gelu"),
        # odd sizes: K no multiple of 128, N odd; activations in 32 bits
        _linear("ragged_relu", 777, 1184, 1001, "float32", "e4m3", "e5m2", bias=True, act="relu", extra="residual"),
        # a prompt through the gated projection
        _linear("prompt_gate", 8192, 4096, 14336, "bfloat16", "e4m3", "e4m3", act="silu", extra="multiplier"),
        # a prompt with both operands in four bits
        _linear("prompt_fp4", 4096, 4096, 4096, "bfloat16", "e2m1", "e2m1", extra="residual"),
        # one token and the two experts it is routed to
        _grouped("token_experts", 2, 8, 4096, 14336, "bfloat16", "e4m3", "e4m3", top=2, act="silu", extra="multiplier"),
        # a decoding batch over many small experts: a few rows each, some none
        _grouped("decode_experts", 256, 64, 2048, 1024, "bfloat16", "e4m3", "e4m3", top=8, act="silu", extra="multiplier"),
        # the same rows back to the model width
        _grouped("decode_down", 256, 64, 1024, 2048, "bfloat16", "e4m3", "e3m2"),
        # odd sizes, a padded batch, bias per expert
        _grouped("ragged_experts", 3001, 17, 1184, 520, "float16", "e4m3", "e2m3", pad=39, bias=True, act="gelu_tanh", extra="residual"),
        # a prompt over experts in four bits
        _grouped("prompt_fp4_experts", 8192, 32, 2048, 2048, "bfloat16", "e2m1", "e2m1", top=4, act="silu", extra="multiplier"),
        # a prompt over large experts, each token to two of them
        _grouped("prompt_experts", 16384, 8, 4096, 14336, "bfloat16", "e4m3", "e4m3", top=2, act="silu", extra="multiplier"),
    ]


def draw(rng):
    def size(lo, hi, step=1):
        v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
        return max(step, int(v) // step * step)

    while True:
        x, w = rng.choice(["e4m3", "e4m3", "e5m2", "e2m3", "e3m2", "e2m1"]), rng.choice(["e4m3", "e4m3", "e5m2", "e2m3", "e3m2", "e2m1"])
        if rng.random() < 0.2:
            x = w = "e2m1"
        common = dict(dtype=rng.choice(["bfloat16", "bfloat16", "float16"]), x=x, w=w, bias=rng.random() < 0.4,
                      act=rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]), extra=rng.choice(["none", "multiplier", "residual"]))
        K, N = size(32, 14336, rng.choice([32, 128, 256])), size(8, 14336, rng.choice([1, 8, 64]))
        if K <= 4096 and rng.random() < 0.2:
            common["dtype"] = "float32"
        if rng.random() < 0.5:
            M = size(1, 8192)
            if 2 * M * K * N > MOST_FLOPS or M * K * N < 1 << 16:
                continue
            c = _linear("", M, K, N, **common)
        else:
            E, top = size(2, 128), rng.choice([0, 1, 2, 4, 8])
            T = max(1, size(1, 16384) // max(1, top)) * max(1, top)
            if T > 16384 or E * K * N > 1 << 29 or 2 * T * K * N > MOST_FLOPS or T * K * N < 1 << 16:
                continue
            c = _grouped("", T, E, K, N, top=top, pad=rng.choice([0, 0, 7, 130]) if top == 0 else 0, **common)
        c.pop("name")
        return c


# ---------------------------------------------------------------------------------------------------------------------
# plain form
# ---------------------------------------------------------------------------------------------------------------------
def _encode(x, fmt):
    """MXFP codes and scale bytes of ``x [..., K]``, blocks of 32 along K: ``(scales [..., K / 32], codes [..., K])``, whole numbers.

    The shared exponent is that of the block's largest magnitude less the format's largest exponent; the quotient's
    mantissa is cut to 15 bits and rounded half to even to the format's fraction, and the rounded field is OR-ed under
    the exponent field, so that a carry out of it is kept where the biased exponent is even and lost where it is odd."""
    eb, fb = FORMATS[fmt]
    bias, top = (1 << (eb - 1)) - 1, (1 << eb) - 1
    b = x.to(torch.float32).reshape(*x.shape[:-1], -1, 32)
    most = b.abs().amax(-1, keepdim=True)
    # 64 bits: the logarithm of a value just below a power of two, rounded once to 32 bits
    shared = (torch.log2(most.to(torch.float64)).to(torch.float32).floor() - (top - bias)).clamp(-127, 127)
    shared = torch.where(most > 0, shared, torch.zeros_like(shared))
    bits = (b * torch.exp2(-shared)).view(torch.int32)
    m, e = (bits >> 8) & 0x7FFF, ((bits >> 23) & 0xFF) - 127 + bias
    d = 15 - fb
    f = (m + ((1 << (d - 1)) - 1) + ((m >> d) & 1)) >> d
    f = torch.where((e == 0) & (f != 0), (f | (1 << fb)) >> 1, f)
    code = (e << fb) | f
    code = torch.where(e < 0, 0, torch.where(e > top, (top << fb) | ((1 << fb) - 1), code))
    code = code | ((bits < 0) & (b != 0)).to(torch.int32) * (1 << (eb + fb))
    scale = torch.where(most > 0, shared + 127, torch.zeros_like(shared)).squeeze(-1)
    return scale.to(torch.int32), code.reshape(x.shape)


def _decode(scales, codes, fmt):
    """The values in 32 bits that the codes ``[..., K]`` and the scale bytes ``[..., K / 32]`` stand for."""
    eb, fb = FORMATS[fmt]
    bias = (1 << (eb - 1)) - 1
    c = codes.to(torch.int32)
    e, f = (c >> fb) & ((1 << eb) - 1), (c & ((1 << fb) - 1)).to(torch.float32)
    v = torch.where(e == 0, f * 2.0 ** (1 - bias - fb), (f * 2.0**-fb + 1) * torch.exp2((e - bias).to(torch.float32)))
    v = torch.where((c >> (eb + fb)) & 1 == 1, -v, v)
    v = v.reshape(*v.shape[:-1], -1, 32) * torch.exp2(scales.to(torch.float32) - 127).unsqueeze(-1)
    return v.reshape(codes.shape)


def _activate(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _epilogue(z, s, wide):
    y = _activate(z, s["act"])
    if s["extra"] == "multiplier":
        y = y * s["other"].to(wide)
    elif s["extra"] == "residual":
        y = y + s["other"].to(wide)
    return y


def _plain_linear(s):
    z = _decode(*_encode(s["values"], s["x"]), s["x"]) @ _decode(s["scales"], s["codes"], s["w"]).t()
    if s["bias"] is not None:
        z = z + s["bias"].to(torch.float32)
    return _epilogue(z, s, torch.float32).to(s["dtype"])


def _plain_grouped(s):
    # the experts' rows side by side, each expert filled up to the longest with rows of zeros: one batched product
    x = s["values"] if s["row_index"] is None else s["values"].index_select(0, s["row_index"].to(torch.int64))
    offsets = s["offsets"].to(torch.int64)
    x = _decode(*_encode(x, s["x"]), s["x"])
    place = offsets[:-1, None] + torch.arange(s["most"], device=x.device)
    here = place < offsets[1:, None]
    side = torch.where(here[..., None], x[place.clamp(max=x.shape[0] - 1)], torch.zeros((), device=x.device))
    z = side @ _decode(s["scales"], s["codes"], s["w"]).transpose(1, 2)
    if s["bias"] is not None:
        z = z + s["bias"].to(torch.float32)[:, None]
    row = torch.arange(x.shape[0], device=x.device)
    expert = torch.searchsorted(offsets[1:], row, right=True).clamp(max=offsets.shape[0] - 2)
    z = z[expert, (row - offsets[expert]).clamp(0, s["most"] - 1)]
    y = _epilogue(z, s, torch.float32).to(s["dtype"])
    s["out"].copy_(torch.where((row < offsets[-1])[:, None], y, s["out"]))
    return s["out"]


# ---------------------------------------------------------------------------------------------------------------------
# what the tools call
# ---------------------------------------------------------------------------------------------------------------------
def _counts(case, g, rows):
    """Rows of each expert: the experts are not equally popular, and a small batch leaves some without any."""
    liking = torch.randn(case["E"], generator=g, device="cuda") * 0.5
    picked = torch.multinomial(torch.softmax(liking, 0), rows, replacement=True, generator=g)
    return torch.bincount(picked, minlength=case["E"])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, by=1.0):
        return torch.randn(*shape, generator=g, device="cuda") * by

    K, N, grouped = case["K"], case["N"], case["op"] == "grouped"
    rows = case["T"] if grouped else case["M"]
    tokens = rows // case["top"] if grouped and case["top"] else rows
    s = {"op": case["op"], "dtype": dtype, "x": case["x"], "w": case["w"], "act": case["act"], "extra": case["extra"]}
    # activations: channels differ in scale, as behind a norm with its own weights
    s["values"] = (normal(tokens, K) * torch.exp2(normal(K))).to(dtype)
    experts = case["E"] if grouped else 1
    scales, codes = torch.empty(experts, N, K // 32, dtype=torch.uint8, device="cuda"), torch.empty(experts, N, K, dtype=torch.uint8, device="cuda")
    for e in range(experts):
        sc, co = _encode(normal(N, K, by=0.5 / math.sqrt(K)).to(torch.bfloat16), case["w"])
        scales[e], codes[e] = sc, co
    s["scales"], s["codes"] = (scales, codes) if grouped else (scales[0], codes[0])
    s["bias"] = None if not case["bias"] else normal(*((experts, N) if grouped else (N,)), by=0.5).to(dtype)
    s["other"] = None if case["extra"] == "none" else normal(rows, N).to(dtype)
    if grouped:
        counts = _counts(case, g, rows - case["pad"] if rows > case["pad"] else rows)
        s["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
        s["most"] = int(counts.max())
        s["row_index"] = None if not case["top"] else torch.argsort(torch.rand(rows, generator=g, device="cuda")).to(torch.int32) // case["top"]
        s["out"] = normal(rows, N).to(dtype)
    if own:
        from mase_triton_b200.mxfp import layers, meta

        x_meta, w_meta = (meta.MXFPMeta(32, 8, *FORMATS[f], True, "rn") for f in (case["x"], case["w"]))
        shape = (experts, N, K) if grouped else (N, K)
        tensor_meta = meta.MXFPTensorMeta("cuda:0", case["dtype"], shape, -1, w_meta)
        stored = (scales.reshape(-1, 1), codes.reshape(-1, 32), tensor_meta, s["bias"])
        if grouped:
            s["layer"] = layers.MXFPGroupedLinearPTQ.from_quantized(*stored, x_mxfp_meta=x_meta)
        else:
            s["layer"] = layers.MXFPLinearPTQ.from_quantized(*stored, None, None, None, x_meta, "XqWqB", "fused")
    return s


def run(s):
    if not own:
        return _plain_grouped(s) if s["op"] == "grouped" else _plain_linear(s)
    epilogue = {"activation": None if s["act"] == "none" else s["act"]}
    if s["extra"] != "none":
        epilogue[s["extra"]] = s["other"]
    if s["op"] == "grouped":
        return s["layer"](s["values"], s["offsets"], row_index=s["row_index"], out=s["out"], **epilogue)
    return s["layer"](s["values"], **epilogue)


def work(case):
    """The activation, the codes and scales of the weights that have rows, bias and second operand read once, the output
    written once; the products."""
    K, N, grouped = case["K"], case["N"], case["op"] == "grouped"
    rows = case["T"] - (case["pad"] if case["T"] > case["pad"] else 0) if grouped else case["M"]
    size = 4 if case["dtype"] == "float32" else 2
    experts = min(case["E"], rows) if grouped else 1
    tokens = rows // case["top"] if grouped and case["top"] else rows
    bits = 1 + sum(FORMATS[case["w"]])
    weights = experts * N * K * (bits / 8 + 1 / 32)
    return {"bytes": tokens * K * size + weights + (experts * N * size if case["bias"] else 0) + rows * N * size * (1 if case["extra"] == "none" else 2),
            "flops": 2 * rows * N * K}


# ---------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def _grid(x, fmt):
    """Q(x) in 64 bits, by the values of the format's grid and not by its bit fields."""
    eb, fb = FORMATS[fmt]
    bias, top = (1 << (eb - 1)) - 1, (1 << eb) - 1
    b = x.to(torch.float64).unflatten(-1, (-1, 32))
    most = b.abs().amax(-1, keepdim=True)
    level = torch.log2(most.clamp(min=2.0**-140)).to(torch.float32).to(torch.float64).floor() - (top - bias)
    scale = torch.ldexp(torch.ones_like(level), level.clamp(min=-127))
    mantissa, exponent = torch.frexp(b.abs() / scale)                 # in [0.5, 1): the binade below
    mantissa, exponent = torch.floor(mantissa * 2.0**16) * 2.0**-15, exponent - 1
    steps = torch.round((mantissa - 1) * 2.0**fb)                     # 0 .. 2^fb above the binade's lower end, half to even
    biased = exponent + bias
    full = steps == 2**fb
    lower = torch.ldexp(torch.ones_like(mantissa), exponent)
    normal = torch.where(full, torch.where(biased % 2 == 0, 2 * lower, lower), lower * (1 + steps * 2.0**-fb))
    small = torch.where(steps == 0, steps, torch.floor((steps + torch.where(full, 0.0, 2.0**fb)) / 2)) * 2.0 ** (1 - bias - fb)
    v = torch.where(biased < 0, torch.zeros_like(normal), torch.where(biased == 0, small, normal))
    v = torch.where(biased > top, torch.full_like(v, 2.0 ** (top - bias) * (2 - 2.0**-fb)), v)
    v = torch.where(b == 0, torch.zeros_like(v), v)
    return (torch.sign(b) * v * scale).flatten(-2)


def _values(scales, codes, fmt):
    """The stored weights in 64 bits: a table of the format's values, times the blocks' scales."""
    eb, fb = FORMATS[fmt]
    bias = (1 << (eb - 1)) - 1
    table = []
    for c in range(256):
        e, f = (c >> fb) & ((1 << eb) - 1), c & ((1 << fb) - 1)
        v = math.ldexp(f, 1 - bias - fb) if e == 0 else math.ldexp(f + (1 << fb), e - bias - fb)
        table.append(-v if (c >> (eb + fb)) & 1 else v)
    v = torch.tensor(table, dtype=torch.float64, device=codes.device)[codes.to(torch.int64)]
    scale = torch.ldexp(torch.ones(scales.shape, dtype=torch.float64, device=codes.device), scales.to(torch.int32) - 127)
    return (v.unflatten(-1, (-1, 32)) * scale.unsqueeze(-1)).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    wide = torch.float64
    if case["op"] == "linear":
        z = _grid(s["values"], case["x"]) @ _values(s["scales"], s["codes"], case["w"]).t()
        z = z if s["bias"] is None else z + s["bias"].to(wide)
        return _epilogue(z, s, wide)
    x = s["values"] if s["row_index"] is None else s["values"][s["row_index"].to(torch.int64)]
    y = s["out"].to(wide)
    ends = s["offsets"].tolist()
    for e in range(case["E"]):
        lo, hi = ends[e], ends[e + 1]
        if lo < hi:
            z = _grid(x[lo:hi], case["x"]) @ _values(s["scales"][e], s["codes"][e], case["w"]).t()
            z = z if s["bias"] is None else z + s["bias"][e].to(wide)
            y[lo:hi] = _epilogue(z, {**s, "other": None if s["other"] is None else s["other"][lo:hi]}, wide)
    return y
