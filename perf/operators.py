"""What the performance of the 4-bit serving operators is measured on (``mpserve_b200.mx4``).

A serving process keeps its weights in MXFP4 (E2M1 codes, one power-of-two scale per 32 columns), quantises what it
decoded from a compressed checkpoint once, and then, per step and per layer, normalises the residual stream, multiplies
by the weights and joins the block's result to the stream again.  Steps have one token (a lone conversation), some tens
(a batch of conversations) or thousands (prompts).

Plain forms are elementary torch operations in 32 bits.  What is held in 4 bits is returned as the values it stands for.
"""
import math

import torch

own = False

BLOCK = 32
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
BITS = 4.25 / 8      # bytes of an element in MXFP4, its share of the scale included
EPS = 1e-5
# One 8B layer: hidden 4096, inter 14336; a 70B layer split over 8 ranks: hidden 8192, inter 28672 / 8 = 3584.
MOST = 4096 * 4096 * 14336   # multiply-adds of the largest listed product


def quantize(name, rows, cols, dtype):
    return dict(name=name, kind="quantize", rows=rows, cols=cols, dtype=dtype)


def linear(name, tokens, cols, rows, dtype="bf16"):
    return dict(name=name, kind="linear", tokens=tokens, cols=cols, rows=rows, dtype=dtype)


def gated(name, tokens, cols, rows, activation="silu", dtype="bf16"):
    return dict(name=name, kind="gated", tokens=tokens, cols=cols, rows=rows, activation=activation, dtype=dtype)


def join(name, tokens, cols, dtype="bf16", stream="bf16", gate="channel", post=True, alpha=1.0):
    return dict(name=name, kind="join", tokens=tokens, cols=cols, dtype=dtype, stream=stream, gate=gate, post=post, alpha=alpha)


def mlp(name, tokens, hidden, inter, activation="silu", dtype="bf16"):
    return dict(name=name, kind="mlp", tokens=tokens, hidden=hidden, inter=inter, activation=activation, dtype=dtype)


def listed():
    return [
        # one token's activations: a launch and its host side
        quantize("quantize_token_4096", 1, 4096, "bf16"),
        # an MLP weight, just decoded, on its way into 4 bits: once per weight when a model is loaded
        quantize("quantize_weight_14336x4096", 14336, 4096, "bf16"),
        # rows of no convenient length, in 32 bits
        quantize("quantize_ragged_2047x1337_f32", 2047, 1337, "f32"),
        # a lone conversation's token through an MLP weight: the weight's bytes count
        linear("linear_1x4096x14336", 1, 4096, 14336),
        # a batch of conversations on a tensor-parallel rank's share of a 70B layer, half precision
        linear("linear_64x8192x3584_f16", 64, 8192, 3584, "f16"),
        # odd in every direction: a small model's projection
        linear("linear_333x1000x517", 333, 1000, 517),
        # a prompt's tokens through an MLP weight: the tensor cores count
        linear("linear_4096x4096x14336", 4096, 4096, 14336),
        # both halves of a gated MLP for a batch of conversations
        gated("gated_32x4096x14336", 32, 4096, 14336),
        # the end of a block for one token ...
        join("join_1x4096", 1, 4096),
        # ... and for long prompts whose stream is kept in 32 bits
        join("join_8191x4096_f32_stream", 8191, 4096, "bf16", "f32", "token", True, 0.75),
        # a whole MLP block of an 8B layer: norm, gate and up, activation, down, norm, gate and residual
        mlp("mlp_1_token_8b", 1, 4096, 14336),
        mlp("mlp_2048_tokens_8b", 2048, 4096, 14336),
    ]


def _between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, low, high):
    """Columns: mostly a multiple of 128 as hidden sizes are, or of 32, sometimes any number."""
    step = rng.choice((128, 128, 128, 32, 1))
    return max(step, _between(rng, low, high) // step * step)


def draw(rng):
    kind = rng.choice(("quantize", "linear", "linear", "gated", "join", "join", "mlp"))
    if kind == "quantize":
        cols, dtype = _width(rng, 40, 14336), rng.choice(("bf16", "bf16", "f16", "f32"))
        return quantize(None, _between(rng, 1, max(1, 14336 * 4096 // (cols * (2 if dtype == "f32" else 1)))), cols, dtype)
    if kind in ("linear", "gated"):
        cols, rows = _width(rng, 64, 14336), _width(rng, 64, 14336)
        halves = 2 if kind == "gated" else 1
        tokens = _between(rng, 1, max(1, min(8192, MOST // (cols * rows * halves))))
        if kind == "linear":
            return linear(None, tokens, cols, rows, rng.choice(("bf16", "f16")))
        return gated(None, tokens, cols, rows, rng.choice(("silu", "gelu")), rng.choice(("bf16", "f16")))
    if kind == "join":
        cols, dtype = _width(rng, 64, 8192), rng.choice(("bf16", "bf16", "f16"))
        return join(None, _between(rng, 1, 8192 * 4096 // cols), cols, dtype, rng.choice((dtype, "f32")),
                    rng.choice(("none", "channel", "token", "full")), rng.random() < 0.6, rng.choice((1.0, 0.5)))
    hidden, inter = _width(rng, 64, 8192), _width(rng, 64, 14336)
    tokens = _between(rng, 1, max(1, min(4096, MOST // (3 * hidden * inter))))
    return mlp(None, tokens, hidden, inter, rng.choice(("silu", "gelu")), rng.choice(("bf16", "f16")))


# ---- inputs -----------------------------------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _activations(g, tokens, cols, dtype):
    """Normal, with some channels far larger than the rest, as the streams of trained models have."""
    x = torch.randn((tokens, cols), generator=g, device="cuda")
    loud = torch.rand((cols,), generator=g, device="cuda") < 0.01
    return (x * torch.where(loud, 12.0, 1.0)).to(DTYPES[dtype])


def _weight_parts(g, rows, cols):
    """A weight as checkpoints store MXFP4: two codes a byte, the first in the low half, and a scale byte per 32 columns."""
    w = torch.randn((rows, cols), generator=g, device="cuda") * 0.02
    code, scale = _plain_codes(w)
    code = torch.nn.functional.pad(code, (0, cols % 2)).view(rows, -1, 2)
    return (code[:, :, 0] | (code[:, :, 1] << 4)).contiguous(), scale.contiguous()


def _gain(g, cols):
    return (1 + 0.1 * torch.randn((cols,), generator=g, device="cuda")).to(torch.bfloat16)


def _handle(parts, cols):
    from mpserve_b200 import mx4

    return mx4.from_parts(*parts, cols)


def prepare(case, seed):
    g, s = _generator(seed), dict(case)
    kind = case["kind"]
    if kind == "quantize":
        s["x"] = torch.randn((case["rows"], case["cols"]), generator=g, device="cuda").mul_(0.02).to(DTYPES[case["dtype"]])
    elif kind in ("linear", "gated"):
        s["x"] = _activations(g, case["tokens"], case["cols"], case["dtype"])
        weights = [_weight_parts(g, case["rows"], case["cols"]) for _ in range(2 if kind == "gated" else 1)]
        s["weights"] = [_handle(w, case["cols"]) for w in weights] if own else weights
    elif kind == "join":
        t, d = case["tokens"], case["cols"]
        s["y"], s["h"] = _activations(g, t, d, case["dtype"]), _activations(g, t, d, case["stream"])
        s["post_weight"] = _gain(g, d) if case["post"] else None
        s["next_weight"] = _gain(g, d)
        shape = {"none": None, "channel": (d,), "token": (t, 1), "full": (t, d)}[case["gate"]]
        s["g"] = None if shape is None else torch.randn(shape, generator=g, device="cuda").mul_(0.5).to(DTYPES[case["dtype"]])
    else:
        d, i = case["hidden"], case["inter"]
        s["h"] = _activations(g, case["tokens"], d, case["dtype"])
        weights = [_weight_parts(g, i, d), _weight_parts(g, i, d), _weight_parts(g, d, i)]
        s["pre_weight"], s["post_weight"], s["next_weight"] = _gain(g, d), _gain(g, d), _gain(g, d)
        s["g"] = torch.randn((d,), generator=g, device="cuda").mul_(0.5).to(torch.bfloat16)
        if own:
            from mpserve_b200 import mx4

            s["block"] = mx4.GatedMlp(_handle(weights[0], d), _handle(weights[1], d), _handle(weights[2], i),
                                      pre_weight=s["pre_weight"], post_weight=s["post_weight"], gate=s["g"],
                                      next_weight=s["next_weight"], eps=EPS, activation=case["activation"])
        else:
            s["weights"] = weights
    return s


# ---- a pass -----------------------------------------------------------------------------------------

def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    from mpserve_b200 import mx4

    kind = s["kind"]
    if kind == "quantize":
        return mx4.quantize(s["x"]).dequantize(s["x"].dtype)
    if kind == "linear":
        return mx4.linear(s["x"], s["weights"][0])
    if kind == "gated":
        return mx4.gated_linear(s["x"], s["weights"][0], s["weights"][1], activation=s["activation"])
    if kind == "join":
        return mx4.block_join(s["y"], s["h"], post_weight=s["post_weight"], gate=s["g"], residual_scale=s["alpha"],
                              next_weight=s["next_weight"], eps=EPS)
    return s["block"].forward(s["h"])


def _plain_codes(x):
    """E2M1 codes [rows, cols] and scale bytes [rows, blocks] of a matrix."""
    rows, cols = x.shape
    blocks = -(-cols // BLOCK)
    v = torch.nn.functional.pad(x.float(), (0, blocks * BLOCK - cols)).view(rows, blocks, BLOCK)
    exponent = torch.frexp(v.abs().amax(dim=2))[1] - 1                     # floor(log2)
    exponent = torch.where(v.abs().amax(dim=2) > 0, exponent - 2, -127).clamp(-127, 125)
    a = torch.ldexp(v.abs(), -exponent[:, :, None])
    # nearest of 0, .5, 1, 1.5, 2, 3, 4, 6; halfway to the even code
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)).to(torch.uint8)
    code = code | ((v < 0).to(torch.uint8) << 3)
    return code.view(rows, blocks * BLOCK)[:, :cols], (exponent + 127).to(torch.uint8)


def _plain_values(code, scale):
    """What codes [rows, cols] and scale bytes stand for, in 32 bits."""
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device=code.device)
    s = scale.to(torch.int32).repeat_interleave(BLOCK, dim=1)[:, :code.shape[1]] - 127
    return torch.ldexp(table[code.to(torch.int32)], s)


def _plain_weight(parts, cols):
    packed, scale = parts
    code = torch.stack((packed & 15, packed >> 4), dim=2).view(packed.shape[0], -1)[:, :cols]
    return _plain_values(code, scale)


def _plain_product(x, parts):
    return _plain_values(*_plain_codes(x)) @ _plain_weight(parts, x.shape[1]).t()


def _plain_activation(g, name):
    if name == "silu":
        return g / (1 + torch.exp(-g))
    return 0.5 * g * (1 + torch.tanh(0.7978845608028654 * (g + 0.044715 * g * g * g)))


def _plain_norm(x, weight):
    x = x.float()
    return x * torch.rsqrt((x * x).mean(dim=1, keepdim=True) + EPS) * weight.float()


def _plain_join(y, h, s, alpha, dtype):
    t = y.float() if s["post_weight"] is None else _plain_norm(y, s["post_weight"])
    t = t if s["g"] is None else t * s["g"].float()
    joined = alpha * h.float() + t
    return joined.to(h.dtype), _plain_norm(joined, s["next_weight"]).to(dtype)


def _plain(s):
    kind = s["kind"]
    if kind == "quantize":
        return _plain_values(*_plain_codes(s["x"])).to(s["x"].dtype)
    if kind == "linear":
        return _plain_product(s["x"], s["weights"][0]).to(s["x"].dtype)
    if kind == "gated":
        g, u = (_plain_product(s["x"], w) for w in s["weights"])
        return (_plain_activation(g, s["activation"]) * u).to(s["x"].dtype)
    if kind == "join":
        return _plain_join(s["y"], s["h"], s, s["alpha"], s["y"].dtype)
    x = _plain_norm(s["h"], s["pre_weight"])
    g, u = (_plain_product(x, w) for w in s["weights"][:2])
    y = _plain_product(_plain_activation(g, s["activation"]) * u, s["weights"][2])
    return _plain_join(y, s["h"], s, 1.0, s["h"].dtype)


# ---- the same in 64 bits, from the definitions -------------------------------------------------------

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _exact_round(x):
    """Every block of 32 columns to the nearest multiples of its scale that E2M1 has."""
    x = x.double()
    out = torch.empty_like(x)
    full = x.shape[1] // BLOCK * BLOCK
    for lo, hi, width in ((0, full, BLOCK), (full, x.shape[1], x.shape[1] - full)):
        if hi == lo:
            continue
        v = x[:, lo:hi].reshape(x.shape[0], -1, width)
        m = v.abs().amax(dim=2, keepdim=True)
        _, e = torch.frexp(m)                       # m = f 2^e, f in [1/2, 1)
        e = torch.where(m > 0, e - 3, torch.full_like(e, -127)).clamp(min=-127)
        grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
        a = torch.ldexp(v.abs(), -e)
        up = torch.bucketize(a, grid).clamp(max=7)  # first grid value that is not below a
        down = (up - 1).clamp(min=0)
        over, under = grid[up] - a, a - grid[down]
        even = torch.where(up % 2 == 0, up, down)
        pick = torch.where(over < under, up, torch.where(under < over, down, even))
        pick = torch.where(a >= 6, torch.full_like(pick, 7), pick)
        out[:, lo:hi] = (torch.ldexp(grid[pick], e) * torch.sign(v)).reshape(x.shape[0], -1)
    return out


def _exact_weight(parts, cols):
    packed, scale = parts
    value = torch.tensor(GRID + tuple(-v for v in GRID), dtype=torch.float64, device=packed.device)
    w = torch.empty((packed.shape[0], packed.shape[1] * 2), dtype=torch.float64, device=packed.device)
    w[:, 0::2], w[:, 1::2] = value[(packed % 16).long()], value[(packed // 16).long()]
    w = w[:, :cols]
    column = torch.arange(cols, device=packed.device) // BLOCK
    return w * torch.pow(2.0, scale.double() - 127)[:, column]


def _exact_activation(g, name):
    return g * torch.sigmoid(g) if name == "silu" else g * 0.5 * (1 + torch.tanh((2 / math.pi) ** 0.5 * (g + 0.044715 * g ** 3)))


def _exact_norm(x, weight):
    return x / ((x ** 2).mean(dim=1, keepdim=True) + EPS).sqrt() * weight.double()


def _exact_join(y, h, s, alpha):
    t = y if s["post_weight"] is None else _exact_norm(y, s["post_weight"])
    t = alpha * h + (t if s["g"] is None else t * s["g"].double())
    return t, _exact_norm(t, s["next_weight"])


def exact(case, seed):
    global own
    was, own = own, False      # the inputs, without this repository's code
    try:
        s = prepare(case, seed)
    finally:
        own = was
    kind = case["kind"]
    if kind == "quantize":
        return _exact_round(s["x"])
    if kind == "linear":
        return _exact_round(s["x"]) @ _exact_weight(s["weights"][0], case["cols"]).t()
    if kind == "gated":
        x = _exact_round(s["x"])
        g, u = (x @ _exact_weight(w, case["cols"]).t() for w in s["weights"])
        return _exact_activation(g, case["activation"]) * u
    if kind == "join":
        return _exact_join(s["y"].double(), s["h"].double(), s, case["alpha"])
    h = s["h"].double()
    x = _exact_round(_exact_norm(h, s["pre_weight"]))
    g, u = (x @ _exact_weight(w, case["hidden"]).t() for w in s["weights"][:2])
    a = _exact_round(_exact_activation(g, case["activation"]) * u)
    return _exact_join(a @ _exact_weight(s["weights"][2], case["inter"]).t(), h, s, 1.0)


# ---- the work of a pass ------------------------------------------------------------------------------

def work(case):
    """Every input read once, every output written once; what passes between the parts of a block is neither."""
    kind = case["kind"]
    size = BYTES[case["dtype"]]
    if kind == "quantize":
        return {"bytes": int(case["rows"] * case["cols"] * 2 * size), "flops": 0}
    if kind in ("linear", "gated"):
        t, k, n = case["tokens"], case["cols"], case["rows"]
        halves = 2 if kind == "gated" else 1
        return {"bytes": int(halves * n * k * BITS + t * (k + n) * size), "flops": 2 * halves * t * n * k}
    if kind == "join":
        t, d = case["tokens"], case["cols"]
        gate = {"none": 0, "channel": d, "token": t, "full": t * d}[case["gate"]]
        return {"bytes": int(2 * t * d * (size + BYTES[case["stream"]]) + gate * size + 2 * d * (1 + case["post"])), "flops": 0}
    t, d, i = case["tokens"], case["hidden"], case["inter"]
    return {"bytes": int(3 * d * i * BITS + 3 * t * d * size + 8 * d), "flops": 6 * t * d * i}
