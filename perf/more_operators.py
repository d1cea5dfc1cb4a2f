"""What the performance of the attention half of a decoding step is measured on (``mpserve_b200.int4``, ``mpserve_b200.attention``).

A serving process multiplies a few tokens by INT4 weights (codes, a scale and a zero point per group of columns), normalises
the heads of queries and keys and rotates them by their positions, puts the step's keys and values into a paged cache, and
attends: every sequence to a long prefix that the whole batch shares (a system prompt, a document) and to tokens of its own.

Plain forms are elementary torch operations in 32 bits, angles in 64.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
EPS = 1e-6
BASE = 500000.0
# One 8B layer: hidden 4096, inter 14336, 32 query and 8 key heads of 128; a 70B layer split over 8 ranks: 8 query heads and one key head.
MOST_PRODUCT = 64 * 14336 * 4096
MOST_ELEMENTS = 8192 * 48 * 128
MOST_ATTENTION = 128 * 32 * 128 * (32768 + 1024)


def linear(name, tokens, cols, rows, group=128, dtype="bf16", zeros=True):
    return dict(name=name, kind="linear", tokens=tokens, cols=cols, rows=rows, group=group, dtype=dtype, zeros=zeros)


def rotate(name, tokens, q_heads, kv_heads, dim, dtype="bf16", rotated=None, axes=1, interleaved=False, norm=True, append=False, far=4096):
    """``far``: positions are below it.  ``append``: keys and values go into a cache."""
    return dict(name=name, kind="rotate", tokens=tokens, q_heads=q_heads, kv_heads=kv_heads, dim=dim, dtype=dtype, rotated=rotated or dim, axes=axes,
                interleaved=interleaved, norm=norm, append=append, far=far)


def attend(name, batch, prefix, most_own, q_heads, kv_heads, dim=128, page=16, dtype="bf16"):
    """``most_own``: every sequence has between one and so many tokens of its own."""
    return dict(name=name, kind="attend", batch=batch, prefix=prefix, most_own=most_own, q_heads=q_heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype)


def listed():
    return [
        # a lone conversation's token through the smallest projection of a layer: latency
        linear("linear_1x4096x1024", 1, 4096, 1024),
        # the same token through an MLP weight: the weight's bytes count
        linear("linear_1x4096x14336", 1, 4096, 14336),
        # odd in every direction, symmetric codes, half precision: a small model's projection
        linear("linear_7x1000x517_f16", 7, 1000, 517, 64, "f16", False),
        # a batch of conversations through an MLP weight
        linear("linear_64x14336x4096", 64, 14336, 4096),
        # one token's heads on their way into the cache: a launch and its host side
        rotate("rotate_1_append", 1, 32, 8, 128, append=True, far=131072),
        # a batch of conversations, half precision, far along
        rotate("rotate_64_append_f16", 64, 32, 8, 128, "f16", append=True, far=131072),
        # a small model's odd heads, a part of each rotated, neighbours paired, in 32 bits
        rotate("rotate_333_odd_f32", 333, 5, 3, 80, "f32", 32, 1, True),
        # a prompt of text and pictures: positions have a time, a height and a width
        rotate("rotate_8192_three_axes", 8192, 32, 8, 128, axes=3),
        # a few conversations that have just begun behind a system prompt
        attend("attend_4_behind_1024", 4, 1024, 64, 32, 8),
        # a tensor-parallel rank's heads of a 70B layer, ragged
        attend("attend_33_behind_5001_rank_f16", 33, 5001, 700, 8, 1, 128, 64, "f16"),
        # a batch of conversations about a document
        attend("attend_32_behind_8192", 32, 8192, 512, 32, 8),
        # many conversations about a long document: the tensor cores count, and the cache's bytes
        attend("attend_128_behind_32768", 128, 32768, 1024, 32, 8),
    ]


def _between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("linear", "rotate", "attend", "attend"))
    if kind == "linear":
        group = rng.choice((32, 64, 128, 128, 128))
        cols, rows = (max(s, _between(rng, 64, 14336) // s * s) for s in (rng.choice((128, 128, 32, 1)), rng.choice((128, 128, 16, 1))))
        tokens = _between(rng, 1, max(1, min(64, MOST_PRODUCT // (cols * rows))))
        return linear(None, tokens, cols, rows, group, rng.choice(("bf16", "bf16", "f16")), rng.random() < 0.75)
    if kind == "rotate":
        q_heads, kv_heads = rng.choice(((32, 8), (32, 8), (8, 1), (64, 8), (16, 16), (5, 1)))
        dim, dtype = rng.choice((128, 128, 64, 96, 256)), rng.choice(("bf16", "bf16", "f16", "f32"))
        append = rng.random() < 0.5
        dtype = "bf16" if append and dtype == "f32" else dtype
        most = MOST_ELEMENTS * 2 // BYTES[dtype] // (dim * (q_heads + (2 if append else 1) * kv_heads))
        return rotate(None, _between(rng, 1, most // 2 if append else most), q_heads, kv_heads, dim, dtype, rng.choice((dim, dim, dim // 2)),
                      rng.choice((1, 1, 3)), rng.random() < 0.3, rng.random() < 0.75, append, rng.choice((4096, 131072, 1 << 20)))
    q_heads, kv_heads = rng.choice(((32, 8), (32, 8), (8, 1), (64, 8), (16, 16), (12, 2)))
    dim, page, batch = rng.choice((128, 128, 64)), rng.choice((16, 16, 32, 64, 128)), _between(rng, 1, 128)
    most = MOST_ATTENTION // (batch * q_heads * dim)
    most_own = _between(rng, 1, min(2048, most))
    prefix = _between(rng, 1, max(1, min(32768, most - most_own)))
    return attend(None, batch, prefix, most_own, q_heads, kv_heads, dim, page, rng.choice(("bf16", "bf16", "f16")))


# ---- inputs -----------------------------------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _activations(g, shape, dtype):
    """Normal, with some channels far larger than the rest, as the streams of trained models have."""
    x = torch.randn(shape, generator=g, device="cuda")
    loud = torch.rand((shape[-1],), generator=g, device="cuda") < 0.01
    return (x * torch.where(loud, 12.0, 1.0)).to(DTYPES[dtype])


def _axes(case):
    """Which axis of the positions turns each pair: the first quarter time, then height and width in turn, or one for all."""
    pairs = case["rotated"] // 2
    if case["axes"] == 1:
        return [0] * pairs
    first = pairs // 4
    second = (pairs - first) // 2
    return [0] * first + [1] * second + [2] * (pairs - first - second)


def _pool(g, pages, page, kv_heads, dim, dtype):
    return torch.randn((pages, page, kv_heads, dim), generator=g, device="cuda", dtype=torch.float32).to(DTYPES[dtype])


def prepare(case, seed):
    g, s = _generator(seed), dict(case)
    kind = case["kind"]
    if kind == "linear":
        cols, rows, groups = case["cols"], case["rows"], -(-case["cols"] // case["group"])
        s["x"] = _activations(g, (case["tokens"], cols), case["dtype"])
        codes = (torch.randn((rows, cols), generator=g, device="cuda") * 2.5 + 8).round_().clamp_(0, 15).to(torch.uint8)
        scales = ((torch.rand((rows, groups), generator=g, device="cuda") + 0.5) * 0.008).to(torch.float16)
        zeros = torch.randint(5, 11, (rows, groups), generator=g, device="cuda", dtype=torch.uint8) if case["zeros"] else None
        if own:
            from mpserve_b200 import int4

            s["weight"] = int4.from_parts(codes, scales, zeros, group=case["group"])
        else:
            s["weight"] = (codes, scales, zeros)
    elif kind == "rotate":
        t, dim, q_heads, kv_heads = case["tokens"], case["dim"], case["q_heads"], case["kv_heads"]
        # views of one projection's rows
        heads = _activations(g, (t, (q_heads + 2 * kv_heads) * dim), case["dtype"]).view(t, q_heads + 2 * kv_heads, dim)
        s["q"], s["k"], s["v"] = heads.split((q_heads, kv_heads, kv_heads), dim=1)
        s["positions"] = torch.randint(0, case["far"], (case["axes"], t) if case["axes"] > 1 else (t,), generator=g, device="cuda")
        gains = [(1 + 0.1 * torch.randn((dim,), generator=g, device="cuda")).to(torch.bfloat16) for _ in range(2)]
        s["q_weight"], s["k_weight"] = gains if case["norm"] else (None, None)
        s["frequencies"] = BASE ** (torch.arange(0, case["rotated"], 2, device="cuda", dtype=torch.float64) / -case["rotated"])
        if case["append"]:
            pages = t // 16 + 1
            s["k_pages"], s["v_pages"] = (_pool(g, pages, 16, kv_heads, dim, case["dtype"]) for _ in range(2))
            s["slots"] = torch.randperm(pages * 16, generator=g, device="cuda")[:t]
        if own:
            from mpserve_b200 import attention

            s["rotary"] = attention.Rotary(case["rotated"], frequencies=s["frequencies"], axes=_axes(case), interleaved=case["interleaved"])
            if case["append"]:
                s["cache"] = attention.KvCache(s["k_pages"], s["v_pages"])
    else:
        b, page, dim, kv_heads = case["batch"], case["page"], case["dim"], case["kv_heads"]
        s["q"] = _activations(g, (b, case["q_heads"], dim), case["dtype"])
        per, shared = -(-case["most_own"] // page), -(-case["prefix"] // page)
        pages = per * b + shared
        s["k_pages"], s["v_pages"] = (_pool(g, pages, page, kv_heads, dim, case["dtype"]) for _ in range(2))
        order = torch.randperm(pages, generator=g, device="cuda", dtype=torch.int32)      # a pool that has been in use for a while
        s["prefix_table"], s["tables"] = order[:shared], order[shared:].view(b, per)
        s["lengths"] = torch.randint(1, case["most_own"] + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
        if own:
            from mpserve_b200 import attention

            s["cache"] = attention.KvCache(s["k_pages"], s["v_pages"])
    return s


# ---- a pass -----------------------------------------------------------------------------------------

def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    from mpserve_b200 import attention, int4

    if s["kind"] == "linear":
        return int4.linear(s["x"], s["weight"])
    if s["kind"] == "attend":
        return attention.shared_prefix_attention(s["q"], s["cache"], s["tables"], s["lengths"], prefix_table=s["prefix_table"], prefix_length=s["prefix"])
    if not s["append"]:
        return attention.norm_rotate(s["q"], s["k"], s["positions"], s["rotary"], q_weight=s["q_weight"], k_weight=s["k_weight"], eps=EPS)
    q = attention.norm_rotate_append(s["q"], s["k"], s["v"], s["positions"], s["rotary"], s["cache"], s["slots"], q_weight=s["q_weight"],
                                     k_weight=s["k_weight"], eps=EPS)
    return q, s["k_pages"], s["v_pages"]


def _plain_linear(s):
    codes, scales, zeros = s["weight"]
    groups = s["group"]
    wide = lambda t: t.float().repeat_interleave(groups, dim=1)[:, :s["cols"]]  # noqa: E731
    w = (codes.float() - (8.0 if zeros is None else wide(zeros))) * wide(scales)
    return (s["x"].float() @ w.t()).to(s["x"].dtype)


def _plain_heads(x, weight, cos, sin, rotated, interleaved):
    """[tokens, heads, dim] normalised and rotated, in 32 bits; cos and sin are [tokens, 1, pairs]."""
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(dim=2, keepdim=True) + EPS) * weight.float()
    turned, rest = x[:, :, :rotated], x[:, :, rotated:]
    if interleaved:
        a, b = turned[:, :, 0::2], turned[:, :, 1::2]
        return torch.cat((torch.stack((a * cos - b * sin, b * cos + a * sin), dim=3).flatten(2), rest), dim=2)
    a, b = turned[:, :, :rotated // 2], turned[:, :, rotated // 2:]
    return torch.cat((a * cos - b * sin, b * cos + a * sin, rest), dim=2)


def _plain_rotate(s):
    positions = s["positions"].view(s["axes"], -1)
    angle = positions[_axes(s)].t().double() * s["frequencies"]
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    q, k = (_plain_heads(s[n], s[n + "_weight"], cos, sin, s["rotated"], s["interleaved"]).to(s[n].dtype) for n in "qk")
    if not s["append"]:
        return q, k
    page, at = s["slots"] // 16, s["slots"] % 16
    s["k_pages"][page, at] = k
    s["v_pages"][page, at] = s["v"]
    return q, s["k_pages"], s["v_pages"]


def _plain_attend(s):
    b, heads, dim, prefix, page = s["batch"], s["kv_heads"], s["dim"], s["prefix"], s["page"]
    group, most = s["q_heads"] // heads, s["tables"].shape[1] * page
    q = s["q"].float().view(b, heads, group, dim) / math.sqrt(dim)
    # the prefix, once for all: [heads, batch * group, dim] by [heads, dim, prefix]
    shared_k, shared_v = (s[n][s["prefix_table"]].flatten(0, 1)[:prefix].float().transpose(0, 1) for n in ("k_pages", "v_pages"))
    own_k, own_v = (s[n][s["tables"]].flatten(1, 2).float().transpose(1, 2) for n in ("k_pages", "v_pages"))
    a = (q.transpose(0, 1).reshape(heads, b * group, dim) @ shared_k.transpose(1, 2)).view(heads, b, group, prefix).transpose(0, 1)
    c = q @ own_k.transpose(2, 3)
    beyond = torch.arange(most, device=c.device) >= s["lengths"][:, None]
    c = torch.where(beyond[:, None, None], -math.inf, c)
    top = torch.maximum(a.amax(dim=3, keepdim=True), c.amax(dim=3, keepdim=True))
    a, c = torch.exp(a - top), torch.exp(c - top)
    total = a.sum(dim=3, keepdim=True) + c.sum(dim=3, keepdim=True)
    out = (a.transpose(0, 1).reshape(heads, b * group, prefix) @ shared_v).view(heads, b, group, dim).transpose(0, 1) + c @ own_v
    return (out / total).reshape(b, s["q_heads"], dim).to(s["q"].dtype)


def _plain(s):
    return {"linear": _plain_linear, "rotate": _plain_rotate, "attend": _plain_attend}[s["kind"]](s)


# ---- the same in 64 bits, from the definitions -------------------------------------------------------

def _exact_linear(s):
    codes, scales, zeros = s["weight"]
    column = torch.arange(s["cols"], device=codes.device) // s["group"]
    zero = torch.full(scales.shape, 8, device=codes.device) if zeros is None else zeros
    w = (codes.double() - zero.double()[:, column]) * scales.double()[:, column]
    return s["x"].double() @ w.t()


def _exact_rotate(s):
    t, dim, rotated = s["tokens"], s["dim"], s["rotated"]
    pairs = rotated // 2
    positions = s["positions"].view(s["axes"], t)
    axis = torch.tensor(_axes(s), device=positions.device)
    angle = positions.double().index_select(0, axis) * s["frequencies"][:, None]      # [pairs, tokens]
    turn = torch.polar(torch.ones_like(angle), angle).t()[:, None]
    first = torch.arange(pairs, device=axis.device) * (2 if s["interleaved"] else 1)
    second = first + (1 if s["interleaved"] else pairs)
    done = []
    for name in "qk":
        x = s[name].double()
        if s[name + "_weight"] is not None:
            x = x / (x.pow(2).sum(dim=2, keepdim=True) / dim + EPS).sqrt() * s[name + "_weight"].double()
        z = torch.complex(x[:, :, first], x[:, :, second]) * turn
        x = x.clone()
        x[:, :, first], x[:, :, second] = z.real, z.imag
        done.append(x)
    if not s["append"]:
        return done[0], done[1]
    pools = []
    for pool, new in ((s["k_pages"], done[1]), (s["v_pages"], s["v"].double())):
        flat = pool.double().flatten(0, 1)
        flat[s["slots"]] = new
        pools.append(flat.view(pool.shape))
    return done[0], pools[0], pools[1]


def _exact_attend(s):
    b, heads, dim, prefix = s["batch"], s["kv_heads"], s["dim"], s["prefix"]
    group = s["q_heads"] // heads
    out = torch.empty((b, s["q_heads"], dim), dtype=torch.float64, device="cuda")
    flat = lambda name, h: s[name][:, :, h].double()  # noqa: E731
    for h in range(heads):
        k, v, q = flat("k_pages", h), flat("v_pages", h), s["q"][:, h * group:(h + 1) * group].double()
        pk, pv = (t[s["prefix_table"].long()].reshape(-1, dim)[:prefix] for t in (k, v))
        score = torch.einsum("bgd,pd->bgp", q, pk) / dim ** 0.5
        mine = torch.einsum("bgd,bld->bgl", q, k[s["tables"].long()].reshape(b, -1, dim)) / dim ** 0.5
        mine.masked_fill_((torch.arange(mine.shape[2], device="cuda")[None] >= s["lengths"][:, None])[:, None], -math.inf)
        p = torch.softmax(torch.cat((score, mine), dim=2), dim=2)
        out[:, h * group:(h + 1) * group] = (torch.einsum("bgp,pd->bgd", p[:, :, :prefix], pv) +
                                             torch.einsum("bgl,bld->bgd", p[:, :, prefix:], v[s["tables"].long()].reshape(b, -1, dim)))
    return out


def exact(case, seed):
    global own
    was, own = own, False      # the inputs, without this repository's code
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"linear": _exact_linear, "rotate": _exact_rotate, "attend": _exact_attend}[case["kind"]](s)


# ---- the work of a pass ------------------------------------------------------------------------------

def work(case):
    """Every input read once, every output written once; the tokens of their own that sequences have are counted at their mean."""
    size = BYTES[case["dtype"]]
    if case["kind"] == "linear":
        t, k, n = case["tokens"], case["cols"], case["rows"]
        groups = -(-k // case["group"])
        return {"bytes": int(n * k / 2 + n * groups * (2.5 if case["zeros"] else 2) + t * (k + n) * size), "flops": 2 * t * n * k}
    if case["kind"] == "rotate":
        heads = case["q_heads"] + (2 if case["append"] else 1) * case["kv_heads"]
        return {"bytes": int(2 * case["tokens"] * heads * case["dim"] * size), "flops": 0}
    b, dim, heads, tokens = case["batch"], case["dim"], case["q_heads"], case["batch"] * (case["most_own"] + 1) / 2
    return {"bytes": int(2 * (case["prefix"] + tokens) * case["kv_heads"] * dim * size + 2 * b * heads * dim * size),
            "flops": int(4 * heads * dim * (b * case["prefix"] + tokens))}
