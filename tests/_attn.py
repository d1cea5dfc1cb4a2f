"""INT4 products, head norms with rotation and attention behind a shared prefix in 64 bits, from their formulas, and how far FP32 arithmetic may be from them."""
import math

import torch

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
# half the distance of neighbouring numbers, relative
ROUND = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
# half the distance of a type's smallest numbers
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}
STEP = 2.0 ** -24


def generator(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def within(got: torch.Tensor, want: torch.Tensor, off: torch.Tensor) -> None:
    """``got`` is ``want``, off by at most ``off`` before it was rounded to its type."""
    assert got.shape == want.shape
    most = off + ROUND[got.dtype] * (want.abs() + off) + TINY[got.dtype]
    far = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    assert (far <= most).all(), f"{(far / most).max().item():.3g} times what rounding explains"


# ---- INT4 -----------------------------------------------------------------------------------------

def int4_parts(g, rows: int, cols: int, group: int, zeros: bool = True, scale_dtype=torch.float16):
    groups = -(-cols // group)
    codes = torch.randint(0, 16, (rows, cols), generator=g, device="cuda", dtype=torch.uint8)
    scales = ((torch.rand((rows, groups), generator=g, device="cuda") + 0.5) * 0.01).to(scale_dtype)
    return codes, scales, torch.randint(0, 16, (rows, groups), generator=g, device="cuda", dtype=torch.uint8) if zeros else None


def int4_values(codes, scales, zeros, group: int) -> torch.Tensor:
    """In 64 bits."""
    column = torch.arange(codes.shape[1], device=codes.device) // group
    zero = 8.0 if zeros is None else zeros.double()[:, column]
    return (codes.double() - zero) * scales.double()[:, column]


def int4_off(x, values, group: int) -> torch.Tensor:
    """A product's error: a multiplication adds 16 products to a sum, each off by at most one step of the largest, group / 16 times (a half group of 32 columns
    likewise); groups and the eight warps' parts are then added one by one."""
    steps = 17 * (max(group, 32) // 16) + -(-values.shape[1] // group) + 10
    return steps * STEP * (x.double().abs() @ values.abs().t())


# ---- norms and rotation -----------------------------------------------------------------------------

def rotated(x, weight, positions, frequencies, axes, interleaved, scale, eps):
    """(values in 64 bits, how far FP32's may be)."""
    x = x.double()
    dim, pairs = x.shape[2], frequencies.numel()
    off = torch.zeros_like(x)
    if weight is not None:
        x = x / (x.pow(2).mean(dim=2, keepdim=True) + eps).sqrt() * weight.double()
        off = x.abs() * (dim + 8) * STEP      # `dim` additions under a root, the root, three products
    positions = positions.view(-1, x.shape[0])
    axis = torch.tensor([0] * pairs if axes is None else axes, device=x.device, dtype=torch.long)
    angle = (positions[axis].double() * frequencies.double()[:, None]).t()[:, None]
    first = torch.arange(pairs, device=x.device) * (2 if interleaved else 1)
    second = first + (1 if interleaved else pairs)
    a, b = x[:, :, first], x[:, :, second]
    out, far = x.clone(), off.clone()
    out[:, :, first] = scale * (a * angle.cos() - b * angle.sin())
    out[:, :, second] = scale * (b * angle.cos() + a * angle.sin())
    # the angle is rounded to FP32 (half a turn at most: 2 pi 2^-26), sine and cosine are off by a step or two, and there are two products and a sum
    both = abs(scale) * (off[:, :, first] + off[:, :, second] + (a.abs() + b.abs()) * 10 * STEP)
    far[:, :, first] = far[:, :, second] = both
    return out, far


# ---- attention ----------------------------------------------------------------------------------------

def attend(q, k_pages, v_pages, tables, lengths, prefix_table=None, prefix_length=0, scale=None):
    """(out, logarithms of the denominators, how far FP32 with weights in the cache's type may be from either), sequence by sequence, in 64 bits."""
    batch, heads, dim = q.shape
    pages, page, kv_heads, _ = k_pages.shape
    scale = dim ** -0.5 if scale is None else scale
    out, far = (torch.zeros((batch, heads, dim), dtype=torch.float64, device=q.device) for _ in range(2))
    lse, lse_far = torch.full((batch, heads), -math.inf, dtype=torch.float64, device=q.device), torch.zeros((batch, heads), dtype=torch.float64, device=q.device)
    slot = torch.arange(page, device=q.device)
    for b in range(batch):
        at = []
        for table, n in ((prefix_table, prefix_length), (tables[b], max(0, min(int(lengths[b]), tables.shape[1] * page)))):
            if n:
                number = table.long()[:-(-n // page), None].expand(-1, page).reshape(-1)[:n]
                place = slot.repeat(-(-n // page))[:n]
                there = (number >= 0) & (number < pages)
                at.append((number[there], place[there]))
        if not at or not sum(n.numel() for n, _ in at):
            continue
        number, place = (torch.cat([pair[i] for pair in at]) for i in range(2))
        k, v = (t[number, place].double().repeat_interleave(heads // kv_heads, dim=1) for t in (k_pages, v_pages))
        logit = torch.einsum("hd,nhd->hn", q[b].double(), k) * scale
        size = torch.einsum("hd,nhd->hn", q[b].double().abs(), k.abs()) * abs(scale)
        lse[b] = torch.logsumexp(logit, dim=1)
        weight = torch.exp(logit - lse[b][:, None])
        out[b] = torch.einsum("hn,nhd->hd", weight, v)
        # a logit: dim / 16 additions of 16 products each, a scaling, the difference to the largest one; the exponential two steps
        shift = ((17 * dim / 16 + 4) * STEP * size + 4 * STEP * (logit - logit.amax(dim=1, keepdim=True)).abs() + 4 * STEP).amax(dim=1)
        keys = logit.shape[1]
        sums = (17 * keys / 16 + 40) * STEP      # of weights or weighted values, and of the parts
        relative = 2 * shift + 2 * sums
        far[b] = torch.einsum("hn,nhd->hd", weight, v.abs()) * (relative + ROUND[q.dtype])[:, None]
        lse_far[b] = relative + 4 * STEP * lse[b].abs()
    return out, lse, far, lse_far
