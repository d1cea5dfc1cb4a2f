"""Softmax weights far below a row's largest, in a cache of 16-bit types."""
import pytest
import torch

from mpserve_b200 import attention
from tests import _attn as ref

pytestmark = pytest.mark.gpu


def _call(q, k, v, where, keys, page=16):
    """``keys`` keys of pages in order, as a prefix or as every sequence's own; scale 1."""
    batch = q.shape[0]
    table = torch.arange(-(-keys // page), dtype=torch.int32, device="cuda")
    if where == "prefix":
        tables, lengths = torch.zeros((batch, 0), dtype=torch.int32, device="cuda"), torch.zeros(batch, dtype=torch.int32, device="cuda")
        shared = dict(prefix_table=table, prefix_length=keys)
    else:
        tables, lengths = table.expand(batch, -1).contiguous(), torch.full((batch,), keys, dtype=torch.int32, device="cuda")
        shared = {}
    got = attention.shared_prefix_attention(q, attention.KvCache(k, v), tables, lengths, scale=1.0, return_lse=True, **shared)
    return got, (tables, lengths, shared.get("prefix_table"), shared.get("prefix_length", 0))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("where,keys", [("prefix", 100), ("prefix", 1000), ("own", 60), ("own", 1000)])
@pytest.mark.parametrize("nats", [10, 16, 17, 20, 24])
@pytest.mark.parametrize("place", [0, 37, -1])
def test_one_key_that_dominates_and_has_no_value(dtype, where, keys, nats, place):
    # 74 key heads: a head's prefix has two stretches
    g, kind, heads, page = ref.generator(nats + keys), ref.TYPES[dtype], 74, 16
    shape = (-(-keys // page), page, heads, 64)
    k, v = ref.randn(g, *shape, dtype=kind), (1000 + 100 * ref.randn(g, *shape)).to(kind)
    k[..., 0] = torch.rand(shape[:3], generator=g, device="cuda") * 0.5 - 0.25      # the other keys' logits
    at = place % keys
    k[at // page, at % page, :, 0], v[at // page, at % page] = nats, 0
    q = torch.zeros((2, heads, 64), dtype=kind, device="cuda")
    q[..., 0] = 1
    (out, lse), rest = _call(q, k, v, where, keys)
    want, want_lse, off, lse_off = ref.attend(q, k, v, *rest, 1.0)
    if dtype == "f16":
        # A weight is rounded by half an F16 step: 2^-11 of itself, counted in `off`, or 2^-25 where it is subnormal.  The largest weight of those that are rounded
        # against one another is 2^12 at least, so the latter is 2^-37 of it, and it is at most 1 of the sum.
        mass = v.flatten(0, 1)[:keys].double().abs().sum(dim=0)
        off = off + 2.0 ** -37 * mass
    ref.within(out, want, off)
    assert ((lse.double() - want_lse).abs() <= lse_off + ref.STEP * want_lse.abs()).all()


@pytest.mark.parametrize("dtype,size", [("f16", 2.0 ** 15), ("bf16", 2.0 ** 15), ("bf16", 2.0 ** 40)])
@pytest.mark.parametrize("where", ["prefix", "own"])
@pytest.mark.parametrize("sign", [1, -1])
def test_logits_with_no_digits_behind_the_point(dtype, size, where, sign):
    """Logits whose FP32 steps are far apart: one key has all the weight, and its value is the result."""
    g, kind, heads, page, keys = ref.generator(5), ref.TYPES[dtype], 8, 16, 300
    shape = (-(-keys // page), page, heads, 64)
    k, v = torch.zeros(shape, dtype=kind, device="cuda"), ref.randn(g, *shape, dtype=kind)
    others = -1 if sign == 1 else -1.5      # times the best one's, or below it
    k[..., 0] = others * size
    k[150 // page, 150 % page, :, 0] = sign * size
    q = torch.zeros((40, heads, 64), dtype=kind, device="cuda")
    q[..., 0] = ((torch.rand((40, heads), generator=g, device="cuda") + 0.9) * size).to(kind)
    q[7] = 0      # between such rows one whose keys have equal weights
    (out, lse), rest = _call(q, k, v, where, keys)
    best = v[150 // page, 150 % page]
    keep = [b for b in range(40) if b != 7]
    assert torch.equal(out[keep], best.expand(40, heads, 64)[keep])
    want = q[..., 0].double() * size * sign
    assert ((lse.double() - want).abs() <= 8 * ref.STEP * want.abs())[keep].all()
    want, want_lse, off, _ = ref.attend(q[7:8], k, v, rest[0][7:8], rest[1][7:8], rest[2], rest[3], 1.0)
    ref.within(out[7:8], want, off)
