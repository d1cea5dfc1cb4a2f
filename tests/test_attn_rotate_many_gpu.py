"""Norms, rotation and the cache for more tokens than CTAs are given one each, against the formula in 64 bits."""
import pytest
import torch

from mpserve_b200 import attention
from tests import _attn as ref

pytestmark = pytest.mark.gpu

EPS = 1e-6


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim,turned,heads", [(128, 128, (32, 8)), (64, 64, (7, 7)), (256, 64, (4, 2)), (128, 64, (1, 1)), (80, 32, (3, 1)), (34, 10, (2, 2))])
@pytest.mark.parametrize("tokens", [888, 889, 1500, 4097])
def test_many_tokens(dtype, dim, turned, heads, tokens):
    g, kind, page = ref.generator(dim + tokens), ref.TYPES[dtype], 16
    q, k, v = ref.randn(g, tokens, heads[0] + 2 * heads[1], dim, dtype=kind).split((heads[0], heads[1], heads[1]), dim=1)
    qw, kw = ((1 + 0.1 * ref.randn(g, dim)).to(torch.bfloat16) for _ in range(2))
    positions = torch.randint(0, 100000, (3, tokens), generator=g, device="cuda")
    frequencies = torch.rand((turned // 2,), generator=g, device="cuda", dtype=torch.float64)
    axes = [j % 3 for j in range(turned // 2)]
    rotary = attention.Rotary(turned, frequencies=frequencies, axes=axes, interleaved=tokens % 2 == 1)
    q_new, k_new = attention.norm_rotate(q, k, positions, rotary, q_weight=qw, k_weight=kw, eps=EPS)
    for got, x, w in ((q_new, q, qw), (k_new, k, kw)):
        ref.within(got, *ref.rotated(x, w, positions, frequencies, axes, rotary.interleaved, 1.0, EPS))
    pages, width = -(-tokens // page) + 2, -(-dim // 8) * 8
    stores = [ref.randn(g, pages, page, heads[1], width, dtype=kind) for _ in range(2)]
    want = [t.clone() for t in stores]
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens]
    slots[5] = -1
    cache = attention.KvCache(*(t[..., :dim] for t in stores))
    again = attention.norm_rotate_append(q, k, v, positions, rotary, cache, slots, q_weight=qw, k_weight=kw, eps=EPS)
    assert torch.equal(again, q_new)
    there = slots >= 0
    for store, old, new in ((stores[0], want[0], k_new), (stores[1], want[1], v)):
        old[slots[there] // page, slots[there] % page, :, :dim] = new[there]
        assert torch.equal(store, old)
