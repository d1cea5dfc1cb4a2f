"""Attention behind a shared prefix for more tiles of rows and key heads than there are SMs, where the host settles who has what."""
import math

import pytest
import torch

from mpserve_b200 import attention
from tests import _attn as ref

pytestmark = pytest.mark.gpu


def _check(batch, q_heads, kv_heads, prefix, own, dim=64, page=16, dtype="bf16", look_at=None):
    g, kind = ref.generator(batch + q_heads + prefix), ref.TYPES[dtype]
    columns, shared = -(-own // page), -(-prefix // page)
    pages = 64 + shared      # sequences have pages in common
    k, v = (ref.randn(g, pages, page, kv_heads, dim, dtype=kind) for _ in range(2))
    q = ref.randn(g, batch, q_heads, dim, dtype=kind)
    tables = torch.randint(0, pages, (batch, columns), generator=g, device="cuda", dtype=torch.int32)
    lengths = torch.randint(0, own + 1, (batch,), generator=g, device="cuda", dtype=torch.int32)
    table = torch.randperm(pages, generator=g, device="cuda", dtype=torch.int32)[:shared].clone()
    out, lse = attention.shared_prefix_attention(q, attention.KvCache(k, v), tables, lengths, prefix_table=table, prefix_length=prefix, return_lse=True)
    at = list(range(batch)) if look_at is None else look_at
    want, want_lse, off, lse_off = ref.attend(q[at], k, v, tables[at], lengths[at], table, prefix)
    ref.within(out[at], want, off)
    assert (want_lse > -math.inf).all() and ((lse[at].double() - want_lse).abs() <= lse_off + ref.STEP * want_lse.abs()).all()
    assert out.isfinite().all() and lse.isfinite().all()


@pytest.mark.parametrize("heads", [146, 147, 148, 149, 160, 300])
@pytest.mark.parametrize("prefix", [1, 129, 500])
@pytest.mark.parametrize("own", [0, 100])
def test_heads_on_both_sides_of_the_number_of_sms(heads, prefix, own):
    _check(2, heads, heads, prefix, own)


@pytest.mark.parametrize("prefix", [1, 129, 700])
@pytest.mark.parametrize("own", [0, 90])
@pytest.mark.parametrize("batch,dim,dtype", [(1152, 128, "bf16"), (1200, 64, "f16"), (1217, 128, "bf16")])
def test_many_sequences(prefix, own, batch, dim, dtype):
    # a pair of tiles has 64 sequences: 18, 19 and 20 pairs for each of 8 key heads, the last of 1217 sequences with one tile
    _check(batch, 32, 8, prefix, own, dim, dtype=dtype, look_at=[*range(0, batch, 41), *range(batch - 3, batch)])


def test_a_wide_batch_with_long_sequences():
    _check(1300, 32, 8, 300, 3000, 128, look_at=[0, 1, 650, 1298, 1299])
