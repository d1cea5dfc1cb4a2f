"""Attention behind a prefix that a batch shares, against the formula in 64 bits."""
import math

import pytest
import torch

from mpserve_b200 import attention
from tests import _attn as ref

pytestmark = pytest.mark.gpu


def _case(seed, lengths, prefix, q_heads=8, kv_heads=2, dim=128, page=16, dtype="bf16", spare=3, columns=None):
    g, kind, batch = ref.generator(seed), ref.TYPES[dtype], len(lengths)
    columns = max(1, -(-max(lengths, default=0) // page)) if columns is None else columns
    shared = -(-prefix // page)
    pages = batch * columns + shared + spare
    k, v = (ref.randn(g, pages, page, kv_heads, dim, dtype=kind) for _ in range(2))
    order = torch.randperm(pages, generator=g, device="cuda", dtype=torch.int32)
    return dict(q=ref.randn(g, batch, q_heads, dim, dtype=kind), k=k, v=v, tables=order[shared:shared + batch * columns].view(batch, columns).clone(),
                lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"), prefix_table=order[:shared].clone(), prefix_length=prefix)


def _run(c, scale=None):
    return attention.shared_prefix_attention(c["q"], attention.KvCache(c["k"], c["v"]), c["tables"], c["lengths"], prefix_table=c["prefix_table"],
                                             prefix_length=c["prefix_length"], scale=scale, return_lse=True)


def _check(c, scale=None):
    out, lse = _run(c, scale)
    want, want_lse, off, lse_off = ref.attend(c["q"], c["k"], c["v"], c["tables"], c["lengths"], c["prefix_table"], c["prefix_length"], scale)
    assert out.dtype == c["q"].dtype and lse.dtype == torch.float32
    ref.within(out, want, off)
    none = want_lse == -math.inf
    assert torch.equal(lse == -math.inf, none) and (out[none] == 0).all()
    assert ((lse.double() - want_lse)[~none].abs() <= (lse_off + ref.STEP * want_lse.abs())[~none]).all()
    return out, lse


LENGTHS = [1, 0, 15, 16, 17, 64, 65, 127, 128, 129, 300, 1, 777]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q_heads,kv_heads", [(1, 1), (8, 2), (8, 8), (12, 2), (16, 1), (20, 1), (9, 3)])
@pytest.mark.parametrize("prefix", [0, 1, 1000])
def test_heads(dtype, dim, q_heads, kv_heads, prefix):
    _check(_case(q_heads + prefix, LENGTHS, prefix, q_heads, kv_heads, dim, dtype=dtype))


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 1024])
@pytest.mark.parametrize("prefix", [5, 128, 129, 2047])
def test_pages(page, prefix):
    _check(_case(page + prefix, LENGTHS, prefix, page=page))


@pytest.mark.parametrize("batch", [1, 2, 15, 16, 17, 31, 32, 33, 40, 64, 100, 300])
@pytest.mark.parametrize("prefix", [63, 4096, 5001])
def test_batches(batch, prefix):
    _check(_case(batch + prefix, [(7 * i * i) % 90 for i in range(batch)], prefix))


@pytest.mark.parametrize("prefix", [1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 191, 192, 193, 255, 256, 257, 383, 384, 385, 511, 513, 1023, 1025])
def test_lengths_of_the_prefix(prefix):
    _check(_case(prefix, [3] * 40, prefix, 4, 1))


@pytest.mark.parametrize("batch,q_heads,kv_heads", [(1, 4, 1), (3, 8, 8), (70, 8, 1), (70, 32, 8)])
def test_long_prefix(batch, q_heads, kv_heads):
    _check(_case(batch, [1 + i for i in range(batch)], 20000 + batch, q_heads, kv_heads))


def test_one_long_sequence_among_short_ones():
    _check(_case(1, [5, 40000, 3, 0, 1, 7], 0))
    _check(_case(2, [40000], 100, 32, 8))


def test_nothing_to_attend_to():
    c = _case(3, [0, 5, 0], 0)
    out, lse = _check(c)
    assert (out[0] == 0).all() and (out[2] == 0).all() and (lse[0] == -math.inf).all()
    c["lengths"].zero_()
    assert (_run(c)[0] == 0).all()
    c = _case(4, [0, 0], 0, columns=0)
    assert (_run(c)[0] == 0).all()
    c = _case(5, [0, 0], 50, columns=0)
    _check(c)
    empty = _case(6, [], 50)
    assert _run(empty)[0].shape == (0, 8, 128)


def test_lengths_out_of_range():
    c = _case(7, [40, 40, 40], 20)
    c["lengths"].copy_(torch.tensor([-5, 1 << 30, 33]))
    _check(c)


@pytest.mark.parametrize("prefix", [0, 70, 300])
def test_pages_outside_the_cache(prefix):
    c = _case(8, [100, 100, 16, 33], prefix)
    c["tables"][0, 2], c["tables"][1, 0], c["tables"][2, 0], c["tables"][3, 2] = -1, 1 << 30, -(1 << 31), c["k"].shape[0]
    if prefix:
        c["prefix_table"][1], c["prefix_table"][-1] = -1, c["k"].shape[0]
    _check(c)


@pytest.mark.parametrize("prefix", [10, 129, 300])
def test_what_lies_beyond_a_length_is_not_read_as_keys(prefix):
    lengths = [1, 17, 100, 31, 0, 64]
    c = _case(9, lengths, prefix, columns=8)
    want = _run(c)
    keep_k, keep_v = torch.zeros(c["k"].shape[:2], dtype=torch.bool, device="cuda"), None
    flat = keep_k.view(-1)
    for table, n in [(c["prefix_table"], prefix)] + [(c["tables"][b], n) for b, n in enumerate(lengths)]:
        at = torch.arange(n, device="cuda")
        flat[table.long()[at // 16] * 16 + at % 16] = True
    for bad in (float("nan"), float("inf"), -float("inf")):
        c["k"][~keep_k], c["v"][~keep_k] = bad, bad
        got = _run(c)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("where", ["prefix", "own"])
@pytest.mark.parametrize("bad", ["nan", "inf"])
def test_nans_and_infinities_in_what_is_attended_to(where, bad):
    c = _case(10, [20, 30, 40], 200)
    table = c["prefix_table"] if where == "prefix" else c["tables"][1]
    c["v"][table[1].long(), 3, 0, 5] = float(bad)
    out, lse = _run(c)
    touched = [0, 1, 2] if where == "prefix" else [1]
    for b in range(3):
        hit = out[b, :4, 5]
        assert ((hit.isnan() if bad == "nan" else hit.isinf()) if b in touched else hit.isfinite()).all()
    rest = out.clone()
    rest[:, :4, 5] = 0
    assert rest.isfinite().all() and lse.isfinite().all()
    # a query that is NaN gets NaN, the others what they had
    c = _case(11, [20, 30, 40], 200)
    want = _run(c)[0]
    c["q"][1, 2, 7] = float("nan")
    out, lse = _run(c)
    assert out[1, 2].isnan().all() and lse[1, 2].isnan()
    out[1, 2], want[1, 2] = 0, 0
    assert torch.equal(out, want)


@pytest.mark.parametrize("scale", [0.0, 1.0, -0.2, 5.0])
def test_scales(scale):
    # with 1 and 5 the largest logits lie far apart, parts of the keys weigh nothing
    _check(_case(12, [50, 100, 200], 500), scale)


def test_logits_that_grow_and_fall_along_the_keys():
    for sign in (1, -1):
        c = _case(13, [300] * 40, 3000, 8, 2)
        ramp = torch.linspace(0, 8 * sign, c["k"].shape[0], device="cuda").to(torch.bfloat16)
        c["prefix_table"] = torch.sort(c["prefix_table"])[0].contiguous()
        c["k"][..., 0] = ramp[:, None, None]
        c["q"][..., 0] = 6.0
        _check(c)


def test_views_of_queries_and_pages():
    c = _case(14, [30, 200, 5], 333)
    want = _run(c)[0]
    wide = ref.randn(ref.generator(1), 3, 20, 128, dtype=torch.bfloat16)
    wide[:, 4:12] = c["q"]
    c["q"] = wide[:, 4:12]
    assert torch.equal(_run(c)[0], want)
    # heads outside, both halves of one buffer
    both = torch.stack((c["k"], c["v"])).transpose(2, 3).contiguous()
    c["k"], c["v"] = both[0].transpose(1, 2), both[1].transpose(1, 2)
    assert torch.equal(_run(c)[0], want)


def test_a_captured_call_follows_lengths_and_tables():
    c = _case(15, [10, 20, 30, 0], 500, columns=20)
    cache = attention.KvCache(c["k"], c["v"])
    call = lambda: attention.shared_prefix_attention(c["q"], cache, c["tables"], c["lengths"], prefix_table=c["prefix_table"], prefix_length=500)  # noqa: E731
    call()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call())
        graphs.append(graph)
    for lengths in ([10, 20, 30, 0], [320, 0, 1, 319], [0, 0, 0, 0], [200, 200, 200, 200]):
        c["lengths"].copy_(torch.tensor(lengths))
        c["q"].normal_(generator=ref.generator(sum(lengths)))
        streams = [torch.cuda.Stream() for _ in graphs]
        for s, graph in zip(streams, graphs):      # both at once: they share nothing that either writes
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                graph.replay()
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        want = call()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


def test_the_same_call_gives_the_same_bits():
    c = _case(16, [100] * 50, 3000, 32, 8)
    first = _run(c)
    for _ in range(5):
        again = _run(c)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_a_cache_beyond_32_bit_offsets():
    pages, page, heads, dim = 40000, 128, 4, 128      # 2.6 G values each
    k, v = (torch.zeros((pages, page, heads, dim), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    g = ref.generator(6)
    used = torch.tensor([pages - 1, 1, pages // 2 + 7, 0, pages - 2, 3], dtype=torch.int32, device="cuda")
    for t in (k, v):
        t[used.long()] = ref.randn(g, 6, page, heads, dim, dtype=torch.bfloat16)
    c = dict(q=ref.randn(g, 2, 8, dim, dtype=torch.bfloat16), k=k, v=v, tables=used[:4].view(2, 2).clone(), lengths=torch.tensor([200, 130], dtype=torch.int32, device="cuda"),
             prefix_table=used[4:].clone(), prefix_length=250)
    _check(c)
