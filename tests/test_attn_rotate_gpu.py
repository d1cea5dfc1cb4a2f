"""Norms and rotation of heads, and the step's keys and values in the cache, against the formula in 64 bits."""
import pytest
import torch

from mpserve_b200 import attention
from tests import _attn as ref

pytestmark = pytest.mark.gpu
EPS = 1e-6


def _heads(g, tokens, heads, dim, dtype):
    """Views of one projection's rows: queries, keys, values."""
    x = ref.randn(g, tokens, sum(heads), dim, dtype=dtype)
    return x.split(heads, dim=1)


def _weights(g, dim, dtype=torch.bfloat16):
    return [(1 + 0.1 * ref.randn(g, dim)).to(dtype) for _ in range(2)]


def _check(got, x, weight, positions, rotary, frequencies, axes=None):
    ref.within(got, *ref.rotated(x, weight, positions, frequencies, axes, rotary.interleaved, rotary.scale, EPS))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim,turned", [(128, 128), (64, 64), (256, 256), (256, 64), (128, 64), (80, 32), (96, 96), (16, 16), (8, 0), (34, 10), (7, 6), (1, 0)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens", [1, 5, 200])
def test_norms_and_rotation(dtype, dim, turned, interleaved, tokens):
    g = ref.generator(dim + turned + tokens)
    q, k, _ = _heads(g, tokens, (5, 2, 2), dim, ref.TYPES[dtype])
    qw, kw = _weights(g, dim)
    positions = torch.randint(0, 5000, (tokens,), generator=g, device="cuda")
    frequencies = torch.rand((turned // 2,), generator=g, device="cuda", dtype=torch.float64)
    rotary = attention.Rotary(turned, frequencies=frequencies, interleaved=interleaved, scale=1.25)
    q_new, k_new = attention.norm_rotate(q, k, positions, rotary, q_weight=qw, k_weight=kw, eps=EPS)
    assert q_new.is_contiguous() and k_new.is_contiguous() and q_new.dtype == q.dtype
    _check(q_new, q, qw, positions, rotary, frequencies)
    _check(k_new, k, kw, positions, rotary, frequencies)


@pytest.mark.parametrize("heads", [(1, 1), (32, 8), (64, 8), (40, 40), (100, 3), (512, 512)])
@pytest.mark.parametrize("tokens", [1, 149, 400])
def test_numbers_of_heads(heads, tokens):
    g = ref.generator(sum(heads) + tokens)
    q, k = (ref.randn(g, tokens, n, 128, dtype=torch.bfloat16) for n in heads)
    qw, kw = _weights(g, 128, torch.float32)
    positions = torch.arange(tokens, device="cuda", dtype=torch.int32)
    rotary = attention.Rotary(128, base=500000.0)
    frequencies = 500000.0 ** (torch.arange(0, 128, 2, device="cuda", dtype=torch.float64) / -128)
    q_new, k_new = attention.norm_rotate(q, k, positions, rotary, q_weight=qw, k_weight=kw, eps=EPS)
    _check(q_new, q, qw, positions, rotary, frequencies)
    _check(k_new, k, kw, positions, rotary, frequencies)


@pytest.mark.parametrize("which", ["none", "q", "k"])
def test_without_norms(which):
    g = ref.generator(4)
    q, k, _ = _heads(g, 9, (4, 2, 2), 64, torch.float16)
    qw, kw = _weights(g, 64)
    qw, kw = qw if which == "q" else None, kw if which == "k" else None
    positions = torch.randint(0, 100, (9,), generator=g, device="cuda")
    rotary = attention.Rotary(64)
    frequencies = 10000.0 ** (torch.arange(0, 64, 2, device="cuda", dtype=torch.float64) / -64)
    q_new, k_new = attention.norm_rotate(q, k, positions, rotary, q_weight=qw, k_weight=kw, eps=EPS)
    _check(q_new, q, qw, positions, rotary, frequencies)
    _check(k_new, k, kw, positions, rotary, frequencies)


@pytest.mark.parametrize("far", [1 << 20, 1 << 31, 1 << 40])
def test_far_and_negative_positions(far):
    # with FP32 angles the result would have nothing to do with the formula's
    g = ref.generator(far)
    q, k, _ = _heads(g, 50, (3, 1, 1), 128, torch.float32)
    positions = torch.randint(-far, far, (50,), generator=g, device="cuda")
    frequencies = 10000.0 ** (torch.arange(0, 128, 2, device="cuda", dtype=torch.float64) / -128)
    rotary = attention.Rotary(128, frequencies=frequencies)
    q_new, k_new = attention.norm_rotate(q, k, positions, rotary)
    # the 64-bit angle itself, position times frequency, is off by far 2^-53, and so are the turns
    slack = 8 * far * 2.0 ** -53
    for new, x in ((q_new, q), (k_new, k)):
        want, off = ref.rotated(x, None, positions, frequencies, None, False, 1.0, EPS)
        ref.within(new, want, off + slack * 2 * x.double().abs().amax())


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("sections", [(16, 24, 24), (64, 0, 0), (0, 1, 63)])
def test_several_axes(interleaved, sections):
    g = ref.generator(sum(sections[:2]))
    q, k, _ = _heads(g, 70, (4, 2, 2), 128, torch.bfloat16)
    positions = torch.randint(0, 3000, (3, 70), generator=g, device="cuda")
    frequencies = 1000.0 ** (torch.arange(0, 128, 2, device="cuda", dtype=torch.float64) / -128)
    rotary = attention.Rotary(128, frequencies=frequencies, sections=sections, interleaved=interleaved)
    axes = [i for i, n in enumerate(sections) for _ in range(n)]
    q_new, k_new = attention.norm_rotate(q, k, positions, rotary)
    _check(q_new, q, None, positions, rotary, frequencies, axes)
    _check(k_new, k, None, positions, rotary, frequencies, axes)
    mixed = [j % 3 for j in range(64)]
    rotary = attention.Rotary(128, frequencies=frequencies, axes=mixed, interleaved=interleaved)
    _check(attention.norm_rotate(q, k, positions, rotary)[0], q, None, positions, rotary, frequencies, mixed)


def test_one_row_of_positions_serves_one_axis():
    g = ref.generator(8)
    q, k, _ = _heads(g, 6, (2, 1, 1), 32, torch.bfloat16)
    positions = torch.randint(0, 100, (6,), generator=g, device="cuda")
    rotary = attention.Rotary(32, axes=[0] * 16)
    a = attention.norm_rotate(q, k, positions, rotary)
    b = attention.norm_rotate(q, k, torch.stack((positions, positions + 7)), rotary)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("dim,page,dtype", [(128, 16, "bf16"), (64, 1, "f16"), (72, 64, "bf16"), (10, 8, "f32"), (256, 32, "f32")])
@pytest.mark.parametrize("permuted", [False, True])
@pytest.mark.parametrize("tokens", [1, 60])
def test_appended(dim, page, dtype, permuted, tokens):
    if dim == 10 and permuted:
        pytest.skip("rows of ten values keep no alignment")
    g, kind, pages, width = ref.generator(dim + tokens), ref.TYPES[dtype], 70, -(-dim // 8) * 8
    q, k, v = _heads(g, tokens, (6, 2, 2), dim, kind)
    qw, kw = _weights(g, dim)
    shape = (pages, 2, page, width) if permuted else (pages, page, 2, width)
    stores = [ref.randn(g, *shape, dtype=kind) for _ in range(2)]
    before = [t.clone() for t in stores]
    view = lambda t: (t.transpose(1, 2) if permuted else t)[..., :dim]  # noqa: E731
    cache = attention.KvCache(*(view(t) for t in stores))
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens]
    if tokens > 3:
        slots[0], slots[1], slots[2] = -1, pages * page, 1 << 40
    positions = torch.randint(0, 5000, (tokens,), generator=g, device="cuda")
    turned = dim // 2 // 2 * 2
    rotary = attention.Rotary(turned)
    q_new = attention.norm_rotate_append(q, k, v, positions, rotary, cache, slots, q_weight=qw, k_weight=kw, eps=EPS)
    want_q, want_k = attention.norm_rotate(q, k, positions, rotary, q_weight=qw, k_weight=kw, eps=EPS)
    ref.within(want_k, *ref.rotated(k, kw, positions, 10000.0 ** (torch.arange(0, turned, 2, device="cuda", dtype=torch.float64) / -max(turned, 1)), None, False, 1.0, EPS))
    assert torch.equal(q_new, want_q)
    # every other place keeps what it had
    for store, old, new in ((stores[0], before[0], want_k), (stores[1], before[1], v)):
        for t in range(tokens):
            if 0 <= slots[t] < pages * page:
                view(old)[slots[t] // page, slots[t] % page] = new[t]
        assert torch.equal(store, old)


def test_replayed_and_on_another_stream():
    g = ref.generator(2)
    q, k, v = _heads(g, 8, (4, 2, 2), 128, torch.bfloat16)
    positions, slots = torch.arange(8, device="cuda"), torch.arange(8, device="cuda")
    rotary, cache = attention.Rotary(128), attention.KvCache(*(torch.zeros((2, 16, 2, 128), dtype=torch.bfloat16, device="cuda") for _ in range(2)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q_new = attention.norm_rotate_append(q, k, v, positions, rotary, cache, slots)
    for step in range(3):
        positions.add_(1000 * step)
        slots.add_(step)
        graph.replay()
        want_q, want_k = attention.norm_rotate(q, k, positions, rotary)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            side_q, _ = attention.norm_rotate(q, k, positions, rotary)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(q_new, want_q) and torch.equal(side_q, want_q)
        assert torch.equal(cache.k_pages.flatten(0, 1)[slots], want_k) and torch.equal(cache.v_pages.flatten(0, 1)[slots], v)


def test_a_cache_beyond_32_bit_offsets():
    pages, page, heads, dim = 70000, 64, 4, 128      # 2.3 G values each
    stores = [torch.zeros((pages, page, heads, dim), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    g = ref.generator(6)
    q, k, v = _heads(g, 4, (4, 4, 4), dim, torch.bfloat16)
    slots = torch.tensor([0, pages * page - 1, pages * page // 2 + 3, pages * page - 64], device="cuda")
    positions, rotary = torch.arange(4, device="cuda"), attention.Rotary(dim)
    attention.norm_rotate_append(q, k, v, positions, rotary, attention.KvCache(*stores), slots)
    _, want = attention.norm_rotate(q, k, positions, rotary)
    assert torch.equal(stores[0].flatten(0, 1)[slots], want) and torch.equal(stores[1].flatten(0, 1)[slots], v)


def test_no_tokens():
    rotary, none = attention.Rotary(64), torch.empty((0, 2, 64), dtype=torch.bfloat16, device="cuda")
    cache = attention.KvCache(*(torch.zeros((2, 16, 2, 64), dtype=torch.bfloat16, device="cuda") for _ in range(2)))
    empty = torch.empty((0,), dtype=torch.int64, device="cuda")
    assert attention.norm_rotate(none, none, empty, rotary)[0].shape == (0, 2, 64)
    assert attention.norm_rotate_append(none, none, none, empty, rotary, cache, empty).shape == (0, 2, 64)
