"""INT4 weights and their products on a GPU, against the formula in 64 bits."""
import pytest
import torch

from mpserve_b200 import int4
from tests import _attn as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows,cols", [(1, 1), (16, 64), (17, 63), (5, 129), (130, 1000), (256, 512)])
@pytest.mark.parametrize("zeros", [True, False])
def test_values_come_back(group, rows, cols, zeros):
    codes, scales, z = ref.int4_parts(ref.generator(rows * cols), rows, cols, group, zeros)
    want = ref.int4_values(codes, scales, z, group)
    for s in (scales, scales.view(torch.uint16)):
        w = int4.from_parts(codes, s, z, group=group)
        assert w.shape == (rows, cols) and w.group == group
        assert torch.equal(w.dequantize(torch.float32).double(), want)      # 5 bits times 11: exact
    for dtype in (torch.bfloat16, torch.float16):
        assert torch.equal(w.dequantize(dtype), want.to(dtype))


def test_values_with_bfloat16_scales():
    codes, scales, z = ref.int4_parts(ref.generator(5), 40, 200, 64, True, torch.bfloat16)
    assert torch.equal(int4.from_parts(codes, scales, z, group=64).dequantize(torch.float32).double(), ref.int4_values(codes, scales, z, 64))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("tokens", [1, 2, 7, 8, 9, 16, 17, 31, 33, 64, 65, 130])
@pytest.mark.parametrize("rows,cols", [(16, 128), (37, 1000), (200, 2048)])
def test_products(dtype, group, tokens, rows, cols):
    g = ref.generator(tokens * rows + cols + group)
    parts = ref.int4_parts(g, rows, cols, group, tokens % 2 == 0)
    values = ref.int4_values(*parts, group)
    x = ref.randn(g, tokens, cols, dtype=ref.TYPES[dtype])
    y = int4.linear(x, int4.from_parts(*parts, group=group))
    assert y.dtype == x.dtype and y.shape == (tokens, rows)
    ref.within(y, x.double() @ values.t(), ref.int4_off(x, values, group))


@pytest.mark.parametrize("tokens,rows,cols", [(1, 1, 1), (3, 5, 7), (1, 14336, 4096), (8, 1024, 4096), (5, 300, 14336), (64, 129, 14336), (40, 4097, 520)])
def test_products_of_other_sizes(tokens, rows, cols):
    g = ref.generator(rows)
    parts = ref.int4_parts(g, rows, cols, 128)
    values = ref.int4_values(*parts, 128)
    x = ref.randn(g, tokens, cols, dtype=torch.bfloat16)
    w = int4.from_parts(*parts)
    ref.within(int4.linear(x, w), x.double() @ values.t(), ref.int4_off(x, values, 128))
    ref.within(int4.linear(x, w, dtype=torch.float16), x.double() @ values.t(), ref.int4_off(x, values, 128))


@pytest.mark.parametrize("tokens", [1, 3, 20, 50])
def test_rows_of_any_stride_and_alignment(tokens):
    g = ref.generator(tokens)
    parts = ref.int4_parts(g, 100, 333, 64)
    values = ref.int4_values(*parts, 64)
    w = int4.from_parts(*parts, group=64)
    wide = ref.randn(g, tokens, 1001, dtype=torch.float16)
    wide[:, 500:] = float("nan")      # what lies beside a row is not read as a part of it
    for first in (0, 1, 8, 100):
        x = wide[:, first:first + 333]
        ref.within(int4.linear(x, w), x.double() @ values.t(), ref.int4_off(x, values, 64))
    x = wide[:, 7:340].reshape(tokens, 1, 333).contiguous()
    assert int4.linear(x, w).shape == (tokens, 1, 100)


def test_no_tokens_and_memory_that_was_used_before():
    parts = ref.int4_parts(ref.generator(1), 50, 70, 32)
    w = int4.from_parts(*parts, group=32)
    assert int4.linear(torch.empty((0, 70), dtype=torch.bfloat16, device="cuda"), w).shape == (0, 50)
    x = ref.randn(ref.generator(2), 4, 70, dtype=torch.bfloat16)
    want = int4.linear(x, w)
    for _ in range(3):
        trash = torch.full((1 << 20,), float("nan"), device="cuda")
        del trash
        assert torch.equal(int4.linear(x, w), want)


def test_infinities_and_nans_stay_in_their_token():
    g = ref.generator(3)
    parts = ref.int4_parts(g, 40, 256, 128)
    w, x = int4.from_parts(*parts), ref.randn(g, 12, 256, dtype=torch.bfloat16)
    x[3, 17], x[9, 200] = float("nan"), float("inf")
    y = int4.linear(x, w)
    keep = [i for i in range(12) if i not in (3, 9)]
    assert y[3].isnan().all()
    code = parts[0][:, 200].int() - parts[2][:, 1].int()      # infinity times a weight, which may be 0
    assert torch.equal(y[9].isnan(), code == 0) and torch.equal(y[9][code != 0] > 0, code[code != 0] > 0)
    assert torch.equal(y[keep], int4.linear(x[keep], w))


@pytest.mark.parametrize("tokens", [1, 64])
def test_replayed_graphs_and_other_streams(tokens):
    g = ref.generator(tokens)
    parts = ref.int4_parts(g, 500, 1024, 128)
    w, x = int4.from_parts(*parts), ref.randn(g, tokens, 1024, dtype=torch.bfloat16)
    want = int4.linear(x, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = int4.linear(x, w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(on_side, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = int4.linear(x, w)
    fresh = ref.randn(g, tokens, 1024, dtype=torch.bfloat16)
    for new in (fresh, x):
        x.copy_(new)
        graph.replay()
        assert torch.equal(y, int4.linear(x, w))


def test_a_weight_beyond_32_bit_offsets():
    rows, cols = (1 << 20) + 5, 8192      # 4.25 GB
    g = ref.generator(9)
    codes = torch.randint(0, 16, (rows, cols), generator=g, device="cuda", dtype=torch.uint8)
    scales = torch.full((rows, cols // 128), 0.01, dtype=torch.float16, device="cuda")
    w = int4.from_parts(codes, scales)
    x = ref.randn(g, 2, cols, dtype=torch.bfloat16)
    y = int4.linear(x, w)
    for at in (slice(0, 100), slice(1 << 19, (1 << 19) + 50), slice(rows - 100, rows)):
        values = ref.int4_values(codes[at], scales[at], None, 128)
        ref.within(y[:, at], x.double() @ values.t(), ref.int4_off(x, values, 128))


def test_refusals():
    parts = ref.int4_parts(ref.generator(1), 8, 64, 32)
    w, x = int4.from_parts(*parts, group=32), torch.zeros((2, 64), dtype=torch.bfloat16, device="cuda")
    for call, match in ((lambda: int4.linear(x[:, :63], w), "columns"), (lambda: int4.linear(x.float(), w), "bfloat16 or float16"),
                        (lambda: int4.linear(x, w, dtype=torch.float32), "bfloat16 or float16"), (lambda: int4.linear(x.cpu(), w), "CUDA"),
                        (lambda: int4.linear(x.t()[:2], w), "unit stride|columns"), (lambda: int4.linear(x, parts[0]), "Int4Tensor"),
                        (lambda: int4.from_parts(parts[0] + 100, *parts[1:], group=32), "below 16"),
                        (lambda: int4.from_parts(*parts[:2], parts[2] + 16, group=32), "below 16"), (lambda: int4.from_parts(*parts, group=64), "shape"),
                        (lambda: int4.from_parts(parts[0].cpu(), *parts[1:], group=32), "CUDA"), (lambda: w.dequantize(torch.float64), "dtype")):
        with pytest.raises(ValueError, match=match):
            call()
