"""Products of MXFP4 matrices against 64 bits.

The operands' values are exact in 64 bits, and so are products of two.  A step of the tensor cores adds 64 products to an FP32
accumulator; taking each of its two blocks of 32 as one rounded or cut addition, a sum over ``cols`` is off by at most (cols / 32 + parts) 2^-23 of the sum of
magnitudes, parts being the pieces that several CTAs add up (at most 256).  The result rounds to its type.
"""
import numpy as np
import pytest
import torch

from mpserve_b200 import mx4
from tests import _mx4 as ref

pytestmark = pytest.mark.gpu


def _inputs(tokens, cols, rows, seed=0, dtype="bf16"):
    g = torch.Generator(device="cuda").manual_seed(seed * 1000003 + tokens * 9176 + cols * 31 + rows)
    x = torch.randn((tokens, cols), generator=g, device="cuda") * torch.exp2(torch.randint(-6, 6, (tokens, 1), generator=g, device="cuda").float())
    w = torch.randn((rows, cols), generator=g, device="cuda") * torch.exp2(torch.randint(-6, 6, (rows, 1), generator=g, device="cuda").float()) * 0.02
    return x.to(ref.TYPES[dtype]), mx4.quantize(w.to(torch.bfloat16))


def _values(q):
    return torch.from_numpy(ref.values(q)).cuda()


def _sum_off(x, w):
    return (x.abs() @ w.abs().t()) * ((x.shape[1] / 32 + 256) * 2.0 ** -23)


def _check(y, x, w, dtype):
    want = x @ w.t()
    off = _sum_off(x, w) + want.abs() * ref.ROUND[dtype] * (1 + 2.0 ** -8) + (2.0 ** -25 if dtype == torch.float16 else 0)
    assert y.dtype == dtype and y.shape == want.shape
    worst = ((y.double() - want).abs() / off.clamp_min(1e-300)).max().item()
    assert worst <= 1, worst


SIZES = [(1, 256, 128), (1, 64, 1), (1, 1, 3), (2, 33, 31), (1, 4096, 4096), (5, 255, 127), (16, 257, 129), (17, 512, 300), (31, 1000, 517), (32, 4096, 256),
         (33, 96, 1000), (64, 2048, 384), (65, 300, 260), (100, 4097, 130), (128, 256, 128), (129, 1024, 640), (256, 512, 256), (257, 770, 511), (333, 1000, 517),
         (512, 4096, 1024), (700, 256, 2000), (1025, 1280, 385), (2048, 512, 512), (1, 14336, 4096), (3, 20000, 40), (4, 32, 30000)]


@pytest.mark.parametrize("tokens,cols,rows", SIZES)
def test_linear(tokens, cols, rows):
    x, w = _inputs(tokens, cols, rows)
    ref.poison()
    y = mx4.linear(x, w)
    q = mx4.quantize(x)
    _check(y, _values(q), _values(w), torch.bfloat16)
    assert torch.equal(y, mx4.linear(q, w)), "a quantised input gives what the call quantises itself"
    assert torch.equal(y, mx4.linear(x, w)), "the same call again gives the same bits"
    assert mx4.product_timed_out() is False


# so many rows that a tile of the output is one CTA's, whose ring goes round several times over the columns
@pytest.mark.parametrize("tokens,cols,rows", [(1, 5000, 38000), (9, 8192, 20000), (16, 4097, 37900), (40, 3000, 38000), (64, 6144, 20000), (128, 4096, 19999)])
def test_linear_with_long_rows_in_one_cta(tokens, cols, rows):
    x, w = _inputs(tokens, cols, rows, 11)
    ref.poison()
    y = mx4.linear(x, w)
    q = mx4.quantize(x)
    pick = torch.randint(0, rows, (1500,), device="cuda")
    want = _values(q) @ _sampled(w, pick).t()
    off = _values(q).abs() @ _sampled(w, pick).abs().t() * ((cols / 32 + 256) * 2.0 ** -23) + want.abs() * ref.ROUND[torch.bfloat16] * (1 + 2.0 ** -8)
    assert ((y[:, pick].double() - want).abs() <= off).all()
    assert torch.equal(y, mx4.linear(q, w)) and torch.equal(y, mx4.linear(x, w))
    gated = mx4.gated_linear(x, w, w)
    assert torch.equal(gated, mx4.gated_linear(q, w, w))
    want, off = _gated_off(_values(q), _sampled(w, pick), _sampled(w, pick), "silu")
    assert ((gated[:, pick].double() - want).abs() <= off + want.abs() * ref.ROUND[torch.bfloat16] * (1 + 2.0 ** -8)).all()
    assert mx4.product_timed_out() is False


def _sampled(w, rows):
    """Some of a weight's rows, as values in 64 bits."""
    codes, scales = w.parts()
    return torch.from_numpy(ref.decode(ref.unpack(codes[rows].cpu().numpy(), w.cols), scales[rows].cpu().numpy())).cuda()


@pytest.mark.parametrize("tokens,cols,rows", [(1, 512, 300), (40, 1000, 129), (300, 640, 517)])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_linear_types(tokens, cols, rows, dtype):
    x, w = _inputs(tokens, cols, rows, 1, dtype)
    q = _values(mx4.quantize(x))
    _check(mx4.linear(x, w), q, _values(w), torch.bfloat16 if dtype == "f32" else torch.float16)
    _check(mx4.linear(x, w, dtype=torch.float16), q, _values(w), torch.float16)


def test_layouts_are_where_they_belong():
    """Weights that pick single columns: every element of x comes out at its place, exactly."""
    cols, tokens = 700, 300
    rng = np.random.default_rng(5)
    x = mx4.from_parts(torch.from_numpy(ref.pack(rng.integers(0, 16, (tokens, cols), dtype=np.uint8))).cuda(),
                       torch.from_numpy(rng.integers(120, 134, (tokens, 22), dtype=np.uint8)).cuda(), cols)
    pick = torch.eye(cols, device="cuda").to(torch.bfloat16)[torch.randperm(cols, device="cuda")]
    want = _values(x) @ pick.double().t()
    for t in (1, 16, 20, 64, 128, 200, 300):
        part = mx4.from_parts(*(p[:t].contiguous() for p in x.parts()), cols)
        assert torch.equal(mx4.linear(part, mx4.quantize(pick)).double(), want[:t])


def _gated_off(x, wg, wu, name):
    g, u = x @ wg.t(), x @ wu.t()
    a = g * torch.sigmoid(g) if name == "silu" else 0.5 * g * (1 + torch.tanh((2 / np.pi) ** 0.5 * (g + 0.044715 * g ** 3)))
    dg, du = _sum_off(x, wg), _sum_off(x, wu)
    # neither function is steeper than 1.13; their FP32 evaluation is off by some 2^-19 of themselves, or of g where 1 + tanh cancels
    da = 1.13 * dg + a.abs() * 2.0 ** -19 + (g.abs() * 2.0 ** -21 if name == "gelu" else 0)
    return a * u, da * (u.abs() + du) + a.abs() * du


@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("tokens,cols,rows", [(1, 256, 128), (1, 4096, 1000), (7, 100, 33), (16, 1024, 384), (32, 512, 129), (50, 2000, 517), (64, 256, 640),
                                              (65, 512, 128), (129, 300, 260), (300, 1024, 1100), (1030, 640, 385)])
def test_gated_linear(tokens, cols, rows, activation):
    x, wg = _inputs(tokens, cols, rows, 2)
    _, wu = _inputs(tokens, cols, rows, 3)
    want, off = _gated_off(_values(mx4.quantize(x)), _values(wg), _values(wu), activation)
    ref.poison()
    y = mx4.gated_linear(x, wg, wu, activation=activation)
    bound = off + want.abs() * ref.ROUND[torch.bfloat16] * (1 + 2.0 ** -8)
    assert ((y.double() - want).abs() <= bound).all()
    ref.poison()
    q = mx4.gated_linear(mx4.quantize(x), wg, wu, activation=activation, quantized=True)
    assert q.shape == (tokens, rows)
    ref.check_rounded(q, want.cpu().numpy(), off.cpu().numpy())
    # what fills up the last tile is zeros: a product with it is finite and right
    w = mx4.quantize(torch.randn((70, rows), device="cuda").to(torch.bfloat16))
    _check(mx4.linear(q, w), _values(q), _values(w), torch.bfloat16)
    assert mx4.product_timed_out() is False


@pytest.mark.parametrize("tokens", [3, 40, 300])
def test_nan_and_infinity_stay_in_their_row_and_column(tokens):
    x, _ = _inputs(tokens, 512, 200, 4)
    w = torch.randn((200, 512), device="cuda").to(torch.bfloat16)
    x[1, 100], x[2, 511], w[150, 3] = float("nan"), float("inf"), -float("inf")
    y = mx4.linear(x, mx4.quantize(w))
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[1], bad[2], bad[:, 150] = True, True, True
    assert torch.equal(y.isnan(), bad) and y[~bad].isfinite().all()


def test_shapes_no_tokens_and_extreme_scales():
    x, w = _inputs(30, 96, 50)
    assert torch.equal(mx4.linear(x.view(5, 6, 96), w).view(30, 50), mx4.linear(x, w))
    assert mx4.linear(x[0], w).shape == (50,)
    assert mx4.linear(x[:0], w).shape == (0, 50) and mx4.gated_linear(x[:0], w, w, quantized=True).rows == 0
    assert torch.equal(mx4.linear(x[:, :96][::2], w), mx4.linear(x[::2].contiguous(), w))
    # zeros times whatever is zero, and the least scales give no NaN
    assert (mx4.linear(torch.zeros_like(x), w) == 0).all()
    tiny = torch.full((4, 96), 2.0 ** -126, device="cuda")
    huge = mx4.quantize(torch.full((8, 96), 2.0 ** 100, device="cuda"))
    np.testing.assert_allclose(ref.to64(mx4.linear(tiny, huge)), 96 * 2.0 ** -26, rtol=2.0 ** -8)


def test_two_streams_at_once():
    x, w = _inputs(20, 4096, 3000, 5)
    want = mx4.linear(x, w)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(8):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(mx4.linear(x, w))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_captured_in_a_graph():
    x, w = _inputs(3, 1024, 700, 6)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        mx4.linear(x, w)                                    # the stream's scratch, outside of the capture
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y = mx4.linear(x, w)
    x2, _ = _inputs(3, 1024, 700, 7)
    x.copy_(x2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, mx4.linear(x2, w))


def test_refusals():
    x, w = _inputs(4, 64, 32)
    for call, match in (
            (lambda: mx4.linear(x.cpu(), w), "CUDA tensor"),
            (lambda: mx4.linear(x, x), "Mx4Tensor"),
            (lambda: mx4.linear(x[:, :32], w), "32 columns, the weight 64"),
            (lambda: mx4.linear(x, w, dtype=torch.float32), "bfloat16 or float16"),
            (lambda: mx4.linear(x.t(), w), "unit stride"),
            (lambda: mx4.gated_linear(x, w, None), "Mx4Tensor"),
            (lambda: mx4.gated_linear(x, w, mx4.quantize(x)), "same shape"),
            (lambda: mx4.gated_linear(x, w, w, activation="relu"), "activation"),
            (lambda: mx4.linear(x, mx4.quantize(x[:0])), "at least one row"),
            (lambda: mx4.GatedMlp(w, w, w, pre_weight=x[0]), "down_proj")):
        with pytest.raises(ValueError, match=match):
            call()


@pytest.mark.parametrize("tokens,hidden,inter", [(1, 256, 640), (9, 300, 1000), (140, 512, 385)])
def test_gated_mlp(tokens, hidden, inter):
    """The block is its operators, one after the other."""
    h, gate = _inputs(tokens, hidden, inter, 8)
    _, up = _inputs(tokens, hidden, inter, 9)
    _, down = _inputs(tokens, inter, hidden, 10)
    pre, post, nxt = (torch.rand(hidden, device="cuda") + 0.5 for _ in range(3))
    block = mx4.GatedMlp(gate, up, down, pre_weight=pre, post_weight=post, gate=post, residual_scale=0.5, next_weight=nxt, eps=1e-6)
    joined, n = block(h)
    x = mx4.rms_norm(h, pre, eps=1e-6, quantized=True)
    y = mx4.linear(mx4.gated_linear(x, gate, up, quantized=True), down)
    want = mx4.block_join(y, h, post_weight=post, gate=post, residual_scale=0.5, next_weight=nxt, eps=1e-6)
    assert torch.equal(joined, want[0]) and torch.equal(n, want[1])
    assert torch.equal(block(h, inplace=True)[0], want[0]) and torch.equal(h, want[0])


@pytest.mark.parametrize("tokens", [1, 33, 200])
@pytest.mark.parametrize("stream,gate,activation", [("f32", "row", "gelu"), ("f16", "full", "silu"), ("bf16", None, "gelu")])
def test_gated_mlp_forms(tokens, stream, gate, activation):
    """Streams of every type, gates that are checked with every call, strided streams."""
    hidden, inter = 384, 1000
    whole, gp = _inputs(tokens, hidden + 64, inter, 12, stream)
    h = whole[:, 32:32 + hidden]
    gp, up, down = (mx4.quantize(torch.randn(s, device="cuda") * 0.05) for s in ((inter, hidden), (inter, hidden), (hidden, inter)))
    pre, nxt = (torch.rand(hidden, device="cuda").to(torch.bfloat16) for _ in range(2))
    g = None if gate is None else torch.randn((tokens, 1) if gate == "row" else (tokens, hidden), device="cuda")
    block = mx4.GatedMlp(gp, up, down, pre_weight=pre, gate=g, next_weight=nxt, eps=1e-6, activation=activation)
    joined, n = block(h)
    kept = torch.bfloat16 if stream == "f32" else h.dtype
    x = mx4.rms_norm(h, pre, eps=1e-6, quantized=True)
    y = mx4.linear(mx4.gated_linear(x, gp, up, activation=activation, quantized=True), down, dtype=kept)
    want = mx4.block_join(y, h, gate=g, next_weight=nxt, eps=1e-6)
    assert torch.equal(joined, want[0]) and torch.equal(n, want[1]) and n.dtype == kept and joined.dtype == h.dtype
    if g is not None and tokens > 1:      # (one row's gate fits any number of rows)
        with pytest.raises(ValueError, match="gate must be contiguous"):
            block(torch.cat([h, h]))


def test_gated_mlp_of_no_tokens():
    w = mx4.quantize(torch.ones((64, 64), device="cuda"))
    one = torch.ones(64, device="cuda")
    joined, n = mx4.GatedMlp(w, w, w, pre_weight=one, next_weight=one)(torch.empty((0, 64), dtype=torch.bfloat16, device="cuda"))
    assert joined.shape == n.shape == (0, 64)
