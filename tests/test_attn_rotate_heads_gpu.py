"""The rotation's kernels for few tokens of many heads: values, and which kernel has them."""
import ctypes
import re

import pytest
import torch

from mpserve_b200 import attention
from tests import _attn as ref

pytestmark = pytest.mark.gpu


def _kernels(call) -> set:
    """Names of the rotation's kernels that ``call`` launches: those of a captured graph, from the driver."""
    cuda = ctypes.CDLL("libcuda.so.1")
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    handle, count = ctypes.c_void_p(graph.raw_cuda_graph()), ctypes.c_size_t(0)
    assert cuda.cuGraphGetNodes(handle, None, ctypes.byref(count)) == 0
    nodes, names = (ctypes.c_void_p * count.value)(), set()
    assert cuda.cuGraphGetNodes(handle, nodes, ctypes.byref(count)) == 0
    for node in nodes:
        kind = ctypes.c_int(-1)
        assert cuda.cuGraphNodeGetType(ctypes.c_void_p(node), ctypes.byref(kind)) == 0
        if kind.value:      # not a kernel
            continue
        params, name = (ctypes.c_uint64 * 16)(), ctypes.c_char_p()      # the function first, a library's kernel in the eighth word
        assert cuda.cuGraphKernelNodeGetParams_v2(ctypes.c_void_p(node), params) == 0
        rc = cuda.cuFuncGetName(ctypes.byref(name), ctypes.c_void_p(params[0])) if params[0] else cuda.cuKernelGetName(ctypes.byref(name), ctypes.c_void_p(params[7]))
        assert rc == 0
        names.update(re.findall(r"rotate_(?:many_|any_)?kernel", name.value.decode()))
    return names


@pytest.mark.parametrize("q_heads,kv_heads,dim", [(64, 8, 128), (40, 40, 128), (64, 8, 64), (32, 8, 256), (16, 16, 256), (128, 128, 64), (128, 8, 128), (100, 100, 256)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("tokens", [1, 64, 400, 888])
def test_many_heads(q_heads, kv_heads, dim, dtype, tokens):
    g, kind = ref.generator(q_heads + tokens), ref.TYPES[dtype]
    q, k, v = ref.randn(g, tokens, q_heads + 2 * kv_heads, dim, dtype=kind).split((q_heads, kv_heads, kv_heads), dim=1)
    qw, kw = (1 + 0.1 * ref.randn(g, dim) for _ in range(2))
    positions = torch.randint(0, 5000, (tokens,), generator=g, device="cuda")
    frequencies = 10000.0 ** (torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / -dim)
    rotary = attention.Rotary(dim, frequencies=frequencies, interleaved=tokens == 64)
    plain = lambda: attention.norm_rotate(q, k, positions, rotary, q_weight=qw, k_weight=kw, eps=1e-6)  # noqa: E731
    q_new, k_new = plain()
    for got, x, w in ((q_new, q, qw), (k_new, k, kw)):
        ref.within(got, *ref.rotated(x, w, positions, frequencies, None, rotary.interleaved, 1.0, 1e-6))
    stores = [ref.randn(g, -(-tokens // 16) + 1, 16, kv_heads, dim, dtype=kind) for _ in range(2)]
    want = [t.clone() for t in stores]
    slots = torch.randperm(stores[0].shape[0] * 16, generator=g, device="cuda")[:tokens]
    cache = attention.KvCache(*stores)
    append = lambda: attention.norm_rotate_append(q, k, v, positions, rotary, cache, slots, q_weight=qw, k_weight=kw, eps=1e-6)  # noqa: E731
    assert torch.equal(append(), q_new)
    for store, old, new in ((stores[0], want[0], k_new), (stores[1], want[1], v)):
        old[slots // 16, slots % 16] = new
        assert torch.equal(store, old)
    # heads of whole, aligned eights are never taken value by value
    for call in (plain, append):
        names = _kernels(call)
        assert names and names <= {"rotate_kernel", "rotate_many_kernel"}


def test_odd_heads_are_taken_value_by_value():
    q, k = (torch.zeros((3, n, 34), dtype=torch.bfloat16, device="cuda") for n in (4, 2))
    positions, rotary = torch.arange(3, device="cuda"), attention.Rotary(34)
    assert _kernels(lambda: attention.norm_rotate(q, k, positions, rotary)) == {"rotate_any_kernel"}
