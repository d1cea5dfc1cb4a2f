"""A decoding step's attention half as it is used: products, norms with rotation into the cache, attention and the product behind it, eagerly, captured and from threads."""
import threading

import pytest
import torch

from mpserve_b200 import attention, int4, mx4
from tests import _attn as ref

pytestmark = pytest.mark.gpu

HIDDEN, Q_HEADS, KV_HEADS, DIM, PAGE, PREFIX, OWN_COLUMNS = 512, 8, 2, 64, 16, 37, 3


class _Layer:
    """Weights, a cache whose first pages hold the prefix, and one layer's calls."""

    def __init__(self, seed, batch):
        g = ref.generator(seed)
        self.batch, heads = batch, Q_HEADS + 2 * KV_HEADS
        self.qkv_parts = ref.int4_parts(g, heads * DIM, HIDDEN, 64)
        self.out_parts = ref.int4_parts(g, HIDDEN, Q_HEADS * DIM, 64)
        self.qkv, self.out = int4.from_parts(*self.qkv_parts, group=64), int4.from_parts(*self.out_parts, group=64)
        self.q_weight, self.k_weight = (torch.rand(DIM, generator=g, device="cuda") + 0.5 for _ in range(2))
        self.frequencies = torch.rand((DIM // 2,), generator=g, device="cuda", dtype=torch.float64)
        self.rotary = attention.Rotary(DIM, frequencies=self.frequencies)
        self.prefix_pages = -(-PREFIX // PAGE)
        pages = self.prefix_pages + batch * OWN_COLUMNS
        self.k, self.v = (ref.randn(g, pages, PAGE, KV_HEADS, DIM, dtype=torch.bfloat16) for _ in range(2))
        self.cache = attention.KvCache(self.k, self.v)
        order = torch.randperm(pages, generator=g, device="cuda").int()
        self.prefix_table, self.tables = order[:self.prefix_pages].clone(), order[self.prefix_pages:].view(batch, OWN_COLUMNS).clone()
        self.lengths = torch.randint(0, PAGE * OWN_COLUMNS - 4, (batch,), generator=g, device="cuda", dtype=torch.int32)      # before the step
        self.x = ref.randn(g, batch, HIDDEN, dtype=torch.bfloat16)

    def step(self):
        """The layer's call for one more token of each sequence, all on the device."""
        n, heads = self.batch, Q_HEADS + 2 * KV_HEADS
        qkv = int4.linear(self.x, self.qkv).view(n, heads, DIM)
        at = self.lengths.long()
        pages = self.tables.gather(1, (at // PAGE)[:, None])[:, 0].long()
        slots = pages * PAGE + at % PAGE
        q = attention.norm_rotate_append(qkv[:, :Q_HEADS], qkv[:, Q_HEADS:Q_HEADS + KV_HEADS], qkv[:, Q_HEADS + KV_HEADS:], PREFIX + at, self.rotary, self.cache, slots,
                                         q_weight=self.q_weight, k_weight=self.k_weight)
        a = attention.shared_prefix_attention(q, self.cache, self.tables, self.lengths + 1, prefix_table=self.prefix_table, prefix_length=PREFIX)
        return qkv, q, a, int4.linear(a.view(n, -1), self.out)

    def slots(self):
        at = self.lengths.long()
        return self.tables.gather(1, (at // PAGE)[:, None])[:, 0].long(), at % PAGE

    def check(self, got):
        """Every call's result against its formula in 64 bits, from what the call was given."""
        qkv, q, a, y = got
        n = self.batch
        values = ref.int4_values(*self.qkv_parts, 64)
        ref.within(qkv.reshape(n, -1), self.x.double() @ values.t(), ref.int4_off(self.x, values, 64))
        own_q, own_k, own_v = qkv.split((Q_HEADS, KV_HEADS, KV_HEADS), dim=1)
        at, (page, slot) = PREFIX + self.lengths.long(), self.slots()
        for new, x, weight in ((q, own_q, self.q_weight), (self.k[page, slot], own_k, self.k_weight)):
            ref.within(new, *ref.rotated(x, weight, at, self.frequencies, None, False, 1.0, 1e-6))
        assert torch.equal(self.v[page, slot], own_v)
        want, _, off, _ = ref.attend(q, self.k, self.v, self.tables, self.lengths + 1, self.prefix_table, PREFIX)
        ref.within(a, want, off)
        values = ref.int4_values(*self.out_parts, 64)
        ref.within(y, a.reshape(n, -1).double() @ values.t(), ref.int4_off(a.reshape(n, -1), values, 64))


@pytest.mark.parametrize("batch", [1, 3, 33])
def test_a_step(batch):
    layer = _Layer(batch, batch)
    layer.check(layer.step())


def test_a_captured_step_goes_on_from_token_to_token():
    layer = _Layer(5, 5)
    layer.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layer.step()
    for _ in range(3):      # the same graph for the next tokens: lengths and inputs are read on the GPU
        graph.replay()
        torch.cuda.synchronize()
        layer.check(got)
        layer.lengths += 1
        layer.x.mul_(-0.5)


def test_two_captured_steps_share_the_workspace():
    layers = [_Layer(seed, 4) for seed in (6, 7)]
    graphs, results = [], []
    for layer in layers:
        layer.step()
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            results.append(layer.step())
    streams = [torch.cuda.Stream() for _ in layers]
    for _ in range(4):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for layer, got in zip(layers, results):
        layer.check(got)
    assert not mx4.product_timed_out()


def test_steps_from_two_threads():
    layers = [_Layer(seed, 3 + seed) for seed in (8, 9)]
    torch.cuda.synchronize()
    results, errors = [None, None], []

    def run(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(20):
                    results[i] = layers[i].step()
            stream.synchronize()
        except Exception as e:
            errors.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for layer, got in zip(layers, results):
        layer.check(got)


def test_two_tokens_with_one_slot_leave_one_of_them():
    layer = _Layer(10, 2)
    layer.tables[1] = layer.tables[0]
    layer.lengths[1] = layer.lengths[0]
    qkv = layer.step()[0]
    page, slot = layer.slots()
    kept, own_v = layer.v[page[0], slot[0]], qkv[:, Q_HEADS + KV_HEADS:]
    assert ((kept == own_v[0]) | (kept == own_v[1])).all()


def test_gradients_do_not_pass():
    layer = _Layer(11, 2)
    layer.x.requires_grad_()
    assert not any(t.requires_grad for t in layer.step())


def test_a_cache_brings_the_workspace(monkeypatch):
    """A first call that is captured must not allocate it: it would be the graph's."""
    monkeypatch.setattr(mx4, "_workspaces", {})
    pages = torch.zeros((2, PAGE, KV_HEADS, DIM), dtype=torch.bfloat16, device="cuda")
    attention.KvCache(pages, pages.clone())
    kept = mx4._workspaces[pages.get_device()]
    assert not kept.any()
