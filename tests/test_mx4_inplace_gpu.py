"""``inplace`` with operands that lie beside the stream, are the stream, or share memory with it."""
import pytest
import torch

from mpserve_b200 import mx4

pytestmark = pytest.mark.gpu


def _both(make):
    y, h, kw = make()
    want = mx4.block_join(y.clone(), h.clone(), **{k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in kw.items()})
    got = mx4.block_join(y, h, inplace=True, **kw)
    assert got[0] is h and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_operands_beside_the_stream_and_the_stream_itself(dtype):
    g = torch.Generator(device="cuda").manual_seed(3)
    buf = torch.randn((700, 1024), generator=g, device="cuda").to(dtype)
    w = torch.rand(512, generator=g, device="cuda") + 0.5
    _both(lambda: (buf[:, 512:], buf[:, :512], dict(post_weight=w, next_weight=w)))
    _both(lambda: (buf[300:600, :512], buf[:300, :512], dict(gate=w, next_weight=w)))
    h = buf[:, :512].contiguous()
    _both(lambda: (h, h, dict(post_weight=w, gate=h, next_weight=w)))
    _both(lambda: (buf[:, 512:].contiguous(), h[:1].clone().expand(700, 512).contiguous(), dict(gate=buf[:, :1].contiguous(), next_weight=w)))


def test_refusals():
    buf = torch.zeros((9, 128), device="cuda", dtype=torch.bfloat16)
    w = torch.ones(64, device="cuda", dtype=torch.bfloat16)
    h = torch.zeros((8, 64), device="cuda", dtype=torch.bfloat16)
    for call, name in ((lambda: mx4.block_join(buf[1:], buf[:8], inplace=True), "y"),
                       (lambda: mx4.block_join(buf[:, 32:96], buf[:, :64], inplace=True), "y"),
                       (lambda: mx4.block_join(w.expand(8, 64), h, gate=h[2], inplace=True), "gate"),
                       (lambda: mx4.block_join(w.expand(8, 64), h, gate=h.view(-1)[8:16].view(8, 1), inplace=True), "gate"),
                       (lambda: mx4.block_join(w.expand(8, 64), h, post_weight=h[0], inplace=True), "post_weight"),
                       (lambda: mx4.block_join(w.expand(8, 64), h, next_weight=h[7], inplace=True), "next_weight")):
        with pytest.raises(ValueError, match=f"{name} shares memory with h"):
            call()
    q = mx4.quantize(torch.ones((64, 64), device="cuda"))
    block = mx4.GatedMlp(q, q, q, pre_weight=w, gate=h[3], next_weight=w)
    with pytest.raises(ValueError, match="gate shares memory with h"):
        block(h, inplace=True)
    assert (h == 0).all() and block(h)[0].isfinite().all()
