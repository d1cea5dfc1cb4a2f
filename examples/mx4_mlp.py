"""A gated MLP block served in 4 bits from a compressed checkpoint.

    python examples/mx4_mlp.py [--tokens 1 64 2048] [--hidden 1024] [--inter 3584]

The block's three weights are random (no checkpoint is needed), quantised to FP8 with a scale per channel and compressed as a
checkpoint would be; ``FusedDecoder`` gives them back as BF16, ``mx4.quantize`` takes them to MXFP4 once, and ``mx4.GatedMlp`` serves the
block from then on.  For every number of tokens the block's result is held against the same block in FP32 with the decoded weights, and
against one that has the 4-bit weights and activations but multiplies in FP32: the first difference is what 4 bits cost, the second is
rounding.
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

if __package__ is None:
    sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import MPServe_cuda  # noqa: E402
from mpserve_b200 import mx4, sidecar  # noqa: E402
from mpserve_b200 import workloads as wl  # noqa: E402

EPS = 1e-5


def decoded_weights(hidden: int, inter: int, device) -> list[torch.Tensor]:
    """gate, up and down projection in BF16, by way of a compressed checkpoint."""
    groups = []
    for i, (rows, cols) in enumerate(((inter, hidden), (inter, hidden), (hidden, inter))):
        c = wl.quantize_fp8(wl.random_weight(rows, cols, i, device=device), "channel")
        art = MPServe_cuda.huffman_build_fp8_decode_tables(c.bf16, c.fp8_u8, c.scales_u16, max_len=7, threads_per_block=1024)
        groups.append([(c.fp8_u8, art)])
    return sidecar.FusedDecoder(groups).decode()


def _norm(x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
    return x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS) * weight.float()


def plain_block(h, weights, pre, post, through=lambda t: t) -> torch.Tensor:
    """The block in FP32; ``through`` is what a product's left operand goes through."""
    gate, up, down = (w.float() for w in weights)
    x = through(_norm(h.float(), pre))
    a = through(torch.nn.functional.silu(x @ gate.t()) * (x @ up.t()))
    return h.float() + _norm(a @ down.t(), post)


def run(tokens: int, hidden: int, inter: int, device="cuda") -> tuple[float, float]:
    """The relative differences (2-norm) to the FP32 block and to the FP32 block of 4-bit operands."""
    weights = decoded_weights(hidden, inter, device)
    packed = [mx4.quantize(w) for w in weights]                                 # once, when the model is loaded
    pre, post = (torch.ones(hidden, device=device) for _ in range(2))
    block = mx4.GatedMlp(*packed, pre_weight=pre, post_weight=post, eps=EPS)
    g = torch.Generator(device=device).manual_seed(tokens)
    h = torch.randn((tokens, hidden), generator=g, device=device).to(torch.bfloat16)
    joined, _ = block(h)                                                        # every step
    exact = plain_block(h, weights, pre, post)
    rounded = plain_block(h, [q.dequantize() for q in packed], pre, post, lambda t: mx4.quantize(t).dequantize(torch.float32))
    off = [((joined.float() - want).norm() / want.norm()).item() for want in (exact, rounded)]
    return off[0], off[1]


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--tokens", type=int, nargs="+", default=[1, 64, 2048])
    ap.add_argument("--hidden", type=int, default=1024)
    ap.add_argument("--inter", type=int, default=3584)
    args = ap.parse_args()
    torch.backends.cuda.matmul.allow_tf32 = False
    for tokens in args.tokens:
        bits, rounding = run(tokens, args.hidden, args.inter)
        print(f"{tokens:6d} tokens: {bits:.3f} off FP32, {rounding:.5f} off FP32 of the same 4-bit operands")


if __name__ == "__main__":
    main()
