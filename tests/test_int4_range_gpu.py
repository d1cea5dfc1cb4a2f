"""INT4 products of the largest tokens that their sums have room for."""
import pytest
import torch

from mpserve_b200 import int4
from tests import _attn as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [1, 9, 40])
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("dtype,size", [("bf16", 2.0 ** 116), ("f16", 65504.0)])
def test_tokens_at_the_end_of_the_range(tokens, group, dtype, size):
    # every product of a group has the same sign and 15 for its whole number: group * 15 * 2^116 is just inside FP32
    g = ref.generator(tokens)
    x = torch.full((tokens, 256), size, device="cuda").to(ref.TYPES[dtype])
    x[:, group:] = 0
    codes, zeros = torch.full((70, 256), 15, dtype=torch.uint8, device="cuda"), torch.zeros((70, 256 // group), dtype=torch.uint8, device="cuda")
    scales = ((torch.rand((70, 256 // group), generator=g, device="cuda") + 0.5) * 1e-3).to(torch.float16)
    values = ref.int4_values(codes, scales, zeros, group)
    # F16 tokens' results are up to 65504 * 15 * 128 * 0.0015 = 1.9e5, beyond F16: in BF16
    y = int4.linear(x, int4.from_parts(codes, scales, zeros, group=group), dtype=torch.bfloat16)
    ref.within(y, x.double() @ values.t(), ref.int4_off(x, values, group))
