"""How exact the angles of far positions are, against products of whole numbers and fractions."""
from fractions import Fraction
import math

import pytest
import torch

from mpserve_b200 import attention

pytestmark = pytest.mark.gpu

# 2 pi to 50 digits
TURN = Fraction(628318530717958647692528676655900576839433879875021, 10 ** 50)


@pytest.mark.parametrize("far", [1 << 10, 1 << 20, 1 << 25, 1 << 28, 1 << 35, 1 << 45])
@pytest.mark.parametrize("tokens", [40, 900])
def test_angles(far, tokens):
    g = torch.Generator().manual_seed(far % 1000003)
    positions = torch.randint(-far, far, (tokens,), generator=g)
    frequencies = torch.cat((torch.ones(1, dtype=torch.float64), torch.rand((7,), generator=g, dtype=torch.float64)))
    rotary = attention.Rotary(16, frequencies=frequencies.cuda())
    x = torch.zeros((tokens, 1, 16), device="cuda")
    x[:, :, :8] = 1      # becomes (cosine, sine)
    q, _ = attention.norm_rotate(x, x, positions.cuda(), rotary)
    got = q[:, 0].double().cpu()
    for t, p in enumerate(positions.tolist()):
        for j, f in enumerate(frequencies.tolist()):
            turns = Fraction(f) * p / TURN
            angle = float((turns - round(turns)) * TURN)
            # The frequency in turns is off by 2^-52 of itself, its product with the position by another 2^-53: 2^-51 of the angle at most.  What is left of it below half a turn is
            # rounded to FP32 (2 pi 2^-26), sine and cosine are off by two of FP32's steps at most.
            off = abs(p * f) * 2.0 ** -51 + 2 * math.pi * 2.0 ** -26 + 2 * 2.0 ** -23
            assert abs(got[t, j].item() - math.cos(angle)) <= off and abs(got[t, 8 + j].item() - math.sin(angle)) <= off
