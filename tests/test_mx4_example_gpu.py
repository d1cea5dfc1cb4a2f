"""The example runs as a user runs it, and the block from a compressed checkpoint is the block of its 4-bit operands."""
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [1, 37, 300])
def test_block_from_a_compressed_checkpoint(tokens):
    from examples import mx4_mlp

    bits, rounding = mx4_mlp.run(tokens, 512, 1152)
    # a value in E2M1 is off by at most a quarter of itself or of the grid's first step, some 0.12 in the mean square; four such operands meet in the block
    assert 0 < bits < 0.5
    # BF16 rounding of the block's result and of the stream, 2^-8 each at most, and activations that round to a neighbouring code
    assert rounding < 2 * 2.0 ** -8


def test_the_command():
    done = subprocess.run([sys.executable, "examples/mx4_mlp.py", "--tokens", "1", "130", "--hidden", "256", "--inter", "640"], cwd=ROOT,
                          capture_output=True, text=True, timeout=600)
    assert done.returncode == 0, done.stderr
    assert len([line for line in done.stdout.splitlines() if "tokens:" in line]) == 2
