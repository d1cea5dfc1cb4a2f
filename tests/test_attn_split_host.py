"""The arithmetic that splits attention's work, compiled for the host: stretches of own keys and cycles of the prefix at the sizes that the entries accept."""
import random
import subprocess

import pytest

from mpserve_b200 import build

MOST_KEYS, MOST_SEQUENCES, LEAST = 1 << 30, 1 << 16, 64

PROGRAM = """
#include "attn.cuh"
#include <cstdio>
int main() {
    long long a, b;
    char what;
    while (scanf(" %c %lld %lld", &what, &a, &b) == 3)
        printf("%lld\\n", what == 's' ? (long long)mps::own_stretch(a, b) : (long long)mps::prefix_cycles((int)a, (int)b));
}
"""


@pytest.fixture(scope="module")
def split(tmp_path_factory):
    at = tmp_path_factory.mktemp("split")
    (at / "split.cu").write_text(PROGRAM)
    subprocess.run([build.nvcc_path(), "-std=c++17", *build.ARCH_FLAGS, "-I", str(build.CSRC), "-o", str(at / "split"), str(at / "split.cu")], check=True, capture_output=True)

    def ask(rows):
        done = subprocess.run([str(at / "split")], input="\n".join(f"{what} {a} {b}" for what, a, b in rows), check=True, capture_output=True, text=True)
        return [int(line) for line in done.stdout.split()]

    return ask


def test_stretches_of_own_keys(split):
    rng = random.Random(1)
    asked = [(0, 1), (1, 1), (64, 1), (65, 1), (MOST_KEYS, 1), (MOST_KEYS + 1, 1), ((1 << 31) - 64, 1), (1 << 31, 1), (1 << 32, 1), (MOST_KEYS * MOST_SEQUENCES, 9),
             (MOST_KEYS * MOST_SEQUENCES, 8288), (MOST_KEYS * 64, 9)]
    asked += [(rng.randrange(1 << rng.randrange(1, 47)), rng.randrange(1, 1 << rng.randrange(1, 14))) for _ in range(500)]
    for (keys, places), step in zip(asked, split([("s", *pair) for pair in asked])):
        assert step == min(MOST_KEYS, max(LEAST, -(-(-(-keys // places)) // 64) * 64))
        # lengths that add up to so many: no more stretches than there are places for
        left, count, sequences = keys, 0, 0
        if keys <= MOST_KEYS * 64:
            while left:
                length = min(left, MOST_KEYS)
                count, sequences, left = count - (-length // step), sequences + 1, left - length
            assert count <= places + sequences


def test_cycles_of_the_prefix(split):
    asked = [(tiles, cycles) for tiles in (1, 2, 1000, (1 << 31) // 3000, (1 << 31) // 1800 + 1, 1 << 23) for cycles in (1800, 3000)]
    got = split([("c", *pair) for pair in asked])
    assert all(b > a for (t, a), (u, b) in zip(zip(asked[::2], got[::2]), zip(asked[2::2], got[2::2])))
    start = got[0] - 1800
    assert got == [start + tiles * cycles for tiles, cycles in asked]
