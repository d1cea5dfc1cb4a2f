"""No scratch of a product outlives its call: what the C entry takes and refuses, without a launch."""
import pytest

from mpserve_b200 import _lib


@pytest.fixture(scope="module")
def lib():
    from mpserve_b200 import build

    build.build()
    return _lib.load()


def test_the_workspace_holds_a_record_and_no_tokens(lib):
    assert 4 <= lib.mps_mx4_workspace_bytes() < 17408


@pytest.mark.parametrize("tokens", [9, 64, 100000])
@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_tokens_to_quantise_come_with_a_place_of_their_own(lib, tokens, dtype):
    args = _lib.MX4_LINEAR.pack(256, 0, 256, 0, 256, tokens, 256, 128, 256, 128, dtype, 0, 0, 0)
    assert lib.mps_mx4_product(args, 256, 1 << 30, None) == _lib.MPS_ERR_WORKSPACE
    assert b"x_tiles" in lib.mps_last_error()


@pytest.mark.parametrize("tokens,hidden,inter", [(1, 64, 64), (3, 300, 1000), (35, 256, 640), (2048, 4096, 14336), (100000, 512, 512)])
def test_scratch_of_a_block_holds_its_result_in_32_bits(lib, tokens, hidden, inter):
    """The result takes the place of the normalised tokens, which have been multiplied by then."""
    need = lib.mps_mx4_mlp_scratch_bytes(tokens, hidden, inter)
    a, x = lib.mps_mx4_bytes(tokens, inter), lib.mps_mx4_bytes(tokens, hidden)
    assert need >= a + 4 * tokens * hidden and need >= a + x + 2 * tokens * hidden
