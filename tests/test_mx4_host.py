"""What the 4-bit operators' host side does without a GPU: refusals that come before any launch, sizes, the layout of packed arguments."""
import ctypes

import pytest
import torch

from mpserve_b200 import _lib, mx4


@pytest.fixture(scope="module")
def lib():
    from mpserve_b200 import build

    build.build()
    return _lib.load()


def test_packed_arguments_have_the_sizes_of_their_structs():
    assert _lib.MX4_NORM.size == 7 * 8 + 7 * 8 + 6 * 4 + 2 * 4
    assert _lib.MX4_LINEAR.size == 5 * 8 + 5 * 8 + 4 * 4
    assert ctypes.sizeof(_lib.Mx4Mlp) == 7 * 8 + 3 * 8 + 5 * 4 + 2 * 4 + 4      # and four bytes to a multiple of 8


@pytest.mark.parametrize("rows,cols", [(0, 1), (1, 1), (128, 256), (129, 257), (14336, 4096), (1 << 31, 1 << 24)])
def test_bytes_of_tiles(lib, rows, cols):
    want = -(-rows // 128) * -(-cols // 256) * 17408
    assert lib.mps_mx4_bytes(rows, cols) == want == mx4._tile_bytes(rows, cols)


def test_sizes_out_of_range(lib):
    assert lib.mps_mx4_bytes(1, 0) == lib.mps_mx4_bytes(-1, 5) == lib.mps_mx4_bytes((1 << 31) + 1, 5) == lib.mps_mx4_bytes(1, (1 << 24) + 1) == -1
    assert lib.mps_mx4_mlp_scratch_bytes(3, 0, 5) == -1
    assert lib.mps_mx4_mlp_scratch_bytes(3, 300, 1000) == mx4._tile_bytes(3, 300) + mx4._tile_bytes(3, 1000) + 3 * 300 * 2


def test_errors_come_back_from_the_c_entries(lib):
    for call, code, text in (
            (lambda: lib.mps_mx4_quantize(None, 0, 4, 0, 0, None, None), _lib.MPS_ERR_INVALID, b"cols"),
            (lambda: lib.mps_mx4_quantize(None, 9, 4, 8, 8, None, None), _lib.MPS_ERR_INVALID, b"dtype"),
            (lambda: lib.mps_mx4_quantize(None, 0, 4, 8, 8, None, None), _lib.MPS_ERR_INVALID, b"null"),
            (lambda: lib.mps_mx4_dequantize(16, 4, 8, 3, 16, None), _lib.MPS_ERR_INVALID, b"dtype"),
            (lambda: lib.mps_mx4_pack(None, None, 4, 8, None, None), _lib.MPS_ERR_INVALID, b"null"),
            (lambda: lib.mps_mx4_unpack(None, 4, 8, None, None, None), _lib.MPS_ERR_INVALID, b"null"),
            (lambda: lib.mps_mx4_norm_rows(None, None), _lib.MPS_ERR_INVALID, b"null"),
            (lambda: lib.mps_mx4_product(None, None, 0, None), _lib.MPS_ERR_INVALID, b"null"),
            (lambda: lib.mps_mx4_product(_lib.MX4_LINEAR.pack(16, 0, 16, 0, 16, 1, 8, 8, 8, 8, 0, 0, 0, 0), None, 0, None), _lib.MPS_ERR_WORKSPACE, b"workspace"),
            (lambda: lib.mps_mx4_product(_lib.MX4_LINEAR.pack(16, 0, 16, 0, 16, 1, 8, 8, 8, 8, 0, 3, 0, 0), 256, 1 << 30, None), _lib.MPS_ERR_INVALID, b"gated"),
            (lambda: lib.mps_mx4_product(_lib.MX4_LINEAR.pack(16, 0, 8, 0, 16, 1, 8, 8, 8, 8, 3, 0, 0, 0), 256, 1 << 30, None), _lib.MPS_ERR_INVALID, b"aligned"),
            (lambda: lib.mps_mx4_gated_mlp(None, None, 0, 0, 1, None, 0, None, 0, None, 0, None, 0, None), _lib.MPS_ERR_INVALID, b"null")):
        assert call() == code
        assert text in lib.mps_last_error()


def test_cpu_tensors_are_refused():
    x, w = torch.zeros((4, 64)), torch.ones(64)
    q = mx4.Mx4Tensor(torch.zeros(17408, dtype=torch.uint8), 4, 64)
    for call, match in ((lambda: mx4.quantize(x), "CUDA tensor"), (lambda: mx4.rms_norm(x, w), "CUDA tensor"), (lambda: mx4.block_join(x, x), "CUDA tensor"),
                        (lambda: mx4.linear(x, q), "CUDA tensor"), (lambda: mx4.linear(x, x), "Mx4Tensor"), (lambda: mx4.dequantize(x), "Mx4Tensor"),
                        (lambda: mx4.from_parts(x, x, 64), "uint8"), (lambda: mx4.gated_linear(x, q, q, activation="x"), "activation")):
        with pytest.raises(ValueError, match=match):
            call()
