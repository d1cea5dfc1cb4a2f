"""Sizes whose products pass 64 bits are refused by the C entries, not wrapped round to something small."""
import pytest

from mpserve_b200 import _lib
from tests.test_attn_host import _attend, lib  # noqa: F401


@pytest.mark.parametrize("columns,page", [((1 << 26) + 1, 16), (1 << 59, 16), (1 << 60, 16), ((1 << 60) + 1, 16), (1 << 44, 1 << 20), ((1 << 63) - 1, 32)])
def test_tables_of_too_many_keys(lib, columns, page):  # noqa: F811
    args = _attend(columns=columns, page=page)
    assert lib.mps_prefix_attend_scratch_bytes(args) == -1 and b"keys" in lib.mps_last_error()
    assert lib.mps_prefix_attend_tokens(args, None, 0, None, 0, None) == _lib.MPS_ERR_INVALID and b"keys" in lib.mps_last_error()
