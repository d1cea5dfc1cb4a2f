"""The block's C entry refuses what one of its parts would refuse before it launches the first of them."""
import pytest

from mpserve_b200 import _lib

GOOD = dict(gate_proj=256, up_proj=256, down_proj=256, pre_weight=256, post_weight=256, gate=256, next_weight=256, hidden=256, inter=640,
            gate_row_stride=0, gate_col_stride=1, gate_dtype=0, pre_dtype=0, weight_dtype=0, activation=0, eps=1e-5, residual_scale=1.0, wide_result=0)
CALL = dict(h=256, h_dtype=0, tokens=3, h_out=256, n_out=256, n_dtype=0, scratch=256, scratch_bytes=1 << 30, workspace=256, workspace_bytes=1 << 20)


@pytest.fixture(scope="module")
def lib():
    from mpserve_b200 import build

    build.build()
    return _lib.load()


@pytest.mark.parametrize("bad,code,text", [
    (dict(pre_weight=0), _lib.MPS_ERR_INVALID, b"null"),
    (dict(h=0), _lib.MPS_ERR_INVALID, b"null"),
    (dict(h_out=0), _lib.MPS_ERR_INVALID, b"null"),
    (dict(n_out=0), _lib.MPS_ERR_INVALID, b"null"),
    (dict(hidden=32769), _lib.MPS_ERR_INVALID, b"hidden"),
    (dict(hidden=0), _lib.MPS_ERR_INVALID, b"sizes"),
    (dict(inter=0), _lib.MPS_ERR_INVALID, b"sizes"),
    (dict(tokens=-1), _lib.MPS_ERR_INVALID, b"sizes"),
    (dict(tokens=1 << 31, scratch_bytes=1 << 62), _lib.MPS_ERR_INVALID, b"tokens"),
    (dict(h_dtype=3), _lib.MPS_ERR_INVALID, b"dtype"),
    (dict(n_dtype=4), _lib.MPS_ERR_INVALID, b"dtype"),
    (dict(gate_dtype=3), _lib.MPS_ERR_INVALID, b"dtype"),
    (dict(weight_dtype=-1), _lib.MPS_ERR_INVALID, b"dtype"),
    (dict(pre_dtype=7), _lib.MPS_ERR_INVALID, b"dtype"),
    (dict(activation=2), _lib.MPS_ERR_INVALID, b"activation"),
    (dict(down_proj=264), _lib.MPS_ERR_INVALID, b"aligned"),
    (dict(n_dtype=3, n_out=264), _lib.MPS_ERR_INVALID, b"aligned"),
    (dict(scratch=0), _lib.MPS_ERR_WORKSPACE, b"scratch"),
    (dict(scratch=272), _lib.MPS_ERR_WORKSPACE, b"scratch"),
    (dict(scratch_bytes=17408), _lib.MPS_ERR_WORKSPACE, b"scratch"),
    (dict(workspace=0), _lib.MPS_ERR_WORKSPACE, b"workspace"),
    (dict(workspace_bytes=3), _lib.MPS_ERR_WORKSPACE, b"workspace"),
])
def test_refusals_come_before_the_first_kernel(lib, bad, code, text):
    block = _lib.Mx4Mlp(**{k: bad.get(k, v) for k, v in GOOD.items()})
    c = {k: bad.get(k, v) for k, v in CALL.items()}
    rc = lib.mps_mx4_gated_mlp(block, c["h"], c["h_dtype"], 256, c["tokens"], c["h_out"], 256, c["n_out"], c["n_dtype"], c["scratch"], c["scratch_bytes"],
                               c["workspace"], c["workspace_bytes"], None)
    assert rc == code and text in lib.mps_last_error()


def test_no_tokens_are_no_work(lib):
    assert lib.mps_mx4_gated_mlp(_lib.Mx4Mlp(**GOOD), None, 0, 256, 0, None, 256, None, 0, None, 0, None, 0, None) == _lib.MPS_OK
