"""What the host side of INT4 products and of the attention operators does without a GPU: refusals that come before any launch, sizes, packed arguments."""
import pytest
import torch

from mpserve_b200 import _lib, attention, int4


@pytest.fixture(scope="module")
def lib():
    from mpserve_b200 import build

    build.build()
    return _lib.load()


def test_packed_arguments_have_the_sizes_of_their_structs():
    assert _lib.INT4_LINEAR.size == 4 * 8 + 5 * 8 + 4 * 4
    assert _lib.HEAD_ROTATE.size == 12 * 8 + 15 * 8 + 8 * 4 + 2 * 4
    assert _lib.PREFIX_ATTEND.size == 8 * 8 + 13 * 8 + 4 * 4 + 4 + 4      # the last four fill up to a multiple of 8


@pytest.mark.parametrize("rows,cols,group", [(0, 1, 32), (1, 1, 128), (16, 64, 64), (17, 65, 32), (14336, 4096, 128), (1 << 27, 1 << 24, 32)])
def test_bytes_of_a_weight(lib, rows, cols, group):
    want = -(-rows // 128) * -(-cols // 128) * (128 * 128 // 2 + 128 * (128 // group) * 4)
    assert lib.mps_int4_bytes(rows, cols, group) == want == int4._bytes(rows, cols, group)


def test_sizes_out_of_range(lib):
    for rows, cols, group in ((-1, 5, 32), (5, 0, 32), (5, 5, 48), (5, 5, 256), ((1 << 27) + 1, 5, 32), (5, (1 << 24) + 1, 32)):
        assert lib.mps_int4_bytes(rows, cols, group) == -1


def _rotate(**kw):
    a = dict(q=16, k=16, v=0, q_out=16, k_out=16, v_out=0, qw=0, kw=0, positions=16, turns=16, axis=0, slots=0, tokens=1, pages=0, page=0, q_heads=1, kv_heads=1, dim=64,
             rotated=64, dtype=0, weight_dtype=0) | kw
    return _lib.HEAD_ROTATE.pack(*(a[n] for n in "q k v q_out k_out v_out qw kw positions turns axis slots tokens".split()), *([64] * 12), a["pages"], a["page"],
                                 a["q_heads"], a["kv_heads"], a["dim"], a["rotated"], 0, 1, a["dtype"], a["weight_dtype"], 1e-6, 1.0)


def _attend(**kw):
    a = dict(q=16, k=16, v=16, out=16, tables=16, lengths=16, prefix=16, batch=1, columns=1, prefix_length=1, pages=4, page=16, stride=64, q_heads=2, kv_heads=1, dim=64,
             dtype=0) | kw
    return _lib.PREFIX_ATTEND.pack(a["q"], a["k"], a["v"], a["out"], 0, a["tables"], a["lengths"], a["prefix"], a["batch"], a["columns"], a["prefix_length"], a["pages"],
                                   a["page"], a["stride"], 64, *([64] * 6), a["q_heads"], a["kv_heads"], a["dim"], a["dtype"], 1.0)


def test_errors_come_back_from_the_c_entries(lib):
    bad = _lib.MPS_ERR_INVALID
    linear = lambda x, *a: lib.mps_int4_product(_lib.INT4_LINEAR.pack(x, 0, *a), None, 0, None)  # noqa: E731
    rotate = lambda **kw: lib.mps_head_rotate_rows(_rotate(**kw), None)  # noqa: E731
    attend = lambda **kw: lib.mps_prefix_attend_tokens(_attend(**kw), None, 0, None, 0, None)  # noqa: E731
    for call, text in (
            (lambda: lib.mps_int4_product(None, None, 0, None), b"null"), (lambda: linear(16, 16, 16, 1, 64, 8, 64, 8, 100, 0, 0, 0), b"group"),
            (lambda: linear(16, 16, 16, 1, 64, 0, 64, 8, 64, 0, 0, 0), b"rows"), (lambda: linear(16, 16, 16, -1, 64, 8, 64, 8, 64, 0, 0, 0), b"tokens"),
            (lambda: linear(16, 16, 16, 1, 64, 8, 64, 8, 64, 2, 0, 0), b"dtypes"), (lambda: linear(16, 16, 16, 1, 64, 8, 64, 8, 64, 0, 0, 2), b"dtypes"),
            (lambda: linear(0, 16, 16, 1, 64, 8, 64, 8, 64, 0, 0, 0), b"null"), (lambda: linear(16, 8, 16, 1, 64, 8, 64, 8, 64, 0, 0, 0), b"unaligned"),
            (lambda: lib.mps_int4_pack(None, None, None, 4, 64, 64, None, None), b"null"), (lambda: lib.mps_int4_pack(16, 16, 0, 4, 64, 65, 16, None), b"group"),
            (lambda: lib.mps_int4_dequantize(16, 4, 64, 64, 2, 0, 16, None), b"dtype"), (lambda: lib.mps_int4_dequantize(16, 4, 64, 64, 0, 3, 16, None), b"dtype"),
            (lambda: lib.mps_int4_dequantize(None, 4, 64, 64, 0, 0, None, None), b"null"),
            (lambda: lib.mps_head_rotate_rows(None, None), b"null"), (lambda: rotate(dim=257), b"dim"), (lambda: rotate(rotated=66), b"rotated"),
            (lambda: rotate(rotated=63), b"even"), (lambda: rotate(dtype=3), b"dtype"), (lambda: rotate(qw=16, weight_dtype=3), b"dtype"), (lambda: rotate(q_heads=1025), b"heads"),
            (lambda: rotate(q=0), b"missing"), (lambda: rotate(positions=0), b"missing"), (lambda: rotate(v=16), b"missing"), (lambda: rotate(slots=16), b"missing"),
            (lambda: rotate(slots=16, v=16, v_out=16, pages=2, page=24), b"power of two"),
            (lambda: lib.mps_prefix_attend_tokens(None, None, 0, None, 0, None), b"null"), (lambda: attend(dim=96), b"64 or 128"), (lambda: attend(dtype=2), b"BF16 or F16"),
            (lambda: attend(page=8), b"power of two"), (lambda: attend(page=48), b"power of two"), (lambda: attend(q_heads=3, kv_heads=2), b"multiple"),
            (lambda: attend(batch=-1), b"batch"), (lambda: attend(prefix_length=(1 << 30) + 1), b"keys"), (lambda: attend(columns=1 << 27), b"keys"),
            (lambda: attend(q=0), b"missing"), (lambda: attend(prefix=0), b"missing"), (lambda: attend(tables=0), b"missing"), (lambda: attend(k=8), b"aligned"),
            (lambda: attend(stride=4, batch=2), b"aligned")):
        assert call() == bad
        assert text in lib.mps_last_error()
    # nothing to do is no error, and touches nothing
    assert linear(0, 0, 0, 0, 64, 8, 64, 8, 64, 0, 0, 0) == rotate(tokens=0, q=0) == attend(batch=0, q=0) == 0


def test_cpu_tensors_are_refused():
    x, codes = torch.zeros((2, 64), dtype=torch.bfloat16), torch.zeros((4, 64), dtype=torch.uint8)
    heads, positions = torch.zeros((2, 4, 64), dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int64)
    rotary = attention.Rotary(64, device="cpu")
    for call, match in ((lambda: int4.from_parts(codes, torch.ones((4, 1), dtype=torch.float16), group=64), "CUDA"), (lambda: int4.linear(x, codes), "Int4Tensor"),
                        (lambda: int4.dequantize(codes), "Int4Tensor"), (lambda: attention.norm_rotate(heads, heads, positions, rotary), "CUDA"),
                        (lambda: attention.KvCache(*[torch.zeros((2, 16, 1, 64), dtype=torch.bfloat16)] * 2), "CUDA")):
        with pytest.raises(ValueError, match=match):
            call()


def test_parts_that_do_not_fit():
    codes, scales = torch.zeros((4, 100), dtype=torch.uint8), torch.ones((4, 1), dtype=torch.float16)
    for call, match in ((lambda: int4.from_parts(codes, scales, group=48), "group"), (lambda: int4.from_parts(codes.int(), scales), "uint8"),
                        (lambda: int4.from_parts(codes[0], scales), "matrix"), (lambda: int4.from_parts(codes, scales, group=64), "shape"),
                        (lambda: int4.from_parts(codes, scales.float()), "float16"), (lambda: int4.from_parts(codes, scales, scales), "zeros")):
        with pytest.raises(ValueError, match=match):
            call()


def test_rotary():
    r = attention.Rotary(8, base=100.0, device="cpu")
    want = torch.tensor([100.0 ** (-j / 4) for j in range(4)], dtype=torch.float64) / (2 * torch.pi)
    assert torch.allclose(r._turns, want, rtol=1e-15, atol=0) and r.axes == 1 and r._axis is None
    r = attention.Rotary(8, sections=(1, 2, 1), device="cpu").to("cpu")
    assert r.axes == 3 and r._axis.tolist() == [0, 1, 1, 2]
    assert attention.Rotary(0, device="cpu").dims == 0
    for kw, match in ((dict(dims=7), "even"), (dict(dims=258), "even"), (dict(dims=8, axes=[0, 1], device="cpu"), "axis"), (dict(dims=8, axes=[0, 1, 2, 256], device="cpu"), "axis"),
                      (dict(dims=8, sections=(4, 4)), "axis"), (dict(dims=8, axes=[0] * 4, sections=(4,)), "exclude"), (dict(dims=8, frequencies=torch.ones(3)), "frequencies"),
                      (dict(dims=8, frequencies=torch.ones(4, dtype=torch.int32)), "frequencies")):
        with pytest.raises(ValueError, match=match):
            attention.Rotary(**kw)


class _Elsewhere(torch.Tensor):
    """A CPU tensor that says it is on a GPU: for refusals that come after the check of the device, and before anything is launched."""

    is_cuda = property(lambda self: True)
    get_device = lambda self: 0  # noqa: E731


def _there(t):
    return t.as_subclass(_Elsewhere)


def _cache(pages=2, page=16, heads=2, dim=64, dtype=torch.bfloat16):
    return attention.KvCache(*(_there(torch.zeros((pages, page, heads, dim), dtype=dtype)) for _ in range(2)))


def test_caches_that_are_refused():
    ok = torch.zeros((2, 16, 2, 64), dtype=torch.bfloat16)
    wide = torch.zeros((2, 16, 2, 68), dtype=torch.bfloat16)
    for k, match in ((ok[0], "dimensions"), (ok.int(), "bfloat16"), (torch.zeros((2, 24, 2, 64), dtype=torch.bfloat16), "power of two"),
                     (torch.zeros((2, 16, 2, 264), dtype=torch.bfloat16), "heads"), (ok.transpose(2, 3), "power|heads|unit"), (wide[..., :64], "aligned"), (wide[..., 4:], "aligned"),
                     (ok[:1].expand(2, 16, 2, 64), "share memory"), (torch.zeros(4096, dtype=torch.bfloat16).as_strided((2, 16, 2, 64), (128, 64, 64, 1)), "share memory")):
        with pytest.raises(ValueError, match=match):
            attention.KvCache(_there(k), _there(k))
    with pytest.raises(ValueError, match="same shape"):
        attention.KvCache(_there(ok), _there(ok[:1]))
    c = attention.KvCache(_there(ok.transpose(1, 2).contiguous().transpose(1, 2)), _there(ok))
    assert (c.pages, c.page_size, c.kv_heads, c.head_dim) == (2, 16, 2, 64)


def test_calls_of_norm_rotate_that_are_refused():
    q, k, w = _there(torch.zeros((3, 4, 64))), _there(torch.zeros((3, 2, 64))), _there(torch.ones(64))
    positions, slots, rotary = _there(torch.zeros(3, dtype=torch.int64)), _there(torch.zeros(3, dtype=torch.int64)), attention.Rotary(64, device="cpu")
    rotate, append = attention.norm_rotate, attention.norm_rotate_append
    two = attention.Rotary(64, sections=(16, 16), device="cpu")
    for call, match in ((lambda: rotate(q[0], k, positions, rotary), "dimensions"), (lambda: rotate(q.double(), k, positions, rotary), "bfloat16"),
                        (lambda: rotate(q, k[:2], positions, rotary), "same tokens"), (lambda: rotate(q, k.half(), positions, rotary), "same tokens"),
                        (lambda: rotate(q.transpose(1, 2), k, positions, rotary), "unit stride"), (lambda: rotate(q, k, positions, None), "Rotary"),
                        (lambda: rotate(q, k, positions, attention.Rotary(128, device="cpu")), "turns 128"), (lambda: rotate(q, k, positions.float(), rotary), "int32 or int64"),
                        (lambda: rotate(q, k, positions[:2], rotary), "positions"), (lambda: rotate(q, k, positions, two), "2 axes"),
                        (lambda: rotate(q, k, positions.reshape(1, 3), two), "2 axes"), (lambda: rotate(q, k, positions, rotary), "same CUDA device"),
                        (lambda: append(q, k, k, positions, rotary, None, slots), "KvCache")):
        with pytest.raises(ValueError, match=match):
            call()
    rotary._turns = _there(rotary._turns)      # as if it were beside them
    for call, match in ((lambda: rotate(q, k, positions, rotary, q_weight=w[:5]), "q_weight"), (lambda: rotate(q, k, positions, rotary, q_weight=w, k_weight=w.half()), "same dtype"),
                        (lambda: append(q, k, k[:, :1], positions, rotary, _cache(dtype=torch.float32), slots), "same shape"),
                        (lambda: append(q, k, k, positions, rotary, _cache(heads=1, dtype=torch.float32), slots), "cache must have"),
                        (lambda: append(q, k, k, positions, rotary, _cache(), slots), "cache must have"),
                        (lambda: append(q, k, k, positions, rotary, _cache(dtype=torch.float32), slots.int()), "slots"),
                        (lambda: append(q, k, k, positions, rotary, _cache(dtype=torch.float32), slots[:2]), "slots")):
        with pytest.raises(ValueError, match=match):
            call()


def test_calls_of_attention_that_are_refused():
    q = _there(torch.zeros((3, 4, 64), dtype=torch.bfloat16))
    tables, lengths, shared = (_there(torch.zeros(s, dtype=torch.int32)) for s in ((3, 2), (3,), (2,)))

    def call(q=q, cache=None, tables=tables, lengths=lengths, **kw):
        return attention.shared_prefix_attention(q, _cache() if cache is None else cache, tables, lengths, **kw)

    wide = _there(torch.zeros((3, 4, 68), dtype=torch.bfloat16))
    for kw, match in ((dict(cache=3), "KvCache"), (dict(q=q.float()), "bfloat16 or float16"), (dict(q=q.half()), "dtype"), (dict(q=q[:, :3]), "multiple"),
                      (dict(q=q[..., :32], cache=_cache(dim=32)), "64 or 128"), (dict(cache=_cache(page=8)), "16 to"), (dict(tables=tables[:2]), "tables"),
                      (dict(tables=tables.long()), "tables"), (dict(lengths=lengths.long()), "lengths"), (dict(lengths=lengths[:2]), "lengths"),
                      (dict(prefix_length=-1), "negative"), (dict(prefix_length=5), "prefix_table"), (dict(prefix_length=33, prefix_table=shared), "prefix_table"),
                      (dict(prefix_length=5, prefix_table=shared.long()), "prefix_table"), (dict(q=wide[..., :64]), "aligned"), (dict(q=wide[..., 4:]), "aligned")):
        with pytest.raises(ValueError, match=match):
            call(**kw)
