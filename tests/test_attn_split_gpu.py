"""How the work of attention behind a shared prefix is split: the longest prefixes."""
import math

import pytest
import torch

from mpserve_b200 import _lib, attention, mx4
from tests import _attn as ref

pytestmark = pytest.mark.gpu


def test_a_prefix_beyond_32_bits_of_cycles_is_split():
    # 160 times the same page of 2^20 keys: the softmax over one of them, and a denominator that is 160 times as large
    page, times = 1 << 20, 160
    g = ref.generator(1)
    k, v = ref.randn(g, 1, page, 1, 64, dtype=torch.bfloat16), (1 + 0.1 * ref.randn(g, 1, page, 1, 64)).to(torch.bfloat16)
    q = ref.randn(g, 1, 1, 64, dtype=torch.bfloat16)
    table = torch.zeros(times, dtype=torch.int32, device="cuda")
    tables, lengths = torch.zeros((1, 0), dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    cache, index = attention.KvCache(k, v), q.get_device()
    out, lse = attention.shared_prefix_attention(q, cache, tables, lengths, prefix_table=table, prefix_length=page * times, return_lse=True)
    one, one_lse = attention.shared_prefix_attention(q, cache, tables, lengths, prefix_table=table, prefix_length=page, return_lse=True)
    want, want_lse, off, _ = ref.attend(q, k, v, tables, lengths, table, page)
    ref.within(one, want, off)
    # a stretch is at most two SMs' share of the keys: 16 of them are one addition to a sum of values (off by 17 steps), one of them to each fourth of the denominator
    sms = torch.cuda.get_device_properties(index).multi_processor_count
    keys = 2 * page * times / sms
    far = (17 * keys / 16 + keys / 4 + sms + 100) * ref.STEP
    assert ((out.double() - want).abs() <= off + (far + ref.ROUND[out.dtype]) * v.double().abs().amax()).all()
    assert ((lse.double() - want_lse - math.log(times)).abs() <= 2 * far).all()
    # the number of stretches that the call chose is the first word of its scratch
    lib, need = _lib.load(), attention._scratch_bytes(index, 1, 0, page * times, page, 1, 1, 64, 0)
    scratch, ws = torch.zeros(need, dtype=torch.uint8, device="cuda"), mx4._workspace(index)
    args = _lib.PREFIX_ATTEND.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), 0, 0, 0, table.data_ptr(), 1, 0, page * times, 1, page, 64, 64,
                                   *k.stride()[:3], *v.stride()[:3], 1, 1, 64, 0, 0.125)
    _lib.check(lib.mps_prefix_attend_tokens(args, scratch.data_ptr(), need, ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream))
    assert sms // 2 < int(scratch[:4].view(torch.int32)) <= sms
