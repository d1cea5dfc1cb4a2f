"""What uint16 scales are: bits of no particular type to the AWQ entries, float16's to the INT4 products."""
import pytest
import torch

from mpserve_b200 import encoder, workloads


def test_the_awq_entries_name_no_type():
    w, codes, scales = torch.zeros((4, 128), dtype=torch.bfloat16), torch.zeros((4, 128), dtype=torch.uint8), torch.zeros((4, 1), dtype=torch.bfloat16)
    for call in (lambda: encoder.build_awq_bucket(w, codes, scales, 11, 256), lambda: encoder.build_awq_by_scale(w, codes, scales, 11, 256, 1024),
                 lambda: encoder.build_awq_shared(w, codes, scales, 11)):
        with pytest.raises(ValueError, match=r"scales_u16 must be torch.uint16 \(raw bits\)"):
            call()


@pytest.mark.gpu
def test_a_weight_of_the_awq_path_has_the_same_values_in_products():
    from mpserve_b200 import int4

    c = workloads.quantize_awq(workloads.random_weight(64, 512, 3, "normal"))
    codes, scales, zeros = c.int4_u8.cuda(), c.scales_u16.cuda(), c.zeros_u8.cuda()
    column = torch.arange(512, device="cuda") // c.group
    difference = codes.double() - zeros.double()[:, column]
    for given, scale in ((scales, scales.view(torch.float16)), (scales.view(torch.float16), scales.view(torch.float16)), (scales.view(torch.bfloat16), scales.view(torch.bfloat16))):
        got = int4.from_parts(codes, given, zeros, group=c.group).dequantize(torch.float32)
        assert torch.equal(got.double(), difference * scale.double()[:, column])      # a whole number of 5 bits times 11 or 8: exact
    # the rounded weight is within half a step of a scale, and a step of the zero point's, of what was quantised
    got = int4.from_parts(codes, scales, zeros, group=c.group).dequantize(torch.float32)
    assert ((got - c.bf16.cuda().float()).abs() <= 1.01 * scales.view(torch.float16).float()[:, column]).all()
