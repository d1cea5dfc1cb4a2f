"""``GatedMlp`` as users keep one: what it holds is replaced, moved and refilled between calls."""
import pytest
import torch

from mpserve_b200 import mx4
from tests import _mx4 as ref

pytestmark = pytest.mark.gpu
HIDDEN, INTER = 256, 640


def _weight(rows, cols, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return mx4.quantize(torch.randn((rows, cols), generator=g, device="cuda") * 0.05)


def _vector(seed, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.rand(HIDDEN, generator=g, device="cuda") + 0.5).to(dtype)


def _fields(seed):
    return dict(gate_proj=_weight(INTER, HIDDEN, seed), up_proj=_weight(INTER, HIDDEN, seed + 1), down_proj=_weight(HIDDEN, INTER, seed + 2),
                pre_weight=_vector(seed + 3), post_weight=_vector(seed + 4), gate=_vector(seed + 5), next_weight=_vector(seed + 6))


def _block(fields):
    f = dict(fields)
    return mx4.GatedMlp(f.pop("gate_proj"), f.pop("up_proj"), f.pop("down_proj"), **f)


def _h(tokens, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn((tokens, HIDDEN), generator=g, device="cuda").to(torch.bfloat16)


def _equal(got, want):
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("tokens", [1, 40])
@pytest.mark.parametrize("field", ["gate_proj", "up_proj", "down_proj", "pre_weight", "post_weight", "gate", "next_weight"])
def test_a_replaced_attribute_counts_from_the_next_call_on(field, tokens):
    fields, others, h = _fields(10), _fields(20), _h(tokens)
    block = _block(fields)
    old = [t.clone() for t in block(h)]
    fields[field] = others[field]
    setattr(block, field, others[field])
    ref.poison()                        # the memory of what was replaced holds something else
    got = block(h)
    _equal(got, _block(fields)(h))
    assert not torch.equal(got[1], old[1])


@pytest.mark.parametrize("field", ["pre_weight", "post_weight", "gate", "next_weight"])
def test_a_storage_swapped_under_a_tensor_counts_too(field):
    fields, others, h = _fields(10), _fields(20), _h(3)
    fields = {k: torch.nn.Parameter(v, requires_grad=False) if isinstance(v, torch.Tensor) else v for k, v in fields.items()}
    block = _block(fields)
    block(h)
    if field in ("pre_weight", "gate"):                     # (the other two share a dtype)
        fields[field].data = others[field].float()
    else:
        fields[field].data = others[field]
    ref.poison()
    _equal(block(h), _block({**fields, field: fields[field].data})(h))


def test_scalars_and_absent_parts_are_attributes_as_well():
    fields, h = _fields(10), _h(5)
    block = _block(fields)
    block.residual_scale, block.eps, block.activation, block.gate, block.post_weight = 0.5, 1e-3, "gelu", None, None
    want = mx4.GatedMlp(fields["gate_proj"], fields["up_proj"], fields["down_proj"], pre_weight=fields["pre_weight"], next_weight=fields["next_weight"],
                        residual_scale=0.5, eps=1e-3, activation="gelu")(h)
    _equal(block(h), want)
    block.next_weight = None
    joined, n = block(h)
    assert n is None and torch.equal(joined, want[0])
    assert (block.hidden, block.inter) == (HIDDEN, INTER)


def test_what_does_not_fit_is_refused_when_it_is_used():
    fields, h = _fields(10), _h(5)
    for field, value, match in (("down_proj", fields["up_proj"], "down_proj"), ("up_proj", None, "Mx4Tensor"), ("pre_weight", torch.ones(8, device="cuda"), "vector of 256"),
                                ("post_weight", _vector(1, torch.float32), "same dtype"), ("gate", torch.ones((4, 1), device="cuda"), "gate must be contiguous"),
                                ("next_weight", torch.ones(HIDDEN), "same CUDA device"), ("activation", "relu", "activation")):
        block = _block(fields)
        setattr(block, field, value)
        with pytest.raises(ValueError, match=match):
            block(h)
