"""What may be read while ``h`` is updated in place: nothing that another row's CTA writes.  Addresses alone decide, so this runs anywhere."""
import pytest
import torch

from mpserve_b200 import mx4

BUF = torch.zeros((12, 64))


def _check(h, *others):
    mx4._check_inplace(h, *_extent(h), [(f"t{i}", t, *_extent(t)) for i, t in enumerate(others)])


def _extent(t):
    if t.dim() == 1:
        return 1, t.numel(), t.numel()
    return t.shape[0], t.shape[1], t.stride(0) if t.shape[0] > 1 else t.shape[1]


@pytest.mark.parametrize("h,other", [
    (BUF[:4], BUF[4:8]), (BUF[4:8], BUF[:4]),                       # rows apart
    (BUF[:, :32], BUF[:, 32:]), (BUF[:, 32:], BUF[:, :32]),         # columns of one matrix
    (BUF[:, 8:24], BUF[:, 40:]), (BUF[1:5, 40:], BUF[2:9, 8:24]),   # rows shifted, columns apart
    (BUF, BUF), (BUF[:, :32], BUF[:, :32]), (BUF[3:4], BUF[3:4]),   # itself
    (BUF[:1], BUF[1:2]), (BUF[2:2], BUF), (BUF[:5], BUF[5]),
    (BUF[:, :32], torch.zeros((12, 32))),
])
def test_allowed(h, other):
    _check(h, other)


@pytest.mark.parametrize("h,other", [
    (BUF[:4], BUF[1:5]), (BUF[1:5], BUF[:4]),                       # a row on
    (BUF[:, :32], BUF[:, 16:48]), (BUF[:, 16:48], BUF[:, :32]),     # some columns
    (BUF[:, 8:40], BUF[1:, :9]),
    (BUF, BUF.view(24, 32)), (BUF[:6], BUF[::2]),                   # another pitch
    (BUF[:6], BUF[2]), (BUF[:6], BUF.view(-1)[70:80]),              # a vector out of it
    (BUF[:4], BUF.view(torch.bfloat16)[:4, :64]),                   # another type in the same place
    (BUF[3:4], BUF[3:4, :32]),
    (BUF, BUF[:1].expand(12, 64)),
])
def test_refused(h, other):
    with pytest.raises(ValueError, match="shares memory with h"):
        _check(h, torch.zeros(3), other)


def test_rows_that_share_memory():
    with pytest.raises(ValueError, match="rows that share memory"):
        _check(BUF[:1].expand(4, 64))
