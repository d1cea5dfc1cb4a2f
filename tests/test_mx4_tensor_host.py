"""An ``Mx4Tensor`` whose memory the kernels could not read is refused, when it is made or where it is used, before any launch."""
import pytest
import torch

from mpserve_b200 import mx4

TILE = 17408


def _data(nbytes, **kw):
    return torch.zeros(nbytes, dtype=torch.uint8, **kw)


@pytest.mark.parametrize("data,rows,cols,shape,match", [
    (_data(TILE - 1), 1, 1, None, "17407 bytes"),
    (_data(TILE), 129, 256, None, "17408 bytes"),
    (_data(TILE), 128, 257, None, "17408 bytes"),
    (_data(0), 1, 1, None, "0 bytes"),
    (_data(2 * TILE).view(2, TILE), 129, 256, None, "flat"),
    (_data(2 * TILE)[::2], 4, 64, None, "flat"),
    (_data(TILE).view(torch.int8), 4, 64, None, "uint8"),
    ([0] * TILE, 4, 64, None, "uint8"),
    (_data(TILE), -1, 64, None, "rows"),
    (_data(TILE), 4, 0, None, "column"),
    (_data(TILE), 4, (1 << 24) + 1, None, "2\\^24"),
    (_data(TILE), 4, 64, (5, 64), "shape"),
    (_data(TILE), 4, 64, (4, 65), "shape"),
    (_data(TILE), 4, 64, (2, 3, 64), "shape"),
    (_data(TILE), 4, 64, (-2, -2, 64), "shape"),
    (_data(TILE), 4, 64, (), "shape"),
])
def test_what_does_not_fit_is_refused_when_it_is_made(data, rows, cols, shape, match):
    with pytest.raises(ValueError, match=match):
        mx4.Mx4Tensor(data, rows, cols, shape)


def test_what_fits_is_taken_and_kept():
    q = mx4.Mx4Tensor(_data(3 * TILE), 130, 200, (2, 65, 200))
    assert (q.rows, q.cols, q.shape, q.data.numel()) == (130, 200, (2, 65, 200), 3 * TILE)
    assert mx4.Mx4Tensor(_data(0), 0, 64).shape == (0, 64) and mx4.Mx4Tensor(_data(TILE), 1, 64, torch.Size([64])).shape == (64,)
    for name in ("data", "rows", "cols", "shape"):
        with pytest.raises(AttributeError):
            setattr(q, name, getattr(q, name))


def test_matrices_in_host_memory_are_refused_everywhere():
    q = mx4.Mx4Tensor(_data(TILE), 64, 64)
    w = torch.ones(64)
    for call in (lambda: q.dequantize(), lambda: mx4.dequantize(q), lambda: q.parts(), lambda: mx4.linear(q, q), lambda: mx4.gated_linear(q, q, q),
                 lambda: mx4.GatedMlp(q, q, q, pre_weight=w)):
        with pytest.raises(ValueError, match="CUDA tensor"):
            call()


def test_a_tensor_cut_off_later_is_refused(monkeypatch):
    """As if its memory were a GPU's: the check comes before anything else is done with it."""
    data = _data(TILE)
    q = mx4.Mx4Tensor(data, 4, 64)
    data.resize_(100)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda self: 0)
    for call in (lambda: q.dequantize(), lambda: q.parts(), lambda: mx4.linear(q, q)):
        with pytest.raises(ValueError, match="lost a part"):
            call()
