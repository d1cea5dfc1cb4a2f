"""MXFP4 in 64 bits, from the format's definition, for the tests of ``mpserve_b200.mx4``."""
import numpy as np
import torch

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
# half the distance of neighbouring numbers, relative
ROUND = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def encode(x: np.ndarray):
    """float64 ``[rows, cols]`` -> codes ``uint8 [rows, cols]`` and scale bytes ``[rows, ceil(cols / 32)]``."""
    rows, cols = x.shape
    codes = np.zeros((rows, cols), np.uint8)
    scales = np.zeros((rows, -(-cols // 32)), np.uint8)
    for b in range(scales.shape[1]):
        v = x[:, b * 32:(b + 1) * 32]
        a = np.abs(v)
        bad = ~np.isfinite(v).all(axis=1)
        m = np.where(bad, 0.0, a.max(axis=1))
        e = np.full(rows, -127, np.int64)
        pos = m > 0
        e[pos] = np.maximum(np.floor(np.log2(m[pos])).astype(np.int64) - 2, -127)
        # log2 of a number just below a power of two may round up to it
        e[pos] -= ((np.ldexp(1.0, e[pos] + 2) > m[pos]) & (e[pos] > -127)).astype(np.int64)
        with np.errstate(invalid="ignore", over="ignore"):
            y = np.where(bad[:, None], 0.0, np.ldexp(np.where(np.isfinite(a), a, 0.0), -e[:, None].astype(np.int32)))
        d = np.abs(y[:, :, None] - GRID)
        near = d == d.min(axis=2, keepdims=True)
        # of two equally near ones the even code
        code = np.where(near.sum(axis=2) == 2, (np.argmax(near, axis=2) + 1) // 2 * 2, np.argmax(near, axis=2))
        codes[:, b * 32:(b + 1) * 32] = code + 8 * (np.signbit(v) & ~bad[:, None])
        scales[:, b] = np.where(bad, 255, e + 127)
    return codes, scales


def decode(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int32) - 127))
    v = np.where(codes >= 8, -1.0, 1.0) * GRID[codes & 7]
    return v * np.repeat(s, 32, axis=1)[:, :codes.shape[1]]


def pack(codes: np.ndarray) -> np.ndarray:
    c = np.pad(codes, ((0, 0), (0, codes.shape[1] % 2)))
    return (c[:, 0::2] | (c[:, 1::2] << 4)).astype(np.uint8)


def unpack(packed: np.ndarray, cols: int) -> np.ndarray:
    c = np.empty((packed.shape[0], packed.shape[1] * 2), np.uint8)
    c[:, 0::2], c[:, 1::2] = packed & 15, packed >> 4
    return c[:, :cols]


def to64(t: torch.Tensor) -> np.ndarray:
    return t.detach().cpu().double().numpy()


def values(q) -> np.ndarray:
    """What an ``Mx4Tensor`` stands for, in 64 bits, by way of its parts."""
    codes, scales = (t.cpu().numpy() for t in q.parts())
    return decode(unpack(codes, q.cols), scales)


def spacing(units: np.ndarray) -> np.ndarray:
    return np.where(units < 2, 0.5, np.where(units < 4, 1.0, 2.0))


def check_rounded(q, exact: np.ndarray, off: np.ndarray) -> None:
    """``q`` is what some values within ``off`` of ``exact`` are quantised to."""
    got = values(q)
    codes, scales = (t.cpu().numpy() for t in q.parts())
    assert got.shape == exact.shape
    pad = (-exact.shape[1]) % 32
    blocks = lambda v: np.pad(v, ((0, 0), (0, pad))).reshape(v.shape[0], -1, 32).max(axis=2)  # noqa: E731
    top, slack = blocks(np.abs(exact)), blocks(off)

    def scale_of(m):
        return np.where(m > 0, np.maximum(np.floor(np.log2(np.maximum(m, 1e-300))) - 2, -127), -127) + 127

    assert ((scales >= scale_of(np.maximum(top - slack, 0))) & (scales <= scale_of(top + slack))).all()
    s = np.repeat(np.ldexp(1.0, scales.astype(np.int32) - 127), 32, axis=1)[:, :exact.shape[1]]
    units = np.abs(exact) / s
    low = np.maximum(units - off / s, 0)
    # the nearest code's distance, or that to 6 for what lies above it
    most = np.maximum(np.maximum(spacing(low), spacing(units + off / s)) / 2, units - 6) * s + off
    assert (np.abs(got - exact) <= most * (1 + 1e-12)).all()


def poison(nbytes: int = 1 << 26) -> None:
    """Memory that the allocator hands out next holds NaN scales and full codes."""
    del_me = [torch.full((size,), 255, dtype=torch.uint8, device="cuda") for size in (nbytes, 1 << 20, 1 << 20, 1 << 20, 1 << 16, 1 << 16)]
    torch.cuda.synchronize()
    del del_me
