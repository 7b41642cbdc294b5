"""The microscaled format stated once more, in float64 on the CPU and element by element where that is clearest."""
import numpy as np
import torch

BLOCK, CHUNK = 32, 128
E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
E4M3 = np.array([(c % 8) * 2.0 ** -9 if c < 8 else (8 + c % 8) * 2.0 ** (c // 8 - 10) for c in range(127)])
VALUES = {4: E2M1, 8: E4M3}
EMAX = {4: 2, 8: 8}


def padded(k):
    return -(-k // CHUNK) * CHUNK


def quantize(x, bits):
    """Codes ``[rows, padded]`` (one per element) and scales ``[rows, padded / 32]`` of float64 rows, as int arrays."""
    x = np.asarray(x, dtype=np.float64)
    rows, k = x.shape
    full = np.zeros((rows, padded(k)))
    full[:, :k] = x
    blocks = full.reshape(rows, -1, BLOCK)
    finite = np.isfinite(blocks).all(axis=2)
    top = np.where(finite, np.abs(np.where(np.isfinite(blocks), blocks, 0.0)).max(axis=2), 1.0)
    exponent = np.frexp(top)[1] - 1 + 127                            # biased; below float32's normal range it counts as 0
    exponent = np.where((top == 0) | (exponent < 0), 0, exponent)
    scales = np.where(finite, np.maximum(exponent - EMAX[bits], 0), 255)
    values = VALUES[bits]
    y = np.where(finite[:, :, None], blocks, 0.0) / np.ldexp(1.0, scales - 127)[:, :, None]
    a = np.abs(y)
    above = np.clip(np.searchsorted(values, a, side="left"), 1, len(values) - 1)
    below = above - 1
    down, up = a - values[below], values[above] - a
    code = np.where((up < down) | ((up == down) & (above % 2 == 0)), above, below)   # ties to the even mantissa
    code = code + np.signbit(y) * (1 << (bits - 1))
    return code.reshape(rows, -1).astype(np.int64), scales.astype(np.int64)


def numbers(codes, scales, bits):
    """float64 numbers that codes and scales (as ``quantize`` gives them) stand for, NaN where the scale is 255."""
    mag, sign = codes % (1 << (bits - 1)), codes >> (bits - 1)
    q = VALUES[bits][np.minimum(mag, len(VALUES[bits]) - 1)] * (1 - 2 * sign)
    f = np.where(scales == 255, np.nan, np.ldexp(1.0, scales - 127))
    return q * np.repeat(f, BLOCK, axis=1)


def pack(codes, scales, bits):
    """``codes`` and ``scales`` tensors of an ``MxRows`` (CPU)."""
    rows, kp = codes.shape
    c = codes.astype(np.uint8)
    held = c if bits == 8 else c[:, 0::2] | (c[:, 1::2] << 4)
    tiles = np.zeros((-(-rows // 128), kp // CHUNK, 512), dtype=np.uint8)
    for r in range(rows):
        for b in range(kp // BLOCK):
            tiles[r // 128, b // 4, r % 32 * 16 + r // 32 % 4 * 4 + b % 4] = scales[r, b]
    return torch.from_numpy(np.ascontiguousarray(held)), torch.from_numpy(tiles)


def unpack(q):
    """Codes and scales of an ``MxRows`` as ``quantize`` gives them."""
    held, tiles = q.codes.cpu().numpy().astype(np.int64), q.scales.cpu().numpy().astype(np.int64)
    rows = held.shape[0]
    codes = held
    if q.bits == 4:
        codes = np.empty((rows, held.shape[1] * 2), dtype=np.int64)
        codes[:, 0::2], codes[:, 1::2] = held & 15, held >> 4
    blocks = tiles.shape[1] * 4
    r, b = np.arange(rows)[:, None], np.arange(blocks)[None, :]
    return codes, tiles[r // 128, b // 4, r % 32 * 16 + r // 32 % 4 * 4 + b % 4]


def values_of(q):
    """float64 numbers of an ``MxRows``, its own columns."""
    codes, scales = unpack(q)
    return numbers(codes, scales, q.bits)[:, : q.cols]


def rounding(exact, bits):
    """How far the nearest number of the format may lie from each of ``exact``, given that the format's scale may follow from
    a block's largest magnitude that is off in its last bits: half a step of the element type relative to the number (1/16 or
    1/4), half a step of its smallest numbers, and what saturation cuts off (448 of 512, 6 of 8).  A scale that falls on the
    other side of a power of two doubles the steps."""
    exact = np.asarray(exact, dtype=np.float64)
    rows, k = exact.shape
    full = np.zeros((rows, padded(k)))
    full[:, :k] = np.abs(exact)
    top = full.reshape(rows, -1, BLOCK).max(axis=2)
    unit = np.ldexp(1.0, np.frexp(top * (1 + 1e-4))[1] - 1 - EMAX[bits])
    unit = np.repeat(unit, BLOCK, axis=1)[:, :k]
    relative, smallest = (1 / 8, 2.0 ** -10) if bits == 8 else (1 / 4, 0.25)
    return relative * np.abs(exact) + smallest * unit
