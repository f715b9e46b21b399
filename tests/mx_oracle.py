"""MXFP4 and the quantized cache in NumPy, from their definitions (float64 unless a step is defined in
float32): the oracle of the microscaled and cache tests."""

import numpy as np

VALUES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def encode(x):
    """(element codes (rows, K) uint8, scale bytes (rows, K / 32) uint8, whether an element fits)."""
    x = np.asarray(x, dtype=np.float64)
    b = x.reshape(x.shape[0], -1, 32)
    bad = ~np.isfinite(b).all(-1)
    b = np.where(bad[..., None], 0.0, b)
    top = np.abs(b).max(-1)
    _, e = np.frexp(top)
    exponent = np.where(top > 0, np.maximum(e.astype(np.int64) - 1 - 2, -127), -127)
    a = np.ldexp(np.abs(b), -exponent[..., None])
    # nearest element; of two equally near ones the one with the even index
    dist = np.abs(a[..., None] - VALUES)
    near = dist.min(-1, keepdims=True)
    is_near = dist == near
    first = is_near.argmax(-1)
    both = is_near.sum(-1) == 2
    code = np.where(both & (first % 2 == 1), first + 1, first).astype(np.uint8)
    code = code | (np.signbit(b).astype(np.uint8) << 3)
    code[bad] = 0
    byte = np.where(bad, 255, exponent + 127).astype(np.uint8)
    return code.reshape(x.shape), byte, ((a < 7.0) & ~bad[..., None]).reshape(x.shape)


def decode(code, byte):
    v = np.where(code & 8, -VALUES[code & 7], VALUES[code & 7])
    s = np.where(byte == 255, np.nan, np.ldexp(1.0, byte.astype(np.int64) - 127))
    return v * np.repeat(s, 32, axis=-1)


def pack(code):
    return code[..., 0::2] | (code[..., 1::2] << 4)


def unpack(packed):
    return np.stack((packed & 15, packed >> 4), -1).reshape(*packed.shape[:-1], -1)


def tile(byte):
    rows, blocks = byte.shape
    out = np.zeros(((rows + 127) // 128, (blocks + 7) // 8, 1024), dtype=np.uint8)
    r, b = np.meshgrid(np.arange(rows), np.arange(blocks), indexing="ij")
    out[r // 128, b // 8, b % 8 // 4 * 512 + r % 32 * 16 + r % 128 // 32 * 4 + b % 4] = byte
    return out


def quantize(x):
    code, byte, _ = encode(x)
    return pack(code), tile(byte)


def int8_rows(x):
    """Per-row int8 codes and float32 scales: the steps are binary32, as the encode defines them."""
    x = np.asarray(x, dtype=np.float32)
    scale = np.maximum(np.abs(x).max(-1) / np.float32(127.5), np.float32(1e-8)).astype(np.float32)
    q = np.rint((x / scale[..., None]).astype(np.float32))
    return np.clip(q, -128, 127).astype(np.int8), scale
