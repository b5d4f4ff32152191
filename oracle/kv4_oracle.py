"""The 4-bit KV cache restated in float64 numpy, from the format's definition (used as checker only).

Every function walks dims, tokens or bytes by their place in the format; none shares code or layout
tricks with the kernels."""
import functools

import numpy as np

MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
MIN_EXP, MAX_EXP = -120, 125


def code_values():
    """Value of each of the 16 codes."""
    return np.concatenate([MAGNITUDES, -MAGNITUDES])


def round_code(a):
    """Code 0..7 of magnitudes a >= 0: nearest value, ties to the even code, 6 from 5 on up."""
    a = np.asarray(a, dtype=np.float64)
    best = np.zeros(a.shape, dtype=np.uint8)
    gap = np.abs(a - MAGNITUDES[0])
    for code in range(1, 8):
        d = np.abs(a - MAGNITUDES[code])
        take = (d < gap) | ((d == gap) & (code % 2 == 0))
        best = np.where(take, code, best).astype(np.uint8)
        gap = np.where(take, d, gap)
    return best


def quantise(x):
    """x [..., D] float64 -> codes [..., D] (0..15) and scale bytes [..., D // 32]."""
    x = np.asarray(x, dtype=np.float64)
    blocks = x.reshape(x.shape[:-1] + (-1, 32))
    top = np.abs(blocks).max(-1)
    bad = ~np.isfinite(blocks).all(-1)
    e = np.full(top.shape, MIN_EXP)
    for k in range(MIN_EXP, MAX_EXP):                # the smallest power of two with top <= 6 * 2^e
        e = np.where(top > 6.0 * 2.0 ** k, k + 1, e)
    byte = np.where(bad, 255, e + 127).astype(np.uint8)
    scaled = np.where(bad[..., None], 0.0, np.abs(np.where(bad[..., None], 0.0, blocks))) / (2.0 ** e)[..., None]
    code = round_code(scaled)
    code = np.where(np.signbit(blocks) & ~bad[..., None], code + 8, code).astype(np.uint8)
    return code.reshape(x.shape), byte


def dequantise(code, byte):
    """Codes and scale bytes -> float64 values (byte 255: NaN)."""
    v = code_values()[code]
    with np.errstate(over='ignore'):
        s = np.where(byte == 255, np.nan, 2.0 ** (byte.astype(np.float64) - 127))
    return v * np.repeat(s, 32, axis=-1)


def code_place(D, row, dim, value_form):
    """(byte offset within a record, shift) of the code of token `row` (0..15) and dim."""
    if value_form:
        block, pair = dim // 32, (dim % 32) // 2
        group, j = row // 4, row % 4
        return ((group * 16 + pair) * (D // 32) + block) * 4 + j, 4 * (dim % 2)
    return row * (D // 2) + dim // 2, 4 * (dim % 2)


def scale_place(D, row, block, value_form):
    """Byte offset within a record of the scale of token `row`'s dims 32 block .. + 31."""
    if value_form:
        return 8 * D + (row // 4 * (D // 32) + block) * 4 + row % 4
    return 8 * D + row * (D // 32) + block


def record_bytes(D):
    return 8 * D + 16 * (D // 32)


def write_row(record, row, code, byte, value_form):
    """Put one token's codes [D] and scale bytes [D // 32] into record (uint8 [record_bytes])."""
    D = code.shape[0]
    for d in range(D):
        at, shift = code_place(D, row, d, value_form)
        record[at] = (int(record[at]) & (0xF0 >> shift)) | int(code[d]) << shift
    for b in range(D // 32):
        record[scale_place(D, row, b, value_form)] = byte[b]


@functools.lru_cache(None)
def _places(D, value_form):
    at = np.array([[code_place(D, r, d, value_form)[0] for d in range(D)] for r in range(16)])
    shift = np.array([[code_place(D, r, d, value_form)[1] for d in range(D)] for r in range(16)])
    scale = np.array([[scale_place(D, r, b, value_form) for b in range(D // 32)] for r in range(16)])
    return at, shift, scale


def pack(code, byte, value_form):
    """codes [..., 16, D], scale bytes [..., 16, D // 32] -> records [..., record_bytes]."""
    D = code.shape[-1]
    at, shift, scale = _places(D, value_form)
    out = np.zeros(code.shape[:-2] + (record_bytes(D),), dtype=np.uint8)
    for r in range(16):
        for d in range(D):
            out[..., at[r, d]] |= (code[..., r, d] << shift[r, d]).astype(np.uint8)
        for b in range(D // 32):
            out[..., scale[r, b]] = byte[..., r, b]
    return out


def unpack(record, value_form):
    """records [..., record_bytes] -> values [..., 16, D]."""
    D = record.shape[-1] * 2 // 17
    at, shift, scale = _places(D, value_form)
    return dequantise((record[..., at] >> shift) & 15, record[..., scale])


def gather(cache, table, n, head, value_form):
    """Positions 0 .. n - 1 of one head through a block table; cache [blocks, heads, tiles, bytes] -> [n, D]."""
    tiles = cache.shape[2]
    rows = [unpack(cache[table[t // (16 * tiles)], head, t // 16 % tiles], value_form) for t in range(0, n, 16)]
    return np.concatenate(rows)[:n]


def rotate(x, cos, sin, interleaved):
    """x [T, H, D] float64, cos / sin [T, R / 2]."""
    out = np.array(x, dtype=np.float64)
    half = cos.shape[1]
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        c, s = cos[:, None, i].astype(np.float64), sin[:, None, i].astype(np.float64)
        out[..., a] = x[..., a] * c - x[..., b] * s
        out[..., b] = x[..., b] * c + x[..., a] * s
    return out


def attend(q, k, v, scale, limits):
    """q [n, D] over k / v [m, D]; query i sees rows 0 .. limits[i] (none: zeros).  Returns (out, the
    weighted mean of |v|, the largest sum |q| |k| |scale| of a score): what an error bound needs."""
    out, size = np.zeros(q.shape), np.zeros(q.shape)
    big = np.zeros((q.shape[0], 1))
    for i in range(q.shape[0]):
        m = limits[i] + 1
        if m <= 0:
            continue
        s = k[:m] @ q[i] * scale
        w = np.exp(s - s.max())
        w /= w.sum()
        out[i], size[i] = w @ v[:m], w @ np.abs(v[:m])
        big[i] = (np.abs(k[:m]) @ np.abs(q[i])).max() * abs(scale)
    return out, size, big
