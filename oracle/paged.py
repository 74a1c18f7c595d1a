"""Oracle (test infrastructure only): the paged KV cache held in 4 bits.

The format is OCP MX FP4 (blocks of 32 channels, E2M1 elements, one E8M0 scale), restated in numpy;
attention is the f64 softmax over the rows that the codes stand for. No counterpart in the
reference, whose cache is packed 16-bit rows.
"""

from __future__ import annotations

import numpy as np

MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def scale_exponent(amax: np.ndarray, f16: bool) -> np.ndarray:
    """log2 of a block's scale: the largest X = 2^e with 4 X <= amax, doubled where amax >= 7 X."""
    amax = np.asarray(amax, np.float64)
    significand, exponent = np.frexp(amax)  # amax = significand * 2^exponent, in [0.5, 1)
    e = exponent - 1 - 2 + (significand >= 7 / 8)
    low, high = (-23, 13) if f16 else (-125, 125)
    return np.clip(np.where(amax == 0, low, e), low, high).astype(np.int64)


def quantise(rows: np.ndarray, f16: bool = False):
    """rows [..., dim] -> (codes uint8 [..., dim / 2], scales uint8 [..., dim / 32]). By search for
    the nearest magnitude, ties to the even code."""
    blocks = np.asarray(rows, np.float64).reshape(rows.shape[:-1] + (rows.shape[-1] // 32, 32))
    finite = np.isfinite(blocks).all(-1)
    blocks = np.where(finite[..., None], blocks, 0.0)
    e = scale_exponent(np.abs(blocks).max(-1), f16)
    ratio = np.abs(blocks) / np.exp2(e)[..., None]
    distance = np.abs(ratio[..., None] - MAGNITUDES)
    nearest = distance == distance.min(-1, keepdims=True)
    even = nearest & (np.arange(8) % 2 == 0)
    code = np.where(even.any(-1), even.argmax(-1), nearest.argmax(-1))
    code = code + 8 * np.signbit(blocks)
    code = np.where(finite[..., None], code, 0).reshape(rows.shape).astype(np.uint8)
    scales = np.where(finite, e + 127, 255).astype(np.uint8)
    return code[..., 0::2] | code[..., 1::2] << 4, scales


def values(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """f64 rows [..., dim]."""
    nibbles = np.stack((codes & 15, codes >> 4), -1)
    nibbles = nibbles.reshape(codes.shape[:-1] + (codes.shape[-1] // 16, 32))
    size = MAGNITUDES[nibbles & 7] * np.exp2(scales.astype(np.float64) - 127)[..., None]
    rows = np.where(nibbles >= 8, -size, size)
    rows = np.where((scales == 255)[..., None], np.nan, rows)
    return rows.reshape(codes.shape[:-1] + (2 * codes.shape[-1],))


def rotate(rows: np.ndarray, cos: np.ndarray, sin: np.ndarray) -> np.ndarray:
    """f32 rows [..., dim], tables [..., half]: each product and sum rounded to f32."""
    half = cos.shape[-1]
    a, b = rows[..., :half], rows[..., half:2 * half]
    return np.concatenate((a * cos - b * sin, b * cos + a * sin, rows[..., 2 * half:]), -1)


def page_bytes(page_size: int, dim: int) -> int:
    return page_size * (dim + dim // 16 + 4)


def store(pages: np.ndarray, page, slot, page_size: int, keys, key_scales, vals, value_scales,
          positions) -> None:
    """Rows' codes, scales and positions into uint8 [pages, page_bytes], row i in slot slot[i] of
    page page[i]."""
    count, half = keys.shape
    sections = (keys, vals, key_scales, value_scales,
                np.asarray(positions, np.float32).reshape(count, 1).view(np.uint8))
    start = 0
    for section in sections:
        size = section.shape[1]
        at = start + np.asarray(slot)[:, None] * size + np.arange(size)
        pages[np.asarray(page)[:, None], at] = section
        start += page_size * size
    assert start == page_bytes(page_size, 2 * half)


def load(pages: np.ndarray, table_row: np.ndarray, count: int, page_size: int, dim: int):
    """f64 keys and values [count, dim] and f32 positions [count] of a segment."""
    half, blocks = dim // 2, dim // 32
    index = np.arange(count)
    raw, slot = pages[table_row[index // page_size]], index % page_size
    cut, start = [], 0
    for width in (half, half, blocks, blocks, 4):
        section = raw[:, start:start + page_size * width].reshape(count, page_size, width)
        cut.append(section[index, slot])
        start += page_size * width
    positions = np.ascontiguousarray(cut[4]).view(np.float32).reshape(count)
    return values(cut[0], cut[2]), values(cut[1], cut[3]), positions


def attention(queries: np.ndarray, rows, lengths, counts, kv_heads: int, scale=None) -> np.ndarray:
    """queries [B, Hq, L, d]; rows[s] = (keys, values) f64 of segment s, new rows included ->
    f64 [B, L, Hq * d]."""
    batch, query_heads, length, dim = queries.shape
    groups = query_heads // kv_heads
    scale = dim ** -0.5 if scale is None else scale
    out = np.zeros((batch, length, query_heads, dim))
    for b in range(batch):
        for head in range(query_heads):
            s = b * kv_heads + head // groups
            keys, vals = rows[s]
            for i in range(min(int(counts[b]), length)):
                n = min(int(lengths[s]) + i + 1, len(keys))
                if n <= 0:
                    continue
                scores = keys[:n] @ queries[b, head, i].astype(np.float64) * scale
                weights = np.exp(scores - scores.max())
                out[b, i, head] = weights @ vals[:n] / weights.sum()
    return out.reshape(batch, length, query_heads * dim)
