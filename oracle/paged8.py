"""Oracle (test infrastructure only): the paged KV cache held in 8 bits.

Rows of E4M3 codes with a power-of-two scale for each 16 rows of a head, restated in numpy by search
over the codes' magnitudes; attention, rotation and rows in 4 bits are oracle.paged's. No counterpart
in the reference, whose cache is packed 16-bit rows.
"""

from __future__ import annotations

import numpy as np

from .paged import attention, rotate  # noqa: F401

BLOCK = 16
MAGNITUDES = np.array([m * 2.0 ** -9 for m in range(8)]
                      + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)][:-1])
assert len(MAGNITUDES) == 127 and MAGNITUDES[-1] == 448.0


def scale_exponent(amax, f16: bool = False):
    """The smallest e with amax < 464 2^e (464 is halfway from 448 to the next such number)."""
    significand, power = np.frexp(np.asarray(amax, np.float64) / 464.0)
    e = np.where(significand == 0.0, -2000, power)  # amax / 464 < 2^power, and not < 2^(power - 1)
    return np.clip(e, -117, 7 if f16 else 119).astype(np.int64)


def four_bits(rows):
    """Rounded to four significant bits, ties to even; below f32's normal numbers to their 2^-129."""
    _, power = np.frexp(rows)
    unit = np.exp2(np.maximum(power, -125) - 4.0)
    return np.round(rows / unit) * unit


def encode(rows, exponent):
    """Codes uint8 of finite or non-finite elements at scale 2^exponent (broadcast)."""
    rows = np.asarray(rows, np.float64)
    finite = np.isfinite(rows)
    size = np.abs(four_bits(np.where(finite, rows, 0.0))) * np.exp2(-np.asarray(exponent, np.float64))
    code = np.searchsorted(MAGNITUDES, size, side="right") - 1  # cut to the code at or below
    return np.where(finite, code + 128 * np.signbit(rows), 255).astype(np.uint8)


def values(codes, exponent):
    """f64 elements of codes at scale 2^exponent (broadcast)."""
    size = np.append(MAGNITUDES, np.nan)[codes & 127] * np.exp2(np.asarray(exponent, np.float64))
    return np.where(codes >= 128, -size, size)


def page_bytes(page_size: int, dim: int) -> int:
    return page_size * (2 * dim + 8)


def places(slot, page_size: int, dim: int):
    """Byte offsets in a page of rows' keys and values [..., dim], positions [..., 4] and their blocks'
    scales [..., 2]."""
    slot, c = np.asarray(slot)[..., None], np.arange(dim)
    block, row = slot // BLOCK, slot % BLOCK
    keys = block * BLOCK * dim + c // 16 * 256 + row * 16 + c % 16
    quads = page_size * dim + slot // 4 * 4 * dim + 4 * c + slot % 4
    positions = 2 * page_size * dim + 4 * slot + np.arange(4)
    return keys, quads, positions, page_size * (2 * dim + 4) + 2 * block + np.arange(2)


def append(pages, table_row, length: int, page_size: int, keys, vals, positions, f16: bool = False):
    """Stores rows [n, dim] behind a segment's `length` rows, in place."""
    n, dim = keys.shape
    for first in range(length // BLOCK * BLOCK, length + n, BLOCK):
        index = np.arange(first, min(first + BLOCK, length + n))
        page, slot = table_row[first // page_size], index % page_size
        spots = places(slot, page_size, dim)
        fresh = index >= length
        for which, rows in enumerate((keys, vals)):
            new = rows[index[fresh] - length]
            e = scale_exponent(np.abs(np.where(np.isfinite(new), new, 0.0)).max(), f16)
            at = spots[3][0, which]
            if not fresh[0]:  # older rows: theirs, or codes cut to the larger scale
                was = int(pages[page, at]) - 127
                e = max(e, was)
                old = pages[page, spots[which][~fresh]]
                pages[page, spots[which][~fresh]] = np.where(
                    old & 127 == 127, 255, encode(values(old, was), e) & 127 | old & 128)
            pages[page, spots[which][fresh]] = encode(new, e)
            pages[page, at] = e + 127
        pages[page, spots[2][fresh]] = np.asarray(
            positions, np.float32)[index[fresh] - length].reshape(-1, 1).view(np.uint8)


def codes(pages, table_row, rows, page_size: int, dim: int):
    """Rows' codes of keys and values [n, dim], exponents [n, 2] and positions [n]."""
    rows = np.asarray(rows, np.int64)
    page, slot = table_row[rows // page_size][:, None], rows % page_size
    keys, quads, where, scales = places(slot, page_size, dim)
    positions = np.ascontiguousarray(pages[page, where]).view(np.float32).reshape(-1)
    return pages[page, keys], pages[page, quads], pages[page, scales].astype(int) - 127, positions


def load(pages, table_row, count: int, page_size: int, dim: int):
    """f64 keys and values [count, dim] and f32 positions [count] of a segment."""
    k, v, e, positions = codes(pages, table_row, np.arange(count), page_size, dim)
    return values(k, e[:, :1]), values(v, e[:, 1:]), positions


def compact(pages, table_row, kept, target_row, page_size: int, dim: int):
    """Moves a segment's rows `kept` to the pages of target_row, in place."""
    k, v, e, positions = codes(pages, table_row, kept, page_size, dim)
    for first in range(0, len(kept), BLOCK):
        part = slice(first, min(first + BLOCK, len(kept)))
        page, slot = target_row[first // page_size], np.arange(part.start, part.stop) % page_size
        spots = places(slot, page_size, dim)
        for which, old in enumerate((k[part], v[part])):
            was = e[part, which:which + 1]
            top = was.max()
            pages[page, spots[which]] = np.where(old & 127 == 127, 255,
                                                 encode(values(old, was), top) & 127 | old & 128)
            pages[page, spots[3][0, which]] = top + 127
        pages[page, spots[2]] = positions[part].astype(np.float32).reshape(-1, 1).view(np.uint8)
