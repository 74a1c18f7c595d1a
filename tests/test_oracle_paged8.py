"""The 8-bit cache's oracle against independent statements of the format: torch's E4M3 conversion where
no small code is involved, exactness in the 16-bit types, the byte layout, and that a block's bytes do
not depend on the calls that its rows came in."""

import numpy as np
import pytest
import torch
from hypothesis import given, settings
from hypothesis import strategies as st

from oracle import paged8 as opaged


def test_scale_rule():
    got = opaged.scale_exponent(np.array([448.0, 463.9, 464.0, 465.0, 256.0, 232.0, 231.9, 1.0, 0.0, 3.4e38]))
    assert got.tolist() == [0, 0, 1, 1, 0, 0, -1, -8, -117, 119]
    assert opaged.scale_exponent(np.array([65504.0, 57344.0, 0.0]), True).tolist() == [7, 7, -117]


def test_magnitudes_are_torchs():
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    got = opaged.values(np.arange(256, dtype=np.uint8), 0)
    assert np.array_equal(got, codes, equal_nan=True)


@settings(max_examples=60, deadline=None)
@given(st.integers(0, 2 ** 32 - 1), st.integers(-20, 20))
def test_codes_are_torchs_rounding_but_for_the_small_ones(seed, exponent):
    rows = np.random.default_rng(seed).standard_normal((16, 64)) * 100 * 2.0 ** exponent
    rows = rows.astype(np.float32).astype(np.float64)
    e = opaged.scale_exponent(np.abs(rows).max())
    got = opaged.values(opaged.encode(rows, e), e)
    nearest = torch.from_numpy(rows * 2.0 ** -e).float().to(torch.float8_e4m3fn).double().numpy() * 2.0 ** e
    normal = np.abs(rows) >= 2.0 ** (e - 6)
    assert np.array_equal(got[normal], nearest[normal])
    # half of a step of the four bits, and less than the smallest code
    assert np.all(np.abs(got - rows) <= np.abs(rows) * 2.0 ** -4 + 2.0 ** (e - 9) * ~normal)
    assert np.array_equal(opaged.values(opaged.encode(got, e), e), got)


def test_ties_go_to_even_and_what_lies_under_the_smallest_code_is_cut():
    x = np.array([448.0, 1.0625, 1.1875, -1.0625, 2.0 ** -7 * 1.9, 2.0 ** -9 * 1.99, -(2.0 ** -10), 463.0])
    got = opaged.values(opaged.encode(x, 0), 0)
    expect = [448, 1, 1.25, -1, 2.0 ** -9 * 7, 2.0 ** -9 * 2, 0, 448]  # (1.99 is 2 in four bits)
    assert got.tolist() == expect


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_values_are_exact_in_the_16_bit_type(dtype):
    rng = np.random.default_rng(0)
    for power in range(-20, 15):
        rows = torch.from_numpy(rng.standard_normal((16, 64)) * 2.0 ** power).to(dtype).double().numpy()
        rows = np.clip(rows, -65504, 65504)
        e = opaged.scale_exponent(np.abs(rows).max(), dtype == torch.float16)
        got = opaged.values(opaged.encode(rows, e), e)
        assert np.array_equal(torch.from_numpy(got).to(dtype).double().numpy(), got)


def random_rows(rng, n, dim):
    return [rng.standard_normal((n, dim)) * np.exp2(rng.uniform(-9, 9, (n, 1))) for _ in range(2)]


@settings(max_examples=40, deadline=None)
@given(st.integers(0, 2 ** 32 - 1))
def test_a_blocks_bytes_do_not_depend_on_the_calls(seed):
    rng = np.random.default_rng(seed)
    page_size, dim, n = 32, 64, int(rng.integers(1, 70))
    rows, positions = random_rows(rng, n, dim), np.arange(n) + 2.0
    table, blank = np.array([2, 0, 3]), rng.integers(0, 256, (4, opaged.page_bytes(page_size, dim)),
                                                     dtype=np.uint8)
    once, parts = blank.copy(), blank.copy()
    opaged.append(once, table, 0, page_size, *rows, positions)
    at = 0
    while at < n:
        take = int(min(rng.integers(1, 20), n - at))
        opaged.append(parts, table, at, page_size, *(r[at:at + take] for r in rows), positions[at:at + take])
        at += take
    assert np.array_equal(once, parts)


def test_layout():
    rng = np.random.default_rng(1)
    page_size, dim = 32, 64
    pages = rng.integers(0, 256, (3, opaged.page_bytes(page_size, dim)), dtype=np.uint8)
    rows = random_rows(rng, 40, dim)
    opaged.append(pages, np.array([1, 2]), 0, page_size, *rows, np.arange(40))
    page = pages[1]
    keys = page[:32 * 64].reshape(2, 4, 16, 16).transpose(0, 2, 1, 3).reshape(32, 64)
    vals = page[32 * 64:2 * 32 * 64].reshape(8, 64, 4).transpose(0, 2, 1).reshape(32, 64)
    where = page[2 * 32 * 64:2 * 32 * 64 + 128].view(np.float32)
    scales = page[2 * 32 * 64 + 128:][:4].astype(int) - 127
    for block in range(2):
        part = slice(16 * block, 16 * block + 16)
        for got, x, e in ((keys, rows[0], scales[2 * block]), (vals, rows[1], scales[2 * block + 1])):
            assert e == opaged.scale_exponent(np.abs(x[part]).max())
            assert np.array_equal(got[part], opaged.encode(x[part], e))
    assert where.tolist() == list(range(32))
    got = opaged.load(pages, np.array([1, 2]), 40, page_size, dim)
    for x, y in zip(got, rows):
        assert np.all(np.abs(x - y) <= 2.0 ** -4 * np.abs(y) + 2.0 ** -16 * np.abs(y).max())


def test_non_finite_elements_read_as_nan_and_leave_the_scale():
    rows = np.ones((20, 64))
    rows[3, 5], rows[4, 6], rows[17, 7] = np.nan, np.inf, -np.inf
    pages = np.zeros((1, opaged.page_bytes(32, 64)), np.uint8)
    opaged.append(pages, np.array([0]), 0, 32, rows, rows, np.arange(20))
    keys, vals, _ = opaged.load(pages, np.array([0]), 20, 32, 64)
    bad = ~np.isfinite(rows)
    assert np.array_equal(np.isnan(keys), bad) and np.array_equal(np.isnan(vals), bad)
    assert np.array_equal(keys[~bad], rows[~bad])
    # a larger row moves the block's scale and leaves its NaN
    opaged.append(pages, np.array([0]), 20, 32, rows[:1] * 2.0 ** 12, rows[:1], np.arange(1))
    keys, _, _ = opaged.load(pages, np.array([0]), 21, 32, 64)
    assert np.array_equal(np.isnan(keys[:20]), bad) and keys[20, 0] == 4096 and keys[19, 0] == 1


def test_compact_takes_the_largest_scale():
    rng = np.random.default_rng(4)
    page_size, dim = 16, 64
    pages = np.zeros((6, opaged.page_bytes(page_size, dim)), np.uint8)
    rows = random_rows(rng, 48, dim)
    rows[0][:16] *= 2.0 ** -12
    opaged.append(pages, np.array([0, 1, 2]), 0, page_size, *rows, np.arange(48))
    before = opaged.load(pages, np.array([0, 1, 2]), 48, page_size, dim)
    kept = np.sort(rng.permutation(48)[:29])
    opaged.compact(pages, np.array([0, 1, 2]), kept, np.array([4, 3]), page_size, dim)
    after = opaged.load(pages, np.array([4, 3]), 29, page_size, dim)
    assert after[2].tolist() == kept.tolist()
    for got, was in zip(after[:2], before[:2]):
        for part in (slice(0, 16), slice(16, 29)):
            x, y = got[part], was[kept[part]]
            # a cut is below the smallest code of the largest scale among the blocks that the rows come
            # from, 2^(e - 9), and those blocks' largest element is 232 2^e at least
            source = np.concatenate([was[b:b + 16] for b in set(kept[part] // 16 * 16)])
            assert np.all(np.abs(x) <= np.abs(y))
            assert np.all(np.abs(x - y) < np.abs(source).max() * 2.0 ** -16)
