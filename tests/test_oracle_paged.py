"""The paged cache's oracle against independent statements of the format: the nearest of the
representable values, exactness in the 16-bit types, idempotence, the byte layout."""

import numpy as np
import pytest
import torch
from hypothesis import given, settings
from hypothesis import strategies as st

from oracle import paged as opaged


def test_scale_rule():
    x = np.array([1.0, 4.0, 5.9, 6.0, 6.99, 7.0, 7.01, 8.0, 0.4375, 0.43])
    got = np.exp2(opaged.scale_exponent(x, False))
    assert got.tolist() == [0.25, 1, 1, 1, 1, 2, 2, 2, 0.125, 0.0625]
    assert opaged.scale_exponent(np.array([0.0, 65504.0, 1e30]), True).tolist() == [-23, 13, 13]
    assert opaged.scale_exponent(np.array([0.0, 3.4e38]), False).tolist() == [-125, 125]


def test_ties_go_to_the_even_code():
    row = np.zeros(32)
    row[:10] = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -0.75, -2.5]
    codes, scales = opaged.quantise(row)
    assert scales.tolist() == [127]
    assert opaged.values(codes, scales)[:10].tolist() == [0, 1, 1, 2, 2, 4, 4, 6, -1, -2]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_values_are_exact_in_the_16_bit_type(dtype):
    rng = np.random.default_rng(0)
    rows = torch.from_numpy(rng.standard_normal((64, 128)) * np.exp2(rng.uniform(-22, 14, (64, 1))))
    rows = rows.to(dtype).double().numpy()
    got = opaged.values(*opaged.quantise(rows, dtype == torch.float16))
    assert np.array_equal(torch.from_numpy(got).to(dtype).double().numpy(), got)


@settings(max_examples=60, deadline=None)
@given(st.integers(0, 2 ** 32 - 1), st.floats(-20, 20))
def test_quantising_twice_changes_nothing(seed, power):
    rows = np.random.default_rng(seed).standard_normal((4, 64)) * 2.0 ** power
    once = opaged.values(*opaged.quantise(rows))
    assert np.array_equal(opaged.values(*opaged.quantise(once)), once)
    # no element is further off than half the widest spacing under the block's scale
    amax = np.abs(rows.reshape(4, 2, 32)).max(-1)
    step = np.exp2(opaged.scale_exponent(amax, False))
    assert np.all(np.abs(once - rows).reshape(4, 2, 32) <= step[..., None])


def test_non_finite_blocks_read_as_nan():
    rows = np.ones((3, 64))
    rows[0, 3], rows[1, 40], rows[2, 63] = np.nan, np.inf, -np.inf
    got = opaged.values(*opaged.quantise(rows))
    assert np.isnan(got[0, :32]).all() and np.isfinite(got[0, 32:]).all()
    assert np.isfinite(got[1:, :32]).all() and np.isnan(got[1:, 32:]).all()


@pytest.mark.parametrize("page_size,dim", [(16, 64), (32, 128), (64, 256)])
def test_store_and_load(page_size, dim):
    rng = np.random.default_rng(1)
    pages = rng.integers(0, 256, (4, opaged.page_bytes(page_size, dim)), dtype=np.uint8)
    count = page_size + 5
    rows = rng.standard_normal((2, count, dim))
    table = np.array([2, 0])
    quantised = [opaged.quantise(r) for r in rows]
    index = np.arange(count)
    opaged.store(pages, table[index // page_size], index % page_size, page_size, *quantised[0],
                 *quantised[1], 7.0 + index)
    keys, values, positions = opaged.load(pages, table, count, page_size, dim)
    assert np.array_equal(keys, opaged.values(*quantised[0]))
    assert np.array_equal(values, opaged.values(*quantised[1]))
    assert positions.tolist() == [7.0 + i for i in range(count)]


def test_rotation_keeps_lengths_and_the_unrotated_channels():
    rng = np.random.default_rng(2)
    rows = rng.standard_normal((5, 64)).astype(np.float32)
    angle = rng.uniform(0, 7, (5, 8))
    got = opaged.rotate(rows, np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32))
    assert np.array_equal(got[:, 16:], rows[:, 16:])
    z = (rows[:, :8] + 1j * rows[:, 8:16]) * np.exp(1j * angle)
    np.testing.assert_allclose(got[:, :8] + 1j * got[:, 8:16], z, rtol=1e-5, atol=1e-6)


def test_attention_is_the_softmax_over_the_visible_rows():
    rng = np.random.default_rng(3)
    q = rng.standard_normal((1, 4, 3, 64))
    rows = [(rng.standard_normal((n, 64)), rng.standard_normal((n, 64))) for n in (5, 3)]
    got = opaged.attention(q, rows, [2, 0], [3], 2)
    scores = torch.from_numpy(rows[1][0][:2] @ q[0, 3, 1] / 8)
    expect = torch.softmax(scores, 0).numpy() @ rows[1][1][:2]
    np.testing.assert_allclose(got.reshape(3, 4, 64)[1, 3], expect, rtol=1e-12)
    padded = opaged.attention(q, rows, [2, 0], [1], 2)
    assert not padded[0, 1:].any() and np.array_equal(padded[0, 0], got[0, 0])
