"""The paged 8-bit cache's kernels against the numpy oracle: append (whole pages compared byte by
byte), read and compact (bit-exact), attention (f64 softmax over the rows the codes stand for), and
a run of them together as a decode loop with evictions uses them.

Attention's tolerance. Products of a 16-bit query element and a stored value (or its code, times the
scale afterwards) are exact in f32, as are those of the probabilities' pieces, so the errors are: D f32
additions of a score (each at most 2^-24 of the sum A of the score's absolute terms) and its scaling,
the scaled exponent's rounding and the exponential (a few 2^-24 of A + 1), n additions of the sums, and
the output's rounding, half a step of the value and of its error. All but the last weigh in with E,
the same average of |V|: |got - ref| <= eps / 2 |ref| + (1 + eps) (2 2^-24 E ((D + 9) (A + 1) + n + 64)
+ 2^-126 n max(1, |V|)) + 2^-25 in f16; the terms at the end for exponentials (of which a row's largest
is 1 at least) and products below f32's normal numbers, and for half of f16's subnormal step.
"""

import dataclasses

import numpy as np
import pytest
import torch

from code_for_iclr27_amd import _lib
from code_for_iclr27_amd import attention as packed
from code_for_iclr27_amd import paged
from oracle import paged8 as opaged

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


class Cache:
    """A cache on the host and on the device: pages of random bytes, shuffled tables, stored rows."""

    def __init__(self, device, lengths, kv_heads, dim, page_size, room=None, dtype=BF16, seed=0,
                 fill=True):
        rng = np.random.default_rng(seed)
        self.rng, self.device, self.f16 = rng, device, dtype == F16
        self.kv_heads, self.dim, self.page_size = kv_heads, dim, page_size
        self.lengths = np.asarray(lengths, np.int32)
        room = self.lengths if room is None else np.asarray(room)
        used = -(-room // page_size)
        width = max(int(used.max()), 1)
        order = rng.permutation(int(used.sum()) + 2).astype(np.int32)
        self.table = np.full((len(self.lengths), width), -1, np.int32)
        self.table[np.arange(width) < used[:, None]] = order[:used.sum()]
        self.spare = order[used.sum():]
        self.pages = rng.integers(0, 256, (len(order), opaged.page_bytes(page_size, dim)),
                                  dtype=np.uint8)
        for s, n in enumerate(self.lengths if fill else []):
            rows = [torch.from_numpy(rng.standard_normal((n, dim))
                                     * np.exp2(rng.uniform(-3, 1, (n, 1)))).to(dtype) for _ in range(2)]
            self.store(s, 0, *(r.double().numpy() for r in rows), np.arange(n) + 3.0 * s)
        self.upload()

    def store(self, segment, length, keys, values, positions):
        opaged.append(self.pages, self.table[segment], int(length), self.page_size, keys, values,
                      positions, self.f16)

    def upload(self):
        put = lambda a: torch.from_numpy(a.copy()).to(self.device)  # noqa: E731
        self.layer = paged.PagedLayer(put(self.pages), put(self.table), put(self.lengths),
                                      self.kv_heads, self.dim, self.page_size, bits=8)

    def rows(self, segment, count):
        return opaged.load(self.pages, self.table[segment], int(count), self.page_size, self.dim)

    def check_pages(self):
        got = self.layer.pages.cpu().numpy()
        bad = np.nonzero((got != self.pages).any(1))[0]
        assert bad.size == 0, (bad[:5], [np.nonzero(got[p] != self.pages[p])[0][:8] for p in bad[:3]])


def tables(rows, half, device, seed=0):
    angle = np.random.default_rng(seed).uniform(-9, 9, (rows, half))
    host = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    return host, tuple(torch.from_numpy(t).to(device) for t in host)


def randn(rng, shape, dtype):
    return torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(dtype)


# ---- append -----------------------------------------------------------------------------------

def check_append(device, lengths, kv_heads, groups, added, dim, page_size, dtype, half, counts=None,
                 layout="rows", edit=None, seed=0):
    batch = len(lengths) // kv_heads
    room = np.maximum(np.asarray(lengths), 0) + added
    cache = Cache(device, lengths, kv_heads, dim, page_size, room, dtype, seed)
    rng = cache.rng
    heads = kv_heads * groups
    keys, values = (randn(rng, (batch, kv_heads, added, dim), dtype) for _ in range(2))
    queries = randn(rng, (batch, heads, added, dim), dtype) if groups else None
    if edit is not None:
        edit(keys, values)
    positions = torch.from_numpy(rng.integers(0, 50, (batch, added)))
    (cos, sin), rotary = tables(50, max(half, 8), device, seed)
    where = positions.numpy()[:, None, :]

    def turned(x):
        x = x.float().numpy()
        with np.errstate(all="ignore"):
            return opaged.rotate(x, cos[where], sin[where]) if half else x

    def there(x):  # the layouts a model hands over
        x = x.to(device)
        if layout == "heads":
            return x.transpose(1, 2).contiguous().transpose(1, 2)
        if layout == "padded":
            wide = torch.zeros(x.shape[:3] + (dim + 16,), dtype=dtype, device=device)
            wide[..., :dim] = x
            return wide[..., :dim]
        return x

    got = paged.append(cache.layer, there(keys), there(values), positions.to(device),
                       rotary=rotary if half else None,
                       queries=None if queries is None else there(queries),
                       counts=None if counts is None else
                       torch.tensor(counts, dtype=torch.int32, device=device))
    k, v = turned(keys), values.float().numpy()
    for s in range(len(lengths)):
        b, h = divmod(s, kv_heads)
        n = added if counts is None else min(max(counts[b], 0), added)
        if n:
            cache.store(s, lengths[s], k[b, h, :n], v[b, h, :n], positions[b, :n].numpy())
    torch.cuda.synchronize()
    cache.check_pages()
    assert cache.layer.lengths.cpu().tolist() == list(lengths)
    if groups:
        expect = torch.from_numpy(turned(queries)).to(dtype)
        assert got.shape == queries.shape and got.is_contiguous()
        assert torch.equal(got.cpu().float().nan_to_num(7e7), expect.float().nan_to_num(7e7))
    else:
        assert got is None


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("dim,half,page_size", [(64, 32, 16), (128, 64, 32), (256, 32, 64), (128, 24, 16),
                                                (128, 8, 128), (256, 128, 16), (64, 0, 256), (256, 0, 32)])
@pytest.mark.parametrize("added", [1, 2, 37])
def test_append(device, dtype, dim, half, page_size, added):
    check_append(device, [0, 1, 15, 16, 31, 33, 18, 14, 13], 3, 2, added, dim, page_size, dtype, half,
                 seed=dim + half)


@pytest.mark.parametrize("layout", ["heads", "padded"])
def test_append_layouts(device, layout):
    check_append(device, [5, 0, 9, 40], 2, 3, 6, 128, 16, BF16, 64, layout=layout)
    check_append(device, [5, 0, 9, 40], 2, 0, 6, 64, 16, F32, 16, layout=layout)


def test_append_of_a_padded_batch(device):
    check_append(device, [4, 0, 9, 40, 7, 2, 1, 0], 2, 4, 9, 128, 32, BF16, 64,
                 counts=[9, 0, 4, -3])
    check_append(device, [4, 0], 1, 1, 3, 64, 16, F16, 32, counts=[2, 100])


@pytest.mark.parametrize("dtype,dim,half", [(BF16, 64, 32), (F32, 128, 32), (F16, 128, 64),
                                            (BF16, 256, 0)])
def test_append_of_many_rows_takes_several_heads_a_thread(device, dtype, dim, half):
    """From 32,768 query rows on; six and fourteen heads are no multiple of the four that a thread takes."""
    check_append(device, [100, 3, 0], 3, 2, 5500, dim, 64, dtype, half, counts=[5499], seed=dim)
    check_append(device, [100, 0], 1, 14, 1300, dim, 64, dtype, half, counts=[1300, 17], seed=dim)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("length", [0, 3])
def test_append_edge_values(device, dtype, length):
    top = float(torch.finfo(dtype).max)
    tiny = 2.0 ** -24 if dtype == F16 else 2.0 ** -133 if dtype == BF16 else 2.0 ** -149

    def edit(keys, values):  # blocks of their own, 16 rows each
        for h, row in enumerate([1.0, top, -top, tiny, tiny * 8, 0.0, -0.0, 2.0 ** -14]):
            values[0, h] = row
        values[0, 0, 5, 3], values[0, 0, 6, 40], values[0, 0, 7, 31] = float("nan"), float("inf"), -float("inf")
        values[0, 1, 0, 3], values[0, 1, 1] = float("nan"), 2.0 ** -10
        values[0, 4] *= torch.randint(0, 200, values[0, 4].shape).to(dtype)
        grid = torch.tensor([0.25, 0.75, 1.0625, 1.1875, 1.3125, 448.0, 2.0 ** -9 * 1.5, 2.0 ** -9 * 7.5])
        values[0, 7, :, :16] = torch.cat((grid, -grid)).to(dtype)  # ties, and under the smallest codes
        values[0, 8, :, 0] = 463.0  # under the step to the next scale, and on it
        values[0, 9, :, 0] = 464.0
        values[0, 10] = float("nan")
        values[0, 11] = float("inf")
        keys[0] = values[0]
    check_append(device, [length] * 12, 12, 1, 16 - length, 64, 16, dtype, 0, edit=edit)


@pytest.mark.parametrize("dim,page_size", [(64, 16), (128, 32), (256, 64)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_blocks_bytes_do_not_depend_on_the_calls(device, dim, page_size, dtype):
    """Rows of very different sizes, with NaN among them, at once, in parts and one by one."""
    rng = np.random.default_rng(dim)
    segments, n = 6, 45
    sizes = np.exp2(rng.uniform(-12, 12, (1, segments, n, 1)))
    sizes[0, 0] = np.exp2(np.arange(n) / 2 - 20).reshape(-1, 1)  # ever larger
    rows = [torch.from_numpy(rng.standard_normal((1, segments, n, dim)) * sizes).to(dtype) for _ in range(2)]
    rows[0][0, 1, 7, 5] = rows[1][0, 2, 20, 9] = float("nan")
    cache = Cache(device, [0] * segments, segments, dim, page_size, [n] * segments, dtype)
    for s in range(segments):
        cache.store(s, 0, *(r[0, s].double().numpy() for r in rows), np.arange(n))
    blank = cache.layer.pages.clone()
    there, where = [r.to(device) for r in rows], torch.arange(n, device=device)[None]
    for parts in ([n], [1] * n, [16, 16, 13], [5, 1, 30, 2, 7], [15, 2, 15, 13]):
        cache.layer.pages.copy_(blank)
        at = 0
        for take in parts:
            part = slice(at, at + take)
            layer = cache.layer.with_lengths(cache.layer.lengths + at)
            paged.append(layer, *(t[:, :, part] for t in there), where[:, part].contiguous())
            at += take
        cache.check_pages()


def test_rows_written_again_keep_the_scale(device):
    """A draft of large rows given up and written over: the block stays at the scale they needed."""
    cache = Cache(device, [20], 1, 64, 16, [40])
    keys = randn(cache.rng, (1, 1, 3, 64), BF16) * 500
    small = randn(cache.rng, (1, 1, 2, 64), BF16)
    at = torch.arange(3, device=device)[None]
    for rows in (keys, small):
        n = rows.shape[2]
        paged.append(cache.layer, rows.to(device), rows.to(device), at[:, :n].contiguous())
        cache.store(0, 20, rows[0, 0].double().numpy(), rows[0, 0].double().numpy(), np.arange(n))
        cache.check_pages()


def test_append_outside_the_tables_gives_nan(device):
    cache = Cache(device, [2, 2], 2, 128, 16, [8, 8])
    (_, _), rotary = tables(10, 64, device)
    keys, values = (randn(cache.rng, (1, 2, 3, 128), BF16).to(device) for _ in range(2))
    queries = randn(cache.rng, (1, 2, 3, 128), BF16).to(device)
    positions = torch.tensor([[-1, 4, 10]], device=device)
    got = paged.append(cache.layer, keys, values, positions, rotary=rotary, queries=queries)
    assert got.isnan().all(-1)[0].cpu().tolist() == [[True, False, True]] * 2
    grown = cache.layer.with_lengths(cache.layer.lengths + 3)
    k, v, p, cu = paged.read(grown, 10)
    assert k.isnan().all(-1).cpu().tolist() == [False, False, True, False, True] * 2
    assert k[[0, 1, 3]].isfinite().all() and not v.isnan().any()
    assert p.view(2, 5)[:, 2:].cpu().tolist() == [[-1, 4, 10]] * 2
    assert cu.cpu().tolist() == [0, 5, 10]


def test_append_where_there_is_no_page(device):
    """Rows past the table's end, in pages outside the pool or behind a negative length are not
    stored; the others are."""
    cache = Cache(device, [14, 30, 3, 0], 4, 64, 16, [32, 32, 16, 16])
    cache.table[2, 0] = len(cache.pages)
    cache.table[0, 1] = -5
    before = cache.pages.copy()
    cache.upload()
    cache.layer.lengths[3] = -2
    keys, values = (randn(cache.rng, (1, 4, 4, 64), BF16) for _ in range(2))
    positions = torch.arange(4)[None]
    paged.append(cache.layer, keys.to(device), values.to(device), positions.to(device))
    torch.cuda.synchronize()
    assert np.array_equal(before, cache.pages)
    cache.store(0, 14, keys[0, 0, :2].double().numpy(), values[0, 0, :2].double().numpy(), [0, 1])
    cache.store(1, 30, keys[0, 1, :2].double().numpy(), values[0, 1, :2].double().numpy(), [0, 1])
    cache.check_pages()
    cache.layer.lengths.fill_(2 ** 31 - 1)
    paged.append(cache.layer, keys.to(device), values.to(device), positions.to(device))
    cache.check_pages()


# ---- read -------------------------------------------------------------------------------------

def packed_rows(cache, lengths):
    parts = [cache.rows(s, int(n)) for s, n in enumerate(lengths)]
    return [np.concatenate([p[i] for p in parts]) for i in range(3)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("dim,page_size", [(64, 16), (128, 32), (256, 128)])
def test_read(device, dtype, dim, page_size):
    lengths = [0, 1, 15, 0, 16, 17, 130, 0]
    cache = Cache(device, lengths, 4, dim, page_size, dtype=F16 if dtype == F16 else BF16, seed=dim)
    keys, values, positions = packed_rows(cache, lengths)
    got = paged.read(cache.layer, sum(lengths), dtype)
    assert [t.dtype for t in got] == [dtype, dtype, F32, torch.int32]
    assert np.array_equal(got[0].double().cpu().numpy(), keys)
    assert np.array_equal(got[1].double().cpu().numpy(), values)
    assert np.array_equal(got[2].cpu().numpy().reshape(-1), positions)
    assert got[3].cpu().tolist() == np.concatenate([[0], np.cumsum(lengths)]).tolist()
    cache.check_pages()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_every_code_is_read(device, dtype):
    """All 256 codes at every scale that append writes: exact in bf16 and f32, rounded once in f16."""
    cache = Cache(device, [16 * 237], 1, 256, 256, fill=False)
    lut = np.random.default_rng(0).permuted(np.tile(np.arange(256, dtype=np.uint8), (2, 16 * 237, 1)), axis=2)
    expect = []
    for row in range(0, 16 * 237, 16):
        slot, page = row % 256 + np.arange(16), cache.table[0, row // 256]
        spots = opaged.places(slot, 256, 256)
        cache.pages[page, spots[0]], cache.pages[page, spots[1]] = lut[0, row:row + 16], lut[1, row:row + 16]
        cache.pages[page, spots[3][0]] = 10 + row // 16
        expect.append([opaged.values(x[row:row + 16], row // 16 - 117) for x in lut])
    cache.upload()
    got = paged.read(cache.layer, 16 * 237, dtype)
    for which in range(2):
        rows = torch.from_numpy(np.concatenate([e[which] for e in expect]))
        other = rows.to(F32).to(dtype).double().numpy()  # (exact in f32)
        assert np.array_equal(got[which].double().cpu().numpy(), other, equal_nan=True)
        assert dtype == F16 or np.array_equal(other, rows.numpy(), equal_nan=True)


@pytest.mark.parametrize("dtype,repeats", [(F32, 80), (BF16, 120), (F16, 120)])
def test_read_of_more_than_the_caches_hold(device, dtype, repeats):
    """Rows of more than 256 MB in all, from segments that share pages: the same as one by one."""
    lengths = np.array([1301, 0, 977])
    cache = Cache(device, lengths, 3, 256, 32, dtype=F16 if dtype == F16 else BF16, seed=repeats)
    total = int(lengths.sum())
    assert 2 * repeats * total * 256 * dtype.itemsize > 256 << 20
    keys, values, positions = (torch.from_numpy(x).to(device) for x in packed_rows(cache, lengths))
    layer = dataclasses.replace(cache.layer, table=cache.layer.table.repeat(repeats, 1),
                                lengths=cache.layer.lengths.repeat(repeats))
    got = paged.read(layer, repeats * total, dtype)
    for want, have in ((keys.to(dtype), got[0]), (values.to(dtype), got[1]), (positions.to(F32)[:, None], got[2])):
        assert torch.equal(have.view(repeats, total, -1), want.view(1, total, -1).expand(repeats, -1, -1))
    ends = np.concatenate([[0], np.cumsum(np.tile(lengths, repeats))])
    assert np.array_equal(got[3].cpu().numpy(), ends)


def test_read_many_segments(device):
    """More segments than the summing workgroup has threads, most of them empty."""
    rng = np.random.default_rng(8)
    lengths = np.where(rng.random(2500) < 0.2, rng.integers(1, 20, 2500), 0)
    cache = Cache(device, lengths, 1, 64, 16)
    keys, values, positions = packed_rows(cache, lengths)
    got = paged.read(cache.layer, int(lengths.sum()))
    assert np.array_equal(got[0].double().cpu().numpy(), keys)
    assert np.array_equal(got[1].double().cpu().numpy(), values)
    assert np.array_equal(got[2].cpu().numpy().reshape(-1), positions)
    assert np.array_equal(got[3].cpu().numpy(), np.concatenate([[0], np.cumsum(lengths)]))


def test_read_bounds(device):
    """Fewer or more rows wanted than there are; rows without a page keep what the output held."""
    cache = Cache(device, [20, 7, 5], 3, 64, 16)
    cache.table[0, 1] = len(cache.pages)
    cache.table[2, 0] = -1
    cache.upload()
    keys, _, _ = opaged.load(cache.pages, cache.table[1], 7, 16, 64)
    out = paged.read(cache.layer, 29)
    assert out[0].shape == (29, 64)
    assert np.array_equal(out[0][20:27].double().cpu().numpy(), keys)
    assert paged.read(cache.layer, 0)[0].shape == (0, 64)
    k, v = (torch.full((40, 64), 9.0, dtype=BF16, device=device) for _ in range(2))
    p = torch.full((40,), -1.0, device=device)
    cu = torch.empty(4, dtype=torch.int32, device=device)
    a = cache.layer
    _lib.call("lr_paged8_read", a.pages.data_ptr(), a.pages.shape[0], 16, a.table.data_ptr(),
              a.table.shape[1], a.lengths.data_ptr(), 3, 64, _lib.LR_DTYPE_BF16, 40, k.data_ptr(),
              v.data_ptr(), p.data_ptr(), cu.data_ptr(), _lib.stream_of(k))
    untouched = [(t.view(40, -1) == was).all(1).cpu().tolist()
                 for t, was in ((k, 9.0), (v, 9.0), (p, -1.0))]
    expect = [16 <= i < 20 or i >= 27 for i in range(40)]
    assert untouched == [expect] * 3 and cu.cpu().tolist() == [0, 20, 27, 32]


def test_lengths_past_the_table_are_cut(device):
    cache = Cache(device, [16, 16], 2, 64, 16)
    cache.layer.lengths.copy_(torch.tensor([1000, -4]))
    got = paged.read(cache.layer, 16)
    assert got[3].cpu().tolist() == [0, 16, 16]
    assert np.array_equal(got[0].double().cpu().numpy(), cache.rows(0, 16)[0])


# ---- compact ----------------------------------------------------------------------------------

def check_compact(device, lengths, dim, page_size, share, seed=0, even=False, wide=0):
    rng = np.random.default_rng(seed)
    lengths = np.asarray(lengths)
    cache = Cache(device, lengths, 1, dim, page_size, seed=dim, fill=False)
    for s, n in enumerate(lengths):  # blocks of equal scales, or of very different ones, with NaN
        size = 1.0 if even else np.exp2(rng.uniform(-12, 12, (-(-n // 16), 1))).repeat(16, 0)[:n]
        k, v = rng.uniform(-1, 1, (2, n, dim)) * size
        if n > 5 and not even:
            k[rng.integers(n), 3] = v[rng.integers(n), dim - 1] = np.nan
        cache.store(s, 0, k, v, np.arange(n) + 5.0 * s)
    keep = [np.sort(rng.permutation(n)[:n - int(round(share * n))]) for n in lengths]
    starts = np.concatenate([[0], np.cumsum(lengths)])
    removed = np.concatenate([starts[s] + np.setdiff1d(np.arange(n), keep[s])
                              for s, n in enumerate(lengths)]).astype(np.int64)
    used = np.array([-(-len(k) // page_size) for k in keep])
    width = max(int(used.max()), 1)
    first = len(cache.pages)
    cache.pages = np.concatenate([cache.pages, rng.integers(
        0, 256, (int(used.sum()) + 1, cache.pages.shape[1]), dtype=np.uint8)])
    target = np.full((len(lengths), width), -1, np.int32)
    target[np.arange(width) < used[:, None]] = first + rng.permutation(int(used.sum()))
    if wide:
        cache.table, target = (np.pad(t, ((0, 0), (0, wide - t.shape[1])), constant_values=-1)
                               for t in (cache.table, target))
    cache.upload()
    got = paged.compact(cache.layer, torch.from_numpy(removed).to(device),
                        torch.from_numpy(target).to(device))
    torch.cuda.synchronize()
    assert got.bits == 8 and got.lengths.cpu().tolist() == [len(k) for k in keep]
    assert cache.layer.lengths.cpu().tolist() == lengths.tolist()
    for s, kept in enumerate(keep):
        opaged.compact(cache.pages, cache.table[s], kept, target[s], page_size, dim)
    cache.check_pages()


@pytest.mark.parametrize("dim,page_size", [(64, 16), (128, 32), (256, 64), (128, 256)])
@pytest.mark.parametrize("share", [0.0, 0.1, 0.6, 1.0])
@pytest.mark.parametrize("even", [True, False])
def test_compact(device, dim, page_size, share, even):
    check_compact(device, [0, 1, 16, 33, 64, 65, 200, 150], dim, page_size, share, even=even)


def test_compact_long_and_many_segments(device):
    """Searches of several rounds; more segments than a workgroup sums for itself."""
    check_compact(device, [3000, 0, 5, 2600], 64, 128, 0.4, seed=1)
    check_compact(device, [3000, 0, 5, 2600], 128, 16, 0.02, seed=2)
    lengths = np.random.default_rng(3).integers(0, 12, 700)
    check_compact(device, lengths, 64, 16, 0.5, seed=4)
    check_compact(device, lengths[:256], 64, 16, 0.3, seed=5)
    check_compact(device, lengths[:257], 64, 16, 0.3, seed=6)


@pytest.mark.parametrize("dim,page_size,segments", [(64, 16, 8), (128, 32, 8), (256, 64, 8), (128, 16, 300)])
def test_compact_of_large_tables(device, dim, page_size, segments):
    """Room for a fifth of 256 MB and more (rows are written past the caches), a few rows there."""
    lengths = np.random.default_rng(dim).integers(0, 90, segments)
    lengths[:4] = 0, 1, 200, 33
    wide = -(-(256 << 20) // (5 * segments * paged.page_bytes(page_size, dim, 8)))
    for wide in (wide, wide - 1):
        check_compact(device, lengths, dim, page_size, 0.2, even=False, seed=7, wide=wide)


def test_compact_into_a_short_table_and_missing_pages(device):
    cache = Cache(device, [40, 40, 40], 3, 64, 16)
    extra = len(cache.pages)
    cache.pages = np.concatenate([cache.pages, np.full((4, cache.pages.shape[1]), 77, np.uint8)])
    source = cache.table[2, 1]
    cache.table[2, 1] = -3  # rows 16 .. 31 of the last segment are not there
    cache.upload()
    before = cache.pages.copy()
    target = torch.tensor([[extra, -1], [extra + 99, -1], [extra + 1, extra + 2]], dtype=torch.int32,
                          device=device)
    removed = torch.tensor([0, 41, 80, 81], device=device)
    got = paged.compact(cache.layer, removed, target)
    assert got.lengths.cpu().tolist() == [39, 39, 38]
    after = got.pages.cpu().numpy()
    opaged.compact(before, cache.table[0], np.arange(1, 17), np.array([extra]), 16, 64)
    # the last segment's rows: 2 .. 15 to slots 0 .. 13, 32 .. 39 to slots 30 .. 37 of the table's 32
    untouched = before.copy()
    cache.table[2, 1] = source
    opaged.compact(before, cache.table[2], np.arange(2, 16), np.array([extra + 1]), 16, 64)
    part = opaged.codes(untouched, cache.table[2], np.arange(32, 34), 16, 64)
    spots = opaged.places(np.arange(14, 16), 16, 64)
    for where, rows in ((spots[0], part[0]), (spots[1], part[1])):
        before[extra + 2, where] = rows
    before[extra + 2, spots[2]] = np.array([[32 + 6], [33 + 6]], np.float32).view(np.uint8)
    before[extra + 2, spots[3][0]] = (part[2][0] + 127).astype(np.uint8)
    assert np.array_equal(after, before)


# ---- attention --------------------------------------------------------------------------------

def reference(queries, rows, lengths, counts, kv_heads, scale):
    """The oracle's output, the tolerance's E, its max|V| of a channel and, per row, its A."""
    q = queries.double().numpy()
    with np.errstate(all="ignore"):
        out = opaged.attention(q, rows, lengths, counts, kv_heads, scale)
        average = opaged.attention(q, [(k, np.abs(v)) for k, v in rows], lengths, counts, kv_heads,
                                   scale)
    batch, heads, length, dim = q.shape
    a, top = np.zeros((batch, length, heads)), np.ones((batch, 1, heads, dim))
    for s, (keys, values) in enumerate(rows):
        b, h = divmod(s, kv_heads)
        groups = heads // kv_heads
        mine = np.abs(np.nan_to_num(q[b, h * groups:(h + 1) * groups]))  # [G, L, D]
        terms = mine @ np.abs(np.nan_to_num(keys)).T * scale
        if terms.shape[-1]:
            a[b, :, h * groups:(h + 1) * groups] = terms.max(-1).T
            top[b, 0, h * groups:(h + 1) * groups] = np.abs(np.nan_to_num(values)).max(0).clip(min=1.0)
    shape = (batch, length, heads, dim)
    return out.reshape(shape), average.reshape(shape), top, a


def check_attention(got, queries, rows, lengths, counts, kv_heads, scale=None):
    """Rows that see a NaN are NaN where the oracle's are; the others within the tolerance."""
    batch, heads, length, dim = queries.shape
    scale = dim ** -0.5 if scale is None else scale
    expect, average, top, a = reference(queries, rows, lengths, counts, kv_heads, scale)
    assert got.shape == (batch, length, heads * dim) and got.dtype == queries.dtype
    got = got.double().cpu().numpy().reshape(expect.shape)
    most = max((len(k) for k, _ in rows), default=0)
    eps = torch.finfo(queries.dtype).eps
    bound = eps / 2 * np.abs(expect) + (1 + eps) * (2.0 ** -126 * most * top + average * (
        2 * 2.0 ** -24 * ((dim + 9) * (a[..., None] + 1) + most + 64)))
    bound += 2.0 ** -25 * (queries.dtype == F16)
    fine = ~np.isnan(expect)
    assert np.array_equal(np.isnan(got), ~fine)
    error = np.abs(got - expect)
    assert np.all(error[fine] <= bound[fine]), float((error - bound)[fine].max())
    return expect


def attend(device, lengths, kv_heads, groups, length, dim, page_size, dtype=BF16, counts=None,
           seed=0, amplitude=1.0, scale=None, slack=0, layout="rows", stored=None):
    batch = len(lengths) // kv_heads
    n = np.full(batch, length) if counts is None else np.clip(np.asarray(counts), 0, length)
    grown = np.asarray(lengths) + np.repeat(n, kv_heads)
    cache = Cache(device, grown, kv_heads, dim, page_size, dtype=stored or dtype, seed=seed)
    cache.lengths = np.asarray(lengths, np.int32)
    cache.upload()
    queries = randn(cache.rng, (batch, kv_heads * groups, length, dim), dtype) * amplitude
    there = queries.to(device)
    if layout == "heads":
        there = there.transpose(1, 2).contiguous().transpose(1, 2)
    got = paged.attention(cache.layer, there, int(grown.max()) + slack, scale=scale,
                          counts=None if counts is None else
                          torch.tensor(counts, dtype=torch.int32, device=device))
    rows = [cache.rows(s, int(g))[:2] for s, g in enumerate(grown)]
    torch.cuda.synchronize()
    check_attention(got, queries, rows, lengths, n, kv_heads, scale)
    return got, cache, queries


def plan(segments, groups, length, max_keys, dim=128):
    out = np.zeros(3, np.int64)
    _lib.call("lr_paged8_attention_plan", segments, groups, length, max_keys, dim, out.ctypes.data)
    return out.tolist()


EDGES = [0, 1, 2, 14, 15, 16, 30, 31, 32, 33, 62, 63, 126, 127, 128, 129, 254, 256, 511, 700]

# (segments, groups, queries, longest): calls that take every kernel, its keys split and not
SHAPES = [(8, 4, 1, 90), (8, 4, 1, 2250), (140, 3, 1, 1000), (36, 7, 5, 3000), (144, 3, 43, 243),
          (36, 4, 29, 2500)]


def ragged(segments, length, most):
    """Lengths of segments: most short, a few up to `most` with the call's own rows."""
    lengths = np.random.default_rng(segments).integers(5, 40, segments)
    lengths[[0, 3, 4, 5, -1]] = most - length
    lengths[6] = (most - length) // 2
    return lengths


def test_the_shapes_take_every_form():
    for dim in (64, 128, 256):
        forms = {(rows, splits > 1) for rows, _, splits in (plan(*s, dim) for s in SHAPES)}
        assert {rows for rows, _ in forms} == {16, 32} and {split for _, split in forms} == {True, False}
        assert len(forms) == 4, forms


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim,page_size", [(64, 16), (128, 32), (256, 16), (128, 16), (64, 256)])
@pytest.mark.parametrize("groups", [1, 4, 6])
def test_decode(device, dtype, dim, page_size, groups):
    attend(device, EDGES, 2, groups, 1, dim, page_size, dtype, seed=dim + groups)


@pytest.mark.parametrize("groups,dim", [(16, 128), (17, 64), (32, 128), (33, 256), (64, 64)])
def test_decode_of_many_query_heads(device, groups, dim):
    attend(device, [0, 31, 200, 333], 2, groups, 1, dim, 32, seed=groups)


@pytest.mark.parametrize("batch,lengths", [(1, [2250] * 4), (2, [1499, 33, 2250, 1, 900, 64, 0, 7])])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_decode_split_keys(device, batch, lengths, dim):
    attend(device, lengths, 4, 4, 1, dim, 32, seed=batch)
    attend(device, lengths, 4, 4, 1, dim, 64, seed=batch, slack=5000)


@pytest.mark.parametrize("dim,length,groups", [(64, 1, 3), (128, 2, 1), (256, 1, 16)])
def test_decode_of_many_parts(device, dim, length, groups):
    """More parts than the merge loads in one round; of the second segment's, most see no key."""
    assert plan(2, groups, length, 24000, dim)[2] > 32
    attend(device, [24000 - length, 9000], 2, groups, length, dim, 64, seed=dim)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("length,groups,dim", [(2, 1, 64), (3, 4, 128), (8, 6, 256), (8, 4, 128),
                                               (17, 2, 64), (5, 3, 256), (16, 4, 64), (33, 4, 128),
                                               (70, 2, 128), (40, 6, 256)])
def test_several_queries(device, dtype, length, groups, dim):
    attend(device, [0, 1, 31, 32, 100, 257, 400, 15], 2, groups, length, dim, 16, dtype, seed=length)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("shape", SHAPES)
def test_every_form(device, dtype, dim, shape):
    segments, groups, length, most = shape
    attend(device, ragged(segments, length, most), 4, groups, length, dim, 32 if dim == 64 else 16, dtype,
           seed=length, layout="heads")


@pytest.mark.parametrize("dim,groups", [(64, 4), (128, 4), (256, 6)])
def test_prefill(device, dim, groups):
    attend(device, [0, 60], 2, groups, 250, dim, 32, seed=dim, layout="heads")


def test_padded_batch(device):
    for length in (1, 5, 40, 500):
        assert plan(8, 4, length, 800)[0] == (32 if length == 500 else 16) or length == 40
        attend(device, [0, 5, 100, 33, 64, 0, 7, 300], 2, 4, length, 128, 16,
               counts=[length, 0, length // 2 + 1, -1], seed=length)


def test_scales(device):
    for scale in (1e-3, 1.0, 3.0):
        attend(device, [50, 200], 2, 4, 3, 128, 32, scale=scale)


def test_f16_queries_onto_rows_of_another_type(device):
    """Rows appended as bf16 and f32, also past f16's range."""
    for length in (1, 40):
        cache = Cache(device, [90 + length] * 6, 6, 64, 16, dtype=F32, fill=False)
        held = []
        for s in range(6):
            size = 2.0 ** [-100, -30, 0, 15, 30, 60][s]
            k, v = cache.rng.standard_normal((2, 90 + length, 64))
            cache.store(s, 0, k * size, v, np.arange(90 + length))
            held.append(cache.rows(s, 90 + length)[:2])
        cache.lengths[:] = 90
        cache.upload()
        queries = randn(cache.rng, (1, 24, length, 64), F16)
        for s, power in enumerate([14, 14, 0, -8, -14, -14]):
            queries[:, 4 * s:4 * s + 4] *= 2.0 ** power
        for scale in (0.125, 2.0 ** -20):
            got = paged.attention(cache.layer, queries.to(device), 90 + length, scale=scale)
            check_attention(got, queries, held, [90] * 6, [length], 6, scale)


def test_large_scores_leave_one_key(device):
    attend(device, [300, 40], 2, 4, 1, 128, 32, amplitude=300.0)
    attend(device, [300, 40], 2, 4, 9, 64, 32, amplitude=300.0)


def test_scores_that_rise_key_by_key(device):
    """The running reference has to move at every step."""
    cache = Cache(device, [500], 1, 64, 32)
    keys = np.tile(np.linspace(0, 6, 500)[:, None], (1, 64))
    cache.store(0, 0, keys, cache.rng.standard_normal((500, 64)), np.arange(500))
    cache.lengths[:] = 499
    cache.upload()
    queries = torch.ones(1, 2, 1, 64, dtype=BF16)
    got = paged.attention(cache.layer, queries.to(device), 500)
    check_attention(got, queries, [cache.rows(0, 500)[:2]], [499], [1], 1)


def filled(device, shape, dim, dtype, make, page_size=16, kv_heads=2):
    """A cache of one of SHAPES with rows make(rng, segment, n) -> keys, values, and its rows."""
    segments, _, length, most = shape
    lengths = ragged(segments, length, most)
    cache = Cache(device, lengths + length, kv_heads, dim, page_size, dtype=dtype, fill=False, seed=dim)
    for s, n in enumerate(lengths + length):
        cache.store(s, 0, *make(cache.rng, s, int(n)), np.arange(n))
    cache.lengths = lengths.astype(np.int32)
    cache.upload()
    return cache, [cache.rows(s, int(n) + length)[:2] for s, n in enumerate(lengths)]


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("shape", SHAPES)
def test_values_of_every_size(device, dim, shape):
    """Values of a size of their own in each segment, and of all sizes in one."""
    sizes = [1.0, 2e-4, 3e-6, 1e-9, 1e-30, 4e4, 1e30, 0.0, None]

    def make(rng, s, n):
        keys, values = rng.standard_normal((2, n, dim))
        size = sizes[s % 9]
        if size is None:
            size = rng.choice(sizes[:7], (-(-n // 16), 1), p=[.94, .01, .01, .01, .01, .01, .01])
            size = size.repeat(16, 0)[:n]
        return keys, values * size
    segments, groups, length, most = shape
    cache, rows = filled(device, shape, dim, BF16, make)
    queries = randn(cache.rng, (segments // 2, 2 * groups, length, dim), BF16)
    got = paged.attention(cache.layer, queries.to(device), most)
    check_attention(got, queries, rows, cache.lengths, [length] * (segments // 2), 2)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("shape", SHAPES)
def test_a_dominant_key_of_no_value(device, dtype, shape):
    """All of the output is small probabilities on large values, on one side of zero and on both."""
    segments, groups, length, most = shape

    def make(rng, s, n):
        keys, values = np.zeros((n, 128)), 8e3 * rng.random((n, 128)) + 1e3
        keys[n // 3], values[n // 3] = 1.5, 0.0
        values[:, 64:] *= rng.choice([-1, 1], (n, 64))
        return keys, values
    cache, rows = filled(device, shape, 128, dtype, make)
    queries = torch.ones(segments // 2, 2 * groups, length, 128, dtype=dtype)
    for margin in (6, 18, 30, 55):
        scale = margin / 192
        got = paged.attention(cache.layer, queries.to(device), most, scale=scale)
        check_attention(got, queries, rows, cache.lengths, [length] * (segments // 2), 2, scale)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("shape", SHAPES)
def test_probabilities_keep_all_of_their_bits(device, dtype, dim, shape):
    """Two keys of nearly the same score whose values cancel: the output, 2^-12 of the average of
    |V|, is what their probabilities differ by. Scores are exact (two channels), and of the others
    P is below 2^-69 and V 0, so errors are counted without the scores' additions, in units of 2^-24 of
    the average: 7 for the exponents (their products, references and differences, 10 2^-24 in all, times
    ln 2), 6 for three exponentials, 12 for the additions and the weights that join three keys, 3 for
    the division. (Probabilities of 16 to 18 bits miss it by 2 to 3 times.)"""
    segments, groups, length, most = shape

    def make(rng, s, n):
        keys, values = np.zeros((n, dim)), np.zeros((n, dim))
        keys[:, 0] = -192.0
        places = rng.permutation(n - length)[:3]
        keys[places, 0] = 6.0, 4.0, 4.0
        keys[places[2], 32] = 2.0 ** -9  # (a scale of 2^-1 or less: no part of it is cut)
        values[places[1]], values[places[2]] = 96.0, -96.0
        return keys, values
    cache, held = filled(device, shape, dim, dtype, make)
    queries = torch.zeros(segments // 2, 2 * groups, length, dim, dtype=dtype)
    rows = torch.arange(queries[..., 0].numel()).view(queries.shape[:3])
    queries[..., 0], queries[..., 32] = 1 + rows % 97 / 128.0, 0.75
    got = paged.attention(cache.layer, queries.to(device), most, scale=0.25)
    counts = [length] * (segments // 2)
    expect, average = (opaged.attention(queries.double().numpy(), [(k, f(v)) for k, v in held],
                                        cache.lengths, counts, 2, 0.25) for f in (np.asarray, np.abs))
    eps = torch.finfo(dtype).eps
    bound = eps / 2 * np.abs(expect) + (1 + eps) * 28 * 2.0 ** -24 * average
    error = np.abs(got.double().cpu().numpy() - expect)
    assert np.all(error <= bound), float((error / bound).max())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("shape", SHAPES)
def test_scores_of_every_finite_size(device, dtype, dim, shape):
    """Scores of 2^27 to 2^59, whose rounded products with the scale are off by up to 2^35: the keys
    of a row's largest score share the output, the others lie far below. Scores are exact (equal
    channels of a few bits each), so the largest one's probability is one, the output the mean of
    their values: off by its rounding and, in units of 2^-24 of the average of |V|, one for each of up to
    `most` additions to the sum and the products' sum and 64 for the rest."""
    segments, groups, length, most = shape
    codes = np.array([0, .5, 1, 1.5, 2, 3, 4, 6, -.5, -1, -1.5, -2, -3, -4, -6]) * 2.0 ** 13

    def make(rng, s, n):
        keys = np.repeat(rng.choice(codes, (n, 1)), dim, 1)
        if s % 4 == 3:  # all scores of one sign, growing to the end
            keys = np.sort(np.abs(keys), 0)
        return keys, rng.standard_normal((n, dim))
    cache, held = filled(device, shape, dim, dtype, make)
    sizes = 2.0 ** 12 * torch.tensor([1.0, -1.125, 8.0, -8.0, 1.875, -15.0, 13.0])
    queries = torch.ones(segments // 2, 2 * groups, length, dim, dtype=dtype)
    rows = torch.arange(queries[..., 0].numel()).view(queries.shape[:3])
    queries *= sizes[rows % 7].unsqueeze(-1).to(dtype)
    expect, average = np.zeros((2, segments // 2, length, 2 * groups, dim))
    for s, (keys, values) in enumerate(held):
        b, h = divmod(s, 2)
        for i in range(length):
            n = int(cache.lengths[s]) + i + 1
            for sign in (1, -1):
                scores = sign * keys[:n, 0]
                top = scores == scores.max()
                heads = [g for g in range(h * groups, (h + 1) * groups)
                         if float(queries[b, g, i, 0]) * sign > 0]
                expect[b, i, heads] = values[:n][top].mean(0)
                average[b, i, heads] = np.abs(values[:n][top]).mean(0)
    eps = torch.finfo(dtype).eps
    bound = eps / 2 * np.abs(expect) + (1 + eps) * average * 2.0 ** -24 * (2 * most + 64)
    for scale in (2.0 ** -3, 1.0, 2.0 ** 20):
        got = paged.attention(cache.layer, queries.to(device), most, scale=scale)
        error = np.abs(got.double().cpu().numpy().reshape(expect.shape) - expect)
        assert np.all(error <= bound), (scale, np.argwhere(~(error <= bound))[:3].tolist())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("shape", SHAPES)
def test_large_scores_keep_their_differences(device, dtype, dim, shape):
    """Exact scores of 2^27 on either side of zero, that differ by one to eight of f32's steps there: with
    scale 1/8 by factors of e^2 of the probabilities, by e^16 and e^128 with larger ones. An exponent is
    exact but for the scale's rounding and its own (of at most 24: 3 2^-24 24 ln 2), so that in units
    of 2^-24 of the average of |V| the sums' additions count, 2 `most`, and 128 for the rest. Where that
    average is next to nothing: half of f16's smallest step, and what lies below f32's normal numbers (of
    exponentials whose largest is 2^-8 at least, as the reference's rounding is 8 at most at 2^28)."""
    segments, groups, length, most = shape

    def make(rng, s, n):
        keys = np.zeros((n, dim))
        keys[:, 0], keys[:, 32] = 2.0 ** 15, rng.choice([0, .5, 1, 1.5, 2, 3, -.5, -1], n)
        return keys, rng.standard_normal((n, dim))
    cache, held = filled(device, shape, dim, dtype, make)
    queries = torch.zeros(segments // 2, 2 * groups, length, dim, dtype=dtype)
    rows = torch.arange(queries[..., 0].numel()).view(queries.shape[:3])
    queries[..., 0], queries[..., 32] = 4096.0 * (1 - 2 * (rows % 2)), 32.0
    eps = torch.finfo(dtype).eps
    for scale in (0.125, 1.0, 8.0):
        got = paged.attention(cache.layer, queries.to(device), most, scale=scale)
        expect, average = (opaged.attention(
            queries.double().numpy(), [(k, f(v)) for k, v in held], cache.lengths,
            [length] * (segments // 2), 2, scale) for f in (np.asarray, np.abs))
        bound = eps / 2 * np.abs(expect) + (1 + eps) * average * 2.0 ** -24 * (2 * most + 128)
        bound += 2.0 ** -25 * (dtype == F16) + 2.0 ** -118 * most * 8
        error = np.abs(got.double().cpu().numpy() - expect)
        assert np.all(error <= bound), (scale, float((error / bound).max()))


def test_max_length_bounds_the_keys(device):
    cache = Cache(device, [200, 90], 2, 128, 32)
    queries = randn(cache.rng, (1, 4, 1, 128), BF16)
    rows = [cache.rows(s, n)[:2] for s, n in enumerate((100, 90))]
    cache.lengths = np.array([199, 89], np.int32)
    cache.upload()
    got = paged.attention(cache.layer, queries.to(device), 100)
    check_attention(got, queries, rows, [199, 89], [1], 2)
    assert not paged.attention(cache.layer, queries.to(device), 0).any()


@pytest.mark.parametrize("length,groups", [(1, 2), (60, 6)])
def test_keys_in_missing_pages_do_not_count(device, length, groups):
    cache = Cache(device, [70 + length] * 2, 2, 64, 16)
    cache.lengths[:] = 70
    n = 70 + length
    keep = np.ones(n, bool)
    cache.table[0, 1], cache.table[0, n // 16] = -1, len(cache.pages)
    keep[16:32] = keep[n // 16 * 16:n // 16 * 16 + 16] = False
    cache.table[1] = -7
    cache.upload()
    queries = randn(cache.rng, (1, 2 * groups, length, 64), BF16)
    got = paged.attention(cache.layer, queries.to(device), n)
    table = np.where(cache.table < 0, 0, np.minimum(cache.table, len(cache.pages) - 1))
    keys, values, _ = opaged.load(cache.pages, table[0], n, 16, 64)
    got = got.view(length, 2 * groups, 64)
    for i in range(length):
        seen = np.arange(n) <= 70 + i
        rows = [(keys[keep & seen], values[keep & seen]), (np.zeros((0, 64)), np.zeros((0, 64)))]
        check_attention(got[i].reshape(1, 1, -1), queries[:, :, i:i + 1], rows, [n, n], [1], 2)
    assert not got[:, groups:].any()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("shape", SHAPES)
def test_nan_elements_reach_only_the_rows_that_see_them(device, dtype, dim, shape):
    """NaN elements of V and K in the first rows, in the middle of the cache (a part of its own where
    the keys are split), at the diagonal and at the last key: a row that sees a NaN key is NaN, one
    that sees a NaN element of V is NaN in its channel, and all others are within the tolerance."""
    segments, groups, length, most = shape
    lengths = ragged(segments, length, most)
    grown = lengths + length
    cache = Cache(device, grown, 2, dim, 16, dtype=dtype, seed=dim)
    cache.lengths = lengths.astype(np.int32)
    marks = [(0, 1, most // 2, 0), (1, 1, int(grown[1]) - 1, dim - 1), (2, 0, 1, 0),
             (3, 1, most - 1 - length // 2, 1), (3, 1, 0, dim // 2), (4, 0, most - 1, 1),
             (5, 0, most - 1 - length // 2, 0), (5, 1, most // 3, 3), (7, 1, int(grown[7]) - 1, 17),
             (7, 1, int(grown[7]) - 1, 16), (7, 1, 2, 40)]
    for s, which, row, channel in marks:
        at = opaged.places(np.array([row % 16]), 16, dim)[which][0, channel]
        cache.pages[cache.table[s, row // 16], at] |= 127
    cache.upload()
    queries = randn(cache.rng, (segments // 2, 2 * groups, length, dim), dtype)
    got = paged.attention(cache.layer, queries.to(device), most)
    held = [cache.rows(s, int(n))[:2] for s, n in enumerate(grown)]
    with np.errstate(invalid="ignore"):
        expect = check_attention(got, queries, held, lengths, [length] * (segments // 2), 2)
    assert np.isnan(expect).any() and not np.isnan(expect).all()


@pytest.mark.parametrize("length,groups", [(1, 4), (5, 3), (300, 4)])
def test_a_non_finite_query_reaches_its_own_row_only(device, length, groups):
    cache = Cache(device, [90 + length] * 6, 6, 64, 16)
    cache.lengths[:] = 90
    cache.upload()
    queries = randn(cache.rng, (1, 6 * groups, length, 64), BF16)
    spoiled = queries.clone()
    spoiled[0, 1, 0, 3], spoiled[0, groups, length - 1, 60] = float("nan"), float("inf")
    clean = paged.attention(cache.layer, queries.to(device), 90 + length).view(length, -1, 64)
    got = paged.attention(cache.layer, spoiled.to(device), 90 + length).view(length, -1, 64)
    bad = torch.zeros(length, 6 * groups, dtype=torch.bool)
    bad[0, 1] = bad[length - 1, groups] = True
    assert got.isnan().any(-1).cpu().equal(bad) and got.isnan().all(-1).cpu().equal(bad)
    keep = ~bad.to(device)
    assert ((got - clean)[keep].abs() <= 2.0 ** -7 * clean[keep].abs() + 1e-5).all()


@pytest.mark.parametrize("length,groups,most", [(1, 4, 90), (5, 3, 2250), (128, 24, 300)])
def test_a_segment_of_negative_length_has_no_rows_to_attend_to(device, length, groups, most):
    cache = Cache(device, [60, 200, 70, 90], 2, 64, 16)
    cache.lengths = np.array([40, -1, -(2 ** 31), 60], np.int32)
    cache.upload()
    queries = randn(cache.rng, (2, 2 * groups, length, 64), BF16)
    got = paged.attention(cache.layer, queries.to(device), most)
    got = got.view(2, length, 2, groups * 64)
    assert not got[0, :, 1].any() and not got[1, :, 0].any()
    assert got[0, :, 0].any(-1).all() and got[1, :, 1].any(-1).all()
    assert paged.read(cache.layer, 100)[3].cpu().tolist() == [0, 40, 40, 40, 100]


def test_shared_pages_and_wide_tables(device):
    """Requests that share a prefix's pages read the same rows; tables far wider than their segments
    change nothing."""
    cache = Cache(device, [70, 100], 1, 128, 32)
    cache.table[0, :2] = cache.table[1, :2]  # the first 64 rows are one prefix
    cache.lengths = np.array([69, 99], np.int32)
    cache.upload()
    queries = randn(cache.rng, (2, 4, 1, 128), BF16)
    rows = [cache.rows(s, n)[:2] for s, n in enumerate((70, 100))]
    wide = torch.full((2, 5000), 10 ** 9, dtype=torch.int32, device=device)
    wide[:, :cache.table.shape[1]] = cache.layer.table
    for layer, bound in ((cache.layer, 100), (dataclasses.replace(cache.layer, table=wide), 100),
                         (dataclasses.replace(cache.layer, table=wide), 5000 * 32)):
        check_attention(paged.attention(layer, queries.to(device), bound), queries, rows, [69, 99],
                        [1, 1], 1)


def test_attention_equals_packed_attention_over_the_rows_read(device):
    """The same rows give the same output but for the order of sums and half a step of either output."""
    from types import SimpleNamespace
    for length, dim in ((1, 128), (4, 64), (90, 128)):
        got, cache, queries = attend(device, [300, 411, 90, 1000], 2, 4, length, dim, 32)
        grown = cache.layer.lengths + length
        keys, values, _, cu = paged.read(cache.layer.with_lengths(grown), int(grown.sum()))
        meta = SimpleNamespace(cu_seqlens_k=cu, max_seqlen_k=int(grown.max()),
                               decoding_cu_seqlens_q=torch.arange(5, device=device))
        other = packed.packed_attention(queries.to(device), keys, values, meta, length, 2)
        a, b = got.float(), other.float()
        assert ((a - b).abs() <= 2.0 ** -7 * b.abs() + 1e-5).all()


# ---- calls -----------------------------------------------------------------------------------

def test_empty_pool_and_empty_table(device):
    pages = torch.empty(0, paged.page_bytes(32, 128, 8), dtype=torch.uint8, device=device)
    lengths = torch.tensor([5, 0], dtype=torch.int32, device=device)
    for width in (0, 1):
        table = torch.zeros(2, width, dtype=torch.int32, device=device)
        layer = paged.PagedLayer(pages, table, lengths, 2, 128, bits=8)
        queries = torch.ones(1, 2, 1, 128, dtype=BF16, device=device)
        assert not paged.attention(layer, queries, 100).any()
        paged.append(layer, queries, queries, torch.zeros(1, 1, dtype=torch.int64, device=device))
        rows = paged.read(layer, 0)
        assert rows[0].shape == (0, 128)
        assert rows[3].cpu().tolist() == [0, 5 if width else 0, 5 if width else 0]
        out = paged.compact(layer, torch.zeros(0, dtype=torch.int64, device=device), table)
        assert out.lengths.cpu().tolist() == [5 if width else 0, 0]


def test_calls_without_rows(device):
    layer = Cache(device, [3, 4], 2, 64, 16).layer
    none = torch.empty(1, 4, 0, 64, dtype=BF16, device=device)
    assert paged.attention(layer, none, 4).shape == (1, 0, 256)
    got = paged.append(layer, none[:, :2], none[:, :2],
                       torch.empty(1, 0, dtype=torch.int64, device=device), queries=none)
    assert got.shape == none.shape


def test_refusals(device):
    cache = Cache(device, [3, 4], 2, 128, 16)
    layer = cache.layer
    rows = torch.zeros(1, 2, 1, 128, dtype=BF16, device=device)
    at = torch.zeros(1, 1, dtype=torch.int64, device=device)
    change = lambda **o: dataclasses.replace(layer, **o)  # noqa: E731
    table = lambda half: (torch.zeros(4, half, device=device),) * 2  # noqa: E731
    refused = [
        (lambda: paged.append(change(bits=4), rows, rows, at), "Pages must be uint8"),
        (lambda: paged.attention(change(bits=6), rows, 5), "4 or 8 bits"),
        (lambda: paged.read(change(page_size=32), 5), "Pages must be uint8"),
        (lambda: paged.append(change(dim=96), rows, rows, at), "Head dimension must be"),
        (lambda: paged.append(change(lengths=layer.lengths.cpu()), rows, rows, at), "contiguous CUDA"),
        (lambda: paged.append(layer, rows[:, :1], rows[:, :1], at), "New keys and values"),
        (lambda: paged.append(layer, rows.double(), rows.double(), at), "bf16, f16 or f32"),
        (lambda: paged.append(layer, rows, rows, at, rotary=table(12)), "multiple of 16"),
        (lambda: paged.append(layer, rows, rows, at, rotary=table(72)), "at most the head dimension"),
        (lambda: paged.append(layer, torch.zeros(2 * 128 + 1, dtype=BF16, device=device)[1:]
                              .view(1, 2, 1, 128), rows, at), "16-byte aligned"),
        (lambda: paged.attention(layer, rows.float(), 5), "fp16 and bf16"),
        (lambda: paged.attention(layer, rows[:, [0, 0, 1]], 5), "must divide"),
        (lambda: paged.attention(layer, rows, -1), "Invalid max_seqlen_k"),
        (lambda: paged.attention(layer, rows, 5, scale=0.0), "scale must be positive"),
        (lambda: paged.read(layer, 5, torch.float64), "bf16, f16 or f32"),
        (lambda: paged.compact(layer, at.int()[0], layer.table), "Removed indices must be int64"),
        (lambda: paged.compact(layer, at[0], layer.table), "other pages"),
    ]
    for call, message in refused:
        with pytest.raises(RuntimeError, match=message):
            call()
    torch.cuda.synchronize()
    cache.check_pages()


def test_another_stream(device):
    """The launches go on torch's current stream: work there is ordered, other streams wait."""
    side = torch.cuda.Stream(device)
    cache = Cache(device, [100, 50], 2, 128, 32, [200, 200])
    keys, values = (randn(cache.rng, (1, 2, 3, 128), BF16) for _ in range(2))
    queries = randn(cache.rng, (1, 8, 3, 128), BF16)
    on = [t.to(device) for t in (keys, values, queries)]
    positions = torch.arange(3, device=device)[None]
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        filler = torch.randn(2048, 2048, device=device)
        for _ in range(5):
            filler = filler @ filler * 1e-3
        paged.append(cache.layer, on[0], on[1], positions)
        got = paged.attention(cache.layer, on[2], 110)
    torch.cuda.current_stream(device).wait_stream(side)
    for s in range(2):
        cache.store(s, int(cache.lengths[s]), keys[0, s].double().numpy(),
                    values[0, s].double().numpy(), np.arange(3))
    cache.check_pages()
    rows = [cache.rows(s, int(n) + 3)[:2] for s, n in enumerate(cache.lengths)]
    check_attention(got, queries, rows, cache.lengths, [3], 2)


def test_two_calls_at_once(device):
    """Split calls on two streams have workspaces of their own."""
    caches = [Cache(device, [3000, 2500], 2, 64, 64, seed=s) for s in (1, 2)]
    for c in caches:
        c.lengths -= 1
        c.upload()
    queries = [randn(c.rng, (1, 4, 1, 64), BF16) for c in caches]
    streams = [torch.cuda.Stream(device) for _ in caches]
    there = [q.to(device) for q in queries]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i].append(paged.attention(caches[i].layer, there[i], 3000))
    torch.cuda.synchronize()
    for i in (0, 1):
        rows = [caches[i].rows(s, int(n) + 1)[:2] for s, n in enumerate(caches[i].lengths)]
        check_attention(got[i][0], queries[i], rows, caches[i].lengths, [1], 2)
        assert all(torch.equal(got[i][0], other) for other in got[i])


def test_captured_steps(device):
    """A captured decode step (append, attention, the lengths' advance) replayed, with eager work
    and synchronisations between, against the same steps run eagerly; two graphs share no state. The
    rows grow from step to step, so that blocks move to larger scales."""
    def start():
        return Cache(device, [60, 1000], 2, 128, 32, [90, 1030], seed=5).layer
    rng = np.random.default_rng(6)
    steps = 6
    keys, values = (randn(rng, (steps, 1, 2, 1, 128), BF16).to(device) for _ in range(2))
    growth = torch.exp2(torch.arange(steps, device=device)).view(-1, 1, 1, 1, 1).to(BF16)
    keys, values = keys * growth, values * growth
    queries = randn(rng, (steps, 1, 8, 1, 128), BF16).to(device)
    _, rotary = tables(2000, 64, device)
    at = torch.arange(1000, 1000 + steps, device=device).view(steps, 1, 1)

    def step(layer, k, v, q, p):
        turned = paged.append(layer, k, v, p, rotary=rotary, queries=q)
        out = paged.attention(layer, turned, 1030)
        layer.lengths += 1
        return out

    eager = start()
    expect = [step(eager, keys[i], values[i], queries[i], at[i]) for i in range(steps)]
    layers = [start(), start()]
    static = [[t[0].clone() for t in (keys, values, queries, at)] for _ in layers]
    graphs, outs = [], []
    for layer, s in zip(layers, static):
        side = torch.cuda.Stream(device)
        side.wait_stream(torch.cuda.current_stream(device))
        with torch.cuda.stream(side):  # warm up on a throw-away state
            step(start(), *s)
        torch.cuda.current_stream(device).wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(layer, *s))
        graphs.append(graph)
    for i in range(steps):
        for n in (0, 1):
            for s, t in zip(static[n], (keys, values, queries, at)):
                s.copy_(t[i])
            graphs[n].replay()
        torch.randn(512, 512, device=device).sum().item()
        for n in (0, 1):
            assert torch.equal(outs[n], expect[i]), (i, n)
    for layer in layers:
        assert torch.equal(layer.lengths, eager.lengths) and torch.equal(layer.pages, eager.pages)


@pytest.mark.parametrize("dim,groups,dtype", [(128, 4, BF16), (64, 4, F16), (256, 6, BF16)])
def test_decode_loop_with_evictions(device, dim, groups, dtype):
    """Prompt, decode steps and evictions in one pool, as a budgeted generation runs them: every
    step's output against the oracle on the oracle's own cache, and the pages byte by byte."""
    rng = np.random.default_rng(9)
    kv_heads, page_size, batch = 2, 16, 2
    segments = batch * kv_heads
    pool = paged.PagePool(60, dim, page_size, device, bits=8)
    pool.pages.zero_()
    pages = np.zeros(tuple(pool.pages.shape), np.uint8)
    layer, ids = pool.layer(batch, kv_heads, 100)
    assert layer.bits == 8
    (cos, sin), rotary = tables(200, dim // 2, device)
    lengths, position = [0] * segments, 0

    def feed(length, counts=None):
        nonlocal position
        k, v = (randn(rng, (batch, kv_heads, length, dim), dtype) * 2.0 ** rng.integers(-3, 3)
                for _ in range(2))
        q = randn(rng, (batch, kv_heads * groups, length, dim), dtype)
        where = np.tile(position + np.arange(length), (batch, 1))
        at = torch.from_numpy(where).to(device)
        n = np.full(batch, length) if counts is None else np.array(counts)
        c = None if counts is None else torch.tensor(counts, dtype=torch.int32, device=device)
        turned = paged.append(layer, k.to(device), v.to(device), at, rotary=rotary,
                              queries=q.to(device), counts=c)
        got = paged.attention(layer, turned, max(lengths) + length, counts=c)
        rotated = opaged.rotate(k.float().numpy(), cos[where][:, None], sin[where][:, None])
        table = layer.table.cpu().numpy()
        for s in range(segments):
            b, h = divmod(s, kv_heads)
            if n[b]:
                opaged.append(pages, table[s], lengths[s], page_size, rotated[b, h, :n[b]],
                              v[b, h, :n[b]].float().numpy(), where[b, :n[b]], dtype == F16)
        assert np.array_equal(layer.pages.cpu().numpy(), pages)
        rows = [opaged.load(pages, table[s], lengths[s] + int(n[s // kv_heads]), page_size, dim)[:2]
                for s in range(segments)]
        check_attention(got, turned.cpu(), rows, lengths, n, kv_heads)
        layer.lengths += torch.from_numpy(np.repeat(n, kv_heads).astype(np.int32)).to(device)
        lengths[:] = [x + int(n[s // kv_heads]) for s, x in enumerate(lengths)]
        position += length

    feed(50, [50, 31])
    for _ in range(3):
        for _ in range(4):
            feed(1)
        keep = [np.sort(rng.permutation(x)[:rng.integers(20, 35)]) for x in lengths]
        starts = np.concatenate([[0], np.cumsum(lengths)])
        removed = np.concatenate([starts[s] + np.setdiff1d(np.arange(x), keep[s])
                                  for s, x in enumerate(lengths)])
        target, fresh = pool.table([len(k) + 30 for k in keep], width=layer.table.shape[1])
        old = layer.table.cpu().numpy()
        layer = paged.compact(layer, torch.from_numpy(removed).to(device), target)
        pool.release(ids)
        ids = fresh
        for s in range(segments):
            opaged.compact(pages, old[s], keep[s], target[s].cpu().numpy(), page_size, dim)
        assert np.array_equal(layer.pages.cpu().numpy(), pages)
        lengths[:] = [len(k) for k in keep]
        got = paged.read(layer, sum(lengths), dtype)
        held = [opaged.load(pages, target[s].cpu().numpy(), lengths[s], page_size, dim)
                for s in range(segments)]
        for i in range(3):
            expect = np.concatenate([r[i] for r in held])
            assert np.array_equal(got[i].double().cpu().numpy().reshape(expect.shape), expect)
    feed(9)
    pool.release(ids)
    assert pool.free_pages == 60


def test_offsets_past_32_bits(device):
    """Pages beyond 4 GiB of the pool: rows stored, attended to, moved and read there."""
    dim, page_size = 256, 256
    size = paged.page_bytes(page_size, dim, 8)
    count = (5 << 30) // size
    pages = torch.empty(count, size, dtype=torch.uint8, device=device)
    table = torch.tensor([[count - 1, 2], [0, count - 2]], dtype=torch.int32, device=device)
    lengths = torch.zeros(2, dtype=torch.int32, device=device)
    layer = paged.PagedLayer(pages, table, lengths, 2, dim, page_size, bits=8)
    rng = np.random.default_rng(1)
    keys, values = (randn(rng, (1, 2, 300, dim), BF16) for _ in range(2))
    paged.append(layer, keys.to(device), values.to(device), torch.arange(300, device=device)[None])
    host = np.zeros((10, size), np.uint8)
    own = np.array([[0, 1], [2, 3]])
    for s in range(2):
        opaged.append(host, own[s], 0, page_size, keys[0, s].double().numpy(), values[0, s].double().numpy(),
                      np.arange(300))
    rows = [opaged.load(host, own[s], 300, page_size, dim)[:2] for s in range(2)]
    for length in (1, 90):
        queries = randn(rng, (1, 4, length, dim), BF16)
        got = paged.attention(layer.with_lengths(lengths + 300 - length), queries.to(device), 300)
        check_attention(got, queries, rows, [300 - length] * 2, [length], 2)
    target = torch.tensor([[4, count - 3], [count - 4, 5]], dtype=torch.int32, device=device)
    moved = paged.compact(layer.with_lengths(lengths + 300), torch.tensor([0, 599], device=device),
                          target)
    kept = [np.arange(1, 300), np.arange(299)]
    for s in range(2):
        opaged.compact(host, own[s], kept[s], np.array([[4, 5], [6, 7]])[s], page_size, dim)
    k, v, p, _ = paged.read(moved, 598)
    expect = [opaged.load(host, t, 299, page_size, dim) for t in np.array([[4, 5], [6, 7]])]
    assert np.array_equal(k.double().cpu().numpy(), np.concatenate([e[0] for e in expect]))
    assert np.array_equal(v.double().cpu().numpy(), np.concatenate([e[1] for e in expect]))
    assert p.view(-1).cpu().tolist() == list(range(1, 300)) + list(range(299))
