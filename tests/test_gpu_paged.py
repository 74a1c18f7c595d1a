"""The paged 4-bit cache's kernels against the numpy oracle: append (whole pages compared byte by
byte), read and compact (bit-exact), attention (f64 softmax over the rows the codes stand for), and
a run of them together as a decode loop with evictions uses them.

Attention's tolerance. Products of a 16-bit query element and a stored value are exact in f32, as
are those of the probabilities' pieces, so the errors are: D f32 additions of a score (each at most
2^-24 of the sum A of the score's absolute terms), the scaled exponent's rounding and the
exponential (a few 2^-24 of A + 1), n additions of the sums, the rounding of a probability to two
bf16 pieces (2^-16 of it), and the output's rounding, half a step of the value and of its error. All
but the last weigh in with E, the same average of |V|: |got - ref| <= eps / 2 |ref| +
(1 + eps) (E (2^-16 + 2 2^-24 ((D + 8) (A + 1) + n + 64)) + 2^-126 n max(1, |V|)); the last term
for exponentials (of which a row's largest is 1 at least) and products below f32's normal numbers.
"""

import numpy as np
import pytest
import torch

from code_for_iclr27_amd import attention as packed
from code_for_iclr27_amd import paged
from oracle import paged as opaged

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


class Cache:
    """A cache on the host and on the device: pages of random bytes, shuffled tables, stored rows."""

    def __init__(self, device, lengths, kv_heads, dim, page_size, room=None, dtype=BF16, seed=0,
                 amplitude=1.0):
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
        for s, n in enumerate(self.lengths):
            rows = [torch.from_numpy(rng.standard_normal((n, dim)) * amplitude).to(dtype)
                    for _ in range(2)]
            self.store(s, 0, *(r.double().numpy() for r in rows), np.arange(n) + 3.0 * s)
        self.upload()

    def store(self, segment, first, keys, values, positions):
        k, v = opaged.quantise(keys, self.f16), opaged.quantise(values, self.f16)
        page, slot = np.divmod(first + np.arange(len(keys)), self.page_size)
        opaged.store(self.pages, self.table[segment, page], slot, self.page_size, *k, *v, positions)

    def upload(self):
        put = lambda a: torch.from_numpy(a.copy()).to(self.device)  # noqa: E731
        self.layer = paged.PagedLayer(put(self.pages), put(self.table), put(self.lengths),
                                      self.kv_heads, self.dim, self.page_size)

    def rows(self, segment, count):
        return opaged.load(self.pages, self.table[segment], count, self.page_size, self.dim)

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


def check_append(device, lengths, kv_heads, groups, added, dim, page_size, dtype, half, counts=None,
                 layout="rows", edit=None, seed=0):
    batch = len(lengths) // kv_heads
    room = np.asarray(lengths) + added
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
@pytest.mark.parametrize("dim,half,page_size", [(64, 32, 16), (128, 64, 32), (256, 32, 64),
                                                (128, 8, 128), (256, 128, 16), (64, 0, 256)])
@pytest.mark.parametrize("added", [1, 37])
def test_append(device, dtype, dim, half, page_size, added):
    check_append(device, [0, 1, 15, 16, 31, 33], 3, 2, added, dim, page_size, dtype, half,
                 seed=dim + half)


@pytest.mark.parametrize("layout", ["heads", "padded"])
def test_append_layouts(device, layout):
    check_append(device, [5, 0, 9, 40], 2, 3, 6, 128, 16, BF16, 64, layout=layout)
    check_append(device, [5, 0, 9, 40], 2, 0, 6, 64, 16, F32, 16, layout=layout)


def test_append_of_a_padded_batch(device):
    check_append(device, [4, 0, 9, 40, 7, 2, 1, 0], 2, 4, 9, 128, 32, BF16, 64,
                 counts=[9, 0, 4, -3])
    check_append(device, [4, 0], 1, 1, 3, 64, 16, F16, 32, counts=[2, 100])


def test_append_many_rows(device):
    check_append(device, [100, 3], 2, 2, 500, 128, 64, BF16, 64, seed=4)


@pytest.mark.parametrize("dtype,dim,half", [(BF16, 64, 32), (F32, 128, 32), (F16, 128, 64),
                                            (BF16, 256, 0)])
def test_append_of_many_rows_takes_several_heads_a_thread(device, dtype, dim, half):
    """From 32,768 rows on; three and six heads are no multiple of the four that a thread takes."""
    check_append(device, [100, 3, 0], 3, 2, 2800, dim, 64, dtype, half, counts=[2799], seed=dim)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_append_edge_values(device, dtype):
    top = float(torch.finfo(dtype).max)
    tiny = 2.0 ** -24 if dtype == F16 else 2.0 ** -133 if dtype == BF16 else 2.0 ** -149

    def edit(keys, values):
        values[0, 0, 0, 3] = float("nan")
        values[0, 0, 1, 40] = float("inf")
        values[0, 0, 2, 31] = -float("inf")
        values[0, 0, 3] = 0.0
        values[0, 0, 4] = -0.0
        values[0, 0, 5, 7] = top
        values[0, 0, 6, :32] = -top
        values[0, 0, 7] = tiny
        values[0, 0, 8, :32] *= tiny * 8
        grid = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -0.25, -0.75, -1.25,
                             -1.75, -2.5, -3.5, -5.0, -6.0])
        values[0, 0, 9, :32] = torch.cat((grid, grid)).to(dtype)
        values[0, 0, 10, :32] = torch.cat((grid, grid * 0.5)).to(dtype) * 2.0 ** -20
        values[0, 0, 11, 0] = 6.96875  # under the step to the next scale, and on it
        values[0, 0, 12, 0] = 7.0
        keys[0, 0] = values[0, 0]
    check_append(device, [3], 1, 1, 13, 64, 16, dtype, 0, edit=edit)


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
    assert not v.isnan().any() and p.view(2, 5)[:, 2:].cpu().tolist() == [[-1, 4, 10]] * 2
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


def test_read_many_segments(device):
    """More segments than the summing workgroup has threads, most of them empty."""
    rng = np.random.default_rng(8)
    lengths = np.where(rng.random(2500) < 0.2, rng.integers(1, 20, 2500), 0)
    cache = Cache(device, lengths, 1, 64, 16)
    keys, _, positions = packed_rows(cache, lengths)
    got = paged.read(cache.layer, int(lengths.sum()))
    assert np.array_equal(got[0].double().cpu().numpy(), keys)
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
    from code_for_iclr27_amd import _lib
    k, v = (torch.full((40, 64), 9.0, dtype=BF16, device=device) for _ in range(2))
    p = torch.full((40,), -1.0, device=device)
    cu = torch.empty(4, dtype=torch.int32, device=device)
    a = cache.layer
    _lib.call("lr_paged_read", a.pages.data_ptr(), a.pages.shape[0], 16, a.table.data_ptr(),
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


def check_compact(device, lengths, dim, page_size, share, seed=0):
    rng = np.random.default_rng(seed)
    lengths = np.asarray(lengths)
    cache = Cache(device, lengths, 1, dim, page_size, seed=dim)
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
    cache.upload()
    got = paged.compact(cache.layer, torch.from_numpy(removed).to(device),
                        torch.from_numpy(target).to(device))
    torch.cuda.synchronize()
    assert got.lengths.cpu().tolist() == [len(k) for k in keep]
    assert cache.layer.lengths.cpu().tolist() == lengths.tolist()
    for s, kept in enumerate(keep):  # the rows' bytes, section by section
        to, offset = np.arange(len(kept)), 0
        for width in (dim // 2, dim // 2, dim // 32, dim // 32, 4):
            place = lambda table, row: (  # noqa: E731
                table[s, row // page_size][:, None],
                offset + (row % page_size)[:, None] * width + np.arange(width))
            cache.pages[place(target, to)] = cache.pages[place(cache.table, kept)]
            offset += page_size * width
    cache.check_pages()


@pytest.mark.parametrize("dim,page_size", [(64, 16), (128, 32), (256, 64)])
@pytest.mark.parametrize("share", [0.0, 0.1, 0.6, 1.0])
def test_compact(device, dim, page_size, share):
    check_compact(device, [0, 1, 16, 33, 64, 65, 200, 150], dim, page_size, share)


def test_compact_long_and_many_segments(device):
    """Searches of several rounds; more segments than a workgroup sums for itself."""
    check_compact(device, [3000, 0, 5, 2600], 64, 128, 0.4, seed=1)
    check_compact(device, [3000, 0, 5, 2600], 128, 16, 0.02, seed=2)
    lengths = np.random.default_rng(3).integers(0, 12, 700)
    check_compact(device, lengths, 64, 16, 0.5, seed=4)
    check_compact(device, lengths[:256], 64, 16, 0.3, seed=5)
    check_compact(device, lengths[:257], 64, 16, 0.3, seed=6)


def test_compact_into_a_short_table_and_missing_pages(device):
    cache = Cache(device, [40, 40], 2, 64, 16)
    extra = len(cache.pages)
    cache.pages = np.concatenate([cache.pages, np.zeros((3, cache.pages.shape[1]), np.uint8)])
    cache.upload()
    before = cache.pages.copy()
    target = torch.tensor([[extra], [extra + 99]], dtype=torch.int32, device=device)
    removed = torch.tensor([0, 41], device=device)
    got = paged.compact(cache.layer, removed, target)
    assert got.lengths.cpu().tolist() == [39, 39]
    rows = paged.read(got.with_lengths(torch.tensor([16, 0], dtype=torch.int32, device=device)), 16)
    assert np.array_equal(rows[0].double().cpu().numpy(), cache.rows(0, 17)[0][1:])
    after = got.pages.cpu().numpy()
    untouched = [p for p in range(len(before)) if p != extra]
    assert np.array_equal(after[untouched], before[untouched])


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
        mine = np.abs(q[b, h * groups:(h + 1) * groups])  # [G, L, D]
        terms = mine @ np.abs(np.nan_to_num(keys)).T * scale
        if terms.shape[-1]:
            a[b, :, h * groups:(h + 1) * groups] = terms.max(-1).T
            top[b, 0, h * groups:(h + 1) * groups] = np.abs(values).max(0).clip(min=1.0)
    return out, average, top, a


def check_attention(got, queries, rows, lengths, counts, kv_heads, scale=None):
    batch, heads, length, dim = queries.shape
    scale = dim ** -0.5 if scale is None else scale
    expect, average, top, a = reference(queries, rows, lengths, counts, kv_heads, scale)
    assert got.shape == expect.shape and got.dtype == queries.dtype
    got = got.double().cpu().numpy().reshape(batch, length, heads, dim)
    expect, average = expect.reshape(got.shape), average.reshape(got.shape)
    most = max((len(k) for k, _ in rows), default=0)
    eps = torch.finfo(queries.dtype).eps
    bound = eps / 2 * np.abs(expect) + (1 + eps) * (2.0 ** -126 * most * top + average * (
        2.0 ** -16 + 2 * 2.0 ** -24 * ((dim + 8) * (a[..., None] + 1) + most + 64)))
    error = np.abs(got - expect)
    assert np.all(error <= bound), float((error - bound).max())
    return expect


def attend(device, lengths, kv_heads, groups, length, dim, page_size, dtype=BF16, counts=None,
           seed=0, amplitude=1.0, scale=None, slack=0, layout="rows"):
    batch = len(lengths) // kv_heads
    n = np.full(batch, length) if counts is None else np.clip(np.asarray(counts), 0, length)
    grown = np.asarray(lengths) + np.repeat(n, kv_heads)
    cache = Cache(device, grown, kv_heads, dim, page_size, dtype=dtype, seed=seed)
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


EDGES = [0, 1, 2, 14, 15, 16, 30, 31, 32, 33, 62, 63, 126, 127, 128, 129, 254, 256, 511, 700]


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


def test_decode_long(device):
    attend(device, [20001, 17], 2, 2, 1, 64, 128)


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


@pytest.mark.parametrize("dim,groups", [(64, 4), (128, 4), (256, 6)])
def test_prefill(device, dim, groups):
    attend(device, [0, 60], 2, groups, 250, dim, 32, seed=dim, layout="heads")


def plan(segments, groups, length, max_keys, dim=128):
    from code_for_iclr27_amd import _lib
    out = np.zeros(3, np.int64)
    _lib.call("lr_paged_attention_plan", segments, groups, length, max_keys, dim, out.ctypes.data)
    return out.tolist()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim,page_size,groups,length", [(64, 16, 4, 32), (128, 32, 3, 43),
                                                         (256, 64, 4, 32), (128, 16, 7, 19),
                                                         (64, 256, 1, 120), (256, 16, 6, 22)])
def test_tiles_of_32_rows(device, dtype, dim, page_size, groups, length):
    lengths = np.random.default_rng(dim).integers(0, 150, 144)
    lengths[:6] = [0, 1, 31, 32, 33, 200]
    assert plan(144, groups, length, int(lengths.max()) + length, dim)[::2] == [32, 1]
    attend(device, lengths, 24, groups, length, dim, page_size, dtype, seed=length, layout="heads")


@pytest.mark.parametrize("dim,page_size", [(64, 32), (128, 16), (256, 128)])
def test_tiles_of_32_rows_with_split_keys(device, dim, page_size):
    lengths = np.random.default_rng(dim).integers(0, 60, 36)
    lengths[[3, 17, 35]] = [1700, 1013, 2471]
    rows, _, splits = plan(36, 4, 29, 2500, dim)
    assert rows == 32 and splits > 1
    attend(device, lengths, 12, 4, 29, dim, page_size, seed=dim)
    attend(device, lengths, 12, 4, 29, dim, page_size, seed=dim, counts=[29, 11, 0])


@pytest.mark.parametrize("dim,page_size", [(64, 16), (128, 64), (256, 32)])
def test_eight_waves(device, dim, page_size):
    lengths = np.random.default_rng(dim).integers(0, 30, 140)
    lengths[[0, 5, 100, 139]] = [600, 255, 256, 999]
    assert plan(140, 3, 1, 1000, dim) == [16, 8, 1]
    attend(device, lengths, 10, 3, 1, dim, page_size, seed=dim)


@pytest.mark.parametrize("dim,segments,groups,length,rows", [(64, 36, 7, 5, 3000),
                                                             (128, 24, 7, 5, 1500),
                                                             (256, 24, 3, 9, 2200)])
def test_eight_waves_with_split_keys(device, dim, segments, groups, length, rows):
    lengths = np.random.default_rng(dim).integers(0, 90, segments)
    lengths[[1, 9, 22]] = [rows - length, rows // 2, rows // 3]
    assert plan(segments, groups, length, rows, dim)[1] == 8
    assert plan(segments, groups, length, rows, dim)[2] > 1
    attend(device, lengths, 12, groups, length, dim, 32, seed=dim)


def test_padded_batch(device):
    for length in (1, 5, 40, 500):
        assert plan(8, 4, length, 800)[0] == (32 if length == 500 else 16)
        attend(device, [0, 5, 100, 33, 64, 0, 7, 300], 2, 4, length, 128, 16,
               counts=[length, 0, length // 2 + 1, -1], seed=length)


def test_scales(device):
    for scale in (1e-3, 1.0, 3.0):
        attend(device, [50, 200], 2, 4, 3, 128, 32, scale=scale)


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


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("length,groups", [(1, 4), (5, 3), (128, 24)])
def test_values_of_every_size(device, dim, length, groups):
    """Blocks of V that f16 holds as normal or subnormal numbers, that it does not hold, of zeros,
    and all of these in one segment."""
    sizes = [1.0, 2e-4, 3e-6, 1e-9, 1e-30, 4e4, 1e30, 0.0, None, None]
    lengths = np.asarray([0, 33, 75, 75, 75, 75, 75, 90, 140, 300])
    assert plan(10, groups, length, 300 + length, dim)[0] == (32 if length == 128 else 16)
    cache = Cache(device, lengths + length, 10, dim, 16)
    for s, size in enumerate(sizes):
        n = int(lengths[s]) + length
        keys, values = cache.rng.standard_normal((2, n, dim))
        if size is None:
            drawn = cache.rng.choice(sizes[:7], (n, dim // 32), p=[.94, .01, .01, .01, .01, .01, .01])
            size = np.repeat(drawn * (cache.rng.random(drawn.shape) < 0.9), 32, 1)
        cache.store(s, 0, keys, values * size, np.arange(n))
    cache.lengths = lengths.astype(np.int32)
    cache.upload()
    queries = randn(cache.rng, (1, 10 * groups, length, dim), BF16)
    got = paged.attention(cache.layer, queries.to(device), 300 + length)
    rows = [cache.rows(s, int(n) + length)[:2] for s, n in enumerate(lengths)]
    check_attention(got, queries, rows, lengths, [length], 10)
    assert not got[..., 7 * groups * dim:8 * groups * dim].any()


@pytest.mark.parametrize("dtype,margins", [(BF16, (6, 18, 30, 55)), (F16, (6, 12, 18))])
@pytest.mark.parametrize("segments,groups,length,most", [(2, 3, 1, 90), (8, 4, 1, 2250), (140, 3, 1, 1000),
                                                         (144, 3, 43, 243)])
def test_a_dominant_key_of_no_value(device, dtype, margins, segments, groups, length, most):
    """All of the output is small probabilities on large values, on one side of zero and on both."""
    forms = {2: [16, 4, 1], 140: [16, 8, 1], 144: [32, 4, 1]}
    assert plan(segments, groups, length, most) == forms.get(segments, [16, 4, 18])
    lengths = np.random.default_rng(segments).integers(5, 40, segments)
    lengths[0], lengths[-1] = most - length, (most - length) // 2
    cache = Cache(device, lengths + length, 2, 128, 16, dtype=dtype)
    for s in range(segments):
        n = int(lengths[s]) + length
        keys, values = np.zeros((n, 128)), 8e3 * cache.rng.random((n, 128)) + 1e3
        keys[n // 3], values[n // 3] = 1.5, 0.0
        values[:, 64:] *= cache.rng.choice([-1, 1], (n, 64))
        cache.store(s, 0, keys, values, np.arange(n))
    cache.lengths = lengths.astype(np.int32)
    cache.upload()
    queries = torch.ones(segments // 2, 2 * groups, length, 128, dtype=dtype)
    rows = [cache.rows(s, int(n) + length)[:2] for s, n in enumerate(lengths)]
    for margin in margins:
        scale = margin / 192
        got = paged.attention(cache.layer, queries.to(device), most, scale=scale)
        check_attention(got, queries, rows, lengths, [length] * (segments // 2), 2, scale)


def test_max_length_bounds_the_keys(device):
    cache = Cache(device, [200, 90], 2, 128, 32)
    queries = randn(cache.rng, (1, 4, 1, 128), BF16)
    rows = [cache.rows(s, n)[:2] for s, n in enumerate((100, 90))]
    cache.lengths = np.array([199, 89], np.int32)
    cache.upload()
    got = paged.attention(cache.layer, queries.to(device), 100)
    check_attention(got, queries, rows, [199, 89], [1], 2)
    assert not paged.attention(cache.layer, queries.to(device), 0).any()


def test_keys_in_missing_pages_do_not_count(device):
    cache = Cache(device, [70, 70], 2, 64, 16)
    cache.lengths[:] = 69
    keep = np.ones(70, bool)
    cache.table[0, 1], cache.table[0, 4] = -1, len(cache.pages)
    keep[16:32] = keep[64:] = False
    cache.table[1] = -7
    cache.upload()
    queries = randn(cache.rng, (1, 4, 1, 64), BF16)
    got = paged.attention(cache.layer, queries.to(device), 70)
    table = np.where(cache.table < 0, 0, np.minimum(cache.table, len(cache.pages) - 1))
    keys, values, _ = opaged.load(cache.pages, table[0], 70, 16, 64)
    rows = [(keys[keep], values[keep]), (np.zeros((0, 64)), np.zeros((0, 64)))]
    check_attention(got, queries, rows, [69, 69], [1], 2)
    assert not got[..., 128:].any()


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("length,groups", [(1, 4), (6, 2), (40, 3), (128, 24)])
def test_nan_blocks_reach_only_the_rows_that_see_them(device, dim, length, groups):
    """NaN blocks of V (in the last key of all and at the diagonal), and of K: a row that sees a NaN
    key is NaN, one that sees a NaN block of V is NaN in its channels."""
    lengths = [45, 130] + [20] * (6 if length == 128 else 0)
    heads, most = len(lengths), 130 + length
    assert plan(heads, groups, length, most, dim)[0] == (32 if length == 128 else 16)
    grown = np.asarray(lengths) + length
    cache = Cache(device, grown, heads, dim, 16)
    cache.lengths = np.asarray(lengths, np.int32)
    blocks = dim // 32
    scales = lambda which, s, row: (  # noqa: E731
        cache.table[s, row // 16], 16 * dim + which * 16 * blocks + row % 16 * blocks)
    marks = [(1, 0, 45 + length - 1, blocks - 1), (1, 1, 130 + length // 2, 0)]
    if length > 1:
        marks.append((0, 1, 130 + length - 2, 0))
    for which, s, row, block in marks:
        page, at = scales(which, s, row)
        cache.pages[page, at + block] = 255
    cache.upload()
    queries = randn(cache.rng, (1, heads * groups, length, dim), BF16)
    got = paged.attention(cache.layer, queries.to(device), most)
    got = got.view(length, heads, groups, dim).double().cpu().numpy()
    rows = [cache.rows(s, int(n))[:2] for s, n in enumerate(grown)]
    with np.errstate(invalid="ignore"):
        expect = opaged.attention(queries.double().numpy(), rows, lengths, [length], heads)
    expect = expect.reshape(got.shape)
    assert np.isnan(expect).any() and (length == 1 or not np.isnan(expect).all())
    assert np.array_equal(np.isnan(got), np.isnan(expect))
    fine = ~np.isnan(expect)
    np.testing.assert_allclose(got[fine], expect[fine], rtol=2.0 ** -8, atol=1e-3)


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


def test_shared_pages_and_wide_tables(device):
    """Requests that share a prefix's pages read the same rows; tables far wider than their segments
    change nothing."""
    cache = Cache(device, [70, 100], 1, 128, 32)
    cache.table[0, :2] = cache.table[1, :2]  # the first 64 rows are one prefix
    cache.lengths = np.array([69, 99], np.int32)
    cache.upload()
    queries = randn(cache.rng, (2, 4, 1, 128), BF16)
    rows = [cache.rows(s, n)[:2] for s, n in enumerate((70, 100))]
    first = paged.attention(cache.layer, queries.to(device), 100)
    check_attention(first, queries, rows, [69, 99], [1, 1], 1)
    wide = torch.full((2, 5000), 10 ** 9, dtype=torch.int32, device=device)
    wide[:, :cache.table.shape[1]] = cache.layer.table
    import dataclasses
    layer = dataclasses.replace(cache.layer, table=wide)
    for bound in (100, 5000 * 32):
        check_attention(paged.attention(layer, queries.to(device), bound), queries, rows, [69, 99],
                        [1, 1], 1)
    grown = layer.with_lengths(layer.lengths + 1)
    for a, b in zip(paged.read(grown, 170), paged.read(cache.layer.with_lengths(grown.lengths), 170)):
        assert torch.equal(a, b)
    target = torch.full_like(wide, -1)
    target[0, 0], target[1, 0] = (int(p) for p in cache.spare[:2])
    removed = torch.arange(60, 160, device=device)  # ten of the first stay out, ninety of the other
    moved = paged.compact(grown, removed, target)
    assert moved.lengths.cpu().tolist() == [60, 10]
    k = paged.read(moved.with_lengths(moved.lengths.clamp(max=32)), 42)[0].double().cpu().numpy()
    assert np.array_equal(k, np.concatenate((rows[0][0][:32], rows[1][0][90:])))


def test_attention_equals_packed_attention_over_the_rows_read(device):
    """The same rows give the same output but for the order of sums, half a step of either output
    and the paged kernel's probabilities, within 2^-16 of the average of |V| (from the packed kernel,
    rounded once)."""
    for length, dim in ((1, 128), (4, 64), (90, 128)):
        got, cache, queries = attend(device, [300, 411, 90, 1000], 2, 4, length, dim, 32)
        grown = cache.layer.lengths + length
        keys, values, _, cu = paged.read(cache.layer.with_lengths(grown), int(grown.sum()))
        from types import SimpleNamespace
        meta = SimpleNamespace(cu_seqlens_k=cu, max_seqlen_k=int(grown.max()),
                               decoding_cu_seqlens_q=torch.arange(5, device=device))
        other = packed.packed_attention(queries.to(device), keys, values, meta, length, 2)
        average = packed.packed_attention(queries.to(device), keys, values.abs(), meta, length, 2)
        a, b = got.float(), other.float()
        bound = 2.0 ** -7 * b.abs() + 2.0 ** -16 * (1 + 2.0 ** -6) * average.float() + 1e-5
        assert ((a - b).abs() <= bound).all()


def test_empty_pool_and_empty_table(device):
    pages = torch.empty(0, paged.page_bytes(32, 128), dtype=torch.uint8, device=device)
    lengths = torch.tensor([5, 0], dtype=torch.int32, device=device)
    for width in (0, 1):
        table = torch.zeros(2, width, dtype=torch.int32, device=device)
        layer = paged.PagedLayer(pages, table, lengths, 2, 128)
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
    import dataclasses
    change = lambda **o: dataclasses.replace(layer, **o)  # noqa: E731
    refused = [
        (lambda: paged.append(change(dim=96), rows, rows, at), "Head dimension must be"),
        (lambda: paged.append(change(page_size=32), rows, rows, at), "Pages must be uint8"),
        (lambda: paged.append(change(pages=layer.pages.float()), rows, rows, at), "Pages must be"),
        (lambda: paged.append(change(table=layer.table.long()), rows, rows, at), "Page table must"),
        (lambda: paged.append(change(table=layer.table[:1]), rows, rows, at), "Page table must"),
        (lambda: paged.append(change(lengths=layer.lengths.long()), rows, rows, at), "Lengths must"),
        (lambda: paged.append(change(lengths=layer.lengths.cpu()), rows, rows, at), "contiguous CUDA"),
        (lambda: paged.append(layer, rows[:, :1], rows[:, :1], at), "New keys and values"),
        (lambda: paged.append(layer, rows, rows[..., :64], at), "New keys and values"),
        (lambda: paged.append(layer, rows, rows.half(), at), "same dtype"),
        (lambda: paged.append(layer, rows.double(), rows.double(), at), "bf16, f16 or f32"),
        (lambda: paged.append(layer, rows, rows, at, queries=rows[:, :, :, :64]), "New queries"),
        (lambda: paged.append(layer, rows, rows, at, queries=rows[:, [0, 0, 1]]), "must divide"),
        (lambda: paged.append(layer, rows, rows, at.int()), "Positions must be"),
        (lambda: paged.append(layer, rows, rows, at[:, [0, 0]]), "Positions must be"),
        (lambda: paged.append(layer, rows, rows, at, rotary=(torch.zeros(4, 64, device=device), None)),
         "go together"),
        (lambda: paged.append(layer, rows, rows, at, rotary=(torch.zeros(4, 64, device=device),) * 2,
                              counts=torch.zeros(2, dtype=torch.int32, device=device)), "Counts must"),
        (lambda: paged.append(layer, rows, rows, at, rotary=(torch.zeros(4, 12, device=device),) * 2),
         "multiple of 16"),
        (lambda: paged.append(layer, rows, rows, at, rotary=(torch.zeros(4, 72, device=device),) * 2),
         "at most the head dimension"),
        (lambda: paged.append(layer, rows, rows, at,
                              rotary=(torch.zeros(4, 64, device=device).half(),) * 2), "float32"),
        (lambda: paged.append(layer, torch.zeros(1, 2, 128, 1, dtype=BF16, device=device)
                              .transpose(2, 3), rows, at), None),
        (lambda: paged.append(layer, torch.zeros(1, 2, 128, 2, dtype=BF16, device=device)
                              .transpose(2, 3)[:, :, :1], rows, at), "contiguous last dimension"),
        (lambda: paged.append(layer, torch.zeros(2 * 128 + 1, dtype=BF16, device=device)[1:]
                              .view(1, 2, 1, 128), rows, at), "16-byte aligned"),
        (lambda: paged.attention(layer, rows.float(), 5), "fp16 and bf16"),
        (lambda: paged.attention(layer, rows[..., :64], 5), "Queries must be"),
        (lambda: paged.attention(layer, rows[:, [0, 0, 1]], 5), "must divide"),
        (lambda: paged.attention(layer, rows, -1), "Invalid max_seqlen_k"),
        (lambda: paged.attention(layer, rows, 5, scale=0.0), "scale must be positive"),
        (lambda: paged.read(layer, -1), "Invalid packed rows"),
        (lambda: paged.read(layer, 5, torch.float64), "bf16, f16 or f32"),
        (lambda: paged.compact(layer, at.int()[0], layer.table), "Removed indices must be int64"),
        (lambda: paged.compact(layer, at[0], layer.table.long()), "Page table must"),
        (lambda: paged.compact(layer, at[0], layer.table), "other pages"),
    ]
    for call, message in refused:
        if message is None:
            call()
            continue
        with pytest.raises(RuntimeError, match=message):
            call()
    torch.cuda.synchronize()


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
    and synchronisations between, against the same steps run eagerly; two graphs share no state."""
    def start():
        cache = Cache(device, [60, 1000], 2, 128, 32, [90, 1030], seed=5)
        return cache.layer
    rng = np.random.default_rng(6)
    steps = 6
    keys, values = (randn(rng, (steps, 1, 2, 1, 128), BF16).to(device) for _ in range(2))
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
        assert torch.equal(layer.lengths, eager.lengths)


def test_decode_loop_with_evictions(device):
    """Prompt, decode steps and evictions in one pool, as a budgeted generation runs them: every
    step's output and the cache's rows against the oracle's own cache."""
    rng = np.random.default_rng(9)
    kv_heads, groups, dim, page_size, batch = 2, 4, 128, 16, 2
    segments = batch * kv_heads
    pool = paged.PagePool(60, dim, page_size, device)
    layer, ids = pool.layer(batch, kv_heads, 100)
    (cos, sin), rotary = tables(200, 64, device)
    rows = [[np.zeros((0, dim)), np.zeros((0, dim)), np.zeros(0)] for _ in range(segments)]
    position = 0

    def feed(length, counts=None):
        nonlocal position
        k, v = (randn(rng, (batch, kv_heads, length, dim), BF16) for _ in range(2))
        q = randn(rng, (batch, kv_heads * groups, length, dim), BF16)
        where = np.tile(position + np.arange(length), (batch, 1))
        at = torch.from_numpy(where).to(device)
        n = np.full(batch, length) if counts is None else np.array(counts)
        c = None if counts is None else torch.tensor(counts, dtype=torch.int32, device=device)
        turned = paged.append(layer, k.to(device), v.to(device), at, rotary=rotary,
                              queries=q.to(device), counts=c)
        got = paged.attention(layer, turned, max(len(r[0]) for r in rows) + length, counts=c)
        rotated = opaged.rotate(k.float().numpy(), cos[where][:, None], sin[where][:, None])
        lengths = [len(r[0]) for r in rows]
        for s in range(segments):
            b, h = divmod(s, kv_heads)
            new = [opaged.values(*opaged.quantise(x[b, h, :n[b]])) for x in (rotated, v.double().numpy())]
            rows[s] = [np.concatenate((rows[s][0], new[0])), np.concatenate((rows[s][1], new[1])),
                       np.concatenate((rows[s][2], where[b, :n[b]]))]
        check_attention(got, turned.cpu(), [r[:2] for r in rows], lengths, n, kv_heads)
        layer.lengths += torch.from_numpy(np.repeat(n, kv_heads).astype(np.int32)).to(device)
        position += length

    feed(50, [50, 31])
    for turn in range(3):
        for _ in range(4):
            feed(1)
        keep = [np.sort(rng.permutation(len(r[0]))[:rng.integers(20, 35)]) for r in rows]
        starts = np.concatenate([[0], np.cumsum([len(r[0]) for r in rows])])
        removed = np.concatenate([starts[s] + np.setdiff1d(np.arange(len(r[0])), keep[s])
                                  for s, r in enumerate(rows)])
        target, fresh = pool.table([len(k) + 30 for k in keep], width=layer.table.shape[1])
        layer = paged.compact(layer, torch.from_numpy(removed).to(device), target)
        pool.release(ids)
        ids = fresh
        rows = [[part[k] for part in r] for r, k in zip(rows, keep)]
        got = paged.read(layer, sum(len(k) for k in keep))
        for i in range(3):
            expect = np.concatenate([r[i] for r in rows])
            assert np.array_equal(got[i].double().cpu().numpy().reshape(expect.shape), expect)
    feed(9)
    pool.release(ids)
    assert pool.free_pages == 60


def test_offsets_past_32_bits(device):
    """Pages beyond 4 GiB of the pool: rows stored, attended to, moved and read there."""
    dim, page_size = 256, 256
    size = paged.page_bytes(page_size, dim)
    count = (5 << 30) // size
    pages = torch.empty(count, size, dtype=torch.uint8, device=device)
    table = torch.tensor([[count - 1, 2], [0, count - 2]], dtype=torch.int32, device=device)
    lengths = torch.zeros(2, dtype=torch.int32, device=device)
    layer = paged.PagedLayer(pages, table, lengths, 2, dim, page_size)
    rng = np.random.default_rng(1)
    keys, values = (randn(rng, (1, 2, 300, dim), BF16) for _ in range(2))
    paged.append(layer, keys.to(device), values.to(device), torch.arange(300, device=device)[None])
    queries = randn(rng, (1, 4, 1, dim), BF16)
    got = paged.attention(layer.with_lengths(lengths + 299), queries.to(device), 300)
    rows = [tuple(opaged.values(*opaged.quantise(x[0, s].double().numpy())) for x in (keys, values))
            for s in range(2)]
    check_attention(got, queries, rows, [299, 299], [1], 2)
    target = torch.tensor([[4, count - 3], [count - 4, 5]], dtype=torch.int32, device=device)
    moved = paged.compact(layer.with_lengths(lengths + 300), torch.tensor([0, 599], device=device),
                          target)
    k, _, p, _ = paged.read(moved, 598)
    assert np.array_equal(k.double().cpu().numpy(), np.concatenate((rows[0][0][1:], rows[1][0][:-1])))
    assert p.view(-1).cpu().tolist() == list(range(1, 300)) + list(range(299))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("segments,groups,length,most", [(8, 4, 1, 90), (8, 4, 1, 2250),
                                                         (140, 3, 1, 1000), (144, 3, 43, 243)])
def test_probabilities_keep_all_of_their_bits(device, dtype, dim, segments, groups, length, most):
    """Two keys of nearly the same score whose values cancel: the output, 2^-12 of the average of
    |V|, is what their probabilities differ by. Scores are exact (two channels), and of the others
    P is below 2^-69 and V 0, so errors are counted without the scores' additions, in units of 2^-24 of the
    average: 7 for the exponents (their products, references and differences, 10 2^-24 in all, times
    ln 2), 6 for three exponentials, 12 for the additions and the weights that join three keys, 3 for
    the division. (Probabilities of 16 to 18 bits miss it by 2 to 3 times.)"""
    forms = {140: [16, 8, 1], 144: [32, 4, 1]}
    assert plan(segments, groups, length, most, dim) == forms.get(
        segments, [16, 4, 1] if most == 90 else [16, 4, 18])
    lengths = np.random.default_rng(segments).integers(5, 40, segments)
    lengths[0], lengths[-1] = most - length, (most - length) // 2
    cache = Cache(device, lengths + length, 2, dim, 16, dtype=dtype)
    for s in range(segments):
        n = int(lengths[s])
        keys, values = np.zeros((n + length, dim)), np.zeros((n + length, dim))
        keys[:, 0] = -192.0
        places = cache.rng.permutation(n)[:3]
        keys[places, 0] = 6.0, 4.0, 4.0
        keys[places[2], 32] = 6 * 2.0 ** -12
        values[places[1]], values[places[2]] = 96.0, -96.0
        cache.store(s, 0, keys, values, np.arange(n + length))
    cache.lengths = lengths.astype(np.int32)
    cache.upload()
    queries = torch.zeros(segments // 2, 2 * groups, length, dim, dtype=dtype)
    rows = torch.arange(queries[..., 0].numel()).view(queries.shape[:3])
    queries[..., 0], queries[..., 32] = 1 + rows % 97 / 128.0, 1.0
    got = paged.attention(cache.layer, queries.to(device), most, scale=0.25)
    held = [cache.rows(s, int(n) + length)[:2] for s, n in enumerate(lengths)]
    counts = [length] * (segments // 2)
    expect, average = (opaged.attention(queries.double().numpy(), [(k, f(v)) for k, v in held],
                                        lengths, counts, 2, 0.25) for f in (np.asarray, np.abs))
    eps = torch.finfo(dtype).eps
    bound = eps / 2 * np.abs(expect) + (1 + eps) * 28 * 2.0 ** -24 * average
    error = np.abs(got.double().cpu().numpy() - expect)
    assert np.all(error <= bound), float((error / bound).max())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("segments,groups,length,most", [(8, 4, 1, 90), (8, 4, 1, 2250),
                                                         (140, 3, 1, 1000), (144, 3, 43, 243)])
def test_scores_of_every_finite_size(device, dtype, dim, segments, groups, length, most):
    """Scores of 2^27 to 2^59, whose rounded products with the scale are off by up to 2^35: the keys
    of a row's largest score share the output, the others lie far below. Scores are exact (equal
    channels of a few bits each), so the largest one's probability is one, the output the mean of
    their values: off by its rounding and, in units of 2^-24 of the average of |V|, one for each of up to
    `most` additions to the sum and the products' sum and 64 for the rest."""
    forms = {140: [16, 8, 1], 144: [32, 4, 1]}
    assert plan(segments, groups, length, most, dim) == forms.get(
        segments, [16, 4, 1] if most == 90 else [16, 4, 18])
    lengths = np.random.default_rng(segments).integers(5, 40, segments)
    lengths[0], lengths[-1] = most - length, (most - length) // 2
    cache = Cache(device, lengths + length, 2, dim, 16, dtype=dtype)
    codes = np.array([0, .5, 1, 1.5, 2, 3, 4, 6, -.5, -1, -1.5, -2, -3, -4, -6]) * 2.0 ** 13
    for s in range(segments):
        n = int(lengths[s]) + length
        keys = np.repeat(cache.rng.choice(codes, (n, 1)), dim, 1)
        if s % 4 == 3:  # all scores of one sign, growing to the end
            keys = np.sort(np.abs(keys), 0)
        cache.store(s, 0, keys, cache.rng.standard_normal((n, dim)), np.arange(n))
    cache.lengths = lengths.astype(np.int32)
    cache.upload()
    sizes = 2.0 ** 12 * torch.tensor([1.0, -1.125, 8.0, -8.0, 1.875, -15.0, 13.0])
    queries = torch.ones(segments // 2, 2 * groups, length, dim, dtype=dtype)
    rows = torch.arange(queries[..., 0].numel()).view(queries.shape[:3])
    queries *= sizes[rows % 7].unsqueeze(-1).to(dtype)
    held = [cache.rows(s, int(n) + length)[:2] for s, n in enumerate(lengths)]
    expect, average = np.zeros((2, segments // 2, length, 2 * groups, dim))
    for s, (keys, values) in enumerate(held):
        b, h = divmod(s, 2)
        for i in range(length):
            n = int(lengths[s]) + i + 1
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


@pytest.mark.parametrize("length,groups,most", [(1, 4, 90), (5, 3, 2250), (128, 24, 300)])
def test_a_segment_of_negative_length_has_no_rows_to_attend_to(device, length, groups, most):
    """Appends store nothing behind a negative length, so its queries see nothing either: not the
    rows that lie in its pages' first slots."""
    cache = Cache(device, [60, 200, 70, 90], 2, 64, 16)
    cache.lengths = np.array([40, -1, -(2 ** 31), 60], np.int32)
    cache.upload()
    queries = randn(cache.rng, (2, 2 * groups, length, 64), BF16)
    got = paged.attention(cache.layer, queries.to(device), most)
    got = got.view(2, length, 2, groups * 64)
    assert not got[0, :, 1].any() and not got[1, :, 0].any()
    assert got[0, :, 0].any(-1).all() and got[1, :, 1].any(-1).all()
    assert paged.read(cache.layer, 100)[3].cpu().tolist() == [0, 40, 40, 40, 100]


NAN_FORMS = {  # (segments, groups, queries, longest): rows of a tile, waves, split
    (8, 4, 1, 90): (16, 4, False), (8, 4, 1, 2250): (16, 4, True), (140, 3, 1, 1000): (16, 8, False),
    (36, 7, 5, 3000): (16, 8, True), (144, 3, 43, 243): (32, 4, False), (36, 4, 29, 2500): (32, 4, True)}


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("shape", NAN_FORMS)
def test_nan_blocks_in_every_form(device, dtype, dim, shape):
    """NaN blocks of V and K in the first rows, in the middle of the cache (a part of its own where
    the keys are split), at the diagonal and at the last key: a row that sees a NaN key is NaN, one
    that sees a NaN block of V is NaN in its channels, and all others are within the tolerance."""
    segments, groups, length, most = shape
    rows, waves, split = NAN_FORMS[shape]
    chosen = plan(segments, groups, length, most, dim)
    assert chosen[:2] == [rows, waves] and (chosen[2] > 1) == split
    lengths = np.random.default_rng(segments).integers(3, 40, segments)
    lengths[0], lengths[3], lengths[4], lengths[5], lengths[-1] = [most - length] * 5
    grown = lengths + length
    cache = Cache(device, grown, 2, dim, 16, dtype=dtype, seed=dim)
    cache.lengths = lengths.astype(np.int32)
    blocks = dim // 32
    marks = [(0, 1, most // 2, 0), (1, 1, int(grown[1]) - 1, blocks - 1), (2, 0, 1, 0),
             (3, 1, most - 1 - length // 2, 1), (3, 1, 0, blocks - 1), (4, 0, most - 1, 1),
             (5, 0, most - 1 - length // 2, 0), (5, 1, most // 3, 0)]
    for s, which, row, block in marks:
        at = 16 * dim + which * 16 * blocks + row % 16 * blocks + block
        cache.pages[cache.table[s, row // 16], at] = 255
    cache.upload()
    queries = randn(cache.rng, (segments // 2, 2 * groups, length, dim), dtype)
    got = paged.attention(cache.layer, queries.to(device), most)
    held = [cache.rows(s, int(n))[:2] for s, n in enumerate(grown)]
    counts = [length] * (segments // 2)
    with np.errstate(invalid="ignore"):
        expect, average, _, a = reference(queries, held, lengths, counts, 2, dim ** -0.5)
    got = got.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(expect))
    assert np.isnan(expect).any() and not np.isnan(expect).all()
    shape = (segments // 2, length, 2 * groups, dim)
    got, expect, average = (x.reshape(shape) for x in (got, expect, average))
    eps = torch.finfo(dtype).eps
    # (2^-25: half of f16's subnormal step)
    bound = eps / 2 * np.abs(expect) + (1 + eps) * average * (
        2.0 ** -22 * ((dim + 8) * (a[..., None] + 1) + most + 64)) + 2.0 ** -25
    fine = ~np.isnan(expect)
    assert np.all(np.abs(got - expect)[fine] <= bound[fine])


def test_an_audit_of_the_rows_read_back_evicts_the_same_rows(device):
    """Prompt and decode steps in two layers, the rows read back into an audit (scores, selection,
    its own compaction of the packed rows), and the rows that it removes taken out of the cache: the
    pages hold what the audit's compacted layers hold, bit for bit. Twice, so that the second audit
    meets ragged heads."""
    from code_for_iclr27_amd import audit, scoring
    rng = np.random.default_rng(21)
    layers, kv_heads, groups, dim, window, budget = 2, 2, 4, 128, 16, 40
    pool = paged.PagePool(200, dim, 16, device)
    held = [pool.layer(1, kv_heads, 300) for _ in range(layers)]
    lengths = [[0] * kv_heads for _ in range(layers)]
    _, rotary = tables(1000, dim // 2, device)
    position = 0
    for _ in range(2):
        for length in (150, 1, 1, 1):
            at = torch.arange(position, position + length, device=device)[None]
            for n, (layer, _) in enumerate(held):
                k, v = (randn(rng, (1, kv_heads, length, dim), BF16).to(device) for _ in range(2))
                q = randn(rng, (1, kv_heads * groups, length, dim), BF16).to(device)
                q = paged.append(layer, k, v, at, rotary=rotary, queries=q)
                out = paged.attention(layer, q, max(lengths[n]) + length)
                assert out.isfinite().all()
                layer.lengths += length
                lengths[n] = [r + length for r in lengths[n]]
            position += length
        states = []
        for n, (layer, _) in enumerate(held):
            keys, values, where, cu = paged.read(layer, sum(lengths[n]))
            assert cu.cpu().tolist() == np.concatenate([[0], np.cumsum(lengths[n])]).tolist()
            states.append(scoring.LayerState(
                keys, values, where.view(-1), lengths[n], None,
                randn(rng, (kv_heads * groups, window, dim), BF16).to(device),
                randn(rng, (kv_heads * groups, dim), F32).to(device)))
        outcome = audit.AuditStep().run(
            states, torch.arange(position - window, position, device=device),
            torch.ones(1, device=device), layers * kv_heads * budget + 3, protect_recent=8)
        chosen, offsets = (t.cpu().numpy() for t in (outcome.selection.removed_positions,
                                                     outcome.selection.offsets))
        gone = {(s.layer, s.head): chosen[offsets[i]:offsets[i + 1]]
                for i, s in enumerate(outcome.segments)}
        assert sum(len(g) for g in gone.values()) == layers * kv_heads * budget + 3
        for n, (layer, pages) in enumerate(held):
            starts = np.concatenate([[0], np.cumsum(lengths[n])])
            removed = np.concatenate([starts[h] + gone[n, h] for h in range(kv_heads)])
            lengths[n] = [lengths[n][h] - len(gone[n, h]) for h in range(kv_heads)]
            target, fresh = pool.table([r + 160 for r in lengths[n]])
            layer = paged.compact(layer, torch.from_numpy(removed).to(device), target)
            pool.release(pages)
            held[n] = layer, fresh
            kept = outcome.layers[n]
            assert list(kept.head_lens) == lengths[n] and layer.lengths.cpu().tolist() == lengths[n]
            got = paged.read(layer, sum(lengths[n]))
            for a, b in zip(got, (kept.keys, kept.values, kept.positions)):
                assert torch.equal(a.view(-1), b.reshape(-1))
    assert len({*map(tuple, lengths)}) > 1 or len(set(lengths[0])) > 1


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("segments,groups,length,most", [(8, 4, 1, 90), (8, 4, 1, 2250),
                                                         (140, 3, 1, 1000), (144, 3, 43, 243)])
def test_large_scores_keep_their_differences(device, dtype, dim, segments, groups, length, most):
    """Exact scores of 2^27 on either side of zero, that differ by one to eight of f32's steps there: with
    scale 1/8 by factors of e^2 of the probabilities, by e^16 and e^128 with larger ones. An exponent is
    exact but for the scale's rounding and its own (of at most 24: 3 2^-24 24 ln 2), so that in units
    of 2^-24 of the average of |V| the sums' additions count, 2 `most`, and 128 for the rest. Where that average is next to
    nothing: half of f16's smallest step, and what lies below f32's normal numbers (of exponentials whose
    largest is 2^-8 at least, as the reference's rounding is 8 at most at 2^28)."""
    forms = {140: [16, 8, 1], 144: [32, 4, 1]}
    assert plan(segments, groups, length, most, dim) == forms.get(
        segments, [16, 4, 1] if most == 90 else [16, 4, 18])
    lengths = np.random.default_rng(segments).integers(5, 40, segments)
    lengths[0], lengths[-1] = most - length, (most - length) // 2
    cache = Cache(device, lengths + length, 2, dim, 16, dtype=dtype)
    for s in range(segments):
        n = int(lengths[s]) + length
        keys = np.zeros((n, dim))
        keys[:, 0], keys[:, 32] = 2.0 ** 15, cache.rng.choice([0, .5, 1, 1.5, 2, 3, -.5, -1], n)
        cache.store(s, 0, keys, cache.rng.standard_normal((n, dim)), np.arange(n))
    cache.lengths = lengths.astype(np.int32)
    cache.upload()
    queries = torch.zeros(segments // 2, 2 * groups, length, dim, dtype=dtype)
    rows = torch.arange(queries[..., 0].numel()).view(queries.shape[:3])
    queries[..., 0], queries[..., 32] = 4096.0 * (1 - 2 * (rows % 2)), 32.0
    held = [cache.rows(s, int(n) + length)[:2] for s, n in enumerate(lengths)]
    eps = torch.finfo(dtype).eps
    for scale in (0.125, 1.0, 8.0):
        got = paged.attention(cache.layer, queries.to(device), most, scale=scale)
        expect, average = (opaged.attention(
            queries.double().numpy(), [(k, f(v)) for k, v in held], lengths,
            [length] * (segments // 2), 2, scale) for f in (np.asarray, np.abs))
        bound = eps / 2 * np.abs(expect) + (1 + eps) * average * 2.0 ** -24 * (2 * most + 128)
        bound += 2.0 ** -25 * (dtype == F16) + 2.0 ** -118 * most * 8
        error = np.abs(got.double().cpu().numpy() - expect)
        assert np.all(error <= bound), (scale, float((error / bound).max()))
