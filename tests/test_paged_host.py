"""The paged cache's argument checks, on the host (nothing is launched), and the page pool."""

import ctypes

import numpy as np
import pytest
import torch

from code_for_iclr27_amd import _lib, paged
from oracle import paged as opaged

STRIDES = np.array([256, 128, 128], np.int64)


def test_page_bytes():
    for page_size in (16, 32, 64, 128, 256):
        for dim in (64, 128, 256):
            assert paged.page_bytes(page_size, dim) == opaged.page_bytes(page_size, dim)
            assert paged.page_bytes(page_size, dim) % 64 == 0
    for page_size, dim in [(8, 64), (48, 64), (512, 128), (0, 64), (-16, 64), (32, 96), (32, 0)]:
        with pytest.raises(RuntimeError, match="Head dimension must be"):
            paged.page_bytes(page_size, dim)


def append(**over):
    a = dict(keys=256, values=256, queries=None, out_queries=None, batch=1, kv_heads=2,
             query_heads=0, added=1, dim=128, dtype=_lib.LR_DTYPE_BF16, positions=8, cos=None,
             sin=None, table_rows=0, half=0, counts=None, pages=256, page_count=4, page_size=32,
             table=8, max_pages=2, lengths=8, strides=STRIDES)
    a.update(over)
    s = a["strides"].ctypes.data
    return _lib.load().lr_paged_append(
        a["keys"], s, a["values"], s, a["queries"], s, a["out_queries"], a["batch"], a["kv_heads"],
        a["query_heads"], a["added"], a["dim"], a["dtype"], a["positions"], a["cos"], a["sin"],
        a["table_rows"], a["half"], a["counts"], a["pages"], a["page_count"], a["page_size"],
        a["table"], a["max_pages"], a["lengths"], None)


@pytest.mark.parametrize("over,message", [
    (dict(dtype=_lib.LR_DTYPE_F64), "bf16, f16 or f32"),
    (dict(batch=0), "Invalid appended shape"),
    (dict(kv_heads=0), "Invalid appended shape"),
    (dict(added=-1), "Invalid appended shape"),
    (dict(query_heads=4), "Invalid appended shape"),
    (dict(batch=2 ** 31, kv_heads=2), "Invalid appended shape"),
    (dict(dim=96), "Head dimension must be 64, 128 or 256"),
    (dict(page_size=24), "Page size must be"),
    (dict(page_count=-1), "Invalid page table"),
    (dict(table=None), "Invalid page table"),
    (dict(pages=None), "Invalid page table"),
    (dict(lengths=None), "Invalid page table"),
    (dict(max_pages=2 ** 30), "fewer than 2\\^30 rows"),
    (dict(pages=264), "Pages must be 16-byte aligned"),
    (dict(keys=None), "Invalid appended KV"),
    (dict(positions=None), "Invalid appended KV"),
    (dict(queries=256, query_heads=4), "Invalid appended KV"),
    (dict(half=12, cos=256, sin=256, table_rows=9), "multiple of 16"),
    (dict(half=72, cos=256, sin=256, table_rows=9), "at most the head dimension"),
    (dict(half=64), "with tables"),
    (dict(half=64, cos=256, sin=256, table_rows=0), "with tables"),
    (dict(added=2 ** 30), "Appended grid too large"),
    (dict(keys=264), "16-byte aligned"),
    (dict(values=258), "16-byte aligned"),
    (dict(half=64, cos=260, sin=256, table_rows=9), "16-byte aligned"),
    (dict(strides=np.array([256, 132, 128], np.int64)), "16-byte aligned"),
])
def test_append_refusals(over, message):
    import re
    assert append(**over) == 1
    assert re.search(message, _lib.last_error()), _lib.last_error()


def test_append_of_no_rows_enqueues_nothing():
    assert append(added=0, keys=None, values=None, positions=None) == 0


def attend(**over):
    a = dict(queries=256, pages=256, page_count=4, page_size=32, table=8, max_pages=2, lengths=8,
             batch=1, kv_heads=2, groups=4, length=1, dim=128, dtype=_lib.LR_DTYPE_BF16,
             max_keys=64, counts=None, scale=0.1, out=256, workspace=None, size=0, strides=STRIDES)
    a.update(over)
    return _lib.load().lr_paged_attention(
        a["queries"], a["strides"].ctypes.data, a["pages"], a["page_count"], a["page_size"],
        a["table"], a["max_pages"], a["lengths"], a["batch"], a["kv_heads"], a["groups"],
        a["length"], a["dim"], a["dtype"], a["max_keys"], a["counts"],
        ctypes.c_float(a["scale"]), a["out"], a["workspace"], a["size"], None)


@pytest.mark.parametrize("over,message", [
    (dict(dtype=_lib.LR_DTYPE_F32), "fp16 and bf16"),
    (dict(length=0), "Empty attention dimensions"),
    (dict(groups=0), "Empty attention dimensions"),
    (dict(length=2 ** 30), "Attention grid too large"),
    (dict(batch=2 ** 31), "Attention grid too large"),
    (dict(dim=32), "Head dimension must be"),
    (dict(page_size=8), "Page size must be"),
    (dict(max_keys=-1), "Invalid key lengths"),
    (dict(scale=0.0), "Softmax scale must be positive"),
    (dict(scale=-1.0), "Softmax scale must be positive"),
    (dict(scale=float("inf")), "Softmax scale must be positive"),
    (dict(scale=float("nan")), "Softmax scale must be positive"),
    (dict(queries=None), "Invalid attention buffers"),
    (dict(out=None), "Invalid attention buffers"),
    (dict(queries=264), "16-byte aligned"),
    (dict(max_keys=2 ** 30), "Invalid key lengths"),
    (dict(max_pages=2 ** 15, max_keys=2 ** 20), "Attention workspace too small"),
    (dict(max_pages=2, max_keys=4096), "Attention workspace too small"),  # as its size was asked for
    (dict(max_pages=2 ** 15, max_keys=2 ** 20, workspace=128, size=1 << 40), "256-byte aligned"),
])
def test_attention_refusals(over, message):
    assert attend(**over) == 1
    assert message in _lib.last_error()


def test_attention_workspace_grows_with_the_splits():
    size = _lib.load().lr_paged_attention_workspace_bytes
    assert size(8, 4, 1, 64, 128) == 0
    assert size(8, 4, 1, 4096, 128) > 0
    assert size(0, 4, 1, 4096, 128) == 0


def plan(segments, groups, length, max_keys, dim=128):
    out = np.zeros(3, np.int64)
    assert _lib.load().lr_paged_attention_plan(segments, groups, length, max_keys, dim,
                                               out.ctypes.data) == 0
    return out.tolist()


def test_attention_plans():
    """Short calls in one launch, a few rows onto long caches in up to 64 parts, no parts where the
    rows fill the chip, tiles of 32 rows for many."""
    for dim in (64, 128, 256):
        assert plan(8, 4, 1, 0, dim) == plan(8, 4, 1, 100, dim) == [16, 4, 1]
        assert plan(8, 4, 1, 2250, dim) == [16, 4, 18]
        assert plan(8, 4, 1, 130000, dim) == [16, 4, 64]
        assert plan(8, 4, 1, 2 ** 30 - 1, dim)[2] == 64
        assert plan(2048, 4, 1, 2000, dim) == [16, 4, 1]
        assert plan(140, 3, 1, 1000, dim) == [16, 8, 1]
        assert plan(8, 4, 1000, 5000, dim) == [32, 4, 1]
        assert plan(36, 4, 29, 2500, dim)[0] == 32 and plan(36, 4, 29, 2500, dim)[2] > 1
    library, out = _lib.load(), np.zeros(3, np.int64)
    assert library.lr_paged_attention_plan(0, 4, 1, 5, 128, out.ctypes.data) == 1
    assert "Empty attention dimensions" in _lib.last_error()
    assert library.lr_paged_attention_plan(1, 4, 1, 2 ** 30, 128, out.ctypes.data) == 1
    assert "Empty attention dimensions" in _lib.last_error()
    assert library.lr_paged_attention_plan(1, 4, 1, 5, 96, out.ctypes.data) == 1
    assert "Head dimension must be" in _lib.last_error()
    # the workspace holds the parts' states
    for shape in [(8, 4, 1, 2250), (4, 6, 300, 4300), (3, 5, 7, 30000), (64, 4, 1, 2250)]:
        rows, _, splits = plan(*shape)
        tile = min(rows, shape[1] * shape[2])
        tiles = -(-shape[1] * shape[2] // rows)
        size = library.lr_paged_attention_workspace_bytes(*shape, 128)
        assert size == (shape[0] * tiles * splits * tile * 130 * 4 if splits > 1 else 0)


def test_read_and_compact_refusals():
    library = _lib.load()
    read = lambda **o: library.lr_paged_read(  # noqa: E731
        o.get("pages", 256), 4, 32, 8, 2, 8, o.get("segments", 2), 128,
        o.get("dtype", _lib.LR_DTYPE_BF16), o.get("total", 5), o.get("keys", 256), 256, 8,
        o.get("cumulative", 8), None)
    for over, message in [(dict(dtype=_lib.LR_DTYPE_F64), "bf16, f16 or f32"),
                          (dict(segments=0), "Invalid page table"),
                          (dict(total=-1), "Invalid packed buffers"),
                          (dict(total=2 ** 31), "Invalid packed buffers"),
                          (dict(keys=None), "Invalid packed buffers"),
                          (dict(cumulative=None), "Invalid packed buffers"),
                          (dict(keys=264), "16-byte aligned")]:
        assert read(**over) == 1 and message in _lib.last_error(), over
    compact = lambda **o: library.lr_paged_compact(  # noqa: E731
        256, 4, 32, 8, 2, 8, o.get("segments", 2), 128, o.get("removed", 8), o.get("count", 3),
        o.get("target", 8),
        o.get("width", 2), o.get("lengths", 8), o.get("workspace", 256), o.get("size", 64), None)
    for over, message in [(dict(removed=None), "Invalid compaction"),
                          (dict(count=-1), "Invalid compaction"),
                          (dict(target=None), "Invalid compaction"),
                          (dict(width=2 ** 30), "Invalid compaction"),
                          (dict(lengths=None), "Invalid compaction"),
                          (dict(segments=0), "Invalid page table"),
                          (dict(segments=300, workspace=None), "workspace too small"),
                          (dict(segments=300, size=64), "workspace too small"),
                          (dict(segments=300, size=1 << 20, workspace=8), "workspace too small"),
                          (dict(), "other pages"),
                          (dict(target=16), "other pages")]:
        assert compact(**over) == 1 and message in _lib.last_error(), over
    assert library.lr_paged_compact_workspace_bytes(256) == 0
    assert library.lr_paged_compact_workspace_bytes(257) == 258 * 8


def cpu_layer():
    pages = torch.zeros(4, paged.page_bytes(32, 128), dtype=torch.uint8)
    return paged.PagedLayer(pages, torch.zeros(2, 2, dtype=torch.int32),
                            torch.zeros(2, dtype=torch.int32), 2, 128)


def test_cpu_tensors_are_refused():
    layer = cpu_layer()
    rows = torch.zeros(1, 2, 1, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="Expected contiguous CUDA tensor"):
        paged.append(layer, rows, rows, torch.zeros(1, 1, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="Expected contiguous CUDA tensor"):
        paged.attention(layer, rows, 1)
    with pytest.raises(RuntimeError, match="Expected contiguous CUDA tensor"):
        paged.read(layer, 0)
    with pytest.raises(RuntimeError, match="Expected contiguous CUDA tensor"):
        paged.compact(layer, torch.zeros(0, dtype=torch.int64), layer.table)


def test_gradients_are_refused():
    rows = torch.zeros(1, 2, 1, 128, dtype=torch.bfloat16, requires_grad=True)
    plain = rows.detach()
    position = torch.zeros(1, 1, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="forward only"):
        paged.append(cpu_layer(), rows, plain, position)
    with pytest.raises(RuntimeError, match="forward only"):
        paged.append(cpu_layer(), plain, plain, position, queries=rows)
    with pytest.raises(RuntimeError, match="forward only"):
        paged.attention(cpu_layer(), rows, 1)


def test_pool():
    pool = paged.PagePool(10, 128, 32, device="cpu")
    assert pool.pages.shape == (10, paged.page_bytes(32, 128)) and pool.free_pages == 10
    table, ids = pool.table([0, 1, 32, 33, 64])
    assert table.shape == (5, 2) and table.dtype == torch.int32 and pool.free_pages == 4
    assert [(row >= 0).sum().item() for row in table] == [0, 1, 1, 2, 2]
    assert sorted(table[table >= 0].tolist()) == sorted(ids) and len(set(ids)) == 6
    with pytest.raises(RuntimeError, match="Page pool exhausted: 5 pages wanted, 4 free"):
        pool.table([160])
    with pytest.raises(RuntimeError, match="its table holds 1"):
        pool.table([64], width=1)
    with pytest.raises(RuntimeError, match="cannot be negative"):
        pool.table([-1])
    assert pool.free_pages == 4
    pool.release(ids[:2])
    for again in (ids[:1], [ids[2], ids[2]], [99]):
        with pytest.raises(RuntimeError, match="each once"):
            pool.release(again)
    layer, more = pool.layer(2, 3, 32)
    assert layer.table.shape == (6, 1) and len(more) == 6 and pool.free_pages == 0
    assert not layer.lengths.any() and layer.kv_heads == 3 and layer.dim == 128
    wide, none = pool.table([0, 0], width=3)
    assert wide.shape == (2, 3) and none == []


def test_launches_of_2_to_the_32_threads_are_refused():
    """A launch has fewer: larger calls are refused before anything is enqueued."""
    for over in (dict(kv_heads=1, added=2 ** 28, dim=256),
                 dict(kv_heads=1, added=2 ** 27, dim=256, half=8, cos=256, sin=256, table_rows=9)):
        assert append(**over) == 1 and "Appended grid too large" in _lib.last_error(), over
    for over in (dict(batch=2 ** 24, kv_heads=1, groups=1), dict(batch=2 ** 23, kv_heads=1, groups=40),
                 dict(kv_heads=1, batch=1, groups=2 ** 6, length=2 ** 23)):
        assert attend(max_keys=32, **over) == 1, over
        assert "Attention grid too large" in _lib.last_error(), over
    library = _lib.load()
    assert library.lr_paged_read(256, 4, 32, 8, 2, 8, 2, 128, _lib.LR_DTYPE_BF16, 2 ** 30, 256, 256,
                                 8, 8, None) == 1
    assert "Packed rows' grid too large" in _lib.last_error()
    for segments, pages in ((2 ** 24, 1), (5, 2 ** 22 - 1)):
        size = library.lr_paged_compact_workspace_bytes(segments)
        assert library.lr_paged_compact(256, 4, 256, 8, pages, 8, segments, 128, 8, 3, 16, 1, 16,
                                        256, size, None) == 1
        assert "Compaction grid too large" in _lib.last_error(), segments


def test_a_failed_upload_takes_no_pages(monkeypatch):
    """A table that cannot be put on the device leaves the pool as it was."""
    pool = paged.PagePool(10, 128, 32, device="cpu")
    _, ids = pool.table([40])

    def refuse(*args, **kwargs):
        raise RuntimeError("out of memory")

    with monkeypatch.context() as m:
        m.setattr(torch.Tensor, "to", refuse)
        with pytest.raises(RuntimeError, match="out of memory"):
            pool.table([32, 64])
    assert pool.free_pages == 8
    with monkeypatch.context() as m:
        m.setattr(torch, "zeros", refuse)
        with pytest.raises(RuntimeError, match="out of memory"):
            pool.layer(1, 2, 64)
    assert pool.free_pages == 8
    pool.release(ids)
    table, all_pages = pool.table([320])
    assert pool.free_pages == 0 and sorted(all_pages) == list(range(10))
    assert table.tolist() == [all_pages]


def test_gradients_of_the_rotation_tables_are_refused():
    rows = torch.zeros(1, 2, 1, 128, dtype=torch.bfloat16)
    position, angles = torch.zeros(1, 1, dtype=torch.int64), torch.zeros(4, 64, requires_grad=True)
    for rotary in ((angles.cos(), angles.sin()), (angles.detach(), angles), (angles, angles.detach())):
        with pytest.raises(RuntimeError, match="forward only"):
            paged.append(cpu_layer(), rows, rows, position, rotary=rotary)
        with torch.no_grad(), pytest.raises(RuntimeError, match="Expected contiguous CUDA tensor"):
            paged.append(cpu_layer(), rows, rows, position, rotary=rotary)
