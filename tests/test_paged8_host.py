"""The 8-bit paged cache's argument checks, on the host (nothing is launched), its plan and pool."""

import ctypes
import re

import numpy as np
import pytest
import torch

from code_for_iclr27_amd import _lib, paged
from oracle import paged8 as opaged

STRIDES = np.array([256, 128, 128], np.int64)


def test_page_bytes():
    for page_size in (16, 32, 64, 128, 256):
        for dim in (64, 128, 256):
            assert paged.page_bytes(page_size, dim, 8) == opaged.page_bytes(page_size, dim)
            assert paged.page_bytes(page_size, dim, 8) % 128 == 0
    for page_size, dim in [(8, 64), (48, 64), (512, 128), (0, 64), (-16, 64), (32, 96), (32, 0)]:
        with pytest.raises(RuntimeError, match="Head dimension must be"):
            paged.page_bytes(page_size, dim, 8)
    for bits in (0, 3, 16, None):
        with pytest.raises(RuntimeError, match="4 or 8 bits"):
            paged.page_bytes(32, 128, bits)


def append(**over):
    a = dict(keys=256, values=256, queries=None, out_queries=None, batch=1, kv_heads=2,
             query_heads=0, added=1, dim=128, dtype=_lib.LR_DTYPE_BF16, positions=8, cos=None,
             sin=None, table_rows=0, half=0, counts=None, pages=256, page_count=4, page_size=32,
             table=8, max_pages=2, lengths=8, strides=STRIDES)
    a.update(over)
    s = a["strides"].ctypes.data
    return _lib.load().lr_paged8_append(
        a["keys"], s, a["values"], s, a["queries"], s, a["out_queries"], a["batch"], a["kv_heads"],
        a["query_heads"], a["added"], a["dim"], a["dtype"], a["positions"], a["cos"], a["sin"],
        a["table_rows"], a["half"], a["counts"], a["pages"], a["page_count"], a["page_size"],
        a["table"], a["max_pages"], a["lengths"], None)


@pytest.mark.parametrize("over,message", [
    (dict(dtype=_lib.LR_DTYPE_F64), "bf16, f16 or f32"),
    (dict(batch=0), "Invalid appended shape"),
    (dict(added=-1), "Invalid appended shape"),
    (dict(query_heads=4), "Invalid appended shape"),
    (dict(batch=2 ** 31, kv_heads=2), "Invalid appended shape"),
    (dict(dim=96), "Head dimension must be 64, 128 or 256"),
    (dict(page_size=24), "Page size must be"),
    (dict(table=None), "Invalid page table"),
    (dict(max_pages=2 ** 30), "fewer than 2\\^30 rows"),
    (dict(pages=264), "Pages must be 16-byte aligned"),
    (dict(keys=None), "Invalid appended KV"),
    (dict(half=12, cos=256, sin=256, table_rows=9), "multiple of 16"),
    (dict(half=72, cos=256, sin=256, table_rows=9), "at most the head dimension"),
    (dict(half=64), "with tables"),
    (dict(added=2 ** 30), "Appended grid too large"),
    (dict(kv_heads=1, added=2 ** 29, dim=64), "Appended grid too large"),
    (dict(batch=2 ** 26, kv_heads=2, dim=64), "Appended grid too large"),
    (dict(keys=264), "16-byte aligned"),
    (dict(strides=np.array([256, 132, 128], np.int64)), "16-byte aligned"),
])
def test_append_refusals(over, message):
    assert append(**over) == 1
    assert re.search(message, _lib.last_error()), _lib.last_error()


def test_append_of_no_rows_enqueues_nothing():
    assert append(added=0, keys=None, values=None, positions=None) == 0


def attend(**over):
    a = dict(queries=256, pages=256, page_count=4, page_size=32, table=8, max_pages=2, lengths=8,
             batch=1, kv_heads=2, groups=4, length=1, dim=128, dtype=_lib.LR_DTYPE_BF16,
             max_keys=64, counts=None, scale=0.1, out=256, workspace=None, size=0, strides=STRIDES)
    a.update(over)
    return _lib.load().lr_paged8_attention(
        a["queries"], a["strides"].ctypes.data, a["pages"], a["page_count"], a["page_size"],
        a["table"], a["max_pages"], a["lengths"], a["batch"], a["kv_heads"], a["groups"],
        a["length"], a["dim"], a["dtype"], a["max_keys"], a["counts"],
        ctypes.c_float(a["scale"]), a["out"], a["workspace"], a["size"], None)


@pytest.mark.parametrize("over,message", [
    (dict(dtype=_lib.LR_DTYPE_F32), "fp16 and bf16"),
    (dict(length=0), "Empty attention dimensions"),
    (dict(length=2 ** 30), "Attention grid too large"),
    (dict(batch=2 ** 24, kv_heads=1, groups=1, max_keys=32), "Attention grid too large"),
    (dict(dim=32), "Head dimension must be"),
    (dict(page_size=8), "Page size must be"),
    (dict(max_keys=-1), "Invalid key lengths"),
    (dict(scale=0.0), "Softmax scale must be positive"),
    (dict(scale=float("nan")), "Softmax scale must be positive"),
    (dict(out=None), "Invalid attention buffers"),
    (dict(queries=264), "16-byte aligned"),
    (dict(max_keys=2 ** 30), "Invalid key lengths"),
    (dict(max_pages=2 ** 15, max_keys=2 ** 20), "Attention workspace too small"),
    (dict(max_pages=2 ** 15, max_keys=2 ** 20, workspace=128, size=1 << 40), "256-byte aligned"),
])
def test_attention_refusals(over, message):
    assert attend(**over) == 1
    assert message in _lib.last_error()


def test_the_workspace_holds_the_parts_states():
    library, out = _lib.load(), np.zeros(3, np.int64)
    for shape in [(8, 4, 1, 2250), (4, 6, 300, 4300), (3, 5, 7, 30000), (64, 4, 1, 2250), (8, 4, 1, 64)]:
        for dim in (64, 128, 256):
            assert library.lr_paged8_attention_plan(*shape, dim, out.ctypes.data) == 0
            rows, _, splits = out.tolist()
            tile = min(rows, shape[1] * shape[2])
            tiles = -(-shape[1] * shape[2] // rows)
            size = library.lr_paged8_attention_workspace_bytes(*shape, dim)
            assert size == (shape[0] * tiles * splits * tile * (dim + 2) * 4 if splits > 1 else 0)
    assert library.lr_paged8_attention_workspace_bytes(0, 4, 1, 4096, 128) == 0
    assert library.lr_paged8_attention_plan(0, 4, 1, 5, 128, out.ctypes.data) == 1
    assert "Empty attention dimensions" in _lib.last_error()
    assert library.lr_paged8_attention_plan(1, 4, 1, 5, 96, out.ctypes.data) == 1
    assert "Head dimension must be" in _lib.last_error()


def test_read_and_compact_refusals():
    library = _lib.load()
    read = lambda **o: library.lr_paged8_read(  # noqa: E731
        o.get("pages", 256), 4, 32, 8, 2, 8, o.get("segments", 2), 128,
        o.get("dtype", _lib.LR_DTYPE_BF16), o.get("total", 5), o.get("keys", 256), 256, 8,
        o.get("cumulative", 8), None)
    for over, message in [(dict(dtype=_lib.LR_DTYPE_F64), "bf16, f16 or f32"),
                          (dict(segments=0), "Invalid page table"),
                          (dict(total=-1), "Invalid packed buffers"),
                          (dict(total=2 ** 30), "Packed rows' grid too large"),
                          (dict(keys=None), "Invalid packed buffers"),
                          (dict(cumulative=None), "Invalid packed buffers"),
                          (dict(keys=264), "16-byte aligned")]:
        assert read(**over) == 1 and message in _lib.last_error(), over
    compact = lambda **o: library.lr_paged8_compact(  # noqa: E731
        256, 4, 32, 8, o.get("pages", 2), 8, o.get("segments", 2), 128, o.get("removed", 8),
        o.get("count", 3), o.get("target", 8), o.get("width", 2), o.get("lengths", 8),
        o.get("workspace", 256), o.get("size", 64), None)
    for over, message in [(dict(removed=None), "Invalid compaction"),
                          (dict(count=-1), "Invalid compaction"),
                          (dict(target=None), "Invalid compaction"),
                          (dict(width=2 ** 30), "Invalid compaction"),
                          (dict(lengths=None), "Invalid compaction"),
                          (dict(segments=0), "Invalid page table"),
                          (dict(segments=300, workspace=None), "workspace too small"),
                          (dict(segments=300, size=64), "workspace too small"),
                          (dict(segments=2 ** 24, target=16, lengths=16, size=1 << 40),
                           "Compaction grid too large"),
                          (dict(), "other pages"),
                          (dict(target=16), "other pages")]:
        assert compact(**over) == 1 and message in _lib.last_error(), over
    assert library.lr_paged8_compact_workspace_bytes(256) == 0
    assert library.lr_paged8_compact_workspace_bytes(257) == 258 * 8


def cpu_layer():
    pages = torch.zeros(4, paged.page_bytes(32, 128, 8), dtype=torch.uint8)
    return paged.PagedLayer(pages, torch.zeros(2, 2, dtype=torch.int32),
                            torch.zeros(2, dtype=torch.int32), 2, 128, bits=8)


def test_cpu_tensors_and_gradients_are_refused():
    layer = cpu_layer()
    rows = torch.zeros(1, 2, 1, 128, dtype=torch.bfloat16)
    position = torch.zeros(1, 1, dtype=torch.int64)
    for call in (lambda: paged.append(layer, rows, rows, position), lambda: paged.attention(layer, rows, 1),
                 lambda: paged.read(layer, 0),
                 lambda: paged.compact(layer, torch.zeros(0, dtype=torch.int64), layer.table)):
        with pytest.raises(RuntimeError, match="Expected contiguous CUDA tensor"):
            call()
    leaf = rows.clone().requires_grad_()
    for call in (lambda: paged.append(layer, leaf, rows, position), lambda: paged.attention(layer, leaf, 1),
                 lambda: paged.append(layer, rows, rows, position, queries=leaf)):
        with pytest.raises(RuntimeError, match="forward only"):
            call()


def test_pool():
    pool = paged.PagePool(10, 128, 32, device="cpu", bits=8)
    assert pool.pages.shape == (10, opaged.page_bytes(32, 128)) and pool.free_pages == 10
    layer, ids = pool.layer(2, 3, 32)
    assert layer.bits == 8 and layer.with_lengths(layer.lengths + 1).bits == 8 and len(ids) == 6
    assert paged.PagePool(1, 128, 32, device="cpu").layer(1, 1, 3)[0].bits == 4
    with pytest.raises(RuntimeError, match="4 or 8 bits"):
        paged.PagePool(1, 128, 32, device="cpu", bits=5)
