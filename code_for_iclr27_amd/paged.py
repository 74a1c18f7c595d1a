"""A paged KV cache held in 4 or 8 bits: append with the position rotation, attention, compaction,
and the way back to packed rows.

The reference keeps its cache as packed 16-bit rows and copies all of them at every append
(cache.py:33-52). Here a layer's rows lie in pages of a pool, quantised, and an append writes the
step's rows only. A (request, KV head) segment keeps its own rows, so heads may be ragged, as an
eviction leaves them. A pool holds one of two formats (``bits``), and every call takes either:

4  blocks of 32 channels of a row share a scale (OCP MX FP4: E2M1 codes times a power of two). A
   d128 row takes 140 bytes, its position included, in the place of 516; elements are off by up to
   a quarter.
8  16 rows of a head share one scale for their keys and one for their values (E4M3 codes times a
   power of two). A d128 row takes 264 bytes; elements are off by up to 2^-4. An append whose rows
   have larger elements than those in their block moves the block to a larger scale: which bits are
   lost then, all below 2^-17 of the block's largest element, does not depend on the calls that the
   rows came in.

Either's values are exact in the matrix cores' bf16.

One decode step of a layer::

    queries = paged.append(layer, keys, values, positions, rotary=(cos, sin), queries=queries)
    output = paged.attention(layer, queries, max_length)   # over the cached and the new rows
    layer.lengths += 1                                     # once the step is done

(one ``lengths`` tensor for every layer, each layer holding its row of it, makes that one launch a
step). An audit reads the rows back (``read``), scores them as before and removes rows with
``compact``. ``append``, ``attention``, ``read`` and ``compact`` run on torch's current stream and wait
for nothing; all of them can be captured into a HIP graph. (A ``PagePool`` uploads its tables with a copy
that the host waits for, outside of graphs.) There is no CPU path and no backward pass.
"""

from __future__ import annotations

import dataclasses
from collections import deque
from itertools import islice
from typing import Sequence

import torch

from . import _lib


def _format(bits) -> str:
    """The prefix of a format's entry points."""
    if bits not in (4, 8):
        raise RuntimeError("A paged cache holds 4 or 8 bits")
    return "lr_paged_" if bits == 4 else "lr_paged8_"


def page_bytes(page_size: int, dim: int, bits: int = 4) -> int:
    """Bytes of a page: ``page_size`` rows of K and V codes, scales and positions."""
    size = int(getattr(_lib.load(), _format(bits) + "page_bytes")(int(page_size), int(dim)))
    if size == 0:
        raise RuntimeError("Head dimension must be 64, 128 or 256 and page size 16, 32, 64, 128 "
                           "or 256")
    return size


@dataclasses.dataclass
class PagedLayer:
    """A layer's rows: ``pages`` uint8 [pages, page_bytes(page_size, dim, bits)], ``table`` int32
    [batch * kv_heads, max_pages] (row i of a segment: slot i % page_size of page i // page_size),
    ``lengths`` int32 [batch * kv_heads], on one device. ``compact`` and ``read`` take the segments
    of several layers in one table as well. A page that is appended to belongs to one segment;
    segments that only read may share pages."""

    pages: torch.Tensor
    table: torch.Tensor
    lengths: torch.Tensor
    kv_heads: int
    dim: int
    page_size: int = 32
    bits: int = 4

    def with_lengths(self, lengths: torch.Tensor) -> "PagedLayer":
        return dataclasses.replace(self, lengths=lengths)


class PagePool:
    """The pages of one device and the host's list of free ones."""

    def __init__(self, page_count: int, dim: int, page_size: int = 32, device="cuda",
                 bits: int = 4) -> None:
        self.dim, self.page_size, self.bits = int(dim), int(page_size), int(bits)
        self.pages = torch.empty((int(page_count), page_bytes(page_size, dim, bits)),
                                 dtype=torch.uint8, device=device)
        self._free = deque(range(int(page_count)))
        self._taken = set()

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def table(self, rows: Sequence[int], width: int | None = None):
        """Pages for ``rows[s]`` rows of each segment: (table int32 [segments, width] on the
        pool's device, the pages' ids for ``release``). Entries past a segment's pages are -1. The
        room is the table's for good: a segment that needs more moves to another one (``compact``),
        or the caller writes further pages' ids into the table itself."""
        needed = [-(-int(n) // self.page_size) for n in rows]
        if any(int(n) < 0 for n in rows):
            raise RuntimeError("A segment's rows cannot be negative")
        width = max(needed, default=0) if width is None else int(width)
        if max(needed, default=0) > width:
            raise RuntimeError(f"A segment needs {max(needed)} pages, its table holds {width}")
        if sum(needed) > len(self._free):
            raise RuntimeError(f"Page pool exhausted: {sum(needed)} pages wanted, "
                               f"{len(self._free)} free")
        host = torch.full((len(needed), width), -1, dtype=torch.int32)
        ids = list(islice(self._free, sum(needed)))
        first = 0
        for segment, count in enumerate(needed):
            host[segment, :count] = torch.tensor(ids[first:first + count], dtype=torch.int32)
            first += count
        table = host.to(self.pages.device)
        for _ in ids:  # taken once the table is there: an upload that fails takes none
            self._free.popleft()
        self._taken.update(ids)
        return table, ids

    def release(self, ids: Sequence[int]) -> None:
        """Takes pages back. Work that reads them has been enqueued on the stream that their next
        owner writes on (or is waited for there)."""
        ids = [int(i) for i in ids]
        if len(set(ids)) != len(ids) or not self._taken.issuperset(ids):
            raise RuntimeError("Released pages must be taken ones, each once")
        self._taken.difference_update(ids)
        self._free.extend(ids)

    def layer(self, batch: int, kv_heads: int, rows: int):
        """An empty layer with room for ``rows`` rows a segment: (PagedLayer, its pages' ids)."""
        segments = int(batch) * int(kv_heads)
        lengths = torch.zeros(segments, dtype=torch.int32, device=self.pages.device)
        table, ids = self.table([rows] * segments)
        return PagedLayer(self.pages, table, lengths, int(kv_heads), self.dim, self.page_size,
                          self.bits), ids


_native_module = None


def _native():
    """The C++ host module with the paged entry points bound (once)."""
    global _native_module
    if _native_module is None:
        import ctypes
        from .scoring import _planner
        planner = _planner()
        library = _lib.load()
        address = lambda name: ctypes.cast(getattr(library, name), ctypes.c_void_p).value
        for bits in (4, 8):
            planner.bind_paged(bits, *(address(_format(bits) + name) for name in (
                "append", "attention", "attention_workspace_bytes", "read", "compact",
                "compact_workspace_bytes", "page_bytes")), address("lr_last_error"))
        _native_module = planner
    return _native_module


def _forward_only(name):
    raise RuntimeError(f"paged.{name}: the cache has no backward pass (forward only)")


def append(layer, keys, values, positions, rotary=None, queries=None, counts=None):
    """Stores the step's ``keys`` and ``values`` [batch, kv_heads, length, dim] (bf16, f16 or f32;
    any strides of 8 elements with dim contiguous) behind each segment's ``layer.lengths`` rows;
    the lengths stay as they are. ``positions`` int64 [batch, length] are kept with the rows.

    ``rotary``: ``(cos, sin)``, float32 [positions, half]: channels c and c + half of a key, c <
    half, are rotated by the angles of its position before it is stored (half a multiple of 8; the
    channels past 2 * half stay as they are), and so are ``queries`` [batch, query_heads, length,
    dim], which are returned (contiguous, rounded once; None without queries). A position outside
    the tables gives NaN. ``counts`` int32 [batch] on the device: request b brings its first
    counts[b] rows only (a padded batch, or a request that has ended). Rows that the table has no
    page for are not stored. In 8 bits, rows written over later ones that were given up (a draft's)
    leave their block's scale at what these needed."""
    cos, sin = (None, None) if rotary is None else rotary
    if torch.is_grad_enabled() and (
            keys.requires_grad or values.requires_grad or queries is not None and queries.requires_grad
            or cos is not None and cos.requires_grad or sin is not None and sin.requires_grad):
        _forward_only("append")
    return (_native_module or _native()).paged_append(
        layer.pages, layer.table, layer.lengths, layer.kv_heads, layer.dim, layer.page_size,
        layer.bits, keys, values, positions, cos, sin, queries, counts)


def attention(layer, queries, max_length, counts=None, scale=None):
    """Attention of the step's ``queries`` [batch, query_heads, length, dim] (bf16 or f16, rotated)
    over each segment's cached rows and the step's own, appended just before: query i sees the
    first ``lengths + i + 1`` rows. -> [batch, length, query_heads * dim] in the queries' dtype, as
    ``packed_attention`` returns it; rows of padding queries (at or past ``counts[b]``) are zero.

    ``max_length``: a bound on every segment's cached rows plus ``length`` (host int; rows past it
    are not visited, and the keys are split over the chip by it). ``scale`` defaults to dim^-0.5.
    f16 queries are for rows appended as f16, in 4 bits (of others, keys outside f16's range read as
    infinities and zeros); in 8 bits for any. Finite scores may be of any size that f32 holds."""
    if queries.requires_grad and torch.is_grad_enabled():
        _forward_only("attention")
    return (_native_module or _native()).paged_attention(
        layer.pages, layer.table, layer.lengths, layer.kv_heads, layer.dim, layer.page_size,
        layer.bits, queries, int(max_length), counts, float(layer.dim ** -0.5 if scale is None else scale))


def read(layer, total, dtype=torch.bfloat16):
    """The ``total`` rows the cache holds (the host's sum of the lengths), packed by segment:
    (keys [total, dim], values, positions float32 [total, 1], cu_seqlens_k int32 [segments + 1])
    in ``dtype`` (bf16, f16 or f32): what ``scoring.LayerState`` and ``_C`` take. Rows of the outputs
    that the cache does not hold (``total`` past its rows, or a table entry outside the pool) are not
    written: they hold whatever their memory held."""
    return tuple((_native_module or _native()).paged_read(
        layer.pages, layer.table, layer.lengths, layer.dim, layer.page_size, layer.bits, int(total),
        dtype))


def compact(layer, removed, target):
    """Evicts rows: ``removed`` int64 [count] on the device, sorted, unique row numbers in the
    packed order of ``read`` (as for ``_C.compact``). The rows that stay are moved, in order, to the
    pages of ``target`` int32 [segments, max_pages] (pages that the layer does not use, such as
    ``PagePool.table`` gives); the old pages stay as they are. In 8 bits a block of 16 rows takes the
    largest scale of the rows that come together in it. -> the layer in its new pages."""
    lengths = (_native_module or _native()).paged_compact(
        layer.pages, layer.table, layer.lengths, layer.dim, layer.page_size, layer.bits, removed,
        target)
    return dataclasses.replace(layer, table=target, lengths=lengths)
