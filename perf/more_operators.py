"""The paged 8-bit KV cache's operators as a user's program calls them, and their plain forms.

A cache of one layer (or of several, their segments in a row) is a pool of pages and a page table.
A page holds ``page_size`` rows of one (request, KV head) segment. 16 of them form a token block with
one scale for its keys and one for its values: E4M3 codes (a sign, four bits of exponent, three of
significand, up to 448; a magnitude of 127 is NaN) times a power of two, whose exponent plus 127 is
the scale byte. A page's sections:

keys       [blocks, dim / 16, 16 rows, 16 channels] codes
values     [blocks, 4, dim, 4] codes: row 4 i + j of a block at [i, channel, j]
positions  [page_size] f32
scales     [blocks, (keys, values)], in room for 4 page_size bytes

A block's scale is the smallest 2^e that keeps its largest finite magnitude within the codes: e =
floor(log2 amax) - 8, one more from a significand of 1.8125 on. An element is rounded to four
significant bits (ties to even); what lies under the smallest code, 2^(e - 9), is cut off. So codes
at a larger scale follow from those at a smaller one, and a block that grows by a row with larger
elements takes the larger scale as if all of its rows had come at once.

A case is a dict with a ``kind``:

``append``   one layer's new keys and values: keys rotated to their positions, both quantised and
             stored behind each segment's rows; the queries rotated beside them. The outputs are
             the rotated queries and the cache's rows as read back
``attention`` ``length`` queries a head over each segment's cached rows and the ``length`` rows
             appended last (causal)
``compact``  the rows of every segment but the removed ones, into other pages, where a block takes
             the largest scale of its rows; read back
``read``     the rows the cache stands for, packed by segment

``ragged`` cases have a batch whose requests bring fewer rows than the longest (``counts``).
Shapes are the repository's benchmark configurations (8 KV heads of d64 or d128 with 4 query heads
each, 4 KV heads of d256 with 6) and ragged variants around them.
"""

import math

import numpy as np
import torch

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
DEVICE = "cuda"
BLOCK = 16  # rows that share a scale
own = False


def listed():
    return [
        # a decode step's append in a static batch of 16 requests, ragged caches
        {"name": "append8-8b-step-batch16", "kind": "append", "batch": 16, "kv_heads": 8,
         "groups": 4, "dim": 128, "added": 1, "cached": 200, "spread": 150, "half": 64, "page": 32,
         "dtype": "bf16", "ragged": False},
        # a long prompt of the 8B shape in one call
        {"name": "append8-8b-prompt-8192", "kind": "append", "batch": 1, "kv_heads": 8,
         "groups": 4, "dim": 128, "added": 8192, "cached": 0, "spread": 0, "half": 64, "page": 64,
         "dtype": "bf16", "ragged": False},
        # prompts of different lengths in one padded batch of the hybrid shape (64 of 256 channels
        # rotated), behind what the cache holds already
        {"name": "append8-hybrid-padded", "kind": "append", "batch": 4, "kv_heads": 4, "groups": 6,
         "dim": 256, "added": 523, "cached": 700, "spread": 300, "half": 32, "page": 16,
         "dtype": "f16", "ragged": True},
        # a decode step's attention of one request, small model: the smallest call
        {"name": "decode8-1b-f16", "kind": "attention", "batch": 1, "kv_heads": 8, "groups": 4,
         "dim": 64, "length": 1, "cached": 1100, "spread": 0, "page": 16, "dtype": "f16",
         "ragged": False},
        # a static batch of eight, ragged budgets
        {"name": "decode8-8b-batch8", "kind": "attention", "batch": 8, "kv_heads": 8, "groups": 4,
         "dim": 128, "length": 1, "cached": 2000, "spread": 1000, "page": 32, "dtype": "bf16",
         "ragged": False},
        # a long budget of the 8B shape, sixteen requests
        {"name": "decode8-8b-long-batch16", "kind": "attention", "batch": 16, "kv_heads": 8,
         "groups": 4, "dim": 128, "length": 1, "cached": 18000, "spread": 4000, "page": 64,
         "dtype": "bf16", "ragged": False},
        # a few drafted tokens of the hybrid shape, checked in one call
        {"name": "draft8-hybrid-5", "kind": "attention", "batch": 3, "kv_heads": 4, "groups": 6,
         "dim": 256, "length": 5, "cached": 5000, "spread": 900, "page": 32, "dtype": "bf16",
         "ragged": False},
        # a further chunk of a long prompt onto a ragged, already evicted cache
        {"name": "prefill8-8b-chunk", "kind": "attention", "batch": 1, "kv_heads": 8, "groups": 4,
         "dim": 128, "length": 1500, "cached": 4000, "spread": 900, "page": 32, "dtype": "bf16",
         "ragged": False},
        # an eviction in all 16 layers of the 1B shape (a table of 16 x 8 segments)
        {"name": "compact8-1b-all-layers", "kind": "compact", "batch": 16, "kv_heads": 8,
         "dim": 64, "cached": 2000, "spread": 0, "removed": 200, "page": 32, "dtype": "bf16"},
        # an eviction in two layers of a long 8B cache
        {"name": "compact8-8b-long", "kind": "compact", "batch": 2, "kv_heads": 8, "dim": 128,
         "cached": 30000, "spread": 3000, "removed": 1000, "page": 64, "dtype": "bf16"},
        # one layer's rows for the audit's scoring
        {"name": "read8-8b", "kind": "read", "batch": 1, "kv_heads": 8, "dim": 128, "cached": 2000,
         "spread": 500, "page": 16, "dtype": "bf16"},
        # four layers of the hybrid shape, f16
        {"name": "read8-hybrid-f16", "kind": "read", "batch": 4, "kv_heads": 4, "dim": 256,
         "cached": 8000, "spread": 2000, "page": 32, "dtype": "f16"},
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["append", "append", "attention", "attention", "attention", "attention",
                       "attention", "compact", "read"])
    dim = rng.choice([64, 128, 128, 256])
    kv_heads, groups = {64: (8, 4), 128: (8, 4), 256: (4, 6)}[dim]
    if rng.random() < 0.4:
        groups = rng.choice([1, 2, 3, 5, 7, 8, 12, 16])
    case = {"kind": kind, "batch": rng.randint(1, 8), "kv_heads": kv_heads, "dim": dim,
            "page": rng.choice([16, 32, 64, 128, 256]), "dtype": rng.choice(["bf16", "bf16", "f16"])}
    if kind == "append":
        added = rng.choice([1, 1, _log_uniform(rng, 2, 4096)])
        if added > 512:
            case["batch"] = 1
        cached = rng.choice([0, _log_uniform(rng, 1, 2000)])
        if rng.random() < 0.2:
            case["dtype"] = "f32"
        case.update({"groups": min(groups, 8), "added": added, "cached": cached,
                     "spread": rng.randint(0, cached // 2),
                     "half": rng.choice([dim // 2, dim // 2, dim // 4, dim // 8]),
                     "ragged": case["batch"] > 1 and rng.random() < 0.5})
    elif kind == "attention":
        length = rng.choice([1, 1, 1, rng.randint(2, 24), _log_uniform(rng, 25, 1000)])
        cached = _log_uniform(rng, 1, 20000 if length == 1 else 4000)
        if length > 1:
            case["batch"] = rng.randint(1, 4 if length < 25 else 1 if length > 256 else 2)
        case.update({"groups": groups if length < 25 else min(groups, 6), "length": length,
                     "cached": cached, "spread": rng.randint(0, cached // 2),
                     "ragged": case["batch"] > 1 and length > 1 and rng.random() < 0.4})
    else:
        case["batch"] = min(case["batch"], 4)
        cached = _log_uniform(rng, 40, 9000)
        case.update({"cached": cached, "spread": rng.randint(0, cached // 3)})
        if kind == "compact":
            case["removed"] = rng.randint(1, cached // 2)
    return case


# ---- the page format, in elementary operations ------------------------------------------------

def _page_bytes(page, dim):
    return page * (2 * dim + 8)


def _sections(pages, page, dim):
    """Views of the pool: codes of keys [pages, blocks, dim / 16, 16, 16] and values [pages, blocks, 4,
    dim, 4], positions [pages, page], scales [pages, blocks, 2]."""
    blocks, wide = page // BLOCK, page * dim
    keys = pages[:, :wide].unflatten(1, (blocks, dim // 16, BLOCK, 16))
    values = pages[:, wide:2 * wide].unflatten(1, (blocks, 4, dim, 4))
    positions = pages.view(torch.float32)[:, wide // 2:wide // 2 + page]
    at = 2 * wide + 4 * page
    return keys, values, positions, pages[:, at:at + 2 * blocks].unflatten(1, (blocks, 2))


def _get_rows(sections, pid, slot):
    """Codes of the keys and values [..., dim] and positions of rows."""
    keys, values, positions, _ = sections
    block, row = slot // BLOCK, slot % BLOCK
    return (keys[pid, block, :, row].flatten(-2), values[pid, block, row // 4, :, row % 4],
            positions[pid, slot])


def _put_rows(sections, pid, slot, keys, values):
    block, row = slot // BLOCK, slot % BLOCK
    sections[0][pid, block, :, row] = keys.unflatten(-1, (-1, 16))
    sections[1][pid, block, row // 4, :, row % 4] = values


def _exponent(amax, f16):
    """log2 of the scale for a block whose largest finite magnitude is amax (f32)."""
    exponent = ((amax.view(torch.int32) + 0x180000) >> 23) - 127 - 8
    return exponent.clamp(-117, 7 if f16 else 119)


def _encode(units):
    """Magnitude codes of whole numbers of the smallest code."""
    units = units.clamp(max=229376)  # 448 of 2^-9
    top = torch.frexp(units.double())[1] - 1  # of the highest bit
    normal = ((top - 2) << 3) | ((units >> (top - 3).clamp(min=0)) & 7)
    return torch.where(units < 8, units, normal)


def _quantise(x, exponent):
    """Codes of f32 elements at scale 2^exponent (broadcast)."""
    finite = torch.isfinite(x)
    bits = torch.where(finite, x, torch.zeros_like(x)).view(torch.int32) & 0x7fffffff
    bits = (bits + 0x7ffff + ((bits >> 20) & 1)) & ~0xfffff  # four significant bits
    # (a carry to 2^128 is past every scale)
    size = torch.where(bits == 0x7f800000, torch.full_like(x, 2.0 ** 100).double() * 2.0 ** 28,
                       bits.view(torch.float32).double())
    units = torch.ldexp(size, 9 - exponent).clamp(max=1e9).to(torch.int32)
    code = torch.where(finite, _encode(units), torch.full_like(units, 127))
    return (code + 128 * torch.signbit(x)).to(torch.uint8)


def _shift(codes, by):
    """Codes at a scale 2^by times theirs."""
    size = (codes & 127).to(torch.int32)
    units = torch.where(size < 8, size, (8 + (size & 7)) << ((size >> 3) - 1).clamp(min=0))
    moved = _encode(units >> by.clamp(max=31))
    return (torch.where(size == 127, size, moved) + (codes & 128)).to(torch.uint8)


def _values(codes, exponent):
    """f32 rows of codes at scale 2^exponent (broadcast)."""
    size = (codes & 127).to(torch.int32)
    units = torch.where(size < 8, size, (8 + (size & 7)) << ((size >> 3) - 1).clamp(min=0))
    value = torch.ldexp(units.float(), exponent - 9)
    value = torch.where(size == 127, torch.full_like(value, math.nan), value)
    return torch.where(codes >= 128, -value, value)


def _where(table, lengths, page, most):
    """Page and slot of rows 0 .. most - 1 of every segment, and which rows a segment has."""
    row = torch.arange(most, device=table.device)
    held = row[None, :] < lengths[:, None]
    pid = table[:, row // page].long()
    return torch.where(held, pid, torch.zeros_like(pid)), (row % page).expand_as(pid), held


def _row_exponents(sections, pid, slot):
    """Exponents of the keys' and values' scales of rows' blocks."""
    scales = sections[3][pid, slot // BLOCK].to(torch.int32) - 127
    return scales[..., 0], scales[..., 1]


def _plain_rows(pages, table, lengths, page, dim, most):
    """f32 keys and values [segments, most, dim], positions [segments, most], held."""
    pid, slot, held = _where(table, lengths, page, most)
    sections = _sections(pages, page, dim)
    keys, values, positions = _get_rows(sections, pid, slot)
    ek, ev = _row_exponents(sections, pid, slot)
    return _values(keys, ek.unsqueeze(-1)), _values(values, ev.unsqueeze(-1)), positions, held


def _plain_read(pages, table, lengths, page, dim, most, dtype):
    keys, values, positions, held = _plain_rows(pages, table, lengths, page, dim, most)
    return {"keys": keys[held].to(dtype), "values": values[held].to(dtype),
            "positions": positions[held].unsqueeze(-1),
            "cumulative": torch.cat((lengths.new_zeros(1), lengths.cumsum(0))).to(torch.int32)}


def _rotate(x, cos, sin):
    """The first 2 x half channels in pairs (i, i + half); x f32 [batch, heads, rows, dim], the
    tables [batch, rows, half]."""
    half = cos.shape[-1]
    c, s = cos.unsqueeze(1), sin.unsqueeze(1)
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat((a * c - b * s, b * c + a * s, x[..., 2 * half:]), -1)


def _store(pages, table, lengths, page, dim, keys, values, positions, fresh, f16):
    """Stores the `fresh` rows of [segments, rows, dim] (f32; the first ones of each segment) behind
    the segments' rows."""
    sections = _sections(pages, page, dim)
    segments, count = fresh.shape
    first = torch.div(lengths, BLOCK, rounding_mode="floor").long() * BLOCK
    offset = lengths.long() - first
    # the touched blocks, densely: row i of them is row i - offset of the new ones
    blocks = (count + 2 * BLOCK - 2) // BLOCK
    row = torch.arange(blocks * BLOCK, device=pages.device)
    source = row[None, :] - offset[:, None]
    inside = (source >= 0) & (source < count)
    source = source.clamp(0, max(count - 1, 0))
    segment = torch.arange(segments, device=pages.device)[:, None].expand_as(source)
    new = inside & fresh[segment, source]
    old = (row[None, :] < offset[:, None]) & fresh[:, :1]
    at = torch.where(new | old, first[:, None] + row, torch.zeros_like(source))
    pid = table[segment, at // page].long()
    slot = at % page
    pid, slot = torch.where(new | old, pid, torch.zeros_like(pid)), torch.where(new | old, slot, 0)
    stored = _get_rows(sections, pid, slot)[:2]
    scales = _row_exponents(sections, pid, slot)
    out, exponents = [], []
    for x, codes, was in ((keys, stored[0], scales[0]), (values, stored[1], scales[1])):
        x = x[segment, source]
        size = torch.where(new.unsqueeze(-1) & torch.isfinite(x), x, torch.zeros_like(x)).abs()
        exponent = _exponent(size.amax(-1).unflatten(1, (blocks, BLOCK)).amax(-1), f16)
        exponent = exponent.repeat_interleave(BLOCK, 1)
        # the rows that are there already, all of the first block
        before = torch.where((offset[:, None] > 0) & (row[None, :] < BLOCK),
                             was[:, :1].expand_as(was), torch.full_like(was, -127))
        exponent = torch.maximum(exponent, before)
        moved = _shift(codes, (exponent - was).clamp(min=0).unsqueeze(-1))
        out.append(torch.where(new.unsqueeze(-1), _quantise(x, exponent.unsqueeze(-1)), moved))
        exponents.append(exponent)
    touched = new | old
    pid, slot = pid[touched], slot[touched]
    _put_rows(sections, pid, slot, out[0][touched], out[1][touched])
    for which in range(2):
        sections[3][pid, slot // BLOCK, which] = (exponents[which][touched] + 127).to(torch.uint8)
    number = source[new]
    pid, slot = table[segment[new], at[new] // page].long(), at[new] % page
    sections[2][pid, slot] = positions[segment[new], number]


# ---- cases ------------------------------------------------------------------------------------

def prepare(case, seed):
    c, g = case, torch.Generator(device=DEVICE).manual_seed(seed)
    host = np.random.default_rng(seed)
    dim, page, dtype = c["dim"], c["page"], DTYPES[c["dtype"]]
    segments = c["batch"] * c["kv_heads"]
    # the layout goes with the case, so that a case's outputs have one shape
    layout = np.random.default_rng([c["cached"], c["spread"], c["batch"], c["kv_heads"], 8])
    lengths = c["cached"] + layout.integers(0, c["spread"] + 1, segments)
    new = c.get("added", c["length"] if c["kind"] == "attention" else 0)
    counts = np.full(c["batch"], new)
    if c.get("ragged"):
        counts = layout.integers(0, new + 1, c["batch"])
    grown = lengths + np.repeat(counts, c["kv_heads"])
    removed_counts = (np.minimum(c["removed"], lengths) if c["kind"] == "compact"
                      else np.zeros(segments, np.int64))
    most = int(grown.max())
    per = -(-max(most, 1) // page)
    used = -(-grown // page)
    extra = -(-(lengths - removed_counts) // page) if c["kind"] == "compact" else 0 * used
    # pages in any order, as a pool that has been used hands them out; what no row has been
    # stored in holds anything
    total_pages = int(used.sum() + extra.sum()) + 3
    order = host.permutation(total_pages)
    table = np.zeros((segments, per), np.int32)
    table[np.arange(per)[None, :] < used[:, None]] = order[:used.sum()]
    pages = torch.randint(0, 256, (total_pages, _page_bytes(page, dim)), generator=g,
                          dtype=torch.uint8, device=DEVICE)
    put = lambda a, t: torch.from_numpy(np.ascontiguousarray(a)).to(DEVICE, t)  # noqa: E731
    state = {"case": dict(c), "pages": pages, "table": put(table, torch.int32),
             "lengths": put(lengths, torch.int32), "grown": put(grown, torch.int32),
             "counts": put(counts, torch.int32) if c.get("ragged") else None,
             "most": most, "total": int(grown.sum())}
    randn = lambda *shape: torch.randn(shape, generator=g, device=DEVICE)  # noqa: E731
    # a few channels of the keys are large, and so are a few of the values' rows
    channels = 1.0 + 5.0 * (torch.rand(dim, generator=g, device=DEVICE) < 0.04)

    def key_rows(*shape):
        return randn(*shape, dim) * channels

    def value_rows(*shape):
        return randn(*shape, dim) * torch.exp(0.7 * randn(*shape, 1))

    # the rows in the cache: all that the case reads (an attention call's new rows are stored)
    stored = put(grown if c["kind"] == "attention" else lengths, torch.int64)
    longest = int(stored.max())
    step = max(1, 2 ** 25 // max(longest * dim, 1))  # segments at a time, to bound the memory
    for at in range(0, segments if longest else 0, step):
        n = stored[at:at + step]
        row = torch.arange(longest, device=DEVICE)
        _store(pages, state["table"][at:at + step], torch.zeros_like(n), page, dim,
               key_rows(len(n), longest), value_rows(len(n), longest),
               row.float().expand(len(n), longest), row[None, :] < n[:, None],
               dtype == torch.float16)
    if c["kind"] in ("append", "attention"):
        heads = c["kv_heads"] * c["groups"]
        # as a model hands them over: [batch, heads, rows, dim] views of [batch, rows, heads, dim]
        state["queries"] = randn(c["batch"], new, heads, dim).to(dtype).transpose(1, 2)
    if c["kind"] == "append":
        state["keys"] = key_rows(c["batch"], new, c["kv_heads"]).to(dtype).transpose(1, 2)
        state["values"] = value_rows(c["batch"], new, c["kv_heads"]).to(dtype).transpose(1, 2)
        first = torch.randint(0, 5000, (c["batch"], 1), generator=g, device=DEVICE)
        state["positions"] = first + torch.arange(new, device=DEVICE)[None, :]
        angle = (torch.arange(5000 + new, device=DEVICE, dtype=torch.float64)[:, None]
                 * 500000.0 ** -(torch.arange(c["half"], device=DEVICE, dtype=torch.float64)
                                 / c["half"])[None, :])
        state["rotary"] = (angle.cos().float(), angle.sin().float())
    if c["kind"] == "compact":
        starts = np.concatenate([[0], np.cumsum(lengths)])
        state["removed"] = put(np.concatenate(
            [starts[s] + np.sort(host.choice(lengths[s], removed_counts[s], replace=False))
             for s in range(segments)]), torch.int64)
        kept = lengths - removed_counts
        target = np.zeros((segments, per), np.int32)
        target[np.arange(per)[None, :] < extra[:, None]] = order[used.sum():used.sum() + extra.sum()]
        state["target"] = put(target, torch.int32)
        state["total"] = int(kept.sum())
    if own:
        from code_for_iclr27_amd import paged
        state["layer"] = paged.PagedLayer(pages, state["table"], state["lengths"], c["kv_heads"],
                                          dim, page, bits=8)
        state["grown_layer"] = state["layer"].with_lengths(state["grown"])
    return state


def run(state):
    return _own(state) if own else _plain(state)


def _own(state):
    from code_for_iclr27_amd import paged
    c, kind = state["case"], state["case"]["kind"]
    dtype, layer = DTYPES[c["dtype"]], state["layer"]
    out = {}
    if kind == "attention":
        return paged.attention(layer, state["queries"], state["most"], counts=state["counts"])
    if kind == "append":
        out["queries"] = paged.append(layer, state["keys"], state["values"], state["positions"],
                                      rotary=state["rotary"], queries=state["queries"],
                                      counts=state["counts"])
        layer = state["grown_layer"]
    elif kind == "compact":
        layer = paged.compact(layer, state["removed"], state["target"])
        out["lengths"] = layer.lengths
    keys, values, positions, cumulative = paged.read(layer, state["total"], dtype)
    return {**out, "keys": keys, "values": values, "positions": positions,
            "cumulative": cumulative}


def _plain(state):
    c, kind = state["case"], state["case"]["kind"]
    dim, page, dtype = c["dim"], c["page"], DTYPES[c["dtype"]]
    pages, table, lengths = state["pages"], state["table"], state["lengths"]
    out = {}
    if kind == "attention":
        return _plain_attention(state)
    if kind == "append":
        cos, sin = (t[state["positions"]] for t in state["rotary"])
        out["queries"] = _rotate(state["queries"].float(), cos, sin).to(dtype)
        keys, values = _rotate(state["keys"].float(), cos, sin), state["values"].float()
        batch, heads, added, _ = keys.shape
        row = torch.arange(added, device=keys.device)
        fresh = row < (state["counts"][:, None] if c["ragged"] else added)
        fresh = fresh.reshape(-1, 1, added).expand(batch, heads, added).flatten(0, 1)
        positions = state["positions"].float()[:, None, :].expand(batch, heads, added)
        _store(pages, table, lengths, page, dim, keys.flatten(0, 1), values.flatten(0, 1),
               positions.flatten(0, 1), fresh, dtype == torch.float16)
        lengths = state["grown"]
    elif kind == "compact":
        table, lengths = state["target"], _plain_compact(state)
        out["lengths"] = lengths
    return {**out, **_plain_read(pages, table, lengths, page, dim, state["most"], dtype)}


def _plain_compact(state):
    dim, page, most = state["case"]["dim"], state["case"]["page"], state["most"]
    pages, table, lengths = state["pages"], state["table"], state["lengths"]
    pid, slot, held = _where(table, lengths, page, most)
    starts = torch.cat((lengths.new_zeros(1), lengths.cumsum(0)))[:-1]
    number = starts[:, None] + torch.arange(most, device=held.device)
    gone = torch.zeros(held.numel() + 1, dtype=torch.bool, device=held.device)
    gone[state["removed"]] = True
    keep = held & ~gone[torch.where(held, number, torch.full_like(number, held.numel()))]
    to = (keep.cumsum(1) - 1)[keep]
    segment = torch.arange(held.shape[0], device=held.device)[:, None].expand_as(held)[keep]
    sections = _sections(pages, page, dim)
    keys, values, positions = _get_rows(sections, pid[keep], slot[keep])
    blocks = -(-most // BLOCK)
    place = segment * blocks + to // BLOCK
    moved, scales = [], []
    for codes, was in zip((keys, values), _row_exponents(sections, pid[keep], slot[keep])):
        largest = torch.full((held.shape[0] * blocks,), -127, dtype=torch.int32, device=was.device)
        largest = largest.scatter_reduce(0, place, was, "amax")[place]
        moved.append(_shift(codes, (largest - was).unsqueeze(-1)))
        scales.append((largest + 127).to(torch.uint8))
    target, at = state["target"][segment, to // page].long(), to % page
    _put_rows(sections, target, at, *moved)
    sections[2][target, at] = positions
    sections[3][target, at // BLOCK] = torch.stack(scales, -1)
    return keep.sum(1).to(torch.int32)


def _plain_attention(state):
    c = state["case"]
    dim, page, dtype = c["dim"], c["page"], DTYPES[c["dtype"]]
    batch, heads, groups, length = c["batch"], c["kv_heads"], c["groups"], c["length"]
    keys, values, _, held = _plain_rows(state["pages"], state["table"], state["grown"], page, dim,
                                        state["most"])
    keys = torch.where(held.unsqueeze(-1), keys, torch.zeros_like(keys))
    values = torch.where(held.unsqueeze(-1), values, torch.zeros_like(values))
    q = state["queries"].float().reshape(batch * heads, groups * length, dim)
    scores = torch.matmul(q, keys.transpose(1, 2)) * dim ** -0.5
    query = torch.arange(length, device=q.device)
    last = state["lengths"][:, None] + query  # the last key a query sees
    seen = torch.arange(state["most"], device=q.device) <= last.unsqueeze(-1)
    if c["ragged"]:
        seen &= (query < state["counts"].repeat_interleave(heads)[:, None]).unsqueeze(-1)
    seen = seen.unsqueeze(1)
    scores = scores.reshape(batch * heads, groups, length, -1)
    scores = torch.where(seen, scores, torch.full_like(scores, -math.inf))
    top = scores.amax(-1, keepdim=True)
    weight = torch.exp(scores - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    weight = torch.where(seen, weight, torch.zeros_like(weight))
    total = weight.sum(-1, keepdim=True)
    result = torch.matmul(weight.flatten(1, 2), values).reshape(weight.shape[:3] + (dim,))
    result = result / torch.where(total > 0, total, torch.ones_like(total))
    result = result.reshape(batch, heads * groups, length, dim).transpose(1, 2)
    return result.reshape(batch, length, heads * groups * dim).to(dtype)


# ---- what a pass cannot do without ------------------------------------------------------------

def work(case):
    c = case
    segments, dim = c["batch"] * c["kv_heads"], c["dim"]
    cached = c["cached"] + c["spread"] / 2
    size = 4 if c["dtype"] == "f32" else 2
    row, wide = 2 * dim + 2 / BLOCK, 2 * size * dim  # K and V of a row, as codes and as elements
    if c["kind"] == "attention":
        share = 0.5 if c["ragged"] else 1.0  # of the queries, on average
        queries = segments * c["groups"] * c["length"]
        pairs = queries * share * (cached + share * c["length"] / 2 + 0.5)
        return {"bytes": segments * (cached + share * c["length"]) * row + 2 * queries * dim * 2,
                "flops": 4.0 * dim * pairs}
    if c["kind"] == "append":
        share = 0.5 if c["ragged"] else 1.0
        new = segments * c["added"] * share
        queries = segments * c["groups"] * c["added"]
        rows = segments * cached + new
        return {"bytes": new * (wide + row + 4) + 2 * queries * dim * size
                + segments * cached * (row + 4) + rows * (wide + 4),
                "flops": 3.0 * 2 * c["half"] * (queries + new)}
    kept = segments * (cached - c.get("removed", 0))
    moved = kept * (row + 4) if c["kind"] == "compact" else 0.0  # the new pages
    return {"bytes": moved + kept * (row + 4) + kept * (wide + 4), "flops": 0.0}


# ---- the definition in 64 bits ----------------------------------------------------------------

def _magnitudes():
    """The 127 magnitudes of the codes and NaN, from the format's definition."""
    sizes = [m * 2.0 ** -9 for m in range(8)]
    sizes += [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)]
    sizes[127] = math.nan
    return torch.tensor(sizes + [-v for v in sizes], dtype=torch.float64, device=DEVICE)


def _exact_rows(state, segment, table, count):
    """f64 keys, values and positions of one segment's first `count` rows, and the scales of its blocks
    [blocks, 2]."""
    page, dim = state["case"]["page"], state["case"]["dim"]
    raw = state["pages"][table[segment, :-(-count // page)].long()]
    lut, wide = _magnitudes(), page * dim
    keys = lut[raw[:, :wide].long()].reshape(-1, dim // 16, 16, 16).permute(0, 2, 1, 3)
    values = lut[raw[:, wide:2 * wide].long()].reshape(-1, 4, dim, 4).permute(0, 1, 3, 2)
    tail = raw[:, 2 * wide:2 * wide + 4 * page].contiguous().view(torch.float32).double().reshape(-1)
    scales = raw[:, 2 * wide + 4 * page:][:, :page // 8].reshape(-1, 2)
    power = 2.0 ** (scales.double() - 127.0)
    rows = [(x.reshape(-1, 16, dim) * power[:, i].reshape(-1, 1, 1)).reshape(-1, dim)[:count]
            for i, x in enumerate((keys, values))]
    return rows[0], rows[1], tail[:count], power[:-(-count // 16)]


def _exact_power(amax, f16):
    """The smallest power of two whose codes hold amax, with rounding: 2^e with amax < 464 2^e."""
    power = torch.exp2(torch.ceil(torch.log2(amax.clamp(min=2.0 ** -140) / 464.0)))
    power = torch.where(amax >= 464.0 * power, 2 * power, power)
    power = torch.where(amax < 232.0 * power, power / 2, power)
    return power.clamp(2.0 ** -117, 2.0 ** (7 if f16 else 119))


def _exact_round(rows, power):
    """What E4M3 codes at scale `power` make of f64 rows: four significant bits, rounded to even,
    cut at 2^-9."""
    significand, exponent = torch.frexp(rows)
    four = torch.round(significand * 16) * torch.exp2((exponent - 4).double())
    codes = torch.trunc(four / (power * 2.0 ** -9)) * (power * 2.0 ** -9)
    return torch.minimum(torch.maximum(codes, -448.0 * power), 448.0 * power)


def exact(case, seed):
    state = prepare(case, seed)
    c, kind = case, case["kind"]
    dim, f16 = c["dim"], c["dtype"] == "f16"
    heads, segments = c["kv_heads"], c["batch"] * c["kv_heads"]
    lengths, grown = state["lengths"].tolist(), state["grown"].tolist()
    if kind == "attention":
        groups, length = c["groups"], c["length"]
        out = torch.zeros(c["batch"], length, heads * groups, dim, dtype=torch.float64,
                          device=DEVICE)
        for s in range(segments):
            b, h = divmod(s, heads)
            keys, values = _exact_rows(state, s, state["table"], grown[s])[:2]
            for i in range(0, grown[s] - lengths[s], 64):
                n = min(64, grown[s] - lengths[s] - i)
                q = state["queries"][b, h * groups:(h + 1) * groups, i:i + n].double()
                logits = torch.matmul(q, keys.T) / math.sqrt(dim)
                ends = lengths[s] + i + torch.arange(n, device=DEVICE)
                hidden = torch.arange(grown[s], device=DEVICE)[None, :] > ends[:, None]
                p = torch.softmax(logits.masked_fill(hidden, -math.inf), -1)
                out[b, i:i + n, h * groups:(h + 1) * groups] = torch.matmul(p, values).transpose(0, 1)
        return out.reshape(c["batch"], length, -1)
    result, parts = {}, []
    if kind == "append":
        at = state["positions"]
        cos, sin = (t.double()[at][:, None] for t in state["rotary"])
        half = c["half"]

        def turned(x):
            x = x.double().clone()
            a, b = x[..., :half].clone(), x[..., half:2 * half].clone()
            x[..., :half], x[..., half:2 * half] = a * cos - b * sin, a * sin + b * cos
            return x

        result["queries"] = turned(state["queries"])
        fresh = turned(state["keys"]), state["values"].double()

    def blockwise(x, fill=0.0):
        """[blocks, 16, dim] of rows."""
        pad = -x.shape[0] % 16
        return torch.cat((x, x.new_full((pad, x.shape[1]), fill))).reshape(-1, 16, x.shape[1])

    for s in range(segments):
        b, h = divmod(s, heads)
        keys, values, positions, power = _exact_rows(state, s, state["table"], lengths[s])
        if kind == "append":
            n, sides = grown[s] - lengths[s], []
            for which, (old, new) in enumerate(((keys, fresh[0][b, h, :n]),
                                                (values, fresh[1][b, h, :n]))):
                rows = blockwise(torch.cat((old, new)))
                late = blockwise(torch.cat((torch.zeros_like(old), new)))
                scale = _exact_power(late.abs().amax((1, 2)), f16)
                before = torch.zeros_like(scale)
                before[:len(power)] = power[:, which]
                whole = torch.arange(len(scale), device=DEVICE) < lengths[s] // 16
                scale = torch.where(whole if n else before > 0, before, torch.maximum(scale, before))
                sides.append(_exact_round(rows, scale[:, None, None]).reshape(-1, dim)[:grown[s]])
            keys, values = sides
            positions = torch.cat((positions, state["positions"][b, :n].double()))
        if kind == "compact":
            first = sum(lengths[:s])
            mine = state["removed"][(state["removed"] >= first)
                                    & (state["removed"] < first + lengths[s])] - first
            keep = torch.ones(lengths[s], dtype=torch.bool, device=DEVICE)
            keep[mine] = False
            sides = []
            for which, rows in enumerate((keys, values)):
                scale = power[:, which].repeat_interleave(16)[:lengths[s]][keep]
                scale = blockwise(scale[:, None])[..., 0].amax(1)
                sides.append(_exact_round(blockwise(rows[keep]), scale[:, None, None])
                             .reshape(-1, dim)[:int(keep.sum())])
            keys, values = sides
            positions = positions[keep]
        parts.append((keys, values, positions))
    result["keys"], result["values"] = (torch.cat([p[i] for p in parts]) for i in (0, 1))
    result["positions"] = torch.cat([p[2] for p in parts]).unsqueeze(-1)
    if kind == "compact":
        result["lengths"] = torch.tensor([len(p[0]) for p in parts], dtype=torch.int32,
                                         device=DEVICE)
    sizes = torch.tensor([0] + [len(p[0]) for p in parts], device=DEVICE)
    result["cumulative"] = sizes.cumsum(0).to(torch.int32)
    return result
