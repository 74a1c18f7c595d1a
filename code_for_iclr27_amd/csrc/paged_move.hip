// Rows into, out of and within the paged 4-bit KV cache (paged.hpp states its layout).
//
// append: new K and V rows behind each segment's rows, K (and the step's queries) rotated to their
// positions on the way. The rotation pairs channels c and c + half; its products are rounded one by
// one (no fused multiply-add), in f32. Four threads with eight channels each share a block of 32: its
// largest magnitude goes round them in the vector ALU, the scale is the largest power of two X with
// 4 X <= amax, doubled where amax >= 7 X (so that no element loses more to saturation than to
// rounding), and the conversion instruction rounds to the nearest code, ties to even, and saturates.
// Bound by memory: 8,192 tokens of 8 KV and 32 query heads, d128, 177 MB in 36 us (4.9 TB/s; a large
// copy reaches 5.2); a step of eight requests 3.4 us, the time of its chain of loads.
//
// read: the rows as 16- or 32-bit rows packed by segment, the layout of the other operators, with
// its cumulative lengths. Bound by memory: 155,000 rows of d256 as f16, 203 MB in 46.6 us (4.4 TB/s;
// 78 with D / 8 threads a row that each searched for its segment); 19,000 rows of d128 5.9 us.
//
// compact: the rows that stay, in order, into other pages, in one launch. A wave has a chain of about ten
// dependent loads (the lengths, the searches, the tables) ahead of its copies, then reads all of its
// rows and writes them; as nearly all workgroups are resident at once, reads and writes hardly overlap.
// 537,000 rows of d128, 150 MB read and written in 51 us (3.0 TB/s; 35 with the same chain where the
// last-level cache holds them), 256,000 of d64 12.5 us. Two 64-row rounds a wave, one after the other
// (one round of workgroups instead of one and a bit), and non-temporal accesses are no faster with the
// read that follows.

#include "paged_move.hpp"

namespace lr {

int check_paged(const void* pages, int64_t page_count, int64_t page_size, int64_t dim,
                const int32_t* table, int64_t max_pages, const int32_t* lengths,
                int64_t segments) {
  LR_REQUIRE(dim == 64 || dim == 128 || dim == 256, "Head dimension must be 64, 128 or 256");
  LR_REQUIRE(paged_bytes(page_size, dim) > 0, "Page size must be 16, 32, 64, 128 or 256");
  LR_REQUIRE(segments > 0 && segments <= INT32_MAX && page_count >= 0 && max_pages >= 0 &&
                 page_count <= INT32_MAX,
             "Invalid page table");
  LR_REQUIRE(max_pages <= INT32_MAX / 2 / page_size, "A segment holds fewer than 2^30 rows");
  LR_REQUIRE(lengths && (table || max_pages == 0) && (pages || page_count == 0),
             "Invalid page table");
  LR_REQUIRE(reinterpret_cast<uintptr_t>(pages) % 16 == 0, "Pages must be 16-byte aligned");
  return LR_OK;
}

namespace {

template <int BIT>
__device__ __forceinline__ float quad_max(float x) {
  return fmaxf(x, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(
                      0, __builtin_bit_cast(int, x), BIT == 0 ? 0xB1 : 0x4E, 0xF, 0xF, false)));
}

// Eight of a block's elements as codes, with the block's scale byte; four consecutive lanes call it
// with the block's elements.
struct Quantised {
  unsigned codes, scale;
};
__device__ __forceinline__ Quantised quantise(const float (&x)[8], ScaleRange range) {
  float top = 0.0f, sum = 0.0f;  // sum: NaN if an element is not finite
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    top = fmaxf(top, __builtin_fabsf(x[e]));
    sum = __builtin_fmaf(x[e], 0.0f, sum);
  }
  top = sum == sum ? top : __builtin_huge_valf();
  top = quad_max<1>(quad_max<0>(top));
  const bool finite = top < __builtin_huge_valf();
  // 2^(floor(log2 top) - 2), one more where the significand is at least 1.75 (a carry into the exponent)
  int exponent = static_cast<int>((__builtin_bit_cast(unsigned, top) + 0x200000u) >> 23) - 129;
  exponent = exponent < range.low ? range.low : exponent > range.high ? range.high : exponent;
  const unsigned byte = finite ? static_cast<unsigned>(exponent + 127) : kScaleNaN;
  const float scale = scale_of(finite ? byte : 127u);
  unsigned codes = 0;
  if (finite) {
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[0], x[1], scale, 0);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[2], x[3], scale, 1);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[4], x[5], scale, 2);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[6], x[7], scale, 3);
  }
  return {codes, byte};
}

// The page of row lengths[segment] + i, and its slot; NULL where there is none.
struct Spot {
  uint8_t* page;
  int slot;
};
template <int D>
__device__ __forceinline__ Spot new_row(const PagedCache& cache, int64_t segment, unsigned i) {
  const int n = cache.lengths[segment];
  const int64_t at = static_cast<int64_t>(n) + i;
  if (n < 0 || at >= static_cast<int64_t>(cache.max_pages) << cache.shift) return {nullptr, 0};
  const int64_t id = cache.table[segment * cache.max_pages + (at >> cache.shift)];
  if (id < 0 || id >= cache.page_count) return {nullptr, 0};
  return {cache.pages + id * (Page<D>::bytes(1) << cache.shift),
          static_cast<int>(at) & ((1 << cache.shift) - 1)};
}

// Chunk c (eight channels) of a K (what 0) or V (1) row.
template <int D>
__device__ __forceinline__ void store_eight(const PagedCache& cache, const Spot& spot, int what, int c,
                                            const Quantised& q) {
  *reinterpret_cast<unsigned*>(spot.page + Page<D>::codes(cache.shift, what, spot.slot) + 4 * c) = q.codes;
  if (c % 4 == 0)
    spot.page[Page<D>::scales(cache.shift, what, spot.slot) + c / 4] = static_cast<uint8_t>(q.scale);
}
template <int D>
__device__ __forceinline__ void store_position(const PagedCache& cache, const Spot& spot, int64_t position) {
  *reinterpret_cast<float*>(spot.page + Page<D>::position(cache.shift, spot.slot)) =
      static_cast<float>(position);
}

template <typename T, int D>
__global__ __launch_bounds__(kThreads) void paged_append_kernel(AppendArgs a) {
  constexpr int kRowThreads = D / 8, kRowsPerBlock = kThreads / kRowThreads;
  // blocks: the keys', the values', the queries'
  const int what = blockIdx.x < a.kv_blocks ? 0 : blockIdx.x < 2 * a.kv_blocks ? 1 : 2;
  const unsigned block = blockIdx.x - what * a.kv_blocks;
  const unsigned row = block * kRowsPerBlock + threadIdx.x / kRowThreads;
  const int c = threadIdx.x % kRowThreads;
  // whole quads are in or out: the exchanges below stay within a row
  if (row >= (what == 2 ? a.query_rows : a.kv_rows)) return;
  const unsigned heads = what == 2 ? a.query_heads : a.kv_heads;
  const unsigned segment = row / a.added, i = row - segment * a.added;
  const unsigned b = segment / heads, h = segment - b * heads;
  if (what != 2 && a.counts != nullptr && static_cast<int64_t>(i) >= a.counts[b]) return;

  const Rows& rows = what == 0 ? a.keys : what == 1 ? a.values : a.queries;
  const T* source = static_cast<const T*>(rows.base) + b * rows.batch + h * rows.head + i * rows.row;
  float x[8];
  const Eight<T> mine = *reinterpret_cast<const Eight<T>*>(source + 8 * c);
  mine.get(x);
  const int64_t position = a.positions[static_cast<int64_t>(b) * a.added + i];
  if (what != 1 && 8 * c < 2 * a.half) {
    const bool first = 8 * c < a.half;
    float y[8], cosine[8], sine[8];
    const Eight<T> partner =
        *reinterpret_cast<const Eight<T>*>(source + (first ? 8 * c + a.half : 8 * c - a.half));
    partner.get(y);
    const bool known = position >= 0 && position < a.table_rows;
    const int64_t at = (known ? position : 0) * a.half + (first ? 8 * c : 8 * c - a.half);
    reinterpret_cast<const Eight<float>*>(a.cos + at)->get(cosine);
    reinterpret_cast<const Eight<float>*>(a.sin + at)->get(sine);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float p = x[e] * cosine[e], q = y[e] * sine[e];
      x[e] = known ? (first ? p - q : p + q) : __builtin_nanf("");
    }
  }
  if (what == 2) {
    Eight<T> result;
    result.set(x);
    *reinterpret_cast<Eight<T>*>(static_cast<T*>(a.out_queries) + static_cast<int64_t>(row) * D +
                                 8 * c) = result;
    return;
  }

  const Quantised q = quantise(x, a.range);
  const Spot spot = new_row<D>(a.cache, segment, i);
  if (spot.page == nullptr) return;
  store_eight<D>(a.cache, spot, what, c, q);
  if (what == 0 && c == 0) store_position<D>(a.cache, spot, position);
}

// The same where whole blocks are rotated (half a multiple of 32): D / 16 threads a row, each with a
// chunk and its partner (rotated: channels c and c + half; the others: half of them apart), so that
// a cosine and sine are loaded once for both, and for the same chunks of HEADS heads, whose loads
// are in flight together.
template <typename T, int D, int HEADS>
__global__ __launch_bounds__(kThreads) void paged_append_pairs_kernel(AppendArgs a) {
  constexpr int kRowThreads = D / 16, kUnits = kThreads / kRowThreads;
  const int what = blockIdx.x < a.kv_blocks ? 0 : blockIdx.x < 2 * a.kv_blocks ? 1 : 2;
  const unsigned unit = (blockIdx.x - what * a.kv_blocks) * kUnits + threadIdx.x / kRowThreads;
  const unsigned heads = what == 2 ? a.query_heads : a.kv_heads;
  const unsigned head_groups = (heads + HEADS - 1) / HEADS;
  const unsigned place = unit / head_groups, h0 = (unit - place * head_groups) * HEADS;
  const unsigned b = place / a.added, i = place - b * a.added;
  if (b >= a.batch) return;  // whole rows are in or out: the exchanges below stay within a row
  if (what != 2 && a.counts != nullptr && static_cast<int64_t>(i) >= a.counts[b]) return;
  const int t = threadIdx.x % kRowThreads, pairs = what == 1 ? 0 : a.half / 8;
  const bool rotated = t < pairs;
  const int lo = rotated ? t : t + pairs, hi = lo + (rotated ? pairs : D / 16 - pairs);

  const Rows& rows = what == 0 ? a.keys : what == 1 ? a.values : a.queries;
  const T* source = static_cast<const T*>(rows.base) + b * rows.batch + i * rows.row;
  Eight<T> first[HEADS], second[HEADS];
#pragma unroll
  for (int n = 0; n < HEADS; ++n) {
    const T* p = source + min(h0 + n, heads - 1) * rows.head;
    first[n] = *reinterpret_cast<const Eight<T>*>(p + 8 * lo);
    second[n] = *reinterpret_cast<const Eight<T>*>(p + 8 * hi);
  }
  const int64_t position = what == 1 ? 0 : a.positions[static_cast<int64_t>(b) * a.added + i];
  const bool known = position >= 0 && position < a.table_rows;
  float cosine[8], sine[8];
  if (rotated) {
    const int64_t at = (known ? position : 0) * a.half + 8 * t;
    reinterpret_cast<const Eight<float>*>(a.cos + at)->get(cosine);
    reinterpret_cast<const Eight<float>*>(a.sin + at)->get(sine);
  }
#pragma unroll
  for (int n = 0; n < HEADS; ++n) {
    if (h0 + n >= heads) break;
    float x[8], y[8];
    first[n].get(x);
    second[n].get(y);
    if (rotated) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float xc = x[e] * cosine[e], ys = y[e] * sine[e], yc = y[e] * cosine[e], xs = x[e] * sine[e];
        x[e] = known ? xc - ys : __builtin_nanf("");
        y[e] = known ? yc + xs : __builtin_nanf("");
      }
    }
    if (what == 2) {
      T* out = static_cast<T*>(a.out_queries) +
               ((static_cast<int64_t>(b) * heads + h0 + n) * a.added + i) * D;
      Eight<T> result;
      result.set(x);
      *reinterpret_cast<Eight<T>*>(out + 8 * lo) = result;
      result.set(y);
      *reinterpret_cast<Eight<T>*>(out + 8 * hi) = result;
      continue;
    }
    const Quantised p = quantise(x, a.range), q = quantise(y, a.range);
    const Spot spot = new_row<D>(a.cache, static_cast<int64_t>(b) * heads + h0 + n, i);
    if (spot.page == nullptr) continue;
    store_eight<D>(a.cache, spot, what, lo, p);
    store_eight<D>(a.cache, spot, what, hi, q);
    if (what == 0 && t == 0) store_position<D>(a.cache, spot, position);
  }
}

// ---------------------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ Eight<T> eight_values(unsigned codes, float scale) {
  if constexpr (std::is_same<T, float>::value) {
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 0);
    const auto b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 1);
    const auto c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 2);
    const auto d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 3);
    return {move_f32x4{a[0], a[1], b[0], b[1]}, move_f32x4{c[0], c[1], d[0], d[1]}};
  } else {
    return {__builtin_bit_cast(typename Eight<T>::vec, expand8<T>(codes, scale))};
  }
}

// A workgroup takes 64 packed rows: the first wave finds each one's page and slot, then D / 8 threads
// a row expand eight channels each, four rows' loads in flight.
template <typename T, int D, bool FUSED>
__global__ __launch_bounds__(kThreads) void paged_read_kernel(ReadArgs a) {
  constexpr int kRowThreads = D / 8, kRowsAtOnce = kThreads / kRowThreads;
  constexpr int kRounds = kReadRows / kRowsAtOnce, kTogether = kRounds < 4 ? kRounds : 4;
  __shared__ int32_t sums[FUSED ? kFusedSegments + 1 : 1];
  __shared__ int64_t row_page[kReadRows];  // byte offset of the row's page, or -1
  __shared__ int row_slot[kReadRows];
  const PagedCache& cache = a.cache;
  const int segments = static_cast<int>(a.segments);
  const int32_t* cumulative = a.cumulative;
  if constexpr (FUSED) {
    sum_lengths(cache, segments, sums);
    if (blockIdx.x == 0)
      for (int s = threadIdx.x; s <= segments; s += kThreads) a.cumulative[s] = sums[s];
    cumulative = sums;
  }
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kReadRows;
  if (threadIdx.x < kReadRows) {
    const int64_t row = row0 + threadIdx.x;
    int64_t page = -1;
    int slot = 0;
    if (row < a.total && row < cumulative[segments]) {
      const int segment = segment_of(cumulative, segments, static_cast<int>(row));
      const int at = static_cast<int>(row) - cumulative[segment];
      const int64_t id = cache.table[static_cast<int64_t>(segment) * cache.max_pages + (at >> cache.shift)];
      if (id >= 0 && id < cache.page_count) {
        page = id * (Page<D>::bytes(1) << cache.shift);
        slot = at & ((1 << cache.shift) - 1);
        a.positions[row] = *reinterpret_cast<const float*>(cache.pages + page +
                                                           Page<D>::position(cache.shift, slot));
      }
    }
    row_page[threadIdx.x] = page;
    row_slot[threadIdx.x] = slot;
  }
  __syncthreads();
  const int c = threadIdx.x % kRowThreads, first = threadIdx.x / kRowThreads;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    T* const out = static_cast<T*>(which == 0 ? a.keys : a.values) + row0 * D + 8 * c;
#pragma unroll
    for (int r0 = 0; r0 < kRounds; r0 += kTogether) {
      unsigned codes[kTogether], byte[kTogether];
      bool there[kTogether];
#pragma unroll
      for (int i = 0; i < kTogether; ++i) {
        const int r = (r0 + i) * kRowsAtOnce + first, slot = row_slot[r];
        there[i] = row_page[r] >= 0;
        // (a row that is not there reads the pool's first one, and is not written)
        const uint8_t* p = cache.pages + (there[i] ? row_page[r] : 0);
        codes[i] = *reinterpret_cast<const unsigned*>(p + Page<D>::codes(cache.shift, which, slot) + 4 * c);
        byte[i] = p[Page<D>::scales(cache.shift, which, slot) + c / 4];
      }
#pragma unroll
      for (int i = 0; i < kTogether; ++i)
        if (there[i])
          *reinterpret_cast<Eight<T>*>(out + static_cast<int64_t>((r0 + i) * kRowsAtOnce + first) * D) =
              eight_values<T>(codes[i], scale_of(byte[i]));
    }
  }
}

// ---------------------------------------------------------------------------------------
constexpr int kCompactRows = kThreads;  // of a workgroup, 64 a wave

// A wave moves 64 rows of a segment: row r comes from row r + how many removed rows lie at or before
// it. The wave finds that number for its first and its last row, each lane its own between them;
// then all lanes copy 16 bytes each of the rows' codes.
template <int D, bool FUSED>
__global__ __launch_bounds__(kThreads) void paged_compact_kernel(CompactArgs a) {
  constexpr int kPieces = D / 32;  // 16 bytes of a row's codes
  using Scales = std::conditional_t<D == 64, uint16_t, std::conditional_t<D == 128, uint32_t, uint64_t>>;
  __shared__ int64_t lds_sums[FUSED ? kFusedSegments + 1 : 1];
  const PagedCache& cache = a.cache;
  const int lane = threadIdx.x & 63;
  const int64_t segment = blockIdx.x / static_cast<unsigned>(a.chunks);
  const int chunk = static_cast<int>(blockIdx.x - segment * a.chunks);
  const int64_t* sums = a.sums;
  if constexpr (FUSED) {
    sum_lengths(cache, static_cast<int>(a.segments), lds_sums);
    sums = lds_sums;
  }
  const int64_t first = sums[segment];
  const int length = cache.rows(segment);
  const int row0 = chunk * kCompactRows + static_cast<int>(threadIdx.x & ~63u);
  if (chunk > 0 && row0 >= length) return;  // no row can be left there
  // the segment's part of the removed rows
  const int64_t bound = lane < 32 ? first : first + length;
  const int64_t found = half_search(0, a.removed_count, [&](int64_t i) { return a.removed[i] < bound; });
  const int64_t low = __shfl(found, 0);
  const int64_t inside = __shfl(found, 32) - low;  // (negative for rows that are not sorted)
  const int gone = static_cast<int>(inside < 0 ? 0 : inside < length ? inside : length);
  const int left = length - gone;
  if (chunk == 0 && threadIdx.x == 0) a.new_lengths[segment] = left;
  const int rows = min(left, a.target_pages << cache.shift);
  if (row0 >= rows) return;
  const int64_t* removed = a.removed + low;
  // how many removed rows (of this segment) lie at or before kept row `row`
  auto lies_before = [&](int row) { return [=](int64_t i) { return removed[i] - first - i <= row; }; };
  int64_t j = half_search(0, gone, lies_before(lane < 32 ? row0 : row0 + 63));
  const int row = row0 + lane, mask = (1 << cache.shift) - 1;
  {
    int64_t from = __shfl(j, 0), to = __shfl(j, 32);
    while (from < to) {
      const int64_t mid = (from + to) / 2;
      if (lies_before(row)(mid)) from = mid + 1;
      else to = mid;
    }
    j = from;
  }
  // byte offsets of the row's old and new pages (-1: none), and its slots there
  int64_t from = -1, to = -1;
  const int64_t source = row + j;
  if (row < rows && source < length) {
    const int64_t id = cache.table[segment * cache.max_pages + (source >> cache.shift)];
    const int64_t target = a.target[segment * a.target_pages + (row >> cache.shift)];
    if (id >= 0 && id < cache.page_count && target >= 0 && target < cache.page_count) {
      from = id * (Page<D>::bytes(1) << cache.shift);
      to = target * (Page<D>::bytes(1) << cache.shift);
    }
  }
  const int from_slot = static_cast<int>(source) & mask, to_slot = row & mask;
  // All loads before the first store (a row that is not moved reads the pool's first one).
  const uint8_t* const page = cache.pages + (from >= 0 ? from : 0);
  const int read_slot = from >= 0 ? from_slot : 0;
  Scales scales[2];
#pragma unroll
  for (int which = 0; which < 2; ++which)
    scales[which] = *reinterpret_cast<const Scales*>(page + Page<D>::scales(cache.shift, which, read_slot));
  const float position = *reinterpret_cast<const float*>(page + Page<D>::position(cache.shift, read_slot));
  move_u32x4 data[2][kPieces];
  int64_t target[kPieces];
#pragma unroll
  for (int u = 0; u < kPieces; ++u) {
    const int piece = u * 64 + lane, r = piece / kPieces, c = piece % kPieces;
    const int64_t piece_from = __shfl(from, r), piece_to = __shfl(to, r);
    const int slot = __shfl(read_slot, r), target_slot = __shfl(to_slot, r);
    const uint8_t* p = cache.pages + (piece_from >= 0 ? piece_from : 0);
#pragma unroll
    for (int which = 0; which < 2; ++which)
      data[which][u] = *reinterpret_cast<const move_u32x4*>(
          p + Page<D>::codes(cache.shift, which, slot) + 16 * c);
    target[u] = piece_to < 0 ? -1 : piece_to + Page<D>::codes(cache.shift, 0, target_slot) + 16 * c;
  }
#pragma unroll
  for (int u = 0; u < kPieces; ++u)
    if (target[u] >= 0)
#pragma unroll
      for (int which = 0; which < 2; ++which)
        *reinterpret_cast<move_u32x4*>(cache.pages + target[u] + Page<D>::codes(cache.shift, which, 0)) =
            data[which][u];
  if (to < 0) return;
  uint8_t* const out = cache.pages + to;
#pragma unroll
  for (int which = 0; which < 2; ++which)
    *reinterpret_cast<Scales*>(out + Page<D>::scales(cache.shift, which, to_slot)) = scales[which];
  *reinterpret_cast<float*>(out + Page<D>::position(cache.shift, to_slot)) = position;
}

}  // namespace
}  // namespace lr

using namespace lr;

extern "C" int64_t lr_paged_page_bytes(int64_t page_size, int64_t dim) {
  return paged_bytes(page_size, dim);
}

extern "C" int lr_paged_append(const void* keys, const int64_t* key_strides, const void* values,
                               const int64_t* value_strides, const void* queries,
                               const int64_t* query_strides, void* out_queries, int64_t batch,
                               int64_t kv_heads, int64_t query_heads, int64_t added, int64_t dim,
                               int dtype, const int64_t* positions, const float* cos,
                               const float* sin, int64_t table_rows, int64_t half,
                               const int32_t* counts, void* pages, int64_t page_count,
                               int64_t page_size, const int32_t* table, int64_t max_pages,
                               const int32_t* lengths, void* stream) {
  auto launch = [&](AppendArgs& args) {
    args.range = dtype == LR_DTYPE_F16 ? kHalfRange : kWideRange;
    // Rotated blocks whole: the pairs kernel, four heads a thread where there are enough rows to fill
    // the chip with them (8,192 tokens, 393,000 rows: 36 us against 47 with a row's D / 8 threads and
    // one head; a step of eight requests, 384 rows, 3.4 either way).
    const bool pairs = half % kBlock == 0;
    const int64_t all_rows = 2 * static_cast<int64_t>(args.kv_rows) + args.query_rows;
    const int64_t heads = pairs && all_rows >= 32768 ? 4 : 1;
    const int64_t per_block = kThreads / (dim / (pairs ? 16 : 8));
    const int64_t kv_blocks = ceil_div(batch * added * ceil_div(kv_heads, heads), per_block);
    const int64_t blocks = 2 * kv_blocks + ceil_div(batch * added * ceil_div(query_heads, heads), per_block);
    LR_REQUIRE(launchable(blocks, kThreads), "Appended grid too large");
    args.kv_blocks = static_cast<unsigned>(kv_blocks);
    return dispatch_type(dtype, [&]<typename T>() {
      return dispatch_dim(dim, [&]<int D>() {
        auto enqueue = [&](auto kernel) {
          hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0,
                             as_stream(stream), args);
        };
        if (!pairs) enqueue(paged_append_kernel<T, D>);
        else if (heads == 1) enqueue(paged_append_pairs_kernel<T, D, 1>);
        else enqueue(paged_append_pairs_kernel<T, D, 4>);
        return check_launch("paged_append");
      });
    });
  };
  return append_paged(keys, key_strides, values, value_strides, queries, query_strides, out_queries,
                      batch, kv_heads, query_heads, added, dim, dtype, positions, cos, sin, table_rows,
                      half, counts, pages, page_count, page_size, table, max_pages, lengths, launch);
}

extern "C" int lr_paged_read(const void* pages, int64_t page_count, int64_t page_size,
                             const int32_t* table, int64_t max_pages, const int32_t* lengths,
                             int64_t segments, int64_t dim, int dtype, int64_t total, void* keys,
                             void* values, float* positions, int32_t* cumulative, void* stream) {
  auto launch = [&](const ReadArgs& args, int64_t blocks, bool fused) {
    return dispatch_type(dtype, [&]<typename T>() {
      return dispatch_dim(dim, [&]<int D>() {
        auto enqueue = [&](auto kernel) {
          hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0,
                             as_stream(stream), args);
        };
        if (fused) enqueue(paged_read_kernel<T, D, true>);
        else enqueue(paged_read_kernel<T, D, false>);
        return check_launch("paged_read");
      });
    });
  };
  return read_paged(pages, page_count, page_size, table, max_pages, lengths, segments, dim, dtype, total,
                    keys, values, positions, cumulative, stream, launch);
}

extern "C" size_t lr_paged_compact_workspace_bytes(int64_t segments) {
  return compact_paged_workspace(segments);
}

extern "C" int lr_paged_compact(void* pages, int64_t page_count, int64_t page_size,
                                const int32_t* table, int64_t max_pages, const int32_t* lengths,
                                int64_t segments, int64_t dim, const int64_t* removed,
                                int64_t removed_count, const int32_t* target, int64_t target_pages,
                                int32_t* new_lengths, void* workspace, size_t workspace_size,
                                void* stream) {
  auto launch = [&](const CompactArgs& args, unsigned blocks, bool fused) {
    return dispatch_dim(dim, [&]<int D>() {
      auto enqueue = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(blocks), dim3(kThreads), 0, as_stream(stream), args);
      };
      if (fused) enqueue(paged_compact_kernel<D, true>);
      else enqueue(paged_compact_kernel<D, false>);
      return check_launch("paged_compact");
    });
  };
  return compact_paged(kCompactRows, pages, page_count, page_size, table, max_pages, lengths, segments,
                       dim, removed, removed_count, target, target_pages, new_lengths, workspace,
                       workspace_size, stream, launch);
}
