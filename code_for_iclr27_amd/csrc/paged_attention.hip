// Attention over the paged 4-bit KV cache (paged.hpp states its layout): `length` queries a head
// onto each segment's rows. Query i of a request sees the segment's lengths[s] rows and the first
// i + 1 of those appended behind them (counts[b], or `length`, rows): keys j <= lengths[s] + i.
// Queries at or past counts[b] output zeros, as does a query that sees no key.
//
// Work split: row = i * G + g numbers a segment's query rows; a workgroup of four (eight) waves owns a
// tile of 16 rows and a chunk of keys, each wave every fourth (eighth) unit of 32 keys. Calls of many
// rows take tiles of 32 (paged_tile_kernel); plan_paged has the rules. Codes go from memory to
// registers (16 bytes a lane: a block of one row), the conversion instruction makes them 16-bit
// values, and both products run on v_mfma_f32_16x16x32:
//   S^T = K Q^T   A: 16 keys, a lane's eight channels of one key. The contraction's channel order is
//                 free, so a lane's block stays where it was loaded. A lane gets one query's scores
//                 of 4 + 4 keys.
//   O^T += V^T P^T  B: the probabilities where S^T left them (the key order is free as well); A: the
//                 same keys of one channel, read transposed from the wave's V rows in LDS.
// The values are exact in the 16-bit type, and their products exact in f32. P is f32 and stays f32: it
// enters as the sum of three bf16 pieces by truncation, 3 x 8 bits = the whole 24-bit significand, whose
// products with V are exact (a P below 2^-110 keeps what lies above 2^-133, bf16's smallest number), as
// attention over packed rows has it. (Two pieces took 133 us in the place of 157 for 1000 queries onto
// 4,450 rows and 64 in the place of 65 for a long decode, and left 2^-18 to 2^-16 of P out. Three by
// rounding: 161.) Scores, exponentials, their sum and the products' sums are f32 throughout.
//
// The exponentials' reference moves when a row's maximum has outgrown it by 2^kPagedSlack (as in
// attention_tile.hip). The waves' states meet in LDS; tiles whose keys span several chunks leave
// partial states, which a second launch merges.
//
// A masked key contributes nothing: its score becomes -inf, its P 0. As 0 * NaN is NaN, a wave that
// ends with a non-finite sum takes its keys again, with the blocks of V that read as NaN kept out of
// the product and added to the rows that see their key. So does one whose scores are so large that the
// reference's own rounding would show in the exponentials (kLargeReference).
//
// What bounds it. Decode of a long cache: memory (eight requests of 36k rows, 8 heads, G4, d128: 312 MB
// of codes in 65 us, 4.8 TB/s; a large copy reaches 5.2). Short ones: the two launches (8 segments of
// 2,250 rows: 8.8 us, 2,250 rows of eight requests 11.6 us). Prefill: the vector instructions, 268 a
// unit of 32 keys and 32 rows beside 32 MFMAs (a third for the pieces, a quarter for the values), 65% of
// a SIMD's issue slots with 2.3 waves on average: 1000 queries onto 4,450 rows 158 us, where the packed
// kernel on the same rows in 16 bits, with P in as many pieces, takes 206. Tried with two pieces and no
// faster: units in flight two ahead, the exponentials laid between the MFMAs of the last unit's product
// by hand, a raised wave priority for the products, tiles of 64 rows, four waves a SIMD (registers
// spilled), the pieces' rests by two-element dot products.

#include <algorithm>
#include <cmath>

#include "attention_common.hpp"
#include "lds_copy.hpp"
#include "paged.hpp"

namespace lr {
namespace {

typedef short paged_s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned paged_u32x2 __attribute__((ext_vector_type(2)));

constexpr int kUnit = 32;       // keys of a wave's step
constexpr int kSmallRows = 16;  // rows of a tile: decode and a few query rows
constexpr int kTileRows = 32;   // many query rows
constexpr float kPagedSlack = 4.0f;
constexpr int kPieces = 3;      // of a probability
// A row's largest exponent (of two) up to which score * to_log2 - reference is one multiply-add: the
// reference is a rounded product, and the multiply-add keeps the scores' differences exact, but the
// largest P is 2^32 or 2^-32 here, and from 2^31 on f32's exponents do not hold it.
constexpr float kLargeReference = 0x1p30f;

struct PagedAttnArgs {
  const void* queries;  // element strides below; the last dimension is contiguous
  int64_t q_batch, q_head, q_query;
  PagedCache cache;
  const int32_t* counts;  // [batch] or NULL
  int kv_heads, groups, length;
  int max_keys;           // no key at or past it is visited
  unsigned segments, tiles, splits;
  int tile_rows;          // rows of a tile's partial states
  int chunk;              // keys of a split, a multiple of kStep
  float to_log2;          // scale * log2(e)
  void* out;              // [batch, length, kv_heads * groups, D]
  float* part_ml;         // [units * splits, tile_rows, 2]
  float* part_o;          // [units * splits, tile_rows, D]
};

// What the rows of a tile see.
struct TileKeys {
  int cached, count, key_end, needed;  // key_end: past the last key of any row
};
__device__ __forceinline__ TileKeys tile_keys(const PagedAttnArgs& a, unsigned seg, unsigned row0,
                                              unsigned last_row) {
  TileKeys t;
  const unsigned groups = static_cast<unsigned>(a.groups);
  t.cached = a.cache.rows(seg);
  t.count = a.length;
  if (a.counts != nullptr) {
    const int c = a.counts[seg / static_cast<unsigned>(a.kv_heads)];
    t.count = c < 0 ? 0 : c < a.length ? c : a.length;
  }
  if (a.cache.lengths[seg] < 0) t.count = 0;  // (append has stored nothing there)
  const int first = static_cast<int>(row0 / groups), last = static_cast<int>(last_row / groups);
  const int most = min(a.cache.max_pages << a.cache.shift, a.max_keys);
  t.key_end = first < t.count ? min(most, t.cached + min(last, t.count - 1) + 1) : 0;
  t.needed = (t.key_end + a.chunk - 1) / a.chunk;
  return t;
}

template <typename T, int D>
__device__ __forceinline__ T* paged_output(const PagedAttnArgs& a, unsigned seg, unsigned row) {
  const unsigned groups = static_cast<unsigned>(a.groups), heads = static_cast<unsigned>(a.kv_heads);
  const unsigned b = seg / heads, h = seg - b * heads, i = row / groups, g = row - i * groups;
  return static_cast<T*>(a.out) +
         ((static_cast<int64_t>(b) * a.length + i) * (static_cast<int64_t>(heads) * groups) +
          h * groups + g) * D;
}

// Two f32 values as sums of three bf16 pieces each, word `w` of the piece vectors: the top halves of x,
// of x minus that, and of what is left (each difference is exact, the last has at most 8 significant
// bits).
__device__ __forceinline__ void split_bf16(float x, float y, attn_u32x4 (&piece)[kPieces], int w) {
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const unsigned a = __builtin_bit_cast(unsigned, x), b = __builtin_bit_cast(unsigned, y);
    piece[i][w] = __builtin_amdgcn_perm(b, a, 0x07060302u);
    x -= __builtin_bit_cast(float, a & 0xffff0000u);
    y -= __builtin_bit_cast(float, b & 0xffff0000u);
  }
}

// The exponential of a score against its row's reference, the rounded product of its largest score and
// to_log2 (or 0). SAFE: for references of any size; past kLargeReference the score's product is rounded
// as well, so that the largest one's exponent is 0.
template <bool SAFE>
__device__ __forceinline__ float probability(float score, float to_log2, float base) {
  if (SAFE && __builtin_fabsf(base) > kLargeReference)
    return __builtin_amdgcn_exp2f(score * to_log2 - base);
  return __builtin_amdgcn_exp2f(__builtin_fmaf(score, to_log2, -base));
}

// Whether a wave has to take its keys again: a sum that is not finite (`poison` is NaN) or a reference
// past kLargeReference (-inf: the row has seen no key).
__device__ __forceinline__ bool take_again(float poison, float reference) {
  return __any(poison != poison || reference > kLargeReference ||
               (reference < -kLargeReference && reference != kNegInf));
}

// V rows in LDS: 16-byte chunk c of row r in slot c ^ x(r). The eight rows that eight lanes write one
// chunk of lie in different 16-byte places of 128, and the 32 bytes of four rows that 16 lanes read
// transposed in different quarters of it. (Slots that differ in the four rows' 64-byte places alone
// had twice the bank conflicts; the prefill kernel as a whole took 0.6% longer.)
__device__ __forceinline__ int value_swizzle(int row) { return (row & 3) << 1 | ((row >> 2) & 1); }

typedef const __attribute__((address_space(4))) int32_t* PageIds;  // read by scalar loads
__device__ __forceinline__ PageIds page_table(const PagedCache& cache, unsigned seg) {
  return (PageIds)(cache.table + static_cast<int64_t>(seg) * cache.max_pages);
}

// A block's segment, tile and split. Consecutive blocks take consecutive segments, so with 8 segments
// (or a divisor or multiple of it) each XCD's L2 serves its own segments' rows (1000 queries onto
// 4,000 rows: 7% less than with consecutive tiles); within a segment the tiles with the most
// visible keys come first, so that the launch's tail is short.
struct Place {
  unsigned seg, tile, split, unit;
};
__device__ __forceinline__ Place block_place(const PagedAttnArgs& a) {
  Place p;
  const unsigned rest = blockIdx.x / a.segments;
  p.seg = blockIdx.x - rest * a.segments;
  const unsigned back = rest / a.splits;
  p.split = rest - back * a.splits;
  p.tile = a.tiles - 1 - back;
  p.unit = p.seg * a.tiles + p.tile;
  return p;
}

__device__ __forceinline__ int rows_of_tile(const PagedAttnArgs& a, unsigned row0, int most) {
  const unsigned rows = static_cast<unsigned>(a.length) * static_cast<unsigned>(a.groups);
  return static_cast<int>(min(rows - row0, static_cast<unsigned>(most)));
}

// A query row: its query and its place (elements) in the queries.
struct TileRow {
  int query;
  int64_t offset;
};
__device__ __forceinline__ TileRow tile_row(const PagedAttnArgs& a, unsigned seg, unsigned row) {
  const unsigned groups = static_cast<unsigned>(a.groups), heads = static_cast<unsigned>(a.kv_heads);
  const unsigned i = row / groups, g = row - i * groups, b = seg / heads, h = seg - b * heads;
  return {static_cast<int>(i), b * a.q_batch + static_cast<int64_t>(h * groups + g) * a.q_head + i * a.q_query};
}
// The last key that a query sees (-1: none), and the last one that every row of a tile sees.
__device__ __forceinline__ int last_key(const TileKeys& keys, int query) {
  return query < keys.count ? min(keys.cached + query, keys.key_end - 1) : -1;
}
__device__ __forceinline__ int all_rows_see(const PagedAttnArgs& a, const TileKeys& keys, unsigned row0, int rows) {
  const unsigned groups = static_cast<unsigned>(a.groups);
  const int last = static_cast<int>((row0 + rows - 1) / groups);
  return last < keys.count ? min(keys.cached + static_cast<int>(row0 / groups), keys.key_end - 1) : -1;
}

// Zeros for rows that see no key.
template <typename T, int D>
__device__ __forceinline__ void zero_rows(const PagedAttnArgs& a, unsigned seg, unsigned row0, int rows) {
  for (int item = threadIdx.x; item < rows * (D / 8); item += blockDim.x) {
    const int r = item / (D / 8), c = item - r * (D / 8);
    *reinterpret_cast<attn_u32x4*>(paged_output<T, D>(a, seg, row0 + r) + 8 * c) =
        attn_u32x4{0u, 0u, 0u, 0u};
  }
}

// Eight channels of a row from the waves' states: the output, or (`whole` false) the chunk's partial
// state at `slot`.
template <typename T, int D, int WAVES, typename ML, typename State>
__device__ __forceinline__ void finish_item(const PagedAttnArgs& a, unsigned seg, unsigned row,
                                            int channel, int64_t slot, bool whole, ML ml, State state) {
  float top = kNegInf, total = 0.0f, o[8] = {};
#pragma unroll
  for (int w = 0; w < WAVES; ++w) top = fmaxf(top, ml(w, 0));
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    const float reference = ml(w, 0), sum = ml(w, 1);
    attn_f32x4 lo, hi;
    state(w, lo, hi);
    if (reference == kNegInf && sum == 0.0f) continue;  // saw no key
    const float weight = reference == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(reference - top);
    total = __builtin_fmaf(weight, sum, total);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o[e] = __builtin_fmaf(weight, lo[e], o[e]);
      o[4 + e] = __builtin_fmaf(weight, hi[e], o[4 + e]);
    }
  }
  if (whole) {
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] *= inv;
    *reinterpret_cast<attn_u32x4*>(paged_output<T, D>(a, seg, row) + channel) = pack8<T>(o);
    return;
  }
  float* po = a.part_o + slot * D + channel;
  *reinterpret_cast<attn_f32x4*>(po) = attn_f32x4{o[0], o[1], o[2], o[3]};
  *reinterpret_cast<attn_f32x4*>(po + 4) = attn_f32x4{o[4], o[5], o[6], o[7]};
  if (channel == 0) {
    a.part_ml[slot * 2] = top;
    a.part_ml[slot * 2 + 1] = total;
  }
}

// Codes and scales of a unit: two blocks of 16 rows, a lane's words of one row each. Words 4 h ..
// 4 h + 3 (d256: h = 0, 1; else all) belong to one block of channels.
template <int D>
struct UnitCodes {
  static constexpr int kWords = D / 32, kBytes = D == 256 ? 2 : 1;
  unsigned k[2][kWords], v[2][kWords], ks[2][kBytes], vs[2][kBytes];
};

// Memory addressed as a wave-uniform base and a lane's offset. (In the global address space: a generic
// load also counts as an LDS access, and every wait for LDS would be one for memory.)
typedef const __attribute__((address_space(1))) uint8_t* PagedBytes;

template <int D>
__device__ __forceinline__ void load_codes(unsigned (&words)[D / 32], PagedBytes p) {
  if constexpr (D == 64) {
    const paged_u32x2 x = *(const __attribute__((address_space(1))) paged_u32x2*)p;
    words[0] = x[0], words[1] = x[1];
  } else {
#pragma unroll
    for (int half = 0; half < D / 128; ++half) {
      const attn_u32x4 x = *(const __attribute__((address_space(1))) attn_u32x4*)(p + 64 * half);
#pragma unroll
      for (int e = 0; e < 4; ++e) words[4 * half + e] = x[e];
    }
  }
}
// The channel of a lane's word `w`, over 8.
template <int D>
__device__ __forceinline__ int word_chunk(int j, int w) {
  return D == 64 ? 2 * j + w : 16 * (w >> 2) + 4 * j + (w & 3);
}

// Four rows' elements of one column from LDS: lanes 4 k .. 4 k + 3 of each 16 address row k (8 bytes
// each), lane i receives column i of the 16.
__device__ __forceinline__ paged_u32x2 read_transposed(uint32_t p) {
  return __builtin_bit_cast(paged_u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) paged_s16x4*)(uintptr_t)p));
}

__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Tiles of 16 rows: decode, and a few query rows.
template <typename T, int D, int WAVES>
__global__ __launch_bounds__(64 * WAVES) __attribute__((amdgpu_waves_per_eu(
    WAVES == 8 || D == 256 ? 2 : D == 64 ? 4 : 3)))
void paged_attention_kernel(PagedAttnArgs a) {
  constexpr int kStep = kUnit * WAVES;  // keys of the workgroup's step
  using Vec = AttnVec<T>;
  using X8 = typename Vec::x8;
  using Codes = UnitCodes<D>;
  constexpr int KW = D / 32, DT = D / 16;
  __shared__ __align__(1024) uint16_t v_lds[WAVES][kUnit * D];
  __shared__ float wave_ml[WAVES][kSmallRows][2];
  __shared__ __align__(16) attn_u32x4 q_lds[KW][64];

  const int lane = threadIdx.x & 63, m = lane & 15, j = lane >> 4;
  const int wave = static_cast<int>(wave_index());
  const Place place = block_place(a);
  const unsigned seg = place.seg, row0 = place.tile * kSmallRows;
  const int rows_here = rows_of_tile(a, row0, kSmallRows);
  // The pages of the wave's first unit, looked up beside the segment's length (an entry past the
  // segment's last page is not used): the two memory round trips overlap.
  const PagedCache& cache = a.cache;
  const PageIds table = page_table(cache, seg);
  auto in_pool = [&](int id) { return id >= 0 && id < cache.page_count ? id : -1; };
  int first0 = -1, first1 = -1;
  if (a.max_keys > 0) {
    const int key = static_cast<int>(place.split) * a.chunk + kUnit * wave;
    first0 = table[min(key >> cache.shift, cache.max_pages - 1)];
    first1 = table[min((key + 16) >> cache.shift, cache.max_pages - 1)];
  }
  const TileKeys keys = tile_keys(a, seg, row0, row0 + rows_here - 1);
  if (keys.needed == 0) {  // no visible key for any row of this tile
    if (place.split == 0) zero_rows<T, D>(a, seg, row0, rows_here);
    return;
  }
  if (static_cast<int>(place.split) >= keys.needed) return;  // uniform across the workgroup
  const int begin = static_cast<int>(place.split) * a.chunk;
  const int end = min(begin + a.chunk, keys.key_end);
  first0 = in_pool(first0);
  first1 = in_pool(first1);

  // Queries (B operand: row m, the channels of word w of lane group j) in LDS for every wave, and the
  // last key that the lane's row sees.
  const TileRow row = tile_row(a, seg, row0 + (m < rows_here ? m : 0));
  const int limit = m < rows_here ? last_key(keys, row.query) : -1;
  const int all_see = all_rows_see(a, keys, row0, rows_here);
#pragma unroll
  for (int w = 0; w < KW; ++w)
    if (wave == w % WAVES)
      q_lds[w][lane] = load16(static_cast<const T*>(a.queries) + row.offset + 8 * word_chunk<D>(j, w));

  const int64_t page_bytes = Page<D>::bytes(1) << cache.shift;
  const int mask = (1 << cache.shift) - 1;
  // Page of 16 rows from `key` on (one page: page sizes are multiples of 16); -1: outside the pool.
  auto page_id = [&](int key) { return in_pool(table[min(key, keys.key_end - 1) >> cache.shift]); };
  // A page and a slot are the wave's, so addresses are scalar but for the lane's place in 16 rows.
  const unsigned lane_codes = m * Page<D>::kCodes + (D == 64 ? 8 : 16) * j;
  const unsigned lane_scale = m * Page<D>::kScales + (D == 64 ? j >> 1 : j);
  auto load = [&](Codes& u, int key0, int id0, int id1) {
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
      const int id = blk == 0 ? id0 : id1;
      const int slot = (key0 + 16 * blk) & mask;
      const PagedBytes page =
          (PagedBytes)uniform_address(cache.pages + (id < 0 ? 0 : id) * page_bytes);
      load_codes<D>(u.k[blk], page + Page<D>::codes(cache.shift, 0, slot) + lane_codes);
      load_codes<D>(u.v[blk], page + Page<D>::codes(cache.shift, 1, slot) + lane_codes);
#pragma unroll
      for (int i = 0; i < Codes::kBytes; ++i) {
        u.ks[blk][i] = page[Page<D>::scales(cache.shift, 0, slot) + 4 * i + lane_scale];
        u.vs[blk][i] = page[Page<D>::scales(cache.shift, 1, slot) + 4 * i + lane_scale];
      }
    }
  };

  float reference, sum;  // in exponents of two; a row's reference is the same in its four lanes
  attn_f32x4 out[DT];
  char* const my_values = reinterpret_cast<char*>(&v_lds[wave][0]);
  uint32_t read_at;  // of the lane's transposed reads: row 4 j + m / 4, columns 4 (m % 4) .. + 3
  {
    const int r = 4 * j + (m >> 2), chunk = (m & 3) >> 1;
    read_at = lds_address(my_values) + r * (2 * D) + 16 * (chunk ^ value_swizzle(r)) + 8 * (m & 1);
  }
  auto write_values = [&](const Codes& u) {
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
      char* to = my_values + (16 * blk + m) * (2 * D);
#pragma unroll
      for (int w = 0; w < KW; ++w)
        *reinterpret_cast<attn_u32x4*>(to + 16 * (word_chunk<D>(j, w) ^ value_swizzle(m))) =
            expand8<__bf16>(u.v[blk][w], scale_of(u.vs[blk][Codes::kBytes == 2 ? w / 4 : 0]));
    }
  };

  // The wave's units of the chunk. SAFE: blocks of V that read as NaN are kept out of the product and
  // added to the rows that see their key, and no exponential exceeds its row's largest.
  auto pass = [&]<bool SAFE>() {
    reference = kNegInf, sum = 0.0f;
#pragma unroll
    for (int ct = 0; ct < DT; ++ct) out[ct] = attn_f32x4{0.f, 0.f, 0.f, 0.f};
    int key = begin + kUnit * wave;
    if (key >= end) return;
    Codes u;
    int id0 = SAFE ? page_id(key) : first0, id1 = SAFE ? page_id(key + 16) : first1;
    load(u, key, id0, id1);
    int next0 = page_id(key + kStep), next1 = page_id(key + kStep + 16);
    while (true) {
      // the unit after the next: its pages' ids arrive while this one is worked on
      const int later0 = page_id(key + 2 * kStep), later1 = page_id(key + 2 * kStep + 16);
      const bool more = key + kStep < end;
      if (key + kUnit > keys.key_end || id0 < 0 || id1 < 0) {  // rows that are not there: zeros for V
#pragma unroll
        for (int blk = 0; blk < 2; ++blk) {
          const bool there = key + 16 * blk + m < keys.key_end && (blk == 0 ? id0 : id1) >= 0;
#pragma unroll
          for (int w = 0; w < KW; ++w) u.v[blk][w] = there ? u.v[blk][w] : 0u;
#pragma unroll
          for (int i = 0; i < Codes::kBytes; ++i) u.vs[blk][i] = there ? u.vs[blk][i] : 127u;
        }
      }
      if constexpr (SAFE) {
        bool invalid = false;
#pragma unroll
        for (int blk = 0; blk < 2; ++blk)
#pragma unroll
          for (int i = 0; i < Codes::kBytes; ++i) invalid |= u.vs[blk][i] == kScaleNaN;
        if (__any(invalid)) {
#pragma unroll 1
          for (int left = 0; left < kUnit; ++left) {
#pragma unroll
            for (int i = 0; i < Codes::kBytes; ++i)
#pragma unroll
              for (int b = 0; b < 4; ++b) {  // the lane that holds block b + 4 i of row `left`
                if (D == 64 && b >= 2) continue;
                const int from = (D == 64 ? 2 * b : b) * 16 + (left & 15);
                const unsigned byte = __shfl(left < 16 ? u.vs[0][i] : u.vs[1][i], from);
                if (byte == kScaleNaN && key + left <= limit)
#pragma unroll
                  for (int r = 0; r < 4; ++r)
                    out[2 * (b + 4 * i)][r] = out[2 * (b + 4 * i) + 1][r] = __builtin_nanf("");
              }
          }
#pragma unroll
          for (int blk = 0; blk < 2; ++blk)
#pragma unroll
            for (int i = 0; i < Codes::kBytes; ++i)
              if (u.vs[blk][i] == kScaleNaN) {
                u.vs[blk][i] = 127u;
#pragma unroll
                for (int w = 0; w < KW / Codes::kBytes; ++w) u.v[blk][i * 4 + w] = 0u;
              }
        }
      }
      // V rows to LDS (the last unit's reads are done: a wave's LDS accesses stay in order)
      write_values(u);
      // S^T
      attn_f32x4 s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        const X8 q = __builtin_bit_cast(X8, q_lds[w][lane]);
#pragma unroll
        for (int blk = 0; blk < 2; ++blk)
          s[blk] = Vec::mfma(__builtin_bit_cast(X8, expand8<T>(u.k[blk][w], scale_of(
                                 u.ks[blk][Codes::kBytes == 2 ? w / 4 : 0]))), q, s[blk]);
      }
      if (more) load(u, key + kStep, next0, next1);
      if (key + kUnit - 1 > all_see || id0 < 0 || id1 < 0) {
#pragma unroll
        for (int blk = 0; blk < 2; ++blk)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (key + 16 * blk + 4 * j + r > limit || (blk == 0 ? id0 : id1) < 0) s[blk][r] = kNegInf;
      }
      float top = kNegInf;
#pragma unroll
      for (int r = 0; r < 4; ++r) top = fmaxf(fmaxf(top, s[0][r]), s[1][r]);
      LanePair pair = lane_pair<16>(top);
      pair = lane_pair<32>(fmaxf(pair.first, pair.second));
      top = fmaxf(pair.first, pair.second) * a.to_log2;
      if (__any(top > reference + (SAFE ? 0.0f : kPagedSlack))) {
        const float raised = fmaxf(reference, top);
        const float factor = reference == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(reference - raised);
        sum *= factor;
#pragma unroll
        for (int ct = 0; ct < DT; ++ct)
#pragma unroll
          for (int r = 0; r < 4; ++r) out[ct][r] *= factor;
        reference = raised;
      }
      const float base = reference == kNegInf ? 0.0f : reference;
      attn_u32x4 piece[kPieces];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const float x = probability<SAFE>(s[n / 2][2 * (n % 2)], a.to_log2, base);
        const float y = probability<SAFE>(s[n / 2][2 * (n % 2) + 1], a.to_log2, base);
        sum += x;
        sum += y;
        split_bf16(x, y, piece, n);
      }
      // O^T += V^T P^T
      wave_fence();
#pragma unroll
      for (int ct = 0; ct < DT; ++ct) {
        const uint32_t at = read_at ^ (32 * ct);
        const paged_u32x2 lo = read_transposed(at), hi = read_transposed(at + 16 * (2 * D));
        const attn_bf16x8 v = __builtin_bit_cast(attn_bf16x8, attn_u32x4{lo[0], lo[1], hi[0], hi[1]});
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
          out[ct] = AttnVec<__bf16>::mfma(v, __builtin_bit_cast(attn_bf16x8, piece[i]), out[ct]);
      }
      wave_fence();
      if (!more) break;
      key += kStep;
      id0 = next0, id1 = next1;
      next0 = later0, next1 = later1;
    }
  };
  __syncthreads();
  pass.template operator()<false>();
  float poison = 0.0f;  // 0 * NaN is NaN
#pragma unroll
  for (int ct = 0; ct < DT; ++ct)
#pragma unroll
    for (int r = 0; r < 4; ++r) poison = __builtin_fmaf(out[ct][r], 0.0f, poison);
  if (take_again(poison, reference)) pass.template operator()<true>();
  {
    LanePair pair = lane_pair<16>(sum);
    pair = lane_pair<32>(pair.first + pair.second);
    sum = pair.first + pair.second;
  }

  // Wave states to LDS: 16-byte chunk c of row r in slot c ^ r.
  __syncthreads();
  float* const mine = reinterpret_cast<float*>(my_values) + m * D;
#pragma unroll
  for (int ct = 0; ct < DT; ++ct) *reinterpret_cast<attn_f32x4*>(mine + 4 * ((4 * ct + j) ^ m)) = out[ct];
  if (j == 0) {
    wave_ml[wave][m][0] = reference;
    wave_ml[wave][m][1] = sum;
  }
  __syncthreads();
  const int64_t slot = (static_cast<int64_t>(place.unit) * a.splits + place.split) * a.tile_rows;
  for (int item = threadIdx.x; item < rows_here * (D / 8); item += 64 * WAVES) {
    const int r = item / (D / 8), c = item - r * (D / 8);
    auto state = [&](int w, attn_f32x4& lo, attn_f32x4& hi) {
      const float* wo = reinterpret_cast<const float*>(&v_lds[w][0]) + r * D;
      lo = *reinterpret_cast<const attn_f32x4*>(wo + 4 * ((2 * c) ^ r));
      hi = *reinterpret_cast<const attn_f32x4*>(wo + 4 * ((2 * c + 1) ^ r));
    };
    finish_item<T, D, WAVES>(a, seg, row0 + r, 8 * c, slot + r, keys.needed == 1,
                             [&](int w, int i) { return wave_ml[w][r][i]; }, state);
  }
}

// ---- Tiles of 32 rows -------------------------------------------------------------------------
// The same with v_mfma_f32_32x32x16 for calls of many rows: a lane holds one query's scores of 16
// keys, half a row of codes, and an MFMA of twice the work takes no more of the wave's issue slots
// (8 of a SIMD's clocks against 4 a vector instruction, which bound this kernel).

typedef float paged_f32x16 __attribute__((ext_vector_type(16)));

template <typename T>
__device__ __forceinline__ paged_f32x16 mfma32(attn_u32x4 a, attn_u32x4 b, paged_f32x16 c) {
  if constexpr (std::is_same<T, __bf16>::value)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(attn_bf16x8, a),
                                                   __builtin_bit_cast(attn_bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(attn_f16x8, a),
                                                  __builtin_bit_cast(attn_f16x8, b), c, 0, 0, 0);
}

template <typename T, int D>
__global__ __launch_bounds__(kAttnThreads) __attribute__((amdgpu_waves_per_eu(D == 64 ? 4 : D == 128 ? 3 : 2)))
void paged_tile_kernel(PagedAttnArgs a) {
  constexpr int KS = D / 16;      // words of a lane, MFMA steps over the head dimension
  constexpr int DT = D / 32;      // blocks of a row, column tiles of the output
  constexpr int kStep = kUnit * kAttnWaves;
  __shared__ __align__(1024) uint16_t v_lds[kAttnWaves][kUnit * D];
  __shared__ __align__(16) attn_u32x4 q_lds[KS][64];
  // the waves' softmax states at the end, in the place of the queries
  float(*const wave_ml)[kTileRows][2] = reinterpret_cast<float(*)[kTileRows][2]>(&q_lds[0][0]);
  static_assert(sizeof(q_lds) >= sizeof(float) * kAttnWaves * kTileRows * 2, "room for the states");

  const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
  const int wave = static_cast<int>(wave_index());
  const Place place = block_place(a);
  const unsigned seg = place.seg, row0 = place.tile * kTileRows;
  const int rows_here = rows_of_tile(a, row0, kTileRows);
  const TileKeys keys = tile_keys(a, seg, row0, row0 + rows_here - 1);
  if (keys.needed == 0) {  // no visible key for any row of this tile
    if (place.split == 0) zero_rows<T, D>(a, seg, row0, rows_here);
    return;
  }
  if (static_cast<int>(place.split) >= keys.needed) return;  // uniform across the workgroup
  const int begin = static_cast<int>(place.split) * a.chunk;
  const int end = min(begin + a.chunk, keys.key_end);

  // Queries (B operand of step ks: channels half * D / 2 + 8 ks of row `col`) in LDS for every wave,
  // and the last key that the lane's row sees.
  const TileRow row = tile_row(a, seg, row0 + (col < rows_here ? col : 0));
  const int limit = col < rows_here ? last_key(keys, row.query) : -1;
  const int all_see = all_rows_see(a, keys, row0, rows_here);
#pragma unroll
  for (int n = 0; n < KS / kAttnWaves; ++n) {
    const int ks = n * kAttnWaves + wave;
    q_lds[ks][lane] = load16(static_cast<const T*>(a.queries) + row.offset + half * (D / 2) + 8 * ks);
  }

  const PagedCache& cache = a.cache;
  const PageIds table = page_table(cache, seg);
  const int64_t page_bytes = Page<D>::bytes(1) << cache.shift;
  const int mask = (1 << cache.shift) - 1;
  auto page_id = [&](int key) {
    const int id = table[min(key, keys.key_end - 1) >> cache.shift];
    return id >= 0 && id < cache.page_count ? id : -1;
  };
  // Lane (key, half): half a row's codes, words ks of channels half * D / 2 + 8 ks, and its blocks'
  // scales.
  struct Codes {
    unsigned w[KS], scales;
  };
  // Lanes 0 .. 15 and 16 .. 31 read 16 rows each; only pages of 16 rows make them two pages.
  const unsigned lane_slot = col & mask;
  const unsigned lane_codes = lane_slot * Page<D>::kCodes + half * (D / 4);
  const unsigned lane_scales = lane_slot * Page<D>::kScales + half * (DT / 2);
  auto load = [&](Codes& k, Codes& v, int key, int id0, int id1) {
    const PagedBytes page0 = (PagedBytes)(cache.pages + (id0 < 0 ? 0 : id0) * page_bytes);
    const PagedBytes page1 = (PagedBytes)(cache.pages + (id1 < 0 ? 0 : id1) * page_bytes);
    const PagedBytes page = col < 16 ? page0 : page1;
    const int slot = key & mask;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      Codes& u = which == 0 ? k : v;
      const PagedBytes codes = page + (Page<D>::codes(cache.shift, which, slot) + lane_codes);
#pragma unroll
      for (int n = 0; n < KS / 4; ++n) {
        const attn_u32x4 x = *(const __attribute__((address_space(1))) attn_u32x4*)(codes + 16 * n);
#pragma unroll
        for (int e = 0; e < 4; ++e) u.w[4 * n + e] = x[e];
      }
      const PagedBytes scales = page + (Page<D>::scales(cache.shift, which, slot) + lane_scales);
      if constexpr (D == 64) u.scales = *scales;
      else if constexpr (D == 128) u.scales = *(const __attribute__((address_space(1))) uint16_t*)scales;
      else u.scales = *(const __attribute__((address_space(1))) unsigned*)scales;
    }
  };
  auto scale = [&](const Codes& u, int ks) {
    return scale_of(D == 64 ? u.scales : u.scales >> (8 * (ks / 4)) & 255u);
  };

  float reference = kNegInf, sum = 0.0f;  // in exponents of two; the same in both halves
  paged_f32x16 out[DT];
  char* const my_values = reinterpret_cast<char*>(&v_lds[wave][0]);
  auto write_values = [&](const Codes& v) {
    char* row = my_values + col * (2 * D);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      *reinterpret_cast<attn_u32x4*>(row + 16 * ((half * KS + ks) ^ value_swizzle(col))) =
          expand8<__bf16>(v.w[ks], scale(v, ks));
  };
  // Transposed reads: row 4 half + (lane % 16) / 4 of eight, columns 16 (lane / 16 % 2) +
  // 4 (lane % 4) .. + 3 of 32.
  uint32_t read_at;
  {
    const int row = 4 * half + ((lane & 15) >> 2), chunk = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    read_at = lds_address(my_values) + row * (2 * D) + 16 * (chunk ^ value_swizzle(row)) +
              8 * (lane & 1);
  }
  auto read_column = [&](int k, int dt) {  // A operand: keys 16 k .. 16 k + 15 of 32 channels
    // (eight rows on, value_swizzle is the same)
    const uint32_t at = (read_at ^ (64 * dt)) + 16 * k * (2 * D);
    const paged_u32x2 lo = read_transposed(at), hi = read_transposed(at + 8 * (2 * D));
    return attn_u32x4{lo[0], lo[1], hi[0], hi[1]};
  };

  auto pass = [&]<bool SAFE>() {
    reference = kNegInf, sum = 0.0f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) out[dt][r] = 0.0f;
    int key = begin + kUnit * wave;
    if (key >= end) return;
    Codes k, v;
    int id0 = page_id(key), id1 = page_id(key + 16);
    load(k, v, key, id0, id1);
    int next0 = page_id(key + kStep), next1 = page_id(key + kStep + 16);
    while (true) {
      const int later0 = page_id(key + 2 * kStep), later1 = page_id(key + 2 * kStep + 16);
      const bool more = key + kStep < end;
      if (key + kUnit > keys.key_end || id0 < 0 || id1 < 0) {  // rows that are not there: zeros for V
        const bool there = key + col < keys.key_end && (col < 16 ? id0 : id1) >= 0;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) v.w[ks] = there ? v.w[ks] : 0u;
        v.scales = there ? v.scales : 0x7f7f7f7fu;
      }
      if constexpr (SAFE) {
        bool invalid = false;
#pragma unroll
        for (int b = 0; b < DT / 2; ++b) invalid |= (v.scales >> (8 * b) & 255u) == kScaleNaN;
        if (__any(invalid)) {
#pragma unroll 1
          for (int left = 0; left < kUnit; ++left) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
              const unsigned bytes = __shfl(v.scales, left + 32 * (dt / (DT / 2)));
              if ((bytes >> (8 * (dt % (DT / 2))) & 255u) == kScaleNaN && key + left <= limit)
#pragma unroll
                for (int r = 0; r < 16; ++r) out[dt][r] = __builtin_nanf("");
            }
          }
#pragma unroll
          for (int b = 0; b < DT / 2; ++b)
            if ((v.scales >> (8 * b) & 255u) == kScaleNaN) {
              v.scales &= ~(0x80u << (8 * b));  // 127
#pragma unroll
              for (int w = 0; w < 4; ++w) v.w[4 * b + w] = 0u;
            }
        }
      }
      // V rows to LDS (the last unit's reads are done: a wave's LDS accesses stay in order)
      write_values(v);
      // S^T
      paged_f32x16 s;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = 0.0f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) s = mfma32<T>(expand8<T>(k.w[ks], scale(k, ks)), q_lds[ks][lane], s);
      if (more) load(k, v, key + kStep, next0, next1);
      if (key + kUnit - 1 > all_see || id0 < 0 || id1 < 0) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (key + 8 * (r >> 2) + 4 * half + (r & 3) > limit || (r < 8 ? id0 : id1) < 0) s[r] = kNegInf;
      }
      float top = kNegInf;
#pragma unroll
      for (int r = 0; r < 8; ++r) top = fmaxf(fmaxf(top, s[2 * r]), s[2 * r + 1]);
      const LanePair pair = lane_pair<32>(top);
      top = fmaxf(pair.first, pair.second) * a.to_log2;
      if (__any(top > reference + (SAFE ? 0.0f : kPagedSlack))) {
        const float raised = fmaxf(reference, top);
        const float factor = reference == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(reference - raised);
        sum *= factor;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int r = 0; r < 16; ++r) out[dt][r] *= factor;
        reference = raised;
      }
      const float base = reference == kNegInf ? 0.0f : reference;
      attn_u32x4 piece[2][kPieces];
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        const float x = probability<SAFE>(s[2 * n], a.to_log2, base);
        const float y = probability<SAFE>(s[2 * n + 1], a.to_log2, base);
        sum += x;
        sum += y;
        split_bf16(x, y, piece[n / 4], n % 4);
      }
      // O^T += V^T P^T
      wave_fence();
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const attn_u32x4 x = read_column(kk, dt);
#pragma unroll
          for (int n = 0; n < kPieces; ++n) out[dt] = mfma32<__bf16>(x, piece[kk][n], out[dt]);
        }
      wave_fence();
      if (!more) break;
      key += kStep;
      id0 = next0, id1 = next1;
      next0 = later0, next1 = later1;
    }
  };
  __syncthreads();
  pass.template operator()<false>();
  float poison = 0.0f;  // 0 * NaN is NaN
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) poison = __builtin_fmaf(out[dt][r], 0.0f, poison);
  if (take_again(poison, reference)) pass.template operator()<true>();
  {
    const LanePair pair = lane_pair<32>(sum);
    sum = pair.first + pair.second;
  }

  // Wave states to LDS, D / 2 channels at a time: 16-byte chunk c of row r in slot c ^ (r % 8).
  // (Lane (row, half) holds channels 32 dt + 8 c + 4 half + [0, 4).)
  constexpr int DQ = D / 2, kParts = D / DQ, kItems = kTileRows * (DQ / 8);
  const int64_t slot = (static_cast<int64_t>(place.unit) * a.splits + place.split) * a.tile_rows;
#pragma unroll
  for (int part = 0; part < kParts; ++part) {
    __syncthreads();
    float* const mine = reinterpret_cast<float*>(my_values) + col * DQ;
#pragma unroll
    for (int d = 0; d < DQ / 32; ++d)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const paged_f32x16& o = out[DQ / 32 * part + d];
        *reinterpret_cast<attn_f32x4*>(mine + 4 * ((8 * d + 2 * c + half) ^ (col & 7))) =
            attn_f32x4{o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]};
      }
    if (half == 0 && part == 0) {
      wave_ml[wave][col][0] = reference;
      wave_ml[wave][col][1] = sum;
    }
    __syncthreads();
    for (int item = threadIdx.x; item < kItems; item += kAttnThreads) {
      const int r = item / (DQ / 8), c = item - r * (DQ / 8);
      if (r >= rows_here) break;
      auto state = [&](int w, attn_f32x4& lo, attn_f32x4& hi) {
        const float* wo = reinterpret_cast<const float*>(&v_lds[w][0]) + r * DQ;
        lo = *reinterpret_cast<const attn_f32x4*>(wo + 4 * ((2 * c) ^ (r & 7)));
        hi = *reinterpret_cast<const attn_f32x4*>(wo + 4 * ((2 * c + 1) ^ (r & 7)));
      };
      finish_item<T, D, kAttnWaves>(a, seg, row0 + r, DQ * part + 8 * c, slot + r, keys.needed == 1,
                                    [&](int w, int i) { return wave_ml[w][r][i]; }, state);
    }
  }
}

// Second launch of a split call: a thread folds one (row, 8 channels) slice of every fourth chunk of
// a tile, LOADS chunks' states loaded together; the four threads of a slice meet in LDS. The first
// round is loaded before the segment's length is known (the workspace holds every chunk of the
// grid; those past the needed ones are not used), so that the two memory round trips overlap.
constexpr int kMergeItems = 64, kMergeParts = kAttnThreads / kMergeItems;

template <typename T, int D, int LOADS>
__global__ __launch_bounds__(kAttnThreads) void paged_merge_kernel(PagedAttnArgs a, unsigned blocks) {
  __shared__ __align__(16) attn_f32x4 merge_o[2][kMergeParts][kMergeItems];
  __shared__ float merge_ml[2][kMergeParts][kMergeItems];
  const unsigned unit = blockIdx.x / blocks;
  const unsigned seg = unit / a.tiles, tile = unit - seg * a.tiles;
  const unsigned rows = static_cast<unsigned>(a.length) * static_cast<unsigned>(a.groups);
  const unsigned row0 = tile * a.tile_rows;
  const int rows_here = static_cast<int>(min(rows - row0, static_cast<unsigned>(a.tile_rows)));
  const int local = threadIdx.x % kMergeItems, part = threadIdx.x / kMergeItems;
  const int item = static_cast<int>(blockIdx.x - unit * blocks) * kMergeItems + local;
  const int r = item / (D / 8), c = item - r * (D / 8);
  const bool valid = r < rows_here;
  const int64_t first = static_cast<int64_t>(unit) * a.splits * a.tile_rows + (valid ? r : 0);
  float m[LOADS], l[LOADS];
  attn_f32x4 x[LOADS], y[LOADS];
  auto load = [&](int k0) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int k = k0 + i * kMergeParts;
      const int64_t at = first + static_cast<int64_t>(k < static_cast<int>(a.splits) ? k : 0) * a.tile_rows;
      m[i] = a.part_ml[at * 2];
      l[i] = a.part_ml[at * 2 + 1];
      x[i] = *reinterpret_cast<const attn_f32x4*>(a.part_o + at * D + 8 * c);
      y[i] = *reinterpret_cast<const attn_f32x4*>(a.part_o + at * D + 8 * c + 4);
    }
  };
  load(part);
  const int needed = tile_keys(a, seg, row0, row0 + rows_here - 1).needed;
  if (needed <= 1) return;  // the first launch wrote this tile's output
  float top = kNegInf, total = 0.0f, o[8] = {};
  auto fold = [&](float state_m, float state_l, const attn_f32x4& lo, const attn_f32x4& hi) {
    if (state_m == kNegInf && state_l == 0.0f) return;  // saw no key
    const float higher = fmaxf(top, state_m);
    const float ws = top == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(top - higher);
    const float wo = state_m == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(state_m - higher);
    total = __builtin_fmaf(wo, state_l, total * ws);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o[e] = __builtin_fmaf(wo, lo[e], o[e] * ws);
      o[4 + e] = __builtin_fmaf(wo, hi[e], o[4 + e] * ws);
    }
    top = higher;
  };
  for (int k0 = part; k0 < needed; k0 += kMergeParts * LOADS) {
    if (k0 != part) load(k0);
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
      if (k0 + i * kMergeParts < needed) fold(m[i], l[i], x[i], y[i]);
  }
  merge_ml[0][part][local] = top;
  merge_ml[1][part][local] = total;
  merge_o[0][part][local] = attn_f32x4{o[0], o[1], o[2], o[3]};
  merge_o[1][part][local] = attn_f32x4{o[4], o[5], o[6], o[7]};
  __syncthreads();
  if (part != 0 || !valid) return;
#pragma unroll
  for (int p = 1; p < kMergeParts; ++p)
    fold(merge_ml[0][p][local], merge_ml[1][p][local], merge_o[0][p][local], merge_o[1][p][local]);
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] *= inv;
  *reinterpret_cast<attn_u32x4*>(paged_output<T, D>(a, seg, row0 + r) + 8 * c) = pack8<T>(o);
}

struct PagedPlan {
  bool tile_kernel;
  int waves, tile_rows;  // of a workgroup, of a tile's partial states
  int64_t tiles, units, splits, chunk;
};

// Which kernel runs and how many chunks the keys get: the choice with the least estimated time,
//   call + round R + p (step R + share S) [+ merge + megabyte M + state N, when the keys are split],
// where a chunk is p steps (a unit of 32 keys a wave), S workgroups share a compute unit, R rounds of
// them follow one another (`resident` to a compute unit), M is the MB of partial states written and
// read, and a thread of the merge loads N states. The constants (us) are a least-squares fit to measured
// calls (1 to 1,000 queries of 1 to 128 segments onto 100 to 130,000 rows, each kernel, 1 to 64 chunks),
// made when P had two pieces. With three, 17,944 such calls take 6 to 9% longer than estimated (median),
// 7% about that; over their 1,077 shapes the choice takes 0.6% longer than the best one, 15% at most.
// Constants fitted anew choose no better (0.5%). `resident` is a parameter of the fit like the others:
// the registers let five workgroups of four waves share a compute unit at d64 and four at d128, and a
// fit with these numbers comes to 0.6% too. (Rules by the number of workgroups alone take 9% longer,
// up to twice as long: 8 queries of 16 requests onto 300 rows, 4 heads, G6, d256, 21 us against 12; 192
// queries of one onto 9,000 rows 175 against 99.)
struct PagedCost {
  bool tile_kernel;
  int waves, resident;
  double call, round, step, share;
};
struct MergeCost {
  double call, megabyte, state;
};
constexpr PagedCost kPagedCosts[3][3] = {  // d64, d128, d256
    {{false, 4, 4, 4.2, 0.0, 0.446, 0.226},
     {false, 8, 2, 4.5, 0.66, 0.375, 0.48},
     {true, 4, 4, 5.1, 0.0, 0.455, 0.353}},
    {{false, 4, 3, 4.4, 0.0, 0.545, 0.344},
     {false, 8, 2, 4.4, 1.1, 0.2, 0.94},
     {true, 4, 3, 6.0, 0.0, 0.415, 0.62}},
    {{false, 4, 2, 5.1, 1.1, 0.624, 0.88},
     {false, 8, 1, 3.3, 3.3, 2.27, 0.0},
     {true, 4, 2, 8.75, 0.0, 0.632, 1.12}}};
constexpr MergeCost kMergeCosts[3] = {{2.1, 0.34, 0.23}, {2.3, 0.26, 0.24}, {2.45, 0.27, 0.21}};
constexpr int kSplits[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64};
constexpr unsigned kComputeUnits = 256, kMostSplitGroups = 4096;  // (more of them need no splitting)

// Chunks' states that a thread of the merge loads together.
int merge_loads(int64_t splits) {
  return splits <= 2 * kMergeParts ? 2 : splits <= 5 * kMergeParts ? 5 : 8;
}

PagedPlan least_cost(int64_t segments, int64_t groups, int64_t length, int64_t max_keys, int64_t dim) {
  const int row = dim == 64 ? 0 : dim == 128 ? 1 : 2;
  const int64_t rows = length * groups;
  const MergeCost& merge = kMergeCosts[row];
  PagedPlan best{};
  double least = HUGE_VAL;
  for (const PagedCost& cost : kPagedCosts[row]) {
    if (cost.tile_kernel && rows <= kSmallRows) continue;
    PagedPlan p{};
    p.tile_kernel = cost.tile_kernel;
    p.waves = cost.waves;
    const int64_t tile = p.tile_kernel ? kTileRows : kSmallRows;
    p.tile_rows = static_cast<int>(std::min(rows, tile));
    p.tiles = ceil_div(rows, tile);
    p.units = segments * p.tiles;
    const unsigned units = static_cast<unsigned>(std::min<int64_t>(p.units, INT32_MAX));
    const unsigned step = static_cast<unsigned>(kUnit * p.waves);
    const unsigned steps = std::max(1u, (static_cast<unsigned>(max_keys) + step - 1) / step);
    const double state_megabytes = 8e-6 * static_cast<double>(p.tile_rows * dim);
    for (const unsigned wanted : kSplits) {
      const unsigned parts = std::min(steps, wanted), per = (steps + parts - 1) / parts;
      const unsigned splits = (steps + per - 1) / per;
      if (splits > 1 && units > kMostSplitGroups / splits) break;
      if (splits > 4 && p.waves > kAttnWaves) break;  // (never the best, and past the fit)
      const unsigned workgroups = units * splits, resident = kComputeUnits * cost.resident;
      const unsigned rounds = (workgroups + resident - 1) / resident;
      const unsigned shares = (workgroups + kComputeUnits - 1) / kComputeUnits;
      double time = cost.call + cost.round * rounds + per * (cost.step * rounds + cost.share * shares);
      if (splits > 1) {
        const int loads = merge_loads(splits);
        time += merge.call + merge.megabyte * state_megabytes * workgroups +
                merge.state * static_cast<double>(ceil_div(splits, loads * kMergeParts) * loads);
      }
      if (time < least) {
        least = time;
        p.splits = splits;
        p.chunk = static_cast<int64_t>(per) * step;
        best = p;
      }
      if (wanted >= steps) break;
    }
  }
  return best;
}

// The query for the workspace's size and the launch behind it plan the same sizes: the second takes
// the thread's last plan (0.15 us of a call's 7 us of host work).
PagedPlan plan_paged(int64_t segments, int64_t groups, int64_t length, int64_t max_keys, int64_t dim) {
  thread_local int64_t sizes[5] = {};
  thread_local PagedPlan plan;
  const int64_t now[5] = {segments, groups, length, max_keys, dim};
  if (!std::equal(now, now + 5, sizes)) {
    plan = least_cost(segments, groups, length, max_keys, dim);
    std::copy(now, now + 5, sizes);
  }
  return plan;
}

size_t plan_bytes(const PagedPlan& p, int64_t dim) {
  if (p.splits == 1) return 0;
  return static_cast<size_t>(p.units * p.splits * p.tile_rows) * static_cast<size_t>(dim + 2) * 4;
}

template <typename T, int D>
int launch_merge(const PagedAttnArgs& args, const PagedPlan& plan, hipStream_t stream) {
  if (plan.splits == 1) return LR_OK;
  const unsigned blocks =
      static_cast<unsigned>(ceil_div(static_cast<int64_t>(plan.tile_rows) * (D / 8), kMergeItems));
  auto merge = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(plan.units) * blocks), dim3(kAttnThreads),
                       0, stream, args, blocks);
  };
  const int loads = merge_loads(plan.splits);
  if (loads == 2) merge(paged_merge_kernel<T, D, 2>);
  else if (loads == 5) merge(paged_merge_kernel<T, D, 5>);
  else merge(paged_merge_kernel<T, D, 8>);
  return check_launch("paged_attention merge");
}

template <typename T, int D>
int launch_paged(const PagedAttnArgs& args, const PagedPlan& plan, hipStream_t stream) {
  auto attend = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(plan.units * plan.splits)),
                       dim3(static_cast<unsigned>(64 * plan.waves)), 0, stream, args);
  };
  if (plan.tile_kernel) attend(paged_tile_kernel<T, D>);
  else if (plan.waves == kAttnWaves) attend(paged_attention_kernel<T, D, kAttnWaves>);
  else attend(paged_attention_kernel<T, D, 2 * kAttnWaves>);
  if (int status = check_launch("paged_attention")) return status;
  return launch_merge<T, D>(args, plan, stream);
}

}  // namespace
}  // namespace lr

using namespace lr;

extern "C" size_t lr_paged_attention_workspace_bytes(int64_t segments, int64_t groups,
                                                     int64_t length, int64_t max_keys,
                                                     int64_t dim) {
  if (segments <= 0 || groups <= 0 || length <= 0 || max_keys < 0 || max_keys > INT32_MAX / 2 || dim <= 0)
    return 0;
  return plan_bytes(plan_paged(segments, groups, length, max_keys, dim), dim);
}

extern "C" int lr_paged_attention_plan(int64_t segments, int64_t groups, int64_t length,
                                       int64_t max_keys, int64_t dim, int64_t* plan) {
  clear_error();
  LR_REQUIRE(dim == 64 || dim == 128 || dim == 256, "Head dimension must be 64, 128 or 256");
  LR_REQUIRE(segments > 0 && groups > 0 && length > 0 && max_keys >= 0 &&
                 max_keys <= INT32_MAX / 2 && plan,
             "Empty attention dimensions");
  const PagedPlan p = plan_paged(segments, groups, length, max_keys, dim);
  plan[0] = p.tile_kernel ? kTileRows : kSmallRows;
  plan[1] = p.waves;
  plan[2] = p.splits;
  return LR_OK;
}

extern "C" int lr_paged_attention(const void* queries, const int64_t* query_strides,
                                  const void* pages, int64_t page_count, int64_t page_size,
                                  const int32_t* table, int64_t max_pages, const int32_t* lengths,
                                  int64_t batch, int64_t kv_heads, int64_t groups, int64_t length,
                                  int64_t dim, int dtype, int64_t max_keys, const int32_t* counts,
                                  float scale, void* out, void* workspace, size_t workspace_size,
                                  void* stream) {
  clear_error();
  LR_REQUIRE(dtype == LR_DTYPE_BF16 || dtype == LR_DTYPE_F16,
             "FlashAttention only supports fp16 and bf16 data type");
  LR_REQUIRE(batch > 0 && kv_heads > 0 && groups > 0 && length > 0, "Empty attention dimensions");
  LR_REQUIRE(batch <= INT32_MAX / kv_heads && kv_heads <= INT32_MAX / groups &&
                 length <= (INT32_MAX / 2) / groups,
             "Attention grid too large");
  const int64_t segments = batch * kv_heads;
  if (int status = check_paged(pages, page_count, page_size, dim, table, max_pages, lengths, segments))
    return status;
  LR_REQUIRE(max_keys >= 0 && max_keys <= INT32_MAX / 2, "Invalid key lengths");
  LR_REQUIRE(scale > 0.0f && std::isfinite(scale), "Softmax scale must be positive");
  LR_REQUIRE(queries && query_strides && out, "Invalid attention buffers");
  const uintptr_t alignment =
      reinterpret_cast<uintptr_t>(queries) | reinterpret_cast<uintptr_t>(out) |
      static_cast<uintptr_t>((query_strides[0] | query_strides[1] | query_strides[2]) * 2);
  LR_REQUIRE(alignment % 16 == 0, "Attention operands must be 16-byte aligned");
  const PagedPlan plan = plan_paged(segments, groups, length, max_keys, dim);
  const size_t needed = plan_bytes(plan, dim);
  LR_REQUIRE(workspace_size >= needed && (needed == 0 || workspace != nullptr),
             "Attention workspace too small");
  LR_REQUIRE(needed == 0 || reinterpret_cast<uintptr_t>(workspace) % 256 == 0,
             "Attention workspace must be 256-byte aligned");
  // (the merge of a split call, of at most kMostSplitGroups parts, has fewer)
  LR_REQUIRE(launchable(plan.units * plan.splits, 64 * plan.waves), "Attention grid too large");

  PagedAttnArgs args{};
  args.queries = queries;
  args.q_batch = query_strides[0];
  args.q_head = query_strides[1];
  args.q_query = query_strides[2];
  args.cache = paged_cache(pages, page_count, page_size, table, max_pages, lengths);
  args.counts = counts;
  args.kv_heads = static_cast<int>(kv_heads);
  args.groups = static_cast<int>(groups);
  args.length = static_cast<int>(length);
  // keys there can be: what a table holds, of a pool that has pages
  args.max_keys = page_count == 0 ? 0 : static_cast<int>(std::min(max_keys, max_pages * page_size));
  args.segments = static_cast<unsigned>(segments);
  args.tiles = static_cast<unsigned>(plan.tiles);
  args.splits = static_cast<unsigned>(plan.splits);
  args.tile_rows = plan.tile_rows;
  args.chunk = static_cast<int>(plan.chunk);
  args.to_log2 = scale * kAttnLog2e;
  args.out = out;
  if (needed) {
    args.part_o = static_cast<float*>(workspace);  // first, as it is accessed 16 bytes at a time
    args.part_ml = args.part_o + plan.units * plan.splits * plan.tile_rows * dim;
  }
  return dispatch_dim(dim, [&]<int D>() {
    return dtype == LR_DTYPE_BF16 ? launch_paged<__bf16, D>(args, plan, as_stream(stream))
                                  : launch_paged<_Float16, D>(args, plan, as_stream(stream));
  });
}
