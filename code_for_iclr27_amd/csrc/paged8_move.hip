// Rows into, out of and within the paged 8-bit KV cache (paged8.hpp states its layout and its codes).
//
// append: new K and V rows behind each segment's rows, K (and the step's queries) rotated to their
// positions on the way. The rotation pairs channels c and c + half; its products are rounded one by
// one (no fused multiply-add), in f32. A wave owns a token block's keys or values, as their scale
// depends on all of the block's rows: it has the new rows in registers, takes their largest magnitude
// over its lanes, and where that outgrows the scale of rows that are there already, moves these to the
// new one. (A scale a row would spare the decode step that, and cost attention a multiplication for
// each key in the place of one for sixteen, and 2 bytes a row.) Bound by memory: 8,192 tokens of 8 KV
// and 32 query heads, d128, 185 MB in 39 us (4.7 TB/s; a large copy reaches 5.0); a step of sixteen
// requests 4.5 to 5.5 us, the time of its chain of loads (a kernel of its own for single rows, D / 16 threads a
// row, took 5.3 for 5.2 then).
//
// read: the rows as 16- or 32-bit rows packed by segment, the layout of the other operators, with
// its cumulative lengths. Bound by memory: 488,000 rows of d128 as bf16, 381 MB in 63 to 72 us (5.3 to 6
// TB/s); 18,000 rows 6.1 us. Four packed rows a thread, which then fetches a quad of values once where
// four threads do, took 41.7 us for 38.8 (256,000 rows); loads that the caches do not keep, with the lines
// fetched four times, 63.8 for 51.9 (144,000 rows of d256).
//
// compact: the rows that stay, in order, into other pages, in one launch. The rows of a block come from
// several; it takes the largest of their scales. A wave has a chain of about nine dependent loads (5 us:
// the lengths, the searches, the tables) ahead of its copies (6 us), and there are four rounds of waves:
// 488,000 rows of d128, 258 MB read and written in 65 us (4.0 TB/s), 230,000 of d64 19 us. Moving codes to
// another scale one by one took 26 us for the 19, four rows' words of V each in the place of the first and
// the last row's 21 to 25, 16 or 64 rows of d128 a wave 77 to 82 for the 77; searches by one wave of the
// four, with its findings in LDS, the same, of 64 or 128 places a round 80, 86.

#include "attention_common.hpp"
#include "paged8.hpp"
#include "paged_move.hpp"

namespace lr {
namespace {

template <int CONTROL>
__device__ __forceinline__ float dpp_max(float x) {
  return fmaxf(x, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(
                      0, __builtin_bit_cast(int, x), CONTROL, 0xF, 0xF, false)));
}
// The largest of each 16 lanes' values, and of the wave's, in all of them.
__device__ __forceinline__ float row_max(float x) {
  return dpp_max<0x140>(dpp_max<0x141>(dpp_max<0x4E>(dpp_max<0xB1>(x))));
}
__device__ __forceinline__ float wave_max(float x) {
  LanePair pair = lane_pair<16>(row_max(x));
  pair = lane_pair<32>(fmaxf(pair.first, pair.second));
  return fmaxf(pair.first, pair.second);
}

// log2 of the scale for a largest magnitude.
__device__ __forceinline__ int scale_exponent(float top, ScaleRange range) {
  const int exponent = static_cast<int>((__builtin_bit_cast(unsigned, top) + 0x180000u) >> 23) - 135;
  return exponent < range.low ? range.low : exponent > range.high ? range.high : exponent;
}

// The largest finite magnitude of N elements.
template <int N>
__device__ __forceinline__ float finite_max(const float (&x)[N]) {
  float top = 0.0f;
#pragma unroll
  for (int e = 0; e < N; ++e) top = fmaxf(top, __builtin_fabsf(x[e]));  // (takes no NaN)
  if (top == __builtin_huge_valf()) {
    top = 0.0f;
#pragma unroll
    for (int e = 0; e < N; ++e)
      top = __builtin_fabsf(x[e]) < __builtin_huge_valf() ? fmaxf(top, __builtin_fabsf(x[e])) : top;
  }
  return top;
}

// An element's code at scale 2^exponent. Times 2^(-exponent - 120) a code is the exponent and the top
// three bits of the significand of an f32, with the small codes among its subnormal numbers, and the
// cut to whole codes drops the bits below.
__device__ __forceinline__ unsigned encode(float x, int exponent) {
  const unsigned bits = __builtin_bit_cast(unsigned, x), size = bits & 0x7fffffffu;
  const unsigned four = (size + 0x7ffffu + ((size >> 20) & 1u)) & 0xfff00000u;
  const float scaled = __builtin_ldexpf(__builtin_bit_cast(float, four), -exponent - 120);
  const unsigned code = min(__builtin_bit_cast(unsigned, scaled) >> 20, 0x7eu);
  return size >= 0x7f800000u ? kCodeNaN : code | (bits >> 24 & 0x80u);
}
__device__ __forceinline__ unsigned encode4(const float* x, int exponent) {
  return encode(x[0], exponent) | encode(x[1], exponent) << 8 | encode(x[2], exponent) << 16 |
         encode(x[3], exponent) << 24;
}

// Four codes at a scale 2^by times theirs: whole numbers of the smallest code before and, once cut,
// after, so that the conversion back has nothing to round (NaN becomes kCodeNaN).
__device__ __forceinline__ unsigned shift_codes(unsigned codes, int by) {
  typedef short Pair __attribute__((ext_vector_type(2)));
  const float down = scale_of(static_cast<unsigned>(127 + 9 - min(by, 32)));
  const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes, down, false);
  const auto b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes, down, true);
  Pair result{};
  result = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(result, __builtin_truncf(a[0]), __builtin_truncf(a[1]), 512.0f, false);
  result = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(result, __builtin_truncf(b[0]), __builtin_truncf(b[1]), 512.0f, true);
  return __builtin_bit_cast(unsigned, result);
}

// Four words of four codes, each word's bytes of one row, as words of one byte of each: a 4 x 4
// transposition.
__device__ __forceinline__ void transpose4(const unsigned (&in)[4], unsigned (&out)[4]) {
  const unsigned a = __builtin_amdgcn_perm(in[1], in[0], 0x05010400u);  // 0.0 1.0 0.1 1.1
  const unsigned b = __builtin_amdgcn_perm(in[1], in[0], 0x07030602u);
  const unsigned c = __builtin_amdgcn_perm(in[3], in[2], 0x05010400u);
  const unsigned d = __builtin_amdgcn_perm(in[3], in[2], 0x07030602u);
  out[0] = __builtin_amdgcn_perm(c, a, 0x05040100u);
  out[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
  out[2] = __builtin_amdgcn_perm(d, b, 0x05040100u);
  out[3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
}

// A token block that rows are appended to: rows [from, to) of it are new (none: from = to), `first` is
// the number of its row 0 among the new ones (negative where it has older rows), `id` its page as the
// table has it.
struct Target {
  int id, slot, from, to, first;  // slot: of the block's row 0
};
__device__ __forceinline__ Target target_block(const AppendArgs& a, unsigned segment, unsigned b, unsigned n) {
  Target t{-1, 0, 0, 0, 0};
  const PagedCache& cache = a.cache;
  const int length = cache.lengths[segment];
  int count = static_cast<int>(a.added);
  if (a.counts != nullptr) count = max(0, min(count, a.counts[b]));
  const int64_t row = (static_cast<int64_t>(length) & ~int64_t{15}) + 16 * static_cast<int64_t>(n);
  if (length < 0 || row >= static_cast<int64_t>(cache.max_pages) << cache.shift) return t;
  const int64_t behind = static_cast<int64_t>(length) + count - row;  // past the last new row
  t.first = static_cast<int>(row - length);
  t.from = max(0, -t.first);
  t.to = behind < kTokens ? max(t.from, static_cast<int>(behind)) : kTokens;
  t.slot = static_cast<int>(row) & ((1 << cache.shift) - 1);
  t.id = cache.table[static_cast<int64_t>(segment) * cache.max_pages + (row >> cache.shift)];
  return t;
}
// Its page, or NULL where there is none; called behind the loads of the new rows, which do not wait for
// the table.
template <int D>
__device__ __forceinline__ uint8_t* target_page(const AppendArgs& a, const Target& t) {
  if (t.id < 0 || t.id >= a.cache.page_count) return nullptr;
  return a.cache.pages + static_cast<int64_t>(t.id) * (Page8<D>::bytes(1) << a.cache.shift);
}

// The exponent of a block's scale, written to its byte, and by how much older rows' codes move; `was`:
// the byte, of a block with older rows.
struct Scale {
  int exponent, by;
};
__device__ __forceinline__ Scale grow_scale(const AppendArgs& a, const Target& t, uint8_t* byte, unsigned was,
                                            float top) {
  Scale s{scale_exponent(wave_max(top), a.range), 0};
  if (t.from > 0) {
    const int old = static_cast<int>(was) - 127;
    s.by = max(0, s.exponent - old);
    s.exponent = max(s.exponent, old);
  }
  if ((threadIdx.x & 63) == 0) *byte = static_cast<uint8_t>(s.exponent + 127);
  return s;
}

// A chunk's eight channels rotated with its partner's.
__device__ __forceinline__ void rotate_pair(float (&x)[8], float (&y)[8], const float (&cosine)[8],
                                            const float (&sine)[8], bool known) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float xc = x[e] * cosine[e], ys = y[e] * sine[e], yc = y[e] * cosine[e], xs = x[e] * sine[e];
    x[e] = known ? xc - ys : __builtin_nanf("");
    y[e] = known ? yc + xs : __builtin_nanf("");
  }
}

// Eight elements of new rows or queries, each of which is read once. ONCE: the caches do not keep them, and
// have the more room for what the call writes; where a pair's two loads take whole cache lines or the row
// is one. 16,384 tokens (8 KV and 32 query heads, d128) 72 us for 83, behind a kernel that has just made
// them 139 for 155; 8,192 tokens 40.4 for 40.6 and 75.5 for 78.0, of d64 12.7 for 13.4 and 25.6 for 27.2.
// With 32 or 64 of the 128 channels rotated a line is taken in parts, by both loads: 42.8 for 41.4 and 79.6
// for 77.4. (The new rows' loads alone: 73 and 152 for the 16,384, the queries' 73 and 147. Queries written
// past the caches: 80 and 140, but 129 for 124 with a pass over them behind it.)
constexpr int kCacheLine = 128;
template <bool ONCE, typename T>
__device__ __forceinline__ Eight<T> load_eight(const T* p) {
  if constexpr (!ONCE) return *reinterpret_cast<const Eight<T>*>(p);
  Eight<T> x;
  if constexpr (sizeof(T) == 4) {
    x.lo = __builtin_nontemporal_load(reinterpret_cast<const move_f32x4*>(p));
    x.hi = __builtin_nontemporal_load(reinterpret_cast<const move_f32x4*>(p) + 1);
  } else {
    const move_u32x4 bits = __builtin_nontemporal_load(reinterpret_cast<const move_u32x4*>(p));
    x.x = __builtin_bit_cast(typename Eight<T>::vec, bits);
  }
  return x;
}

// The keys of a token block: a lane has eight channels and their partners (rotated: channels c and
// c + half; the others: half of them apart) of D / 64 rows.
template <typename T, int D, bool ONCE>
__device__ __forceinline__ void append_keys(const AppendArgs& a, unsigned segment, unsigned b, unsigned h,
                                            const Target& t) {
  constexpr int kPairs = D / 16, kGroups = 64 / kPairs, kRows = kTokens / kGroups;
  const int lane = threadIdx.x & 63, c = lane % kPairs, group = lane / kPairs;
  const int pairs = a.half / 8;
  const bool rotated = c < pairs;
  const int chunk[2] = {rotated ? c : c + pairs, rotated ? c + pairs : c + kPairs};
  const T* source = static_cast<const T*>(a.keys.base) + b * a.keys.batch + h * a.keys.head;
  const int64_t* positions = a.positions + static_cast<int64_t>(b) * a.added;
  Eight<T> raw[kRows][2];
  int64_t position[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int row = i * kGroups + group, at = t.first + row;
    if (row >= t.from && row < t.to) {
      raw[i][0] = load_eight<ONCE>(source + at * a.keys.row + 8 * chunk[0]);
      raw[i][1] = load_eight<ONCE>(source + at * a.keys.row + 8 * chunk[1]);
      position[i] = positions[at];
    }
  }
  uint8_t* const page = target_page<D>(a, t);
  if (page == nullptr) return;
  uint8_t* const byte = page + Page8<D>::scales(a.cache.shift, t.slot);
  const unsigned was = *byte;
  float x[kRows][2][8], top = 0.0f;
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int row = i * kGroups + group;
    const bool fresh = row >= t.from && row < t.to;
    if (fresh) {
      raw[i][0].get(x[i][0]);
      raw[i][1].get(x[i][1]);
      if (rotated) {
        float cosine[8], sine[8];
        const bool known = position[i] >= 0 && position[i] < a.table_rows;
        const int64_t at = (known ? position[i] : 0) * a.half + 8 * c;
        reinterpret_cast<const Eight<float>*>(a.cos + at)->get(cosine);
        reinterpret_cast<const Eight<float>*>(a.sin + at)->get(sine);
        rotate_pair(x[i][0], x[i][1], cosine, sine, known);
      }
      top = fmaxf(top, fmaxf(finite_max(x[i][0]), finite_max(x[i][1])));
      if (c == 0)
        *reinterpret_cast<float*>(page + Page8<D>::position(a.cache.shift, t.slot + row)) =
            static_cast<float>(position[i]);
    }
  }
  const Scale scale = grow_scale(a, t, byte, was, top);
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int row = i * kGroups + group;
    if (row >= t.to || (row < t.from && scale.by == 0)) continue;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      move_u32x2* const to = reinterpret_cast<move_u32x2*>(
          page + Page8<D>::key(t.slot + row, chunk[p] >> 1) + 8 * (chunk[p] & 1));
      if (row >= t.from) {
        *to = move_u32x2{encode4(&x[i][p][0], scale.exponent), encode4(&x[i][p][4], scale.exponent)};
      } else {
        const move_u32x2 old = *to;
        *to = move_u32x2{shift_codes(old[0], scale.by), shift_codes(old[1], scale.by)};
      }
    }
  }
}

// The values of a token block: a lane has eight channels of four rows, D / 128 times.
template <typename T, int D, bool ONCE>
__device__ __forceinline__ void append_values(const AppendArgs& a, unsigned segment, unsigned b, unsigned h,
                                              const Target& t) {
  constexpr int kChunks = D / 8, kTimes = D == 256 ? 2 : 1;
  const int lane = threadIdx.x & 63;
  const T* source = static_cast<const T*>(a.values.base) + b * a.values.batch + h * a.values.head;
  Eight<T> raw[kTimes][4];
  float top = 0.0f;
#pragma unroll
  for (int u = 0; u < kTimes; ++u) {
    const int c = (u * 64 + lane) % kChunks, quad = (u * 64 + lane) / kChunks;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = 4 * quad + r;
      if (row >= t.from && row < t.to)  // (d64: none for the last 32 lanes)
        raw[u][r] = load_eight<ONCE>(source + (t.first + row) * a.values.row + 8 * c);
    }
  }
  uint8_t* const page = target_page<D>(a, t);
  if (page == nullptr) return;
  uint8_t* const byte = page + Page8<D>::scales(a.cache.shift, t.slot) + 1;
  const unsigned was = *byte;
#pragma unroll
  for (int u = 0; u < kTimes; ++u) {
    const int quad = (u * 64 + lane) / kChunks;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = 4 * quad + r;
      if (row >= t.from && row < t.to) {
        float x[8];
        raw[u][r].get(x);
        top = fmaxf(top, finite_max(x));
      }
    }
  }
  const Scale scale = grow_scale(a, t, byte, was, top);
#pragma unroll
  for (int u = 0; u < kTimes; ++u) {
    const int c = (u * 64 + lane) % kChunks, quad = (u * 64 + lane) / kChunks;
    const int row0 = 4 * quad;
    const bool older = row0 < t.from && scale.by > 0;
    if (quad >= 4 || row0 >= t.to || (row0 + 4 <= t.from && !older)) continue;
    uint8_t* const to = page + Page8<D>::value(a.cache.shift, t.slot + row0) + 32 * c;
    unsigned word[4][2];  // a row's eight codes
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float x[8] = {};
      if (row0 + r >= t.from && row0 + r < t.to) raw[u][r].get(x);
      word[r][0] = encode4(x, scale.exponent);
      word[r][1] = encode4(x + 4, scale.exponent);
    }
    const bool whole = row0 >= t.from && row0 + 4 <= t.to;
    if (whole || older) {
      unsigned fresh = 0;  // bytes of the words that are new
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (row0 + r >= t.from && row0 + r < t.to) fresh |= 0xffu << (8 * r);
      const unsigned old_rows = row0 + 4 <= t.from ? ~0u : row0 >= t.from ? 0u : (1u << (8 * (t.from - row0))) - 1;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const unsigned rows[4] = {word[0][n], word[1][n], word[2][n], word[3][n]};
        unsigned codes[4];
        transpose4(rows, codes);
        move_u32x4* const place = reinterpret_cast<move_u32x4*>(to + 16 * n);
        if (!whole) {
          const move_u32x4 was = *place;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            codes[k] = (codes[k] & fresh) | (shift_codes(was[k], scale.by) & old_rows) |
                       (was[k] & ~(fresh | old_rows));
        }
        *place = move_u32x4{codes[0], codes[1], codes[2], codes[3]};
      }
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (row0 + r >= t.from && row0 + r < t.to)
#pragma unroll
          for (int e = 0; e < 8; ++e) to[4 * e + r] = static_cast<uint8_t>(word[r][e / 4] >> (8 * (e % 4)));
    }
  }
}

// Queries, rotated: D / 16 threads a row, each with a chunk and its partner, for the same chunks of HEADS
// heads, so that a cosine and sine are loaded once.
template <typename T, int D, int HEADS, bool ONCE>
__device__ __forceinline__ void rotate_queries(const AppendArgs& a, unsigned block) {
  constexpr int kRowThreads = D / 16, kUnits = kThreads / kRowThreads;
  const unsigned unit = block * kUnits + threadIdx.x / kRowThreads;
  const unsigned groups = (a.query_heads + HEADS - 1) / HEADS;
  const unsigned place = unit / groups, h0 = (unit - place * groups) * HEADS;
  const unsigned b = place / a.added, i = place - b * a.added;
  if (b >= a.batch) return;
  const int c = threadIdx.x % kRowThreads, pairs = a.half / 8;
  const bool rotated = c < pairs;
  const int lo = rotated ? c : c + pairs, hi = rotated ? c + pairs : c + kRowThreads;
  const T* source = static_cast<const T*>(a.queries.base) + b * a.queries.batch + i * a.queries.row;
  Eight<T> first[HEADS], second[HEADS];
#pragma unroll
  for (int n = 0; n < HEADS; ++n) {
    const T* p = source + min(h0 + n, a.query_heads - 1) * a.queries.head;
    first[n] = load_eight<ONCE>(p + 8 * lo);
    second[n] = load_eight<ONCE>(p + 8 * hi);
  }
  const int64_t position = a.positions[static_cast<int64_t>(b) * a.added + i];
  const bool known = position >= 0 && position < a.table_rows;
  float cosine[8], sine[8];
  if (rotated) {
    const int64_t at = (known ? position : 0) * a.half + 8 * c;
    reinterpret_cast<const Eight<float>*>(a.cos + at)->get(cosine);
    reinterpret_cast<const Eight<float>*>(a.sin + at)->get(sine);
  }
#pragma unroll
  for (int n = 0; n < HEADS; ++n) {
    if (h0 + n >= a.query_heads) break;
    float x[8], y[8];
    first[n].get(x);
    second[n].get(y);
    if (rotated) rotate_pair(x, y, cosine, sine, known);
    T* out = static_cast<T*>(a.out_queries) +
             ((static_cast<int64_t>(b) * a.query_heads + h0 + n) * a.added + i) * D;
    Eight<T> result;
    result.set(x);
    *reinterpret_cast<Eight<T>*>(out + 8 * lo) = result;
    result.set(y);
    *reinterpret_cast<Eight<T>*>(out + 8 * hi) = result;
  }
}

// blocks: the keys', the values', the queries'. A wave takes a token block of one segment, consecutive
// ones those of consecutive heads.
template <typename T, int D, int HEADS, bool ONCE>
__global__ __launch_bounds__(kThreads) void paged8_append_kernel(AppendArgs a, unsigned blocks) {
  if (blockIdx.x >= 2 * a.kv_blocks) return rotate_queries<T, D, HEADS, ONCE>(a, blockIdx.x - 2 * a.kv_blocks);
  const bool keys = blockIdx.x < a.kv_blocks;
  const unsigned unit = __builtin_amdgcn_readfirstlane(
      (blockIdx.x - (keys ? 0 : a.kv_blocks)) * (kThreads / 64) + (threadIdx.x >> 6));
  const unsigned place = unit / a.kv_heads, h = unit - place * a.kv_heads;
  const unsigned b = place / blocks, n = place - b * blocks;
  if (b >= a.batch) return;
  const unsigned segment = b * a.kv_heads + h;
  const Target t = target_block(a, segment, b, n);
  if (t.from >= t.to) return;
  if (keys) append_keys<T, D, ONCE>(a, segment, b, h, t);
  else append_values<T, D, ONCE>(a, segment, b, h, t);
}

// ---------------------------------------------------------------------------------------
// Eight codes times 2^exponent, rounded once to T (codes are exact in f32).
template <typename T>
__device__ __forceinline__ Eight<T> eight_values(move_u32x2 codes, unsigned scale) {
  const float power = scale_of(scale);
  float x[8];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const auto lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes[w], power, false);
    const auto hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes[w], power, true);
    x[4 * w] = lo[0], x[4 * w + 1] = lo[1], x[4 * w + 2] = hi[0], x[4 * w + 3] = hi[1];
  }
  Eight<T> result;
  result.set(x);
  return result;
}

// Byte `row` of each of four words.
__device__ __forceinline__ unsigned gather_bytes(move_u32x4 words, int row) {
  const unsigned two = 0x0c0c0400u + 0x0101u * static_cast<unsigned>(row);
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(words[3], words[2], two),
                               __builtin_amdgcn_perm(words[1], words[0], two), 0x05040100u);
}

// The rows of a read that outgrows the last-level cache are written past it: they would only displace
// each other there. 275 MB of rows (d128, bf16) take 75 us so for 86, and with a pass over them behind it
// 149 for 157; 524 MB 150 for 157, and 284 for 292. Of fewer rows the next pass finds much in the cache
// and loses more than the read gains: 131 MB 32 us for 36, with the pass 71 for 64; 223 MB 65 for 68, and
// 126 for 121. (Two bodies: stores of two branches that differ in this alone are merged.)
constexpr int64_t kLastLevelCache = int64_t{256} << 20;

// To memory (PAST: past the caches).
template <bool PAST, typename T>
__device__ __forceinline__ void store(T* to, const T& x) {
  if constexpr (PAST) __builtin_nontemporal_store(x, to);
  else *to = x;
}
template <bool PAST, typename T>
__device__ __forceinline__ void store_eight(T* to, const Eight<T>& x) {
  if constexpr (sizeof(T) == 4) {
    store<PAST>(reinterpret_cast<move_f32x4*>(to), x.lo);
    store<PAST>(reinterpret_cast<move_f32x4*>(to) + 1, x.hi);
  } else {
    store<PAST>(reinterpret_cast<move_u32x4*>(to), __builtin_bit_cast(move_u32x4, x.x));
  }
}

// A workgroup takes 64 packed rows: the first wave finds each one's page and slot, then D / 8 threads
// a row expand eight channels each, four rows' loads in flight. (Of a value's word a row uses one byte:
// the rows beside it take the others from the same cache lines.)
template <typename T, int D, bool FUSED>
__global__ __launch_bounds__(kThreads) void paged8_read_kernel(ReadArgs a) {
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
        page = id * (Page8<D>::bytes(1) << cache.shift);
        slot = at & ((1 << cache.shift) - 1);
      }
    }
    row_page[threadIdx.x] = page;
    row_slot[threadIdx.x] = slot;
  }
  __syncthreads();
  const int c = threadIdx.x % kRowThreads, first = threadIdx.x / kRowThreads;
  auto expand = [&]<bool PAST>() {
#pragma unroll
    for (int r0 = 0; r0 < kRounds; r0 += kTogether) {
      move_u32x2 keys[kTogether];
      move_u32x4 values[kTogether][2];
      unsigned scales[kTogether];
#pragma unroll
      for (int i = 0; i < kTogether; ++i) {
        const int r = (r0 + i) * kRowsAtOnce + first, slot = row_slot[r];
        // (a row that is not there reads the pool's first one, and is not written)
        const uint8_t* p = cache.pages + (row_page[r] >= 0 ? row_page[r] : 0);
        keys[i] = *reinterpret_cast<const move_u32x2*>(p + Page8<D>::key(slot, c >> 1) + 8 * (c & 1));
        const uint8_t* q = p + Page8<D>::value(cache.shift, slot & ~3) + 32 * c;
        values[i][0] = *reinterpret_cast<const move_u32x4*>(q);
        values[i][1] = *reinterpret_cast<const move_u32x4*>(q + 16);
        scales[i] = *reinterpret_cast<const uint16_t*>(p + Page8<D>::scales(cache.shift, slot));
      }
#pragma unroll
      for (int i = 0; i < kTogether; ++i) {
        const int r = (r0 + i) * kRowsAtOnce + first;
        if (row_page[r] < 0) continue;
        const int64_t at = (row0 + r) * D + 8 * c;
        store_eight<PAST>(static_cast<T*>(a.keys) + at, eight_values<T>(keys[i], scales[i] & 255u));
        const move_u32x2 codes{gather_bytes(values[i][0], row_slot[r] & 3),
                               gather_bytes(values[i][1], row_slot[r] & 3)};
        store_eight<PAST>(static_cast<T*>(a.values) + at, eight_values<T>(codes, scales[i] >> 8));
      }
    }
  };
  if (a.total * static_cast<int64_t>(2 * D * sizeof(T)) > kLastLevelCache) expand.template operator()<true>();
  else expand.template operator()<false>();
  if (threadIdx.x < kReadRows && row_page[threadIdx.x] >= 0)
    a.positions[row0 + threadIdx.x] = *reinterpret_cast<const float*>(
        cache.pages + row_page[threadIdx.x] + Page8<D>::position(cache.shift, row_slot[threadIdx.x]));
}

// ---------------------------------------------------------------------------------------
// A wave moves 4096 channels' rows of a segment (16, 32 or 64): row r comes from row r + how many removed
// rows lie at or before it. The wave finds that number for its first and its last row, each lane its own
// between them; then all lanes move the codes of one token block after the other, all loads before the
// first store.
constexpr int move_rows(int64_t dim) { return static_cast<int>(4096 / dim); }

// PAST: codes are written past the caches, where the tables have room for a fifth of the last one or more.
// They displace no source rows there: 66 MB of rows of d256 29 us for 37, of d64 35 for 42, 129 MB of d128
// 65 for 70, 250 MB 118 for 124; read back at once 73 for 74, 74 for 82, 146 for 150 and 260 for 267. With
// 32 MB a read behind it loses more than it gains (d64: 37.3 us for 34.8 with the read, 17.9 for 18.9 alone).
template <int D, bool FUSED, bool PAST>
__global__ __launch_bounds__(kThreads) void paged8_compact_kernel(CompactArgs a) {
  constexpr int kWaveRows = move_rows(D), kMoveRows = kWaveRows * (kThreads / 64);
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
  const int row0 = chunk * kMoveRows + static_cast<int>(threadIdx.x >> 6) * kWaveRows;
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
  int64_t j = half_search(0, gone, lies_before(lane < 32 ? row0 : row0 + kWaveRows - 1));
  const int row = row0 + lane % kWaveRows, mask = (1 << cache.shift) - 1;
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
      from = id * (Page8<D>::bytes(1) << cache.shift);
      to = target * (Page8<D>::bytes(1) << cache.shift);
    }
  }
  const bool moves = to >= 0;
  const int from_slot = moves ? static_cast<int>(source) & mask : 0;
  if (!moves) from = 0;  // (reads the pool's first row)
  // keys: lane (row, 16 channels of 64); values: lane (four rows, four channels of 64). The four rows
  // come from one or two words of four rows, nearly always: the first row's and the last one's.
  constexpr int kBlocks = kWaveRows / kTokens, kLoads = D / 64;
  const int64_t from_key = from + Page8<D>::key(from_slot, 0);
  const int64_t from_value = (from + Page8<D>::value(cache.shift, from_slot & ~3)) | (from_slot & 3);
  const int c = lane & 15, quad = lane >> 4;
  auto value_words = [&](int64_t packed, int u) {
    return reinterpret_cast<const move_u32x4*>(cache.pages + (packed & ~int64_t{3}) + 256 * u + 16 * c);
  };
  move_u32x4 key_data[kBlocks][kLoads], value_data[kBlocks][2][kLoads];
  int64_t value_from[kBlocks][4];
#pragma unroll
  for (int block = 0; block < kBlocks; ++block) {
    const uint8_t* const p = cache.pages + __shfl(from_key, 16 * block + c) + 256 * quad;
#pragma unroll
    for (int u = 0; u < kLoads; ++u) key_data[block][u] = *reinterpret_cast<const move_u32x4*>(p + 1024 * u);
#pragma unroll
    for (int i = 0; i < 4; ++i) value_from[block][i] = __shfl(from_value, 16 * block + 4 * quad + i);
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      value_data[block][0][u] = *value_words(value_from[block][0], u);
      value_data[block][1][u] = *value_words(value_from[block][3], u);
    }
  }
  const float position = *reinterpret_cast<const float*>(cache.pages + from +
                                                         Page8<D>::position(cache.shift, from_slot));
  // a block's scales, and by how much the row's codes move to them
  const unsigned bytes = *reinterpret_cast<const uint16_t*>(cache.pages + from +
                                                            Page8<D>::scales(cache.shift, from_slot));
  int by[2];
  unsigned largest[2];
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const unsigned mine = bytes >> (8 * which) & 255u;
    largest[which] = static_cast<unsigned>(row_max(moves ? static_cast<float>(mine) : 0.0f));
    by[which] = moves ? static_cast<int>(largest[which] - mine) : 0;
  }
  if (moves && lane < kWaveRows) {
    uint8_t* const out = cache.pages + to;
    *reinterpret_cast<float*>(out + Page8<D>::position(cache.shift, row & mask)) = position;
    // (any of the block's rows that moves: they write the same)
    *reinterpret_cast<uint16_t*>(out + Page8<D>::scales(cache.shift, row & mask)) =
        static_cast<uint16_t>(largest[0] | largest[1] << 8);
  }
  const bool shifts = __any(by[0] > 0 || by[1] > 0);
#pragma unroll
  for (int block = 0; block < kBlocks; ++block) {
    {
      const int64_t row_to = __shfl(to, 16 * block + c);
      const int shift = __shfl(by[0], 16 * block + c);
      uint8_t* const p = cache.pages + row_to + Page8<D>::key((row0 + 16 * block + c) & mask, 0) + 256 * quad;
#pragma unroll
      for (int u = 0; u < kLoads; ++u) {
        if (shifts)
#pragma unroll
          for (int e = 0; e < 4; ++e) key_data[block][u][e] = shift_codes(key_data[block][u][e], shift);
        if (row_to >= 0) store<PAST>(reinterpret_cast<move_u32x4*>(p + 1024 * u), key_data[block][u]);
      }
    }
    int64_t row_to[4];
    int shift[4];
    bool whole = true, apart[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      row_to[i] = __shfl(to, 16 * block + 4 * quad + i);
      shift[i] = __shfl(by[1], 16 * block + 4 * quad + i);
      whole = whole && row_to[i] >= 0;
    }
    const int64_t* const packed = value_from[block];
    auto same = [&](int i, int k) { return ((packed[i] ^ packed[k]) & ~int64_t{3}) == 0; };
#pragma unroll
    for (int i = 0; i < 2; ++i) apart[i] = !same(1 + i, 0) && !same(1 + i, 3);
    const unsigned low = 0x0c0c0400u + static_cast<unsigned>(packed[0] & 3) + (static_cast<unsigned>(packed[1] & 3) << 8);
    const unsigned high = 0x04000c0cu + (static_cast<unsigned>(packed[2] & 3) << 16) +
                          (static_cast<unsigned>(packed[3] & 3) << 24);
    const int at = Page8<D>::value(cache.shift, (row0 + 16 * block + 4 * quad) & mask) + 16 * c;
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      move_u32x4 row[4] = {value_data[block][0][u], value_data[block][0][u], value_data[block][0][u],
                           value_data[block][1][u]};
#pragma unroll
      for (int i = 1; i < 3; ++i) {
        if (!same(i, 0)) row[i] = row[3];
        if (apart[i - 1]) row[i] = *value_words(packed[i], u);
      }
      move_u32x4 codes;
      if (shifts) {  // a row's four codes as a word, moved to their scale
        unsigned word[4], out[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) word[i] = shift_codes(gather_bytes(row[i], packed[i] & 3), shift[i]);
        transpose4(word, out);
        codes = move_u32x4{out[0], out[1], out[2], out[3]};
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          codes[e] = __builtin_amdgcn_perm(row[1][e], row[0][e], low) | __builtin_amdgcn_perm(row[3][e], row[2][e], high);
      }
      if (whole) {
        store<PAST>(reinterpret_cast<move_u32x4*>(cache.pages + row_to[0] + at + 256 * u), codes);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (row_to[i] >= 0)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              cache.pages[row_to[i] + at + 256 * u + 4 * e + i] = static_cast<uint8_t>(codes[e] >> (8 * i));
      }
    }
  }
}

}  // namespace
}  // namespace lr

using namespace lr;

extern "C" int64_t lr_paged8_page_bytes(int64_t page_size, int64_t dim) {
  return paged8_bytes(page_size, dim);
}

extern "C" int lr_paged8_append(const void* keys, const int64_t* key_strides, const void* values,
                                const int64_t* value_strides, const void* queries,
                                const int64_t* query_strides, void* out_queries, int64_t batch,
                                int64_t kv_heads, int64_t query_heads, int64_t added, int64_t dim,
                                int dtype, const int64_t* positions, const float* cos,
                                const float* sin, int64_t table_rows, int64_t half,
                                const int32_t* counts, void* pages, int64_t page_count,
                                int64_t page_size, const int32_t* table, int64_t max_pages,
                                const int32_t* lengths, void* stream) {
  auto launch = [&](AppendArgs& args) {
    args.range = dtype == LR_DTYPE_F16 ? kHalfRange8 : kWideRange8;
    // token blocks that a segment's new rows can touch, from any row of the first one on
    const int64_t token_blocks = (added + 2 * kTokens - 2) / kTokens;
    const int64_t kv_blocks = ceil_div(batch * kv_heads * token_blocks, kThreads / 64);
    // four heads a thread where there are enough rows to fill the chip with them
    const int64_t heads = static_cast<int64_t>(args.query_rows) >= 32768 ? 4 : 1;
    const int64_t per_block = kThreads / (dim / 16);
    const int64_t blocks = 2 * kv_blocks + ceil_div(batch * added * ceil_div(query_heads, heads), per_block);
    LR_REQUIRE(launchable(blocks, kThreads), "Appended grid too large");
    args.kv_blocks = static_cast<unsigned>(kv_blocks);
    return dispatch_type(dtype, [&]<typename T>() {
      return dispatch_dim(dim, [&]<int D>() {
        auto enqueue = [&](auto kernel) {
          hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0,
                             as_stream(stream), args, static_cast<unsigned>(token_blocks));
        };
        auto by_heads = [&]<bool ONCE>() {
          if (heads == 1) enqueue(paged8_append_kernel<T, D, 1, ONCE>);
          else enqueue(paged8_append_kernel<T, D, 4, ONCE>);
        };
        if (D * sizeof(T) <= kCacheLine || half * sizeof(T) % kCacheLine == 0) by_heads.template operator()<true>();
        else by_heads.template operator()<false>();
        return check_launch("paged8_append");
      });
    });
  };
  return append_paged(keys, key_strides, values, value_strides, queries, query_strides, out_queries,
                      batch, kv_heads, query_heads, added, dim, dtype, positions, cos, sin, table_rows,
                      half, counts, pages, page_count, page_size, table, max_pages, lengths, launch);
}

extern "C" int lr_paged8_read(const void* pages, int64_t page_count, int64_t page_size,
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
        if (fused) enqueue(paged8_read_kernel<T, D, true>);
        else enqueue(paged8_read_kernel<T, D, false>);
        return check_launch("paged8_read");
      });
    });
  };
  return read_paged(pages, page_count, page_size, table, max_pages, lengths, segments, dim, dtype, total,
                    keys, values, positions, cumulative, stream, launch);
}

extern "C" size_t lr_paged8_compact_workspace_bytes(int64_t segments) {
  return compact_paged_workspace(segments);
}

extern "C" int lr_paged8_compact(void* pages, int64_t page_count, int64_t page_size,
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
      auto by_sums = [&]<bool PAST>() {
        if (fused) enqueue(paged8_compact_kernel<D, true, PAST>);
        else enqueue(paged8_compact_kernel<D, false, PAST>);
      };
      const int64_t room = segments * std::min(max_pages, target_pages) * paged8_bytes(page_size, dim);
      if (room >= kLastLevelCache / 5) by_sums.template operator()<true>();
      else by_sums.template operator()<false>();
      return check_launch("paged8_compact");
    });
  };
  return compact_paged(move_rows(dim > 0 ? dim : 1) * (kThreads / 64), pages, page_count, page_size, table,
                       max_pages, lengths, segments, dim, removed, removed_count, target, target_pages,
                       new_lengths, workspace, workspace_size, stream, launch);
}
