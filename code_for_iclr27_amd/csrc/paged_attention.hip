// Attention over the paged 4-bit KV cache (paged.hpp states its layout): `length` queries a head
// onto each segment's rows. Query i of a request sees the segment's lengths[s] rows and the first
// i + 1 of those appended behind them (counts[b], or `length`, rows): keys j <= lengths[s] + i.
// Queries at or past counts[b] output zeros, as does a query that sees no key.
//
// Work split: row = i * G + g numbers a segment's query rows; a workgroup of four waves owns a tile
// of 16 * NT rows and a chunk of keys, each wave every fourth unit of 32 keys. Codes go from memory
// to registers (16 bytes a lane: a block of one row), the conversion instruction makes them 16-bit
// values, and both products run on v_mfma_f32_16x16x32:
//   S^T = K Q^T   A: 16 keys, a lane's eight channels of one key. The contraction's channel order is
//                 free, so a lane's block stays where it was loaded. A lane gets one query's scores
//                 of 4 + 4 keys.
//   O^T += V^T P^T  B: the probabilities where S^T left them (the key order is free as well); A: the
//                 same keys of one channel, read transposed from the wave's V rows in LDS.
// The values are exact in the 16-bit type, and P (f32) enters as a sum of three bf16 pieces, 3 x 8
// bits by truncation, whose products with V are exact: scores, probabilities, sums and outputs are
// f32 throughout and only the output is rounded.
//
// The exponentials' reference moves when a row's maximum has outgrown it by 2^kSlack (the tile
// kernel of attention_tile.hip does the same). The waves' states meet in LDS; tiles whose keys span
// several chunks leave partial states, which a second launch merges.
//
// A masked key contributes nothing: its score becomes -inf, and a block of V that reads as NaN is
// kept out of the product and added to the rows that see its key (0 * NaN is NaN).

#include <algorithm>
#include <cmath>

#include "attention_common.hpp"
#include "lds_copy.hpp"
#include "paged.hpp"

namespace lr {
namespace {

typedef short paged_s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned paged_u32x2 __attribute__((ext_vector_type(2)));

constexpr int kUnit = 32;                  // keys of a wave's step
constexpr int kStep = kUnit * kAttnWaves;  // and of the workgroup's
constexpr float kPagedSlack = 4.0f;

struct PagedAttnArgs {
  const void* queries;  // element strides below; the last dimension is contiguous
  int64_t q_batch, q_head, q_query;
  PagedCache cache;
  const int32_t* counts;  // [batch] or NULL
  int kv_heads, groups, length;
  int max_keys;           // no key at or past it is visited
  unsigned tiles, splits;
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

// Two f32 values as sums of three bf16 pieces each, word `w` of the piece vectors: the top halves
// of x, of x minus that, and of what is left (the differences are exact, the last has 8 bits).
__device__ __forceinline__ void split_bf16(float x, float y, attn_u32x4 (&piece)[3], int w) {
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    const unsigned a = __builtin_bit_cast(unsigned, x), b = __builtin_bit_cast(unsigned, y);
    piece[i][w] = __builtin_amdgcn_perm(b, a, 0x07060302u);
    if (i == 2) break;
    x -= __builtin_bit_cast(float, a & 0xffff0000u);
    y -= __builtin_bit_cast(float, b & 0xffff0000u);
  }
}

// V rows in LDS: 16-byte chunk c of row r in slot c ^ x(r). Eight lanes that write one chunk of
// eight rows, and 32 lanes that read 16 columns of eight rows transposed, touch every bank once:
// four consecutive rows go to the four 64-byte quarters of a bank cycle (a d64 row is half of one),
// and groups of four rows to different 16-byte places of a quarter.
template <int D>
__device__ __forceinline__ int value_swizzle(int row) {
  const int quarter = D == 64 ? (row >> 1) & 1 : row & 3, group = (row >> 2) & 3;
  return quarter << 2 ^ ((group & 1) << 1 | group >> 1);
}

// Codes and scales of a unit: two blocks of 16 rows, a lane's words of one row each. Words 4 h ..
// 4 h + 3 (d256: h = 0, 1; else all) belong to one block of channels.
template <int D>
struct UnitCodes {
  static constexpr int kWords = D / 32, kBytes = D == 256 ? 2 : 1;
  unsigned k[2][kWords], v[2][kWords], ks[2][kBytes], vs[2][kBytes];
};

template <int D>
__device__ __forceinline__ void load_codes(unsigned (&words)[D / 32], const uint8_t* p) {
  if constexpr (D == 64) {
    const paged_u32x2 x = *reinterpret_cast<const paged_u32x2*>(p);
    words[0] = x[0], words[1] = x[1];
  } else {
#pragma unroll
    for (int half = 0; half < D / 128; ++half) {
      const attn_u32x4 x = load16(p + 64 * half);
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

__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <typename T, int D, int NT>
__global__ __launch_bounds__(kAttnThreads) __attribute__((amdgpu_waves_per_eu(
    D * NT <= 64 ? 4 : D * NT <= 128 ? 3 : D * NT <= 256 ? 2 : 1))) void paged_attention_kernel(PagedAttnArgs a) {
  using Vec = AttnVec<T>;
  using X8 = typename Vec::x8;
  using Codes = UnitCodes<D>;
  constexpr int KW = D / 32, DT = D / 16;
  constexpr int kRows = 16 * NT;
  constexpr int DH = D == 256 ? 128 : D;  // channels of V in LDS at a time
  constexpr int kHalves = D / DH, kHalfWords = DH / 32;
  __shared__ __align__(1024) uint16_t v_lds[kAttnWaves][kUnit * DH];
  __shared__ float wave_ml[kAttnWaves][16][2];

  const int lane = threadIdx.x & 63, m = lane & 15, j = lane >> 4;
  const int wave = static_cast<int>(wave_index());
  const unsigned unit = blockIdx.x / a.splits, split = blockIdx.x - unit * a.splits;
  const unsigned seg = unit / a.tiles, tile = unit - seg * a.tiles;
  const unsigned groups = static_cast<unsigned>(a.groups);
  const unsigned rows = static_cast<unsigned>(a.length) * groups;
  const unsigned row0 = tile * kRows;
  const int rows_here = static_cast<int>(min(rows - row0, static_cast<unsigned>(kRows)));
  const TileKeys keys = tile_keys(a, seg, row0, row0 + rows_here - 1);
  if (keys.needed == 0) {  // no visible key for any row of this tile: zeros
    if (split != 0) return;
    for (int item = threadIdx.x; item < rows_here * (D / 8); item += kAttnThreads) {
      const int r = item / (D / 8), c = item - r * (D / 8);
      *reinterpret_cast<attn_u32x4*>(paged_output<T, D>(a, seg, row0 + r) + 8 * c) =
          attn_u32x4{0u, 0u, 0u, 0u};
    }
    return;
  }
  if (static_cast<int>(split) >= keys.needed) return;  // uniform across the workgroup
  const int begin = static_cast<int>(split) * a.chunk;
  const int end = min(begin + a.chunk, keys.key_end);

  // Queries (B operand: row m of a tile, the channels of word w of lane group j) and the last key
  // that a lane's rows see; `all_see`: the last one that every row of the workgroup sees.
  X8 q[NT][KW];
  int limit[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const bool valid = 16 * t + m < rows_here;
    const unsigned row = row0 + (valid ? 16 * t + m : 0);
    const unsigned i = row / groups, g = row - i * groups;
    const unsigned b = seg / static_cast<unsigned>(a.kv_heads), h = seg - b * a.kv_heads;
    limit[t] = valid && static_cast<int>(i) < keys.count
                   ? min(keys.cached + static_cast<int>(i), keys.key_end - 1) : -1;
    const T* p = static_cast<const T*>(a.queries) + b * a.q_batch +
                 static_cast<int64_t>(h * groups + g) * a.q_head + i * a.q_query;
#pragma unroll
    for (int w = 0; w < KW; ++w) q[t][w] = __builtin_bit_cast(X8, load16(p + 8 * word_chunk<D>(j, w)));
  }
  const int all_see = static_cast<int>((row0 + rows_here - 1) / groups) < keys.count
                          ? min(keys.cached + static_cast<int>(row0 / groups), keys.key_end - 1)
                          : -1;

  const PagedCache& cache = a.cache;
  const __attribute__((address_space(4))) int32_t* table =
      (const __attribute__((address_space(4))) int32_t*)(cache.table +
                                                         static_cast<int64_t>(seg) * cache.max_pages);
  const int64_t page_bytes = Page<D>::bytes(1) << cache.shift;
  const int mask = (1 << cache.shift) - 1;
  // Page of 16 rows from `key` on (one page: page sizes are multiples of 16); -1: outside the pool.
  auto page_id = [&](int key) {
    const int id = table[min(key, keys.key_end - 1) >> cache.shift];
    return id >= 0 && id < cache.page_count ? id : -1;
  };
  // A page and a slot are the wave's, so addresses are scalar but for the lane's place in 16 rows.
  const unsigned lane_codes = m * Page<D>::kCodes + (D == 64 ? 8 : 16) * j;
  const unsigned lane_scale = m * Page<D>::kScales + (D == 64 ? j >> 1 : j);
  auto load = [&](Codes& u, int key0, int id0, int id1) {
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
      const int id = blk == 0 ? id0 : id1;
      const int slot = (key0 + 16 * blk) & mask;
      const uint8_t* page = reinterpret_cast<const uint8_t*>(
          uniform_address(cache.pages + (id < 0 ? 0 : id) * page_bytes));
      load_codes<D>(u.k[blk], page + Page<D>::codes(cache.shift, 0, slot) + lane_codes);
      load_codes<D>(u.v[blk], page + Page<D>::codes(cache.shift, 1, slot) + lane_codes);
#pragma unroll
      for (int i = 0; i < Codes::kBytes; ++i) {
        u.ks[blk][i] = page[Page<D>::scales(cache.shift, 0, slot) + 4 * i + lane_scale];
        u.vs[blk][i] = page[Page<D>::scales(cache.shift, 1, slot) + 4 * i + lane_scale];
      }
    }
  };

  float reference[NT], sum[NT];  // in exponents of two; a row's reference is the same in its four lanes
  attn_f32x4 out[NT][DT];
  char* const my_values = reinterpret_cast<char*>(&v_lds[wave][0]);
  uint32_t read_at;  // of the lane's transposed reads: row 4 j + m / 4, columns 4 (m % 4) .. + 3
  {
    const int row = 4 * j + (m >> 2), chunk = (m & 3) >> 1;
    read_at = lds_address(my_values) + row * (2 * DH) + 16 * (chunk ^ value_swizzle<DH>(row)) +
              8 * (m & 1);
  }
  auto write_values = [&](const Codes& u, int half) {
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
      char* row = my_values + (16 * blk + m) * (2 * DH);
#pragma unroll
      for (int w = 0; w < kHalfWords; ++w)
        *reinterpret_cast<attn_u32x4*>(row + 16 * (word_chunk<DH>(j, w) ^ value_swizzle<DH>(m))) =
            expand8<__bf16>(u.v[blk][kHalfWords * half + w],
                            scale_of(u.vs[blk][Codes::kBytes == 2 ? half : 0]));
    }
  };

  // The wave's units of the chunk. SAFE: blocks of V that read as NaN are kept out of the product
  // and added to the rows that see their key.
  auto pass = [&]<bool SAFE>() {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      reference[t] = kNegInf, sum[t] = 0.0f;
#pragma unroll
      for (int ct = 0; ct < DT; ++ct) out[t][ct] = attn_f32x4{0.f, 0.f, 0.f, 0.f};
    }
    int key = begin + kUnit * wave;
    if (key >= end) return;
    Codes u;
    int id0 = page_id(key), id1 = page_id(key + 16);
    load(u, key, id0, id1);
    while (true) {
      const bool more = key + kStep < end;
      const int next0 = page_id(key + kStep), next1 = page_id(key + kStep + 16);
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
#pragma unroll 1
        for (int left = 0; left < kUnit; ++left) {
#pragma unroll
          for (int i = 0; i < Codes::kBytes; ++i)
#pragma unroll
            for (int b = 0; b < 4; ++b) {  // the lane that holds block b + 4 i of row `left`
              const int from = (D == 64 ? 2 * b : b) * 16 + (left & 15);
              if (D == 64 && b >= 2) continue;
              const unsigned byte = __shfl(left < 16 ? u.vs[0][i] : u.vs[1][i], from);
              if (byte != kScaleNaN) continue;
#pragma unroll
              for (int t = 0; t < NT; ++t)
                if (key + left <= limit[t])
#pragma unroll
                  for (int r = 0; r < 4; ++r) {
                    out[t][2 * (b + 4 * i)][r] = __builtin_nanf("");
                    out[t][2 * (b + 4 * i) + 1][r] = __builtin_nanf("");
                  }
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
      // V rows to LDS (the last unit's reads are done: a wave's LDS accesses stay in order)
      write_values(u, 0);
      // S^T
      attn_f32x4 s[NT][2];
#pragma unroll
      for (int blk = 0; blk < 2; ++blk) {
#pragma unroll
        for (int t = 0; t < NT; ++t) s[t][blk] = attn_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < KW; ++w) {
          const X8 k = __builtin_bit_cast(
              X8, expand8<T>(u.k[blk][w], scale_of(u.ks[blk][Codes::kBytes == 2 ? w / 4 : 0])));
#pragma unroll
          for (int t = 0; t < NT; ++t) s[t][blk] = Vec::mfma(k, q[t][w], s[t][blk]);
        }
      }
      Codes here;  // d256: the second half's codes of V outlive the next unit's loads
      if constexpr (kHalves == 2) here = u;
      if (more) load(u, key + kStep, next0, next1);
      if (key + kUnit - 1 > all_see || id0 < 0 || id1 < 0) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int blk = 0; blk < 2; ++blk)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (key + 16 * blk + 4 * j + r > limit[t] || (blk == 0 ? id0 : id1) < 0)
                s[t][blk][r] = kNegInf;
      }
      attn_u32x4 piece[NT][3];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float top = kNegInf;
#pragma unroll
        for (int r = 0; r < 4; ++r) top = fmaxf(fmaxf(top, s[t][0][r]), s[t][1][r]);
        LanePair pair = lane_pair<16>(top);
        pair = lane_pair<32>(fmaxf(pair.first, pair.second));
        top = fmaxf(pair.first, pair.second) * a.to_log2;
        if (__any(top > reference[t] + kPagedSlack)) {
          const float raised = fmaxf(reference[t], top);
          const float factor =
              reference[t] == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(reference[t] - raised);
          sum[t] *= factor;
#pragma unroll
          for (int ct = 0; ct < DT; ++ct)
#pragma unroll
            for (int r = 0; r < 4; ++r) out[t][ct][r] *= factor;
          reference[t] = raised;
        }
        const float base = reference[t] == kNegInf ? 0.0f : reference[t];
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][e / 4][e % 4], a.to_log2, -base));
          sum[t] += p[e];
        }
#pragma unroll
        for (int w = 0; w < 4; ++w) split_bf16(p[2 * w], p[2 * w + 1], piece[t], w);
      }
      // O^T += V^T P^T
#pragma unroll
      for (int half = 0; half < kHalves; ++half) {
        if (half > 0) {
          wave_fence();
          if constexpr (kHalves == 2) write_values(here, 1);
        }
        wave_fence();
#pragma unroll
        for (int c = 0; c < DH / 16; ++c) {
          const uint32_t at = read_at ^ (32 * c);
          auto read = [&](uint32_t p) {
            return __builtin_bit_cast(paged_u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) paged_s16x4*)(uintptr_t)p));
          };
          const paged_u32x2 lo = read(at), hi = read(at + 16 * (2 * DH));
          const attn_bf16x8 v = __builtin_bit_cast(attn_bf16x8, attn_u32x4{lo[0], lo[1], hi[0], hi[1]});
          const int ct = DH / 16 * half + c;
#pragma unroll
          for (int i = 0; i < 3; ++i)
#pragma unroll
            for (int t = 0; t < NT; ++t)
              out[t][ct] = AttnVec<__bf16>::mfma(v, __builtin_bit_cast(attn_bf16x8, piece[t][i]), out[t][ct]);
        }
      }
      wave_fence();
      if (!more) break;
      key += kStep;
      id0 = next0, id1 = next1;
    }
  };
  pass.template operator()<false>();
  // 0 * NaN is NaN: a wave with a sum that is not finite takes its keys again.
  float poison = 0.0f;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int ct = 0; ct < DT; ++ct)
#pragma unroll
      for (int r = 0; r < 4; ++r) poison = __builtin_fmaf(out[t][ct][r], 0.0f, poison);
  if (__any(poison != poison)) pass.template operator()<true>();

#pragma unroll
  for (int t = 0; t < NT; ++t) {
    LanePair pair = lane_pair<16>(sum[t]);
    pair = lane_pair<32>(pair.first + pair.second);
    sum[t] = pair.first + pair.second;
  }
  // Wave states to LDS, 16 rows and DH channels at a time: 16-byte chunk c of row r in slot c ^ r.
  constexpr int kItems = 16 * (DH / 8);
  const int64_t slot = (static_cast<int64_t>(unit) * a.splits + split) * a.tile_rows;
#pragma unroll
  for (int step = 0; step < NT * kHalves; ++step) {
    const int t = step / kHalves, half = step % kHalves;
    if (16 * t >= rows_here) break;
    __syncthreads();
    float* const mine = reinterpret_cast<float*>(my_values) + m * DH;
#pragma unroll
    for (int c = 0; c < DH / 16; ++c)
      *reinterpret_cast<attn_f32x4*>(mine + 4 * ((4 * c + j) ^ m)) = out[t][DH / 16 * half + c];
    if (j == 0 && half == 0) {
      wave_ml[wave][m][0] = reference[t];
      wave_ml[wave][m][1] = sum[t];
    }
    __syncthreads();
    for (int item = threadIdx.x; item < kItems; item += kAttnThreads) {
      const int r = item / (DH / 8), c = item - r * (DH / 8);
      if (16 * t + r >= rows_here) break;
      float top = kNegInf, total = 0.0f, o[8] = {};
#pragma unroll
      for (int w = 0; w < kAttnWaves; ++w) top = fmaxf(top, wave_ml[w][r][0]);
#pragma unroll
      for (int w = 0; w < kAttnWaves; ++w) {
        if (wave_ml[w][r][0] == kNegInf && wave_ml[w][r][1] == 0.0f) continue;  // saw no key
        const float weight =
            wave_ml[w][r][0] == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(wave_ml[w][r][0] - top);
        total = __builtin_fmaf(weight, wave_ml[w][r][1], total);
        const float* wo = reinterpret_cast<const float*>(&v_lds[w][0]) + r * DH;
        const attn_f32x4 lo = *reinterpret_cast<const attn_f32x4*>(wo + 4 * ((2 * c) ^ r));
        const attn_f32x4 hi = *reinterpret_cast<const attn_f32x4*>(wo + 4 * ((2 * c + 1) ^ r));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          o[e] = __builtin_fmaf(weight, lo[e], o[e]);
          o[4 + e] = __builtin_fmaf(weight, hi[e], o[4 + e]);
        }
      }
      const int channel = DH * half + 8 * c;
      if (keys.needed == 1) {
        const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] *= inv;
        *reinterpret_cast<attn_u32x4*>(paged_output<T, D>(a, seg, row0 + 16 * t + r) + channel) =
            pack8<T>(o);
      } else {
        float* po = a.part_o + (slot + 16 * t + r) * D + channel;
        *reinterpret_cast<attn_f32x4*>(po) = attn_f32x4{o[0], o[1], o[2], o[3]};
        *reinterpret_cast<attn_f32x4*>(po + 4) = attn_f32x4{o[4], o[5], o[6], o[7]};
        if (channel == 0) {
          a.part_ml[(slot + 16 * t + r) * 2] = top;
          a.part_ml[(slot + 16 * t + r) * 2 + 1] = total;
        }
      }
    }
  }
}

// Second launch of a split call: a thread folds one (row, 8 channels) slice of every fourth chunk of
// a tile, a round of chunks' states loaded together; the four threads of a slice meet in LDS.
constexpr int kMergeItems = 64, kMergeParts = kAttnThreads / kMergeItems, kMergeLoads = 4;

template <typename T, int D>
__global__ __launch_bounds__(kAttnThreads) void paged_merge_kernel(PagedAttnArgs a, unsigned blocks) {
  __shared__ __align__(16) float merge_o[kMergeParts][kMergeItems][8];
  __shared__ float merge_ml[kMergeParts][kMergeItems][2];
  const unsigned unit = blockIdx.x / blocks;
  const unsigned seg = unit / a.tiles, tile = unit - seg * a.tiles;
  const unsigned rows = static_cast<unsigned>(a.length) * static_cast<unsigned>(a.groups);
  const unsigned row0 = tile * a.tile_rows;
  const int rows_here = static_cast<int>(min(rows - row0, static_cast<unsigned>(a.tile_rows)));
  const int needed = tile_keys(a, seg, row0, row0 + rows_here - 1).needed;
  if (needed <= 1) return;  // the first launch wrote this tile's output
  const int local = threadIdx.x % kMergeItems, part = threadIdx.x / kMergeItems;
  const int item = static_cast<int>(blockIdx.x - unit * blocks) * kMergeItems + local;
  const int r = item / (D / 8), c = item - r * (D / 8);
  const bool valid = r < rows_here;
  float top = kNegInf, total = 0.0f, o[8] = {};
  auto fold = [&](float m, float l, const attn_f32x4& x, const attn_f32x4& y) {
    if (m == kNegInf && l == 0.0f) return;  // saw no key
    const float higher = fmaxf(top, m);
    const float ws = top == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(top - higher);
    const float wo = m == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(m - higher);
    total = __builtin_fmaf(wo, l, total * ws);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o[e] = __builtin_fmaf(wo, x[e], o[e] * ws);
      o[4 + e] = __builtin_fmaf(wo, y[e], o[4 + e] * ws);
    }
    top = higher;
  };
  const int64_t first = static_cast<int64_t>(unit) * a.splits * a.tile_rows + (valid ? r : 0);
  for (int k0 = part; k0 < needed; k0 += kMergeParts * kMergeLoads) {
    float m[kMergeLoads], l[kMergeLoads];
    attn_f32x4 x[kMergeLoads], y[kMergeLoads];
#pragma unroll
    for (int i = 0; i < kMergeLoads; ++i) {
      const int k = k0 + i * kMergeParts;
      const int64_t at = first + static_cast<int64_t>(k < needed ? k : k0) * a.tile_rows;
      m[i] = k < needed ? a.part_ml[at * 2] : kNegInf;
      l[i] = k < needed ? a.part_ml[at * 2 + 1] : 0.0f;
      x[i] = *reinterpret_cast<const attn_f32x4*>(a.part_o + at * D + 8 * c);
      y[i] = *reinterpret_cast<const attn_f32x4*>(a.part_o + at * D + 8 * c + 4);
    }
#pragma unroll
    for (int i = 0; i < kMergeLoads; ++i) fold(m[i], l[i], x[i], y[i]);
  }
  merge_ml[part][local][0] = top;
  merge_ml[part][local][1] = total;
#pragma unroll
  for (int e = 0; e < 8; ++e) merge_o[part][local][e] = o[e];
  __syncthreads();
  if (part != 0 || !valid) return;
  for (int p = 1; p < kMergeParts; ++p) {
    const float* w = merge_o[p][local];
    fold(merge_ml[p][local][0], merge_ml[p][local][1], attn_f32x4{w[0], w[1], w[2], w[3]},
         attn_f32x4{w[4], w[5], w[6], w[7]});
  }
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] *= inv;
  *reinterpret_cast<attn_u32x4*>(paged_output<T, D>(a, seg, row0 + r) + 8 * c) = pack8<T>(o);
}

struct PagedPlan {
  int tiles_of_16;       // NT
  int tile_rows;
  int64_t tiles, units, splits, chunk;
};

PagedPlan plan_paged(int64_t segments, int64_t groups, int64_t length, int64_t max_keys, int64_t dim) {
  PagedPlan p{};
  const int64_t rows = length * groups;
  p.tiles_of_16 = rows <= 16 ? 1 : rows <= 32 || dim == 256 ? 2 : 4;
  p.tile_rows = static_cast<int>(std::min<int64_t>(rows, 16 * p.tiles_of_16));
  p.tiles = ceil_div(rows, 16 * p.tiles_of_16);
  p.units = segments * p.tiles;
  const int64_t steps = std::max<int64_t>(1, ceil_div(max_keys, kStep));
  const int64_t wanted = std::min(steps, ceil_div(1024, p.units));
  const int64_t per = ceil_div(steps, wanted);
  p.splits = ceil_div(steps, per);
  p.chunk = per * kStep;
  return p;
}

size_t plan_bytes(const PagedPlan& p, int64_t dim) {
  if (p.splits == 1) return 0;
  return static_cast<size_t>(p.units * p.splits * p.tile_rows) * static_cast<size_t>(dim + 2) * 4;
}

template <typename T, int D, int NT>
int launch_paged(const PagedAttnArgs& args, const PagedPlan& plan, hipStream_t stream) {
  hipLaunchKernelGGL((paged_attention_kernel<T, D, NT>),
                     dim3(static_cast<unsigned>(plan.units * plan.splits)), dim3(kAttnThreads), 0,
                     stream, args);
  if (int status = check_launch("paged_attention")) return status;
  if (plan.splits == 1) return LR_OK;
  const unsigned blocks =
      static_cast<unsigned>(ceil_div(static_cast<int64_t>(plan.tile_rows) * (D / 8), kMergeItems));
  hipLaunchKernelGGL((paged_merge_kernel<T, D>), dim3(static_cast<unsigned>(plan.units) * blocks),
                     dim3(kAttnThreads), 0, stream, args, blocks);
  return check_launch("paged_attention merge");
}

template <typename T, int D>
int launch_paged_rows(const PagedAttnArgs& args, const PagedPlan& plan, hipStream_t stream) {
  if (plan.tiles_of_16 == 1) return launch_paged<T, D, 1>(args, plan, stream);
  if (D == 256 || plan.tiles_of_16 == 2) return launch_paged<T, D, 2>(args, plan, stream);
  if constexpr (D != 256) return launch_paged<T, D, 4>(args, plan, stream);
  return LR_OK;
}

}  // namespace
}  // namespace lr

using namespace lr;

extern "C" size_t lr_paged_attention_workspace_bytes(int64_t segments, int64_t groups,
                                                     int64_t length, int64_t max_keys,
                                                     int64_t dim) {
  if (segments <= 0 || groups <= 0 || length <= 0 || max_keys < 0 || dim <= 0) return 0;
  return plan_bytes(plan_paged(segments, groups, length, max_keys, dim), dim);
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
  LR_REQUIRE(max_keys >= 0, "Invalid key lengths");
  LR_REQUIRE(scale > 0.0f && std::isfinite(scale), "Softmax scale must be positive");
  LR_REQUIRE(queries && query_strides && out, "Invalid attention buffers");
  const uintptr_t alignment =
      reinterpret_cast<uintptr_t>(queries) | reinterpret_cast<uintptr_t>(out) |
      static_cast<uintptr_t>((query_strides[0] | query_strides[1] | query_strides[2]) * 2);
  LR_REQUIRE(alignment % 16 == 0, "Attention operands must be 16-byte aligned");
  // keys there can be: what a table holds, of a pool that has pages
  max_keys = page_count == 0 ? 0 : std::min(max_keys, max_pages * page_size);
  const PagedPlan plan = plan_paged(segments, groups, length, max_keys, dim);
  const size_t needed = plan_bytes(plan, dim);
  LR_REQUIRE(workspace_size >= needed && (needed == 0 || workspace != nullptr),
             "Attention workspace too small");
  LR_REQUIRE(needed == 0 || reinterpret_cast<uintptr_t>(workspace) % 256 == 0,
             "Attention workspace must be 256-byte aligned");
  LR_REQUIRE(plan.units <= INT32_MAX / plan.splits &&
                 plan.units <= INT32_MAX / ceil_div(int64_t{plan.tile_rows} * dim / 8, kMergeItems),
             "Attention grid too large");

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
  args.max_keys = static_cast<int>(max_keys);
  args.tiles = static_cast<unsigned>(plan.tiles);
  args.splits = static_cast<unsigned>(plan.splits);
  args.tile_rows = plan.tile_rows;
  args.chunk = static_cast<int>(plan.chunk);
  args.to_log2 = scale * kAttnLog2e;
  args.out = out;
  if (needed) {
    args.part_ml = static_cast<float*>(workspace);
    args.part_o = args.part_ml + plan.units * plan.splits * plan.tile_rows * 2;
  }
  return dispatch_dim(dim, [&]<int D>() {
    return dtype == LR_DTYPE_BF16 ? launch_paged_rows<__bf16, D>(args, plan, as_stream(stream))
                                  : launch_paged_rows<_Float16, D>(args, plan, as_stream(stream));
  });
}
