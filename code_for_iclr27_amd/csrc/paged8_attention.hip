// Attention over the paged 8-bit KV cache (paged8.hpp states its layout): `length` queries a head onto
// each segment's rows. Query i of a request sees the segment's lengths[s] rows and the first i + 1 of
// those appended behind them (counts[b], or `length`, rows): keys j <= lengths[s] + i. Queries at or
// past counts[b] output zeros, as does a query that sees no key.
//
// Work split: row = i * G + g numbers a segment's query rows; a workgroup of four (eight) waves owns a
// tile of 16 rows and a chunk of keys, each wave every fourth (eighth) unit of 32 keys, two token
// blocks. Calls of many rows take tiles of 32 (paged8_tile_kernel); the plan has the rules. Codes go
// from memory to registers, 1 KB a load, the conversion instruction makes them 16-bit values, and both
// products run on v_mfma_f32_16x16x32:
//   S^T = K Q^T   A: 16 keys, a lane's eight channels of one key. A lane gets one query's scores of
//                 4 + 4 keys.
//   O^T += V^T P^T  B: the probabilities where S^T left them (the contraction's key order is free); A:
//                 the same 4 + 4 keys of one channel, two words of the page.
// Neither operand passes through LDS: the pages hold both as the matrix cores take them.
//
// The keys' scale is a factor of the conversion (bf16 queries) or of the scores (f16 queries: codes are
// exact in f16, their products with a large or small scale are not); the values' scale a factor of the
// conversion to bf16. P is f32 and stays f32: it enters as the sum of three bf16 pieces by truncation,
// the whole significand. Scores, exponentials, their sum and the products' sums are f32 throughout.
//
// The exponentials' reference moves when a row's maximum has outgrown it by 2^kPagedSlack. The waves'
// states meet in LDS; tiles whose keys span several chunks leave partial states, which a second launch
// merges.
//
// A masked key contributes nothing: its score becomes -inf, its P 0. As 0 * NaN is NaN, a wave that
// ends with a non-finite sum takes its keys again, with the codes of V that are NaN kept out of the
// product and added to the rows that see their key. So does one whose scores are so large that the
// reference's own rounding would show in the exponentials (kLargeReference).

#include "paged8.hpp"
#include "paged_attention.hpp"

namespace lr {
namespace {

// A wave's loads of codes: a uniform address and the lane's offset.
__device__ __forceinline__ attn_u32x4 load_piece(PagedBytes p) {
  return *(const __attribute__((address_space(1))) attn_u32x4*)p;
}
// The scales of the token block at `slot`: the keys' in the low byte, the values' in the next.
__device__ __forceinline__ unsigned block_scales(const uint8_t* page, int offset) {
  typedef const __attribute__((address_space(4))) unsigned* Words;
  return *(Words)(page + (offset & ~3)) >> (8 * (offset & 2));
}

// The rows of a quad of keys from `key` on that lie before `end`, as bytes of a word.
__device__ __forceinline__ unsigned quad_mask(int key, int end) {
  const int rows = end - key;
  return rows >= 4 ? ~0u : rows <= 0 ? 0u : (1u << (8 * rows)) - 1u;
}

// Elements of eight bf16 values that are NaN, as ones, and the values with zeros in their place.
__device__ __forceinline__ attn_u32x4 take_out_nan(attn_u32x4& v) {
  attn_u32x4 ones;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned low = (v[i] & 0x7fffu) > 0x7f80u ? 0xffffu : 0u;
    const unsigned high = (v[i] >> 16 & 0x7fffu) > 0x7f80u ? 0xffff0000u : 0u;
    ones[i] = (low | high) & 0x3f803f80u;
    v[i] &= ~(low | high);
  }
  return ones;
}

// Tiles of 16 rows: decode, and a few query rows.
template <typename T, int D, int WAVES>
__global__ __launch_bounds__(64 * WAVES) __attribute__((amdgpu_waves_per_eu(
    WAVES == 8 || D == 256 ? 2 : D == 64 ? 4 : 3)))
void paged8_attention_kernel(PagedAttnArgs a) {
  constexpr int kStep = kUnit * WAVES;  // keys of the workgroup's step
  constexpr int KL = D / 64;            // 16-byte loads of a lane for a token block's keys, or values
  constexpr int DT = D / 16;            // column tiles of the output
  using Vec = AttnVec<T>;
  using X8 = typename Vec::x8;
  __shared__ __align__(16) float state_lds[WAVES][kSmallRows * D];
  __shared__ float wave_ml[WAVES][kSmallRows][2];

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

  // Queries (B operand of step 2 n + h: channels 16 (4 n + j) + 8 h of row m), and the last key that
  // the lane's row sees.
  const TileRow row = tile_row(a, seg, row0 + (m < rows_here ? m : 0));
  const int limit = m < rows_here ? last_key(keys, row.query) : -1;
  const int all_see = all_rows_see(a, keys, row0, rows_here);
  attn_u32x4 q[2 * KL];
#pragma unroll
  for (int s = 0; s < 2 * KL; ++s)
    q[s] = load16(static_cast<const T*>(a.queries) + row.offset + 16 * (4 * (s >> 1) + j) + 8 * (s & 1));

  const int64_t page_bytes = Page8<D>::bytes(1) << cache.shift;
  const int mask = (1 << cache.shift) - 1;
  // Page of 16 rows from `key` on (one page: page sizes are multiples of 16); -1: outside the pool.
  auto page_id = [&](int key) { return in_pool(table[min(key, keys.key_end - 1) >> cache.shift]); };
  auto page_of = [&](int id) {
    return reinterpret_cast<const uint8_t*>(uniform_address(cache.pages + (id < 0 ? 0 : id) * page_bytes));
  };
  // A page and a slot are the wave's, so addresses are scalar but for the lane's place in 16 rows.
  attn_u32x4 k[2][KL], v[2][KL];
  unsigned scales[2];  // of the unit whose keys are loaded
  auto load_keys = [&](int key0, int id0, int id1) {
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
      const uint8_t* page = page_of(blk == 0 ? id0 : id1);
      const int slot = (key0 + 16 * blk) & mask;
#pragma unroll
      for (int n = 0; n < KL; ++n)
        k[blk][n] = load_piece((PagedBytes)page + (Page8<D>::key(slot, 4 * n) + 16 * lane));
      scales[blk] = block_scales(page, Page8<D>::scales(cache.shift, slot));
    }
  };
  // (words 4 n + e: channels 64 n + 4 m + e of keys 4 j .. 4 j + 3)
  auto load_values = [&](int key0, int id0, int id1) {
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
      const uint8_t* page = page_of(blk == 0 ? id0 : id1);
      const int slot = (key0 + 16 * blk) & mask;
#pragma unroll
      for (int n = 0; n < KL; ++n)
        v[blk][n] = load_piece((PagedBytes)page + (Page8<D>::value(cache.shift, slot) + 256 * n) +
                               (j * 4 * D + 16 * m));
    }
  };

  float reference, sum;  // in exponents of two; a row's reference is the same in its four lanes
  attn_f32x4 out[DT];
  // The wave's units of the chunk. SAFE: codes of V that are NaN are kept out of the product and added
  // to the rows that see their key, and no exponential exceeds its row's largest.
  auto pass = [&]<bool SAFE>() {
    reference = kNegInf, sum = 0.0f;
#pragma unroll
    for (int ct = 0; ct < DT; ++ct) out[ct] = attn_f32x4{0.f, 0.f, 0.f, 0.f};
    int key = begin + kUnit * wave;
    if (key >= end) return;
    int id0 = SAFE ? page_id(key) : first0, id1 = SAFE ? page_id(key + 16) : first1;
    load_keys(key, id0, id1);
    load_values(key, id0, id1);
    int next0 = page_id(key + kStep), next1 = page_id(key + kStep + 16);
    while (true) {
      // the unit after the next: its pages' ids arrive while this one is worked on
      const int later0 = page_id(key + 2 * kStep), later1 = page_id(key + 2 * kStep + 16);
      const bool more = key + kStep < end;
      const bool whole = key + kUnit <= keys.key_end && id0 >= 0 && id1 >= 0;
      const bool there1 = key + 16 < keys.key_end && id1 >= 0;
      const float key_scale[2] = {scale_of(scales[0] & 255u), scale_of(scales[1] & 255u)};
      const float value_scale[2] = {id0 >= 0 ? scale_of(scales[0] >> 8 & 255u) : 1.0f,
                                    there1 ? scale_of(scales[1] >> 8 & 255u) : 1.0f};
      // S^T
      attn_f32x4 s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int n = 0; n < 2 * KL; ++n)
#pragma unroll
        for (int blk = 0; blk < 2; ++blk) {
          const float scale = std::is_same<T, __bf16>::value ? key_scale[blk] : 1.0f;
          const paged_u32x2 lo = expand4<T>(k[blk][n >> 1][2 * (n & 1)], scale);
          const paged_u32x2 hi = expand4<T>(k[blk][n >> 1][2 * (n & 1) + 1], scale);
          s[blk] = Vec::mfma(__builtin_bit_cast(X8, attn_u32x4{lo[0], lo[1], hi[0], hi[1]}),
                             __builtin_bit_cast(X8, q[n]), s[blk]);
        }
      if (more) load_keys(key + kStep, next0, next1);
      if constexpr (!std::is_same<T, __bf16>::value)
#pragma unroll
        for (int blk = 0; blk < 2; ++blk)
#pragma unroll
          for (int r = 0; r < 4; ++r) s[blk][r] *= key_scale[blk];
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
      if (!whole) {  // rows that are not there: zeros for V
#pragma unroll
        for (int blk = 0; blk < 2; ++blk) {
          const unsigned rows = (blk == 0 ? id0 : id1) < 0 ? 0u : quad_mask(key + 16 * blk + 4 * j, keys.key_end);
#pragma unroll
          for (int n = 0; n < KL; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[blk][n][e] &= rows;
        }
      }
      // SAFE: ones for the lane's keys that its row sees
      attn_u32x4 seen{0u, 0u, 0u, 0u};
      if constexpr (SAFE)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (key + 16 * (i >> 2) + 4 * j + (i & 3) <= limit) seen[i >> 1] |= 0x3f80u << (16 * (i & 1));
      // O^T += V^T P^T
#pragma unroll
      for (int ct = 0; ct < DT; ++ct) {
        const paged_u32x2 lo = expand4<__bf16>(v[0][ct >> 2][ct & 3], value_scale[0]);
        const paged_u32x2 hi = expand4<__bf16>(v[1][ct >> 2][ct & 3], value_scale[1]);
        attn_u32x4 x{lo[0], lo[1], hi[0], hi[1]};
        if constexpr (SAFE) {
          const attn_u32x4 ones = take_out_nan(x);
          const attn_f32x4 count = AttnVec<__bf16>::mfma(__builtin_bit_cast(attn_bf16x8, ones),
                                                         __builtin_bit_cast(attn_bf16x8, seen),
                                                         attn_f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
          for (int r = 0; r < 4; ++r) out[ct][r] = count[r] > 0.0f ? __builtin_nanf("") : out[ct][r];
        }
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
          out[ct] = AttnVec<__bf16>::mfma(__builtin_bit_cast(attn_bf16x8, x),
                                          __builtin_bit_cast(attn_bf16x8, piece[i]), out[ct]);
      }
      if (!more) break;
      load_values(key + kStep, next0, next1);
      key += kStep;
      id0 = next0, id1 = next1;
      next0 = later0, next1 = later1;
    }
  };
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

  // Wave states to LDS: 16-byte chunk c of row r in slot c ^ r. (Lane (m, j) holds channels
  // 64 n + 16 j + 4 r + e of row m in out[4 n + e][r].)
  float* const mine = &state_lds[wave][m * D];
#pragma unroll
  for (int n = 0; n < KL; ++n)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      *reinterpret_cast<attn_f32x4*>(mine + 4 * ((16 * n + 4 * j + r) ^ m)) =
          attn_f32x4{out[4 * n][r], out[4 * n + 1][r], out[4 * n + 2][r], out[4 * n + 3][r]};
  if (j == 0) {
    wave_ml[wave][m][0] = reference;
    wave_ml[wave][m][1] = sum;
  }
  __syncthreads();
  const int64_t slot = (static_cast<int64_t>(place.unit) * a.splits + place.split) * a.tile_rows;
  for (int item = threadIdx.x; item < rows_here * (D / 8); item += 64 * WAVES) {
    const int r = item / (D / 8), c = item - r * (D / 8);
    auto state = [&](int w, attn_f32x4& lo, attn_f32x4& hi) {
      const float* wo = &state_lds[w][r * D];
      lo = *reinterpret_cast<const attn_f32x4*>(wo + 4 * ((2 * c) ^ r));
      hi = *reinterpret_cast<const attn_f32x4*>(wo + 4 * ((2 * c + 1) ^ r));
    };
    finish_item<T, D, WAVES>(a, seg, row0 + r, 8 * c, slot + r, keys.needed == 1,
                             [&](int w, int i) { return wave_ml[w][r][i]; }, state);
  }
}

// ---- Tiles of 32 rows -------------------------------------------------------------------------
// The same with v_mfma_f32_32x32x16 for calls of many rows: a lane holds one query's scores of 16
// keys, and an MFMA of twice the work takes no more of the wave's issue slots.

template <typename T, int D>
__global__ __launch_bounds__(kAttnThreads) __attribute__((amdgpu_waves_per_eu(D == 64 ? 4 : D == 128 ? 3 : 2)))
void paged8_tile_kernel(PagedAttnArgs a) {
  constexpr int KS = D / 16;      // MFMA steps over the head dimension
  constexpr int KL = D / 32;      // 16-byte loads of a lane for the unit's keys
  constexpr int DT = D / 32;      // column tiles of the output
  constexpr int VW = D == 64 ? 2 : 4;     // channels of a lane's load of values
  constexpr int VL = DT / VW;             // loads of a quad's values
  constexpr int kStep = kUnit * kAttnWaves;
  __shared__ __align__(16) attn_u32x4 q_lds[KS][64];
  __shared__ __align__(16) float state_lds[kAttnWaves][kTileRows * D / 2];
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

  // Queries (B operand of step 2 n + h: channels 16 (2 n + half) + 8 h of row `col`) in LDS for every
  // wave, and the last key that the lane's row sees.
  const TileRow row = tile_row(a, seg, row0 + (col < rows_here ? col : 0));
  const int limit = col < rows_here ? last_key(keys, row.query) : -1;
  const int all_see = all_rows_see(a, keys, row0, rows_here);
#pragma unroll
  for (int n = 0; n < KS / kAttnWaves; ++n) {
    const int ks = n * kAttnWaves + wave;
    q_lds[ks][lane] = load16(static_cast<const T*>(a.queries) + row.offset + 16 * (2 * (ks >> 1) + half) +
                             8 * (ks & 1));
  }

  const PagedCache& cache = a.cache;
  const PageIds table = page_table(cache, seg);
  const int64_t page_bytes = Page8<D>::bytes(1) << cache.shift;
  const int mask = (1 << cache.shift) - 1;
  auto page_id = [&](int key) {
    const int id = table[min(key, keys.key_end - 1) >> cache.shift];
    return id >= 0 && id < cache.page_count ? id : -1;
  };
  auto page_of = [&](int id) {
    return reinterpret_cast<const uint8_t*>(uniform_address(cache.pages + (id < 0 ? 0 : id) * page_bytes));
  };
  // Lane (key, half): 16 channels of every 32, chunks 2 n + half.
  attn_u32x4 k[KL];
  unsigned v[2][2][DT];  // a token block's quads half and 2 + half: the lane's channels
  unsigned scales[2];
  auto load_keys = [&](int key0, int id0, int id1) {
    const uint8_t *const page0 = page_of(id0), *const page1 = page_of(id1);
    const int slot0 = key0 & mask, slot1 = (key0 + 16) & mask;
    const PagedBytes block = col < 16 ? (PagedBytes)page0 + Page8<D>::key(slot0, 0)
                                      : (PagedBytes)page1 + Page8<D>::key(slot1, 0);
#pragma unroll
    for (int n = 0; n < KL; ++n) k[n] = load_piece(block + (512 * n + 256 * half + 16 * (col & 15)));
    scales[0] = block_scales(page0, Page8<D>::scales(cache.shift, slot0));
    scales[1] = block_scales(page1, Page8<D>::scales(cache.shift, slot1));
  };
  // (word VW n + e: channel 32 VW n + VW col + e)
  auto load_values = [&](int key0, int id0, int id1) {
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
      const uint8_t* page = page_of(blk == 0 ? id0 : id1);
      const int slot = (key0 + 16 * blk) & mask;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int n = 0; n < VL; ++n) {
          const PagedBytes p = (PagedBytes)page + (Page8<D>::value(cache.shift, slot) + 8 * D * i + 512 * n) +
                               (4 * D * half + 4 * VW * col);
          if constexpr (VW == 2) {
            const paged_u32x2 x = *(const __attribute__((address_space(1))) paged_u32x2*)p;
            v[blk][i][0] = x[0], v[blk][i][1] = x[1];
          } else {
            const attn_u32x4 x = load_piece(p);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[blk][i][4 * n + e] = x[e];
          }
        }
    }
  };

  float reference = kNegInf, sum = 0.0f;  // in exponents of two; the same in both halves
  paged_f32x16 out[DT];
  auto pass = [&]<bool SAFE>() {
    reference = kNegInf, sum = 0.0f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) out[dt][r] = 0.0f;
    int key = begin + kUnit * wave;
    if (key >= end) return;
    int id0 = page_id(key), id1 = page_id(key + 16);
    load_keys(key, id0, id1);
    load_values(key, id0, id1);
    int next0 = page_id(key + kStep), next1 = page_id(key + kStep + 16);
    while (true) {
      const int later0 = page_id(key + 2 * kStep), later1 = page_id(key + 2 * kStep + 16);
      const bool more = key + kStep < end;
      const bool whole = key + kUnit <= keys.key_end && id0 >= 0 && id1 >= 0;
      const bool there1 = key + 16 < keys.key_end && id1 >= 0;
      const float key_scale[2] = {scale_of(scales[0] & 255u), scale_of(scales[1] & 255u)};
      const float value_scale[2] = {id0 >= 0 ? scale_of(scales[0] >> 8 & 255u) : 1.0f,
                                    there1 ? scale_of(scales[1] >> 8 & 255u) : 1.0f};
      // S^T
      paged_f32x16 s;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = 0.0f;
      const float lane_scale = !std::is_same<T, __bf16>::value ? 1.0f : col < 16 ? key_scale[0] : key_scale[1];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const paged_u32x2 lo = expand4<T>(k[ks >> 1][2 * (ks & 1)], lane_scale);
        const paged_u32x2 hi = expand4<T>(k[ks >> 1][2 * (ks & 1) + 1], lane_scale);
        s = mfma32<T>(attn_u32x4{lo[0], lo[1], hi[0], hi[1]}, q_lds[ks][lane], s);
      }
      if (more) load_keys(key + kStep, next0, next1);
      if constexpr (!std::is_same<T, __bf16>::value)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] *= key_scale[r >> 3];
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
      if (!whole) {  // rows that are not there: zeros for V
#pragma unroll
        for (int blk = 0; blk < 2; ++blk)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const unsigned rows = (blk == 0 ? id0 : id1) < 0
                                      ? 0u : quad_mask(key + 16 * blk + 8 * i + 4 * half, keys.key_end);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) v[blk][i][dt] &= rows;
          }
      }
      // O^T += V^T P^T
#pragma unroll
      for (int blk = 0; blk < 2; ++blk) {
        attn_u32x4 seen{0u, 0u, 0u, 0u};
        if constexpr (SAFE)
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (key + 16 * blk + 8 * (i >> 2) + 4 * half + (i & 3) <= limit) seen[i >> 1] |= 0x3f80u << (16 * (i & 1));
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const paged_u32x2 lo = expand4<__bf16>(v[blk][0][dt], value_scale[blk]);
          const paged_u32x2 hi = expand4<__bf16>(v[blk][1][dt], value_scale[blk]);
          attn_u32x4 x{lo[0], lo[1], hi[0], hi[1]};
          if constexpr (SAFE) {
            paged_f32x16 count;
#pragma unroll
            for (int r = 0; r < 16; ++r) count[r] = 0.0f;
            const attn_u32x4 ones = take_out_nan(x);
            count = mfma32<__bf16>(ones, seen, count);
#pragma unroll
            for (int r = 0; r < 16; ++r) out[dt][r] = count[r] > 0.0f ? __builtin_nanf("") : out[dt][r];
          }
#pragma unroll
          for (int n = 0; n < kPieces; ++n) out[dt] = mfma32<__bf16>(x, piece[blk][n], out[dt]);
        }
      }
      if (!more) break;
      load_values(key + kStep, next0, next1);
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

  // Wave states to LDS, half of a tile's rows at a time (the row's channels are spread over the lanes'
  // registers): 16-byte chunk c of row r in slot c ^ (r % 16). Lane (row, half) holds channels
  // 32 VW n + VW (8 (r / 4) + 4 half + r % 4) + e in out[VW n + e][r].
  constexpr int kHalfRows = kTileRows / 2;
  const int64_t slot = (static_cast<int64_t>(place.unit) * a.splits + place.split) * a.tile_rows;
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    __syncthreads();
    if ((col >> 4) == part) {
      float* const mine = &state_lds[wave][(col & 15) * D];
#pragma unroll
      for (int n = 0; n < VL; ++n)
#pragma unroll
        for (int r = 0; r < 16; r += 4 / VW) {
          attn_f32x4 x;
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = out[VW * n + e % VW][r + e / VW];
          const int channel = 32 * VW * n + VW * (8 * (r >> 2) + 4 * half + (r & 3));
          *reinterpret_cast<attn_f32x4*>(mine + 4 * ((channel >> 2) ^ (col & 15))) = x;
        }
    }
    if (half == 0 && part == 0) {
      wave_ml[wave][col][0] = reference;
      wave_ml[wave][col][1] = sum;
    }
    __syncthreads();
    for (int item = threadIdx.x; item < kHalfRows * (D / 8); item += kAttnThreads) {
      const int local = item / (D / 8), c = item - local * (D / 8), r = kHalfRows * part + local;
      if (r >= rows_here) break;
      auto state = [&](int w, attn_f32x4& lo, attn_f32x4& hi) {
        const float* wo = &state_lds[w][local * D];
        lo = *reinterpret_cast<const attn_f32x4*>(wo + 4 * ((2 * c) ^ local));
        hi = *reinterpret_cast<const attn_f32x4*>(wo + 4 * ((2 * c + 1) ^ local));
      };
      finish_item<T, D, kAttnWaves>(a, seg, row0 + r, 8 * c, slot + r, keys.needed == 1,
                                    [&](int w, int i) { return wave_ml[w][r][i]; }, state);
    }
  }
}

// The plan's constants (us).
constexpr PagedCosts kCosts8 = {
    {{{false, 4, 4, 4.2, 0.0, 0.446, 0.226},
      {false, 8, 2, 4.5, 0.66, 0.375, 0.48},
      {true, 4, 4, 5.1, 0.0, 0.455, 0.353}},
     {{false, 4, 3, 4.4, 0.0, 0.545, 0.344},
      {false, 8, 2, 4.4, 1.1, 0.2, 0.94},
      {true, 4, 3, 6.0, 0.0, 0.415, 0.62}},
     {{false, 4, 2, 5.1, 1.1, 0.624, 0.88},
      {false, 8, 1, 3.3, 3.3, 2.27, 0.0},
      {true, 4, 2, 8.75, 0.0, 0.632, 1.12}}},
    {{2.1, 0.34, 0.23}, {2.3, 0.26, 0.24}, {2.45, 0.27, 0.21}}};

template <typename T, int D>
int launch_paged(const PagedAttnArgs& args, const PagedPlan& plan, hipStream_t stream) {
  auto attend = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(plan.units * plan.splits)),
                       dim3(static_cast<unsigned>(64 * plan.waves)), 0, stream, args);
  };
  if (plan.tile_kernel) attend(paged8_tile_kernel<T, D>);
  else if (plan.waves == kAttnWaves) attend(paged8_attention_kernel<T, D, kAttnWaves>);
  else attend(paged8_attention_kernel<T, D, 2 * kAttnWaves>);
  if (int status = check_launch("paged8_attention")) return status;
  return launch_merge<T, D>(args, plan, stream);
}

}  // namespace
}  // namespace lr

using namespace lr;

extern "C" size_t lr_paged8_attention_workspace_bytes(int64_t segments, int64_t groups,
                                                      int64_t length, int64_t max_keys,
                                                      int64_t dim) {
  return attend_paged_workspace<kCosts8>(segments, groups, length, max_keys, dim);
}

extern "C" int lr_paged8_attention_plan(int64_t segments, int64_t groups, int64_t length,
                                        int64_t max_keys, int64_t dim, int64_t* plan) {
  return describe_paged_plan<kCosts8>(segments, groups, length, max_keys, dim, plan);
}

extern "C" int lr_paged8_attention(const void* queries, const int64_t* query_strides,
                                   const void* pages, int64_t page_count, int64_t page_size,
                                   const int32_t* table, int64_t max_pages, const int32_t* lengths,
                                   int64_t batch, int64_t kv_heads, int64_t groups, int64_t length,
                                   int64_t dim, int dtype, int64_t max_keys, const int32_t* counts,
                                   float scale, void* out, void* workspace, size_t workspace_size,
                                   void* stream) {
  auto launch = [&](const PagedAttnArgs& args, const PagedPlan& plan) {
    return dispatch_dim(dim, [&]<int D>() {
      return dtype == LR_DTYPE_BF16 ? launch_paged<__bf16, D>(args, plan, as_stream(stream))
                                    : launch_paged<_Float16, D>(args, plan, as_stream(stream));
    });
  };
  return attend_paged<kCosts8>(queries, query_strides, pages, page_count, page_size, table, max_pages,
                               lengths, batch, kv_heads, groups, length, dim, dtype, max_keys, counts,
                               scale, out, workspace, workspace_size, launch);
}
