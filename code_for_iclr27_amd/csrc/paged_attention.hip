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

#include "paged_attention.hpp"

namespace lr {
namespace {

typedef short paged_s16x4 __attribute__((ext_vector_type(4)));

// V rows in LDS: 16-byte chunk c of row r in slot c ^ x(r). The eight rows that eight lanes write one
// chunk of lie in different 16-byte places of 128, and the 32 bytes of four rows that 16 lanes read
// transposed in different quarters of it. (Slots that differ in the four rows' 64-byte places alone
// had twice the bank conflicts; the prefill kernel as a whole took 0.6% longer.)
__device__ __forceinline__ int value_swizzle(int row) { return (row & 3) << 1 | ((row >> 2) & 1); }

// Codes and scales of a unit: two blocks of 16 rows, a lane's words of one row each. Words 4 h ..
// 4 h + 3 (d256: h = 0, 1; else all) belong to one block of channels.
template <int D>
struct UnitCodes {
  static constexpr int kWords = D / 32, kBytes = D == 256 ? 2 : 1;
  unsigned k[2][kWords], v[2][kWords], ks[2][kBytes], vs[2][kBytes];
};

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

// The plan's constants (us): a least-squares fit to measured calls (1 to 1,000 queries of 1 to 128
// segments onto 100 to 130,000 rows, each kernel, 1 to 64 chunks), made when P had two pieces. With
// three, 17,944 such calls take 6 to 9% longer than estimated (median), 7% about that; over their 1,077
// shapes the choice takes 0.6% longer than the best one, 15% at most. Constants fitted anew choose no
// better (0.5%). `resident` is a parameter of the fit like the others: the registers let five workgroups
// of four waves share a compute unit at d64 and four at d128, and a fit with these numbers comes to 0.6%
// too. (Rules by the number of workgroups alone take 9% longer, up to twice as long: 8 queries of 16
// requests onto 300 rows, 4 heads, G6, d256, 21 us against 12; 192 queries of one onto 9,000 rows 175
// against 99.)
constexpr PagedCosts kCosts4 = {
    {{{16, 4, 4, 4.2, 0.0, 0.446, 0.226},
      {16, 8, 2, 4.5, 0.66, 0.375, 0.48},
      {32, 4, 4, 5.1, 0.0, 0.455, 0.353}},
     {{16, 4, 3, 4.4, 0.0, 0.545, 0.344},
      {16, 8, 2, 4.4, 1.1, 0.2, 0.94},
      {32, 4, 3, 6.0, 0.0, 0.415, 0.62}},
     {{16, 4, 2, 5.1, 1.1, 0.624, 0.88},
      {16, 8, 1, 3.3, 3.3, 2.27, 0.0},
      {32, 4, 2, 8.75, 0.0, 0.632, 1.12}}},
    {{2.1, 0.34, 0.23}, {2.3, 0.26, 0.24}, {2.45, 0.27, 0.21}}};

template <typename T, int D>
int launch_paged(const PagedAttnArgs& args, const PagedPlan& plan, hipStream_t stream) {
  auto attend = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(plan.units * plan.splits)),
                       dim3(static_cast<unsigned>(64 * plan.waves)), 0, stream, args);
  };
  if (plan.rows == kTileRows) attend(paged_tile_kernel<T, D>);
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
  return attend_paged_workspace<kCosts4>(segments, groups, length, max_keys, dim);
}

extern "C" int lr_paged_attention_plan(int64_t segments, int64_t groups, int64_t length,
                                       int64_t max_keys, int64_t dim, int64_t* plan) {
  return describe_paged_plan<kCosts4>(segments, groups, length, max_keys, dim, plan);
}

extern "C" int lr_paged_attention(const void* queries, const int64_t* query_strides,
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
  return attend_paged<kCosts4>(queries, query_strides, pages, page_count, page_size, table, max_pages,
                               lengths, batch, kv_heads, groups, length, dim, dtype, max_keys, counts,
                               scale, out, workspace, workspace_size, launch);
}
