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
//
// What bounds it. Decode of a long cache: memory (sixteen requests of 20k rows, 8 heads, G4, d128: 657 MB
// of codes in 101 us and the merge's 5, 6.2 TB/s; a large copy reaches 5.0). Short ones: the start of the
// workgroups (2 us until half of them run), a chain of three loads and the two launches (8 segments of
// 1,100 rows of d64 7.6 us, 2,500 rows of eight requests 13.0). Prefill: power. 1500 queries onto 4,450
// rows take 241 to 250 us at 1.9 GHz (2.4 unloaded), where the matrix cores are busy 52% of the cycles
// and the vector instructions (251 a unit of 32 keys and 32 rows beside 32 MFMAs) issue in 61%; eight
// such calls in one run at 1.08 PFLOP/s of matrix work, pieces included, where a large bf16 product of
// the library reaches 1.23. Tried and no faster: the next unit's S^T beside this one's exponentials, with
// and without scheduling barriers (250 to 296), tiles of 64 rows (the same; 5% less on eight such calls),
// two units of codes in flight in the kernel of 16 rows (13.7 -> 15.0 us for the eight requests). Slower:
// queries kept in registers by the tiles of 32 rows (spilled: 270), page addresses of both token blocks
// found apart for pages of more than 16 rows.

#include "paged8.hpp"
#include "paged_attention.hpp"

namespace lr {
namespace {

// Pages of a unit of 32 keys from a multiple of 32 on: one, or (TWO: pages of 16 rows) two.
template <bool TWO>
struct UnitPages {
  int id[TWO ? 2 : 1];  // as the table has them

  __device__ __forceinline__ bool in_pool(int blk, unsigned page_count) const {
    return static_cast<unsigned>(id[TWO ? blk : 0]) < page_count;
  }
};

// What a wave needs to find its units: addresses are scalar, but for a lane's offset.
template <int D, bool TWO>
struct UnitSource {
  PageIds table;
  const uint8_t* pages;
  unsigned page_count, page_bytes;
  int shift, last;  // last: of the rows that a lookup may name

  __device__ __forceinline__ UnitSource(const PagedCache& cache, unsigned seg, int last_row)
      : table(page_table(cache, seg)), pages(cache.pages), page_count(static_cast<unsigned>(cache.page_count)),
        page_bytes(static_cast<unsigned>(Page8<D>::bytes(1) << cache.shift)), shift(cache.shift), last(last_row) {}

  __device__ __forceinline__ UnitPages<TWO> find(int key) const {
    UnitPages<TWO> u;
    u.id[0] = table[min(key, last) >> shift];
    if constexpr (TWO) u.id[1] = table[min(key + 16, last) >> shift];
    return u;
  }
  // The page of a unit's token block (a page outside the pool: the first one, which is not used).
  __device__ __forceinline__ PagedBytes page(const UnitPages<TWO>& u, int blk) const {
    const unsigned id = u.in_pool(blk, page_count) ? static_cast<unsigned>(u.id[TWO ? blk : 0]) : 0u;
    return (PagedBytes)uniform_address(pages + static_cast<uint64_t>(id) * page_bytes);
  }
  // The slot of a unit's token block.
  __device__ __forceinline__ unsigned slot(int key, int blk) const {
    return TWO ? 0u : (static_cast<unsigned>(key) & ((1u << shift) - 1)) + 16 * blk;
  }
};

// The scales of a unit's token blocks, read by scalar loads (they are taken apart where they are used,
// so that nothing waits for them before).
template <int D, bool TWO>
struct UnitScales {
  unsigned word[TWO ? 2 : 1];

  __device__ __forceinline__ void load(const UnitSource<D, TWO>& source, const UnitPages<TWO>& u, int key) {
    typedef const __attribute__((address_space(4))) unsigned* Words;
#pragma unroll
    for (int blk = 0; blk < (TWO ? 2 : 1); ++blk) {
      const PagedBytes p = source.page(u, blk);  // (a unit's two pairs of bytes are an aligned word)
      word[blk] = *(Words)(p + Page8<D>::scales(source.shift, static_cast<int>(source.slot(key, 0))));
    }
  }
  __device__ __forceinline__ float key(int blk) const {
    return scale_of((TWO ? word[blk] : word[0] >> (16 * blk)) & 255u);
  }
  __device__ __forceinline__ float value(int blk) const {
    return scale_of((TWO ? word[blk] : word[0] >> (16 * blk)) >> 8 & 255u);
  }
};

// 16 bytes of a lane from a uniform address on (ONCE: that no other workgroup reads).
template <bool ONCE = false>
__device__ __forceinline__ attn_u32x4 load_piece(PagedBytes p, unsigned lane_offset) {
  typedef const __attribute__((address_space(1))) attn_u32x4* Place;
  if constexpr (ONCE) return __builtin_nontemporal_load((Place)(p + lane_offset));
  else return *(Place)(p + lane_offset);
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

// Tiles of 16 rows: decode, and a few query rows. ONCE: a segment's rows are one tile's, each cached row is
// read once, and its loads ask the caches not to keep it. (Rows that come from memory, as a layer's do
// behind the other layers' and the weights: 676 MB of codes 112 to 114 us for 124 to 127, 338 MB 59 to 60
// for 65 to 68, 169 MB 34 to 35 for 38 to 40, 42 MB 14.1 to 14.6 for 15.4, 2 MB the same. Rows that the
// caches still hold, of one layer's call made again at once: 169 MB 33 to 34 for 31 to 32, 34 MB 13 for 11.
// With two tiles a segment: 20.6 for 17.7 in the drafts of d256. In the tiles of 32 rows: 144 for 151 with
// 676 MB, the same with less, 43 for 39 where the caches hold 169 MB.)
template <typename T, int D, int WAVES, bool TWO, bool ONCE>
__global__ __launch_bounds__(64 * WAVES) __attribute__((amdgpu_waves_per_eu(
    WAVES == 8 || D == 256 ? 2 : D == 64 ? 4 : 3)))
void paged8_attention_kernel(PagedAttnArgs a) {
  constexpr int kStep = kUnit * WAVES;  // keys of the workgroup's step
  constexpr int KL = D / 64;            // 16-byte loads of a lane for a token block's keys, or values
  constexpr int DT = D / 16;            // column tiles of the output
  constexpr bool kFoldScale = std::is_same<T, __bf16>::value;  // the keys' scale into the conversion
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
  UnitSource<D, TWO> source(a.cache, seg, (a.cache.max_pages << a.cache.shift) - 1);
  const int begin = static_cast<int>(place.split) * a.chunk;
  UnitPages<TWO> first{};
  if (a.max_keys > 0) first = source.find(begin + kUnit * wave);
  const TileKeys keys = tile_keys(a, seg, row0, row0 + rows_here - 1);
  if (keys.needed == 0) {  // no visible key for any row of this tile
    if (place.split == 0) zero_rows<T, D>(a, seg, row0, rows_here);
    return;
  }
  if (static_cast<int>(place.split) >= keys.needed) return;  // uniform across the workgroup
  const int end = min(begin + a.chunk, keys.key_end);
  source.last = keys.key_end - 1;

  // Queries (B operand of step 2 n + h: channels 16 (4 n + j) + 8 h of row m), and the last key that
  // the lane's row sees.
  const TileRow row = tile_row(a, seg, row0 + (m < rows_here ? m : 0));
  const int limit = m < rows_here ? last_key(keys, row.query) : -1;
  const int all_see = all_rows_see(a, keys, row0, rows_here);
  attn_u32x4 q[2 * KL];
#pragma unroll
  for (int s = 0; s < 2 * KL; ++s)
    q[s] = load16(static_cast<const T*>(a.queries) + row.offset + 16 * (4 * (s >> 1) + j) + 8 * (s & 1));

  attn_u32x4 k[2][KL], v[2][KL];
  UnitScales<D, TWO> scales;  // of the unit whose keys are loaded
  auto load_keys = [&](const UnitPages<TWO>& u, int key0) {
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
      const PagedBytes block = source.page(u, blk) + D * source.slot(key0, blk);
#pragma unroll
      for (int n = 0; n < KL; ++n) k[blk][n] = load_piece<ONCE>(block + 1024 * n, 16u * lane);
    }
    scales.load(source, u, key0);
  };
  // (words 4 n + e: channels 64 n + 4 m + e of keys 4 j .. 4 j + 3)
  auto load_values = [&](const UnitPages<TWO>& u, int key0) {
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
      const PagedBytes block = source.page(u, blk) + ((D << source.shift) + D * source.slot(key0, blk));
#pragma unroll
      for (int n = 0; n < KL; ++n) v[blk][n] = load_piece<ONCE>(block + 256 * n, 4u * D * j + 16u * m);
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
    UnitPages<TWO> now = SAFE ? source.find(key) : first;
    load_keys(now, key);
    load_values(now, key);
    UnitPages<TWO> next = source.find(key + kStep);
    while (true) {
      // the unit after the next: its pages' ids arrive while this one is worked on
      const UnitPages<TWO> later = source.find(key + 2 * kStep);
      const bool more = key + kStep < end;
      const bool there[2] = {now.in_pool(0, source.page_count), now.in_pool(1, source.page_count)};
      // S^T
      attn_f32x4 s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
      const float key_scale[2] = {scales.key(0), scales.key(1)};
      float value_scale[2] = {scales.value(0), scales.value(1)};
#pragma unroll
      for (int n = 0; n < 2 * KL; ++n)
#pragma unroll
        for (int blk = 0; blk < 2; ++blk) {
          const float scale = kFoldScale ? key_scale[blk] : 1.0f;
          const paged_u32x2 lo = expand4<T>(k[blk][n >> 1][2 * (n & 1)], scale);
          const paged_u32x2 hi = expand4<T>(k[blk][n >> 1][2 * (n & 1) + 1], scale);
          s[blk] = Vec::mfma(__builtin_bit_cast(X8, attn_u32x4{lo[0], lo[1], hi[0], hi[1]}),
                             __builtin_bit_cast(X8, q[n]), s[blk]);
        }
      if (more) load_keys(next, key + kStep);
      if constexpr (!kFoldScale)
#pragma unroll
        for (int blk = 0; blk < 2; ++blk)
#pragma unroll
          for (int r = 0; r < 4; ++r) s[blk][r] *= key_scale[blk];
      if (key + kUnit - 1 > all_see || !there[0] || !there[1]) {
#pragma unroll
        for (int blk = 0; blk < 2; ++blk) {
          const int lane_limit = there[blk] ? limit - (key + 16 * blk + 4 * j) : -1;
#pragma unroll
          for (int r = 0; r < 4; ++r) s[blk][r] = r > lane_limit ? kNegInf : s[blk][r];
        }
        // rows that are not there: zeros for V
        if (key + kUnit > keys.key_end || !there[0] || !there[1]) {
#pragma unroll
          for (int blk = 0; blk < 2; ++blk) {
            const unsigned rows = there[blk] ? quad_mask(key + 16 * blk + 4 * j, keys.key_end) : 0u;
#pragma unroll
            for (int n = 0; n < KL; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) v[blk][n][e] &= rows;
            if (!there[blk] || key + 16 * blk >= keys.key_end) value_scale[blk] = 1.0f;
          }
        }
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
      load_values(next, key + kStep);
      key += kStep;
      now = next;
      next = later;
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

template <typename T, int D, bool TWO>
__global__ __launch_bounds__(kAttnThreads) __attribute__((amdgpu_waves_per_eu(D == 64 ? 4 : D == 128 ? 3 : 2)))
void paged8_tile_kernel(PagedAttnArgs a) {
  constexpr int KS = D / 16;      // MFMA steps over the head dimension
  constexpr int KL = D / 32;      // 16-byte loads of a lane for the unit's keys
  constexpr int DT = D / 32;      // column tiles of the output
  constexpr int VW = D == 64 ? 2 : 4;     // channels of a lane's load of values
  constexpr int VL = DT / VW;             // loads of a quad's values
  constexpr int kStep = kUnit * kAttnWaves;
  constexpr bool kFoldScale = std::is_same<T, __bf16>::value;  // the keys' scale into the conversion
  __shared__ __align__(16) attn_u32x4 q_lds[KS][64];
  __shared__ __align__(16) float state_lds[kAttnWaves][16 * D];
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

  const UnitSource<D, TWO> source(a.cache, seg, keys.key_end - 1);
  // Lane (key, half): 16 channels of every 32, chunks 2 n + half.
  attn_u32x4 k[KL];
  unsigned v[2][2][DT];  // a token block's quads half and 2 + half: the lane's channels
  UnitScales<D, TWO> scales;
  auto load_keys = [&](const UnitPages<TWO>& u, int key0) {
    const unsigned lane_offset = 256u * half + 16u * (col & 15);
    if constexpr (TWO) {
      const PagedBytes block = col < 16 ? source.page(u, 0) : source.page(u, 1);
#pragma unroll
      for (int n = 0; n < KL; ++n) k[n] = load_piece(block + 512 * n, lane_offset);
    } else {
      const PagedBytes block = source.page(u, 0) + D * source.slot(key0, 0);
#pragma unroll
      for (int n = 0; n < KL; ++n) k[n] = load_piece(block + 512 * n, lane_offset + 16u * D * (col >> 4));
    }
    scales.load(source, u, key0);
  };
  // (word VW n + e: channel 32 VW n + VW col + e)
  auto load_values = [&](const UnitPages<TWO>& u, int key0) {
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
      const PagedBytes block = source.page(u, blk) + ((D << source.shift) + D * source.slot(key0, blk));
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int n = 0; n < VL; ++n) {
          const PagedBytes p = block + (8 * D * i + 512 * n);
          const unsigned lane_offset = 4u * D * half + 4u * VW * col;
          if constexpr (VW == 2) {
            const paged_u32x2 x = *(const __attribute__((address_space(1))) paged_u32x2*)(p + lane_offset);
            v[blk][i][0] = x[0], v[blk][i][1] = x[1];
          } else {
            const attn_u32x4 x = load_piece(p, lane_offset);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[blk][i][4 * n + e] = x[e];
          }
        }
    }
  };

  float reference, sum;  // in exponents of two; the same in both halves
  paged_f32x16 out[DT];
  auto pass = [&]<bool SAFE>() {
    reference = kNegInf, sum = 0.0f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) out[dt][r] = 0.0f;
    int key = begin + kUnit * wave;
    if (key >= end) return;
    UnitPages<TWO> now = source.find(key);
    load_keys(now, key);
    load_values(now, key);
    UnitPages<TWO> next = source.find(key + kStep);
    while (true) {
      const UnitPages<TWO> later = source.find(key + 2 * kStep);
      const bool more = key + kStep < end;
      const bool there[2] = {now.in_pool(0, source.page_count), now.in_pool(1, source.page_count)};
      const float key_scale[2] = {scales.key(0), scales.key(1)};
      float value_scale[2] = {scales.value(0), scales.value(1)};
      // S^T
      paged_f32x16 s;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = 0.0f;
      const float lane_scale = !kFoldScale ? 1.0f : col < 16 ? key_scale[0] : key_scale[1];
      asm volatile("" ::: "memory");  // (the queries stay in LDS: as registers they would spill)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const paged_u32x2 lo = expand4<T>(k[ks >> 1][2 * (ks & 1)], lane_scale);
        const paged_u32x2 hi = expand4<T>(k[ks >> 1][2 * (ks & 1) + 1], lane_scale);
        s = mfma32<T>(attn_u32x4{lo[0], lo[1], hi[0], hi[1]}, q_lds[ks][lane], s);
      }
      if (more) load_keys(next, key + kStep);
      if constexpr (!kFoldScale)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] *= key_scale[r >> 3];
      if (key + kUnit - 1 > all_see || !there[0] || !there[1]) {
#pragma unroll
        for (int blk = 0; blk < 2; ++blk) {
          const int lane_limit = there[blk] ? limit - (key + 16 * blk + 4 * half) : -1;
#pragma unroll
          for (int r = 0; r < 8; ++r)
            if (8 * (r >> 2) + (r & 3) > lane_limit) s[8 * blk + r] = kNegInf;
        }
        // rows that are not there: zeros for V
        if (key + kUnit > keys.key_end || !there[0] || !there[1]) {
#pragma unroll
          for (int blk = 0; blk < 2; ++blk) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const unsigned rows = there[blk] ? quad_mask(key + 16 * blk + 8 * i + 4 * half, keys.key_end) : 0u;
#pragma unroll
              for (int dt = 0; dt < DT; ++dt) v[blk][i][dt] &= rows;
            }
            if (!there[blk] || key + 16 * blk >= keys.key_end) value_scale[blk] = 1.0f;
          }
        }
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
      // O^T += V^T P^T, a token block after the other
#pragma unroll
      for (int blk = 0; blk < 2; ++blk) {
        attn_u32x4 piece[kPieces], seen{0u, 0u, 0u, 0u};
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const float x = probability<SAFE>(s[8 * blk + 2 * n], a.to_log2, base);
          const float y = probability<SAFE>(s[8 * blk + 2 * n + 1], a.to_log2, base);
          sum += x;
          sum += y;
          split_bf16(x, y, piece, n);
        }
        if constexpr (SAFE)  // ones for the lane's keys that its row sees
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (key + 16 * blk + 8 * (i >> 2) + 4 * half + (i & 3) <= limit) seen[i >> 1] |= 0x3f80u << (16 * (i & 1));
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const paged_u32x2 lo = expand4<__bf16>(v[blk][0][dt], value_scale[blk]);
          const paged_u32x2 hi = expand4<__bf16>(v[blk][1][dt], value_scale[blk]);
          attn_u32x4 x{lo[0], lo[1], hi[0], hi[1]};
          if constexpr (SAFE) {
            const attn_u32x4 ones = take_out_nan(x);
            paged_f32x16 count;
#pragma unroll
            for (int r = 0; r < 16; ++r) count[r] = 0.0f;
            count = mfma32<__bf16>(ones, seen, count);
#pragma unroll
            for (int r = 0; r < 16; ++r) out[dt][r] = count[r] > 0.0f ? __builtin_nanf("") : out[dt][r];
          }
#pragma unroll
          for (int n = 0; n < kPieces; ++n) out[dt] = mfma32<__bf16>(x, piece[n], out[dt]);
        }
      }
      if (!more) break;
      load_values(next, key + kStep);
      key += kStep;
      now = next;
      next = later;
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

  // Wave states to LDS, 16 rows at a time (a row's channels are spread over the lanes' registers):
  // 16-byte chunk c of row r in slot c ^ (r % 16). Lane (row, half) holds channels
  // 32 VW n + VW (8 (r / 4) + 4 half + r % 4) + e in out[VW n + e][r].
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
    for (int item = threadIdx.x; item < 16 * (D / 8); item += kAttnThreads) {
      const int local = item / (D / 8), c = item - local * (D / 8), r = 16 * part + local;
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

// The plan's constants (us): a least-squares fit to 215,000 measured calls (1 to 1,500 queries of 4 to
// 128 segments onto 1 to 30,000 rows, each kernel, 1 to 64 parts), each weighed by how near it comes to
// the best of its shape (d64: alike). Over their 25,900 shapes the choice takes 1.0 to 1.4% longer than
// the best one (95% of them at most 8%). Without the form of eight waves the best calls take 1.1, 0.7
// and 0.3% longer on average, without the tiles of 32 rows 1.1, 1.6 and 0.3%, and many rows much.
constexpr PagedCosts kCosts8 = {
    {{{16, 4, 5, 3.48, 0.73, 0.433, 0.368},
      {16, 8, 2, 3.38, 1.19, 0.355, 0.623},
      {32, 4, 8, 5.86, 0.00, 0.317, 0.436}},
     {{16, 4, 2, 3.56, 0.70, 0.314, 0.741},
      {16, 8, 1, 3.15, 1.15, 1.582, 0.000},
      {32, 4, 8, 6.25, 0.85, 0.337, 0.736}},
     {{16, 4, 1, 3.60, 1.28, 1.523, 0.000},
      {16, 8, 1, 2.31, 2.58, 2.439, 0.000},
      {32, 4, 8, 7.21, 2.54, 0.132, 1.464}}},
    {{2.24, 0.259, 0.261}, {2.45, 0.185, 0.294}, {2.53, 0.211, 0.282}}};

template <typename T, int D, bool TWO>
int launch_paged(const PagedAttnArgs& args, const PagedPlan& plan, hipStream_t stream) {
  auto attend = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(plan.units * plan.splits)),
                       dim3(static_cast<unsigned>(64 * plan.waves)), 0, stream, args);
  };
  auto small = [&]<bool ONCE>() {
    if (plan.waves == kAttnWaves) attend(paged8_attention_kernel<T, D, kAttnWaves, TWO, ONCE>);
    else attend(paged8_attention_kernel<T, D, 2 * kAttnWaves, TWO, ONCE>);
  };
  if (plan.rows == kTileRows) attend(paged8_tile_kernel<T, D, TWO>);
  else if (plan.tiles == 1) small.template operator()<true>();
  else small.template operator()<false>();
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
      auto by_type = [&]<typename T>() {
        return page_size == kTokens ? launch_paged<T, D, true>(args, plan, as_stream(stream))
                                    : launch_paged<T, D, false>(args, plan, as_stream(stream));
      };
      return dtype == LR_DTYPE_BF16 ? by_type.template operator()<__bf16>()
                                    : by_type.template operator()<_Float16>();
    });
  };
  return attend_paged<kCosts8>(queries, query_strides, pages, page_count, page_size, table, max_pages,
                               lengths, batch, kv_heads, groups, length, dim, dtype, max_keys, counts,
                               scale, out, workspace, workspace_size, launch);
}
