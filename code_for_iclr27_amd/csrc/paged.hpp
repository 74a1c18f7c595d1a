// The paged 4-bit KV cache: what its kernels share (paged_move.hip: append, read, compact;
// paged_attention.hip: attention).
//
// A page holds `size` rows of one (request, KV head) segment, in five sections: the keys' codes
// [size, D / 2], the values' codes, the keys' scales [size, D / 32], the values' scales, the rows'
// positions (f32). A row's 32 channels 32 b .. 32 b + 31 form block b: E2M1 codes (sign, two bits of
// exponent, one of significand: 0, 0.5, 1, 1.5, 2, 3, 4, 6), channel 2 i in the low nibble of byte i,
// times 2^(scale - 127); a scale of 255 makes the block NaN. So a value has at most two significant
// bits and is exact in bf16, and in f16 within the range that append keeps to.
//
// Row i of segment s lies in page table[s * max_pages + i / size], slot i % size. Page ids outside
// [0, page_count) and rows at or past max_pages * size do not exist: nothing is read or written.
#pragma once

#include <type_traits>

#include "lr_common.hpp"

namespace lr {

typedef unsigned paged_u32x4 __attribute__((ext_vector_type(4)));

constexpr int kBlock = 32;  // channels that share a scale
constexpr unsigned kScaleNaN = 255;

// Exponents of the scales that append writes. 6 x 2^125 is finite in bf16 and f32, and half of 2^-125
// is a normal number there; 6 x 2^13 and 0.5 x 2^-23 are f16's largest and smallest.
struct ScaleRange {
  int low, high;
};
constexpr ScaleRange kWideRange{-125, 125}, kHalfRange{-23, 13};

// An E8M0 scale byte as the f32 whose exponent the conversions take (255 gives NaN results).
__device__ __forceinline__ float scale_of(unsigned byte) { return __builtin_bit_cast(float, byte << 23); }

// Eight codes times their scale as eight 16-bit values: exact (T: __bf16 or _Float16).
template <typename T>
__device__ __forceinline__ paged_u32x4 expand8(unsigned codes, float scale) {
  if constexpr (std::is_same<T, __bf16>::value) {
    return paged_u32x4{
        __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0)),
        __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1)),
        __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2)),
        __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3))};
  } else {
    return paged_u32x4{
        __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 0)),
        __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 1)),
        __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 2)),
        __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 3))};
  }
}

template <int D>
struct Page {
  static constexpr int kCodes = D / 2, kScales = D / kBlock;  // bytes a K or V row
  static constexpr int64_t bytes(int size) { return static_cast<int64_t>(size) * (D + D / 16 + 4); }
  // Byte offsets in a page; which: 0 keys, 1 values.
  static __device__ __forceinline__ int codes(int shift, int which, int slot) {
    return (which * kCodes << shift) + slot * kCodes;
  }
  static __device__ __forceinline__ int scales(int shift, int which, int slot) {
    return ((D + which * kScales) << shift) + slot * kScales;
  }
  static __device__ __forceinline__ int position(int shift, int slot) {
    return ((D + 2 * kScales) << shift) + 4 * slot;
  }
};

struct PagedCache {
  uint8_t* pages;
  int64_t page_count;
  int shift;                // log2 of the page size
  int max_pages;            // of a segment
  const int32_t* table;     // [segments, max_pages]
  const int32_t* lengths;   // [segments]

  // rows of a segment, clamped to what its table can hold
  __device__ __forceinline__ int rows(int64_t segment) const {
    const int n = lengths[segment], most = max_pages << shift;
    return n < 0 ? 0 : n < most ? n : most;
  }
};

// Bytes of a page, or 0 for a page size or head dimension that the kernels do not take.
inline int64_t paged_bytes(int64_t page_size, int64_t dim) {
  const bool sizes = page_size == 16 || page_size == 32 || page_size == 64 || page_size == 128 ||
                     page_size == 256;
  if (!sizes || (dim != 64 && dim != 128 && dim != 256)) return 0;
  return page_size * (dim + dim / 16 + 4);
}

// A launch has fewer than 2^32 threads.
inline bool launchable(int64_t blocks, int64_t threads) { return blocks < (int64_t{1} << 32) / threads; }

// The checks every entry point makes of the cache.
int check_paged(const void* pages, int64_t page_count, int64_t page_size, int64_t dim,
                const int32_t* table, int64_t max_pages, const int32_t* lengths, int64_t segments);

inline PagedCache paged_cache(const void* pages, int64_t page_count, int64_t page_size,
                              const int32_t* table, int64_t max_pages, const int32_t* lengths) {
  PagedCache c{};
  c.pages = static_cast<uint8_t*>(const_cast<void*>(pages));
  c.page_count = page_count;
  c.shift = __builtin_ctzll(static_cast<unsigned long long>(page_size));
  c.max_pages = static_cast<int>(max_pages);
  c.table = table;
  c.lengths = lengths;
  return c;
}

template <typename F>
int dispatch_dim(int64_t dim, F&& f) {
  switch (dim) {
    case 64: return f.template operator()<64>();
    case 128: return f.template operator()<128>();
    default: return f.template operator()<256>();
  }
}

}  // namespace lr
