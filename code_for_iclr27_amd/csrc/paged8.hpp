// The paged 8-bit KV cache: what its kernels share (paged8_move.hip: append, read, compact;
// paged8_attention.hip: attention). Tables, lengths and page ids are those of paged.hpp.
//
// 16 rows of a segment, from a multiple of 16 on, are a token block. Its keys share a scale and its
// values another: codes E4M3 (OCP: a sign, four bits of exponent, three of significand; 448 is the
// largest, a magnitude of 127 is NaN) times 2^(scale - 127). A code has at most four significant bits,
// so the values are exact in bf16. A page of `size` rows holds
//   keys       [size / 16][D / 16][16 rows][16 channels]  a wave's 16-byte loads of 16 rows and 64
//                                                         channels are one piece of memory, and are the
//                                                         matrix cores' operand as they are
//   values     [size / 4][D][4 rows]                      four rows of a channel are a word: the other
//                                                         product's operand, without a transposition
//   positions  [size] f32
//   scales     [size / 16] x (keys', values')             in room for 4 size bytes, which makes pages
//                                                         multiples of 128 bytes
//
// The scale of a block is the smallest power of two that holds its largest finite magnitude: 2^e with
// e = floor(log2 amax) - 8, one more from a significand of 1.8125 on (which would round to 480).
// An element is rounded to four significant bits (ties to even), and what then lies under the smallest
// code, 2^(e - 9), is cut off. Both steps and the step to a larger scale (shift_codes) compose: a block
// holds the same bytes whether its rows came at once or one by one.
#pragma once

#include "paged.hpp"

namespace lr {

constexpr int kTokens = 16;          // rows that share a scale
constexpr unsigned kCodeNaN = 0xff;  // the NaN that is written (the conversion instruction's)

// Exponents of the scales that append writes: 2^-9 times the smallest is a normal number in f32 and
// bf16, 448 times the largest is finite there, or (rows appended as f16) in f16.
constexpr ScaleRange kWideRange8{-117, 119}, kHalfRange8{-117, 7};

template <int D>
struct Page8 {
  static constexpr int64_t bytes(int size) { return static_cast<int64_t>(size) * (2 * D + 8); }
  // Byte offsets in a page: 16 channels of a row's key, its values (channel c at 4 c), ...
  static __device__ __forceinline__ int key(int slot, int chunk) {
    return (slot >> 4) * (kTokens * D) + chunk * 256 + (slot & 15) * 16;
  }
  static __device__ __forceinline__ int value(int shift, int slot) {
    return (D << shift) + (slot >> 2) * (4 * D) + (slot & 3);
  }
  static __device__ __forceinline__ int position(int shift, int slot) { return (2 * D << shift) + 4 * slot; }
  // ... and its block's scales: the keys' byte, the values' byte.
  static __device__ __forceinline__ int scales(int shift, int slot) {
    return ((2 * D + 4) << shift) + 2 * (slot >> 4);
  }
};

// Four codes times a scale as four 16-bit values: exact in bf16 (T), and in f16 without a scale.
template <typename T>
__device__ __forceinline__ paged_u32x2 expand4(unsigned codes, float scale) {
  if constexpr (std::is_same<T, __bf16>::value)
    return paged_u32x2{
        __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, false)),
        __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, true))};
  else
    return paged_u32x2{
        __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, false)),
        __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, true))};
}

// Bytes of a page, or 0 for a page size or head dimension that the kernels do not take.
inline int64_t paged8_bytes(int64_t page_size, int64_t dim) {
  return paged_bytes(page_size, dim) == 0 ? 0 : page_size * (2 * dim + 8);
}

}  // namespace lr
