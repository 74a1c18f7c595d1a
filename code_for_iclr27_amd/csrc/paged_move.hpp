// What the operators that move rows of the paged KV caches share (paged_move.hip: 4 bits;
// paged8_move.hip: 8 bits): rows in memory, the calls' arguments, sums of the lengths, searches and the
// entry points' checks.
#pragma once

#include <algorithm>

#include "paged.hpp"

namespace lr {
namespace {

constexpr int kThreads = 256;

typedef float move_f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned move_u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned move_u32x2 __attribute__((ext_vector_type(2)));

template <typename T>
struct Eight;  // eight elements in memory
template <>
struct Eight<float> {
  move_f32x4 lo, hi;
  __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = lo[e], v[4 + e] = hi[e];
  }
  __device__ __forceinline__ void set(const float (&v)[8]) {
    lo = move_f32x4{v[0], v[1], v[2], v[3]};
    hi = move_f32x4{v[4], v[5], v[6], v[7]};
  }
};
template <typename T>
struct Eight {
  typedef T vec __attribute__((ext_vector_type(8)));
  vec x;
  __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = static_cast<float>(x[e]);
  }
  __device__ __forceinline__ void set(const float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = static_cast<T>(v[e]);  // round to nearest even
  }
};

// Rows [batch, heads, added, D] with the strides (elements) of the first three dimensions.
struct Rows {
  const void* base;
  int64_t batch, head, row;
};

struct AppendArgs {
  Rows keys, values, queries;
  void* out_queries;          // [batch, query_heads, added, D], contiguous
  const int64_t* positions;   // [batch, added]
  const float* cos;           // [table_rows, half], or half = 0
  const float* sin;
  int64_t table_rows;
  int half;
  unsigned batch, kv_heads, query_heads, added;
  unsigned kv_rows, query_rows;  // batch * heads * added
  unsigned kv_blocks;            // workgroups of the keys, and of the values
  const int32_t* counts;         // [batch] rows of `added` that are there, or NULL
  ScaleRange range;
  PagedCache cache;
};

// Rows of the segments before each one, sums[s], and of all, sums[segments]: by one workgroup in a launch
// of its own, or (up to kFusedSegments segments, a length a thread) by every workgroup for itself.
constexpr int kSumThreads = 1024;
constexpr int kFusedSegments = kThreads;

// A packed row number as the i32 of the packed layout (rows past 2^31 - 1 are not read).
template <typename Sum>
__device__ __forceinline__ Sum packed_row(int64_t row) {
  if constexpr (sizeof(Sum) == 4) return static_cast<Sum>(row < INT32_MAX ? row : INT32_MAX);
  else return row;
}

// n and what a DPP move brings from another lane (0 where there is none).
template <int CONTROL, int ROWS>
__device__ __forceinline__ int64_t add_lane(int64_t n) {
  const unsigned low = __builtin_amdgcn_update_dpp(0, static_cast<int>(n), CONTROL, ROWS, 0xF, false);
  const int high = __builtin_amdgcn_update_dpp(0, static_cast<int>(n >> 32), CONTROL, ROWS, 0xF, false);
  return n + (static_cast<int64_t>(high) << 32 | low);
}

// The sum of `n` over the workgroup's threads up to and with this one. (In the vector ALU: with the
// lanes' exchange through LDS a read of 18,000 rows in 8 bits took 6.4 us for 6.1.)
template <int THREADS>
__device__ __forceinline__ int64_t running_sum(int64_t n, int64_t (&wave_total)[THREADS / 64]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // shifts within 16 lanes, then their last lane's to the next 16, then lane 31's to the upper 32
  int64_t sum = add_lane<0x114, 0xF>(add_lane<0x112, 0xF>(add_lane<0x111, 0xF>(n)));
  sum = add_lane<0x118, 0xF>(sum);
  sum = add_lane<0x143, 0xC>(add_lane<0x142, 0xA>(sum));
  if (lane == 63) wave_total[wave] = sum;
  __syncthreads();
  for (int w = 0; w < wave; ++w) sum += wave_total[w];
  return sum;
}

template <typename Sum>
__global__ __launch_bounds__(kSumThreads) void paged_sum_kernel(PagedCache cache, int64_t segments, Sum* sums) {
  __shared__ int64_t wave_total[kSumThreads / 64];
  __shared__ int64_t before;  // rows of the segments of earlier rounds
  if (threadIdx.x == 0) before = 0, sums[0] = 0;
  for (int64_t s0 = 0; s0 < segments; s0 += kSumThreads) {
    const int64_t s = s0 + threadIdx.x;
    const int64_t sum = running_sum<kSumThreads>(s < segments ? cache.rows(s) : 0, wave_total) + before;
    if (s < segments) sums[s + 1] = packed_row<Sum>(sum);
    __syncthreads();
    if (threadIdx.x == kSumThreads - 1) before = sum;
    __syncthreads();
  }
}

template <typename Sum>
__device__ __forceinline__ void sum_lengths(const PagedCache& cache, int segments, Sum* sums) {
  __shared__ int64_t wave_total[kThreads / 64];
  const int thread = static_cast<int>(threadIdx.x);
  const int64_t sum = running_sum<kThreads>(thread < segments ? cache.rows(thread) : 0, wave_total);
  if (thread == 0) sums[0] = 0;
  if (thread < segments) sums[thread + 1] = packed_row<Sum>(sum);
  __syncthreads();
}

// ---------------------------------------------------------------------------------------
struct ReadArgs {
  PagedCache cache;
  int64_t segments, total;
  int32_t* cumulative;  // [segments + 1]: written by the fused form, read by the other
  void* keys;
  void* values;
  float* positions;
};

constexpr int kReadRows = 64;  // of a workgroup

// The segment that packed row `row` < cumulative[segments] belongs to: the largest s with
// cumulative[s] <= row.
__device__ __forceinline__ int segment_of(const int32_t* cumulative, int segments, int row) {
  int low = 0, high = segments;
  while (high - low > 1) {
    const int mid = (low + high) >> 1;
    if (cumulative[mid] <= row) low = mid;
    else high = mid;
  }
  return low;
}

// ---------------------------------------------------------------------------------------
struct CompactArgs {
  PagedCache cache;
  int64_t segments;
  int chunks;                   // of a workgroup's rows of a segment
  const int32_t* target;        // [segments, target_pages]
  int target_pages;
  const int64_t* removed;       // sorted packed rows
  int64_t removed_count;
  const int64_t* sums;          // [segments + 1], unless the workgroups sum the lengths themselves
  int32_t* new_lengths;
};

// The first of [low, high) that is not `before` (all of those before it are): 32 lanes look at 32
// places a round, each half of the wave for a range of its own.
template <typename F>
__device__ __forceinline__ int64_t half_search(int64_t low, int64_t high, F before) {
  const int place = threadIdx.x & 31, half = (threadIdx.x >> 5) & 1;
  while (true) {
    const int64_t step = (high - low + 31) / 32;  // 0 once the range is empty
    const int64_t at = low + place * step;
    const bool below = step > 0 && at < high && before(at);
    const unsigned held = static_cast<unsigned>(__ballot(below) >> (32 * half));
    const int count = __builtin_popcount(held);  // of the places looked at, the first ones
    if (step > 0) {
      const int64_t next = low + count * step;
      low = count > 0 ? low + (count - 1) * step + 1 : low;
      high = next < high ? next : high;
    }
    if (!__any(high > low)) return low;
  }
}

// ---------------------------------------------------------------------------------------
template <typename F>
int dispatch_type(int dtype, F&& f) {
  switch (dtype) {
    case LR_DTYPE_BF16: return f.template operator()<__bf16>();
    case LR_DTYPE_F16: return f.template operator()<_Float16>();
    default: return f.template operator()<float>();
  }
}

bool paged_type(int dtype) {
  return dtype == LR_DTYPE_BF16 || dtype == LR_DTYPE_F16 || dtype == LR_DTYPE_F32;
}

// The entry points' common parts: checks and arguments; `launch` gets the arguments.
template <typename Launch>
int append_paged(const void* keys, const int64_t* key_strides, const void* values,
                 const int64_t* value_strides, const void* queries,
                 const int64_t* query_strides, void* out_queries, int64_t batch,
                 int64_t kv_heads, int64_t query_heads, int64_t added, int64_t dim,
                 int dtype, const int64_t* positions, const float* cos,
                 const float* sin, int64_t table_rows, int64_t half,
                 const int32_t* counts, void* pages, int64_t page_count,
                 int64_t page_size, const int32_t* table, int64_t max_pages,
                 const int32_t* lengths, Launch&& launch) {
  clear_error();
  LR_REQUIRE(paged_type(dtype), "Appended rows must be bf16, f16 or f32");
  LR_REQUIRE(batch > 0 && kv_heads > 0 && added >= 0 && query_heads >= 0 &&
                 (query_heads > 0) == (queries != nullptr),
             "Invalid appended shape");
  LR_REQUIRE(batch <= INT32_MAX / kv_heads, "Invalid appended shape");
  if (int status = check_paged(pages, page_count, page_size, dim, table, max_pages, lengths,
                               batch * kv_heads))
    return status;
  if (added == 0) return LR_OK;
  LR_REQUIRE(keys && values && positions && key_strides && value_strides &&
                 (queries == nullptr) == (out_queries == nullptr) &&
                 (queries == nullptr || query_strides != nullptr),
             "Invalid appended KV");
  LR_REQUIRE(half >= 0 && half % 8 == 0 && 2 * half <= dim && table_rows >= 0 &&
                 (half == 0 || (cos && sin && table_rows > 0)),
             "Rotated channels must be a multiple of 16, at most the head dimension, with tables");
  LR_REQUIRE(added <= INT32_MAX / (batch * kv_heads) &&
                 (query_heads == 0 || added <= INT32_MAX / batch / query_heads),
             "Appended grid too large");
  uintptr_t alignment = reinterpret_cast<uintptr_t>(keys) | reinterpret_cast<uintptr_t>(values) |
                        reinterpret_cast<uintptr_t>(queries) |
                        reinterpret_cast<uintptr_t>(out_queries) | reinterpret_cast<uintptr_t>(cos) |
                        reinterpret_cast<uintptr_t>(sin);
  const int64_t elem = dtype == LR_DTYPE_F32 ? 4 : 2;
  for (int i = 0; i < 3; ++i) {
    alignment |= static_cast<uintptr_t>((key_strides[i] | value_strides[i]) * elem);
    if (queries != nullptr) alignment |= static_cast<uintptr_t>(query_strides[i] * elem);
  }
  LR_REQUIRE(alignment % 16 == 0, "Appended operands must be 16-byte aligned");

  AppendArgs args{};
  auto rows = [](const void* base, const int64_t* strides) {
    return base ? Rows{base, strides[0], strides[1], strides[2]} : Rows{};
  };
  args.keys = rows(keys, key_strides);
  args.values = rows(values, value_strides);
  args.queries = rows(queries, query_strides);
  args.out_queries = out_queries;
  args.positions = positions;
  args.cos = cos;
  args.sin = sin;
  args.table_rows = table_rows;
  args.half = static_cast<int>(half);
  args.kv_heads = static_cast<unsigned>(kv_heads);
  args.query_heads = static_cast<unsigned>(query_heads);
  args.added = static_cast<unsigned>(added);
  args.kv_rows = static_cast<unsigned>(batch * kv_heads * added);
  args.query_rows = static_cast<unsigned>(batch * query_heads * added);
  args.counts = counts;
  args.cache = paged_cache(pages, page_count, page_size, table, max_pages, lengths);
  args.batch = static_cast<unsigned>(batch);
  return launch(args);
}

template <typename Launch>
int read_paged(const void* pages, int64_t page_count, int64_t page_size,
               const int32_t* table, int64_t max_pages, const int32_t* lengths,
               int64_t segments, int64_t dim, int dtype, int64_t total, void* keys,
               void* values, float* positions, int32_t* cumulative, void* stream,
               Launch&& launch) {
  clear_error();
  LR_REQUIRE(paged_type(dtype), "Rows are read as bf16, f16 or f32");
  if (int status = check_paged(pages, page_count, page_size, dim, table, max_pages, lengths, segments))
    return status;
  LR_REQUIRE(total >= 0 && total <= INT32_MAX && cumulative &&
                 (total == 0 || (keys && values && positions)),
             "Invalid packed buffers");
  LR_REQUIRE(((reinterpret_cast<uintptr_t>(keys) | reinterpret_cast<uintptr_t>(values)) % 16) == 0,
             "Packed buffers must be 16-byte aligned");
  const int64_t blocks = ceil_div(total, kReadRows);
  LR_REQUIRE(launchable(blocks, kThreads), "Packed rows' grid too large");
  // One launch where a workgroup can sum the lengths itself, beside its rows' lookups; calls without
  // rows or pages have only the sums to write.
  const bool fused = segments <= kFusedSegments && total > 0 && page_count > 0;
  const PagedCache cache = paged_cache(pages, page_count, page_size, table, max_pages, lengths);
  if (!fused) {
    hipLaunchKernelGGL(paged_sum_kernel<int32_t>, dim3(1), dim3(kSumThreads), 0, as_stream(stream),
                       cache, segments, cumulative);
    if (int status = check_launch("paged_read lengths")) return status;
    if (total == 0 || page_count == 0) return LR_OK;
  }
  const ReadArgs args{cache, segments, total, cumulative, keys, values, positions};
  return launch(args, blocks, fused);
}

inline size_t compact_paged_workspace(int64_t segments) {
  return segments > kFusedSegments ? static_cast<size_t>(segments + 1) * sizeof(int64_t) : 0;
}

// (a workgroup takes `group_rows` rows of a segment)
template <typename Launch>
int compact_paged(int group_rows, void* pages, int64_t page_count, int64_t page_size,
                  const int32_t* table, int64_t max_pages, const int32_t* lengths,
                  int64_t segments, int64_t dim, const int64_t* removed,
                  int64_t removed_count, const int32_t* target, int64_t target_pages,
                  int32_t* new_lengths, void* workspace, size_t workspace_size,
                  void* stream,
                  Launch&& launch) {
  clear_error();
  if (int status = check_paged(pages, page_count, page_size, dim, table, max_pages, lengths, segments))
    return status;
  LR_REQUIRE(removed_count >= 0 && (removed_count == 0 || removed) && new_lengths &&
                 target_pages >= 0 && target_pages <= INT32_MAX / 2 / page_size &&
                 (target || target_pages == 0),
             "Invalid compaction");
  const size_t needed = compact_paged_workspace(segments);
  LR_REQUIRE(workspace_size >= needed && (needed == 0 || workspace) &&
                 reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
             "Compaction workspace too small");
  // rows move while other workgroups still read theirs, and the lengths
  LR_REQUIRE((target != table || target_pages == 0 || page_count == 0) && new_lengths != lengths,
             "Compaction needs other pages and lengths than the cache's");
  CompactArgs args{};
  args.cache = paged_cache(pages, page_count, page_size, table, max_pages, lengths);
  args.segments = segments;
  // a segment's rows, kept or not, are at most what its table holds
  args.chunks = static_cast<int>(std::max<int64_t>(1, ceil_div(max_pages * page_size, group_rows)));
  args.target = target;
  // (without a page there is nothing to move: the lengths alone)
  args.target_pages = page_count == 0 ? 0 : static_cast<int>(target_pages);
  args.removed = removed;
  args.removed_count = removed_count;
  args.sums = static_cast<int64_t*>(workspace);
  args.new_lengths = new_lengths;
  LR_REQUIRE(launchable(segments * args.chunks, kThreads), "Compaction grid too large");
  if (needed) {
    hipLaunchKernelGGL(paged_sum_kernel<int64_t>, dim3(1), dim3(kSumThreads), 0, as_stream(stream),
                       args.cache, segments, static_cast<int64_t*>(workspace));
    if (int status = check_launch("paged_compact lengths")) return status;
  }
  return launch(args, static_cast<unsigned>(segments * args.chunks), needed == 0);
}

}  // namespace
}  // namespace lr
