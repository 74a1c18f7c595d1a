// What attention over the paged KV caches shares (paged_attention.hip: 4 bits; paged8_attention.hip: 8
// bits): the call's arguments, the rows and keys of a tile, probabilities, the merge of the parts, the
// plan and the entry point's checks.
#pragma once

#include <algorithm>
#include <cmath>

#include "attention_common.hpp"
#include "lds_copy.hpp"
#include "paged.hpp"

namespace lr {
namespace {

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

// Memory addressed as a wave-uniform base and a lane's offset. (In the global address space: a generic
// load also counts as an LDS access, and every wait for LDS would be one for memory.)
typedef const __attribute__((address_space(1))) uint8_t* PagedBytes;

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
  int rows;              // of a tile
  int waves, tile_rows;  // of a workgroup, of a tile's partial states
  int64_t tiles, units, splits, chunk;
};

// Which kernel runs and how many chunks the keys get: the choice with the least estimated time,
//   call + round R + p (step R + share S) [+ merge + megabyte M + state N, when the keys are split],
// where a chunk is p steps (a unit of 32 keys a wave), S workgroups share a compute unit, R rounds of
// them follow one another (`resident` to a compute unit), M is the MB of partial states written and
// read, and a thread of the merge loads N states. The constants (us) are each cache's own, with its
// kernels.
struct PagedCost {
  int rows, waves, resident;
  double call, round, step, share;
};
struct MergeCost {
  double call, megabyte, state;
};
struct PagedCosts {
  PagedCost kernels[3][3];  // d64, d128, d256
  MergeCost merge[3];
};
constexpr int kSplits[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64};
constexpr unsigned kComputeUnits = 256, kMostSplitGroups = 4096;  // (more of them need no splitting)

// Chunks' states that a thread of the merge loads together.
int merge_loads(int64_t splits) {
  return splits <= 2 * kMergeParts ? 2 : splits <= 5 * kMergeParts ? 5 : 8;
}

PagedPlan least_cost(const PagedCosts& costs, int64_t segments, int64_t groups, int64_t length,
                     int64_t max_keys, int64_t dim) {
  const int row = dim == 64 ? 0 : dim == 128 ? 1 : 2;
  const int64_t rows = length * groups;
  const MergeCost& merge = costs.merge[row];
  PagedPlan best{};
  double least = HUGE_VAL;
  for (const PagedCost& cost : costs.kernels[row]) {
    if (cost.rows > kSmallRows && rows <= kSmallRows) continue;
    PagedPlan p{};
    p.rows = cost.rows;
    p.waves = cost.waves;
    const int64_t tile = p.rows;
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
template <const PagedCosts& COSTS>
PagedPlan plan_paged(int64_t segments, int64_t groups, int64_t length, int64_t max_keys, int64_t dim) {
  thread_local int64_t sizes[5] = {};
  thread_local PagedPlan plan;
  const int64_t now[5] = {segments, groups, length, max_keys, dim};
  if (!std::equal(now, now + 5, sizes)) {
    plan = least_cost(COSTS, segments, groups, length, max_keys, dim);
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

// The entry points' common part: checks, plan and arguments; `launch` gets the arguments and the plan.
template <const PagedCosts& COSTS, typename Launch>
int attend_paged(const void* queries, const int64_t* query_strides, const void* pages,
                 int64_t page_count, int64_t page_size, const int32_t* table, int64_t max_pages,
                 const int32_t* lengths, int64_t batch, int64_t kv_heads, int64_t groups,
                 int64_t length, int64_t dim, int dtype, int64_t max_keys, const int32_t* counts,
                 float scale, void* out, void* workspace, size_t workspace_size, Launch&& launch) {
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
  const PagedPlan plan = plan_paged<COSTS>(segments, groups, length, max_keys, dim);
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
  return launch(args, plan);
}

template <const PagedCosts& COSTS>
size_t attend_paged_workspace(int64_t segments, int64_t groups, int64_t length, int64_t max_keys,
                              int64_t dim) {
  if (segments <= 0 || groups <= 0 || length <= 0 || max_keys < 0 || max_keys > INT32_MAX / 2 || dim <= 0)
    return 0;
  return plan_bytes(plan_paged<COSTS>(segments, groups, length, max_keys, dim), dim);
}

template <const PagedCosts& COSTS>
int describe_paged_plan(int64_t segments, int64_t groups, int64_t length, int64_t max_keys, int64_t dim,
                        int64_t* plan) {
  clear_error();
  LR_REQUIRE(dim == 64 || dim == 128 || dim == 256, "Head dimension must be 64, 128 or 256");
  LR_REQUIRE(segments > 0 && groups > 0 && length > 0 && max_keys >= 0 &&
                 max_keys <= INT32_MAX / 2 && plan,
             "Empty attention dimensions");
  const PagedPlan p = plan_paged<COSTS>(segments, groups, length, max_keys, dim);
  plan[0] = p.rows;
  plan[1] = p.waves;
  plan[2] = p.splits;
  return LR_OK;
}

}  // namespace
}  // namespace lr
