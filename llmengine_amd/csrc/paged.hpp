// paged.hpp -- internal launchers of the paged KV cache behind the C ABI (not exported),
// and its layout.  Every launcher assumes that the caller (capi.hip) has validated
// pointers and shapes; each only enqueues work on `stream` and returns the launch status.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "launch.hpp"

namespace mle {

constexpr int kKvTile = 16;  // tokens of a cache tile
// The write stores an 8-bit V row of this scale or a smaller one as zeros of scale 0, which
// the attention counts as this one: so it has the logarithm of every scale, and the weights
// of such rows, down to 2^-24 of the largest, are there beside scales up to 2^40.
constexpr float kTinyScale = 0x1p-64f;
// A launch of 256 threads a workgroup has fewer than 2^32 of them.
constexpr int64_t kMostBlocks = (int64_t(1) << 24) - 1;
enum class KvType { kF16 = 0, kBF16 = 1, kInt8 = 2 };
struct PagedCache {
  void* k;
  void* v;
  float* k_scale;
  float* v_scale;
  KvType type;
  int num_pages;
  int page_size;
  int kv_heads;
  int head_dim;
};

// x / d for 0 <= x < 2^31 as a product and a shift.
struct Divisor {
  uint32_t magic = 0, shift = 0;
  Divisor() = default;
  explicit Divisor(uint32_t d) {
    while ((1u << shift) < d) ++shift;
    magic = (uint32_t)(((uint64_t(1) << (31 + shift)) + d - 1) / d);
  }
  __host__ __device__ uint32_t of(uint32_t x) const {
    return (uint32_t)((uint64_t)x * magic >> 31) >> shift;
  }
};

struct PlanArgs {
  const int32_t* cached;
  const int32_t* fresh;  // new tokens, or negative: finished
  int sequences;
  int32_t* table;
  int max_pages;
  int page_size;
  int num_pages;
  int32_t* stack;
  const int32_t* count;
  int32_t* count_out;
  int tokens;
  int32_t* kv_lens;
  int32_t* cu;
  int32_t* positions;
  int32_t* slots;
  int32_t* granted;
  Divisor by_page;  // set by the launcher
};
// Many rows take a counter of the workspace.
SplitKNeed paged_plan_workspace(int tokens, int sequences);
hipError_t launch_paged_plan(const PlanArgs& a, const SplitKWorkspace& ws, hipStream_t stream);

int64_t rope_table_blocks(int positions, int rope_dim);
hipError_t launch_rope_table(float* table, int positions, int rope_dim, double theta,
                             const float* freq_factors, hipStream_t stream);

struct KvWriteArgs {
  PagedCache cache;
  const float* q;
  float* q_out;
  const float* k;
  const float* v;
  const float* rope;  // null: no rotation
  const int32_t* positions;
  const int32_t* slots;
  int64_t q_stride, q_out_stride, k_stride, v_stride;
  int heads;
  int rope_positions;
  int rope_dim;
  int rope_halves;
  int tokens;
  uint32_t kv_blocks;  // set by the launcher
};
// Workgroups of the write: for k and v, then for q.
struct KvWriteBlocks {
  int64_t kv, q;
};
KvWriteBlocks paged_kv_write_blocks(int tokens, int heads, int kv_heads, int head_dim);
hipError_t launch_paged_kv_write(const KvWriteArgs& a, hipStream_t stream);

struct AttentionArgs {
  PagedCache cache;
  const float* q;
  float* out;
  int64_t q_stride, out_stride;
  int heads;
  float scale;
  int window;
  const int32_t* table;
  int max_pages;
  const int32_t* kv_lens;
  const int32_t* cu;
  int sequences;
  int tokens;
  // Set by the launcher: heads of a KV head, keys of a table row.
  int group;
  int most;
  Divisor by_group, by_page;
};
constexpr int kAttentionThreads = 256;
constexpr int kFewRows = 16;  // up to this many rows of a tile the waves split the keys

// Places in a part of a tile of few rows: quads of a row's head_dim values, value quad c of
// row r at 16 (16 c + r) bytes, behind them a (maximum, sum) a row.  A group of threads that
// joins 2^bits rows takes quads() of them, thread `at` those of row at % 2^bits from
// at >> bits on, kThreads further on each time.
template <int D>
struct FewPart {
  static constexpr int kQuadsOfThread = D > 128 ? 2 : 1;
  static constexpr uint32_t kMl = kFewRows * D * 4, kBytes = kFewRows * (D + 4) * 4;
  static __host__ __device__ constexpr int quads(int bits) { return (D / 4) << bits; }
  static __host__ __device__ constexpr bool has(int at, int i, int bits) {
    return at + i * kAttentionThreads < quads(bits);
  }
  // Of a quad that the thread does not have, the part's first place: it is not used.
  static __host__ __device__ constexpr uint32_t quad_at(int at, int i, int bits) {
    if (!has(at, i, bits)) return 0;
    const uint32_t quad = (uint32_t)(at + i * kAttentionThreads) >> bits;
    return (quad * kFewRows + (uint32_t)(at & ((1 << bits) - 1))) * 16;
  }
  static __host__ __device__ constexpr uint32_t ml_at(int at, int bits) {
    return kMl + (uint32_t)(at & ((1 << bits) - 1)) * 8;
  }
};

// Workspace of a call with `rows` rows of one KV head (new tokens * heads / kv_heads).
SplitKNeed paged_attention_workspace(int head_dim, int64_t rows);
hipError_t launch_paged_attention(const AttentionArgs& a, const SplitKWorkspace& ws,
                                  hipStream_t stream);

}  // namespace mle
