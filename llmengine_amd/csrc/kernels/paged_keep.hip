// paged_keep.hip -- the accepted path of a tree of drafted tokens takes the places that follow
// the cached tokens, in all layers; the pages past it go back.
//
// Request b has n new rows behind base cached tokens.  keep[b][i] is the row that becomes token
// base + i, for i < keep_counts[b]; rows increase along a path, keep[b][i] >= i, so what a later
// entry reads no earlier one overwrites, and some entries at a time are read before they are
// written.  A path ends before the first entry that is not above the one before it, or not a row.
//
// A wave has one head's path in one layer: the entries of one wave come in order, and nothing of
// a path crosses waves.  What bounds it: a chain of latencies (lengths, entries, page table,
// cells, stores; 1 x 8 nodes in 24 layers 6.4 us, next to 3.3 of an empty launch), and for more
// the lines of the cache that tokens lie in beside others: a token's K is D / 8 pieces of 16
// bytes (8 of 8 bits) 256 bytes apart, its V single elements 16 bytes apart.  32 trees of 64
// nodes, up to 8 of them kept, in 32 layers of 8-bit pages 20 us (13 where the lines are in a
// cache still).  With 48 kept of each 150 us, one entry at a time 232, 4 160; of f16 pages 267,
// 340 and 194, but 4 take 24 us instead of 16 where up to 8 are kept, as most paths are.
// (All with the pieces of 16 bits' K in scratch memory, 144 bytes a lane, where the compiler puts
// an array of class type that is filled under a condition; of 8 bits there is none.)
#include "../paged.hpp"

namespace mle {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kAtOnce = 8;  // entries of a path that are looked up, or moved, together

// The new rows of request b: lengths come from the caller's device memory and may be anything.
struct Rows {
  int base, n, kv_len;
  int entries;  // of its path, not checked yet; -1: every row stays
};

__device__ __forceinline__ Rows rows_of(const KeepArgs& a, int b) {
  const int64_t n = (int64_t)a.cu[b + 1] - a.cu[b];
  const int asked = a.counts[b];
  Rows r;
  r.kv_len = a.kv_lens[b] > 0 ? a.kv_lens[b] : 0;
  const bool there = n > 0 && n <= r.kv_len;
  r.n = there ? (int)n : 0;
  r.base = r.kv_len - r.n;
  r.entries = asked < a.keep_stride ? asked : a.keep_stride;
  if (r.entries > r.n) r.entries = r.n;
  if (asked < 0 || !there) r.entries = -1;
  return r;
}

// The entries [i0, i0 + kAtOnce) of a path, as far as they are rows above the ones before
// them: how many are, and `last` the row of the last one.
__device__ __forceinline__ int next_entries(const KeepArgs& a, int b, const Rows& r, int i0,
                                            int& last, int (&row)[kAtOnce]) {
  const int32_t* keep = a.keep + (int64_t)b * a.keep_stride;
#pragma unroll
  for (int j = 0; j < kAtOnce; ++j)
    row[j] = keep[i0 + j < r.entries ? i0 + j : r.entries - 1];
  int good = 0;
#pragma unroll
  for (int j = 0; j < kAtOnce; ++j) {
    if (good == j && i0 + j < r.entries && row[j] > last && row[j] < r.n) {
      last = row[j];
      ++good;
    }
  }
  return good;
}

// A token of request b as a cell of KV head 0's numbering; -1: in no page of the cache.
__device__ __forceinline__ int64_t cell_of(const KeepArgs& a, int b, int pos, int g) {
  const int at = (int)a.by_page.of((uint32_t)pos);
  if (at >= a.max_pages) return -1;
  const int page = a.table[(int64_t)b * a.max_pages + at];
  if ((uint32_t)page >= (uint32_t)a.num_pages) return -1;
  return ((int64_t)page * a.kv_heads + g) * a.page_size + (pos - at * a.page_size);
}

// The kept lengths, and the pages past them onto the stack, by one workgroup.
__device__ __forceinline__ void keep_lengths(const KeepArgs& a) {
  __shared__ int64_t wave_pages[kWaves];  // up to 31 bits in all, and the stack's
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int most = a.max_pages * a.page_size;
  int64_t top = 0;
  if (a.stack != nullptr) {
    top = *a.count;
    top = top < 0 ? 0 : top < a.num_pages ? top : a.num_pages;
  }
  for (int b0 = 0; b0 < a.sequences; b0 += kThreads) {
    const int b = b0 + tid;
    int first = 0, past = 0;  // pages of the request that go back
    if (b < a.sequences && a.granted[b] != 0) {
      const Rows r = rows_of(a, b);
      int kept = r.kv_len;
      if (r.entries >= 0) {
        kept = r.base;
        int last = -1, row[kAtOnce];
        for (int i0 = 0; i0 < r.entries; i0 += kAtOnce) {
          const int good = next_entries(a, b, r, i0, last, row);
          kept += good;
          if (good < kAtOnce) break;
        }
      }
      a.kept_lens[b] = kept;
      auto pages = [&](int len) {
        return (int)a.by_page.of((uint32_t)((len < most ? len : most) + a.page_size - 1));
      };
      first = pages(kept);
      past = pages(r.kv_len);
    }
    if (a.stack == nullptr) continue;
    const int mine = past - first;
    int64_t upto = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int64_t o = __shfl_up(upto, off);
      if (lane >= off) upto += o;
    }
    if (lane == 63) wave_pages[wave] = upto;
    __syncthreads();
    int64_t at = top + upto - mine;
    for (int w = 0; w < kWaves; ++w) {
      if (w < wave) at += wave_pages[w];
      top += wave_pages[w];
    }
    for (int j = 0; j < mine && at + j < a.num_pages; ++j)
      a.stack[at + j] = a.table[(int64_t)b * a.max_pages + first + j];
    top = top < a.num_pages ? top : a.num_pages;
    __syncthreads();  // wave_pages is written anew
  }
  if (a.stack != nullptr && tid == 0) *a.count_out = (int)top;
}

// E bytes an element; a wave moves one head's path of one layer.  The first workgroup has the
// lengths where they are asked for.
template <int E, int D>
__global__ __launch_bounds__(kThreads) void paged_keep_kernel(KeepArgs a) {
  uint32_t block = blockIdx.x;
  if (a.kept_lens != nullptr) {
    if (block == 0) {
      keep_lengths(a);
      return;
    }
    --block;
  }
  const int lane = threadIdx.x & 63;
  const uint32_t item = block * kWaves + (threadIdx.x >> 6);  // (layer, request, head)
  const uint32_t G = (uint32_t)a.kv_heads;
  if (item >= (uint32_t)a.layers * a.sequences * G) return;
  const int g = (int)(item % G), b = (int)(item / G % a.sequences);
  const int layer = (int)(item / G / a.sequences);
  if (a.granted[b] == 0) return;
  const Rows rows = rows_of(a, b);
  using Piece = std::conditional_t<E == 1, uint2, uint4>;  // 8 elements of K
  using Cell = std::conditional_t<E == 1, uint8_t, uint16_t>;
  constexpr int VL = (D + 63) / 64;
  static_assert(D / 8 <= 64);
  Piece* ck = static_cast<Piece*>(a.layer[layer].k);
  Cell* cv = static_cast<Cell*>(a.layer[layer].v);
  auto k_at = [&](int64_t cell) {
    const int64_t r = cell % kKvTile;
    return (cell - r) * (D / 8) + lane * kKvTile + r;
  };
  auto v_at = [&](int64_t cell, int l) {
    const int64_t r = cell % kKvTile;
    return (cell - r) * D + r / 4 % 2 * (D * 8) + (lane + 64 * l) * 8 + r / 8 * 4 + r % 4;
  };
  int last = -1;
  for (int i0 = 0; i0 < rows.entries; i0 += kAtOnce) {
    int row[kAtOnce];
    const int good = next_entries(a, b, rows, i0, last, row);
    int64_t from[kAtOnce], to[kAtOnce];  // to -1: nothing moves
    Piece k[kAtOnce];
    Cell v[kAtOnce][VL];
    float ks[kAtOnce], vs[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      to[j] = -1;
      if (j >= good || row[j] == i0 + j) continue;
      from[j] = cell_of(a, b, rows.base + row[j], g);
      to[j] = cell_of(a, b, rows.base + i0 + j, g);
      if (from[j] < 0) to[j] = -1;
    }
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      if (to[j] < 0) continue;
      if (lane < D / 8) k[j] = ck[k_at(from[j])];
#pragma unroll
      for (int l = 0; l < VL; ++l)
        if (lane + 64 * l < D) v[j][l] = cv[v_at(from[j], l)];
      if (E == 1 && lane == 0) {
        ks[j] = a.layer[layer].k_scale[from[j]];
        vs[j] = a.layer[layer].v_scale[from[j]];
      }
    }
    // All of it is here before anything is written over.
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0);
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      if (to[j] < 0) continue;
      if (lane < D / 8) ck[k_at(to[j])] = k[j];
#pragma unroll
      for (int l = 0; l < VL; ++l)
        if (lane + 64 * l < D) cv[v_at(to[j], l)] = v[j][l];
      if (E == 1 && lane == 0) {
        a.layer[layer].k_scale[to[j]] = ks[j];
        a.layer[layer].v_scale[to[j]] = vs[j];
      }
    }
    if (good < kAtOnce) break;
  }
}

template <int E>
void launch_moves(const KeepArgs& a, int head_dim, hipStream_t stream) {
  const int64_t blocks = paged_keep_blocks(a.layers, a.sequences, a.kv_heads) +
                         (a.kept_lens != nullptr ? 1 : 0);
  const dim3 grid((unsigned)blocks), block(kThreads);
  switch (head_dim) {
    case 64: hipLaunchKernelGGL((paged_keep_kernel<E, 64>), grid, block, 0, stream, a); break;
    case 96: hipLaunchKernelGGL((paged_keep_kernel<E, 96>), grid, block, 0, stream, a); break;
    case 128: hipLaunchKernelGGL((paged_keep_kernel<E, 128>), grid, block, 0, stream, a); break;
    default: hipLaunchKernelGGL((paged_keep_kernel<E, 256>), grid, block, 0, stream, a);
  }
}

}  // namespace

int64_t paged_keep_blocks(int layers, int sequences, int kv_heads) {
  return ((int64_t)layers * sequences * kv_heads + kWaves - 1) / kWaves;
}

hipError_t launch_paged_keep(const KeepArgs& args, KvType type, int head_dim,
                             hipStream_t stream) {
  KeepArgs a = args;
  a.by_page = Divisor(a.page_size);
  if (type == KvType::kInt8) launch_moves<1>(a, head_dim, stream);
  else launch_moves<2>(a, head_dim, stream);
  return hipGetLastError();
}

}  // namespace mle
