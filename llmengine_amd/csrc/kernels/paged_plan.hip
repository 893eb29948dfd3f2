// paged_plan.hip -- block tables, slot map and row offsets of one serving step.
//
// Everything a request gets follows from prefix sums over the requests: of the pages
// that finished requests give back, of the new tokens (row offsets) and of the pages
// asked for (places in the free stack).  A workgroup makes the three in one scan and
// then walks the pages and rows flat, a thread an entry, finding the entry's request by
// bisecting the sums in LDS, so one long request costs no more than many short ones.
//
// Bound by latency: of the launch, the lengths' loads, the scan and the loads of the pages.
// So that nothing waits for what the launch itself writes, a page that was just given back
// is read from its request's table row instead of the stack, and one that was just taken
// from where the table gets it.  Many rows go to several workgroups, each with the whole
// scan (it is a few us) and a share of the pages and rows.  MI355X: 64 decoding requests
// 6.0 us (8.5 with three scans one after the other and the new entries read back), 512
// requests of which 64 bring prompts, 23000 rows, 9.9 us (16.2 with a second launch for the
// rows); an empty launch takes 3.4 us.  More requests than threads go through one workgroup
// in turns: 2000 decoding 15 us, 2000 of which 64 bring prompts 35 us.
#include "../launch.hpp"
#include "../paged.hpp"

namespace mle {
namespace {

// Sums of clamped terms saturate here: two of them still fit 32 bits.
constexpr uint32_t kCap = 0x40000000u;

__device__ __forceinline__ uint32_t sat_add(uint32_t a, uint32_t b) {
  const uint32_t s = a + b;
  return s < kCap ? s : kCap;
}

struct Sums {
  uint32_t back, rows, add;
};

__device__ __forceinline__ Sums operator+(const Sums& a, const Sums& b) {
  return {sat_add(a.back, b.back), sat_add(a.rows, b.rows), sat_add(a.add, b.add)};
}

// Inclusive saturating prefix sums over the workgroup; *total = the whole sums.  Two
// barriers; `part` holds a Sums of each wave.
template <int kThreads>
__device__ __forceinline__ Sums scan(Sums v, Sums* part, Sums* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const Sums o = {__shfl_up(v.back, off), __shfl_up(v.rows, off), __shfl_up(v.add, off)};
    if (lane >= off) v = v + o;
  }
  if (lane == 63) part[wave] = v;
  __syncthreads();
  Sums before{}, all{};
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    const Sums p = part[w];
    if (w < wave) before = before + p;
    all = all + p;
  }
  __syncthreads();
  *total = all;
  return before + v;
}

// Index of the first of kThreads ascending sums that is above x (kThreads where none is).
template <int kThreads>
__device__ __forceinline__ int first_above(const uint32_t* sums, uint32_t x) {
  int lo = 0;
#pragma unroll
  for (int step = kThreads / 2; step > 0; step >>= 1)
    if (sums[lo + step - 1] <= x) lo += step;
  return lo + (sums[lo] <= x);
}

__device__ __forceinline__ uint32_t pages_of(const PlanArgs& a, uint32_t tokens) {
  return tokens > 0 ? a.by_page.of(tokens - 1) + 1 : 0;
}

__device__ __forceinline__ void row_out(const PlanArgs& a, int64_t row, int pos, int page) {
  a.positions[row] = pos;
  a.slots[row] = (uint32_t)page < (uint32_t)a.num_pages
                     ? page * a.page_size + (pos - (int)a.by_page.of(pos) * a.page_size) : -1;
}

// Pages that a finished request gives back.
__device__ __forceinline__ uint32_t given_back(const PlanArgs& a, int cached, int fresh) {
  if (fresh >= 0 || cached <= 0) return 0;
  const uint32_t have = pages_of(a, cached);
  return have < (uint32_t)a.max_pages ? have : (uint32_t)a.max_pages;
}

// `arrived` counts the workgroups that have read the free count, which may be the place of
// the new one: the last of them writes it.
template <int kThreads>
__global__ __launch_bounds__(kThreads) void paged_plan_kernel(PlanArgs a, uint32_t* arrived) {
  __shared__ Sums part[kThreads / 64];
  __shared__ uint32_t s_back[kThreads], s_rows[kThreads], s_add[kThreads];  // inclusive sums
  __shared__ int32_t s_cached[kThreads], s_have[kThreads], s_granted[kThreads];
  __shared__ uint32_t s_taken;
  const int tid = threadIdx.x;
  // This thread's among the pages.
  const uint32_t first = blockIdx.x * kThreads + tid, step = gridDim.x * kThreads;
  const bool whole = a.sequences <= kThreads;  // one scan holds all requests
  const int cached0 = tid < a.sequences ? a.cached[tid] : 0;
  const int fresh0 = tid < a.sequences ? a.fresh[tid] : 0;
  int32_t n_free = a.count[0];
  n_free = n_free < 0 ? 0 : n_free > a.num_pages ? a.num_pages : n_free;
  if (tid == 0) s_taken = 0;

  // More requests than threads: all given-back pages first, by way of the stack.
  uint32_t top = (uint32_t)n_free;
  for (int base = 0; !whole && base < a.sequences; base += kThreads) {
    const int b = base + tid;
    Sums total;
    const Sums upto =
        scan<kThreads>({b < a.sequences ? given_back(a, a.cached[b], a.fresh[b]) : 0, 0, 0}, part,
                       &total);
    s_back[tid] = upto.back;
    __syncthreads();
    for (uint32_t i = tid; i < total.back; i += kThreads) {
      const int r = first_above<kThreads>(s_back, i);
      const uint32_t at = top + i;
      if (r < kThreads && at < (uint32_t)a.num_pages)  // past the stack's end: dropped
        a.stack[at] = a.table[(int64_t)(base + r) * a.max_pages + (i - (r ? s_back[r - 1] : 0))];
    }
    __syncthreads();
    top = sat_add(top, total.back);
  }
  if (!whole) {
    if (top > (uint32_t)a.num_pages) top = (uint32_t)a.num_pages;
    __syncthreads();  // the stack's new entries are read below
  }

  // Page at place `at` of the stack.
  auto stacked = [&](uint32_t at) {
    if (!whole || at < (uint32_t)n_free) return a.stack[at];
    const uint32_t i = at - (uint32_t)n_free;
    const int r = first_above<kThreads>(s_back, i);
    return a.table[(int64_t)r * a.max_pages + (i - (r ? s_back[r - 1] : 0))];
  };

  const int64_t share = ((int64_t)a.tokens + gridDim.x - 1) / gridDim.x;
  const int64_t row0 = blockIdx.x * share;
  const int64_t row1 = row0 + share < a.tokens ? row0 + share : a.tokens;
  uint32_t rows = 0, asked = 0;
  for (int base = 0; base < a.sequences; base += kThreads) {
    const int b = base + tid;
    const bool in = b < a.sequences;
    const int cached = base == 0 ? cached0 : in ? a.cached[b] : 0;
    const int fresh = base == 0 ? fresh0 : in ? a.fresh[b] : 0;
    const uint32_t want = fresh > 0 ? (uint32_t)fresh : 0;
    uint32_t have = 0, need = 0;
    const uint32_t most = (uint32_t)(cached > 0 ? cached : 0) + want;
    bool valid = in && fresh >= 0 && cached >= 0 && most <= 0x7fffffffu;
    if (valid) {
      have = pages_of(a, cached);
      need = pages_of(a, most);
      valid = need <= (uint32_t)a.max_pages;
    }
    // Whether its rows fit is known once they are counted; one that is cut off there is
    // refused with all after it that have rows, so that its pages in the sum do no harm.
    Sums total;
    const Sums upto = scan<kThreads>({whole ? given_back(a, cached, fresh) : 0,
                                      want < kCap ? want : kCap, valid ? need - have : 0},
                                     part, &total);
    if (whole) {
      top = sat_add((uint32_t)n_free, total.back);
      if (top > (uint32_t)a.num_pages) top = (uint32_t)a.num_pages;
    }
    const uint32_t end = sat_add(rows, upto.rows);
    valid = valid && (want == 0 || end <= (uint32_t)a.tokens);
    const uint32_t add = valid ? need - have : 0;
    const uint32_t until = sat_add(asked, upto.add);
    const bool granted = valid && (add == 0 || until <= top);
    s_back[tid] = upto.back;
    s_rows[tid] = upto.rows;
    s_add[tid] = upto.add;
    s_cached[tid] = cached;
    s_have[tid] = (int32_t)have;
    s_granted[tid] = granted;
    if (granted && add != 0) atomicMax(&s_taken, until);
    if (in && blockIdx.x == 0) {
      a.kv_lens[b] = granted ? cached + (int)want : 0;
      a.granted[b] = granted || fresh < 0;
      a.cu[b + 1] = (int)(end < (uint32_t)a.tokens ? end : (uint32_t)a.tokens);
      if (b == 0) a.cu[0] = 0;
    }
    __syncthreads();
    for (uint32_t i = first; whole && i < total.back; i += step) {
      const uint32_t at = (uint32_t)n_free + i;
      if (at >= (uint32_t)a.num_pages) break;  // past the stack's end: dropped
      const int r = first_above<kThreads>(s_back, i);
      if (r >= kThreads) break;  // a saturated sum
      a.stack[at] = a.table[(int64_t)r * a.max_pages + (i - (r ? s_back[r - 1] : 0))];
    }
    for (uint32_t i = first; i < total.add; i += step) {
      const int r = first_above<kThreads>(s_add, i);
      if (r >= kThreads || !s_granted[r]) continue;
      const uint32_t j = i - (r ? s_add[r - 1] : 0);
      a.table[(int64_t)(base + r) * a.max_pages + s_have[r] + j] = stacked(top - 1 - (asked + i));
    }
    for (int64_t row = (row0 > rows ? row0 : rows) + tid; row < row1; row += kThreads) {
      const uint32_t i = (uint32_t)(row - rows);
      if (i >= total.rows) break;
      const int r = first_above<kThreads>(s_rows, i);
      if (r >= kThreads) break;
      if (!s_granted[r]) {
        row_out(a, row, 0, -1);
        continue;
      }
      const int pos = s_cached[r] + (int)(i - (r ? s_rows[r - 1] : 0));
      const int p = (int)a.by_page.of(pos), fresh_page = p - s_have[r];
      const int page =
          fresh_page >= 0
              ? stacked(top - 1 - (asked + (r ? s_add[r - 1] : 0) + (uint32_t)fresh_page))
              : a.table[(int64_t)(base + r) * a.max_pages + p];
      row_out(a, row, pos, page);
    }
    rows = sat_add(rows, total.rows);
    asked = sat_add(asked, total.add);
    __syncthreads();  // the sums are written again
  }
  for (int64_t row = (row0 > rows ? row0 : rows) + tid; row < row1; row += kThreads)
    row_out(a, row, 0, -1);
  if (tid == 0) {
    bool last = true;
    if (gridDim.x > 1) {
      last = __hip_atomic_fetch_add(arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
             gridDim.x - 1;
      if (last) __hip_atomic_store(arrived, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    if (last) a.count_out[0] = (int)(top - s_taken);
  }
}

// One element a thread, made once for a model: bound by pow and sincos in 64 bits (131072
// positions of 64 pairs 70 us, 1 TB/s of writes).
__global__ __launch_bounds__(256) void rope_table_kernel(float* __restrict__ table,
                                                         int64_t n, int half, double theta,
                                                         const float* __restrict__ factors) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= n) return;
  const int i = (int)(e % half);
  double a = (double)(e / half) * pow(theta, -(double)i / half);
  if (factors != nullptr) a /= (double)factors[i];
  double s, c;
  sincos(a, &s, &c);
  reinterpret_cast<float2*>(table)[e] = make_float2((float)c, (float)s);
}

}  // namespace

// Rows of one workgroup, and of each of several: 512 requests with 23000 rows take 9.8 us in
// 256s, 10.3 in 1024s, 12.8 in 2048s with the pages left to the first.
constexpr int kRowsOfOne = 1024, kRowsOfMany = 256, kMostGroups = 256;

int plan_groups(int tokens, int sequences) {
  // With more requests than threads the given-back pages go by way of the stack, which only
  // one workgroup may write and read.
  if (tokens <= kRowsOfOne || sequences > 1024) return 1;
  const int n = (tokens + kRowsOfMany - 1) / kRowsOfMany;
  return n < kMostGroups ? n : kMostGroups;
}

SplitKNeed paged_plan_workspace(int tokens, int sequences) {
  SplitKNeed need;
  if (plan_groups(tokens, sequences) > 1) {
    need.counters = kCounterStride;
    need.scratch_bytes = 256;  // unused: a need of counters alone counts as none
  }
  return need;
}

hipError_t launch_paged_plan(const PlanArgs& args, const SplitKWorkspace& ws, hipStream_t stream) {
  PlanArgs a = args;
  a.by_page = Divisor((uint32_t)a.page_size);
  const dim3 grid((unsigned)plan_groups(a.tokens, a.sequences));
  if (a.sequences <= 256 && a.tokens <= 1024)
    hipLaunchKernelGGL(paged_plan_kernel<256>, grid, dim3(256), 0, stream, a, ws.counters);
  else
    hipLaunchKernelGGL(paged_plan_kernel<1024>, grid, dim3(1024), 0, stream, a, ws.counters);
  return hipGetLastError();
}

int64_t rope_table_blocks(int positions, int rope_dim) {
  return ((int64_t)positions * (rope_dim / 2) + 255) / 256;
}

hipError_t launch_rope_table(float* table, int positions, int rope_dim, double theta,
                             const float* freq_factors, hipStream_t stream) {
  const int64_t n = (int64_t)positions * (rope_dim / 2);
  hipLaunchKernelGGL(rope_table_kernel, dim3((unsigned)rope_table_blocks(positions, rope_dim)),
                     dim3(256), 0, stream, table, n, rope_dim / 2, theta, freq_factors);
  return hipGetLastError();
}

}  // namespace mle
