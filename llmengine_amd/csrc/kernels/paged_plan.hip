// paged_plan.hip -- block tables, slot map and row offsets of one serving step.
//
// Everything a request gets follows from prefix sums over the requests: of the pages
// that finished requests give back, of the new tokens (row offsets) and of the pages
// asked for (places in the free stack).  One workgroup makes them with wave scans and
// then walks the pages and rows flat, a thread an entry, finding the entry's request by
// bisecting the sums in LDS, so one long request costs no more than many short ones.
// Bound by latency: a chain of a few dependent loads.
#include "../paged.hpp"

namespace mle {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
// Sums of clamped terms saturate here: two of them still fit 32 bits.
constexpr uint32_t kCap = 0x40000000u;

__device__ __forceinline__ uint32_t sat_add(uint32_t a, uint32_t b) {
  const uint32_t s = a + b;
  return s < kCap ? s : kCap;
}

// Inclusive saturating prefix sum over the workgroup; *total = the whole sum.  Two
// barriers; `part` holds kWaves words.
__device__ __forceinline__ uint32_t scan(uint32_t v, uint32_t* part, uint32_t* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t o = __shfl_up(v, off);
    if (lane >= off) v = sat_add(v, o);
  }
  if (lane == 63) part[wave] = v;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const uint32_t p = part[w];
    if (w < wave) before = sat_add(before, p);
    all = sat_add(all, p);
  }
  __syncthreads();
  *total = all;
  return sat_add(before, v);
}

// Index of the first of n ascending sums that is above x (n where none is).
__device__ __forceinline__ int first_above(const uint32_t* sums, int n, uint32_t x) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (sums[mid] > x) hi = mid; else lo = mid + 1;
  }
  return lo;
}

__device__ __forceinline__ int64_t pages_of(int64_t tokens, int page_size) {
  return (tokens + page_size - 1) / page_size;
}

__device__ __forceinline__ void row_out(const PlanArgs& a, int64_t row, int pos, int page) {
  a.positions[row] = pos;
  a.slots[row] = (uint32_t)page < (uint32_t)a.num_pages
                     ? page * a.page_size + pos % a.page_size : -1;
}

// ROWS: the rows' positions and slots too (else paged_rows_kernel makes them).
template <bool ROWS>
__global__ __launch_bounds__(kThreads) void paged_plan_kernel(PlanArgs a) {
  __shared__ uint32_t part[kWaves];
  __shared__ uint32_t sum_a[kThreads], sum_b[kThreads];  // inclusive sums of a chunk
  __shared__ int32_t s_cached[kThreads], s_have[kThreads], s_granted[kThreads];
  __shared__ uint32_t s_taken;
  const int tid = threadIdx.x;
  int32_t n_free = a.count[0];
  n_free = n_free < 0 ? 0 : n_free > a.num_pages ? a.num_pages : n_free;
  if (tid == 0) s_taken = 0;

  // 1. The finished requests' pages go on the stack (past its end: dropped).
  uint32_t top = (uint32_t)n_free;
  for (int base = 0; base < a.sequences; base += kThreads) {
    const int b = base + tid;
    uint32_t back = 0;
    if (b < a.sequences && a.fresh[b] < 0 && a.cached[b] > 0) {
      const int64_t have = pages_of(a.cached[b], a.page_size);
      back = (uint32_t)(have < a.max_pages ? have : a.max_pages);
    }
    uint32_t total;
    const uint32_t upto = scan(back, part, &total);
    if (total != 0) {
      sum_a[tid] = upto;
      __syncthreads();
      for (uint32_t i = tid; i < total; i += kThreads) {
        const int r = first_above(sum_a, kThreads, i);
        if (r >= kThreads) break;  // a saturated sum
        const uint32_t at = top + i;
        if (at < (uint32_t)a.num_pages)
          a.stack[at] = a.table[(int64_t)(base + r) * a.max_pages +
                                (i - (r ? sum_a[r - 1] : 0))];
      }
      __syncthreads();
    }
    top = sat_add(top, total);
  }
  if (top > (uint32_t)a.num_pages) top = (uint32_t)a.num_pages;
  __syncthreads();  // the stack's new entries are read below

  // 2. Row offsets, then the pages asked for and where on the stack they lie.
  uint32_t rows = 0, asked = 0;
  for (int base = 0; base < a.sequences; base += kThreads) {
    const int b = base + tid;
    const bool in = b < a.sequences;
    const int cached = in ? a.cached[b] : 0, fresh = in ? a.fresh[b] : 0;
    const uint32_t want = fresh > 0 ? (uint32_t)fresh : 0;
    uint32_t total_rows, total_add;
    const uint32_t rows_upto = scan(want < kCap ? want : kCap, part, &total_rows);
    const uint32_t end = sat_add(rows, rows_upto);
    int64_t have = 0, need = 0;
    bool valid = in && fresh >= 0 && cached >= 0 && end <= (uint32_t)a.tokens;
    if (valid) {
      have = pages_of(cached, a.page_size);
      need = pages_of((int64_t)cached + want, a.page_size);
      valid = need <= a.max_pages;
    }
    const uint32_t add = valid ? (uint32_t)(need - have) : 0;
    const uint32_t add_upto = scan(add, part, &total_add);
    const uint32_t until = sat_add(asked, add_upto);
    const bool granted = valid && (add == 0 || until <= top);
    sum_a[tid] = rows_upto;
    sum_b[tid] = add_upto;
    s_cached[tid] = cached;
    s_have[tid] = (int32_t)have;
    s_granted[tid] = granted;
    if (granted && add != 0) atomicMax(&s_taken, until);
    if (in) {
      a.kv_lens[b] = granted ? cached + (int)want : 0;
      a.granted[b] = granted || fresh < 0;
      a.cu[b + 1] = (int)(end < (uint32_t)a.tokens ? end : (uint32_t)a.tokens);
      if (b == 0) a.cu[0] = 0;
    }
    __syncthreads();
    for (uint32_t i = tid; i < total_add; i += kThreads) {
      const int r = first_above(sum_b, kThreads, i);
      if (r >= kThreads || !s_granted[r]) continue;
      const uint32_t j = i - (r ? sum_b[r - 1] : 0);
      a.table[(int64_t)(base + r) * a.max_pages + s_have[r] + j] =
          a.stack[top - 1 - (asked + i)];
    }
    if constexpr (ROWS) {
      for (uint32_t i = tid; i < total_rows; i += kThreads) {
        const int64_t row = (int64_t)rows + i;
        if (row >= a.tokens) break;
        const int r = first_above(sum_a, kThreads, i);
        if (r >= kThreads) break;
        if (!s_granted[r]) {
          row_out(a, row, 0, -1);
          continue;
        }
        const int pos = s_cached[r] + (int)(i - (r ? sum_a[r - 1] : 0));
        const int p = pos / a.page_size, fresh_page = p - s_have[r];
        // A new page is read where the table got it from: no wait for those stores.
        const int page =
            fresh_page >= 0
                ? a.stack[top - 1 - (asked + (r ? sum_b[r - 1] : 0) + (uint32_t)fresh_page)]
                : a.table[(int64_t)(base + r) * a.max_pages + p];
        row_out(a, row, pos, page);
      }
    }
    rows = sat_add(rows, total_rows);
    asked = sat_add(asked, total_add);
    __syncthreads();  // the sums are written again
  }
  if constexpr (ROWS)
    for (int64_t row = (int64_t)rows + tid; row < a.tokens; row += kThreads)
      row_out(a, row, 0, -1);
  if (tid == 0) a.count_out[0] = (int)(top - s_taken);
}

// Positions and slots of many rows, after the plan's own launch: a thread a row.
__global__ __launch_bounds__(256) void paged_rows_kernel(PlanArgs a) {
  const int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (row >= a.tokens) return;
  int lo = 0, hi = a.sequences;  // the first b with cu[b + 1] > row
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a.cu[mid + 1] > row) hi = mid; else lo = mid + 1;
  }
  // kv_lens is 0 for a refused request, whose rows are 1 or more.
  if (lo == a.sequences || a.kv_lens[lo] == 0) {
    row_out(a, row, 0, -1);
    return;
  }
  const int pos = a.cached[lo] + (int)(row - a.cu[lo]);
  row_out(a, row, pos, a.table[(int64_t)lo * a.max_pages + pos / a.page_size]);
}

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

// One workgroup's rows: above this many a second launch of a thread a row is made.
constexpr int kRowsInPlan = 8192;

hipError_t launch_paged_plan(const PlanArgs& a, hipStream_t stream) {
  if (a.tokens <= kRowsInPlan) {
    hipLaunchKernelGGL(paged_plan_kernel<true>, dim3(1), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
  }
  hipLaunchKernelGGL(paged_plan_kernel<false>, dim3(1), dim3(kThreads), 0, stream, a);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  hipLaunchKernelGGL(paged_rows_kernel, dim3((unsigned)((a.tokens + 255LL) / 256)), dim3(256), 0,
                     stream, a);
  return hipGetLastError();
}

hipError_t launch_rope_table(float* table, int positions, int rope_dim, double theta,
                             const float* freq_factors, hipStream_t stream) {
  const int64_t n = (int64_t)positions * (rope_dim / 2);
  const int64_t blocks = (n + 255) / 256;
  if (blocks > 0x7fffffff) return hipErrorInvalidValue;
  hipLaunchKernelGGL(rope_table_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, table, n,
                     rope_dim / 2, theta, freq_factors);
  return hipGetLastError();
}

}  // namespace mle
