// paged_attention.hip -- attention of new tokens over the paged KV cache.
//
// One wave per row and query head: 64 keys at a time, a lane per key for the logits, a
// lane per 4 dimensions for the sum over the keys, with the running maximum and sum of
// the softmax between them.
#include "../paged.hpp"
#include "../q8_0_device.hpp"

namespace mle {
namespace {

template <KvType T>
__device__ __forceinline__ float kv_at(const void* base, int64_t at) {
  if constexpr (T == KvType::kF16) return (float)static_cast<const _Float16*>(base)[at];
  else if constexpr (T == KvType::kBF16) return (float)static_cast<const __bf16*>(base)[at];
  else return (float)static_cast<const int8_t*>(base)[at];
}

template <KvType T>
__global__ __launch_bounds__(64) void attention_rows_kernel(AttentionArgs a) {
  __shared__ float s_q[256], s_p[64];
  __shared__ int64_t s_cell[64];
  const int lane = threadIdx.x, row = blockIdx.x, h = blockIdx.y;
  const int D = a.cache.head_dim, P = a.cache.page_size, G = a.cache.kv_heads;
  const int g = h / (a.heads / G);
  int lo = 0, hi = a.sequences;  // the first b with cu[b + 1] > row
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a.cu[mid + 1] > row) hi = mid; else lo = mid + 1;
  }
  if (lo == a.sequences || a.cu[lo] > row) return;
  const int64_t most = (int64_t)a.max_pages * P;
  const int fresh = a.cu[lo + 1] - a.cu[lo];
  const int pos = a.kv_lens[lo] - fresh + (row - a.cu[lo]);
  const int end = (int)(pos + 1LL < most ? pos + 1LL : most);
  const int begin = a.window > 0 && pos - a.window + 1 > 0 ? pos - a.window + 1 : 0;
  for (int d = lane; d < D; d += 64)
    s_q[d] = a.q[row * a.q_stride + (int64_t)h * D + d] * a.scale;
  __syncthreads();
  float m = -INFINITY, l = 0.0f, acc[4] = {};
  for (int j0 = begin; j0 < end; j0 += 64) {
    const int j = j0 + lane;
    float s = -INFINITY, v_scale = 1.0f;
    int64_t cell = -1;
    if (j < end) {
      const int page = a.table[(int64_t)lo * a.max_pages + j / P];
      if ((uint32_t)page < (uint32_t)a.cache.num_pages) {
        cell = ((int64_t)page * G + g) * P + j % P;
        const int64_t at = (cell - j % 16) * D + j % 16 * 8;
        float dot = 0.0f;
        for (int d = 0; d < D; ++d)
          dot = fmaf(s_q[d], kv_at<T>(a.cache.k, at + d / 8 * 128 + d % 8), dot);
        if (T == KvType::kInt8) {
          dot *= a.cache.k_scale[cell];
          v_scale = a.cache.v_scale[cell];
        }
        s = dot;
      }
    }
    float top = s;
    for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
    // A NaN logit (no key with it may be lost in the maximum) makes the row NaN below.
    const float m_new = fmaxf(m, top);
    const bool any = __any(cell >= 0);
    if (!any) continue;
    const float ref = m_new == -INFINITY ? 0.0f : m_new;
    const float keep = expf(m - ref), p = cell >= 0 ? expf(s - ref) : 0.0f;
    float sum = p;
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
    l = l * keep + sum;
    m = m_new;
    s_p[lane] = p * v_scale;
    s_cell[lane] = cell;
    __syncthreads();
    for (int i = 0; i < 4; ++i) {
      const int d = lane + 64 * i;
      if (d >= D) break;
      float o = acc[i] * keep;
      for (int x = 0; x < 64; ++x) {
        const int64_t c = s_cell[x];
        if (c < 0) continue;
        const int r = (j0 + x) % 16;
        o = fmaf(s_p[x],
                 kv_at<T>(a.cache.v, (c - r) * D + r / 4 % 2 * D * 8 + d * 8 + r / 8 * 4 + r % 4),
                 o);
      }
      acc[i] = o;
    }
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i) {
    const int d = lane + 64 * i;
    if (d < D) a.out[row * a.out_stride + (int64_t)h * D + d] = l != 0.0f ? acc[i] / l : 0.0f;
  }
}

}  // namespace

hipError_t launch_paged_attention(const AttentionArgs& a, hipStream_t stream) {
  const dim3 grid((unsigned)a.tokens, (unsigned)a.heads), block(64);
  switch (a.cache.type) {
    case KvType::kF16:
      hipLaunchKernelGGL(attention_rows_kernel<KvType::kF16>, grid, block, 0, stream, a);
      break;
    case KvType::kBF16:
      hipLaunchKernelGGL(attention_rows_kernel<KvType::kBF16>, grid, block, 0, stream, a);
      break;
    default:
      hipLaunchKernelGGL(attention_rows_kernel<KvType::kInt8>, grid, block, 0, stream, a);
  }
  return hipGetLastError();
}

}  // namespace mle
