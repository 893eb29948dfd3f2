// paged_write.hip -- rotary embedding of a step's q and k rows, and the write of k and v
// into the paged cache.
//
// A pair (x, y) turns to (x c - y s, x s + y c).  Both products are exact in 64 bits; their
// sum is rounded to 64 bits (an fma each) and then to 32: the same bits whatever the order,
// and with them the same 8-bit quants, which a last-bit difference could move by a whole step.
// The 64-bit work hides behind memory: the kernel is bound by HBM (q in and out above
// all).  MI355X: 8192 tokens of 32 heads of 128 over 8 KV heads into 8 bits 84 us, 4.25 TB/s
// of the 4.9 that a large copy reaches; 1531 tokens of 14 heads of 64 6.4 us and 32 tokens of
// a 32-head model 6.4 us, next to 3.4 us of an empty launch.
//
// k and v have workgroups of their own, token by token within a head: the lines of a K tile
// hold 8 dimensions of 16 tokens each, and so fill within one workgroup (1531 tokens 7.4 ->
// 6.6 us, 8192 tokens 85.6 -> 83.1).  A group of lanes takes two heads of q of one token,
// whose loads are in flight together (32 tokens 6.6 -> 6.1 us; four heads no better).
//
// A group of lanes takes one head's row, 8 elements a lane, so that the amax of an 8-bit
// row is a few lane exchanges.  A V tile holds 4 tokens of one dimension together: where
// the rows r .. r + 3 fill such a place, the group of the first writes all four, 8 bytes
// at a time, and the others' groups leave it to that one; any other row writes its
// elements one by one.
#include "../paged.hpp"
#include "../q8_0_device.hpp"

namespace mle {
namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));

struct Row8 {
  float x[8];
};

// The 8 elements of lane `s` of a head's row: where the rotation pairs i with i + half,
// two runs of 4 that hold 4 whole pairs, else one run of 8.
struct Span {
  int a, b;  // first elements of the two runs of 4
};
__device__ __forceinline__ Span span_of(int s, int rope_dim, bool halves) {
  if (halves && s * 8 < rope_dim) return {s * 4, rope_dim / 2 + s * 4};
  return {s * 8, s * 8 + 4};
}

__device__ __forceinline__ Row8 load8(const float* p, Span sp) {
  const f32x4 u = *reinterpret_cast<const f32x4*>(p + sp.a);
  const f32x4 v = *reinterpret_cast<const f32x4*>(p + sp.b);
  return {{u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w}};
}

__device__ __forceinline__ void turn(float& x, float& y, float c, float s) {
  const double dx = x, dy = y, dc = c, ds = s;
  x = (float)__builtin_fma(dx, dc, -(dy * ds));
  y = (float)__builtin_fma(dx, ds, dy * dc);
}

// The pairs of lane s: i = 4s .. 4s + 3 either way.
__device__ __forceinline__ void rotate8(Row8& r, const float* rope_row, int s, bool halves) {
  const f32x4 t0 = *reinterpret_cast<const f32x4*>(rope_row + 8 * s);
  const f32x4 t1 = *reinterpret_cast<const f32x4*>(rope_row + 8 * s + 4);
  const float c[4] = {t0.x, t0.z, t1.x, t1.z}, n[4] = {t0.y, t0.w, t1.y, t1.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (halves) turn(r.x[i], r.x[4 + i], c[i], n[i]);
    else turn(r.x[2 * i], r.x[2 * i + 1], c[i], n[i]);
  }
}

// Largest magnitude over a group of LPR lanes as a bit pattern: the order of the patterns
// is that of the magnitudes, infinity and then NaN above all numbers, so neither is lost.
template <int LPR>
__device__ __forceinline__ float amax_of(const Row8& r) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t b = __builtin_bit_cast(uint32_t, r.x[i]) & 0x7fffffffu;
    m = b > m ? b : m;
  }
#pragma unroll
  for (int off = LPR / 2; off > 0; off >>= 1) {
    const uint32_t o = (uint32_t)__shfl_xor((int)m, off);
    m = o > m ? o : m;
  }
  return __builtin_bit_cast(float, m);
}

// Element to the cache's type, as bits.
template <KvType T>
__device__ __forceinline__ uint32_t cell_of(float x, float scale) {
  if constexpr (T == KvType::kF16) {
    return __builtin_bit_cast(uint16_t, (_Float16)x);
  } else if constexpr (T == KvType::kBF16) {
    return __builtin_bit_cast(uint16_t, (__bf16)x);
  } else {
    if (!(scale > 0.0f)) return 0;  // an all-zero row (or a NaN one: its scale is NaN)
    float q = __builtin_rintf(x / scale);
    q = q > 127.0f ? 127.0f : q < -127.0f ? -127.0f : q;  // a NaN (inf / inf) fails both
    return (uint32_t)(q == q ? (int)q : 0) & 0xffu;
  }
}

// Four consecutive cells (4 * size bytes, aligned so) at element `at`.
template <KvType T>
__device__ __forceinline__ void put4(void* base, int64_t at, const uint32_t (&c)[4]) {
  if constexpr (T == KvType::kInt8) {
    *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(base) + at) =
        c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24;
  } else {
    uint2 w = make_uint2(c[0] | c[1] << 16, c[2] | c[3] << 16);
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(base) + at) = w;
  }
}

template <KvType T>
__device__ __forceinline__ void put1(void* base, int64_t at, uint32_t c) {
  if constexpr (T == KvType::kInt8) static_cast<uint8_t*>(base)[at] = (uint8_t)c;
  else static_cast<uint16_t*>(base)[at] = (uint16_t)c;
}

// Heads of q that a group of lanes takes: their loads are in flight together.
constexpr int kQHeads = 2;

// LPR lanes (a power of two, at least head_dim / 8) take one head's row of one token.
template <KvType T, int LPR>
__global__ __launch_bounds__(256) void paged_kv_write_kernel(KvWriteArgs a) {
  const int G = a.cache.kv_heads, D = a.cache.head_dim, P = a.cache.page_size;
  // The first workgroups take k and v, head by head, the others q, token by token.
  const bool is_q = blockIdx.x >= a.kv_blocks;
  const uint32_t item = ((blockIdx.x - (is_q ? a.kv_blocks : 0)) * 256 + threadIdx.x) / LPR;
  const int s = threadIdx.x % LPR;
  // A group's lanes share `item`, and no path below parts them across an exchange.
  const uint32_t q_items = (uint32_t)(a.heads + kQHeads - 1) / kQHeads;  // of a token
  if (item >= (uint32_t)a.tokens * (is_q ? q_items : 2 * G)) return;
  const int t = (int)(is_q ? item / q_items : item % (uint32_t)a.tokens);
  const int h = (int)(is_q ? item % q_items : item / (uint32_t)a.tokens);
  const bool live = s * 8 < D;
  const bool halves = a.rope_halves != 0;
  int pos = 0;
  bool placed = true;
  if (a.rope != nullptr) {
    pos = a.positions[t];
    placed = (uint32_t)pos < (uint32_t)a.rope_positions;
  }
  const float* rope_row = a.rope + (int64_t)pos * a.rope_dim;
  const bool turns = a.rope != nullptr && placed && s * 8 < a.rope_dim;

  if (is_q) {
    if (!live) return;
    const Span sp = span_of(s, a.rope_dim, halves);
    const float* q = a.q + t * a.q_stride + (int64_t)h * kQHeads * D;
    float* o = a.q_out + t * a.q_out_stride + (int64_t)h * kQHeads * D;
    const int n = a.heads - h * kQHeads;  // heads from here on
    Row8 r[kQHeads];
#pragma unroll
    for (int i = 0; i < kQHeads; ++i)
      if (i < n) r[i] = load8(q + i * D, sp);
#pragma unroll
    for (int i = 0; i < kQHeads; ++i) {
      if (i >= n) continue;
      if (turns) rotate8(r[i], rope_row, s, halves);
      if (!placed) r[i] = {};
      float* to = o + i * D;
      *reinterpret_cast<f32x4*>(to + sp.a) =
          f32x4{r[i].x[0], r[i].x[1], r[i].x[2], r[i].x[3]};
      *reinterpret_cast<f32x4*>(to + sp.b) =
          f32x4{r[i].x[4], r[i].x[5], r[i].x[6], r[i].x[7]};
    }
    return;
  }

  const int64_t cells = (int64_t)a.cache.num_pages * P;  // slots of the cache
  const int slot = a.slots[t];
  if (!placed || slot < 0 || slot >= cells) return;
  const int page = slot / P, off = slot - page * P, row = off % kKvTile;

  if (h < G) {  // K
    const int g = h;
    const Span sp = span_of(s, a.rope_dim, halves);
    Row8 r = {};
    if (live) r = load8(a.k + t * a.k_stride + (int64_t)g * D, sp);
    if (turns && live) rotate8(r, rope_row, s, halves);
    const int64_t cell = ((int64_t)page * G + g) * P + off;
    float scale = 1.0f;
    if constexpr (T == KvType::kInt8) {
      scale = amax_of<LPR>(r) * (1.0f / 127.0f);
      if (s == 0) a.cache.k_scale[cell] = scale;
    }
    if (!live) return;
    const int64_t tile = (cell - row) * D + row * 8;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int d = half ? sp.b : sp.a;
      uint32_t c[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] = cell_of<T>(r.x[4 * half + i], scale);
      put4<T>(a.cache.k, tile + (d / 8) * (kKvTile * 8) + d % 8, c);
    }
    return;
  }

  // V: does this row's place of four tokens lie whole in four rows of the step?
  const int g = h - G;
  const int quad = off % 4, first = t - quad;
  bool whole = first >= 0 && first + 4 <= a.tokens;
  if (whole)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      whole = whole && a.slots[first + i] == slot - quad + i;
      if (a.rope != nullptr)  // the rows that are not written at all do not count
        whole = whole && (uint32_t)a.positions[first + i] < (uint32_t)a.rope_positions;
    }
  if (whole && quad != 0) return;
  Row8 r[4] = {};
  float scale[4] = {1.0f, 1.0f, 1.0f, 1.0f};
  const int64_t cell = ((int64_t)page * G + g) * P + off;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (live && (whole || i == 0))
      r[i] = load8(a.v + (int64_t)(t + i) * a.v_stride + (int64_t)g * D, {s * 8, s * 8 + 4});
  if constexpr (T == KvType::kInt8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i != 0 && !whole) break;
      scale[i] = amax_of<LPR>(r[i]) * (1.0f / 127.0f);
      if (scale[i] <= kTinyScale) scale[i] = 0.0f;
      if (s == 0) a.cache.v_scale[cell + i] = scale[i];
    }
  }
  if (!live) return;
  const int64_t tile = (cell - row) * D + (row / 4 % 2) * (D * 8) + (row / 8) * 4 + row % 4;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int64_t at = tile + (int64_t)(s * 8 + e) * 8;
    if (whole) {
      uint32_t c[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] = cell_of<T>(r[i].x[e], scale[i]);
      put4<T>(a.cache.v, at, c);
    } else {
      put1<T>(a.cache.v, at, cell_of<T>(r[0].x[e], scale[0]));
    }
  }
}

// Lanes of a head's row.
int lanes_of(int head_dim) { return head_dim <= 64 ? 8 : head_dim <= 128 ? 16 : 32; }

template <KvType T>
hipError_t launch_typed(const KvWriteArgs& a, hipStream_t stream) {
  const int lpr = lanes_of(a.cache.head_dim);
  KvWriteArgs b = a;
  const KvWriteBlocks n =
      paged_kv_write_blocks(a.tokens, a.heads, a.cache.kv_heads, a.cache.head_dim);
  b.kv_blocks = (uint32_t)n.kv;
  const dim3 grid((unsigned)(n.kv + n.q)), block(256);
  if (lpr == 8)
    hipLaunchKernelGGL((paged_kv_write_kernel<T, 8>), grid, block, 0, stream, b);
  else if (lpr == 16)
    hipLaunchKernelGGL((paged_kv_write_kernel<T, 16>), grid, block, 0, stream, b);
  else
    hipLaunchKernelGGL((paged_kv_write_kernel<T, 32>), grid, block, 0, stream, b);
  return hipGetLastError();
}

}  // namespace

KvWriteBlocks paged_kv_write_blocks(int tokens, int heads, int kv_heads, int head_dim) {
  auto blocks_of = [&](int64_t rows) {
    return (tokens * rows * lanes_of(head_dim) + 255) / 256;
  };
  return {blocks_of(2 * (int64_t)kv_heads), blocks_of(((int64_t)heads + kQHeads - 1) / kQHeads)};
}

hipError_t launch_paged_kv_write(const KvWriteArgs& a, hipStream_t stream) {
  if (a.tokens <= 0) return hipSuccess;
  switch (a.cache.type) {
    case KvType::kF16: return launch_typed<KvType::kF16>(a, stream);
    case KvType::kBF16: return launch_typed<KvType::kBF16>(a, stream);
    default: return launch_typed<KvType::kInt8>(a, stream);
  }
}

}  // namespace mle
