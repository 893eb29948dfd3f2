// select.hpp -- device helpers of the kernels that pick the top tokens of logits rows: keys in
// the order of (value, lower index), reductions, histograms and a sort of few keys.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mle {
namespace {

typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));  // rows are 4-byte aligned


__device__ __forceinline__ uint64_t topk_key(float v, uint32_t i) {
  if (v != v) return 0;      // NaN (the row becomes uniform anyway)
  if (v == 0.0f) v = 0.0f;   // -0 -> +0
  uint32_t u = __builtin_bit_cast(uint32_t, v);
  u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((uint64_t)u << 32) | (uint32_t)~i;
}

__device__ __forceinline__ float key_value(uint64_t k) {
  uint32_t u = (uint32_t)(k >> 32);
  u = (u & 0x80000000u) ? (u & 0x7fffffffu) : ~u;
  return __builtin_bit_cast(float, u);
}

template <int NT, typename T, typename Op>
__device__ T block_reduce(T v, Op op, T* part) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = op(v, __shfl_xor(v, off, 64));
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  __syncthreads();  // part[] may still be read from an earlier reduction
  if (lane == 0) part[wave] = v;
  __syncthreads();
  T r = part[0];
#pragma unroll
  for (int i = 1; i < NT / 64; ++i) r = op(r, part[i]);
  return r;
}

// A logit under the temperature, rounded once.  Never contracted with what uses it: both
// passes have to see the same value, or a row's own maximum could lie above its maximum.
__device__ __forceinline__ float scaled_logit(float v, float inv_temp) {
#pragma clang fp contract(off)
  return v * inv_temp;
}

struct SelectLds {
  uint32_t hist[256];
  uint64_t cand[256];
  uint32_t digit, above, eq, total, ncand;
};

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int m) {
  const uint32_t lo = (uint32_t)__shfl_xor((int)(uint32_t)v, m, 64);
  const uint32_t hi = (uint32_t)__shfl_xor((int)(uint32_t)(v >> 32), m, 64);
  return ((uint64_t)hi << 32) | lo;
}

// Descending bitonic sort of 256 keys held by one wave, 4 per lane (element
// 4 lane + j), in registers.
__device__ void wave_sort256_desc(uint64_t (&v)[4]) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int size = 2; size <= 256; size <<= 1)
#pragma unroll
    for (int stride = size >> 1; stride > 0; stride >>= 1) {
      if (stride >= 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int e = 4 * lane + j;
          const uint64_t o = shfl_xor64(v[j], stride >> 2);
          const bool lower = (e & stride) == 0;
          const bool keep_max = lower == ((e & size) == 0);
          v[j] = keep_max ? (o > v[j] ? o : v[j]) : (o < v[j] ? o : v[j]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (j & stride) continue;  // handle each in-lane pair once, from its lower element
          const int e = 4 * lane + j;
          const bool desc = (e & size) == 0;
          const uint64_t a = v[j], c = v[j + stride];
          const bool swap = desc ? a < c : a > c;
          v[j] = swap ? c : a;
          v[j + stride] = swap ? a : c;
        }
      }
    }
}

// hist[bin] += 1 for every lane with `in`.  Lanes that all name one bin (ties, the leading
// digits) add once: 16384 single adds to one LDS word took 7 us a digit (MI355X).
__device__ __forceinline__ void count_bin(uint32_t* hist, uint32_t bin, bool in) {
  const uint64_t lanes = __builtin_amdgcn_ballot_w64(in);
  if (lanes == 0) return;  // uniform
  const int first = __builtin_ctzll(lanes);
  const uint32_t one = (uint32_t)__builtin_amdgcn_readlane((int)bin, first);
  if (__builtin_amdgcn_ballot_w64(in && bin == one) == lanes) {
    if ((int)(threadIdx.x & 63) == first) atomicAdd(&hist[one], (uint32_t)__builtin_popcountll(lanes));
  } else if (in) {
    atomicAdd(&hist[bin], 1u);
  }
}

// The digit of the histogram's bins from the top in which the `need`-th key lies, by one wave.
__device__ __forceinline__ void find_digit(SelectLds& sm, int need) {
  const int lane = threadIdx.x & 63;
  uint32_t h[4], local = 0;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    h[t] = sm.hist[255 - (4 * lane + t)];
    local += h[t];
  }
  uint32_t incl = local;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t o = (uint32_t)__shfl_up((int)incl, off, 64);
    if (lane >= off) incl += o;
  }
  uint32_t run = incl - local;  // keys in the bins above this lane's first bin
  if (lane == 63) sm.total = incl;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    if (run < (uint32_t)need && (uint32_t)need <= run + h[t]) {
      sm.digit = 255u - (uint32_t)(4 * lane + t);
      sm.above = run;
      sm.eq = h[t];
    }
    run += h[t];
  }
}

// The candidates' first k, largest first, by one wave.
__device__ __forceinline__ void sort_candidates(SelectLds& sm, int k, uint64_t* __restrict__ out) {
  const int lane = threadIdx.x & 63;
  uint64_t v[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = sm.cand[4 * lane + j];
  wave_sort256_desc(v);
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (4 * lane + j < k) out[4 * lane + j] = v[j];
}

}  // namespace
}  // namespace mle
