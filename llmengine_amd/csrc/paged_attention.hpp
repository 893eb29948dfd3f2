// paged_attention.hpp -- attention of new tokens over the paged KV cache.
//
// A source file includes it once, behind the definition of mle::kTrees: whether the new
// tokens of a request may be a tree (the caller's masks say which of them a row sees) or are
// a run of text, each seeing those before it.  The two are kernels of their own, so that the
// second has nothing of what only the first needs.
//
// out = sum_j softmax_j(scale q . k_j) v_j in one pass over the keys, with the running
// maximum m and sum l of the softmax beside the output.  Both products are transposed,
// S^T = K q^T and O^T = V^T P^T, so that a lane keeps one row of q throughout: row maxima
// and sums are sums over its registers, and with the cache's layout (include/mle_paged.h)
// the registers of S^T are those of the P operand, without a transpose of K, V or P.
//
// fp32 accuracy from 16-bit matrix instructions: q and P go in as sums of 16-bit parts, two
// f16 (22 bits) against f16 and 8-bit caches, three bf16 (24 bits) against bf16, whose
// range f16 does not have.  For f16 a row of q is first brought near 2^10 (row_scale) and P
// carries a factor 2^6, so the parts keep 22 bits down to 2^-12 of the largest.
//
// 8-bit caches: s_j = (q . k_j) ks_j; the V row's scale goes into the exponent, p_j vs_j =
// 2^(s_j + log2 vs_j - m), with m the maximum of those sums, so that the parts have their
// bits where the row's contributions are; l gets p_j vs_j * (1 / vs_j).
//
// A workgroup is four waves, two workgroups a CU (one at head size 256), so that one's softmax
// runs beside the other's products; the loop over segments makes what it can anew in each
// (fresh, fresh_args, forget), since values kept across it cost the inner loops their
// registers: with them kept the 128-wide kernels spilled.
//
// A value of V that is not finite must reach the rows that see it and no others, and 0 times
// it, or the parts of P times it, are NaN; so are the parts of q times an infinity in K, whose
// product may be minus infinity, a weight of 0.  Where a sum comes out non-finite, the keys are
// gone through again, with such values of V taken out of the product and added to the rows that
// see them, and with products that came out NaN made again one by one.  Places that no row
// sees, which may hold anything, always count as zero.  The second pass is code of its own,
// which the first keeps nothing for: together in one loop, the 128-wide kernels spilled and 4
// prompts of 512 took 39.7 us instead of 38.7.  With infinities in two of three pages of V the
// 2048 tokens over 10240 below take 5.8 ms, with one in K of every token 33.
//
// The maximum moves only when a logit passes it by 2^8 (P and l stay far from their limits),
// so that the rescaling of O is rare.  It stays finite, so that a logit past 2^128 makes NaN of
// its row, not a row of no weights.
//
// Work is laid out on the device, from the lengths there (the host knows only bounds, and a
// launch shaped by those would be mostly empty workgroups): units of 64 keys of one (sequence,
// KV head, row tile), cut into as many equal runs as there are workgroups, whatever the mix
// of short and long sequences, decoding and prompts.  A tile cut by a run's end is joined,
// in order, by the workgroup that finishes last.
//
// What bounds it (MI355X; 2 GiB are read at 6.1 TB/s, a large f16 product reaches 1.32
// PFLOP/s in a row of calls):
//   decoding: HBM.  32 sequences of up to 4096 tokens, 32 heads of 128, 182 us = 5.3 TB/s;
//     8 of up to 32768 of 8 bits, 8 KV heads, 64 us = 4.1 TB/s, of which about 10 are the
//     beginning and 5 the joins.
//   prompts: power, and the softmax beside the products.  2048 tokens over 10240, 32 heads
//     over 8, 555-575 us = 1.08-1.11 PFLOP/s of parts in a row of calls; the first 40 after a
//     rest 600-780, while the card settles its clock (a library product of 8192^3 likewise,
//     0.83 and 0.85-1.07 ms).  The matrix cores are busy in 56% of 1.06 million cycles (in 69%
//     of the library's), with 4.2 vector instructions to each of theirs; of the two waves of a
//     SIMD 1.65 are there on average, which wait for it 43% of their time, for memory and
//     barriers 19%.  Priorities of the waves, a second accumulator for the low parts, and loads
//     issued between the matrix instructions changed nothing.
//   short calls: a chain of latencies (lengths, run, page table, keys) of 6 us for few rows
//     and 12 for many: 129 tokens of 14 heads 8.7 us.
//   trees: as few or many rows, by the query heads of their nodes.  8 nodes over 129 tokens, 14
//     heads 11.4 us.  16 trees of 26 over up to 4096, 32 heads (383 MB) 90 us = 4.3 TB/s: 5 us
//     of beginning, units of 2.4 us beside another workgroup, runs that end between 64 and 94.
//     8 trees of 64 over up to 32768 of 8 bits, 32 heads over 8 198-200 us = 0.79 PFLOP/s of parts:
//     matrix cores busy in 35% of the cycles, 1.5 waves a SIMD, since of the two workgroups of a
//     CU the older one's waves go first and it is done at 165 us, the other by 206.  Priorities
//     that changed from unit to unit brought their ends together, longer runs for the older ones
//     likewise, and the call was no shorter by either.
#pragma once

#include "launch.hpp"
#include "paged.hpp"
#include "q8_0_device.hpp"

namespace mle {
namespace {

constexpr int kThreads = kAttentionThreads;
constexpr int kUnit = 64;         // keys of a unit of work, and of a stage in LDS
// kFewRows is what one matrix instruction holds.  At 16 rows over 32 sequences of 4096 (f16, 8
// KV heads of 128) that form takes 37 us against 42 with the tiles of many rows, at 7 over
// 32768 of 8 bits (2 heads of 64) 22 against 148, and nowhere longer.
constexpr int kTileRows = 128;    // above kFewRows: four waves of 32 rows share the keys in LDS
// Between: rows of trees, of which a request seldom has more, in tiles of kSomeRows, whose keys
// the waves split as those of few rows.
constexpr int kSomeRows = 2 * kFewRows;
constexpr float kLargest = 0x1.fffffep127f;
constexpr float kSlack = 8.0f;    // log2 of what a logit may pass the kept maximum by
constexpr int kDeviceScope = 16;  // cache policy of loads and stores

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// ---- element types ----

// 8-bit caches are computed in f16, which holds their whole numbers.
template <KvType T>
constexpr int kParts = T == KvType::kBF16 ? 3 : 2;
template <KvType T>
constexpr bool kBytes = T == KvType::kInt8;
// log2 of P's factor: f16 parts reach further down with 6.  bf16 parts need none for that; with
// -16, P is at most 2^-8, and sums over 256 keys of the largest bf16 values stay finite (over
// 65536 where the maximum does not lag).
template <KvType T>
constexpr float kHeadroom = T == KvType::kBF16 ? -16.0f : 6.0f;

// Two fp32 values as pairs of 16-bit parts that add up to them.
template <KvType T>
__device__ __forceinline__ void split2(float a, float b, uint32_t* part, int stride) {
  if constexpr (T == KvType::kBF16) {
    // Truncation leaves 8 bits a part: three hold all 24.
    const uint32_t ua = __builtin_bit_cast(uint32_t, a), ub = __builtin_bit_cast(uint32_t, b);
    part[0] = top_halves(ua, ub);
    const float ra = a - __builtin_bit_cast(float, ua & 0xffff0000u);
    const float rb = b - __builtin_bit_cast(float, ub & 0xffff0000u);
    const uint32_t va = __builtin_bit_cast(uint32_t, ra), vb = __builtin_bit_cast(uint32_t, rb);
    part[stride] = top_halves(va, vb);
    const float sa = ra - __builtin_bit_cast(float, va & 0xffff0000u);
    const float sb = rb - __builtin_bit_cast(float, vb & 0xffff0000u);
    part[2 * stride] =
        top_halves(__builtin_bit_cast(uint32_t, sa), __builtin_bit_cast(uint32_t, sb));
  } else {
    const f16x2 hi = __builtin_convertvector((f32x2{a, b}), f16x2);
    const f32x2 rest = {a - (float)hi.x, b - (float)hi.y};
    part[0] = __builtin_bit_cast(uint32_t, hi);
    part[stride] = __builtin_bit_cast(uint32_t, __builtin_convertvector(rest, f16x2));
  }
}

template <KvType T>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (T == KvType::kBF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <KvType T>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (T == KvType::kBF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Four 8-bit quants to f16 (exact): 0x6400 | u is 1024 + u.
__device__ __forceinline__ u32x2 quants_to_f16(uint32_t w) {
  const uint32_t u = w ^ 0x80808080u;  // q + 128
  const f16x2 lo = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u));
  const f16x2 hi = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u));
  const f16x2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
  return u32x2{__builtin_bit_cast(uint32_t, lo - off), __builtin_bit_cast(uint32_t, hi - off)};
}
__device__ __forceinline__ u32x4 quants_to_f16(u32x2 w) {
  const u32x2 a = quants_to_f16(w.x), b = quants_to_f16(w.y);
  return u32x4{a.x, a.y, b.x, b.y};
}

// Bit 15 of each 16-bit half whose value is an infinity or a NaN.
template <KvType T>
__device__ __forceinline__ uint32_t non_finite(uint32_t w) {
  constexpr uint32_t e = T == KvType::kBF16 ? 0x7f807f80u : 0x7c007c00u;
  constexpr uint32_t one = T == KvType::kBF16 ? 0x00800080u : 0x04000400u;
  return ((w & e) + one) & 0x80008000u;
}

template <KvType T>
__device__ __forceinline__ float value_of(uint32_t half) {
  if constexpr (T == KvType::kBF16) return __builtin_bit_cast(float, half << 16);
  else return (float)__builtin_bit_cast(_Float16, (uint16_t)half);
}

template <KvType T>
__device__ __forceinline__ bool is_non_finite(uint32_t half) {
  constexpr uint32_t e = T == KvType::kBF16 ? 0x7f80u : 0x7c00u;
  return (half & e) == e;
}

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// q . k of a key for which the matrix cores give NaN: they make that of an infinity in K,
// times the low parts of q, whatever the product is.  It is not finite, so that the finite
// terms do not count.
template <KvType T, int D>
__device__ __forceinline__ float product_of(const float* q, const uint16_t* k) {
  float sum = 0.0f;
#pragma unroll 1
  for (int d = 0; d < D; d += 8) {
    const u32x4 w = *reinterpret_cast<const u32x4*>(k + d * kKvTile);
    const f32x4 v[2] = {*reinterpret_cast<const f32x4*>(q + d),
                        *reinterpret_cast<const f32x4*>(q + d + 4)};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float term = v[i / 4][i % 4] * value_of<T>(w[i / 2] >> (i % 2 * 16) & 0xffffu);
      if (term - term != 0.0f) sum += term;
    }
  }
  return sum;
}

// Bits where one of a lane's values of q, as parts, is not finite.
template <KvType T, int N>
__device__ __forceinline__ uint32_t non_finite(const u32x4 (&q)[N]) {
  uint32_t bits = 0;
#pragma unroll
  for (int kk = 0; kk < N; ++kk)
#pragma unroll
    for (int i = 0; i < 4; ++i) bits |= non_finite<T>(q[kk][i]);
  return bits;
}

// The scale of a V row as its logarithm and inverse; a scale of 0 counts as a tiny one (the
// row's quants are 0).  NaN and infinity stay in the logarithm, which hidden keys
// do not use; the inverse, times their weight of 0, is always finite.
__device__ __forceinline__ float scale_log2(float v) {
  return __builtin_amdgcn_logf(v <= kTinyScale ? kTinyScale : v);
}
__device__ __forceinline__ float scale_inverse(float v) {
  return __builtin_amdgcn_rcpf(v > kTinyScale ? v : v <= kTinyScale ? kTinyScale : 1.0f);
}

// Factor that brings a row of q to some 2^9 or 2^10, the mantissa of scale log2(e) in it, so that
// logits in units of log2 are products times a power of two, c: they have no rounding of their
// own then, and the largest one, less itself, is 0 however large it is.  Over a bf16 cache it
// brings it to 2^-12 or 2^-11: the products of 256 elements with the largest values of the cache
// stay below 2^126, and no part loses bits to the type's range.
template <KvType T>
__device__ __forceinline__ void row_scale(uint32_t amax_bits, float scale, float* up, float* c) {
  constexpr int kTop = T == KvType::kBF16 ? 115 : 136;
  const int ex = (int)(amax_bits >> 23);
  const int es = __builtin_amdgcn_frexp_expf(scale);  // mantissa in [1/2, 1); 0 of a scale of 0
  int f = 0;  // non-finite rows: any
  if (amax_bits != 0 && ex != 255) {
    f = kTop - ex < 126 ? kTop - ex : 126;
    f = f < es + 126 ? f : es + 126;  // c is at least 2^-126
  }
  int e = es - f < 127 ? es - f : 127;
  e = e > -126 ? e : -126;
  *up = __builtin_ldexpf(__builtin_amdgcn_frexp_mantf(scale) * 1.44269504f, f);
  *c = __builtin_bit_cast(float, (uint32_t)(127 + e) << 23);
}

__device__ __forceinline__ uint32_t magnitude(f32x4 v) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v[i]) & 0x7fffffffu;
    m = b > m ? b : m;
  }
  return m;
}

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ uint64_t uniform(uint64_t x) {
  return (uint64_t)(uint32_t)uniform((int)(x >> 32)) << 32 | (uint32_t)uniform((int)x);
}
// A value, made anew: what is computed from it is computed there, instead of before a loop
// and kept in registers across it.
__device__ __forceinline__ int fresh(int x) {
  asm volatile("" : "+v"(x));
  return x;
}
__device__ __forceinline__ int fresh_tid() { return fresh((int)threadIdx.x); }
__device__ __forceinline__ int from_lane(int v, int lane) {
  return __builtin_amdgcn_ds_bpermute(lane << 2, v);
}
__device__ __forceinline__ int64_t from_lane(int64_t v, int lane) {
  return (int64_t)((uint64_t)(uint32_t)from_lane((int)(v >> 32), lane) << 32 |
                   (uint32_t)from_lane((int)v, lane));
}

// f of a value and that of the lane 32 (16) away, in both.
template <class F>
__device__ __forceinline__ uint32_t with_32(uint32_t v, F f) {
  const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return f((uint32_t)r[0], (uint32_t)r[1]);
}
template <class F>
__device__ __forceinline__ uint32_t with_16(uint32_t v, F f) {
  const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return f((uint32_t)r[0], (uint32_t)r[1]);
}
__device__ __forceinline__ uint32_t max_bits(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint32_t max_float(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(
      uint32_t, fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)));
}
__device__ __forceinline__ uint32_t sum_float(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t,
                            __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b));
}
template <class F>
__device__ __forceinline__ float with_32(float v, F f) {
  return __builtin_bit_cast(float, with_32(__builtin_bit_cast(uint32_t, v), f));
}
template <class F>
__device__ __forceinline__ float with_16(float v, F f) {
  return __builtin_bit_cast(float, with_16(__builtin_bit_cast(uint32_t, v), f));
}

// The kernel's first argument, read anew for the same reason.
__device__ __forceinline__ AttentionArgs fresh_args() {
  typedef const __attribute__((address_space(4))) AttentionArgs* Ptr;
  Ptr p = (Ptr)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const AttentionArgs*)p;
}
__device__ __forceinline__ int64_t lane_of(int64_t x, int lane) {
  return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), lane) << 32 |
                   (uint32_t)__builtin_amdgcn_readlane((int)x, lane));
}

// ---- the work ----

struct Run {
  int row0, n, pos0;  // first row, rows, position of the first row
};
struct Tree : Run {
  int masked;  // whether the rows are a tree, or a run after all
};
using Seq = std::conditional_t<kTrees, Tree, Run>;

__device__ __forceinline__ bool is_tree(const Run&) { return false; }
__device__ __forceinline__ bool is_tree(const Tree& s) { return s.masked != 0; }
__device__ __forceinline__ Run uniform(const Run& s) {
  return {uniform(s.row0), uniform(s.n), uniform(s.pos0)};
}
__device__ __forceinline__ Tree uniform(const Tree& s) {
  return {uniform(static_cast<const Run&>(s)), uniform(s.masked)};
}

__device__ __forceinline__ void read_kind(const AttentionArgs&, int, Run&) {}
__device__ __forceinline__ void read_kind(const AttentionArgs& a, int b, Tree& s) {
  s.masked = a.trees == nullptr || a.trees[b] != 0;
}
__device__ __forceinline__ Seq seq_of(const AttentionArgs& a, int b) {
  // Offsets and lengths come from the caller's device memory: held to their range.
  int c0 = a.cu[b], c1 = a.cu[b + 1], len = a.kv_lens[b];
  c0 = c0 < 0 ? 0 : c0 < a.tokens ? c0 : a.tokens;
  c1 = c1 < c0 ? c0 : c1 < a.tokens ? c1 : a.tokens;
  Seq s{};
  s.row0 = c0;
  s.n = c1 - c0;
  s.pos0 = (len < 0 ? 0 : len) - s.n;
  read_kind(a, b, s);
  return s;
}

// Up to this many rows a request's tiles are of kSomeRows.  They begin and end sooner than those
// of kTileRows, but two of them read the keys twice: of f16 caches, whose steps have the least to
// compute, that costs more once the requests together read some 512 MB (as if all were as long as
// this one).  64 rows of 8 requests, 8 KV heads of 128: up to 1024 keys 21 us against 29, 4096 30
// against 41; of 16 requests up to 8192 72 against 61.  65 rows and more: of 8 requests of 8192
// 103 against 66.  At head size 256, 16 x 12 rows of 16 heads over 8 (24 a tile) over 8192 of f16,
// bf16 and 8 bits 101, 106 and 62 us against 129, 190 and 135 with the tiles of many rows, whose one
// workgroup a CU hides less; so there f16 ones take two as well, 16 x 26 of them 129 against 135.
template <KvType T, int D>
__device__ __forceinline__ int most_some_rows(const AttentionArgs& a, const Seq& s) {
  if (!kTrees) return 0;
  if (T != KvType::kF16 || D > 128) return 2 * kSomeRows;
  const int64_t keys = (int64_t)s.pos0 + s.n;
  return keys * a.sequences * a.cache.kv_heads < (int64_t(1) << 29) / (4 * D) ? 2 * kSomeRows
                                                                             : kSomeRows;
}

__device__ __forceinline__ int clamp_key(int64_t x, int most) {
  return (int)(x < 0 ? 0 : x < most ? x : most);
}

// Keys of the rows [r0, r1) of a sequence: any row sees [lo, hi), every row [lo_all, hi_all).
// Of a tree's rows any may see every new token, and none has to; the cached ones are seen
// through the window from positions that lie among those of the new rows.
struct Span {
  int lo, hi, lo_all, hi_all;
};

__device__ __forceinline__ Span span_of(const AttentionArgs& a, const Seq& s, int r0, int r1) {
  if (is_tree(s)) {
    Span x;
    x.hi = clamp_key((int64_t)s.pos0 + s.n, a.most);
    x.hi_all = clamp_key(s.pos0, a.most);
    x.lo = a.window > 0 ? clamp_key((int64_t)s.pos0 - a.window + 1, x.hi) : 0;
    x.lo_all = a.window > 0 ? clamp_key((int64_t)s.pos0 + s.n - a.window, a.most) : 0;
    return x;
  }
  const int64_t first = (int64_t)s.pos0 + (int)a.by_group.of(r0);
  const int64_t last = (int64_t)s.pos0 + (int)a.by_group.of(r1 - 1);
  Span x;
  x.hi = clamp_key(last + 1, a.most);
  x.hi_all = clamp_key(first + 1, a.most);
  x.lo = a.window > 0 ? clamp_key(first - a.window + 1, x.hi) : 0;
  x.lo_all = a.window > 0 ? clamp_key(last - a.window + 1, a.most) : 0;
  return x;
}

// What one row sees: a run of keys, and of a tree's new tokens those of its mask.
struct Sight {
  int lo;          // the run
  uint32_t width;
  int pos0, hi;    // a tree's new tokens are the keys [pos0, hi)
  const uint32_t* mask;  // null: no tree
  int words;

  // Of the 32 keys from `from` on, those that the row sees, a bit each.
  __device__ __forceinline__ uint32_t of(int from) const {
    uint32_t bits = below(lo + (int)width - from) & ~below(lo - from);
    if (kTrees && mask != nullptr) {
      const int j = from - pos0;  // the first of them, as a new token
      if (j > -32 && from < hi) {
        const int w = j >> 5;
        const uint32_t a = w >= 0 && w < words ? mask[w] : 0;
        const uint32_t b = w + 1 < words ? mask[w + 1] : 0;
        bits |= __builtin_amdgcn_alignbit(b, a, (uint32_t)j & 31) & below(hi - from);
      }
    }
    return bits;
  }
  // The lowest n bits.
  static __device__ __forceinline__ uint32_t below(int n) {
    return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1;
  }
  __device__ __forceinline__ bool sees(int key) const {
    if (kTrees) return of(key) & 1;
    return (uint32_t)(key - lo) < width;
  }
};

__device__ __forceinline__ Sight sight_of(const AttentionArgs& a, const Seq& s, int row) {
  Sight x{};
  if (is_tree(s)) {
    const int in = s.row0 + (int)a.by_group.of(row);
    x.hi = clamp_key((int64_t)s.pos0 + s.n, a.most);
    x.pos0 = s.pos0;
    if (a.window > 0) {
      int64_t pos = a.row_positions[in];
      pos = pos > s.pos0 ? pos : s.pos0;
      pos = pos < (int64_t)s.pos0 + s.n ? pos : (int64_t)s.pos0 + s.n - 1;
      x.lo = clamp_key(pos - a.window + 1, x.hi);
    }
    const int cached = clamp_key(s.pos0, a.most);
    x.width = cached > x.lo ? (uint32_t)(cached - x.lo) : 0;
    x.words = 2 * a.mask_words;
    x.mask = a.mask + (int64_t)in * x.words;
  } else {
    const Span mine = span_of(a, s, row, row + 1);
    x.lo = mine.lo;
    x.width = mine.hi > mine.lo ? (uint32_t)(mine.hi - mine.lo) : 0;
  }
  return x;
}

// What the row tiles of a (sequence, KV head) cost: tile t counts min(first + t slope, cap),
// a linear account of its units (causality adds keys from tile to tile, a window ends that)
// and of its beginning and end.  Only the balance depends on how close it is.
struct Cost {
  int tiles;
  int first, slope, cap;
  int fixed;  // of a tile's cost, what is not its units
  int least;  // the least piece of a tile worth a workgroup of its own, its fixed cost in it

  // The least one at a tile's end.  A tile's fixed cost is in the account where it begins, so a
  // run that takes up only its end, and goes on with the next, is no longer than others; one
  // prolonged to the tile's end is, and the next is shorter (2 x 40 rows of 32 heads over 600 keys
  // 27 us so and 22 with this, 64 of 28 over 20000 73 and 64; but 32 x 8 of 14 over
  // up to 8192 29 and 31).
  __device__ __forceinline__ int last() const { return kTrees ? least - fixed : least; }

  __device__ __forceinline__ int of(int t) const {
    const int64_t v = (int64_t)first + (int64_t)t * slope;
    return (int)(v < cap ? v : cap);
  }
  // Of the tiles before t.
  __device__ __forceinline__ uint64_t before(int t) const {
    int ramp = t;  // tiles below the cap
    if (first >= cap) ramp = 0;
    else if (slope > 0 && (cap - first) / slope + 1 < t) ramp = (cap - first) / slope + 1;
    return (uint64_t)ramp * first + (uint64_t)slope * ((uint64_t)ramp * (ramp - 1) / 2) +
           (uint64_t)(t - ramp) * cap;
  }
};

// Cost of a unit of many and of few rows, and of a tile besides its units: beside another
// workgroup, 64 keys of 128 rows take 3.5 us (5.6 with three parts) and of few rows 1.2
// (0.9 of 8 bits), 3 where all of them wait for memory; a tile's beginning and end 8 us.
template <KvType T>
struct Weights {
  static constexpr int kMany = kParts<T> * 16;
  static constexpr int kFew = kBytes<T> ? 8 : 11;
  static constexpr int kSome = kFew + 2;
  static constexpr int kTileMany = 80, kTileFew = 40;
  // The least piece of a tile worth a workgroup of its own.
  static constexpr int kLeastMany = kTileMany + kMany, kLeastFew = kTileFew + 20;
};

template <KvType T, int D>
__device__ __forceinline__ Cost cost_of(const AttentionArgs& a, const Seq& s) {
  constexpr int kMax = 1 << 29;
  const int rows = s.n * a.group;
  const bool few = rows <= kFewRows, some = !few && rows <= most_some_rows<T, D>(a, s);
  const int tile_rows = some ? kSomeRows : kTileRows;
  int unit = few ? Weights<T>::kFew : some ? Weights<T>::kSome : Weights<T>::kMany;
  // Waves without rows take no time.
  if (kTrees && !few && !some && rows < kTileRows)
    unit = Weights<T>::kSome + (unit - Weights<T>::kSome) * ((rows + 31) / 32 - 1) / 3;
  const int fixed = few || some ? Weights<T>::kTileFew : Weights<T>::kTileMany;
  auto units = [&](int64_t keys) {  // at least a partial one
    const int64_t v = (keys > 0 ? (keys * unit) / kUnit : 0) + unit / 2 + fixed;
    return (int)(v < kMax ? v : kMax);
  };
  Cost c;
  c.tiles = few ? rows > 0 : (rows + tile_rows - 1) / tile_rows;
  const int tokens = c.tiles > 1 ? (int)a.by_group.of(tile_rows + a.group - 1) : s.n;
  const int reach = is_tree(s) ? s.n : tokens;
  c.cap = a.window > 0 ? units((int64_t)a.window + reach) : kMax;
  c.first = units((int64_t)s.pos0 + reach);
  // From tile to tile tile_rows / group keys more.
  c.slope = is_tree(s) ? 0
            : some     ? (int)a.by_group.of(Weights<T>::kSome / 2)
                       : (int)a.by_group.of(2 * Weights<T>::kMany);
  c.fixed = fixed;
  c.least = few || some ? Weights<T>::kLeastFew : Weights<T>::kLeastMany;
  return c;
}

// floor(x / d).
__device__ __forceinline__ uint64_t quotient(uint64_t x, uint64_t d) {
  double r = __builtin_amdgcn_rcp((double)d);
  r = __builtin_fma(r, __builtin_fma(-(double)d, r, 1.0), r);
  uint64_t q = (uint64_t)((double)x * r);
  while (q * d > x) --q;
  while ((q + 1) * d <= x) ++q;
  return q;
}

// What one workgroup does in one go: some units of one row tile.
struct Segment {
  int b, g;
  Seq seq;
  int r0, rows;       // the tile's first row, and its rows
  Span span;
  int k0, k1;         // keys of the segment, multiples of kUnit
  int parts;          // workgroups that share the tile
  int part, first;    // which of them this is, and the first one's index
};

// The same in every lane, and told so: the fields stay in scalar registers.
__device__ __forceinline__ Segment uniform(const Segment& s) {
  return {uniform(s.b), uniform(s.g), uniform(s.seq),
          uniform(s.r0), uniform(s.rows),
          {uniform(s.span.lo), uniform(s.span.hi), uniform(s.span.lo_all),
           uniform(s.span.hi_all)},
          uniform(s.k0), uniform(s.k1), uniform(s.parts), uniform(s.part), uniform(s.first)};
}

struct Shared {
  float* partials;
  uint32_t* counters;
  int slot_floats;
  uint32_t bytes;  // of the partials: no access of a part goes past them
};

// What is written to LDS before is read from there, not kept in registers.
__device__ __forceinline__ void forget() { asm volatile("" ::: "memory"); }

// The sequences as a workgroup keeps them: thread i those from i * chunk on.
struct Schedule {
  uint64_t sum[kThreads];  // of the costs up to and with the thread's
  Seq seq[kThreads];       // where chunk is 1
  uint64_t wave_sum[4];
  int wave_tiles[4];
};

// A workgroup's way through its run of the work.  The whole work, `total`, is cut at
// multiples of `run`; a cut that leaves less than cost.least of a tile before it, or cost.last()
// behind it, moves to the tile's begin or end.
template <KvType T, int D>
struct Cursor {
  int b, g, t;
  Seq seq;
  Cost cost;
  uint64_t i0, i1;         // the current tile's place in the work
  uint64_t begin;          // where this workgroup takes it up
  uint64_t end, total, run;
  int w;
  bool done;

  // The sequence `b` or the first one after it that has rows; skips *base over the others.
  __device__ __forceinline__ void seek(const AttentionArgs& a, const Schedule& sch, int chunk) {
    for (;; ++b) {
      seq = chunk == 1 ? sch.seq[b] : seq_of(a, b);
      seq = uniform(seq);
      if (seq.n > 0) break;
    }
    cost = cost_of<T, D>(a, seq);
  }

  __device__ __forceinline__ void advance(const AttentionArgs& a, const Schedule& sch,
                                          int chunk) {
    if (++t == cost.tiles) {
      t = 0;
      if (++g == a.cache.kv_heads) {
        g = 0;
        ++b;
        seek(a, sch, chunk);
      }
    }
    i0 = i1;
    begin = i0;
    i1 = i0 + cost.of(t);
  }

  // The tile with the work's place `at`, and where in it the cut there lies.  `before`
  // threads' sequences come wholly before it.
  __device__ __forceinline__ void locate(const AttentionArgs& a, const Schedule& sch, int chunk,
                                         int before, uint64_t at) {
    b = before * chunk;
    i0 = before > 0 ? uniform(sch.sum[before - 1]) : 0;
    uint64_t of_head;
    for (;;) {
      seek(a, sch, chunk);
      of_head = cost.before(cost.tiles);
      if (at < i0 + of_head * a.cache.kv_heads) break;
      i0 += of_head * a.cache.kv_heads;
      ++b;
    }
    g = (int)quotient(at - i0, of_head);
    i0 += g * of_head;
    t = 0;
    for (int past = cost.tiles; past - t > 1;) {
      const int mid = t + (past - t) / 2;
      if (i0 + cost.before(mid) <= at) t = mid; else past = mid;
    }
    i0 += cost.before(t);
    i1 = i0 + cost.of(t);
    done = false;
    begin = i0;
    if (at - i0 >= (uint64_t)cost.least) {
      begin = at;
      if (i1 - at < (uint64_t)cost.last()) {
        if (i1 < total) advance(a, sch, chunk);
        else done = true;
      }
    }
  }

  // Units of the tile that lie before place x of it; its fixed cost comes first.
  __device__ __forceinline__ int units_at(uint64_t x, uint64_t of, int units) const {
    if (x >= of) return units;
    const float u = ((float)(uint32_t)x - (float)cost.fixed) *
                    ((float)units * __builtin_amdgcn_rcpf((float)((uint32_t)of - cost.fixed)));
    return u <= 0.0f ? 0 : u < (float)units ? (int)u : units;
  }

  __device__ __forceinline__ Cursor uniform_copy() const {
    Cursor c;
    c.b = uniform(b);
    c.g = uniform(g);
    c.t = uniform(t);
    c.seq = uniform(seq);
    c.cost = {uniform(cost.tiles), uniform(cost.first), uniform(cost.slope), uniform(cost.cap),
              uniform(cost.fixed), uniform(cost.least)};
    c.i0 = uniform(i0);
    c.i1 = uniform(i1);
    c.begin = uniform(begin);
    c.end = uniform(end);
    c.total = uniform(total);
    c.w = uniform(w);
    c.run = uniform(run);
    c.done = uniform((int)done) != 0;
    return c;
  }

  // The next piece of this workgroup's run; false at its end.
  __device__ __forceinline__ bool next(const AttentionArgs& a, const Schedule& sch, int chunk,
                                       Segment* out) {
    if (done || end <= i0 || (end < i1 && end - i0 < (uint64_t)cost.least)) return false;
    const uint64_t stop = (int64_t)(i1 - end) < cost.last() ? i1 : end;
    Segment s;
    s.b = b;
    s.g = g;
    s.seq = seq;
    const int rows = seq.n * a.group;
    const int tr = rows <= kFewRows                        ? kFewRows
                   : rows <= most_some_rows<T, D>(a, seq) ? kSomeRows
                                                          : kTileRows;
    s.r0 = t * tr;
    s.rows = rows - s.r0 < tr ? rows - s.r0 : tr;
    s.span = span_of(a, seq, s.r0, s.r0 + s.rows);
    const int u0 = s.span.lo / kUnit, units = (s.span.hi + kUnit - 1) / kUnit - u0;
    s.k0 = (u0 + (begin == i0 ? 0 : units_at(begin - i0, i1 - i0, units))) * kUnit;
    s.k1 = (u0 + units_at(stop - i0, i1 - i0, units)) * kUnit;
    s.parts = 1;
    s.part = s.first = 0;
    if (begin != i0 || stop != i1) {
      // The cuts inside the tile.
      const uint64_t lo = i0 + cost.least, hi = i1 - cost.last();
      const int c0 = (int)quotient(lo + run - 1, run), c1 = (int)quotient(hi, run);
      s.first = c0 - 1;
      s.part = w - s.first;
      s.parts = c1 - c0 + 2;
    }
    *out = uniform(s);
    if (stop != i1 || i1 >= end) done = true;
    else advance(a, sch, chunk);
    return true;
  }
};

// Device memory of a tile's part: workgroup `first + part` has two slots, for a tile that
// came from the workgroup before and for one that goes on in the next.
__device__ __forceinline__ uint32_t slot_at(const Shared& sh, const Segment& s, int part) {
  return (uint32_t)((s.first + part) * 2 + (part == 0)) * (uint32_t)sh.slot_floats * 4u;
}

// The same in every lane, and told so: an access goes lane by lane otherwise.
__device__ __forceinline__ uint32_t same_slot_at(const Shared& sh, const Segment& s, int part) {
  return (uint32_t)uniform((int)slot_at(sh, s, part));
}

// Whether this workgroup is the last of `all` at a counter.
__device__ __forceinline__ bool last_to_arrive(uint32_t* c, int all, int* shared) {
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_s_waitcnt(0);  // this wave's part has reached the coherence point
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __syncthreads();
  if (threadIdx.x == 0) {
    const int n = (int)__hip_atomic_fetch_add(c, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *shared = n;
    if (n == all - 1)  // nobody else comes: zero again for the next launch
      __hip_atomic_store(c, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  return *shared == all - 1;
}

// Parts of a tile that are joined before all of them are.  One workgroup alone reads a part of
// 128 rows of 256 in about a microsecond: 20 tokens of 8 heads over 8000 keys took 135 us, and 59
// in groups; 64 of 14 heads of 64 over 20000 54 and 37.  Up to 12 parts a second wait for the
// counter costs what it saves.
__device__ __forceinline__ int parts_of_group(int parts) {
  return !kTrees || parts <= 12 ? parts : parts <= 64 ? 8 : parts <= 144 ? 12 : 24;
}

// Joins a tile's parts, in order, whichever workgroup comes last: join(first, step, count) adds
// up the parts first, first + step, .. into registers, keep(part) makes them that part.  Says
// whether this workgroup has them all.  A group's counter lies beside that of a tile that would
// begin with the group's first workgroup; a last part alone, whose workgroup may begin one, needs
// none.
template <class Join, class Keep>
__device__ __forceinline__ bool join_parts(const Shared& sh, const Segment& s, int* shared,
                                           Join join, Keep keep) {
  uint32_t* tile = sh.counters + s.first * kCounterStride;
  const int size = parts_of_group(s.parts);
  if (!kTrees || size >= s.parts) {
    if (!last_to_arrive(tile, s.parts, shared)) return false;
    join(0, 1, s.parts);
    return true;
  }
  const int first = s.part / size * size;
  const int count = s.parts - first < size ? s.parts - first : size;
  if (count > 1) {
    if (!last_to_arrive(tile + first * kCounterStride + 1, count, shared)) return false;
    join(first, 1, count);
    // Every wave has read the part `first` before it is written over: all of them read the maxima
    // and sums of few rows, and one writes them.
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0);
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __syncthreads();
    keep(first);
  }
  const int groups = (s.parts + size - 1) / size;
  if (!last_to_arrive(tile, groups, shared)) return false;
  join(0, size, groups);
  return true;
}

// Parts lie at `slot` + `at` bytes: what lanes share, and what they do not.
__device__ __forceinline__ f32x4 load_part(__amdgpu_buffer_rsrc_t rs, uint32_t at, uint32_t slot) {
  return __builtin_bit_cast(f32x4,
                            __builtin_amdgcn_raw_buffer_load_b128(rs, at, slot, kDeviceScope));
}
__device__ __forceinline__ f32x2 load_part2(__amdgpu_buffer_rsrc_t rs, uint32_t at,
                                            uint32_t slot) {
  return __builtin_bit_cast(f32x2,
                            __builtin_amdgcn_raw_buffer_load_b64(rs, at, slot, kDeviceScope));
}
__device__ __forceinline__ void store_part(f32x4 v, __amdgpu_buffer_rsrc_t rs, uint32_t at,
                                           uint32_t slot) {
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), rs, at, slot, kDeviceScope);
}
__device__ __forceinline__ void store_part2(f32x2 v, __amdgpu_buffer_rsrc_t rs, uint32_t at,
                                            uint32_t slot) {
  __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, v), rs, at, slot, kDeviceScope);
}

// Weight of a partial result with maximum m beside the maximum M of all.
__device__ __forceinline__ float weight(float m, float M) {
  return M == -INFINITY ? 0.0f : exp2_of(m - M);
}

// The tiles of 64 lanes' places: tile index in the cache (of 16 tokens), and whether the
// lane's tile is there at all.
struct Tiles {
  int64_t index;
  bool bad;
};

// Finding them waits for the table; the load goes out with page_of, long before.
__device__ __forceinline__ int page_of(const AttentionArgs& a, const Segment& s, int key) {
  int page = -1;
  if (key < s.span.hi) page = a.table[(int64_t)s.b * a.max_pages + a.by_page.of(key)];
  return page;
}

__device__ __forceinline__ Tiles tile_of(const AttentionArgs& a, const Segment& s, int key,
                                         int page) {
  const int P = a.cache.page_size;
  Tiles t;
  t.bad = (uint32_t)page >= (uint32_t)a.cache.num_pages;
  const int64_t first = ((int64_t)page * a.cache.kv_heads + s.g) * P;
  t.index = t.bad ? 0 : (first + (key - (int)a.by_page.of(key) * P)) / kKvTile;
  return t;
}

__device__ __forceinline__ Tiles find_tile(const AttentionArgs& a, const Segment& s, int key) {
  return tile_of(a, s, key, page_of(a, s, key));
}

// ---- few rows: the workgroup's waves split the keys ----
//
// Bound by HBM, so by bytes in flight: a wave has a step's K and V (16 KB of 32 keys, or of 64
// of 8 bits, at head size 128) under way in registers, straight from the cache, whose layout
// makes each load one run of memory.  16 columns of q are 16 rows or copies of the last one:
// the matrix cores are idle for most of the time anyway.  The next tile's first loads go out
// before the present one is joined and written (32 x <= 4096: 200 -> 182 us).
//
// R times 16 rows: a step's keys are multiplied by R operands of q, which then lie in LDS, read
// anew for each step: in registers beside the loads, the sums of 32 rows of 128 spilled.

template <KvType T, int D, int R>
struct FewRows {
  // Cache tiles of a wave's step.
  static constexpr int kTiles = kBytes<T> && R == 1 ? 4 : 2;
  static constexpr int kStep = kTiles * kKvTile;
  static constexpr int KK = D / 32, DB = D / 16;
  static constexpr int NQ = (4 * D + kThreads - 1) / kThreads;  // quads of the result a thread
  using Raw = std::conditional_t<kBytes<T>, u32x2, u32x4>;

  struct Loads {
    Raw k[kTiles][KK];
    Raw v[kTiles / 2][DB];
    f32x4 ks[kBytes<T> ? kTiles : 1], vs[kBytes<T> ? kTiles : 1];
  };
  // What goes out for a segment before the one in front of it has been joined and written.
  struct Ahead {
    Loads x;
    Tiles held;     // the tiles of this wave's first steps, a lane each
    bool started;
  };
  // No loads ahead.  The registers are said to be set here, to anything: left unset, they
  // would be reserved throughout the kernel.
  static __device__ __forceinline__ void none_ahead(Ahead& n) {
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) asm volatile("" : "=v"(n.x.k[t][kk]));
      if constexpr (kBytes<T>) asm volatile("" : "=v"(n.x.ks[t]), "=v"(n.x.vs[t]));
    }
#pragma unroll
    for (int u = 0; u < kTiles / 2; ++u)
#pragma unroll
      for (int db = 0; db < DB; ++db) asm volatile("" : "=v"(n.x.v[u][db]));
    n.held = {0, true};
    n.started = false;
  }
  static constexpr int kAhead = 64 / kTiles;  // steps whose tiles the lanes hold

  static __device__ __forceinline__ Tiles look_up(const AttentionArgs& a, const Segment& s,
                                                  int lane, int from) {
    return find_tile(a, s, key_of(lane, from));
  }
  // First key of the lane's tile among the tiles of a wave's steps.
  static __device__ __forceinline__ int key_of(int lane, int from) {
    lane = fresh(lane);
    return from + (lane / kTiles) * 4 * kStep + (lane % kTiles) * kKvTile;
  }
  static __device__ __forceinline__ void take(const Tiles& held, int step, int64_t* tile) {
#pragma unroll
    for (int t = 0; t < kTiles; ++t) tile[t] = lane_of(held.index, step * kTiles + t);
  }
  static __device__ __forceinline__ int last_key(const Segment& s) {
    return s.k1 < s.span.hi ? s.k1 : s.span.hi;
  }
  // The first step's loads.
  static __device__ __forceinline__ void start(const AttentionArgs& a, const Segment& s, int lane,
                                               int wave, Ahead& n) {
    if (s.k0 + wave * kStep >= last_key(s)) return;
    int64_t tile[kTiles];
    take(n.held, 0, tile);
    load_k(a, lane, tile, n.x);
    load_v(a, lane, tile, n.x);
  }

  // Whether the lane's row of q is finite; lanes l, l + 16 .. have it, and all of them come here.
  static __device__ __forceinline__ bool finite_q(const u32x4 (&qp)[kParts<T>][KK]) {
    return with_32(with_16(non_finite<T>(qp[0]), max_bits), max_bits) == 0;
  }
  static __device__ __forceinline__ bool any_nan(const float (&sc)[kTiles][4]) {
    bool nan = false;
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) nan |= sc[t][i] != sc[t][i];
    return nan;
  }

  static __device__ __forceinline__ u32x4 operand(Raw r) {
    if constexpr (kBytes<T>) return quants_to_f16(r);
    else return r;
  }

  static __device__ __forceinline__ void load_k(const AttentionArgs& a, int lane,
                                                const int64_t* tile, Loads& x) {
    constexpr int E = kBytes<T> ? 1 : 2;
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      const uint8_t* p = static_cast<const uint8_t*>(a.cache.k) + tile[t] * (kKvTile * D * E);
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
        x.k[t][kk] = *reinterpret_cast<const Raw*>(p + (uint32_t)(kk * 512 * E + lane * 8 * E));
      if constexpr (kBytes<T>)
        x.ks[t] = *reinterpret_cast<const f32x4*>(a.cache.k_scale + tile[t] * kKvTile +
                                                  (lane >> 4) * 4);
    }
  }

  // Lane group l / 16 is (tile of the pair, half of the places of four tokens).
  static __device__ __forceinline__ void load_v(const AttentionArgs& a, int lane,
                                                const int64_t* tile, Loads& x) {
    constexpr int E = kBytes<T> ? 1 : 2;
#pragma unroll
    for (int u = 0; u < kTiles / 2; ++u) {
      const int64_t mine = lane < 32 ? tile[2 * u] : tile[2 * u + 1];
      const uint8_t* p = static_cast<const uint8_t*>(a.cache.v) + mine * (kKvTile * D * E) +
                         (uint32_t)(((lane >> 4 & 1) * D + (lane & 15)) * 8 * E);
#pragma unroll
      for (int db = 0; db < DB; ++db)
        x.v[u][db] = *reinterpret_cast<const Raw*>(p + db * 128 * E);
      if constexpr (kBytes<T>)
#pragma unroll
        for (int t = 2 * u; t < 2 * u + 2; ++t)
          x.vs[t] = *reinterpret_cast<const f32x4*>(a.cache.v_scale + tile[t] * kKvTile +
                                                    (lane >> 4) * 4);
    }
  }

  static __device__ __forceinline__ float* out_row(const AttentionArgs& a, const Segment& s,
                                                   int r) {
    if constexpr (R > 1) r += s.r0;
    const int tok = (int)a.by_group.of(r);
    return a.out + (int64_t)(s.seq.row0 + tok) * a.out_stride +
           (int64_t)(s.g * a.group + r - tok * a.group) * D;
  }
  using Part = FewPart<D>;
  static constexpr uint32_t kMl = Part::kMl;  // of a part: where its (m, l) are

  // Joins and writes a tile of up to 8 rows that came in many parts: groups of threads as many
  // as there is room for, (rows to a power of two) D / 4 threads each, take some parts each.
  static __device__ __forceinline__ void join_many(const AttentionArgs& a, const Segment& s,
                                                   const Shared& sh, int tid, uint8_t* smem) {
    constexpr int NJ = Part::kQuadsOfThread, kAtOnce = 16 / NJ;
    const __amdgpu_buffer_rsrc_t rs = buffer_rsrc(sh.partials, sh.bytes);
    const int bits = s.rows > 4 ? 3 : s.rows > 2 ? 2 : s.rows > 1 ? 1 : 0;
    const int quads = Part::quads(bits);
    const int groups = quads < kThreads ? kThreads / quads : 1;
    const int group =
        groups > 1 ? (int)(((float)tid + 0.5f) * __builtin_amdgcn_rcpf((float)quads)) : 0;
    const int at = tid - group * quads, r = at & ((1 << bits) - 1);
    uint32_t quad_at[NJ];
#pragma unroll
    for (int i = 0; i < NJ; ++i) quad_at[i] = Part::quad_at(at, i, bits);
    const uint32_t ml_at = Part::ml_at(at, bits);
    float M = -INFINITY, L = 0.0f;
    f32x4 out[NJ] = {};
    for (int p0 = group; p0 < s.parts && group < groups; p0 += kAtOnce * groups) {
      f32x2 ml[kAtOnce];
      f32x4 v[kAtOnce][NJ];
#pragma unroll
      for (int p = 0; p < kAtOnce; ++p) {
        // Past the last part: that one again, not used.
        const int part = p0 + p * groups < s.parts ? p0 + p * groups : s.parts - 1;
        const uint32_t from = slot_at(sh, s, part);
        ml[p] = load_part2(rs, from + ml_at, 0);
#pragma unroll
        for (int i = 0; i < NJ; ++i) v[p][i] = load_part(rs, from + quad_at[i], 0);
      }
      float top = M;
#pragma unroll
      for (int p = 0; p < kAtOnce; ++p) top = fmaxf(top, ml[p].x);
      const float keep = weight(M, top);
      M = top;
      L *= keep;
#pragma unroll
      for (int i = 0; i < NJ; ++i) out[i] *= keep;
#pragma unroll
      for (int p = 0; p < kAtOnce; ++p) {
        if (p0 + p * groups < s.parts) {
          const float f = weight(ml[p].x, M);
          L = __builtin_fmaf(ml[p].y, f, L);
#pragma unroll
          for (int i = 0; i < NJ; ++i) out[i] += v[p][i] * f;
        }
      }
    }
    if (groups > 1) {  // NJ's first quad is all there is
      f32x4* g_acc = reinterpret_cast<f32x4*>(smem + 1024);
      f32x2* g_ml = reinterpret_cast<f32x2*>(smem + 1024 + kThreads * 16);
      __syncthreads();  // the arrival count has been read
      g_acc[tid] = out[0];
      g_ml[tid] = f32x2{M, L};
      __syncthreads();
      M = -INFINITY;
      L = 0.0f;
      out[0] = f32x4{};
      if (group == 0) {
        for (int g = 0; g < groups; ++g) M = fmaxf(M, g_ml[g * quads + tid].x);
        for (int g = 0; g < groups; ++g) {
          const f32x2 ml = g_ml[g * quads + tid];
          const float f = weight(ml.x, M);
          L = __builtin_fmaf(ml.y, f, L);
          out[0] += g_acc[g * quads + tid] * f;
        }
      }
    }
    if (group == 0 && r < s.rows) {
      float* o = out_row(a, s, r);
      const float inv = L != 0.0f ? 1.0f / L : 0.0f;
#pragma unroll
      for (int i = 0; i < NJ; ++i)
        if (Part::has(at, i, bits))
          *reinterpret_cast<f32x4*>(o + ((at + i * kThreads) >> bits) * 4) =
              L != 0.0f ? out[i] * inv : f32x4{};
    }
  }

  // One segment; `n` holds its first loads if n.started.  find_next() puts the next one into
  // `then`; if that is of few rows too, it comes next (true) and `n` gets its first loads.
  template <class F>
  static __device__ __forceinline__ bool run(const Segment& s, const Shared& sh, uint8_t* smem,
                                             const Segment* then, F find_next, Ahead& n) {
    const AttentionArgs a = fresh_args();
    forget();
    const int tid = fresh_tid(), lane = tid & 63, wave = uniform(tid >> 6);
    const int quad = lane >> 4;
    // The rows of q as operands, of R > 1 in LDS, with their factors and whether they are finite.
    constexpr int kC = R * kParts<T> * KK * 1024;
    float* s_c = reinterpret_cast<float*>(smem + kC);
    uint32_t* s_odd = reinterpret_cast<uint32_t*>(smem + kC + R * 64);
    // The lane's rows among the request's, or copies of the last one.
    auto row_of = [&](int r) {
      const int in = r * 16 + (lane & 15);
      return (R > 1 ? s.r0 : 0) + (in < s.rows ? in : s.rows - 1);
    };
    Sight mine[R];
#pragma unroll
    for (int r = 0; r < R; ++r) mine[r] = sight_of(a, s.seq, row_of(r));

    // Steps of this wave: s.k0 + (wave + 4 i) kStep.
    const int hi = last_key(s);
    Loads& x = n.x;
    Tiles& held = n.held;
    f32x4 qv[KK][2];
    auto load_q = [&](int row) {
      const int token = (int)a.by_group.of(row);
      const float* q = a.q + (int64_t)(s.seq.row0 + token) * a.q_stride +
                       (int64_t)(s.g * a.group + row - token * a.group) * D + quad * 8;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          qv[kk][h] = *reinterpret_cast<const f32x4*>(q + kk * 32 + h * 4);
    };
    // Ahead of the first keys, which wait for the table.
    if (R == 1 || wave < R) load_q(row_of(R == 1 ? 0 : wave));
    int base = s.k0 + wave * kStep;
    if (!n.started) {
      held = look_up(a, s, lane, base);
      start(a, s, lane, wave, n);
    }
    uint64_t bad = __ballot(held.bad);
    int at = 0;  // step among the held ones
    int64_t tile[kTiles];
    take(held, 0, tile);
    int then_page = 0;
    const bool go_on = find_next();
    if (go_on) {
      const Segment t = uniform(*then);
      then_page = page_of(a, t, key_of(lane, t.k0 + wave * kStep));
    }

    // q as the right operand: element 8 (l / 16) + e of each run of 32.
    u32x4 qp[kParts<T>][KK];
    float c[R];  // logits in units of log2 are S * c
    auto convert = [&](float* c) {
      uint32_t amax = 0;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
#pragma unroll
        for (int h = 0; h < 2; ++h) amax = max_bits(amax, magnitude(qv[kk][h]));
      amax = with_32(with_16(amax, max_bits), max_bits);
      float up;
      row_scale<T>(amax, a.scale, &up, c);
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        uint32_t w[kParts<T>][4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          split2<T>(qv[kk][i >> 1][(i & 1) * 2] * up, qv[kk][i >> 1][(i & 1) * 2 + 1] * up,
                    &w[0][i], 4);
#pragma unroll
        for (int p = 0; p < kParts<T>; ++p)
          qp[p][kk] = u32x4{w[p][0], w[p][1], w[p][2], w[p][3]};
      }
    };
    if constexpr (R == 1) {
      convert(&c[0]);
    } else {
      __syncthreads();  // the memory's earlier readers
      if (wave < R) {   // a block of 16 rows each
        float mine;
        convert(&mine);
        const bool finite = finite_q(qp);
#pragma unroll
        for (int p = 0; p < kParts<T>; ++p)
#pragma unroll
          for (int kk = 0; kk < KK; ++kk)
            reinterpret_cast<u32x4*>(smem)[((wave * kParts<T> + p) * KK + kk) * 64 + lane] =
                qp[p][kk];
        if (lane < 16) {
          s_c[wave * 16 + lane] = mine;
          s_odd[wave * 16 + lane] = !finite;
        }
      }
      __syncthreads();
#pragma unroll
      for (int r = 0; r < R; ++r) c[r] = s_c[r * 16 + (lane & 15)];
    }
    auto finite = [&](int r) {
      if constexpr (R == 1) return finite_q(qp);
      else return s_odd[r * 16 + (fresh(lane) & 15)] == 0;
    };

    float m[R], l[R];
    f32x4 acc[R][DB];
    auto begin = [&] {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.0f;
#pragma unroll
        for (int db = 0; db < DB; ++db) acc[r][db] = f32x4{};
      }
    };
    begin();
    // The sums of 32 rows of 256 lie where only matrix instructions reach them, as far as it
    // goes: beside 16-bit loads in flight they would take all the others, and those loads were
    // spilled as they came (16 x 26 rows of 16 heads over 8192: 278 us, so 134).
    auto set_aside = [&] {
      if constexpr (R == 2 && D > 128 && !kBytes<T>)
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int db = 0; db < DB; ++db) asm("" : "+a"(acc[r][db]));
    };
    // Twice in the code, so that the first pass has nothing of what only the second does.
    auto pass = [&](auto second) __attribute__((always_inline)) {
      constexpr bool careful = decltype(second)::value;
      for (; base < hi; base += 4 * kStep) {
        // The step's keys are whole for every row, or each lane's keys are checked.
        const uint32_t bad_now = (uint32_t)(bad >> (at * kTiles)) & ((1u << kTiles) - 1);
        const bool whole = base >= s.span.lo_all && base + kStep <= s.span.hi_all && bad_now == 0;

        set_aside();
        float sc[R][kTiles][4];
        if constexpr (R == 1) {
#pragma unroll
          for (int t = 0; t < kTiles; ++t) {
            f32x4 sum = {};
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
              const u32x4 kf = operand(x.k[t][kk]);
#pragma unroll
              for (int p = 0; p < kParts<T>; ++p) sum = mfma16<T>(kf, qp[p][kk], sum);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[0][t][i] = sum[i];
          }
        } else {
          const u32x4* s_q = reinterpret_cast<const u32x4*>(smem) + fresh(lane);
          f32x4 sum[R][kTiles] = {};
#pragma unroll
          for (int kk = 0; kk < KK; ++kk) {
            u32x4 kf[kTiles];
#pragma unroll
            for (int t = 0; t < kTiles; ++t) kf[t] = operand(x.k[t][kk]);
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
              for (int p = 0; p < kParts<T>; ++p) {
                const u32x4 qf = s_q[((r * kParts<T> + p) * KK + kk) * 64];
#pragma unroll
                for (int t = 0; t < kTiles; ++t) sum[r][t] = mfma16<T>(kf[t], qf, sum[r][t]);
              }
          }
#pragma unroll
          for (int r = 0; r < R; ++r)
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
#pragma unroll
              for (int i = 0; i < 4; ++i) sc[r][t][i] = sum[r][t][i];
        }
        if constexpr (kBytes<T>) {
#pragma unroll
          for (int t = 0; t < kTiles; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float log2_scale = scale_log2(x.vs[t][i]);
#pragma unroll
              for (int r = 0; r < R; ++r)
                sc[r][t][i] = __builtin_fmaf(sc[r][t][i] * c[r], x.ks[t][i], log2_scale);
            }
        } else if (careful) {
#pragma unroll
          for (int r = 0; r < R; ++r) {
            if (!__any((int)any_nan(sc[r]) & (int)finite(r))) continue;
            const AttentionArgs a = fresh_args();
            const int me = fresh(lane), place = r * 16 + (me & 15);
            const int in = (R > 1 ? s.r0 : 0) + (place < s.rows ? place : s.rows - 1);
            const int tok = (int)a.by_group.of(in);
            const float* q = a.q + (int64_t)(s.seq.row0 + tok) * a.q_stride +
                             (int64_t)(s.g * a.group + in - tok * a.group) * D;
#pragma unroll 1
            for (int j = 0; j < kTiles * 4; ++j) {
              const uint16_t* k = static_cast<const uint16_t*>(a.cache.k) +
                                  (j < 4 ? tile[0] : tile[1]) * (kKvTile * D) +
                                  ((me >> 4) * 4 + j % 4) * 8;
              const float exact = product_of<T, D>(q, k);
#pragma unroll
              for (int i = 0; i < kTiles * 4; ++i)
                if (i == j && sc[r][i / 4][i % 4] != sc[r][i / 4][i % 4])
                  sc[r][i / 4][i % 4] = exact * a.scale;
            }
          }
        }

        // The next step's K goes out before the softmax.
        const bool more = base + 4 * kStep < hi;
        const int64_t tile_now[2] = {tile[0], tile[1]};
        if (more) {
          if (++at == kAhead) {
            held = look_up(a, s, lane, base + 4 * kStep);
            bad = __ballot(held.bad);
            at = 0;
          }
          take(held, at, tile);
          load_k(a, lane, tile, x);
        }

        if (!whole) {
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const int from = fresh(base + quad * 4 - (kTrees ? 0 : mine[r].lo));
            uint32_t bits = 0;
#pragma unroll
            for (int t = 0; t < kTiles; ++t) {
              if (kTrees && t % 2 == 0) bits = mine[r].of(from + t * kKvTile);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const bool in = kTrees ? bits >> (t % 2 * kKvTile + i) & 1
                                       : (uint32_t)(from + t * kKvTile + i) < mine[r].width;
                const bool seen = in && !(bad_now >> t & 1);
                sc[r][t][i] = seen ? sc[r][t][i] : -INFINITY;
              }
            }
          }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float to_log2 = kBytes<T> ? 1.0f : c[r];
          float top = -INFINITY;
#pragma unroll
          for (int t = 0; t < kTiles; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) top = fmaxf(top, sc[r][t][i]);
          top *= to_log2;
          if (__any(top - m[r] > kSlack)) {
            top = with_32(with_16(top, max_float), max_float);
            const float to = fminf(fmaxf(m[r], top), kLargest);
            const float keep = to == -INFINITY ? 1.0f : exp2_of(m[r] - to);
            m[r] = to;
            l[r] *= keep;
#pragma unroll
            for (int db = 0; db < DB; ++db) acc[r][db] *= keep;
          }
          const float ref = (m[r] == -INFINITY ? 0.0f : m[r]) - kHeadroom<T>;
#pragma unroll
          for (int t = 0; t < kTiles; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float p = exp2_of(__builtin_fmaf(sc[r][t][i], to_log2, -ref));
              if constexpr (kBytes<T>) l[r] = __builtin_fmaf(p, scale_inverse(x.vs[t][i]), l[r]);
              else l[r] += p;
              sc[r][t][i] = p;
            }
        }

        bool odd = false;  // a value of V that is not finite
        if constexpr (!kBytes<T>) {
          if (careful || base < s.span.lo || base + kStep > s.span.hi || bad_now != 0) {
            // Values that no row sees count as zero.
            const int from = fresh(base + (lane >> 4 & 1) * 4);
            uint32_t found = 0;
#pragma unroll
            for (int u = 0; u < kTiles / 2; ++u) {
              const int t = 2 * u + (lane >> 5);
#pragma unroll
              for (int w = 0; w < 4; ++w) {
                const int key = from + t * kKvTile + (w >> 1) * 8 + (w & 1) * 2;
                const bool tile_ok = !(bad_now >> t & 1);
                const uint32_t keep =
                    (tile_ok && key >= s.span.lo && key < s.span.hi ? 0x0000ffffu : 0u) |
                    (tile_ok && key + 1 >= s.span.lo && key + 1 < s.span.hi ? 0xffff0000u : 0u);
#pragma unroll
                for (int db = 0; db < DB; ++db) {
                  x.v[u][db][w] &= keep;
                  found |= non_finite<T>(x.v[u][db][w]);
                }
              }
            }
            odd = careful && __any(found != 0);
            if (odd)
#pragma unroll
              for (int u = 0; u < kTiles / 2; ++u)
#pragma unroll
                for (int db = 0; db < DB; ++db)
#pragma unroll
                  for (int w = 0; w < 4; ++w)
                    x.v[u][db][w] &= ~((non_finite<T>(x.v[u][db][w]) >> 15) * 0xffffu);
          }
        }

        set_aside();
        // P as the right operand: tokens 4 h' .. of a pair of tiles, by one exchange of the
        // wave's halves.
#pragma unroll
        for (int u = 0; u < kTiles / 2; ++u) {
          u32x4 pp[R][kParts<T>];
#pragma unroll
          for (int r = 0; r < R; ++r) {
            uint32_t w[2][2][kParts<T>];  // [tile][pair][part]
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
              for (int h = 0; h < 2; ++h)
                split2<T>(sc[r][2 * u + t][2 * h], sc[r][2 * u + t][2 * h + 1], &w[t][h][0], 1);
#pragma unroll
            for (int p = 0; p < kParts<T>; ++p) {
              const auto e0 =
                  __builtin_amdgcn_permlane32_swap(w[0][0][p], w[1][0][p], false, false);
              const auto e1 =
                  __builtin_amdgcn_permlane32_swap(w[0][1][p], w[1][1][p], false, false);
              pp[r][p] =
                  u32x4{(uint32_t)e0[0], (uint32_t)e1[0], (uint32_t)e0[1], (uint32_t)e1[1]};
            }
          }
#pragma unroll
          for (int db = 0; db < DB; ++db) {
            const u32x4 vf = operand(x.v[u][db]);
#pragma unroll
            for (int p = 0; p < kParts<T>; ++p)
#pragma unroll
              for (int r = 0; r < R; ++r) acc[r][db] = mfma16<T>(vf, pp[r][p], acc[r][db]);
          }
        }
        if constexpr (!kBytes<T>) {
          if (odd) {  // values that are not finite, for the rows that see them
#pragma unroll 1
            for (int j = 0; j < kStep; ++j) {
              const int64_t ti = j < kKvTile ? tile_now[0] : tile_now[1];
              const int tok = j % kKvTile, key = base + j;
              const bool there = !(bad_now >> (j / kKvTile) & 1);
              bool seen[R];
#pragma unroll
              for (int r = 0; r < R; ++r) seen[r] = mine[r].sees(key) && there;
              const uint16_t* p = static_cast<const uint16_t*>(a.cache.v) + ti * (kKvTile * D) +
                                  (tok / 4 % 2) * (D * 8) + (tok / 8) * 4 + tok % 4;
#pragma unroll
              for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const uint32_t v = p[(db * 16 + quad * 4 + i) * 8];
#pragma unroll
                  for (int r = 0; r < R; ++r)
                    if (seen[r] && is_non_finite<T>(v)) acc[r][db][i] += value_of<T>(v);
                }
            }
          }
        }
        if (more) load_v(a, lane, tile, x);
      }
    };
    pass(std::false_type{});
    if constexpr (!kBytes<T>) {
      bool again = false;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float zero = 0.0f;  // NaN where a sum is not finite
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int i = 0; i < 4; ++i) zero = __builtin_fmaf(acc[r][db][i], 0.0f, zero);
        // A row of q that is not finite is NaN either way.
        if (__any(zero != zero) && __any((int)(zero != zero) & (int)finite(r))) again = true;
      }
      if (again) {
        begin();
        base = s.k0 + wave * kStep;
        held = look_up(a, s, lane, base);
        start(a, s, lane, wave, n);
        bad = __ballot(held.bad);
        at = 0;
        take(held, 0, tile);
        pass(std::true_type{});
      }
    }
    // The next segment's first loads are under way while this one is joined and written.
    n.started = go_on;
    if (go_on) {
      forget();
      const Segment t = uniform(*then);
      held = tile_of(a, t, key_of(lane, t.k0 + wave * kStep), then_page);
      start(a, t, lane, wave, n);
    }
    f32x4* s_acc = reinterpret_cast<f32x4*>(smem);                // [wave][4 D]
    f32x2* s_ml = reinterpret_cast<f32x2*>(smem + 4 * 4 * D * 16);  // [wave][16]
    const int here = fresh(tid), row = here & 15;
    auto in_range = [&](int i) { return 4 * D % kThreads == 0 || here + i * kThreads < 4 * D; };
    auto write = [&](int r, const f32x4 (&out)[NQ], float L) {
      if (r * 16 + row < s.rows) {
        float* o = out_row(a, s, r * 16 + row);
        const float inv = L != 0.0f ? 1.0f / L : 0.0f;
#pragma unroll
        for (int i = 0; i < NQ; ++i)
          if (in_range(i))
            *reinterpret_cast<f32x4*>(o + (here + i * kThreads) / 16 * 4) =
                L != 0.0f ? out[i] * inv : f32x4{};
      }
    };
    // A row's part, of which the rows past the tile's are not read.
    auto store = [&](int r, int part, const f32x4 (&out)[NQ], float M, float L) {
      const __amdgpu_buffer_rsrc_t rs = buffer_rsrc(sh.partials, sh.bytes);
      const uint32_t to = same_slot_at(sh, s, part) + r * Part::kBytes;
      if (r * 16 + row < s.rows) {
#pragma unroll
        for (int i = 0; i < NQ; ++i)
          if (in_range(i)) store_part(out[i], rs, here * 16, to + i * kThreads * 16);
        if (here < 16) store_part2(f32x2{M, L}, rs, here * 8, to + kMl);
      }
    };
#pragma unroll
    for (int r = 0; r < R; ++r) {
      l[r] = with_32(with_16(l[r], sum_float), sum_float);

      // Join the four waves; thread tid has the quads tid + 256 i: row tid % 16.
      __syncthreads();  // the memory's earlier readers
#pragma unroll
      for (int db = 0; db < DB; ++db)
        s_acc[wave * 4 * D + db * 64 + (here & 63)] = acc[r][db];
      if ((here & 63) < 16) s_ml[wave * 16 + row] = f32x2{m[r], l[r]};
      __syncthreads();
      f32x4 out[NQ] = {};
      float M = -INFINITY, L = 0.0f;
#pragma unroll
      for (int w = 0; w < 4; ++w) M = fmaxf(M, s_ml[w * 16 + row].x);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const f32x2 ml = s_ml[w * 16 + row];
        const float f = weight(ml.x, M);
        // A NaN row's sum is NaN whatever its weight.
        L = __builtin_fmaf(ml.y, f, L);
#pragma unroll
        for (int i = 0; i < NQ; ++i)
          if (in_range(i)) out[i] += s_acc[w * 4 * D + here + i * kThreads] * f;
      }
      if (s.parts > 1) store(r, s.part, out, M, L);
      else write(r, out, L);
    }
    if (s.parts == 1) return go_on;

    int* arrived = reinterpret_cast<int*>(smem);
    if (R == 1 && s.rows <= 8 && s.parts > 8) {
      if (last_to_arrive(sh.counters + s.first * kCounterStride, s.parts, arrived))
        join_many(a, s, sh, here, smem);
      return go_on;
    }
    const __amdgpu_buffer_rsrc_t rs = buffer_rsrc(sh.partials, sh.bytes);
    float M[R], L[R];
    f32x4 out[R][NQ];
    const bool whole = join_parts(
        sh, s, arrived,
        [&](int first, int step, int count) {
#pragma unroll
          for (int r = 0; r < R; ++r) {
            // Some at a time, whose loads are in flight together.
            constexpr int kAtOnce = 12 / NQ;
            M[r] = -INFINITY;
            L[r] = 0.0f;
#pragma unroll
            for (int i = 0; i < NQ; ++i) out[r][i] = f32x4{};
            for (int p0 = 0; p0 < count; p0 += kAtOnce) {
              f32x2 ml[kAtOnce];
              f32x4 v[kAtOnce][NQ];
#pragma unroll
              for (int p = 0; p < kAtOnce; ++p) {
                // Past the last part: that one again, not used.
                const int part = first + step * (p0 + p < count ? p0 + p : count - 1);
                const uint32_t from = same_slot_at(sh, s, part) + r * Part::kBytes;
                ml[p] = load_part2(rs, row * 8, from + kMl);
#pragma unroll
                for (int i = 0; i < NQ; ++i)
                  if (in_range(i)) v[p][i] = load_part(rs, here * 16, from + i * kThreads * 16);
              }
              float top = M[r];
#pragma unroll
              for (int p = 0; p < kAtOnce; ++p) top = fmaxf(top, ml[p].x);
              const float keep = weight(M[r], top);
              M[r] = top;
              L[r] *= keep;
#pragma unroll
              for (int i = 0; i < NQ; ++i) out[r][i] *= keep;
#pragma unroll
              for (int p = 0; p < kAtOnce; ++p) {
                if (p0 + p < count) {
                  const float f = weight(ml[p].x, M[r]);
                  L[r] = __builtin_fmaf(ml[p].y, f, L[r]);
#pragma unroll
                  for (int i = 0; i < NQ; ++i)
                    if (in_range(i)) out[r][i] += v[p][i] * f;
                }
              }
            }
          }
        },
        [&](int part) {
#pragma unroll
          for (int r = 0; r < R; ++r) store(r, part, out[r], M[r], L[r]);
        });
    if (whole)
#pragma unroll
      for (int r = 0; r < R; ++r) write(r, out[r], L[r]);
    return go_on;
  }
};

// 16 bytes a lane from global memory to LDS, a wave's 1024 in one run, without registers.
// Not the builtin: with that every later read of LDS first waits for all loads in flight.
// The caller waits (wait_for_loads) before the barrier behind which the bytes are read.
// m0 holds the place in LDS: the compiler writes it there, so it knows what m0 holds.
__device__ __forceinline__ void load_to_lds(const uint8_t* from, uint8_t* to) {
  const uint32_t at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)to;
  register int m0 asm("m0") = uniform((int)at);
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :: "s"(m0), "v"(from) : "memory");
}

__device__ __forceinline__ void wait_for_loads() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// ---- many rows: four waves of 32 rows share the keys in LDS ----
//
// 32 rows a wave, so that a fragment of K or V from LDS feeds all parts' products (32 KB of
// LDS reads for 2048 cycles of the matrix cores a unit); stages of 64 keys, two of them, one
// loading while the other is used; one barrier a stage.  8-bit stages go through registers
// and become f16 on the way, once for all four waves.

template <KvType T, int D>
struct ManyRows {
  static constexpr int KK = D / 16, DB = D / 32;
  static constexpr int kTilesUnit = kUnit / kKvTile;
  static constexpr int kTileBytes = kKvTile * D * 2;         // in LDS: 16-bit elements
  static constexpr int kHalf = kUnit * D * 2;                // K or V of a stage
  static constexpr int kStage = 2 * kHalf;
  static constexpr int kScales = 2 * kStage;                 // [2][3][64] floats (8-bit caches)
  static constexpr int kFlags = kScales + (kBytes<T> ? 2 * 3 * kUnit * 4 : 0);  // two of any_of
  static constexpr int kLdsBytes = kFlags + 32;
  // 16-byte loads of a stage's K, a thread (8-bit head sizes of 96: some threads none).
  static constexpr int kChunks = kUnit * D * (kBytes<T> ? 1 : 2) / 16;
  static constexpr int kLoads = (kChunks + kThreads - 1) / kThreads;

  struct Staged {  // 8-bit caches: a stage on its way through registers
    u32x4 k[kBytes<T> ? kLoads : 1], v[kBytes<T> ? kLoads : 1];
    float ks, vs;
  };

  // Whether a thread of the workgroup has `mine`; a barrier.  `flags` is written again only
  // behind a later barrier.
  static __device__ __forceinline__ bool any_of(bool mine, int wave, uint8_t* flags) {
    reinterpret_cast<uint32_t*>(flags)[wave] = __any(mine);
    __syncthreads();
    const u32x4 all = *reinterpret_cast<const u32x4*>(flags);
    return uniform((int)(all.x | all.y | all.z | all.w)) != 0;
  }

  // Whether the lane's row of q is finite; lanes l and l + 32 have it, and both come here.
  static __device__ __forceinline__ bool finite_q(const u32x4 (&qp)[kParts<T>][KK]) {
    return with_32(non_finite<T>(qp[0]), max_bits) == 0;
  }
  static __device__ __forceinline__ bool any_nan(const f32x16& sc) {
    bool nan = false;
#pragma unroll
    for (int i = 0; i < 16; ++i) nan |= sc[i] != sc[i];
    return nan;
  }

  static __device__ __forceinline__ bool has_chunk(int chunk) {
    return kChunks % kThreads == 0 || chunk < kChunks;
  }

  // Starts the loads of the unit whose first tile is lane `first` of `tiles`.
  static __device__ __forceinline__ void issue(const AttentionArgs& a, int tid, int64_t tiles,
                                               int first, uint8_t* stage, Staged& x) {
    tid = fresh(tid);
    const int lane = tid & 63, wave = uniform(tid >> 6);
    if constexpr (kBytes<T>) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int chunk = tid + i * kThreads, tile = chunk / D;
        const int64_t at = from_lane(tiles, first + tile) * (kKvTile * D) + (chunk - tile * D) * 16;
        if (has_chunk(chunk)) {
          x.k[i] = *reinterpret_cast<const u32x4*>(static_cast<const uint8_t*>(a.cache.k) + at);
          x.v[i] = *reinterpret_cast<const u32x4*>(static_cast<const uint8_t*>(a.cache.v) + at);
        }
      }
      if (wave == 0) {
        const int64_t mine =
            from_lane(tiles, first + lane / kKvTile) * kKvTile + lane % kKvTile;
        x.ks = a.cache.k_scale[mine];
        x.vs = a.cache.v_scale[mine];
      }
    } else {
      constexpr int kPerTile = kTileBytes / 1024;  // wave loads of a tile
      static_assert(kTileBytes % 1024 == 0 && kTilesUnit * kPerTile == 4 * kLoads);
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int n = i * 4 + wave;  // the wave's load of the stage's K or V
        const int tile = n / kPerTile, part = n - tile * kPerTile;
        const int64_t at = lane_of(tiles, first + tile) * kTileBytes + part * 1024 + lane * 16;
        uint8_t* to = stage + n * 1024;
        load_to_lds(static_cast<const uint8_t*>(a.cache.k) + at, to);
        load_to_lds(static_cast<const uint8_t*>(a.cache.v) + at, to + kHalf);
      }
    }
  }

  // 8-bit caches: the staged unit into LDS as f16.
  static __device__ __forceinline__ void commit(int tid, uint8_t* smem, int buf,
                                                const Staged& x) {
    if constexpr (kBytes<T>) {
      tid = fresh(tid);
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int chunk = tid + i * kThreads;
        if (!has_chunk(chunk)) break;
        u32x4* k = reinterpret_cast<u32x4*>(smem + buf * kStage) + chunk * 2;
        u32x4* v = reinterpret_cast<u32x4*>(smem + buf * kStage + kHalf) + chunk * 2;
        k[0] = quants_to_f16(u32x2{x.k[i].x, x.k[i].y});
        k[1] = quants_to_f16(u32x2{x.k[i].z, x.k[i].w});
        v[0] = quants_to_f16(u32x2{x.v[i].x, x.v[i].y});
        v[1] = quants_to_f16(u32x2{x.v[i].z, x.v[i].w});
      }
      if (tid < kUnit) {
        float* sc = reinterpret_cast<float*>(smem + kScales) + buf * 3 * kUnit;
        sc[tid] = x.ks;
        sc[kUnit + tid] = scale_log2(x.vs);
        sc[2 * kUnit + tid] = scale_inverse(x.vs);
      }
    }
  }

  // V's places that no row sees become zero; where asked for, so do values that are not
  // finite, which the caller adds to the rows that see them.  Returns whether there were any.
  static __device__ __forceinline__ bool clear_v(const Segment& s, int tid, int base,
                                                 uint32_t bad, bool careful, uint8_t* stage) {
    bool found = false;
    if constexpr (!kBytes<T>) {
      tid = fresh(tid);
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int chunk = tid + i * kThreads;
        const int tile = chunk / (2 * D), in = chunk - tile * 2 * D, half = in / D;
        u32x4* p = reinterpret_cast<u32x4*>(stage + kHalf) + chunk;
        u32x4 v = *p;
        const bool tile_ok = !(bad >> tile & 1);
        uint32_t odd = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int key = base + tile * kKvTile + (w >> 1) * 8 + half * 4 + (w & 1) * 2;
          v[w] &= (tile_ok && key >= s.span.lo && key < s.span.hi ? 0x0000ffffu : 0u) |
                  (tile_ok && key + 1 >= s.span.lo && key + 1 < s.span.hi ? 0xffff0000u : 0u);
          odd |= non_finite<T>(v[w]);
        }
        if (careful && odd != 0) {
          found = true;
#pragma unroll
          for (int w = 0; w < 4; ++w) v[w] &= ~((non_finite<T>(v[w]) >> 15) * 0xffffu);
        }
        *p = v;
      }
    }
    return found;
  }

  // The segment's keys for the tile's rows: their maxima m, sums l (a share of it a lane) and
  // products acc.  Says whether a sum is not finite; the second pass, a function of its own so
  // that the first has none of what only it needs, then does the same with values that are not
  // finite row by row.
  template <bool kSecond>
  static __device__ __forceinline__ bool attend(const Segment& s, uint8_t* smem, float& m,
                                                float& l, f32x16 (&acc)[DB]) {
    const AttentionArgs a = fresh_args();
    const int tid = fresh_tid(), lane = tid & 63, wave = uniform(tid >> 6);
    const int half = lane >> 5;
    const int wrow = wave * 32 + (lane & 31);
    const int row = s.r0 + (wrow < s.rows ? wrow : s.rows - 1);
    const int token = (int)a.by_group.of(row);
    const bool live = wave * 32 < s.rows;
    const Sight mine = sight_of(a, s.seq, row);
    // What the wave's rows see together and alone.
    const int w0 = live ? wave * 32 : 0, w1 = s.rows < w0 + 32 ? s.rows : w0 + 32;
    const Span ours = span_of(a, s.seq, s.r0 + w0, s.r0 + w1);

    const int hi = s.k1 < s.span.hi ? s.k1 : s.span.hi;
    Staged staged;
    Tiles held;
    uint64_t bad = 0;
    int at = 0;  // unit among the 16 whose tiles the lanes hold
    auto look_up = [&](int from) {
      held = find_tile(a, s, from + fresh(lane) * kKvTile);
      bad = __ballot(held.bad);
      at = 0;
    };
    // q ahead of the first keys, which wait for the table.
    const float* q = a.q + (int64_t)(s.seq.row0 + token) * a.q_stride +
                     (int64_t)(s.g * a.group + row - token * a.group) * D + half * 8;
    f32x4 qv[KK][2];
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        qv[kk][h] = *reinterpret_cast<const f32x4*>(q + kk * 16 + h * 4);
    look_up(s.k0);
    __syncthreads();  // the memory's earlier readers
    if (s.k0 < hi) issue(a, tid, held.index, 0, smem, staged);

    u32x4 qp[kParts<T>][KK];
    float c = 0.0f;
    {
      uint32_t amax = 0;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
#pragma unroll
        for (int h = 0; h < 2; ++h) amax = max_bits(amax, magnitude(qv[kk][h]));
      amax = with_32(amax, max_bits);
      float up;
      row_scale<T>(amax, a.scale, &up, &c);
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        uint32_t w[kParts<T>][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const f32x4 v = qv[kk][h];
          split2<T>(v.x * up, v.y * up, &w[0][2 * h], 4);
          split2<T>(v.z * up, v.w * up, &w[0][2 * h + 1], 4);
        }
#pragma unroll
        for (int p = 0; p < kParts<T>; ++p) qp[p][kk] = u32x4{w[p][0], w[p][1], w[p][2], w[p][3]};
      }
    }
    if (s.k0 < hi) commit(tid, smem, 0, staged);

    // Operands of 32 keys: K's of all steps, or V's of two tiles; as many either way, all at
    // once or some of them, as registers allow.
    constexpr bool kLean = kParts<T> == 3 || kBytes<T>;
    constexpr int FB = KK / ((kLean ? 2 : 1) * (D > 128 ? 2 : 1));
    u32x4 f[FB];
    const uint32_t k_at = (lane >> 4 & 1) * kTileBytes + half * 256 + (lane & 15) * 16;
    const uint32_t v_at = kHalf + (half * D + (lane & 31)) * 16;
    auto read_k = [&](const uint8_t* stage, int u, int from) {
#pragma unroll
      for (int n = 0; n < FB; ++n)
        f[n] = *reinterpret_cast<const u32x4*>(stage + k_at + 2 * u * kTileBytes +
                                               (from + n) * 512);
    };
    auto read_v = [&](const uint8_t* stage, int u, int from) {
#pragma unroll
      for (int n = 0; n < FB; ++n)
        f[n] = *reinterpret_cast<const u32x4*>(
            stage + v_at + (2 * u + (from + n) / DB) * kTileBytes + (from + n) % DB * 512);
    };

    m = -INFINITY;
    l = 0.0f;
#pragma unroll
    for (int db = 0; db < DB; ++db) acc[db] = f32x16{};
    int buf = 0;
    for (int base = s.k0; base < hi; base += kUnit, buf ^= 1) {
      const uint32_t bad_now = (uint32_t)(bad >> (at * kTilesUnit)) & ((1u << kTilesUnit) - 1);
      const int64_t tiles_now = held.index;
      const int at_now = at;
      uint8_t* stage = smem + buf * kStage;
      wait_for_loads();  // this wave's loads of the stage
      __syncthreads();   // everyone's; and the other stage's readers are done
      const bool more = base + kUnit < hi;
      if (more) {
        if (++at == 64 / kTilesUnit) look_up(base + kUnit);
        issue(a, tid, held.index, at * kTilesUnit, smem + (buf ^ 1) * kStage, staged);
      }
      bool odd = false;
      if (!kBytes<T> && (kSecond || base < s.span.lo || base + kUnit > s.span.hi || bad_now != 0))
      {
        const bool found = clear_v(s, tid, base, bad_now, kSecond, stage);
        if constexpr (kSecond) odd = any_of(found, wave, smem + kFlags);
        else __syncthreads();
      }

      if (live && base < ours.hi && base + kUnit > ours.lo) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {  // 32 keys: two tiles
          const int from_key = base + u * 32;
          if (from_key >= ours.hi || from_key + 32 <= ours.lo) continue;
          const bool whole =
              from_key >= ours.lo_all && from_key + 32 <= ours.hi_all && bad_now == 0;
          f32x16 sc = {};
#pragma unroll
          for (int from = 0; from < KK; from += FB) {
            read_k(stage, u, from);
#pragma unroll
            for (int n = 0; n < FB; ++n)
#pragma unroll
              for (int p = 0; p < kParts<T>; ++p) sc = mfma32<T>(f[n], qp[p][from + n], sc);
          }
          read_v(stage, u, 0);  // on its way during the softmax
          const float* ks = reinterpret_cast<const float*>(smem + kScales) + buf * 3 * kUnit +
                            u * 32 + half * 4;
          if constexpr (kBytes<T>) {
#pragma unroll
            for (int b4 = 0; b4 < 4; ++b4) {
              const f32x4 k4 = *reinterpret_cast<const f32x4*>(ks + b4 * 8);
              const f32x4 l4 = *reinterpret_cast<const f32x4*>(ks + kUnit + b4 * 8);
#pragma unroll
              for (int i = 0; i < 4; ++i)
                sc[b4 * 4 + i] = __builtin_fmaf(sc[b4 * 4 + i] * c, k4[i], l4[i]);
            }
          }
          if (!kBytes<T> && kSecond && __any((int)any_nan(sc) & (int)finite_q(qp))) {
            const AttentionArgs a = fresh_args();
            const int me = fresh_tid(), in = (me >> 6) * 32 + (me & 31);
            const int row = s.r0 + (in < s.rows ? in : s.rows - 1);
            const int token = (int)a.by_group.of(row);
            const float* q = a.q + (int64_t)(s.seq.row0 + token) * a.q_stride +
                             (int64_t)(s.g * a.group + row - token * a.group) * D;
#pragma unroll 1
            for (int j = 0; j < 16; ++j) {
              const int key = (j >> 2) * 8 + (me >> 3 & 4) + (j & 3);
              const uint16_t* k = reinterpret_cast<const uint16_t*>(
                                      stage + (2 * u + key / kKvTile) * kTileBytes) +
                                  key % kKvTile * 8;
              const float exact = product_of<T, D>(q, k);
#pragma unroll
              for (int i = 0; i < 16; ++i)
                if (i == j && sc[i] != sc[i]) sc[i] = exact * a.scale;
            }
          }
          if (!whole) {
            const int from = fresh(base + half * 4 - (kTrees ? 0 : mine.lo));
            const uint32_t bits = kTrees ? mine.of(from + u * 32) : 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const bool in = kTrees
                                  ? bits >> ((i >> 2) * 8 + (i & 3)) & 1
                                  : (uint32_t)(from + u * 32 + (i >> 2) * 8 + (i & 3)) < mine.width;
              const bool seen = in && !(bad_now >> (2 * u + (i >> 3)) & 1);
              sc[i] = seen ? sc[i] : -INFINITY;
            }
          }
          const float to_log2 = kBytes<T> ? 1.0f : c;
          float top = -INFINITY;
#pragma unroll
          for (int i = 0; i < 16; ++i) top = fmaxf(top, sc[i]);
          top *= to_log2;
          if (__any(top - m > kSlack)) {
            top = with_32(top, max_float);
            const float to = fminf(fmaxf(m, top), kLargest);
            const float keep = to == -INFINITY ? 1.0f : exp2_of(m - to);
            m = to;
            l *= keep;
#pragma unroll
            for (int db = 0; db < DB; ++db) acc[db] *= keep;
          }
          const float ref = (m == -INFINITY ? 0.0f : m) - kHeadroom<T>;
          uint32_t w[kParts<T>][8];
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            const float p0 = exp2_of(__builtin_fmaf(sc[i], to_log2, -ref));
            const float p1 = exp2_of(__builtin_fmaf(sc[i + 1], to_log2, -ref));
            if constexpr (kBytes<T>) {
              const f32x2 inv = *reinterpret_cast<const f32x2*>(ks + 2 * kUnit + (i >> 2) * 8 +
                                                                (i & 3));
              l = __builtin_fmaf(p0, inv.x, l);
              l = __builtin_fmaf(p1, inv.y, l);
            } else {
              l += p0;
              l += p1;
            }
            split2<T>(p0, p1, &w[0][i / 2], 8);
          }
#pragma unroll
          for (int from = 0; from < KK; from += FB) {
            if (from > 0) read_v(stage, u, from);
#pragma unroll
            for (int n = 0; n < FB; ++n) {
              const int t = (from + n) / DB, db = (from + n) % DB;
#pragma unroll
              for (int p = 0; p < kParts<T>; ++p)
                acc[db] = mfma32<T>(
                    f[n], u32x4{w[p][4 * t], w[p][4 * t + 1], w[p][4 * t + 2], w[p][4 * t + 3]},
                    acc[db]);
            }
          }
        }
        if constexpr (!kBytes<T>) {
          if (odd) {  // values that are not finite, for the rows that see them
#pragma unroll 1
            for (int j = 0; j < kUnit; ++j) {
              const int tok = j % kKvTile, key = base + j;
              const bool seen = mine.sees(key) && !(bad_now >> (j / kKvTile) & 1);
              const int64_t ti = lane_of(tiles_now, at_now * kTilesUnit + j / kKvTile);
              const uint16_t* p = static_cast<const uint16_t*>(a.cache.v) + ti * (kKvTile * D) +
                                  (tok / 4 % 2) * (D * 8) + (tok / 8) * 4 + tok % 4;
#pragma unroll
              for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                  const uint32_t v = p[(db * 32 + (i >> 2) * 8 + half * 4 + (i & 3)) * 8];
                  if (seen && is_non_finite<T>(v)) acc[db][i] += value_of<T>(v);
                }
            }
          }
        }
      }
      if (more) commit(tid, smem, buf ^ 1, staged);
    }
    if constexpr (!kBytes<T> && !kSecond) {
      float zero = 0.0f;  // NaN where a sum is not finite
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) zero = __builtin_fmaf(acc[db][i], 0.0f, zero);
      // A row of q that is not finite is NaN either way.
      bool odd = false;
      if (__any(zero != zero)) odd = (zero != zero) & finite_q(qp);
      return any_of(odd, wave, smem + kFlags + 16);
    }
    return false;
  }

  static __device__ __forceinline__ void run(const Segment& s, const Shared& sh,
                                             uint8_t* smem) {
    float m, l;
    f32x16 acc[DB];
    if (attend<false>(s, smem, m, l, acc)) attend<true>(s, smem, m, l, acc);
    l = with_32(l, sum_float);
    const AttentionArgs a = fresh_args();
    const int tid = fresh_tid(), half = tid >> 5 & 1;
    const int wrow = (tid >> 6) * 32 + (tid & 31);
    const int row = s.r0 + (wrow < s.rows ? wrow : s.rows - 1);
    const int token = (int)a.by_group.of(row);

    if (s.parts > 1) {
      constexpr uint32_t kMl = kTileRows * D * 4;
      const int at = fresh(tid);
      const __amdgpu_buffer_rsrc_t rs = buffer_rsrc(sh.partials, sh.bytes);
      auto store = [&](int part) {
        const uint32_t to = same_slot_at(sh, s, part);
        if (wrow < s.rows) {
#pragma unroll
          for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int q = 0; q < 4; ++q)
              store_part(f32x4{acc[db][4 * q], acc[db][4 * q + 1], acc[db][4 * q + 2],
                               acc[db][4 * q + 3]},
                         rs, at * 16, to + (db * 4 + q) * kThreads * 16);
          store_part2(f32x2{m, l}, rs, at * 8, to + kMl);
        }
      };
      store(s.part);
      const bool whole = join_parts(
          sh, s, reinterpret_cast<int*>(smem),
          [&](int first, int step, int count) {
            if (wrow >= s.rows) return;
            // Some at a time: their loads are in flight together.
            constexpr int kAtOnce = D <= 64 ? 4 : D <= 128 ? 2 : 1, kQuads = D / 8;
            m = -INFINITY;
            l = 0.0f;
#pragma unroll
            for (int db = 0; db < DB; ++db) acc[db] = f32x16{};
#pragma unroll 1
            for (int p0 = 0; p0 < count; p0 += kAtOnce) {
              f32x2 ml[kAtOnce];
              f32x4 v[kAtOnce][kQuads];
#pragma unroll
              for (int p = 0; p < kAtOnce; ++p) {
                // Past the last part: that one again, with no weight.
                const int part = first + step * (p0 + p < count ? p0 + p : count - 1);
                const uint32_t from = same_slot_at(sh, s, part);
                ml[p] = load_part2(rs, at * 8, from + kMl);
#pragma unroll
                for (int q = 0; q < kQuads; ++q)
                  v[p][q] = load_part(rs, at * 16, from + q * kThreads * 16);
              }
              float to = m;
#pragma unroll
              for (int p = 0; p < kAtOnce; ++p) to = fmaxf(to, ml[p].x);
              const float keep = weight(m, to);
              m = to;
              l *= keep;
#pragma unroll
              for (int db = 0; db < DB; ++db) acc[db] *= keep;
#pragma unroll
              for (int p = 0; p < kAtOnce; ++p) {
                if (p0 + p < count) {
                  const float f = weight(ml[p].x, m);
                  l = __builtin_fmaf(ml[p].y, f, l);
#pragma unroll
                  for (int q = 0; q < kQuads; ++q)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[q / 4][q % 4 * 4 + i] += v[p][q][i] * f;
                }
              }
            }
          },
          store);
      if (!whole || wrow >= s.rows) return;
    }
    if (wrow < s.rows) {
      const float inv = 1.0f / l;
      float* o = a.out + (int64_t)(s.seq.row0 + token) * a.out_stride +
                 (int64_t)(s.g * a.group + row - token * a.group) * D + half * 4;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          f32x4 v = {acc[db][4 * q], acc[db][4 * q + 1], acc[db][4 * q + 2], acc[db][4 * q + 3]};
          v = l != 0.0f ? v * inv : f32x4{};
          *reinterpret_cast<f32x4*>(o + db * 32 + q * 8) = v;
        }
    }
  }
};

constexpr int kCus = 256, kMostGroups = 2 * kCus;  // workgroups: two a CU up to size 128

template <KvType T, int D>
constexpr int kLds = ManyRows<T, D>::kLdsBytes > 4 * 16 * (D * 4 + 8)
                         ? ManyRows<T, D>::kLdsBytes : 4 * 16 * (D * 4 + 8);

template <KvType T, int D>
__global__ __launch_bounds__(kThreads, D <= 128 ? 2 : 1) void attention_kernel(AttentionArgs a,
                                                                               Shared sh) {
  __shared__ __attribute__((aligned(16))) uint8_t smem[kLds<T, D>];
  __shared__ Schedule sch;
  // A wave's cursor and next segment, here rather than in registers that its loops need.
  __shared__ Cursor<T, D> s_cursor[4];
  __shared__ Segment s_then[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);

  // Costs of all sequences, summed over the threads.
  const int chunk = (a.sequences + kThreads - 1) / kThreads;
  uint64_t sum = 0;
  int tiles = 0;
  for (int i = 0; i < chunk; ++i) {
    const int b = tid * chunk + i;
    Seq s{};
    if (b < a.sequences) s = seq_of(a, b);
    sch.seq[tid] = s;
    const Cost c = cost_of<T, D>(a, s);
    sum += c.before(c.tiles) * a.cache.kv_heads;
    // More than workgroups are no matter.
    const int64_t n = (int64_t)c.tiles * a.cache.kv_heads;
    tiles = tiles + n < kMostGroups ? tiles + (int)n : kMostGroups;
  }
#pragma unroll 1
  for (int off = 1; off < 64; off <<= 1) {
    const uint64_t o = (uint64_t)from_lane((int64_t)sum, lane - off);
    const int n = from_lane(tiles, lane - off);
    if (lane >= off) {
      sum += o;
      tiles += n;
    }
  }
  if (lane == 63) {
    sch.wave_sum[wave] = sum;
    sch.wave_tiles[wave] = tiles;
  }
  __syncthreads();
  for (int i = 0; i < wave; ++i) sum += sch.wave_sum[i];
  sch.sum[tid] = sum;
  __syncthreads();

  // Runs of equal cost; neighbours on one XCD, whose L2 they share.
  Cursor<T, D> cur;
  cur.total = uniform(sch.sum[kThreads - 1]);
  if (cur.total == 0) return;
  // One for each tile, or each least piece of the work if that is more, in eights.
  tiles = sch.wave_tiles[0] + sch.wave_tiles[1] + sch.wave_tiles[2] + sch.wave_tiles[3];
  const uint64_t pieces = cur.total / Weights<T>::kLeastFew;
  uint64_t used = (uint64_t)tiles > pieces ? (uint64_t)tiles : pieces;
  used = used < gridDim.x ? (used + 7) / 8 * 8 : gridDim.x;
  if (blockIdx.x >= used) return;
  cur.run = uniform(quotient(cur.total + used - 1, used));
  cur.w = (int)(blockIdx.x % 8) * (int)(used / 8) + (int)(blockIdx.x / 8);
  const uint64_t from = cur.w * cur.run;
  if (from >= cur.total) return;
  cur.end = from + cur.run < cur.total ? from + cur.run : cur.total;

  // Threads whose sequences come wholly before the run.
  int before = 0;
#pragma unroll
  for (int i = 0; i < kThreads; i += 64)
    before += __builtin_popcountll(__ballot(sch.sum[i + lane] <= from));
  cur.locate(fresh_args(), sch, chunk, uniform(before), from);

  s_cursor[wave] = cur;
  // The next segment into s_then; false at the run's end.
  auto next = [&] {
    forget();
    const AttentionArgs args = fresh_args();
    const int mine = uniform(fresh_tid() >> 6);
    Cursor<T, D> c = s_cursor[mine].uniform_copy();
    Segment then;
    if (!c.next(args, sch, (args.sequences + kThreads - 1) / kThreads, &then)) return false;
    s_cursor[mine] = c;
    s_then[mine] = then;
    forget();
    return true;
  };
  auto take = [&] {
    forget();
    return uniform(s_then[uniform(fresh_tid() >> 6)]);
  };
  // 0: few rows, 1: some, 2: many.
  auto kind_of = [](const Segment& s) {
    const AttentionArgs a = fresh_args();
    const int rows = s.seq.n * a.group;
    return rows <= kFewRows ? 0 : rows <= most_some_rows<T, D>(a, s.seq) ? 1 : 2;
  };
  // Segments of one kind, whose loads go out ahead; false at the run's end.
  bool have = false;
  auto go = [&]<class Rows>(Rows, int kind, Segment s) __attribute__((always_inline)) {
    typename Rows::Ahead ahead;
    Rows::none_ahead(ahead);
    for (;;) {
      const bool go_on = Rows::run(
          s, sh, smem, &s_then[uniform(fresh_tid() >> 6)],
          [&] {
            have = next();
            return have && kind_of(take()) == kind;
          },
          ahead);
      if (!go_on) return have;
      s = take();
    }
  };
  for (;;) {
    if (!have && !next()) return;
    have = false;
    const Segment s = take();
    const int kind = kind_of(s);
    if (kind == 0) {
      if (!go(FewRows<T, D, 1>{}, 0, s)) return;
    } else if (kTrees && kind == 1) {
      if constexpr (kTrees)
        if (!go(FewRows<T, D, 2>{}, 1, s)) return;
    } else {
      ManyRows<T, D>::run(s, sh, smem);
    }
  }
}

int grid_of(int head_dim) { return head_dim <= 128 ? kMostGroups : kCus; }

int slot_floats_of(int head_dim, int64_t rows) {
  return (rows <= kFewRows ? kFewRows : kTileRows) * (head_dim + 4);
}

template <KvType T>
hipError_t launch_typed(const AttentionArgs& a, const Shared& sh, hipStream_t stream) {
  const dim3 grid((unsigned)grid_of(a.cache.head_dim)), block(kThreads);
  switch (a.cache.head_dim) {
    case 64: hipLaunchKernelGGL((attention_kernel<T, 64>), grid, block, 0, stream, a, sh); break;
    case 96: hipLaunchKernelGGL((attention_kernel<T, 96>), grid, block, 0, stream, a, sh); break;
    case 128: hipLaunchKernelGGL((attention_kernel<T, 128>), grid, block, 0, stream, a, sh); break;
    default: hipLaunchKernelGGL((attention_kernel<T, 256>), grid, block, 0, stream, a, sh);
  }
  return hipGetLastError();
}

SplitKNeed workspace_of(int head_dim, int64_t rows) {
  SplitKNeed need;
  need.splits = grid_of(head_dim);
  need.partial_floats = (size_t)need.splits * 2 * slot_floats_of(head_dim, rows);
  need.counters = (size_t)need.splits * kCounterStride;
  return need;
}

hipError_t launch_attention(const AttentionArgs& args, const SplitKWorkspace& ws,
                            hipStream_t stream) {
  AttentionArgs a = args;
  a.group = a.heads / a.cache.kv_heads;
  a.most = a.max_pages * a.cache.page_size;
  a.by_group = Divisor(a.group);
  a.by_page = Divisor(a.cache.page_size);
  const int64_t rows = (int64_t)a.tokens * a.group;
  const SplitKNeed need = workspace_of(a.cache.head_dim, rows);
  const Shared sh{ws.partials, ws.counters, slot_floats_of(a.cache.head_dim, rows),
                  (uint32_t)(need.partial_floats * sizeof(float))};
  switch (a.cache.type) {
    case KvType::kF16: return launch_typed<KvType::kF16>(a, sh, stream);
    case KvType::kBF16: return launch_typed<KvType::kBF16>(a, sh, stream);
    default: return launch_typed<KvType::kInt8>(a, sh, stream);
  }
}

}  // namespace
}  // namespace mle
