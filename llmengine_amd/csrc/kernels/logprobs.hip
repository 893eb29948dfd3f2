// logprobs.hip -- log probabilities of given tokens, entropies and top alternatives of logits
// rows, in one pass over the logits and one launch.
//
// log p(t) = x_t - m - log S and H = log S - W / S, with m the row's maximum,
// S = sum e^(x - m) and W = sum (x - m) e^(x - m).  A thread keeps a maximum and sums of its
// own, brought to a new maximum when one comes: with f = e^(m - m'), W <- f (W + (m - m') S)
// and S <- f S.  S is of 64 bits (their additions cost what those of 32 do): log p of a likely
// token is near 0 and S near 1, and what counts is S's difference from 1.  The exponent is
// (x - m) log2 e, so that the largest terms are exactly 1 and the others off by 2^-23 |x - m|.
// A NaN or an infinite maximum makes S NaN, which is how such rows are found.
//
// Alternatives: the top_n tokens lie in the top_n groups of 128 values of largest maximum, so the
// pass writes the groups' maxima, 1/128 of the row.  The top_n-th largest of 256 threads' largest
// maxima is a bound that at least top_n groups reach, and seldom many more; their values are
// read again, and those that reach it are ranked by counting the larger keys.  Where too many
// groups or values reach it (ties), a radix select over keys, whose low half is the id,
// picks exactly.
//
// A row is cut into pieces, one workgroup each; the one that arrives last at the row's counter
// joins their statistics in order and does the rest.  What the others wrote passes their XCD's
// cache (device-scope stores and loads).  No result depends on the order of arrival.
//
// What bounds it (MI355X; 622 MB are read at 5.65 TB/s): reading the logits, for many rows.  1024
// rows of 151936 with 20 alternatives 127 us, 4.9 TB/s, 110 for a plain read; an exponential, a
// 64-bit addition and an fma a value take a SIMD's time beside it.  208 rows of 32000 14.6 us (5
// for a read) and one of 151936 without alternatives 5.7 us are latencies: loads, the counter,
// the join and the selection, one after the other.
#include "../launch.hpp"
#include "../paged.hpp"
#include "../select.hpp"

namespace mle {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 2048;     // values of a workgroup's step
constexpr int kValues = kChunk / kThreads;  // side by side, a thread's
constexpr int kQuads = kValues / 4;
constexpr int kAhead = 4;        // steps whose loads are in flight
constexpr int kGroup = 16 * kValues;
constexpr int kChunkGroups = kChunk / kGroup;
constexpr int kBlock = 16;       // steps whose maxima are stored together
constexpr int kHeldMaxima = 8;   // a thread keeps this many of the row's maxima in registers
constexpr int kList = 256;       // groups whose values are looked at
constexpr int kCands = 512;      // values that are ranked by counting
// A row's pieces take turns at its counter, and two of them are a lane's.
constexpr int kPiecesRow = 96;
constexpr float kLog2E = 1.44269504088896340736f;
constexpr float kLowest = -0x1.fffffep127f;
constexpr float kFarBelow = -1e30f;  // stands for distances of -Inf, whose terms are 0

// Statistics of a piece: its maximum (+Inf: the row has no distribution), S in two parts, W.
struct Piece {
  float max, sum, rest, weighted;
};

struct Sums {
  float m = kLowest;  // of all values but -Inf
  double s = 0.0, w = 0.0;

  __device__ __forceinline__ void to(float top) {
    if (!(top > m)) return;
    const float low = fmaxf(m - top, kFarBelow);
    const double f = __builtin_amdgcn_exp2f(low * kLog2E);
    w = f * (w + (double)low * s);
    s *= f;
    m = top;
  }
  __device__ __forceinline__ void add(const f4 (&x)[kQuads]) {
    float part = 0.0f;
#pragma unroll
    for (int j = 0; j < kQuads; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float low = x[j][e] - m;
        const float p = __builtin_amdgcn_exp2f(low * kLog2E);
        s += (double)p;
        part = __builtin_fmaf(fmaxf(low, kFarBelow), p, part);
      }
    w += (double)part;
  }
};

// A lane's value as the lane 8, 4, 2 or 1 further on in a row of 16 has it, or 16 or 32 lanes
// away.
template <int kCtrl>
__device__ __forceinline__ int in_row(int x) {
  return __builtin_amdgcn_update_dpp(0, x, kCtrl, 0xf, 0xf, false);
}
template <int kOff>
__device__ __forceinline__ int across(int x) {
  if constexpr (kOff == 8) return in_row<0x128>(x);
  else if constexpr (kOff == 4) return in_row<0x124>(x);
  else if constexpr (kOff == 2) return in_row<0x122>(x);
  else if constexpr (kOff == 1) return in_row<0x121>(x);
  else return __shfl_xor(x, kOff, 64);
}
template <int kOff>
__device__ __forceinline__ float across(float x) {
  return __builtin_bit_cast(float, across<kOff>(__builtin_bit_cast(int, x)));
}
template <int kOff>
__device__ __forceinline__ double across(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = (uint32_t)across<kOff>((int)(uint32_t)u);
  const uint32_t hi = (uint32_t)across<kOff>((int)(uint32_t)(u >> 32));
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// Without the instruction that fmaxf has the compiler quiet a NaN by, which no caller has.
__device__ __forceinline__ float max_of(float a, float b) {
  return __builtin_amdgcn_fmed3f(a, b, __builtin_inff());
}
__device__ __forceinline__ float max_of_16(float g) {
  g = max_of(g, across<8>(g));
  g = max_of(g, across<4>(g));
  g = max_of(g, across<2>(g));
  return max_of(g, across<1>(g));
}
__device__ __forceinline__ float max_of_64(float g) {
  g = max_of(g, across<32>(g));
  return max_of_16(max_of(g, across<16>(g)));
}
__device__ __forceinline__ double sum_of_64(double v) {
  v += across<32>(v);
  v += across<16>(v);
  v += across<8>(v);
  v += across<4>(v);
  v += across<2>(v);
  return v + across<1>(v);
}

__device__ __forceinline__ void store_device(float* p, float v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float load_device(const float* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

struct Args {
  const float* x;
  int rows;
  int64_t n;
  int chunks, span, pieces;  // of a row; chunks of a piece
  float inv_temp;  // 1: the logits as they are
  const int32_t* tokens;
  int given;
  float* logprobs;
  float* entropy;
  int top_n;                 // at most n
  int32_t* top_ids;
  float* top_logprobs;
  float* maxima;             // [row][pieces] x the piece's, where there are alternatives
  Piece* stats;              // [row][pieces]
  Divisor by_piece;          // places of a piece's maxima
  uint32_t* counters;        // [row] x kCounterStride, where there is more than one piece
};

__device__ __forceinline__ float scaled(const Args& a, float v) {
  return scaled_logit(v, a.inv_temp);
}

// A thread's values of a chunk; past the row -Inf.
__device__ __forceinline__ void load_chunk(const Args& a, const float* row, int c,
                                           f4 (&t)[kQuads]) {
  const int64_t b = (int64_t)c * kChunk;
  if (b + kChunk <= a.n) {
#pragma unroll
    for (int j = 0; j < kQuads; ++j)
      t[j] = *reinterpret_cast<const f4*>(row + b + kValues * (int)threadIdx.x + 4 * j);
    return;
  }
#pragma unroll
  for (int j = 0; j < kQuads; ++j) {
    const int64_t i = b + kValues * (int)threadIdx.x + 4 * j;
#pragma unroll
    for (int e = 0; e < 4; ++e) t[j][e] = i + e < a.n ? row[i + e] : -__builtin_inff();
  }
}

// A row's maximum, log S and entropy, in every thread.
struct RowLog {
  float max;
  double log_sum, entropy;
  bool uniform;  // no distribution: every token 1 / n
};

__device__ __forceinline__ float log_prob(const RowLog& row, float x) {
  return (float)((row.uniform ? 0.0 : (double)x - (double)row.max) - row.log_sum);
}

struct Scratch {
  float max[kThreads / 64];
  double sum[kThreads / 64], weighted[kThreads / 64];
  int arrived;
};

// The statistics of a row's pieces, two a lane in every wave.
struct Pieces {
  Piece p[2];

  __device__ __forceinline__ Pieces(const Args& a, int64_t r) {
    const float* st = reinterpret_cast<const float*>(a.stats + r * a.pieces);
    const int lane = threadIdx.x & 63;
    static_assert(kPiecesRow <= 128);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float* at = st + 4 * (lane + 64 * i);
      p[i] = Piece{-__builtin_inff(), 0.0f, 0.0f, 0.0f};
      if (lane + 64 * i < a.pieces)
        p[i] = Piece{load_device(at), load_device(at + 1), load_device(at + 2),
                     load_device(at + 3)};
    }
  }
};

__device__ __forceinline__ RowLog row_log(const Args& a, const Piece (&p)[2]) {
  RowLog row;
  row.max = max_of_64(fmaxf(p[0].max, p[1].max));
  row.uniform = !(row.max > -__builtin_inff() && row.max < __builtin_inff());
  double s = 0.0, w = 0.0;
  if (!row.uniform) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float low = fmaxf(p[i].max - row.max, kFarBelow);  // of no values: S and W are 0
      const double f = __builtin_amdgcn_exp2f(low * kLog2E);
      const double sum = (double)p[i].sum + p[i].rest;
      s += f * sum;
      w += f * (p[i].weighted + (double)low * sum);
    }
  }
  s = sum_of_64(s);
  w = sum_of_64(w);
  row.log_sum = log(row.uniform ? (double)a.n : s);
  row.entropy = row.uniform ? row.log_sum : row.log_sum - w / s;
  return row;
}

// Unsigned numbers in the order of the values, -0 as +0.
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// The k largest of the distinct keys key(0) .. key(count - 1) (0: none), sorted, to out; keys are
// made anew for each digit.
template <class F>
__device__ void select_of(int count, F key, int k, uint64_t* out, SelectLds& sm) {
  const int tid = threadIdx.x;
  const int past = (count + kThreads - 1) / kThreads * kThreads;  // the same for all threads
  uint64_t prefix = 0, mask = 0;
  int need = k;
  bool all = false;
  for (int shift = 56; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += kThreads) sm.hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < past; i += kThreads) {
      const uint64_t v = i < count ? key(i) : 0;
      count_bin(sm.hist, (uint32_t)(v >> shift) & 255u, v != 0 && (v & mask) == prefix);
    }
    __syncthreads();
    if (tid < 64) find_digit(sm, need);
    __syncthreads();
    if (shift == 56 && sm.total <= (uint32_t)k) {
      all = true;
      break;
    }
    need -= (int)sm.above;
    prefix |= (uint64_t)sm.digit << shift;
    mask |= (uint64_t)255u << shift;
    if ((uint32_t)(k - need) + sm.eq <= 256u) break;  // always so once the key is whole
    __syncthreads();  // the digit has been read
  }
  __syncthreads();
  if (tid == 0) sm.ncand = 0;
  for (int i = tid; i < 256; i += kThreads) sm.cand[i] = 0;
  __syncthreads();
#pragma unroll 4
  for (int i = tid; i < count; i += kThreads) {
    const uint64_t v = key(i);
    if (v != 0 && (all || v >= prefix)) sm.cand[atomicAdd(&sm.ncand, 1u)] = v;
  }
  __syncthreads();
  if (tid < 64) sort_candidates(sm, k, out);
  __syncthreads();
}

typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));

struct SelectMemory {
  f4 of_thread[kThreads / 4];  // the threads' largest maxima
  int list[kList];
  u64x2 cand[kCands / 2];  // 0 behind the last one of an odd number
  uint64_t top[kTopTokensMax];
  SelectLds sm;
  uint32_t listed, cands;
};

// The group behind place i of a row's maxima.  A piece has those of its steps one after the
// other, in blocks of kBlock steps: of each of 16 lane rows in turn the block's steps.
__device__ __forceinline__ int group_at(const Args& a, int i) {
  const int piece = (int)a.by_piece.of((uint32_t)i), in = i - piece * a.span * kChunkGroups;
  const int block = in / (kBlock * kChunkGroups), at = in - block * kBlock * kChunkGroups;
  const int first = piece * a.span + block * kBlock;  // the block's first chunk
  int past = (piece + 1) * a.span;
  past = past < a.chunks ? past : a.chunks;
  const int steps = past - first < kBlock ? past - first : kBlock;
  const int row = (int)(((float)at + 0.5f) * __builtin_amdgcn_rcpf((float)steps));
  return (first + at - row * steps) * kChunkGroups + row;
}

// The row's maxima as a thread has them: the first ones ahead, in registers.
struct Maxima {
  const float* at;
  int count;
  float held[kHeldMaxima];

  __device__ __forceinline__ Maxima(const Args& a, int64_t r)
      : at(a.maxima + r * a.chunks * kChunkGroups), count(a.chunks * kChunkGroups) {
#pragma unroll
    for (int e = 0; e < kHeldMaxima; ++e)
      held[e] = kThreads * e < count
                    ? load_device(at + min((int)threadIdx.x + kThreads * e, count - 1))
                    : -__builtin_inff();
  }
  // f(place, maximum) of the thread's.
  template <class F>
  __device__ __forceinline__ void each(F f) const {
#pragma unroll
    for (int e = 0; e < kHeldMaxima; ++e)
      if ((int)threadIdx.x + kThreads * e < count) f((int)threadIdx.x + kThreads * e, held[e]);
#pragma unroll 4
    for (int i = threadIdx.x + kThreads * kHeldMaxima; i < count; i += kThreads)
      f(i, load_device(at + i));
  }
};

// The largest bound, but for its lowest bits, that kk of the waves' 64 lanes' values reach.
template <int N>
__device__ __forceinline__ uint32_t reached_by(const uint32_t (&key)[N], int kk) {
  uint32_t bound = 0;
#pragma unroll
  for (int bit = 31; bit >= 15; --bit) {
    const uint32_t with = bound | 1u << bit;
    int reach = 0;
#pragma unroll
    for (int i = 0; i < N; ++i)
      reach += __builtin_popcountll(__builtin_amdgcn_ballot_w64(key[i] >= with));
    bound = reach >= kk ? with : bound;
  }
  return bound;
}

// A bound that the kk largest of the threads' maxima reach, or (all have some) of four threads'
// each; every wave for itself.
__device__ __forceinline__ uint32_t bound_of(const SelectMemory& mem, int kk, bool all) {
  const f4 mine = mem.of_thread[threadIdx.x & 63];
  if (all && kk <= 24) {
    const uint32_t key[1] = {ordered(max_of(max_of(mine.x, mine.y), max_of(mine.z, mine.w)))};
    return reached_by(key, kk);
  }
  const uint32_t key[4] = {ordered(mine.x), ordered(mine.y), ordered(mine.z), ordered(mine.w)};
  return reached_by(key, kk);
}

// f(i, the place in the list) for the items i < kItems that a wave's lanes have, bit i of `has`:
// one addition to the list's length for all.
template <int kItems, class F>
__device__ __forceinline__ void append(uint32_t* length, uint32_t has, F f) {
  uint64_t lanes[kItems];
  int all = 0;
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    lanes[i] = __builtin_amdgcn_ballot_w64(has >> i & 1);
    all += __builtin_popcountll(lanes[i]);
  }
  if (all == 0) return;
  uint32_t at = 0;
  if ((threadIdx.x & 63) == 0) at = atomicAdd(length, (uint32_t)all);
  at = (uint32_t)__builtin_amdgcn_readfirstlane((int)at);
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const uint32_t before = __builtin_amdgcn_mbcnt_hi(
        (uint32_t)(lanes[i] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)lanes[i], 0));
    if (has >> i & 1) f(i, at + before);
    at += (uint32_t)__builtin_popcountll(lanes[i]);
  }
}

// The keys of the row's top_n tokens into mem.top; every thread comes here.  A row without a
// distribution gives any.
__device__ __forceinline__ void select_tokens(const Args& a, int64_t r, const Maxima& maxima,
                                              SelectMemory& mem) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const float* x = a.x + r * a.n;
  const int kk = a.top_n;
  const uint32_t n = (uint32_t)a.n;
  auto value_at = [&](uint32_t i) { return scaled(a, x[i < n ? i : n - 1]); };
  // f(j, first ids, values), f_end() of the listed groups, four values a lane of some groups at
  // once; j < kAtOnce, not all of them where there are no more groups.
  constexpr int kAtOnce = 4, kPairs = 256 / kGroup;  // groups of a load
  constexpr int kApart = kPairs * (kThreads / 64);
  auto scan = [&](int listed, auto f, auto f_end) {
    for (int l0 = wave * kPairs; l0 < listed; l0 += kAtOnce * kApart) {
      uint32_t at[kAtOnce];
      f4 v[kAtOnce];
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        if (l0 + j * kApart >= listed) break;
        const int l = l0 + j * kApart + lane / (64 / kPairs);
        at[j] = n;
        if (l < listed)
          at[j] = (uint32_t)mem.list[l] * kGroup + (uint32_t)(lane % (64 / kPairs) * 4);
        v[j] = f4{};
        if (at[j] + 4 <= n)
          v[j] = *reinterpret_cast<const f4*>(x + at[j]);
        else if (at[j] < n)
#pragma unroll
          for (int e = 0; e < 3; ++e) v[j][e] = x[at[j] + e < n ? at[j] + e : n - 1];
      }
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        if (l0 + j * kApart >= listed) break;
        f(j, at[j], v[j]);
      }
      f_end(at, v);
    }
  };
  // As many groups as twice the tokens leave a bound between them; of fewer, every value is
  // looked at, the threads' largest first.
  const bool few = maxima.count < 2 * kk;
  float most = -__builtin_inff();
  int listed = (int)((n + kGroup - 1) / kGroup);
  if (few) {
    for (int j = tid; j < listed; j += kThreads) mem.list[j] = j;
    __syncthreads();
    scan(
        listed,
        [&](int, uint32_t at, f4& v) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (at + e < n) most = fmaxf(most, scaled(a, v[e]));
        },
        [](const uint32_t (&)[kAtOnce], const f4 (&)[kAtOnce]) {});
  } else {
    maxima.each([&](int, float v) { most = fmaxf(most, v); });
  }
  reinterpret_cast<float*>(mem.of_thread)[tid] = most;
  if (tid == 0) {
    mem.listed = 0;
    mem.cands = 0;
  }
  __syncthreads();
  const uint32_t bound = bound_of(mem, kk, !few && maxima.count >= kThreads);
  if (!few) {
    auto list = [&](uint32_t at, int i) {
      if (at < (uint32_t)kList) mem.list[at] = group_at(a, i);
    };
    uint32_t reach = 0;
#pragma unroll
    for (int e = 0; e < kHeldMaxima; ++e)
      reach |= (uint32_t)(tid + kThreads * e < maxima.count && ordered(maxima.held[e]) >= bound)
               << e;
    append<kHeldMaxima>(&mem.listed, reach,
                        [&](int e, uint32_t at) { list(at, tid + kThreads * e); });
    for (int i0 = kThreads * kHeldMaxima; i0 < maxima.count; i0 += kThreads) {
      const int i = i0 + tid;
      const bool in = i < maxima.count && ordered(load_device(maxima.at + i)) >= bound;
      append<1>(&mem.listed, in, [&](int, uint32_t at) { list(at, i); });
    }
    __syncthreads();
    listed = (int)mem.listed;
  }
  if (listed > kList) {  // ties: the kk groups of largest maximum, the lower ones first
    listed = kk < maxima.count ? kk : maxima.count;
    select_of(
        maxima.count,
        [&](int i) { return topk_key(load_device(maxima.at + i), (uint32_t)group_at(a, i)); },
        listed, mem.top, mem.sm);
    for (int j = tid; j < listed; j += kThreads) mem.list[j] = (int)~(uint32_t)mem.top[j];
    __syncthreads();
  }
  // The listed values that reach the bound are candidates, all kk winners among them.
  auto reaches = [&](uint32_t i, float v) { return i < n && ordered(v) >= bound; };
  uint64_t* cand = reinterpret_cast<uint64_t*>(mem.cand);
  uint32_t has = 0;  // of a lane's 4 kAtOnce values those that reach it
  scan(
      listed,
      [&](int j, uint32_t at, f4& v) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] = scaled(a, v[e]);
          has |= (uint32_t)reaches(at + e, v[e]) << (4 * j + e);
        }
      },
      [&](const uint32_t (&at)[kAtOnce], const f4 (&v)[kAtOnce]) {
        if (__ballot(has != 0) == 0) return;
        // The lanes' places among the wave's, one addition to the number of all.
        const int mine = __builtin_popcount(has);
        int upto = mine;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
          const int o = __shfl_up(upto, off, 64);
          if (lane >= off) upto += o;
        }
        uint32_t slot = 0;
        if (lane == 63) slot = atomicAdd(&mem.cands, (uint32_t)upto);
        slot = (uint32_t)__builtin_amdgcn_readlane((int)slot, 63) + (uint32_t)(upto - mine);
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {
          if (__ballot((has >> (4 * j) & 15) != 0) == 0) continue;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (has >> (4 * j + e) & 1) {
              if (slot < (uint32_t)kCands) cand[slot] = topk_key(v[j][e], at[j] + e);
              ++slot;
            }
        }
        has = 0;
      });
  __syncthreads();
  const int cands = (int)mem.cands;
  if (cands <= kCands) {
    if (tid == 0 && cands % 2 != 0) cand[cands] = 0;
    __syncthreads();
    // Four, two or one neighbouring threads count a candidate's larger ones.
    const int shift = cands <= kThreads / 4 ? 2 : cands <= kThreads / 2 ? 1 : 0;
    for (int c = tid >> shift; c < ((cands + 63) & ~63); c += kThreads) {
      const uint64_t mine = c < cands ? cand[c] : 0;
      int rank = 0;
#pragma unroll 4
      for (int j = tid & ((1 << shift) - 1); j < (cands + 1) / 2; j += 1 << shift) {
        const u64x2 other = mem.cand[j];
        rank += (other.x > mine) + (other.y > mine);
      }
      if (shift > 0) rank += __shfl_xor(rank, 1, 64);
      if (shift > 1) rank += __shfl_xor(rank, 2, 64);
      if (mine != 0 && rank < kk) mem.top[rank] = mine;
    }
    __syncthreads();
  } else {
    select_of(
        listed * kGroup,
        [&](int j) -> uint64_t {
          const uint32_t i = (uint32_t)mem.list[j / kGroup] * kGroup + (uint32_t)(j % kGroup);
          const float v = value_at(i);
          return reaches(i, v) ? topk_key(v, i) : 0;
        },
        kk, mem.top, mem.sm);
  }
}

template <bool kTop>
struct Memory {
  SelectMemory m;
};
template <>
struct Memory<false> {};

// A workgroup takes a row's chunks from piece * span on.  Workgroups go to the XCDs in turn: of
// eight rows together each has an XCD of its own, so that the last pieces to arrive, which
// come last in a row, are on all of them (on one: 1024 rows of 151936 in 16 pieces took 188 us
// with 20 alternatives).
template <bool kTop>
__global__ __launch_bounds__(kThreads) void logprobs_kernel(Args a) {
  __shared__ Scratch sc;
  __shared__ Memory<kTop> mem;
  const int first_row = (int)(blockIdx.x / (8u * (uint32_t)a.pieces)) * 8;
  const int in = (int)blockIdx.x - first_row * a.pieces;
  const int together = a.rows - first_row < 8 ? a.rows - first_row : 8, piece = in / together;
  const int64_t r = first_row + in - piece * together;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const float* row = a.x + r * a.n;
  const int first = piece * a.span;
  const int past = first + a.span < a.chunks ? first + a.span : a.chunks;
  float* maxima = a.maxima + (r * a.chunks + first) * kChunkGroups;
  Sums sums;
  float mine = 0.0f;  // of a block's maxima of this row of 16 lanes the lane's
  f4 t[kAhead][kQuads];
#pragma unroll
  for (int u = 0; u < kAhead; ++u)
    if (first + u < past) load_chunk(a, row, first + u, t[u]);
  for (int c0 = first; c0 < past; c0 += kAhead) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int c = c0 + u, step = (c - first) % kBlock;
      if (c >= past) break;
      f4 v[kQuads];
      float top = -__builtin_inff();
#pragma unroll
      for (int j = 0; j < kQuads; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[j][e] = scaled(a, t[u][j][e]);
          top = fmaxf(top, v[j][e]);  // but for NaN
        }
      if constexpr (kTop) {
        const float g = max_of_16(top);
        mine = (tid & 15) == step ? g : mine;
      }
      if (c + kAhead < past) load_chunk(a, row, c + kAhead, t[u]);
      sums.to(top);
      sums.add(v);
      if constexpr (kTop) {
        const int steps = step + 1;
        if (steps == kBlock || c + 1 == past) {
          if ((tid & 15) < steps) store_device(maxima + tid / 16 * steps + (tid & 15), mine);
          maxima += kBlock * kChunkGroups;
        }
      }
    }
  }
  // The wave's, and then the workgroup's.
  sums.to(max_of_64(sums.m));
  sums.s = sum_of_64(sums.s);
  sums.w = sum_of_64(sums.w);
  if (lane == 0) {
    sc.max[wave] = sums.m;
    sc.sum[wave] = sums.s;
    sc.weighted[wave] = sums.w;
  }
  __syncthreads();
  if (tid == 0) {
#pragma unroll
    for (int w = 1; w < kThreads / 64; ++w) {
      Sums other;
      other.m = sc.max[w];
      other.s = sc.sum[w];
      other.w = sc.weighted[w];
      sums.to(other.m);
      other.to(sums.m);
      sums.s += other.s;
      sums.w += other.w;
    }
    const double s = sums.s;
    float* st = reinterpret_cast<float*>(a.stats + r * a.pieces + piece);
    store_device(st, s != s ? __builtin_inff() : s == 0.0 ? -__builtin_inff() : sums.m);
    store_device(st + 1, (float)s);
    store_device(st + 2, (float)(s - (double)(float)s));
    store_device(st + 3, (float)sums.w);
  }
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_s_waitcnt(0);  // what this wave wrote has passed its XCD's cache
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __syncthreads();
  if (a.pieces > 1) {
    if (tid == 0) {
      uint32_t* c = a.counters + r * kCounterStride;
      sc.arrived = (int)__hip_atomic_fetch_add(c, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (sc.arrived == a.pieces - 1)  // nobody else comes: zero again for the next launch
        __hip_atomic_store(c, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    if (sc.arrived != a.pieces - 1) return;
  }

  // The statistics and the first given token's logit are on their way during the selection.
  const Pieces pieces(a, r);
  const int32_t id = tid < a.given ? a.tokens[r * a.given + tid] : -1;
  const float logit = id >= 0 && id < a.n ? row[id] : 0.0f;
  if constexpr (kTop) {
    const Maxima all(a, r);
    select_tokens(a, r, all, mem.m);
  }
  const RowLog log = row_log(a, pieces.p);
  if (tid == 0 && a.entropy != nullptr) a.entropy[r] = (float)log.entropy;
  // An id outside the vocabulary has no probability.
  if (tid < a.given)
    a.logprobs[r * a.given + tid] =
        id >= 0 && id < a.n ? log_prob(log, scaled(a, logit)) : -__builtin_inff();
  for (int j = tid + kThreads; j < a.given; j += kThreads) {
    const int32_t other = a.tokens[r * a.given + j];
    a.logprobs[r * a.given + j] =
        other >= 0 && other < a.n ? log_prob(log, scaled(a, row[other])) : -__builtin_inff();
  }
  if constexpr (kTop) {
    for (int j = tid; j < a.top_n; j += kThreads) {
      const uint64_t key = mem.m.top[j];
      a.top_ids[r * a.top_n + j] = log.uniform ? j : (int32_t)~(uint32_t)key;
      a.top_logprobs[r * a.top_n + j] = log_prob(log, key_value(key));
    }
  }
}

// From this many rows on a row is one piece, fewer are cut into about kPiecesAll in all.  With 20
// alternatives: 512 rows of 32000 whole 22 us, cut in 8 26, 1024 of 151936 127 and (in 2) 137;
// 208 of 32000 in 5 pieces each 15.9, in 9 16.9.
constexpr int kRowsAlone = 512, kPiecesAll = 1024;

int span_of(int rows, int chunks) {
  if (rows >= kRowsAlone) return chunks;
  const int64_t all = ((int64_t)rows * chunks + kPiecesAll - 1) / kPiecesAll;
  const int64_t row = (chunks + kPiecesRow - 1) / kPiecesRow;
  const int64_t span = all > row ? all : row;
  return (int)(span < chunks ? span : chunks);
}

int chunks_of(int64_t n) { return (int)((n + kChunk - 1) / kChunk); }

}  // namespace

SplitKNeed token_logprobs_workspace(int rows, int64_t n, int top_n) {
  // No more pieces than this for these or smaller sizes: an odd number of each row.
  const int64_t chunks = chunks_of(n), all = rows * chunks;
  const int64_t most = rows + 2 * (kPiecesAll + (int64_t)kRowsAlone);
  SplitKNeed need;
  need.partial_floats = (size_t)most * 4 +
                        (top_n > 0 ? (size_t)all * kChunkGroups : 0);
  need.counters = (size_t)rows * kCounterStride;
  return need;
}

hipError_t launch_token_logprobs(const float* x, int rows, int64_t n, float temperature,
                                 const int32_t* tokens, int given, int top_n, float* logprobs,
                                 float* entropy, int32_t* top_ids, float* top_logprobs,
                                 const SplitKWorkspace& ws, hipStream_t stream) {
  if (rows <= 0 || rows > 65535 || n <= 0 || given < 0 || top_n < 0 || top_n > kTopTokensMax)
    return hipErrorInvalidValue;
  Args a{};
  a.x = x;
  a.rows = rows;
  a.n = n;
  a.chunks = chunks_of(n);
  a.span = span_of(rows, a.chunks);
  a.pieces = (a.chunks + a.span - 1) / a.span;
  // An odd number, so that the last ones of the rows are on all of an XCD's units too; one of
  // them may be empty.
  if (a.pieces > 1) a.pieces |= 1;
  a.inv_temp = temperature > 0.0f && temperature != 1.0f ? 1.0f / temperature : 1.0f;
  a.tokens = tokens;
  a.given = given;
  a.logprobs = logprobs;
  a.entropy = entropy;
  a.top_n = (int)(top_n < n ? top_n : n);
  a.top_ids = top_ids;
  a.top_logprobs = top_logprobs;
  a.stats = reinterpret_cast<Piece*>(ws.partials);
  a.maxima = ws.partials + (size_t)rows * a.pieces * 4;
  a.by_piece = Divisor((uint32_t)(a.span * kChunkGroups));
  a.counters = ws.counters;
  const dim3 grid((unsigned)rows * (unsigned)a.pieces), block(kThreads);
  if (a.top_n > 0)
    hipLaunchKernelGGL(logprobs_kernel<true>, grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL(logprobs_kernel<false>, grid, block, 0, stream, a);
  return hipGetLastError();
}

}  // namespace mle
