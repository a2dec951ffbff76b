// beams.cuh -- a beam search's step: the best continuations of each request, and the beams' states moved.
//
// select.  Request b has K beams (rows b K .. b K + K - 1 of the logits x [R, V]) with scores s.  With
//   lse_k = ln sum_v exp x[k, v]
// candidate (k, v) has the total s_k + (x[k, v] - lse_k); a finished beam has one candidate, its pad token
// with the total s_k.  The n best of a request come out in order, equal totals by k V + v.  A total of -inf
// (a masked token, an empty beam) is none; places left over have the score -inf, the pad token and
// the row b K + j mod K.  A NaN logit counts as -inf, +inf as its type's largest finite number; a NaN or +inf score as -inf.
//
// Which candidate comes first is an answer of whole numbers, so totals are compared in 64 bits and lse must
// be good to some 1e-7: what the rounding of the row's largest logit times log2 e moves is put right in the sum, sixteen values are added in fp32 and the rest in 64 bits.  Within a row
// the order is that of the logits themselves, which needs no exp.
//
// One pass over the logits, bound by HBM in principle.  A block holds a slice of one row in shared memory (2 to 16 16-byte
// pieces a thread), so maximum, sum and selection read it once.  Selection: each warp's t-th largest of its threads' maxima
// (8 t >= n) gives a bound that at least n elements reach and few more (37 of 32,768 for n = 16); those are ranked by
// counting.  Where many elements reach it (ties, a constant row) the n-th largest key is found by bisection of its
// bits and its equals are taken in the order of their index, which bounds the work for every row.  A second launch
// takes the best of a request's lists in the same way, or merges the lists where too many totals meet the bound.
// Measured (B200): 256 rows of 127,999 bf16 logits, n = 16, one in seven finished: 31.4 us, of which the slices 26 (the bytes need 8.5):
// loads, sums (8 special-function results a piece) and ranks follow one another in a block, and three blocks an SM do
// not cover them (8 pieces a thread 33 us, 512 threads 33, blocks that stay with the next slice on its way 49).  4 rows of
// 32,000: 8.2 us, two dependent launches of some ten dependent steps each.
//
// reorder.  Row r of each state becomes row parent[r], a row of the same request, as it was before the call.  A thread reads
// its 16 bytes of all the request's moving rows and then writes them: in place without a copy of the state, and
// rows that stay cost nothing.  384 rows of 135 KB, two thirds of them moving: 15.0 us, 4.6 TB/s by the bytes of the moving rows, 70 % of
// what a copy gets here.  Rows of one parent read it each for themselves (from L2 in part), and a thread has one piece in flight a row.
#pragma once

#include <cfloat>
#include <cmath>

#include "rope.cuh"

namespace specq {

constexpr int kSelThreads = 256;
constexpr int kSelMaxN = 128;
constexpr int kSelMaxBeams = 64;
constexpr int kSelBuf = 512;       // candidates of a slice that are ranked by counting
constexpr int kSelMaxPieces = 16;  // 16-byte pieces a thread: 64 KB of a row, three blocks an SM
constexpr uint32_t kKeyNone = 0x007FFFFFu;   // the key of -inf, which is no candidate

// Unsigned keys in the order of the floats (no NaN; -0 and +0 are one value).
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
__device__ __forceinline__ uint64_t order_key64(double x) {
  const uint64_t u = static_cast<uint64_t>(__double_as_longlong(x + 0.0));
  return u ^ (static_cast<uint64_t>(static_cast<int64_t>(u) >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ double key64_value(uint64_t k) {
  return __longlong_as_double(static_cast<int64_t>(k & 0x8000000000000000ull ? k ^ 0x8000000000000000ull : ~k));
}

// Two 16-bit logits, or one fp32 one, of a word: the larger of each; the same with NaN kept; and the words that
// the selection has in place of a NaN (-inf) and of +inf (the type's largest finite number).
template <typename T>
struct LogitWord;
template <>
struct LogitWord<float> {
  static __device__ __forceinline__ uint32_t max(uint32_t a, uint32_t b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }
  static __device__ __forceinline__ uint32_t max_nan(uint32_t a, uint32_t b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(__uint_as_float(a)), "f"(__uint_as_float(b)));
    return __float_as_uint(y);
  }
  static __device__ __forceinline__ float top(uint32_t w) { return __uint_as_float(w); }
  static __device__ __forceinline__ bool strange(uint32_t w) { return !(__uint_as_float(w) < INFINITY); }
  static __device__ __forceinline__ uint32_t plain(uint32_t w) {
    const float x = __uint_as_float(w);
    return __float_as_uint(fminf(fmaxf(x, -INFINITY), FLT_MAX));
  }
  static constexpr uint32_t kNone = 0xFF800000u;
};
template <>
struct LogitWord<__half> {
  static __device__ __forceinline__ __half2 h(uint32_t w) { return *reinterpret_cast<const __half2*>(&w); }
  static __device__ __forceinline__ uint32_t u(__half2 w) { return *reinterpret_cast<const uint32_t*>(&w); }
  static __device__ __forceinline__ uint32_t max(uint32_t a, uint32_t b) { return u(__hmax2(h(a), h(b))); }
  static __device__ __forceinline__ uint32_t max_nan(uint32_t a, uint32_t b) { return u(__hmax2_nan(h(a), h(b))); }
  static __device__ __forceinline__ float top(uint32_t w) { return fmaxf(__low2float(h(w)), __high2float(h(w))); }
  static __device__ __forceinline__ bool strange(uint32_t w) { return !(__low2float(h(w)) < INFINITY && __high2float(h(w)) < INFINITY); }
  static __device__ __forceinline__ uint32_t plain(uint32_t w) { return u(__hmin2(__hmax2(h(w), h(kNone)), h(0x7BFF7BFFu))); }
  static constexpr uint32_t kNone = 0xFC00FC00u;
};
template <>
struct LogitWord<__nv_bfloat16> {
  static __device__ __forceinline__ __nv_bfloat162 h(uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); }
  static __device__ __forceinline__ uint32_t u(__nv_bfloat162 w) { return *reinterpret_cast<const uint32_t*>(&w); }
  static __device__ __forceinline__ uint32_t max(uint32_t a, uint32_t b) { return u(__hmax2(h(a), h(b))); }
  static __device__ __forceinline__ uint32_t max_nan(uint32_t a, uint32_t b) { return u(__hmax2_nan(h(a), h(b))); }
  static __device__ __forceinline__ float top(uint32_t w) { return fmaxf(__low2float(h(w)), __high2float(h(w))); }
  static __device__ __forceinline__ bool strange(uint32_t w) { return !(__low2float(h(w)) < INFINITY && __high2float(h(w)) < INFINITY); }
  static __device__ __forceinline__ uint32_t plain(uint32_t w) { return u(__hmin2(__hmax2(h(w), h(kNone)), h(0x7F7F7F7Fu))); }
  static constexpr uint32_t kNone = 0xFF80FF80u;
};

// exp(x - top) of two logits added up: 2^(x c - top c), one rounding a term.  `shift` is fp32(top c); what its rounding moves is
// the same factor in every term, which shift_factor gives.  c is log2 e less 1.9e-8, so a term far below the top is off by 1.3e-8
// of its distance: in rows alike an error alike, beside which an order of beams is not lost.  (-inf goes through as 0.)
constexpr float kFarTop = 1024.f;      // above it the moved factor is no longer 1 + a little (and fp32(top c) may be infinite)
constexpr float kLog2eF = 1.44269502162933349609375f;
__device__ __forceinline__ void add_exp(float x, float y, float2 minus_shift, float2& sum) {
  const float2 t = __ffma2_rn(make_float2(x, y), make_float2(kLog2eF, kLog2eF), minus_shift);
  float2 e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(t.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(t.y));
  sum = __fadd2_rn(sum, e);
}
__device__ __forceinline__ double shift_factor(float top, float shift) {
  return 1.0 + 0.6931471805599453 * (static_cast<double>(shift) - static_cast<double>(top) * static_cast<double>(kLog2eF));
}

// exp(x) for |x| < 700, to 1e-9 of itself: 2^k times Taylor's sum of the rest (|r| <= ln 2 / 2, r^9 / 9! < 2.1e-10); in place of the
// library's, whose code is longer than all of the merge.
__device__ __forceinline__ double exp64(double x) {
  const double k = rint(x * 1.4426950408889634);
  const double r = fma(k, -0.6931471805599453, x);
  double y = 1.0 / 40320;
  y = fma(y, r, 1.0 / 5040);
  y = fma(y, r, 1.0 / 720);
  y = fma(y, r, 1.0 / 120);
  y = fma(y, r, 1.0 / 24);
  y = fma(y, r, 1.0 / 6);
  y = fma(y, r, 0.5);
  y = fma(y, r, 1.0);
  y = fma(y, r, 1.0);
  return __longlong_as_double(__double_as_longlong(y) + (static_cast<int64_t>(static_cast<int>(k)) << 52));
}
// ln(x), 1 <= x < 2^100: a Newton step for exp(y) = x from fp32's logarithm, which is good to 1e-6.
__device__ __forceinline__ double log64(double x) {
  const double y = static_cast<double>(__logf(static_cast<float>(x)));
  return y + (x * exp64(-y) - 1.0);
}

struct BeamSelectParams {
  const void* logits;     // [R, V], unit stride along V
  const float* scores;    // [R]
  const uint8_t* done;    // optional [R]
  float* part_max;        // workspace [R, S]
  double* part_sum;       // workspace [R, S]
  uint64_t* cand;         // workspace [R, S, n]: order key << 32 | ~index, best first, 0: none
  float* out_scores;      // [B, n]
  int32_t* out_parent;
  int32_t* out_token;
  int* status;
  int64_t ld;
  int K, V, n, S, slice, pieces, pad;
  uint32_t lists_inv, beams_inv;   // 2^32 / (K S) and / K, rounded up: exact quotients of a staged candidate's index
};

__device__ __forceinline__ bool beam_alive(float score) { return score > -INFINITY && score < INFINITY; }

// Sum over the block's 256 threads, to every thread.  red: 9 words of T.
template <typename T>
__device__ __forceinline__ T block_total(T v, T* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  T sum = red[0];
#pragma unroll
  for (int w = 1; w < kSelThreads / 32; ++w) sum += red[w];
  __syncthreads();
  return sum;
}

// Exclusive sum over the block's threads; *sum: the total.
__device__ __forceinline__ int block_before(int v, int* red, int* sum) {
  const int lane = static_cast<int>(threadIdx.x & 31), warp = static_cast<int>(threadIdx.x >> 5);
  int inc = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += up;
  }
  if (lane == 31) red[warp] = inc;
  __syncthreads();
  int base = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kSelThreads / 32; ++w) {
    if (w == warp) base = all;
    all += red[w];
  }
  __syncthreads();
  *sum = all;
  return base + inc - v;
}

template <typename T>
__global__ void __launch_bounds__(kSelThreads) beam_slice_kernel(const __grid_constant__ BeamSelectParams p) {
  constexpr int E = Row16<T>::N;
  using W = LogitWord<T>;
  extern __shared__ uint4 held[];                 // [pieces, threads]: a thread reads back its own pieces
  __shared__ uint64_t buf[kSelBuf];
  __shared__ uint32_t warp_top[kSelThreads / 32], warp_least[kSelThreads / 32];
  __shared__ int warp_with[kSelThreads / 32];
  __shared__ double redd[kSelThreads / 32];
  __shared__ int redi[kSelThreads / 32];
  __shared__ int found;
  pdl_launch_dependents();
  pdl_wait();
  const int row = blockIdx.y, s = blockIdx.x, tid = static_cast<int>(threadIdx.x), lane = tid & 31, warp = tid >> 5;
  if (!beam_alive(p.scores[row]) || (p.done != nullptr && p.done[row] != 0)) return;   // no logits are needed
  const T* x = static_cast<const T*>(p.logits) + static_cast<int64_t>(row) * p.ld;
  // pieces begin at the 16-byte boundary before the row: element 0 of the slice is index `first`, and the slices of a row
  // meet at first + slice
  const int shift = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T));
  const int first = s * p.slice - shift;
  const int NP = p.pieces;                        // even
  auto fetch = [&](int j, int i) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(held + j * kSelThreads + tid)), "l"(x + i) : "memory");
  };
  const bool whole = first >= 0 && first + p.slice <= p.V;
  if (whole) {
#pragma unroll 4
    for (int j = 0; j < NP / 2; ++j) fetch(j, first + (j * kSelThreads + tid) * E);
    asm volatile("cp.async.commit_group;" ::: "memory");
#pragma unroll 4
    for (int j = NP / 2; j < NP; ++j) fetch(j, first + (j * kSelThreads + tid) * E);
    asm volatile("cp.async.commit_group;" ::: "memory");
  } else {                                        // a row's ends: -inf outside, its cut pieces by elements
#pragma unroll 1
    for (int j = 0; j < NP; ++j) {
      const int i = first + (j * kSelThreads + tid) * E;
      if (i >= 0 && i + E <= p.V) fetch(j, i);
      else if (i >= p.V) held[j * kSelThreads + tid] = make_uint4(W::kNone, W::kNone, W::kNone, W::kNone);
    }
    const int last = (p.V - first) / E * E;       // the piece that the row's end cuts, if it does: two warps' lanes take the two
    const int at = tid < 32 ? lane : last + lane;
    if (lane < E && (tid < 32 ? first < 0 : tid < 64 && last < p.slice && first + last < p.V)) {
      const int i = first + at;
      reinterpret_cast<T*>(held)[at] = i >= 0 && i < p.V ? x[i] : f32_to_row<T>(-INFINITY);
    }
  }
  if (tid == 0) found = 0;
  // (loops over the pieces are not unrolled: the kernel is short against its code)
  float m = -INFINITY;
  uint32_t seen = W::kNone;
  auto top_of = [&](const uint4& u) { return W::top(W::max(W::max(u.x, u.y), W::max(u.z, u.w))); };
  auto look = [&](int j0, int j1) {
#pragma unroll 2
    for (int j = j0; j < j1; ++j) {
      const uint4 u = held[j * kSelThreads + tid];
      seen = W::max_nan(seen, W::max_nan(W::max_nan(u.x, u.y), W::max_nan(u.z, u.w)));
      m = fmaxf(m, top_of(u));
    }
  };
  if (whole) {
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    look(0, NP / 2);
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    look(NP / 2, NP);
  } else {
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    look(0, NP);
  }
  if (W::strange(seen)) {                         // rewritten once, by the only thread that reads them
    m = -INFINITY;
#pragma unroll 1
    for (int j = 0; j < NP; ++j) {
      uint4& u = held[j * kSelThreads + tid];
      u = make_uint4(W::plain(u.x), W::plain(u.y), W::plain(u.z), W::plain(u.w));
      m = fmaxf(m, top_of(u));
    }
  }
  const uint32_t mine = order_key(m);
  // Each warp's t-th largest of its threads' maxima (of those that have a candidate, if they are fewer): where the warps have n
  // of them together, n elements reach the least of these.
  const uint32_t with = __ballot_sync(0xffffffffu, mine > kKeyNone);
  auto bound_of = [&](int t) {
    uint32_t left = mine, at = 0xffffffffu;       // (a warp without candidates bounds nothing)
    for (int i = min(t, __popc(with)); i > 0; --i) {
      at = __reduce_max_sync(0xffffffffu, left);
      if (lane == __ffs(__ballot_sync(0xffffffffu, left == at)) - 1) left = 0;
    }
    if (lane == 0) warp_least[warp] = at;
  };
  int t = (p.n + kSelThreads / 32 - 1) / (kSelThreads / 32);
  bound_of(t);
  {
    const uint32_t top = __reduce_max_sync(0xffffffffu, mine);
    if (lane == 0) warp_top[warp] = top, warp_with[warp] = __popc(with);
  }
  __syncthreads();
  uint32_t best = 0, least = 0xffffffffu;
  int have = 0;
#pragma unroll
  for (int w = 0; w < kSelThreads / 32; ++w) {
    best = max(best, warp_top[w]);
    least = min(least, warp_least[w]);
    have += min(warp_with[w], t);
  }
  // A short row, or a short end of one: fewer warps give more each. (Bounded by the empty warps it collected all it had, and
  // ranked it: 8 beams of 362 symbols, 16 taken, 28 us against 12.7; 104 rows of 1299, 34 against 22.)
  if (have < p.n) {
    while (have < p.n && t < 32) {
      ++t;
      have = 0;
#pragma unroll
      for (int w = 0; w < kSelThreads / 32; ++w) have += min(warp_with[w], t);
    }
    __syncthreads();                              // everyone has read the first bounds
    if (have >= p.n) bound_of(t);
    __syncthreads();
    least = have >= p.n ? 0xffffffffu : 0u;
#pragma unroll
    for (int w = 0; w < kSelThreads / 32; ++w) least = min(least, warp_least[w]);
  }
  least = max(least, kKeyNone + 1);               // fewer than n threads with candidates: every one is taken
  const float row_max = key_value(best), bound = key_value(least);
  auto values = [&](int j, float (&v)[E]) {
    Row16<T> r;
    r.raw = held[j * kSelThreads + tid];
    r.get(v);
  };
  // the warp goes through the pieces of its threads that reach the bound, a lane half a piece
  if (best > kKeyNone) {
    static_assert(2 * kSelMaxPieces <= 32, "a lane for each half piece");
    constexpr int EH = E / 2;
    for (uint32_t todo = __ballot_sync(0xffffffffu, mine >= least); todo != 0u; todo &= todo - 1u) {
      const int from = warp * 32 + __ffs(todo) - 1;
      if (lane >= 2 * NP) continue;
      const int slot = (lane >> 1) * kSelThreads + from;
      const uint2 u = reinterpret_cast<const uint2*>(held + slot)[lane & 1];
      const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
      for (int k = 0; k < EH; ++k) {
        const float v = weight_to_f32<T>(e[k]);
        if (v >= bound) {
          const int at = atomicAdd(&found, 1);    // their order does not matter: they are ranked
          if (at < kSelBuf) buf[at] = static_cast<uint64_t>(order_key(v)) << 32 | static_cast<uint32_t>(~(first + slot * E + (lane & 1) * EH + k));
        }
      }
    }
  }
  double sum = 0.0;
  if (best > kKeyNone) {
    const float shift = row_max * kLog2eF;
    const float2 minus_shift = make_float2(-shift, -shift);
    const bool far = fabsf(row_max) > kFarTop;
#pragma unroll 1
    for (int j = 0; j < NP; j += 2) {             // two pieces in fp32, the rest in 64 bits
      float2 e = {0.f, 0.f};
      if (far) {
        for (int i = 0; i < 2; ++i) {
          float v[E];
          values(j + i, v);
#pragma unroll
          for (int k = 0; k < E; ++k) e.x += exp2f((v[k] - row_max) * kLog2eF);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float v[E];
          values(j + i, v);
#pragma unroll
          for (int k = 0; k < E; k += 2) add_exp(v[k], v[k + 1], minus_shift, e);
        }
      }
      sum += static_cast<double>(e.x + e.y);
    }
    if (!far) sum *= shift_factor(row_max, shift);
  }
  sum = block_total(sum, redd);                   // (its barriers publish buf and found)
  const int64_t list = static_cast<int64_t>(row) * p.S + s;
  if (tid == 0) {
    p.part_max[list] = best > kKeyNone ? row_max : -INFINITY;
    p.part_sum[list] = sum;
  }
  int total = found;
  if (total > kSelBuf) {
    auto count_from = [&](uint32_t key) {
      int c = 0;
#pragma unroll 1
      for (int j = 0; j < NP; ++j) {
        float v[E];
        values(j, v);
#pragma unroll
        for (int k = 0; k < E; ++k) c += order_key(v[k]) >= key;
      }
      return c;
    };
    auto put = [&](int at, uint32_t key, int j, int k) {
      buf[at] = static_cast<uint64_t>(key) << 32 | static_cast<uint32_t>(~(first + (j * kSelThreads + tid) * E + k));
    };
    // the n-th largest key: the largest one that at least n elements reach
    uint32_t lo = least, hi = best;
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo) / 2 + 1;
      if (block_total(mine >= mid ? count_from(mid) : 0, redi) >= p.n) lo = mid;
      else hi = mid - 1;
    }
    const int cnt = mine > lo ? count_from(lo + 1) : 0;     // fewer than n are above it
    int at = block_before(cnt, redi, &total);
    int left = p.n - total, next = total;         // its equals fill up, lowest index first
#pragma unroll 1
    for (int j = 0; j < NP; ++j) {
      float v[E];
      values(j, v);
      int same = 0;
#pragma unroll
      for (int k = 0; k < E; ++k) {
        const uint32_t key = order_key(v[k]);
        if (key > lo) put(at++, key, j, k);
        same += key == lo;
      }
      int all;
      int before = block_before(same, redi, &all);
#pragma unroll
      for (int k = 0; k < E; ++k)
        if (order_key(v[k]) == lo) {
          if (before < left) put(next + before, lo, j, k);
          ++before;
        }
      const int took = min(all, left);
      left -= took;
      next += took;
    }
    total = next;
    __syncthreads();
  }
  uint64_t* out = p.cand + list * p.n;
  for (int c = tid; c < total; c += kSelThreads) {
    const uint64_t me = buf[c];
    int ahead = 0;
#pragma unroll 4
    for (int o = 0; o < total; ++o) ahead += buf[o] > me;
    if (ahead < p.n) out[ahead] = me;
  }
  for (int c = total + tid; c < p.n; c += kSelThreads) out[c] = 0;
}

constexpr int kMergeThreads = 256;
constexpr int kMergeWarps = kMergeThreads / 32;
constexpr int kMergeRank = 256;         // candidates that are ranked by counting
constexpr int kMergeSmem = 96 * 1024;   // a request's candidates up to this size are staged in shared memory

struct Merged {                         // a candidate of a request
  uint64_t key;                         // order_key64 of its total; 0: none
  uint32_t at;                          // k V + v
};

// The lane with the first of the warp's candidates, or -1 when no lane has one.
__device__ __forceinline__ int warp_first(const Merged& mine) {
  const uint32_t hi = static_cast<uint32_t>(mine.key >> 32);
  const uint32_t mh = __reduce_max_sync(0xffffffffu, hi);
  if (mh == 0u) return -1;              // (the key of a finite total has a high word above 0)
  uint32_t who = __ballot_sync(0xffffffffu, hi == mh);
  if (who & (who - 1)) {
    const uint32_t lo = static_cast<uint32_t>(mine.key);
    const uint32_t ml = __reduce_max_sync(0xffffffffu, hi == mh ? lo : 0u);
    const bool tie = hi == mh && lo == ml;
    const uint32_t mi = __reduce_min_sync(0xffffffffu, tie ? mine.at : 0xffffffffu);
    who = __ballot_sync(0xffffffffu, tie && mine.at == mi);
  }
  return __ffs(who) - 1;
}

__global__ void __launch_bounds__(kMergeThreads) beam_merge_kernel(const __grid_constant__ BeamSelectParams p, int staged) {
  extern __shared__ __align__(16) uint8_t dyn[];   // staged: totals' keys [K, S, n] and places [K, S, n]; a position a list
  __shared__ double top[kSelMaxBeams];  // a beam's largest logit and the logarithm of its sum: their sum would round
  __shared__ double ln[kSelMaxBeams];   // the small one away beside logits of 1e16 and more
  __shared__ float score[kSelMaxBeams];
  __shared__ int mode[kSelMaxBeams];    // 0: has lists, 1: finished, 2: no candidate
  __shared__ Merged warp_list[kMergeWarps * kSelMaxN];
  __shared__ Merged final_list[kSelMaxN];
  __shared__ uint32_t warp_least[kMergeWarps];
  __shared__ int found;
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.x, tid = static_cast<int>(threadIdx.x), lane = tid & 31, warp = tid >> 5;
  const int lists = p.K * p.S, all = lists * p.n;
  uint64_t* keys = reinterpret_cast<uint64_t*>(dyn);
  uint32_t* places = reinterpret_cast<uint32_t*>(keys + all);
  int* pos = staged ? reinterpret_cast<int*>(places + all) : reinterpret_cast<int*>(dyn);
  const uint64_t* cand = p.cand + static_cast<int64_t>(b) * all;
  if (tid == 0) found = 0;
  if (staged) {                         // on their way while the sums are made
#pragma unroll 4
    for (int i = tid; i < all; i += kMergeThreads)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(keys + i)), "l"(cand + i) : "memory");
  }
  // a warp a beam: maximum and sum over its slices
  for (int k = warp; k < p.K; k += kMergeWarps) {
    const int row = b * p.K + k;
    const float sc = p.scores[row];
    int md = !beam_alive(sc) ? 2 : p.done != nullptr && p.done[row] != 0 ? 1 : 0;
    double l = 0.0;
    float m = -INFINITY;
    if (md == 0) {
      const float* pm = p.part_max + static_cast<int64_t>(row) * p.S;
      const double* ps = p.part_sum + static_cast<int64_t>(row) * p.S;
      float m0 = lane < p.S ? pm[lane] : -INFINITY;
      double s0 = lane < p.S ? ps[lane] : 0.0;
      m = m0;
      for (int s = lane + 32; s < p.S; s += 32) m = fmaxf(m, pm[s]);
      m = warp_max_f32(m);
      auto share = [&](float v, double sum) {    // below e^-100 it is nothing beside the largest one's
        const double d = static_cast<double>(v) - static_cast<double>(m);
        return d > -100.0 ? sum * exp64(d) : 0.0;
      };
      if (m > -INFINITY) {
        double sum = m0 > -INFINITY ? share(m0, s0) : 0.0;
        for (int s = lane + 32; s < p.S; s += 32)
          if (pm[s] > -INFINITY) sum += share(pm[s], ps[s]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        l = log64(sum);
      } else {
        md = 2;
      }
    }
    if (lane == 0) {
      top[k] = static_cast<double>(m);
      ln[k] = l;
      score[k] = sc;
      mode[k] = md;
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  // i / d by d's inverse
  auto div = [](int i, int d, uint32_t inv) { return d == 1 ? i : static_cast<int>(__umulhi(static_cast<uint32_t>(i), inv)); };
  // candidate i of list `list` of beam k
  auto total_of = [&](int k, bool first, uint64_t u) {
    Merged c = {0, 0xffffffffu};
    if (mode[k] == 1) {
      if (first) {
        c.key = order_key64(static_cast<double>(score[k]));
        c.at = static_cast<uint32_t>(k) * static_cast<uint32_t>(p.V) + static_cast<uint32_t>(p.pad);
      }
    } else if (mode[k] == 0 && u != 0) {
      c.key = order_key64(static_cast<double>(score[k]) + (static_cast<double>(key_value(static_cast<uint32_t>(u >> 32))) - top[k] - ln[k]));
      c.at = static_cast<uint32_t>(k) * static_cast<uint32_t>(p.V) + ~static_cast<uint32_t>(u);
    }
    return c;
  };
  bool ranked = false;
  if (staged) {
    // A thread takes its candidates in the order rank, slice, beam, so that each warp sees good ones of all beams.
    uint32_t high = 0;                        // the high word of this thread's best key
#pragma unroll 2
    for (int i = tid; i < all; i += kMergeThreads) {
      const int j = div(i, lists, p.lists_inv), list = i - j * lists, s = div(list, p.K, p.beams_inv), k = list - s * p.K;
      const int at = (k * p.S + s) * p.n + j;
      const Merged c = total_of(k, s == 0 && j == 0, keys[at]);
      keys[at] = c.key;
      places[at] = c.at;
      high = max(high, static_cast<uint32_t>(c.key >> 32));
    }
    // As in a slice: the t-th largest of its threads' bests of each of the `full` warps whose threads all have
    // candidates, t full >= n; n candidates reach the least of these.
    const int full = min(all / 32, kMergeWarps), t = full > 0 ? (p.n + full - 1) / full : 33;
    if (warp < full && t <= 32) {
      uint32_t left = high, at = 0;
      for (int i = 0; i < t; ++i) {
        at = __reduce_max_sync(0xffffffffu, left);
        if (lane == __ffs(__ballot_sync(0xffffffffu, left == at)) - 1) left = 0;
      }
      if (lane == 0) warp_least[warp] = at;
    }
    __syncthreads();
    uint32_t bound = t <= 32 ? 0xffffffffu : 0u;
    for (int w = 0; w < full && t <= 32; ++w) bound = min(bound, warp_least[w]);
    bound = max(bound, 1u);                   // none has the key 0
    if (high >= bound)
      for (int i = tid; i < all; i += kMergeThreads) {
        const int j = div(i, lists, p.lists_inv), list = i - j * lists, s = div(list, p.K, p.beams_inv), k = list - s * p.K;
        const int at = (k * p.S + s) * p.n + j;
        const uint64_t key = keys[at];
        if (static_cast<uint32_t>(key >> 32) < bound) continue;
        const int o = atomicAdd(&found, 1);
        if (o < kMergeRank) warp_list[o] = Merged{key, places[at]};
      }
    __syncthreads();
    const int total = found;
    if (total <= kMergeRank) {
      ranked = true;
      for (int j = total + tid; j < p.n; j += kMergeThreads) final_list[j] = Merged{0, 0xffffffffu};
      for (int c = tid; c < total; c += kMergeThreads) {
        const Merged me = warp_list[c];
        int ahead = 0;
#pragma unroll 4
        for (int o = 0; o < total; ++o) {
          const Merged x = warp_list[o];
          ahead += x.key > me.key || (x.key == me.key && x.at < me.at);
        }
        if (ahead < p.n) final_list[ahead] = me;
      }
    }
  }
  if (!ranked) {                              // very many candidates, or very many that meet the bound
    for (int i = tid; i < lists; i += kMergeThreads) pos[i] = 0;
    __syncthreads();
  }
  auto head = [&](int list) {
    const int i = pos[list];
    if (i >= p.n) return Merged{0, 0xffffffffu};
    if (staged) return Merged{keys[list * p.n + i], places[list * p.n + i]};
    const int k = list / p.S;
    return total_of(k, list == k * p.S && i == 0, cand[static_cast<int64_t>(list) * p.n + i]);
  };
  // a warp merges the lists from, from + step, ..., spread over its lanes
  auto merge = [&](int from, int step, Merged* out) {
    Merged mine;
    int which;
    auto look = [&]() {                       // the first of this lane's heads
      mine = Merged{0, 0xffffffffu};
      which = 0;
      for (int l = from + lane * step; l < lists; l += 32 * step) {
        const Merged c = head(l);
        if (c.key > mine.key || (c.key == mine.key && c.at < mine.at)) mine = c, which = l;
      }
    };
    look();
    int j = 0;
    for (; j < p.n; ++j) {
      const int who = warp_first(mine);
      if (who < 0) break;
      if (lane == who) {
        out[j] = mine;
        ++pos[which];
        look();
      }
      __syncwarp();
    }
    for (j += lane; j < p.n; j += 32) out[j] = Merged{0, 0xffffffffu};
  };
  if (!ranked) {
    merge(warp, kMergeWarps, warp_list + warp * kSelMaxN);
    __syncthreads();
    if (warp == 0) {
      int i = 0, j = 0;
      const Merged* mine_list = warp_list + lane * kSelMaxN;
      Merged mine = lane < kMergeWarps ? mine_list[0] : Merged{0, 0xffffffffu};
      for (; j < p.n; ++j) {
        const int who = warp_first(mine);
        if (who < 0) break;
        if (lane == who) {
          final_list[j] = mine;
          ++i;
          mine = i < p.n ? mine_list[i] : Merged{0, 0xffffffffu};
        }
      }
      for (j += lane; j < p.n; j += 32) final_list[j] = Merged{0, 0xffffffffu};
    }
  }
  __syncthreads();
  for (int j = tid; j < p.n; j += kMergeThreads) {
    const Merged c = final_list[j];
    const int64_t o = static_cast<int64_t>(b) * p.n + j;
    if (c.key == 0) {                         // a place without a candidate
      p.out_scores[o] = -INFINITY;
      p.out_parent[o] = b * p.K + j % p.K;
      p.out_token[o] = p.pad;
    } else {
      const uint32_t k = c.at / static_cast<uint32_t>(p.V);
      p.out_scores[o] = static_cast<float>(key64_value(c.key));
      p.out_parent[o] = b * p.K + static_cast<int>(k);
      p.out_token[o] = static_cast<int>(c.at - k * static_cast<uint32_t>(p.V));
    }
  }
}

// Pieces a thread takes of a row, elements a block, and blocks a row: the least of an SM's blocks * (pieces + what a block costs
// besides, about twenty pieces' time) and of the merge's work, a few of a block's pieces for each 256 candidates.
inline void beam_slices(int rows, int K, int V, int n, int elem, int sm_count, int* pieces, int* slice, int* S) {
  const int E = 16 / elem;
  double best = 0;
  *pieces = 0;
  for (int c = 2; c <= kSelMaxPieces; c += 2) {
    const int len = kSelThreads * E * c;
    const int64_t count = (static_cast<int64_t>(V) + E - 1 + len - 1) / len;   // a row may begin E - 1 elements into its first piece
    const double per_sm = std::max(1.0, static_cast<double>(rows) * static_cast<double>(count) / sm_count);
    const double cost = per_sm * (c + 20) + 2.0 * static_cast<double>(K) * static_cast<double>(count) * n / 256;
    if (*pieces == 0 || cost < best) {
      best = cost;
      *pieces = c;
      *slice = len;
      *S = static_cast<int>(count);
    }
  }
}

inline int beam_select_check(int B, int K, int V, int n, int dtype) {
  if (B < 0 || K < 1 || V < 1 || n < 1) return fail(SPECQ_ERR_INVALID_ARG, "beam_select: B=%d beams=%d V=%d n=%d", B, K, V, n);
  if (K > kSelMaxBeams || n > kSelMaxN)
    return fail(SPECQ_ERR_UNSUPPORTED, "beam_select: %d beams (at most %d), %d candidates (at most %d)", K, kSelMaxBeams, n, kSelMaxN);
  if (static_cast<int64_t>(K) * V >= 0x7fffffffll || V > 0x40000000 || static_cast<int64_t>(B) * K > 65535)
    return fail(SPECQ_ERR_UNSUPPORTED, "beam_select: %d x %d beams of %d tokens", B, K, V);
  if (dtype < 0 || dtype > 2) return fail(SPECQ_ERR_INVALID_ARG, "beam_select: dtype code %d", dtype);
  return SPECQ_OK;
}

inline int run_beam_select_workspace(int B, int K, int V, int n, int dtype, int64_t* bytes) {
  if (bytes == nullptr) return fail(SPECQ_ERR_INVALID_ARG, "beam_select_workspace: null pointer");
  if (int rc = beam_select_check(B, K, V, n, dtype)) return rc;
  DeviceState* dev = nullptr;
  if (int rc = get_device_state(&dev)) return rc;
  int pieces, slice, S;
  beam_slices(B * K, K, V, n, dtype == SPECQ_DTYPE_F32 ? 4 : 2, dev->sm_count, &pieces, &slice, &S);
  *bytes = static_cast<int64_t>(B) * K * S * (static_cast<int64_t>(n) * 8 + 8 + 4);
  return SPECQ_OK;
}

inline int run_beam_select(const void* logits, int64_t ld, int dtype, const float* scores, const uint8_t* done, int pad, float* out_scores,
                           int32_t* out_parent, int32_t* out_token, int B, int K, int V, int n, void* workspace, int64_t workspace_bytes,
                           void* stream) {
  if (int rc = beam_select_check(B, K, V, n, dtype)) return rc;
  if (pad < 0 || pad >= V) return fail(SPECQ_ERR_INVALID_ARG, "beam_select: pad %d is no token of %d", pad, V);
  if (B == 0) return SPECQ_OK;
  if (logits == nullptr || scores == nullptr || out_scores == nullptr || out_parent == nullptr || out_token == nullptr)
    return fail(SPECQ_ERR_INVALID_ARG, "beam_select: null pointer");
  if (B * K > 1 && ld < V) return fail(SPECQ_ERR_INVALID_ARG, "beam_select: rows of %d tokens %lld apart", V, static_cast<long long>(ld));
  int64_t need = 0;
  if (int rc = run_beam_select_workspace(B, K, V, n, dtype, &need)) return rc;
  if (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 16))
    return fail(SPECQ_ERR_INVALID_ARG, "beam_select: a workspace of %lld bytes is needed", static_cast<long long>(need));
  DeviceState* dev = nullptr;
  if (int rc = get_device_state(&dev)) return rc;
  BeamSelectParams p = {};
  beam_slices(B * K, K, V, n, dtype == SPECQ_DTYPE_F32 ? 4 : 2, dev->sm_count, &p.pieces, &p.slice, &p.S);
  const int64_t lists = static_cast<int64_t>(B) * K * p.S;
  p.logits = logits; p.ld = ld; p.scores = scores; p.done = done; p.status = dev->status;
  p.cand = static_cast<uint64_t*>(workspace);
  p.part_sum = reinterpret_cast<double*>(p.cand + lists * n);
  p.part_max = reinterpret_cast<float*>(p.part_sum + lists);
  p.out_scores = out_scores; p.out_parent = out_parent; p.out_token = out_token;
  p.K = K; p.V = V; p.n = n; p.pad = pad;
  // i (ceil(2^32 / d) d - 2^32) < i d < 2^32 for i below the number of staged candidates, 8192, and d up to 8192
  auto inverse = [](int64_t d) { return static_cast<uint32_t>((0x100000000ll + d - 1) / d); };
  p.lists_inv = inverse(static_cast<int64_t>(K) * p.S);
  p.beams_inv = inverse(K);
  const int64_t lists_b = static_cast<int64_t>(K) * p.S;
  const int staged = lists_b * n * 12 <= kMergeSmem ? 1 : 0;
  const int64_t smem = (staged ? lists_b * n * 12 : 0) + lists_b * 4;
  if (smem > dev->max_smem_optin - 32 * 1024) return fail(SPECQ_ERR_UNSUPPORTED, "beam_select: %d beams of %d tokens", K, V);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid(p.S, B * K), block(kSelThreads);
  const int held = p.pieces * kSelThreads * 16;
  auto launch = [&](auto kern) {
    cudaError_t e = ensure_dyn_smem(reinterpret_cast<const void*>(kern), kSelMaxPieces * kSelThreads * 16);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t c = {};
    c.gridDim = grid;
    c.blockDim = block;
    c.dynamicSmemBytes = static_cast<size_t>(held);
    c.stream = st;
    LaunchAttrs a(1);
    a.apply(c);
    return cudaLaunchKernelEx(&c, kern, p);
  };
  cudaError_t e;
  if (dtype == SPECQ_DTYPE_F16) e = launch(beam_slice_kernel<__half>);
  else if (dtype == SPECQ_DTYPE_F32) e = launch(beam_slice_kernel<float>);
  else e = launch(beam_slice_kernel<__nv_bfloat16>);
  SPECQ_CUDA_TRY(e);
  SPECQ_CUDA_TRY(ensure_dyn_smem(reinterpret_cast<const void*>(beam_merge_kernel), static_cast<int>(smem)));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(B);
  cfg.blockDim = dim3(kMergeThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = st;
  LaunchAttrs at(1);
  at.apply(cfg);
  SPECQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, beam_merge_kernel, p, staged));
  return SPECQ_OK;
}

// ---- reorder --------------------------------------------------------------------------------------
constexpr int kReorderThreads = 256;
constexpr int kReorderStates = 32;   // states of one launch

struct BeamReorderParams {
  uint8_t* ptr[kReorderStates];
  int64_t stride[kReorderStates];    // bytes between rows
  int64_t pieces[kReorderStates];    // of a row, `width` bytes each
  int first[kReorderStates + 1];     // the state's first block along x
  int width[kReorderStates];         // 16, 8, 4, 2 or 1
  const int32_t* parent;             // [R]
  int* status;
  int K, states;
};

template <typename U, int KMAX>
__device__ __forceinline__ void reorder_piece(const BeamReorderParams& p, int i, int64_t piece, const int* from, int row0) {
  uint8_t* base = p.ptr[i] + row0 * p.stride[i] + piece * static_cast<int64_t>(sizeof(U));
  U v[KMAX];
#pragma unroll
  for (int r = 0; r < KMAX; ++r)
    if (r < p.K && from[r] != r) v[r] = *reinterpret_cast<const U*>(base + from[r] * p.stride[i]);
#pragma unroll
  for (int r = 0; r < KMAX; ++r)
    if (r < p.K && from[r] != r) *reinterpret_cast<U*>(base + r * p.stride[i]) = v[r];
}

template <int KMAX>
__global__ void __launch_bounds__(kReorderThreads) beam_reorder_kernel(const __grid_constant__ BeamReorderParams p) {
  __shared__ int from[KMAX];
  pdl_launch_dependents();
  pdl_wait();
  const int row0 = blockIdx.y * p.K, tid = static_cast<int>(threadIdx.x);
  int moves = 0;
  if (tid < p.K) {
    const int w = p.parent[row0 + tid];
    int f = tid;
    if (w >= row0 && w < row0 + p.K) f = w - row0;
    else if (w >= 0) report_status(p.status, SPECQ_STATUS_BAD_INDEX);
    from[tid] = f;
    moves = f != tid;
  }
  if (!__syncthreads_or(moves)) return;
  int i = 0;
  while (i + 1 < p.states && static_cast<int>(blockIdx.x) >= p.first[i + 1]) ++i;
  const int64_t piece = static_cast<int64_t>(static_cast<int>(blockIdx.x) - p.first[i]) * kReorderThreads + tid;
  if (piece >= p.pieces[i]) return;
  switch (p.width[i]) {
    case 16: if constexpr (KMAX <= 32) reorder_piece<uint4, KMAX>(p, i, piece, from, row0); break;
    case 8: reorder_piece<uint2, KMAX>(p, i, piece, from, row0); break;
    case 4: reorder_piece<uint32_t, KMAX>(p, i, piece, from, row0); break;
    case 2: reorder_piece<uint16_t, KMAX>(p, i, piece, from, row0); break;
    default: reorder_piece<uint8_t, KMAX>(p, i, piece, from, row0); break;
  }
}

inline int run_beam_reorder(void* const* ptr, const int64_t* stride, const int64_t* row_bytes, int states, const int32_t* parent, int B,
                            int K, void* stream) {
  if (states < 0 || B < 0 || K < 1) return fail(SPECQ_ERR_INVALID_ARG, "beam_reorder: %d states, B=%d beams=%d", states, B, K);
  if (K > kSelMaxBeams || B > 65535) return fail(SPECQ_ERR_UNSUPPORTED, "beam_reorder: %d requests of %d beams (at most %d)", B, K, kSelMaxBeams);
  if (states == 0 || B == 0) return SPECQ_OK;
  if (ptr == nullptr || stride == nullptr || row_bytes == nullptr || parent == nullptr)
    return fail(SPECQ_ERR_INVALID_ARG, "beam_reorder: null pointer");
  for (int i = 0; i < states; ++i) {
    if (row_bytes[i] < 0 || (row_bytes[i] > 0 && ptr[i] == nullptr)) return fail(SPECQ_ERR_INVALID_ARG, "beam_reorder: state %d", i);
    if (B * static_cast<int64_t>(K) > 1 && stride[i] < row_bytes[i])
      return fail(SPECQ_ERR_INVALID_ARG, "beam_reorder: state %d has rows of %lld bytes %lld apart", i,
                  static_cast<long long>(row_bytes[i]), static_cast<long long>(stride[i]));
  }
  DeviceState* dev = nullptr;
  if (int rc = get_device_state(&dev)) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  for (int i0 = 0; i0 < states;) {
    BeamReorderParams p = {};
    p.parent = parent; p.status = dev->status; p.K = K;
    int64_t blocks = 0;
    for (; i0 < states && p.states < kReorderStates; ++i0) {
      if (row_bytes[i0] == 0) continue;
      int w = common_vec_width({reinterpret_cast<uint64_t>(ptr[i0]), static_cast<uint64_t>(stride[i0]), static_cast<uint64_t>(row_bytes[i0])});
      if (K > 32) w = std::min(w, 8);               // 64 rows of 16 bytes are more than a thread's registers
      const int64_t pieces = row_bytes[i0] / w, need = (pieces + kReorderThreads - 1) / kReorderThreads;
      if (need > 0x40000000ll) return fail(SPECQ_ERR_UNSUPPORTED, "beam_reorder: state %d has rows of %lld bytes", i0, static_cast<long long>(row_bytes[i0]));
      if (blocks + need > 0x7fffffffll) break;
      const int j = p.states++;
      p.ptr[j] = static_cast<uint8_t*>(ptr[i0]);
      p.stride[j] = stride[i0];
      p.width[j] = w;
      p.pieces[j] = pieces;
      p.first[j] = static_cast<int>(blocks);
      blocks += need;
      p.first[p.states] = static_cast<int>(blocks);
    }
    if (p.states == 0) continue;
    const dim3 grid(static_cast<unsigned>(blocks), B), block(kReorderThreads);
    cudaError_t e;
    if (K <= 4) e = launch_plain(beam_reorder_kernel<4>, grid, block, st, p);
    else if (K <= 8) e = launch_plain(beam_reorder_kernel<8>, grid, block, st, p);
    else if (K <= 16) e = launch_plain(beam_reorder_kernel<16>, grid, block, st, p);
    else if (K <= 32) e = launch_plain(beam_reorder_kernel<32>, grid, block, st, p);
    else e = launch_plain(beam_reorder_kernel<64>, grid, block, st, p);
    SPECQ_CUDA_TRY(e);
  }
  return SPECQ_OK;
}

}  // namespace specq
