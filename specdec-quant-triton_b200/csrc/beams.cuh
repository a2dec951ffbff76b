// beams.cuh -- a beam search's step: the best continuations of each request, and the beams' states moved.
//
// select.  Request b has K beams (rows b K .. b K + K - 1 of the logits x [R, V]) with scores s.  With
//   lse_k = ln sum_v exp x[k, v]
// candidate (k, v) has the total s_k + (x[k, v] - lse_k); a finished beam has one candidate, its pad token
// with the total s_k.  The n best of a request come out in order, equal totals by k V + v.  A total of -inf
// (a masked token, an empty beam) is none; places left over have the score -inf, the pad token and
// the row b K + j mod K.  A NaN logit counts as -inf, +inf as the largest finite number; a NaN or +inf score as -inf.
//
// Which candidate comes first is an answer of whole numbers, so totals are compared in 64 bits and lse must
// be good to some 1e-7: exp is made with the product by log2 e in two parts (the rounding of that product
// is the error that would not average out), eight values are added in fp32 and the rest in 64 bits.  Within a row
// the order is that of the logits themselves, which needs no exp.
//
// Bound by HBM: one pass over the logits.  A block holds a slice of one row in shared memory (8 or 2
// 16-byte pieces a thread, which only that thread reads back), so maximum, sum and selection read it once.  Selection: the n-th largest of the
// threads' maxima is a bound that at least n elements reach and few more; those are ranked by
// counting.  Where many elements reach it (ties, a constant row) the n-th largest key is found by bisection
// of its bits and its equals are taken in the order of their index, which bounds the work for every row.  A second
// launch merges a request's sorted lists, the best of the lists' heads at a time, by one warp up to 128
// lists, by eight and then one beyond.
//
// reorder.  Row r of each state becomes row parent[r], a row of the same request, as it was before the call.  A thread reads
// its 16 bytes of all the request's moving rows and then writes them: in place without a copy of the state, and
// rows that stay cost nothing.  Bound by HBM.
#pragma once

#include <cfloat>

#include "rope.cuh"

namespace specq {

constexpr int kSelThreads = 256;
constexpr int kSelMaxN = 128;
constexpr int kSelMaxBeams = 64;
constexpr int kSelBuf = 512;       // candidates of a slice that are ranked by counting
constexpr int kSelPieces = 8;      // 16-byte pieces a thread; kSelFewPieces where there are few rows
constexpr int kSelFewPieces = 2;
constexpr int kSelOneWarp = 128;   // lists that one warp merges
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

// A logit as the selection sees it: NaN is -inf, +inf the largest finite number.
__device__ __forceinline__ float plain_logit(float x) { return fminf(fmaxf(x, -INFINITY), FLT_MAX); }

// exp(d), d <= 0: 2^(d log2 e) with the product's low part kept.  log2 e = kLog2eHi + kLog2eLo to 2^-50.
__device__ __forceinline__ float exp_wide(float d) {
  constexpr float kLog2eHi = 1.44269502162933349609375f, kLog2eLo = 1.92596303e-8f, kLn2 = 0.693147182f;
  d = fmaxf(d, -200.f);             // exp(-200) is below fp32; -inf would make a NaN of the low part
  const float hi = d * kLog2eHi;
  const float lo = fmaf(d, kLog2eLo, fmaf(d, kLog2eHi, -hi));
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(hi));
  return fmaf(e, lo * kLn2, e);
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
  extern __shared__ uint4 held[];                 // [pieces, threads]: a thread reads back its own pieces
  __shared__ uint64_t buf[kSelBuf];
  __shared__ uint32_t top[kSelThreads];
  __shared__ double redd[kSelThreads / 32];
  __shared__ int redi[kSelThreads / 32];
  __shared__ uint32_t bound;
  pdl_launch_dependents();
  pdl_wait();
  const int row = blockIdx.y, s = blockIdx.x, tid = static_cast<int>(threadIdx.x);
  if (!beam_alive(p.scores[row]) || (p.done != nullptr && p.done[row] != 0)) return;   // no logits are needed
  const T* x = static_cast<const T*>(p.logits) + static_cast<int64_t>(row) * p.ld;
  // pieces begin at the 16-byte boundary before the row: element 0 of the slice is index `first`
  const int shift = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T));
  const int first = s * p.slice - shift;
  const int end = min(p.V, first + p.slice);      // the slices of a row meet at first + slice
  const int begin = max(first, 0);
  const int pieces = p.pieces;
#pragma unroll 4
  for (int j = 0; j < pieces; ++j) {
    const int i = first + (j * kSelThreads + tid) * E;
    uint4* to = held + j * kSelThreads + tid;
    if (i >= begin && i + E <= end) {
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(x + i) : "memory");
    } else {                                      // the row's ends, by elements; -inf outside
      T* e = reinterpret_cast<T*>(to);
#pragma unroll
      for (int k = 0; k < E; ++k) e[k] = i + k >= begin && i + k < end ? x[i + k] : f32_to_row<T>(-INFINITY);
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  auto piece = [&](int j, float (&v)[E]) {
    Row16<T> r;
    r.raw = held[j * kSelThreads + tid];
    r.get(v);
#pragma unroll
    for (int k = 0; k < E; ++k) v[k] = plain_logit(v[k]);
  };
  float m = -INFINITY;
#pragma unroll 2
  for (int j = 0; j < pieces; ++j) {
    float v[E];
    piece(j, v);
#pragma unroll
    for (int k = 0; k < E; ++k) m = fmaxf(m, v[k]);
  }
  const uint32_t mine = order_key(m);
  top[tid] = mine;
  if (tid == 0) bound = kKeyNone + 1;             // fewer than n threads with a candidate: every one is taken
  __syncthreads();
  // rank of this thread's maximum, equal ones by thread; the block's maximum on the way
  int rank = 0;
  uint32_t best = 0;
  for (int t = 0; t < kSelThreads; t += 4) {
    const uint4 u = *reinterpret_cast<const uint4*>(top + t);
    rank += (u.x > mine || (u.x == mine && t < tid)) + (u.y > mine || (u.y == mine && t + 1 < tid)) +
            (u.z > mine || (u.z == mine && t + 2 < tid)) + (u.w > mine || (u.w == mine && t + 3 < tid));
    best = max(best, max(max(u.x, u.y), max(u.z, u.w)));
  }
  if (rank == p.n - 1 && mine > kKeyNone) bound = mine;
  const float row_max = key_value(best);
  double sum = 0.0;
  if (best > kKeyNone) {
#pragma unroll 1
    for (int j = 0; j < pieces; ++j) {
      float v[E], e8 = 0.f;
      piece(j, v);
#pragma unroll
      for (int k = 0; k < E; ++k) e8 += exp_wide(v[k] - row_max);
      sum += static_cast<double>(e8);
    }
  }
  sum = block_total(sum, redd);                   // (its barriers publish `bound`)
  const int64_t list = static_cast<int64_t>(row) * p.S + s;
  if (tid == 0) {
    p.part_max[list] = best > kKeyNone ? row_max : -INFINITY;
    p.part_sum[list] = sum;
  }
  uint32_t least = bound;
  auto count_from = [&](uint32_t key) {
    int c = 0;
#pragma unroll 1
    for (int j = 0; j < pieces; ++j) {
      float v[E];
      piece(j, v);
#pragma unroll
      for (int k = 0; k < E; ++k) c += order_key(v[k]) >= key;
    }
    return c;
  };
  auto put = [&](int at, uint32_t key, int index) { buf[at] = static_cast<uint64_t>(key) << 32 | static_cast<uint32_t>(~index); };
  int cnt = mine >= least ? count_from(least) : 0, total;
  int at = block_before(cnt, redi, &total);
  if (total <= kSelBuf) {
    if (cnt > 0) {
#pragma unroll 1
      for (int j = 0; j < pieces; ++j) {
        float v[E];
        piece(j, v);
#pragma unroll
        for (int k = 0; k < E; ++k) {
          const uint32_t key = order_key(v[k]);
          if (key >= least) put(at++, key, first + (j * kSelThreads + tid) * E + k);
        }
      }
    }
  } else {
    // the n-th largest key: the largest one that at least n elements reach
    uint32_t lo = least, hi = best;
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo) / 2 + 1;
      if (block_total(mine >= mid ? count_from(mid) : 0, redi) >= p.n) lo = mid;
      else hi = mid - 1;
    }
    cnt = mine > lo ? count_from(lo + 1) : 0;     // fewer than n are above it
    at = block_before(cnt, redi, &total);
    int left = p.n - total, next = total;         // its equals fill up, lowest index first
#pragma unroll 1
    for (int j = 0; j < pieces; ++j) {
      float v[E];
      piece(j, v);
      int same = 0;
#pragma unroll
      for (int k = 0; k < E; ++k) {
        const uint32_t key = order_key(v[k]);
        if (key > lo) put(at++, key, first + (j * kSelThreads + tid) * E + k);
        same += key == lo;
      }
      int all;
      int before = block_before(same, redi, &all);
#pragma unroll
      for (int k = 0; k < E; ++k)
        if (order_key(v[k]) == lo) {
          if (before < left) put(next + before, lo, first + (j * kSelThreads + tid) * E + k);
          ++before;
        }
      const int took = min(all, left);
      left -= took;
      next += took;
    }
    total = next;
  }
  __syncthreads();
  uint64_t* out = p.cand + list * p.n;
  for (int c = tid; c < total; c += kSelThreads) {
    const uint64_t me = buf[c];
    int ahead = 0;
    for (int o = 0; o < total; ++o) ahead += buf[o] > me;
    if (ahead < p.n) out[ahead] = me;
  }
  for (int c = total + tid; c < p.n; c += kSelThreads) out[c] = 0;
}

constexpr int kMergeThreads = 256;
constexpr int kMergeSmem = 64 * 1024;   // candidates up to this size are staged in shared memory

struct Merged {                         // a candidate of a request
  uint64_t key;                         // order_key64 of its total; 0: none
  uint32_t at;                          // k V + v
  __device__ __forceinline__ bool before(const Merged& o) const { return key > o.key || (key == o.key && at < o.at); }
};

// The lane with the warp's first candidate, or -1 when no lane has one; *got: that candidate.
__device__ __forceinline__ int warp_first(const Merged& mine, Merged* got) {
  const uint32_t hi = static_cast<uint32_t>(mine.key >> 32), lo = static_cast<uint32_t>(mine.key);
  const uint32_t mh = __reduce_max_sync(0xffffffffu, hi);
  if (mh == 0u) return -1;              // (the key of a finite total has a high word above 0)
  const uint32_t ml = __reduce_max_sync(0xffffffffu, hi == mh ? lo : 0u);
  const bool tie = hi == mh && lo == ml;
  const uint32_t mi = __reduce_min_sync(0xffffffffu, tie ? mine.at : 0xffffffffu);
  got->key = static_cast<uint64_t>(mh) << 32 | ml;
  got->at = mi;
  return __ffs(__ballot_sync(0xffffffffu, tie && mine.at == mi)) - 1;
}

__global__ void __launch_bounds__(kMergeThreads) beam_merge_kernel(const __grid_constant__ BeamSelectParams p, int staged) {
  extern __shared__ uint64_t dyn[];     // staged candidates [K, S, n], then a position for each list
  __shared__ double top[kSelMaxBeams];  // a beam's largest logit and the logarithm of its sum: their sum would round
  __shared__ double ln[kSelMaxBeams];   // the small one away beside logits of 1e16 and more
  __shared__ float score[kSelMaxBeams];
  __shared__ int mode[kSelMaxBeams];    // 0: has lists, 1: finished, 2: no candidate
  __shared__ Merged warp_list[kMergeThreads / 32][kSelMaxN];
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.x, tid = static_cast<int>(threadIdx.x), lane = tid & 31, warp = tid >> 5;
  const int lists = p.K * p.S;
  uint64_t* staged_cand = dyn;
  int* pos = reinterpret_cast<int*>(dyn + (staged ? static_cast<int64_t>(lists) * p.n : 0));
  const uint64_t* cand = p.cand + static_cast<int64_t>(b) * lists * p.n;
  if (staged) {
    for (int i = tid; i < lists * p.n; i += kMergeThreads) staged_cand[i] = cand[i];
    cand = staged_cand;
  }
  for (int i = tid; i < lists; i += kMergeThreads) pos[i] = 0;
  // a warp a beam: maximum and sum over its slices
  for (int k = warp; k < p.K; k += kMergeThreads / 32) {
    const int row = b * p.K + k;
    const float sc = p.scores[row];
    int md = !beam_alive(sc) ? 2 : p.done != nullptr && p.done[row] != 0 ? 1 : 0;
    double l = 0.0;
    float m = -INFINITY;
    if (md == 0) {
      for (int s = lane; s < p.S; s += 32) m = fmaxf(m, p.part_max[static_cast<int64_t>(row) * p.S + s]);
      m = warp_max_f32(m);
      double sum = 0.0;
      if (m > -INFINITY)
        for (int s = lane; s < p.S; s += 32) {
          const float pm = p.part_max[static_cast<int64_t>(row) * p.S + s];
          if (pm > -INFINITY) sum += p.part_sum[static_cast<int64_t>(row) * p.S + s] * exp(static_cast<double>(pm) - static_cast<double>(m));
        }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (m > -INFINITY) l = log(sum);
      else md = 2;
    }
    if (lane == 0) {
      top[k] = static_cast<double>(m);
      ln[k] = l;
      score[k] = sc;
      mode[k] = md;
    }
  }
  __syncthreads();
  // the candidate at the head of a list
  auto head = [&](int list) {
    const int k = list / p.S, s = list - k * p.S, i = pos[list];
    Merged c = {0, 0xffffffffu};
    if (mode[k] == 1) {
      if (s == 0 && i == 0) {
        c.key = order_key64(static_cast<double>(score[k]));
        c.at = static_cast<uint32_t>(k) * static_cast<uint32_t>(p.V) + static_cast<uint32_t>(p.pad);
      }
    } else if (mode[k] == 0 && i < p.n) {
      const uint64_t u = cand[static_cast<int64_t>(list) * p.n + i];
      if (u != 0) {
        c.key = order_key64(static_cast<double>(score[k]) + (static_cast<double>(key_value(static_cast<uint32_t>(u >> 32))) - top[k] - ln[k]));
        c.at = static_cast<uint32_t>(k) * static_cast<uint32_t>(p.V) + ~static_cast<uint32_t>(u);
      }
    }
    return c;
  };
  auto emit = [&](int j, const Merged& c) {   // c.key 0: a place without a candidate
    const int64_t o = static_cast<int64_t>(b) * p.n + j;
    if (c.key == 0) {
      p.out_scores[o] = -INFINITY;
      p.out_parent[o] = b * p.K + j % p.K;
      p.out_token[o] = p.pad;
    } else {
      const uint32_t k = c.at / static_cast<uint32_t>(p.V);
      p.out_scores[o] = static_cast<float>(key64_value(c.key));
      p.out_parent[o] = b * p.K + static_cast<int>(k);
      p.out_token[o] = static_cast<int>(c.at - k * static_cast<uint32_t>(p.V));
    }
  };
  // a warp merges the lists warp0, warp0 + step, ... of its lanes
  auto merge = [&](int from, int step, auto use) {
    Merged mine = {0, 0xffffffffu};
    int which = -1;
    auto look = [&]() {                       // the first of this lane's heads
      mine.key = 0;
      mine.at = 0xffffffffu;
      for (int l = from + lane * step; l < lists; l += 32 * step) {
        const Merged c = head(l);
        if (c.before(mine)) mine = c, which = l;
      }
    };
    look();
    int j = 0;
    for (; j < p.n; ++j) {
      Merged got;
      const int who = warp_first(mine, &got);
      if (who < 0) break;
      if (lane == who) {
        use(j, got);
        ++pos[which];
        look();
      }
      __syncwarp();
    }
    const Merged no = {0, 0xffffffffu};
    for (j += lane; j < p.n; j += 32) use(j, no);
  };
  if (lists <= kSelOneWarp) {
    if (warp == 0) merge(0, 1, emit);
    return;
  }
  merge(warp, kMergeThreads / 32, [&](int j, const Merged& c) { warp_list[warp][j] = c; });
  __syncthreads();
  if (warp != 0) return;
  int i = 0;
  Merged mine = {0, 0xffffffffu};
  if (lane < kMergeThreads / 32) mine = warp_list[lane][0];
  for (int j = 0; j < p.n; ++j) {
    Merged got;
    const int who = warp_first(mine, &got);
    if (who < 0) {
      const Merged no = {0, 0xffffffffu};
      for (j += lane; j < p.n; j += 32) emit(j, no);
      return;
    }
    if (lane == who) {
      emit(j, got);
      ++i;
      mine = i < p.n ? warp_list[lane][i] : Merged{0, 0xffffffffu};
    }
  }
}

// Elements a block takes of a row, and blocks a row.  Small slices while the large ones leave SMs idle.
inline void beam_slices(int rows, int V, int elem, int sm_count, int* pieces, int* slice, int* S) {
  const int E = 16 / elem;
  *pieces = kSelPieces;
  *slice = kSelThreads * E * kSelPieces;
  // a row may begin E - 1 elements into its first piece
  auto count = [&] { return static_cast<int>((static_cast<int64_t>(V) + E - 1 + *slice - 1) / *slice); };
  if (static_cast<int64_t>(rows) * count() < 2 * sm_count) {
    *pieces = kSelFewPieces;
    *slice = kSelThreads * E * kSelFewPieces;
  }
  *S = count();
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
  beam_slices(B * K, V, dtype == SPECQ_DTYPE_F32 ? 4 : 2, dev->sm_count, &pieces, &slice, &S);
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
  beam_slices(B * K, V, dtype == SPECQ_DTYPE_F32 ? 4 : 2, dev->sm_count, &p.pieces, &p.slice, &p.S);
  const int64_t lists = static_cast<int64_t>(B) * K * p.S;
  p.logits = logits; p.ld = ld; p.scores = scores; p.done = done; p.status = dev->status;
  p.cand = static_cast<uint64_t*>(workspace);
  p.part_sum = reinterpret_cast<double*>(p.cand + lists * n);
  p.part_max = reinterpret_cast<float*>(p.part_sum + lists);
  p.out_scores = out_scores; p.out_parent = out_parent; p.out_token = out_token;
  p.K = K; p.V = V; p.n = n; p.pad = pad;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid(p.S, B * K), block(kSelThreads);
  const size_t held = static_cast<size_t>(p.pieces) * kSelThreads * 16;   // 32 KB at most, below the 48 that need no leave
  auto launch = [&](auto kern) {
    cudaLaunchConfig_t c = {};
    c.gridDim = grid;
    c.blockDim = block;
    c.dynamicSmemBytes = held;
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
  const int64_t lists_b = static_cast<int64_t>(K) * p.S;
  const int staged = lists_b * n * 8 <= kMergeSmem ? 1 : 0;
  const int64_t smem = (staged ? lists_b * n * 8 : 0) + lists_b * 4;
  if (smem > dev->max_smem_optin - 32 * 1024) return fail(SPECQ_ERR_UNSUPPORTED, "beam_select: %d beams of %d tokens", K, V);
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
