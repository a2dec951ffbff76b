// mass.cuh -- how much attention the cached tokens get: the column sums of the softmax over the
// block-scaled cache (block_cache.cuh), added to a running total.
//
// For sequence b and KV head h with G query heads, rows r = (new token i, head g), and token t's key k_t (8-bit
// numbers times their page's scale):
//   s_rt = q_r . k_t sm_scale,   lse_r = ln sum_t exp s_rt   over the tokens that row i sees
//   mass[b, h, t] <- decay mass[b, h, t] + sum_r exp(s_rt - lse_r)          for t < ctx_len[b]
// Row i of n stands at place ctx_len - n + i and sees the tokens up to it.  A row with a NaN or an infinity adds
// nothing, nor does a token of a page outside the cache get anything; a page of scale 0 gives scores of 0.
//
// The products run on the tensor cores, rows on M and tokens on N.  A warp takes 32 tokens at a time: each lane copies
// the bytes that the B fragments want in it to shared memory (asynchronously, 16 at a time; nobody else reads them), and
// widens them to fp16 in its registers, exactly; the order of the elements along D is free as long as q has the
// same.  q stands in shared memory as fp16 (bf16 rows times a power of two that brings their largest element to
// 2^14: exact down to 2^-31 of it).  A thread has two rows and eight tokens of a product, so a row's maximum and sum over
// 32 tokens and a token's sum over rows are nearly all its own.  Scores, maxima and sums are fp32; a score is the
// product times its scale, rounded once, before anything is taken off it.
//
// A column needs its rows' sums over all tokens first.  Where a cluster of up to 8 blocks of 512 tokens holds the whole
// table, the blocks exchange their maxima and sums through distributed shared memory and each key is read from
// HBM once; up to 16 rows the scores stay in registers, more rows' products are made again from the keys in shared
// memory.  For longer tables, and up to 16 rows where the SMs are busy anyway, a first launch leaves each block's maxima and
// sums (and, up to 16 rows, the scores: 8 bytes a row and token against D for reading the key again), and a later one
// takes the sums.  No atomics: a token's sum is made in a fixed order.
//
// Measured (B200, 8 KV heads of 128).  One row of 4 heads: 32 sequences of 1 to 8192 tokens 49 us (2.9 TB/s), 32 x 4096 51, one of
// 37 tokens 4.9: the bytes of the first two need some 22.  Their instructions (a tile of 32 tokens costs a warp some 450, 128 of them to
// widen bytes) are some 13 us of issue, 38 % of the time: two blocks an SM (registers) do not cover their waits, the blocks are 1.7 to 1.9
// turns of the machine, and 32 bytes of scores a token go to HBM and back beside 128 of key.  36 rows (9 of 4 heads), 8 x 4096: 44 us
// where the bytes need 5.5; 64 rows of the same: 52: each product is made twice, on the warp-level pipe, and each key widened twice.
// More rows' products are made on tcgen05 (mass_wide.cuh): made here, twice, at the warp-level pipe's 8.5 cycles each, those of
// 256 rows and two sequences of 12 to 16 thousand tokens took 55 of 163 us.
#pragma once

#include "block_cache.cuh"

namespace specq {

constexpr int kMassThreads = 256;
constexpr int kMassWarps = kMassThreads / 32;
constexpr int kMassTiles = 2;                // tiles of 32 tokens that a warp takes of a block's
constexpr int kMassChunk = 32 * kMassWarps * kMassTiles;   // tokens of a block
constexpr int kMassFew = 16;                 // rows of one product
constexpr int kMassWide = 96;                // rows from which the products go to tcgen05 (mass_wide.cuh)
constexpr int kMassRows = kMassWide;         // rows of q in shared memory where there are more than kMassFew
constexpr int kMassStages = 2;               // tiles of a warp on their way, up to 16 rows
constexpr int kMassCluster = 8;              // blocks that share their sums
constexpr int kMassSms = 148;                // how a call is cut does not ask the device: its workspace is known without one
constexpr float kLog2E = 1.44269504f;

struct MassParams {
  const void* q;           // [B, q_len, H, D]; q_sb = 0: packed rows
  const uint8_t* kc;
  const float* ks;
  const int32_t* bt;
  const int32_t* ctx;
  const int32_t* n_rows;   // optional [B]
  float* mass;             // [B, H_KV, N]
  float2* stats;           // workspace [B, H_KV, chunks, rows]: maximum (of score log2 e) and sum
  float* lse;              // workspace [B, H_KV, rows], log2 (more than 16 rows)
  float* score;            // workspace [B, H_KV, rows, chunks * chunk_tiles * 256], times log2 e (up to 16 rows)
  int* status;
  int64_t q_sb, q_st, q_sh, kv_sp, kv_so, kv_sh, s_sp, s_sh, bt_sb, m_sb, m_sh;
  int q_len, group, h_kv, page_log2, n_pages, bt_cols, chunks, rows;   // rows = q_len * group
  int chunk_tiles;         // a block's tokens in several launches, 256 each
  float sm_log2, decay;
};

enum MassMode { kMassStats = 0, kMassWeights = 1, kMassWhole = 2 };

template <int CT>   // four stored numbers to fp16, exactly, in order
__device__ __forceinline__ void widen4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (CT == 0) {          // 1024 + (byte ^ 0x80), less 1152
    const uint32_t x = w ^ 0x80808080u;
    const uint32_t a = __byte_perm(x, 0x64646464u, 0x4140), b = __byte_perm(x, 0x64646464u, 0x4342);
    const __half2 off = __half2(__half_raw{0x6480}, __half_raw{0x6480});
    const __half2 u = __hsub2(*reinterpret_cast<const __half2*>(&a), off), v = __hsub2(*reinterpret_cast<const __half2*>(&b), off);
    lo = *reinterpret_cast<const uint32_t*>(&u);
    hi = *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 u = __half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w & 0xFFFFu), __NV_E4M3));
    const __half2 v = __half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> 16), __NV_E4M3));
    lo = *reinterpret_cast<const uint32_t*>(&u);
    hi = *reinterpret_cast<const uint32_t*>(&v);
  }
}

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// What a bf16 row's halves times 2^k stand for: 2^-k, but no more than 2^80, so that the scores of rows past 2^94 stay within fp32 (a
// product of halves and keys is below 2^32).  Such a row's weight is on its largest score either way: its products are multiples of
// 2^-33, and 2^47 times the least scale that the append writes is beyond the reach of an exponential.
__device__ __forceinline__ float row_factor(int k) { return __int_as_float((127 + min(-k, 80)) << 23); }

// Two products, each rounded.  (Scalar ones: __fmul2_rn and mul.rn.f32x2 came out fused with the sums that they go into.)
__device__ __forceinline__ float2 mul2_rounded(float2 a, float2 b) { return make_float2(__fmul_rn(a.x, b.x), __fmul_rn(a.y, b.y)); }

template <int D, int ROWS>
struct MassSmem {
  static constexpr int kQStride = D + 8;     // halves: 16 more bytes a row put a quarter-warp's reads on all banks
  uint4 keys[kMassTiles][kMassWarps][D / 16][32];   // the 16-byte pieces of a lane: its token of eight, n-tile by n-tile
  __half q[ROWS * kQStride];
  float2 part[kMassWarps][ROWS];             // each warp's maximum and sum for a row
  float2 all[ROWS];                          // the block's
  float lse[ROWS];
  float factor[ROWS];
  int lim[ROWS];                             // the last token that a row sees; -1: none
};

__device__ __forceinline__ float2 join_stats(float2 a, float2 b) {
  const float m = fmaxf(a.x, b.x);
  if (m == -INFINITY) return make_float2(-INFINITY, 0.f);
  return make_float2(m, a.y * exp2_fast(a.x - m) + b.y * exp2_fast(b.x - m));
}
// log2 of a row's sum; +inf where it has none, so that exp2(s - lse) is 0
__device__ __forceinline__ float stats_lse(float2 x) { return x.y > 0.f ? x.x + log2f(x.y) : INFINITY; }

// What a sequence has: tokens (within its table) and counted rows; 0 rows: its mass stays.
__device__ __forceinline__ void mass_extent(const MassParams& p, int b, bool tell, int& n, int& nr) {
  n = p.ctx[b];
  const int most = p.bt_cols << p.page_log2;
  if (n > most) {
    if (tell) report_status(p.status, SPECQ_STATUS_PLAN_CLAMPED);
    n = most;
  }
  nr = n <= 0 ? 0 : p.n_rows == nullptr ? p.q_len : min(max(p.n_rows[b], 0), p.q_len);
}

// A sequence's rows of q of the KV head, padded with zeros to `pad`, to fp16 in shared memory; their factors and limits.
template <bool BF, int D, int ROWS, typename Smem>
__device__ __forceinline__ void mass_queries(const MassParams& p, Smem& sm, int b, int h, int rows, int pad, int base) {
  constexpr int kPieces = D / 8, kLanes = 2, kMine = D / kLanes;   // threads of a row, elements of each
  static_assert(ROWS * kLanes <= kMassThreads, "every row has its threads");
  const int tid = static_cast<int>(threadIdx.x);
  for (int i = tid; i < pad * kPieces; i += kMassThreads) {
    const int r = i / kPieces, c = i - r * kPieces;
    __half* dst = sm.q + r * Smem::kQStride + c * 8;
    if (r < rows) {
      const int row = r / p.group, head = h * p.group + r - row * p.group;
      const int64_t at = (p.q_sb != 0 ? b * p.q_sb + row * p.q_st : (static_cast<int64_t>(b) * p.q_len + row) * p.q_st) + head * p.q_sh;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(static_cast<const __half*>(p.q) + at + c * 8) : "memory");
    } else {
      *reinterpret_cast<uint4*>(dst) = make_uint4(0u, 0u, 0u, 0u);
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  const int r = tid / kLanes, lane = tid - r * kLanes;
  if (r < pad) {                       // (pad is a multiple of 16 rows: whole warps)
    uint4* at = reinterpret_cast<uint4*>(sm.q + r * Smem::kQStride + lane * kMine);
    uint32_t top = 0u;                 // the larger of the halves' magnitudes, a NaN kept
#pragma unroll
    for (int i = 0; i < kMine / 8; ++i) {
      const uint4 u = at[i];
      const uint32_t w[4] = {u.x & 0x7FFF7FFFu, u.y & 0x7FFF7FFFu, u.z & 0x7FFF7FFFu, u.w & 0x7FFF7FFFu};
#pragma unroll
      for (int k = 0; k < 4; ++k) top = __vmaxu2(top, w[k]);      // magnitudes order as integers, infinity and NaN last
    }
    top = max(top & 0xFFFFu, top >> 16);
#pragma unroll
    for (int o = 1; o < kLanes; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    const bool finite = top < (BF ? 0x7F80u : 0x7C00u);
    float factor = 1.f;
    if constexpr (BF) {
      const float amax = __uint_as_float(top << 16);
      // amax 2^k in [2^14, 2^15); 2^126 suffices for what is not zero beside any key
      const int k = top != 0u && finite ? min(14 - ilogbf(amax), 126) : 0;
      const float up = __int_as_float((127 + k) << 23);           // k >= 14 - 127
      factor = row_factor(k);
#pragma unroll
      for (int i = 0; i < kMine / 8; ++i) {
        uint4 u = at[i];
        uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const __half2 v = __floats2half2_rn(__uint_as_float(w[j] << 16) * up, __uint_as_float(w[j] & 0xFFFF0000u) * up);
          w[j] = finite ? *reinterpret_cast<const uint32_t*>(&v) : 0u;
        }
        at[i] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    } else if (!finite) {
#pragma unroll
      for (int i = 0; i < kMine / 8; ++i) at[i] = make_uint4(0u, 0u, 0u, 0u);
    }
    if (lane == 0) {
      sm.factor[r] = factor;
      sm.lim[r] = r < rows && finite ? base + r / p.group : -1;
    }
  }
  __syncthreads();
}

// The same for up to 16 rows in two steps, so that nothing waits between them: a 16-byte piece for each thread (asked for with the
// lengths), and later its row's factor and the piece in shared memory (the caller's barrier publishes them).
template <int D>
__device__ __forceinline__ uint4 few_queries_load(const MassParams& p, int b, int h) {
  const int r = static_cast<int>(threadIdx.x) / (D / 8), c = static_cast<int>(threadIdx.x) % (D / 8);
  if (r >= p.rows) return make_uint4(0u, 0u, 0u, 0u);
  const int row = r / p.group, head = h * p.group + r - row * p.group;
  const int64_t at = (p.q_sb != 0 ? b * p.q_sb + row * p.q_st : (static_cast<int64_t>(b) * p.q_len + row) * p.q_st) + head * p.q_sh;
  return *reinterpret_cast<const uint4*>(static_cast<const __half*>(p.q) + at + c * 8);
}
template <bool BF, int D, typename Smem>
__device__ __forceinline__ void few_queries_store(const MassParams& p, Smem& sm, uint4 u, int rows, int base) {
  constexpr int kLanes = D / 8;              // threads of a row
  const int r = static_cast<int>(threadIdx.x) / kLanes, c = static_cast<int>(threadIdx.x) % kLanes;
  uint32_t w[4] = {u.x, u.y, u.z, u.w}, top = 0u;   // the larger of the halves' magnitudes: infinity and NaN last
#pragma unroll
  for (int k = 0; k < 4; ++k) top = max(top, max(w[k] & 0x7FFFu, w[k] >> 16 & 0x7FFFu));
#pragma unroll
  for (int o = 1; o < kLanes; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  const bool counts = r < rows && top < (BF ? 0x7F80u : 0x7C00u);
  float factor = 1.f;
  if constexpr (BF) {
    // the largest element times 2^k in [2^14, 2^15); 2^126 suffices for what is not zero beside any key
    const int k = top != 0u && counts ? min(14 - ilogbf(__uint_as_float(top << 16)), 126) : 0;
    const float up = __int_as_float((127 + k) << 23);             // k >= 14 - 127
    factor = row_factor(k);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __half2 v = __floats2half2_rn(__uint_as_float(w[j] << 16) * up, __uint_as_float(w[j] & 0xFFFF0000u) * up);
      w[j] = *reinterpret_cast<const uint32_t*>(&v);
    }
  }
  if (r >= kMassFew) return;                 // (D = 64: half the threads have a piece)
  *reinterpret_cast<uint4*>(sm.q + r * Smem::kQStride + c * 8) = counts ? make_uint4(w[0], w[1], w[2], w[3]) : make_uint4(0u, 0u, 0u, 0u);
  if (c == 0) {
    sm.factor[r] = factor;
    sm.lim[r] = counts ? base + r / p.group : -1;
  }
}

template <bool BF, int CT, int D, int ROWS, int MODE>
__global__ void __launch_bounds__(kMassThreads, ROWS == kMassFew ? 3 : 2) mass_kernel(const __grid_constant__ MassParams p) {
  using Smem = MassSmem<D, ROWS>;
  constexpr bool kFew = ROWS == kMassFew;
  constexpr int C = D / 64;                  // 16-byte pieces of a lane's token
  extern __shared__ __align__(16) uint8_t raw_smem[];
  Smem& sm = *reinterpret_cast<Smem*>(raw_smem);
  pdl_launch_dependents();
  pdl_wait();
  const int chunk = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int lane = static_cast<int>(threadIdx.x & 31), warp = static_cast<int>(threadIdx.x >> 5);
  const int g = lane >> 2, tq = lane & 3;
  uint4 my_q = make_uint4(0u, 0u, 0u, 0u);
  if constexpr (kFew) my_q = few_queries_load<D>(p, b, h);
  int n, nr;
  mass_extent(p, b, chunk == 0 && h == 0 && threadIdx.x == 0 && MODE != kMassWeights, n, nr);
  // A block without tokens leaves; a cluster's barriers count only the threads that have not left, and no
  // block looks at the sums of one that has no tokens.
  if (nr == 0 || chunk * kMassChunk >= n) return;
  const int64_t bh = static_cast<int64_t>(b) * p.h_kv + h;

  // This warp's tiles: a page for each n-tile of eight tokens (a page holds eight or more), its scale, the lane's keys.
  int t0[kMassTiles];
  float tscale[kMassTiles][4];
  uint32_t bad[kMassTiles];                  // bit j: n-tile j is of no page
#pragma unroll
  for (int i = 0; i < kMassTiles; ++i) {
    t0[i] = chunk * kMassChunk + (i * kMassWarps + warp) * 32;
    bad[i] = 0u;
    int pg = -1;
    float sc = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int t = t0[i] + j * 8;
      uint4* dst = &sm.keys[i][warp][j * C][lane];
      if (j == 0 || (t & ((1 << p.page_log2) - 1)) == 0) {      // another page
        pg = -1;
        sc = 0.f;
        if (t < n) {
          pg = p.bt[b * p.bt_sb + (t >> p.page_log2)];
          if (pg < 0 || pg >= p.n_pages) {
            if (lane == 0) report_status(p.status, SPECQ_STATUS_BAD_INDEX);
            pg = -1;
          } else {
            sc = p.ks[pg * p.s_sp + h * p.s_sh] * p.sm_log2;
          }
        }
      }
      tscale[i][j] = pg < 0 ? 1.f : sc;
      if (pg < 0 || t >= n) bad[i] |= 1u << j;
      if (pg >= 0 && t + g < n) {
        const uint8_t* k = p.kc + pg * p.kv_sp + ((t + g) & ((1 << p.page_log2) - 1)) * p.kv_so + h * p.kv_sh + tq * 16;
#pragma unroll
        for (int c = 0; c < C; ++c)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst + c * 32)), "l"(k + c * 64) : "memory");
      } else {
#pragma unroll
        for (int c = 0; c < C; ++c) dst[c * 32] = make_uint4(0u, 0u, 0u, 0u);
      }
    }
  }
  const int base = n - nr, rows = nr * p.group;
  const int active = min((n - 1) / kMassChunk + 1, static_cast<int>(gridDim.x));   // of this sequence's blocks
  float weight[kMassTiles][4][2];            // of this thread's tokens, over its rows
#pragma unroll
  for (int i = 0; i < kMassTiles; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) weight[i][j][0] = weight[i][j][1] = 0.f;

  // Fragments of q for rows r0 + g and r0 + g + 8.
  auto fragments = [&](int r0, uint32_t (&a)[C][4][4]) {
    const __half* lo = sm.q + (r0 + g) * Smem::kQStride + tq * 16;
    const __half* hi = lo + 8 * Smem::kQStride;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int jj = 0; jj < 2; ++jj) {
        const uint4 u = *reinterpret_cast<const uint4*>(lo + c * 64 + jj * 8), v = *reinterpret_cast<const uint4*>(hi + c * 64 + jj * 8);
        a[c][2 * jj][0] = u.x; a[c][2 * jj][1] = v.x; a[c][2 * jj][2] = u.y; a[c][2 * jj][3] = v.y;
        a[c][2 * jj + 1][0] = u.z; a[c][2 * jj + 1][1] = v.z; a[c][2 * jj + 1][2] = u.w; a[c][2 * jj + 1][3] = v.w;
      }
  };
  auto widen = [&](int i, int j, uint32_t (&k)[C][4][2]) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const uint4 u = sm.keys[i][warp][j * C + c][lane];
      widen4<CT>(u.x, k[c][0][0], k[c][0][1]);
      widen4<CT>(u.y, k[c][1][0], k[c][1][1]);
      widen4<CT>(u.z, k[c][2][0], k[c][2][1]);
      widen4<CT>(u.w, k[c][3][0], k[c][3][1]);
    }
  };
  auto product = [&](const uint32_t (&a)[C][4][4], const uint32_t (&k)[C][4][2], float (&s)[4]) {
    s[0] = s[1] = s[2] = s[3] = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int jj = 0; jj < 4; ++jj) mma_f16(s, a[c][jj], k[c][jj][0], k[c][jj][1]);
  };
  // s: the products of rows r0 + g (0, 1) and r0 + g + 8 (2, 3) with tokens 8 j + 2 tq + 0, 1, made scores times log2 e.  They are
  // rounded once here: a maximum of rounded scores leaves its own score with the difference 0, whatever its size, where a fused
  // s x - max would leave what the rounding cut off (2^36 of 2^60).
  auto scale = [&](int i, int r0, float (&s)[4][4]) {
    const float f0 = BF ? sm.factor[r0 + g] : 1.f, f1 = BF ? sm.factor[r0 + g + 8] : 1.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float x = BF ? tscale[i][j] * f0 : tscale[i][j], y = BF ? tscale[i][j] * f1 : tscale[i][j];
      const float2 u = mul2_rounded(make_float2(s[j][0], s[j][1]), make_float2(x, x)), v = mul2_rounded(make_float2(s[j][2], s[j][3]), make_float2(y, y));
      s[j][0] = u.x;
      s[j][1] = u.y;
      s[j][2] = v.x;
      s[j][3] = v.y;
    }
  };
  // s becomes -inf where a row does not see a token: after the scaling, since a scale of 0 (or a product of small ones that leaves
  // fp32) times -inf is NaN
  auto hide = [&](int i, int r0, float (&s)[4][4]) {
    if (bad[i] == 0u && t0[i] + 31 <= base) return;
    const int l0 = sm.lim[r0 + g], l1 = sm.lim[r0 + g + 8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int t = bad[i] >> j & 1u ? INT_MAX - 1 : t0[i] + j * 8 + 2 * tq;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if (t + e > l0) s[j][e] = -INFINITY;
        if (t + e > l1) s[j][2 + e] = -INFINITY;
      }
    }
  };
  // a row's maximum and sum over this thread's eight tokens, then over the quad's 32
  auto row_stats = [&](const float (&s)[4][4], int e) {
    float m = fmaxf(s[0][e], s[0][e + 1]);
#pragma unroll
    for (int j = 1; j < 4; ++j) m = fmaxf(m, fmaxf(s[j][e], s[j][e + 1]));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
    const float z = m == -INFINITY ? 0.f : -m;
    float2 l = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 d = __fadd2_rn(make_float2(s[j][e], s[j][e + 1]), make_float2(z, z));
      l = __fadd2_rn(l, make_float2(exp2_fast(d.x), exp2_fast(d.y)));
    }
    float sum = l.x + l.y;
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    return make_float2(m, sum);
  };
  auto add_weights = [&](int i, int r0, const float (&s)[4][4]) {
    const float l0 = -sm.lse[r0 + g], l1 = -sm.lse[r0 + g + 8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 u = __fadd2_rn(make_float2(s[j][0], s[j][1]), make_float2(l0, l0));
      const float2 v = __fadd2_rn(make_float2(s[j][2], s[j][3]), make_float2(l1, l1));
      const float2 w = __fadd2_rn(__fadd2_rn(make_float2(weight[i][j][0], weight[i][j][1]), make_float2(exp2_fast(u.x), exp2_fast(u.y))),
                                  make_float2(exp2_fast(v.x), exp2_fast(v.y)));
      weight[i][j][0] = w.x;
      weight[i][j][1] = w.y;
    }
  };
  // the warps' sums to the block's, and (a cluster) the blocks' to lse
  auto block_stats = [&](int pad) {
    __syncthreads();
    for (int r = threadIdx.x; r < pad; r += kMassThreads) {
      float2 x = make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int w = 0; w < kMassWarps; ++w) x = join_stats(x, sm.part[w][r]);
      if (sm.lim[r] < 0) x = make_float2(-INFINITY, 0.f);
      if (MODE == kMassStats) {
        if (r < rows) p.stats[(bh * p.chunks + chunk) * p.rows + r] = x;
      } else {
        sm.all[r] = x;
      }
    }
    if (MODE != kMassWhole) return;
    if (active == 1) {
      __syncthreads();
      for (int r = threadIdx.x; r < pad; r += kMassThreads) sm.lse[r] = stats_lse(sm.all[r]);
    } else {
      cluster_sync();
      for (int r = threadIdx.x; r < pad; r += kMassThreads) {
        const uint32_t mine = smem_u32(&sm.all[r]);
        float2 x = make_float2(-INFINITY, 0.f);
#pragma unroll 4
        for (int c = 0; c < active; ++c) {
          const uint32_t at = dsmem_map(mine, static_cast<uint32_t>(c));
          x = join_stats(x, make_float2(dsmem_ld_f32(at), dsmem_ld_f32(at + 4)));
        }
        sm.lse[r] = stats_lse(x);
      }
      __syncthreads();
      cluster_arrive();                       // this block has read its peers' sums (waited for at the end)
      return;
    }
    __syncthreads();
  };

  if constexpr (kFew) {
    few_queries_store<BF, D>(p, sm, my_q, rows, base);
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    const bool half = rows <= 8;              // rows 8 to 15 are padding
    float s[kMassTiles][4][4];
    if (t0[0] < n) {                          // (a warp's first tile is the one that has tokens if any has)
      uint32_t a[C][4][4];
      fragments(0, a);
#pragma unroll
      for (int i = 0; i < kMassTiles; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t k[C][4][2];
          widen(i, j, k);
          product(a, k, s[i][j]);
        }
        scale(i, 0, s[i]);
        hide(i, 0, s[i]);
      }
    }
    // a quad's largest score of rows g and g + 8, -inf where they see none of its tokens (their factor is then 0, however small the
    // rows' sums are); the scores become 2^(s - top)
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
      float2 x = make_float2(-INFINITY, 0.f);
      if (t0[0] < n && !(half && e == 2)) {
#pragma unroll
        for (int i = 0; i < kMassTiles; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) x.x = fmaxf(x.x, fmaxf(s[i][j][e], s[i][j][e + 1]));
        x.x = fmaxf(x.x, __shfl_xor_sync(0xffffffffu, x.x, 1));
        x.x = fmaxf(x.x, __shfl_xor_sync(0xffffffffu, x.x, 2));
        const float z = x.x == -INFINITY ? 0.f : x.x;
        top[e / 2] = x.x;
#pragma unroll
        for (int i = 0; i < kMassTiles; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float u = exp2_fast(s[i][j][e] - z), v = exp2_fast(s[i][j][e + 1] - z);
            x.y += u + v;
            s[i][j][e] = u;
            s[i][j][e + 1] = v;
          }
        x.y += __shfl_xor_sync(0xffffffffu, x.y, 1);
        x.y += __shfl_xor_sync(0xffffffffu, x.y, 2);
      }
      if (tq == 0) sm.part[warp][g + 4 * e] = x;
    }
    block_stats(kMassFew);
    {
      if (t0[0] < n) {
        const float f0 = exp2_fast(top[0] - sm.lse[g]), f1 = exp2_fast(top[1] - sm.lse[g + 8]);
#pragma unroll
        for (int i = 0; i < kMassTiles; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) weight[i][j][e] = half ? s[i][j][e] * f0 : fmaf(s[i][j][2 + e], f1, s[i][j][e] * f0);
      }
    }
  } else {
    const int pad = (rows + 15) & ~15;
    mass_queries<BF, D, ROWS>(p, sm, b, h, rows, pad, base);
    if constexpr (MODE == kMassWeights) {
      for (int r = threadIdx.x; r < pad; r += kMassThreads) sm.lse[r] = r < rows ? p.lse[bh * p.rows + r] : INFINITY;
      __syncthreads();
    } else {
#pragma unroll
      for (int i = 0; i < kMassTiles; ++i) {
        uint32_t k[4][C][4][2];
#pragma unroll
        for (int j = 0; j < 4; ++j) widen(i, j, k[j]);
#pragma unroll 1
        for (int r0 = 0; r0 < pad; r0 += 16) {
          asm volatile("" : "+r"(r0));         // addresses from r0 alone: a pointer each for q, factors, limits and sums spilled (36 rows 49 us)
          uint32_t a[C][4][4];
          float s[4][4];
          fragments(r0, a);
#pragma unroll
          for (int j = 0; j < 4; ++j) product(a, k[j], s[j]);
          scale(i, r0, s);
          hide(i, r0, s);
          const float2 u = row_stats(s, 0), v = row_stats(s, 2);
          if (tq == 0) {
            float2* at = &sm.part[warp][r0 + g];
            at[0] = i == 0 ? u : join_stats(at[0], u);
            at[8] = i == 0 ? v : join_stats(at[8], v);
          }
        }
      }
      block_stats(pad);
    }
    if constexpr (MODE != kMassStats) {
#pragma unroll
      for (int i = 0; i < kMassTiles; ++i) {
        uint32_t k[4][C][4][2];
#pragma unroll
        for (int j = 0; j < 4; ++j) widen(i, j, k[j]);
#pragma unroll 1
        for (int r0 = 0; r0 < pad; r0 += 16) {
          asm volatile("" : "+r"(r0));
          uint32_t a[C][4][4];
          float s[4][4];
          fragments(r0, a);
#pragma unroll
          for (int j = 0; j < 4; ++j) product(a, k[j], s[j]);
          scale(i, r0, s);
          hide(i, r0, s);
          add_weights(i, r0, s);
        }
      }
    }
  }
  if constexpr (MODE != kMassStats) {
    // Eight tokens' sums over the eight lanes of a column, halving: lane g keeps token 8 (g >> 1) + 2 tq + (g & 1).
#pragma unroll
    for (int i = 0; i < kMassTiles; ++i) {
      if (t0[i] >= n) continue;
      float u[4], v[2];
#pragma unroll
      for (int j = 0; j < 4; ++j) {           // e by bit 0 of g
        const bool odd = g & 1;
        u[j] = (odd ? weight[i][j][1] : weight[i][j][0]) + __shfl_xor_sync(0xffffffffu, odd ? weight[i][j][0] : weight[i][j][1], 4);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {           // n-tiles 2 j, 2 j + 1 by bit 1
        const bool odd = g & 2;
        v[j] = (odd ? u[2 * j + 1] : u[2 * j]) + __shfl_xor_sync(0xffffffffu, odd ? u[2 * j] : u[2 * j + 1], 8);
      }
      const bool odd = g & 4;
      const float w = (odd ? v[1] : v[0]) + __shfl_xor_sync(0xffffffffu, odd ? v[0] : v[1], 16);
      const int t = t0[i] + 8 * (g >> 1) + 2 * tq + (g & 1);
      if (t < n) {
        float* at = p.mass + b * p.m_sb + h * p.m_sh + t;
        *at = fmaf(*at, p.decay, w);
      }
    }
  }
  if (MODE == kMassWhole && active > 1) cluster_wait();   // the peers have read this block's sums
}

// log2 of each row's sum from its blocks' maxima and sums: a warp a row.
__global__ void __launch_bounds__(256) mass_join_kernel(const __grid_constant__ MassParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int r = blockIdx.x * 8 + static_cast<int>(threadIdx.x >> 5), lane = static_cast<int>(threadIdx.x & 31), h = blockIdx.y, b = blockIdx.z;
  int n, nr;
  mass_extent(p, b, false, n, nr);
  if (r >= nr * p.group) return;
  const int64_t bh = static_cast<int64_t>(b) * p.h_kv + h;
  const int chunks = (n - 1) / (p.chunk_tiles * kMassThreads) + 1;
  float2 x = make_float2(-INFINITY, 0.f);
  for (int c = lane; c < chunks; c += 32) x = join_stats(x, p.stats[(bh * p.chunks + c) * p.rows + r]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x = join_stats(x, make_float2(__shfl_xor_sync(0xffffffffu, x.x, o), __shfl_xor_sync(0xffffffffu, x.y, o)));
  if (lane == 0) p.lse[bh * p.rows + r] = stats_lse(x);
}

// Up to 16 rows, a table longer than a cluster: scores, and each block's maxima and sums.  A warp goes through its tiles of
// 32 tokens with the keys of the next two on their way; what q costs is paid once for all of them.
template <int D>
struct MassStreamSmem {
  static constexpr int kQStride = D + 8;
  uint4 keys[kMassStages][kMassWarps][D / 16][32];
  __half q[kMassFew * kQStride];
  float2 part[kMassWarps][kMassFew];
  float factor[kMassFew];
  int lim[kMassFew];
};

template <bool BF, int CT, int D>
__global__ void __launch_bounds__(kMassThreads, 2) mass_stream_kernel(const __grid_constant__ MassParams p) {
  using Smem = MassStreamSmem<D>;
  constexpr int C = D / 64;
  extern __shared__ __align__(16) uint8_t raw_smem[];
  Smem& sm = *reinterpret_cast<Smem*>(raw_smem);
  pdl_launch_dependents();
  pdl_wait();
  const int chunk = blockIdx.x, h = blockIdx.y, b = blockIdx.z, len = p.chunk_tiles * kMassThreads;
  const int lane = static_cast<int>(threadIdx.x & 31), warp = static_cast<int>(threadIdx.x >> 5);
  const int g = lane >> 2, tq = lane & 3;
  const uint4 my_q = few_queries_load<D>(p, b, h);
  int n, nr;
  mass_extent(p, b, chunk == 0 && h == 0 && threadIdx.x == 0, n, nr);
  if (nr == 0 || static_cast<int64_t>(chunk) * len >= n) return;
  const int64_t bh = static_cast<int64_t>(b) * p.h_kv + h;
  const int base = n - nr, rows = nr * p.group, first = chunk * len;
  const int tiles = min(p.chunk_tiles, (n - first + kMassThreads - 1) / kMassThreads);
  auto start = [&](int i) { return first + (i * kMassWarps + warp) * 32; };
  // lane's n-tile (lane & 3) of tile i: its page, or -1
  auto page_of = [&](int i) {
    const int t = start(i) + 8 * (lane & 3);
    if (i >= tiles || t >= n) return -1;
    const int pg = p.bt[b * p.bt_sb + (t >> p.page_log2)];
    if (pg >= 0 && pg < p.n_pages) return pg;
    if (lane < 4) report_status(p.status, SPECQ_STATUS_BAD_INDEX);
    return -1;
  };
  constexpr float kNoPage = -INFINITY;        // (a page's own scale may be 0; a bit beside it in a word of its own cost 1.5 us of 49)
  auto scale_of = [&](int pg) { return pg < 0 ? kNoPage : p.ks[pg * p.s_sp + h * p.s_sh] * p.sm_log2; };
  const int mask = (1 << p.page_log2) - 1;
  const uint8_t* heads = p.kc + h * p.kv_sh + tq * 16;
  auto fetch = [&](int stage, int i, int pg) {
    if (i < tiles) {
      const int t = start(i) + g;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int of = __shfl_sync(0xffffffffu, pg, j);
        uint4* dst = &sm.keys[stage][warp][j * C][lane];
        if (of >= 0 && t + 8 * j < n) {
          const uint8_t* k = heads + of * p.kv_sp + ((t + 8 * j) & mask) * p.kv_so;
#pragma unroll
          for (int c = 0; c < C; ++c)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst + c * 32)), "l"(k + c * 64) : "memory");
        } else {
#pragma unroll
          for (int c = 0; c < C; ++c) dst[c * 32] = make_uint4(0u, 0u, 0u, 0u);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  int pg[kMassStages];
  float sc[kMassStages];                      // the lane's n-tile's scale of each tile on its way, or kNoPage
#pragma unroll
  for (int i = 0; i < kMassStages; ++i) pg[i] = page_of(i);
  int ahead = page_of(kMassStages);
#pragma unroll
  for (int i = 0; i < kMassStages; ++i) {
    fetch(i, i, pg[i]);
    sc[i] = scale_of(pg[i]);
  }
  few_queries_store<BF, D>(p, sm, my_q, rows, base);
  __syncthreads();
  uint32_t a[C][4][4];
  {
    const __half* lo = sm.q + g * Smem::kQStride + tq * 16;
    const __half* hi = lo + 8 * Smem::kQStride;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int jj = 0; jj < 2; ++jj) {
        const uint4 u = *reinterpret_cast<const uint4*>(lo + c * 64 + jj * 8), v = *reinterpret_cast<const uint4*>(hi + c * 64 + jj * 8);
        a[c][2 * jj][0] = u.x; a[c][2 * jj][1] = v.x; a[c][2 * jj][2] = u.y; a[c][2 * jj][3] = v.y;
        a[c][2 * jj + 1][0] = u.z; a[c][2 * jj + 1][1] = v.z; a[c][2 * jj + 1][2] = u.w; a[c][2 * jj + 1][3] = v.w;
      }
  }
  const float f0 = sm.factor[g], f1 = sm.factor[g + 8];
  const int l0 = sm.lim[g], l1 = sm.lim[g + 8];
  const bool half = rows <= 8;
  const int64_t width = static_cast<int64_t>(p.chunks) * len;
  float* out0 = p.score + (bh * p.rows + g) * width + 2 * tq;
  float* out1 = out0 + 8 * width;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  int stage = 0;
#pragma unroll 1
  for (int i = 0; i < tiles; ++i) {
    const int t = start(i);
    const float scl = sc[0];
    const bool bad = __any_sync(0xffffffffu, scl == kNoPage);
    asm volatile("cp.async.wait_group %0;" ::"n"(kMassStages - 1) : "memory");
    float s[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const uint4 u = sm.keys[stage][warp][j * C + c][lane];
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) {
          uint32_t b0, b1;
          widen4<CT>(w[jj], b0, b1);
          mma_f16(s[j], a[c][jj], b0, b1);
        }
      }
    }
    // the stage is read: its next tile, and the page after that
    fetch(stage, i + kMassStages, ahead);
    stage = stage + 1 == kMassStages ? 0 : stage + 1;
#pragma unroll
    for (int k = 0; k + 1 < kMassStages; ++k) sc[k] = sc[k + 1];
    sc[kMassStages - 1] = scale_of(ahead);
    ahead = page_of(i + kMassStages + 1);
    if (t >= n) continue;                     // (the warp has no tokens here)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float x = __shfl_sync(0xffffffffu, scl, j), x0 = BF ? x * f0 : x, x1 = BF ? x * f1 : x;
      s[j][0] = __fmul_rn(s[j][0], x0); s[j][1] = __fmul_rn(s[j][1], x0);   // rounded once, as by `scale` above
      s[j][2] = __fmul_rn(s[j][2], x1); s[j][3] = __fmul_rn(s[j][3], x1);
    }
    if (bad || t + 31 > base) {
      const uint32_t gone = __ballot_sync(0xffffffffu, scl == kNoPage);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int at = gone >> j & 1u ? INT_MAX - 1 : t + 8 * j + 2 * tq;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (at + e > l0) s[j][e] = -INFINITY;
          if (at + e > l1) s[j][2 + e] = -INFINITY;
        }
      }
    }
    auto take = [&](int e) {
      float top = m[e / 2];
#pragma unroll
      for (int j = 0; j < 4; ++j) top = fmaxf(top, fmaxf(s[j][e], s[j][e + 1]));
      const float z = top == -INFINITY ? 0.f : top;
      float sum = l[e / 2] * exp2_fast(m[e / 2] - z);
#pragma unroll
      for (int j = 0; j < 4; ++j) sum += exp2_fast(s[j][e] - z) + exp2_fast(s[j][e + 1] - z);
      m[e / 2] = top;
      l[e / 2] = sum;
    };
    take(0);
    if (g < rows)
#pragma unroll
      for (int j = 0; j < 4; ++j) *reinterpret_cast<float2*>(out0 + t + 8 * j) = make_float2(s[j][0], s[j][1]);
    if (!half) {
      take(2);
      if (g + 8 < rows)
#pragma unroll
        for (int j = 0; j < 4; ++j) *reinterpret_cast<float2*>(out1 + t + 8 * j) = make_float2(s[j][2], s[j][3]);
    }
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    float2 x = make_float2(m[e], l[e]);
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) x = join_stats(x, make_float2(__shfl_xor_sync(0xffffffffu, x.x, o), __shfl_xor_sync(0xffffffffu, x.y, o)));
    if (tq == 0) sm.part[warp][g + 8 * e] = x;
  }
  __syncthreads();
  const int r = threadIdx.x;
  if (r >= rows) return;
  float2 x = make_float2(-INFINITY, 0.f);
#pragma unroll
  for (int w = 0; w < kMassWarps; ++w) x = join_stats(x, sm.part[w][r]);
  if (sm.lim[r] < 0) x = make_float2(-INFINITY, 0.f);
  p.stats[(bh * p.chunks + chunk) * p.rows + r] = x;
}

// The sums over rows from those scores.
constexpr int kMassSumTokens = 4 * kMassThreads;
__global__ void __launch_bounds__(kMassThreads) mass_sum_kernel(const __grid_constant__ MassParams p) {
  __shared__ float lse[kMassFew];
  pdl_launch_dependents();
  pdl_wait();
  const int h = blockIdx.y, b = blockIdx.z, lane = static_cast<int>(threadIdx.x & 31), warp = static_cast<int>(threadIdx.x >> 5);
  int n, nr;
  mass_extent(p, b, false, n, nr);
  if (nr == 0 || static_cast<int64_t>(blockIdx.x) * kMassSumTokens >= n) return;
  const int64_t bh = static_cast<int64_t>(b) * p.h_kv + h;
  const int len = p.chunk_tiles * kMassThreads, chunks = (n - 1) / len + 1, rows = nr * p.group;
  const int64_t width = static_cast<int64_t>(p.chunks) * len;
  const int t = static_cast<int>(blockIdx.x) * kMassSumTokens + static_cast<int>(threadIdx.x);
  const float* score = p.score + bh * p.rows * width + t;
  float* at = p.mass + b * p.m_sb + h * p.m_sh + t;
  // the first rows' scores and the masses are on their way while the rows' sums are joined
  float v[4][4], old[4], w[4] = {0.f, 0.f, 0.f, 0.f};
  auto load = [&](int r0) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int i = 0; i < 4; ++i) v[r][i] = r0 + r < rows && t + i * kMassThreads < n ? score[(r0 + r) * width + i * kMassThreads] : -INFINITY;
  };
  load(0);
#pragma unroll
  for (int i = 0; i < 4; ++i) old[i] = t + i * kMassThreads < n ? at[i * kMassThreads] : 0.f;
  for (int r = warp; r < kMassFew; r += kMassWarps) {
    float2 x = make_float2(-INFINITY, 0.f);
    if (r < rows)
      for (int c = lane; c < chunks; c += 32) x = join_stats(x, p.stats[(bh * p.chunks + c) * p.rows + r]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x = join_stats(x, make_float2(__shfl_xor_sync(0xffffffffu, x.x, o), __shfl_xor_sync(0xffffffffu, x.y, o)));
    if (lane == 0) lse[r] = stats_lse(x);
  }
  __syncthreads();
  for (int r0 = 0; r0 < rows; r0 += 4) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] += exp2_fast(v[r][i] - lse[r0 + r]);
    if (r0 + 4 < rows) load(r0 + 4);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (t + i * kMassThreads < n) at[i * kMassThreads] = fmaf(old[i], p.decay, w[i]);
}

}  // namespace specq
