// mass.cuh -- how much attention the cached tokens get: the column sums of the softmax over the
// block-scaled cache (block_cache.cuh), added to a running total.
//
// For sequence b and KV head h with G query heads, rows r = (new token i, head g), and token t's key k_t (8-bit
// numbers times their page's scale):
//   s_rt = q_r . k_t sm_scale,   lse_r = ln sum_t exp s_rt   over the tokens that row i sees
//   mass[b, h, t] <- decay mass[b, h, t] + sum_r exp(s_rt - lse_r)          for t < ctx_len[b]
// Row i of n stands at place ctx_len - n + i and sees the tokens up to it.  A row with a NaN or an infinity adds
// nothing, nor does a token of a page outside the cache get anything.
//
// The products run on the tensor cores with the tokens on M: the keys' bytes go from global memory into the
// registers of the thread that the A fragment wants them in (the order of the elements along D is free as long as q
// has the same), are widened to fp16 there, exactly, and stay for all rows; q stands in shared memory as fp16 (bf16
// rows times a power of two that brings their largest element to 2^14: exact down to 2^-31 of it).  Scores,
// maxima and sums are fp32, nothing is rounded in between.
//
// A column needs its rows' sums over all tokens first.  Where one cluster of blocks holds the whole context,
// the blocks exchange their maxima and sums through distributed shared memory and each key is read once;
// else a first launch leaves each tile's maxima and sums, a second joins them, and a third makes the
// products again.  No atomics: a token's sum is one thread's, over the rows in their order.
#pragma once

#include "block_cache.cuh"

namespace specq {

constexpr int kMassThreads = 256;
constexpr int kMassWarps = kMassThreads / 32;
constexpr int kMassTile = 32 * kMassWarps;   // tokens of a block
constexpr int kMassRows = 128;               // rows of q in shared memory at a time
constexpr float kLog2E = 1.44269504f;

struct MassParams {
  const void* q;           // [B, q_len, H, D]; q_sb = 0: packed rows
  const uint8_t* kc;
  const float* ks;
  const int32_t* bt;
  const int32_t* ctx;
  const int32_t* n_rows;   // optional [B]
  float* mass;             // [B, H_KV, N]
  float2* stats;           // workspace [B, H_KV, tiles, rows]: maximum (of score log2 e) and sum
  float* lse;              // workspace [B, H_KV, rows], log2
  int* status;
  int64_t q_sb, q_st, q_sh, kv_sp, kv_so, kv_sh, s_sp, s_sh, bt_sb, m_sb, m_sh;
  int q_len, group, h_kv, page_log2, n_pages, bt_cols, tiles, rows;   // rows = q_len * group
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

// One row of q to fp16 in shared memory, by a warp; *factor: what its scores are to be multiplied by.
// Returns whether every element is finite (else the row is zeros).
template <bool BF, int D>
__device__ __forceinline__ bool mass_query_row(const void* src, __half* dst, float* factor, int lane) {
  constexpr int E = D / 32;
  float v[E], top = 0.f;
  bool finite = true;
  if constexpr (BF) {
    const __nv_bfloat16* s = static_cast<const __nv_bfloat16*>(src) + lane * E;
#pragma unroll
    for (int i = 0; i < E; i += 2) {
      const __nv_bfloat162 u = *reinterpret_cast<const __nv_bfloat162*>(s + i);
      v[i] = __low2float(u);
      v[i + 1] = __high2float(u);
    }
  } else {
    const __half* s = static_cast<const __half*>(src) + lane * E;
#pragma unroll
    for (int i = 0; i < E; i += 2) {
      const __half2 u = *reinterpret_cast<const __half2*>(s + i);
      v[i] = __low2float(u);
      v[i + 1] = __high2float(u);
    }
  }
#pragma unroll
  for (int i = 0; i < E; ++i) {
    finite = finite && fabsf(v[i]) < INFINITY;
    top = fmaxf(top, fabsf(v[i]));
  }
  finite = __all_sync(0xffffffffu, finite);
  *factor = 1.f;
  if constexpr (BF) {
    top = warp_max_f32(top);
    // top 2^k in [2^14, 2^15); 2^126 suffices for what is not zero beside any key
    const int k = top > 0.f && finite ? min(14 - ilogbf(top), 126) : 0;
    const float up = __int_as_float((127 + k) << 23);            // k >= 14 - 127
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] *= up;
    *factor = __int_as_float((127 - k) << 23);
  }
#pragma unroll
  for (int i = 0; i < E; i += 2)
    *reinterpret_cast<__half2*>(dst + lane * E + i) = finite ? __floats2half2_rn(v[i], v[i + 1]) : __floats2half2_rn(0.f, 0.f);
  return finite;
}

template <int D>
struct MassSmem {
  static constexpr int kQStride = D + 8;     // halves: 16 more bytes a row put a quarter-warp's reads on all banks
  __half q[kMassRows * kQStride];
  float2 part[kMassWarps][kMassRows];        // each warp's maximum and sum for a row
  float2 all[kMassRows];                     // the block's
  float lse[kMassRows];
  float factor[kMassRows];
  int lim[kMassRows];                        // the last token that a row sees; -1: none
};

__device__ __forceinline__ float2 join_stats(float2 a, float2 b) {
  const float m = fmaxf(a.x, b.x);
  if (m == -INFINITY) return make_float2(-INFINITY, 0.f);
  return make_float2(m, a.y * exp2_fast(a.x - m) + b.y * exp2_fast(b.x - m));
}

template <bool BF, int CT, int D, int MODE>
__global__ void __launch_bounds__(kMassThreads, 2) mass_kernel(const __grid_constant__ MassParams p) {
  using Smem = MassSmem<D>;
  extern __shared__ __align__(16) uint8_t raw_smem[];
  Smem& sm = *reinterpret_cast<Smem*>(raw_smem);
  pdl_launch_dependents();
  pdl_wait();
  const int tile = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int lane = static_cast<int>(threadIdx.x & 31), warp = static_cast<int>(threadIdx.x >> 5);
  const int g = lane >> 2, tq = lane & 3;
  int n = p.ctx[b];
  const int most = p.bt_cols << p.page_log2;
  if (n > most) {
    if (tile == 0 && h == 0 && threadIdx.x == 0) report_status(p.status, SPECQ_STATUS_PLAN_CLAMPED);
    n = most;
  }
  const int nr = p.n_rows == nullptr ? p.q_len : min(max(p.n_rows[b], 0), p.q_len);
  const bool idle = n <= 0 || nr == 0 || tile * kMassTile >= n;
  // (a cluster's blocks stay together: an idle one still takes part in the barriers)
  if (MODE != kMassWhole && idle) return;

  // this lane's four tokens of the warp's 32: page, scale, keys
  constexpr int C = D / 64;
  uint32_t a[2][C][4][4];
  float tscale[2][2];
  int tok[2][2];             // a token that no row sees: INT_MAX
  const int t0 = tile * kMassTile + warp * 32;
  bool good = true;
  {
    uint4 w[2][2][C];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int t = t0 + mt * 16 + half * 8 + g;
        tok[mt][half] = INT_MAX;
        tscale[mt][half] = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c) w[mt][half][c] = make_uint4(0u, 0u, 0u, 0u);
        if (!idle && t < n) {
          const int pg = p.bt[b * p.bt_sb + (t >> p.page_log2)];
          if (pg >= 0 && pg < p.n_pages) {
            tok[mt][half] = t;
            const uint8_t* k = p.kc + pg * p.kv_sp + (t & ((1 << p.page_log2) - 1)) * p.kv_so + h * p.kv_sh + tq * 16;
#pragma unroll
            for (int c = 0; c < C; ++c) w[mt][half][c] = *reinterpret_cast<const uint4*>(k + c * 64);
            tscale[mt][half] = p.ks[pg * p.s_sp + h * p.s_sh] * p.sm_log2;
          } else {
            report_status(p.status, SPECQ_STATUS_BAD_INDEX);
            good = false;
          }
        } else {
          good = false;
        }
      }
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const uint32_t* u = reinterpret_cast<const uint32_t*>(&w[mt][0][c]);
        const uint32_t* v = reinterpret_cast<const uint32_t*>(&w[mt][1][c]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          widen4<CT>(u[j], a[mt][c][j][0], a[mt][c][j][2]);
          widen4<CT>(v[j], a[mt][c][j][1], a[mt][c][j][3]);
        }
      }
  }
  const int base = n - nr;
  good = __all_sync(0xffffffffu, good);
  float weight[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
  const int64_t bh = static_cast<int64_t>(b) * p.h_kv + h;
  const int rows = nr * p.group;

  // scores of eight rows from `r0` of the block, times log2 e; -inf where a row does not see a token
  auto scores = [&](int r0, float (&s)[2][4]) {
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[mt][i] = 0.f;
    const __half* qrow = sm.q + (r0 + g) * Smem::kQStride + tq * 16;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int jj = 0; jj < 2; ++jj) {
        const uint4 u = *reinterpret_cast<const uint4*>(qrow + c * 64 + jj * 8);
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          mma_f16(s[mt], a[mt][c][2 * jj], u.x, u.y);
          mma_f16(s[mt], a[mt][c][2 * jj + 1], u.z, u.w);
        }
      }
    const float f0 = sm.factor[r0 + 2 * tq], f1 = sm.factor[r0 + 2 * tq + 1];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        // a NaN among the keys weighs nothing
        s[mt][2 * half] = fmaxf(s[mt][2 * half] * tscale[mt][half] * (BF ? f0 : 1.f), -INFINITY);
        s[mt][2 * half + 1] = fmaxf(s[mt][2 * half + 1] * tscale[mt][half] * (BF ? f1 : 1.f), -INFINITY);
      }
    if (!good || t0 + 31 > base) {
      const int l0 = sm.lim[r0 + 2 * tq], l1 = sm.lim[r0 + 2 * tq + 1];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (tok[mt][half] > l0) s[mt][2 * half] = -INFINITY;
          if (tok[mt][half] > l1) s[mt][2 * half + 1] = -INFINITY;
        }
    }
  };

  for (int first = 0; first < rows; first += kMassRows) {
    const int here = min(kMassRows, rows - first), padded = (here + 7) & ~7;
    if (first > 0) __syncthreads();
    for (int r = warp; r < padded; r += kMassWarps) {
      __half* dst = sm.q + r * Smem::kQStride;
      if (r < here) {
        const int i = (first + r) / p.group, head = h * p.group + (first + r) - i * p.group;
        const int64_t at = (p.q_sb != 0 ? b * p.q_sb + i * p.q_st : (static_cast<int64_t>(b) * p.q_len + i) * p.q_st) + head * p.q_sh;
        float factor;
        const bool finite = mass_query_row<BF, D>(static_cast<const __half*>(p.q) + at, dst, &factor, lane);
        if (lane == 0) {
          sm.factor[r] = factor;
          sm.lim[r] = finite ? base + i : -1;
        }
      } else {
        for (int e = lane * 2; e < D; e += 64) *reinterpret_cast<uint32_t*>(dst + e) = 0u;
        if (lane == 0) {
          sm.factor[r] = 1.f;
          sm.lim[r] = -1;
        }
      }
    }
    if constexpr (MODE == kMassWeights)
      for (int r = threadIdx.x; r < padded; r += kMassThreads) sm.lse[r] = r < here ? p.lse[bh * p.rows + first + r] : INFINITY;
    __syncthreads();
    if constexpr (MODE != kMassWeights) {
      for (int r0 = 0; r0 < padded; r0 += 8) {
        float s[2][4];
        scores(r0, s);
        float m0 = fmaxf(fmaxf(s[0][0], s[0][2]), fmaxf(s[1][0], s[1][2]));
        float m1 = fmaxf(fmaxf(s[0][1], s[0][3]), fmaxf(s[1][1], s[1][3]));
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, o));
          m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, o));
        }
        const float z0 = m0 == -INFINITY ? 0.f : m0, z1 = m1 == -INFINITY ? 0.f : m1;
        float l0 = 0.f, l1 = 0.f;
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            l0 += exp2_fast(s[mt][2 * half] - z0);
            l1 += exp2_fast(s[mt][2 * half + 1] - z1);
          }
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          l0 += __shfl_xor_sync(0xffffffffu, l0, o);
          l1 += __shfl_xor_sync(0xffffffffu, l1, o);
        }
        if (g == 0) {
          sm.part[warp][r0 + 2 * tq] = make_float2(m0, l0);
          sm.part[warp][r0 + 2 * tq + 1] = make_float2(m1, l1);
        }
      }
      __syncthreads();
      for (int r = threadIdx.x; r < padded; r += kMassThreads) {
        float2 x = make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int w = 0; w < kMassWarps; ++w) x = join_stats(x, sm.part[w][r]);
        if (sm.lim[r] < 0) x = make_float2(-INFINITY, 0.f);
        if (MODE == kMassStats) {
          if (r < here) p.stats[(bh * p.tiles + tile) * p.rows + first + r] = x;
        } else {
          sm.lse[r] = x.y > 0.f ? x.x + log2f(x.y) : INFINITY;   // +inf: exp2(s - lse) is 0
        }
      }
      if (MODE == kMassWhole) __syncthreads();
    }
    if constexpr (MODE != kMassStats) {
      for (int r0 = 0; r0 < padded; r0 += 8) {
        float s[2][4];
        scores(r0, s);
        const float l0 = sm.lse[r0 + 2 * tq], l1 = sm.lse[r0 + 2 * tq + 1];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int half = 0; half < 2; ++half)
            weight[mt][half] += exp2_fast(s[mt][2 * half] - l0) + exp2_fast(s[mt][2 * half + 1] - l1);
      }
    }
  }
  if constexpr (MODE != kMassStats) {
    if (idle) return;
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float w = weight[mt][half];
        w += __shfl_xor_sync(0xffffffffu, w, 1);
        w += __shfl_xor_sync(0xffffffffu, w, 2);
        const int t = t0 + mt * 16 + half * 8 + g;
        if (tq == 0 && t < n) {
          float* at = p.mass + b * p.m_sb + h * p.m_sh + t;
          *at = fmaf(*at, p.decay, w);
        }
      }
  }
}

// log2 of each row's sum from its tiles' maxima and sums, in their order.
__global__ void __launch_bounds__(128) mass_join_kernel(const __grid_constant__ MassParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int r = blockIdx.x * 128 + threadIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int n = min(p.ctx[b], p.bt_cols << p.page_log2);
  const int nr = p.n_rows == nullptr ? p.q_len : min(max(p.n_rows[b], 0), p.q_len);
  if (r >= nr * p.group || n <= 0) return;
  const int64_t bh = static_cast<int64_t>(b) * p.h_kv + h;
  const int tiles = (n + kMassTile - 1) / kMassTile;
  const float2* at = p.stats + bh * p.tiles * p.rows + r;
  float2 x = make_float2(-INFINITY, 0.f);
  for (int t = 0; t < tiles; ++t) x = join_stats(x, at[static_cast<int64_t>(t) * p.rows]);
  p.lse[bh * p.rows + r] = x.y > 0.f ? x.x + log2f(x.y) : INFINITY;
}

inline int mass_check(int B, int q_len, int H, int H_KV, int D, int page, int bt_cols) {
  const char* who = "attention_mass";
  if (B < 0 || q_len < 0 || H < 1 || H_KV < 1 || H % H_KV || bt_cols < 0)
    return fail(SPECQ_ERR_INVALID_ARG, "%s: B=%d q_len=%d H=%d H_KV=%d bt_cols=%d", who, B, q_len, H, H_KV, bt_cols);
  if (D != 64 && D != 128) return fail(SPECQ_ERR_UNSUPPORTED, "%s: head_dim %d (64 or 128)", who, D);
  if (page < 8 || page > 128 || (page & (page - 1))) return fail(SPECQ_ERR_UNSUPPORTED, "%s: page %d (a power of two, 8 to 128)", who, page);
  if (B > 65535 || H_KV > 65535 || static_cast<int64_t>(bt_cols) * page > 0x7ffffeffll || static_cast<int64_t>(q_len) * (H / H_KV) > 0x7fffff00ll)
    return fail(SPECQ_ERR_UNSUPPORTED, "%s: B=%d H_KV=%d, %d pages of %d, %d rows of %d heads", who, B, H_KV, bt_cols, page, q_len, H / H_KV);
  return SPECQ_OK;
}

inline int run_attention_mass_workspace(int B, int q_len, int H, int H_KV, int D, int page, int bt_cols, int64_t* bytes) {
  if (bytes == nullptr) return fail(SPECQ_ERR_INVALID_ARG, "attention_mass_workspace: null pointer");
  if (int rc = mass_check(B, q_len, H, H_KV, D, page, bt_cols)) return rc;
  const int tiles = ceil_div(bt_cols * page, kMassTile);
  const int64_t rows = static_cast<int64_t>(B) * H_KV * q_len * (H / H_KV);
  *bytes = tiles > 1 ? rows * tiles * 8 + rows * 4 : 0;
  return SPECQ_OK;
}

inline int run_attention_mass(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, int dtype, const void* kc, int64_t kv_sp,
                              int64_t kv_so, int64_t kv_sh, int cache_dtype, int n_pages, const float* ks, int64_t s_sp, int64_t s_sh,
                              const int32_t* block_tbl, int64_t bt_sb, int bt_cols, const int32_t* ctx_len, const int32_t* n_rows,
                              float sm_scale, float decay, float* mass, int64_t m_sb, int64_t m_sh, int B, int q_len, int H, int H_KV,
                              int D, int page, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* who = "attention_mass";
  if (int rc = mass_check(B, q_len, H, H_KV, D, page, bt_cols)) return rc;
  if (dtype != SPECQ_DTYPE_F16 && dtype != SPECQ_DTYPE_BF16) return fail(SPECQ_ERR_INVALID_ARG, "%s: dtype code %d", who, dtype);
  if (cache_dtype != SPECQ_CACHE_INT8 && cache_dtype != SPECQ_CACHE_E4M3) return fail(SPECQ_ERR_INVALID_ARG, "%s: cache dtype code %d", who, cache_dtype);
  if (!(sm_scale > 0.f)) return fail(SPECQ_ERR_INVALID_ARG, "%s: sm_scale %g", who, static_cast<double>(sm_scale));
  if (B == 0 || q_len == 0 || bt_cols == 0) return SPECQ_OK;
  if (q == nullptr || kc == nullptr || ks == nullptr || block_tbl == nullptr || ctx_len == nullptr || mass == nullptr)
    return fail(SPECQ_ERR_INVALID_ARG, "%s: null pointer", who);
  if (!aligned(q, 16) || q_sb % 8 || q_st % 8 || q_sh % 8) return fail(SPECQ_ERR_UNSUPPORTED, "%s: query rows must be 16-byte aligned", who);
  if (!aligned(kc, 16) || kv_sp % 16 || kv_so % 16 || kv_sh % 16) return fail(SPECQ_ERR_UNSUPPORTED, "%s: cache rows must be 16-byte aligned", who);
  int64_t need = 0;
  if (int rc = run_attention_mass_workspace(B, q_len, H, H_KV, D, page, bt_cols, &need)) return rc;
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 16)))
    return fail(SPECQ_ERR_INVALID_ARG, "%s: a workspace of %lld bytes is needed", who, static_cast<long long>(need));
  DeviceState* dev = nullptr;
  if (int rc = get_device_state(&dev)) return rc;
  MassParams p = {};
  p.q = q; p.kc = static_cast<const uint8_t*>(kc); p.ks = ks; p.bt = block_tbl; p.ctx = ctx_len; p.n_rows = n_rows; p.mass = mass;
  p.status = dev->status;
  p.q_sb = q_sb; p.q_st = q_st; p.q_sh = q_sh; p.kv_sp = kv_sp; p.kv_so = kv_so; p.kv_sh = kv_sh; p.s_sp = s_sp; p.s_sh = s_sh;
  p.bt_sb = bt_sb; p.m_sb = m_sb; p.m_sh = m_sh;
  p.q_len = q_len; p.group = H / H_KV; p.h_kv = H_KV; p.page_log2 = __builtin_ctz(static_cast<unsigned>(page));
  p.n_pages = n_pages; p.bt_cols = bt_cols; p.tiles = ceil_div(bt_cols * page, kMassTile); p.rows = q_len * p.group;
  p.sm_log2 = sm_scale * kLog2E; p.decay = decay;
  p.stats = static_cast<float2*>(workspace);
  p.lse = reinterpret_cast<float*>(p.stats + (p.tiles > 1 ? static_cast<int64_t>(B) * H_KV * p.tiles * p.rows : 0));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid(p.tiles, H_KV, B);
  auto launch = [&](auto kern, size_t smem) {
    const cudaError_t e = ensure_dyn_smem(reinterpret_cast<const void*>(kern), static_cast<int>(smem));
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kMassThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    LaunchAttrs at(1);
    at.apply(cfg);
    return cudaLaunchKernelEx(&cfg, kern, p);
  };
  auto all = [&](auto bf, auto ct, auto d) -> int {
    constexpr bool BF = decltype(bf)::value;
    constexpr int CT = decltype(ct)::value, DD = decltype(d)::value;
    const size_t smem = sizeof(MassSmem<DD>);
    if (p.tiles == 1) {
      SPECQ_CUDA_TRY(launch(mass_kernel<BF, CT, DD, kMassWhole>, smem));
      return SPECQ_OK;
    }
    SPECQ_CUDA_TRY(launch(mass_kernel<BF, CT, DD, kMassStats>, smem));
    SPECQ_CUDA_TRY(launch_plain(mass_join_kernel, dim3(ceil_div(p.rows, 128), H_KV, B), dim3(128), st, p));
    SPECQ_CUDA_TRY(launch(mass_kernel<BF, CT, DD, kMassWeights>, smem));
    return SPECQ_OK;
  };
  auto by_d = [&](auto bf, auto ct) { return D == 64 ? all(bf, ct, std::integral_constant<int, 64>{}) : all(bf, ct, std::integral_constant<int, 128>{}); };
  auto by_ct = [&](auto bf) {
    return cache_dtype == SPECQ_CACHE_INT8 ? by_d(bf, std::integral_constant<int, 0>{}) : by_d(bf, std::integral_constant<int, 1>{});
  };
  return dtype == SPECQ_DTYPE_F16 ? by_ct(std::false_type{}) : by_ct(std::true_type{});
}

}  // namespace specq
