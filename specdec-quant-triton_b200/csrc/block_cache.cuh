// block_cache.cuh -- writing a KV cache held in 8 bits with one fp32 scale for each page and
// KV head: the append of new tokens and the compaction of a verified draft tree.
//
// Cache: kc, vc [P, page, H_KV, D] of int8 or e4m3 numbers q (q_max = 127 or 448) and ks, vs
// [P, H_KV] fp32 scales s; the value is q * s.
//
// append.  Token t of sequence b (row b * q_len + t) goes to position ctx_len[b] - q_len + t.
// For each page that receives tokens and each KV head, with a = max |x| over its new tokens
// (K after its rotary turn, in fp32):
//   need = max(a, 1e-8) * fp32(1 / q_max)
//   s'   = need               if the page's first slot is among the new tokens
//          max(s, need)       otherwise; the page's older tokens become rn(q * (s / s'))
//   q'   = rn(x * (1 / s'))   saturated, for the new tokens
// Older tokens are rewritten only when the scale grows; slots past the new tokens are not
// touched.  An 8-bit number has no NaN or infinity here: a NaN is stored as 0, an infinity as
// +-q_max, neither takes part in a, and SPECQ_STATUS_KV_NONFINITE is reported.
//
// A warp holds 8 (16 at D = 64) slots of one page and head in registers, 32 fp32 a thread,
// so the rotated values are made once and used twice, for the maximum and for the numbers; the
// warps that share a larger page are of one CTA and exchange their maxima through shared memory.
// The same launch turns the tokens' queries: they come from the same rows, and a launch of their
// own costs a short verification step as much as the work.  Bound by HBM for prompts and by latency
// for a few tokens.  Measured (32 query and 8 KV heads of 128): 4 x 2047 tokens, page 64: 36.9 us,
// 5.1 TB/s (keys and values of 64 values a thread and half the blocks an SM took 6 us more, blocks of
// queries among those of keys and values 0.7); 8 x 9 tokens: 4.5 us.
//
// compact.  After verification the accepted drafts of sequence b sit at base + accept[b, j]
// (base = ctx_len - q_len); they move to base + j.  A target page's scale becomes
//   s' = max(s, max over its arriving tokens of (max |q| * fp32(1 / q_max)) * s_source)
// and numbers whose scale differs are requantised, rn(q * (s_source / s')).  One warp per
// (layer, sequence, head, K or V) walks its tokens in order, 4 or 8 at a time: accept[j] >= j
// and both grow, so a token never lands on one that has yet to be read.  Bound by scattered reads
// and writes of 128 bytes.  Measured: 48 trees of 33 nodes, 32 layers, 8 heads of 128: 26.3 us for
// some 83 MB, 3.2 TB/s (40 warps an SM in place of 28: the same; two to eight heads a warp, the next
// one's tokens read ahead: 31 to 46; half as many tokens in flight: 31); 8 chains of 9, one layer:
// 3.0 us, the three loads of its chain.
//
// Lengths, tables, scales and numbers are written by the kernels that come before these in a stream, and under
// programmatic launch a kernel's blocks may be resident while those still run.  They are read by plain
// loads after the wait; the read-only path (__ldg) is for what no such kernel writes: rotary tables and
// positions, plans, accepted indices.
#pragma once

#include <cuda_fp8.h>

#include "rope.cuh"

namespace specq {

constexpr int kAppendThreads = 256;
constexpr int kAppendWarps = kAppendThreads / 32;
// Slots of a page that one warp holds: 8 x 128 or 16 x 64 values are 32 fp32 a thread, which leaves
// room for four blocks an SM (64 for 16 x 128 left room for two); a page of 128 slots of 128 needs 16.
__host__ __device__ constexpr int append_slots(int D, int page) { return D == 128 && page <= 64 ? 8 : 16; }
constexpr float kKvFloor = 1e-8f;

template <int CT>   // 0 = int8, 1 = e4m3
__host__ __device__ constexpr float cache_inv_max() { return CT == 0 ? 1.0f / 127.0f : 1.0f / 448.0f; }

// Four fp32 to four 8-bit numbers (round to nearest even).  None of them is NaN; int8: none rounds
// to more than 127 in magnitude.
template <int CT>
__device__ __forceinline__ uint32_t pack_cache4(float a, float b, float c, float d) {
  if constexpr (CT == 0) {
    uint32_t lo, w;
    asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, 0;" : "=r"(lo) : "r"(__float2int_rn(d)), "r"(__float2int_rn(c)));
    asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, %3;" : "=r"(w) : "r"(__float2int_rn(b)), "r"(__float2int_rn(a)), "r"(lo));
    return w;
  } else {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
  }
}

template <int CT>
__device__ __forceinline__ void unpack_cache4(uint32_t w, float (&v)[4]) {
  if constexpr (CT == 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = static_cast<float>(static_cast<int8_t>((w >> (8 * i)) & 0xFFu));
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>((w >> (16 * i)) & 0xFFFFu), __NV_E4M3);
      const float2 f = __half22float2(__half2(r));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
}

// rn(q * r) of four stored numbers, r <= 1 (a stored -128 is not one of this cache's)
template <int CT>
__device__ __forceinline__ uint32_t requant4(uint32_t w, float r) {
  float v[4];
  unpack_cache4<CT>(w, v);
  return pack_cache4<CT>(v[0] * r, v[1] * r, v[2] * r, v[3] * r);
}

// The largest magnitude of 16 stored numbers; exact in fp16, two at a time.
template <int CT>
__device__ __forceinline__ float absmax16(const uint4& u) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  __half2 m = __half2(__half_raw{0}, __half_raw{0});
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    __half2 a, b;
    if constexpr (CT == 0) {          // 1024 + (byte ^ 0x80), less 1152
      const uint32_t x = w[i] ^ 0x80808080u;
      const uint32_t lo = __byte_perm(x, 0x64646464u, 0x4140), hi = __byte_perm(x, 0x64646464u, 0x4342);
      const __half2 off = __half2(__half_raw{0x6480}, __half_raw{0x6480});
      a = __hsub2(*reinterpret_cast<const __half2*>(&lo), off);
      b = __hsub2(*reinterpret_cast<const __half2*>(&hi), off);
    } else {
      a = __half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w[i] & 0xFFFFu), __NV_E4M3));
      b = __half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w[i] >> 16), __NV_E4M3));
    }
    m = __hmax2(m, __hmax2(__habs2(a), __habs2(b)));
  }
  return __half2float(__hmax(__low2half(m), __high2half(m)));
}

struct BlockAppendParams {
  const void* k;         // [T, H_KV, D] packed token rows
  const void* v;
  const void* q;         // optional [T, H, D]: turned into q_out
  void* q_out;
  const float* table;    // optional [n_pos, rot]
  const int32_t* pos;    // optional [T] rotary positions (default: the token's cache position)
  uint8_t* kc;
  uint8_t* vc;
  float* ks;
  float* vs;
  const int32_t* bt;
  const int32_t* ctx;
  const int32_t* plan;   // plan[0] = n_seqs, plan[1] = q_len
  int* status;
  int64_t kt, kh, vt, vh, qt, qh, ot, oh, kv_sp, kv_so, kv_sh, s_sp, s_sh, bt_sb;
  int n_seqs, q_len, b_grid, ql_max, h_kv, h_q, page_log2, n_pages, bt_cols, rot, n_pos, half;
  int wide;                           // rows of K and V are 16-byte aligned
  int n_win, win_blocks, kv_blocks;   // pages a sequence may touch, blocks of one of them, blocks of all
  int q_items, q_groups;
};

template <typename T>
__device__ __forceinline__ void load_row4(const T* p, float* v) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = weight_to_f32<T>(e[i]);
}

__device__ __forceinline__ void append_extents(const BlockAppendParams& p, int& n_seqs, int& q_len) {
  n_seqs = p.n_seqs;
  q_len = p.q_len;
  if (p.plan != nullptr) {
    const int a = __ldg(p.plan), b = __ldg(p.plan + 1);
    n_seqs = min(max(a, 0), p.b_grid);
    q_len = min(max(b, 0), p.ql_max);
    if ((a != n_seqs || b != q_len) && blockIdx.x == 0 && threadIdx.x == 0)
      report_status(p.status, SPECQ_STATUS_PLAN_CLAMPED);
  }
}

// Thread id of the tokens' queries: one 16-byte item of HP heads of a token.
template <typename T, int HP>
__device__ __forceinline__ void append_queries(const BlockAppendParams& p, uint32_t id, int n_seqs, int q_len) {
  const uint32_t th = id / static_cast<uint32_t>(p.q_items);
  const int item = static_cast<int>(id - th * p.q_items);
  const int t = static_cast<int>(th / static_cast<uint32_t>(p.q_groups));
  const int h0 = static_cast<int>(th - static_cast<uint32_t>(t) * p.q_groups) * HP;
  if (t >= n_seqs * q_len) return;
  int pos;
  if (p.pos != nullptr) {
    pos = __ldg(p.pos + t);
  } else {
    const int b = t / q_len;
    pos = p.ctx[b] - q_len + (t - b * q_len);
  }
  const float* row = rope_row(p.table, pos, p.n_pos, p.rot, p.status);
  const T* x = static_cast<const T*>(p.q) + t * p.qt + h0 * p.qh;
  T* out = static_cast<T*>(p.q_out) + t * p.ot + h0 * p.oh;
  const int n = min(HP, p.h_q - h0);
  if (p.half) rope_item<T, true, HP>(x, p.qh, out, p.oh, row, p.rot, 1.f, item, n);
  else rope_item<T, false, HP>(x, p.qh, out, p.oh, row, p.rot, 1.f, item, n);
}

template <typename T, int D, int CT, int SLOTS, int HP>
__global__ void __launch_bounds__(kAppendThreads, SLOTS * D <= 1024 ? 4 : 2)
block_append_kernel(const __grid_constant__ BlockAppendParams p) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ float red[kAppendWarps];
  int n_seqs, q_len;
  append_extents(p, n_seqs, q_len);
  if (static_cast<int>(blockIdx.x) >= p.kv_blocks) {
    append_queries<T, HP>(p, (blockIdx.x - p.kv_blocks) * kAppendThreads + threadIdx.x, n_seqs, q_len);
    return;
  }

  // ---- keys and values: (sequence, page of its window, group of (head, K|V) units)
  const int page = 1 << p.page_log2;
  const int wpu = max(1, page / SLOTS);                     // warps of a unit
  const int warp = static_cast<int>(threadIdx.x >> 5), lane = static_cast<int>(threadIdx.x & 31);
  const int bw = static_cast<int>(blockIdx.x) / p.win_blocks;
  const int part = static_cast<int>(blockIdx.x) - bw * p.win_blocks;
  const int b = bw / p.n_win, win = bw - b * p.n_win;
  if (b >= n_seqs || q_len == 0) return;
  const int ctx = p.ctx[b];
  const int base = ctx - q_len;
  if (base < 0 || ctx > p.bt_cols * page) {                 // tokens outside the table: not written
    if (threadIdx.x == 0 && win == 0 && part == 0) report_status(p.status, SPECQ_STATUS_PLAN_CLAMPED);
    return;
  }
  const int col = (base >> p.page_log2) + win;
  const int start = col << p.page_log2;                     // position of the page's slot 0
  if (start >= ctx) return;
  const int pg = p.bt[b * p.bt_sb + col];           // looked at after the rows' loads
  const int unit = part * (kAppendWarps / wpu) + warp / wpu;
  const bool live = unit < 2 * p.h_kv;
  const bool is_v = unit >= p.h_kv;
  const int head = is_v ? unit - p.h_kv : unit;
  const int sub = warp % wpu;                               // this warp's slots of the page

  constexpr int LPT = D / 8;            // lanes of a token
  constexpr int TPS = 32 / LPT;         // tokens of a step
  constexpr int STEPS = SLOTS / TPS;
  const int l = lane % LPT;
  const bool turn = !is_v && p.table != nullptr && 8 * l < p.rot;
  // the thread's 8 elements are two runs of 4: partners in the half layout
  const int o1 = turn && p.half ? 4 * l : 8 * l;
  const int o2 = turn && p.half ? (p.rot >> 1) + 4 * l : 8 * l + 4;
  const int slot0 = sub * SLOTS + lane / LPT;
  // steps i with a new token: lo <= i < hi (slots past a small page are past every token)
  const int first = start + slot0;
  const int lo = max(0, (base - first + TPS - 1) / TPS);
  const int end = min(ctx, start + page);
  const int hi = live ? min(STEPS, max(0, (end - first + TPS - 1) / TPS)) : 0;
  float x[STEPS][8];
  const int64_t row0 = b * q_len + (first - base);
  {
    const int64_t st = is_v ? p.vt : p.kt;
    const T* r = static_cast<const T*>(is_v ? p.v : p.k) + head * (is_v ? p.vh : p.kh) + row0 * st;
    // one 16-byte load for both runs where they adjoin (41.0 -> 36.9 us for 4 x 2047 tokens)
    if (p.wide && o2 == o1 + 4) {
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        Row16<T> w;
        w.raw = make_uint4(0u, 0u, 0u, 0u);
        if (i >= lo && i < hi) w.load(r + i * TPS * st + o1);
        w.get(x[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[i][e] = 0.f;
        if (i >= lo && i < hi) {
          load_row4<T>(r + i * TPS * st + o1, x[i]);
          load_row4<T>(r + i * TPS * st + o2, x[i] + 4);
        }
      }
    }
  }
  if (pg < 0 || pg >= p.n_pages) {
    if (threadIdx.x == 0 && part == 0) report_status(p.status, SPECQ_STATUS_BAD_INDEX);
    return;
  }
  float s_old = 0.f;
  float* scale = nullptr;
  uint8_t* dst = nullptr;
  if (live) {
    scale = (is_v ? p.vs : p.ks) + static_cast<int64_t>(pg) * p.s_sp + head * p.s_sh;
    dst = (is_v ? p.vc : p.kc) + static_cast<int64_t>(pg) * p.kv_sp + head * p.kv_sh;
    s_old = *scale;
  }
  if (turn) {
    auto each = [&](auto is_half) {
      constexpr bool HALF = decltype(is_half)::value;
#pragma unroll
      for (int i = 0; i < STEPS; ++i)
        if (i >= lo && i < hi) {
          const int pos = p.pos != nullptr ? __ldg(p.pos + row0 + i * TPS) : first + i * TPS;
          const float* row = rope_row(p.table, pos, p.n_pos, p.rot, p.status);
          float c[4], s[4];
          load_f32_run<4>(row + 4 * l, c);
          load_f32_run<4>(row + (p.rot >> 1) + 4 * l, s);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float& xa = x[i][HALF ? e : 2 * e];
            float& xb = x[i][HALF ? e + 4 : 2 * e + 1];
            const float a = xa, bb = xb;
            xa = fmaf(a, c[e], -bb * s[e]);
            xb = fmaf(bb, c[e], a * s[e]);
          }
        }
    };
    if (p.half) each(std::true_type{});
    else each(std::false_type{});
  }
  // the maximum of the magnitudes as bits: a NaN or an infinity shows as 0x7f800000 or more
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < STEPS; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[i][e]) & 0x7fffffffu);
  float amax = __uint_as_float(top);
  const bool odd = __any_sync(0xffffffffu, top >= 0x7f800000u);
  if (odd) {                            // NaN becomes 0; infinities have no part in the maximum
    amax = 0.f;
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (!(x[i][e] == x[i][e])) x[i][e] = 0.f;
        const float a = fabsf(x[i][e]);
        if (a <= 3.402823466e38f) amax = fmaxf(amax, a);
      }
    if (lane == 0) report_status(p.status, SPECQ_STATUS_KV_NONFINITE);
  }
  amax = warp_max_f32(amax);
  if (wpu > 1) {
    if (lane == 0) red[warp] = amax;
    __syncthreads();                    // also: every warp has read the old scale
    for (int w = 0; w < wpu; ++w) amax = fmaxf(amax, red[warp - sub + w]);
  } else {
    __syncwarp();
  }
  if (!live) return;
  const float need = fmaxf(amax, kKvFloor) * cache_inv_max<CT>();
  const bool fresh = start >= base;
  const float s_new = fresh ? need : fmaxf(s_old, need);
  const float rs = __frcp_rn(s_new);
  if (odd) {                            // an infinity is stored as the largest number
    const float lim = s_new * (1.f / cache_inv_max<CT>());
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (fabsf(x[i][e]) > 3.402823466e38f) x[i][e] = copysignf(lim, x[i][e]);
  }
  {
    uint8_t* d = dst + static_cast<int64_t>(slot0) * p.kv_so;
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
      if (i >= lo && i < hi) {
        const float* y = x[i];
        const uint32_t w0 = pack_cache4<CT>(y[0] * rs, y[1] * rs, y[2] * rs, y[3] * rs);
        const uint32_t w1 = pack_cache4<CT>(y[4] * rs, y[5] * rs, y[6] * rs, y[7] * rs);
        uint8_t* q = d + static_cast<int64_t>(i * TPS) * p.kv_so;
        if (turn && p.half) {
          *reinterpret_cast<uint32_t*>(q + o1) = w0;
          *reinterpret_cast<uint32_t*>(q + o2) = w1;
        } else {
          *reinterpret_cast<uint2*>(q + o1) = make_uint2(w0, w1);
        }
      }
  }
  if (!fresh && s_new > s_old) {        // the page's older tokens under the grown scale
    const float r = __fdiv_rn(s_old, s_new);
    for (int slot = slot0; slot < min(base - start, (sub + 1) * SLOTS); slot += TPS) {
      uint2* d = reinterpret_cast<uint2*>(dst + static_cast<int64_t>(slot) * p.kv_so + 8 * l);
      uint2 w = *d;
      w.x = requant4<CT>(w.x, r);
      w.y = requant4<CT>(w.y, r);
      *d = w;
    }
  }
  if (sub == 0 && lane == 0 && s_new != s_old) *scale = s_new;
}

inline bool page_ok(int page) { return page >= 8 && page <= 128 && (page & (page - 1)) == 0; }

inline int run_block_append(const void* k, int64_t kt, int64_t kh, const void* v, int64_t vt, int64_t vh,
                            const void* q, int64_t qt, int64_t qh, void* q_out, int64_t ot, int64_t oh, int dtype,
                            const float* table, int n_pos, int rot, int layout, const int32_t* pos, void* kc,
                            void* vc, int64_t kv_sp, int64_t kv_so, int64_t kv_sh, int cache_dtype, int n_pages,
                            float* ks, float* vs, int64_t s_sp, int64_t s_sh, const int32_t* bt, int64_t bt_sb,
                            int bt_cols, const int32_t* ctx, const int32_t* plan, int B, int n_seqs, int q_len,
                            int ql_max, int H, int H_KV, int D, int page, void* stream) {
  if (B < 0 || n_seqs < 0 || q_len < 0 || ql_max < 0 || H < 0 || H_KV <= 0 || n_pages < 0 || bt_cols < 0)
    return fail(SPECQ_ERR_INVALID_ARG, "block_append: negative size");
  if (dtype != 0 && dtype != 2) return fail(SPECQ_ERR_INVALID_ARG, "block_append: row dtype code %d", dtype);
  if (cache_dtype != SPECQ_CACHE_INT8 && cache_dtype != SPECQ_CACHE_E4M3)
    return fail(SPECQ_ERR_INVALID_ARG, "block_append: cache dtype code %d", cache_dtype);
  if (D != 64 && D != 128) return fail(SPECQ_ERR_UNSUPPORTED, "block_append: head_dim %d (this build supports 64 and 128)", D);
  if (!page_ok(page)) return fail(SPECQ_ERR_UNSUPPORTED, "block_append: page %d (a power of two in 8..128)", page);
  if (plan == nullptr && (n_seqs > B || q_len > ql_max))
    return fail(SPECQ_ERR_INVALID_ARG, "block_append: n_seqs/q_len exceed the grid");
  if (layout < 0 || layout > 1) return fail(SPECQ_ERR_INVALID_ARG, "block_append: layout %d", layout);
  if (table != nullptr && (rot < 2 || rot > D || n_pos <= 0))
    return fail(SPECQ_ERR_INVALID_ARG, "block_append: rot=%d n_pos=%d", rot, n_pos);
  if (table != nullptr && rot % 16)
    return fail(SPECQ_ERR_UNSUPPORTED, "block_append: rot=%d must be a multiple of 16 (rope takes any even one)", rot);
  if (table == nullptr && (q != nullptr || pos != nullptr))
    return fail(SPECQ_ERR_INVALID_ARG, "block_append: queries and positions need a rotary table");
  const int b_grid = plan ? B : n_seqs;
  const int ql = plan ? ql_max : q_len;
  if (b_grid == 0 || ql == 0) return SPECQ_OK;
  if (k == nullptr || v == nullptr || kc == nullptr || vc == nullptr || ks == nullptr || vs == nullptr ||
      bt == nullptr || ctx == nullptr || (q != nullptr && q_out == nullptr))
    return fail(SPECQ_ERR_INVALID_ARG, "block_append: null pointer");
  if (!aligned(k, 8) || !aligned(v, 8) || kt % 4 || kh % 4 || vt % 4 || vh % 4)
    return fail(SPECQ_ERR_UNSUPPORTED, "block_append: K and V rows must be 8-byte aligned");
  if (!aligned(kc, 8) || !aligned(vc, 8) || kv_sp % 8 || kv_so % 8 || kv_sh % 8)
    return fail(SPECQ_ERR_UNSUPPORTED, "block_append: cache rows must be 8-byte aligned");
  if (table != nullptr && !aligned(table, 16)) return fail(SPECQ_ERR_UNSUPPORTED, "block_append: table not 16-byte aligned");
  if (q != nullptr && H > 0 && (!aligned(q, 16) || !aligned(q_out, 16) || qt % 8 || qh % 8 || ot % 8 || oh % 8))
    return fail(SPECQ_ERR_UNSUPPORTED, "block_append: query rows must be 16-byte aligned");
  if (q != nullptr && q == q_out && (qt != ot || qh != oh))
    return fail(SPECQ_ERR_INVALID_ARG, "block_append: in place, the strides of q and q_out must be the same");
  if (static_cast<int64_t>(b_grid) * ql > 0x7FFFFFFFll) return fail(SPECQ_ERR_UNSUPPORTED, "block_append: too many tokens");
  DeviceState* dev = nullptr;
  if (int rc = get_device_state(&dev)) return rc;
  BlockAppendParams p = {};
  p.k = k; p.v = v; p.q = q; p.q_out = q_out; p.table = table; p.pos = pos;
  p.kc = static_cast<uint8_t*>(kc); p.vc = static_cast<uint8_t*>(vc); p.ks = ks; p.vs = vs;
  p.bt = bt; p.ctx = ctx; p.plan = plan; p.status = dev->status;
  p.kt = kt; p.kh = kh; p.vt = vt; p.vh = vh; p.qt = qt; p.qh = qh; p.ot = ot; p.oh = oh;
  p.kv_sp = kv_sp; p.kv_so = kv_so; p.kv_sh = kv_sh; p.s_sp = s_sp; p.s_sh = s_sh; p.bt_sb = bt_sb;
  p.n_seqs = n_seqs; p.q_len = q_len; p.b_grid = b_grid; p.ql_max = ql; p.h_kv = H_KV; p.h_q = H;
  p.page_log2 = __builtin_ctz(static_cast<unsigned>(page));
  p.n_pages = n_pages; p.bt_cols = bt_cols; p.rot = rot; p.n_pos = n_pos; p.half = layout == 0;
  p.wide = aligned(k, 16) && aligned(v, 16) && kt % 8 == 0 && kh % 8 == 0 && vt % 8 == 0 && vh % 8 == 0;
  const int slots = append_slots(D, page);
  const int wpu = std::max(1, page / slots);
  p.n_win = (ql - 1) / page + 2;
  p.win_blocks = ceil_div(2 * H_KV, kAppendWarps / wpu);
  const int64_t kv_blocks = static_cast<int64_t>(b_grid) * p.n_win * p.win_blocks;
  int64_t q_blocks = 0;
  bool many = false;
  if (q != nullptr && H > 0) {
    const int64_t tokens = static_cast<int64_t>(b_grid) * ql;
    const bool tail = q_out != q;
    p.q_items = rope_items<__half>(D, rot, p.half != 0, tail);
    many = tokens * H * p.q_items >= static_cast<int64_t>(dev->sm_count) * 2048;
    p.q_groups = ceil_div(H, many ? kRopeHeads : 1);
    const int64_t threads = tokens * p.q_groups * p.q_items;
    if (threads > 0x7FFFFF00ll) return fail(SPECQ_ERR_UNSUPPORTED, "block_append: too many query rows");
    q_blocks = (threads + kAppendThreads - 1) / kAppendThreads;
  }
  if (kv_blocks + q_blocks > 0x7FFFFFFFll) return fail(SPECQ_ERR_UNSUPPORTED, "block_append: too many tokens");
  p.kv_blocks = static_cast<int>(kv_blocks);
  const dim3 grid(static_cast<unsigned>(kv_blocks + q_blocks));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto launch = [&](auto t, auto d, auto c, auto hp) -> cudaError_t {
    using T = decltype(t);
    constexpr int DD = decltype(d)::value, CT = decltype(c)::value, HP = decltype(hp)::value;
    if constexpr (DD == 128) {
      if (slots == 8) return launch_plain(block_append_kernel<T, DD, CT, 8, HP>, grid, dim3(kAppendThreads), st, p);
    }
    return launch_plain(block_append_kernel<T, DD, CT, 16, HP>, grid, dim3(kAppendThreads), st, p);
  };
  auto by_hp = [&](auto t, auto d, auto c) {
    return many ? launch(t, d, c, std::integral_constant<int, kRopeHeads>{}) : launch(t, d, c, std::integral_constant<int, 1>{});
  };
  auto by_cache = [&](auto t, auto d) {
    return cache_dtype == SPECQ_CACHE_INT8 ? by_hp(t, d, std::integral_constant<int, 0>{})
                                           : by_hp(t, d, std::integral_constant<int, 1>{});
  };
  auto by_dim = [&](auto t) {
    return D == 64 ? by_cache(t, std::integral_constant<int, 64>{}) : by_cache(t, std::integral_constant<int, 128>{});
  };
  SPECQ_CUDA_TRY(dtype == 0 ? by_dim(__half{}) : by_dim(__nv_bfloat16{}));
  return SPECQ_OK;
}

struct BlockCompactParams {
  uint8_t* kc;
  uint8_t* vc;
  float* ks;
  float* vs;
  const int32_t* bt;
  const int32_t* ctx;
  const int32_t* accept;   // [B, A]
  const int32_t* n_accept; // [B]
  int32_t* ctx_out;        // [B]
  int* status;
  int64_t kv_sl, kv_sp, kv_so, kv_sh, s_sl, s_sp, s_sh, bt_sb, acc_sb;
  int L, B, h_kv, q_len, acc_cols, page_log2, n_pages, bt_cols;
};

constexpr int kCompactThreads = 128;
constexpr int kCompactTokens = 64;   // accepted ones, whose indices a warp holds, two a lane

// The indices, page numbers and scales of a warp's drafts stand in its lanes' registers, so the
// chain of dependent loads is: lengths and indices; page numbers; scales and tokens.  Up to 16
// (D = 128) or 32 (D = 64) moving tokens are read once, before the first is written.
template <int D, int CT>
__global__ void __launch_bounds__(kCompactThreads) block_compact_kernel(const __grid_constant__ BlockCompactParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t id = (blockIdx.x * kCompactThreads + threadIdx.x) >> 5;
  const int lane = static_cast<int>(threadIdx.x & 31);
  const uint32_t hu = 2u * p.h_kv;
  const uint32_t lb = id / hu;
  const int unit = static_cast<int>(id - lb * hu);
  const int layer = static_cast<int>(lb / static_cast<uint32_t>(p.B));
  const int b = static_cast<int>(lb - static_cast<uint32_t>(layer) * p.B);
  if (layer >= p.L) return;
  const int page = 1 << p.page_log2, mask = page - 1;
  const bool first_unit = layer == 0 && unit == 0 && lane == 0;
  const int32_t* acc = p.accept + b * p.acc_sb;
  const int a0 = lane < p.acc_cols ? __ldg(acc + lane) : 0;
  const int a1 = lane + 32 < p.acc_cols ? __ldg(acc + lane + 32) : 0;
  const int ctx = p.ctx[b];
  const int n_raw = __ldg(p.n_accept + b);
  const int base = ctx - p.q_len;
  const int n = min(max(n_raw, 0), min(p.acc_cols, p.q_len));
  const bool in_table = base >= 0 && ctx <= p.bt_cols * page;
  // the drafts' pages, one a lane
  const int col0 = base >> p.page_log2, n_win = ((ctx - 1) >> p.page_log2) - col0 + 1;
  int pg = 0;
  if (in_table && lane < n_win) pg = p.bt[b * p.bt_sb + col0 + lane];
  // accept must grow strictly within the drafts, the drafts lie in the table on pages of the cache
  const int before0 = __shfl_up_sync(0xffffffffu, a0, 1), last0 = __shfl_sync(0xffffffffu, a0, 31);
  const int before1 = __shfl_up_sync(0xffffffffu, a1, 1);
  const bool good0 = lane >= n || (a0 > (lane == 0 ? -1 : before0) && a0 < p.q_len);
  const bool good1 = lane + 32 >= n || (a1 > (lane == 0 ? last0 : before1) && a1 < p.q_len);
  const unsigned moves0 = __ballot_sync(0xffffffffu, lane < n && a0 != lane);
  const unsigned moves1 = __ballot_sync(0xffffffffu, lane + 32 < n && a1 != lane + 32);
  // leading tokens that already stand where they belong
  const int same = moves0 != 0u ? __ffs(moves0) - 1 : moves1 != 0u ? 31 + __ffs(moves1) : n;
  bool ok = in_table && n == n_raw && __all_sync(0xffffffffu, good0 && good1);
  if (same < n) ok = ok && __all_sync(0xffffffffu, lane >= n_win || (pg >= 0 && pg < p.n_pages));
  if (first_unit) {
    p.ctx_out[b] = ok ? base + n : ctx;
    if (!ok) report_status(p.status, SPECQ_STATUS_BAD_INDEX);
  }
  if (!ok || same == n) return;   // not ok: nothing of this sequence moves

  const bool is_v = unit >= p.h_kv;
  const int head = is_v ? unit - p.h_kv : unit;
  uint8_t* cache = (is_v ? p.vc : p.kc) + layer * p.kv_sl + head * p.kv_sh;
  float* scale = (is_v ? p.vs : p.ks) + layer * p.s_sl + head * p.s_sh;
  float sc = 0.f;                                // of window page `lane`
  if (lane < n_win) sc = scale[static_cast<int64_t>(pg) * p.s_sp];
  constexpr int LPT = D / 16, TPS = 32 / LPT;    // lanes of a token (16 bytes each), tokens of a step
  constexpr int BATCH = 4;                       // steps in flight
  const int sub = lane / LPT;
  const int byte = (lane % LPT) * 16;

  uint4 w[BATCH];
  int swin[BATCH];
  auto load = [&](int jb, int end) {
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int j = jb + i * TPS + sub;
      const int lo = __shfl_sync(0xffffffffu, a0, j & 31), hi = __shfl_sync(0xffffffffu, a1, j & 31);
      const int pos = base + (j < 32 ? lo : hi);
      const int win = j < end ? (pos >> p.page_log2) - col0 : 0;
      const int spg = __shfl_sync(0xffffffffu, pg, win);
      swin[i] = win;
      w[i] = make_uint4(0u, 0u, 0u, 0u);
      if (j < end)
        w[i] = *reinterpret_cast<const uint4*>(cache + static_cast<int64_t>(spg) * p.kv_sp +
                                               static_cast<int64_t>(pos & mask) * p.kv_so + byte);
    }
  };
  // few enough tokens: all are read at once, for every target page
  const bool once = n - same <= BATCH * TPS;
  if (once) load(same, n);
  for (int j0 = same; j0 < n;) {
    const int dpos = base + j0;
    const int dwin = (dpos >> p.page_log2) - col0;
    const int j1 = min(n, ((col0 + dwin + 1) << p.page_log2) - base);   // this target page takes tokens j0 .. j1 - 1
    uint8_t* dst = cache + static_cast<int64_t>(__shfl_sync(0xffffffffu, pg, dwin)) * p.kv_sp;
    const float s_old = __shfl_sync(0xffffffffu, sc, dwin);
    // the arriving tokens' need; a number is at most q_max, so those of pages whose scale is no larger
    // (the page itself among them) fit already
    float need = 0.f;
    const int jf = once ? same : j0;             // the first batch's first token
    for (int jb = jf; jb < j1; jb += BATCH * TPS) {
      if (!once) load(jb, j1);
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const float ss = __shfl_sync(0xffffffffu, sc, swin[i]);
        const int j = jb + i * TPS + sub;
        if (j >= j0 && j < j1 && ss > s_old) need = fmaxf(need, absmax16<CT>(w[i]) * cache_inv_max<CT>() * ss);
      }
    }
    need = warp_max_f32(need);
    const float s_new = fmaxf(s_old, need);
    if (s_new > s_old) {        // what the page held before the arriving tokens
      const float r = __fdiv_rn(s_old, s_new);
      const int keep = dpos & mask;
      for (int slot = sub; slot < keep; slot += TPS) {
        uint4* d = reinterpret_cast<uint4*>(dst + static_cast<int64_t>(slot) * p.kv_so + byte);
        uint4 x = *d;
        x.x = requant4<CT>(x.x, r); x.y = requant4<CT>(x.y, r);
        x.z = requant4<CT>(x.z, r); x.w = requant4<CT>(x.w, r);
        *d = x;
      }
    }
    for (int jb = jf; jb < j1; jb += BATCH * TPS) {
      if (!once && j1 - j0 > BATCH * TPS) load(jb, j1);   // otherwise they are in the registers still
      __syncwarp();             // every read of the batch before its writes
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const int j = jb + i * TPS + sub;
        const float ss = __shfl_sync(0xffffffffu, sc, swin[i]);
        if (j >= j0 && j < j1) {
          uint4 x = w[i];
          if (ss != s_new) {
            const float r = __fdiv_rn(ss, s_new);
            x.x = requant4<CT>(x.x, r); x.y = requant4<CT>(x.y, r);
            x.z = requant4<CT>(x.z, r); x.w = requant4<CT>(x.w, r);
          }
          *reinterpret_cast<uint4*>(dst + static_cast<int64_t>((base + j) & mask) * p.kv_so + byte) = x;
        }
      }
      __syncwarp();
    }
    if (lane == dwin && s_new != s_old) scale[static_cast<int64_t>(pg) * p.s_sp] = s_new;
    j0 = j1;
  }
}

inline int run_block_compact(void* kc, void* vc, int64_t kv_sl, int64_t kv_sp, int64_t kv_so, int64_t kv_sh,
                             int cache_dtype, int L, int n_pages, float* ks, float* vs, int64_t s_sl, int64_t s_sp,
                             int64_t s_sh, const int32_t* bt, int64_t bt_sb, int bt_cols, const int32_t* ctx,
                             const int32_t* accept, int64_t acc_sb, int acc_cols, const int32_t* n_accept,
                             int32_t* ctx_out, int B, int q_len, int H_KV, int D, int page, void* stream) {
  if (B < 0 || q_len < 0 || H_KV <= 0 || n_pages < 0 || bt_cols < 0 || L <= 0 || acc_cols < 0)
    return fail(SPECQ_ERR_INVALID_ARG, "block_compact: negative size");
  if (cache_dtype != SPECQ_CACHE_INT8 && cache_dtype != SPECQ_CACHE_E4M3)
    return fail(SPECQ_ERR_INVALID_ARG, "block_compact: cache dtype code %d", cache_dtype);
  if (D != 64 && D != 128) return fail(SPECQ_ERR_UNSUPPORTED, "block_compact: head_dim %d (this build supports 64 and 128)", D);
  if (!page_ok(page)) return fail(SPECQ_ERR_UNSUPPORTED, "block_compact: page %d (a power of two in 8..128)", page);
  if (acc_cols > kCompactTokens || (q_len - 1) / page + 2 > 32)
    return fail(SPECQ_ERR_UNSUPPORTED, "block_compact: %d accepted tokens > %d, or %d drafts over more than 32 pages of %d",
                acc_cols, kCompactTokens, q_len, page);
  if (B == 0) return SPECQ_OK;
  if (kc == nullptr || vc == nullptr || ks == nullptr || vs == nullptr || bt == nullptr || ctx == nullptr ||
      n_accept == nullptr || ctx_out == nullptr || (acc_cols > 0 && accept == nullptr))
    return fail(SPECQ_ERR_INVALID_ARG, "block_compact: null pointer");
  if (ctx == ctx_out) return fail(SPECQ_ERR_INVALID_ARG, "block_compact: ctx_out must not be ctx_len (every warp reads ctx_len)");
  if (!aligned(kc, 16) || !aligned(vc, 16) || kv_sl % 16 || kv_sp % 16 || kv_so % 16 || kv_sh % 16)
    return fail(SPECQ_ERR_UNSUPPORTED, "block_compact: cache rows must be 16-byte aligned");
  const int64_t warps = static_cast<int64_t>(L) * B * 2 * H_KV;
  if (warps > (0x7FFFFFFFll >> 5)) return fail(SPECQ_ERR_UNSUPPORTED, "block_compact: too many (layer, sequence, head) units");
  DeviceState* dev = nullptr;
  if (int rc = get_device_state(&dev)) return rc;
  BlockCompactParams p = {};
  p.kc = static_cast<uint8_t*>(kc); p.vc = static_cast<uint8_t*>(vc); p.ks = ks; p.vs = vs; p.bt = bt; p.ctx = ctx;
  p.accept = accept; p.n_accept = n_accept; p.ctx_out = ctx_out; p.status = dev->status;
  p.kv_sl = kv_sl; p.kv_sp = kv_sp; p.kv_so = kv_so; p.kv_sh = kv_sh;
  p.s_sl = s_sl; p.s_sp = s_sp; p.s_sh = s_sh; p.bt_sb = bt_sb; p.acc_sb = acc_sb;
  p.L = L; p.B = B; p.h_kv = H_KV; p.q_len = q_len; p.acc_cols = acc_cols;
  p.page_log2 = __builtin_ctz(static_cast<unsigned>(page));
  p.n_pages = n_pages; p.bt_cols = bt_cols;
  const dim3 grid(static_cast<unsigned>((warps + kCompactThreads / 32 - 1) / (kCompactThreads / 32)));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (cache_dtype == SPECQ_CACHE_INT8)
    e = D == 64 ? launch_plain(block_compact_kernel<64, 0>, grid, dim3(kCompactThreads), st, p)
                : launch_plain(block_compact_kernel<128, 0>, grid, dim3(kCompactThreads), st, p);
  else
    e = D == 64 ? launch_plain(block_compact_kernel<64, 1>, grid, dim3(kCompactThreads), st, p)
                : launch_plain(block_compact_kernel<128, 1>, grid, dim3(kCompactThreads), st, p);
  SPECQ_CUDA_TRY(e);
  return SPECQ_OK;
}

}  // namespace specq
