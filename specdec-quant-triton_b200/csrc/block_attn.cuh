// block_attn.cuh -- attention over the block-scaled 8-bit paged KV cache (block_cache.cuh).
//
// Row (b, qi, head) with L = ctx_len[b] sees cached token t when t <= L - q_len + qi, or, under
// a draft tree, when t < L - q_len or bit t - (L - q_len) of tree[b, qi] is set (and t < L).  A
// row that sees nothing is 0.
//
// Mathematics.  In log2 units, with x = (q . k8) * sK * sm_scale * log2(e) + log2(sV) and m the
// running maximum of x over the row,
//   p = 2^(x - m) = 2^(score - m) * sV,   O = sum p v8,   l = sum p / sV,   out = O / l,
// so neither scale costs a pass over a tile: sK is a factor of the exponent's fused
// multiply-add, sV part of its addend, and the normaliser divides by a number that is the same
// for a whole page.  p is rounded to fp16 for the tensor core; l sums the unrounded p in fp32.
// q is exact in fp16 (bf16 rows are first scaled by a power of two), and so are k8 and v8; the
// products accumulate in fp32.  m lags: p may reach 2^8 before the running maximum is raised
// (one warp vote a tile), which fp16 holds without loss.
//
// Tile.  A warp owns 16 tokens at a time and up to 24 query rows, and works alone:
//   S^T [16 tokens x rows] = K Q^T      mma.m16n8k16, K converted 8 -> 16 bits in registers
//   P^T = 2^(S^T - m)                   in the accumulator's registers
//   O^T [D x rows] += V^T P^T           P^T turned by movmatrix, V by a transposing ldmatrix
// Rows are the N side of both products, so they pad to 8 and not to 16 or 128.  Everything
// but the 8-bit tiles stays in registers; no barrier joins the warps inside the loop.  Tiles
// arrive by TMA (one box of 16 slots of a page for K, one for V) in a ring of its own for each
// group of warps that shares tokens; the lane that issues takes page numbers from a register
// file of the next 32 boxes, loaded a batch ahead with their scales.  Groups of more than 24
// rows split their rows over 2 or 4 warps that read the same ring; rows beyond 96 go to other
// blocks, which find the pages in L2.
//
// Why mma.sync: a 16-token tile is 16 x 8n x 128 twice, 16 n instructions.  The warp-level
// tensor pipe makes one every 2 cycles an SM (measured; 1024 multiply-adds a cycle), so one
// token costs 2 n cycles an SM for 8 n rows, against the 11.6 cycles in which HBM delivers its
// 256 bytes: up to 5 groups of 8 rows stay below the memory time, without the round trips
// through tensor memory and the block-wide hand-overs of a tcgen05 pipeline.
//
// Work.  The tiles of all (sequence, KV head, row chunk) segments form one line, cut into equal
// pieces, one for each resident block, whatever the sequences' lengths; each block finds its
// piece from ctx_len on the device.  A segment inside one piece is written at once; the parts of
// a cut one go to the workspace and a second, dependent launch joins them in the pieces' order.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "block_cache.cuh"
#include "sm100.cuh"
#include "specq_host.cuh"

namespace specq {

constexpr int kBAThreads = 256;
constexpr int kBAWarps = kBAThreads / 32;
constexpr int kBATok = 16;              // tokens of a warp's tile
constexpr int kBAMaxStages = 8;
constexpr float kBARaise = 8.f;         // log2 of how far p may pass 1 before the maximum is raised
constexpr float kBANone = -1e30f;        // the running maximum of a row that has seen no token: finite, so that a
                                         // masked score, -inf, less it is -inf and not NaN
constexpr float kBALeastV = 8.077935669463161e-28f;   // 2^-90: a smaller V scale reads as this

struct BlockAttnParams {
  const void* q;
  void* out;
  const float* ks;
  const float* vs;
  const int32_t* bt;
  const int32_t* ctx;
  const uint64_t* tree;     // optional [B, q_len] bit sets
  const int32_t* plan;      // plan[0] = n_seqs, plan[1] = q_len
  float* part_o;            // [2 grid][rows][D]
  float* part_ml;           // [2 grid][rows][2]
  int* status;
  int64_t q_sb, q_st, q_sh, o_sb, o_st, o_sh, s_sp, s_sh, bt_sb, tree_sb, tree_st;
  float scale_log2;         // sm_scale * log2(e)
  int n_seqs, q_len, b_max, ql_max, h_kv, group, page_log2, n_pages, bt_cols;
  int bf16, stages, grid, rows, tile;   // rows: of a block's chunk; tile: tokens of a block's tile
};

__device__ __forceinline__ void tma_box(void* dst, const CUtensorMap* map, uint64_t* bar, int head, int slot, int page) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(0), "r"(head), "r"(slot), "r"(page)
      : "memory");
}

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t movm_t(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Bytes 0..3 of w as two half2: (0, 1) and (2, 3), or with SPLIT (0, 2) and (1, 3).
// int8: byte ^ 0x80 becomes the low byte of 1024 + u, and 1024 + u - 1152 = the signed value,
// exactly.  e4m3: the conversion instruction, exact.
template <int CT, bool SPLIT>
__device__ __forceinline__ void widen4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (CT == 0) {
    const uint32_t u = w ^ 0x80808080u;
    const uint32_t a = __byte_perm(u, 0x64646464u, SPLIT ? 0x4240 : 0x4140);
    const uint32_t b = __byte_perm(u, 0x64646464u, SPLIT ? 0x4341 : 0x4342);
    const __half2 off = __half2(__half_raw{0x6480}, __half_raw{0x6480});   // 1152
    const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), off);
    const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&b), off);
    lo = *reinterpret_cast<const uint32_t*>(&x);
    hi = *reinterpret_cast<const uint32_t*>(&y);
  } else {
    const uint32_t u = SPLIT ? __byte_perm(w, 0u, 0x3120) : w;
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(u));
  }
}

// Where the segments of a call lie on the line of tiles.
struct BALine {
  int n_seqs, q_len, q_rows, rc;   // rc: row chunks of a (sequence, KV head)
  int chunk_rows;                  // rows of a chunk (a multiple of 8)
  int64_t total;                   // tiles in all
};

__device__ __forceinline__ int ba_ctx(const BlockAttnParams& p, int b) {
  const int c = __ldg(p.ctx + b);
  return min(max(c, 0), p.bt_cols << p.page_log2);
}
__device__ __forceinline__ int ba_tiles(const BlockAttnParams& p, int ctx) { return max(1, (ctx + p.tile - 1) / p.tile); }

__device__ __forceinline__ BALine ba_line(const BlockAttnParams& p, bool tell) {
  BALine a;
  a.n_seqs = p.n_seqs;
  a.q_len = p.q_len;
  if (p.plan != nullptr) {
    const int n = __ldg(p.plan), q = __ldg(p.plan + 1);
    a.n_seqs = min(max(n, 0), p.b_max);
    a.q_len = min(max(q, 0), p.ql_max);
    if (tell && (n != a.n_seqs || q != a.q_len)) report_status(p.status, SPECQ_STATUS_PLAN_CLAMPED);
  }
  a.q_rows = a.q_len * p.group;
  const int groups = (a.q_rows + 7) >> 3;
  a.rc = (groups * 8 + p.rows - 1) / p.rows;
  a.chunk_rows = a.rc > 0 ? (groups + a.rc - 1) / a.rc * 8 : 0;
  int64_t t = 0;
  const int lane = static_cast<int>(threadIdx.x & 31);
  for (int b0 = 0; b0 < a.n_seqs; b0 += 32) {
    const int b = b0 + lane;
    int n = 0;
    if (b < a.n_seqs) {
      const int c = __ldg(p.ctx + b);
      if (tell && (c < 0 || c > (p.bt_cols << p.page_log2))) report_status(p.status, SPECQ_STATUS_PLAN_CLAMPED);
      n = ba_tiles(p, ba_ctx(p, b));
    }
    t += __reduce_add_sync(0xffffffffu, n);
  }
  a.total = t * (p.h_kv * a.rc);
  return a;
}

// The sequence that holds line position u (every lane of the warp calls), and where it begins.
__device__ __forceinline__ int ba_find(const BlockAttnParams& p, const BALine& a, int64_t u, int64_t* begin) {
  const int lane = static_cast<int>(threadIdx.x & 31);
  const int per = p.h_kv * a.rc;
  int64_t at = 0;
  for (int b0 = 0; b0 < a.n_seqs; b0 += 32) {
    const int b = b0 + lane;
    const int n = b < a.n_seqs ? ba_tiles(p, ba_ctx(p, b)) : 0;
    int inc = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, inc, d);
      if (lane >= d) inc += up;
    }
    const int64_t end = at + static_cast<int64_t>(inc) * per;
    const unsigned over = __ballot_sync(0xffffffffu, b < a.n_seqs && end > u);
    if (over != 0u) {
      const int first = __ffs(over) - 1;
      *begin = at + static_cast<int64_t>(__shfl_sync(0xffffffffu, inc - n, first)) * per;
      return b0 + first;
    }
    at += static_cast<int64_t>(__shfl_sync(0xffffffffu, inc, 31)) * per;
  }
  *begin = at;
  return a.n_seqs;
}

__device__ __forceinline__ void ba_store(const BlockAttnParams& p, int64_t off, float a, float b, float c, float d) {
  if (p.bf16) {
    const __nv_bfloat162 x = __floats2bfloat162_rn(a, b), y = __floats2bfloat162_rn(c, d);
    *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.out) + off) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
  } else {
    const __half2 x = __floats2half2_rn(a, b), y = __floats2half2_rn(c, d);
    *reinterpret_cast<uint2*>(static_cast<__half*>(p.out) + off) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
  }
}

// Row rr of (sequence b, KV head h) in out, in elements.  o_sb = 0: packed token rows.
__device__ __forceinline__ int64_t ba_out_at(const BlockAttnParams& p, const BALine& a, int b, int h, int rr) {
  const int qi = rr / p.group, g = rr - qi * p.group;
  const int64_t tok = p.o_sb == 0 ? static_cast<int64_t>(b) * a.q_len + qi : qi;
  return b * p.o_sb + tok * p.o_st + static_cast<int64_t>(h * p.group + g) * p.o_sh;
}

// One block's view of the segment it works on.
struct BASeg {
  int b, h, row_lo;        // sequence, KV head, first row of the chunk
  int ctx, old;            // tokens; tokens before the drafts (every row sees them)
  int ta, tb, nt;          // tiles of this piece, tiles of the segment
};

// A group's place in its ring, carried from segment to segment.
struct BARing {
  uint64_t* full;          // [stages]
  uint64_t* empty;
  uint8_t* base;
  int get, put;            // next stage to read, to fill
  uint32_t get_ph, put_ph; // their phases
  bool ok;                 // no wait has run out
};

// One warp's part of a segment: its rows (NT groups of 8 from row lr0 of the chunk, nts of them
// in use), its group's tokens; leaves its part of O in the merge buffer, m and l beside it.
template <int D, int CT, int NT, int RG>
__device__ __forceinline__ void ba_segment(const BlockAttnParams& p, const CUtensorMap& mk, const CUtensorMap& mv,
                                           const BALine& a, const BASeg& sg, BARing& ring, int tg, int rg, int lr0, int nts,
                                           float* sm_m, float* sm_l, float* merge) {
  constexpr int TG = kBAWarps / RG;
  constexpr int KC = D / 16;                 // 16-byte pieces of a token
  constexpr int KB = kBATok * D;             // bytes of a K (or V) tile
  constexpr int PITCH = D + 12;              // of the merge buffer, in floats: its stores hit each bank once
  const int lane = static_cast<int>(threadIdx.x & 31);
  const int gq = lane >> 2, tq = lane & 3;
  const int stages = p.stages;

  // ---- boxes: box e of the group's tile i (page 8: two boxes a tile) and their registers
  const int two = p.page_log2 == 3 ? 1 : 0;
  const int first_tok = sg.ta * p.tile + tg * kBATok;
  int n_tiles = sg.tb - sg.ta;                                 // of this group, those with a token
  if (n_tiles > 0 && first_tok + (n_tiles - 1) * p.tile >= sg.ctx) --n_tiles;
  const int boxes = n_tiles << two;
  const int32_t* bt = p.bt + sg.b * p.bt_sb;
  int pg_c = 0, pg_n = 0;
  float ck_c = 0.f, lv_c = 0.f, iv_c = 0.f, ck_n = 0.f, lv_n = 0.f, iv_n = 0.f;
  auto load_batch = [&](int e0, int& pg, float& ck, float& lv, float& iv) {
    const int e = e0 + lane;
    pg = 0;
    ck = 1e-37f; lv = -INFINITY; iv = 0.f;     // a box that is not there weighs nothing
    if (e < boxes) {
      const int tok = first_tok + (e >> two) * p.tile + (two ? (e & 1) * 8 : 0);
      if (tok < sg.ctx) {
        const int x = __ldg(bt + (tok >> p.page_log2));
        if (x >= 0 && x < p.n_pages) {
          pg = x;
          const int64_t at = static_cast<int64_t>(x) * p.s_sp + sg.h * p.s_sh;
          ck = __ldg(p.ks + at) * p.scale_log2;
          if (ck < 1e-37f) ck = 1e-37f;        // a masked score, -inf, times it stays -inf
          float v = __ldg(p.vs + at);
          v = v < kBALeastV ? kBALeastV : v;
          lv = __log2f(v);
          iv = 1.f / v;
        } else {
          report_status(p.status, SPECQ_STATUS_BAD_INDEX);
        }
      }
    }
  };
  load_batch(0, pg_c, ck_c, lv_c, iv_c);
  load_batch(32, pg_n, ck_n, lv_n, iv_n);
  int batch0 = 0;                                              // first box of the current batch

  auto issue = [&](int i) {                                    // tile i into the next stage (rg 0's warp)
    const int e = i << two;
    const int pg = e - batch0 < 32 ? pg_c : pg_n;
    const int p0 = __shfl_sync(0xffffffffu, pg, e & 31);
    const int p1 = two ? __shfl_sync(0xffffffffu, pg, (e + 1) & 31) : 0;
    if (RG > 1)
      ring.ok = ring.ok && mbar_wait(&ring.empty[ring.put], ring.put_ph ^ 1u, p.status, SPECQ_STATUS_TIMEOUT_PIPELINE);
    if (lane == 0 && ring.ok) {
      uint8_t* d = ring.base + ring.put * 2 * KB;
      uint64_t* bar = &ring.full[ring.put];
      const int slot = two ? 0 : (first_tok + i * p.tile) & ((1 << p.page_log2) - 1);
      mbar_arrive_expect_tx(bar, 2 * KB);
      tma_box(d, &mk, bar, sg.h, slot, p0);
      tma_box(d + KB, &mv, bar, sg.h, slot, p0);
      if (two) {
        tma_box(d + KB / 2, &mk, bar, sg.h, 0, p1);
        tma_box(d + KB + KB / 2, &mv, bar, sg.h, 0, p1);
      }
    }
    __syncwarp();
    if (++ring.put == stages) {
      ring.put = 0;
      ring.put_ph ^= 1u;
    }
  };
  if (rg == 0)
    for (int i = 0; i < min(stages - 1, n_tiles); ++i) issue(i);

  // ---- Q^T as the B operand: thread (gq, tq) holds row gq of each group, d = 16 c + 4 tq + 0..3
  uint32_t qf[NT][KC][2];
  float fac = 1.f;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int lr = lr0 + n * 8 + gq;
    const int rr = sg.row_lo + lr;
#pragma unroll
    for (int c = 0; c < KC; ++c) qf[n][c][0] = qf[n][c][1] = 0u;
    if (n < nts && lr < a.chunk_rows && rr < a.q_rows) {
      const int qi = rr / p.group, g = rr - qi * p.group;
      const int64_t tok = p.q_sb == 0 ? static_cast<int64_t>(sg.b) * a.q_len + qi : qi;
      const int64_t off = sg.b * p.q_sb + tok * p.q_st + static_cast<int64_t>(sg.h * p.group + g) * p.q_sh;
      const uint2* src = reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p.q) + off + 4 * tq);
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        const uint2 w = __ldg(src + 4 * c);
        qf[n][c][0] = w.x;
        qf[n][c][1] = w.y;
      }
    }
  }
  if (p.bf16) {
    // to fp16 under one power of two that brings the warp's largest to [1, 2): bf16's 8 bits are
    // exact down to 2^-17 of it, and what is smaller is off by 2^-25 of it at most
    float top = 0.f;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < KC; ++c)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          top = fmaxf(top, fmaxf(fabsf(__uint_as_float(qf[n][c][i] << 16)), fabsf(__uint_as_float(qf[n][c][i] & 0xffff0000u))));
    top = warp_max_f32(top);
    const uint32_t ex = min(max(__float_as_uint(top) >> 23, 1u), 253u);
    fac = __uint_as_float(ex << 23);
    const float inv = __uint_as_float((254u - ex) << 23);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < KC; ++c)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const __half2 y = __floats2half2_rn(__uint_as_float(qf[n][c][i] << 16) * inv,
                                              __uint_as_float(qf[n][c][i] & 0xffff0000u) * inv);
          qf[n][c][i] = *reinterpret_cast<const uint32_t*>(&y);
        }
  }

  float o[KC][NT][4], m[NT][2], l[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    m[n][0] = m[n][1] = kBANone;
    l[n][0] = l[n][1] = 0.f;
#pragma unroll
    for (int c = 0; c < KC; ++c) o[c][n][0] = o[c][n][1] = o[c][n][2] = o[c][n][3] = 0.f;
  }
  // this lane's ldmatrix row: matrix lane / 8 = (token half, piece), swizzled as the box was stored
  const int mr = (lane & 7) + ((lane >> 3) & 1) * 8, mc = lane >> 4;
  const uint32_t row_off = static_cast<uint32_t>(mr * D + ((mc ^ (D == 128 ? (mr & 7) : ((mr >> 1) & 3))) << 4));
  const uint32_t ring_s = smem_u32(ring.base) + row_off;

  for (int i = 0; i < n_tiles; ++i) {
    const int e = (i << two) & 31;
    if (e == 0 && i > 0) {                                      // the next batch of boxes
      batch0 += 32;
      pg_c = pg_n; ck_c = ck_n; lv_c = lv_n; iv_c = iv_n;
      load_batch(batch0 + 32, pg_n, ck_n, lv_n, iv_n);
    }
    if (rg == 0 && i + stages - 1 < n_tiles) issue(i + stages - 1);
    const int s = ring.get;
    ring.ok = ring.ok && mbar_wait(&ring.full[s], ring.get_ph, p.status, SPECQ_STATUS_TIMEOUT_PIPELINE);
    if (++ring.get == stages) {
      ring.get = 0;
      ring.get_ph ^= 1u;
    }
    const uint32_t kt = ring_s + static_cast<uint32_t>(s * 2 * KB), vt = kt + KB;

    // S^T = K Q^T
    float sc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
#pragma unroll
    for (int c = 0; c < KC; c += 2) {
      uint32_t r[4];
      ldsm4(kt ^ static_cast<uint32_t>(c << 4), r);
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        uint32_t l0, h0, l1, h1;
        widen4<CT, false>(r[2 * hf], l0, h0);
        widen4<CT, false>(r[2 * hf + 1], l1, h1);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma16816(sc[n], l0, l1, h0, h1, qf[n][c + hf][0], qf[n][c + hf][1]);
      }
    }

    // softmax of the tile: rows 2 tq, 2 tq + 1 of each group, tokens gq and gq + 8
    const float ck = __shfl_sync(0xffffffffu, ck_c, e) * fac;
    const float lv = __shfl_sync(0xffffffffu, lv_c, e);
    const float iv = __shfl_sync(0xffffffffu, iv_c, e);
    float lv1 = lv, iv_rel = 1.f;                               // tokens 8 .. 15: the same page, or
    if (two) {                                                  // another one with its own scales
      const float ck1 = __shfl_sync(0xffffffffu, ck_c, e + 1) * fac;
      lv1 = __shfl_sync(0xffffffffu, lv_c, e + 1);
      const float iv1 = __shfl_sync(0xffffffffu, iv_c, e + 1);
      const float rel = ck1 / ck;
      iv_rel = iv > 0.f ? iv1 / iv : 0.f;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        sc[n][2] *= rel;
        sc[n][3] *= rel;
      }
    }
    const int t0 = first_tok + i * p.tile;
    if (t0 + kBATok > sg.old) {                                 // some row may not see some token
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int rr = sg.row_lo + lr0 + n * 8 + 2 * tq + r;
          const int qi = rr / p.group;
          if (p.tree == nullptr) {
            const int lim = min(sg.ctx, sg.old + qi + 1);
            if (t0 + gq >= lim) sc[n][r] = -INFINITY;
            if (t0 + gq + 8 >= lim) sc[n][2 + r] = -INFINITY;
          } else {
            const uint64_t word = qi < a.q_len ? __ldg(reinterpret_cast<const unsigned long long*>(p.tree) + sg.b * p.tree_sb + qi * p.tree_st) : 0ull;
            const int j0 = t0 + gq - sg.old, j1 = j0 + 8;
            if (j0 >= a.q_len || (j0 >= 0 && ((word >> (j0 & 63)) & 1ull) == 0ull)) sc[n][r] = -INFINITY;
            if (j1 >= a.q_len || (j1 >= 0 && ((word >> (j1 & 63)) & 1ull) == 0ull)) sc[n][2 + r] = -INFINITY;
          }
        }
      if (CT == 1 && t0 + kBATok > sg.ctx) {
        // slots past the last token may hold anything, NaN bytes too: their V reads as 0
        uint8_t* v = ring.base + s * 2 * KB + KB;
        for (int x = max(sg.ctx - t0, 0) * KC + lane; x < kBATok * KC; x += 32) *reinterpret_cast<uint4*>(v + x * 16) = make_uint4(0u, 0u, 0u, 0u);
        fence_proxy_async_smem();                               // before the stage is filled again
        __syncwarp();
      }
    }
    // x - m in log2 units, x = score + log2(sV)
    float y[NT][4], top = -INFINITY;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        y[n][r] = fmaf(sc[n][r], ck, lv - m[n][r]);
        y[n][2 + r] = fmaf(sc[n][2 + r], ck, lv1 - m[n][r]);
        top = fmaxf(top, fmaxf(y[n][r], y[n][2 + r]));
      }
    if (__any_sync(0xffffffffu, top > kBARaise)) {              // raise the maxima and what they scale
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float x0 = fmaf(sc[n][r], ck, lv), x1 = fmaf(sc[n][2 + r], ck, lv1);
          float v = fmaxf(x0, x1);
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
          const float mn = fmaxf(m[n][r], v);
          const float f = ex2(m[n][r] - mn);
          m[n][r] = mn;
          l[n][r] *= f;
#pragma unroll
          for (int c = 0; c < KC; ++c) {
            o[c][n][r] *= f;
            o[c][n][2 + r] *= f;
          }
          y[n][r] = x0 - mn;
          y[n][2 + r] = x1 - mn;
        }
    }
    uint32_t pb[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        y[n][r] = ex2(y[n][r]);
        y[n][2 + r] = ex2(y[n][2 + r]);
        l[n][r] = fmaf(fmaf(y[n][2 + r], iv_rel, y[n][r]), iv, l[n][r]);
      }
      const __half2 h0 = __floats2half2_rn(y[n][0], y[n][1]), h1 = __floats2half2_rn(y[n][2], y[n][3]);
      pb[n][0] = movm_t(*reinterpret_cast<const uint32_t*>(&h0));
      pb[n][1] = movm_t(*reinterpret_cast<const uint32_t*>(&h1));
    }

    // O^T += V^T P^T
#pragma unroll
    for (int c = 0; c < KC; c += 2) {
      uint32_t r[4];
      ldsm4_t(vt ^ static_cast<uint32_t>(c << 4), r);
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        uint32_t e0, d0, e1, d1;
        widen4<CT, true>(r[2 * hf], e0, d0);
        widen4<CT, true>(r[2 * hf + 1], e1, d1);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma16816(o[c + hf][n], e0, d0, e1, d1, pb[n][0], pb[n][1]);
      }
    }
    __syncwarp();                                               // every lane has read the stage
    if (RG > 1 && lane == 0) mbar_arrive(&ring.empty[s]);
  }

  // ---- this warp's part of the join
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float v = l[n][r];
      v += __shfl_xor_sync(0xffffffffu, v, 4);
      v += __shfl_xor_sync(0xffffffffu, v, 8);
      v += __shfl_xor_sync(0xffffffffu, v, 16);
      const int lr = lr0 + n * 8 + 2 * tq + r;
      if (gq == 0 && n < nts) {
        sm_m[tg * p.rows + lr] = m[n][r];
        sm_l[tg * p.rows + lr] = v;
      }
    }
  named_barrier_sync(1, kBAThreads);                            // also: every group is done with the ring
#pragma unroll
  for (int n = 0; n < NT; ++n)
    if (n < nts) {
      float f[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int lr = lr0 + n * 8 + 2 * tq + r;
        float top = -INFINITY;
#pragma unroll
        for (int t = 0; t < TG; ++t) top = fmaxf(top, sm_m[t * p.rows + lr]);
        f[r] = ex2(m[n][r] - top);
      }
      float* d0 = merge + (tg * p.rows + lr0 + n * 8 + 2 * tq) * PITCH + 2 * gq;
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        *reinterpret_cast<float2*>(d0 + 16 * c) = make_float2(o[c][n][0] * f[0], o[c][n][2] * f[0]);
        *reinterpret_cast<float2*>(d0 + PITCH + 16 * c) = make_float2(o[c][n][1] * f[1], o[c][n][3] * f[1]);
      }
    }
}

template <int D, int CT, int NT, int RG>
__global__ void __launch_bounds__(kBAThreads, NT == 1 ? 2 : 1)
block_attn_kernel(const __grid_constant__ BlockAttnParams p, const __grid_constant__ CUtensorMap mk,
                  const __grid_constant__ CUtensorMap mv) {
  constexpr int TG = kBAWarps / RG;          // groups of warps with tokens of their own
  constexpr int KB = kBATok * D;
  constexpr int ROWS = RG * NT * 8;
  constexpr int PITCH = D + 12;
  extern __shared__ uint8_t smem_raw[];
  __shared__ float sm_m[TG * ROWS], sm_l[TG * ROWS];
  __shared__ __align__(8) uint64_t full[TG][kBAMaxStages], empty[TG][kBAMaxStages];
  uint8_t* base = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  float* merge = reinterpret_cast<float*>(base);

  const int warp = static_cast<int>(threadIdx.x >> 5), lane = static_cast<int>(threadIdx.x & 31);
  const int tg = warp % TG, rg = warp / TG;
  const int stages = p.stages;
  if (threadIdx.x == 0) {
    for (int t = 0; t < TG; ++t)
      for (int s = 0; s < stages; ++s) {
        mbar_init(&full[t][s], 1u);
        mbar_init(&empty[t][s], RG);
      }
    fence_barrier_init();
    tma_prefetch_desc(&mk);
    tma_prefetch_desc(&mv);
  }
  __syncthreads();
  pdl_wait();

  const BALine a = ba_line(p, blockIdx.x == 0 && warp == 0);
  const int64_t u0 = a.total * blockIdx.x / p.grid, u1 = a.total * (blockIdx.x + 1) / p.grid;
  BARing ring = {full[tg], empty[tg], base + tg * stages * 2 * KB, 0, 0, 0u, 0u, true};
  BASeg sg = {};
  int64_t seq_begin = 0;
  if (u0 < u1) sg.b = ba_find(p, a, u0, &seq_begin);
  for (int64_t u = u0; u < u1;) {
    sg.ctx = ba_ctx(p, sg.b);
    sg.old = sg.ctx - a.q_len;
    sg.nt = ba_tiles(p, sg.ctx);
    const int in_seq = static_cast<int>(u - seq_begin);
    const int hr = in_seq / sg.nt;                             // (KV head, row chunk)
    sg.ta = in_seq - hr * sg.nt;
    sg.h = hr / a.rc;
    sg.row_lo = (hr - sg.h * a.rc) * a.chunk_rows;
    const int64_t seg_begin = u - sg.ta;
    sg.tb = static_cast<int>(min(static_cast<int64_t>(sg.nt), u1 - seg_begin));

    // rows of this warp: groups of 8 dealt evenly over the RG warps, so NT or NT - 1 (fewer only
    // under a plan whose q_len is below the largest: the spare groups then compute on zeros)
    const int groups = min(a.chunk_rows, a.q_rows - sg.row_lo + 7) >> 3;
    const int nts = groups / RG + (rg < groups % RG ? 1 : 0);
    const int lr0 = 8 * (rg * (groups / RG) + min(rg, groups % RG));
    if (NT == 1 || RG == 1 || nts == NT)
      ba_segment<D, CT, NT, RG>(p, mk, mv, a, sg, ring, tg, rg, lr0, nts, sm_m, sm_l, merge);
    else
      ba_segment<D, CT, NT == 1 ? 1 : NT - 1, RG>(p, mk, mv, a, sg, ring, tg, rg, lr0, nts, sm_m, sm_l, merge);
    __syncthreads();

    const bool whole = sg.ta == 0 && sg.tb == sg.nt;
    const int slot = 2 * static_cast<int>(blockIdx.x) + (sg.ta == 0 ? 1 : 0);
    const int live = min(a.chunk_rows, a.q_rows - sg.row_lo);
    for (int x = static_cast<int>(threadIdx.x); x < live * (D / 4); x += kBAThreads) {
      const int lr = x / (D / 4), d = (x - lr * (D / 4)) * 4;
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int t = 0; t < TG; ++t) top = fmaxf(top, sm_m[t * ROWS + lr]);
#pragma unroll
      for (int t = 0; t < TG; ++t) {
        sum += ex2(sm_m[t * ROWS + lr] - top) * sm_l[t * ROWS + lr];
      }
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int t = 0; t < TG; ++t) {
        const float4 w = *reinterpret_cast<const float4*>(merge + (t * ROWS + lr) * PITCH + d);
        v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
      }
      if (whole) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        ba_store(p, ba_out_at(p, a, sg.b, sg.h, sg.row_lo + lr) + d, v.x * inv, v.y * inv, v.z * inv, v.w * inv);
      } else {
        *reinterpret_cast<float4*>(p.part_o + (static_cast<int64_t>(slot) * ROWS + lr) * D + d) = v;
        if (d == 0)
          *reinterpret_cast<float2*>(p.part_ml + (static_cast<int64_t>(slot) * ROWS + lr) * 2) = make_float2(top, sum);
      }
    }
    fence_proxy_async_smem();                                   // the merge buffer becomes a TMA target again
    __syncthreads();

    u = seg_begin + sg.tb;
    if (hr + 1 == p.h_kv * a.rc && sg.tb == sg.nt) {
      seq_begin = u;
      ++sg.b;
    }
  }
  pdl_launch_dependents();
  if (!ring.ok && rg == 0 && lane == 0) {   // a wait ran out: leave no copy of this block in flight
    for (int s = 0; s < stages; ++s) {
      (void)mbar_wait(&full[tg][s], 0u, p.status, SPECQ_STATUS_TIMEOUT_PIPELINE);
      (void)mbar_wait(&full[tg][s], 1u, p.status, SPECQ_STATUS_TIMEOUT_PIPELINE);
    }
  }
}

// Join the parts of cut segments: block (segment, group of 8 rows), one warp a row.
template <int D>
__global__ void __launch_bounds__(256) block_attn_join_kernel(const __grid_constant__ BlockAttnParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int warp = static_cast<int>(threadIdx.x >> 5), lane = static_cast<int>(threadIdx.x & 31);
  const BALine a = ba_line(p, false);
  if (a.rc == 0) return;
  const int seg = blockIdx.x;
  const int b = seg / (p.h_kv * a.rc), hr = seg - b * (p.h_kv * a.rc);
  if (b >= a.n_seqs) return;
  const int h = hr / a.rc, rc = hr - h * a.rc;
  // where the segment lies on the line
  int64_t before = 0;
  for (int b0 = 0; b0 < b; b0 += 32) {
    const int x = b0 + lane;
    before += __reduce_add_sync(0xffffffffu, x < b ? ba_tiles(p, ba_ctx(p, x)) : 0);
  }
  const int nt = ba_tiles(p, ba_ctx(p, b));
  const int64_t s0 = before * (p.h_kv * a.rc) + static_cast<int64_t>(hr) * nt, s1 = s0 + nt;
  const int c0 = static_cast<int>(((s0 + 1) * p.grid - 1) / a.total), c1 = static_cast<int>((s1 * p.grid - 1) / a.total);
  if (c0 == c1) return;                                         // inside one piece: written already
  const int row_lo = rc * a.chunk_rows;
  const int lr = blockIdx.y * 8 + warp;
  if (lr >= min(a.chunk_rows, a.q_rows - row_lo)) return;
  auto slot_of = [&](int c) { return 2 * c + (a.total * c / p.grid <= s0 ? 1 : 0); };
  auto empty_piece = [&](int c) { return a.total * c / p.grid == a.total * (c + 1) / p.grid; };
  float top = -INFINITY;
  for (int c = c0 + lane; c <= c1; c += 32)
    if (!empty_piece(c)) top = fmaxf(top, __ldg(p.part_ml + (static_cast<int64_t>(slot_of(c)) * p.rows + lr) * 2));
  top = warp_max_f32(top);
  constexpr int V = D / 32;
  float v[V];
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = 0.f;
  float sum = 0.f;
  for (int c = c0; c <= c1; ++c) {
    if (empty_piece(c)) continue;
    const int64_t at = static_cast<int64_t>(slot_of(c)) * p.rows + lr;
    const float2 ml = __ldg(reinterpret_cast<const float2*>(p.part_ml + at * 2));
    const float f = ex2(ml.x - top);
    sum += f * ml.y;
    const float* src = p.part_o + at * D + lane * V;
    if constexpr (V == 4) {
      const float4 w = __ldg(reinterpret_cast<const float4*>(src));
      v[0] += f * w.x; v[1] += f * w.y; v[2] += f * w.z; v[3] += f * w.w;
    } else {
      const float2 w = __ldg(reinterpret_cast<const float2*>(src));
      v[0] += f * w.x; v[1] += f * w.y;
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int64_t off = ba_out_at(p, a, b, h, row_lo + lr) + lane * V;
  if constexpr (V == 4) {
    ba_store(p, off, v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
  } else if (p.bf16) {
    *reinterpret_cast<__nv_bfloat162*>(static_cast<__nv_bfloat16*>(p.out) + off) = __floats2bfloat162_rn(v[0] * inv, v[1] * inv);
  } else {
    *reinterpret_cast<__half2*>(static_cast<__half*>(p.out) + off) = __floats2half2_rn(v[0] * inv, v[1] * inv);
  }
}

// How a call is launched: the variant for its rows, the grid and the workspace, from the sizes
// that the host knows (maxima under a plan).
struct BAShape {
  int nt, rg, rows, tile, rc, grid, stages, smem;
  bool join;
  int64_t o_floats, ml_floats;
};

inline int ba_shape(int B, int ql, int H_KV, int group, int D, int page, int bt_cols, int sm_count, BAShape* s) {
  const int groups = ceil_div(ql * group, 8);
  s->rc = ceil_div(groups, 12);
  const int g = ceil_div(groups, s->rc);
  // up to 3 groups of 8 rows are one warp's (its accumulators and Q fill the registers); more
  // are dealt to 2 or 4 warps that share a ring
  s->rg = g <= 3 ? 1 : g <= 6 ? 2 : 4;
  s->nt = std::max(g <= 3 ? 1 : 2, ceil_div(g, s->rg));
  s->rows = s->rg * s->nt * 8;
  const int tg = kBAWarps / s->rg;
  s->tile = tg * kBATok;
  const int per_sm = s->nt == 1 ? 2 : 1;
  const int64_t max_tiles = std::max<int64_t>(1, (static_cast<int64_t>(bt_cols) * page + s->tile - 1) / s->tile);
  const int64_t line = static_cast<int64_t>(B) * H_KV * s->rc * max_tiles;
  s->grid = static_cast<int>(std::min<int64_t>(line, static_cast<int64_t>(per_sm) * sm_count));
  s->join = max_tiles > 1;
  const int stage = tg * 2 * kBATok * D;
  const int merge = tg * s->rows * (D + 12) * 4;
  const int room = (per_sm == 2 ? 110 * 1024 : 216 * 1024);
  s->stages = std::min(kBAMaxStages, room / stage);
  s->smem = 1024 + std::max(s->stages * stage, merge);
  if (s->smem > 224 * 1024) return fail(SPECQ_ERR_UNSUPPORTED, "block_attention: shared memory %d", s->smem);
  s->o_floats = s->join ? 2ll * s->grid * s->rows * D : 0;
  s->ml_floats = s->join ? 2ll * s->grid * s->rows * 2 : 0;
  return SPECQ_OK;
}

template <int D, int CT, int NT, int RG>
inline int launch_block_attn(const BlockAttnParams& p, const BAShape& s, const CUtensorMap& mk, const CUtensorMap& mv,
                             cudaStream_t st) {
  auto kern = block_attn_kernel<D, CT, NT, RG>;
  SPECQ_CUDA_TRY(ensure_dyn_smem(reinterpret_cast<const void*>(kern), s.smem));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(s.grid));
  cfg.blockDim = dim3(kBAThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(s.smem);
  cfg.stream = st;
  LaunchAttrs at(1);
  at.apply(cfg);
  SPECQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, p, mk, mv));
  return SPECQ_OK;
}

template <int D, int CT>
inline int launch_block_attn_rows(const BlockAttnParams& p, const BAShape& s, const CUtensorMap& mk,
                                  const CUtensorMap& mv, cudaStream_t st) {
  if (s.rg == 1) {
    if (s.nt == 1) return launch_block_attn<D, CT, 1, 1>(p, s, mk, mv, st);
    if (s.nt == 2) return launch_block_attn<D, CT, 2, 1>(p, s, mk, mv, st);
    return launch_block_attn<D, CT, 3, 1>(p, s, mk, mv, st);
  }
  if (s.rg == 2) return s.nt == 2 ? launch_block_attn<D, CT, 2, 2>(p, s, mk, mv, st) : launch_block_attn<D, CT, 3, 2>(p, s, mk, mv, st);
  return s.nt == 2 ? launch_block_attn<D, CT, 2, 4>(p, s, mk, mv, st) : launch_block_attn<D, CT, 3, 4>(p, s, mk, mv, st);
}

inline int check_block_attn_sizes(int B, int n_seqs, int q_len, int ql_max, int H, int H_KV, int D, int page, int bt_cols,
                                  bool plan) {
  if (B < 0 || n_seqs < 0 || q_len < 0 || ql_max < 0 || H < 0 || H_KV <= 0 || bt_cols < 0)
    return fail(SPECQ_ERR_INVALID_ARG, "block_attention: negative size");
  if (H % H_KV) return fail(SPECQ_ERR_INVALID_ARG, "block_attention: H=%d is not a multiple of H_KV=%d", H, H_KV);
  if (D != 64 && D != 128) return fail(SPECQ_ERR_UNSUPPORTED, "block_attention: head_dim %d (this build supports 64 and 128)", D);
  if (!page_ok(page)) return fail(SPECQ_ERR_UNSUPPORTED, "block_attention: page %d (a power of two in 8..128)", page);
  if (!plan && (n_seqs > B || q_len > ql_max))
    return fail(SPECQ_ERR_INVALID_ARG, "block_attention: n_seqs/q_len exceed the grid");
  if (static_cast<int64_t>(bt_cols) * page > 0x7FFFFF00ll || static_cast<int64_t>(ql_max) * H > (1 << 24))
    return fail(SPECQ_ERR_UNSUPPORTED, "block_attention: %d columns of %d tokens, %d x %d query rows", bt_cols, page, ql_max, H);
  return SPECQ_OK;
}

inline int run_block_attention_workspace(int B, int n_seqs, int q_len, int ql_max, int H, int H_KV, int D, int page,
                                         int bt_cols, int plan, int64_t* bytes) {
  if (bytes == nullptr) return fail(SPECQ_ERR_INVALID_ARG, "block_attention_workspace: null pointer");
  *bytes = 0;
  if (int rc = check_block_attn_sizes(B, n_seqs, q_len, ql_max, H, H_KV, D, page, bt_cols, plan != 0)) return rc;
  const int bg = plan ? B : n_seqs, ql = plan ? ql_max : q_len;
  if (bg == 0 || ql == 0 || H == 0) return SPECQ_OK;
  DeviceState* dev = nullptr;
  if (int rc = get_device_state(&dev)) return rc;
  BAShape s;
  if (int rc = ba_shape(bg, ql, H_KV, H / H_KV, D, page, bt_cols, dev->sm_count, &s)) return rc;
  *bytes = (s.o_floats + s.ml_floats) * static_cast<int64_t>(sizeof(float));
  return SPECQ_OK;
}

inline int run_block_attention(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, int dtype, const void* kc,
                               const void* vc, int64_t kv_sp, int64_t kv_so, int64_t kv_sh, int cache_dtype,
                               int n_pages, const float* ks, const float* vs, int64_t s_sp, int64_t s_sh,
                               const int32_t* bt, int64_t bt_sb, int bt_cols, const int32_t* ctx, const uint64_t* tree,
                               int64_t tree_sb, int64_t tree_st, float sm_scale, void* out, int64_t o_sb, int64_t o_st,
                               int64_t o_sh, const int32_t* plan, int B, int n_seqs, int q_len, int ql_max, int H,
                               int H_KV, int D, int page, void* workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = check_block_attn_sizes(B, n_seqs, q_len, ql_max, H, H_KV, D, page, bt_cols, plan != nullptr)) return rc;
  if (dtype != 0 && dtype != 2) return fail(SPECQ_ERR_INVALID_ARG, "block_attention: query dtype code %d", dtype);
  if (!(sm_scale > 0.f)) return fail(SPECQ_ERR_INVALID_ARG, "block_attention: sm_scale %g must be positive", sm_scale);
  if (cache_dtype != SPECQ_CACHE_INT8 && cache_dtype != SPECQ_CACHE_E4M3)
    return fail(SPECQ_ERR_INVALID_ARG, "block_attention: cache dtype code %d", cache_dtype);
  const int bg = plan ? B : n_seqs, ql = plan ? ql_max : q_len;
  if (bg == 0 || ql == 0 || H == 0) return SPECQ_OK;
  if (tree != nullptr && ql > 64) return fail(SPECQ_ERR_UNSUPPORTED, "block_attention: a draft tree of %d > 64 tokens", ql);
  if (q == nullptr || out == nullptr || kc == nullptr || vc == nullptr || ks == nullptr || vs == nullptr ||
      ctx == nullptr || (bt == nullptr && bt_cols > 0))
    return fail(SPECQ_ERR_INVALID_ARG, "block_attention: null pointer");
  if (n_pages <= 0) return fail(SPECQ_ERR_INVALID_ARG, "block_attention: a cache of %d pages", n_pages);
  if (!aligned(q, 8) || q_sb % 4 || q_st % 4 || q_sh % 4 || !aligned(out, 8) || o_sb % 4 || o_st % 4 || o_sh % 4)
    return fail(SPECQ_ERR_UNSUPPORTED, "block_attention: query and output rows must be 8-byte aligned");
  if (!aligned(kc, 16) || !aligned(vc, 16) || kv_sp % 16 || kv_so % 16 || kv_sh % 16 || kv_sp <= 0 || kv_so <= 0 || kv_sh <= 0)
    return fail(SPECQ_ERR_UNSUPPORTED, "block_attention: cache rows must be 16-byte aligned (TMA)");
  DeviceState* dev = nullptr;
  if (int rc = get_device_state(&dev)) return rc;
  BAShape s;
  if (int rc = ba_shape(bg, ql, H_KV, H / H_KV, D, page, bt_cols, dev->sm_count, &s)) return rc;
  const int64_t need = (s.o_floats + s.ml_floats) * static_cast<int64_t>(sizeof(float));
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 16)))
    return fail(SPECQ_ERR_INVALID_ARG, "block_attention: a 16-byte aligned workspace of %lld bytes is needed, got %lld",
                (long long)need, (long long)workspace_bytes);
  CUtensorMap mk, mv;
  const uint64_t dims[4] = {static_cast<uint64_t>(D), static_cast<uint64_t>(H_KV), static_cast<uint64_t>(page),
                            static_cast<uint64_t>(n_pages)};
  const uint64_t strides[3] = {static_cast<uint64_t>(kv_sh), static_cast<uint64_t>(kv_so), static_cast<uint64_t>(kv_sp)};
  const uint32_t box[4] = {static_cast<uint32_t>(D), 1, static_cast<uint32_t>(std::min(kBATok, page)), 1};
  const CUtensorMapSwizzle sw = D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
  if (int rc = encode_tiled(&mk, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, kc, dims, strides, box, sw)) return rc;
  if (int rc = encode_tiled(&mv, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, vc, dims, strides, box, sw)) return rc;
  BlockAttnParams p = {};
  p.q = q; p.out = out; p.ks = ks; p.vs = vs; p.bt = bt; p.ctx = ctx; p.tree = tree; p.plan = plan;
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = p.part_o + s.o_floats;
  p.status = dev->status;
  p.q_sb = q_sb; p.q_st = q_st; p.q_sh = q_sh; p.o_sb = o_sb; p.o_st = o_st; p.o_sh = o_sh;
  p.s_sp = s_sp; p.s_sh = s_sh; p.bt_sb = bt_sb; p.tree_sb = tree_sb; p.tree_st = tree_st;
  p.scale_log2 = sm_scale * 1.4426950408889634f;
  p.n_seqs = n_seqs; p.q_len = q_len; p.b_max = bg; p.ql_max = ql; p.h_kv = H_KV; p.group = H / H_KV;
  p.page_log2 = __builtin_ctz(static_cast<unsigned>(page));
  p.n_pages = n_pages; p.bt_cols = bt_cols;
  p.bf16 = dtype == 2; p.stages = s.stages; p.grid = s.grid; p.rows = s.rows; p.tile = s.tile;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int rc;
  if (D == 128)
    rc = cache_dtype == SPECQ_CACHE_INT8 ? launch_block_attn_rows<128, 0>(p, s, mk, mv, st) : launch_block_attn_rows<128, 1>(p, s, mk, mv, st);
  else
    rc = cache_dtype == SPECQ_CACHE_INT8 ? launch_block_attn_rows<64, 0>(p, s, mk, mv, st) : launch_block_attn_rows<64, 1>(p, s, mk, mv, st);
  if (rc != SPECQ_OK || !s.join) return rc;
  const dim3 grid(static_cast<unsigned>(bg * H_KV * s.rc), static_cast<unsigned>(s.rows / 8));
  SPECQ_CUDA_TRY(D == 128 ? launch_plain(block_attn_join_kernel<128>, grid, dim3(256), st, p)
                          : launch_plain(block_attn_join_kernel<64>, grid, dim3(256), st, p));
  return SPECQ_OK;
}

}  // namespace specq
