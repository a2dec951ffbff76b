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
// for a whole page.  What a row may not see becomes -inf after that multiply-add: the factor may
// underflow, and 0 times -inf is NaN.  p is rounded to fp16 for the tensor core; l sums the unrounded p in fp32.
// k8 and v8 are exact in fp16, and so is q (bf16 rows are first scaled by a power of two, and keep their 8
// bits down to 2^-17 of the row's largest element whatever the other rows hold); the products
// accumulate in fp32.  m lags: p may reach 2^8 before the running maximum is raised
// (one warp vote a tile), which fp16 holds without loss.
//
// Tile.  A tile is 128 tokens (64 up to 16 rows) of one KV head against up to 40 query rows, the work of
// a group of four warps.  A block has two groups, which take tiles in turn, each with its own
// running maxima.  Within a group
//   S^T [tokens x rows] = K Q^T   each warp its own quarter of the tokens; Q^T stays in registers, K
//                                 is converted 8 -> 16 bits in registers, once
//   P^T = 2^(S^T - m)             in the accumulator's registers, turned by stmatrix on its way to
//                                 shared memory, where every warp of the group reads it
//   O^T [D x rows] += V^T P^T     each warp its own quarter of D over all of the tokens; V by a
//                                 transposing ldmatrix, converted once
// so O costs 8 registers for 8 rows (D = 128), and a segment ends with a sum of two halves.  Two
// barriers of the group a tile: one carries the vote that raises the running maxima, one joins
// the products.  Rows are the N side of both products and pad to 8.  Feeding warps walk the same
// segments ahead of the others: they read page numbers and scales, start the TMA boxes (up to 64
// slots of a page) into a ring and copy the next queries, so a new segment finds its first tiles
// in shared memory.  The piece's first queries are copied by the computing warps: behind the ring's
// first filling they came 2.5 us later.
//
// Why mma.sync: a 16-token tile of 8n rows is 16 n instructions, and the warp-level tensor pipe
// takes one every 2 cycles an SM (measured; 1024 multiply-adds a cycle): 2 n cycles a token,
// against the 11.6 in which HBM delivers its 256 bytes, so up to n = 5 the products fit under the
// memory time.  A tcgen05 tile would be 128 tokens x 16n padded rows at 64-76 cycles an
// instruction, with round trips through tensor memory between the steps.  More than 40 rows go to
// several blocks, which find the pages in L2; there the products are the bound.
//
// Measured (D = 128, 8 KV heads, group 4, page 64): B = 32, q = 1, context 4096: 55.0 us, 4.9 TB/s (heads
// before slots in a page: 49.5 us, 5.4 TB/s, of the 6.44 that a copy reaches), bound by HBM.  B = 8,
// q = 9, context 4096: 35.4 us (bf16 queries 37.9), of which some 15 are set-up and the join (a launch runs its set-up once,
// from cold instruction caches), and some 2,400 cycles a tile where the products alone would take 1,525: two
// warps a quarter of the SM are all that the registers hold (Q and O of 40 rows), too few to cover
// their own latencies.  The registers spill from 17 rows on (-Xptxas -v: 268 to 368 bytes of stores a thread,
// the feeding warps' among them) and at 9 to 16 rows of D = 128 (128 to 132).  D = 64: two blocks of 24 rows an SM were 35 us for q = 9, one of 40 rows is 27.
//
// Work.  The tiles of all (sequence, KV head, row chunk) segments form one line, each segment's after
// some places that stand for the time its beginning takes; the line is cut into equal pieces, one
// for each resident block, whatever the sequences' lengths, and each block finds its piece from
// ctx_len on the device.  A segment inside one piece is written at once; the parts of a cut one,
// two groups' for each piece, go to the workspace, and a second, dependent launch joins them in the
// pieces' order.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "block_cache.cuh"
#include "paged_attn.cuh"
#include "sm100.cuh"
#include "specq_host.cuh"

namespace specq {

constexpr int kBAGroupWarps = 4;                  // of a group
constexpr int kBAWarps = 2 * kBAGroupWarps;       // that compute
constexpr int kBACompute = 32 * kBAWarps;
// And those that feed them.  A TMA box holds its warp for some 180 cycles whatever its size
// (measured: 2 KB boxes from one warp an SM come at 2.8 TB/s, from two at 4.7, from four at 5.1), so
// an SM has four of them, two a block where two blocks share it.  The registers of an SM's quarter
// divide among whole warps: from 3 row groups on the block launches 12 warps of 168 and splits
// their 64,512 as 224 for the computing ones (8 x 32 x 224) and 56 for the feeding ones (4 x 32 x 56).
__host__ __device__ constexpr bool ba_split(int nt) { return nt >= 3; }
__host__ __device__ constexpr int ba_feeders(int nt) { return ba_split(nt) ? 4 : 2; }
__host__ __device__ constexpr int ba_threads(int nt) { return kBACompute + 32 * ba_feeders(nt); }
// Tokens of a tile: up to 16 rows two blocks share an SM, and half as many tokens leave each a ring
// of six stages.
__host__ __device__ constexpr int ba_tile(int nt) { return ba_split(nt) ? 128 : 64; }
// Places of the line that a segment takes before its tiles: a block that begins a segment spends
// 6,000 to 8,000 cycles on it (the part before, the next queries, a first tile that raises the maxima),
// a tile some 2,400 at D = 128 and 1,500 at D = 64.  Measured without, with these and with 6 and 8: B = 8
// q = 9 ctx 4096 39 / 36.0 / 37.8 us; D = 64, 24 ragged lengths of up to 4000, q = 5: 48 / 30.4 / 31.7 us.
__host__ __device__ constexpr int ba_switch(int d) { return d == 64 ? 4 : 3; }
// Fewest places of a piece.  Measured with 1, 2, 3, 4 and 6: one sequence of 3000 tokens, q = 1, D = 128
// 29.0 / 18.7 / 15.7 / 14.3 / 13.3 us; 16 drafts on 2500 tokens, one KV head, D = 64 19.9 / 14.5 / 13.4 /
// 13.1 / 14.0; 6 x 23 rows, context 286 10.0 / 10.0 / 10.5 / 12.2 / 10.4; one short sequence 5.1, with 6 7.0.
constexpr int kBAPiece = 3;
constexpr int kBAComputeRegs = 224, kBAFeedRegs = 56;
constexpr int kBAMaxGroups = 5;                   // groups of 8 query rows a block holds at most
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
  float* part_o;            // [grid][2 cut segments][2 groups][rows][ba_part(D)]
  int* status;
  int64_t q_sb, q_st, q_sh, o_sb, o_st, o_sh, s_sp, s_sh, bt_sb, tree_sb, tree_st;
  float scale_log2;         // sm_scale * log2(e)
  int n_seqs, q_len, b_max, ql_max, h_kv, group, page_log2, n_pages, bt_cols;
  int bf16, stages, grid, rows, box;    // rows: of a block's chunk; box: slots of a TMA box
  int tile, tile_log2;                  // tokens of a tile
  int places;                           // of the line, before a segment's tiles
  int rc, chunk_rows;                   // row chunks of a (sequence, KV head) and their rows, without a plan
  uint32_t group_magic;                 // ceil(2^32 / group), for group > 1
};

__device__ __forceinline__ void tma_box(void* dst, const CUtensorMap* map, uint64_t* bar, int head, int slot, int page,
                                        uint64_t hint) {
  tma_load_4d(dst, map, bar, 0, head, slot, page, hint);
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
__device__ __forceinline__ void stsm4_t(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d)
               : "memory");
}
__device__ __forceinline__ void stsm2_t(uint32_t addr, uint32_t a, uint32_t b) {
  asm volatile("stmatrix.sync.aligned.m8n8.x2.trans.shared.b16 [%0], {%1, %2};" ::"r"(addr), "r"(a), "r"(b) : "memory");
}
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
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

// qi of query row rr = qi * group + g (rr * group < 2^32: check_block_attn_sizes)
__device__ __forceinline__ int ba_token(const BlockAttnParams& p, int rr) {
  return p.group == 1 ? rr : static_cast<int>(__umulhi(static_cast<uint32_t>(rr), p.group_magic));
}

// a / b for non-negative a and positive b.  A launch executes its set-up code once, from cold
// instruction caches, so its length is its time: the quotient by the reciprocal is a third of an
// integer division's (exact after one correction below 2^22, where the product is off by < 1).
__device__ __forceinline__ int ba_div(int a, int b) {
  if (a >= (1 << 22)) return a / b;
  int q = static_cast<int>(__fmul_rz(static_cast<float>(a), __frcp_rn(static_cast<float>(b))));
  const int r = a - q * b;
  if (r >= b) ++q;
  if (r < 0) --q;
  return q;
}

// Where the segments of a call lie on the line.  A segment takes p.places places, in which nothing
// is done, and then one for each of its tiles: beginning a segment costs a block about as much.
// Piece c of the line (one a block) is [start(c), start(c + 1)): the first `more` pieces have one
// place more than the others.  A piece has kBAPiece places at least: a block's two groups take two
// tiles in the time of one, and every piece is two more parts to join.
struct BALine {
  int n_seqs, q_len, q_rows, rc;   // rc: row chunks of a (sequence, KV head)
  int chunk_rows;                  // rows of a chunk (a multiple of 8)
  int pieces, each, more;
  __device__ __forceinline__ int start(int c) const { return each * c + min(c, more); }
  __device__ __forceinline__ int piece_of(int u) const {
    const int wide = more * (each + 1);
    return u < wide ? ba_div(u, each + 1) : more + ba_div(u - wide, each);   // each > 0 past the wide ones
  }
};

// A length or plan value.  JOIN: from L2.  The joining blocks read these before their own wait: by then the
// kernels that wrote them have completed (the attention blocks have all passed theirs), but only a block's
// own wait says anything about what its SM's L1 holds.  (From L2 everywhere: 32 x 4096 55.5 -> 58.6 us.)
template <bool JOIN>
__device__ __forceinline__ int ba_read(const int32_t* at) {
  if constexpr (!JOIN) return *at;
  int v;
  asm volatile("ld.relaxed.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(at) : "memory");
  return v;
}
template <bool JOIN = false>
__device__ __forceinline__ int ba_ctx(const BlockAttnParams& p, int b) {
  const int c = ba_read<JOIN>(p.ctx + b);
  return min(max(c, 0), p.bt_cols << p.page_log2);
}
__device__ __forceinline__ int ba_tiles(const BlockAttnParams& p, int ctx) { return max(1, (ctx + p.tile - 1) >> p.tile_log2); }
__device__ __forceinline__ int ba_places(const BlockAttnParams& p, int ctx) { return p.places + ba_tiles(p, ctx); }

template <bool JOIN = false>
__device__ __forceinline__ BALine ba_line(const BlockAttnParams& p, bool tell) {
  BALine a;
  a.n_seqs = p.n_seqs;
  a.q_len = p.q_len;
  if (p.plan != nullptr) {
    const int n = ba_read<JOIN>(p.plan), q = ba_read<JOIN>(p.plan + 1);
    a.n_seqs = min(max(n, 0), p.b_max);
    a.q_len = min(max(q, 0), p.ql_max);
    if (tell && (n != a.n_seqs || q != a.q_len)) report_status(p.status, SPECQ_STATUS_PLAN_CLAMPED);
  }
  int t = 0;
  const int lane = static_cast<int>(threadIdx.x & 31);
  for (int b0 = 0; b0 < a.n_seqs; b0 += 32) {
    const int b = b0 + lane;
    int n = 0;
    if (b < a.n_seqs) {
      const int c = ba_read<JOIN>(p.ctx + b);
      if (tell && (c < 0 || c > (p.bt_cols << p.page_log2))) report_status(p.status, SPECQ_STATUS_PLAN_CLAMPED);
      n = ba_places(p, min(max(c, 0), p.bt_cols << p.page_log2));
    }
    t += __reduce_add_sync(0xffffffffu, n);
  }
  a.q_rows = a.q_len * p.group;
  a.rc = p.rc;
  a.chunk_rows = p.chunk_rows;
  if (p.plan != nullptr) {
    const int groups = (a.q_rows + 7) >> 3;
    a.rc = ba_div(groups * 8 + p.rows - 1, p.rows);
    a.chunk_rows = a.rc > 0 ? ba_div(groups + a.rc - 1, a.rc) * 8 : 0;
  }
  const int total = t * (p.h_kv * a.rc);
  a.pieces = min(p.grid, max(1, ba_div(total, kBAPiece)));
  a.each = ba_div(total, a.pieces);
  a.more = total - a.each * a.pieces;
  return a;
}

// The sequence that holds line position u (every lane of the warp calls), and where it begins.
__device__ __forceinline__ int ba_find(const BlockAttnParams& p, const BALine& a, int u, int* begin) {
  const int lane = static_cast<int>(threadIdx.x & 31);
  const int per = p.h_kv * a.rc;
  int at = 0;
  for (int b0 = 0; b0 < a.n_seqs; b0 += 32) {
    const int b = b0 + lane;
    const int n = b < a.n_seqs ? ba_places(p, ba_ctx(p, b)) * per : 0;
    int inc = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, inc, d);
      if (lane >= d) inc += up;
    }
    const unsigned over = __ballot_sync(0xffffffffu, b < a.n_seqs && at + inc > u);
    if (over != 0u) {
      const int first = __ffs(over) - 1;
      *begin = at + __shfl_sync(0xffffffffu, inc - n, first);
      return b0 + first;
    }
    at += __shfl_sync(0xffffffffu, inc, 31);
  }
  *begin = at;
  return a.n_seqs;
}

__device__ __forceinline__ void ba_store2(const BlockAttnParams& p, int64_t off, float a, float b) {
  if (p.bf16) *reinterpret_cast<__nv_bfloat162*>(static_cast<__nv_bfloat16*>(p.out) + off) = __floats2bfloat162_rn(a, b);
  else *reinterpret_cast<__half2*>(static_cast<__half*>(p.out) + off) = __floats2half2_rn(a, b);
}

// Row rr of (sequence b, KV head h) in out, in elements.  o_sb = 0: packed token rows.
__device__ __forceinline__ int64_t ba_out_at(const BlockAttnParams& p, const BALine& a, int b, int h, int rr) {
  const int qi = ba_token(p, rr), g = rr - qi * p.group;
  const int64_t tok = p.o_sb == 0 ? static_cast<int64_t>(b) * a.q_len + qi : qi;
  return b * p.o_sb + tok * p.o_st + static_cast<int64_t>(h * p.group + g) * p.o_sh;
}

// One block's view of the segment it works on.
struct BASeg {
  int b, h, row_lo;        // sequence, KV head, first row of the chunk
  int ctx, old;            // tokens; tokens before the drafts (every row sees them)
  int ta, tb, nt;          // tiles of this piece, tiles of the segment
};

// The segments of a block's piece [u, u1) of the line, in order.  (The divisions are in start():
// what a block executes once runs from cold instruction caches, some 20 cycles an instruction.)
struct BAWalk {
  int u, u1;
  int b, h, chunk, from;   // of the segment at u, and u's place in it
  int ctx, ctx_next;       // of sequences b and b + 1, read before they are needed
  __device__ __forceinline__ void start(const BlockAttnParams& p, const BALine& a) {
    u = a.start(static_cast<int>(blockIdx.x));
    u1 = a.start(static_cast<int>(blockIdx.x) + 1);
    b = h = chunk = from = ctx = ctx_next = 0;
    if (static_cast<int>(blockIdx.x) >= a.pieces) u = u1;
    if (u >= u1) return;
    int begin;
    b = ba_find(p, a, u, &begin);
    ctx = ba_ctx(p, b);
    if (b + 1 < a.n_seqs) ctx_next = ba_ctx(p, b + 1);
    const int len = ba_places(p, ctx), hr = ba_div(u - begin, len);
    from = u - begin - hr * len;
    h = a.rc == 1 ? hr : ba_div(hr, a.rc);
    chunk = hr - h * a.rc;
  }
  __device__ __forceinline__ bool next(const BlockAttnParams& p, const BALine& a, BASeg& s) {
    do {
      if (u >= u1) return false;
      s.b = b;
      s.h = h;
      s.row_lo = chunk * a.chunk_rows;
      s.ctx = ctx;
      s.old = ctx - a.q_len;
      s.nt = ba_tiles(p, ctx);
      const int to = min(p.places + s.nt, from + u1 - u);
      s.ta = max(0, from - p.places);
      s.tb = max(0, to - p.places);
      u += to - from;
      from = 0;
      if (++chunk == a.rc) {
        chunk = 0;
        if (++h == p.h_kv) {
          h = 0;
          ++b;
          ctx = ctx_next;
          if (b + 1 < a.n_seqs) ctx_next = ba_ctx(p, b + 1);
        }
      }
    } while (s.tb == s.ta);                  // the piece may end before the segment's first tile
    return true;
  }
};

// A place in the ring of stages.  The number of stages is a multiple of 2 and of the feeding warps, and
// tile n of a piece goes to group n % 2 and comes from warp n % feeders: so a stage has one reader and
// one writer for good.  (With others in between, a waiter would not see every phase of a barrier,
// and a parity would name two.)
struct BAPlace {
  int s;
  uint32_t ph;
  __device__ __forceinline__ void step(int stages) {
    if (++s == stages) {
      s = 0;
      ph ^= 1u;
    }
  }
  __device__ __forceinline__ void back(int stages) {
    if (s == 0) {
      s = stages;
      ph ^= 1u;
    }
    --s;
  }
};

// A group's barrier that also tells whether any of its threads says so.
__device__ __forceinline__ bool ba_vote(int id, bool x) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.red.or.pred q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(x ? 1u : 0u), "r"(id), "n"(32 * kBAGroupWarps)
      : "memory");
  return r != 0u;
}

// A row's part in the workspace: O [D], l of the group's four warps, m, and padding to 16 bytes.
__host__ __device__ constexpr int ba_part(int D) { return D + 8; }

template <int D, int NT>
struct BASmem {
  static constexpr int TOK = ba_tile(NT);
  static constexpr int U = TOK / 16 / kBAGroupWarps;           // 16 tokens that a warp multiplies with Q
  static constexpr int MT = D / 16 / kBAGroupWarps;            // 16-element pieces of D a warp accumulates
  static constexpr int ROWS = NT * 8;
  static constexpr int KB = TOK * D;                       // bytes of a K (or V) tile
  static constexpr int STAGE = 2 * KB;
  static constexpr int PPITCH = 2 * TOK + 16;                  // rows of P shift by 4 banks
  static constexpr int P = ROWS * PPITCH;  // a tile's P [row][token], fp16
  static constexpr int QPITCH = 2 * D + 16;
  static constexpr int TREE = ROWS * QPITCH;                   // behind the queries: the rows' tree words
  static constexpr int Q = TREE + ROWS * 8;
  static constexpr int SC = TOK / 8;                           // scales of a stage: ck, lv, iv for each 8 tokens
  static constexpr int SCALES = SC * 16;
  static constexpr int PART = ba_part(D);                      // floats of a row's part
  static constexpr int MERGE = kBAGroupWarps * MT * NT * 32 * 16;   // one group's O
  static constexpr int fixed = 2 * P + MERGE + 2 * Q + kBAMaxStages * SCALES + 2 * kBAWarps * ROWS * 4 + 512;
};

template <int D, int CT, int NT>
__global__ void __launch_bounds__(ba_threads(NT), ba_split(NT) ? 1 : 2)
block_attn_kernel(const __grid_constant__ BlockAttnParams p, const __grid_constant__ CUtensorMap mk,
                  const __grid_constant__ CUtensorMap mv) {
  SPECQ_TRACE_INIT();
  if (threadIdx.x == 0) SPECQ_TRACE_POINT(0, 0);
  using S = BASmem<D, NT>;
  constexpr int KC = D / 16;                 // 16-byte pieces of a token
  constexpr int MT = S::MT, U = S::U, TOK = S::TOK, ROWS = S::ROWS, NF = ba_feeders(NT);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const int stages = p.stages;
  uint8_t* ring = base;
  uint8_t* pbuf = ring + stages * S::STAGE;                    // one for each group
  float4* merge = reinterpret_cast<float4*>(pbuf + 2 * S::P);
  uint8_t* qbuf = pbuf + 2 * S::P + S::MERGE;
  float4* scales = reinterpret_cast<float4*>(qbuf + 2 * S::Q);
  float* sm_l = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(scales) + kBAMaxStages * S::SCALES);   // [warp][row]
  float* sm_m = sm_l + kBAWarps * ROWS;                                                                   // [warp][row]
  // A block that has the SM to itself has few stages, and frees a tile's K when its scores are made;
  // where two share it, a tile is one stage with one barrier (59 -> 56 us for B=32 q=1 ctx 4096)
  constexpr bool TWO = ba_split(NT);
  uint64_t* k_full = reinterpret_cast<uint64_t*>(sm_m + kBAWarps * ROWS);
  uint64_t* k_empty = k_full + kBAMaxStages;
  uint64_t* v_full = k_empty + kBAMaxStages;
  uint64_t* v_empty = v_full + kBAMaxStages;
  uint64_t* q_full = v_empty + kBAMaxStages;
  uint64_t* q_empty = q_full + 2;

  const int warp = static_cast<int>(threadIdx.x >> 5), lane = static_cast<int>(threadIdx.x & 31);
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&k_full[s], 2u);             // the boxes' expected bytes, and the scales
      mbar_init(&v_full[s], 1u);
      mbar_init(&k_empty[s], kBAGroupWarps); // the group that reads it
      mbar_init(&v_empty[s], kBAGroupWarps);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&q_full[s], 32u * NF);
      mbar_init(&q_empty[s], kBAWarps);
    }
    fence_barrier_init();
    tma_prefetch_desc(&mk);
    tma_prefetch_desc(&mv);
  }
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();                   // the joining blocks set themselves up as these leave the SMs
  if (threadIdx.x == 0) SPECQ_TRACE_POINT(1, 0);
  const BALine a = ba_line(p, blockIdx.x == 0 && warp == 0);
  BAWalk walk;
  walk.start(p, a);
  if (threadIdx.x == 0) SPECQ_TRACE_POINT(2, 0);
  BASeg sg = {};
  BAPlace at = {0, 0u}, qat = {0, 0u};       // stage of the piece's next tile, of its next queries
  bool ok = true;
  // The queries of segment s into the next buffer, a quarter (NF = 2: half) by each of NF warps.
  auto copy_queries = [&](int f, const BASeg& s) {
    const int rows = min(a.chunk_rows, a.q_rows - s.row_lo);
    constexpr int CH = D / 8;                // 16-byte pieces of a query row: a lane keeps its piece
    const int c = lane % CH;
    for (int lr = f * (32 / CH) + lane / CH; lr < ROWS; lr += NF * (32 / CH)) {
      uint8_t* d = qbuf + qat.s * S::Q + lr * S::QPITCH + c * 16;
      const int rr = s.row_lo + min(lr, rows - 1);
      const int qi = ba_token(p, rr), g = rr - qi * p.group;
      const int64_t row = p.q_sb == 0 ? static_cast<int64_t>(s.b) * a.q_len + qi : qi;
      const uint16_t* src = static_cast<const uint16_t*>(p.q) + s.b * p.q_sb + row * p.q_st +
                            static_cast<int64_t>(s.h * p.group + g) * p.q_sh + c * 8;
      // padding rows take 0 of the 16 bytes: zeros
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(d)), "l"(src), "r"(lr < rows ? 16 : 0)
                   : "memory");
    }
    if (p.tree != nullptr && f == NF - 1) {
      for (int lr = lane; lr < ROWS; lr += 32) {
        const int qi = ba_token(p, s.row_lo + min(lr, rows - 1));
        const uint64_t* src = p.tree + s.b * p.tree_sb + qi * p.tree_st;
        const uint32_t d = smem_u32(qbuf + qat.s * S::Q + S::TREE + lr * 8);
        asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(d), "l"(src) : "memory");
      }
    }
    cp_async_mbar_arrive(&q_full[qat.s]);
    if (lane == 0 && f == 0) SPECQ_TRACE_POINT(4, qat.s);
  };

  if (warp >= kBAWarps) {                    // ---- the feeding warps: warp f takes tiles f, f + NF, ... of the piece
    if constexpr (ba_split(NT)) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kBAFeedRegs));
    const int f = warp - kBAWarps;
    const int nb = TOK >> (31 - __clz(p.box));          // boxes of a tile; a batch of 32 is `tpb` of the warp's tiles
    const int tpb = 32 / nb;                 // (all powers of two)
    const int lt = lane >> (31 - __clz(nb)), lb = lane & (nb - 1);
    bool q_done = true;                      // the computing warps copy the piece's first queries
    qat.step(2);
    int skip = f;                            // tiles of the segment before the warp's next one
    // pages that one block reads are read once; of several row chunks the first leaves them in L2
    const uint64_t hint = a.rc == 1 ? policy_evict_first() : policy_evict_last();
    while (walk.next(p, a, sg)) {
      const int32_t* bt = p.bt + sg.b * p.bt_sb;
      int t0 = sg.ta + skip;                 // the batch's first tile
      int pg = -1, tok = 0;
      auto load_pages = [&]() {
        const int t = t0 + lt * NF;
        tok = t * TOK + lb * p.box;
        pg = t < sg.tb && tok < sg.ctx ? bt[tok >> p.page_log2] : -1;
      };
      load_pages();
      if (!q_done) {
        ok = ok && mbar_wait(&q_empty[qat.s], qat.ph ^ 1u, p.status, SPECQ_STATUS_TIMEOUT_PIPELINE);
        copy_queries(f, sg);
        qat.step(2);
      }
      q_done = false;
      int stepped = sg.ta;                   // `at` is the stage of this tile
      for (; t0 < sg.tb;) {
        const int my_tile = t0 + lt * NF, my_tok = tok;
        const bool load = my_tile < sg.tb && tok < sg.ctx;
        const bool there = pg >= 0 && pg < p.n_pages;
        if (load && !there) report_status(p.status, SPECQ_STATUS_BAD_INDEX);
        // a page that is not there weighs nothing: its box lies past the map's last page, which TMA fills with
        // zeros (another page's bytes may be e4m3 NaN)
        const int page = there ? pg : p.n_pages;
        float ks = 0.f, vs = 0.f;
        const int t1 = min(sg.tb, t0 + tpb * NF);
        const int tb0 = t0;
        t0 += tpb * NF;
        if (t0 < sg.tb) load_pages();
        for (int t = tb0; t < t1; t += NF) {
          for (; stepped < t; ++stepped) at.step(stages);
          ok = ok && mbar_wait(&k_empty[at.s], at.ph ^ 1u, p.status, SPECQ_STATUS_TIMEOUT_PIPELINE);
          const bool mine = t == my_tile;
          const unsigned boxes = __ballot_sync(0xffffffffu, mine && load);
          if (ok) {
            if (lane == 0) mbar_arrive_expect_tx(&k_full[at.s], (TWO ? 1u : 2u) * __popc(boxes) * p.box * D);
            __syncwarp();
            // one lane starts all boxes: their operands are the warp's, not a lane's
            const int first = (t - tb0) / NF * nb;
            const int slot0 = (t * TOK) & ((1 << p.page_log2) - 1);
            const int n_box = __popc(boxes);
            auto start = [&](uint8_t* d, const CUtensorMap* map, uint64_t* bar) {
              int slot = slot0;
              for (int x = 0; x < n_box; ++x) {
                const int pgx = __shfl_sync(0xffffffffu, page, first + x);
                if (elect_one()) tma_box(d, map, bar, sg.h, slot, pgx, hint);
                d += p.box * D;
                slot = (slot + p.box) & ((1 << p.page_log2) - 1);
              }
            };
            start(ring + at.s * S::KB, &mk, &k_full[at.s]);
            if (t == tb0 && there) {         // the batch's scales, behind its first boxes
              const int64_t x = static_cast<int64_t>(page) * p.s_sp + sg.h * p.s_sh;
              ks = p.ks[x];
              vs = p.vs[x];
            }
            if constexpr (!TWO) start(ring + (stages + at.s) * S::KB, &mv, &k_full[at.s]);
            if (mine) {
              float4 w = make_float4(0.f, -INFINITY, 0.f, 0.f);   // what is not there weighs nothing
              if (there) {
                const float v = vs < kBALeastV ? kBALeastV : vs;
                w.x = ks * p.scale_log2;
                w.y = __log2f(v);
                w.z = __frcp_rn(v);
              }
              float4* d = scales + at.s * S::SC + lb * (p.box >> 3);
              for (int i = 0; i < p.box >> 3; ++i) d[i] = w;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&k_full[at.s]);
            if (lane == 0) SPECQ_TRACE_POINT(5, t);
            if constexpr (TWO)
              ok = ok && mbar_wait(&v_empty[at.s], at.ph ^ 1u, p.status, SPECQ_STATUS_TIMEOUT_PIPELINE);
            if (TWO && ok) {
              if (lane == 0) mbar_arrive_expect_tx(&v_full[at.s], __popc(boxes) * p.box * D);
              __syncwarp();
              start(ring + (stages + at.s) * S::KB, &mv, &v_full[at.s]);
            }
          }
        }
      }
      for (; stepped < sg.tb; ++stepped) at.step(stages);
      skip = (skip + NF - (sg.tb - sg.ta) % NF) % NF;
    }
    if (!ok) {                               // a wait ran out: leave no copy of this block in flight
      for (int s = 0; s < stages; ++s) {
        for (uint32_t ph = 0; ph < 2u; ++ph) {
          (void)mbar_wait(&k_full[s], ph, p.status, SPECQ_STATUS_TIMEOUT_PIPELINE);
          if (TWO) (void)mbar_wait(&v_full[s], ph, p.status, SPECQ_STATUS_TIMEOUT_PIPELINE);
        }
      }
    }
    return;
  }

  // ---- the computing warps
  if constexpr (ba_split(NT)) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kBAComputeRegs));
  const int grp = warp >> 2, gw = warp & 3;  // group, warp of the group
  const int gq = lane >> 2, tq = lane & 3;
  // ldmatrix rows of this lane: matrix lane / 8 = (token half, piece); pieces are swizzled
  const int mr = (lane & 7) + ((lane >> 3) & 1) * 8, mc = lane >> 4;
  const uint32_t ring_s = smem_u32(ring);
  const uint32_t k_off =
      ring_s + static_cast<uint32_t>((gw * 16 * U + mr) * D + ((mc ^ (D == 128 ? (mr & 7) : ((mr >> 1) & 3))) << 4));
  // V: MT = 2, matrices (token half, piece); MT = 1, (token half, next 16 tokens)
  const int vr = MT == 2 ? mr : mr + mc * 16;
  const int vc = MT == 2 ? 2 * gw + mc : gw;
  const uint32_t v_off =
      ring_s + static_cast<uint32_t>(stages * S::KB + vr * D + ((vc ^ (D == 128 ? (vr & 7) : ((vr >> 1) & 3))) << 4));
  // P: this lane's row of the matrices that it stores (group pair, token half) and loads (32 tokens of a group)
  const uint32_t p_base = smem_u32(pbuf + grp * S::P);
  const uint32_t p_put =
      p_base + static_cast<uint32_t>(((lane >> 4) * 8 + (lane & 7)) * S::PPITCH + (U * gw * 16 + ((lane >> 3) & 1) * 8) * 2);
  const uint32_t p_get = p_base + static_cast<uint32_t>((lane & 7) * S::PPITCH + (lane >> 3) * 16);

  int tile_no = 0;                           // of the piece
  for (bool first = true; walk.next(p, a, sg); first = false) {
    // The piece's first queries are on their way before any tile, so they do not queue behind the
    // ring's first filling; the feeding warps copy the others, ahead.
    if (first && warp < NF) copy_queries(warp, sg);
    // ---- Q^T as the B operand: thread (gq, tq) holds row gq of each group, d = 16 c + 4 tq + 0..3
    uint32_t qf[NT][KC][2];
    ok = ok && mbar_wait(&q_full[qat.s], qat.ph, p.status, SPECQ_STATUS_TIMEOUT_PIPELINE);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const uint8_t* src = qbuf + qat.s * S::Q + (n * 8 + gq) * S::QPITCH + 8 * tq;
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        const uint2 w = *reinterpret_cast<const uint2*>(src + 32 * c);
        qf[n][c][0] = w.x;
        qf[n][c][1] = w.y;
      }
    }
    const uint64_t* tree_rows = reinterpret_cast<const uint64_t*>(qbuf + qat.s * S::Q + S::TREE);
    if (threadIdx.x == 0) SPECQ_TRACE_POINT(9, sg.ta);
    // bf16 to fp16: under one power of two that brings the largest finite element to [2^15, 2^16), so that a
    // row 2^15 below it still keeps bf16's 8 bits down to 2^-17 of its own largest element (what is smaller
    // is off by 2^-25 of it at most).  Rows further apart than that have a power each: no row costs another
    // its bits.  (Each row its own always: D = 128, 8 x 16384, 36 rows 92 -> 98 us, D = 64 trees 38 -> 41.)
    float fac = 1.f;
    float* facs = sm_l + warp * ROWS;        // free until the segment's sums are written
    if (p.bf16) {
      uint32_t tops[NT], hi = 0u, lo = 0x7f80u;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        uint32_t top = 0;
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const uint32_t mag = (half ? qf[n][c][i] >> 16 : qf[n][c][i]) & 0x7fffu;
              top = max(top, mag >= 0x7f80u ? 0u : mag);
            }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));   // the row's elements lie in four lanes
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        tops[n] = top;
        hi = max(hi, top);
        lo = min(lo, top == 0u ? 0x7f80u : top);                // a row of zeros goes with any
      }
      hi = __reduce_max_sync(0xffffffffu, hi) >> 7;             // biased exponents
      lo = __reduce_min_sync(0xffffffffu, lo) >> 7;
      const bool apart = hi > lo + 15u;
      const uint32_t all = max(hi, 16u);
      fac = apart ? 0.f : __uint_as_float((all - 15u) << 23);   // 0: look in facs
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint32_t own = min(max(tops[n] >> 7, 1u), 253u);
        const float inv = __uint_as_float((254u - (apart ? own : all - 15u)) << 23);
        if (apart && tq == 0) facs[n * 8 + gq] = __uint_as_float(own << 23);
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const __half2 y = __floats2half2_rn(__uint_as_float(qf[n][c][i] << 16) * inv,
                                                __uint_as_float(qf[n][c][i] & 0xffff0000u) * inv);
            qf[n][c][i] = *reinterpret_cast<const uint32_t*>(&y);
          }
      }
      __syncwarp();
    }
    float o[MT][NT][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n][0] = m[n][1] = kBANone;
      l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int c = 0; c < MT; ++c) o[c][n][0] = o[c][n][1] = o[c][n][2] = o[c][n][3] = 0.f;
    }

    float sc[U][NT][4];                      // a tile's scores
    auto scores = [&](uint32_t stage) {
      // S^T = K Q^T for tokens 16 (U gw + u) + 0..15
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int n = 0; n < NT; ++n) sc[u][n][0] = sc[u][n][1] = sc[u][n][2] = sc[u][n][3] = 0.f;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        uint32_t r[KC / 2][4];               // the whole 16 tokens are on their way before the first product
#pragma unroll
        for (int c = 0; c < KC / 2; ++c)
          ldsm4(((k_off + stage) ^ static_cast<uint32_t>(c << 5)) + static_cast<uint32_t>(u * 16 * D), r[c]);
#pragma unroll
        for (int c = 0; c < KC; ++c) {
          uint32_t l0, h0, l1, h1;
          widen4<CT, false>(r[c >> 1][2 * (c & 1)], l0, h0);
          widen4<CT, false>(r[c >> 1][2 * (c & 1) + 1], l1, h1);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma16816(sc[u][n], l0, l1, h0, h1, qf[n][c][0], qf[n][c][1]);
        }
      }
    };
    // masks, raises the maxima where the vote says so, leaves P in shared memory (after the vote, which is
    // also the barrier after which the group has read the P before)
    BAPlace pl = at;
    auto softmax = [&](int t) {              // of tile t, whose place is pl
      // softmax: rows 2 tq, 2 tq + 1 of each group, tokens gq and gq + 8 of each 16
      // x = score in log2 units + log2(sV); what a row may not see is masked after, since a factor that
      // underflows times a masked -inf would be NaN
      float iv[U], iv1[U];                   // 1: of tokens gq + 8
      {
        float ck[U], lv[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const float4 w0 = scales[pl.s * S::SC + 2 * (U * gw + u)];
          ck[u] = w0.x;
          lv[u] = w0.y;
          iv[u] = iv1[u] = w0.z;
        }
        if (fac == 0.f || p.page_log2 == 3) {     // a factor for each row; tokens 8 .. 15 are another page's at page 8
          float ck1[U], lv1[U];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            ck1[u] = ck[u];
            lv1[u] = lv[u];
            if (p.page_log2 == 3) {
              const float4 w1 = scales[pl.s * S::SC + 2 * (U * gw + u) + 1];
              ck1[u] = w1.x;
              lv1[u] = w1.y;
              iv1[u] = w1.z;
            }
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const float2 f = fac == 0.f ? *reinterpret_cast<const float2*>(&facs[n * 8 + 2 * tq]) : make_float2(fac, fac);
#pragma unroll
            for (int u = 0; u < U; ++u) {
              sc[u][n][0] = fmaf(sc[u][n][0], ck[u] * f.x, lv[u]);
              sc[u][n][1] = fmaf(sc[u][n][1], ck[u] * f.y, lv[u]);
              sc[u][n][2] = fmaf(sc[u][n][2], ck1[u] * f.x, lv1[u]);
              sc[u][n][3] = fmaf(sc[u][n][3], ck1[u] * f.y, lv1[u]);
            }
          }
        } else {
#pragma unroll
          for (int u = 0; u < U; ++u) ck[u] *= fac;
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int i = 0; i < 4; ++i) sc[u][n][i] = fmaf(sc[u][n][i], ck[u], lv[u]);
        }
      }
      const int tw = t * TOK + 16 * U * gw;  // the warp's first token
      if (tw + 16 * U > sg.old) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int t0 = tw + 16 * u;
          if (t0 + 16 > sg.old) {            // some row may not see some token
            // bits 4n + 2r + half of what this thread's rows see of its two tokens
            uint32_t sees = 0;
            const int j0 = t0 + gq - sg.old, j1 = j0 + 8;       // draft numbers
#pragma unroll 1
            for (int x = 0; x < 2 * NT; ++x) {
              const int lr = (x >> 1) * 8 + 2 * tq + (x & 1);
              uint32_t s0, s1;
              if (p.tree == nullptr) {
                const int qi = min(ba_token(p, sg.row_lo + lr), a.q_len - 1);
                s0 = j0 <= qi;
                s1 = j1 <= qi;
              } else {
                const uint64_t word = tree_rows[lr];
                s0 = j0 < 0 || (j0 < a.q_len && ((word >> (j0 & 63)) & 1ull) != 0ull);
                s1 = j1 < 0 || (j1 < a.q_len && ((word >> (j1 & 63)) & 1ull) != 0ull);
              }
              sees |= (s0 | s1 << 1) << (2 * x);
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int r = 0; r < 2; ++r) {
                if (((sees >> (4 * n + 2 * r)) & 1u) == 0u) sc[u][n][r] = -INFINITY;
                if (((sees >> (4 * n + 2 * r)) & 2u) == 0u) sc[u][n][2 + r] = -INFINITY;
              }
            if (CT == 1 && t0 + 16 > sg.ctx) {
              // slots past the last token may hold anything, NaN bytes too: their V reads as 0
              if constexpr (TWO) ok = ok && mbar_wait(&v_full[pl.s], pl.ph, p.status, SPECQ_STATUS_TIMEOUT_PIPELINE);
              uint8_t* v = ring + (stages + pl.s) * S::KB + 16 * (U * gw + u) * D;
              for (int x = max(sg.ctx - t0, 0) * KC + lane; x < 16 * KC; x += 32)
                *reinterpret_cast<uint4*>(v + x * 16) = make_uint4(0u, 0u, 0u, 0u);
              fence_proxy_async_smem();      // before the stage is filled again
            }
          }
        }
      }
      // against the lagging m; one chain of maxima a group of rows
      float tops[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        tops[n] = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int r = 0; r < 2; ++r) tops[n] = fmaxf(tops[n], fmaxf(sc[u][n][r], sc[u][n][2 + r]) - m[n][r]);
      }
      float top = tops[0];
#pragma unroll
      for (int n = 1; n < NT; ++n) top = fmaxf(top, tops[n]);
      if (ba_vote(1 + grp, top > kBARaise)) {                   // raise the maxima and what they scale
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float v = fmaxf(sc[0][n][r], sc[0][n][2 + r]);
            if constexpr (U == 2) v = fmaxf(v, fmaxf(sc[U - 1][n][r], sc[U - 1][n][2 + r]));
            v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
            v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
            v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
            if (gq == 0) sm_m[warp * ROWS + n * 8 + 2 * tq + r] = v;
          }
        named_barrier_sync(1 + grp, 32 * kBAGroupWarps);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float2 top2 = make_float2(m[n][0], m[n][1]);
#pragma unroll
          for (int w = 0; w < kBAGroupWarps; ++w) {
            const float2 v = *reinterpret_cast<const float2*>(&sm_m[(grp * kBAGroupWarps + w) * ROWS + n * 8 + 2 * tq]);
            top2.x = fmaxf(top2.x, v.x);
            top2.y = fmaxf(top2.y, v.y);
          }
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float mn = r == 0 ? top2.x : top2.y;
            const float f = ex2(m[n][r] - mn);
            m[n][r] = mn;
            l[n][r] *= f;
#pragma unroll
            for (int c = 0; c < MT; ++c) {
              o[c][n][r] *= f;
              o[c][n][2 + r] *= f;
            }
          }
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        uint32_t h[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float y[4];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            y[r] = ex2(sc[u][n][r] - m[n][r]);
            y[2 + r] = ex2(sc[u][n][2 + r] - m[n][r]);
            l[n][r] = fmaf(y[2 + r], iv1[u], fmaf(y[r], iv[u], l[n][r]));
          }
          const __half2 h0 = __floats2half2_rn(y[0], y[1]), h1 = __floats2half2_rn(y[2], y[3]);
          h[n][0] = *reinterpret_cast<const uint32_t*>(&h0);
          h[n][1] = *reinterpret_cast<const uint32_t*>(&h1);
        }
        // (token, row) fragments turned on the way to P [row][token]
        const uint32_t d = p_put + static_cast<uint32_t>(u * 32);
#pragma unroll
        for (int n = 0; n + 1 < NT; n += 2)
          stsm4_t(d + static_cast<uint32_t>(n * 8 * S::PPITCH), h[n][0], h[n][1], h[n + 1][0], h[n + 1][1]);
        if constexpr (NT % 2 == 1) stsm2_t(d + static_cast<uint32_t>((NT - 1) * 8 * S::PPITCH), h[NT - 1][0], h[NT - 1][1]);
      }
    };
    auto products = [&](uint32_t stage) {
      // O^T += V^T P^T
      // 32 tokens at a time; V of the next 32 is on its way
      constexpr int NK = TOK / 32;
      uint32_t vn[MT][4];
#pragma unroll
      for (int c = 0; c < MT; ++c) ldsm4_t(v_off + stage + static_cast<uint32_t>(c * 16 * D), vn[c]);
#pragma unroll
      for (int k = 0; k < NK; ++k) {
        uint32_t pf[NT][4], r[MT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) ldsm4(p_get + static_cast<uint32_t>(n * 8 * S::PPITCH + k * 64), pf[n]);
#pragma unroll
        for (int c = 0; c < MT; ++c) {
#pragma unroll
          for (int i = 0; i < 4; ++i) r[c][i] = vn[c][i];
          if (k + 1 < NK) ldsm4_t(v_off + stage + static_cast<uint32_t>(((k + 1) * 2 + c) * 16 * D), vn[c]);
        }
        // MT = 2: r[s] is 16-token step s, two pieces of D; MT = 1: both steps of the one piece
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int c = 0; c < MT; ++c) {
            uint32_t e0, d0, e1, d1;
            widen4<CT, true>(r[MT == 2 ? s : 0][2 * (MT == 2 ? c : s)], e0, d0);
            widen4<CT, true>(r[MT == 2 ? s : 0][2 * (MT == 2 ? c : s) + 1], e1, d1);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma16816(o[c][n], e0, d0, e1, d1, pf[n][2 * s], pf[n][2 * s + 1]);
          }
      }
    };
    auto release = [&](uint64_t* bar) {
      __syncwarp();                          // every lane has read the stage
      if (lane == 0) mbar_arrive(bar);
    };

    // the group's tiles are every other one of the piece
    const int n_all = sg.tb - sg.ta, first_mine = ((tile_no & 1) != grp) ? 1 : 0;
    const int n_mine = (n_all - first_mine + 1) >> 1;
    tile_no += n_all;
    if (first_mine) pl.step(stages);
    for (int x = 0; x < n_mine; ++x) {
      ok = ok && mbar_wait(&k_full[pl.s], pl.ph, p.status, SPECQ_STATUS_TIMEOUT_PIPELINE);
      if (threadIdx.x == 0) SPECQ_TRACE_POINT(10, x);
      scores(static_cast<uint32_t>(pl.s * S::KB));
      if (threadIdx.x == 0) SPECQ_TRACE_POINT(11, x);
      softmax(sg.ta + first_mine + 2 * x);
      if constexpr (TWO) release(&k_empty[pl.s]);               // its scales are read too
      named_barrier_sync(1 + grp, 32 * kBAGroupWarps);          // the group's P is written
      if (threadIdx.x == 0) SPECQ_TRACE_POINT(13, x);
      if constexpr (TWO) ok = ok && mbar_wait(&v_full[pl.s], pl.ph, p.status, SPECQ_STATUS_TIMEOUT_PIPELINE);
      products(static_cast<uint32_t>(pl.s * S::KB));
      release(TWO ? &v_empty[pl.s] : &k_empty[pl.s]);
      if (threadIdx.x == 0) SPECQ_TRACE_POINT(14, x);
      pl.step(stages);
      pl.step(stages);
    }
    at = pl;                                 // of the tile after the segment's last:
    if (first_mine + 2 * n_mine > n_all) at.back(stages);

    __syncwarp();                            // the queries' buffer (and its tree words) may be filled again
    if (lane == 0) mbar_arrive(&q_empty[qat.s]);
    qat.step(2);

    // ---- the group's part of the segment
    const int live = min(a.chunk_rows, a.q_rows - sg.row_lo);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float v = l[n][r];
        v += __shfl_xor_sync(0xffffffffu, v, 4);
        v += __shfl_xor_sync(0xffffffffu, v, 8);
        v += __shfl_xor_sync(0xffffffffu, v, 16);
        l[n][r] = v;
      }
    if (sg.ta > 0 || sg.tb < sg.nt) {
      // a piece of a cut segment: each group writes its part to the workspace (O of each warp's
      // elements, l of each warp's tokens, m; a group that had no tile has l = 0) and goes on
      {
        float* part = p.part_o + (2 * (2 * static_cast<int64_t>(blockIdx.x) + (sg.ta == 0 ? 1 : 0)) + grp) * (ROWS * S::PART);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float* d = part + (n * 8 + 2 * tq + r) * S::PART;
            if (n * 8 + 2 * tq + r < live) {
#pragma unroll
              for (int c = 0; c < MT; ++c)
                *reinterpret_cast<float2*>(d + (gw * MT + c) * 16 + 2 * gq) = make_float2(o[c][n][r], o[c][n][2 + r]);
              if (gq == 0) {
                d[D + gw] = l[n][r];
                if (gw == 0) d[D + kBAGroupWarps] = m[n][r];
              }
            }
          }
      }
    } else {
      // all of it: the second group's part goes to the first, and out
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 2; ++r)
          if (gq == 0) {
            sm_l[warp * ROWS + n * 8 + 2 * tq + r] = l[n][r];
            if (warp == kBAGroupWarps) sm_m[warp * ROWS + n * 8 + 2 * tq + r] = m[n][r];
          }
      if (grp == 1) {
#pragma unroll
        for (int c = 0; c < MT; ++c)
#pragma unroll
          for (int n = 0; n < NT; ++n)
            merge[((gw * MT + c) * NT + n) * 32 + lane] = make_float4(o[c][n][0], o[c][n][1], o[c][n][2], o[c][n][3]);
      }
      named_barrier_sync(3, kBACompute);
      if (grp == 0) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int lr = n * 8 + 2 * tq + r;
            const float m1 = sm_m[kBAGroupWarps * ROWS + lr];
            const float mx = fmaxf(m[n][r], m1), f0 = ex2(m[n][r] - mx), f1 = ex2(m1 - mx);
            float l0 = 0.f, l1 = 0.f;
#pragma unroll
            for (int x = 0; x < kBAGroupWarps; ++x) {
              l0 += sm_l[x * ROWS + lr];
              l1 += sm_l[(kBAGroupWarps + x) * ROWS + lr];
            }
            const float sum = l0 * f0 + l1 * f1;
            const float inv = sum == 0.f ? 0.f : __frcp_rn(sum);
            if (lr < live) {
              const int64_t off = ba_out_at(p, a, sg.b, sg.h, sg.row_lo + lr) + gw * MT * 16 + 2 * gq;
#pragma unroll
              for (int c = 0; c < MT; ++c) {
                const float4 w = merge[((gw * MT + c) * NT + n) * 32 + lane];
                ba_store2(p, off + 16 * c, (o[c][n][r] * f0 + (r == 0 ? w.x : w.y) * f1) * inv,
                          (o[c][n][2 + r] * f0 + (r == 0 ? w.z : w.w) * f1) * inv);
              }
            }
          }
      }
      named_barrier_sync(3, kBACompute);                        // sm_l, sm_m and the merge buffer may be written again
    }
    if (threadIdx.x == 0) SPECQ_TRACE_POINT(15, sg.ta);
  }
}

// Join the parts of cut segments: block (segment, group of 8 rows), one warp a row.
template <int D>
__global__ void __launch_bounds__(256) block_attn_join_kernel(const __grid_constant__ BlockAttnParams p) {
  pdl_launch_dependents();
  const int warp = static_cast<int>(threadIdx.x >> 5), lane = static_cast<int>(threadIdx.x & 31);
  // The lengths and the plan were there before the attention kernel started (these blocks start when
  // all of its have passed their own wait), so the block finds its rows while that still runs.
  const BALine a = ba_line<true>(p, false);
  const int per = max(1, p.h_kv * a.rc);
  const int b = ba_div(static_cast<int>(blockIdx.x), per), hr = static_cast<int>(blockIdx.x) - b * per;
  const int h = a.rc > 1 ? ba_div(hr, a.rc) : hr, row_lo = (hr - h * a.rc) * a.chunk_rows;
  const int lr = blockIdx.y * 8 + warp;
  bool work = a.rc > 0 && b < a.n_seqs && lr < min(a.chunk_rows, a.q_rows - row_lo);
  int c0 = 0, c1 = 0;
  if (work) {
    // where the segment lies on the line
    int before = 0;
    for (int b0 = 0; b0 < b; b0 += 32) {
      const int x = b0 + lane;
      before += __reduce_add_sync(0xffffffffu, x < b ? ba_places(p, ba_ctx<true>(p, x)) : 0);
    }
    const int nt = ba_tiles(p, ba_ctx<true>(p, b));
    const int s0 = before * per + hr * (p.places + nt) + p.places;      // its first tile
    c0 = a.piece_of(s0);
    c1 = a.piece_of(s0 + nt - 1);
    work = c0 != c1;                                            // else inside one piece: written already
  }
  pdl_wait();                                                   // every block, or the next kernel could pass this one
  if (!work) return;
  // piece c0 holds the segment's beginning (its second slot), the others begin inside it
  constexpr int V = D / 32, PART = ba_part(D);
  float v[V];
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = 0.f;
  float sum = 0.f, top = kBANone;
  constexpr int U = 8;                                          // parts in flight (4: verify 36.0 us, 8: 35.2, 16: 38.1)
  for (int x0 = 2 * c0; x0 <= 2 * c1 + 1; x0 += U) {
    float m[U], l[U], w[U][V];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int x = x0 + i, c = x >> 1, grp = x & 1;
      m[i] = kBANone;
      l[i] = 0.f;
#pragma unroll
      for (int y = 0; y < V; ++y) w[i][y] = 0.f;
      if (c <= c1) {
        const float* src = p.part_o + (static_cast<int64_t>(2 * (2 * c + (c == c0 ? 1 : 0)) + grp) * p.rows + lr) * PART;
        const float4 l4 = *reinterpret_cast<const float4*>(src + D);
        m[i] = src[D + kBAGroupWarps];
        l[i] = (l4.x + l4.y) + (l4.z + l4.w);
        if constexpr (V == 4) {
          const float4 u = *reinterpret_cast<const float4*>(src + lane * V);
          w[i][0] = u.x; w[i][1] = u.y; w[i][2] = u.z; w[i][3] = u.w;
        } else {
          const float2 u = *reinterpret_cast<const float2*>(src + lane * V);
          w[i][0] = u.x; w[i][1] = u.y;
        }
      }
    }
    float mx = top;
#pragma unroll
    for (int i = 0; i < U; ++i) mx = fmaxf(mx, m[i]);
    const float f0 = ex2(top - mx);
    sum *= f0;
#pragma unroll
    for (int y = 0; y < V; ++y) v[y] *= f0;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const float f = ex2(m[i] - mx);
      sum = fmaf(f, l[i], sum);
#pragma unroll
      for (int y = 0; y < V; ++y) v[y] = fmaf(f, w[i][y], v[y]);
    }
    top = mx;
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int64_t off = ba_out_at(p, a, b, h, row_lo + lr) + lane * V;
#pragma unroll
  for (int i = 0; i < V; i += 2) ba_store2(p, off + i, v[i] * inv, v[i + 1] * inv);
}

// How a call is launched: the variant for its rows, the grid and the workspace, from the sizes
// that the host knows (maxima under a plan).
struct BAShape {
  int nt, rows, tile, rc, grid, stages, smem;
  bool join;
  int64_t ws_floats;
};

template <int D>
inline void ba_smem(int nt, int* fixed, int* stage) {
  switch (nt) {
    case 1: *fixed = BASmem<D, 1>::fixed; break;
    case 2: *fixed = BASmem<D, 2>::fixed; break;
    case 3: *fixed = BASmem<D, 3>::fixed; break;
    case 4: *fixed = BASmem<D, 4>::fixed; break;
    default: *fixed = BASmem<D, 5>::fixed; break;
  }
  *stage = 2 * ba_tile(nt) * D;
}

inline int ba_shape(int B, int ql, int H_KV, int group, int D, int page, int bt_cols, int sm_count, BAShape* s) {
  const int groups = ceil_div(ql * group, 8);
  s->rc = ceil_div(groups, kBAMaxGroups);
  s->nt = ceil_div(groups, s->rc);
  s->rows = s->nt * 8;
  // up to 16 rows two blocks fit an SM's registers and fill each other's pauses
  const int per_sm = ba_split(s->nt) ? 1 : 2;
  s->tile = ba_tile(s->nt);
  const int64_t max_tiles = std::max<int64_t>(1, (static_cast<int64_t>(bt_cols) * page + s->tile - 1) / s->tile);
  const int64_t line = static_cast<int64_t>(B) * H_KV * s->rc * max_tiles;
  if (line + static_cast<int64_t>(B) * H_KV * s->rc * ba_switch(D) > 0x7FFFFFFFll)
    return fail(SPECQ_ERR_UNSUPPORTED, "block_attention: %lld tiles", (long long)line);
  s->grid = static_cast<int>(std::min<int64_t>(line, static_cast<int64_t>(per_sm) * sm_count));
  s->join = max_tiles > 1;
  int fixed, stage;
  if (D == 64) ba_smem<64>(s->nt, &fixed, &stage);
  else ba_smem<128>(s->nt, &fixed, &stage);
  const int room = (per_sm == 2 ? 112 * 1024 : 226 * 1024) - 1024 - fixed;
  const int of = std::max(2, ba_feeders(s->nt));               // stages have one reader and one writer each
  s->stages = std::min(kBAMaxStages, room / stage) / of * of;
  if (s->stages < of) return fail(SPECQ_ERR_UNSUPPORTED, "block_attention: %d rows do not fit shared memory", s->rows);
  s->smem = 1024 + fixed + s->stages * stage;
  s->ws_floats = s->join ? 4ll * s->grid * s->rows * ba_part(D) : 0;
  return SPECQ_OK;
}

template <int D, int CT, int NT>
inline int launch_block_attn(const BlockAttnParams& p, const BAShape& s, const CUtensorMap& mk, const CUtensorMap& mv,
                             cudaStream_t st) {
  auto kern = block_attn_kernel<D, CT, NT>;
  if constexpr (ba_split(NT)) {
    // The computing warps wait for registers that the launch has to bring: fewer would be waited for without end.
    static const int regs = [&] {
      cudaFuncAttributes fa = {};
      return cudaFuncGetAttributes(&fa, reinterpret_cast<const void*>(kern)) == cudaSuccess ? fa.numRegs : 0;
    }();
    if (regs * ba_threads(NT) < 32 * (kBAWarps * kBAComputeRegs + ba_feeders(NT) * kBAFeedRegs))
      return fail(SPECQ_ERR_UNSUPPORTED, "block_attention: built with %d registers a thread, too few to split", regs);
  }
  SPECQ_CUDA_TRY(ensure_dyn_smem(reinterpret_cast<const void*>(kern), s.smem));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(s.grid));
  cfg.blockDim = dim3(ba_threads(NT));
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
  switch (s.nt) {
    case 1: return launch_block_attn<D, CT, 1>(p, s, mk, mv, st);
    case 2: return launch_block_attn<D, CT, 2>(p, s, mk, mv, st);
    case 3: return launch_block_attn<D, CT, 3>(p, s, mk, mv, st);
    case 4: return launch_block_attn<D, CT, 4>(p, s, mk, mv, st);
    default: return launch_block_attn<D, CT, 5>(p, s, mk, mv, st);
  }
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
  const int64_t group = H / H_KV, rows = static_cast<int64_t>(ql_max) * group;
  if (static_cast<int64_t>(bt_cols) * page > 0x7FFFFF00ll || static_cast<int64_t>(ql_max) * H > (1 << 24) ||
      (rows + 8 * kBAMaxGroups) * group > 0x100000000ll)   // ba_token's product, a chunk's padding rows included
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
  *bytes = s.ws_floats * static_cast<int64_t>(sizeof(float));
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
  if (!aligned(q, 16) || q_sb % 8 || q_st % 8 || q_sh % 8 || !aligned(out, 4) || o_sb % 2 || o_st % 2 || o_sh % 2)
    return fail(SPECQ_ERR_UNSUPPORTED, "block_attention: query rows must be 16-byte aligned, output rows 4-byte");
  if (!aligned(kc, 16) || !aligned(vc, 16) || kv_sp % 16 || kv_so % 16 || kv_sh % 16 || kv_sp <= 0 || kv_so <= 0 || kv_sh <= 0)
    return fail(SPECQ_ERR_UNSUPPORTED, "block_attention: cache rows must be 16-byte aligned (TMA)");
  DeviceState* dev = nullptr;
  if (int rc = get_device_state(&dev)) return rc;
  BAShape s;
  if (int rc = ba_shape(bg, ql, H_KV, H / H_KV, D, page, bt_cols, dev->sm_count, &s)) return rc;
  const int64_t need = s.ws_floats * static_cast<int64_t>(sizeof(float));
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 16)))
    return fail(SPECQ_ERR_INVALID_ARG, "block_attention: a 16-byte aligned workspace of %lld bytes is needed, got %lld",
                (long long)need, (long long)workspace_bytes);
  CUtensorMap mk, mv;
  const uint64_t dims[4] = {static_cast<uint64_t>(D), static_cast<uint64_t>(H_KV), static_cast<uint64_t>(page),
                            static_cast<uint64_t>(n_pages)};
  const uint64_t strides[3] = {static_cast<uint64_t>(kv_sh), static_cast<uint64_t>(kv_so), static_cast<uint64_t>(kv_sp)};
  const uint32_t box[4] = {static_cast<uint32_t>(D), 1, static_cast<uint32_t>(std::min(64, page)), 1};
  const CUtensorMapSwizzle sw = D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
  if (int rc = encode_tiled(&mk, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, kc, dims, strides, box, sw)) return rc;
  if (int rc = encode_tiled(&mv, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, vc, dims, strides, box, sw)) return rc;
  BlockAttnParams p = {};
  p.q = q; p.out = out; p.ks = ks; p.vs = vs; p.bt = bt; p.ctx = ctx; p.tree = tree; p.plan = plan;
  p.part_o = static_cast<float*>(workspace);
  p.status = dev->status;
  p.q_sb = q_sb; p.q_st = q_st; p.q_sh = q_sh; p.o_sb = o_sb; p.o_st = o_st; p.o_sh = o_sh;
  p.s_sp = s_sp; p.s_sh = s_sh; p.bt_sb = bt_sb; p.tree_sb = tree_sb; p.tree_st = tree_st;
  p.scale_log2 = sm_scale * 1.4426950408889634f;
  p.n_seqs = n_seqs; p.q_len = q_len; p.b_max = bg; p.ql_max = ql; p.h_kv = H_KV; p.group = H / H_KV;
  p.page_log2 = __builtin_ctz(static_cast<unsigned>(page));
  p.n_pages = n_pages; p.bt_cols = bt_cols;
  p.bf16 = dtype == 2; p.stages = s.stages; p.grid = s.grid; p.rows = s.rows; p.box = std::min(64, page); p.tile = s.tile;
  p.places = ba_switch(D);
  p.tile_log2 = 31 - __builtin_clz(static_cast<unsigned>(s.tile));
  p.rc = s.rc; p.chunk_rows = ceil_div(ceil_div(ql * p.group, 8), s.rc) * 8;
  p.group_magic = p.group > 1 ? 0xFFFFFFFFu / static_cast<uint32_t>(p.group) + 1u : 0u;
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
