// evict.cuh -- a row of the block-scaled cache cut down to its heaviest and its newest tokens.
//
// For each layer, sequence b of n = ctx_len[b] > keep tokens and KV head (heads choose for themselves):
//   kept: the `recent` newest tokens and of the others the keep - recent of largest mass[b, h, t],
//         equal ones the earliest first (a NaN counts as -inf)
//   they move to places 0 .. keep - 1 in their order, their masses with them; mass becomes 0 from keep to n
//   a page's scale becomes the largest scale of the pages that its tokens come from, and numbers of
//   another scale are requantised, rn(q * (s_source / s'))
// Each number moved from a page of the largest scale keeps its bits, and no maximum over the numbers is needed.
//
// A block selects for one (layer, sequence, head): the bound's 32 bits two at a time by counting, then one
// ordered pass that writes the kept tokens' places in the cache.  A block then moves K or V of one (layer, sequence,
// head), 32 KB at a time, the next batch read ahead of the writes: a token's place never grows, and the
// batches hold whole pages, so what is read later lies behind what is written.  Bound by scattered runs of D bytes where
// there are some hundred (layer, sequence, head)s, by latency below.  Measured (B200): 4 layers, 12 sequences of up to 2500
// tokens, 8 heads of 128, 1024 kept: 69 us for 206 MB, of which the moves some 47 (4.3 TB/s; runs of 128 bytes 1 KB apart do not
// get more, whatever is in flight) and the selection the rest; one layer, 8 sequences of up to 700, 256 kept: 13.2 us.
// (Selection by histograms of 8 bits in place of counting 18 us more; 256 threads in place of 512 for a move 3 more.)
#pragma once

#include "beams.cuh"
#include "block_cache.cuh"

namespace specq {

constexpr int kEvictSelThreads = 256;
static_assert(kEvictSelThreads == kSelThreads, "block_before's threads");
constexpr int kEvictRun = 4;                                        // tokens a thread takes in the ordered pass
// Keys held in shared memory: 192 KB of them where the rows leave each SM one block or two, else 48 KB, so that four blocks of
// a wide table's short rows stay on an SM. (8 rows of 16384 tokens 75 us against 123 with 48 KB, 256 rows of 32768 213 against
// 278; past the limit each digit reads the masses again.)
constexpr int kEvictStage = 48 * 1024;
constexpr int kEvictStageMany = 12 * 1024;
constexpr int kEvictMoveThreads = 512;
constexpr int kEvictPieces = 4;                                     // 16-byte pieces a thread moves at a time

struct EvictParams {
  uint8_t* kc;
  uint8_t* vc;
  float* ks;
  float* vs;
  const int32_t* bt;
  const int32_t* ctx;
  const int32_t* ref;      // optional [P]: rows that hold a page
  float* mass;             // [L, B, H_KV, N]
  int32_t* ctx_out;        // [B]
  int32_t* place;          // workspace [L, B, H_KV, keep]: page * page size + slot of the kept tokens
  int32_t* first;          // workspace [L, B, H_KV]: the first kept token that moves; keep: none; -1: the row stays
  int* status;
  int64_t kv_sl, kv_sp, kv_so, kv_sh, s_sl, s_sp, s_sh, bt_sb, m_sl, m_sb, m_sh;
  int n_pages, bt_cols, B, h_kv, page_log2, keep, recent;
  int staged;              // keys that the shared memory holds
  int linear;              // kv_sp is a page of kv_so
};

__global__ void __launch_bounds__(kEvictSelThreads) evict_select_kernel(const __grid_constant__ EvictParams p) {
  extern __shared__ uint32_t staged[];
  __shared__ int4 counts[2][kEvictSelThreads / 32];
  __shared__ int red[kEvictSelThreads / 32];
  __shared__ int lowest;
  pdl_launch_dependents();
  pdl_wait();
  const int h = blockIdx.x, b = blockIdx.y, l = blockIdx.z, tid = static_cast<int>(threadIdx.x);
  const int64_t id = (static_cast<int64_t>(l) * p.B + b) * p.h_kv + h;
  const int n = p.ctx[b], page = 1 << p.page_log2, keep = p.keep;
  if (n <= keep) {
    if (tid == 0) p.first[id] = -1;
    return;
  }
  // a row that reaches past its table, has a page outside the cache or shares one stays as it is
  const int32_t* row = p.bt + b * p.bt_sb;
  const int cols = (n - 1) / page + 1;
  bool bad = cols > p.bt_cols;
  for (int c = tid; c < min(cols, p.bt_cols); c += kEvictSelThreads) {
    const int pg = row[c];
    bad = bad || pg < 0 || pg >= p.n_pages || (p.ref != nullptr && p.ref[pg] > 1);
  }
  if (__syncthreads_or(bad)) {
    if (tid == 0) {
      p.first[id] = -1;
      report_status(p.status, SPECQ_STATUS_BAD_INDEX);
    }
    return;
  }
  float* mass = p.mass + l * p.m_sl + b * p.m_sb + h * p.m_sh;
  const int others = n - p.recent, want = keep - p.recent;     // others > want
  const bool in_smem = p.staged != 0 && others <= p.staged;
  auto key_at = [&](int t) { return in_smem ? staged[t] : order_key(fmaxf(mass[t], -INFINITY)); };
  if (in_smem) {
    for (int t = tid; t < others; t += kEvictSelThreads) staged[t] = order_key(fmaxf(mass[t], -INFINITY));
    __syncthreads();
  }
  // The want-th largest key, two bits at a time: how many keys reach each of the next three bounds.
  uint32_t bound = 0xffffffffu;
  int equal = 0;                                               // keys equal to the bound that are kept
  if (want > 0) {
    uint32_t prefix = 0;
    int above = 0;                                             // keys above prefix's range
    for (int shift = 30; shift >= 0; shift -= 2) {
      const uint32_t b1 = prefix + (1u << shift), b2 = prefix + (2u << shift), b3 = prefix + (3u << shift);
      const uint32_t last = prefix + ((4u << shift) - 1u);     // (wraps to all ones at the top)
      int n1 = 0, n2 = 0, n3 = 0;
      for (int t = tid; t < others; t += kEvictSelThreads) {
        const uint32_t k = key_at(t);
        if (k > last) continue;
        n1 += k >= b1;
        n2 += k >= b2;
        n3 += k >= b3;
      }
      n1 = __reduce_add_sync(0xffffffffu, n1);
      n2 = __reduce_add_sync(0xffffffffu, n2);
      n3 = __reduce_add_sync(0xffffffffu, n3);
      int4* sums = counts[shift >> 1 & 1];                     // the other one may still be read
      if ((tid & 31) == 0) sums[tid >> 5] = make_int4(n1, n2, n3, 0);
      __syncthreads();
      n1 = n2 = n3 = 0;
#pragma unroll
      for (int w = 0; w < kEvictSelThreads / 32; ++w) {
        const int4 u = sums[w];
        n1 += u.x;
        n2 += u.y;
        n3 += u.z;
      }
      // as many as wanted reach a bound: the keys above it less one are the ones
      const uint32_t exact = above + n3 == want ? b3 : above + n2 == want ? b2 : above + n1 == want ? b1 : 0u;
      if (exact != 0u) {
        prefix = exact - 1u;
        above = want;
        break;
      }
      // the largest bound that `want` keys reach; those at or above the next one are above its range
      if (above + n3 >= want) prefix = b3;
      else if (above + n2 >= want) prefix = b2, above += n3;
      else if (above + n1 >= want) prefix = b1, above += n2;
      else above += n1;
    }
    bound = prefix;
    equal = want - above;
  }
  if (tid == 0) lowest = keep;
  // kept tokens in order: those above the bound and the first `equal` at it
  int32_t* place = p.place + id * keep;
  auto put = [&](int j, int t, float m) {
    place[j] = row[t >> p.page_log2] * page + (t & (page - 1));
    mass[j] = m;               // j <= t, and what lies before this tile has been read
    if (t != j) atomicMin(&lowest, j);
  };
  int above = 0, same = 0;
  for (int t0 = 0; want > 0 && t0 < others; t0 += kEvictSelThreads * kEvictRun) {
    float m[kEvictRun];
    uint32_t k[kEvictRun];
    int mine = 0;
#pragma unroll
    for (int i = 0; i < kEvictRun; ++i) {
      const int t = t0 + tid * kEvictRun + i;
      m[i] = t < others ? mass[t] : 0.f;
      k[i] = t < others ? order_key(fmaxf(m[i], -INFINITY)) : 0u;
      mine += (t < others && k[i] > bound) + (t < others && k[i] == bound ? 1 << 16 : 0);
    }
    int all;
    const int before = block_before(mine, red, &all);          // (its barriers: every thread has read its masses)
    int up = above + (before & 0xffff), eq = same + (before >> 16);
#pragma unroll
    for (int i = 0; i < kEvictRun; ++i) {
      const int t = t0 + tid * kEvictRun + i;
      if (t >= others || k[i] < bound) continue;
      if (k[i] > bound) put(up++ + min(eq, equal), t, m[i]);
      else if (eq++ < equal) put(up + eq - 1, t, m[i]);
    }
    above += all & 0xffff;
    same += all >> 16;
    __syncthreads();
  }
  for (int i0 = 0; i0 < p.recent; i0 += kEvictSelThreads) {
    const int i = i0 + tid;
    const float m = i < p.recent ? mass[others + i] : 0.f;
    __syncthreads();
    if (i < p.recent) put(want + i, others + i, m);
  }
  __syncthreads();
  for (int t = keep + tid; t < n; t += kEvictSelThreads) mass[t] = 0.f;
  if (tid == 0) p.first[id] = lowest;
}

// A piece of 16 stored numbers times r <= 1, rounded: fp32 products, two at a time.
template <int CT>
__device__ __forceinline__ uint4 requant16(uint4 w, float r) {
  uint32_t u[4] = {w.x, w.y, w.z, w.w};
  const float2 rr = make_float2(r, r);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float v[4];
    unpack_cache4<CT>(u[i], v);
    const float2 a = __fmul2_rn(make_float2(v[0], v[1]), rr), b = __fmul2_rn(make_float2(v[2], v[3]), rr);
    u[i] = pack_cache4<CT>(a.x, a.y, b.x, b.y);
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}

template <int CT, int D>
__global__ void __launch_bounds__(kEvictMoveThreads) evict_move_kernel(const __grid_constant__ EvictParams p) {
  constexpr int U = kEvictPieces, kPer = D / 16;                       // pieces of a token
  constexpr int kBatch = kEvictMoveThreads * U / kPer;                 // tokens: 256 (D = 128) or 512
  static_assert(kEvictMoveThreads % kPer == 0, "a thread's pieces stand at one place of their tokens");
  static_assert(kBatch >= 128 && kBatch <= kEvictMoveThreads, "a batch holds whole pages, a thread a token's scale");
  __shared__ float from[kBatch];
  __shared__ float to[kBatch];
  __shared__ int dest[kBatch];
  __shared__ float wide[kEvictMoveThreads / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int h = static_cast<int>(blockIdx.x >> 1), is_v = blockIdx.x & 1, b = blockIdx.y, l = blockIdx.z, tid = static_cast<int>(threadIdx.x);
  const int64_t id = (static_cast<int64_t>(l) * p.B + b) * p.h_kv + h;
  const int first = p.first[id];
  if (blockIdx.x == 0 && l == 0 && tid == 0) {     // the only reader of ctx here, so ctx_out may be ctx
    const int n = p.ctx[b];
    p.ctx_out[b] = first < 0 ? n : p.keep;
  }
  if (first < 0 || first >= p.keep) return;
  const int page = 1 << p.page_log2, mask = page - 1;
  uint8_t* cache = (is_v ? p.vc : p.kc) + l * p.kv_sl + h * p.kv_sh;
  float* scale = (is_v ? p.vs : p.ks) + l * p.s_sl + h * p.s_sh;
  const int32_t* place = p.place + id * p.keep;
  const int32_t* row = p.bt + b * p.bt_sb;
  // Batches in registers: the tokens of one while the one before is written, and the places of the one after.
  uint4 w[2][U];
  float s[2];                                       // this thread's token's scale
  int at[U], at_scale;
  uint8_t* mine = cache + (tid % kPer) * 16;
  // where a place of the cache stands; pages that follow one another without gaps need one product
  auto token = [&](int where) {
    return p.linear ? where * p.kv_so : (where >> p.page_log2) * p.kv_sp + (where & mask) * p.kv_so;
  };
  auto look = [&](int j0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + (u * kEvictMoveThreads + tid) / kPer;
      at[u] = j < p.keep ? place[j] : -1;
    }
    at_scale = tid < kBatch && j0 + tid < p.keep ? place[j0 + tid] : -1;
  };
  auto load = [&](uint4 (&v)[U], float& sc) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (at[u] >= 0)
        v[u] = *reinterpret_cast<const uint4*>(mine + token(at[u]));
    sc = at_scale >= 0 ? scale[(at_scale >> p.page_log2) * p.s_sp] : 0.f;
  };
  auto store = [&](int j0, uint4 (&v)[U], float sc) {
    // the largest scale of each page: over its lanes, then (pages of 64 and 128) its warps
    float m = sc;
    for (int o = 1; o < min(page, 32); o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if ((tid & 31) == 0) wide[tid >> 5] = m;
    __syncthreads();                                // (every thread's loads of this batch are done as well)
    if (page > 32) {
      const int warps = page >> 5, w0 = (tid >> 5) & ~(warps - 1);
      m = wide[w0];
      for (int i = 1; i < warps; ++i) m = fmaxf(m, wide[w0 + i]);
    }
    if (tid < kBatch) {
      from[tid] = sc;
      to[tid] = m;
      if (j0 + tid < p.keep) {
        const int pg = row[(j0 + tid) >> p.page_log2];
        dest[tid] = pg * page + (tid & mask);       // (a batch begins with a page)
        if ((tid & mask) == 0) scale[pg * p.s_sp] = m;
      }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = (u * kEvictMoveThreads + tid) / kPer;
      if (j0 + t < p.keep) {
        const float a = from[t], z = to[t];
        *reinterpret_cast<uint4*>(mine + token(dest[t])) = a == z ? v[u] : requant16<CT>(v[u], a / z);
      }
    }
  };
  int j0 = first & ~mask;
  look(j0);
  load(w[0], s[0]);
  look(j0 + kBatch);
  while (true) {
    load(w[1], s[1]);                               // (nothing past the last token)
    look(j0 + 2 * kBatch);
    store(j0, w[0], s[0]);
    j0 += kBatch;
    if (j0 >= p.keep) break;
    load(w[0], s[0]);
    look(j0 + 2 * kBatch);
    store(j0, w[1], s[1]);
    j0 += kBatch;
    if (j0 >= p.keep) break;
  }
}

inline int evict_check(int L, int B, int H_KV, int D, int page, int keep, int recent, int n_pages) {
  const char* who = "block_evict";
  if (L < 1 || B < 0 || H_KV < 1 || keep < 1 || recent < 0 || recent > keep || n_pages < 0)
    return fail(SPECQ_ERR_INVALID_ARG, "%s: layers=%d B=%d H_KV=%d keep=%d recent=%d", who, L, B, H_KV, keep, recent);
  if (D != 64 && D != 128) return fail(SPECQ_ERR_UNSUPPORTED, "%s: head_dim %d (64 or 128)", who, D);
  if (page < 8 || page > 128 || (page & (page - 1))) return fail(SPECQ_ERR_UNSUPPORTED, "%s: page %d (a power of two, 8 to 128)", who, page);
  if (B > 65535 || L > 65535 || H_KV > 65535 || static_cast<int64_t>(n_pages) * page > 0x7fffffffll)
    return fail(SPECQ_ERR_UNSUPPORTED, "%s: layers=%d B=%d H_KV=%d, %d pages of %d", who, L, B, H_KV, n_pages, page);
  return SPECQ_OK;
}

// Sequences of a turn: a place for each token that may be kept, by layers and heads, goes by `keep`, whatever the sequences hold.  (A budget
// of 131072 tokens in 32 layers of 64 sequences and 8 heads would be 8.6 GB.)
inline int evict_turn(int L, int B, int H_KV, int keep) {
  return even_turn(B, kTurnSpace / (static_cast<int64_t>(L) * H_KV * (static_cast<int64_t>(keep) + 1) * 4));
}

inline int run_block_evict_workspace(int L, int B, int H_KV, int keep, int64_t* bytes) {
  if (bytes == nullptr) return fail(SPECQ_ERR_INVALID_ARG, "block_evict_workspace: null pointer");
  if (int rc = evict_check(L, B, H_KV, 64, 8, keep, 0, 0)) return rc;
  *bytes = static_cast<int64_t>(L) * evict_turn(L, B, H_KV, keep) * H_KV * (static_cast<int64_t>(keep) + 1) * 4;
  return SPECQ_OK;
}

inline int run_block_evict(void* kc, void* vc, int64_t kv_sl, int64_t kv_sp, int64_t kv_so, int64_t kv_sh, int cache_dtype, int L,
                           int n_pages, float* ks, float* vs, int64_t s_sl, int64_t s_sp, int64_t s_sh, const int32_t* block_tbl,
                           int64_t bt_sb, int bt_cols, const int32_t* ctx_len, const int32_t* ref, float* mass, int64_t m_sl,
                           int64_t m_sb, int64_t m_sh, int keep, int recent, int32_t* ctx_out, int B, int H_KV, int D, int page,
                           void* workspace, int64_t workspace_bytes, void* stream) {
  const char* who = "block_evict";
  if (int rc = evict_check(L, B, H_KV, D, page, keep, recent, n_pages)) return rc;
  if (cache_dtype != SPECQ_CACHE_INT8 && cache_dtype != SPECQ_CACHE_E4M3) return fail(SPECQ_ERR_INVALID_ARG, "%s: cache dtype code %d", who, cache_dtype);
  if (bt_cols < 0) return fail(SPECQ_ERR_INVALID_ARG, "%s: bt_cols=%d", who, bt_cols);
  if (B == 0) return SPECQ_OK;
  if (kc == nullptr || vc == nullptr || ks == nullptr || vs == nullptr || block_tbl == nullptr || ctx_len == nullptr || mass == nullptr ||
      ctx_out == nullptr)
    return fail(SPECQ_ERR_INVALID_ARG, "%s: null pointer", who);
  if (!aligned(kc, 16) || !aligned(vc, 16) || kv_sl % 16 || kv_sp % 16 || kv_so % 16 || kv_sh % 16)
    return fail(SPECQ_ERR_UNSUPPORTED, "%s: cache rows must be 16-byte aligned", who);
  int64_t need = 0;
  if (int rc = run_block_evict_workspace(L, B, H_KV, keep, &need)) return rc;
  if (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 16))
    return fail(SPECQ_ERR_INVALID_ARG, "%s: a workspace of %lld bytes is needed", who, static_cast<long long>(need));
  DeviceState* dev = nullptr;
  if (int rc = get_device_state(&dev)) return rc;
  EvictParams p = {};
  p.kc = static_cast<uint8_t*>(kc); p.vc = static_cast<uint8_t*>(vc); p.ks = ks; p.vs = vs;
  p.ref = ref; p.status = dev->status;
  p.place = static_cast<int32_t*>(workspace);
  p.kv_sl = kv_sl; p.kv_sp = kv_sp; p.kv_so = kv_so; p.kv_sh = kv_sh; p.s_sl = s_sl; p.s_sp = s_sp; p.s_sh = s_sh;
  p.bt_sb = bt_sb; p.m_sl = m_sl; p.m_sb = m_sb; p.m_sh = m_sh;
  p.n_pages = n_pages; p.bt_cols = bt_cols; p.h_kv = H_KV; p.page_log2 = __builtin_ctz(static_cast<unsigned>(page));
  p.keep = keep; p.recent = recent; p.linear = kv_sp == page * kv_so;
  const int turn = evict_turn(L, B, H_KV, keep);
  const bool few = static_cast<int64_t>(H_KV) * turn * L <= 2 * static_cast<int64_t>(dev->sm_count);
  p.staged = static_cast<int>(std::min<int64_t>(static_cast<int64_t>(bt_cols) * page, few ? kEvictStage : kEvictStageMany));
  SPECQ_CUDA_TRY(ensure_dyn_smem(reinterpret_cast<const void*>(evict_select_kernel), kEvictStage * 4));
  const bool i8 = cache_dtype == SPECQ_CACHE_INT8;
  LaunchAttrs at(1);
  for (int b0 = 0; b0 < B; b0 += turn) {
    p.B = std::min(turn, B - b0);
    p.first = p.place + static_cast<int64_t>(L) * p.B * H_KV * keep;
    p.bt = block_tbl + b0 * bt_sb;
    p.ctx = ctx_len + b0;
    p.ctx_out = ctx_out + b0;
    p.mass = mass + b0 * m_sb;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(H_KV, p.B, L);
    cfg.blockDim = dim3(kEvictSelThreads);
    cfg.dynamicSmemBytes = static_cast<size_t>(p.staged) * 4;
    cfg.stream = static_cast<cudaStream_t>(stream);
    at.apply(cfg);
    SPECQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, evict_select_kernel, p));
    cfg.gridDim = dim3(2 * H_KV, p.B, L);
    cfg.blockDim = dim3(kEvictMoveThreads);
    cfg.dynamicSmemBytes = 0;
    cudaError_t e;
    if (D == 64) e = i8 ? cudaLaunchKernelEx(&cfg, evict_move_kernel<0, 64>, p) : cudaLaunchKernelEx(&cfg, evict_move_kernel<1, 64>, p);
    else e = i8 ? cudaLaunchKernelEx(&cfg, evict_move_kernel<0, 128>, p) : cudaLaunchKernelEx(&cfg, evict_move_kernel<1, 128>, p);
    SPECQ_CUDA_TRY(e);
  }
  return SPECQ_OK;
}

}  // namespace specq
