// mass_api.cuh -- how attention_mass is cut into launches: clusters, streams of tiles, or tcgen05 products, by rows and table; and into
// turns over one workspace where its sums or scores would fill more.
#pragma once

#include "mass_wide.cuh"

namespace specq {

inline int mass_check(int B, int q_len, int H, int H_KV, int D, int page, int bt_cols) {
  const char* who = "attention_mass";
  if (B < 0 || q_len < 0 || H < 1 || H_KV < 1 || H % H_KV || bt_cols < 0)
    return fail(SPECQ_ERR_INVALID_ARG, "%s: B=%d q_len=%d H=%d H_KV=%d bt_cols=%d", who, B, q_len, H, H_KV, bt_cols);
  if (D != 64 && D != 128) return fail(SPECQ_ERR_UNSUPPORTED, "%s: head_dim %d (64 or 128)", who, D);
  if (page < 8 || page > 128 || (page & (page - 1))) return fail(SPECQ_ERR_UNSUPPORTED, "%s: page %d (a power of two, 8 to 128)", who, page);
  if (B > 65535 || H_KV > 65535 || static_cast<int64_t>(bt_cols) * page > 0x7ffff000ll || static_cast<int64_t>(q_len) * (H / H_KV) > 0x7fffff00ll)
    return fail(SPECQ_ERR_UNSUPPORTED, "%s: B=%d H_KV=%d, %d pages of %d, %d rows of %d heads", who, B, H_KV, bt_cols, page, q_len, H / H_KV);
  return SPECQ_OK;
}

// Why from kMassWide rows on the products go to tcgen05: 96 rows of one short sequence 16 us against 23, 256 rows of 4 x 1500 tokens 40 against 75,
// of two long prompts 128 against 163; but 64 rows of 8 x 4096 tokens 73 against 52 (half of the 128 lanes have no row).

// How a call is cut: whether clusters hold the whole table, else the tokens of a block (chunk_tiles * 256) and blocks a head.
inline bool mass_plan(int B, int H_KV, int rows, int tokens, int* chunk_tiles, int* chunks) {
  *chunk_tiles = kMassChunk / kMassThreads;
  *chunks = ceil_div(tokens, kMassChunk);
  // up to 16 rows a cluster is the faster only while most SMs would be idle: 1 x 4096 tokens of 8 heads 8.5 us against 9.2, but 8 x 1024
  // 10.8 against 9.9 and 32 x 4096 76 against 52
  if (rows >= kMassWide) {
    *chunk_tiles = kWideChunk / kMassThreads;
    *chunks = ceil_div(tokens, kWideChunk);
    return false;
  }
  if (*chunks <= kMassCluster && (rows > kMassFew || *chunks == 1 || static_cast<int64_t>(B) * H_KV * *chunks <= kMassSms / 2)) return true;
  if (rows <= kMassFew) {            // long blocks pay for q once; three blocks an SM at least, if the call has them
    int tiles = 8;
    while (tiles > 2 && static_cast<int64_t>(B) * H_KV * ceil_div(tokens, tiles * kMassThreads) < 3 * kMassSms) tiles /= 2;
    *chunk_tiles = tiles;
    *chunks = ceil_div(tokens, tiles * kMassThreads);
  }
  return false;
}

// What a call keeps in its workspace goes by the table's width, whatever is cached of it: 4 bytes for each row and token (up to 16 rows),
// or 8 for each row and block of 256 or 512 tokens, of every KV head of every sequence.  Past kTurnSpace it goes through its sequences, or
// the KV heads of one, in several turns of one size over the same workspace, which is then at most that or what one KV head of one
// sequence takes.  (16 rows of 64 sequences, 8 heads and a table of 131072 tokens: 512 MB in place of 4.3 GB.  A turn costs some 10 us: the
// same rows of 32 sequences of 32768 tokens take 454 us in one turn of 540 MB, 470 in two and 497 in three.)

struct MassCut {
  bool whole;                  // in one launch, without a workspace
  int chunk_tiles, chunks;
  int seqs, heads;             // of a turn
  int64_t bytes;               // of a turn
};

inline MassCut mass_cut(int B, int H_KV, int rows, int tokens) {
  MassCut c = {};
  c.whole = mass_plan(B, H_KV, rows, tokens, &c.chunk_tiles, &c.chunks);
  c.seqs = B;
  c.heads = H_KV;
  if (c.whole || B == 0) return c;
  const int64_t stats = static_cast<int64_t>(rows) * c.chunks * 8;
  const int64_t one = stats + (rows <= kMassFew ? static_cast<int64_t>(rows) * c.chunks * c.chunk_tiles * kMassThreads * 4 : static_cast<int64_t>(rows) * 4);
  if (one > 0) {
    c.seqs = even_turn(B, kTurnSpace / (one * H_KV));
    if (one * H_KV > kTurnSpace) c.heads = even_turn(H_KV, kTurnSpace / one);
  }
  c.bytes = one * c.seqs * c.heads;
  return c;
}

inline int run_attention_mass_workspace(int B, int q_len, int H, int H_KV, int D, int page, int bt_cols, int64_t* bytes) {
  if (bytes == nullptr) return fail(SPECQ_ERR_INVALID_ARG, "attention_mass_workspace: null pointer");
  if (int rc = mass_check(B, q_len, H, H_KV, D, page, bt_cols)) return rc;
  *bytes = mass_cut(B, H_KV, q_len * (H / H_KV), bt_cols * page).bytes;
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
  if (!(sm_scale > 0.f) || !(sm_scale < 2e38f)) return fail(SPECQ_ERR_INVALID_ARG, "%s: sm_scale %g", who, static_cast<double>(sm_scale));
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
  p.kc = static_cast<const uint8_t*>(kc);
  p.status = dev->status;
  p.q_sb = q_sb; p.q_st = q_st; p.q_sh = q_sh; p.kv_sp = kv_sp; p.kv_so = kv_so; p.kv_sh = kv_sh; p.s_sp = s_sp; p.s_sh = s_sh;
  p.bt_sb = bt_sb; p.m_sb = m_sb; p.m_sh = m_sh;
  p.q_len = q_len; p.group = H / H_KV; p.page_log2 = __builtin_ctz(static_cast<unsigned>(page));
  p.n_pages = n_pages; p.bt_cols = bt_cols; p.rows = q_len * p.group;
  p.sm_log2 = sm_scale * kLog2E; p.decay = decay;
  const MassCut cut = mass_cut(B, H_KV, p.rows, bt_cols * page);
  const bool whole = cut.whole;
  p.chunk_tiles = cut.chunk_tiles;
  p.chunks = cut.chunks;
  p.stats = static_cast<float2*>(workspace);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int here = B;                // sequences of this turn (its KV heads: p.h_kv)
  auto launch = [&](auto kern, size_t smem, int threads = kMassThreads) {
    int cluster = 1;
    cudaError_t e = ensure_dyn_smem(reinterpret_cast<const void*>(kern), static_cast<int>(smem));
    if (e != cudaSuccess) return e;
    if (whole) cluster = next_pow2(p.chunks);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(whole ? cluster : p.chunks, p.h_kv, here);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    LaunchAttrs at(cluster);
    at.apply(cfg);
    return cudaLaunchKernelEx(&cfg, kern, p);
  };
  auto all = [&](auto bf, auto ct, auto d) -> int {
    constexpr bool BF = decltype(bf)::value;
    constexpr int CT = decltype(ct)::value, DD = decltype(d)::value;
    const size_t few = sizeof(MassSmem<DD, kMassFew>), many = sizeof(MassSmem<DD, kMassRows>);
    if (p.rows <= kMassFew) {
      if (whole) {
        SPECQ_CUDA_TRY(launch(mass_kernel<BF, CT, DD, kMassFew, kMassWhole>, few));
        return SPECQ_OK;
      }
      SPECQ_CUDA_TRY(launch(mass_stream_kernel<BF, CT, DD>, sizeof(MassStreamSmem<DD>)));
      SPECQ_CUDA_TRY(launch_plain(mass_sum_kernel, dim3(ceil_div(bt_cols * page, kMassSumTokens), p.h_kv, here), dim3(kMassThreads), st, p));
      return SPECQ_OK;
    }
    if (p.rows >= kMassWide) {
      const size_t wide = sizeof(WideSmem<DD>) + 1024;
      SPECQ_CUDA_TRY(launch(mass_wide_kernel<BF, CT, DD, kMassStats>, wide, kWideThreads));
      SPECQ_CUDA_TRY(launch_plain(mass_join_kernel, dim3(ceil_div(p.rows, 8), p.h_kv, here), dim3(256), st, p));
      SPECQ_CUDA_TRY(launch(mass_wide_kernel<BF, CT, DD, kMassWeights>, wide, kWideThreads));
      return SPECQ_OK;
    }
    if (whole) {
      SPECQ_CUDA_TRY(launch(mass_kernel<BF, CT, DD, kMassRows, kMassWhole>, many));
      return SPECQ_OK;
    }
    SPECQ_CUDA_TRY(launch(mass_kernel<BF, CT, DD, kMassRows, kMassStats>, many));
    SPECQ_CUDA_TRY(launch_plain(mass_join_kernel, dim3(ceil_div(p.rows, 8), p.h_kv, here), dim3(256), st, p));
    SPECQ_CUDA_TRY(launch(mass_kernel<BF, CT, DD, kMassRows, kMassWeights>, many));
    return SPECQ_OK;
  };
  auto by_d = [&](auto bf, auto ct) { return D == 64 ? all(bf, ct, std::integral_constant<int, 64>{}) : all(bf, ct, std::integral_constant<int, 128>{}); };
  auto by_ct = [&](auto bf) {
    return cache_dtype == SPECQ_CACHE_INT8 ? by_d(bf, std::integral_constant<int, 0>{}) : by_d(bf, std::integral_constant<int, 1>{});
  };
  const MassParams every = p;
  for (int b0 = 0; b0 < B; b0 += cut.seqs)
    for (int h0 = 0; h0 < H_KV; h0 += cut.heads) {
      here = std::min(cut.seqs, B - b0);
      p.h_kv = std::min(cut.heads, H_KV - h0);
      p.q = static_cast<const __half*>(q) + b0 * (q_sb != 0 ? q_sb : q_len * q_st) + h0 * every.group * q_sh;
      p.kc = every.kc + h0 * kv_sh;
      p.ks = ks + h0 * s_sh;
      p.bt = block_tbl + b0 * bt_sb;
      p.ctx = ctx_len + b0;
      p.n_rows = n_rows == nullptr ? nullptr : n_rows + b0;
      p.mass = mass + b0 * m_sb + h0 * m_sh;
      p.score = p.lse = reinterpret_cast<float*>(p.stats + (whole ? 0 : static_cast<int64_t>(here) * p.h_kv * p.chunks * p.rows));
      if (int rc = dtype == SPECQ_DTYPE_F16 ? by_ct(std::false_type{}) : by_ct(std::true_type{})) return rc;
    }
  return SPECQ_OK;
}

}  // namespace specq
