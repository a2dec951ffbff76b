// mass_wide.cuh -- the products of many query rows with the cached keys for attention_mass (mass.cuh) on tcgen05.
//
// A block takes 256 tokens of one sequence and KV head.  It widens their keys once, exactly, to fp16 tiles of [128 tokens x D] in
// shared memory (128-byte swizzle) and goes through the rows of q, 128 at a time.  Both tiles are
// K-major, so the same bytes serve as either operand: for the rows' maxima and sums the rows stand on the lanes of
// tensor memory (A = q, B = keys) and a thread owns a row; for the tokens' sums the tokens stand there (A = keys, B = q) and a thread
// owns a token.  Neither needs a shuffle.  One warp issues the two 128 x 128 products, two warpgroups take one
// each; the next rows of q come into their place as soon as both products are done.
//
// 256 rows (64 of 4 heads), 8 KV heads of 128, two sequences of 12 to 16 thousand tokens, B200: 128 us for both passes (mma.sync
// 163).  The exponentials, one for each score and pass, 16 a clock and SM, are 26 of them and keep their pipe 25 to
// 30 % busy, the products theirs 13 %; the rest is a block's start (lengths, table, keys, their widening: 9 of its 26
// thousand cycles) and waits for products and barriers.  Two blocks an SM cover that for one another: blocks of 512 tokens,
// one an SM, took 138 us.
#pragma once

#include <type_traits>

#include "mass.cuh"

namespace specq {

constexpr int kWideWork = 256;              // two warpgroups, one for each product
constexpr int kWideThreads = kWideWork + 32;   // and a warp that issues the products
constexpr int kWideTile = 128;
constexpr int kWideTiles = kWideWork / kWideTile;
constexpr int kWideChunk = kWideTiles * kWideTile;   // tokens of a block
constexpr uint32_t kWideColumns = 128u * kWideTiles; // of tensor memory: half of it

template <int D>
struct WideSmem {
  static constexpr int kTileBytes = (D / 64) * kWideTile * 128;
  uint8_t keys[kWideTiles][kTileBytes];
  uint8_t q[kTileBytes];
  float scale[kWideChunk / 8];              // of each eight tokens: their page's scale, times sm_scale log2 e
  // of each of the 128 rows at work and, while some warps are not yet done with those, of the next
  float factor[2][kWideTile];
  float minus_lse[2][kWideTile];
  int lim[2][kWideTile];                    // the last token that a row sees; -1: none
  float2 part[kWideTiles][kWideTile];       // each warpgroup's maxima and sums
  uint32_t bad[(kWideChunk / 8 + 31) / 32]; // a bit for each eight tokens that no page gives
  uint64_t full[kWideTiles];
  uint32_t tmem;
};

// 16 stored numbers to 16 halves.
template <int CT>
__device__ __forceinline__ void widen16(const uint4& u, uint4& lo, uint4& hi) {
  widen4<CT>(u.x, lo.x, lo.y);
  widen4<CT>(u.y, lo.z, lo.w);
  widen4<CT>(u.z, hi.x, hi.y);
  widen4<CT>(u.w, hi.z, hi.w);
}

// Where 16-byte chunk `c` of row `r` of a [128 x D] tile of halves stands.
__device__ __forceinline__ uint32_t wide_at(int r, int c) {
  return static_cast<uint32_t>(c >> 3) * (kWideTile * 128u) + sw128_offset(static_cast<uint32_t>(r), static_cast<uint32_t>(c & 7));
}

template <bool BF, int CT, int D, int MODE>
__global__ void __launch_bounds__(kWideThreads, 2) mass_wide_kernel(const __grid_constant__ MassParams p) {
  using Smem = WideSmem<D>;
  extern __shared__ uint8_t raw_smem[];
  Smem& sm = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~uintptr_t(1023));
  pdl_wait();
  const int chunk = blockIdx.x, h = blockIdx.y, b = blockIdx.z, tid = static_cast<int>(threadIdx.x);
  const int warp = tid >> 5, lane = tid & 31, group = warp >> 2;       // the last group: the issuing warp
  int n, nr;
  mass_extent(p, b, chunk == 0 && h == 0 && tid == 0 && MODE == kMassStats, n, nr);
  const int first_token = chunk * kWideChunk;
  if (nr == 0 || first_token >= n) return;
  const int64_t bh = static_cast<int64_t>(b) * p.h_kv + h;
  const int rows = nr * p.group, base = n - nr;
  const int tiles = min(kWideTiles, (n - first_token + kWideTile - 1) / kWideTile);
  const int mask = (1 << p.page_log2) - 1;

  if (group == kWideTiles) {
    tmem_alloc(&sm.tmem, kWideColumns);
    tmem_relinquish();
    if (lane < kWideTiles) mbar_init(&sm.full[lane], 1u);
    fence_barrier_init();
  }
  // q's rows [first, first + 128) of this head, as they are, two threads a row; rows past the last are zeros
  constexpr int kMine = D / 16;              // 16-byte chunks of a thread
  const int my_row = tid >> 1, my_chunk = (tid & 1) * kMine;
  auto request = [&](int first) {
    const int r = first + my_row;
    if (r < rows) {
      const int row = r / p.group, head = h * p.group + r - row * p.group;
      const __half* src = static_cast<const __half*>(p.q) + my_chunk * 8 + head * p.q_sh +
                          (p.q_sb != 0 ? b * p.q_sb + row * p.q_st : (static_cast<int64_t>(b) * p.q_len + row) * p.q_st);
#pragma unroll
      for (int c = 0; c < kMine; ++c)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(sm.q + wide_at(my_row, my_chunk + c))), "l"(src + c * 8) : "memory");
    } else {
#pragma unroll
      for (int c = 0; c < kMine; ++c) *reinterpret_cast<uint4*>(sm.q + wide_at(my_row, my_chunk + c)) = make_uint4(0u, 0u, 0u, 0u);
    }
  };
  // each row's factor (and the halves it stands for, in place), limit and lse, by the threads that asked for it
  auto finish = [&](int first, int side, float lse) {
    using W2 = typename std::conditional<BF, __nv_bfloat162, __half2>::type;
    uint32_t seen = 0u;                      // the largest magnitudes, a NaN kept
    auto add = [&](uint32_t w) {
      const W2 m = __hmax2_nan(*reinterpret_cast<const W2*>(&seen), __habs2(*reinterpret_cast<const W2*>(&w)));
      seen = *reinterpret_cast<const uint32_t*>(&m);
    };
#pragma unroll
    for (int c = 0; c < kMine; ++c) {
      const uint4 u = *reinterpret_cast<const uint4*>(sm.q + wide_at(my_row, my_chunk + c));
      add(u.x);
      add(u.y);
      add(u.z);
      add(u.w);
    }
    uint32_t top = max(seen & 0x7FFFu, seen >> 16 & 0x7FFFu);     // magnitudes order as integers: infinity and NaN last
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    const bool finite = top < (BF ? 0x7F80u : 0x7C00u);
    float factor = 1.f;
    if (BF || !finite) {
      float up = 1.f;
      if constexpr (BF) {
        // the largest element times 2^k in [2^14, 2^15); 2^126 suffices for what is not zero beside any key
        const int k = top != 0u && finite ? min(14 - ilogbf(__uint_as_float(top << 16)), 126) : 0;
        up = __int_as_float((127 + k) << 23);                      // k >= 14 - 127
        factor = row_factor(k);
      }
#pragma unroll
      for (int c = 0; c < kMine; ++c) {
        uint4* at = reinterpret_cast<uint4*>(sm.q + wide_at(my_row, my_chunk + c));
        const uint4 u = *at;
        uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const __half2 v = __floats2half2_rn(__uint_as_float(w[j] << 16) * up, __uint_as_float(w[j] & 0xFFFF0000u) * up);
          w[j] = finite ? *reinterpret_cast<const uint32_t*>(&v) : 0u;
        }
        *at = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    if ((tid & 1) == 0) {
      const bool there = first + my_row < rows;
      sm.factor[side][my_row] = factor;
      sm.lim[side][my_row] = there && finite ? base + (first + my_row) / p.group : -1;
      sm.minus_lse[side][my_row] = there ? -lse : -INFINITY;
    }
  };
  auto lse_of = [&](int first) {
    const int r = first + my_row;
    return MODE == kMassWeights && tid < kWideWork && r < rows ? p.lse[bh * p.rows + r] : INFINITY;
  };

  float next_lse = lse_of(0);
  if (tid < kWideWork) {
    request(0);
    // scales of the chunk's 32 runs of eight tokens
    if (tid < kWideChunk / 8) {
      const int t = first_token + tid * 8;
      int pg = -1;
      if (t < n) {
        pg = p.bt[b * p.bt_sb + (t >> p.page_log2)];
        if (pg < 0 || pg >= p.n_pages) {
          report_status(p.status, SPECQ_STATUS_BAD_INDEX);
          pg = -1;
        }
      }
      sm.scale[tid] = pg >= 0 ? p.ks[pg * p.s_sp + h * p.s_sh] * p.sm_log2 : 1.f;
      const uint32_t gone = __ballot_sync(0xffffffffu, pg < 0);
      if (lane == 0) sm.bad[warp] = gone;
    }
    // the keys, two threads a token, 32 bytes side by side at a time
    static_assert(kWideChunk == kWideWork, "two tokens for each pair of threads");
    constexpr int kPieces = D / 32;
    uint4 w[2][kPieces];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int t = first_token + i * kWideTile + (tid >> 1);
      int pg = -1;
      if (t < n) pg = p.bt[b * p.bt_sb + (t >> p.page_log2)];
      const bool there = pg >= 0 && pg < p.n_pages;
      const uint8_t* src = p.kc + (there ? pg * p.kv_sp + (t & mask) * p.kv_so + h * p.kv_sh : 0) + (tid & 1) * 16;
#pragma unroll
      for (int j = 0; j < kPieces; ++j) w[i][j] = there ? *reinterpret_cast<const uint4*>(src + j * 32) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < kPieces; ++j) {
        const int c = 4 * j + 2 * (tid & 1);
        uint4 lo, hi;
        widen16<CT>(w[i][j], lo, hi);
        *reinterpret_cast<uint4*>(sm.keys[i] + wide_at(tid >> 1, c)) = lo;
        *reinterpret_cast<uint4*>(sm.keys[i] + wide_at(tid >> 1, c + 1)) = hi;
      }
  }

  float weight = 0.f;                        // of this thread's token
  const uint32_t quarter = static_cast<uint32_t>(warp & 3) * 32u;      // this warp's lanes of tensor memory
  const int me = static_cast<int>(quarter) + lane;
  uint32_t tmem = 0, phase = 0;
  for (int first = 0; first < rows; first += kWideTile, phase ^= 1u) {
    const int here = min(kWideTile, rows - first), pad = (here + 15) & ~15;
    const int side = static_cast<int>(phase);
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (tid < kWideWork) finish(first, side, next_lse);   // (a thread's own bytes)
    fence_proxy_async_smem();
    tc_fence_before();
    __syncthreads();                         // both operands are there; the products before have been read
    tc_fence_after();
    tmem = sm.tmem;
    if (first == 0) pdl_launch_dependents(); // (tensor memory is taken: what may start now cannot keep it from this block)
    if (group == kWideTiles) {
      if (elect_one()) {
        const uint64_t qd = sdesc_sw128(smem_u32(sm.q), 16u, 1024u);
        const uint32_t idesc = idesc_f16(128u, MODE == kMassStats ? 128u : static_cast<uint32_t>(pad));
        for (int t = 0; t < tiles; ++t) {
          const uint64_t kd = sdesc_sw128(smem_u32(sm.keys[t]), 16u, 1024u);
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {   // 32 bytes of a 128-byte row each, then the next 64 elements' rows
            const uint64_t step = static_cast<uint64_t>((k >> 2) * (kWideTile * 128 / 16) + (k & 3) * 2);
            umma_f16_ss(tmem + 128u * t, MODE == kMassStats ? qd + step : kd + step, MODE == kMassStats ? kd + step : qd + step, idesc, k > 0);
          }
          umma_commit(&sm.full[t]);
        }
      }
      __syncwarp();
    } else {
      float m = -INFINITY, l = 0.f;
      const int t = group;
      const bool more = first + kWideTile < rows;
      if (more) {                              // q's place is free when every product has read it
        for (int i = 0; i < tiles; ++i) (void)mbar_wait(&sm.full[i], phase, p.status, SPECQ_STATUS_TIMEOUT_MMA);
        request(first + kWideTile);
        next_lse = lse_of(first + kWideTile);
      }
      if (t < tiles) {
        if (!more) (void)mbar_wait(&sm.full[t], phase, p.status, SPECQ_STATUS_TIMEOUT_MMA);
        tc_fence_after();
        const uint32_t at = tmem + (quarter << 16) + 128u * t;
        const int token0 = first_token + t * kWideTile;
        const uint32_t gone = sm.bad[t >> 1] >> ((t & 1) * 16) & 0xFFFFu;   // 16 runs of eight tokens a tile
        const bool hidden = gone != 0u || token0 + kWideTile - 1 > base;
        if constexpr (MODE == kMassStats) {
          if (static_cast<int>(quarter) < here) {              // (a warp with rows)
            const float* scale = sm.scale + t * (kWideTile / 8);
            const float mine = sm.factor[side][me];
            const int my_lim = sm.lim[side][me];
            uint32_t v[2][16];
            tmem_ld16(at, v[0]);
#pragma unroll
            for (int c = 0; c < kWideTile; c += 16) {          // the next 16 columns on their way
              uint32_t(&u)[16] = v[(c / 16) & 1];
              tmem_wait_ld();
              if (c + 16 < kWideTile) tmem_ld16(at + c + 16, v[(c / 16 + 1) & 1]);
              const float2 xs = *reinterpret_cast<const float2*>(scale + c / 8);
              const float x[2] = {BF ? xs.x * mine : xs.x, BF ? xs.y * mine : xs.y};
#pragma unroll
              for (int k = 0; k < 16; ++k) u[k] = __float_as_uint(__fmul_rn(__uint_as_float(u[k]), x[k / 8]));   // see `scale` in mass.cuh
              if (hidden) {                                     // after the scaling: see `hide` there
#pragma unroll
                for (int k = 0; k < 16; ++k)
                  if ((gone >> ((c + k) / 8) & 1u) != 0u || token0 + c + k > my_lim) u[k] = 0xFF800000u;
              }
              float top = m;
#pragma unroll
              for (int k = 0; k < 16; ++k) top = fmaxf(top, __uint_as_float(u[k]));
              const float z = top == -INFINITY ? 0.f : -top;
              float2 sum = {l * exp2_fast(m + z), 0.f};         // m = -inf: 0
#pragma unroll
              for (int k = 0; k < 16; k += 2) {
                const float2 d = __fadd2_rn(make_float2(__uint_as_float(u[k]), __uint_as_float(u[k + 1])), make_float2(z, z));
                sum = __fadd2_rn(sum, make_float2(exp2_fast(d.x), exp2_fast(d.y)));
              }
              l = sum.x + sum.y;
              m = top;
            }
          }
        } else {
          const float x = sm.scale[t * (kWideTile / 8) + me / 8];
          float2 sum = {0.f, 0.f};
          uint32_t v[2][16];
          tmem_ld16(at, v[0]);
#pragma unroll
          for (int c = 0; c < kWideTile; c += 16) {
            if (c >= pad) break;
            uint32_t(&u)[16] = v[(c / 16) & 1];
            tmem_wait_ld();
            if (c + 16 < pad) tmem_ld16(at + c + 16, v[(c / 16 + 1) & 1]);
#pragma unroll
            for (int k = 0; k < 16; k += 4) {
              float4 lse = *reinterpret_cast<const float4*>(sm.minus_lse[side] + c + k);
              float2 s0 = make_float2(__uint_as_float(u[k]), __uint_as_float(u[k + 1])), s1 = make_float2(__uint_as_float(u[k + 2]), __uint_as_float(u[k + 3]));
              if constexpr (BF) {
                const float4 f = *reinterpret_cast<const float4*>(sm.factor[side] + c + k);
                s0 = __fmul2_rn(s0, make_float2(f.x, f.y));
                s1 = __fmul2_rn(s1, make_float2(f.z, f.w));
              }
              if (hidden) {
                const int4 lim = *reinterpret_cast<const int4*>(sm.lim[side] + c + k);
                if (token0 + me > lim.x) lse.x = -INFINITY;
                if (token0 + me > lim.y) lse.y = -INFINITY;
                if (token0 + me > lim.z) lse.z = -INFINITY;
                if (token0 + me > lim.w) lse.w = -INFINITY;
              }
              // (s f) x is s (f x) to the bit, f being a power of two: the scores of the other pass
              s0 = mul2_rounded(s0, make_float2(x, x));
              s1 = mul2_rounded(s1, make_float2(x, x));
              const float2 d0 = __fadd2_rn(s0, make_float2(lse.x, lse.y)), d1 = __fadd2_rn(s1, make_float2(lse.z, lse.w));
              sum = __fadd2_rn(sum, make_float2(exp2_fast(d0.x), exp2_fast(d0.y)));
              sum = __fadd2_rn(sum, make_float2(exp2_fast(d1.x), exp2_fast(d1.y)));
            }
          }
          if ((gone >> (me / 8) & 1u) == 0u) weight += sum.x + sum.y;
        }
      }
      if constexpr (MODE == kMassStats) sm.part[group][me] = make_float2(m, l);
    }
    if constexpr (MODE == kMassStats) {
      __syncthreads();
      if (tid < here) {
        float2 x = sm.part[0][tid];
#pragma unroll
        for (int g = 1; g < kWideTiles; ++g) x = join_stats(x, sm.part[g][tid]);
        if (sm.lim[side][tid] < 0) x = make_float2(-INFINITY, 0.f);
        p.stats[(bh * p.chunks + chunk) * p.rows + first + tid] = x;
      }
    }
  }
  if constexpr (MODE == kMassWeights) {
    const int t = first_token + tid;         // group * 128 + me
    if (tid < kWideWork && t < n) {
      float* at = p.mass + b * p.m_sb + h * p.m_sh + t;
      *at = fmaf(*at, p.decay, weight);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (group == kWideTiles) {
    tc_fence_after();
    tmem_dealloc(tmem, kWideColumns);
  }
}

}  // namespace specq
