// mass_wide.cuh -- the products of many query rows with the cached keys for attention_mass (mass.cuh) on tcgen05.
//
// A block takes 512 tokens of one sequence and KV head.  It widens their keys once, exactly, to fp16 tiles of [128 tokens x D] in
// shared memory (128-byte swizzle) and goes through the rows of q, 128 at a time, the next ones on their way.  Both tiles are
// K-major, so the same bytes serve as either operand: for the rows' maxima and sums the rows stand on the lanes of
// tensor memory (A = q, B = keys) and a thread owns a row; for the tokens' sums the tokens stand there (A = keys, B = q) and a thread
// owns a token.  Neither needs a shuffle.  Four 128 x 128 products fill the tensor memory; one warp issues them, four
// warpgroups take one each.
//
// Bound by the exponentials: one for each score and pass, 16 a clock and SM, against 8192 products; what the block does before
// its first product (lengths, table, keys, their widening) is not covered by another block of its SM.
#pragma once

#include "mass.cuh"

namespace specq {

constexpr int kWideWork = 512;              // four warpgroups, one for each product
constexpr int kWideThreads = kWideWork + 32;   // and a warp that issues the products
constexpr int kWideTile = 128;
constexpr int kWideTiles = kMassChunk / kWideTile;
static_assert(kWideTiles == 4 && kMassRows == kWideTile, "four products of 128 columns fill the tensor memory");

template <int D>
struct WideSmem {
  static constexpr int kTileBytes = (D / 64) * kWideTile * 128;
  uint8_t keys[kWideTiles][kTileBytes];
  uint8_t q[2][kTileBytes];
  float4 dummy_align;
  float scale[kMassChunk / 8];              // of each eight tokens: their page's scale, times sm_scale log2 e
  float factor[kWideTile];                  // of each row
  float minus_lse[kWideTile];
  int lim[kWideTile];                       // the last token that a row sees; -1: none
  float2 part[kWideTiles][kWideTile];       // each warpgroup's maxima and sums
  uint32_t bad[kMassChunk / 8 / 32];        // a bit for each eight tokens that no page gives
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
__global__ void __launch_bounds__(kWideThreads, 1) mass_wide_kernel(const __grid_constant__ MassParams p) {
  using Smem = WideSmem<D>;
  extern __shared__ uint8_t raw_smem[];
  Smem& sm = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~uintptr_t(1023));
  pdl_wait();
  const int chunk = blockIdx.x, h = blockIdx.y, b = blockIdx.z, tid = static_cast<int>(threadIdx.x);
  const int warp = tid >> 5, lane = tid & 31, group = warp >> 2;       // group 4: the issuing warp
  int n, nr;
  mass_extent(p, b, chunk == 0 && h == 0 && tid == 0 && MODE == kMassStats, n, nr);
  const int first_token = chunk * kMassChunk;
  if (nr == 0 || first_token >= n) return;
  const int64_t bh = static_cast<int64_t>(b) * p.h_kv + h;
  const int rows = nr * p.group, base = n - nr;
  const int tiles = min(kWideTiles, (n - first_token + kWideTile - 1) / kWideTile);
  const int mask = (1 << p.page_log2) - 1;

  if (group == 4) {
    tmem_alloc(&sm.tmem, 512u);
    tmem_relinquish();
    if (lane < kWideTiles) mbar_init(&sm.full[lane], 1u);
    fence_barrier_init();
  }
  // q's rows [first, first + 128) of this head, as they are, into buffer `side`; rows past the last are zeros
  auto request = [&](int first, int side) {
    constexpr int kChunks = D / 8;
    const int here = min(kWideTile, rows - first);
#pragma unroll
    for (int i = tid; i < kWideTile * kChunks; i += kWideWork) {
      const int r = i / kChunks, c = i - r * kChunks;
      uint8_t* dst = sm.q[side] + wide_at(r, c);
      if (r < here) {
        const int row = (first + r) / p.group, head = h * p.group + (first + r) - row * p.group;
        const int64_t at = (p.q_sb != 0 ? b * p.q_sb + row * p.q_st : (static_cast<int64_t>(b) * p.q_len + row) * p.q_st) + head * p.q_sh;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(static_cast<const __half*>(p.q) + at + c * 8) : "memory");
      } else {
        *reinterpret_cast<uint4*>(dst) = make_uint4(0u, 0u, 0u, 0u);
      }
    }
  };
  // each row's factor (and the halves it stands for, in place), limit and lse; four threads a row
  auto finish = [&](int first, int side, float lse) {
    constexpr int kMine = D / 32;            // chunks of a thread
    const int r = tid >> 2, c0 = (tid & 3) * kMine, here = min(kWideTile, rows - first);
    uint32_t top = 0u;                       // the larger of the halves' magnitudes: infinity and NaN last
#pragma unroll
    for (int c = 0; c < kMine; ++c) {
      const uint4 u = *reinterpret_cast<const uint4*>(sm.q[side] + wide_at(r, c0 + c));
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) top = max(top, max(w[k] & 0x7FFFu, w[k] >> 16 & 0x7FFFu));
    }
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const bool finite = top < (BF ? 0x7F80u : 0x7C00u);
    float factor = 1.f;
    if (BF || !finite) {
      float up = 1.f;
      if constexpr (BF) {
        // the largest element times 2^k in [2^14, 2^15); 2^126 suffices for what is not zero beside any key
        const int k = top != 0u && finite ? min(14 - ilogbf(__uint_as_float(top << 16)), 126) : 0;
        up = __int_as_float((127 + k) << 23);                      // k >= 14 - 127
        factor = __int_as_float((127 - k) << 23);
      }
#pragma unroll
      for (int c = 0; c < kMine; ++c) {
        uint4* at = reinterpret_cast<uint4*>(sm.q[side] + wide_at(r, c0 + c));
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
    if ((tid & 3) == 0) {
      sm.factor[r] = factor;
      sm.lim[r] = r < here && finite ? base + (first + r) / p.group : -1;
      sm.minus_lse[r] = r < here ? -lse : -INFINITY;
    }
  };
  auto lse_of = [&](int first) {
    const int r = first + (tid >> 2);
    return MODE == kMassWeights && tid < kWideWork && r < rows ? p.lse[bh * p.rows + r] : INFINITY;
  };

  float next_lse = lse_of(0);
  if (tid < kWideWork) {
    request(0, 0);
    // scales of the chunk's 64 runs of eight tokens
    if (tid < kMassChunk / 8) {
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
    // the keys: 16 bytes a thread and turn, all turns' loads in flight
    constexpr int kPer = D / 16, kTurns = kMassChunk * kPer / kWideWork;
    uint4 w[kTurns];
#pragma unroll
    for (int j = 0; j < kTurns; ++j) {
      const int i = tid + j * kWideWork, t = first_token + i / kPer;
      w[j] = make_uint4(0u, 0u, 0u, 0u);
      if (t < n) {
        const int pg = p.bt[b * p.bt_sb + (t >> p.page_log2)];
        if (pg >= 0 && pg < p.n_pages)
          w[j] = *reinterpret_cast<const uint4*>(p.kc + pg * p.kv_sp + (t & mask) * p.kv_so + h * p.kv_sh + (i % kPer) * 16);
      }
    }
#pragma unroll
    for (int j = 0; j < kTurns; ++j) {
      const int i = tid + j * kWideWork, t = i / kPer, c = (i % kPer) * 2;
      uint4 lo, hi;
      widen16<CT>(w[j], lo, hi);
      uint8_t* tile = sm.keys[t / kWideTile];
      *reinterpret_cast<uint4*>(tile + wide_at(t % kWideTile, c)) = lo;
      *reinterpret_cast<uint4*>(tile + wide_at(t % kWideTile, c + 1)) = hi;
    }
  }

  float weight = 0.f;                        // of this thread's token
  const uint32_t quarter = static_cast<uint32_t>(warp & 3) * 32u;      // this warp's lanes of tensor memory
  const int me = static_cast<int>(quarter) + lane;
  uint32_t tmem = 0, phase = 0;
  for (int first = 0, side = 0; first < rows; first += kWideTile, side ^= 1, phase ^= 1u) {
    const int here = min(kWideTile, rows - first), pad = (here + 15) & ~15;
    asm volatile("cp.async.wait_all;" ::: "memory");
    tc_fence_before();
    __syncthreads();                         // q's bytes are there; the products before have been read
    tc_fence_after();
    tmem = sm.tmem;
    if (first == 0) pdl_launch_dependents(); // (tensor memory is taken: what may start now cannot keep it from this block)
    if (tid < kWideWork) finish(first, side, next_lse);
    fence_proxy_async_smem();
    __syncthreads();
    if (group == 4) {
      if (elect_one()) {
        const uint64_t qd = sdesc_sw128(smem_u32(sm.q[side]), 16u, 1024u);
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
      if (first + kWideTile < rows) {
        request(first + kWideTile, side ^ 1);
        next_lse = lse_of(first + kWideTile);
      }
      float m = -INFINITY, l = 0.f;
      const int t = group;
      if (t < tiles) {
        (void)mbar_wait(&sm.full[t], phase, p.status, SPECQ_STATUS_TIMEOUT_MMA);
        tc_fence_after();
        const uint32_t at = tmem + (quarter << 16) + 128u * t;
        const int token0 = first_token + t * kWideTile;
        const uint32_t gone = sm.bad[t >> 1] >> ((t & 1) * 16) & 0xFFFFu;   // 16 runs of eight tokens a tile
        const bool hidden = gone != 0u || token0 + kWideTile - 1 > base;
        if constexpr (MODE == kMassStats) {
          if (static_cast<int>(quarter) < here) {              // (a warp with rows)
            const float* scale = sm.scale + t * (kWideTile / 8);
            const float mine = sm.factor[me];
            const int my_lim = sm.lim[me];
            uint32_t v[2][16];
            tmem_ld16(at, v[0]);
#pragma unroll
            for (int c = 0; c < kWideTile; c += 16) {          // the next 16 columns on their way
              uint32_t(&u)[16] = v[(c / 16) & 1];
              tmem_wait_ld();
              if (c + 16 < kWideTile) tmem_ld16(at + c + 16, v[(c / 16 + 1) & 1]);
              const float2 xs = *reinterpret_cast<const float2*>(scale + c / 8);
              const float x[2] = {BF ? xs.x * mine : xs.x, BF ? xs.y * mine : xs.y};
              if (hidden) {
#pragma unroll
                for (int k = 0; k < 16; ++k)
                  if ((gone >> ((c + k) / 8) & 1u) != 0u || token0 + c + k > my_lim) u[k] = 0xFF800000u;
              }
              float top = m;
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                float y = __uint_as_float(u[j * 8]);
#pragma unroll
                for (int k = 1; k < 8; ++k) y = fmaxf(y, __uint_as_float(u[j * 8 + k]));
                top = fmaxf(top, y * x[j]);
              }
              const float z = top == -INFINITY ? 0.f : -top;
              float2 sum = {l * exp2_fast(m + z), 0.f};         // m = -inf: 0
#pragma unroll
              for (int k = 0; k < 16; k += 2) {
                const float2 d = __ffma2_rn(make_float2(__uint_as_float(u[k]), __uint_as_float(u[k + 1])), make_float2(x[k / 8], x[k / 8]), make_float2(z, z));
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
              float4 lse = *reinterpret_cast<const float4*>(sm.minus_lse + c + k);
              float2 s0 = make_float2(__uint_as_float(u[k]), __uint_as_float(u[k + 1])), s1 = make_float2(__uint_as_float(u[k + 2]), __uint_as_float(u[k + 3]));
              if constexpr (BF) {
                const float4 f = *reinterpret_cast<const float4*>(sm.factor + c + k);
                s0 = __fmul2_rn(s0, make_float2(f.x, f.y));
                s1 = __fmul2_rn(s1, make_float2(f.z, f.w));
              }
              if (hidden) {
                const int4 lim = *reinterpret_cast<const int4*>(sm.lim + c + k);
                if (token0 + me > lim.x) lse.x = -INFINITY;
                if (token0 + me > lim.y) lse.y = -INFINITY;
                if (token0 + me > lim.z) lse.z = -INFINITY;
                if (token0 + me > lim.w) lse.w = -INFINITY;
              }
              const float2 d0 = __ffma2_rn(s0, make_float2(x, x), make_float2(lse.x, lse.y)), d1 = __ffma2_rn(s1, make_float2(x, x), make_float2(lse.z, lse.w));
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
        if (sm.lim[tid] < 0) x = make_float2(-INFINITY, 0.f);
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
  if (group == 4) {
    tc_fence_after();
    tmem_dealloc(tmem, 512u);
  }
}

}  // namespace specq
