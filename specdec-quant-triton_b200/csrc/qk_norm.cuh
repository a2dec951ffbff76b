// qk_norm.cuh -- RMS norm of every query and key head with its rotary turn, and the gradients.
//
// For a head x of D elements with weights w, a token at position p (R: the turn of rope.cuh):
//   r = (mean x^2 + eps)^(-1/2),  y = R(p) (x r w)
// and, from g = dL/dy, u = R(p)^T g and xh = x r:
//   dx = r (u w - xh mean(u w xh)),   dw = sum over tokens and heads of u xh
// All in fp32, one rounding at each output.  A sum of squares that overflows fp32 (elements from
// some 2^60 on) is made again of x 2^-70.
//
// Bound by HBM: forward reads and writes each element once, backward reads x and g and writes dx; the
// turned and normalised values never leave the registers, and r is made again in the backward pass
// instead of being kept (8 more bytes for each head against 3 shuffles).  A head is D / (2 V) lanes of one warp
// (V = 16 bytes of elements); each lane holds the two 16-byte pieces that the turn pairs, so the norm
// costs log2(lanes) shuffles and the turn none.  A forward thread takes kNormHeads heads of one token,
// whose loads are in flight together and share angles and weights; short calls take one head a thread.
// The backward kernel runs a fixed grid whose threads keep the sums for dw of their own elements in
// registers over all their heads, the next heads' pieces being copied meanwhile; a block adds its lanes' sums in a fixed order, a
// second small kernel adds the blocks': no atomics, the same bits each time.
//
// Measured (B200, 32 + 8 heads of 128, bf16): 8190 tokens forward 37.8 us, 4.5 TB/s: a thread's angles and weights in fp32 take half of
// its 128 registers and are live from before the reduction, though needed after it, so that 16 warps an SM have loads in flight (2, 1,
// 8 heads a thread: 42, 46, 46 us; blocks that stay and copy ahead: 47; rope.cuh moves the same bytes in 28.7).  4093 tokens forward and backward 54.4 us, of which backward some 30 (without the copies ahead 56, three stages 57,
// one head a thread 57).  One token: 2.2 us in a stream of launches.
#pragma once

#include "rope.cuh"

namespace specq {

struct QkNormParams {
  const void* x[2];      // q [T, H, D], k [T, H_KV, D], unit stride along D
  void* out[2];          // forward: y; backward: dx (null: not wanted)
  const void* g[2];      // backward: dL/dy
  const void* w[2];      // [D], of the rows' type or fp32 (null: ones)
  float* part[2];        // backward: the blocks' sums for dw, [blocks, D] (null: not wanted)
  const int32_t* pos;
  const float* table;    // [n_pos, rot]: cosines | sines
  const int32_t* plan;
  int* status;
  int64_t xt[2], xh[2], ot[2], oh[2], gt[2], gh[2];
  int heads[2];
  int blocks[2];         // backward: blocks for q, for k
  int T, D, rot, n_pos, w_f32;
  float eps, inv_d;
};

constexpr int kNormThreads = 128;
constexpr int kNormHeads = 4;
constexpr int kNormGradThreads = 256;
constexpr int kNormGradHeads = 2;
constexpr int kNormMaxD = 2048;
constexpr float kNormSmall = 8.470329472543003e-22f;   // 2^-70

// Sums of N values over the `lanes` lanes (a power of two) that share a head.
template <int N>
__device__ __forceinline__ void lanes_sum(float (&v)[N], int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
}

// Where the two pieces of lane `item` of a head stand, whether the turn pairs them, and where their
// angles begin in the table's row.
template <bool HALF, int V>
struct NormPieces {
  int a, b, angle;
  bool turned;
  __device__ __forceinline__ NormPieces(int item, int rot) {
    if constexpr (HALF) {
      turned = item * 2 * V < rot;
      a = turned ? item * V : item * 2 * V;        // past rot / 2V items of pairs come those of the tail
      b = turned ? (rot >> 1) + item * V : a + V;
    } else {
      turned = item * 2 * V < rot;
      a = item * 2 * V;
      b = a + V;
    }
    angle = item * V;
  }
};

// Turn two pieces (sgn -1: back).  Half layout: element i of a with element i of b; interleaved: neighbours.
template <bool HALF, int V>
__device__ __forceinline__ void turn_pieces(float (&a)[V], float (&b)[V], const float (&c)[V], const float (&s)[V], float sgn) {
  if constexpr (HALF) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float si = s[i] * sgn, x = a[i], y = b[i];
      a[i] = fmaf(x, c[i], -y * si);
      b[i] = fmaf(y, c[i], x * si);
    }
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const float s0 = s[i] * sgn, s1 = s[V / 2 + i] * sgn, c0 = c[i], c1 = c[V / 2 + i];
      const float x = a[2 * i], y = a[2 * i + 1], z = b[2 * i], w = b[2 * i + 1];
      a[2 * i] = fmaf(x, c0, -y * s0);
      a[2 * i + 1] = fmaf(y, c0, x * s0);
      b[2 * i] = fmaf(z, c1, -w * s1);
      b[2 * i + 1] = fmaf(w, c1, z * s1);
    }
  }
}

template <typename T, int V>
__device__ __forceinline__ void load_weights(const void* w, int w_f32, int at, float (&v)[V]) {
  if (w == nullptr) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = 1.f;
  } else if (w_f32) {
    load_f32_run<V>(static_cast<const float*>(w) + at, v);
  } else {
    Row16<T> r;
    r.load(static_cast<const T*>(w) + at);
    r.get(v);
  }
}

template <typename T>
__device__ __forceinline__ float weight_at(const void* w, int w_f32, int i) {
  return w == nullptr ? 1.f : w_f32 ? static_cast<const float*>(w)[i] : weight_to_f32<T>(static_cast<const T*>(w)[i]);
}

// r of N heads from their lanes' squares; `sq(h, scale)` is a lane's own sum of (x scale)^2 of head h.
template <int N, typename Sq>
__device__ __forceinline__ void inverse_rms(const QkNormParams& p, int lanes, float (&r)[N], Sq sq) {
#pragma unroll
  for (int h = 0; h < N; ++h) r[h] = sq(h, 1.f);
  lanes_sum<N>(r, lanes);
  uint32_t over = 0;                   // heads whose sum left fp32 (or is NaN, and stays so)
#pragma unroll
  for (int h = 0; h < N; ++h) {
    if (!(r[h] < 3e38f)) over |= 1u << h;
    r[h] = __frsqrt_rn(fmaf(r[h], p.inv_d, p.eps));
  }
  if (__any_sync(0xffffffffu, over != 0u)) {
    float s[N];
#pragma unroll
    for (int h = 0; h < N; ++h) s[h] = sq(h, kNormSmall);
    lanes_sum<N>(s, lanes);
#pragma unroll
    for (int h = 0; h < N; ++h)        // eps is nothing beside such squares
      if (over >> h & 1u) r[h] = kNormSmall * __frsqrt_rn(s[h] * p.inv_d);
  }
}

// Lane-groups in order: token, then groups of HP heads, first q's and then k's.
template <typename T, bool HALF, int HP>
__global__ void __launch_bounds__(kNormThreads) qk_norm_vec_kernel(const __grid_constant__ QkNormParams p, int lane_bits) {
  constexpr int V = Row16<T>::N;
  pdl_launch_dependents();
  pdl_wait();
  const int rows = rope_active_rows(p.plan, p.T, p.status);
  const int lanes = 1 << lane_bits;
  const int groups_q = (p.heads[0] + HP - 1) / HP, groups = groups_q + (p.heads[1] + HP - 1) / HP;
  const uint32_t id = blockIdx.x * kNormThreads + threadIdx.x;
  const uint32_t unit = id >> lane_bits;
  const int t = static_cast<int>(unit / static_cast<uint32_t>(groups));
  const int gi = static_cast<int>(unit - static_cast<uint32_t>(t) * groups);
  const int is_k = gi >= groups_q;
  const int h0 = (gi - (is_k ? groups_q : 0)) * HP;
  const int n = t < rows ? min(HP, p.heads[is_k] - h0) : 0;   // the others only take part in the shuffles
  const NormPieces<HALF, V> at(static_cast<int>(id) & (lanes - 1), p.rot);
  const T* x = static_cast<const T*>(p.x[is_k]) + t * p.xt[is_k] + h0 * p.xh[is_k];
  Row16<T> a[HP], b[HP];
#pragma unroll
  for (int h = 0; h < HP; ++h) {
    a[h].raw = b[h].raw = make_uint4(0u, 0u, 0u, 0u);
    if (h < n) {
      a[h].load(x + h * p.xh[is_k] + at.a);
      b[h].load(x + h * p.xh[is_k] + at.b);
    }
  }
  float c[V], s[V], wa[V], wb[V];
  if (at.turned && n > 0) {
    const float* row = rope_row(p.table, __ldg(p.pos + t), p.n_pos, p.rot, p.status);
    load_f32_run<V>(row + at.angle, c);
    load_f32_run<V>(row + (p.rot >> 1) + at.angle, s);
  }
  load_weights<T, V>(p.w[is_k], p.w_f32, at.a, wa);
  load_weights<T, V>(p.w[is_k], p.w_f32, at.b, wb);
  float r[HP];
  inverse_rms<HP>(p, lanes, r, [&](int h, float scale) {
    float av[V], bv[V], q = 0.f;
    a[h].get(av);
    b[h].get(bv);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float u = av[i] * scale, v = bv[i] * scale;
      q = fmaf(u, u, q);
      q = fmaf(v, v, q);
    }
    return q;
  });
  T* out = static_cast<T*>(p.out[is_k]) + t * p.ot[is_k] + h0 * p.oh[is_k];
#pragma unroll
  for (int h = 0; h < HP; ++h)
    if (h < n) {
      float av[V], bv[V];
      a[h].get(av);
      b[h].get(bv);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        av[i] = av[i] * r[h] * wa[i];
        bv[i] = bv[i] * r[h] * wb[i];
      }
      if (at.turned) turn_pieces<HALF, V>(av, bv, c, s, 1.f);
      a[h].set(av);
      b[h].set(bv);
      a[h].store(out + h * p.oh[is_k] + at.a);
      b[h].store(out + h * p.oh[is_k] + at.b);
    }
}

// Sum of a value over the warp.
__device__ __forceinline__ float warp_sum_f32(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Elements of pair i, or (i >= rot / 2) the single element of the tail at rot + i - rot / 2.
__device__ __forceinline__ void norm_pair(int i, int rot, bool half_layout, int& ia, int& ib) {
  const int half = rot >> 1;
  if (i >= half) ia = ib = rot + i - half;
  else if (half_layout) ia = i, ib = i + half;
  else ia = 2 * i, ib = 2 * i + 1;
}

// r of one head, by a warp.
template <typename T>
__device__ __forceinline__ float warp_inverse_rms(const QkNormParams& p, const T* x, int lane) {
  float q = 0.f;
  for (int i = lane; i < p.D; i += 32) {
    const float v = weight_to_f32<T>(x[i]);
    q = fmaf(v, v, q);
  }
  q = warp_sum_f32(q);
  float r = __frsqrt_rn(fmaf(q, p.inv_d, p.eps));
  if (!(q < 3e38f)) {
    q = 0.f;
    for (int i = lane; i < p.D; i += 32) {
      const float v = weight_to_f32<T>(x[i]) * kNormSmall;
      q = fmaf(v, v, q);
    }
    q = warp_sum_f32(q);
    r = kNormSmall * __frsqrt_rn(q * p.inv_d);
  }
  return r;
}

// Any head size, alignment and even rot: a warp a head.
template <typename T>
__global__ void __launch_bounds__(kNormThreads) qk_norm_any_kernel(const __grid_constant__ QkNormParams p, int half_layout) {
  pdl_launch_dependents();
  pdl_wait();
  const int rows = rope_active_rows(p.plan, p.T, p.status);
  const uint32_t unit = blockIdx.x * (kNormThreads / 32) + (threadIdx.x >> 5);
  const int lane = static_cast<int>(threadIdx.x & 31), all = p.heads[0] + p.heads[1];
  const int t = static_cast<int>(unit / static_cast<uint32_t>(all));
  int h = static_cast<int>(unit - static_cast<uint32_t>(t) * all);
  if (t >= rows) return;
  const int is_k = h >= p.heads[0];
  if (is_k) h -= p.heads[0];
  const T* x = static_cast<const T*>(p.x[is_k]) + t * p.xt[is_k] + h * p.xh[is_k];
  T* out = static_cast<T*>(p.out[is_k]) + t * p.ot[is_k] + h * p.oh[is_k];
  const float r = warp_inverse_rms<T>(p, x, lane);
  const float* row = rope_row(p.table, __ldg(p.pos + t), p.n_pos, p.rot, p.status);
  const int half = p.rot >> 1;
  for (int i = lane; i < p.D - half; i += 32) {   // in place: a lane reads its pair before it writes it
    int ia, ib;
    norm_pair(i, p.rot, half_layout != 0, ia, ib);
    const float u = weight_to_f32<T>(x[ia]) * r * weight_at<T>(p.w[is_k], p.w_f32, ia);
    if (i >= half) {
      out[ia] = f32_to_row<T>(u);
      continue;
    }
    const float v = weight_to_f32<T>(x[ib]) * r * weight_at<T>(p.w[is_k], p.w_f32, ib);
    const float c = __ldg(row + i), s = __ldg(row + half + i);
    out[ia] = f32_to_row<T>(fmaf(u, c, -v * s));
    out[ib] = f32_to_row<T>(fmaf(v, c, u * s));
  }
}

// ---- gradients ------------------------------------------------------------------------------------
// A thread's stages: the 16-byte pieces of the units to come, copied asynchronously; nobody else reads them.
constexpr int kNormStages = 2;
template <int THREADS, int PIECES>
struct NormStages {
  uint4 (*at)[PIECES][THREADS];
  __device__ __forceinline__ void fetch(int stage, int piece, const void* src) const {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(&at[stage][piece][threadIdx.x])), "l"(src) : "memory");
  }
  __device__ __forceinline__ uint4 get(int stage, int piece, bool there) const {
    return there ? at[stage][piece][threadIdx.x] : make_uint4(0u, 0u, 0u, 0u);
  }
};
__device__ __forceinline__ void norm_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void norm_arrived() { asm volatile("cp.async.wait_group %0;" ::"n"(kNormStages - 1) : "memory"); }

template <typename T, bool HALF>
__global__ void __launch_bounds__(kNormGradThreads, 2)
    qk_norm_grad_vec_kernel(const __grid_constant__ QkNormParams p, int lane_bits) {
  constexpr int V = Row16<T>::N, HP = kNormGradHeads;
  extern __shared__ uint4 ring[];      // [stages, 4 HP, threads]; at the end the warps' sums [warps, D]
  float* red = reinterpret_cast<float*>(ring);
  const NormStages<kNormGradThreads, 4 * HP> stages{reinterpret_cast<uint4 (*)[4 * HP][kNormGradThreads]>(ring)};
  pdl_launch_dependents();
  pdl_wait();
  const int rows = rope_active_rows(p.plan, p.T, p.status);
  const int lanes = 1 << lane_bits;
  const int is_k = static_cast<int>(blockIdx.x) >= p.blocks[0];
  const int block = static_cast<int>(blockIdx.x) - (is_k ? p.blocks[0] : 0);
  const int per_block = kNormGradThreads >> lane_bits;
  const int groups = (p.heads[is_k] + HP - 1) / HP;
  const int64_t units = static_cast<int64_t>(rows) * groups, step = static_cast<int64_t>(p.blocks[is_k]) * per_block;
  const int item = static_cast<int>(threadIdx.x) & (lanes - 1);
  const NormPieces<HALF, V> at(item, p.rot);
  const T* x0 = static_cast<const T*>(p.x[is_k]);
  const T* g0 = static_cast<const T*>(p.g[is_k]);
  T* d0 = static_cast<T*>(p.out[is_k]);
  float wa[V], wb[V], sa[V], sb[V];
  load_weights<T, V>(p.w[is_k], p.w_f32, at.a, wa);
  load_weights<T, V>(p.w[is_k], p.w_f32, at.b, wb);
#pragma unroll
  for (int i = 0; i < V; ++i) sa[i] = sb[i] = 0.f;
  const int mine = static_cast<int>(threadIdx.x) >> lane_bits;
  auto place = [&](int64_t u0, int& t, int& h0) {    // -> heads
    const int64_t unit = u0 + mine;
    t = static_cast<int>(unit / groups);
    h0 = static_cast<int>(unit - static_cast<int64_t>(t) * groups) * HP;
    return unit < units ? min(HP, p.heads[is_k] - h0) : 0;
  };
  auto fetch = [&](int stage, int64_t u0) {
    if (u0 < units) {
      int t, h0;
      const int n = place(u0, t, h0);
      const T* x = x0 + t * p.xt[is_k] + h0 * p.xh[is_k];
      const T* g = g0 + t * p.gt[is_k] + h0 * p.gh[is_k];
#pragma unroll
      for (int h = 0; h < HP; ++h)
        if (h < n) {
          stages.fetch(stage, 4 * h, x + h * p.xh[is_k] + at.a);
          stages.fetch(stage, 4 * h + 1, x + h * p.xh[is_k] + at.b);
          stages.fetch(stage, 4 * h + 2, g + h * p.gh[is_k] + at.a);
          stages.fetch(stage, 4 * h + 3, g + h * p.gh[is_k] + at.b);
        }
    }
    norm_commit();
  };
  // a block's lane groups take neighbouring units; all warps make the same number of turns
  const int64_t first = static_cast<int64_t>(block) * per_block;
#pragma unroll
  for (int i = 0; i < kNormStages - 1; ++i) fetch(i, first + i * step);
  int stage = 0;
  for (int64_t u0 = first; u0 < units; u0 += step) {
    fetch(stage == 0 ? kNormStages - 1 : stage - 1, u0 + (kNormStages - 1) * step);
    int t, h0;
    const int n = place(u0, t, h0);
    norm_arrived();
    Row16<T> xa[HP], xb[HP], ga[HP], gb[HP];
#pragma unroll
    for (int h = 0; h < HP; ++h) {
      xa[h].raw = stages.get(stage, 4 * h, h < n);
      xb[h].raw = stages.get(stage, 4 * h + 1, h < n);
      ga[h].raw = stages.get(stage, 4 * h + 2, h < n);
      gb[h].raw = stages.get(stage, 4 * h + 3, h < n);
    }
    stage = stage + 1 == kNormStages ? 0 : stage + 1;
    float c[V], s[V];
    if (at.turned && n > 0) {
      const float* row = rope_row(p.table, __ldg(p.pos + t), p.n_pos, p.rot, p.status);
      load_f32_run<V>(row + at.angle, c);
      load_f32_run<V>(row + (p.rot >> 1) + at.angle, s);
    }
    float r[HP];
    inverse_rms<HP>(p, lanes, r, [&](int h, float scale) {
      float av[V], bv[V], q = 0.f;
      xa[h].get(av);
      xb[h].get(bv);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float u = av[i] * scale, v = bv[i] * scale;
        q = fmaf(u, u, q);
        q = fmaf(v, v, q);
      }
      return q;
    });
    float ua[HP][V], ub[HP][V], dot[HP];
#pragma unroll
    for (int h = 0; h < HP; ++h) {
      float av[V], bv[V];
      ga[h].get(ua[h]);
      gb[h].get(ub[h]);
      if (at.turned && n > 0) turn_pieces<HALF, V>(ua[h], ub[h], c, s, -1.f);
      xa[h].get(av);
      xb[h].get(bv);
      dot[h] = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float ea = ua[h][i] * (av[i] * r[h]), eb = ub[h][i] * (bv[i] * r[h]);
        if (h < n) {
          sa[i] += ea;
          sb[i] += eb;
        }
        dot[h] = fmaf(ea, wa[i], dot[h]);
        dot[h] = fmaf(eb, wb[i], dot[h]);
      }
    }
    lanes_sum<HP>(dot, lanes);
    if (d0 != nullptr) {
      T* d = d0 + t * p.ot[is_k] + h0 * p.oh[is_k];
#pragma unroll
      for (int h = 0; h < HP; ++h)
        if (h < n) {
          const float mean = dot[h] * p.inv_d;
          float av[V], bv[V];
          xa[h].get(av);
          xb[h].get(bv);
#pragma unroll
          for (int i = 0; i < V; ++i) {
            av[i] = r[h] * fmaf(-(av[i] * r[h]), mean, ua[h][i] * wa[i]);
            bv[i] = r[h] * fmaf(-(bv[i] * r[h]), mean, ub[h][i] * wb[i]);
          }
          xa[h].set(av);
          xb[h].set(bv);
          xa[h].store(d + h * p.oh[is_k] + at.a);
          xb[h].store(d + h * p.oh[is_k] + at.b);
        }
    }
  }
  if (p.part[is_k] == nullptr) return;
  __syncthreads();                     // the stages are read
  // the warp's lanes of one item, then the warps
  for (int o = 16; o >= lanes; o >>= 1)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      sa[i] += __shfl_xor_sync(0xffffffffu, sa[i], o);
      sb[i] += __shfl_xor_sync(0xffffffffu, sb[i], o);
    }
  const int warp = static_cast<int>(threadIdx.x >> 5);
  if (static_cast<int>(threadIdx.x & 31) < lanes) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      red[warp * p.D + at.a + i] = sa[i];
      red[warp * p.D + at.b + i] = sb[i];
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.D; e += kNormGradThreads) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kNormGradThreads / 32; ++w) sum += red[w * p.D + e];
    p.part[is_k][static_cast<int64_t>(block) * p.D + e] = sum;
  }
}

// Any head size, alignment and even rot: a warp a head, its sums for dw in its own row of shared memory,
// whose elements belong to the lane that takes their pair.
template <typename T>
__global__ void __launch_bounds__(kNormThreads) qk_norm_grad_any_kernel(const __grid_constant__ QkNormParams p, int half_layout) {
  extern __shared__ float red[];       // [warps, D]
  pdl_launch_dependents();
  pdl_wait();
  constexpr int kWarps = kNormThreads / 32;
  const int rows = rope_active_rows(p.plan, p.T, p.status);
  const int lane = static_cast<int>(threadIdx.x & 31), warp = static_cast<int>(threadIdx.x >> 5);
  const int is_k = static_cast<int>(blockIdx.x) >= p.blocks[0];
  const int block = static_cast<int>(blockIdx.x) - (is_k ? p.blocks[0] : 0);
  const int heads = p.heads[is_k], half = p.rot >> 1;
  float* mine = red + warp * p.D;
  for (int e = threadIdx.x; e < kWarps * p.D; e += kNormThreads) red[e] = 0.f;
  __syncthreads();
  const int64_t units = static_cast<int64_t>(rows) * heads;
  for (int64_t unit = static_cast<int64_t>(block) * kWarps + warp; unit < units; unit += static_cast<int64_t>(p.blocks[is_k]) * kWarps) {
    const int t = static_cast<int>(unit / heads), h = static_cast<int>(unit - static_cast<int64_t>(t) * heads);
    const T* x = static_cast<const T*>(p.x[is_k]) + t * p.xt[is_k] + h * p.xh[is_k];
    const T* g = static_cast<const T*>(p.g[is_k]) + t * p.gt[is_k] + h * p.gh[is_k];
    const float* row = rope_row(p.table, __ldg(p.pos + t), p.n_pos, p.rot, p.status);
    const float r = warp_inverse_rms<T>(p, x, lane);
    auto back = [&](int i, int& ia, int& ib, float& ua, float& ub) {   // u of a pair (of the tail: ub = 0)
      norm_pair(i, p.rot, half_layout != 0, ia, ib);
      const float a = weight_to_f32<T>(g[ia]);
      if (i >= half) {
        ua = a;
        ub = 0.f;
        return;
      }
      const float b = weight_to_f32<T>(g[ib]), c = __ldg(row + i), s = __ldg(row + half + i);
      ua = fmaf(a, c, b * s);
      ub = fmaf(b, c, -a * s);
    };
    float dot = 0.f;
    for (int i = lane; i < p.D - half; i += 32) {
      int ia, ib;
      float ua, ub;
      back(i, ia, ib, ua, ub);
      const float ea = ua * (weight_to_f32<T>(x[ia]) * r);
      mine[ia] += ea;
      dot = fmaf(ea, weight_at<T>(p.w[is_k], p.w_f32, ia), dot);
      if (i < half) {
        const float eb = ub * (weight_to_f32<T>(x[ib]) * r);
        mine[ib] += eb;
        dot = fmaf(eb, weight_at<T>(p.w[is_k], p.w_f32, ib), dot);
      }
    }
    const float mean = warp_sum_f32(dot) * p.inv_d;
    if (p.out[is_k] == nullptr) continue;
    T* d = static_cast<T*>(p.out[is_k]) + t * p.ot[is_k] + h * p.oh[is_k];
    for (int i = lane; i < p.D - half; i += 32) {
      int ia, ib;
      float ua, ub;
      back(i, ia, ib, ua, ub);
      d[ia] = f32_to_row<T>(r * fmaf(-(weight_to_f32<T>(x[ia]) * r), mean, ua * weight_at<T>(p.w[is_k], p.w_f32, ia)));
      if (i < half)
        d[ib] = f32_to_row<T>(r * fmaf(-(weight_to_f32<T>(x[ib]) * r), mean, ub * weight_at<T>(p.w[is_k], p.w_f32, ib)));
    }
  }
  if (p.part[is_k] == nullptr) return;
  __syncthreads();
  for (int e = threadIdx.x; e < p.D; e += kNormThreads) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) sum += red[w * p.D + e];
    p.part[is_k][static_cast<int64_t>(block) * p.D + e] = sum;
  }
}

struct QkNormWeightGradParams {
  const float* part[2];  // [blocks, D]
  void* dw[2];           // [D], of the weights' type
  int blocks[2];
  int D, dtype;
};

// dw of 32 elements: 32 warps take the blocks' rows in turn, their sums are added in order, in 64 bits.
__global__ void __launch_bounds__(1024) qk_norm_weight_grad_kernel(const __grid_constant__ QkNormWeightGradParams p) {
  __shared__ double red[32][33];
  pdl_launch_dependents();
  pdl_wait();
  const int is_k = blockIdx.y, lane = static_cast<int>(threadIdx.x & 31), warp = static_cast<int>(threadIdx.x >> 5);
  const int e = blockIdx.x * 32 + lane;
  if (p.dw[is_k] == nullptr) return;
  double sum = 0.0;
  if (e < p.D)
    for (int b = warp; b < p.blocks[is_k]; b += 32) sum += p.part[is_k][static_cast<int64_t>(b) * p.D + e];
  red[warp][lane] = sum;
  __syncthreads();
  if (warp != 0 || e >= p.D) return;
  for (int w = 1; w < 32; ++w) sum += red[w][lane];
  const float v = static_cast<float>(sum);
  if (p.dtype == SPECQ_DTYPE_F16) static_cast<__half*>(p.dw[is_k])[e] = __float2half_rn(v);
  else if (p.dtype == SPECQ_DTYPE_BF16) static_cast<__nv_bfloat16*>(p.dw[is_k])[e] = __float2bfloat16_rn(v);
  else static_cast<float*>(p.dw[is_k])[e] = v;
}

// ---- host -------------------------------------------------------------------------------------------
// Lanes of a head as a power of two's exponent, or -1 where the 16-byte form does not fit.
template <typename T>
inline int norm_lane_bits(const QkNormParams& p) {
  constexpr int V = Row16<T>::N;
  const int es = static_cast<int>(sizeof(T));
  if (p.D % (2 * V) || p.rot % (2 * V) || !aligned(p.table, 16)) return -1;
  const int lanes = p.D / (2 * V);
  if (lanes > 32 || (lanes & (lanes - 1))) return -1;
  for (int i = 0; i < 2; ++i) {
    if (p.heads[i] == 0) continue;
    if (!aligned(p.x[i], 16) || !aligned(p.out[i], 16) || !aligned(p.g[i], 16) || !aligned(p.w[i], 16) || (p.xt[i] * es) % 16 ||
        (p.xh[i] * es) % 16 || (p.ot[i] * es) % 16 || (p.oh[i] * es) % 16 || (p.gt[i] * es) % 16 || (p.gh[i] * es) % 16)
      return -1;
  }
  return __builtin_ctz(static_cast<unsigned>(lanes));
}

inline int norm_check(const char* who, const QkNormParams& p, int dtype, int layout, bool grad) {
  if (p.T < 0 || p.heads[0] < 0 || p.heads[1] < 0 || p.D <= 0 || p.n_pos <= 0)
    return fail(SPECQ_ERR_INVALID_ARG, "%s: bad shape T=%d H=%d H_KV=%d D=%d n_pos=%d", who, p.T, p.heads[0], p.heads[1], p.D, p.n_pos);
  if (p.rot < 2 || p.rot % 2 || p.rot > p.D)
    return fail(SPECQ_ERR_INVALID_ARG, "%s: rot=%d must be even and in 2..D=%d", who, p.rot, p.D);
  if (p.D > kNormMaxD) return fail(SPECQ_ERR_UNSUPPORTED, "%s: head size %d > %d", who, p.D, kNormMaxD);
  if (layout < 0 || layout > 1) return fail(SPECQ_ERR_INVALID_ARG, "%s: layout %d", who, layout);
  if (dtype < 0 || dtype > 2) return fail(SPECQ_ERR_INVALID_ARG, "%s: dtype code %d", who, dtype);
  if (!(p.eps > 0.f) || !(p.eps < 3e38f)) return fail(SPECQ_ERR_INVALID_ARG, "%s: eps must be positive (in fp32) and finite", who);
  if (static_cast<int64_t>(p.heads[0]) + p.heads[1] > 1 << 20) return fail(SPECQ_ERR_UNSUPPORTED, "%s: %d + %d heads", who, p.heads[0], p.heads[1]);
  if (p.T > 0 && (p.pos == nullptr || p.table == nullptr)) return fail(SPECQ_ERR_INVALID_ARG, "%s: null pointer", who);
  for (int i = 0; i < 2 && p.T > 0; ++i)
    if (p.heads[i] > 0 && (p.x[i] == nullptr || (grad ? p.g[i] == nullptr : p.out[i] == nullptr)))
      return fail(SPECQ_ERR_INVALID_ARG, "%s: null pointer", who);
  return SPECQ_OK;
}

template <typename T>
inline int launch_qk_norm(const QkNormParams& all, bool half, int sm_count, cudaStream_t st) {
  const int bits = norm_lane_bits<T>(all);
  // Several heads a thread once one head a thread would fill the SMs' 2048 threads, as in rope.cuh.
  const int heads = all.heads[0] + all.heads[1];
  const bool many = bits >= 0 && ((static_cast<int64_t>(all.T) * heads) << bits) >= static_cast<int64_t>(sm_count) * 2048;
  const int hp = many ? kNormHeads : 1;
  const int64_t per_row = bits >= 0 ? static_cast<int64_t>(ceil_div(all.heads[0], hp) + ceil_div(all.heads[1], hp)) << bits
                                    : static_cast<int64_t>(heads) * 32;
  const int64_t step = std::max<int64_t>(1, 0x7FFFFF00ll / per_row);   // thread indices are 32-bit
  if (all.plan != nullptr && all.T > step) return fail(SPECQ_ERR_UNSUPPORTED, "qk_norm_rope: %d rows under a plan", all.T);
  for (int64_t t0 = 0; t0 < all.T; t0 += step) {
    QkNormParams p = all;
    p.T = static_cast<int>(std::min<int64_t>(step, all.T - t0));
    for (int i = 0; i < 2; ++i) {
      if (p.heads[i] == 0) continue;
      p.x[i] = static_cast<const T*>(all.x[i]) + t0 * all.xt[i];
      p.out[i] = static_cast<T*>(all.out[i]) + t0 * all.ot[i];
    }
    p.pos = all.pos + t0;
    const dim3 grid(static_cast<unsigned>((p.T * per_row + kNormThreads - 1) / kNormThreads)), block(kNormThreads);
    cudaError_t e;
    if (bits < 0) e = launch_plain(qk_norm_any_kernel<T>, grid, block, st, p, half ? 1 : 0);
    else if (many) e = half ? launch_plain(qk_norm_vec_kernel<T, true, kNormHeads>, grid, block, st, p, bits)
                            : launch_plain(qk_norm_vec_kernel<T, false, kNormHeads>, grid, block, st, p, bits);
    else e = half ? launch_plain(qk_norm_vec_kernel<T, true, 1>, grid, block, st, p, bits)
                  : launch_plain(qk_norm_vec_kernel<T, false, 1>, grid, block, st, p, bits);
    SPECQ_CUDA_TRY(e);
  }
  return SPECQ_OK;
}

// Blocks of the gradient kernel for q and for k: two an SM in all, shared as the heads are.
inline void norm_grad_blocks(int T, int H, int H_KV, int sm_count, int (&blocks)[2]) {
  const int heads = H + H_KV, all = 2 * sm_count;
  blocks[0] = blocks[1] = 0;
  if (T == 0 || heads == 0) return;
  blocks[0] = H == 0 ? 0 : H_KV == 0 ? all : std::min(all - 1, std::max(1, static_cast<int>(static_cast<int64_t>(all) * H / heads)));
  blocks[1] = H_KV == 0 ? 0 : all - blocks[0];
  const int h[2] = {H, H_KV};
  for (int i = 0; i < 2; ++i)   // no block without a head
    blocks[i] = static_cast<int>(std::min<int64_t>(blocks[i], static_cast<int64_t>(T) * h[i]));
}

template <typename T>
inline int launch_qk_norm_grad(QkNormParams p, bool half, cudaStream_t st) {
  const int bits = norm_lane_bits<T>(p);
  const dim3 grid(p.blocks[0] + p.blocks[1]);
  auto launch = [&](auto kern, int threads, int last) {
    const size_t smem = std::max<size_t>(static_cast<size_t>(threads / 32) * p.D * sizeof(float), bits < 0 ? 0 : static_cast<size_t>(kNormStages) * 4 * kNormGradHeads * kNormGradThreads * 16);
    cudaError_t e = ensure_dyn_smem(reinterpret_cast<const void*>(kern), static_cast<int>(smem));
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    LaunchAttrs at(1);
    at.apply(cfg);
    return cudaLaunchKernelEx(&cfg, kern, p, last);
  };
  if (bits < 0) SPECQ_CUDA_TRY(launch(qk_norm_grad_any_kernel<T>, kNormThreads, half ? 1 : 0));
  else if (half) SPECQ_CUDA_TRY(launch(qk_norm_grad_vec_kernel<T, true>, kNormGradThreads, bits));
  else SPECQ_CUDA_TRY(launch(qk_norm_grad_vec_kernel<T, false>, kNormGradThreads, bits));
  return SPECQ_OK;
}

inline int run_qk_norm_rope(const void* q, int64_t qt, int64_t qh, void* q_out, int64_t qot, int64_t qoh, const void* k, int64_t kt,
                            int64_t kh, void* k_out, int64_t kot, int64_t koh, int dtype, const void* qw, const void* kw,
                            int weight_f32, float eps, const int32_t* pos, const float* table, int n_pos, int T, int H, int H_KV,
                            int D, int rot, int layout, const int32_t* plan, void* stream) {
  QkNormParams p = {};
  p.x[0] = q; p.x[1] = k; p.out[0] = q_out; p.out[1] = k_out; p.w[0] = qw; p.w[1] = kw;
  p.xt[0] = qt; p.xh[0] = qh; p.ot[0] = qot; p.oh[0] = qoh; p.xt[1] = kt; p.xh[1] = kh; p.ot[1] = kot; p.oh[1] = koh;
  p.pos = pos; p.table = table; p.plan = plan;
  p.heads[0] = H; p.heads[1] = H_KV;
  p.T = T; p.D = D; p.rot = rot; p.n_pos = n_pos; p.w_f32 = weight_f32 != 0 || dtype == SPECQ_DTYPE_F32;
  p.eps = eps; p.inv_d = D > 0 ? 1.f / static_cast<float>(D) : 0.f;
  if (int rc = norm_check("qk_norm_rope", p, dtype, layout, false)) return rc;
  for (int i = 0; i < 2; ++i)
    if (p.x[i] == p.out[i] && p.x[i] != nullptr && (p.xt[i] != p.ot[i] || p.xh[i] != p.oh[i]))
      return fail(SPECQ_ERR_INVALID_ARG, "qk_norm_rope: in place, the strides of input and output must be the same");
  if (T == 0 || H + H_KV == 0) return SPECQ_OK;
  DeviceState* dev = nullptr;
  if (int rc = get_device_state(&dev)) return rc;
  p.status = dev->status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool half = layout == SPECQ_ROPE_HALF;
  if (dtype == SPECQ_DTYPE_F16) return launch_qk_norm<__half>(p, half, dev->sm_count, st);
  if (dtype == SPECQ_DTYPE_F32) return launch_qk_norm<float>(p, half, dev->sm_count, st);
  return launch_qk_norm<__nv_bfloat16>(p, half, dev->sm_count, st);
}

inline int run_qk_norm_rope_grad_workspace(int T, int H, int H_KV, int D, int64_t* bytes) {
  if (bytes == nullptr || T < 0 || H < 0 || H_KV < 0 || D <= 0)
    return fail(SPECQ_ERR_INVALID_ARG, "qk_norm_rope_grad_workspace: T=%d H=%d H_KV=%d D=%d", T, H, H_KV, D);
  DeviceState* dev = nullptr;
  if (int rc = get_device_state(&dev)) return rc;
  int blocks[2];
  norm_grad_blocks(T, H, H_KV, dev->sm_count, blocks);
  *bytes = static_cast<int64_t>(blocks[0] + blocks[1]) * D * static_cast<int64_t>(sizeof(float));
  return SPECQ_OK;
}

inline int run_qk_norm_rope_grad(const void* q, int64_t qt, int64_t qh, const void* gq, int64_t gqt, int64_t gqh, void* dq,
                                 int64_t dqt, int64_t dqh, const void* k, int64_t kt, int64_t kh, const void* gk, int64_t gkt,
                                 int64_t gkh, void* dk, int64_t dkt, int64_t dkh, int dtype, const void* qw, const void* kw, void* dqw,
                                 void* dkw, int weight_f32, float eps, const int32_t* pos, const float* table, int n_pos, int T, int H,
                                 int H_KV, int D, int rot, int layout, const int32_t* plan, void* workspace, int64_t workspace_bytes,
                                 void* stream) {
  const char* who = "qk_norm_rope_grad";
  QkNormParams p = {};
  p.x[0] = q; p.x[1] = k; p.out[0] = dq; p.out[1] = dk; p.g[0] = gq; p.g[1] = gk; p.w[0] = qw; p.w[1] = kw;
  p.xt[0] = qt; p.xh[0] = qh; p.ot[0] = dqt; p.oh[0] = dqh; p.gt[0] = gqt; p.gh[0] = gqh;
  p.xt[1] = kt; p.xh[1] = kh; p.ot[1] = dkt; p.oh[1] = dkh; p.gt[1] = gkt; p.gh[1] = gkh;
  p.pos = pos; p.table = table; p.plan = plan;
  p.heads[0] = H; p.heads[1] = H_KV;
  p.T = T; p.D = D; p.rot = rot; p.n_pos = n_pos; p.w_f32 = weight_f32 != 0 || dtype == SPECQ_DTYPE_F32;
  p.eps = eps; p.inv_d = D > 0 ? 1.f / static_cast<float>(D) : 0.f;
  if (int rc = norm_check(who, p, dtype, layout, true)) return rc;
  if ((dqw != nullptr && qw == nullptr) || (dkw != nullptr && kw == nullptr))
    return fail(SPECQ_ERR_INVALID_ARG, "%s: a gradient of weights that are not there", who);
  DeviceState* dev = nullptr;
  if (int rc = get_device_state(&dev)) return rc;
  p.status = dev->status;
  norm_grad_blocks(T, H, H_KV, dev->sm_count, p.blocks);
  QkNormWeightGradParams s = {};
  s.dw[0] = dqw; s.dw[1] = dkw;
  s.D = D;
  s.dtype = p.w_f32 ? SPECQ_DTYPE_F32 : dtype;
  const int64_t need = static_cast<int64_t>(p.blocks[0] + p.blocks[1]) * D * static_cast<int64_t>(sizeof(float));
  const bool weights = dqw != nullptr || dkw != nullptr;
  if (weights && need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 16)))
    return fail(SPECQ_ERR_INVALID_ARG, "%s: a workspace of %lld bytes is needed", who, static_cast<long long>(need));
  float* ws = static_cast<float*>(workspace);
  for (int i = 0; i < 2; ++i) {
    s.blocks[i] = p.blocks[i];
    if (s.dw[i] != nullptr) s.part[i] = p.part[i] = i == 0 ? ws : ws + static_cast<int64_t>(p.blocks[0]) * D;
    if (p.out[i] == nullptr && s.dw[i] == nullptr) p.heads[i] = 0;   // nothing is wanted of these
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool half = layout == SPECQ_ROPE_HALF;
  for (int i = 0; i < 2; ++i)
    if (p.heads[i] == 0) p.blocks[i] = 0;
  if (p.blocks[0] + p.blocks[1] > 0) {
    int rc;
    if (dtype == SPECQ_DTYPE_F16) rc = launch_qk_norm_grad<__half>(p, half, st);
    else if (dtype == SPECQ_DTYPE_F32) rc = launch_qk_norm_grad<float>(p, half, st);
    else rc = launch_qk_norm_grad<__nv_bfloat16>(p, half, st);
    if (rc) return rc;
  }
  if (weights) SPECQ_CUDA_TRY(launch_plain(qk_norm_weight_grad_kernel, dim3(ceil_div(D, 32), 2), dim3(1024), st, s));
  return SPECQ_OK;
}

}  // namespace specq
