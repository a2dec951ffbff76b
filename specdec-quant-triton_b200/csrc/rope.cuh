// rope.cuh -- rotary positions of the heads of packed token rows.
//
// The first `rot` elements of a head are rot/2 pairs, and pair i of a token at position p is
// turned by the angle whose cosine and sine stand in row p of the table:
//   (a, b) -> (a cos - b sin, b cos + a sin)
// Pairs are (i, i + rot/2) in the half layout and (2i, 2i + 1) in the interleaved one.  The
// inverse turns by the negative angle; a rotation is orthogonal, so that is also its gradient.
// The products are made in fp32 whatever the rows' type and rounded once.
//
// Bound by HBM (3 flops an element): each element is read and written once.  A thread takes 16
// bytes (half layout: the 16 bytes of both partners) of kRopeHeads heads of one token, so the
// pair's cosines and sines are loaded once for all of them and the heads' loads are in flight
// together; short calls, whose time is the latency of one load, take one head a thread.
// Measured (B200): 8190 x 40 x 128 bf16, interleaved, first 64 turned: 28.7 us, 5.9 TB/s of the 6.44
// that a copy reaches; one token of 40 heads: 1.5 us in a stream of launches.
#pragma once

#include <cuda_bf16.h>

#include "rowops.cuh"
#include "sm100.cuh"
#include "specq_host.cuh"

namespace specq {

struct RopeParams {
  const void* x;        // [T, H, D], unit stride along D
  void* out;            // [T, H, D] (may be x itself)
  const int32_t* pos;   // [T]
  const float* table;   // [n_pos, rot]: cosines | sines
  const int32_t* plan;  // plan[0] = active T
  int* status;
  int64_t xt, xh, ot, oh;
  int T, H, D, rot, n_pos;
  int copy_tail;        // elements past rot are copied (out is not x)
  float sgn;            // -1: the inverse rotation
};

template <typename T>
__device__ __forceinline__ T f32_to_row(float v);
template <>
__device__ __forceinline__ __half f32_to_row<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ float f32_to_row<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 f32_to_row<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// 16 bytes of a row as fp32, and back.
template <typename T>
struct Row16 {
  static constexpr int N = 16 / sizeof(T);
  uint4 raw;
  __device__ __forceinline__ void load(const T* p) { raw = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<uint4*>(p) = raw; }
  __device__ __forceinline__ void get(float (&v)[N]) const {
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = weight_to_f32<T>(e[i]);
  }
  __device__ __forceinline__ void set(const float (&v)[N]) {
    T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] = f32_to_row<T>(v[i]);
  }
};

template <int N>
__device__ __forceinline__ void load_f32_run(const float* p, float (&v)[N]) {
  static_assert(N == 2 || N % 4 == 0, "run of 2 or of fours");
  if constexpr (N == 2) {
    const float2 u = __ldg(reinterpret_cast<const float2*>(p));
    v[0] = u.x; v[1] = u.y;
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 u = __ldg(reinterpret_cast<const float4*>(p + i));
      v[i] = u.x; v[i + 1] = u.y; v[i + 2] = u.z; v[i + 3] = u.w;
    }
  }
}

// One 16-byte item of `n` heads (x, out: the first head's row; row = the token's table row).
// Item i < half_items rotates elements; the later ones are 16-byte pieces of the tail.
template <typename T, bool HALF, int HP>
__device__ __forceinline__ void rope_item(const T* x, int64_t xh, T* out, int64_t oh, const float* row, int rot,
                                          float sgn, int item, int n) {
  constexpr int V = Row16<T>::N;
  const int half = rot >> 1;
  if (item * (HALF ? 2 : 1) * V >= rot) {   // past the rotated part: a copy
    const int o = rot + (item - rot / (HALF ? 2 * V : V)) * V;
    Row16<T> a[HP];
#pragma unroll
    for (int h = 0; h < HP; ++h)
      if (h < n) a[h].load(x + h * xh + o);
#pragma unroll
    for (int h = 0; h < HP; ++h)
      if (h < n) a[h].store(out + h * oh + o);
    return;
  }
  if constexpr (HALF) {
    const int o = item * V;
    Row16<T> a[HP], b[HP];
#pragma unroll
    for (int h = 0; h < HP; ++h)
      if (h < n) {
        a[h].load(x + h * xh + o);
        b[h].load(x + h * xh + half + o);
      }
    float c[V], s[V];
    load_f32_run<V>(row + o, c);
    load_f32_run<V>(row + half + o, s);
#pragma unroll
    for (int h = 0; h < HP; ++h)
      if (h < n) {
        float av[V], bv[V], y[V], z[V];
        a[h].get(av);
        b[h].get(bv);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float si = s[i] * sgn;
          y[i] = fmaf(av[i], c[i], -bv[i] * si);
          z[i] = fmaf(bv[i], c[i], av[i] * si);
        }
        a[h].set(y);
        b[h].set(z);
        a[h].store(out + h * oh + o);
        b[h].store(out + h * oh + half + o);
      }
  } else {
    const int o = item * V;
    Row16<T> a[HP];
#pragma unroll
    for (int h = 0; h < HP; ++h)
      if (h < n) a[h].load(x + h * xh + o);
    float c[V / 2], s[V / 2];
    load_f32_run<V / 2>(row + o / 2, c);
    load_f32_run<V / 2>(row + half + o / 2, s);
#pragma unroll
    for (int h = 0; h < HP; ++h)
      if (h < n) {
        float v[V], y[V];
        a[h].get(v);
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
          const float si = s[i] * sgn;
          y[2 * i] = fmaf(v[2 * i], c[i], -v[2 * i + 1] * si);
          y[2 * i + 1] = fmaf(v[2 * i + 1], c[i], v[2 * i] * si);
        }
        a[h].set(y);
        a[h].store(out + h * oh + o);
      }
  }
}

// 16-byte items of a head: both partners (half layout) or one run of pairs, then the tail.
template <typename T>
__host__ __device__ inline int rope_items(int D, int rot, bool half, bool tail) {
  const int V = 16 / static_cast<int>(sizeof(T));
  return rot / (half ? 2 * V : V) + (tail ? (D - rot) / V : 0);
}

// The token's table row; a position outside the table is clamped into it and reported.
__device__ __forceinline__ const float* rope_row(const float* table, int pos, int n_pos, int rot, int* status) {
  if (pos < 0 || pos >= n_pos) {
    report_status(status, SPECQ_STATUS_PLAN_CLAMPED);
    pos = min(max(pos, 0), n_pos - 1);
  }
  return table + static_cast<int64_t>(pos) * rot;
}

__device__ __forceinline__ int rope_active_rows(const int32_t* plan, int T, int* status) {
  if (plan == nullptr) return T;
  const int m = __ldg(plan);
  if ((m < 0 || m > T) && blockIdx.x == 0 && threadIdx.x == 0) report_status(status, SPECQ_STATUS_PLAN_CLAMPED);
  return min(max(m, 0), T);
}

constexpr int kRopeThreads = 128;
constexpr int kRopeHeads = 4;

template <typename T, bool HALF, int HP>
__global__ void __launch_bounds__(kRopeThreads) rope_vec_kernel(const __grid_constant__ RopeParams p, int items, int groups) {
  pdl_launch_dependents();
  pdl_wait();
  const int rows = rope_active_rows(p.plan, p.T, p.status);
  const uint32_t id = blockIdx.x * kRopeThreads + threadIdx.x;
  const uint32_t th = id / static_cast<uint32_t>(items);
  const int item = static_cast<int>(id - th * items);
  const int t = static_cast<int>(th / static_cast<uint32_t>(groups));
  const int h0 = static_cast<int>(th - static_cast<uint32_t>(t) * groups) * HP;
  if (t >= rows) return;
  const float* row = rope_row(p.table, __ldg(p.pos + t), p.n_pos, p.rot, p.status);
  rope_item<T, HALF, HP>(static_cast<const T*>(p.x) + t * p.xt + h0 * p.xh, p.xh,
                         static_cast<T*>(p.out) + t * p.ot + h0 * p.oh, p.oh, row, p.rot, p.sgn, item,
                         min(HP, p.H - h0));
}

// Any alignment, any even rot: one pair, or one element of the tail, a thread.
template <typename T>
__global__ void __launch_bounds__(kRopeThreads) rope_any_kernel(const __grid_constant__ RopeParams p, int half_layout, int items) {
  pdl_launch_dependents();
  pdl_wait();
  const int rows = rope_active_rows(p.plan, p.T, p.status);
  const uint32_t id = blockIdx.x * kRopeThreads + threadIdx.x;
  const uint32_t th = id / static_cast<uint32_t>(items);
  const int item = static_cast<int>(id - th * items);
  const int t = static_cast<int>(th / static_cast<uint32_t>(p.H));
  const int h = static_cast<int>(th - static_cast<uint32_t>(t) * p.H);
  if (t >= rows) return;
  const T* x = static_cast<const T*>(p.x) + t * p.xt + h * p.xh;
  T* out = static_cast<T*>(p.out) + t * p.ot + h * p.oh;
  const int half = p.rot >> 1;
  if (item >= half) {
    const int o = p.rot + item - half;
    out[o] = x[o];
    return;
  }
  const float* row = rope_row(p.table, __ldg(p.pos + t), p.n_pos, p.rot, p.status);
  const int ia = half_layout ? item : 2 * item, ib = half_layout ? item + half : 2 * item + 1;
  const float a = weight_to_f32<T>(x[ia]), b = weight_to_f32<T>(x[ib]);
  const float c = __ldg(row + item), s = __ldg(row + half + item) * p.sgn;
  out[ia] = f32_to_row<T>(fmaf(a, c, -b * s));
  out[ib] = f32_to_row<T>(fmaf(b, c, a * s));
}

template <typename T>
inline int launch_rope(const RopeParams& all, bool half, int sm_count, cudaStream_t st) {
  constexpr int V = Row16<T>::N;
  const int es = static_cast<int>(sizeof(T));
  const bool vec = all.rot % (half ? 2 * V : V) == 0 && all.D % V == 0 && aligned(all.x, 16) && aligned(all.out, 16) &&
                   aligned(all.table, 16) && (all.xt * es) % 16 == 0 && (all.xh * es) % 16 == 0 &&
                   (all.ot * es) % 16 == 0 && (all.oh * es) % 16 == 0;
  const int items = vec ? rope_items<T>(all.D, all.rot, half, all.copy_tail)
                        : all.rot / 2 + (all.copy_tail ? all.D - all.rot : 0);
  // Several heads a thread once one head a thread would fill the SMs' 2048 threads: below that
  // the extra threads hide latency, above it the table's loads are what they save.
  const bool many = vec && static_cast<int64_t>(all.T) * all.H * items >= static_cast<int64_t>(sm_count) * 2048;
  const int hp = many ? kRopeHeads : 1;
  const int groups = vec ? ceil_div(all.H, hp) : all.H;
  // thread indices are 32-bit: token rows go in launches of fewer than 2^31 threads
  const int64_t per_row = static_cast<int64_t>(groups) * items;
  const int64_t step = std::max<int64_t>(1, 0x7FFFFF00ll / per_row);
  if (per_row > 0x7FFFFF00ll) return fail(SPECQ_ERR_UNSUPPORTED, "rope: a row of %d heads is too wide", all.H);
  if (all.plan != nullptr && all.T > step) return fail(SPECQ_ERR_UNSUPPORTED, "rope: %d rows under a plan", all.T);
  for (int64_t t0 = 0; t0 < all.T; t0 += step) {
    RopeParams p = all;
    p.T = static_cast<int>(std::min<int64_t>(step, all.T - t0));
    p.x = static_cast<const T*>(all.x) + t0 * all.xt;
    p.out = static_cast<T*>(all.out) + t0 * all.ot;
    p.pos = all.pos + t0;
    const unsigned grid = static_cast<unsigned>((p.T * per_row + kRopeThreads - 1) / kRopeThreads);
    cudaError_t e;
    if (!vec) {
      e = launch_plain(rope_any_kernel<T>, dim3(grid), dim3(kRopeThreads), st, p, half ? 1 : 0, items);
    } else if (many) {
      e = half ? launch_plain(rope_vec_kernel<T, true, kRopeHeads>, dim3(grid), dim3(kRopeThreads), st, p, items, groups)
               : launch_plain(rope_vec_kernel<T, false, kRopeHeads>, dim3(grid), dim3(kRopeThreads), st, p, items, groups);
    } else {
      e = half ? launch_plain(rope_vec_kernel<T, true, 1>, dim3(grid), dim3(kRopeThreads), st, p, items, groups)
               : launch_plain(rope_vec_kernel<T, false, 1>, dim3(grid), dim3(kRopeThreads), st, p, items, groups);
    }
    SPECQ_CUDA_TRY(e);
  }
  return SPECQ_OK;
}

inline int run_rope(const void* x, int64_t xt, int64_t xh, void* out, int64_t ot, int64_t oh, int dtype,
                    const int32_t* pos, const float* table, int n_pos, int T, int H, int D, int rot, int layout,
                    int inverse, const int32_t* plan, void* stream) {
  if (T < 0 || H < 0 || D <= 0 || n_pos <= 0)
    return fail(SPECQ_ERR_INVALID_ARG, "rope: bad shape T=%d H=%d D=%d rot=%d n_pos=%d", T, H, D, rot, n_pos);
  if (rot < 2 || rot % 2 || rot > D)
    return fail(SPECQ_ERR_INVALID_ARG, "rope: rot=%d must be even and in 2..D=%d", rot, D);
  if (layout < 0 || layout > 1) return fail(SPECQ_ERR_INVALID_ARG, "rope: layout %d", layout);
  if (dtype < 0 || dtype > 2) return fail(SPECQ_ERR_INVALID_ARG, "rope: dtype code %d", dtype);
  if (T == 0 || H == 0) return SPECQ_OK;
  if (x == nullptr || out == nullptr || pos == nullptr || table == nullptr)
    return fail(SPECQ_ERR_INVALID_ARG, "rope: null pointer");
  if (x == out && (xt != ot || xh != oh))
    return fail(SPECQ_ERR_INVALID_ARG, "rope: in place, the strides of x and out must be the same");
  DeviceState* dev = nullptr;
  if (int rc = get_device_state(&dev)) return rc;
  RopeParams p = {};
  p.x = x; p.out = out; p.pos = pos; p.table = table; p.plan = plan; p.status = dev->status;
  p.xt = xt; p.xh = xh; p.ot = ot; p.oh = oh;
  p.T = T; p.H = H; p.D = D; p.rot = rot; p.n_pos = n_pos;
  p.copy_tail = x != out;
  p.sgn = inverse ? -1.f : 1.f;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool half = layout == 0;
  if (dtype == 0) return launch_rope<__half>(p, half, dev->sm_count, st);
  if (dtype == 1) return launch_rope<float>(p, half, dev->sm_count, st);
  return launch_rope<__nv_bfloat16>(p, half, dev->sm_count, st);
}

}  // namespace specq
