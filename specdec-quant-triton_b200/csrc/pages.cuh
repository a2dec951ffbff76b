// pages.cuh -- the page pool of a paged KV cache on the device: release, reserve, fork.
//
// State: ref [P] (how many rows hold a page; 0 = free), tbl [S, C] (the rows' pages, -1 past
// the held ones, which every call keeps so) and held [S] (pages a row holds).  There is no free
// list: a page is free when its count is 0, and pages are handed out lowest index first, row by
// row, so the result of every call is a function of the state alone (the atomics below add
// integers, whose order does not matter, or claim nothing).
//
// release  every held page of a dropped row counts one less; the row empties.
// reserve  row r is extended to ceil(want[r] / page) pages.  All rows or, when the free pages
//          do not suffice, none; short = the missing pages (0: granted).
// fork     row r with parent[r] = p (p >= 0, p != r) becomes a copy of row p's first
//          length[p] tokens: p's full pages are shared (count + 1), a part-filled last page is
//          copied (its filled slots and its scales, in every layer) to the lowest free page,
//          and what r held before is released.  All rows at once: parents are read as they
//          were, so beams can be permuted.  Again all or none, short = the missing pages.
//
// The work is a few kilobytes of integers, so what counts is the number of dependent steps.
// reserve is one CTA that reads ref in runs of 8 counts a thread (8,192 pages a step, one
// block scan each, the free ones listed in shared memory and placed by a warp a row) and stops when
// it has found enough.  fork is that CTA and beside it others that snapshot the parents' rows, and
// then a grid that copies the pages (bound by HBM) and rewrites the rows.  The kernels follow one
// another by programmatic launch.  Measured, release + reserve + fork: 8 rows, one layer 9.2 us; 192 rows in
// beams of 4, 16 layers of pages of 16 x 8 x 128: 24.5 us, of which the copies' bytes need 8.8.
#pragma once

#include "sm100.cuh"
#include "specq_host.cuh"

namespace specq {

constexpr int kPoolThreads = 1024;
constexpr int kPoolRun = 8;        // counts a thread reads in one step
constexpr int kPoolMaxRows = 8192; // rows of a table: their prefix sums stand in shared memory

struct PagePool {
  int32_t* ref;
  int32_t* tbl;
  int32_t* held;
  int* status;
  int64_t ld;      // row stride of tbl
  int P, S, C;
};

// held[r], within the table's columns
__device__ __forceinline__ int pool_held(const PagePool& p, int r) { return min(max(p.held[r], 0), p.C); }

__global__ void __launch_bounds__(128) pages_release_kernel(const __grid_constant__ PagePool p, const uint8_t* drop) {
  pdl_launch_dependents();
  pdl_wait();
  const int r = blockIdx.x;
  if (drop[r] == 0) return;
  const int n = pool_held(p, r);
  int32_t* row = p.tbl + r * p.ld;
  for (int c = threadIdx.x; c < n; c += 128) {
    const int pg = row[c];
    if (pg < 0 || pg >= p.P) report_status(p.status, SPECQ_STATUS_BAD_INDEX);
    else if (atomicSub(p.ref + pg, 1) <= 0) {   // a count that was already 0 stays 0
      atomicAdd(p.ref + pg, 1);
      report_status(p.status, SPECQ_STATUS_BAD_INDEX);
    }
    row[c] = -1;
  }
  __syncthreads();       // every thread has read held[r]
  if (threadIdx.x == 0) p.held[r] = 0;
}

// Exclusive sum over the block's threads; total in *sum.  red: 33 ints.
__device__ __forceinline__ int block_exclusive(int v, int* red, int* sum) {
  const int lane = static_cast<int>(threadIdx.x & 31), warp = static_cast<int>(threadIdx.x >> 5);
  int inc = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += up;
  }
  if (lane == 31) red[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    const int w = red[lane];
    int winc = w;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, winc, d);
      if (lane >= d) winc += up;
    }
    red[lane] = winc - w;
    if (lane == 31) red[32] = winc;
  }
  __syncthreads();
  const int out = red[warp] + inc - v;
  *sum = red[32];
  __syncthreads();       // red may be used again
  return out;
}

// Row r needs `need` pages: fills start[S + 1] with the exclusive sums and returns the total.
template <typename Need>
__device__ __forceinline__ int pool_starts(int S, int* start, int* red, Need need) {
  int total = 0;
  for (int r0 = 0; r0 < S; r0 += kPoolThreads) {
    const int r = r0 + static_cast<int>(threadIdx.x);
    const int n = r < S ? need(r) : 0;
    int sum;
    const int at = block_exclusive(n, red, &sum);
    if (r < S) start[r] = total + at;
    total += sum;
  }
  if (threadIdx.x == 0) start[S] = total;
  __syncthreads();
  return total;
}

// Finds the `total` lowest free pages, if there are as many, and hands them over a step at a time:
// use(rank, list, count) by every thread, list[i] being the free page of rank `rank` + i.  Returns
// how many pages are missing.  A call whose first step finds enough looks at the counts once;
// others count first, since nothing may be handed over when pages are missing.
template <typename Use>
__device__ __forceinline__ int pool_take(const PagePool& p, int total, int* red, int* list, Use use) {
  const int step = kPoolThreads * kPoolRun;
  for (int pass = 0; pass < 2; ++pass) {
    int found = 0;
    for (int p0 = 0; p0 < p.P && found < total; p0 += step) {
      const int first = p0 + static_cast<int>(threadIdx.x) * kPoolRun;
      uint32_t free_bits = 0;
      if (first + kPoolRun <= p.P) {
#pragma unroll
        for (int i = 0; i < kPoolRun; i += 4) {
          const int4 u = *reinterpret_cast<const int4*>(p.ref + first + i);
          free_bits |= (u.x == 0 ? 1u : 0u) << i | (u.y == 0 ? 2u : 0u) << i | (u.z == 0 ? 4u : 0u) << i | (u.w == 0 ? 8u : 0u) << i;
        }
      } else {
        for (int i = 0; i < kPoolRun; ++i)
          if (first + i < p.P && p.ref[first + i] == 0) free_bits |= 1u << i;
      }
      int sum;
      int at = block_exclusive(__popc(free_bits), red, &sum);
      if (pass == 1 || (p0 == 0 && sum >= total)) {
        for (; free_bits != 0u; free_bits &= free_bits - 1u) list[at++] = first + __ffs(free_bits) - 1;
        __syncthreads();
        use(found, list, min(sum, total - found));
        __syncthreads();
        if (pass == 0) return 0;
      }
      found += sum;
    }
    if (found < total) return total - found;
  }
  return 0;
}

inline size_t pool_smem(int S) { return (static_cast<size_t>(kPoolThreads) * kPoolRun + S + 1) * sizeof(int); }

__global__ void __launch_bounds__(kPoolThreads) pages_reserve_kernel(const __grid_constant__ PagePool p, const int32_t* want,
                                                                     int page, int32_t* short_out) {
  pdl_launch_dependents();
  pdl_wait();
  extern __shared__ int list[];           // [kPoolThreads * kPoolRun], then start [S + 1]
  int* start = list + kPoolThreads * kPoolRun;
  __shared__ int red[33];
  const int warp = static_cast<int>(threadIdx.x >> 5), lane = static_cast<int>(threadIdx.x & 31);
  auto need = [&](int r) {
    const int w = want[r];
    int cols = w <= 0 ? 0 : (w - 1) / page + 1;
    if (cols > p.C) {
      report_status(p.status, SPECQ_STATUS_PLAN_CLAMPED);
      cols = p.C;
    }
    return max(cols - pool_held(p, r), 0);
  };
  const int total = pool_starts(p.S, start, red, need);
  int missing = 0;
  if (total > 0) {
    missing = pool_take(p, total, red, list, [&](int rank, const int* pages, int count) {
      for (int r = warp; r < p.S; r += kPoolThreads / 32) {
        const int lo = max(start[r], rank), hi = min(start[r + 1], rank + count);
        if (lo >= hi) continue;
        int32_t* cell = p.tbl + r * p.ld + pool_held(p, r) - start[r];
        for (int k = lo + lane; k < hi; k += 32) {
          const int pg = pages[k - rank];
          cell[k] = pg;
          p.ref[pg] = 1;
        }
      }
    });
  }
  __syncthreads();                        // the pages are placed by the old held
  if (missing == 0)
    for (int r = threadIdx.x; r < p.S; r += kPoolThreads) {
      const int n = start[r + 1] - start[r];
      if (n > 0) p.held[r] = pool_held(p, r) + n;
    }
  if (threadIdx.x == 0) *short_out = missing;
}

struct PageForkParams {
  PagePool pool;
  const int32_t* parent;   // [S]
  const int32_t* length;   // [S]
  int32_t* snap;           // [S, C] scratch: the rows to be
  int32_t* fresh;          // [S] scratch: the copied page, -1 without one, -2 where the row stays
  int32_t* from;           // [S] scratch: the page it is copied from
  int32_t* short_out;
  uint8_t* kc;
  uint8_t* vc;
  float* ks;
  float* vs;
  int64_t kv_sl, kv_sp, kv_so, kv_sh, s_sl, s_sp, s_sh;
  int page, h_kv, D, L;
  int planes;              // blocks that copy a row's page
  int dense;               // a page's tokens and heads are contiguous
};

// Row r, which is forked with `to` as its copied page, takes its share of the parent's pages:
// snapshot (before any row is rewritten) and rewrite, each by `step` threads from `c0`.  The rows'
// additions to the counts and subtractions from them may come in any order: a page is subtracted
// at most once for each row that held it.
__device__ __forceinline__ void fork_snapshot(const PageForkParams& f, int r, int c0, int step) {
  const int p = f.parent[r], full = f.length[p] / f.page;
  const int32_t* from_row = f.pool.tbl + p * f.pool.ld;
  int32_t* snap = f.snap + static_cast<int64_t>(r) * f.pool.C;
  for (int c = c0; c < full; c += step) snap[c] = from_row[c];
}
__device__ __forceinline__ void fork_rewrite(const PageForkParams& f, int r, int to, int c0, int step) {
  const int full = f.length[f.parent[r]] / f.page, had = pool_held(f.pool, r);
  int32_t* row = f.pool.tbl + r * f.pool.ld;
  const int32_t* snap = f.snap + static_cast<int64_t>(r) * f.pool.C;
  for (int c = c0; c < max(had, full + (to >= 0 ? 1 : 0)); c += step) {
    if (c < had) {
      const int pg = row[c];
      if (pg < 0 || pg >= f.pool.P) report_status(f.pool.status, SPECQ_STATUS_BAD_INDEX);
      else if (atomicSub(f.pool.ref + pg, 1) <= 0) {
        atomicAdd(f.pool.ref + pg, 1);
        report_status(f.pool.status, SPECQ_STATUS_BAD_INDEX);
      }
    }
    int now = c == full && to >= 0 ? to : -1;
    if (c < full) {
      now = snap[c];
      if (now < 0 || now >= f.pool.P) report_status(f.pool.status, SPECQ_STATUS_BAD_INDEX);
      else atomicAdd(f.pool.ref + now, 1);
    }
    row[c] = now;
  }
}
__device__ __forceinline__ int fork_held(const PageForkParams& f, int r, int to) {
  return f.length[f.parent[r]] / f.page + (to >= 0 ? 1 : 0);
}

// parent of row r, or -1 where the row stays as it is
__device__ __forceinline__ int fork_parent(const PageForkParams& f, int r, bool tell) {
  const int p = f.parent[r];
  if (p < 0 || p == r) return -1;
  bool bad = p >= f.pool.S;
  if (!bad) {
    const int n = f.length[p];
    bad = n < 0 || (n > 0 && (n - 1) / f.page + 1 > pool_held(f.pool, p));
  }
  if (bad && tell) report_status(f.pool.status, SPECQ_STATUS_BAD_INDEX);
  return bad ? -1 : p;
}

__global__ void __launch_bounds__(kPoolThreads) pages_fork_plan_kernel(const __grid_constant__ PageForkParams f) {
  pdl_launch_dependents();
  pdl_wait();
  const int warp = static_cast<int>(threadIdx.x >> 5), lane = static_cast<int>(threadIdx.x & 31);
  if (blockIdx.x > 0) {                   // beside the planning CTA: the parents' rows
    const int r = (static_cast<int>(blockIdx.x) - 1) * (kPoolThreads / 32) + warp;
    if (r < f.pool.S && fork_parent(f, r, false) >= 0) fork_snapshot(f, r, lane, 32);
    return;
  }
  extern __shared__ int list[];
  int* start = list + kPoolThreads * kPoolRun;
  __shared__ int red[33];
  auto need = [&](int r) {
    const int p = fork_parent(f, r, true);
    f.fresh[r] = p < 0 ? -2 : -1;
    if (p < 0) return 0;
    const int n = f.length[p], full = n / f.page;
    if (n == full * f.page) return 0;
    f.from[r] = f.pool.tbl[p * f.pool.ld + full];
    return 1;
  };
  const int total = pool_starts(f.pool.S, start, red, need);
  int missing = 0;
  if (total > 0) {
    missing = pool_take(f.pool, total, red, list, [&](int rank, const int* pages, int count) {
      for (int r = threadIdx.x; r < f.pool.S; r += kPoolThreads) {
        const int k = start[r];
        if (start[r + 1] > k && k >= rank && k < rank + count) {
          f.fresh[r] = pages[k - rank];
          f.pool.ref[pages[k - rank]] = 1;
        }
      }
    });
  }
  if (missing > 0)
    for (int r = threadIdx.x; r < f.pool.S; r += kPoolThreads) f.fresh[r] = -2;
  if (threadIdx.x == 0) *f.short_out = missing;
}

constexpr int kForkThreads = 256;

// Block (row, y) copies the row's page in the (layer, K|V) pairs y, y + planes, ...; the blocks of
// y = planes rewrite the rows.
__global__ void __launch_bounds__(kForkThreads) pages_fork_copy_kernel(const __grid_constant__ PageForkParams f) {
  pdl_launch_dependents();
  pdl_wait();
  const int r = blockIdx.x;
  const int to = f.fresh[r];
  if (to == -2) return;
  if (blockIdx.y == static_cast<unsigned>(f.planes)) {
    fork_rewrite(f, r, to, threadIdx.x, kForkThreads);
    __syncthreads();       // every thread has read held[r]
    if (threadIdx.x == 0) f.pool.held[r] = fork_held(f, r, to);
    return;
  }
  if (to < 0) return;
  const int n = f.length[f.parent[r]];
  const int rest = n - n / f.page * f.page;
  const int from = f.from[r];
  if (from < 0 || from >= f.pool.P) {
    if (threadIdx.x == 0) report_status(f.pool.status, SPECQ_STATUS_BAD_INDEX);
    return;
  }
  // all pairs' 16-byte pieces as one run, several loads in flight
  const unsigned chunks = f.D >> 4, per_slot = f.h_kv * chunks, items = rest * per_slot;
  const unsigned pairs = (2 * f.L - blockIdx.y + f.planes - 1) / f.planes;
  constexpr int U = 8;
  for (unsigned i0 = threadIdx.x; i0 < items * pairs; i0 += U * kForkThreads) {
    uint4 w[U];
    uint8_t* at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const unsigned i = i0 + u * kForkThreads;
      at[u] = nullptr;
      if (i < items * pairs) {
        const unsigned pair = i / items, in = i - pair * items;
        const unsigned y = blockIdx.y + pair * f.planes;
        int64_t off;
        if (f.dense) {
          off = static_cast<int64_t>(in) * 16;
        } else {
          const unsigned slot = in / per_slot, rest_in = in - slot * per_slot, h = rest_in / chunks;
          off = slot * f.kv_so + h * f.kv_sh + (rest_in - h * chunks) * 16;
        }
        uint8_t* base = ((y & 1) ? f.vc : f.kc) + (y >> 1) * f.kv_sl + off;
        at[u] = base + to * f.kv_sp;
        w[u] = *reinterpret_cast<const uint4*>(base + from * f.kv_sp);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (at[u] != nullptr) *reinterpret_cast<uint4*>(at[u]) = w[u];
  }
  for (unsigned i = threadIdx.x; i < pairs * f.h_kv; i += kForkThreads) {
    const unsigned pair = i / f.h_kv, h = i - pair * f.h_kv, y = blockIdx.y + pair * f.planes;
    float* scale = ((y & 1) ? f.vs : f.ks) + (y >> 1) * f.s_sl + h * f.s_sh;
    scale[to * f.s_sp] = scale[from * f.s_sp];
  }
}

inline int make_pool(const char* who, PagePool* p, int32_t* ref, int P, int32_t* tbl, int64_t ld, int32_t* held,
                     int S, int C) {
  if (P < 0 || S < 0 || C < 0 || ld < C) return fail(SPECQ_ERR_INVALID_ARG, "%s: bad sizes P=%d S=%d C=%d", who, P, S, C);
  if (S > kPoolMaxRows) return fail(SPECQ_ERR_UNSUPPORTED, "%s: %d rows > %d", who, S, kPoolMaxRows);
  if (S > 0 && (ref == nullptr || tbl == nullptr || held == nullptr))
    return fail(SPECQ_ERR_INVALID_ARG, "%s: null pointer", who);
  if (!aligned(ref, 16)) return fail(SPECQ_ERR_UNSUPPORTED, "%s: the page counts must be 16-byte aligned", who);
  p->ref = ref; p->tbl = tbl; p->held = held; p->ld = ld;
  p->P = P; p->S = S; p->C = C;
  return SPECQ_OK;
}

inline int pool_device(PagePool* p) {
  DeviceState* dev = nullptr;
  if (int rc = get_device_state(&dev)) return rc;
  p->status = dev->status;
  return SPECQ_OK;
}

inline cudaError_t launch_pool(void (*kern)(PagePool, const int32_t*, int, int32_t*), const PagePool& p, const int32_t* want,
                               int page, int32_t* short_out, cudaStream_t st) {
  const cudaError_t e = ensure_dyn_smem(reinterpret_cast<const void*>(kern), static_cast<int>(pool_smem(p.S)));
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(1);
  cfg.blockDim = dim3(kPoolThreads);
  cfg.dynamicSmemBytes = pool_smem(p.S);
  cfg.stream = st;
  LaunchAttrs at(1);
  at.apply(cfg);
  return cudaLaunchKernelEx(&cfg, kern, p, want, page, short_out);
}

inline int run_pages_release(int32_t* ref, int P, int32_t* tbl, int64_t ld, int32_t* held, int S, int C,
                             const uint8_t* drop, void* stream) {
  PagePool p = {};
  if (int rc = make_pool("pages_release", &p, ref, P, tbl, ld, held, S, C)) return rc;
  if (S == 0) return SPECQ_OK;
  if (drop == nullptr) return fail(SPECQ_ERR_INVALID_ARG, "pages_release: null pointer");
  if (int rc = pool_device(&p)) return rc;
  SPECQ_CUDA_TRY(launch_plain(pages_release_kernel, dim3(S), dim3(128), static_cast<cudaStream_t>(stream), p, drop));
  return SPECQ_OK;
}

inline int run_pages_reserve(int32_t* ref, int P, int32_t* tbl, int64_t ld, int32_t* held, int S, int C,
                             const int32_t* want, int page, int32_t* short_out, void* stream) {
  PagePool p = {};
  if (page <= 0) return fail(SPECQ_ERR_INVALID_ARG, "pages_reserve: page %d", page);
  if (int rc = make_pool("pages_reserve", &p, ref, P, tbl, ld, held, S, C)) return rc;
  if (short_out == nullptr || (S > 0 && want == nullptr)) return fail(SPECQ_ERR_INVALID_ARG, "pages_reserve: null pointer");
  if (int rc = pool_device(&p)) return rc;
  SPECQ_CUDA_TRY(launch_pool(pages_reserve_kernel, p, want, page, short_out, static_cast<cudaStream_t>(stream)));
  return SPECQ_OK;
}

inline int run_pages_fork(void* kc, void* vc, int64_t kv_sl, int64_t kv_sp, int64_t kv_so, int64_t kv_sh, int L,
                          float* ks, float* vs, int64_t s_sl, int64_t s_sp, int64_t s_sh, int32_t* ref, int P,
                          int32_t* tbl, int64_t ld, int32_t* held, int S, int C, const int32_t* parent,
                          const int32_t* length, int32_t* scratch, int32_t* short_out, int H_KV, int D, int page,
                          void* stream) {
  PageForkParams f = {};
  if (page <= 0 || L < 0 || L > 32767 || H_KV <= 0 || D <= 0)
    return fail(SPECQ_ERR_INVALID_ARG, "pages_fork: page=%d layers=%d H_KV=%d D=%d", page, L, H_KV, D);
  if (D % 16) return fail(SPECQ_ERR_UNSUPPORTED, "pages_fork: head_dim %d must be a multiple of 16", D);
  if (int rc = make_pool("pages_fork", &f.pool, ref, P, tbl, ld, held, S, C)) return rc;
  if (short_out == nullptr || (S > 0 && (parent == nullptr || length == nullptr || scratch == nullptr)) ||
      (L > 0 && S > 0 && (kc == nullptr || vc == nullptr || ks == nullptr || vs == nullptr)))
    return fail(SPECQ_ERR_INVALID_ARG, "pages_fork: null pointer");
  if (!aligned(kc, 16) || !aligned(vc, 16) || kv_sl % 16 || kv_sp % 16 || kv_so % 16 || kv_sh % 16)
    return fail(SPECQ_ERR_UNSUPPORTED, "pages_fork: cache rows must be 16-byte aligned");
  if (int rc = pool_device(&f.pool)) return rc;
  f.parent = parent; f.length = length; f.short_out = short_out;
  f.fresh = scratch; f.from = scratch + S; f.snap = scratch + 2 * static_cast<int64_t>(S);
  f.kc = static_cast<uint8_t*>(kc); f.vc = static_cast<uint8_t*>(vc); f.ks = ks; f.vs = vs;
  f.kv_sl = kv_sl; f.kv_sp = kv_sp; f.kv_so = kv_so; f.kv_sh = kv_sh; f.s_sl = s_sl; f.s_sp = s_sp; f.s_sh = s_sh;
  f.page = page; f.h_kv = H_KV; f.D = D; f.L = L;
  f.dense = kv_sh == D && kv_so == static_cast<int64_t>(H_KV) * D;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  SPECQ_CUDA_TRY(ensure_dyn_smem(reinterpret_cast<const void*>(pages_fork_plan_kernel), static_cast<int>(pool_smem(S))));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(1 + ceil_div(S, kPoolThreads / 32));
  cfg.blockDim = dim3(kPoolThreads);
  cfg.dynamicSmemBytes = pool_smem(S);
  cfg.stream = st;
  LaunchAttrs at(1);
  at.apply(cfg);
  // enough blocks for eight an SM; each then copies several layers' pages with its loads in flight
  DeviceState* dev = nullptr;
  if (int rc = get_device_state(&dev)) return rc;
  f.planes = S > 0 ? std::min(2 * L, std::max(1, ceil_div(8 * dev->sm_count, S))) : 0;
  SPECQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, pages_fork_plan_kernel, f));
  if (S > 0) SPECQ_CUDA_TRY(launch_plain(pages_fork_copy_kernel, dim3(S, f.planes + 1), dim3(kForkThreads), st, f));
  return SPECQ_OK;
}

}  // namespace specq
