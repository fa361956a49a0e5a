// hcg_norm.hip -- layer norm by rows and its gradient (include/hcg_lm.h).
//
//   mean = sum x / D, var = sum (x - mean)^2 / D, r = 1 / sqrt(var + eps),
//   y = (x - mean) r w + b
// and, with xh = (x - mean) r and g = dy w,
//   dx = r (g - sum g / D - xh sum(g xh) / D), dw = sum_t dy xh, db = sum_t dy.
//
// Both are bound by HBM: a row is read once (the gradient reads two) and held in
// registers, so the variance is the sum of squares about the mean, without the
// cancellation of E[x^2] - mean^2 and without a second read.  A row takes as
// few lanes as hold it with 16 bytes each.  8192 x 4096 bf16: forward 24.4 us
// (5.5 TB/s), gradient 43.7 + 4.7 (4.2 TB/s); the sums' divisions are true
// ones, so that a row of equal values gives exactly 0.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "hcg_vec.h"

namespace {

using hcg::ElemOf;
using hcg::kVec;
using hcg::raw4;

struct NormArgs {
  const void* x;
  const void* weight;
  const void* bias;
  void* y;
  float* mean;
  float* rstd;
  int64_t ldx, ldy, rows;
  int width;
  float eps;
};

// Sum over the LANES lanes of a row that share a wave, the same value in each.
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int m = (LANES < 64 ? LANES : 64) / 2; m >= 1; m >>= 1) v += __shfl_xor(v, m);
  return v;
}
// Sum over the LANES lanes of a row (a part of a wave, or whole waves).  `slot`:
// LDS words of the row group, not in use by a wave still behind the last barrier.
template <int LANES>
__device__ __forceinline__ float row_sum(float v, float* slot, int tir) {
  v = lanes_sum<LANES>(v);
  if constexpr (LANES > 64) {
    if (tir % 64 == 0) slot[tir / 64] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < LANES / 64; ++i) v += slot[i];
  }
  return v;
}

template <int LANES>
constexpr int norm_threads() {
  return LANES > 256 ? LANES : 256;
}

// One row by LANES lanes, held in registers as NV vectors per lane between the
// two passes of the variance.
template <class T, class P, int LANES, int NV>
__global__ __launch_bounds__(norm_threads<LANES>()) void norm_kernel(NormArgs g) {
  constexpr int E = kVec<T>, kRowsPerWg = norm_threads<LANES>() / LANES;
  constexpr int kSlots = LANES > 64 ? LANES / 64 : 1;
  __shared__ float slots[2][kRowsPerWg * kSlots];
  const int group = threadIdx.x / LANES, tir = threadIdx.x % LANES;
  const int64_t row = hcg::workgroup() * kRowsPerWg + group;
  const bool live = row < g.rows;
  const T* x = static_cast<const T*>(g.x) + (live ? row : 0) * g.ldx;
  const int first = tir * E;
  raw4 raw[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = first + i * LANES * E;
    raw[i] = c < g.width ? hcg::load_raw(x + c, g.width - c) : raw4{0, 0, 0, 0};
  }
  float v[NV][E];
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    hcg::unpack<T>(raw[i], v[i]);
#pragma unroll
    for (int e = 0; e < E; ++e) sum += v[i][e];
  }
  const float count = (float)g.width;
  const float mean = row_sum<LANES>(sum, slots[0] + group * kSlots, tir) / count;
  float sq = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int left = g.width - (first + i * LANES * E);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      v[i][e] -= mean;
      if (e < left) sq += v[i][e] * v[i][e];
    }
  }
  const float var = row_sum<LANES>(sq, slots[1] + group * kSlots, tir) / count;
  const float rstd = 1.f / sqrtf(var + g.eps);
  if (!live) return;
  if (tir == 0) {
    if (g.mean) g.mean[row] = mean;
    if (g.rstd) g.rstd[row] = rstd;
  }
  T* y = static_cast<T*>(g.y) + row * g.ldy;
  const P* w = static_cast<const P*>(g.weight);
  const P* b = static_cast<const P*>(g.bias);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = first + i * LANES * E;
    if (c < g.width) {
      float o[E], wf[E], bf[E];
#pragma unroll
      for (int e = 0; e < E; ++e) wf[e] = 1.f, bf[e] = 0.f;
      if (w) hcg::load_floats<P, E>(w + c, g.width - c, wf);
      if (b) hcg::load_floats<P, E>(b + c, g.width - c, bf);
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = v[i][e] * rstd * wf[e] + bf[e];
      hcg::store_raw(y + c, hcg::pack<T>(o), g.width - c);
    }
  }
}

// Rows too wide for registers (more than 4096 vectors): three passes over the
// row (the second and third from the L2), 1024 threads.
template <class T, class P>
__global__ __launch_bounds__(1024) void norm_wide_kernel(NormArgs g) {
  constexpr int E = kVec<T>;
  __shared__ float slots[2][16];
  const int64_t row = hcg::workgroup();
  if (row >= g.rows) return;
  const T* x = static_cast<const T*>(g.x) + row * g.ldx;
  float sum = 0.f;
  for (int64_t c = (int64_t)threadIdx.x * E; c < g.width; c += 1024 * E) {
    float f[E];
    hcg::unpack<T>(hcg::load_raw(x + c, (int)(g.width - c)), f);
#pragma unroll
    for (int e = 0; e < E; ++e) sum += f[e];
  }
  const float count = (float)g.width;
  const float mean = row_sum<1024>(sum, slots[0], threadIdx.x) / count;
  float sq = 0.f;
  for (int64_t c = (int64_t)threadIdx.x * E; c < g.width; c += 1024 * E) {
    float f[E];
    hcg::unpack<T>(hcg::load_raw(x + c, (int)(g.width - c)), f);
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (c + e < g.width) sq += (f[e] - mean) * (f[e] - mean);
  }
  const float rstd = 1.f / sqrtf(row_sum<1024>(sq, slots[1], threadIdx.x) / count + g.eps);
  if (threadIdx.x == 0) {
    if (g.mean) g.mean[row] = mean;
    if (g.rstd) g.rstd[row] = rstd;
  }
  T* y = static_cast<T*>(g.y) + row * g.ldy;
  const P* w = static_cast<const P*>(g.weight);
  const P* b = static_cast<const P*>(g.bias);
  for (int64_t c = (int64_t)threadIdx.x * E; c < g.width; c += 1024 * E) {
    float f[E], wf[E], bf[E];
    const int left = (int)(g.width - c);
    hcg::unpack<T>(hcg::load_raw(x + c, left), f);
#pragma unroll
    for (int e = 0; e < E; ++e) wf[e] = 1.f, bf[e] = 0.f;
    if (w) hcg::load_floats<P, E>(w + c, left, wf);
    if (b) hcg::load_floats<P, E>(b + c, left, bf);
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = (f[e] - mean) * rstd * wf[e] + bf[e];
    hcg::store_raw(y + c, hcg::pack<T>(f), left);
  }
}

// ---------------------------------------------------------------------------
// Gradient
// ---------------------------------------------------------------------------

struct NormGradArgs {
  const void* dy;
  const void* x;
  const float* mean;
  const float* rstd;
  const void* weight;
  void* dx;
  float* part;  // [gridDim.x][2][width]: each workgroup's sums of dy xh and dy
  int64_t lddy, ldx, lddx, rows;
  int width;
  bool stream;  // dx past the caches: non-temporal stores
};

// 256 workgroups (one per CU; 512 or 1024 write more parts and were no faster).
// GROUPS row groups of LANES lanes; group q of workgroup b takes rows
// b * GROUPS + q, + gridDim.x * GROUPS, ... and keeps its columns' sums of
// dy xh and dy in registers; the groups' sums meet in LDS once, at the end.
// LEAN (1024 threads, so 128 registers, with 16 16-bit columns each): the
// weights come from the L2 for every row and no loads run ahead; held, they
// spill 65 registers.
template <class T, class P, int LANES, int NV, int GROUPS, bool LEAN = false>
__global__ __launch_bounds__(LANES * GROUPS) void norm_grad_kernel(NormGradArgs g) {
  constexpr int E = kVec<T>, kWaves = LANES / 64;
  __shared__ float slots[2][kWaves > 1 ? GROUPS * kWaves * 2 : 1];
  // The column sums of groups that share a wave meet by exchanges, the waves'
  // in LDS.
  constexpr int kShare = LANES < 64 ? 64 / LANES : 1, kMeet = GROUPS / kShare;
  __shared__ float meet[kMeet > 1 ? kMeet * LANES * E : 1];
  const int group = threadIdx.x / LANES, tir = threadIdx.x % LANES;
  const T* px = static_cast<const T*>(g.x);
  const T* pdy = static_cast<const T*>(g.dy);
  const P* w = static_cast<const P*>(g.weight);
  const int first = tir * E;
  const float count = (float)g.width;

  float wf[LEAN ? 1 : NV][E], dw[NV][E], db[NV][E];
  auto load_weight = [&](int i, float(&f)[E]) {
    const int c = first + i * LANES * E;
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = 1.f;
    if (w && c < g.width) hcg::load_floats<P, E>(w + c, g.width - c, f);
  };
#pragma unroll
  for (int i = 0; i < NV; ++i) {
#pragma unroll
    for (int e = 0; e < E; ++e) dw[i][e] = 0.f, db[i][e] = 0.f;
    if constexpr (!LEAN) load_weight(i, wf[i]);
  }

  const int64_t step = (int64_t)gridDim.x * GROUPS;
  const int64_t first_row = (int64_t)blockIdx.x * GROUPS + group;
  // Loads run kAhead rows ahead of the work (two where a lane has one vector of
  // a row: 64 KB in flight per CU).
  constexpr int kAhead = LEAN ? 0 : NV == 1 ? 2 : 1, kSlots = kAhead > 0 ? kAhead : 1;
  raw4 rx[kSlots][NV], rdy[kSlots][NV];
  float rmean[kSlots], rrstd[kSlots];
  auto load = [&](auto slot, int64_t row) {
    constexpr int S = decltype(slot)::value;
    const bool live = row < g.rows;
    rmean[S] = live ? g.mean[row] : 0.f;
    rrstd[S] = live ? g.rstd[row] : 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = first + i * LANES * E;
      const bool in = live && c < g.width;
      rx[S][i] = in ? hcg::load_raw(px + row * g.ldx + c, g.width - c) : raw4{0, 0, 0, 0};
      rdy[S][i] = in ? hcg::load_raw(pdy + row * g.lddy + c, g.width - c) : raw4{0, 0, 0, 0};
    }
  };
  int parity = 0;
  auto turn = [&](auto slot, int64_t row) {
    constexpr int S = decltype(slot)::value;
    if constexpr (kAhead == 0) load(slot, row);
    const float mean = rmean[S], rstd = rrstd[S];
    float xh[NV][E], dy[NV][E];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      hcg::unpack<T>(rx[S][i], xh[i]);
      hcg::unpack<T>(rdy[S][i], dy[i]);
    }
    if constexpr (kAhead > 0) load(slot, row + kAhead * step);
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float (&wi)[E] = wf[LEAN ? 0 : i];
      if constexpr (LEAN) load_weight(i, wi);
      // Past the row's end dy is 0 and x must be the mean: -mean * rstd may
      // overflow where no column's (x - mean) * rstd does.
      const int left = g.width - (first + i * LANES * E);
      if (left < E) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (e >= left) xh[i][e] = mean;
      }
#pragma unroll
      for (int e = 0; e < E; ++e) {
        xh[i][e] = (xh[i][e] - mean) * rstd;
        dw[i][e] += dy[i][e] * xh[i][e];
        db[i][e] += dy[i][e];
        dy[i][e] *= wi[e];
        s1 += dy[i][e];
        s2 += dy[i][e] * xh[i][e];
      }
    }
    s1 = lanes_sum<LANES>(s1);
    s2 = lanes_sum<LANES>(s2);
    if constexpr (kWaves > 1) {
      float* slot_sums = slots[parity] + group * kWaves * 2;
      if (tir % 64 == 0) slot_sums[tir / 64 * 2] = s1, slot_sums[tir / 64 * 2 + 1] = s2;
      __syncthreads();
      s1 = s2 = 0.f;
#pragma unroll
      for (int i = 0; i < kWaves; ++i) s1 += slot_sums[i * 2], s2 += slot_sums[i * 2 + 1];
      parity ^= 1;
    }
    if (row < g.rows) {
      s1 /= count;
      s2 /= count;
      T* dx = static_cast<T*>(g.dx) + row * g.lddx;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = first + i * LANES * E;
        if (c < g.width) {
          float o[E];
#pragma unroll
          for (int e = 0; e < E; ++e) o[e] = rstd * (dy[i][e] - s1 - xh[i][e] * s2);
          if (g.stream)
            hcg::store_raw<true>(dx + c, hcg::pack<T>(o), g.width - c);
          else
            hcg::store_raw(dx + c, hcg::pack<T>(o), g.width - c);
        }
      }
    }
  };
  typedef std::integral_constant<int, 0> Slot0;
  typedef std::integral_constant<int, kSlots - 1> Slot1;
  if constexpr (kAhead > 0) load(Slot0{}, first_row);
  if constexpr (kAhead > 1) load(Slot1{}, first_row + step);
  // (Every group runs as many turns as the workgroup's first: barriers.)
  for (int64_t row0 = (int64_t)blockIdx.x * GROUPS; row0 < g.rows; row0 += step) {
    turn(Slot0{}, row0 + group);
    if constexpr (kSlots > 1) {
      row0 += step;
      if (row0 < g.rows) turn(Slot1{}, row0 + group);
    }
  }

  if (g.part == nullptr) return;
  float* part = g.part + (int64_t)blockIdx.x * 2 * g.width;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float (&v)[E] = which ? db[i] : dw[i];
#pragma unroll
      for (int m = LANES; m < 64; m <<= 1)
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] += __shfl_xor(v[e], m);
      if constexpr (kMeet > 1) {
        __syncthreads();
        if (group > 0 && group % kShare == 0) {
#pragma unroll
          for (int e = 0; e < E; ++e) meet[(group / kShare * E + e) * LANES + tir] = v[e];
        }
        __syncthreads();
        if (group == 0) {
#pragma unroll
          for (int q = 1; q < kMeet; ++q)
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] += meet[(q * E + e) * LANES + tir];
        }
      }
      const int c = first + i * LANES * E;
      if (group == 0) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (c + e < g.width) part[(int64_t)which * g.width + c + e] = v[e];
      }
    }
  }
}

// Rows too wide for registers: a workgroup per row for dx (three passes); the
// column sums follow by norm_columns_kernel.
template <class T, class P>
__global__ __launch_bounds__(1024) void norm_grad_wide_kernel(NormGradArgs g) {
  constexpr int E = kVec<T>;
  __shared__ float slots[2][16];
  const int64_t row = hcg::workgroup();
  if (row >= g.rows) return;
  const T* x = static_cast<const T*>(g.x) + row * g.ldx;
  const T* dy = static_cast<const T*>(g.dy) + row * g.lddy;
  T* dx = static_cast<T*>(g.dx) + row * g.lddx;
  const P* w = static_cast<const P*>(g.weight);
  const float mean = g.mean[row], rstd = g.rstd[row], count = (float)g.width;
  float s1 = 0.f, s2 = 0.f;
  for (int pass = 0; pass < 2; ++pass) {
    for (int64_t c = (int64_t)threadIdx.x * E; c < g.width; c += 1024 * E) {
      const int left = (int)(g.width - c);
      float xf[E], df[E], wf[E];
      hcg::unpack<T>(hcg::load_raw(x + c, left), xf);
      hcg::unpack<T>(hcg::load_raw(dy + c, left), df);
#pragma unroll
      for (int e = 0; e < E; ++e) wf[e] = 1.f;
      if (w) hcg::load_floats<P, E>(w + c, left, wf);
      if (pass == 0) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          s1 += df[e] * wf[e];
          if (e < left) s2 += df[e] * wf[e] * ((xf[e] - mean) * rstd);  // (past the row's end: 0 * -mean * rstd)
        }
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) df[e] = rstd * (df[e] * wf[e] - s1 - (xf[e] - mean) * rstd * s2);
        hcg::store_raw(dx + c, hcg::pack<T>(df), left);
      }
    }
    if (pass == 0) {
      s1 = row_sum<1024>(s1, slots[0], threadIdx.x) / count;
      s2 = row_sum<1024>(s2, slots[1], threadIdx.x) / count;
    }
  }
}

// The wide rows' column sums: workgroup (b, q) sums 256 columns over the rows
// q, q + gridDim.y, ...
template <class T>
__global__ __launch_bounds__(256) void norm_columns_kernel(NormGradArgs g) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= g.width) return;
  float dw = 0.f, db = 0.f;
  for (int64_t row = blockIdx.y; row < g.rows; row += gridDim.y) {
    const float dy = (float)static_cast<const T*>(g.dy)[row * g.lddy + c];
    const float x = (float)static_cast<const T*>(g.x)[row * g.ldx + c];
    dw += dy * ((x - g.mean[row]) * g.rstd[row]);
    db += dy;
  }
  float* part = g.part + (int64_t)blockIdx.y * 2 * g.width;
  part[c] = dw;
  part[g.width + c] = db;
}

// dw and db from the workgroups' sums (8 MB from the L2 at a width of 4096: 4.7
// us, 3.9 at 1027): 64 columns by 16 waves, wave q adding
// the parts q, q + 16, ..., the waves' sums added in order.
template <class P>
__global__ __launch_bounds__(1024) void norm_reduce_kernel(const float* part, int parts, int width, P* dweight,
                                                           P* dbias) {
  __shared__ float meet[16][64];
  P* out = blockIdx.y ? dbias : dweight;
  if (out == nullptr) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = (int64_t)blockIdx.x * 64 + lane;
  float sum = 0.f;
  if (c < width) {
    const float* p = part + (int64_t)blockIdx.y * width + c;
#pragma unroll 16
    for (int q = wave; q < parts; q += 16) sum += p[(int64_t)q * 2 * width];
  }
  meet[wave][lane] = sum;
  __syncthreads();
  if (wave == 0 && c < width) {
    sum = meet[0][lane];
#pragma unroll
    for (int q = 1; q < 16; ++q) sum += meet[q][lane];
    out[c] = (P)sum;
  }
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------

constexpr int kGradParts = 256;       // workgroups of the gradient, each with one part
constexpr int64_t kMaxWidth = 1 << 30;

template <class T, class P, int LANES, int NV>
void launch_norm(const NormArgs& a, hipStream_t s) {
  constexpr int rows = norm_threads<LANES>() / LANES;
  norm_kernel<T, P, LANES, NV><<<hcg::grid_of((a.rows + rows - 1) / rows), norm_threads<LANES>(), 0, s>>>(a);
}

template <class T, class P>
void run_norm(const NormArgs& a, hipStream_t s) {
  const int64_t vecs = ((int64_t)a.width + kVec<T> - 1) / kVec<T>;  // 16-byte vectors in a row
  if (vecs <= 16) return launch_norm<T, P, 16, 1>(a, s);
  if (vecs <= 32) return launch_norm<T, P, 32, 1>(a, s);
  if (vecs <= 64) return launch_norm<T, P, 64, 1>(a, s);
  // As few lanes as hold the row.  us, 64 / 16 lanes (65536 x 128 bf16) 23.6 / 9.1,
  // 64 / 32 (16384 x 256) 7.8 / 5.5, 256 / 128 (16384 x 1024) 22.0 / 16.1.
  if (vecs <= 128) return launch_norm<T, P, 128, 1>(a, s);
  if (vecs <= 256) return launch_norm<T, P, 256, 1>(a, s);
  if (vecs <= 512) return launch_norm<T, P, 256, 2>(a, s);
  if (vecs <= 1024) return launch_norm<T, P, 256, 4>(a, s);
  if (vecs <= 4096) return launch_norm<T, P, 1024, 4>(a, s);
  norm_wide_kernel<T, P><<<hcg::grid_of(a.rows), 1024, 0, s>>>(a);
}

template <class T, class P, int LANES, int NV, int GROUPS, bool LEAN = false>
int launch_norm_grad(const NormGradArgs& a, hipStream_t s) {
  const int64_t wgs = std::min<int64_t>(kGradParts, (a.rows + GROUPS - 1) / GROUPS);
  norm_grad_kernel<T, P, LANES, NV, GROUPS, LEAN><<<dim3((unsigned)wgs), LANES * GROUPS, 0, s>>>(a);
  return (int)wgs;
}

// Returns the number of parts the column sums were left in.
template <class T, class P>
int run_norm_grad(const NormGradArgs& a, hipStream_t s) {
  const int64_t vecs = ((int64_t)a.width + kVec<T> - 1) / kVec<T>;
  // As few lanes per row as hold it, and as many rows as fit 1024 threads (512,
  // where a row is one wave or less: 16 rows of 64 lanes took 2048 x 512 bf16 from
  // 8.0 to 13.0 us): idle lanes are loads that are not in flight.  us, 64 / 16
  // lanes (65536 x 128 bf16) 37.0 / 16.4, 256 / 128 (16384 x 768) 33.1 / 23.1, 256 /
  // 192 (16384 x 1536) 36.2 / 33.0, 512 / 320 (8192 x 2560) 35.5 / 30.2, 512 / 384
  // (8192 x 2880) 37.2 / 35.9; the few rows of 100 x 128 8.0 / 8.0.
  if (vecs <= 16) return launch_norm_grad<T, P, 16, 1, 32>(a, s);
  if (vecs <= 32) return launch_norm_grad<T, P, 32, 1, 16>(a, s);
  if (vecs <= 64) return launch_norm_grad<T, P, 64, 1, 8>(a, s);
  if (vecs <= 128) return launch_norm_grad<T, P, 128, 1, 8>(a, s);
  if (vecs <= 192) return launch_norm_grad<T, P, 192, 1, 5>(a, s);
  if (vecs <= 256) return launch_norm_grad<T, P, 256, 1, 4>(a, s);
  if (vecs <= 320) return launch_norm_grad<T, P, 320, 1, 3>(a, s);
  if (vecs <= 384) return launch_norm_grad<T, P, 384, 1, 2>(a, s);
  if (vecs <= 512) return launch_norm_grad<T, P, 512, 1, 2>(a, s);
  if (vecs <= 1024) return launch_norm_grad<T, P, 512, 2, 1>(a, s);
  if (vecs <= 2048) return launch_norm_grad<T, P, 1024, 2, 1, sizeof(T) == 2>(a, s);
  norm_grad_wide_kernel<T, P><<<hcg::grid_of(a.rows), 1024, 0, s>>>(a);
  const int parts = (int)std::min<int64_t>(64, a.rows);
  if (a.part)
    norm_columns_kernel<T><<<dim3((unsigned)((a.width + 255) / 256), parts), 256, 0, s>>>(a);
  return parts;
}

template <class F>
int with_types(int dtype, int param_dtype, F f) {
  const auto inner = [&](auto t) {
    switch (param_dtype) {
      case HCG_F16: return f(t, ElemOf<HCG_F16>::type{});
      case HCG_BF16: return f(t, ElemOf<HCG_BF16>::type{});
      default: return f(t, float{});
    }
  };
  switch (dtype) {
    case HCG_F16: return inner(ElemOf<HCG_F16>::type{});
    case HCG_BF16: return inner(ElemOf<HCG_BF16>::type{});
    default: return inner(float{});
  }
}

// Parameters have the rows' type or float32.
bool param_ok(int dtype, int param_dtype) { return param_dtype == dtype || param_dtype == HCG_F32; }

}  // namespace

extern "C" {

int hcg_layer_norm(int dtype, const void* x, int64_t ldx, int64_t rows, int64_t width, int param_dtype,
                   const void* weight, const void* bias, float eps, void* y, int64_t ldy, float* mean, float* rstd,
                   void* stream) {
  HCG_LM_REQUIRE(hcg::elem_ok(dtype), "dtype %d is not HCG_F16, HCG_BF16 or HCG_F32", dtype);
  HCG_LM_REQUIRE(param_ok(dtype, param_dtype), "weight and bias must have the rows' type or float32");
  HCG_LM_REQUIRE(rows >= 0 && rows < ((int64_t)1 << 31) && width >= 0 && width <= kMaxWidth,
                 "%lld rows of %lld elements are out of range", (long long)rows, (long long)width);
  if (rows == 0) return HCG_OK;
  HCG_LM_REQUIRE(width > 0, "layer norm of rows without elements");
  HCG_LM_REQUIRE(x && y, "null pointer");
  HCG_LM_REQUIRE(rows == 1 || (ldx >= width && ldy >= width), "row stride below the width %lld", (long long)width);
  HCG_LM_REQUIRE(hcg::elem_aligned(x, hcg::elem_bytes(dtype)) && hcg::elem_aligned(y, hcg::elem_bytes(dtype)),
                 "rows must be aligned to their elements");
  const int pb = hcg::elem_bytes(param_dtype);
  HCG_LM_REQUIRE(hcg::elem_aligned(weight, pb) && hcg::elem_aligned(bias, pb) && hcg::elem_aligned(mean, 4) &&
                     hcg::elem_aligned(rstd, 4),
                 "parameters and statistics must be aligned to their elements");
  const NormArgs a{x, weight, bias, y, mean, rstd, ldx, ldy, rows, (int)width, eps};
  with_types(dtype, param_dtype, [&](auto t, auto p) {
    if constexpr (std::is_same_v<decltype(p), float> || std::is_same_v<decltype(p), decltype(t)>)
      run_norm<decltype(t), decltype(p)>(a, static_cast<hipStream_t>(stream));
    return 0;
  });
  HCG_LM_HIP_CHECK(hipGetLastError());
  return HCG_OK;
}

int64_t hcg_layer_norm_grad_workspace(int64_t rows, int64_t width) {
  return rows > 0 && width > 0 ? (int64_t)kGradParts * 2 * width * 4 : 0;
}

int hcg_layer_norm_grad(int dtype, const void* dy, int64_t lddy, const void* x, int64_t ldx, int64_t rows,
                        int64_t width, const float* mean, const float* rstd, int param_dtype, const void* weight,
                        void* dx, int64_t lddx, void* dweight, void* dbias, void* workspace, int64_t workspace_bytes,
                        void* stream) {
  HCG_LM_REQUIRE(hcg::elem_ok(dtype), "dtype %d is not HCG_F16, HCG_BF16 or HCG_F32", dtype);
  HCG_LM_REQUIRE(param_ok(dtype, param_dtype), "weight and bias must have the rows' type or float32");
  HCG_LM_REQUIRE(rows >= 0 && rows < ((int64_t)1 << 31) && width >= 0 && width <= kMaxWidth,
                 "%lld rows of %lld elements are out of range", (long long)rows, (long long)width);
  if (width == 0) {
    HCG_LM_REQUIRE(rows == 0, "layer norm of rows without elements");
    return HCG_OK;
  }
  HCG_LM_REQUIRE(rows == 0 || (dy && x && mean && rstd && dx), "null pointer");
  HCG_LM_REQUIRE(rows <= 1 || (lddy >= width && ldx >= width && lddx >= width), "row stride below the width %lld",
                 (long long)width);
  const int eb = hcg::elem_bytes(dtype);
  HCG_LM_REQUIRE(hcg::elem_aligned(dy, eb) && hcg::elem_aligned(x, eb) && hcg::elem_aligned(dx, eb),
                 "rows must be aligned to their elements");
  const int pb = hcg::elem_bytes(param_dtype);
  HCG_LM_REQUIRE(hcg::elem_aligned(weight, pb) && hcg::elem_aligned(dweight, pb) && hcg::elem_aligned(dbias, pb) &&
                     hcg::elem_aligned(mean, 4) && hcg::elem_aligned(rstd, 4),
                 "parameters and statistics must be aligned to their elements");
  const bool params = dweight || dbias;
  if (params && rows > 0) {
    HCG_LM_REQUIRE(workspace && workspace_bytes >= hcg_layer_norm_grad_workspace(rows, width) &&
                       hcg::elem_aligned(workspace, 256),
                   "workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
                   (long long)hcg_layer_norm_grad_workspace(rows, width));
  }
  const NormGradArgs a{dy,   x,   mean, rstd, weight,     dx, params ? static_cast<float*>(workspace) : nullptr,
                       lddy, ldx, lddx, rows, (int)width,
                       // (past the L2s' 32 MB, where rows are whole lines: 8192 x 4096 bf16 45.1 -> 44.8 us)
                       rows * width * eb > (32 << 20) && hcg::elem_aligned(dx, 128) && lddx * eb % 128 == 0};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  with_types(dtype, param_dtype, [&](auto t, auto p) {
    using T = decltype(t);
    using P = decltype(p);
    if constexpr (std::is_same_v<P, float> || std::is_same_v<P, T>) {
      const int parts = rows > 0 ? run_norm_grad<T, P>(a, s) : 0;
      if (params)
        norm_reduce_kernel<P><<<dim3((unsigned)((width + 63) / 64), 2), 1024, 0, s>>>(
            a.part, parts, (int)width, static_cast<P*>(dweight), static_cast<P*>(dbias));
    }
    return 0;
  });
  HCG_LM_HIP_CHECK(hipGetLastError());
  return HCG_OK;
}

}  // extern "C"
