// hcg_rms.hip -- root-mean-square norm by rows with the residual's addition, its
// form with an 8-bit result, and its gradient (include/hcg_lm.h, hcg_fp8.h).
//
//   h = x + residual, r = 1 / sqrt(sum h^2 / D + eps), y = h r w
// and, with xh = h r and g = dy w,
//   dh = r (g - xh sum(g xh) / D) + dresidual, dw = sum_t dy xh.
//
// All are bound by HBM: a row is read once and held in registers by as few lanes
// as hold it with 16 bytes each, between the sum of squares and the result.  h
// is rounded before the norm, so that the gradient, which reads it, is of the
// same function.  The 8-bit form takes each 128 columns' largest magnitude from
// the 16 or 32 lanes that hold them, by exchanges.  8192 x 4096: to 8 bits with a
// bf16 residual 45 us (5.2 TB/s), f16 with a float32 residual 82 us (4.9), bf16
// gradient with the residual's 46.5 us (5.8) and 4.7 for the columns' sums; one row
// 3.8 us, a launch and its latency.  Wider rows, whole passes: 4096 x 8192 to 8 bits
// 55, 2048 x 16384 70 (1024 lanes of four vectors, half of them idle).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "hcg_scale8.h"
#include "hcg_vec.h"

namespace {

using hcg::ElemOf;
using hcg::kVec;
using hcg::raw4;

struct RmsArgs {
  const void* x;
  const void* residual;  // or null
  const void* weight;    // or null
  void* y;
  void* h;
  float* rstd;  // or null
  int64_t ldx, ldr, ldy, ldh, rows;
  int width;
  float eps;
  bool wide_weight;  // float32, else of x's type
  hcg::fp8::Out out;
};

// E elements of S as they lie in memory.
template <class S, int E>
struct Raws {
  static constexpr int kPer = kVec<S>, kN = E / kPer;
  raw4 v[kN];
  __device__ __forceinline__ void load(const S* p, int valid) {
#pragma unroll
    for (int i = 0; i < kN; ++i)
      v[i] = valid > i * kPer ? hcg::load_raw(p + i * kPer, valid - i * kPer) : raw4{0, 0, 0, 0};
  }
  // The same without a branch, of a row of at least kPer elements, in two steps: a
  // vector past the row's end, or over it, is read as the row's last one, and settle()
  // moves what it holds of the row (`left` columns) to its place.
  __device__ __forceinline__ void load_whole(const S* row, int c, int width) {
    typedef typename hcg::RawAt<sizeof(S)>::type raw4a;
#pragma unroll
    for (int i = 0; i < kN; ++i)
      v[i] = *reinterpret_cast<const raw4a*>(row + min(c + i * kPer, width - kPer));
  }
  __device__ __forceinline__ void settle(int left, bool ragged) {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int away = kPer - max(min(left - i * kPer, kPer), 0);
      raw4 r = v[i];
      if (ragged) {
        constexpr int kWord = 4 / sizeof(S);  // elements
        if (away & 2 * kWord) r = raw4{r[2], r[3], 0, 0};
        if (away & kWord) r = raw4{r[1], r[2], r[3], 0};
        if constexpr (kWord == 2)
          if (away & 1) {
            r = raw4{r[0] >> 16 | r[1] << 16, r[1] >> 16 | r[2] << 16, r[2] >> 16 | r[3] << 16, r[3] >> 16};
          }
      }
      v[i] = away == kPer ? raw4{0, 0, 0, 0} : r;
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kN; ++i) v[i] = raw4{0, 0, 0, 0};
  }
  __device__ __forceinline__ void floats(float (&f)[E]) const {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      float part[kPer];
      hcg::unpack<S>(v[i], part);
#pragma unroll
      for (int e = 0; e < kPer; ++e) f[i * kPer + e] = part[e];
    }
  }
  __device__ __forceinline__ void round(const float (&f)[E]) {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      float part[kPer];
#pragma unroll
      for (int e = 0; e < kPer; ++e) part[e] = f[i * kPer + e];
      v[i] = hcg::pack<S>(part);
    }
  }
  __device__ __forceinline__ void store(S* p, int valid) const {
#pragma unroll
    for (int i = 0; i < kN; ++i)
      if (valid > i * kPer) hcg::store_raw(p + i * kPer, v[i], valid - i * kPer);
  }
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

// E weights from column c on (ones without any; zeros past the row's end).
template <class T, int E>
__device__ __forceinline__ void load_weights(const void* w, bool wide, int c, int left, float (&f)[E]) {
#pragma unroll
  for (int e = 0; e < E; ++e) f[e] = e < left ? 1.f : 0.f;
  if (w == nullptr || left <= 0) return;
  if (wide)
    hcg::load_floats<float, E>(static_cast<const float*>(w) + c, left, f);
  else
    hcg::load_floats<T, E>(static_cast<const T*>(w) + c, left, f);
}

// E columns from c on of row `row`, quantised: G neighbouring lanes hold a block.
template <int E, int G>
__device__ __forceinline__ void emit_q(const hcg::fp8::Out& o, int64_t row, int c, int left, const float (&f)[E],
                                       bool live) {
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (e < left) top = max(top, hcg::fp8::magnitude(f[e]));
#pragma unroll
  for (int m = G / 2; m >= 1; m >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, m));
  if (!live || left <= 0) return;
  const hcg::fp8::Scale s = hcg::fp8::scale_of(top, o.e5m2, o.e8m0);
  hcg::fp8::store_q<E>(o.q + row * o.ldq + c, f, s.inverse, left, o.e5m2);
  if (c % hcg::fp8::kBlock == 0) hcg::fp8::put_scale(o, row, c / hcg::fp8::kBlock, s.held);
}

template <int LANES>
constexpr int rms_threads() {
  return LANES > 256 ? LANES : 256;
}

// One row by LANES lanes, held in registers as NV vectors per lane.  T: x's type,
// H: the residual's, Q: the result in 8 bits.
template <class T, class H, int LANES, int NV, bool Q>
__global__ __launch_bounds__(rms_threads<LANES>()) void rms_kernel(RmsArgs g) {
  constexpr int E = kVec<T>, kRowsPerWg = rms_threads<LANES>() / LANES;
  constexpr int kGroup = hcg::fp8::kBlock / E < LANES ? hcg::fp8::kBlock / E : LANES;
  __shared__ float slots[kRowsPerWg * (LANES > 64 ? LANES / 64 : 1)];
  const int group = threadIdx.x / LANES, tir = threadIdx.x % LANES;
  const int64_t row = hcg::workgroup() * kRowsPerWg + group;
  const bool live = row < g.rows;
  const T* x = static_cast<const T*>(g.x) + (live ? row : 0) * g.ldx;
  const H* res = static_cast<const H*>(g.residual) + (live && g.residual ? row : 0) * g.ldr;
  const int first = tir * E;
  Raws<T, E> raw[NV];
  Raws<H, E> add[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = first + i * LANES * E;
    raw[i].load(x + c, g.width - c);
    if (g.residual)
      add[i].load(res + c, g.width - c);
    else
      add[i].clear();
  }
  float w[NV][E];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = first + i * LANES * E;
    load_weights<T, E>(g.weight, g.wide_weight, c, g.width - c, w[i]);
  }
  float v[NV][E];
  float sq = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    raw[i].floats(v[i]);
    if (g.residual) {
      float r[E];
      add[i].floats(r);
#pragma unroll
      for (int e = 0; e < E; ++e) v[i][e] += r[e];
      add[i].round(v[i]);
      add[i].floats(v[i]);
      const int c = first + i * LANES * E;
      if (live && c < g.width) add[i].store(static_cast<H*>(g.h) + row * g.ldh + c, g.width - c);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) sq += v[i][e] * v[i][e];
  }
  const float rstd = 1.f / sqrtf(row_sum<LANES>(sq, slots + group * (LANES > 64 ? LANES / 64 : 1), tir) /
                                     (float)g.width + g.eps);
  if (live && tir == 0 && g.rstd) g.rstd[row] = rstd;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = first + i * LANES * E;
    float o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = v[i][e] * rstd * w[i][e];
    if constexpr (Q) {
      emit_q<E, kGroup>(g.out, row, c, g.width - c, o, live);
    } else if (live && c < g.width) {
      hcg::store_raw(static_cast<T*>(g.y) + row * g.ldy + c, hcg::pack<T>(o), g.width - c);
    }
  }
}

// Rows too wide for registers (more than 4096 vectors): two passes over the row,
// 1024 threads, the second one adding (and rounding) again.
template <class T, class H, bool Q>
__global__ __launch_bounds__(1024) void rms_wide_kernel(RmsArgs g) {
  constexpr int E = kVec<T>, kStep = 1024 * E;
  __shared__ float slots[16];
  const int64_t row = hcg::workgroup();
  if (row >= g.rows) return;
  const T* x = static_cast<const T*>(g.x) + row * g.ldx;
  const H* res = static_cast<const H*>(g.residual) + (g.residual ? row : 0) * g.ldr;
  H* h = static_cast<H*>(g.h) + (g.residual ? row : 0) * g.ldh;
  const int64_t first = (int64_t)threadIdx.x * E;
  // (h may be the residual: the sums are read back, not made twice.)
  float sq = 0.f;
  for (int64_t c = first; c < g.width; c += kStep) {
    const int left = (int)(g.width - c);
    Raws<T, E> raw;
    float f[E];
    raw.load(x + c, left);
    raw.floats(f);
    if (g.residual) {
      Raws<H, E> add;
      float r[E];
      add.load(res + c, left);
      add.floats(r);
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] += r[e];
      add.round(f);
      add.floats(f);
      add.store(h + c, left);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) sq += f[e] * f[e];
  }
  const float rstd = 1.f / sqrtf(row_sum<1024>(sq, slots, threadIdx.x) / (float)g.width + g.eps);
  if (threadIdx.x == 0 && g.rstd) g.rstd[row] = rstd;
  for (int64_t c0 = 0; c0 < g.width; c0 += kStep) {  // (whole waves: exchanges)
    const int64_t c = c0 + first;
    const int left = c < g.width ? (int)(g.width - c) : 0;
    float f[E], w[E];
    if (g.residual) {
      Raws<H, E> sum;
      sum.load(h + c, left);
      sum.floats(f);
    } else {
      Raws<T, E> raw;
      raw.load(x + c, left);
      raw.floats(f);
    }
    load_weights<T, E>(g.weight, g.wide_weight, (int)c, left, w);
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = f[e] * rstd * w[e];
    if constexpr (Q)
      emit_q<E, hcg::fp8::kBlock / E>(g.out, row, (int)c, left, f, true);
    else if (left > 0)
      hcg::store_raw(static_cast<T*>(g.y) + row * g.ldy + c, hcg::pack<T>(f), left);
  }
}

// ---------------------------------------------------------------------------
// Gradient
// ---------------------------------------------------------------------------

struct RmsGradArgs {
  const void* dy;
  const void* h;
  const float* rstd;
  const void* weight;  // or null
  const void* dres;    // or null
  void* dh;
  float* part;  // [gridDim.x][width]: each workgroup's sums of dy xh; or null
  int64_t lddy, ldh, lddr, lddh, rows;
  int width;
  bool wide_weight;
};

// 256 workgroups, one per CU.  GROUPS row groups of LANES lanes; group q of
// workgroup b takes rows b * GROUPS + q, + gridDim.x * GROUPS, ... and keeps its
// columns' sums of dy xh in registers; the groups' sums meet in LDS once, at the
// end.  AHEAD: a row's loads go out before the work on the row before it.  Not by 1024
// threads with two vectors each, whose registers do not hold both; with a float32 h
// beside a 16-bit dy they do not hold one either (22 of them spill): 2048 x 16384 bf16
// 66.8 us (4.0 TB/s with the sums), with a float32 h 127 (3.7).  Rows hold a
// vector or more, so that no load is behind a branch: the number of those in flight
// would not be known after it, and a row would wait for the next row's as well (8192 x
// 4096 bf16 51.2 -> 46.5 us, 3001 x 1027 float32 12.6 -> 12.0; with the sums 55.2 ->
// 53.4 and 14.6 -> 13.1).
template <class T, class H, int LANES, int NV, int GROUPS, bool AHEAD>
__global__ __launch_bounds__(LANES * GROUPS) void rms_grad_kernel(RmsGradArgs g) {
  constexpr int E = kVec<T>, kWaves = LANES / 64;
  __shared__ float slots[2][kWaves > 1 ? GROUPS * kWaves : 1];
  constexpr int kShare = LANES < 64 ? 64 / LANES : 1, kMeet = GROUPS / kShare;
  __shared__ float meet[kMeet > 1 ? kMeet * LANES * E : 1];
  const int group = threadIdx.x / LANES, tir = threadIdx.x % LANES;
  const int first = tir * E;
  const float count = (float)g.width;
  float w[NV][E], dw[NV][E];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = first + i * LANES * E;
    load_weights<T, E>(g.weight, g.wide_weight, c, g.width - c, w[i]);
#pragma unroll
    for (int e = 0; e < E; ++e) dw[i][e] = 0.f;
  }
  const int64_t step = (int64_t)gridDim.x * GROUPS;
  const bool ragged = g.width % E != 0;
  // (Without a residual's gradient one vector of h is read in its place, and left out.)
  const H* const dres_rows = static_cast<const H*>(g.dres ? g.dres : g.h);
  const int64_t dres_step = g.dres ? g.lddr : 0;
  int parity = 0;
  struct Row {
    float rstd;
    Raws<T, E> dy[NV];
    Raws<H, E> h[NV], dres[NV];
  };
  auto load = [&](Row& r, int64_t row) {
    const int64_t at = min(row, g.rows - 1);
    r.rstd = g.rstd[at];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = first + i * LANES * E;
      r.dy[i].load_whole(static_cast<const T*>(g.dy) + at * g.lddy, c, g.width);
      r.h[i].load_whole(static_cast<const H*>(g.h) + at * g.ldh, c, g.width);
      r.dres[i].load_whole(dres_rows + at * dres_step, g.dres ? c : 0, g.width);
    }
  };
  Row next;
  if constexpr (AHEAD) load(next, (int64_t)blockIdx.x * GROUPS + group);
  // (Every group runs as many turns as the workgroup's first: barriers.)
  for (int64_t row0 = (int64_t)blockIdx.x * GROUPS; row0 < g.rows; row0 += step) {
    const int64_t row = row0 + group;
    const bool live = row < g.rows;
    if constexpr (!AHEAD) load(next, row);
    const float rstd = live ? next.rstd : 0.f;
    float dy[NV][E], xh[NV][E];
    Raws<H, E> dres[NV];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int left = live ? g.width - (first + i * LANES * E) : 0;
      next.dy[i].settle(left, ragged);
      next.h[i].settle(left, ragged);
      next.dres[i].settle(g.dres ? left : 0, ragged);
      next.dy[i].floats(dy[i]);
      next.h[i].floats(xh[i]);
      dres[i] = next.dres[i];
    }
    if constexpr (AHEAD) load(next, row + step);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        xh[i][e] *= rstd;
        dw[i][e] += dy[i][e] * xh[i][e];
        dy[i][e] *= w[i][e];
        s += dy[i][e] * xh[i][e];
      }
    }
    s = lanes_sum<LANES>(s);
    if constexpr (kWaves > 1) {
      float* slot = slots[parity] + group * kWaves;
      if (tir % 64 == 0) slot[tir / 64] = s;
      __syncthreads();
      s = 0.f;
#pragma unroll
      for (int i = 0; i < kWaves; ++i) s += slot[i];
      parity ^= 1;
    }
    s /= count;
    if (live) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = first + i * LANES * E;
        if (c < g.width) {
          float o[E], r[E];
          dres[i].floats(r);
#pragma unroll
          for (int e = 0; e < E; ++e) o[e] = rstd * (dy[i][e] - xh[i][e] * s) + r[e];
          Raws<H, E> out;
          out.round(o);
          out.store(static_cast<H*>(g.dh) + row * g.lddh + c, g.width - c);
        }
      }
    }
  }
  if (g.part == nullptr) return;
  float* part = g.part + (int64_t)blockIdx.x * g.width;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float(&v)[E] = dw[i];
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
        if (c + e < g.width) part[c + e] = v[e];
    }
  }
}

// Rows too wide for registers: a workgroup per row for dh (two passes); the
// column sums follow by rms_columns_kernel.  Three readings of dy and h: 2048 x 16384
// float32 174 us, 3.1 TB/s of what one reading takes.
template <class T, class H>
__global__ __launch_bounds__(1024) void rms_grad_wide_kernel(RmsGradArgs g) {
  constexpr int E = kVec<T>;
  __shared__ float slots[16];
  const int64_t row = hcg::workgroup();
  if (row >= g.rows) return;
  const T* dy = static_cast<const T*>(g.dy) + row * g.lddy;
  const H* h = static_cast<const H*>(g.h) + row * g.ldh;
  const H* dres = static_cast<const H*>(g.dres) + (g.dres ? row : 0) * g.lddr;
  H* dh = static_cast<H*>(g.dh) + row * g.lddh;
  const float rstd = g.rstd[row], count = (float)g.width;
  float s = 0.f;
  for (int pass = 0; pass < 2; ++pass) {
    for (int64_t c = (int64_t)threadIdx.x * E; c < g.width; c += 1024 * E) {
      const int left = (int)(g.width - c);
      Raws<T, E> a;
      Raws<H, E> b;
      float d[E], x[E], w[E];
      a.load(dy + c, left);
      b.load(h + c, left);
      a.floats(d);
      b.floats(x);
      load_weights<T, E>(g.weight, g.wide_weight, (int)c, left, w);
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] *= rstd, d[e] *= w[e];
      if (pass == 0) {
#pragma unroll
        for (int e = 0; e < E; ++e) s += d[e] * x[e];
      } else {
        float r[E];
        Raws<H, E> past;
        if (g.dres)
          past.load(dres + c, left);
        else
          past.clear();
        past.floats(r);
#pragma unroll
        for (int e = 0; e < E; ++e) d[e] = rstd * (d[e] - x[e] * s) + r[e];
        b.round(d);
        b.store(dh + c, left);
      }
    }
    if (pass == 0) s = row_sum<1024>(s, slots, threadIdx.x) / count;
  }
}

// The wide rows' column sums: workgroup (b, q) sums 256 columns over the rows q,
// q + gridDim.y, ...
template <class T, class H>
__global__ __launch_bounds__(256) void rms_columns_kernel(RmsGradArgs g) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= g.width) return;
  float dw = 0.f;
  for (int64_t row = blockIdx.y; row < g.rows; row += gridDim.y)
    dw += (float)static_cast<const T*>(g.dy)[row * g.lddy + c] *
          ((float)static_cast<const H*>(g.h)[row * g.ldh + c] * g.rstd[row]);
  g.part[(int64_t)blockIdx.y * g.width + c] = dw;
}

// dw from the workgroups' sums (4 MB at a width of 4096: 4.6 us): 64 columns by 16 waves, wave q adding the parts
// q, q + 16, ..., the waves' sums added in order.
template <class P>
__global__ __launch_bounds__(1024) void rms_reduce_kernel(const float* part, int parts, int width, P* dweight) {
  __shared__ float meet[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = hcg::workgroup_short() * 64 + lane;
  float sum = 0.f;
  if (c < width) {
#pragma unroll 16
    for (int q = wave; q < parts; q += 16) sum += part[(int64_t)q * width + c];
  }
  meet[wave][lane] = sum;
  __syncthreads();
  if (wave == 0 && c < width) {
    sum = meet[0][lane];
#pragma unroll
    for (int q = 1; q < 16; ++q) sum += meet[q][lane];
    dweight[c] = (P)sum;
  }
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------

constexpr int kGradParts = 256;  // workgroups of the gradient, each with one part
constexpr int kWideParts = 64;   // row sums of the wide form's columns
constexpr int kMaxVecs = 2048;   // in a row that the gradient holds in registers
constexpr int64_t kMaxWidth = 1 << 30;

// Parts that the column sums are left in, at most: a row has no more than one, and
// rows over kMaxVecs vectors of any type are the wide form's.
int64_t grad_parts(int64_t rows, int64_t width) {
  return std::min<int64_t>(rows, width > kMaxVecs * kVec<_Float16> ? kWideParts : kGradParts);
}

template <class T, class H, int LANES, int NV, bool Q>
void launch_rms(const RmsArgs& a, hipStream_t s) {
  constexpr int rows = rms_threads<LANES>() / LANES;
  rms_kernel<T, H, LANES, NV, Q><<<hcg::grid_of((a.rows + rows - 1) / rows), rms_threads<LANES>(), 0, s>>>(a);
}

template <class T, class H, bool Q>
void run_rms(const RmsArgs& a, hipStream_t s) {
  const int64_t vecs = ((int64_t)a.width + kVec<T> - 1) / kVec<T>;  // 16-byte vectors in a row
  // As few lanes as hold a row (as for layer norm, whose figures for idle lanes are
  // beside its launch).
  if (vecs <= 16) return launch_rms<T, H, 16, 1, Q>(a, s);
  if (vecs <= 32) return launch_rms<T, H, 32, 1, Q>(a, s);
  if (vecs <= 64) return launch_rms<T, H, 64, 1, Q>(a, s);
  if (vecs <= 128) return launch_rms<T, H, 128, 1, Q>(a, s);
  if (vecs <= 256) return launch_rms<T, H, 256, 1, Q>(a, s);
  if (vecs <= 512) return launch_rms<T, H, 256, 2, Q>(a, s);
  if (vecs <= 1024) return launch_rms<T, H, 256, 4, Q>(a, s);
  if (vecs <= 4096) return launch_rms<T, H, 1024, 4, Q>(a, s);
  rms_wide_kernel<T, H, Q><<<hcg::grid_of(a.rows), 1024, 0, s>>>(a);
}

template <class T, class H, int LANES, int NV, int GROUPS, bool AHEAD = true>
int launch_rms_grad(const RmsGradArgs& a, hipStream_t s) {
  const int64_t wgs = std::min<int64_t>(kGradParts, (a.rows + GROUPS - 1) / GROUPS);
  rms_grad_kernel<T, H, LANES, NV, GROUPS, AHEAD><<<dim3((unsigned)wgs), LANES * GROUPS, 0, s>>>(a);
  return (int)wgs;
}

template <class T, class H>
int run_rms_grad_wide(const RmsGradArgs& a, hipStream_t s) {
  rms_grad_wide_kernel<T, H><<<hcg::grid_of(a.rows), 1024, 0, s>>>(a);
  const int parts = (int)std::min<int64_t>(kWideParts, a.rows);
  if (a.part) rms_columns_kernel<T, H><<<dim3((unsigned)((a.width + 255) / 256), parts), 256, 0, s>>>(a);
  return parts;
}

// Returns the number of parts the column sums were left in.
template <class T, class H>
int run_rms_grad(const RmsGradArgs& a, hipStream_t s) {
  const int64_t vecs = ((int64_t)a.width + kVec<T> - 1) / kVec<T>;
  if (a.width < kVec<T>) return run_rms_grad_wide<T, H>(a, s);
  // As few lanes as hold a row, and as many rows as fit 1024 threads (512, where a
  // row is one wave or less): idle lanes are loads that are not in flight.
  if (vecs <= 16) return launch_rms_grad<T, H, 16, 1, 32>(a, s);
  if (vecs <= 32) return launch_rms_grad<T, H, 32, 1, 16>(a, s);
  if (vecs <= 64) return launch_rms_grad<T, H, 64, 1, 8>(a, s);
  if (vecs <= 128) return launch_rms_grad<T, H, 128, 1, 8>(a, s);
  if (vecs <= 192) return launch_rms_grad<T, H, 192, 1, 5>(a, s);
  if (vecs <= 256) return launch_rms_grad<T, H, 256, 1, 4>(a, s);
  if (vecs <= 320) return launch_rms_grad<T, H, 320, 1, 3>(a, s);
  if (vecs <= 384) return launch_rms_grad<T, H, 384, 1, 2>(a, s);
  if (vecs <= 512) return launch_rms_grad<T, H, 512, 1, 2>(a, s);
  if (vecs <= 1024) return launch_rms_grad<T, H, 512, 2, 1>(a, s);
  if (vecs <= kMaxVecs) return launch_rms_grad<T, H, 1024, 2, 1, false>(a, s);
  return run_rms_grad_wide<T, H>(a, s);
}

// f(x's type, the residual's type).
template <class F>
void with_types(int dtype, int wide, F f) {
  const auto inner = [&](auto t) {
    if (wide == HCG_F32)
      f(t, float{});
    else
      f(t, t);
  };
  switch (dtype) {
    case HCG_F16: return inner(ElemOf<HCG_F16>::type{});
    case HCG_BF16: return inner(ElemOf<HCG_BF16>::type{});
    default: return f(float{}, float{});
  }
}

// Parameters and residuals have the rows' type or float32.
bool with_ok(int dtype, int other) { return other == dtype || other == HCG_F32; }

// What both forms of the norm ask of their arguments but the result.
int check_rms(int dtype, const void* x, int64_t ldx, int64_t rows, int64_t width, int residual_dtype,
              const void* residual, int64_t ldr, int param_dtype, const void* weight, const void* h, int64_t ldh,
              const float* rstd) {
  HCG_LM_REQUIRE(hcg::elem_ok(dtype), "dtype %d is not HCG_F16, HCG_BF16 or HCG_F32", dtype);
  HCG_LM_REQUIRE(with_ok(dtype, param_dtype), "weight must have the rows' type or float32");
  HCG_LM_REQUIRE(residual == nullptr || with_ok(dtype, residual_dtype), "residual must have the rows' type or float32");
  HCG_LM_REQUIRE(rows >= 0 && rows < ((int64_t)1 << 31) && width >= 0 && width <= kMaxWidth,
                 "%lld rows of %lld elements are out of range", (long long)rows, (long long)width);
  if (rows == 0) return HCG_OK;
  HCG_LM_REQUIRE(width > 0, "norm of rows without elements");
  HCG_LM_REQUIRE(x && (residual == nullptr || h), "null pointer");
  HCG_LM_REQUIRE(rows == 1 || (ldx >= width && (residual == nullptr || (ldr >= width && ldh >= width))),
                 "row stride below the width %lld", (long long)width);
  const int eb = hcg::elem_bytes(dtype), rb = residual ? hcg::elem_bytes(residual_dtype) : 1;
  HCG_LM_REQUIRE(hcg::elem_aligned(x, eb) && hcg::elem_aligned(residual, rb) &&
                     (residual == nullptr || hcg::elem_aligned(h, rb)),
                 "rows must be aligned to their elements");
  HCG_LM_REQUIRE(hcg::elem_aligned(weight, hcg::elem_bytes(param_dtype)) && hcg::elem_aligned(rstd, 4),
                 "weight and statistics must be aligned to their elements");
  return HCG_OK;
}

}  // namespace

extern "C" {

int hcg_rms_norm(int dtype, const void* x, int64_t ldx, int64_t rows, int64_t width, int residual_dtype,
                 const void* residual, int64_t ldr, int param_dtype, const void* weight, float eps, void* y,
                 int64_t ldy, void* h, int64_t ldh, float* rstd, void* stream) {
  const int rc = check_rms(dtype, x, ldx, rows, width, residual_dtype, residual, ldr, param_dtype, weight, h, ldh, rstd);
  if (rc != HCG_OK || rows == 0) return rc;
  HCG_LM_REQUIRE(y, "null pointer");
  HCG_LM_REQUIRE(rows == 1 || ldy >= width, "row stride below the width %lld", (long long)width);
  HCG_LM_REQUIRE(hcg::elem_aligned(y, hcg::elem_bytes(dtype)), "rows must be aligned to their elements");
  RmsArgs a{x, residual, weight, y, h, rstd, ldx, ldr, ldy, ldh, rows, (int)width, eps, param_dtype == HCG_F32, {}};
  with_types(dtype, residual ? residual_dtype : dtype, [&](auto t, auto r) {
    run_rms<decltype(t), decltype(r), false>(a, static_cast<hipStream_t>(stream));
  });
  HCG_LM_HIP_CHECK(hipGetLastError());
  return HCG_OK;
}

int hcg_rms_norm_fp8(int dtype, const void* x, int64_t ldx, int64_t rows, int64_t width, int residual_dtype,
                     const void* residual, int64_t ldr, int param_dtype, const void* weight, float eps, int q_dtype,
                     void* q, int64_t ldq, int scale_dtype, void* scale, int64_t scale_row, int64_t scale_block,
                     void* h, int64_t ldh, float* rstd, void* stream) {
  HCG_LM_REQUIRE(hcg::fp8::type_ok(q_dtype), "q's type %d is not HCG_E4M3 or HCG_E5M2", q_dtype);
  HCG_LM_REQUIRE(hcg::fp8::scale_ok(scale_dtype), "scales of type %d are not HCG_F32 or HCG_E8M0", scale_dtype);
  const int rc = check_rms(dtype, x, ldx, rows, width, residual_dtype, residual, ldr, param_dtype, weight, h, ldh, rstd);
  if (rc != HCG_OK || rows == 0) return rc;
  HCG_LM_REQUIRE(q && scale, "null pointer");
  HCG_LM_REQUIRE(rows == 1 || ldq >= width, "row stride below the width %lld", (long long)width);
  HCG_LM_REQUIRE(hcg::elem_aligned(scale, hcg::fp8::scale_bytes(scale_dtype)), "scales must be aligned");
  RmsArgs a{x,
            residual,
            weight,
            nullptr,
            h,
            rstd,
            ldx,
            ldr,
            0,
            ldh,
            rows,
            (int)width,
            eps,
            param_dtype == HCG_F32,
            {static_cast<unsigned char*>(q), scale, ldq, scale_row, scale_block, q_dtype == HCG_E5M2,
             scale_dtype == HCG_E8M0}};
  with_types(dtype, residual ? residual_dtype : dtype, [&](auto t, auto r) {
    run_rms<decltype(t), decltype(r), true>(a, static_cast<hipStream_t>(stream));
  });
  HCG_LM_HIP_CHECK(hipGetLastError());
  return HCG_OK;
}

int64_t hcg_rms_norm_grad_workspace(int64_t rows, int64_t width) {
  return rows > 0 && width > 0 ? grad_parts(rows, width) * width * 4 : 0;
}

int hcg_rms_norm_grad(int dtype, const void* dy, int64_t lddy, int h_dtype, const void* h, int64_t ldh, int64_t rows,
                      int64_t width, const float* rstd, int param_dtype, const void* weight, const void* dresidual,
                      int64_t lddr, void* dh, int64_t lddh, void* dweight, void* workspace, int64_t workspace_bytes,
                      void* stream) {
  HCG_LM_REQUIRE(hcg::elem_ok(dtype), "dtype %d is not HCG_F16, HCG_BF16 or HCG_F32", dtype);
  HCG_LM_REQUIRE(with_ok(dtype, param_dtype) && with_ok(dtype, h_dtype), "weight and h must have dy's type or float32");
  HCG_LM_REQUIRE(rows >= 0 && rows < ((int64_t)1 << 31) && width >= 0 && width <= kMaxWidth,
                 "%lld rows of %lld elements are out of range", (long long)rows, (long long)width);
  if (width == 0) {
    HCG_LM_REQUIRE(rows == 0, "norm of rows without elements");
    return HCG_OK;
  }
  HCG_LM_REQUIRE(rows == 0 || (dy && h && rstd && dh), "null pointer");
  HCG_LM_REQUIRE(rows <= 1 || (lddy >= width && ldh >= width && lddh >= width && (dresidual == nullptr || lddr >= width)),
                 "row stride below the width %lld", (long long)width);
  const int hb = hcg::elem_bytes(h_dtype), pb = hcg::elem_bytes(param_dtype);
  HCG_LM_REQUIRE(hcg::elem_aligned(dy, hcg::elem_bytes(dtype)) && hcg::elem_aligned(h, hb) &&
                     hcg::elem_aligned(dresidual, hb) && hcg::elem_aligned(dh, hb),
                 "rows must be aligned to their elements");
  HCG_LM_REQUIRE(hcg::elem_aligned(weight, pb) && hcg::elem_aligned(dweight, pb) && hcg::elem_aligned(rstd, 4),
                 "weight, its gradient and statistics must be aligned to their elements");
  if (dweight && rows > 0) {
    HCG_LM_REQUIRE(workspace && workspace_bytes >= hcg_rms_norm_grad_workspace(rows, width) &&
                       hcg::elem_aligned(workspace, 256),
                   "workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
                   (long long)hcg_rms_norm_grad_workspace(rows, width));
  }
  const RmsGradArgs a{dy,   h,   rstd, weight, dresidual, dh,         dweight ? static_cast<float*>(workspace) : nullptr,
                      lddy, ldh, lddr, lddh,   rows,      (int)width, param_dtype == HCG_F32};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  with_types(dtype, h_dtype, [&](auto t, auto r) {
    using T = decltype(t);
    const int parts = rows > 0 ? run_rms_grad<T, decltype(r)>(a, s) : 0;
    if (dweight == nullptr) return;
    const dim3 grid = hcg::grid_of((width + 63) / 64);
    if (param_dtype == HCG_F32)
      rms_reduce_kernel<float><<<grid, 1024, 0, s>>>(a.part, parts, (int)width, static_cast<float*>(dweight));
    else
      rms_reduce_kernel<T><<<grid, 1024, 0, s>>>(a.part, parts, (int)width, static_cast<T*>(dweight));
  });
  HCG_LM_HIP_CHECK(hipGetLastError());
  return HCG_OK;
}

}  // extern "C"
