// hcg_quantize.hip -- quantises a matrix to 8-bit floating point with a scale
// for each 128 columns of a row or each 128 x 128 tile, also transposed
// (include/hcg_fp8.h).
//
//   a = max |x| over the block, s = a / F, q = rne(x F / a).
//
// Bound by HBM: a workgroup reads a 128 x 128 tile of x once, whole 16-byte
// vectors, all of them in flight, and holds it in registers (8 x 8 values per
// thread) between the maximum and the result.  Transposed, the bytes pass
// through LDS, so that both sides are whole lines.  8192 x 8192 float32 by tiles
// 64.2 us (5.2 TB/s), 8192 x 4096 bf16 by rows 19.0 (5.3 TB/s), transposed 18.2 (5.6
// TB/s; 24.5 with loads that waited for each other and scales found by every lane,
// 27.1 with padded instead of swizzled rows in LDS as well), 64 x 8192 bf16 4.5.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "hcg_scale8.h"
#include "hcg_vec.h"

namespace {

using hcg::ElemOf;
using hcg::fp8::kBlock;

struct QuantArgs {
  const void* x;
  int64_t ldx, rows, cols;
  int64_t tiles_c;  // tiles along x's columns
  hcg::fp8::Out out;
};

constexpr int kThreads = 256;
constexpr int kSide = 8;                     // a thread's rows and columns
constexpr int kAcross = kBlock / kSide;      // threads along either side of a tile

// Where row c of a turned tile has its 8 bytes i in LDS: the 16 threads that write
// one i of rows 8 apart cover 32 banks (side by side they would share two).
__device__ __forceinline__ int turned_at(int c, int i) { return c * kBlock + (i ^ (c / kSide)) * kSide; }

__device__ __forceinline__ uint32_t shfl_max(uint32_t v, int mask) {
  return max(v, (uint32_t)__shfl_xor((int)v, mask));
}

// Joins 2 H values of two lanes `mask` apart; each is left with H of them, the lane
// with that bit with the upper ones.  (A scale, with its division, is then found by
// as few lanes as there are.)
template <int H>
__device__ __forceinline__ void halve(uint32_t (&top)[kSide], int lane, int mask) {
  const bool upper = lane & mask;
#pragma unroll
  for (int k = 0; k < H; ++k) {
    const uint32_t away = upper ? top[k] : top[k + H];
    top[k] = max(upper ? top[k + H] : top[k], (uint32_t)__shfl_xor((int)away, mask));
  }
}

// Thread (i, j) = (tid / 16, tid % 16) holds rows 8 i ... and columns 8 j ... of
// the workgroup's tile.
template <class T, bool TRANS, bool TILE>
__global__ __launch_bounds__(kThreads) void quantize_kernel(QuantArgs g) {
  __shared__ uint32_t meet[4 * kBlock];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int i = tid / kAcross, j = tid % kAcross;
  const int64_t tile = hcg::workgroup();
  // (64-bit division is a long sequence of instructions; few matrices need it.)
  const int64_t tr = tile >> 32 ? tile / g.tiles_c : (uint32_t)tile / (uint32_t)g.tiles_c;
  const int64_t tc = tile - tr * g.tiles_c;
  const int64_t row0 = tr * kBlock + i * kSide, col0 = tc * kBlock + j * kSide;
  const int rows = (int)min((int64_t)kSide, g.rows - row0), cols = (int)min((int64_t)kSide, g.cols - col0);
  if (tr * kBlock >= g.rows) return;  // (a whole workgroup past the grid's last tile)

  // Loads without a branch between them, of the last row where there is none, but in
  // a last column of tiles: a load that ends a branch is waited for there.
  constexpr int kEach = hcg::kVec<T>, kParts = kSide / kEach;
  const T* const x = static_cast<const T*>(g.x) + col0;
  hcg::raw4 raw[kSide][kParts];
  if ((tc + 1) * kBlock <= g.cols) {
#pragma unroll
    for (int r = 0; r < kSide; ++r)
#pragma unroll
      for (int p = 0; p < kParts; ++p)
        raw[r][p] = hcg::load_raw(x + min(row0 + r, g.rows - 1) * g.ldx + p * kEach, kEach);
  } else {
#pragma unroll
    for (int r = 0; r < kSide; ++r)
#pragma unroll
      for (int p = 0; p < kParts; ++p) {
        raw[r][p] = hcg::raw4{0, 0, 0, 0};
        if (r < rows && cols > p * kEach)
          raw[r][p] = hcg::load_raw(x + (row0 + r) * g.ldx + p * kEach, cols - p * kEach);
        asm volatile("" : "+v"(raw[r][p]));  // (whole words, not values of 16 bits: they took 200 registers)
      }
  }
  float v[kSide][kSide];
#pragma unroll
  for (int r = 0; r < kSide; ++r)
#pragma unroll
    for (int p = 0; p < kParts; ++p) {
      float part[kEach];
      hcg::unpack<T>(r < rows ? raw[r][p] : hcg::raw4{0, 0, 0, 0}, part);
#pragma unroll
      for (int e = 0; e < kEach; ++e) v[r][p * kEach + e] = part[e];
    }

  float inverse[TILE ? 1 : kSide];  // per row of q that the thread holds
  if constexpr (TILE) {
    uint32_t top = 0;
#pragma unroll
    for (int r = 0; r < kSide; ++r)
#pragma unroll
      for (int e = 0; e < kSide; ++e) top = max(top, hcg::fp8::magnitude(v[r][e]));
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) top = shfl_max(top, m);
    if (lane == 0) meet[wave] = top;
    __syncthreads();
    top = max(max(meet[0], meet[1]), max(meet[2], meet[3]));
    const hcg::fp8::Scale s = hcg::fp8::scale_of(top, g.out.e5m2, g.out.e8m0);
    inverse[0] = s.inverse;
    if (tid == 0) hcg::fp8::put_scale(g.out, TRANS ? tc : tr, TRANS ? tr : tc, s.held);
  } else if constexpr (TRANS) {
    // A row of q is a column of x.
    __shared__ __attribute__((aligned(16))) float found[kBlock];
    uint32_t top[kSide] = {};
#pragma unroll
    for (int e = 0; e < kSide; ++e)
#pragma unroll
      for (int r = 0; r < kSide; ++r) top[e] = max(top[e], hcg::fp8::magnitude(v[r][e]));
    halve<4>(top, lane, 16);
    halve<2>(top, lane, 32);
    uint32_t* const to = meet + wave * kBlock + j * kSide + (lane & 16 ? 4 : 0) + (lane & 32 ? 2 : 0);
    to[0] = top[0], to[1] = top[1];
    __syncthreads();
    if (tid < kBlock) {
      const uint32_t most = max(max(meet[tid], meet[kBlock + tid]), max(meet[2 * kBlock + tid], meet[3 * kBlock + tid]));
      const hcg::fp8::Scale s = hcg::fp8::scale_of(most, g.out.e5m2, g.out.e8m0);
      if (tc * kBlock + tid < g.cols) hcg::fp8::put_scale(g.out, tc * kBlock + tid, tr, s.held);
      found[tid] = s.inverse;
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kSide; ++e) inverse[e] = found[j * kSide + e];
  } else {
    uint32_t top[kSide] = {};
#pragma unroll
    for (int r = 0; r < kSide; ++r)
#pragma unroll
      for (int e = 0; e < kSide; ++e) top[r] = max(top[r], hcg::fp8::magnitude(v[r][e]));
    halve<4>(top, lane, 4);
    halve<2>(top, lane, 2);
    halve<1>(top, lane, 1);
    const hcg::fp8::Scale s = hcg::fp8::scale_of(shfl_max(top[0], 8), g.out.e5m2, g.out.e8m0);  // of row j % 8
    if (j < rows && j < kSide) hcg::fp8::put_scale(g.out, row0 + j, tc, s.held);
#pragma unroll
    for (int r = 0; r < kSide; ++r) inverse[r] = __shfl(s.inverse, (lane & -kAcross) + r);
  }

  if constexpr (!TRANS) {
    if (cols <= 0) return;
#pragma unroll
    for (int r = 0; r < kSide; ++r)
      if (r < rows)
        hcg::fp8::store_q<kSide>(g.out.q + (row0 + r) * g.out.ldq + col0, v[r], inverse[TILE ? 0 : r], cols,
                                 g.out.e5m2);
  } else {
    __shared__ __attribute__((aligned(16))) unsigned char turned[kBlock * kBlock];
#pragma unroll
    for (int e = 0; e < kSide; ++e) {
      float f[kSide];
#pragma unroll
      for (int r = 0; r < kSide; ++r) f[r] = v[r][e];
      hcg::fp8::store_q<kSide>(turned + turned_at(j * kSide + e, i), f, inverse[TILE ? 0 : e], kSide,
                               g.out.e5m2);
    }
    __syncthreads();
    // Rows of q by 8 lanes each, 16 bytes a lane.
    const int part = tid & 7;
    const int left = (int)min((int64_t)16, g.rows - (tr * kBlock + part * 16));
    typedef uint32_t u32x4a __attribute__((ext_vector_type(4), aligned(1)));
#pragma unroll
    for (int c = tid >> 3; c < kBlock; c += kThreads / 8) {
      if (tc * kBlock + c >= g.cols || left <= 0) continue;
      // (Two neighbouring pieces of 8 bytes, in either order.)
      const hcg::raw4 v = *reinterpret_cast<const hcg::raw4*>(turned + (turned_at(c, 2 * part) & ~15));
      const bool swapped = c / kSide & 1;
      const hcg::raw4 q = swapped ? hcg::raw4{v[2], v[3], v[0], v[1]} : v;
      unsigned char* to = g.out.q + (tc * kBlock + c) * g.out.ldq + tr * kBlock + part * 16;
      if (left == 16) {
        *reinterpret_cast<u32x4a*>(to) = q;
      } else {
#pragma unroll
        for (int b = 0; b < 16; ++b)
          if (b < left) to[b] = (unsigned char)(q[b >> 2] >> (8 * (b & 3)));
      }
    }
  }
}

template <class T>
void launch(const QuantArgs& a, bool transpose, bool tile, hipStream_t s) {
  const dim3 grid = hcg::grid_of(a.tiles_c * ((a.rows + kBlock - 1) / kBlock));
  if (transpose && tile)
    quantize_kernel<T, true, true><<<grid, kThreads, 0, s>>>(a);
  else if (transpose)
    quantize_kernel<T, true, false><<<grid, kThreads, 0, s>>>(a);
  else if (tile)
    quantize_kernel<T, false, true><<<grid, kThreads, 0, s>>>(a);
  else
    quantize_kernel<T, false, false><<<grid, kThreads, 0, s>>>(a);
}

}  // namespace

extern "C" int hcg_quantize_fp8(int dtype, const void* x, int64_t ldx, int64_t rows, int64_t cols, int transpose,
                                int tile, int q_dtype, void* q, int64_t ldq, int scale_dtype, void* scale,
                                int64_t scale_row, int64_t scale_block, void* stream) {
  HCG_LM_REQUIRE(hcg::elem_ok(dtype), "dtype %d is not HCG_F16, HCG_BF16 or HCG_F32", dtype);
  HCG_LM_REQUIRE(hcg::fp8::type_ok(q_dtype), "q's type %d is not HCG_E4M3 or HCG_E5M2", q_dtype);
  HCG_LM_REQUIRE(hcg::fp8::scale_ok(scale_dtype), "scales of type %d are not HCG_F32 or HCG_E8M0", scale_dtype);
  constexpr int64_t kMost = (int64_t)1 << 31;
  HCG_LM_REQUIRE(rows >= 0 && rows < kMost && cols >= 0 && cols < kMost, "a matrix of %lld x %lld is out of range",
                 (long long)rows, (long long)cols);
  if (rows == 0 || cols == 0) return HCG_OK;
  HCG_LM_REQUIRE(x && q && scale, "null pointer");
  const int64_t qrows = transpose ? cols : rows, qcols = transpose ? rows : cols;
  HCG_LM_REQUIRE((rows == 1 || ldx >= cols) && (qrows == 1 || ldq >= qcols), "row stride below the width");
  HCG_LM_REQUIRE(hcg::elem_aligned(x, hcg::elem_bytes(dtype)), "rows must be aligned to their elements");
  HCG_LM_REQUIRE(hcg::elem_aligned(scale, hcg::fp8::scale_bytes(scale_dtype)), "scales must be aligned");
  const int64_t tiles_c = (cols + kBlock - 1) / kBlock, tiles_r = (rows + kBlock - 1) / kBlock;
  HCG_LM_REQUIRE(tiles_c * tiles_r < (int64_t)1 << 36, "a matrix of %lld x %lld is out of range", (long long)rows,
                 (long long)cols);
  const QuantArgs a{x,
                    ldx,
                    rows,
                    cols,
                    tiles_c,
                    {static_cast<unsigned char*>(q), scale, ldq, scale_row, scale_block, q_dtype == HCG_E5M2,
                     scale_dtype == HCG_E8M0}};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case HCG_F16: launch<ElemOf<HCG_F16>::type>(a, transpose, tile, s); break;
    case HCG_BF16: launch<ElemOf<HCG_BF16>::type>(a, transpose, tile, s); break;
    default: launch<float>(a, transpose, tile, s);
  }
  HCG_LM_HIP_CHECK(hipGetLastError());
  return HCG_OK;
}
