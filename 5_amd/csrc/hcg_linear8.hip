// hcg_linear8.hip -- the product of two quantised matrices, y = x w^T
// (include/hcg_fp8.h):
//
//   y[t][v] = sum_b sx[t][b] sw[v][b] sum_{k in b} x[t][k] w[v][k]
//
// over blocks b of 128 inputs (sw per row v or per 128 of them).  One
// v_mfma_f32_16x16x128 takes a block: w's rows on its M side (a lane's four
// registers, consecutive outputs of a token), tokens on its N side (lanes), so
// that a token's scale is one value per lane.  Both operands' lanes hold the
// same 32 of a block's inputs, l / 16 of them; which, makes no difference.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "hcg_scale8.h"
#include "hcg_tile8.h"
#include "hcg_vec.h"

namespace {

using hcg::ElemOf;
using hcg::u32x4;
using hcg::fp8::Args;
using hcg::fp8::by_power;
using hcg::fp8::by_tile;
using hcg::fp8::f32x4;
using hcg::fp8::Halves;
using hcg::fp8::halves;
using hcg::fp8::i32x8;
using hcg::fp8::join;
using hcg::fp8::kBlock;
using hcg::fp8::kPowerRow;
using hcg::fp8::kPowerTile;
using hcg::fp8::kRow;
using hcg::fp8::kTile;
using hcg::fp8::mfma;
using hcg::fp8::Scaling;

typedef uint32_t u32x4b __attribute__((ext_vector_type(4), aligned(1)));

// 16 bytes at p, of which the first `left` are in the row (the rest zero, not
// read).  before: the row has bytes in front of p (at least 16 in all): a part is
// then one load of the row's last 16, shifted.
__device__ __forceinline__ u32x4 load16(const unsigned char* p, int left, bool before) {
  if (left >= 16) return *reinterpret_cast<const u32x4b*>(p);
  u32x4 r{0, 0, 0, 0};
  if (left <= 0) return r;
  if (before) {
    const u32x4 v = *reinterpret_cast<const u32x4b*>(p + left - 16);
    const int gone = 16 - left, words = gone >> 2;
    uint32_t w[5];
#pragma unroll
    for (int i = 0; i < 5; ++i) {
      w[i] = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + words == e) w[i] = v[e];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __builtin_amdgcn_alignbyte(w[i + 1], w[i], gone & 3);
    return r;
  }
#pragma unroll
  for (int b = 0; b < 16; ++b)
    if (b < left) r[b >> 2] |= (uint32_t)p[b] << (8 * (b & 3));
  return r;
}

// Four consecutive outputs of a token, the first `valid` of them in the row.
__device__ __forceinline__ void store4(const Args& g, int64_t t, int v, f32x4 f) {
  const int valid = g.V - v;
  if (valid <= 0) return;
  if (g.y_dtype == HCG_F32) {
    float* p = static_cast<float*>(g.y) + t * g.ldy + v;
    typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
    if (valid >= 4) {
      *reinterpret_cast<f32x4u*>(p) = f;
    } else {
      for (int e = 0; e < valid; ++e) p[e] = f[e];
    }
    return;
  }
  uint16_t h[4];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    h[e] = g.y_dtype == HCG_F16 ? __builtin_bit_cast(uint16_t, (_Float16)f[e])
                                : __builtin_bit_cast(uint16_t, (__bf16)f[e]);
  uint16_t* p = static_cast<uint16_t*>(g.y) + t * g.ldy + v;
  typedef uint32_t u32x2h __attribute__((ext_vector_type(2), aligned(2)));
  if (valid >= 4) {
    *reinterpret_cast<u32x2h*>(p) =
        u32x2h{(uint32_t)h[0] | (uint32_t)h[1] << 16, (uint32_t)h[2] | (uint32_t)h[3] << 16};
  } else {
    for (int e = 0; e < valid; ++e) p[e] = h[e];
  }
}

// ---------------------------------------------------------------------------
// Operands straight into registers
// ---------------------------------------------------------------------------

// A scale as a float.
__device__ __forceinline__ float power(uint32_t byte) {
  return __builtin_bit_cast(float, byte == 0 ? 0x00400000u : byte == 255 ? 0x7fc00000u : byte << 23);
}
template <Scaling SC>
__device__ __forceinline__ float scale_at(const void* p, int64_t at) {
  if constexpr (by_power(SC)) return power(static_cast<const unsigned char*>(p)[at]);
  return static_cast<const float*>(p)[at];
}

// For few tokens, bound by reading the weight (8192 x 8192: one token 12.8 us, 5.2
// TB/s, 16 tokens 14.5).  A workgroup takes 16 R rows of the weight and 16 NI tokens;
// its waves take the blocks of K in turn, each an own load of both operands, a block
// ahead, and their sums meet in LDS, in the order of the waves.  Workgroups start at
// blocks of their own (a golden-ratio sequence) and wrap: rows a power of two apart
// put what is read at one k on a few HBM channels (4096 x 4096, one token: 5.9 -> 4.7
// us in one run; passes over several weights take 5.4, and 6.8 for 16 tokens).
// Waves, that is, parts of K: as many again where a workgroup has 16 rows.
constexpr int stream_waves(int r) { return r == 1 ? 8 : 4; }

template <bool X5, Scaling SC, bool EXACT, int NI, int R>
__global__ __launch_bounds__(64 * stream_waves(R)) void stream_kernel(Args g) {
  constexpr int kStreamWaves = stream_waves(R);
  __shared__ f32x4 meet[kStreamWaves][R * NI][64];
  const int lane = threadIdx.x & 63, quad = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // (Fewer than 2^32 workgroups.)
  const uint32_t tiles_v = (g.V + 16 * R - 1) / (16 * R), tiles = tiles_v * ((g.T + 16 * NI - 1) / (16 * NI));
  const int64_t number = hcg::workgroup();
  if (number >= (int64_t)tiles * g.splits) return;
  const uint32_t wg = (uint32_t)number, tile = wg % tiles;
  const int split = (int)(wg / tiles);
  const int v0 = (int)(tile % tiles_v) * 16 * R;
  const int64_t t0 = (int64_t)(tile / tiles_v) * (16 * NI);
  // (Rows past the ends read the last one; their results go nowhere.)
  const unsigned char* w[R];
  int64_t sw[R][by_power(SC) && !EXACT ? 1 : 4];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int v = min(v0 + 16 * i + (lane & 15), g.V - 1);
    w[i] = g.w + v * g.ldw + quad * 16;
    if constexpr (by_power(SC) && !EXACT) {
      sw[i][0] = (by_tile(SC) ? v / kBlock : v) * g.sw_row;
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int vr = min(v0 + 16 * i + 4 * quad + r, g.V - 1);
        sw[i][r] = (by_tile(SC) ? vr / kBlock : vr) * g.sw_row;
      }
    }
  }
  const unsigned char* x[NI];
  int64_t sx[NI];
#pragma unroll
  for (int j = 0; j < NI; ++j) {
    const int64_t t = min(t0 + j * 16 + (lane & 15), (int64_t)g.T - 1);
    x[j] = g.x + t * g.ldx + quad * 16;
    sx[j] = t * g.sx_row;
  }
  f32x4 acc[R][NI];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j) acc[i][j] = f32x4{};

  // Blocks of this split: `first` on, `whole` of them of kBlock inputs.
  const int first = split * (g.chunk / kBlock), K = min(g.K - split * g.chunk, g.chunk), whole = K / kBlock;
  const int start = (int)(((uint64_t)(wg * 2654435769u) * (uint32_t)whole) >> 32);
  struct Block {
    u32x4 w[R][2], x[NI][2];
    float sx[NI], sw[R][by_tile(SC) ? 1 : 4];
    int ex[NI], ew[R];
  };
  // A lane's bytes of a block are chunks l / 16 and l / 16 + 4: 64 neighbouring bytes
  // of a row per load.
  auto load = [&](Block& q, int b, auto full) {
    const int64_t k = (int64_t)b * kBlock;
    const int left = decltype(full)::value ? kBlock : g.K - (int)k - quad * 16;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int i = 0; i < R; ++i)
        q.w[i][h] = decltype(full)::value ? *reinterpret_cast<const u32x4b*>(w[i] + k + 64 * h)
                                          : load16(w[i] + k + 64 * h, left - 64 * h, g.K >= 16);
#pragma unroll
      for (int j = 0; j < NI; ++j)
        q.x[j][h] = decltype(full)::value ? *reinterpret_cast<const u32x4b*>(x[j] + k + 64 * h)
                                          : load16(x[j] + k + 64 * h, left - 64 * h, g.K >= 16);
    }
    if constexpr (by_power(SC) && !EXACT) {
#pragma unroll
      for (int j = 0; j < NI; ++j) q.ex[j] = static_cast<const unsigned char*>(g.sx)[sx[j] + b * g.sx_block];
#pragma unroll
      for (int i = 0; i < R; ++i) q.ew[i] = static_cast<const unsigned char*>(g.sw)[sw[i][0] + b * g.sw_block];
    } else {
#pragma unroll
      for (int j = 0; j < NI; ++j) q.sx[j] = scale_at<SC>(g.sx, sx[j] + b * g.sx_block);
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int r = 0; r < (by_tile(SC) ? 1 : 4); ++r) q.sw[i][r] = scale_at<SC>(g.sw, sw[i][r] + b * g.sw_block);
    }
  };
  auto add = [&](const Block& q) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const i32x8 fw = join(q.w[i][0], q.w[i][1]);
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        const i32x8 fx = join(q.x[j][0], q.x[j][1]);
        if constexpr (by_power(SC) && !EXACT) {
          acc[i][j] = mfma<X5>(fw, fx, acc[i][j], q.ew[i], q.ex[j]);
        } else {
          f32x4 part;
          if constexpr (EXACT)
            part = mfma(halves<false>(fw), halves<X5>(fx));
          else
            part = mfma<X5>(fw, fx, f32x4{});
#pragma unroll
          for (int r = 0; r < 4; ++r)
            acc[i][j][r] = __builtin_fmaf(part[r], q.sx[j] * q.sw[i][by_tile(SC) ? 0 : r], acc[i][j][r]);
        }
      }
    }
  };
  auto place = [&](int n) {  // of a wave's n-th block
    const int b = n + start;
    return first + (b >= whole ? b - whole : b);
  };
  // Two blocks in turn, so that a block's loads never wait for a move of the one
  // before; a load past the end reads the last block again.
  Block now, next;
  const int last = (whole - 1 - wave) / kStreamWaves * kStreamWaves + wave;
  if (wave < whole) {
    load(now, place(wave), std::true_type{});
    for (int n = wave; n < whole; n += 2 * kStreamWaves) {
      load(next, place(min(n + kStreamWaves, last)), std::true_type{});
      __builtin_amdgcn_sched_barrier(0);
      add(now);
      __builtin_amdgcn_sched_barrier(0);
      load(now, place(min(n + 2 * kStreamWaves, last)), std::true_type{});
      __builtin_amdgcn_sched_barrier(0);
      if (n + kStreamWaves < whole) add(next);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  if (K % kBlock && wave == whole % kStreamWaves) {
    load(now, first + whole, std::false_type{});
    add(now);
  }

#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j) meet[wave][i * NI + j][lane] = acc[i][j];
  __syncthreads();
  for (int u = wave; u < R * NI; u += kStreamWaves) {
    f32x4 sum = meet[0][u][lane];
#pragma unroll
    for (int q = 1; q < kStreamWaves; ++q) sum += meet[q][u][lane];
    const int64_t t = t0 + u % NI * 16 + (lane & 15);
    const int v = v0 + u / NI * 16 + 4 * quad;
    if (t >= g.T) continue;
    if (g.splits > 1) {
      if (v < g.V) *reinterpret_cast<f32x4*>(g.part + ((int64_t)split * g.T + t) * g.ld_part + v) = sum;
    } else {
      store4(g, t, v, sum);
    }
  }
}

// ---------------------------------------------------------------------------
// What the tiled kernel does not take as it is
// ---------------------------------------------------------------------------

// Rows of `width` bytes at any address into rows of whole 16 bytes (zeros past
// the width).
__global__ __launch_bounds__(256) void copy_rows_kernel(const unsigned char* from, int64_t ld, int64_t rows, int width,
                                                        unsigned char* to, int64_t ldt) {
  const int64_t vecs = ldt / 16, total = rows * vecs;
  for (int64_t at = hcg::workgroup() * 256 + threadIdx.x; at < total; at += (int64_t)gridDim.x * gridDim.y * 256) {
    const int64_t row = at / vecs;
    const int c = (int)(at - row * vecs) * 16;
    *reinterpret_cast<u32x4*>(to + row * ldt + c) = load16(from + row * ld + c, width - c, width >= 16);
  }
}

// Scales in any strides to rows next to each other, block by block, as floats or
// (e8m0 to e8m0) bytes; zeros in rows past `rows`.
__global__ __launch_bounds__(256) void copy_scales_kernel(const void* from, int64_t row_stride, int64_t block_stride,
                                                          int64_t rows, int64_t blocks, void* to, int64_t ldt,
                                                          bool from_e8m0, bool to_e8m0) {
  const int64_t total = blocks * ldt;
  for (int64_t at = hcg::workgroup() * 256 + threadIdx.x; at < total; at += (int64_t)gridDim.x * gridDim.y * 256) {
    const int64_t block = at / ldt, row = at - block * ldt;
    const int64_t src = row * row_stride + block * block_stride;
    if (to_e8m0)
      static_cast<unsigned char*>(to)[at] = row < rows ? static_cast<const unsigned char*>(from)[src] : 0;
    else
      static_cast<float*>(to)[at] = row >= rows  ? 0.f
                                    : from_e8m0 ? power(static_cast<const unsigned char*>(from)[src])
                                                : static_cast<const float*>(from)[src];
  }
}

// The splits' sums, added in order, rounded.
template <class T>
__global__ __launch_bounds__(256) void join_kernel(const float* part, int64_t ld_part, int splits, int64_t tokens, int V,
                                                   T* y, int64_t ldy) {
  const int64_t vecs = ld_part / 4, total = tokens * vecs;
  for (int64_t at = hcg::workgroup() * 256 + threadIdx.x; at < total; at += (int64_t)gridDim.x * gridDim.y * 256) {
    const int64_t t = at / vecs;
    const int v = (int)(at - t * vecs) * 4;
    const float* p = part + t * ld_part + v;
    f32x4 sum{};
#pragma unroll 4
    for (int s = 0; s < splits; ++s) sum += *reinterpret_cast<const f32x4*>(p + s * tokens * ld_part);
    T* row = y + t * ldy;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (v + e < V) row[v + e] = (T)sum[e];
  }
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------

constexpr int64_t kMaxInputs = 4000000;  // and row strides: a tile's offsets stay in 31 bits
constexpr int64_t kMaxRows = (int64_t)1 << 26;

int64_t round_up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Forms of the product: tiles of outputs and tokens, and the workgroups that share
// a CU.
enum Shape { kStream, kLarge, kMedium, kSmall, kNumShapes };
struct ShapeInfo {
  int tm, tn, per_cu;
};
constexpr ShapeInfo kShapes[kNumShapes] = {{0, 0, 2}, {256, 256, 1}, {128, 128, 2}, {128, 64, 2}};
constexpr int kMaxSplits = 16;
constexpr int kCus = 256;
constexpr int64_t kMaxTiles = (int64_t)1 << 22;  // of a launch: its threads are fewer than 2^32

// A model of a form's time in us.  Tiles: a launch, and per round of workgroups a
// tile's start and end and its stages, one of which takes `lo` on an idle chip and
// `hi` on a busy one, or a start and the weight from HBM (`rate`, MB per us).  Stream:
// a launch, and a CU's reading of 16 rows (of the weight and of x's), per block, by
// eight waves (`fixed`) or by four (`lo`), or the weight from HBM.  Split sums: a
// launch, and their MB per us.  Fitted to 100000 times of 9000 random sizes of up to
// 16384, every form and 1 to 16 splits; the pick is within 2.1% of the fastest in the
// mean, and within 10% at 90% of the sizes.  (It ranks forms and foretells no times:
// one token by 8192 x 8192 comes out at 18.9 us for 12.8.  Where it loses, us picked /
// best: 32 tokens by 8192 x 8192 19.2 / 17.2, 64 by it 20.9 / 18.9, 256 by 4096 x 4096
// 20.4 / 17.6.)
struct Cost {
  double launch, fixed, lo, hi, join, join_rate, rate;
};
// 16-bit results, those of weights scaled by rows in float32, float32 results.
enum Kind { kEightBit, kByRows, kExact };
constexpr Cost kCosts[3][kNumShapes] = {
    {{3.501, 0.06312, 0.06408, 0, 2.493, 0.7264, 4.346},
     {2.441, 4.915, 1.041, 1.47, 1.095, 2.883, 5.371},
     {1.471, 3.126, 0.5236, 1.092, 2.125, 2.53, 5.047},
     {0.8981, 3.142, 0.4686, 0.7523, 2.162, 2.272, 5.164}},
    {{3.533, 0.06905, 0.06739, 0, 2.522, 0.6559, 3.862},
     {},
     {2.985, 2.664, 0.6613, 1.294, 1.688, 2.596, 4.44},
     {1.861, 2.786, 0.552, 0.9062, 2.285, 2.311, 4.965}},
    {{3.57, 0.07146, 0.08228, 0, 2.481, 0.5148, 4.034},
     {},
     {1.761, 3.908, 1.068, 2.036, 1.858, 2.495, 2.848},
     {1.722, 3.517, 0.7111, 1.298, 2.425, 2.274, 3.875}}};

struct Problem {
  int algo;
  int64_t tokens, outputs, inputs;
  const void* x;
  int64_t ldx;
  const void* w;
  int64_t ldw;
  bool w_tile, e8m0, exact;
  int64_t sx_row, sw_row, sw_block;
  const void* sw;
};

// 16 rows per workgroup of the streaming form (by eight waves), or 32 (by four),
// which read x half as often: what gives a CU less to read.  us, 16 / 32 rows, one
// token by 8192 x 8192 12.2 / 11.4, 16 tokens 16.7 / 12.9, 64 tokens 37.9 / 24.3; one
// by 4096 x 4096 4.6 / 6.1, 16 by it 5.8 / 7.4 (both sides in one run; passes over
// several weights take 12.8, 14.5, 5.4 and 6.8).
int stream_rows(int64_t tokens, int64_t outputs, int splits) {
  const int64_t tiles = ceil_div(tokens, 64) * splits, n = std::min<int64_t>(tokens, 64);
  const int64_t one = ceil_div(ceil_div(outputs, 16) * tiles, kCus) * (16 + n);
  const int64_t two = ceil_div(ceil_div(outputs, 32) * tiles, kCus) * (32 + n);
  return two < one ? 2 : 1;
}
int stream_groups(int64_t tokens) { return tokens <= 16 ? 1 : tokens <= 32 ? 2 : 4; }

// us; `chunk` blocks of K per split.
double cost_of(Shape shape, Kind kind, const Problem& q, int chunk, int splits) {
  const Cost& c = kCosts[kind][shape];
  const uint32_t T = (uint32_t)q.tokens, V = (uint32_t)q.outputs;
  const double from_hbm = (double)V * q.inputs * 1e-6 / c.rate;
  double us = 0;
  if (shape == kStream) {
    const uint32_t r = stream_rows(T, V, splits), wgs = (V + 16 * r - 1) / (16 * r) * splits;  // (up to 64 tokens)
    us = std::max((double)((wgs + kCus - 1) / kCus) * chunk * (r + T / 16.0) * (r == 1 ? c.fixed : c.lo), from_hbm);
  } else {
    const ShapeInfo& s = kShapes[shape];
    const uint32_t units = ((V + s.tm - 1) / s.tm) * ((T + s.tn - 1) / s.tn) * splits, room = kCus * s.per_cu;
    const uint32_t rest = units % room;
    us = (double)(units / room) * (c.fixed + chunk * c.hi);
    if (rest) {
      const double busy = s.per_cu == 1 ? (double)rest / room : std::max(0.0, ((double)rest - kCus) / kCus);
      us += c.fixed + chunk * (c.lo + (c.hi - c.lo) * busy);
    }
    us = std::max(us, c.fixed + from_hbm);
  }
  us += c.launch;
  if (splits > 1) us += c.join + (splits + 0.5) * T * V * 4e-6 / c.join_rate;
  return us;
}

int64_t tiles_of(Shape s, const Problem& q) {
  return ceil_div(q.outputs, kShapes[s].tm) * ceil_div(q.tokens, kShapes[s].tn);
}

void pick(const Problem& q, Shape& shape, int& splits) {
  const Kind kind = q.exact ? kExact : !q.w_tile && !q.e8m0 ? kByRows : kEightBit;
  const int blocks = (int)ceil_div(q.inputs, kBlock);
  double best = -1;
  for (int i = 0; i < kNumShapes; ++i) {
    const Shape s = (Shape)i;
    if (s == kStream && q.tokens > 64) continue;  // (past that a weight is read too often)
    if (s == kLarge && kind != kEightBit) continue;
    const int64_t tiles = s == kStream ? 1 : tiles_of(s, q);
    if (tiles >= kMaxTiles) continue;
    for (const int n : {1, 2, 3, 4, 6, 8, 12, 16}) {
      if (n > 1 && (blocks / n < 2 || tiles * n > 5 * kCus)) break;
      const int chunk = (blocks + n - 1) / n;
      const double us = cost_of(s, kind, q, chunk, (blocks + chunk - 1) / chunk);
      if (best >= 0 && us >= best) continue;
      best = us;
      shape = s;
      splits = n;
    }
  }
}

struct Plan {
  Shape shape;
  int splits, chunk;
  bool copy_x, copy_w, copy_sx, copy_sw;
  int64_t ldx, ldw, lds_x, lds_w, ld_part;                // of the copies
  int64_t x, w, sx, sw, part, total;                      // offsets into the workspace
};

// What a plan can be made for, and whether a launch holds it.
bool algo_ok(int algo) {
  return algo >= 0 && algo % HCG_FP8_SPLITS <= HCG_FP8_128x64 && algo / HCG_FP8_SPLITS <= kMaxSplits &&
         (algo % HCG_FP8_SPLITS != HCG_FP8_AUTO || algo == HCG_FP8_AUTO);
}
bool sizes_ok(int64_t tokens, int64_t outputs, int64_t inputs) {
  return tokens >= 0 && tokens < kMaxRows && outputs >= 0 && outputs < kMaxRows && inputs >= 0 && inputs < kMaxInputs;
}
bool launch_ok(const Plan& p, const Problem& q) {
  return p.shape == kStream ? ceil_div(q.tokens, 16) * ceil_div(q.outputs, 16) * p.splits < (int64_t)1 << 32
                            : tiles_of(p.shape, q) * p.splits < kMaxTiles;
}

bool in_place(const void* p, int64_t ld, int64_t rows) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (rows == 1 || ld % 16 == 0);
}

Plan make_plan(const Problem& q) {
  Plan p{};
  const int64_t blocks = ceil_div(q.inputs, kBlock);
  int splits = q.algo / HCG_FP8_SPLITS;
  if (q.algo % HCG_FP8_SPLITS == HCG_FP8_AUTO) {
    p.shape = kMedium;
    pick(q, p.shape, splits);
  } else {
    p.shape = (Shape)(q.algo % HCG_FP8_SPLITS - HCG_FP8_STREAM);
  }
  if (p.shape == kLarge && (q.exact || (!q.w_tile && !q.e8m0))) p.shape = kMedium;
  p.chunk = (int)ceil_div(blocks, std::max(1, splits)) * kBlock;
  p.splits = (int)ceil_div(q.inputs, p.chunk);
  const bool stream = p.shape == kStream;
  const bool floats = q.exact || !q.e8m0;  // scales that the kernel takes
  p.copy_x = !stream && !in_place(q.x, q.ldx, q.tokens);
  p.copy_w = !stream && !in_place(q.w, q.ldw, q.outputs);
  p.ldx = p.ldw = round_up(q.inputs, 16);
  p.copy_sx = !stream && ((q.tokens > 1 && q.sx_row != 1) || (q.e8m0 && floats));
  p.lds_x = q.tokens;
  // The weight's rows are read in whole, aligned fours.
  const int64_t rows = q.w_tile ? ceil_div(q.outputs, kBlock) : q.outputs;
  p.copy_sw = !stream && ((rows > 1 && q.sw_row != 1) || (q.e8m0 && floats) ||
                          (floats && !q.w_tile &&
                           (rows % 4 || (blocks > 1 && q.sw_block % 4) || (reinterpret_cast<uintptr_t>(q.sw) & 15))));
  p.lds_w = round_up(rows, 4);
  p.ld_part = round_up(q.outputs, 4);
  int64_t at = 0;
  const auto take = [&](bool wanted, int64_t bytes) {
    const int64_t here = at;
    if (wanted) at += round_up(bytes, 256);
    return here;
  };
  p.x = take(p.copy_x, q.tokens * p.ldx);
  p.w = take(p.copy_w, q.outputs * p.ldw);
  p.sx = take(p.copy_sx, blocks * p.lds_x * 4);
  p.sw = take(p.copy_sw, blocks * p.lds_w * 4);
  p.part = take(p.splits > 1, p.splits * q.tokens * p.ld_part * 4);
  p.total = at;
  return p;
}

template <bool X5, Scaling SC, bool EXACT, int NI, int R>
void launch_stream(const Args& a, hipStream_t s) {
  const int64_t wgs = ceil_div(a.V, 16 * R) * ceil_div(a.T, 16 * NI) * a.splits;
  stream_kernel<X5, SC, EXACT, NI, R><<<hcg::grid_of(wgs), 64 * stream_waves(R), 0, s>>>(a);
}

template <bool X5, Scaling SC, bool EXACT>
void run_stream(const Args& a, hipStream_t s) {
  const bool two = stream_rows(a.T, a.V, a.splits) == 2;
  const int groups = stream_groups(a.T);
  if (groups == 1)
    two ? launch_stream<X5, SC, EXACT, 1, 2>(a, s) : launch_stream<X5, SC, EXACT, 1, 1>(a, s);
  else if (groups == 2)
    two ? launch_stream<X5, SC, EXACT, 2, 2>(a, s) : launch_stream<X5, SC, EXACT, 2, 1>(a, s);
  else
    two ? launch_stream<X5, SC, EXACT, 4, 2>(a, s) : launch_stream<X5, SC, EXACT, 4, 1>(a, s);
}

template <bool X5, Scaling SC, bool EXACT>
void run_tiles(Shape shape, const Args& a, hipStream_t s) {
  const dim3 grid((unsigned)(ceil_div(a.V, kShapes[shape].tm) * ceil_div(a.T, kShapes[shape].tn) * a.splits));
  if constexpr (SC != kRow && !EXACT) {
    if (shape == kLarge)
      return hcg::fp8::tile_kernel<X5, SC, EXACT, 256, 256, 2, 4><<<grid, 512, 0, s>>>(a);
  }
  if (shape == kSmall)
    return hcg::fp8::tile_kernel<X5, SC, EXACT, 128, 64, 4, 2><<<grid, 512, 0, s>>>(a);
  if constexpr (SC == kRow || EXACT)
    hcg::fp8::tile_kernel<X5, SC, EXACT, 128, 128, 2, 2><<<grid, 256, 0, s>>>(a);
  else
    hcg::fp8::tile_kernel<X5, SC, EXACT, 128, 128, 2, 4><<<grid, 512, 0, s>>>(a);
}

}  // namespace

extern "C" {

int64_t hcg_linear_fp8_workspace(int algo, int64_t tokens, int64_t outputs, int64_t inputs, const void* x, int64_t ldx,
                                 const void* weight, int64_t ldw, int scale_dtype, int64_t xs_row, int w_tile,
                                 const void* w_scale, int64_t ws_row, int64_t ws_block, int out_dtype) {
  // (What the call refuses needs none: the call says why.)
  if (!algo_ok(algo) || !sizes_ok(tokens, outputs, inputs) || tokens == 0 || outputs == 0 || inputs == 0) return 0;
  const Problem q{algo,        tokens, outputs, inputs, x,
                  ldx,         weight, ldw,     w_tile != 0, scale_dtype == HCG_E8M0,
                  out_dtype == HCG_F32, xs_row, ws_row, ws_block, w_scale};
  const Plan p = make_plan(q);
  return launch_ok(p, q) ? p.total : 0;
}

int hcg_linear_fp8(int algo, int x_dtype, const void* x, int64_t ldx, int64_t tokens, const void* weight, int64_t ldw,
                   int64_t outputs, int64_t inputs, int scale_dtype, const void* x_scale, int64_t xs_row,
                   int64_t xs_block, int w_tile, const void* w_scale, int64_t ws_row, int64_t ws_block, int out_dtype,
                   void* y, int64_t ldy, void* workspace, int64_t workspace_bytes, void* stream) {
  HCG_LM_REQUIRE(algo_ok(algo), "unknown algo %d", algo);
  HCG_LM_REQUIRE(hcg::fp8::type_ok(x_dtype), "x's type %d is not HCG_E4M3 or HCG_E5M2", x_dtype);
  HCG_LM_REQUIRE(hcg::fp8::scale_ok(scale_dtype), "scales of type %d are not HCG_F32 or HCG_E8M0", scale_dtype);
  HCG_LM_REQUIRE(hcg::elem_ok(out_dtype), "the output's type %d is not HCG_F16, HCG_BF16 or HCG_F32", out_dtype);
  HCG_LM_REQUIRE(sizes_ok(tokens, outputs, inputs), "%lld tokens, %lld outputs and %lld inputs are out of range",
                 (long long)tokens, (long long)outputs, (long long)inputs);
  if (tokens == 0 || outputs == 0) return HCG_OK;
  HCG_LM_REQUIRE(inputs > 0, "a product over no inputs");
  HCG_LM_REQUIRE(x && weight && x_scale && w_scale && y, "null pointer");
  HCG_LM_REQUIRE((tokens == 1 || (ldx >= inputs && ldy >= outputs)) && (outputs == 1 || ldw >= inputs),
                 "row stride below the width");
  HCG_LM_REQUIRE((tokens == 1 || ldx < kMaxInputs) && (outputs == 1 || ldw < kMaxInputs),
                 "row strides of %lld and %lld are out of range", (long long)ldx, (long long)ldw);
  HCG_LM_REQUIRE(hcg::elem_aligned(y, hcg::elem_bytes(out_dtype)), "rows must be aligned to their elements");
  const int sb = hcg::fp8::scale_bytes(scale_dtype);
  HCG_LM_REQUIRE(hcg::elem_aligned(x_scale, sb) && hcg::elem_aligned(w_scale, sb), "scales must be aligned");
  const bool e8m0 = scale_dtype == HCG_E8M0, exact = out_dtype == HCG_F32;
  const Problem q{algo, tokens, outputs, inputs, x,      ldx,    weight,   ldw,
                  w_tile != 0, e8m0, exact, xs_row, ws_row, ws_block, w_scale};
  const Plan p = make_plan(q);
  HCG_LM_REQUIRE(launch_ok(p, q), "%lld tokens by %lld outputs are out of range", (long long)tokens,
                 (long long)outputs);
  HCG_LM_REQUIRE(p.total == 0 || (workspace && workspace_bytes >= p.total && hcg::elem_aligned(workspace, 256)),
                 "workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)p.total);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  char* const ws = static_cast<char*>(workspace);
  Args a{static_cast<const unsigned char*>(x),
         static_cast<const unsigned char*>(weight),
         tokens == 1 ? 0 : ldx,
         outputs == 1 ? 0 : ldw,
         x_scale,
         w_scale,
         xs_row,
         xs_block,
         ws_row,
         ws_block,
         (int)tokens,
         (int)outputs,
         (int)inputs,
         y,
         ldy,
         out_dtype,
         p.splits,
         p.chunk,
         reinterpret_cast<float*>(ws + p.part),
         p.ld_part};
  const auto grid = [](int64_t items) { return dim3((unsigned)std::min<int64_t>(ceil_div(items, 256), 1 << 14)); };
  const int64_t blocks = ceil_div(inputs, kBlock), w_rows = w_tile ? ceil_div(outputs, kBlock) : outputs;
  if (p.copy_x) {
    unsigned char* to = reinterpret_cast<unsigned char*>(ws + p.x);
    copy_rows_kernel<<<grid(tokens * p.ldx / 16), 256, 0, s>>>(a.x, a.ldx, tokens, a.K, to, p.ldx);
    a.x = to;
    a.ldx = p.ldx;
  }
  if (p.copy_w) {
    unsigned char* to = reinterpret_cast<unsigned char*>(ws + p.w);
    copy_rows_kernel<<<grid(outputs * p.ldw / 16), 256, 0, s>>>(a.w, a.ldw, outputs, a.K, to, p.ldw);
    a.w = to;
    a.ldw = p.ldw;
  }
  const bool bytes = e8m0 && !exact;
  if (p.copy_sx) {
    void* to = ws + p.sx;
    copy_scales_kernel<<<grid(blocks * p.lds_x), 256, 0, s>>>(x_scale, xs_row, xs_block, tokens, blocks, to, p.lds_x, e8m0,
                                                              bytes);
    a.sx = to;
    a.sx_block = p.lds_x;
  }
  if (p.copy_sw) {
    void* to = ws + p.sw;
    copy_scales_kernel<<<grid(blocks * p.lds_w), 256, 0, s>>>(w_scale, ws_row, ws_block, w_rows, blocks, to, p.lds_w, e8m0,
                                                              bytes);
    a.sw = to;
    a.sw_block = p.lds_w;
  }
  const auto with = [&](auto x5, auto scaling, auto exactly) {
    constexpr bool X5 = decltype(x5)::value, EXACT = decltype(exactly)::value;
    constexpr Scaling SC = decltype(scaling)::value;
    if (p.shape == kStream) {
      run_stream<X5, SC, EXACT>(a, s);
    } else if constexpr (by_power(SC) && EXACT) {
      run_tiles<X5, by_tile(SC) ? kTile : kRow, true>(p.shape, a, s);  // (scales copied to floats)
    } else {
      run_tiles<X5, SC, EXACT>(p.shape, a, s);
    }
  };
  const auto with_scales = [&](auto x5, auto exactly) {
    if (e8m0 && w_tile)
      with(x5, std::integral_constant<Scaling, kPowerTile>{}, exactly);
    else if (e8m0)
      with(x5, std::integral_constant<Scaling, kPowerRow>{}, exactly);
    else if (w_tile)
      with(x5, std::integral_constant<Scaling, kTile>{}, exactly);
    else
      with(x5, std::integral_constant<Scaling, kRow>{}, exactly);
  };
  const auto with_x = [&](auto exactly) {
    if (x_dtype == HCG_E5M2)
      with_scales(std::true_type{}, exactly);
    else
      with_scales(std::false_type{}, exactly);
  };
  if (exact)
    with_x(std::true_type{});
  else
    with_x(std::false_type{});
  if (p.splits > 1) {
    const dim3 all = grid(tokens * p.ld_part / 4);
    switch (out_dtype) {
      case HCG_F16:
        join_kernel<<<all, 256, 0, s>>>(a.part, p.ld_part, p.splits, tokens, a.V, static_cast<_Float16*>(y), ldy);
        break;
      case HCG_BF16:
        join_kernel<<<all, 256, 0, s>>>(a.part, p.ld_part, p.splits, tokens, a.V, static_cast<__bf16*>(y), ldy);
        break;
      default: join_kernel<<<all, 256, 0, s>>>(a.part, p.ld_part, p.splits, tokens, a.V, static_cast<float*>(y), ldy);
    }
  }
  HCG_LM_HIP_CHECK(hipGetLastError());
  return HCG_OK;
}

}  // extern "C"
