// hcg_loss.hip -- softmax cross entropy of a linear head, and its gradient
// (include/hcg_lm.h).
//
//   l[t][v] = x_t . w_v,  lse_t = log sum_v exp l[t][v],  loss_t = lse_t - l[t][y_t]
//   g[t][v] = c (exp(l[t][v] - lse_t) - [v = y_t]),  dx = g w,  dw = g^T x
// with c = grad_scale, over the number of tokens that count for a mean.
//
// The tokens that count are packed first (their number stays on the device),
// so that ignored ones cost no product and may hold anything.  The product x
// w^T keeps its logits in accumulators: it leaves, per token and block of a
// wave's vocabulary rows, the maximum and the sum of exp(l - maximum), and for
// the gradient the exponentials themselves as f16, relative to their block's
// maximum (within 2^-11 of the value, or 2^-40 of that maximum).  One pass over
// those makes the row's lse and the probabilities (minus the one-hot) in the
// operands' type, from which dx and dw are two more products: three in all,
// where recomputing the logits would take four.  Exponentials and
// probabilities are held for kPieceBytes' worth of tokens at a time.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "hcg_head.h"
#include "hcg_vec.h"

namespace {

using hcg::ElemOf;
using hcg::raw4;
namespace head = hcg::head;
typedef head::f32x2 f32x2;

// (16-bit values, without the rows' padding; at least 256 tokens, however large the
// vocabulary)
constexpr int64_t kPieceBytes = (int64_t)1 << 30;
// ... and no more than so many tokens, whose launches stay below 2^32 threads
// (a loss alone holds no probabilities, and its pieces kPieceLogits logits).
constexpr int64_t kPieceTokens = (int64_t)1 << 22, kPieceLogits = (int64_t)1 << 32;
constexpr int64_t kMaxTokens = (int64_t)1 << 26;
constexpr int64_t kMaxExtent = 4000000;  // of vocabulary and width: a tile's offsets stay in 31 bits
// f16 probabilities are held times 2^15 (a uniform one over a vocabulary past
// 2^14 would be subnormal; so they are normal down to 2^-29, and held to 2^-40
// below), undone in the products' float32 factor.
constexpr float kF16Scale = 32768.f;

// ---------------------------------------------------------------------------
// Packing
// ---------------------------------------------------------------------------

struct PackArgs {
  const void* targets;
  int64_t ignore, vocab;
  int tokens, per_wg, mean;
  float grad_scale;
  int* token;   // per place among those that count: the token
  int* target;  // per place: its target, -1 outside the vocabulary
  int* count;
  const int* counts;  // how many count among each kCountRun tokens, where there are more (or null)
  float* scale;  // [0]: the gradient's factor, [1]: the loss's
  float* loss;   // per token, zeroed where ignored (or null)
  float* lse;
  // The rows: x to its place, zeros past the width; zeros in dx where ignored.
  const uint16_t* x;
  int64_t ldx;
  uint16_t* rows;
  int64_t ldr;
  int width, vecs;
  uint16_t* dx;  // or null
  int64_t lddx;
  unsigned* counters;  // cleared for the dx product
  int num_counters;
};

constexpr int kPackThreads = 256;
constexpr int kPackRun = 128;  // tokens per workgroup at most: their places are in LDS

// Past so many tokens, a launch counts them by runs of that many first.  us of
// hcg_linear_cross_entropy over 64 x 16, counted first / not: 98304 tokens 159 /
// 181, 262144 316 / 468, 1048576 1092 / 4734.
constexpr int kCountRun = 1 << 16;
constexpr int kCountThreads = 1024;
template <class I>
__global__ __launch_bounds__(kCountThreads) void count_kernel(const I* targets, int tokens, int64_t ignore,
                                                              int* counts) {
  __shared__ int waves[kCountThreads / 64];
  const int from = blockIdx.x * kCountRun, to = min(from + kCountRun, tokens);
  int sum = 0;
#pragma unroll 8
  for (int t = from + threadIdx.x; t < to; t += kCountThreads) sum += (int64_t)targets[t] != ignore;
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) sum += __shfl_xor(sum, m);
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kCountThreads / 64; ++w) sum += waves[w];
    counts[blockIdx.x] = sum;
  }
}

// A workgroup packs a run of tokens (8192 x 4096 bf16: 29 us for 134 MB, read and
// written, 4.6 TB/s).  It counts the tokens before its run
// itself, from the L2 (64 KB of targets at 8192 tokens), so that packing is one
// launch without anything to wait for.
template <class I>
__global__ __launch_bounds__(kPackThreads) void pack_kernel(PackArgs g) {
  __shared__ int waves[kPackThreads / 64];
  __shared__ int slot[kPackRun];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int from = blockIdx.x * g.per_wg, n = min(g.per_wg, g.tokens - from);
  const I* targets = static_cast<const I*>(g.targets);
  for (int i = blockIdx.x * kPackThreads + tid; i < g.num_counters; i += gridDim.x * kPackThreads)
    g.counters[i * hcg::kSplitCounterStride] = 0;
  int before = 0, counted = 0;
  if (g.counts) {
    counted = from / kCountRun * kCountRun;
    for (int i = tid; i < from / kCountRun; i += kPackThreads) before += g.counts[i];
  }
  for (int t0 = counted + tid; t0 < from; t0 += kPackThreads * 8) {
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int t = t0 + u * kPackThreads;
      before += t < from && (int64_t)targets[t] != g.ignore;
    }
  }
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) before += __shfl_xor(before, m);
  if (lane == 0) waves[wave] = before;
  __syncthreads();
  int place = 0;
#pragma unroll
  for (int w = 0; w < kPackThreads / 64; ++w) place += waves[w];
  // Every wave places the run; the first one writes it down.
  for (int j0 = 0; j0 < n; j0 += 64) {
    const int j = j0 + lane, t = from + j;
    const int64_t y = j < n ? (int64_t)targets[t] : g.ignore;
    const uint64_t counts = __ballot(y != g.ignore);
    if (wave == 0 && j < n) {
      const int at = place + __popcll(counts & (((uint64_t)1 << lane) - 1));
      slot[j] = y == g.ignore ? -1 : at;
      if (y == g.ignore) {
        if (g.loss) g.loss[t] = 0.f;
        if (g.lse) g.lse[t] = 0.f;
      } else {
        g.token[at] = t;
        g.target[at] = y >= 0 && y < g.vocab ? (int)y : -1;
      }
    }
    place += __popcll(counts);
  }
  if (tid == 0 && from + n == g.tokens) {
    *g.count = place;
    const float share = g.mean ? 1.f / (float)max(place, 1) : 1.f;
    g.scale[0] = g.grad_scale * share;
    g.scale[1] = share;
  }
  __syncthreads();
  typedef _Float16 h;
  const int total = n * g.vecs;
  constexpr int kPer = 8;  // loads in flight
  for (int i0 = tid; i0 < total; i0 += kPackThreads * kPer) {
    raw4 v[kPer];
    int row[kPer], col[kPer], to[kPer];
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      const int i = i0 + u * kPackThreads;
      row[u] = i / g.vecs;
      col[u] = (i - row[u] * g.vecs) * 8;
      to[u] = i < total ? slot[row[u]] : -2;
      v[u] = raw4{0, 0, 0, 0};
      if (to[u] >= 0)
        v[u] = hcg::load_raw(reinterpret_cast<const h*>(g.x + (int64_t)(from + row[u]) * g.ldx + col[u]),
                             g.width - col[u]);
    }
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      if (to[u] >= 0)
        *reinterpret_cast<raw4*>(g.rows + (int64_t)to[u] * g.ldr + col[u]) = v[u];
      else if (to[u] == -1 && g.dx)
        hcg::store_raw(reinterpret_cast<h*>(g.dx + (int64_t)(from + row[u]) * g.lddx + col[u]), v[u],
                       g.width - col[u]);
    }
  }
}

// Rows of 16-bit elements into rows of `ldo` (a multiple of 8) elements, zeros
// past the width, for weights whose rows are not 16-byte aligned: the products
// read them many times, by 16-byte DMA.  50021 x 1027: 42 us (4.9 TB/s).
struct CopyArgs {
  const uint16_t* src;
  int64_t lds;
  uint16_t* dst;
  int64_t ldo;
  int rows, width, vecs;
};

__global__ __launch_bounds__(256) void copy_rows_kernel(CopyArgs g) {
  const int64_t total = (int64_t)g.rows * g.vecs;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / g.vecs;
    const int c = (int)(i - row * g.vecs) * 8;
    typedef _Float16 h;
    *reinterpret_cast<raw4*>(g.dst + row * g.ldo + c) =
        hcg::load_raw(reinterpret_cast<const h*>(g.src + row * g.lds + c), g.width - c);
  }
}

// ---------------------------------------------------------------------------
// Softmax
// ---------------------------------------------------------------------------

struct SoftmaxArgs {
  const f32x2* stats;
  int64_t ld_stats;
  int blocks, block;  // statistics per row, and the vocabulary rows each covers
  const float* hit;
  const int* target;
  const int* count;
  int count0;
  // The losses, by place, or by token through `token`.
  const int* token;
  float* loss;
  float* lse;
  uint16_t* e;  // exponentials in, probabilities out
  int64_t lde;
  int vocab;
};

// One row by one workgroup: lse from the blocks' statistics, the loss, and
// (GRAD) the probabilities in place of the exponentials.  With block maxima m_b
// and sums s_b, lse = ref + log2 sum_b s_b 2^(m_b - ref) in powers of two, and a
// probability is its exponential times 2^(m_b - ref) / (sum exp_factor): one
// multiply-add per element.  Bound by HBM, 2 bytes read and written per
// probability: 8192 x 65536 447 us (4.8 TB/s), 8192 x 32768 215 (5.0).
template <int DT, bool GRAD>
__global__ __launch_bounds__(256) void softmax_kernel(SoftmaxArgs g) {
  constexpr double kLn2 = 0.693147180559945309;
  __shared__ float slots[2][4];
  const int n = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (n >= *g.count - g.count0) return;
  const f32x2* stats = g.stats + (int64_t)n * g.ld_stats;
  float top = -__builtin_inff();
  for (int j = tid; j < g.blocks; j += 256) top = fmaxf(top, stats[j].x);
  top = hcg::wave_max(top);
  if (lane == 0) slots[0][wave] = top;
  __syncthreads();
  top = fmaxf(fmaxf(slots[0][0], slots[0][1]), fmaxf(slots[0][2], slots[0][3]));
  const float ref = top == -__builtin_inff() ? 0.f : top;
  float sum = 0.f;
  for (int j = tid; j < g.blocks; j += 256) {
    const f32x2 s = stats[j];
    // (a block of -inf alone has sum 0, a NaN sum stays)
    sum += s.y * __builtin_amdgcn_exp2f(s.x == -__builtin_inff() ? -1e30f : s.x - ref);
  }
  sum = hcg::wave_sum(sum);
  if (lane == 0) slots[1][wave] = sum;
  __syncthreads();
  sum = (slots[1][0] + slots[1][1]) + (slots[1][2] + slots[1][3]);
  // (in doubles: one rounding of a value that may be some hundreds)
  const float lse = (float)(((double)ref + (double)log2f(sum)) * kLn2);
  const int target = g.target[n];
  if (tid == 0) {
    const int64_t to = g.token ? g.token[n] : n;
    g.loss[to] = target < 0 ? __builtin_nanf("") : lse - g.hit[n];
    if (g.lse) g.lse[to] = lse;
  }
  if constexpr (GRAD) {
    uint16_t* row = g.e + (int64_t)n * g.lde;
    const float scale = DT == HCG_F16 ? kF16Scale : 1.f;
    const float rest = scale / sum;
    for (int c = tid * 8; c < g.vocab; c += 256 * 8) {
      const float m = stats[c / g.block].x;
      const float down = 1.f / head::exp_factor(m);
      const float f = rest * __builtin_amdgcn_exp2f(m == -__builtin_inff() ? -1e30f : m - ref) * down;
      float v[8];
      hcg::unpack<_Float16>(*reinterpret_cast<const raw4*>(row + c), v);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = v[e] * f - (c + e == target ? scale : 0.f);
      *reinterpret_cast<raw4*>(row + c) = hcg::pack<typename ElemOf<DT>::type>(v);
    }
  }
}

// Rows of dx from the K splits' sums (where head_kernel split K in large tiles).
// The parts come from the L2s and the Infinity Cache: 1300 x 1027 in 8 parts 11
// us; a launch with nothing to add (few splits on the host's count of tokens, none
// on the device's) 3 to 5.
struct JoinArgs {
  const float* part;  // [splits][live tokens][ld]
  int64_t ld;
  int units, max_splits, tiles_m, tile_n, tokens, K;  // as head_kernel has them
  int width, vecs;
  const int* count;
  int count0;
  const int* token;
  const float* scale;
  float post;
  uint16_t* dx;
  int64_t lddx;
};

template <int DT>
__global__ __launch_bounds__(256) void join_kernel(JoinArgs g) {
  const int live = min(max(*g.count - g.count0, 0), g.tokens);
  int chunk;
  const int splits =
      head::splits_of(g.units, g.max_splits, g.tiles_m * ((live + g.tile_n - 1) / g.tile_n), g.K, &chunk);
  if (splits == 1) return;
  const float f = *g.scale * g.post;
  typedef typename ElemOf<DT>::type T;
  const int64_t total = (int64_t)live * g.vecs;
  for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < total; at += (int64_t)gridDim.x * 256) {
    const int n = (int)(at / g.vecs), i = (int)(at - (int64_t)n * g.vecs);
    T* row = reinterpret_cast<T*>(g.dx) + (int64_t)g.token[n] * g.lddx;
    const float* p = g.part + (int64_t)n * g.ld + i * 8;  // (rows are padded to 8)
    float sum[8] = {};
#pragma unroll 4
    for (int s = 0; s < splits; ++s) {
      const head::f32x4 a = *reinterpret_cast<const head::f32x4*>(p + (int64_t)s * live * g.ld);
      const head::f32x4 b = *reinterpret_cast<const head::f32x4*>(p + (int64_t)s * live * g.ld + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += a[e], sum[4 + e] += b[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[e] *= f;
    hcg::store_raw(row + i * 8, hcg::pack<T>(sum), g.width - i * 8);
  }
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------

int64_t round_up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Tile shapes of head_kernel: rows of M and N, waves over M in the softmax's
// product, and a model of its time in us: a tile's start and end, and one
// stage of K on an idle and on a busy chip, per round of workgroups
// (per_cu of which share a CU).  Fitted to 10 sizes with every shape and 1 to 8
// K splits: its choice is the fastest, or within 8% of it, at nine of them.  Both
// sides, us (a launch that adds up parts included): dx of 1300 x 50000 x 1032
// large in 8 parts 158, medium in 4 196; of 256 x 4096 x 512 large in 8 parts 28,
// few in 4 11; of 1000 x 30000 x 1000 large in 8 parts 88, medium in 4 77; logits
// of 128 x 6000 x 700 large 18, few 7; of 1024 x 32768 x 2048 large 121, medium
// 159; dw of 64 x 32768 x 4096 large 110, medium 80, small 127; of 4096 x 32768 x
// 512 113, 142, 188.
enum Shape { kLarge, kMedium, kSmall, kFew };
struct ShapeInfo {
  int tm, tn, wm, per_cu;
  double fixed, lo, hi;
};
constexpr ShapeInfo kShapes[] = {
    {256, 256, 2, 1, 10.0, 0.92, 1.5},
    {128, 128, 2, 2, 4.0, 0.55, 1.05},
    {128, 64, 4, 2, 3.2, 0.35, 0.78},
    {128, 32, 4, 2, 3.5, 0.28, 0.74}};  // (not dw: its rows of vocabulary are read 64 at a time)
constexpr int kNumShapes = 4;
constexpr int kCus = 256;
constexpr int kMaxSplits = 32;
constexpr int kMinKPerSplit = 256, kMinKPerFusedSplit = 128;

int64_t tiles(Shape s, int64_t m, int64_t n) { return ceil_div(m, kShapes[s].tm) * ceil_div(n, kShapes[s].tn); }

double cost_of(Shape s, int64_t m, int64_t n, int64_t k, int splits) {
  const ShapeInfo& t = kShapes[s];
  const int64_t units = tiles(s, m, n) * splits, room = kCus * t.per_cu, rest = units % room;
  const double stages = (double)ceil_div(ceil_div(k, splits), head::kStep);
  // Full rounds, and what is left: with one workgroup per CU a stage slows as the
  // chip fills, with two once CUs are shared.
  double us = (double)(units / room) * (t.fixed + stages * t.hi);
  if (rest) {
    const double busy = t.per_cu == 1 ? (double)rest / room : std::max(0.0, (double)(rest - kCus) / kCus);
    us += t.fixed + stages * (t.lo + (t.hi - t.lo) * busy);
  }
  if (splits > 1) {
    // The parts written and read, and a launch, or their reading by one CU.
    us += 2.0 * splits * m * n * 4 / 6.0e6;
    us += head::can_fuse(t.tm, t.tn) ? 1.0 + (splits - 1) * std::max(0.5, t.tm * t.tn * 4 / 4.5e4) : 4.0;
  }
  return us;
}

bool fuses(Shape s) { return head::can_fuse(kShapes[s].tm, kShapes[s].tn); }

enum ProductKind { kLogits, kDx, kDw };

// How a product of m x n over k runs: the shape with the least modelled time, and
// into how many parts K may be split (by the tile's last workgroup, or, dx in
// large tiles, by a launch).
struct Product {
  Shape shape;
  int units, max_splits;  // as head::Args has them
  int counters;           // tiles that may be split and summed by their last workgroup
  int64_t part_bytes;
  int64_t wgs(int64_t m, int64_t n) const {
    return std::max<int64_t>(tiles(shape, m, n), max_splits > 1 ? units : 0);
  }
};

Product pick_product(ProductKind kind, int64_t m, int64_t n, int64_t k) {
  Product best{};
  double best_cost = -1;
  for (int i = 0; i < kNumShapes; ++i) {
    const Shape s = (Shape)i;
    if (kind == kDw && s == kFew) continue;
    const int64_t most = fuses(s) ? std::min<int64_t>(hcg::kMaxSummedSplits, k / kMinKPerFusedSplit)
                         : kind == kDx ? std::min<int64_t>(kMaxSplits, k / kMinKPerSplit)
                                       : 1;
    for (int splits = 1; splits <= std::max<int64_t>(1, most); ++splits) {
      const double cost = cost_of(s, m, n, k, splits);
      if (best_cost >= 0 && cost >= best_cost) continue;
      best_cost = cost;
      best.shape = s;
      best.max_splits = (int)std::max<int64_t>(1, most);
      // (where fewer tokens count, the fewer tiles are split up to as many; more
      // than some rounds of workgroups gain nothing and would take scratch)
      best.units = (int)std::min<int64_t>(tiles(s, m, n) * splits, 8 * kCus);
    }
  }
  if (best.max_splits > 1) {
    const ShapeInfo& t = kShapes[best.shape];
    if (fuses(best.shape)) {
      // Whole tiles of at most `units` workgroups.
      best.counters = (int)std::min<int64_t>(best.units, tiles(best.shape, m, n));
      best.part_bytes = (int64_t)best.units * t.tm * t.tn * 4;
    } else {
      // K is split while the parts' tiles are at most `units`: no more rows
      // (padded to 8) than those tiles have, nor than max_splits times n.
      best.part_bytes = std::min(best.units / ceil_div(m, t.tm) * t.tn, best.max_splits * n) * round_up(m, 8) * 4;
    }
  }
  return best;
}

struct Plan {
  int64_t tokens, vocab, width;
  bool grad, copy_weight;
  int64_t ldx, lde;    // padded rows of X and of the probabilities
  int64_t piece;       // tokens per piece
  int pieces;
  Product logits, dx, dw;
  int counters;        // of the products (which run one after the other), the most
  int64_t blocks;      // statistics per token
  // Offsets into the workspace.
  int64_t token, target, count, counts, scale, rows, weight, stats, hit, loss, exps, part, counter, sums, total;
};

Plan make_plan(int64_t tokens, int64_t vocab, int64_t width, bool copy_weight, bool grad) {
  Plan p{};
  p.tokens = tokens;
  p.vocab = vocab;
  p.width = width;
  p.grad = grad;
  p.copy_weight = copy_weight;
  p.ldx = round_up(width, 8);
  // Whole 128-byte lines, and not a multiple of 1 KB: rows a power of two apart
  // put the pieces that are read at one k on a few HBM channels (dx of 4096 x
  // 32768 x 512 bf16 167 us, so 126).
  p.lde = round_up(vocab, 64) + (round_up(vocab, 64) % 512 ? 0 : 64);
  const int64_t fit = (grad ? kPieceBytes / 2 : kPieceLogits) / vocab / 256 * 256;
  p.piece = std::min({tokens, std::max<int64_t>(256, fit), kPieceTokens});
  p.pieces = (int)ceil_div(tokens, p.piece);
  p.logits = pick_product(kLogits, vocab, p.piece, width);
  p.blocks = ceil_div(vocab, kShapes[p.logits.shape].tm) * kShapes[p.logits.shape].wm;
  if (grad) {
    p.dx = pick_product(kDx, width, p.piece, vocab);
    p.dw = pick_product(kDw, width, vocab, p.piece);
  }
  p.counters = std::max({p.logits.counters, p.dx.counters, p.dw.counters});
  const int64_t part_bytes = std::max({p.logits.part_bytes, p.dx.part_bytes, p.dw.part_bytes});
  int64_t at = 0;
  const auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += round_up(bytes, 256);
    return here;
  };
  p.token = take(tokens * 4);
  p.target = take(tokens * 4);
  p.count = take(4);
  p.counts = take(tokens > kCountRun ? ceil_div(tokens, kCountRun) * 4 : 0);
  p.scale = take(8);
  p.rows = take(tokens * p.ldx * 2);
  p.weight = take(copy_weight ? vocab * p.ldx * 2 : 0);
  p.stats = take(p.piece * p.blocks * 8);
  p.hit = take(p.piece * 4);
  if (grad) {
    p.loss = take(tokens * 4);
    p.exps = take(p.piece * p.lde * 2);
    p.sums = take(p.pieces > 1 ? vocab * width * 4 : 0);
  }
  p.part = take(part_bytes);
  p.counter = take((int64_t)p.counters * hcg::kSplitCounterStride * 4);
  p.total = at;
  return p;
}

bool weight_in_place(const void* w, int64_t ldw, int64_t vocab, int64_t width) {
  return (reinterpret_cast<uintptr_t>(w) & 15) == 0 && width % 8 == 0 && (vocab == 1 || ldw % 8 == 0) &&
         ldw <= kMaxExtent;
}

// extra: workgroups beside the product's.
template <int DT, int EPI, bool AKC, bool BKC, bool COUNT_K>
void launch_head(const Product& p, head::Args a, hipStream_t s, int extra = 0) {
  const Shape shape = p.shape;
  a.tiles_m = (int)ceil_div(a.M, kShapes[shape].tm);
  a.units = p.units;
  a.max_splits = p.max_splits;
  a.part_bytes = (int)p.part_bytes;
  const dim3 grid((unsigned)(p.wgs(a.M, a.N) + extra));
  // Large tiles: four waves read the least LDS (128 KB per stage against 192 KB
  // by eight), and the board runs at its power limit; the softmax's epilogue is
  // faster by eight.  8192 x 65536 x 4096 bf16, us, four / eight waves: logits
  // 3464 / 3333, dx 2938 / 2964, dw 3082 / 3116.
  constexpr bool kSoftmax = EPI == head::kStats || EPI == head::kExp;
  if (shape == kLarge) {
    head::head_kernel<DT, 256, 256, 2, kSoftmax ? 4 : 2, 5, AKC, BKC, EPI, COUNT_K, false>
        <<<grid, kSoftmax ? 512 : 256, 0, s>>>(a);
  } else if (shape == kMedium) {
    // A ring of 5 units, 80 KB: two workgroups share a CU, and one computes while
    // the other starts or ends.  Eight units at one per CU / five, us: logits of
    // 4096 x 32768 x 512 233 / 201, dw of 64 x 32768 x 4096 127 / 80, dx of 1024 x
    // 32768 x 2048 156 / 151.
    head::head_kernel<DT, 128, 128, 2, 4, 5, AKC, BKC, EPI, COUNT_K, false><<<grid, 512, 0, s>>>(a);
  } else if (shape == kSmall) {
    // (one tile of tokens: bound by reading the weights)
    if (kSoftmax && a.N <= 64)
      head::head_kernel<DT, 128, 64, 4, 2, 6, AKC, BKC, EPI, COUNT_K, kSoftmax><<<grid, 512, 0, s>>>(a);
    else
      head::head_kernel<DT, 128, 64, 4, 2, 6, AKC, BKC, EPI, COUNT_K, false><<<grid, 512, 0, s>>>(a);
  } else if constexpr (BKC) {
    head::head_kernel<DT, 128, 32, 4, 1, 6, AKC, BKC, EPI, COUNT_K, kSoftmax><<<grid, 256, 0, s>>>(a);
  }
}

struct Call {
  const void* x;
  int64_t ldx;
  const void* weight;
  int64_t ldw;
  int id_bytes;
  const void* targets;
  int64_t ignore;
  int mean;
  float grad_scale;
  float* loss;
  float* lse;
  void* dx;
  int64_t lddx;
  void* dw;
  int64_t lddw;
  char* ws;
};

template <int DT>
int run_loss(const Plan& p, const Call& c, hipStream_t s) {
  const auto at = [&](int64_t offset) { return static_cast<void*>(c.ws + offset); };
  const int T = (int)p.tokens, V = (int)p.vocab, D = (int)p.width;
  int* token = static_cast<int*>(at(p.token));
  int* target = static_cast<int*>(at(p.target));
  int* count = static_cast<int*>(at(p.count));
  int* counts = T > kCountRun ? static_cast<int*>(at(p.counts)) : nullptr;
  float* scale = static_cast<float*>(at(p.scale));
  uint16_t* rows = static_cast<uint16_t*>(at(p.rows));

  // At most 1024 runs, four workgroups per CU, while a run fits.
  const int per_wg = (int)std::min<int64_t>(kPackRun, ceil_div(T, 1024));
  const PackArgs pk{c.targets,
                    c.ignore,
                    p.vocab,
                    T,
                    per_wg,
                    c.mean,
                    c.grad_scale,
                    token,
                    target,
                    count,
                    counts,
                    scale,
                    p.grad ? nullptr : c.loss,
                    p.grad ? nullptr : c.lse,
                    static_cast<const uint16_t*>(c.x),
                    c.ldx,
                    rows,
                    p.ldx,
                    D,
                    (int)(p.ldx / 8),
                    static_cast<uint16_t*>(c.dx),
                    c.lddx,
                    static_cast<unsigned*>(at(p.counter)),
                    p.counters};
  const dim3 runs((unsigned)ceil_div(T, per_wg));
  if (counts) {
    const dim3 grid((unsigned)ceil_div(T, kCountRun));
    if (c.id_bytes == 8)
      count_kernel<<<grid, kCountThreads, 0, s>>>(static_cast<const int64_t*>(c.targets), T, c.ignore, counts);
    else
      count_kernel<<<grid, kCountThreads, 0, s>>>(static_cast<const int32_t*>(c.targets), T, c.ignore, counts);
  }
  if (c.id_bytes == 8)
    pack_kernel<int64_t><<<runs, kPackThreads, 0, s>>>(pk);
  else
    pack_kernel<int32_t><<<runs, kPackThreads, 0, s>>>(pk);
  const uint16_t* weight = static_cast<const uint16_t*>(c.weight);
  int64_t ldw = p.vocab == 1 ? p.ldx : c.ldw;
  if (p.copy_weight) {
    const CopyArgs a{weight, c.ldw, static_cast<uint16_t*>(at(p.weight)), p.ldx, V, D, (int)(p.ldx / 8)};
    const int64_t wgs = std::min<int64_t>(ceil_div((int64_t)V * a.vecs, 256), 16384);
    copy_rows_kernel<<<dim3((unsigned)wgs), 256, 0, s>>>(a);
    weight = static_cast<const uint16_t*>(at(p.weight));
    ldw = p.ldx;
  }

  float* sums = p.pieces > 1 ? static_cast<float*>(at(p.sums)) : nullptr;
  for (int i = 0; i < p.pieces; ++i) {
    const int64_t t0 = (int64_t)i * p.piece;
    const int n = (int)std::min<int64_t>(p.piece, p.tokens - t0);
    const uint16_t* x = rows + t0 * p.ldx;
    // The logits' statistics (and exponentials).
    head::Args a{};
    a.A = weight;
    a.lda = ldw;
    a.B = x;
    a.ldb = p.ldx;
    a.M = V;
    a.N = n;
    a.K = (int)p.ldx;
    a.count = count;
    a.count0 = (int)t0;
    a.part = static_cast<float*>(at(p.part));
    a.counters = static_cast<unsigned*>(at(p.counter));
    a.stats = static_cast<f32x2*>(at(p.stats));
    a.ld_stats = p.blocks;
    a.target = target + t0;
    a.hit = static_cast<float*>(at(p.hit));
    a.out = p.grad ? at(p.exps) : nullptr;
    a.ldo = p.lde;
    if (p.grad)
      launch_head<DT, head::kExp, true, true, false>(p.logits, a, s);
    else
      launch_head<DT, head::kStats, true, true, false>(p.logits, a, s);

    SoftmaxArgs sm{a.stats, p.blocks, (int)p.blocks, kShapes[p.logits.shape].tm / kShapes[p.logits.shape].wm, a.hit, a.target,
                   count, (int)t0, p.grad ? nullptr : token + t0, p.grad ? static_cast<float*>(at(p.loss)) + t0 : c.loss,
                   p.grad ? nullptr : c.lse, static_cast<uint16_t*>(a.out), p.lde, V};
    if (!p.grad) {
      softmax_kernel<DT, false><<<dim3((unsigned)n), 256, 0, s>>>(sm);
      continue;
    }
    softmax_kernel<DT, true><<<dim3((unsigned)n), 256, 0, s>>>(sm);
    const uint16_t* probs = static_cast<const uint16_t*>(a.out);
    const float post = DT == HCG_F16 ? 1.f / kF16Scale : 1.f;

    head::Args d{};
    d.A = weight;
    d.lda = ldw;
    d.B = probs;
    d.ldb = p.lde;
    d.M = D;
    d.N = n;
    d.K = V;
    d.count = count;
    d.count0 = (int)t0;
    d.scale = scale;
    d.post = post;
    d.out = c.dx;
    d.ldo = c.lddx;
    d.row_of = token + t0;
    d.part = a.part;
    d.ld_part = p.ldx;
    d.counters = a.counters;
    launch_head<DT, head::kSplit, false, true, false>(p.dx, d, s);
    if (p.dx.max_splits > 1 && !fuses(p.dx.shape)) {
      const ShapeInfo& t = kShapes[p.dx.shape];
      const JoinArgs j{d.part,     p.ldx, p.dx.units, p.dx.max_splits,  (int)ceil_div(D, t.tm),
                       t.tn,       n,     V,          D,                (int)(p.ldx / 8),
                       count,      (int)t0, token + t0, scale,          post,
                       static_cast<uint16_t*>(c.dx), c.lddx};
      const int64_t wgs = std::min<int64_t>(ceil_div((int64_t)n * j.vecs, 256), 4 * kCus);
      join_kernel<DT><<<dim3((unsigned)wgs), 256, 0, s>>>(j);
    }

    head::Args w{};
    w.A = x;
    w.lda = p.ldx;
    w.B = probs;
    w.ldb = p.lde;
    w.M = D;
    w.N = V;
    w.K = n;
    w.count = count;
    w.count0 = (int)t0;
    w.counters = a.counters;
    w.part = a.part;
    w.scale = scale;
    w.post = post;
    w.add = i > 0 ? sums : nullptr;
    if (i + 1 == p.pieces) {
      w.out = c.dw;
      w.ldo = c.lddw;
      w.loss = static_cast<const float*>(at(p.loss));
      w.loss_scale = scale + 1;
      w.loss_out = c.loss;
      launch_head<DT, head::kRound, false, false, true>(p.dw, w, s, 1);
    } else {
      w.part = sums;
      w.ld_part = D;
      launch_head<DT, head::kPartial, false, false, true>(p.dw, w, s);
    }
  }
  HCG_LM_HIP_CHECK(hipGetLastError());
  return HCG_OK;
}

int check_call(int dtype, const Call& c, int64_t tokens, int64_t vocab, int64_t width, bool grad, int64_t ws_bytes,
               Plan* plan) {
  HCG_LM_REQUIRE(dtype == HCG_F16 || dtype == HCG_BF16, "dtype %d is not HCG_F16 or HCG_BF16", dtype);
  HCG_LM_REQUIRE(c.id_bytes == 4 || c.id_bytes == 8, "targets are 4 or 8 bytes, not %d", c.id_bytes);
  HCG_LM_REQUIRE(tokens >= 0 && tokens < kMaxTokens && vocab >= 0 && vocab < kMaxExtent - 8 && width >= 0 &&
                     width < kMaxExtent - 8,
                 "%lld tokens, %lld rows of %lld elements are out of range", (long long)tokens, (long long)vocab,
                 (long long)width);
  HCG_LM_REQUIRE(vocab > 0 || tokens == 0, "a softmax over no vocabulary");
  HCG_LM_REQUIRE(width > 0 || tokens == 0, "hidden states without elements");
  HCG_LM_REQUIRE(c.loss || (!grad && tokens == 0), "null pointer");
  HCG_LM_REQUIRE(tokens == 0 || (c.x && c.weight && c.targets && (grad ? c.dx != nullptr : c.lse != nullptr)),
                 "null pointer");
  HCG_LM_REQUIRE(!grad || c.dw || vocab == 0 || width == 0, "null pointer");
  HCG_LM_REQUIRE((tokens <= 1 || (c.ldx >= width && (!grad || c.lddx >= width))) &&
                     (vocab <= 1 || (c.ldw >= width && (!grad || c.lddw >= width))),
                 "row stride below the width %lld", (long long)width);
  HCG_LM_REQUIRE(hcg::elem_aligned(c.x, 2) && hcg::elem_aligned(c.weight, 2) && hcg::elem_aligned(c.dx, 2) &&
                     hcg::elem_aligned(c.dw, 2) && hcg::elem_aligned(c.targets, c.id_bytes) &&
                     hcg::elem_aligned(c.loss, 4) && hcg::elem_aligned(c.lse, 4),
                 "rows, targets and losses must be aligned to their elements");
  if (tokens == 0 || vocab == 0 || width == 0) return HCG_OK;
  *plan = make_plan(tokens, vocab, width, !weight_in_place(c.weight, c.ldw, vocab, width), grad);
  const int64_t most = ((int64_t)1 << 31) - 1;
  HCG_LM_REQUIRE(plan->logits.wgs(vocab, plan->piece) < most &&
                     (!grad || (plan->dw.wgs(width, vocab) < most && plan->dx.wgs(width, plan->piece) < most)),
                 "too many tiles");
  HCG_LM_REQUIRE(c.ws && ws_bytes >= plan->total && hcg::elem_aligned(c.ws, 256),
                 "workspace of %lld bytes, %lld needed (256-byte aligned)", (long long)ws_bytes,
                 (long long)plan->total);
  return HCG_OK;
}

// What a call without tokens leaves: no loss, no gradient.
__global__ __launch_bounds__(256) void clear_kernel(uint16_t* dw, int64_t lddw, int64_t vocab, int64_t width,
                                                    float* loss) {
  const int64_t total = vocab * width;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256)
    dw[i / width * lddw + i % width] = 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) *loss = 0.f;
}

}  // namespace

extern "C" {

int64_t hcg_linear_cross_entropy_workspace(int64_t tokens, int64_t vocab, int64_t width, const void* weight,
                                           int64_t ldw, int grad) {
  if (tokens <= 0 || vocab <= 0 || width <= 0 || tokens >= kMaxTokens || vocab >= kMaxExtent - 8 ||
      width >= kMaxExtent - 8)
    return 0;
  return make_plan(tokens, vocab, width, !weight_in_place(weight, ldw, vocab, width), grad != 0).total;
}

int hcg_linear_cross_entropy_plan(int64_t tokens, int64_t vocab, int64_t width, int grad, int* plan) {
  HCG_LM_REQUIRE(plan, "null pointer");
  HCG_LM_REQUIRE(tokens > 0 && tokens < kMaxTokens && vocab > 0 && vocab < kMaxExtent - 8 && width > 0 &&
                     width < kMaxExtent - 8,
                 "%lld tokens, %lld rows of %lld elements are out of range", (long long)tokens, (long long)vocab,
                 (long long)width);
  const Plan p = make_plan(tokens, vocab, width, false, grad != 0);
  *plan++ = p.pieces;
  const auto put = [&](bool made, const Product& q, int64_t m, int64_t n) {
    *plan++ = made ? kShapes[q.shape].tm : 0;
    *plan++ = made ? kShapes[q.shape].tn : 0;
    *plan++ = made ? (int)std::max<int64_t>(1, std::min<int64_t>(q.max_splits, q.units / tiles(q.shape, m, n))) : 0;
  };
  put(true, p.logits, vocab, p.piece);
  put(grad != 0, p.dx, width, p.piece);
  put(grad != 0, p.dw, width, vocab);
  return HCG_OK;
}

int hcg_linear_cross_entropy(int dtype, const void* x, int64_t ldx, int64_t tokens, const void* weight, int64_t ldw,
                             int64_t vocab, int64_t width, int id_bytes, const void* targets, int64_t ignore_index,
                             float* loss, float* lse, void* workspace, int64_t workspace_bytes, void* stream) {
  const Call c{x,    ldx, weight,  ldw, id_bytes, targets, ignore_index, 0, 1.f,
               loss, lse, nullptr, 0,   nullptr,  0,       static_cast<char*>(workspace)};
  Plan plan{};
  const int rc = check_call(dtype, c, tokens, vocab, width, false, workspace_bytes, &plan);
  if (rc != HCG_OK || tokens == 0) return rc;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return dtype == HCG_F16 ? run_loss<HCG_F16>(plan, c, s) : run_loss<HCG_BF16>(plan, c, s);
}

int hcg_linear_cross_entropy_grad(int dtype, const void* x, int64_t ldx, int64_t tokens, const void* weight,
                                  int64_t ldw, int64_t vocab, int64_t width, int id_bytes, const void* targets,
                                  int64_t ignore_index, int mean, float grad_scale, float* loss, void* dx,
                                  int64_t lddx, void* dweight, int64_t lddw, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  const Call c{x,    ldx,     weight, ldw,  id_bytes, targets, ignore_index, mean, grad_scale,
               loss, nullptr, dx,     lddx, dweight,  lddw,    static_cast<char*>(workspace)};
  Plan plan{};
  const int rc = check_call(dtype, c, tokens, vocab, width, true, workspace_bytes, &plan);
  if (rc != HCG_OK) return rc;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (tokens == 0) {
    const int64_t wgs = std::min<int64_t>(std::max<int64_t>(1, ceil_div(vocab * width, 256)), 4096);
    clear_kernel<<<dim3((unsigned)wgs), 256, 0, s>>>(static_cast<uint16_t*>(dweight), vocab > 1 ? lddw : width, vocab, width, loss);
    HCG_LM_HIP_CHECK(hipGetLastError());
    return HCG_OK;
  }
  return dtype == HCG_F16 ? run_loss<HCG_F16>(plan, c, s) : run_loss<HCG_BF16>(plan, c, s);
}

}  // extern "C"
