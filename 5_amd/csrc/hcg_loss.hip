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
// maximum (so within 2^-12 of the value wherever they matter).  One pass over
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

constexpr int64_t kPieceBytes = (int64_t)1 << 30;
constexpr int64_t kMaxTokens = (int64_t)1 << 26;
constexpr int64_t kMaxExtent = 4000000;  // of vocabulary and width: a tile's offsets stay in 31 bits
// f16 probabilities are held times 2^12 (a uniform one over a vocabulary past
// 2^14 would be subnormal), undone in the products' float32 factor.
constexpr float kF16Scale = 4096.f;

// ---------------------------------------------------------------------------
// Packing
// ---------------------------------------------------------------------------

struct PackArgs {
  const void* targets;
  int64_t ignore, vocab;
  int tokens, mean;
  float grad_scale;
  int* slot;    // per token: its place among those that count, or -1
  int* token;   // per place: the token
  int* target;  // per place: its target, -1 outside the vocabulary
  int* count;
  float* scale;  // [0]: the gradient's factor, [1]: the loss's
  float* loss;   // per token, zeroed where ignored (or null)
  float* lse;
};

// One workgroup; each thread a contiguous run of tokens.
template <class I>
__global__ __launch_bounds__(1024) void pack_kernel(PackArgs g) {
  __shared__ int waves[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int per = (g.tokens + 1023) / 1024;
  const int from = min(tid * per, g.tokens), to = min(from + per, g.tokens);
  const I* targets = static_cast<const I*>(g.targets);
  int mine = 0;
  for (int t = from; t < to; ++t) mine += (int64_t)targets[t] != g.ignore;
  int sum = mine;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const int up = __shfl_up(sum, m);
    if (lane >= m) sum += up;
  }
  if (lane == 63) waves[wave] = sum;
  __syncthreads();
  int place = sum - mine, total = 0;
#pragma unroll
  for (int w = 0; w < 16; ++w) {
    if (w < wave) place += waves[w];
    total += waves[w];
  }
  for (int t = from; t < to; ++t) {
    const int64_t y = (int64_t)targets[t];
    if (y == g.ignore) {
      g.slot[t] = -1;
      if (g.loss) g.loss[t] = 0.f;
      if (g.lse) g.lse[t] = 0.f;
    } else {
      g.slot[t] = place;
      g.token[place] = t;
      g.target[place] = y >= 0 && y < g.vocab ? (int)y : -1;
      ++place;
    }
  }
  if (tid == 0) {
    *g.count = total;
    const float share = g.mean ? 1.f / (float)max(total, 1) : 1.f;
    g.scale[0] = g.grad_scale * share;
    g.scale[1] = share;
  }
}

// Rows of 16-bit elements into rows of `ldo` (a multiple of 8) elements, zeros
// past the width.  With `slot`, row t goes to place slot[t], or (-1) leaves
// zeros in row t of dx.
struct CopyArgs {
  const uint16_t* src;
  int64_t lds;
  uint16_t* dst;
  int64_t ldo;
  int rows, width, vecs;
  const int* slot;
  uint16_t* dx;  // or null
  int64_t lddx;
};

__global__ __launch_bounds__(256) void copy_rows_kernel(CopyArgs g) {
  const int64_t total = (int64_t)g.rows * g.vecs;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / g.vecs;
    const int c = (int)(i - row * g.vecs) * 8;
    const int64_t to = g.slot ? g.slot[row] : row;
    typedef _Float16 h;
    if (to >= 0) {
      const raw4 v = hcg::load_raw(reinterpret_cast<const h*>(g.src + row * g.lds + c), g.width - c);
      *reinterpret_cast<raw4*>(g.dst + to * g.ldo + c) = v;
    } else if (g.dx) {
      hcg::store_raw(reinterpret_cast<h*>(g.dx + row * g.lddx + c), raw4{0, 0, 0, 0}, g.width - c);
    }
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
  float scale;
};

// One row by one workgroup: lse from the blocks' statistics, the loss, and
// (GRAD) the probabilities in place of the exponentials.
template <int DT, bool GRAD>
__global__ __launch_bounds__(256) void softmax_kernel(SoftmaxArgs g) {
  constexpr float kLog2e = 1.44269504088896341f;
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
    sum += s.y * __builtin_amdgcn_exp2f((s.x == -__builtin_inff() ? -1e30f : s.x - ref) * kLog2e);
  }
  sum = hcg::wave_sum(sum);
  if (lane == 0) slots[1][wave] = sum;
  __syncthreads();
  sum = (slots[1][0] + slots[1][1]) + (slots[1][2] + slots[1][3]);
  const float lse = ref + logf(sum);
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
      const float f = rest * __builtin_amdgcn_exp2f((m == -__builtin_inff() ? -1e30f : m - ref) * kLog2e);
      float v[8];
      hcg::unpack<_Float16>(*reinterpret_cast<const raw4*>(row + c), v);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = v[e] * f - (c + e == target ? scale : 0.f);
      *reinterpret_cast<raw4*>(row + c) = hcg::pack<typename ElemOf<DT>::type>(v);
    }
  }
}

// The loss over all places, in one order.
__global__ __launch_bounds__(1024) void loss_sum_kernel(const float* loss, const int* count, const float* scale,
                                                        float* out) {
  __shared__ float waves[16];
  float sum = 0.f;
  for (int n = threadIdx.x; n < *count; n += 1024) sum += loss[n];
  sum = hcg::wave_sum(sum);
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = 0.f;
    for (int w = 0; w < 16; ++w) sum += waves[w];
    *out = sum * scale[1];
  }
}

// Rows of dx from the K splits' sums.
struct JoinArgs {
  const float* part;  // [splits][rows][ld]
  int64_t ld, stride;
  int splits, width, vecs;
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
  const int n = blockIdx.x;
  if (n >= *g.count - g.count0) return;
  const float f = *g.scale * g.post;
  typedef typename ElemOf<DT>::type T;
  T* row = reinterpret_cast<T*>(g.dx) + (int64_t)g.token[n] * g.lddx;
  for (int i = blockIdx.y * 256 + threadIdx.x; i < g.vecs; i += gridDim.y * 256) {
    const float* p = g.part + (int64_t)n * g.ld + i * 8;  // (rows are padded to 8)
    float sum[8] = {};
    for (int s = 0; s < g.splits; ++s) {
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] += p[s * g.stride + e];
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

// Tile shapes of head_kernel: rows of M and N, waves over them, LDS stages.
enum Shape { kLarge, kMedium, kFew };
struct ShapeInfo {
  int tm, tn, wm;
};
constexpr ShapeInfo kShapes[] = {{256, 256, 2}, {128, 128, 2}, {128, 32, 4}};

// The whole chip is 256 CUs with one workgroup each.
constexpr int kCus = 256;

int64_t tiles(Shape s, int64_t m, int64_t n) { return ceil_div(m, kShapes[s].tm) * ceil_div(n, kShapes[s].tn); }

Shape pick_shape(int64_t m, int64_t n, bool few) {
  if (few && n <= 32) return kFew;
  return tiles(kLarge, m, n) >= kCus / 2 ? kLarge : kMedium;
}

struct Plan {
  int64_t tokens, vocab, width;
  bool grad, copy_weight;
  int64_t ldx, lde;    // padded rows of X and of the probabilities
  int64_t piece;       // tokens per piece
  int pieces;
  Shape logits, dx, dw;
  int splits, kchunk;  // of dx
  int64_t blocks;      // statistics per token
  // Offsets into the workspace.
  int64_t slot, token, target, count, scale, rows, weight, stats, hit, loss, exps, part, sums, total;
};

Plan make_plan(int64_t tokens, int64_t vocab, int64_t width, bool copy_weight, bool grad) {
  Plan p{};
  p.tokens = tokens;
  p.vocab = vocab;
  p.width = width;
  p.grad = grad;
  p.copy_weight = copy_weight;
  p.ldx = round_up(width, 8);
  p.lde = round_up(vocab, 8);
  p.piece = tokens;
  if (grad) p.piece = std::min(tokens, std::max<int64_t>(256, kPieceBytes / (p.lde * 2) / 256 * 256));
  p.pieces = (int)ceil_div(tokens, p.piece);
  p.logits = pick_shape(vocab, p.piece, true);
  p.blocks = ceil_div(vocab, kShapes[p.logits].tm) * kShapes[p.logits].wm;
  p.splits = 1;
  if (grad) {
    p.dx = pick_shape(width, p.piece, true);
    p.dw = pick_shape(width, vocab, false);
    const int64_t t = tiles(p.dx, width, p.piece);
    if (t < kCus) p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(kCus / t, 32), vocab / 512));
    p.kchunk = (int)round_up(ceil_div(vocab, p.splits), head::kStep);
    p.splits = (int)ceil_div(vocab, p.kchunk);
  }
  int64_t at = 0;
  const auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += round_up(bytes, 256);
    return here;
  };
  p.slot = take(tokens * 4);
  p.token = take(tokens * 4);
  p.target = take(tokens * 4);
  p.count = take(4);
  p.scale = take(8);
  p.rows = take(tokens * p.ldx * 2);
  p.weight = take(copy_weight ? vocab * p.ldx * 2 : 0);
  p.stats = take(p.piece * p.blocks * 8);
  p.hit = take(p.piece * 4);
  if (grad) {
    p.loss = take(tokens * 4);
    p.exps = take(p.piece * p.lde * 2);
    p.part = take(p.splits > 1 ? p.splits * p.piece * p.ldx * 4 : 0);
    p.sums = take(p.pieces > 1 ? vocab * width * 4 : 0);
  }
  p.total = at;
  return p;
}

bool weight_in_place(const void* w, int64_t ldw, int64_t vocab, int64_t width) {
  return (reinterpret_cast<uintptr_t>(w) & 15) == 0 && width % 8 == 0 && (vocab == 1 || ldw % 8 == 0) &&
         ldw <= kMaxExtent;
}

template <int DT, int EPI, bool AKC, bool BKC, bool COUNT_K>
void launch_head(Shape shape, const head::Args& a, int64_t wgs, hipStream_t s) {
  const dim3 grid((unsigned)wgs);
  if (shape == kLarge) {
    head::head_kernel<DT, 256, 256, 2, 4, 2, AKC, BKC, EPI, COUNT_K><<<grid, 512, 0, s>>>(a);
  } else if (shape == kMedium) {
    head::head_kernel<DT, 128, 128, 2, 4, 4, AKC, BKC, EPI, COUNT_K><<<grid, 512, 0, s>>>(a);
  } else if constexpr (BKC) {
    head::head_kernel<DT, 128, 32, 4, 1, 4, AKC, BKC, EPI, COUNT_K><<<grid, 256, 0, s>>>(a);
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
  int* token = static_cast<int*>(at(p.token));
  int* target = static_cast<int*>(at(p.target));
  int* count = static_cast<int*>(at(p.count));
  float* scale = static_cast<float*>(at(p.scale));
  uint16_t* rows = static_cast<uint16_t*>(at(p.rows));
  const int T = (int)p.tokens, V = (int)p.vocab, D = (int)p.width;

  PackArgs pk{c.targets, c.ignore, p.vocab, T, c.mean, c.grad_scale, static_cast<int*>(at(p.slot)), token, target,
              count, scale, p.grad ? nullptr : c.loss, p.grad ? nullptr : c.lse};
  if (c.id_bytes == 8)
    pack_kernel<int64_t><<<1, 1024, 0, s>>>(pk);
  else
    pack_kernel<int32_t><<<1, 1024, 0, s>>>(pk);
  const auto copy = [&](const CopyArgs& a) {
    const int64_t wgs = std::min<int64_t>(ceil_div((int64_t)a.rows * a.vecs, 256), 16384);
    copy_rows_kernel<<<dim3((unsigned)wgs), 256, 0, s>>>(a);
  };
  copy(CopyArgs{static_cast<const uint16_t*>(c.x), c.ldx, rows, p.ldx, T, D, (int)(p.ldx / 8),
                static_cast<const int*>(at(p.slot)), static_cast<uint16_t*>(c.dx), c.lddx});
  const uint16_t* weight = static_cast<const uint16_t*>(c.weight);
  int64_t ldw = p.vocab == 1 ? p.ldx : c.ldw;
  if (p.copy_weight) {
    copy(CopyArgs{weight, c.ldw, static_cast<uint16_t*>(at(p.weight)), p.ldx, V, D, (int)(p.ldx / 8), nullptr,
                  nullptr, 0});
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
    a.splits = 1;
    a.kchunk = a.K;
    a.tiles_m = (int)ceil_div(V, kShapes[p.logits].tm);
    a.stats = static_cast<f32x2*>(at(p.stats));
    a.ld_stats = p.blocks;
    a.target = target + t0;
    a.hit = static_cast<float*>(at(p.hit));
    a.out = p.grad ? at(p.exps) : nullptr;
    a.ldo = p.lde;
    const int64_t wgs = tiles(p.logits, V, n);
    if (p.grad)
      launch_head<DT, head::kExp, true, true, false>(p.logits, a, wgs, s);
    else
      launch_head<DT, head::kStats, true, true, false>(p.logits, a, wgs, s);

    SoftmaxArgs sm{a.stats, p.blocks, (int)p.blocks, kShapes[p.logits].tm / kShapes[p.logits].wm, a.hit, a.target,
                   count, (int)t0, p.grad ? nullptr : token + t0, p.grad ? static_cast<float*>(at(p.loss)) + t0 : c.loss,
                   p.grad ? nullptr : c.lse, static_cast<uint16_t*>(a.out), p.lde, V, 1.f};
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
    d.splits = p.splits;
    d.kchunk = p.kchunk;
    d.tiles_m = (int)ceil_div(D, kShapes[p.dx].tm);
    d.scale = scale;
    d.post = post;
    const int64_t dx_wgs = tiles(p.dx, D, n) * p.splits;
    if (p.splits == 1) {
      d.out = c.dx;
      d.ldo = c.lddx;
      d.row_of = token + t0;
      launch_head<DT, head::kRound, false, true, false>(p.dx, d, dx_wgs, s);
    } else {
      d.out = at(p.part);
      d.ldo = p.ldx;
      d.split_stride = p.piece * p.ldx;
      launch_head<DT, head::kPartial, false, true, false>(p.dx, d, dx_wgs, s);
      const JoinArgs j{static_cast<const float*>(d.out), p.ldx, d.split_stride, p.splits, D, (int)(p.ldx / 8), count,
                       (int)t0, token + t0, scale, post, static_cast<uint16_t*>(c.dx), c.lddx};
      join_kernel<DT><<<dim3((unsigned)n, (unsigned)ceil_div(p.ldx / 8, 256)), 256, 0, s>>>(j);
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
    w.splits = 1;
    w.kchunk = n;
    w.tiles_m = (int)ceil_div(D, kShapes[p.dw].tm);
    w.scale = scale;
    w.post = post;
    w.add = i > 0 ? sums : nullptr;
    const int64_t dw_wgs = tiles(p.dw, D, V);
    if (i + 1 == p.pieces) {
      w.out = c.dw;
      w.ldo = c.lddw;
      launch_head<DT, head::kRound, false, false, true>(p.dw, w, dw_wgs, s);
    } else {
      w.out = sums;
      w.ldo = D;
      launch_head<DT, head::kPartial, false, false, true>(p.dw, w, dw_wgs, s);
    }
  }
  if (p.grad)
    loss_sum_kernel<<<1, 1024, 0, s>>>(static_cast<const float*>(at(p.loss)), count, scale, c.loss);
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
                     hcg::elem_aligned(c.dw, 2) && hcg::elem_aligned(c.targets, c.id_bytes),
                 "rows and targets must be aligned to their elements");
  if (tokens == 0 || vocab == 0 || width == 0) return HCG_OK;
  *plan = make_plan(tokens, vocab, width, !weight_in_place(c.weight, c.ldw, vocab, width), grad);
  HCG_LM_REQUIRE(tiles(plan->logits, vocab, plan->piece) < ((int64_t)1 << 31) &&
                     tiles(plan->dw, width, vocab) < ((int64_t)1 << 31) &&
                     tiles(plan->dx, width, plan->piece) * std::max(plan->splits, 1) < ((int64_t)1 << 31),
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
