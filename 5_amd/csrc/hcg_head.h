// hcg_head.h -- the products of a linear head's loss on gfx950 (device code).
//
// Three products share one kernel: with W (vocab x width), X (tokens x width)
// and the probabilities P (tokens x vocab),
//   logits^T = W X^T,  dX^T = W^T P^T,  dW^T = X^T P.
// Each is computed transposed, its "N" index (a token, or a vocabulary row)
// across the lanes of an accumulator and its "M" index in the registers
// (32x32x16 layout: register r of lane l is row 8 (r/4) + 4 (l/32) + r%4,
// column l%32).  So a lane holds runs of one output row: a softmax's maximum
// and sum over the vocabulary are reductions over registers plus one exchange
// between the wave's halves (across lanes they would take five exchanges per
// row and register), and outputs leave as 16-byte pieces of a row.
//
// TM x TN tiles by WM x WN waves; K advances 64 at a time.  A stage is two
// units, A's part and B's; a ring of UNITS LDS units is filled by
// global-to-LDS DMA.  One barrier per stage: past it every wave has read the
// stage before, whose two units are refilled UNITS units ahead.  Operand
// layouts, swizzles and fragment reads are those of hcg_wg8.h.
//
// Large products are bound by the board's power: MFMAs issue in 90% of the cycles
// of dX, 85% of dW's and 80% of the logits' at 1.6 GHz (8192 x 65536 x 4096 bf16:
// 2.9, 3.0 and 3.2 ms, 1.52, 1.46 and 1.37 PFLOP/s; the logits' epilogue takes the
// exponentials and writes 1 GB), without LDS bank conflicts.  The 5-unit ring of 160
// KB carries them: with four units (128 KB) 3355, 3544 and 3654 us on a card that
// takes 2938, 3082 and 3333 with five.
// Products of few tokens are bound by HBM (16 x 65536 x 4096: 90.5 us, 5.9 TB/s) or,
// the smallest, by a launch and a tile's start and end.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "hcg_lm.h"
#include "hcg_splitsum.h"
#include "hcg_tile.h"

namespace hcg {
namespace head {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int kStep = 64;  // K per stage

enum Epilogue {
  kStats,    // softmax statistics of the logits
  kExp,      // and exp(logit - block maximum) times exp_factor as f16
  kRound,    // scaled, rounded to DT, as rows of the output
  kPartial,  // float32, into scratch
  kSplit,    // kRound, or where K is split and the tile too large to fuse kPartial
};

// Tiles whose K splits the tile's last workgroup sums itself (hcg_splitsum.h);
// larger ones are added up by a launch of their own (dx of 256 x 4096 x 512 in
// 128x128 tiles and 8 parts: 21.7 us by the last workgroup, 14.6 with a launch; in
// 128x32 tiles and 4 parts 11 by the last one).
constexpr bool can_fuse(int tm, int tn) { return tm * tn <= 128 * 64; }

struct Args {
  const uint16_t* A;  // M side
  const uint16_t* B;  // N side
  int64_t lda, ldb;   // elements between rows as stored
  int M, N, K;
  // The live tokens, on the device: N (or, COUNT_K, K) is at most *count - count0.
  const int* count;
  int count0;
  int tiles_m;
  // kSplit, and tiles that can_fuse: K is split while there are fewer tiles (of
  // live tokens) than units, into at most max_splits parts.
  int units, max_splits;
  unsigned* counters;  // can_fuse: one per tile, kSplitCounterStride apart, all zero
  int part_bytes;
  // kRound: row n of the output is out + (row_of ? row_of[n] : n) * ldo;
  // kPartial: part + (split * N + n) * ld_part.
  void* out;
  int64_t ldo;
  float* part;
  int64_t ld_part;
  const int* row_of;
  const float* add;    // [N][M] floats added to the sums, or null
  const float* scale;  // kRound: the factor *scale * post
  float post;
  // kStats, kExp: per token n and block of TM / WM vocabulary rows its largest
  // logit times log2 e, c, and the sum of 2^(logit * log2 e - c), and the
  // target's logit.
  f32x2* stats;
  int64_t ld_stats;
  const int* target;
  float* hit;
  // kRound, where loss_out is not null: one workgroup more, which adds up the
  // losses of the live tokens.
  const float* loss;
  const float* loss_scale;
  float* loss_out;
};

template <int DT>
__device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (DT == HCG_F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                  0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
}

// What kExp multiplies the exponentials of a block with largest exponent `top`
// by: 2^15, so that f16 holds them to 11 bits down to 2^-29 of the largest, and
// to 2^-40 of it below.  Past 2^20 `top` is itself rounded by more than 2^-4 and
// the largest exponential is no longer close enough to 1 for that.
__device__ __forceinline__ float exp_factor(float top) { return fabsf(top) < 0x1p20f ? 0x1p15f : 1.f; }

template <int N>
__device__ __forceinline__ void wait_vm() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  __builtin_amdgcn_s_waitcnt(0x0f70 | (N & 15) | ((N >> 4) << 14));
}
__device__ __forceinline__ void wait_lgkm() { __builtin_amdgcn_s_waitcnt(0xc07f); }

// Each unit is an LDS object of its own, named at compile time, so that the
// compiler does not serialize a DMA into one with reads of another.
template <int BYTES, int S>
__device__ __forceinline__ unsigned char* ring_unit() {
  __shared__ __attribute__((aligned(1024))) unsigned char buf[BYTES];
  return buf;
}

// Two floats rounded to DT, packed.
template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (DT == HCG_F16)
    return __builtin_bit_cast(uint32_t, f16x2{(_Float16)a, (_Float16)b});
  else
    return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)a, (__bf16)b});
}

// The parts that K is split into, of *chunk (a multiple of kStep) each but the
// last.
__device__ __forceinline__ int splits_of(int units, int max_splits, int tiles, int K, int* chunk) {
  const int want = max(1, min(units / max(tiles, 1), max_splits));
  *chunk = ((K + want - 1) / want + kStep - 1) / kStep * kStep;
  return max(1, (K + *chunk - 1) / max(*chunk, 1));
}

// blockIdx -> (K split, tile): each XCD (id % 8) takes a contiguous run of
// units, within a split in groups of 4 tile rows, so that the workgroups
// sharing an L2 share operand rows (as hcg_wg8.h's unit_of).
__device__ __forceinline__ void unit_of(int tiles_m, int tiles_n, int splits, int wg, int& split, int& tm, int& tn) {
  const int nt = tiles_m * tiles_n, n = nt * splits;
  const int per = n >> 3, rem = n & 7, xcd = wg & 7, idx = wg >> 3;
  const int unit = xcd < rem ? xcd * (per + 1) + idx : rem * (per + 1) + (xcd - rem) * per + idx;
  split = unit / nt;
  const int logical = unit - split * nt;
  const int span = 4 * tiles_n;
  const int group = logical / span, first = group * 4;
  const int size = min(tiles_m - first, 4);
  const int in_group = logical - group * span;
  tm = first + in_group % size;
  tn = in_group / size;
}

// One operand's part of a stage, T rows of the output's M or N by kStep of K,
// loaded by NW waves.  KC: K-contiguous rows as stored (LDS rows of 64
// elements, one per output row, a fragment is one ds_read_b128).  Otherwise K
// rows of T contiguous output rows (LDS rows of T elements, one per k, a
// fragment is two transposing reads).  The 16-byte chunks of an LDS row are
// XOR-swizzled to cover all banks.
template <int T, bool KC, int NW>
struct Operand {
  static constexpr int kBytes = T * kStep * 2;
  static constexpr int kInst = kBytes / 1024 / NW;  // DMA instructions per wave per stage
  static constexpr int kRowBytes = KC ? kStep * 2 : T * 2;
  static constexpr int kChunks = kRowBytes / 16;
  static constexpr int kRowsPerInst = 64 / kChunks;
  static_assert(kInst >= 1 && kInst * NW * 1024 == kBytes, "a stage is whole DMA instructions of every wave");
  static_assert(KC || T >= 64, "swizzle");

  static __device__ __forceinline__ int swz(int row, int c) {
    if constexpr (KC) {
      return c ^ ((row >> 1) & 7);
    } else {
      const int m = row & 3;
      if constexpr (T == 64) return c ^ ((m >> 1) * 4);
      return c ^ ((m >> 1) * 10 + (m & 1) * 4);
    }
  }

  int off[kInst];  // byte offset of the lane's chunk from the stage's first element, or kOobOffset
  int key[kInst];  // the chunk's first k from the stage's first

  // extent: output rows from the tile's first on.
  __device__ __forceinline__ void init(int wave, int lane, int extent, int64_t ld) {
#pragma unroll
    for (int i = 0; i < kInst; ++i) {
      const int row = (wave * kInst + i) * kRowsPerInst + lane / kChunks;
      const int c = swz(row, lane % kChunks);
      const bool live = KC ? row < extent : c * 8 < extent;
      off[i] = live ? (row * (int)ld + c * 8) * 2 : kOobOffset;
      key[i] = KC ? c * 8 : row;
    }
  }

  // The stage whose first element is at p, `left` of K from there on (FULL: a
  // whole stage).  The resource starts at the stage, so offsets stay in 31
  // bits whatever the matrix's size; chunks out of range are redirected past
  // its extent and load zeros.
  // Instructions FROM to TO - 1 of the wave's.
  template <bool FULL, int FROM, int TO>
  __device__ __forceinline__ void issue(const uint16_t* p, unsigned char* st, int wave, int left) const {
    const __amdgpu_buffer_rsrc_t r = make_rsrc(p, 0x7fffffe0);
#pragma unroll
    for (int i = FROM; i < TO; ++i) {
      lds_void* dst = (lds_void*)(st + (wave * kInst + i) * 1024);
      if constexpr (FULL)
        dma16(r, dst, off[i]);
      else
        dma16(r, dst, dma_offset(key[i] < left, off[i]));
    }
  }

  int fa;
  int fb[2];
  __device__ __forceinline__ void frag_init(int lane, int first) {
    if constexpr (KC) {
      const int row = first + (lane & 31);
      fa = row * kRowBytes + swz(row, lane >> 5) * 16;
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int sl = lane & 15, grp = lane >> 4;
        const int krow = 8 * (grp >> 1) + 4 * h + (sl >> 2);
        const int col = first + 16 * (grp & 1) + 4 * (sl & 3);
        fb[h] = krow * kRowBytes + swz(krow, col >> 3) * 16 + (col & 7) * 2;
      }
    }
  }
  // Fragment of 32-row block b and 16-wide K step s.
  __device__ __forceinline__ u32x4 frag(const unsigned char* st, int b, int s) const {
    if constexpr (KC) {
      return *reinterpret_cast<const u32x4*>(st + (fa ^ (s * 32)) + b * 32 * kRowBytes);
    } else {
      const int x = s * 16 * kRowBytes;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) s16x4*)(st + (fb[0] ^ (b * 64)) + x));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) s16x4*)(st + (fb[1] ^ (b * 64)) + x));
      const uint64_t l = __builtin_bit_cast(uint64_t, lo), h = __builtin_bit_cast(uint64_t, hi);
      return u32x4{(uint32_t)l, (uint32_t)(l >> 32), (uint32_t)h, (uint32_t)(h >> 32)};
    }
  }
};

template <int I>
using Int = std::integral_constant<int, I>;

// A wave's 32 rows by 32 * MI columns of 16-bit results on their way out, in
// LDS: row r's 16-byte chunk c lies at chunk c ^ (r % the row's chunks), so that
// both the writes (a lane per row) and the reads (a row per group of lanes)
// cover all banks.
template <int MI>
struct RowStage {
  static constexpr int kChunks = 4 * MI;  // 16-byte chunks per row
  static constexpr int kBytes = 32 * kChunks * 16;
  static __device__ __forceinline__ int at(int row, int chunk) {
    return (row * kChunks + (chunk ^ (row & (kChunks - 1)))) * 16;
  }
  // value(r), r = 0 .. 15: the lane's accumulator registers of block mi, in
  // row lane % 32, columns 32 mi + 8 (r / 4) + 4 (lane / 32) + r % 4.  The
  // wave's halves exchange groups of four, so that each lane holds whole
  // chunks.
  template <int DT, class F>
  static __device__ __forceinline__ void put(unsigned char* st, int lane, int mi, F value) {
    const int row = lane & 31, half = lane >> 5;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      uint32_t w[2][2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t a = pack2<DT>(value(8 * p + 2 * i), value(8 * p + 2 * i + 1));
        const uint32_t b = pack2<DT>(value(8 * p + 4 + 2 * i), value(8 * p + 5 + 2 * i));
        const auto x = __builtin_amdgcn_permlane32_swap(a, b, false, false);
        w[0][i] = x[0];
        w[1][i] = x[1];
      }
      *reinterpret_cast<u32x4*>(st + at(row, 4 * mi + 2 * p + half)) = u32x4{w[0][0], w[0][1], w[1][0], w[1][1]};
    }
  }
  // The wave's rows as 16-byte stores, a row's chunks in neighbouring lanes.
  // base(row): the output row's element 0, or null; columns m0 ... below
  // `extent` (a chunk that reaches past it is cut, or, in padded scratch,
  // stored whole).
  template <bool CUT, class F>
  static __device__ __forceinline__ void store(const unsigned char* st, int lane, int m0, int extent, F base) {
    typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(2)));
    constexpr int kPer = 64 / kChunks;  // rows per instruction
    const int chunk = lane % kChunks, m = m0 + chunk * 8;
#pragma unroll
    for (int i = 0; i < 32 / kPer; ++i) {
      const int row = i * kPer + lane / kChunks;
      const u32x4 v = *reinterpret_cast<const u32x4*>(st + at(row, chunk));
      uint16_t* p = base(row);
      if (p == nullptr || m >= extent) continue;
      if (!CUT || m + 8 <= extent) {
        *reinterpret_cast<u32x4u*>(p + m) = v;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (m + e < extent) p[m + e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
      }
    }
  }
};

// AKC, BKC: the operand is stored with K contiguous.  COUNT_K: the live
// tokens bound K, else N.  ROTATE (few tokens, bound by reading A's rows): a
// workgroup starts at a stage of its own (a golden-ratio sequence) and wraps.
// With all of them at one k, rows a power of two apart put every piece that is
// read at one offset, and the reads pile onto a few HBM channels: logits of 16 x
// 65536 x 4096 bf16 109 us, rotated 94 (on another card 90.5, 5.9 TB/s).
template <int DT, int TM, int TN, int WM, int WN, int UNITS, bool AKC, bool BKC, int EPI, bool COUNT_K, bool ROTATE>
__device__ __forceinline__ void head_tile(Args g, int wg) {
  constexpr int NW = WM * WN;
  constexpr int MI = TM / WM / 32, NI = TN / WN / 32;
  static_assert(MI >= 1 && NI >= 1 && MI * WM * 32 == TM && NI * WN * 32 == TN, "wave tile");
  constexpr int NSUB = kStep / 16;
  using OpA = Operand<TM, AKC, NW>;
  using OpB = Operand<TN, BKC, NW>;
  // (In a ring of an even number of units a place holds units of one operand.)
  constexpr int kUnitA = UNITS % 2 && OpB::kBytes > OpA::kBytes ? OpB::kBytes : OpA::kBytes;
  constexpr int kUnitB = UNITS % 2 && OpA::kBytes > OpB::kBytes ? OpA::kBytes : OpB::kBytes;
  static_assert(UNITS >= 4 && kUnitA * ((UNITS + 1) / 2) + kUnitB * (UNITS / 2) <= 160 * 1024, "ring");
  auto place = [](auto uc) {
    constexpr int P = decltype(uc)::value % UNITS;
    return ring_unit<P % 2 ? kUnitB : kUnitA, P>();
  };
  constexpr int kPeriod = UNITS % 2 ? UNITS : UNITS / 2;  // stages until the units' places repeat

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;

  const int live = min(max(*g.count - g.count0, 0), COUNT_K ? g.K : g.N);
  const int N = COUNT_K ? g.N : live;
  const int tiles_n = (N + TN - 1) / TN;
  const int K_all = COUNT_K ? live : g.K;
  int chunk = K_all, splits = 1;
  constexpr bool kFuse = can_fuse(TM, TN) && EPI != kPartial;
  if constexpr (EPI == kSplit || kFuse) splits = splits_of(g.units, g.max_splits, g.tiles_m * tiles_n, K_all, &chunk);
  if (wg >= g.tiles_m * tiles_n * splits) return;
  int split, tm, tn;
  unit_of(g.tiles_m, tiles_n, splits, wg, split, tm, tn);
  const int m0 = tm * TM, n0 = tn * TN;
  const int kbeg = split * chunk;
  const int K = min(K_all - kbeg, chunk);
  const int nk = max((K + kStep - 1) / kStep, 0);

  const uint16_t* pa = g.A + (AKC ? (int64_t)m0 * g.lda + kbeg : (int64_t)kbeg * g.lda + m0);
  const uint16_t* pb = g.B + (BKC ? (int64_t)n0 * g.ldb + kbeg : (int64_t)kbeg * g.ldb + n0);
  const int64_t step_a = AKC ? kStep : kStep * g.lda, step_b = BKC ? kStep : kStep * g.ldb;
  OpA a;
  OpB b;
  a.init(wave, lane, g.M - m0, g.lda);
  b.init(wave, lane, N - n0, g.ldb);
  a.frag_init(lane, wm * (TM / WM));
  b.frag_init(lane, wn * (TN / WN));

  f32x16 acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j) acc[i][j] = f32x16{};

  u32x4 fa[2][MI], fb[2][NI];
  // Instructions FROM to TO - 1 of the next unit U of its operand (even units
  // are A's).
  int left_a = K, left_b = K;
  const int stage0 = ROTATE ? (int)(((uint64_t)((uint32_t)tm * 2654435769u) * (uint32_t)nk) >> 32) : 0;
  int at_a = stage0, at_b = stage0, issued_a = 0, issued_b = 0;
  if constexpr (ROTATE) {
    pa += stage0 * step_a;
    pb += stage0 * step_b;
    left_a -= stage0 * kStep;
    left_b = left_a;
  }
  auto advance = [&](const uint16_t*& p, int64_t step, int& left, int& at, int& issued) {
    p += step;
    left -= kStep;
    if constexpr (ROTATE) {
      if (++at == nk) {
        at = 0;
        p -= nk * step;
        left = K;
      }
      if (++issued >= nk) left = 0;
    }
  };
  auto issue = [&](auto uc, auto full, auto from, auto to) {
    constexpr int U = decltype(uc)::value, F = decltype(from)::value, T = decltype(to)::value;
    constexpr bool kFull = decltype(full)::value;
    unsigned char* st = place(uc);
    if constexpr (U % 2 == 0) {
      a.template issue<kFull, F, T>(pa, st, wave, left_a);
      if constexpr (T == OpA::kInst) advance(pa, step_a, left_a, at_a, issued_a);
    } else {
      b.template issue<kFull, F, T>(pb, st, wave, left_b);
      if constexpr (T == OpB::kInst) advance(pb, step_b, left_b, at_b, issued_b);
    }
  };
  // DMA instructions of n units from unit u on.
  constexpr auto dmas = [](int u, int n) {
    int c = 0;
    for (int i = 0; i < n; ++i) c += (u + i) % 2 ? OpB::kInst : OpA::kInst;
    return c;
  };
  auto read = [&](auto kc, int s) {
    constexpr int K0 = decltype(kc)::value;
    const unsigned char* sa = place(Int<2 * K0>{});
    const unsigned char* sb = place(Int<2 * K0 + 1>{});
#pragma unroll
    for (int i = 0; i < MI; ++i) fa[s & 1][i] = a.frag(sa, i, s);
#pragma unroll
    for (int j = 0; j < NI; ++j) fb[s & 1][j] = b.frag(sb, j, s);
  };
  auto multiply = [&](int s) {
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[i][j] = mfma<DT>(fa[s & 1][i], fb[s & 1][j], acc[i][j]);
  };
  constexpr int kReads = MI * (AKC ? 1 : 2) + NI * (BKC ? 1 : 2);
  constexpr int kMfmas = MI * NI;
  // Instruction order of one 16-wide K step: fragment reads behind the first
  // MFMAs, DMA loads spread over all.
  auto schedule = [&](auto nv_c) {
    constexpr int nv = decltype(nv_c)::value;
    constexpr int per = (kReads + kMfmas - 1) / kMfmas > 2 ? (kReads + kMfmas - 1) / kMfmas : 2;
#pragma unroll
    for (int m = 0; m < kMfmas; ++m) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      if (per * m < kReads) __builtin_amdgcn_sched_group_barrier(0x100, per, 0);
      int loads = 0;
#pragma unroll
      for (int v = 0; v < nv; ++v) loads += (v * kMfmas / (nv > 0 ? nv : 1) == m) ? 1 : 0;
      if (loads == 1) __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
      if (loads == 2) __builtin_amdgcn_sched_group_barrier(0x020, 2, 0);
      if (loads > 2) __builtin_amdgcn_sched_group_barrier(0x020, 4, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  using Full = std::true_type;
  using Checked = std::false_type;
  // Stage k (known modulo kPeriod): on entry fragment 0 is in registers, on
  // exit the next stage's.  The DMA of unit 2 k + UNITS goes out behind the
  // barrier, that of the unit after it over the next stage's K steps: 64 DMA
  // instructions take the CU's address unit 1024 cycles, and issued within one
  // K step (512 cycles of MFMA) they held the waves up.
  auto iteration = [&](auto kc, auto full) {
    constexpr int k = decltype(kc)::value;
    constexpr int kLast = 2 * k + UNITS - 1;  // the unit that the stage before left to issue
    constexpr int kParts = kLast % 2 ? OpB::kInst : OpA::kInst;
    constexpr int kNext = 2 * k + UNITS;
    constexpr int kNextParts = kNext % 2 ? OpB::kInst : OpA::kInst;
    auto step = [&](auto sc) {
      constexpr int s = decltype(sc)::value;
      constexpr int from = kParts * s / (NSUB - 1), to = kParts * (s + 1) / (NSUB - 1);
      read(Int<k>{}, s + 1);
      if constexpr (to > from) issue(Int<kLast>{}, full, Int<from>{}, Int<to>{});
      multiply(s);
      schedule(Int<to - from>{});
    };
    step(Int<0>{});
    step(Int<1>{});
    step(Int<2>{});
    static_assert(NSUB == 4, "K steps");
    wait_vm<dmas(2 * k + 4, UNITS - 4)>();  // the next stage's two units have landed
    wait_lgkm();
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    read(Int<k + 1>{}, 0);
    issue(Int<kNext>{}, full, Int<0>{}, Int<kNextParts>{});
    multiply(NSUB - 1);
    schedule(Int<kNextParts>{});
  };

  auto first = [&](auto uc) {
    constexpr int U = decltype(uc)::value;
    if constexpr (U < UNITS - 1) issue(uc, Checked{}, Int<0>{}, Int<(U % 2 ? OpB::kInst : OpA::kInst)>{});
  };
  first(Int<0>{});
  first(Int<1>{});
  first(Int<2>{});
  first(Int<3>{});
  first(Int<4>{});
  first(Int<5>{});
  first(Int<6>{});
  first(Int<7>{});
  first(Int<8>{});
  static_assert(UNITS <= 10, "ring");
  wait_vm<dmas(2, UNITS - 3)>();
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  read(Int<0>{}, 0);

  int kt = 0;
  // (A rotated walk passes a partial stage somewhere inside.)
  const int nfull = ROTATE && K % kStep ? 0 : K / kStep;
  for (; kt + kPeriod + UNITS / 2 <= nfull; kt += kPeriod) {
    iteration(Int<0>{}, Full{});
    iteration(Int<1>{}, Full{});
    if constexpr (kPeriod > 2) iteration(Int<2>{}, Full{});
    if constexpr (kPeriod > 3) iteration(Int<3>{}, Full{});
    if constexpr (kPeriod > 4) iteration(Int<4>{}, Full{});
  }
  static_assert(kPeriod <= 5, "ring");
  while (kt < nk) {
    iteration(Int<0>{}, Checked{});
    if (++kt >= nk) break;
    iteration(Int<1>{}, Checked{});
    if (++kt >= nk) break;
    if constexpr (kPeriod > 2) {
      iteration(Int<2>{}, Checked{});
      if (++kt >= nk) break;
    }
    if constexpr (kPeriod > 3) {
      iteration(Int<3>{}, Checked{});
      if (++kt >= nk) break;
    }
    if constexpr (kPeriod > 4) {
      iteration(Int<4>{}, Checked{});
      ++kt;
    }
  }
  wait_vm<0>();  // no DMA may still be writing LDS
  wait_lgkm();
  __builtin_amdgcn_s_barrier();  // every wave has read its last fragments: the stages are free
  // Rows on their way out: a part of the first units for each wave.
  typedef RowStage<MI> Stage;
  constexpr int kWavesPerUnit = kUnitA / Stage::kBytes;  // (in the places 0, 2, 4 of A's units)
  static_assert(kWavesPerUnit * ((UNITS + 1) / 2) >= NW && kWavesPerUnit * 3 >= NW, "staging");
  unsigned char* const rows_out = (wave < kWavesPerUnit       ? place(Int<0>{})
                                   : wave < 2 * kWavesPerUnit ? place(Int<2>{})
                                                              : place(Int<4 % UNITS>{})) +
                                  wave % kWavesPerUnit * Stage::kBytes;

  if constexpr (kFuse) {
    if (splits > 1) {
      constexpr int P = MI * NI * 4;
      split_f32x4 v[P];
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[p][e] = acc[p / 4 / NI][p / 4 % NI][p % 4 * 4 + e];
      if (!sum_splits<P, 64 * NW, 16>(v, make_rsrc(g.part, g.part_bytes), g.tiles_m * tiles_n, tm * tiles_n + tn, splits,
                                  split, g.counters, reinterpret_cast<unsigned*>(place(Int<1>{}))))
        return;
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[p / 4 / NI][p / 4 % NI][p % 4 * 4 + e] = v[p][e];
      splits = 1;
    }
  }

  // Accumulator block (mi, ni) of a lane: row n of the output, columns
  // m = mfirst + 32 mi + 8 (r / 4) + 4 (lane / 32) + r % 4.
  const int half = lane >> 5;
  const int mfirst = m0 + wm * (TM / WM);
#pragma unroll
  for (int ni = 0; ni < NI; ++ni) {
    const int nfirst = n0 + wn * (TN / WN) + ni * 32, n = nfirst + (lane & 31);
    const bool live_n = n < N;
    if constexpr (EPI == kStats || EPI == kExp) {
      constexpr float kLog2e = 1.44269504088896341f;
      constexpr int kBlock = TM / WM;
      const bool edge = mfirst + kBlock > g.M;
      if (edge) {
#pragma unroll
        for (int mi = 0; mi < MI; ++mi)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (mfirst + mi * 32 + 8 * (r / 4) + 4 * half + r % 4 >= g.M) acc[mi][ni][r] = -__builtin_inff();
      }
      // The target's logit, where it lies in this block (few waves have one).
      const int t = live_n ? g.target[n] : -1;
      const int at = t - mfirst;
      if (__any(at >= 0 && at < kBlock && live_n)) {
        float v = 0.f;
#pragma unroll
        for (int mi = 0; mi < MI; ++mi)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (at == mi * 32 + 8 * (r / 4) + 4 * half + r % 4) v = acc[mi][ni][r];
        if (live_n && at >= 0 && at < kBlock && ((at >> 2) & 1) == half) g.hit[n] = v;
      }
      // In powers of two: exp(l) = 2^(l log2 e), relative to the block's largest
      // exponent c, whose float32 value is the reference itself, so that one
      // fused multiply-add per logit loses nothing.
      float top = -__builtin_inff();
#pragma unroll
      for (int mi = 0; mi < MI; ++mi)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, acc[mi][ni][r]);
      top = fmaxf(top, __shfl_xor(top, 32)) * kLog2e;
      // (a block without a finite maximum: 2^(-inf - 0) = 0)
      const float ref = top == -__builtin_inff() ? 0.f : top;
      float sum = 0.f;
#pragma unroll
      for (int mi = 0; mi < MI; ++mi)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[mi][ni][r], kLog2e, -ref));
          acc[mi][ni][r] = e;
          sum += e;
        }
      sum += __shfl_xor(sum, 32);
      if (half == 0 && live_n) g.stats[(int64_t)n * g.ld_stats + tm * WM + wm] = f32x2{top, sum};
      if constexpr (EPI == kExp) {
        const float up = exp_factor(top);
#pragma unroll
        for (int mi = 0; mi < MI; ++mi)
          Stage::template put<HCG_F16>(rows_out, lane, mi, [&](int r) { return acc[mi][ni][r] * up; });
        Stage::template store<false>(rows_out, lane, mfirst, g.M, [&](int row) -> uint16_t* {
          const int to = nfirst + row;
          return to < N ? static_cast<uint16_t*>(g.out) + (int64_t)to * g.ldo : nullptr;
        });
      }
    } else {
      if (EPI != kSplit && g.add && live_n) {
#pragma unroll
        for (int mi = 0; mi < MI; ++mi)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int m = mfirst + mi * 32 + 8 * q + 4 * half;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (m + e < g.M) acc[mi][ni][4 * q + e] += g.add[(int64_t)n * g.M + m + e];
          }
      }
      if (EPI == kRound || (EPI == kSplit && splits == 1)) {
        const float f = *g.scale * g.post;
#pragma unroll
        for (int mi = 0; mi < MI; ++mi)
          Stage::template put<DT>(rows_out, lane, mi, [&](int r) { return acc[mi][ni][r] * f; });
        Stage::template store<true>(rows_out, lane, mfirst, g.M, [&](int row) -> uint16_t* {
          const int to = nfirst + row;
          if (to >= N) return nullptr;
          return static_cast<uint16_t*>(g.out) + (int64_t)(g.row_of ? g.row_of[to] : to) * g.ldo;
        });
      } else {
        typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
        float* row = g.part + ((int64_t)split * N + n) * g.ld_part;
        if (live_n) {
#pragma unroll
          for (int mi = 0; mi < MI; ++mi)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const int m = mfirst + mi * 32 + 8 * q + 4 * half;
              const f32x4 v{acc[mi][ni][4 * q], acc[mi][ni][4 * q + 1], acc[mi][ni][4 * q + 2], acc[mi][ni][4 * q + 3]};
              if (m + 4 <= g.M) {
                *reinterpret_cast<f32x4u*>(row + m) = v;
              } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (m + e < g.M) row[m + e] = v[e];
              }
            }
        }
      }
    }
  }
}

// The sum of the losses over the live tokens by one wave, in one order, into
// *out (times *scale).  It runs beside the tiles of a product.  In doubles: a lane
// adds up n / 64 values, and like ones would all be rounded the same way.
__device__ __forceinline__ void sum_losses(const float* loss, int n, const float* scale, float* out) {
  double sum = 0.0;
#pragma unroll 16
  for (int i = threadIdx.x; i < n; i += 64) sum += loss[i];
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) sum += __shfl_xor(sum, m);
  if (threadIdx.x == 0) *out = (float)(sum * (double)*scale);
}

// Waves per SIMD: two workgroups per CU where the ring takes at most half its LDS.
constexpr int waves_per_simd(int tm, int tn, int waves, int units) {
  return waves / 4 * ((tm + tn) * kStep * 2 * units / 2 <= 80 * 1024 ? 2 : 1);
}

template <int DT, int TM, int TN, int WM, int WN, int UNITS, bool AKC, bool BKC, int EPI, bool COUNT_K, bool ROTATE>
__global__ __launch_bounds__(64 * WM * WN, waves_per_simd(TM, TN, WM * WN, UNITS)) void head_kernel(Args g) {
  if (EPI == kRound && g.loss_out && blockIdx.x + 1 == gridDim.x) {
    if (threadIdx.x < 64) sum_losses(g.loss, *g.count, g.loss_scale, g.loss_out);
    return;
  }
  head_tile<DT, TM, TN, WM, WN, UNITS, AKC, BKC, EPI, COUNT_K, ROTATE>(g, blockIdx.x);
}

}  // namespace head
}  // namespace hcg
