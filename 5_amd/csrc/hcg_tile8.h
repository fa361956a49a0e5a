// hcg_tile8.h -- the tiled product of two quantised matrices on gfx950 (device
// code).
//
// A TM x TN tile of outputs x tokens by WM x WN waves; K advances one block of 128
// (a scale each) per stage.  A stage is two units, the weight's rows and x's, of
// 128 bytes a row, filled by global-to-LDS DMA two stages ahead: three places for
// the weight's, two for x's (160 KB for 256 x 256).  The 16-byte chunks of an LDS
// row are XOR-swizzled so that the lanes that an LDS cycle serves cover all banks.
//
// 256 x 256 tiles by eight waves, 8192^3, passes back to back on one card: 450 us
// with float32 scales (2.44 PFLOP/s), 398 with e8m0 ones (2.76; 381 on another
// card); a library's product of the same size with one scale for all 350 (3.14), so
// that the scaling of a block's sums (16 multiply-adds per lane and four products)
// costs an eighth.  Float32 scales of the weight's rows 657 us in 128 x 128 tiles, a
// multiplication more per sum; exact products with them 1039 (1.06 PFLOP/s; a 16-bit
// product 809): of 21 instructions per 128-deep product 4 are MFMAs, 8 scale and 8
// convert, every fragment in the two waves that hold it.  Alone on a CU a 256 x 256
// stage takes 1.04 us (2500 cycles for 2048 of MFMA issue), on a busy chip 1.47 at a
// lower clock.  Four-wave tiles spill; sixteen-wave ones took 478 us where eight took
// 412.
//
// A 16-bit result takes v_mfma_f32_16x16x128 on the bytes as they are: a block's
// products in one instruction, whose sum is multiplied by both scales into the
// accumulators, or whose scales are the instruction's own (e8m0), which then
// adds up all of K.  The instruction cuts each product of 8 neighbours to
// multiples of 2^-13 of the largest exponent among them (measured: beside 448 *
// 448 the bits below 2^3 are lost), 1.5e-5 of a sum of normal products, and up to 8e-5
// where one column in a hundred is sixteen times the others: less than a 16-bit
// result's rounding (2.1e-4 for f16), but not float32.  So a float32 result (EXACT)
// takes the bytes as f16, which holds both formats, in v_mfma_f32_16x16x32,
// whose sums are within 2^-22 of the magnitudes.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "hcg_scale8.h"
#include "hcg_tile.h"

namespace hcg {
namespace fp8 {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// How scales are held and used.
enum Scaling {
  kTile,       // float32, the weight's by tiles
  kRow,        // float32, the weight's by rows
  kPowerTile,  // exponent bytes, which the MFMA takes itself
  kPowerRow
};
constexpr bool by_power(Scaling s) { return s == kPowerTile || s == kPowerRow; }
constexpr bool by_tile(Scaling s) { return s == kTile || s == kPowerTile; }

struct Args {
  const unsigned char* x;
  const unsigned char* w;
  int64_t ldx, ldw;
  const void* sx;
  const void* sw;
  int64_t sx_row, sx_block, sw_row, sw_block;  // (tiled: the rows' strides are 1)
  int T, V, K;
  void* y;
  int64_t ldy;
  int y_dtype;
  // Tiled: K in splits of `chunk` (a multiple of kBlock); where there are more than
  // one, float32 sums go to part[split][T][ld_part].
  int splits, chunk;
  float* part;
  int64_t ld_part;
};

// c + w-block . x-block, 128 deep.  X5: x is e5m2.
template <bool X5>
__device__ __forceinline__ f32x4 mfma(i32x8 w, i32x8 x, f32x4 c) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, c, 0, X5 ? 1 : 0, 0, 0, 0, 0);
}
template <bool X5>
__device__ __forceinline__ f32x4 mfma(i32x8 w, i32x8 x, f32x4 c, int sw, int sx) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, c, 0, X5 ? 1 : 0, 0, sw, 0, sx);
}

// 8 bytes as f16, exactly (a byte of e5m2 is an f16's upper one).
template <bool E5>
__device__ __forceinline__ f16x8 halves(int lo, int hi) {
  uint32_t r[4];
  if constexpr (E5) {
    r[0] = __builtin_amdgcn_perm(0u, (uint32_t)lo, 0x010c000cu);
    r[1] = __builtin_amdgcn_perm(0u, (uint32_t)lo, 0x030c020cu);
    r[2] = __builtin_amdgcn_perm(0u, (uint32_t)hi, 0x010c000cu);
    r[3] = __builtin_amdgcn_perm(0u, (uint32_t)hi, 0x030c020cu);
  } else {
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((uint32_t)lo, 1.f, false));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((uint32_t)lo, 1.f, true));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((uint32_t)hi, 1.f, false));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((uint32_t)hi, 1.f, true));
  }
  return __builtin_bit_cast(f16x8, u32x4{r[0], r[1], r[2], r[3]});
}
struct Halves {
  f16x8 v[4];
};
template <bool E5>
__device__ __forceinline__ Halves halves(i32x8 b) {
  Halves h;
#pragma unroll
  for (int q = 0; q < 4; ++q) h.v[q] = halves<E5>(b[2 * q], b[2 * q + 1]);
  return h;
}
// The same sum of 128 products, exactly.
__device__ __forceinline__ f32x4 mfma(const Halves& w, const Halves& x) {
  f32x4 c{};
#pragma unroll
  for (int q = 0; q < 4; ++q) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(w.v[q], x.v[q], c, 0, 0, 0);
  return c;
}

__device__ __forceinline__ i32x8 join(u32x4 a, u32x4 b) {
  return i32x8{(int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)b[0], (int)b[1], (int)b[2], (int)b[3]};
}

__device__ __forceinline__ uint32_t pack_out(float a, float b, int dtype) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  if (dtype == HCG_F16) return __builtin_bit_cast(uint32_t, f16x2{(_Float16)a, (_Float16)b});
  return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)a, (__bf16)b});
}

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

// blockIdx -> (K split, tile): each XCD (id % 8) takes a contiguous run of
// units, within a split in groups of 4 tile rows, so that the workgroups
// sharing an L2 share operand rows.
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

// One operand's unit: ROWS rows of a block's 128 bytes, loaded by NW waves.
template <int ROWS, int NW>
struct Side {
  static constexpr int kBytes = ROWS * kBlock;
  static constexpr int kInst = kBytes / 1024 / NW;  // DMA instructions per wave per unit
  static_assert(kInst >= 1 && kInst * NW * 1024 == kBytes, "a unit is whole DMA instructions of every wave");
  static __device__ __forceinline__ int swz(int row, int c) { return c ^ ((row >> 1) & 7); }

  int64_t ld;
  int rows;       // of the matrix, from the tile's first on
  int key;        // the lane's first byte in the rows of the wave's even instructions; in an odd one's key ^ 64
  int at[2];      // and its place from the instruction's first row in either

  __device__ __forceinline__ void init(int wave, int lane, int extent, int64_t stride) {
    ld = stride;
    rows = min(extent, ROWS);
    key = swz(wave * kInst * 8 + (lane >> 3), lane & 7) * 16;  // (8 rows on the swizzle differs by 4 chunks)
    at[0] = (lane >> 3) * (int)ld + key;
    at[1] = (lane >> 3) * (int)ld + (key ^ 64);
  }
  // Instructions FROM to TO - 1 of the wave's, of the unit whose first byte is at p
  // and whose rows have `left` bytes from there on (FULL: all of them).  The
  // resource starts at the unit and ends with the matrix's last row, so that
  // offsets stay in 31 bits whatever the matrix's size and rows past it load
  // zeros; chunks past a row's end are redirected past it.  The chunk with a
  // row's last byte is loaded whole, from within its own 16-byte granule.
  template <bool FULL, int FROM, int TO>
  __device__ __forceinline__ void issue(const unsigned char* p, unsigned char* st, int wave, int left) const {
    const int end = (int)((rows - 1) * ld) + (FULL ? kBlock : min((left + 15) & ~15, kBlock));
    const __amdgpu_buffer_rsrc_t r = make_rsrc(p, max(end, 0));
#pragma unroll
    for (int i = FROM; i < TO; ++i) {
      lds_void* dst = (lds_void*)(st + (wave * kInst + i) * 1024);
      // (All of the offset is the lane's: what is checked against the extent.)
      const int off = at[i & 1] + (wave * kInst + i) * 8 * (int)ld;
      if constexpr (FULL)
        dma16(r, dst, off);
      else
        dma16(r, dst, dma_offset((i & 1 ? key ^ 64 : key) < left, off));
    }
  }
  // Zeros in place of what lies past `left` bytes in the chunk that holds them.
  static __device__ __forceinline__ void cut(unsigned char* st, int tid, int left) {
    for (int row = tid; row < ROWS; row += 64 * NW) {
      u32x4* chunk = reinterpret_cast<u32x4*>(st + row * kBlock + swz(row, left >> 4) * 16);
      u32x4 v = *chunk;
      const int valid = left & 15;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int bytes = min(max(valid - 4 * e, 0), 4);
        v[e] &= bytes == 4 ? 0xffffffffu : (1u << (8 * bytes)) - 1;
      }
      *chunk = v;
    }
  }
  // The lane's fragment of rows 16 i ... past `base` (made from the wave's first):
  // chunks l / 16 and l / 16 + 4.  An LDS cycle serves lanes 0 - 3, 12 - 15 and 20 -
  // 27 together, or 4 - 11, 16 - 19 and 28 - 31 (and so on): with neighbouring
  // chunks in lanes 16 apart those are 16 places in different banks (with chunks
  // 2 (l / 16) half of all LDS cycles were conflicts).
  static __device__ __forceinline__ int base_of(int lane, int first) {
    const int row = lane & 15;
    return (first + row) * kBlock + swz(row, lane >> 4) * 16;
  }
  static __device__ __forceinline__ i32x8 frag(const unsigned char* st, int base, int i) {
    return join(*reinterpret_cast<const u32x4*>(st + base + i * 16 * kBlock),
                *reinterpret_cast<const u32x4*>(st + (base ^ 64) + i * 16 * kBlock));
  }
};

template <int I>
using Int = std::integral_constant<int, I>;

// Places in LDS for units of the weight and of x.
constexpr int kPlacesA = 3, kPlacesB = 2;

// Waves per SIMD: two workgroups per CU where the rings take at most half its LDS.
constexpr int waves_per_simd(int tm, int tn, int waves) {
  return waves / 4 * ((tm * kPlacesA + tn * kPlacesB) * kBlock <= 80 * 1024 ? 2 : 1);
}

template <bool X5, Scaling SC, bool EXACT, int TM, int TN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN, waves_per_simd(TM, TN, WM* WN)) void tile_kernel(Args g) {
  constexpr int NW = WM * WN;
  constexpr int MI = TM / WM / 16, NI = TN / WN / 16;
  static_assert(MI >= 2 && NI >= 1 && MI * WM * 16 == TM && NI * WN * 16 == TN, "wave tile");
  static_assert(kBlock % (TM / WM) == 0, "a wave's outputs share a tile's scale");
  static_assert(!EXACT || !by_power(SC), "exact products take float32 scales");
  using OpA = Side<TM, NW>;
  using OpB = Side<TN, NW>;
  static_assert(OpA::kBytes * kPlacesA + OpB::kBytes * kPlacesB <= 160 * 1024, "rings");
  auto place_a = [](auto kc) { return ring_unit<OpA::kBytes, decltype(kc)::value % kPlacesA>(); };
  auto place_b = [](auto kc) { return ring_unit<OpB::kBytes, kPlacesA + decltype(kc)::value % kPlacesB>(); };
  constexpr int kPeriod = 6;  // stages until the places repeat

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int tiles_m = (g.V + TM - 1) / TM, tiles_n = (g.T + TN - 1) / TN;
  int split, tm, tn;
  unit_of(tiles_m, tiles_n, g.splits, blockIdx.x, split, tm, tn);
  const int m0 = tm * TM, n0 = tn * TN;
  const int mfirst = m0 + wm * (TM / WM), nfirst = n0 + wn * (TN / WN);
  const int kbeg = split * g.chunk;
  const int K = min(g.K - kbeg, g.chunk);
  const int nk = (K + kBlock - 1) / kBlock;

  const unsigned char* pa = g.w + (int64_t)m0 * g.ldw + kbeg;
  const unsigned char* pb = g.x + (int64_t)n0 * g.ldx + kbeg;
  OpA a;
  OpB b;
  a.init(wave, lane, g.V - m0, g.ldw);
  b.init(wave, lane, g.T - n0, g.ldx);
  const int first_a = OpA::base_of(lane, wm * (TM / WM)), first_b = OpB::base_of(lane, wn * (TN / WN));

  // Scales: a stage's are loaded two stages ahead, those of rows past the last as
  // zeros.
  constexpr int kHeld = by_power(SC) ? 1 : 4;
  const int quad = lane >> 4;
  static_assert(NI == 2 || NI == 4, "tokens' scales");
  const int at_x = (nfirst + (lane & (16 * NI - 1))) * kHeld;
  const int at_w = by_tile(SC)    ? mfirst / kBlock * kHeld
                   : by_power(SC) ? mfirst + (lane & (16 * MI - 1) & 63)
                                  : (mfirst + 4 * quad) * kHeld;
  const int rows_w = by_tile(SC) ? (g.V + kBlock - 1) / kBlock : SC == kRow ? (g.V + 3) & ~3 : g.V;
  int block = kbeg / kBlock;  // of the scales that are loaded next
  const int last_block = block + nk - 1;
  constexpr int kWs = SC == kPowerRow ? MI : 1;
  // As loaded: of 64 of the wave's tokens or outputs, one a lane (a load for each
  // group of 16 would take as many of the CU's address cycles as a third of the
  // operands' DMA).
  constexpr int kXs = (NI + 3) / 4, kEws = SC == kPowerRow ? (MI + 3) / 4 : 1;
  struct Loaded {
    uint32_t x[kXs], ew[kEws];
    f32x4 w[SC == kRow ? MI : 1];
  };
  // As used: x[j] in every lane that holds a sum of token 16 j + lane % 16.
  struct Scales {
    float x[NI];
    f32x4 w[SC == kRow ? MI : 1];
    int ex[NI], ew[kWs];
  };
  // v[j] = lane % 16 of each 16 lanes' values, j of `groups`.
  auto fan = [](auto groups, const uint32_t* l, uint32_t* v) {
    constexpr int G = decltype(groups)::value;
    static_assert(G == 2 || G % 4 == 0, "groups");
#pragma unroll
    for (int q = 0; q < (G + 3) / 4; ++q) {
      const auto rows = __builtin_amdgcn_permlane16_swap(l[q], l[q], false, false);
      if constexpr (G == 2) {
        v[0] = rows[0], v[1] = rows[1];
      } else {
        const auto even = __builtin_amdgcn_permlane32_swap(rows[0], rows[0], false, false);
        const auto odd = __builtin_amdgcn_permlane32_swap(rows[1], rows[1], false, false);
        v[4 * q] = even[0], v[4 * q + 1] = odd[0], v[4 * q + 2] = even[1], v[4 * q + 3] = odd[1];
      }
    }
  };
  auto spread = [&](const Loaded& l) {
    Scales s;
    uint32_t x[NI];
    fan(Int<NI>{}, l.x, x);
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      if constexpr (by_power(SC))
        s.ex[j] = (int)x[j];
      else
        s.x[j] = SC == kTile ? __builtin_bit_cast(float, x[j]) * l.w[0][0] : __builtin_bit_cast(float, x[j]);
    }
#pragma unroll
    for (int i = 0; i < (SC == kRow ? MI : 1); ++i) s.w[i] = l.w[i];
    if constexpr (SC == kPowerRow) {
      uint32_t w[MI];
      fan(Int<MI>{}, l.ew, w);
#pragma unroll
      for (int i = 0; i < MI; ++i) s.ew[i] = (int)w[i];
    } else {
      s.ew[0] = (int)l.ew[0];
    }
    return s;
  };
  auto load_scales = [&](Loaded& s) {
    const __amdgpu_buffer_rsrc_t rx =
        make_rsrc(static_cast<const unsigned char*>(g.sx) + block * g.sx_block * kHeld, g.T * kHeld);
    const __amdgpu_buffer_rsrc_t rw =
        make_rsrc(static_cast<const unsigned char*>(g.sw) + block * g.sw_block * kHeld, rows_w * kHeld);
#pragma unroll
    for (int q = 0; q < kXs; ++q) {
      if constexpr (by_power(SC))
        s.x[q] = __builtin_amdgcn_raw_buffer_load_b8(rx, at_x + 64 * q, 0, 0);
      else
        s.x[q] = __builtin_amdgcn_raw_buffer_load_b32(rx, at_x + 256 * q, 0, 0);
    }
    if constexpr (by_power(SC)) {
#pragma unroll
      for (int q = 0; q < kEws; ++q)
        s.ew[q] = __builtin_amdgcn_raw_buffer_load_b8(rw, at_w + 64 * q, 0, 0);
    } else if constexpr (SC == kTile) {
      s.w[0][0] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rw, at_w, 0, 0));
    } else {
#pragma unroll
      for (int i = 0; i < MI; ++i)
        s.w[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rw, at_w + 64 * i, 0, 0));
    }
    block = min(block + 1, last_block);
  };

  f32x4 acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j) acc[i][j] = f32x4{};

  int left_a = K, left_b = K;
  // DMA instructions FROM to TO - 1 of the next unit of the weight, or of x, which is
  // stage kc's.
  auto issue_a = [&](auto kc, auto full, auto from, auto to) {
    constexpr int F = decltype(from)::value, T = decltype(to)::value;
    if constexpr (T > F) a.template issue<decltype(full)::value, F, T>(pa, place_a(kc), wave, left_a);
    if constexpr (T > F && T == OpA::kInst) pa += kBlock, left_a -= kBlock;
  };
  auto issue_b = [&](auto kc, auto full, auto from, auto to) {
    constexpr int F = decltype(from)::value, T = decltype(to)::value;
    if constexpr (T > F) b.template issue<decltype(full)::value, F, T>(pb, place_b(kc), wave, left_b);
    if constexpr (T > F && T == OpB::kInst) pb += kBlock, left_b -= kBlock;
  };

  using FragA = std::conditional_t<EXACT, Halves, i32x8>;
  using FragB = std::conditional_t<EXACT, Halves, i32x8>;
  i32x8 ra, rb[NI];  // fragments as read
  Loaded next;  // of the stage after the next one
  Scales now;
  // Sums of a block that are not yet in the accumulators: the scaling of a sum runs
  // kLag products behind, so that it does not wait for its own.  Everything is
  // issued in the order written here: left to itself the compiler starts all
  // products of a stage and spills.
  constexpr int kLag = EXACT ? NI : NI - 1, kSums = EXACT ? 2 * NI : NI;
  f32x4 parts[kSums];
  // The stage's products in their order: the last kLate groups of outputs are taken
  // token group by token group, so that x's fragments come free one by one.
  constexpr int kLate = MI > 2 ? 2 : 1, kEarly = MI - kLate;
  constexpr auto group_of = [](int n) { return n < kEarly * NI ? n / NI : kEarly + n % kLate; };
  constexpr auto tokens_of = [](int n) { return n < kEarly * NI ? n % NI : (n - kEarly * NI) / kLate; };
  auto scale = [&](auto nc, const Scales& s) {
    constexpr int n = decltype(nc)::value, i = group_of(n), j = tokens_of(n);
    const f32x4 part = parts[n % kSums];
#pragma unroll
    for (int r = 0; r < 4; ++r)
      acc[i][j][r] = __builtin_fmaf(part[r], SC == kTile ? s.x[j] : s.x[j] * s.w[i][r], acc[i][j][r]);
    asm volatile("" : "+v"(acc[i][j]));  // (here and not where the sums are used next)
  };
  auto product = [&](auto nc, const FragA& fa, const FragB& fb, const Scales& s) {
    constexpr int n = decltype(nc)::value, i = group_of(n), j = tokens_of(n);
    if constexpr (by_power(SC)) {
      acc[i][j] = mfma<X5>(fa, fb, acc[i][j], s.ew[SC == kPowerRow ? i : 0], s.ex[j]);
      asm volatile("" : "+v"(acc[i][j]));
    } else {
      if constexpr (EXACT)
        parts[n % kSums] = mfma(fa, fb);
      else
        parts[n % kSums] = mfma<X5>(fa, fb, f32x4{});
      if constexpr (n >= kLag) scale(Int<n - kLag>{}, s);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  auto finish = [&](const Scales& s) {
    if constexpr (!by_power(SC)) {
      constexpr int n = MI * NI;
      if constexpr (kLag > 3) scale(Int<n - 4>{}, s);
      if constexpr (kLag > 2) scale(Int<n - 3>{}, s);
      if constexpr (kLag > 1) scale(Int<n - 2>{}, s);
      scale(Int<n - 1>{}, s);
    }
  };
  auto as_a = [](i32x8 v) -> FragA {
    if constexpr (EXACT)
      return halves<false>(v);
    else
      return v;
  };
  auto as_b = [](i32x8 v) -> FragB {
    if constexpr (EXACT)
      return halves<X5>(v);
    else
      return v;
  };
  using Full = std::true_type;
  using Checked = std::false_type;
  // Where K ends inside a chunk, the last stage's bytes past it are cleared once
  // they have landed (in both operands: they may be NaNs).
  const bool ragged = (K & 15) != 0;
  auto cut = [&](auto kc) {
    OpA::cut(place_a(kc), tid, K & (kBlock - 1));
    OpB::cut(place_b(kc), tid, K & (kBlock - 1));
    wait_lgkm();
    __builtin_amdgcn_s_barrier();
  };
  // Stage k (known modulo kPeriod): on entry its scales, its tokens' fragments and
  // the first of its outputs' are in registers or on their way, on exit the next
  // stage's.  Its steps take 16 outputs each, the last kLate of them as one.  The
  // weight's unit of stage k + 2 goes out over the first half (its place held stage
  // k - 1's); x's over the second half: its place held this stage's, whose
  // fragments every wave has read once all have met in the middle.  So DMA
  // instructions, each 16 cycles of the CU's address unit, never queue up in front
  // of a wave's products.  Before the last step all have read this stage's
  // fragments and the next one's have landed: they are read between its products.
  constexpr int kHalf = MI / 2;
  auto iteration = [&](auto kc, auto full, int kt) {
    constexpr int k = decltype(kc)::value;
    const unsigned char* sa = place_a(kc);
    const Scales s = now;
    // (Fresh every stage: the compiler would hold an address for each read whose
    // place lies past the 64 KB that an LDS instruction's offset reaches.)
    int base_a = first_a, base_b = first_b;
    asm volatile("" : "+v"(base_a), "+v"(base_b));
    FragB fb[NI];
#pragma unroll
    for (int j = 0; j < NI; ++j) fb[j] = as_b(rb[j]);
    i32x8 rz = ra;  // of the last group of outputs
    auto dma = [&](auto ic) {
      constexpr int i = decltype(ic)::value;
      if constexpr (i < kHalf)
        issue_a(Int<k + 2>{}, full, Int<OpA::kInst * i / kHalf>{}, Int<OpA::kInst*(i + 1) / kHalf>{});
      else
        issue_b(Int<k + 2>{}, full, Int<OpB::kInst*(i - kHalf) / kHalf>{}, Int<OpB::kInst*(i - kHalf + 1) / kHalf>{});
    };
    auto step = [&](auto ic) {
      constexpr int i = decltype(ic)::value;
      const FragA fa = as_a(ra);
      ra = OpA::frag(sa, base_a, i + 1);
      if constexpr (kLate > 1 && i == kEarly - 1) rz = OpA::frag(sa, base_a, i + 2);
      dma(ic);
      product(Int<i * NI>{}, fa, fb[0], s);
      product(Int<i * NI + 1>{}, fa, fb[1], s);
      if constexpr (NI > 2) product(Int<i * NI + 2>{}, fa, fb[2], s);
      if constexpr (NI > 3) product(Int<i * NI + 3>{}, fa, fb[3], s);
      if constexpr (i == kHalf - 1) {
        wait_vm<OpA::kInst>();  // the next stage's two units have landed
        if constexpr (i < kEarly - 1) {
          __builtin_amdgcn_s_barrier();
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    };
    step(Int<0>{});
    if constexpr (kEarly > 1) step(Int<1>{});
    if constexpr (kEarly > 2) step(Int<2>{});
    if constexpr (kEarly > 3) step(Int<3>{});
    if constexpr (kEarly > 4) step(Int<4>{});
    if constexpr (kEarly > 5) step(Int<5>{});
    static_assert(MI == 2 || MI == 4 || MI == 8, "steps");
    wait_lgkm();
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (!decltype(full)::value) {
      if (ragged && kt + 2 == nk) cut(Int<k + 1>{});
    }
    const FragA fa = as_a(ra), fz = as_a(rz);
    const unsigned char* nb = place_b(Int<k + 1>{});
    ra = OpA::frag(place_a(Int<k + 1>{}), base_a, 0);
    if constexpr (kLate > 1) dma(Int<kEarly>{});
    auto late = [&](auto jc) {
      constexpr int j = decltype(jc)::value, n = kEarly * NI + j * kLate;
      if constexpr (j == NI / 2) dma(Int<MI - 1>{});
      if constexpr (kLate > 1) product(Int<n>{}, fa, fb[j], s);
      product(Int<n + kLate - 1>{}, kLate > 1 ? fz : fa, fb[j], s);
      rb[j] = OpB::frag(nb, base_b, j);
      __builtin_amdgcn_sched_barrier(0);
    };
    late(Int<0>{});
    late(Int<1>{});
    if constexpr (NI > 2) late(Int<2>{});
    if constexpr (NI > 3) late(Int<3>{});
    now = spread(next);
    load_scales(next);
    finish(s);
    __builtin_amdgcn_sched_barrier(0);
  };

  load_scales(next);
  issue_a(Int<0>{}, Checked{}, Int<0>{}, Int<OpA::kInst>{});
  issue_b(Int<0>{}, Checked{}, Int<0>{}, Int<OpB::kInst>{});
  issue_a(Int<1>{}, Checked{}, Int<0>{}, Int<OpA::kInst>{});
  issue_b(Int<1>{}, Checked{}, Int<0>{}, Int<OpB::kInst>{});
  wait_vm<OpA::kInst + OpB::kInst>();
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  now = spread(next);
  load_scales(next);
  __builtin_amdgcn_sched_barrier(0);
  if (ragged && nk == 1) cut(Int<0>{});
  ra = OpA::frag(place_a(Int<0>{}), first_a, 0);
#pragma unroll
  for (int j = 0; j < NI; ++j) rb[j] = OpB::frag(place_b(Int<0>{}), first_b, j);

  int kt = 0;
  const int nfull = K / kBlock;
  for (; kt + kPeriod + 2 <= nfull; kt += kPeriod) {
    iteration(Int<0>{}, Full{}, 0);
    iteration(Int<1>{}, Full{}, 0);
    iteration(Int<2>{}, Full{}, 0);
    iteration(Int<3>{}, Full{}, 0);
    iteration(Int<4>{}, Full{}, 0);
    iteration(Int<5>{}, Full{}, 0);
  }
  while (kt < nk) {
    iteration(Int<0>{}, Checked{}, kt);
    if (++kt >= nk) break;
    iteration(Int<1>{}, Checked{}, kt);
    if (++kt >= nk) break;
    iteration(Int<2>{}, Checked{}, kt);
    if (++kt >= nk) break;
    iteration(Int<3>{}, Checked{}, kt);
    if (++kt >= nk) break;
    iteration(Int<4>{}, Checked{}, kt);
    if (++kt >= nk) break;
    iteration(Int<5>{}, Checked{}, kt);
    ++kt;
  }
  wait_vm<0>();  // no DMA may still be writing LDS
  wait_lgkm();
  __builtin_amdgcn_s_barrier();  // every wave has read its last fragments: the units are free

  // Block (i, j) of a lane: token nfirst + 16 j + lane % 16, outputs mfirst + 16 i +
  // 4 (lane / 16) + r.
  if (g.splits > 1) {
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int t = nfirst + 16 * j + (lane & 15);
      if (t >= g.T) continue;
      float* row = g.part + ((int64_t)split * g.T + t) * g.ld_part;  // (rows of whole fours)
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const int v = mfirst + 16 * i + 4 * quad;
        if (v < g.V) *reinterpret_cast<f32x4*>(row + v) = acc[i][j];
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    return;
  }
  // A wave's 16 tokens at a time pass through LDS, so that rows leave in pieces of
  // 16 bytes that are neighbours.
  constexpr int kSize = EXACT ? 4 : 2;
  constexpr int kRow = MI * 16 * kSize, kChunks = kRow / 16, kStage = 16 * kRow;
  constexpr int kPerUnit = OpA::kBytes / kStage;
  static_assert(kPerUnit * kPlacesA >= NW && kChunks <= 64, "staging");
  unsigned char* const out = (wave < kPerUnit       ? place_a(Int<0>{})
                              : wave < 2 * kPerUnit ? place_a(Int<1>{})
                                                    : place_a(Int<2>{})) +
                             wave % kPerUnit * kStage;
  // (Chunk c of row t lies at c ^ t, within the row's chunks.)
  auto chunk_at = [](int t, int c) { return t * kRow + (c ^ (t & (kChunks - 1))) * 16; };
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  typedef uint32_t u32x4w __attribute__((ext_vector_type(4), aligned(4)));
  typedef uint32_t u32x4h __attribute__((ext_vector_type(4), aligned(2)));
  using u32x4u = std::conditional_t<EXACT, u32x4w, u32x4h>;
#pragma unroll
  for (int j = 0; j < NI; ++j) {
    const int t = lane & 15;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const f32x4 v = acc[i][j];
      if constexpr (EXACT)
        *reinterpret_cast<f32x4*>(out + chunk_at(t, 4 * i + quad)) = v;
      else
        *reinterpret_cast<u32x2*>(out + chunk_at(t, 2 * i + (quad >> 1)) + 8 * (quad & 1)) =
            u32x2{pack_out(v[0], v[1], g.y_dtype), pack_out(v[2], v[3], g.y_dtype)};
    }
    __builtin_amdgcn_sched_barrier(0);
    constexpr int kRows = 64 / kChunks;  // per instruction
    const int c = lane % kChunks, v0 = mfirst + c * (16 / kSize);
#pragma unroll
    for (int q = 0; q < 16 / kRows; ++q) {
      const int row = q * kRows + lane / kChunks, to = nfirst + 16 * j + row;
      const u32x4 v = *reinterpret_cast<const u32x4*>(out + chunk_at(row, c));
      if (to >= g.T || v0 >= g.V) continue;
      unsigned char* p = static_cast<unsigned char*>(g.y) + ((int64_t)to * g.ldy + v0) * kSize;
      if (v0 + 16 / kSize <= g.V) {
        *reinterpret_cast<u32x4u*>(p) = v;
      } else if constexpr (EXACT) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (v0 + e < g.V) reinterpret_cast<uint32_t*>(p)[e] = v[e];
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (v0 + e < g.V) reinterpret_cast<uint16_t*>(p)[e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
      }
    }
  }
}

}  // namespace fp8
}  // namespace hcg
