// hcg_embed.hip -- the embedding lookup and its gradient (include/hcg_lm.h).
//
// Forward: out[i] = scale * table[ids[i]], a gather of whole rows; bound by
// HBM.  Every thread has four 16-byte loads in flight, whatever the row's width:
// the rows of a workgroup are one range of vectors.  8192 of 65536 x 4096 bf16
// 19.1 us, of which the writes (67 MB) alone are 13.
//
// Gradient: grad[v] = scale * sum of dy[i] over ids[i] == v.  Each workgroup
// owns a few rows of the table.  It reads all ids (64 KB for 8192 tokens, from
// the L2), keeps those of its rows in the order of i, groups them by row and
// writes every row once: zeros, or the float32 sum over ascending i.  No
// atomics on values, no sorting passes and no launch between them; a row's
// order of additions depends on the ids alone.  A row that many tokens name
// (natural text: one word is several percent of a batch) would keep one
// workgroup busy long after the others, so the tokens of rows with more than
// kLong of them are left in a list, in the order of (row, i), which a second
// launch sums in windows of kWindow entries and a third adds up by rows.
// Bound by the table's writes, most of them zeros: a pass over 65536 x 4096 bf16
// with 8192 tokens 115 us on the same inputs and 125 on new ones, for 537 MB (and
// 67 MB read); its first launch 105.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "hcg_vec.h"

namespace {

using hcg::ElemOf;
using hcg::kVec;
using hcg::raw4;

// ---------------------------------------------------------------------------
// Lookup
// ---------------------------------------------------------------------------

struct EmbedArgs {
  const void* table;
  const void* ids;
  void* out;
  int64_t ldt, ldo, vocab, n;
  int width, vecs, rows_per_wg;  // vecs: 16-byte vectors in a row
  float scale;
};

constexpr int kEmbedPer = 4;  // vectors per thread and turn

template <class T, class I>
__global__ __launch_bounds__(256) void embed_kernel(EmbedArgs g) {
  constexpr int E = kVec<T>;
  const int64_t row0 = hcg::workgroup() * g.rows_per_wg;
  if (row0 >= g.n) return;
  const int rows = (int)min((int64_t)g.rows_per_wg, g.n - row0);
  const int total = rows * g.vecs;
  const I* ids = static_cast<const I*>(g.ids) + row0;
  const T* table = static_cast<const T*>(g.table);
  T* out = static_cast<T*>(g.out);
  for (int base = threadIdx.x; base < total; base += 256 * kEmbedPer) {
    raw4 raw[kEmbedPer];
    int at_row[kEmbedPer], at_col[kEmbedPer];
    bool known[kEmbedPer];
#pragma unroll
    for (int u = 0; u < kEmbedPer; ++u) {
      const int i = base + u * 256;
      if (i < total) {
        const int r = i / g.vecs, c = (i - r * g.vecs) * E;
        const int64_t id = (int64_t)ids[r];
        at_row[u] = r;
        at_col[u] = c;
        known[u] = id >= 0 && id < g.vocab;
        raw[u] = known[u] ? hcg::load_raw(table + id * g.ldt + c, g.width - c) : raw4{0, 0, 0, 0};
      }
    }
#pragma unroll
    for (int u = 0; u < kEmbedPer; ++u) {
      if (base + u * 256 < total) {
        float f[E];
        hcg::unpack<T>(raw[u], f);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          f[e] = known[u] ? f[e] * g.scale : __builtin_nanf("");
          // The product is a float32 before it is rounded to T.  (For f16 the
          // compiler would make both one mixed-precision instruction, which
          // rounds once and turns -0 into 0.)
          asm("" : "+v"(f[e]));
        }
        hcg::store_raw(out + (row0 + at_row[u]) * g.ldo + at_col[u], hcg::pack<T>(f), g.width - at_col[u]);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Gradient
// ---------------------------------------------------------------------------

constexpr int kGradThreads = 512;
constexpr int kGradWaves = kGradThreads / 64;
constexpr int kScan = 4;           // pairs of ids in flight per lane
constexpr int kMaxRows = 64;       // table rows per workgroup
constexpr int kListPerWave = 256;  // ids of a workgroup's rows kept in LDS, per wave that scans
// Rows of dy in flight per thread.  (16 take registers that leave two workgroups
// per CU instead of four: 999 tokens of 515 f32 into 5003 rows 13.6 us with 8,
// 18.7 with 16.)
constexpr int kSumLoads = 8;
constexpr int kLong = 16;
constexpr int kWindow = 32;
// Runs of long rows in one window: those that lie inside it have more than
// kLong entries each, and one more may enter and one leave.
constexpr int kRuns = kWindow / (kLong + 1) + 2;
// Few tokens of narrow rows: a workgroup sums its long rows too, in parts that
// meet in LDS, and one launch does it all.  Up to kOneLaunch tokens where a row has
// at most half as many items as there are threads, up to twice as many, by lists
// twice as long (54 KB of LDS: 3 workgroups per CU, not 4), where it has at most a
// quarter.  us, one launch / three: 3160 into 5065 x 131 f32 14.6 / 24.9, 2273 into
// 6920 x 463 f32 17.0 / 24.8, but 3720 into 731 x 1336 f16 (167 items) 28.6 / 23.7;
// long lists / short ones: 2048 into 13384 x 128 bf16 15.0 / 12.1.
constexpr int kOneLaunch = 2048;
// Past so many tokens they are first parted by ranges of the table (a launch of
// kBuckets workgroups, stable), and a workgroup scans its range's tokens only:
// 4096 workgroups that scan them all read 1 GB from the L2s at 32768 tokens.
// us, all scanned / parted: 32768 into 108888 x 512 f16 80 / 71, 65536 into 32768
// x 1024 bf16 181 / 141, 8192 into 65536 x 4096 117 / 119, 5000 into 5000 x 512
// f32 25.8 / 26.4.
constexpr int kBucketTokens = 8192;
constexpr int kBuckets = 64;

// Runs of empty rows of up to so many vectors are filled by a wave each, longer
// ones by the workgroup.
constexpr int kShortRun = 64 * 4;

struct EmbedGradArgs {
  const void* dy;
  const void* ids;
  void* grad;
  int64_t lddy, ldg, vocab, padding;
  int n;
  int width, items;  // items: dy's whole 16-byte vectors in a row, and the elements past them
  int rows;         // table rows per workgroup
  float scale;
  // Lists over the tokens in the order of (row, i).
  int* token;     // i (null: one launch)
  int* row;       // the long row it belongs to, or -1
  int* run_len;   // (at a long row's first entry) its tokens
  int* found;     // tokens of a workgroup's rows in the order of i, where LDS is too small ...
  uint16_t* found_row;  // ... and which of its rows
  float* part;    // [windows][kRuns][width]
  // Parted tokens, or null: their rows and indexes by bucket of bucket_rows
  // table rows, and each bucket's first place and number of tokens.
  int* bucket_id;
  int* bucket_token;
  int* bucket;  // [kBuckets][2]
  int bucket_rows;
};

__device__ __forceinline__ int lanes_below(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi((unsigned)(mask >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)mask, 0));
}

// f[0..E) of dy scaled, as the sum's rounding to G and one 16- or 32-byte store.
template <bool WHOLE, class T, class G>
__device__ __forceinline__ void store_grad(G* p, const float (&f)[kVec<T>], float scale) {
  constexpr int E = kVec<T>, EG = kVec<G>;
  if constexpr (!WHOLE) {
    *p = (G)(f[0] * scale);
  } else {
#pragma unroll
    for (int h = 0; h < E / EG; ++h) {
      float o[EG];
#pragma unroll
      for (int e = 0; e < EG; ++e) o[e] = f[h * EG + e] * scale;
      hcg::store_raw(p + h * EG, hcg::pack<G>(o), EG);
    }
  }
}

// n zeros from p on by `threads` threads (64 or more), this one number `thread`:
// whole 128-byte lines as non-temporal vectors, the elements before and after
// them one by one.
template <class G>
__device__ __forceinline__ void fill_zeros(G* p, int64_t n, int thread, int threads) {
  constexpr int kLine = 128 / (int)sizeof(G);
  const int64_t to_line = (kLine - (int)(reinterpret_cast<uintptr_t>(p) % 128) / (int)sizeof(G)) % kLine;
  const int head = (int)min(n, to_line);
  if (thread < head) p[thread] = (G)0.f;
  p += head;
  const int64_t vecs = (n - head) / kLine * 8, tail = n - head - vecs * kVec<G>;
  for (int64_t i = thread; i < vecs; i += threads)
    hcg::store_raw<true>(p + i * kVec<G>, raw4{0, 0, 0, 0}, kVec<G>);
  if (thread < tail) p[vecs * kVec<G> + thread] = (G)0.f;
}

// A row as whole vectors and, one by one, the elements past them: items
// 0 .. items - 1.  A thread's item is WHOLE (E elements) or one element, so that
// no load asks how much of it is in the row.
struct Items {
  int whole, items;
  __device__ Items(int width, int E) : whole(width / E), items(width / E + width % E) {}
};

// sum[e] += the rows of dy (from the item's first element on) that entries
// 0 .. n - 1 name, in order.
template <bool WHOLE, class T, class F>
__device__ __forceinline__ void sum_rows(float (&sum)[kVec<T>], const T* dy, int64_t lddy, int n, F entry) {
  constexpr int E = kVec<T>, W = WHOLE ? E : 1;
  // (The last rows go out together as well, each if there is one: in batches
  // of 4, 2 and 1 they waited for each other, 129 us against 104.)
  for (int j = 0; j < n; j += kSumLoads) {
    raw4 raw[kSumLoads];
    T one[kSumLoads];
#pragma unroll
    for (int u = 0; u < kSumLoads; ++u)
      if (j + u < n) {
        const T* p = dy + (int64_t)entry(j + u) * lddy;
        if constexpr (WHOLE)
          raw[u] = hcg::load_raw(p, E);
        else
          one[u] = *p;
      }
#pragma unroll
    for (int u = 0; u < kSumLoads; ++u)
      if (j + u < n) {
        float f[E];
        if constexpr (WHOLE)
          hcg::unpack<T>(raw[u], f);
        else
          f[0] = (float)one[u];
#pragma unroll
        for (int e = 0; e < W; ++e) sum[e] += f[e];
      }
  }
}

// The ids [from, to) by one wave, two neighbours per lane: f(i, a, b) with the
// ids of i and i + 1, -1 past the end and for the padding row; kScan loads in
// flight.
template <class I, class F>
__device__ __forceinline__ void scan_ids(const I* ids, int from, int to, int64_t padding, F f) {
  typedef I pair __attribute__((ext_vector_type(2), aligned(sizeof(I))));
  const int lane = threadIdx.x & 63;
  for (int i0 = from; i0 < to; i0 += 128 * kScan) {
    int64_t a[kScan], b[kScan];
#pragma unroll
    for (int u = 0; u < kScan; ++u) {
      const int i = i0 + u * 128 + lane * 2;
      a[u] = b[u] = -1;
      if (i + 1 < to) {
        const pair v = *reinterpret_cast<const pair*>(ids + i);
        a[u] = (int64_t)v.x;
        b[u] = (int64_t)v.y;
      } else if (i < to) {
        a[u] = (int64_t)ids[i];
      }
      if (a[u] == padding) a[u] = -1;
      if (b[u] == padding) b[u] = -1;
    }
#pragma unroll
    for (int u = 0; u < kScan; ++u)
      if (i0 + u * 128 < to) f(i0 + u * 128 + lane * 2, a[u], b[u]);
  }
}

// Over scan_ids: counts the ids below `lo` into *below and those in [lo, hi)
// into *finds, which it hands over in order: keep(number, i, id).
template <class I, class F>
__device__ __forceinline__ void find_ids(const I* ids, int from, int to, int64_t padding, int64_t lo, int64_t hi,
                                         int* finds, int* below, F keep) {
  const int lane = threadIdx.x & 63;
  int found = 0, under = 0;
  scan_ids<I>(ids, from, to, padding, [&](int i, int64_t a, int64_t b) {
    under += __popcll(__ballot(a >= 0 && a < lo)) + __popcll(__ballot(b >= 0 && b < lo));
    const uint64_t hit_a = __ballot(a >= lo && a < hi), hit_b = __ballot(b >= lo && b < hi);
    if (hit_a | hit_b) {
      const int at = found + lanes_below(hit_a) + lanes_below(hit_b);
      const bool mine_a = hit_a >> lane & 1;
      if (mine_a) keep(at, i, a);
      if (hit_b >> lane & 1) keep(at + mine_a, i + 1, b);
      found += __popcll(hit_a) + __popcll(hit_b);
    }
  });
  *finds = found;
  *below = under;
}

// Parts the tokens: workgroup b takes those of its bucket_rows rows of the
// table, in order, to the places after all of lower rows.  The finds wait in
// LDS until their place is known; where they do not fit (a hot row) the ids are
// scanned again, from the L2.  Bound by the latency of reading all ids once by
// each of 64 workgroups (32768 tokens: about 10 us).
constexpr int kPartThreads = 1024;
constexpr int kPartWaves = kPartThreads / 64;
constexpr int kPartList = 512;  // finds per wave
template <class I>
__global__ __launch_bounds__(kPartThreads) void embed_bucket_kernel(EmbedGradArgs g) {
  __shared__ int wave_found[kPartWaves], wave_below[kPartWaves];
  __shared__ int list_id[kPartWaves * kPartList], list_token[kPartWaves * kPartList];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t lo = (int64_t)blockIdx.x * g.bucket_rows, hi = min(lo + g.bucket_rows, g.vocab);
  const I* ids = static_cast<const I*>(g.ids);
  const int quota = (g.n + kPartWaves * 128 - 1) / (kPartWaves * 128) * 128;
  const int from = min(wave * quota, g.n), to = min(from + quota, g.n);
  int finds, below;
  find_ids<I>(ids, from, to, g.padding, lo, hi, &finds, &below, [&](int at, int i, int64_t id) {
    if (at < kPartList) {
      list_id[wave * kPartList + at] = (int)id;
      list_token[wave * kPartList + at] = i;
    }
  });
  if (lane == 0) wave_found[wave] = finds, wave_below[wave] = below;
  __syncthreads();
  int total = 0, first = 0, base = 0;
#pragma unroll
  for (int w = 0; w < kPartWaves; ++w) {
    if (w < wave) first += wave_found[w];
    total += wave_found[w];
    base += wave_below[w];
  }
  if (threadIdx.x == 0) g.bucket[2 * blockIdx.x] = base, g.bucket[2 * blockIdx.x + 1] = total;
  first += base;
  if (finds <= kPartList) {  // (this wave's own finds)
    for (int j = lane; j < finds; j += 64) {
      g.bucket_id[first + j] = list_id[wave * kPartList + j];
      g.bucket_token[first + j] = list_token[wave * kPartList + j];
    }
  } else {
    find_ids<I>(ids, from, to, g.padding, lo, hi, &finds, &below, [&](int at, int i, int64_t id) {
      g.bucket_id[first + at] = (int)id;
      g.bucket_token[first + at] = i;
    });
  }
}

// ONE: no lists are kept (g.token is null), the workgroup sums its long rows too;
// the finds per wave that LDS has room for.
// PARTED: the tokens come from the workgroup's bucket (I is int).
template <class T, class G, class I, int ONE, bool PARTED>
__global__ __launch_bounds__(kGradThreads, ONE > kListPerWave ? 6 : 8) void embed_grad_kernel(EmbedGradArgs g) {
  constexpr int E = kVec<T>, kList = ONE ? ONE : kListPerWave;
  __shared__ float meet[ONE ? kGradThreads * E : 1];
  __shared__ int found[kGradWaves * kList], grouped[kGradWaves * kList];
  __shared__ uint8_t found_row[kGradWaves * kList];
  __shared__ int wave_found[kGradWaves], wave_below[kGradWaves];
  __shared__ int count[kMaxRows], start[kMaxRows];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t lo = (int64_t)blockIdx.x * g.rows;
  const int rows = (int)min((int64_t)g.rows, g.vocab - lo);
  const int bucket = PARTED ? (int)(lo / g.bucket_rows) : 0;
  const int base = PARTED ? g.bucket[2 * bucket] : 0, tokens = PARTED ? g.bucket[2 * bucket + 1] : g.n;
  const I* ids = PARTED ? reinterpret_cast<const I*>(g.bucket_id + base) : static_cast<const I*>(g.ids);
  for (int r = tid; r < kMaxRows; r += kGradThreads) count[r] = 0;

  // Wave w scans the tokens [w * quota, (w + 1) * quota): its finds and, for
  // the place of this workgroup's tokens in the lists, how many name a row
  // before the first of these.  `keep` takes the find at its place.
  const int quota = (tokens + kGradWaves * 128 - 1) / (kGradWaves * 128) * 128;
  const int from = min(wave * quota, tokens), to = min(from + quota, tokens);
  auto scan = [&](auto keep) {
    int finds, below;
    find_ids<I>(ids, from, to, g.padding, lo, lo + rows, &finds, &below, [&](int at, int i, int64_t id) {
      keep(at, PARTED ? g.bucket_token[base + i] : i, (int)(id - lo));
    });
    if (lane == 0) wave_found[wave] = finds, wave_below[wave] = below;
  };
  scan([&](int at, int i, int r) {
    if (at < kList) {
      found[wave * kList + at] = i;
      found_row[wave * kList + at] = (uint8_t)r;
    }
  });
  __syncthreads();
  int total = 0, before = 0, below = base;
  bool fits = true;
#pragma unroll
  for (int w = 0; w < kGradWaves; ++w) {
    if (w < wave) before += wave_found[w];
    total += wave_found[w];
    below += wave_below[w];
    fits = fits && wave_found[w] <= kList;
  }
  if (!ONE && !fits) {
    // (wave_found and wave_below are written again with the same values)
    scan([&](int at, int i, int r) {
      g.found[below + before + at] = i;
      g.found_row[below + before + at] = (uint16_t)r;
    });
    __syncthreads();
  }

  // Find number j of wave w.
  auto find = [&](int w, int off, int j, int& i) -> int {
    if (ONE || fits) {
      i = found[w * kList + j];
      return found_row[w * kList + j];
    }
    i = g.found[below + off + j];
    return g.found_row[below + off + j];
  };
  for (int j = lane; j < wave_found[wave]; j += 64) {
    int i;
    atomicAdd(&count[find(wave, before, j, i)], 1);
  }
  __syncthreads();
  if (wave == 0) {
    int c = lane < kMaxRows ? count[lane] : 0, sum = c;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const int up = __shfl_up(sum, m);
      if (lane >= m) sum += up;
    }
    start[lane] = sum - c;
  }
  __syncthreads();
  // Group by row, stably: a wave takes every kGradWaves-th row and passes
  // over all finds.
  for (int r = wave; r < rows; r += kGradWaves) {
    const int c = count[r];
    if (c == 0) continue;
    int put = start[r], off = 0;
    for (int w = 0; w < kGradWaves; ++w) {
      for (int j0 = 0; j0 < wave_found[w]; j0 += 64) {
        int i = 0;
        const bool mine = j0 + lane < wave_found[w] && find(w, off, j0 + lane, i) == r;
        const uint64_t hit = __ballot(mine);
        if (mine) {
          const int at = put + lanes_below(hit);
          if (ONE || fits) grouped[at] = i;
          if (!ONE) g.token[below + at] = i;
        }
        put += __popcll(hit);
      }
      off += wave_found[w];
    }
    if (!ONE) {
      for (int j = lane; j < c; j += 64) g.row[below + start[r] + j] = c > kLong ? (int)(lo + r) : -1;
      if (c > kLong && lane == 0) g.run_len[below + start[r]] = c;
    }
  }
  // The places past all tokens (ids that name no row) belong to no long row.
  if (!ONE && lo + rows == g.vocab)
    for (int j = below + total + tid; j < g.n; j += kGradThreads) g.row[j] = -1;
  __syncthreads();

  // The rows without tokens: neighbours together, where the gradient has no
  // gaps, so that lines are written whole whatever the width, and past the
  // caches.  us of a pass, row by row / so / so without non-temporal stores: 8192
  // tokens into 65536 x 4096 bf16 117 / 115 / 146, 200 into 36696 x 3400 f32 102 /
  // 102 / 110, 1353 into 24661 x 1367 f32 49 / 45 / 44, 2048 into 13384 x 128 bf16
  // 15.3 / 11.8 / 11.8.
  const T* dy = static_cast<const T*>(g.dy);
  G* grad = static_cast<G*>(g.grad);
  uint64_t empty = __ballot(lane < rows && count[lane] == 0);
  for (int run = 0; empty; ++run) {
    const int first = __ffsll((unsigned long long)empty) - 1;
    const uint64_t past = ~(empty >> first);  // (0: all 64 rows)
    const int len = g.ldg != g.width ? 1 : past ? __ffsll((unsigned long long)past) - 1 : 64;
    G* p = grad + (lo + first) * g.ldg;
    const int64_t n = (int64_t)len * g.width;
    if (n > kShortRun * kVec<G>)
      fill_zeros<G>(p, n, tid, kGradThreads);
    else if (run % kGradWaves == wave)
      fill_zeros<G>(p, n, lane, 64);
    empty &= first + len >= 64 ? 0 : ~(uint64_t)0 << (first + len);
  }

  // Every row that is neither empty nor long, its items over the threads.
  const Items it(g.width, E);
  const auto entry = [&](int j) { return ONE || fits ? grouped[j] : g.token[below + j]; };
  const int work = rows * it.items;
  for (int at = tid; at < work; at += kGradThreads) {
    const int r = at / it.items, i = at - r * it.items;
    const int n = count[r], first = start[r];
    if (n == 0 || n > kLong) continue;
    const auto one_item = [&](auto whole, int c) {
      constexpr bool WHOLE = decltype(whole)::value;
      float sum[E] = {};
      sum_rows<WHOLE, T>(sum, dy + c, g.lddy, n, [&](int j) { return entry(first + j); });
      store_grad<WHOLE, T, G>(grad + (lo + r) * g.ldg + c, sum, g.scale);
    };
    if (i < it.whole)
      one_item(std::true_type{}, i * E);
    else
      one_item(std::false_type{}, it.whole * E + i - it.whole);
  }
  if constexpr (!ONE) return;

  // A long row's entries in `parts` runs, a group of threads each (the row's
  // items are at most half the threads, and few tokens always fit the lists).
  const int parts = kGradThreads / it.items, part = tid / it.items, i = tid - part * it.items;
  for (int r = 0; r < rows; ++r) {
    const int n = count[r];
    if (n <= kLong) continue;
    const int first = start[r] + n * part / parts, len = start[r] + n * (part + 1) / parts - first;
    const auto one_item = [&](auto whole, int c) {
      constexpr bool WHOLE = decltype(whole)::value;
      constexpr int W = WHOLE ? E : 1;
      float sum[E] = {};
      if (part < parts)
        sum_rows<WHOLE, T>(sum, dy + c, g.lddy, len, [&](int j) { return entry(first + j); });
#pragma unroll
      for (int e = 0; e < W; ++e) meet[e * kGradThreads + tid] = sum[e];
    };
    const bool whole = i < it.whole;
    const int c = whole ? i * E : it.whole * E + i - it.whole;
    if (whole)
      one_item(std::true_type{}, c);
    else
      one_item(std::false_type{}, c);
    __syncthreads();
    if (part == 0) {
      float sum[E];
#pragma unroll
      for (int e = 0; e < E; ++e) sum[e] = meet[e * kGradThreads + tid];
      for (int q = 1; q < parts; ++q)
#pragma unroll
        for (int e = 0; e < E; ++e) sum[e] += meet[e * kGradThreads + q * it.items + tid];
      G* p = grad + (lo + r) * g.ldg + c;
      if (whole)
        store_grad<true, T, G>(p, sum, g.scale);
      else
        store_grad<false, T, G>(p, sum, g.scale);
    }
    __syncthreads();
  }
}

// The entries of a window (a lane each): which belong to a long row, and of
// these which are the first of a run in the window.
struct Window {
  uint64_t in_long, starts;
};
__device__ __forceinline__ Window window_of(const EmbedGradArgs& g, int from, int n, int lane, int* row) {
  const int mine = lane < n ? g.row[from + lane] : -1;
  const int left = __shfl_up(mine, 1);
  *row = mine;
  return Window{__ballot(mine >= 0), __ballot(mine >= 0 && (lane == 0 || mine != left))};
}

// Window blockIdx.x of the lists, items blockIdx.y * 256 ...: the sum of
// each run of one long row in it.  A run is at most 32 rows by one thread per
// 16 bytes, eight loads in flight: bound by their latency where a few words make
// up most of the windows (8192 tokens x 4096 bf16, a third in long rows: 8 us).
template <class T>
__global__ __launch_bounds__(256) void embed_window_kernel(EmbedGradArgs g) {
  constexpr int E = kVec<T>;
  __shared__ int token[kWindow];
  const int from = blockIdx.x * kWindow, n = min(kWindow, g.n - from), lane = threadIdx.x & 63;
  int row;
  const Window w = window_of(g, from, n, lane, &row);
  if (w.in_long == 0) return;
  if ((int)threadIdx.x < n) token[threadIdx.x] = g.token[from + threadIdx.x];
  __syncthreads();
  const Items it(g.width, E);
  const int i = blockIdx.y * 256 + threadIdx.x;
  if (i >= it.items) return;
  const bool whole = i < it.whole;
  const int c = whole ? i * E : it.whole * E + i - it.whole;
  float* part = g.part + (int64_t)blockIdx.x * kRuns * g.width + c;
  for (uint64_t starts = w.starts; starts; starts &= starts - 1) {
    const int first = __ffsll((unsigned long long)starts) - 1;
    // The run ends before the next start or the next entry of no long row.
    const uint64_t ends = ((starts & (starts - 1)) | ~w.in_long) >> first >> 1;
    const int len = __ffsll((unsigned long long)ends);
    const T* dy = static_cast<const T*>(g.dy) + c;
    const auto entry = [&](int j) { return token[first + j]; };
    float sum[E] = {};
    if (whole) {
      sum_rows<true, T>(sum, dy, g.lddy, len, entry);
#pragma unroll
      for (int e = 0; e < E; ++e) part[e] = sum[e];
    } else {
      sum_rows<false, T>(sum, dy, g.lddy, len, entry);
      part[0] = sum[0];
    }
    part += g.width;
  }
}

// The long rows that start in window blockIdx.x, columns blockIdx.y * 256 ...:
// their windows' sums, in order (7 us at the size above: one chain of float32
// loads, 16 in flight, of the most frequent row's windows).
template <class G>
__global__ __launch_bounds__(256) void embed_long_kernel(EmbedGradArgs g) {
  const int from = blockIdx.x * kWindow, n = min(kWindow, g.n - from), lane = threadIdx.x & 63;
  int row;
  const Window w = window_of(g, from, n, lane, &row);
  // A run that goes on from the window before is that window's business.
  const int before = from > 0 ? g.row[from - 1] : -1;
  uint64_t starts = w.starts;
  int run = 0;
  if ((starts & 1) && before == __shfl(row, 0)) starts &= ~(uint64_t)1, run = 1;
  const int64_t c = (int64_t)blockIdx.y * 256 + threadIdx.x;
  for (; starts; starts &= starts - 1, ++run) {
    const int first = __ffsll((unsigned long long)starts) - 1;
    const int v = __shfl(row, first);
    if (c >= g.width) continue;
    const int len = g.run_len[from + first];
    const int windows = (from + first + len - 1) / kWindow - (int)blockIdx.x;  // after this one
    float sum = g.part[((int64_t)blockIdx.x * kRuns + run) * g.width + c];
    const float* next = g.part + (int64_t)(blockIdx.x + 1) * kRuns * g.width + c;
#pragma unroll 16
    for (int q = 0; q < windows; ++q) sum += next[(int64_t)q * kRuns * g.width];
    static_cast<G*>(g.grad)[(int64_t)v * g.ldg + c] = (G)(sum * g.scale);
  }
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------

constexpr int64_t kMaxTokens = (int64_t)1 << 30;
// Tokens and rows of the gradient: fewer than 2^32 threads to a launch.
constexpr int64_t kMaxGrad = (int64_t)1 << 28;

int64_t items_of(int dtype, int64_t width) {
  const int64_t e = 16 / hcg::elem_bytes(dtype);
  return width / e + width % e;
}
bool one_launch(int64_t n, int64_t items) {
  return n <= kLong || (n <= kOneLaunch && items <= kGradThreads / 2) ||
         (n <= 2 * kOneLaunch && items <= kGradThreads / 4);
}
int64_t windows_of(int64_t n) { return (n + kWindow - 1) / kWindow; }
int64_t round256(int64_t b) { return (b + 255) / 256 * 256; }

template <class F>
void with_elem(int dtype, F f) {
  if (dtype == HCG_F16)
    f(ElemOf<HCG_F16>::type{});
  else if (dtype == HCG_BF16)
    f(ElemOf<HCG_BF16>::type{});
  else
    f(float{});
}

template <class T, class G, class I>
void run_embed_grad(const EmbedGradArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)((a.vocab + a.rows - 1) / a.rows));
  if (a.token == nullptr) {
    if (a.n <= kOneLaunch)
      embed_grad_kernel<T, G, I, kListPerWave, false><<<grid, kGradThreads, 0, s>>>(a);
    else
      embed_grad_kernel<T, G, I, 2 * kListPerWave, false><<<grid, kGradThreads, 0, s>>>(a);
    return;
  }
  if (a.bucket) {
    const dim3 buckets((unsigned)((a.vocab + a.bucket_rows - 1) / a.bucket_rows));
    embed_bucket_kernel<I><<<buckets, kPartThreads, 0, s>>>(a);
    embed_grad_kernel<T, G, int32_t, 0, true><<<grid, kGradThreads, 0, s>>>(a);
  } else {
    embed_grad_kernel<T, G, I, 0, false><<<grid, kGradThreads, 0, s>>>(a);
  }
  const unsigned windows = (unsigned)windows_of(a.n);
  embed_window_kernel<T><<<dim3(windows, (unsigned)((a.items + 255) / 256)), 256, 0, s>>>(a);
  embed_long_kernel<G><<<dim3(windows, (unsigned)((a.width + 255) / 256)), 256, 0, s>>>(a);
}

}  // namespace

extern "C" {

int hcg_embedding(int dtype, const void* table, int64_t ldt, int64_t vocab, int64_t width, int id_bytes,
                  const void* ids, int64_t n, float scale, void* out, int64_t ldo, void* stream) {
  HCG_LM_REQUIRE(hcg::elem_ok(dtype), "dtype %d is not HCG_F16, HCG_BF16 or HCG_F32", dtype);
  HCG_LM_REQUIRE(id_bytes == 4 || id_bytes == 8, "ids are 4 or 8 bytes, not %d", id_bytes);
  HCG_LM_REQUIRE(n >= 0 && n < kMaxTokens && vocab >= 0 && width >= 0 && width < ((int64_t)1 << 30),
                 "%lld ids into %lld rows of %lld elements are out of range", (long long)n, (long long)vocab,
                 (long long)width);
  if (n == 0 || width == 0) return HCG_OK;
  const int eb = hcg::elem_bytes(dtype);
  HCG_LM_REQUIRE((table || vocab == 0) && ids && out, "null pointer");
  HCG_LM_REQUIRE((vocab <= 1 || ldt >= width) && (n == 1 || ldo >= width), "row stride below the width %lld",
                 (long long)width);
  HCG_LM_REQUIRE(hcg::elem_aligned(table, eb) && hcg::elem_aligned(out, eb) && hcg::elem_aligned(ids, id_bytes),
                 "rows and ids must be aligned to their elements");
  EmbedArgs a{table, ids, out, ldt, ldo, vocab, n, (int)width, 0, 0, scale};
  a.vecs = (int)((width * eb + 15) / 16);
  a.rows_per_wg = std::max(1, 256 * kEmbedPer / a.vecs);
  const dim3 grid = hcg::grid_of((n + a.rows_per_wg - 1) / a.rows_per_wg);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  with_elem(dtype, [&](auto t) {
    using T = decltype(t);
    if (id_bytes == 8)
      embed_kernel<T, int64_t><<<grid, 256, 0, s>>>(a);
    else
      embed_kernel<T, int32_t><<<grid, 256, 0, s>>>(a);
  });
  HCG_LM_HIP_CHECK(hipGetLastError());
  return HCG_OK;
}

int64_t hcg_embedding_grad_workspace(int dtype, int64_t n, int64_t vocab, int64_t width) {
  if (vocab <= 0 || width <= 0 || n >= kMaxGrad || one_launch(n, items_of(dtype, width))) return 0;
  const int64_t parted = n > kBucketTokens ? 2 * round256(n * 4) + round256(kBuckets * 8) : 0;
  return 4 * round256(n * 4) + round256(n * 2) + parted + windows_of(n) * kRuns * width * 4;
}

int hcg_embedding_grad(int dtype, const void* dy, int64_t lddy, int64_t n, int64_t width, int id_bytes,
                       const void* ids, int64_t vocab, int64_t padding_idx, float scale, int grad_dtype,
                       void* grad, int64_t ldg, void* workspace, int64_t workspace_bytes, void* stream) {
  HCG_LM_REQUIRE(hcg::elem_ok(dtype), "dtype %d is not HCG_F16, HCG_BF16 or HCG_F32", dtype);
  HCG_LM_REQUIRE(grad_dtype == dtype || grad_dtype == HCG_F32, "the gradient has the type of dy or float32");
  HCG_LM_REQUIRE(id_bytes == 4 || id_bytes == 8, "ids are 4 or 8 bytes, not %d", id_bytes);
  HCG_LM_REQUIRE(n >= 0 && n < kMaxGrad && vocab >= 0 && vocab < kMaxGrad && width >= 0 &&
                     width < ((int64_t)1 << 23),
                 "%lld ids into %lld rows of %lld elements are out of range", (long long)n, (long long)vocab,
                 (long long)width);
  if (vocab == 0 || width == 0) return HCG_OK;
  const int eb = hcg::elem_bytes(dtype);
  HCG_LM_REQUIRE(grad && (n == 0 || (dy && ids)), "null pointer");
  HCG_LM_REQUIRE((n <= 1 || lddy >= width) && (vocab == 1 || ldg >= width), "row stride below the width %lld",
                 (long long)width);
  HCG_LM_REQUIRE(hcg::elem_aligned(dy, eb) && hcg::elem_aligned(grad, hcg::elem_bytes(grad_dtype)) &&
                     hcg::elem_aligned(ids, id_bytes),
                 "rows and ids must be aligned to their elements");
  const int64_t need = hcg_embedding_grad_workspace(dtype, n, vocab, width);
  HCG_LM_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && hcg::elem_aligned(workspace, 256)),
                 "workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
  EmbedGradArgs a{};
  a.dy = dy;
  a.ids = ids;
  a.grad = grad;
  a.lddy = lddy;
  a.ldg = ldg;
  a.vocab = vocab;
  a.padding = padding_idx < 0 ? -1 : padding_idx;
  a.n = (int)n;
  a.width = (int)width;
  a.items = (int)items_of(dtype, width);
  // A small table in one round of workgroups (1024), a large one in up to four,
  // so that some scan the ids while others write (65536 x 4096 bf16: 1024
  // workgroups 130 us, 4096 115).
  const int64_t quick = std::min((vocab + 1023) / 1024, std::max<int64_t>(1, (128 << 10) / (width * eb)));
  a.rows = (int)std::min<int64_t>(kMaxRows, std::max((vocab + 4095) / 4096, quick));
  a.scale = scale;
  if (need > 0) {
    char* p = static_cast<char*>(workspace);
    a.token = reinterpret_cast<int*>(p);
    a.row = reinterpret_cast<int*>(p += round256(n * 4));
    a.run_len = reinterpret_cast<int*>(p += round256(n * 4));
    a.found = reinterpret_cast<int*>(p += round256(n * 4));
    a.found_row = reinterpret_cast<uint16_t*>(p += round256(n * 4));
    p += round256(n * 2);
    if (n > kBucketTokens) {
      a.bucket_id = reinterpret_cast<int*>(p);
      a.bucket_token = reinterpret_cast<int*>(p += round256(n * 4));
      a.bucket = reinterpret_cast<int*>(p += round256(n * 4));
      p += round256(kBuckets * 8);
      // (whole workgroups' rows: a workgroup's lie in one bucket)
      a.bucket_rows = (int)((vocab + (int64_t)kBuckets * a.rows - 1) / ((int64_t)kBuckets * a.rows) * a.rows);
    }
    a.part = reinterpret_cast<float*>(p);
  }
  const hipStream_t s = static_cast<hipStream_t>(stream);
  with_elem(dtype, [&](auto t) {
    using T = decltype(t);
    const auto by_ids = [&](auto g) {
      using G = decltype(g);
      if (id_bytes == 8)
        run_embed_grad<T, G, int64_t>(a, s);
      else
        run_embed_grad<T, G, int32_t>(a, s);
    };
    if (grad_dtype == HCG_F32)
      by_ids(float{});
    else
      by_ids(t);
  });
  HCG_LM_HIP_CHECK(hipGetLastError());
  return HCG_OK;
}

}  // extern "C"
