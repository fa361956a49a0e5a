// hcg_embed.hip -- the embedding lookup and its gradient (include/hcg_lm.h).
//
// Forward: out[i] = scale * table[ids[i]], a gather of whole rows; bound by
// HBM.
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
  const int64_t row0 = (int64_t)blockIdx.x * g.rows_per_wg;
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

constexpr int kGradThreads = 256;
constexpr int kGradWaves = kGradThreads / 64;
constexpr int kScan = 8;           // ids in flight per lane
constexpr int kMaxRows = 64;       // table rows per workgroup
constexpr int kListPerWave = 512;  // ids of a workgroup's rows kept in LDS, per wave that scans
constexpr int kLong = 32;
constexpr int kWindow = 64;
// Runs of long rows in one window: those that lie inside it have more than
// kLong entries each, and one more may enter and one leave.
constexpr int kRuns = kWindow / (kLong + 1) + 2;

struct EmbedGradArgs {
  const void* dy;
  const void* ids;
  void* grad;
  int64_t lddy, ldg, vocab, padding;
  int n;
  int width, vecs;  // vecs: 16-byte vectors of dy in a row
  int rows;         // table rows per workgroup
  float scale;
  // Lists over the tokens in the order of (row, i).
  int* token;     // i
  int* row;       // the long row it belongs to, or -1
  int* run_len;   // (at a long row's first entry) its tokens
  int* found;     // tokens of a workgroup's rows in the order of i, where LDS is too small ...
  uint16_t* found_row;  // ... and which of its rows
  float* part;    // [windows][kRuns][width]
};

__device__ __forceinline__ int lanes_below(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi((unsigned)(mask >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)mask, 0));
}

// f[0..E) of dy scaled, as the sum's rounding to G and one 16- or 32-byte store.
template <class T, class G>
__device__ __forceinline__ void store_grad(G* p, const float (&f)[kVec<T>], float scale, int valid) {
  constexpr int E = kVec<T>, EG = kVec<G>;
#pragma unroll
  for (int h = 0; h < E / EG; ++h) {
    float o[EG];
#pragma unroll
    for (int e = 0; e < EG; ++e) o[e] = f[h * EG + e] * scale;
    if (h * EG < valid) hcg::store_raw(p + h * EG, hcg::pack<G>(o), valid - h * EG);
  }
}

template <class T, class G, class I>
__global__ __launch_bounds__(kGradThreads) void embed_grad_kernel(EmbedGradArgs g) {
  constexpr int E = kVec<T>;
  __shared__ int found[kGradWaves * kListPerWave], grouped[kGradWaves * kListPerWave];
  __shared__ uint8_t found_row[kGradWaves * kListPerWave];
  __shared__ int wave_found[kGradWaves], wave_below[kGradWaves];
  __shared__ int count[kMaxRows], start[kMaxRows];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t lo = (int64_t)blockIdx.x * g.rows;
  const int rows = (int)min((int64_t)g.rows, g.vocab - lo);
  const I* ids = static_cast<const I*>(g.ids);
  for (int r = tid; r < kMaxRows; r += kGradThreads) count[r] = 0;

  // Wave w scans the tokens [w * quota, (w + 1) * quota): its finds and, for
  // the place of this workgroup's tokens in the lists, how many name a row
  // before the first of these.  `keep` takes the find at its place.
  const int quota = (g.n + kGradWaves * 64 - 1) / (kGradWaves * 64) * 64;
  const int from = min(wave * quota, g.n), to = min(from + quota, g.n);
  auto scan = [&](auto keep) {
    int finds = 0, below = 0;
    for (int i0 = from; i0 < to; i0 += 64 * kScan) {
      int64_t id[kScan];
#pragma unroll
      for (int u = 0; u < kScan; ++u) {
        const int i = i0 + u * 64 + lane;
        id[u] = i < to ? (int64_t)ids[i] : -1;
        if (id[u] == g.padding) id[u] = -1;
      }
#pragma unroll
      for (int u = 0; u < kScan; ++u) {
        const int64_t r = id[u] - lo;
        below += __popcll(__ballot(id[u] >= 0 && r < 0));
        const uint64_t hit = __ballot(r >= 0 && r < rows);
        if (hit) {
          if (hit >> lane & 1) keep(finds + lanes_below(hit), i0 + u * 64 + lane, (int)r);
          finds += __popcll(hit);
        }
      }
    }
    if (lane == 0) wave_found[wave] = finds, wave_below[wave] = below;
  };
  scan([&](int at, int i, int r) {
    if (at < kListPerWave) {
      found[wave * kListPerWave + at] = i;
      found_row[wave * kListPerWave + at] = (uint8_t)r;
    }
  });
  __syncthreads();
  int total = 0, before = 0, below = 0;
  bool fits = true;
#pragma unroll
  for (int w = 0; w < kGradWaves; ++w) {
    if (w < wave) before += wave_found[w];
    total += wave_found[w];
    below += wave_below[w];
    fits = fits && wave_found[w] <= kListPerWave;
  }
  if (!fits) {
    // (wave_found and wave_below are written again with the same values)
    scan([&](int at, int i, int r) {
      g.found[below + before + at] = i;
      g.found_row[below + before + at] = (uint16_t)r;
    });
    __syncthreads();
  }

  // Find number j of wave w.
  auto find = [&](int w, int off, int j, int& i) -> int {
    if (fits) {
      i = found[w * kListPerWave + j];
      return found_row[w * kListPerWave + j];
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
          if (fits) grouped[at] = i;
          if (g.token) g.token[below + at] = i;
        }
        put += __popcll(hit);
      }
      off += wave_found[w];
    }
    if (g.row) {
      for (int j = lane; j < c; j += 64) g.row[below + start[r] + j] = c > kLong ? (int)(lo + r) : -1;
      if (c > kLong && lane == 0) g.run_len[below + start[r]] = c;
    }
  }
  // The places past all tokens (ids that name no row) belong to no long row.
  if (g.row && lo + rows == g.vocab)
    for (int j = below + total + tid; j < g.n; j += kGradThreads) g.row[j] = -1;
  __syncthreads();

  // Every row that is not long, as vectors over the threads.
  const T* dy = static_cast<const T*>(g.dy);
  G* grad = static_cast<G*>(g.grad);
  const int work = rows * g.vecs;
  for (int at = tid; at < work; at += kGradThreads) {
    const int r = at / g.vecs, c = (at - r * g.vecs) * E;
    const int n = count[r];
    if (n > kLong) continue;
    float sum[E];
#pragma unroll
    for (int e = 0; e < E; ++e) sum[e] = 0.f;
    const int first = start[r];
    for (int j0 = 0; j0 < n; j0 += 4) {
      raw4 raw[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (j0 + u < n) {
          const int i = fits ? grouped[first + j0 + u] : g.token[below + first + j0 + u];
          raw[u] = hcg::load_raw(dy + (int64_t)i * g.lddy + c, g.width - c);
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (j0 + u < n) {
          float f[E];
          hcg::unpack<T>(raw[u], f);
#pragma unroll
          for (int e = 0; e < E; ++e) sum[e] += f[e];
        }
      }
    }
    store_grad<T, G>(grad + (lo + r) * g.ldg + c, sum, g.scale, g.width - c);
  }
}

// Window blockIdx.x of the lists, vectors blockIdx.y * 256 ...: the sum of
// each run of one long row in it.
template <class T>
__global__ __launch_bounds__(256) void embed_window_kernel(EmbedGradArgs g) {
  constexpr int E = kVec<T>;
  __shared__ int token[kWindow], row[kWindow];
  const int from = blockIdx.x * kWindow, n = min(kWindow, g.n - from);
  if ((int)threadIdx.x < n) {
    token[threadIdx.x] = g.token[from + threadIdx.x];
    row[threadIdx.x] = g.row[from + threadIdx.x];
  }
  __syncthreads();
  const int c = (blockIdx.y * 256 + threadIdx.x) * E;
  if (c >= g.width) return;
  const T* dy = static_cast<const T*>(g.dy) + c;
  float* part = g.part + (int64_t)blockIdx.x * kRuns * g.width + c;
  const int left = g.width - c;
  int j = 0;
  while (j < n) {
    const int r = row[j];
    if (r < 0) {
      ++j;
      continue;
    }
    float sum[E];
#pragma unroll
    for (int e = 0; e < E; ++e) sum[e] = 0.f;
    int end = j + 1;
    while (end < n && row[end] == r) ++end;
    for (; j < end; j += 8) {
      raw4 raw[8];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (j + u < end) raw[u] = hcg::load_raw(dy + (int64_t)token[j + u] * g.lddy, left);
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (j + u < end) {
          float f[E];
          hcg::unpack<T>(raw[u], f);
#pragma unroll
          for (int e = 0; e < E; ++e) sum[e] += f[e];
        }
    }
    j = end;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (e < left) part[e] = sum[e];
    part += g.width;
  }
}

// The long rows that start in window blockIdx.x, columns blockIdx.y * 256 ...:
// their windows' sums, in order.
template <class G>
__global__ __launch_bounds__(256) void embed_long_kernel(EmbedGradArgs g) {
  __shared__ int row[kWindow + 1];  // [0]: the entry before the window
  const int from = blockIdx.x * kWindow, n = min(kWindow, g.n - from);
  for (int j = threadIdx.x; j <= n; j += 256) row[j] = from + j > 0 ? g.row[from + j - 1] : -1;
  __syncthreads();
  const int64_t c = (int64_t)blockIdx.y * 256 + threadIdx.x;
  if (c >= g.width) return;
  int run = row[1] >= 0 ? 0 : -1;  // of the entry looked at, counted over the long rows of the window
  for (int j = 1; j <= n; ++j) {
    const bool starts = row[j] >= 0 && row[j] != row[j - 1];
    if (j > 1 && starts) ++run;
    if (!starts) continue;
    const int len = g.run_len[from + j - 1];
    const int windows = (from + j - 1 + len - 1) / kWindow - (int)blockIdx.x;  // after this one
    float sum = g.part[((int64_t)blockIdx.x * kRuns + run) * g.width + c];
    const float* next = g.part + (int64_t)(blockIdx.x + 1) * kRuns * g.width + c;
#pragma unroll 8
    for (int w = 0; w < windows; ++w) sum += next[(int64_t)w * kRuns * g.width];
    static_cast<G*>(g.grad)[(int64_t)row[j] * g.ldg + c] = (G)(sum * g.scale);
  }
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------

constexpr int64_t kMaxTokens = (int64_t)1 << 30;

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
  embed_grad_kernel<T, G, I><<<dim3((unsigned)((a.vocab + a.rows - 1) / a.rows)), kGradThreads, 0, s>>>(a);
  if (a.token == nullptr) return;  // too few tokens for a long row
  const unsigned windows = (unsigned)windows_of(a.n);
  embed_window_kernel<T><<<dim3(windows, (unsigned)((a.vecs + 255) / 256)), 256, 0, s>>>(a);
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
  const dim3 grid((unsigned)((n + a.rows_per_wg - 1) / a.rows_per_wg));
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

int64_t hcg_embedding_grad_workspace(int64_t n, int64_t vocab, int64_t width) {
  if (n <= kLong || vocab <= 0 || width <= 0 || n >= kMaxTokens) return 0;
  return 4 * round256(n * 4) + round256(n * 2) + windows_of(n) * kRuns * width * 4;
}

int hcg_embedding_grad(int dtype, const void* dy, int64_t lddy, int64_t n, int64_t width, int id_bytes,
                       const void* ids, int64_t vocab, int64_t padding_idx, float scale, int grad_dtype,
                       void* grad, int64_t ldg, void* workspace, int64_t workspace_bytes, void* stream) {
  HCG_LM_REQUIRE(hcg::elem_ok(dtype), "dtype %d is not HCG_F16, HCG_BF16 or HCG_F32", dtype);
  HCG_LM_REQUIRE(grad_dtype == dtype || grad_dtype == HCG_F32, "the gradient has the type of dy or float32");
  HCG_LM_REQUIRE(id_bytes == 4 || id_bytes == 8, "ids are 4 or 8 bytes, not %d", id_bytes);
  HCG_LM_REQUIRE(n >= 0 && n < kMaxTokens && vocab >= 0 && vocab < kMaxTokens && width >= 0 &&
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
  const int64_t need = hcg_embedding_grad_workspace(n, vocab, width);
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
  a.vecs = (int)((width * eb + 15) / 16);
  a.rows = (int)std::min<int64_t>(kMaxRows, (vocab + 1023) / 1024);
  a.scale = scale;
  if (need > 0) {
    char* p = static_cast<char*>(workspace);
    a.token = reinterpret_cast<int*>(p);
    a.row = reinterpret_cast<int*>(p += round256(n * 4));
    a.run_len = reinterpret_cast<int*>(p += round256(n * 4));
    a.found = reinterpret_cast<int*>(p += round256(n * 4));
    a.found_row = reinterpret_cast<uint16_t*>(p += round256(n * 4));
    a.part = reinterpret_cast<float*>(p + round256(n * 2));
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
