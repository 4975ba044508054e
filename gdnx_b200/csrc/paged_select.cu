// The pages of a paged cache that a query's key head reads, by a score that the bounds of a page's keys give:
//   score = max over the head's queries of  sum_d max(q_d lo_d, q_d hi_d),
// which no product q.k of a key on the page exceeds.  Taken are the pages of the first `sinks` and the last `window`
// tokens, then those with the largest scores, the lower page first among equals, `k` in all; they come in rising order.
//
// A score decides by comparison, so a rounding could change which page is taken: products and sums are in 64 bits
// (exact products of 16-bit values, and sums whose error is far below the scores' distances), and score pages at 4
// lanes a page with a fixed order of sums, so that equal pages have equal scores.  max(q lo, q hi) is q hi for q >= 0,
// else q lo.  The scores are kept as 64-bit words that order alike: all ones for a page that is always taken, 0 for one
// that the sequence does not hold.
//
// The k-th largest word is found bit by bit from the highest in which the words differ: a bit stays set where at least k
// words lie at or above; the search ends as soon as just k do.
#include "paged_cache.cuh"

namespace gdnx {
namespace {

constexpr int NT = 256;
constexpr int LANES = 4;      // of a page
constexpr int GH = 8;         // query heads that one reading of the bounds serves
constexpr int SMEM_KEYS = 24 * 1024;

struct SelParams {
  gdnx_paged_select_args a;
  unsigned long long* keys;  // [B, Hk, width]; null: the words stay in shared memory
  int splits;                // CTAs that share a query head's pages
};

struct Query {
  int row, len, pages;
};
GDNX_DEV Query query_of(const gdnx_paged_select_args& a, int64_t b) {
  const gdnx_cache& c = a.cache;
  Query q;
  q.row = a.rows ? a.rows[b] : (int)b;
  if (q.row < 0 || q.row >= c.slots) return {0, 0, 0};
  int64_t n = length_of(c, q.row);
  if (a.positions) n = min(n, max((int64_t)a.positions[b] + 1, (int64_t)0));
  q.len = (int)n;
  q.pages = (int)pages_of(c, n);
  return q;
}

// NaN counts as +inf.
GDNX_DEV unsigned long long ordered(double x) {
  if (x != x) x = INFINITY;
  const long long u = __double_as_longlong(x + 0.0);  // -0 as 0
  return u < 0 ? ~(unsigned long long)u : (unsigned long long)u | 0x8000000000000000ull;
}

template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
};
GDNX_DEV void widen(float (&x)[4], uint4 u, float) {
  x[0] = __uint_as_float(u.x);
  x[1] = __uint_as_float(u.y);
  x[2] = __uint_as_float(u.z);
  x[3] = __uint_as_float(u.w);
}
GDNX_DEV void widen(float (&x)[8], uint4 u, __nv_bfloat16) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
GDNX_DEV void widen(float (&x)[8], uint4 u, __half) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}

// The words of this CTA's pages x, x = first, first + stride, ... of NT / LANES at a time.
template <typename T>
GDNX_DEV void score_pages(const SelParams& P, const Query& q, int64_t b, int64_t hk, double (*qs)[128],
                          unsigned long long* keys) {
  const gdnx_paged_select_args& a = P.a;
  const gdnx_cache& c = a.cache;
  const int G = (int)(a.H / c.Hk), D = (int)c.D, per = D / Vec<T>::N, lane = threadIdx.x % LANES;
  const uint4* bounds = static_cast<const uint4*>(a.bounds);
  const int64_t lo0 = a.layer * 2 * c.pages, hi0 = lo0 + c.pages;
  constexpr int STEP = NT / LANES;
  for (int g0 = 0; g0 < G; g0 += GH) {
    __syncthreads();
    for (int i = threadIdx.x; i < GH * D; i += NT) {
      const int g = i / D, d = i % D;
      // a head that is not there repeats the first
      qs[g][d] = ld_as_f32(a.q.ptr, a.q.dtype, b * a.q.sb + (hk * G + (g0 + g < G ? g0 + g : 0)) * a.q.sh + d);
    }
    __syncthreads();
    for (int x0 = blockIdx.x * STEP; x0 < q.pages; x0 += P.splits * STEP) {
      const int x = x0 + threadIdx.x / LANES;
      const int p = x < q.pages ? c.table[(int64_t)q.row * c.width + x] : -1;
      double s[GH];
#pragma unroll
      for (int g = 0; g < GH; ++g) s[g] = 0.0;
      if (page_ok(c, p)) {
        const uint4* lo = bounds + ((lo0 + p) * c.Hk + hk) * per;
        const uint4* hi = bounds + ((hi0 + p) * c.Hk + hk) * per;
        for (int e = lane; e < per; e += LANES) {
          float l[Vec<T>::N], h[Vec<T>::N];
          widen(l, lo[e], T());
          widen(h, hi[e], T());
#pragma unroll
          for (int i = 0; i < Vec<T>::N; ++i) {
            const double dl = l[i], dh = h[i];
#pragma unroll
            for (int g = 0; g < GH; ++g) {
              const double v = qs[g][e * Vec<T>::N + i];
              s[g] = fma(v, v >= 0.0 ? dh : dl, s[g]);
            }
          }
        }
      }
      unsigned long long key = 0;
#pragma unroll
      for (int g = 0; g < GH; ++g) {
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) s[g] += __shfl_xor_sync(0xffffffffu, s[g], o);
        const unsigned long long w = ordered(s[g]);
        key = w > key ? w : key;
      }
      if (lane == 0 && x < q.pages) {
        const int64_t at = (int64_t)x * c.page;
        if (!page_ok(c, p)) key = 0;
        else if (at < a.sinks || at + c.page > q.len - a.window) key = ~0ull;
        else if (g0 > 0) key = key > keys[x] ? key : keys[x];
        keys[x] = key;
      }
    }
  }
}

// Exclusive prefix sum of 0 or 1 per thread over the CTA, and the total.
GDNX_DEV int rank_of(bool on, int* warp_sums, int* total) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const uint32_t bits = __ballot_sync(0xffffffffu, on);
  __syncthreads();
  if (lane == 0) warp_sums[warp] = __popc(bits);
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < NT / 32; ++i) {
    before += i < warp ? warp_sums[i] : 0;
    all += warp_sums[i];
  }
  *total = all;
  return before + __popc(bits & ((1u << lane) - 1));
}

// f(word) summed over the n words, in every thread.
template <typename F>
GDNX_DEV int count_words(const unsigned long long* keys, int n, int* warp_sums, F f) {
  int mine = 0;
  for (int i = threadIdx.x; i < n; i += NT) mine += f(keys[i]);
  mine = __reduce_add_sync(0xffffffffu, mine);
  __syncthreads();
  if (threadIdx.x % 32 == 0) warp_sums[threadIdx.x / 32] = mine;
  __syncthreads();
  int all = 0;
#pragma unroll
  for (int i = 0; i < NT / 32; ++i) all += warp_sums[i];
  return all;
}

// The k largest of n words (0: none), the lower index first among equals, in rising order; -1 behind them.
GDNX_DEV void take_largest(const unsigned long long* keys, int n, int k, int32_t* out) {
  __shared__ int sums[NT / 32];
  __shared__ unsigned long long ends[2][NT / 32];
  unsigned long long least = ~0ull, most = 0;
  for (int i = threadIdx.x; i < n; i += NT) {
    const unsigned long long w = keys[i];
    if (w == 0) continue;
    least = w < least ? w : least;
    most = w > most ? w : most;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long x = __shfl_xor_sync(0xffffffffu, least, o), y = __shfl_xor_sync(0xffffffffu, most, o);
    least = x < least ? x : least;
    most = y > most ? y : most;
  }
  if (threadIdx.x % 32 == 0) {
    ends[0][threadIdx.x / 32] = least;
    ends[1][threadIdx.x / 32] = most;
  }
  const int there = count_words(keys, n, sums, [](unsigned long long w) { return w != 0; });  // synchronises
#pragma unroll
  for (int i = 0; i < NT / 32; ++i) {
    least = ends[0][i] < least ? ends[0][i] : least;
    most = ends[1][i] > most ? ends[1][i] : most;
  }
  unsigned long long bar = 1;  // at least this is taken
  int above = there;           // words at or above it
  if (there > k) {
    const int top = least == most ? -1 : 63 - __clzll(least ^ most);
    bar = top < 0 ? most : most >> top >> 1 << top << 1;
    for (int bit = top; bit >= 0 && above != k; --bit) {
      const unsigned long long t = bar | 1ull << bit;
      const int m = count_words(keys, n, sums, [=](unsigned long long w) { return w >= t; });
      if (m >= k) {
        bar = t;
        above = m;
      }
    }
  }
  // of the words equal to the bar, the first ones
  int equal = n;
  if (above > k) equal = k - count_words(keys, n, sums, [=](unsigned long long w) { return w > bar; });
  int taken = 0, ties = 0;
  for (int i0 = 0; i0 < n && taken < k; i0 += NT) {
    const int i = i0 + threadIdx.x;
    const unsigned long long w = i < n ? keys[i] : 0;
    int all;
    bool on = w >= bar;
    if (above > k) {
      const int r = rank_of(w == bar, sums, &all);
      if (w == bar) on = ties + r < equal;
      ties += all;
    }
    const int r = rank_of(on, sums, &all);
    if (on) out[taken + r] = i;
    taken += all;
  }
  for (int i = taken + threadIdx.x; i < k; i += NT) out[i] = -1;
}

// FUSED: one CTA for each query and key head scores its pages and takes the largest; else CTA (x, unit) leaves the
// words of its share of the pages to the next kernel.
template <typename T, bool FUSED>
__global__ void __launch_bounds__(NT) paged_select_kernel(const SelParams P) {
  extern __shared__ unsigned long long words[];
  __shared__ double qs[GH][128];
  dependents_may_start();
  wait_for_earlier();
  const int64_t unit = blockIdx.y + (int64_t)blockIdx.z * gridDim.y, Hk = P.a.cache.Hk;
  if (unit >= P.a.B * Hk) return;
  const Query q = query_of(P.a, unit / Hk);
  unsigned long long* keys = FUSED ? words : P.keys + unit * P.a.cache.width;
  score_pages<T>(P, q, unit / Hk, unit % Hk, qs, keys);
  if (!FUSED) return;
  __syncthreads();
  take_largest(keys, q.pages, (int)P.a.k, P.a.selected + unit * P.a.k);
}

__global__ void __launch_bounds__(NT) paged_take_kernel(const SelParams P) {
  extern __shared__ unsigned long long words[];
  dependents_may_start();
  wait_for_earlier();
  const int64_t unit = blockIdx.x, Hk = P.a.cache.Hk;
  const Query q = query_of(P.a, unit / Hk);
  const unsigned long long* keys = P.keys + unit * P.a.cache.width;
  if (q.pages <= SMEM_KEYS) {
    for (int i = threadIdx.x; i < q.pages; i += NT) words[i] = keys[i];
    __syncthreads();
    keys = words;
  }
  take_largest(keys, q.pages, (int)P.a.k, P.a.selected + unit * P.a.k);
}

// Pages that a sequence can have.
int64_t most_pages(const gdnx_paged_select_args& a) {
  const gdnx_cache& c = a.cache;
  const int64_t n = a.max_len > 0 ? (a.max_len + c.page - 1) / c.page : c.width;
  return n < c.width ? n : c.width;
}
// One kernel does both where the query heads fill the device by themselves, or have few pages each.
bool fused(const gdnx_paged_select_args& a) {
  const int64_t n = most_pages(a);
  return a.cache.width <= SMEM_KEYS && (a.B * a.cache.Hk >= sm_count() || n <= 4 * NT / LANES);
}

template <typename F>
bool allow(F kernel, size_t bytes) {
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) == cudaSuccess) return true;
  cudaGetLastError();
  return false;
}

template <typename T>
gdnx_status select_of(const gdnx_paged_select_args& a, cudaStream_t st) {
  const int64_t units = a.B * a.cache.Hk, n = most_pages(a);
  SelParams P = {a, static_cast<unsigned long long*>(a.workspace), 1};
  const unsigned y = (unsigned)(units < 65535 ? units : 65535), z = (unsigned)((units + y - 1) / y);
  const size_t bytes = (size_t)(a.cache.width < SMEM_KEYS ? a.cache.width : SMEM_KEYS) * 8;
  if (fused(a)) {
    if (!allow(paged_select_kernel<T, true>, SMEM_KEYS * 8)) return GDNX_ELAUNCH;
    return launched(launch_early(paged_select_kernel<T, true>, dim3(1, y, z), dim3(NT), bytes, st, P));
  }
  const int64_t want = ((int64_t)sm_count() * 4 + units - 1) / units, have = (n + NT / LANES - 1) / (NT / LANES);
  P.splits = (int)(want < have ? want : have);
  if (launch_early(paged_select_kernel<T, false>, dim3((unsigned)P.splits, y, z), dim3(NT), 0, st, P) != cudaSuccess)
    return GDNX_ELAUNCH;
  if (!allow(paged_take_kernel, SMEM_KEYS * 8)) return GDNX_ELAUNCH;
  return launched(launch_early(paged_take_kernel, dim3((unsigned)units), dim3(NT), bytes, st, P));
}

}  // namespace

size_t paged_select_workspace_bytes(const gdnx_paged_select_args& a) {
  return fused(a) ? 0 : (size_t)(a.B * a.cache.Hk * a.cache.width) * 8;
}

gdnx_status launch_paged_select(const gdnx_paged_select_args& a, cudaStream_t st) {
  switch (a.cache.dtype) {
    case GDNX_BF16: return select_of<__nv_bfloat16>(a, st);
    case GDNX_F16: return select_of<__half>(a, st);
    default: return select_of<float>(a, st);
  }
}

}  // namespace gdnx
