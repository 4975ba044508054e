// The pages of a paged cache that a query's key head reads, by a score that the bounds of a page's keys give:
//   score = max over the head's queries of  sum_d max(q_d lo_d, q_d hi_d),
// which no product q.k of a key on the page exceeds.  Taken are the pages of the first `sinks` and the last `window`
// tokens, then those with the largest scores, the lower page first among equals, `k` in all; they come in rising order.
//
// A score decides by comparison, so a rounding could change which page is taken: products and sums are in 64 bits
// (exact products of 16-bit values, and sums whose error is far below the scores' distances) with a fixed order of sums,
// so that equal pages have equal scores.  max(q lo, q hi) is q hi for q >= 0, else q lo.  The scores are kept as 64-bit
// words that order alike: all ones for a page that is always taken, 0 for one that the sequence does not hold.
//
// Issue slots bound it.  A lane holds the queries of four dims in registers and reads 8 or 16 bytes of a page's
// bounds; the sums of several pages and heads are reduced over the lanes together, each step handing half of them to
// the lane's partner.  (With a page to four lanes and the queries in shared memory, the reads of these took 70 us for
// 64 x 4 key heads of up to 256 pages, which take 18 now.)  The two words of a lane's query value, from 0 on and below,
// stand for the choice of lo or hi: one of two products is 0.
//
// Of up to RANKED words each thread ranks one against all others.  Of more, the words are counted in 256 parts of their
// range, and those of the part that the k-th largest lies in again, until they are few enough to be ranked.
//
// Measured: 64 requests of up to 256 pages of 64, 16 heads over 4 of 128: 18 us (33 MB of bounds: 5 us at a copy's rate);
// one of 4096 pages over 2 key heads: 17 us, two launches, of which the latency of each is most.  A CTA of 240
// registers a thread has an SM to itself, and its 36 % of issue slots are the chain from page id to score.
#include <type_traits>

#include "attn_tc.cuh"
#include "paged_cache.cuh"

namespace gdnx {
namespace {

constexpr int NT = 256;         // threads of a CTA that scores
constexpr int TAKE_NT = 1024;   // of one that only takes
constexpr int RANKED = 256;
constexpr int SMEM_KEYS = 24 * 1024;

struct SelParams {
  gdnx_paged_select_args a;
  unsigned long long* keys;  // [B, Hk, width]; null: the words stay in shared memory
  int splits;                // CTAs that share a query head's pages
  int vec_q;                 // four values of q lie aligned
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

// Four values of a row of bounds, as they lie and widened.
template <typename T>
struct Four {
  uint2 u;
  GDNX_DEV void clear() { u = make_uint2(0, 0); }
  GDNX_DEV void load(const void* base, int64_t at) { u = *reinterpret_cast<const uint2*>(static_cast<const char*>(base) + at * 2); }
  GDNX_DEV void gather(const void* base, int64_t at) {  // not aligned
    const uint16_t* p = static_cast<const uint16_t*>(base) + at;
    u = make_uint2(p[0] | (uint32_t)p[1] << 16, p[2] | (uint32_t)p[3] << 16);
  }
  GDNX_DEV void widen(double (&x)[4]) const {
    if constexpr (std::is_same<T, __half>::value) {
      const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
      x[0] = a.x;
      x[1] = a.y;
      x[2] = b.x;
      x[3] = b.y;
    } else {
      x[0] = __uint_as_float(u.x << 16);
      x[1] = __uint_as_float(u.x & 0xffff0000u);
      x[2] = __uint_as_float(u.y << 16);
      x[3] = __uint_as_float(u.y & 0xffff0000u);
    }
  }
};
template <>
struct Four<float> {
  float4 u;
  GDNX_DEV void clear() { u = make_float4(0.f, 0.f, 0.f, 0.f); }
  GDNX_DEV void load(const void* base, int64_t at) { u = *reinterpret_cast<const float4*>(static_cast<const float*>(base) + at); }
  GDNX_DEV void gather(const void* base, int64_t at) {
    const float* p = static_cast<const float*>(base) + at;
    u = make_float4(p[0], p[1], p[2], p[3]);
  }
  GDNX_DEV void widen(double (&x)[4]) const {
    x[0] = u.x;
    x[1] = u.y;
    x[2] = u.z;
    x[3] = u.w;
  }
};

constexpr int log2_of(int n) { return n <= 1 ? 0 : 1 + log2_of(n / 2); }

// The words of this CTA's share of the pages.  LANES lanes share a page, 32 / LANES pages lie side by side, and a warp
// takes PB of these at a time; GH query heads at a time.
template <typename T, int LANES, int GH>
GDNX_DEV void score_pages(const SelParams& P, const Query& q, int64_t b, int64_t hk, unsigned long long* keys) {
  constexpr int PB = GH == 1 ? 8 : 16 / GH, V = PB * GH, SIDE = 32 / LANES;
  // of the sums' number v = page GH + head, the lane's upper bits are the upper ones, REST sums stay with a lane
  constexpr int LV = log2_of(V), LG = log2_of(LANES), L = LV < LG ? LV : LG, REST = 1 << (LV - L);
  static_assert(REST <= GH, "a lane's sums are one page's");
  const gdnx_paged_select_args& a = P.a;
  const gdnx_cache& c = a.cache;
  const int G = (int)(a.H / c.Hk), D = (int)c.D, in = threadIdx.x % LANES, sub = threadIdx.x % 32 / LANES, d = in * 4;
  const int64_t lo0 = a.layer * 2 * c.pages, hi0 = lo0 + c.pages;
  const int32_t* table = c.table + (int64_t)q.row * c.width;
  constexpr int BATCH = SIDE * PB;
  static_assert(32 % BATCH == 0, "a batch's ids lie in one reading");
  // the warp's pages r0..r1-1: an even share in whole batches
  const int lane = threadIdx.x % 32, warps = P.splits * (NT / 32), warp = (int)blockIdx.x * (NT / 32) + (int)threadIdx.x / 32;
  const int share = ((q.pages + BATCH - 1) / BATCH + warps - 1) / warps * BATCH;
  const int r0 = min(warp * share, q.pages), r1 = min(r0 + share, q.pages);
  for (int g0 = 0; g0 < G; g0 += GH) {
    double up[GH][4], dn[GH][4];  // the queries' values from 0 on (the others 0), and those below
#pragma unroll
    for (int g = 0; g < GH; ++g) {
      // a head that is not there repeats the first; a dim that is not there counts nothing
      const int64_t at = b * a.q.sb + (hk * G + (g0 + g < G ? g0 + g : 0)) * a.q.sh + d;
      Four<T> w;
      w.clear();
      if (d < D && P.vec_q) w.load(a.q.ptr, at);
      else if (d < D) w.gather(a.q.ptr, at);
      double x[4];
      w.widen(x);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        up[g][i] = x[i] >= 0.0 ? x[i] : 0.0;
        dn[g][i] = x[i] >= 0.0 ? 0.0 : x[i];
      }
    }
    // ids of 32 of the warp's pages, a lane's each, and of the 32 behind them; bounds of a batch, read one ahead
    const auto read = [&](int x) { return x + lane < r1 ? table[x + lane] : -1; };
    int base = r0, ids = read(r0), more = read(r0 + 32);
    int id[PB], next_id[PB];
    Four<T> lo[PB], hi[PB], next_lo[PB], next_hi[PB];
    const auto fetch = [&](int x0) {
      if (x0 >= base + 32) {
        base += 32;
        ids = more;
        more = read(base + 32);
      }
#pragma unroll
      for (int j = 0; j < PB; ++j) {
        next_id[j] = __shfl_sync(0xffffffffu, ids, (x0 - base + j * SIDE + sub) & 31);
        next_lo[j].clear();
        next_hi[j].clear();
        if (page_ok(c, next_id[j]) && d < D) {
          next_lo[j].load(a.bounds, ((lo0 + next_id[j]) * c.Hk + hk) * D + d);
          next_hi[j].load(a.bounds, ((hi0 + next_id[j]) * c.Hk + hk) * D + d);
        }
      }
    };
    if (r0 < r1) fetch(r0);
    for (int x0 = r0; x0 < r1; x0 += BATCH) {
#pragma unroll
      for (int j = 0; j < PB; ++j) {
        id[j] = next_id[j];
        lo[j] = next_lo[j];
        hi[j] = next_hi[j];
      }
      if (x0 + BATCH < r1) fetch(x0 + BATCH);
      double s[V];
      const auto sum = [&](auto term) {
#pragma unroll
        for (int j = 0; j < PB; ++j) {
          double l[4], h[4];
          lo[j].widen(l);
          hi[j].widen(h);
#pragma unroll
          for (int g = 0; g < GH; ++g) {
            double t = 0.0;
#pragma unroll
            for (int i = 0; i < 4; ++i) t = term(t, g, i, l[i], h[i]);
            s[j * GH + g] = t;
          }
        }
        int left = V;
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) {
          if (left > 1) {
            left /= 2;
            const bool upper = in & o;
#pragma unroll
            for (int i = 0; i < V / 2; ++i)
              if (i < left) {
                const double give = upper ? s[i] : s[i + left], keep = upper ? s[i + left] : s[i];
                s[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
              }
          } else {
            s[0] += __shfl_xor_sync(0xffffffffu, s[0], o);
          }
        }
      };
      // one of the two products is 0; with a bound that is not finite it may be NaN, which shows in the sum
      sum([&](double t, int g, int i, double l, double h) { return fma(dn[g][i], l, fma(up[g][i], h, t)); });
      bool odd = false;
#pragma unroll
      for (int i = 0; i < REST; ++i) odd |= !(fabs(s[i]) < INFINITY);
      if (__any_sync(0xffffffffu, odd))
        sum([&](double t, int g, int i, double l, double h) {
          const bool below = !(dn[g][i] == 0.0);
          return fma(below ? dn[g][i] : up[g][i], below ? l : h, t);
        });
      unsigned long long key = 0;
#pragma unroll
      for (int i = 0; i < REST; ++i) {
        const unsigned long long w = ordered(s[i]);
        key = w > key ? w : key;
      }
#pragma unroll
      for (int n = REST, o = 1 << (LG - L); n < GH; n *= 2, o *= 2) {
        const unsigned long long w = __shfl_xor_sync(0xffffffffu, key, o);
        key = w > key ? w : key;
      }
      const int v = (in >> (LG - L)) << (LV - L), j = v / GH;
      if (v % GH == 0 && (in & ((1 << (LG - L)) - 1)) == 0) {
        const int at = x0 + j * SIDE + sub;
        int p = -1;
#pragma unroll
        for (int e = 0; e < PB; ++e) p = e == j ? id[e] : p;
        if (at < r1) {
          const int64_t first = (int64_t)at * c.page;
          if (!page_ok(c, p)) key = 0;
          else if (first < a.sinks || first + c.page > q.len - a.window) key = ~0ull;
          else if (g0 > 0) key = key > keys[at] ? key : keys[at];
          keys[at] = key;
        }
      }
    }
  }
}

// Exclusive prefix sum of 0 or 1 per thread over the CTA, and the total.
template <int THREADS>
GDNX_DEV int rank_of(bool on, int* warp_sums, int* total) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const uint32_t bits = __ballot_sync(0xffffffffu, on);
  __syncthreads();
  if (lane == 0) warp_sums[warp] = __popc(bits);
  __syncthreads();
  const int mine = lane < THREADS / 32 ? warp_sums[lane] : 0;
  *total = __reduce_add_sync(0xffffffffu, mine);
  return __reduce_add_sync(0xffffffffu, lane < warp ? mine : 0) + __popc(bits & ((1u << lane) - 1));
}

// The k largest of n words (0: none), the lower index first among equals, in rising order; -1 behind them.
template <int THREADS>
GDNX_DEV void take_largest(const unsigned long long* keys, int n, int k, int32_t* out) {
  constexpr int WARPS = THREADS / 32;
  static_assert(RANKED <= THREADS, "a word for each thread");
  __shared__ int sums[2][WARPS];
  __shared__ unsigned long long ends[2][WARPS], few[RANKED], last;
  __shared__ int few_at[RANKED], hist[256], found[3];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  if (n <= RANKED) {
    const unsigned long long w = (int)threadIdx.x < n ? keys[threadIdx.x] : 0;
    int above = 0;
    if (warp * 32 < n && n > k) {
      // those before this warp's words go first among equals, those behind them do not
      const int a0 = warp * 32, a1 = min(a0 + 32, n);
#pragma unroll 8
      for (int i = 0; i < a0; ++i) above += keys[i] >= w;
#pragma unroll 8
      for (int i = a0; i < a1; ++i) above += keys[i] > w || (keys[i] == w && i < (int)threadIdx.x);
#pragma unroll 8
      for (int i = a1; i < n; ++i) above += keys[i] > w;
    }
    int all;
    const bool on = w != 0 && above < k;
    const int r = rank_of<THREADS>(on, sums[0], &all);
    if (on) out[r] = (int)threadIdx.x;
    for (int i = all + threadIdx.x; i < k; i += THREADS) out[i] = -1;
    return;
  }
  // The ends of the words that are there and not taken always, and the numbers of both.
  unsigned long long least = ~0ull, most = 0;
  int there = 0, always = 0;
  for (int i = threadIdx.x; i < n; i += THREADS) {
    const unsigned long long w = keys[i];
    there += w != 0;
    always += w == ~0ull;
    if (w == 0 || w == ~0ull) continue;
    least = w < least ? w : least;
    most = w > most ? w : most;
  }
  const auto span = [](unsigned long long& a, unsigned long long& z) {  // over the warp
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long x = __shfl_xor_sync(0xffffffffu, a, o), y = __shfl_xor_sync(0xffffffffu, z, o);
      a = x < a ? x : a;
      z = y > z ? y : z;
    }
  };
  span(least, most);
  there = __reduce_add_sync(0xffffffffu, there);
  always = __reduce_add_sync(0xffffffffu, always);
  if (lane == 0) {
    ends[0][warp] = least;
    ends[1][warp] = most;
    sums[0][warp] = there;
    sums[1][warp] = always;
  }
  __syncthreads();
  least = lane < WARPS ? ends[0][lane] : ~0ull;
  most = lane < WARPS ? ends[1][lane] : 0;
  span(least, most);
  there = __reduce_add_sync(0xffffffffu, lane < WARPS ? sums[0][lane] : 0);
  always = __reduce_add_sync(0xffffffffu, lane < WARPS ? sums[1][lane] : 0);
  // Taken is what lies above `bar`, and of the words equal to it those up to index `end`.
  unsigned long long bar = 0;
  int end = -1;
  if (there > k) {
    // the need-th largest of the `inside` words from least to most is the last that is taken
    int need = k - always, inside = there - always;
    while (need > 0 && inside > RANKED && least < most) {
      // how many of them lie in each 256th of their range
      const int shift = max(0, 56 - __clzll(most - least));
      for (int i = threadIdx.x; i < 256; i += THREADS) hist[i] = 0;
      __syncthreads();
      for (int i = threadIdx.x; i < n; i += THREADS) {
        const unsigned long long w = keys[i];
        if (w >= least && w <= most) atomicAdd(&hist[(int)((w - least) >> shift)], 1);
      }
      __syncthreads();
      if (warp == 0) {  // from the highest: a lane has eight parts
        int mine = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) mine += hist[255 - (lane * 8 + e)];
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int x = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += x;
        }
        if (upto >= need && upto - mine < need) {
          int before = upto - mine, e = 0;
          while (before + hist[255 - (lane * 8 + e)] < need) before += hist[255 - (lane * 8 + e++)];
          found[0] = 255 - (lane * 8 + e);
          found[1] = before;
          found[2] = hist[255 - (lane * 8 + e)];
        }
      }
      __syncthreads();
      need -= found[1];
      inside = found[2];
      least += (unsigned long long)found[0] << shift;
      const unsigned long long top = least + ((1ull << shift) - 1);
      most = top < most ? top : most;
      __syncthreads();  // found and hist may be written again
    }
    if (need <= 0) {
      bar = ~0ull - 1;  // those always taken are all
    } else if (inside <= RANKED) {
      if (threadIdx.x == 0) found[0] = 0;
      __syncthreads();
      for (int i = threadIdx.x; i < n; i += THREADS) {
        const unsigned long long w = keys[i];
        if (w >= least && w <= most) {
          const int at = atomicAdd(&found[0], 1);  // in any order: the ranks do not depend on it
          few[at] = w;
          few_at[at] = i;
        }
      }
      __syncthreads();
      if ((int)threadIdx.x < inside) {
        const unsigned long long w = few[threadIdx.x];
        const int at = few_at[threadIdx.x];
        int above = 0;
        for (int i = 0; i < inside; ++i) above += few[i] > w || (few[i] == w && few_at[i] < at);
        if (above == need - 1) {
          last = w;
          found[1] = at;
        }
      }
      __syncthreads();
      bar = last;
      end = found[1];
    } else {  // all alike: the need-th of them
      bar = least;
      int before = 0;
      for (int i0 = 0; i0 < n && before < need; i0 += THREADS) {
        const int i = i0 + threadIdx.x;
        const bool on = i < n && keys[i] == bar;
        int all;
        const int r = rank_of<THREADS>(on, sums[0], &all);
        if (on && before + r == need - 1) found[1] = i;
        before += all;
      }
      __syncthreads();
      end = found[1];
    }
  }
  int taken = 0;
  for (int i0 = 0; i0 < n && taken < k; i0 += THREADS) {
    const int i = i0 + threadIdx.x;
    const unsigned long long w = i < n ? keys[i] : 0;
    const bool on = w > bar || (w == bar && w != 0 && i <= end);
    int all;
    const int r = rank_of<THREADS>(on, sums[0], &all);
    if (on && taken + r < k) out[taken + r] = i;
    taken += all;
  }
  for (int i = min(taken, k) + threadIdx.x; i < k; i += THREADS) out[i] = -1;
}

// FUSED: one CTA for each query and key head scores its pages and takes the largest; else CTA (x, unit) leaves the
// words of its share of the pages to the next kernel.
template <typename T, int LANES, int GH, bool FUSED>
__global__ void __launch_bounds__(NT) paged_select_kernel(const SelParams P) {
  extern __shared__ unsigned long long words[];
  dependents_may_start();
  wait_for_earlier();
  const int64_t unit = blockIdx.y + (int64_t)blockIdx.z * gridDim.y, Hk = P.a.cache.Hk;
  if (unit >= P.a.B * Hk) return;
  const Query q = query_of(P.a, unit / Hk);
  unsigned long long* keys = FUSED ? words : P.keys + unit * P.a.cache.width;
  score_pages<T, LANES, GH>(P, q, unit / Hk, unit % Hk, keys);
  if (!FUSED) return;
  __syncthreads();
  take_largest<NT>(keys, q.pages, (int)P.a.k, P.a.selected + unit * P.a.k);
}

__global__ void __launch_bounds__(TAKE_NT) paged_take_kernel(const SelParams P) {
  extern __shared__ unsigned long long words[];
  dependents_may_start();
  wait_for_earlier();
  const int64_t unit = blockIdx.x, Hk = P.a.cache.Hk;
  const Query q = query_of(P.a, unit / Hk);
  const unsigned long long* keys = P.keys + unit * P.a.cache.width;
  if (q.pages <= SMEM_KEYS) {
    for (int i = threadIdx.x; i < q.pages; i += TAKE_NT) words[i] = keys[i];
    __syncthreads();
    keys = words;
  }
  take_largest<TAKE_NT>(keys, q.pages, (int)P.a.k, P.a.selected + unit * P.a.k);
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
  return a.cache.width <= SMEM_KEYS && (a.B * a.cache.Hk >= sm_count() || n <= RANKED);
}

template <typename T, int LANES, int GH>
gdnx_status select_of(const gdnx_paged_select_args& a, cudaStream_t st) {
  static std::atomic<uint64_t> done[2];
  const int64_t units = a.B * a.cache.Hk, n = most_pages(a);
  const size_t four = 4 * sizeof(T);
  SelParams P = {a, static_cast<unsigned long long*>(a.workspace), 1,
                 reinterpret_cast<uintptr_t>(a.q.ptr) % four == 0 && a.q.sb % 4 == 0 && a.q.sh % 4 == 0};
  const unsigned y = (unsigned)(units < 65535 ? units : 65535), z = (unsigned)((units + y - 1) / y);
  const size_t bytes = (size_t)(a.cache.width < SMEM_KEYS ? a.cache.width : SMEM_KEYS) * 8;
  if (fused(a)) {
    const auto kernel = paged_select_kernel<T, LANES, GH, true>;
    if (bytes > 32 * 1024 && !attn::allow_smem(kernel, SMEM_KEYS * 8, done[0])) return GDNX_ELAUNCH;
    return launched(launch_early(kernel, dim3(1, y, z), dim3(NT), bytes, st, P));
  }
  // CTAs that fill the device twice over, of two batches of pages for each warp at least: reading q costs about one
  constexpr int64_t STEP = 2 * NT / LANES * (GH == 1 ? 8 : 16 / GH);
  const int64_t want = ((int64_t)sm_count() * 2 + units - 1) / units, have = (n + STEP - 1) / STEP;
  P.splits = (int)(want < have ? want : have);
  if (launch_early(paged_select_kernel<T, LANES, GH, false>, dim3((unsigned)P.splits, y, z), dim3(NT), 0, st, P) != cudaSuccess)
    return GDNX_ELAUNCH;
  if (bytes > 32 * 1024 && !attn::allow_smem(paged_take_kernel, SMEM_KEYS * 8, done[1])) return GDNX_ELAUNCH;
  return launched(launch_early(paged_take_kernel, dim3((unsigned)units), dim3(TAKE_NT), bytes, st, P));
}

template <typename T, int LANES>
gdnx_status select_heads(const gdnx_paged_select_args& a, cudaStream_t st) {
  const int64_t G = a.H / a.cache.Hk;
  return G == 1 ? select_of<T, LANES, 1>(a, st) : select_of<T, LANES, 4>(a, st);
}

template <typename T>
gdnx_status select_type(const gdnx_paged_select_args& a, cudaStream_t st) {
  const int64_t D = a.cache.D;
  return D > 64 ? select_heads<T, 32>(a, st) : D > 32 ? select_heads<T, 16>(a, st) : select_heads<T, 8>(a, st);
}

}  // namespace

size_t paged_select_workspace_bytes(const gdnx_paged_select_args& a) {
  return fused(a) ? 0 : (size_t)(a.B * a.cache.Hk * a.cache.width) * 8;
}

gdnx_status launch_paged_select(const gdnx_paged_select_args& a, cudaStream_t st) {
  switch (a.cache.dtype) {
    case GDNX_BF16: return select_type<__nv_bfloat16>(a, st);
    case GDNX_F16: return select_type<__half>(a, st);
    default: return select_type<float>(a, st);
  }
}

}  // namespace gdnx
