// What a serving step writes into a paged cache: the packed new tokens' keys and values at the places that the step
// gave them, and the bounds of the keys on the pages they touched.
//
// append: bytes bound it.  A thread keeps one 16-byte piece of a token (side, head and part of the head's row are found
// once) and walks over the tokens, four at a time in flight.
// bounds: lo_d = min_j k_jd, hi_d = max_j k_jd over a page's tokens, exact in the cache's type, NaN where a key is.
// Bytes bound it: every key of the touched pages is read once, by one CTA for each page and head whose threads take
// 16 bytes of a row each and every so many rows.
//
// Measured (4 heads of 128, bf16): append of 24,500 tokens (100 MB moved) 16 us, 6.2 TB/s; of 64 tokens 2.0 us.  bounds of
// 8 x 4096 tokens 10.5 us (3.3 TB/s), behind one token in each of 64 slots 4.9 us: the check of the call, under which the
// first page's keys come, and the chain from slot to page to keys.  Behind one token in each of 4096 slots 63 us: checked
// by every CTA, such a call took 599, which grew with the square of the rows.
#include "paged_cache.cuh"

namespace gdnx {
namespace {

constexpr int APPEND_NT = 256;
constexpr int TOKENS = 4;  // of a thread in flight
constexpr int BOUNDS_NT = 128;
constexpr int CHECK_NT = 1024;

template <typename V>
__global__ void __launch_bounds__(APPEND_NT) cache_append_kernel(const gdnx_cache c, int64_t layer, int64_t tokens,
                                                                 const gdnx_view k, const gdnx_view v,
                                                                 const int64_t* places, int es) {
  dependents_may_start();
  wait_for_earlier();
  if (*c.status != 0) return;
  const int per = (int)(c.D * es / sizeof(V)), all = 2 * (int)c.Hk * per;  // pieces of a head's row, of a token
  const int together = all < APPEND_NT ? APPEND_NT / all : 1;               // tokens side by side in a CTA
  const int shift = 31 - __clz(c.page);
  const int64_t row = c.D * es, head = row << shift, page = c.Hk * head, most = c.pages << shift;
  const int64_t step = (int64_t)gridDim.x * together;
  for (int x = threadIdx.x; x < all * together; x += APPEND_NT) {
    const int e = x % all, piece = e % per, h = e / per % (int)c.Hk, side = e / (per * (int)c.Hk);
    const gdnx_view& in = side ? v : k;
    const char* src = static_cast<const char*>(in.ptr) + h * in.sh * es + piece * (int)sizeof(V);
    char* dst = static_cast<char*>(c.kv) + (layer * 2 + side) * c.pages * page + h * head + piece * (int)sizeof(V);
    for (int64_t t0 = (int64_t)blockIdx.x * together + x / all; t0 < tokens; t0 += TOKENS * step) {
      int64_t place[TOKENS];
      V w[TOKENS];
#pragma unroll
      for (int i = 0; i < TOKENS; ++i) {
        const int64_t t = t0 + i * step;
        place[i] = t < tokens ? places[t] : -1;
        if (place[i] >= most) place[i] = -1;
        if (t < tokens) w[i] = *reinterpret_cast<const V*>(src + t * in.st * es);
      }
#pragma unroll
      for (int i = 0; i < TOKENS; ++i)
        if (place[i] >= 0)
          *reinterpret_cast<V*>(dst + (place[i] >> shift) * page + (place[i] & (c.page - 1)) * row) = w[i];
    }
  }
}

GDNX_DEV uint32_t least(uint32_t a, uint32_t b, float) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(__uint_as_float(a)), "f"(__uint_as_float(b)));
  return __float_as_uint(r);
}
GDNX_DEV uint32_t most(uint32_t a, uint32_t b, float) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(__uint_as_float(a)), "f"(__uint_as_float(b)));
  return __float_as_uint(r);
}
GDNX_DEV uint32_t least(uint32_t a, uint32_t b, __nv_bfloat16) {
  uint32_t r;
  asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
GDNX_DEV uint32_t most(uint32_t a, uint32_t b, __nv_bfloat16) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
GDNX_DEV uint32_t least(uint32_t a, uint32_t b, __half) {
  uint32_t r;
  asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
GDNX_DEV uint32_t most(uint32_t a, uint32_t b, __half) {
  uint32_t r;
  asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <typename T>
GDNX_DEV uint4 least4(uint4 a, uint4 b) {
  return make_uint4(least(a.x, b.x, T()), least(a.y, b.y, T()), least(a.z, b.z, T()), least(a.w, b.w, T()));
}
template <typename T>
GDNX_DEV uint4 most4(uint4 a, uint4 b) {
  return make_uint4(most(a.x, b.x, T()), most(a.y, b.y, T()), most(a.z, b.z, T()), most(a.w, b.w, T()));
}

// True in every thread when the bounds of these rows' newest tokens can be found: no operation was refused before, each slot
// once and in range, no more tokens than the slot has, and no partly filled last page that another slot holds too (which
// may see more of it).
GDNX_DEV bool bounds_ok(uint32_t* seen, const gdnx_cache& c, int64_t n, const int32_t* rows, const int32_t* counts) {
  bool bad = *c.status != 0;  // (voted on below: another CTA may set it meanwhile)
  if (!rows_ok(seen, c, n, rows, nullptr, counts)) return false;
  for (int64_t i = threadIdx.x; i < n; i += blockDim.x) {
    const int64_t len = length_of(c, rows[i]);
    bad |= counts[i] > len;
    if (counts[i] > 0 && !bad && len % c.page) {
      const int p = c.table[rows[i] * c.width + len / c.page];
      bad |= page_ok(c, p) && c.refs[p] > 1;
    }
  }
  return !__syncthreads_or(bad);
}

// The check by one CTA, for calls of many rows.
__global__ void __launch_bounds__(CHECK_NT) cache_bounds_check_kernel(const gdnx_cache c, int64_t n, const int32_t* rows,
                                                                      const int32_t* counts) {
  extern __shared__ uint32_t seen[];
  dependents_may_start();
  wait_for_earlier();
  if (!bounds_ok(seen, c, n, rows, counts) && threadIdx.x == 0 && *c.status == 0) *c.status = GDNX_EINVAL;
}

// CTA (h, i, z): head h of every gridDim.z-th page that holds one of the newest tokens of slot rows[i].  CHECK: every CTA
// checks the call itself and decides like the others; it reads its first page's keys before, and writes after.
template <typename T, bool CHECK>
__global__ void __launch_bounds__(BOUNDS_NT) cache_bounds_kernel(const gdnx_cache c, int64_t layer, int64_t n,
                                                                 const int32_t* rows, const int32_t* counts,
                                                                 uint4* bounds) {
  extern __shared__ uint32_t seen[];
  __shared__ uint4 part[2][BOUNDS_NT];
  dependents_may_start();
  wait_for_earlier();
  const int per = (int)(c.D * sizeof(T) / 16), groups = BOUNDS_NT / per;  // pieces of a row, rows side by side
  const int piece = threadIdx.x % per, group = threadIdx.x / per, h = blockIdx.x;
  const bool first_cta = blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0;
  bool checked = !CHECK;
  if (!CHECK && *c.status != 0) return;
  for (int64_t i = blockIdx.y; i < n; i += gridDim.y) {
    const int row = rows[i];
    if (row < 0 || row >= c.slots) continue;  // refused by the CTAs that have work
    const int64_t len = length_of(c, row), count = min((int64_t)counts[i], len);
    if (count <= 0) continue;
    for (int64_t x = (len - count) / c.page + blockIdx.z; x * c.page < len; x += gridDim.z) {
      const int p = c.table[row * c.width + x];
      if (!page_ok(c, p)) continue;
      const int have = (int)min((int64_t)c.page, len - x * c.page);
      const uint4* src = static_cast<const uint4*>(c.kv) + ((layer * 2 * c.pages + p) * c.Hk + h) * c.page * per + piece;
      constexpr int AHEAD = 8;  // rows in flight, those of the first page under the checks
      uint4 k[AHEAD];
#pragma unroll
      for (int e = 0; e < AHEAD; ++e)
        if (group < groups && group + e * groups < have) k[e] = src[(group + e * groups) * per];
      if (!checked) {
        if (!bounds_ok(seen, c, n, rows, counts)) {
          if (first_cta && threadIdx.x == 0 && *c.status == 0) *c.status = GDNX_EINVAL;
          return;
        }
        checked = true;
      }
      if (group < groups) {
        uint4 lo = k[0], hi = k[0];
        for (int r = group; r < have; r += AHEAD * groups) {
          if (r > group) {
#pragma unroll
            for (int e = 0; e < AHEAD; ++e)
              if (r + e * groups < have) k[e] = src[(r + e * groups) * per];
          }
#pragma unroll
          for (int e = 0; e < AHEAD; ++e)
            if (r + e * groups < have) {
              lo = least4<T>(lo, k[e]);
              hi = most4<T>(hi, k[e]);
            }
        }
        part[0][threadIdx.x] = lo;
        part[1][threadIdx.x] = hi;
      }
      __syncthreads();
      if (threadIdx.x < 2 * per) {
        const int side = threadIdx.x / per, e = threadIdx.x % per;
        uint4 r = part[side][e];
        for (int g = 1; g < groups && g < have; ++g) {
          const uint4 k = part[side][g * per + e];
          r = side ? most4<T>(r, k) : least4<T>(r, k);
        }
        bounds[(((layer * 2 + side) * c.pages + p) * c.Hk + h) * per + e] = r;
      }
      __syncthreads();
    }
  }
  if (!checked && first_cta && !bounds_ok(seen, c, n, rows, counts) && threadIdx.x == 0 && *c.status == 0)
    *c.status = GDNX_EINVAL;
}

template <typename T, bool CHECK>
cudaError_t bounds_of(const gdnx_cache& c, int64_t layer, int64_t n, const int32_t* rows, const int32_t* counts,
                      void* bounds, cudaStream_t st) {
  // as many CTAs as keep the device busy; where the pages of a call are fewer, the others find none
  const int64_t y = n < 65535 ? n : 65535, fill = (int64_t)sm_count() * 8 / (c.Hk * y), z = fill < 1 ? 1 : fill < c.width ? fill : c.width;
  return launch_early(cache_bounds_kernel<T, CHECK>, dim3((unsigned)c.Hk, (unsigned)y, (unsigned)(z < 65535 ? z : 65535)),
                      dim3(BOUNDS_NT), CHECK ? seen_bytes(c) : 0, st, c, layer, n, rows, counts, static_cast<uint4*>(bounds));
}

// A check that takes every thread of a CTA one step runs in the CTAs that find the bounds; longer ones run once, in a CTA
// of their own before them (one new token in each of 128 slots: 4.8 us in the CTAs; of 200 slots 9.7 in the CTAs, 6.6 in
// its own; of 1024 slots 53 and 16).
template <typename T>
gdnx_status bounds_call(const gdnx_cache& c, int64_t layer, int64_t n, const int32_t* rows, const int32_t* counts,
                        void* bounds, cudaStream_t st) {
  if (n <= BOUNDS_NT && seen_bytes(c) <= BOUNDS_NT * 4) return launched(bounds_of<T, true>(c, layer, n, rows, counts, bounds, st));
  if (launch_early(cache_bounds_check_kernel, dim3(1), dim3(CHECK_NT), seen_bytes(c), st, c, n, rows, counts) != cudaSuccess)
    return GDNX_ELAUNCH;
  return launched(bounds_of<T, false>(c, layer, n, rows, counts, bounds, st));
}

}  // namespace

gdnx_status launch_cache_append(const gdnx_cache& c, int64_t layer, int64_t tokens, const gdnx_view& k,
                                const gdnx_view& v, const int64_t* places, cudaStream_t st) {
  const int es = elem(c.dtype), vec = 16 / es;
  const auto wide = [&](const gdnx_view& x) {
    return reinterpret_cast<uintptr_t>(x.ptr) % 16 == 0 && x.st % vec == 0 && x.sh % vec == 0;
  };
  const bool v16 = wide(k) && wide(v);
  const int64_t all = 2 * c.Hk * (v16 ? c.D / vec : c.D), together = all < APPEND_NT ? APPEND_NT / all : 1;
  const int64_t need = (tokens + together - 1) / together, most = (int64_t)sm_count() * 8;
  const auto kernel = v16 ? cache_append_kernel<uint4> : es == 4 ? cache_append_kernel<uint32_t> : cache_append_kernel<uint16_t>;
  return launched(launch_early(kernel, dim3((unsigned)(need < most ? need : most)), dim3(APPEND_NT), 0, st, c, layer, tokens,
                               k, v, places, es));
}

gdnx_status launch_cache_bounds(const gdnx_cache& c, int64_t layer, int64_t n, const int32_t* rows,
                                const int32_t* counts, void* bounds, cudaStream_t st) {
  switch (c.dtype) {
    case GDNX_BF16: return bounds_call<__nv_bfloat16>(c, layer, n, rows, counts, bounds, st);
    case GDNX_F16: return bounds_call<__half>(c, layer, n, rows, counts, bounds, st);
    default: return bounds_call<float>(c, layer, n, rows, counts, bounds, st);
  }
}

}  // namespace gdnx
