// Page operations of a paged key/value cache (gdnx_cache): fork, extend, write, truncate,
// trim, compact.  The page table, the lengths and the reference counts live on the device,
// so that a serving step needs no host synchronisation and can be captured in a graph.
//
// Every operation is decided before it changes anything.  The row operations (fork,
// truncate, trim) have one CTA per row, each of which checks the whole list of rows
// itself, so that all CTAs decide alike without a word between them; counts move by
// integer atomics, whose order does not show.  extend and compact are planned by one CTA
// (the free pages are ranked by a scan over refs, so allocation is lowest index first
// whatever the thread order); a second kernel moves the pages.
//
// Bytes moved bound extend's copies and compact.  write of whole prompts is bound by its index arithmetic (77 % of
// issue slots, 15 % of DRAM).  The row operations are one short launch for up to some hundreds of rows (trim of 64:
// 2.3 us), but every CTA reads the whole list (4096 rows: 69 us).  The scans over refs grow with the pool: where
// only its last pages are free, extend takes 17 us with 4096 pages and 98 us with 262,144 (compact with nothing to
// move: 11 and 170 us).
// Measured: 32 requests of up to 1500 tokens forked, extended by 5 tokens (their last pages copied in 24
// layers), written in one layer and trimmed: 57 us (198 MB); compaction after waves of requests moves
// pages at 85 % of a copy's rate; write of 64 x 1 tokens 4.2 us (its checks: 1.1), of 8 x 4096 tokens of 4 heads of
// 128 in bf16 56 us.
#include "common.cuh"
#include "kernels.h"
#include "launch.cuh"

namespace gdnx {
namespace {

constexpr int NT = 1024;      // threads of a planning CTA
constexpr int ROW_NT = 128;   // threads of a row CTA
constexpr int COPY_NT = 256;
constexpr int WRITE_NT = 256;
constexpr int COPY_VEC = 4;   // 16-byte words in flight for each thread of a copy
constexpr int HEAD = 64;      // workspace words before the lists: [0] copies, [1] live pages

// Workspace (int32): HEAD words, the copies' sources and destinations, then for extend
// the free pages in order and each row's first free-page rank, for compact the new place
// of each moved page.
struct Plan {
  int32_t *head, *src, *dst, *list, *off;
  __host__ __device__ Plan(void* ws, int64_t pages, int64_t n) {
    const int64_t m = n > pages ? n : pages;
    head = static_cast<int32_t*>(ws);
    src = head + HEAD;
    dst = src + m;
    list = dst + m;
    off = list + pages;
  }
  static size_t bytes(int64_t pages, int64_t n) {
    const int64_t m = n > pages ? n : pages;
    return (size_t)(HEAD + 2 * m + pages + n) * sizeof(int32_t);
  }
};

// True in every thread when all rows are slots and none is named twice (and, where
// `other` is given, its rows are slots not among `rows`).  `seen` has slots bits.
GDNX_DEV bool rows_ok(uint32_t* seen, const gdnx_cache& c, int64_t n, const int32_t* rows, const int32_t* other,
                      const int32_t* counts) {
  for (int64_t i = threadIdx.x; i < (c.slots + 31) / 32; i += blockDim.x) seen[i] = 0;
  __syncthreads();
  bool bad = false;
  for (int64_t i = threadIdx.x; i < n; i += blockDim.x) {
    const int r = rows[i];
    if (r < 0 || r >= c.slots) bad = true;
    else bad |= (atomicOr(&seen[r / 32], 1u << (r % 32)) >> (r % 32)) & 1u;
    if (counts) bad |= counts[i] < 0;
  }
  __syncthreads();
  if (other)
    for (int64_t i = threadIdx.x; i < n; i += blockDim.x) {
      const int r = other[i];
      if (r < 0 || r >= c.slots) bad = true;
      else bad |= (seen[r / 32] >> (r % 32)) & 1u;
    }
  return !__syncthreads_or(bad);
}

GDNX_DEV bool page_ok(const gdnx_cache& c, int p) { return p >= 0 && p < c.pages; }

GDNX_DEV int64_t pages_of(const gdnx_cache& c, int64_t tokens) { return (tokens + c.page - 1) / c.page; }

// A slot's length, kept within what its row can hold.
GDNX_DEV int64_t length_of(const gdnx_cache& c, int row) {
  const int64_t n = c.lengths[row], most = c.width * c.page;
  return n < 0 ? 0 : (n > most ? most : n);
}

enum RowOp { kFork, kTruncate, kTrim };

template <int OP>
__global__ void __launch_bounds__(ROW_NT) cache_rows_kernel(const gdnx_cache c, int64_t n, const int32_t* rows,
                                                            const int32_t* arg, int64_t window, int64_t sinks) {
  extern __shared__ uint32_t seen[];
  dependents_may_start();
  wait_for_earlier();
  if (*c.status != 0) return;
  if (!rows_ok(seen, c, n, rows, OP == kFork ? arg : nullptr, OP == kTruncate ? arg : nullptr)) {
    if (blockIdx.x == 0 && threadIdx.x == 0) *c.status = GDNX_EINVAL;
    return;
  }
  const int row = rows[blockIdx.x];
  int32_t* mine = c.table + row * c.width;
  const int64_t len = length_of(c, row);
  if (OP == kFork) {
    const int from = arg[blockIdx.x];
    const int32_t* theirs = c.table + from * c.width;
    for (int64_t i = threadIdx.x; i < c.width; i += ROW_NT) {
      const int was = mine[i], now = theirs[i];
      if (page_ok(c, was)) atomicSub(&c.refs[was], 1);
      if (page_ok(c, now)) atomicAdd(&c.refs[now], 1);
      mine[i] = now;
    }
    if (threadIdx.x == 0) c.lengths[row] = c.lengths[from];
    return;
  }
  const int64_t keep = OP == kTruncate ? min(len, (int64_t)arg[blockIdx.x]) : len;
  for (int64_t i = threadIdx.x; i < c.width; i += ROW_NT) {
    const int p = mine[i];
    const int64_t first = i * c.page;
    const bool drop = OP == kTruncate ? i >= pages_of(c, keep) : first >= sinks && first + c.page <= len - window;
    if (drop && p != -1) {
      if (page_ok(c, p)) atomicSub(&c.refs[p], 1);
      mine[i] = -1;
    }
  }
  __syncthreads();  // every thread has read the length
  if (OP == kTruncate && threadIdx.x == 0) c.lengths[row] = (int32_t)keep;
}

// Exclusive prefix sum of one value per thread over the CTA, and the total.
GDNX_DEV int block_scan(int x, int* warp_sums, int* total) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  int s = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += y;
  }
  if (lane == 31) warp_sums[warp] = s;
  __syncthreads();
  if (warp == 0) {
    int w = warp_sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += y;
    }
    warp_sums[lane] = w;
  }
  __syncthreads();
  const int before = warp > 0 ? warp_sums[warp - 1] : 0;
  *total = warp_sums[31];
  __syncthreads();
  return before + s - x;
}

// refs of pages p..p+3 (as many as there are; beyond the pool: `fill`)
GDNX_DEV void load4(int (&r)[4], const gdnx_cache& c, int64_t p, int fill) {
#pragma unroll
  for (int e = 0; e < 4; ++e) r[e] = p + e < c.pages ? c.refs[p + e] : fill;
}

__global__ void __launch_bounds__(NT) cache_extend_kernel(const gdnx_cache c, int64_t n, const int32_t* rows,
                                                          const int32_t* counts, void* ws) {
  extern __shared__ uint32_t seen[];
  __shared__ int sums[32];
  __shared__ int ncopy;
  const Plan w(ws, c.pages, n);
  dependents_may_start();
  wait_for_earlier();
  if (threadIdx.x == 0) {
    w.head[0] = 0;
    ncopy = 0;
  }
  if (*c.status != 0) return;
  if (!rows_ok(seen, c, n, rows, nullptr, counts)) {
    if (threadIdx.x == 0) *c.status = GDNX_EINVAL;
    return;
  }
  // what each row needs: its new pages, and one more where a shared last page is copied; `lost`: the new
  // tokens would begin on a page that was released (trimmed, and the slot cut back into it since)
  const auto ask = [&](int64_t i, int64_t& first, int64_t& need, int& shared, bool& lost) {
    const int64_t len = length_of(c, rows[i]);
    const int64_t have = pages_of(c, len), want = pages_of(c, len + counts[i]);
    shared = -1;
    if (counts[i] > 0 && len % c.page) {
      const int tail = c.table[rows[i] * c.width + have - 1];
      if (!page_ok(c, tail)) lost = true;
      else if (c.refs[tail] > 1) shared = tail;
    }
    first = have - (shared >= 0);
    need = want - first;
    return want <= c.width;
  };
  bool full = false, lost = false;
  int64_t total = 0;
  for (int64_t base = 0; base < n; base += NT) {
    const int64_t i = base + threadIdx.x;
    int64_t first = 0, need = 0;
    int shared, sum;
    if (i < n) full |= !ask(i, first, need, shared, lost);
    if (full) need = 0;  // refused below; keeps the sums small
    const int at = block_scan((int)need, sums, &sum);
    if (i < n) w.off[i] = (int)(total + at);
    total += sum;
  }
  if (__syncthreads_or(lost)) {
    if (threadIdx.x == 0) *c.status = GDNX_EINVAL;
    return;
  }
  if (__syncthreads_or(full || total > c.pages)) {
    if (threadIdx.x == 0) *c.status = GDNX_ENOPAGES;
    return;
  }
  int64_t found = 0;
  for (int64_t base = 0; base < c.pages && found < total; base += 4 * NT) {
    int r[4], sum;
    load4(r, c, base + 4 * threadIdx.x, 1);
    int at = block_scan((r[0] == 0) + (r[1] == 0) + (r[2] == 0) + (r[3] == 0), sums, &sum);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (r[e] == 0) {
        if (found + at < total) w.list[found + at] = (int)(base + 4 * threadIdx.x + e);
        ++at;
      }
    found += sum;
  }
  if (found < total) {
    if (threadIdx.x == 0) *c.status = GDNX_ENOPAGES;
    return;
  }
  __syncthreads();  // the list is whole
  // refs of shared pages are read above and below by every row before any is changed
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  for (int64_t i0 = 0; i0 < n; i0 += NT / 32) {
    const int64_t i = i0 + warp;
    int64_t first = 0, need = 0;
    int shared = -1;
    if (i < n) ask(i, first, need, shared, lost);
    if (i < n) w.off[i] |= shared >= 0 ? (int)0x80000000 : 0;
  }
  __syncthreads();
  for (int64_t i = warp; i < n; i += NT / 32) {
    const int row = rows[i];
    const int64_t len = length_of(c, row), have = pages_of(c, len), want = pages_of(c, len + counts[i]);
    const bool cow = w.off[i] < 0;
    const int off = w.off[i] & 0x7fffffff;
    int32_t* mine = c.table + row * c.width;
    const int64_t first = have - cow;
    if (cow && lane == 0) {
      const int k = atomicAdd(&ncopy, 1), tail = mine[first];
      w.src[k] = tail;
      w.dst[k] = w.list[off];
      atomicSub(&c.refs[tail], 1);
    }
    __syncwarp();
    for (int64_t k = lane; k < want - first; k += 32) {
      const int p = w.list[off + k];
      mine[first + k] = p;
      c.refs[p] = 1;
    }
    __syncwarp();
    if (lane == 0) c.lengths[row] = (int32_t)(len + counts[i]);
  }
  __syncthreads();
  if (threadIdx.x == 0) w.head[0] = ncopy;
}

__global__ void __launch_bounds__(NT) cache_compact_kernel(const gdnx_cache c, void* ws) {
  __shared__ int sums[32];
  const Plan w(ws, c.pages, 0);
  dependents_may_start();
  wait_for_earlier();
  if (threadIdx.x == 0) w.head[0] = 0;
  if (*c.status != 0) return;
  int64_t live = 0;
  for (int64_t base = 0; base < c.pages; base += 4 * NT) {
    int r[4], sum;
    load4(r, c, base + 4 * threadIdx.x, 0);
    block_scan((r[0] > 0) + (r[1] > 0) + (r[2] > 0) + (r[3] > 0), sums, &sum);
    live += sum;
  }
  int64_t holes = 0, moved = 0;
  for (int64_t base = 0; base < c.pages; base += 4 * NT) {
    int r[4], nh = 0, nm = 0, sh, sm;
    const int64_t p = base + 4 * threadIdx.x;
    load4(r, c, p, 0);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      nh += p + e < live && r[e] <= 0;
      nm += p + e >= live && r[e] > 0;
    }
    int h = block_scan(nh, sums, &sh), m = block_scan(nm, sums, &sm);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (p + e < live && r[e] <= 0) w.dst[holes + h++] = (int)(p + e);
      if (p + e >= live && r[e] > 0) w.src[moved + m++] = (int)(p + e);
    }
    holes += sh;
    moved += sm;
  }
  __syncthreads();  // both lists are whole, and as long as one another
  for (int64_t i = threadIdx.x; i < moved; i += NT) {
    const int from = w.src[i], to = w.dst[i];
    c.refs[to] = c.refs[from];
    c.refs[from] = 0;
    w.list[from] = to;
  }
  if (threadIdx.x == 0) {
    w.head[0] = (int)moved;
    w.head[1] = (int)live;
  }
}

// Moves the planned pages in every layer; for compact also renames them in the table.
// A page of one layer's keys or values is one contiguous run.  Sources and destinations
// are different pages, so the moves are independent.
__global__ void __launch_bounds__(COPY_NT) cache_copy_kernel(const gdnx_cache c, void* ws, int64_t n, int64_t run,
                                                             int rename) {
  const Plan w(ws, c.pages, n);
  dependents_may_start();
  wait_for_earlier();
  const int m = w.head[0];
  if (m == 0) return;
  if (rename) {
    const int live = w.head[1];
    for (int64_t i = (int64_t)blockIdx.x * COPY_NT + threadIdx.x; i < c.slots * c.width;
         i += (int64_t)gridDim.x * COPY_NT) {
      const int p = c.table[i];
      if (p >= live && p < c.pages) c.table[i] = w.list[p];
    }
  }
  constexpr int UNIT = COPY_NT * COPY_VEC;  // 16-byte words
  const int64_t words = run / 16, per = (words + UNIT - 1) / UNIT, sides = c.L * 2;
  uint4* kv = static_cast<uint4*>(c.kv);
  for (int64_t u = blockIdx.x; u < per * sides * m; u += gridDim.x) {
    const int64_t part = u % per, side = u / per % sides, k = u / (per * sides);
    const uint4* src = kv + (side * c.pages + w.src[k]) * words;
    uint4* dst = kv + (side * c.pages + w.dst[k]) * words;
    uint4 x[COPY_VEC];
#pragma unroll
    for (int e = 0; e < COPY_VEC; ++e) {
      const int64_t i = part * UNIT + e * COPY_NT + threadIdx.x;
      if (i < words) x[e] = __ldcs(src + i);
    }
#pragma unroll
    for (int e = 0; e < COPY_VEC; ++e) {
      const int64_t i = part * UNIT + e * COPY_NT + threadIdx.x;
      if (i < words) __stcs(dst + i, x[e]);
    }
  }
}

// Pages that a write of T tokens touches in a slot, at most.
__host__ __device__ inline int64_t pages_touched(const gdnx_cache& c, int64_t T) {
  const int64_t most = (T + c.page - 2) / c.page + 1;
  return most < c.width ? most : c.width;
}

// True in every thread when a write can be carried out: no operation was refused before, each slot once and in range, 0 <= count <= T tokens
// that the slot has, and every page they lie on held by this slot alone.  `seen` has slots bits.
GDNX_DEV bool write_ok(uint32_t* seen, const gdnx_cache& c, int64_t n, int64_t T, const int32_t* rows,
                       const int32_t* counts) {
  for (int64_t i = threadIdx.x; i < (c.slots + 31) / 32; i += blockDim.x) seen[i] = 0;
  bool bad = *c.status != 0;
  __syncthreads();
  const int64_t span = pages_touched(c, T);
  for (int64_t x = threadIdx.x; x < n * span; x += blockDim.x) {
    const int64_t i = x / span, k = x % span, count = counts ? counts[i] : T;
    const int row = rows[i];
    if (row < 0 || row >= c.slots || count < 0 || count > T) {
      bad = true;
      continue;
    }
    if (k == 0) bad |= (atomicOr(&seen[row / 32], 1u << (row % 32)) >> (row % 32)) & 1u;
    const int64_t len = length_of(c, row), at = (len - count) / c.page + k;
    if (count > len) bad = true;
    else if (count > 0 && at <= (len - 1) / c.page) {
      const int p = c.table[row * c.width + at];
      bad |= !page_ok(c, p) || c.refs[p] != 1;
    }
  }
  return !__syncthreads_or(bad);
}

// The check by one CTA, for writes of many pages.
__global__ void __launch_bounds__(NT) cache_write_check_kernel(const gdnx_cache c, int64_t n, int64_t T,
                                                               const int32_t* rows, const int32_t* counts) {
  extern __shared__ uint32_t seen[];
  dependents_may_start();
  wait_for_earlier();
  if (!write_ok(seen, c, n, T, rows, counts) && threadIdx.x == 0 && *c.status == 0) *c.status = GDNX_EINVAL;
}

// One V-typed piece of a token's key or value for each thread.  CHECK: every CTA checks the call itself and
// decides like the others.
template <typename V, bool CHECK>
__global__ void __launch_bounds__(WRITE_NT) cache_write_kernel(const gdnx_cache c, int64_t layer, int64_t n, int64_t T,
                                                               const gdnx_view k, const gdnx_view v,
                                                               const int32_t* rows, const int32_t* counts, int es) {
  extern __shared__ uint32_t seen[];
  dependents_may_start();
  wait_for_earlier();
  if (CHECK ? !write_ok(seen, c, n, T, rows, counts) : *c.status != 0) {
    if (CHECK && blockIdx.x == 0 && threadIdx.x == 0 && *c.status == 0) *c.status = GDNX_EINVAL;
    return;
  }
  const int per = (int)(c.D * es / sizeof(V));  // pieces of one head
  const int64_t all = n * T * c.Hk * per * 2;
  for (int64_t x = (int64_t)blockIdx.x * WRITE_NT + threadIdx.x; x < all; x += (int64_t)gridDim.x * WRITE_NT) {
    const int64_t e = x % per, h = x / per % c.Hk, t = x / (per * c.Hk) % T, i = x / (per * c.Hk * T) % n;
    const int side = (int)(x / (per * c.Hk * T * n));
    const int row = rows[i];
    const int64_t count = counts ? counts[i] : T;
    if (t >= count) continue;
    const int64_t pos = length_of(c, row) - count + t;
    const int p = c.table[row * c.width + pos / c.page];
    const gdnx_view& in = side ? v : k;
    const V* src = reinterpret_cast<const V*>(static_cast<const char*>(in.ptr) + (i * in.sb + t * in.st + h * in.sh) * es);
    char* at = static_cast<char*>(c.kv) +
               ((((layer * 2 + side) * c.pages + p) * c.Hk + h) * c.page + pos % c.page) * c.D * es;
    reinterpret_cast<V*>(at)[e] = src[e];
  }
}

size_t seen_bytes(const gdnx_cache& c) { return (size_t)((c.slots + 31) / 32) * 4; }

gdnx_status launched(cudaError_t e) { return e == cudaSuccess ? GDNX_OK : GDNX_ELAUNCH; }

int elem(int dtype) { return dtype == GDNX_F32 ? 4 : 2; }

gdnx_status copy_pages(const gdnx_cache& c, void* ws, int64_t n, int rename, cudaStream_t st) {
  const int64_t run = c.Hk * c.page * c.D * elem(c.dtype);
  return launched(launch_early(cache_copy_kernel, dim3(sm_count() * 8), dim3(COPY_NT), 0, st, c, ws, n, run, rename));
}

}  // namespace

size_t cache_workspace_bytes(const gdnx_cache& c, int64_t n) { return Plan::bytes(c.pages, n); }

gdnx_status launch_cache_fork(const gdnx_cache& c, int64_t n, const int32_t* src, const int32_t* dst, cudaStream_t st) {
  return launched(launch_early(cache_rows_kernel<kFork>, dim3((unsigned)n), dim3(ROW_NT), seen_bytes(c), st, c, n, dst,
                               src, 0, 0));
}

gdnx_status launch_cache_truncate(const gdnx_cache& c, int64_t n, const int32_t* rows, const int32_t* lengths,
                                  cudaStream_t st) {
  return launched(launch_early(cache_rows_kernel<kTruncate>, dim3((unsigned)n), dim3(ROW_NT), seen_bytes(c), st, c, n,
                               rows, lengths, 0, 0));
}

gdnx_status launch_cache_trim(const gdnx_cache& c, int64_t n, const int32_t* rows, int64_t window, int64_t sinks,
                              cudaStream_t st) {
  return launched(launch_early(cache_rows_kernel<kTrim>, dim3((unsigned)n), dim3(ROW_NT), seen_bytes(c), st, c, n, rows,
                               nullptr, window, sinks));
}

gdnx_status launch_cache_extend(const gdnx_cache& c, int64_t n, const int32_t* rows, const int32_t* counts, void* ws,
                                cudaStream_t st) {
  if (launch_early(cache_extend_kernel, dim3(1), dim3(NT), seen_bytes(c), st, c, n, rows, counts, ws) != cudaSuccess)
    return GDNX_ELAUNCH;
  return copy_pages(c, ws, n, 0, st);
}

gdnx_status launch_cache_compact(const gdnx_cache& c, void* ws, cudaStream_t st) {
  if (launch_early(cache_compact_kernel, dim3(1), dim3(NT), 0, st, c, ws) != cudaSuccess) return GDNX_ELAUNCH;
  return copy_pages(c, ws, 0, 1, st);
}

namespace {

template <bool CHECK>
cudaError_t write_pieces(const gdnx_cache& c, int64_t layer, int64_t n, int64_t T, const gdnx_view& k,
                         const gdnx_view& v, const int32_t* rows, const int32_t* counts, cudaStream_t st) {
  const int es = elem(c.dtype), vec = 16 / es;
  const auto wide = [&](const gdnx_view& x) {
    return reinterpret_cast<uintptr_t>(x.ptr) % 16 == 0 && x.sb % vec == 0 && x.st % vec == 0 && x.sh % vec == 0;
  };
  const bool v16 = wide(k) && wide(v);
  const int64_t all = n * T * c.Hk * (v16 ? c.D / vec : c.D) * 2;
  const int64_t most = sm_count() * 64;
  const unsigned grid = (unsigned)((all + WRITE_NT - 1) / WRITE_NT < most ? (all + WRITE_NT - 1) / WRITE_NT : most);
  const auto kernel = v16 ? cache_write_kernel<uint4, CHECK>
                      : es == 4 ? cache_write_kernel<uint32_t, CHECK> : cache_write_kernel<uint16_t, CHECK>;
  return launch_early(kernel, dim3(grid), dim3(WRITE_NT), CHECK ? seen_bytes(c) : 0, st, c, layer, n, T, k, v, rows,
                      counts, es);
}

}  // namespace

// A check that takes every thread of a CTA one step runs in the CTAs that write; longer ones run once, in a
// CTA of their own before them.
gdnx_status launch_cache_write(const gdnx_cache& c, int64_t layer, int64_t n, int64_t T, const gdnx_view& k,
                               const gdnx_view& v, const int32_t* rows, const int32_t* counts, cudaStream_t st) {
  if (n * pages_touched(c, T) <= WRITE_NT && seen_bytes(c) <= WRITE_NT * 4)
    return launched(write_pieces<true>(c, layer, n, T, k, v, rows, counts, st));
  if (launch_early(cache_write_check_kernel, dim3(1), dim3(NT), seen_bytes(c), st, c, n, T, rows, counts) != cudaSuccess)
    return GDNX_ELAUNCH;
  return launched(write_pieces<false>(c, layer, n, T, k, v, rows, counts, st));
}

}  // namespace gdnx
