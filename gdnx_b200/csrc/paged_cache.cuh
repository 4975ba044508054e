// What the cache's page operations share: checks of a call's rows, and pages and lengths of slots.
#pragma once

#include "common.cuh"
#include "kernels.h"
#include "launch.cuh"

namespace gdnx {
namespace {  // one copy for each kernel file

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

// (A page has a power of two tokens.)
GDNX_DEV int64_t pages_of(const gdnx_cache& c, int64_t tokens) { return (tokens + c.page - 1) >> (31 - __clz(c.page)); }

// A slot's length, kept within what its row can hold.
GDNX_DEV int64_t length_of(const gdnx_cache& c, int row) {
  const int64_t n = c.lengths[row], most = c.width * c.page;
  return n < 0 ? 0 : (n > most ? most : n);
}

size_t seen_bytes(const gdnx_cache& c) { return (size_t)((c.slots + 31) / 32) * 4; }

gdnx_status launched(cudaError_t e) { return e == cudaSuccess ? GDNX_OK : GDNX_ELAUNCH; }

int elem(int dtype) { return dtype == GDNX_F32 ? 4 : 2; }

}  // namespace
}  // namespace gdnx
