// Tiles of the CUDA-core attention kernels: 32 rows of a block's own, 64 of what streams past, 128 threads.  A thread
// holds a 4 x 4 piece of the products and a 4 x DP/16 piece of the accumulators, a warp eight rows.
#pragma once

#include <type_traits>

#include "attn_tc.cuh"

namespace gdnx {
namespace {  // one copy for each kernel file

using namespace attn;

constexpr int BR = 32;        // rows of a block's own tiles
constexpr int BT = 64;        // rows of the tiles that stream past
constexpr int NT = 128;       // threads
constexpr int LDP = BT + 4;   // row stride of the weight tile (16-byte rows, conflict-free)

template <typename T>
GDNX_DEV float to_f32(T x);
template <>
GDNX_DEV float to_f32<float>(float x) { return x; }
template <>
GDNX_DEV float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
GDNX_DEV float to_f32<__half>(__half x) { return __half2float(x); }

// This thread's asynchronous copies have landed (a barrier makes them everyone's).
GDNX_DEV void wait_tiles() {
  asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
}

// The groups of 16 of a streamed tile's rows that a warp's own eight rows meet: first, first + n - 1.
struct Groups {
  int first, n;
  GDNX_DEV Groups(int lo, int hi) {  // rows lo..hi of the tile, any integers
    lo = max(lo, 0);
    hi = min(hi, BT - 1);
    first = lo / 16;
    n = lo > hi ? 0 : hi / 16 - first + 1;
  }
};
// Keys of the tile at j0 that the queries at positions p..p+7 see.
GDNX_DEV Groups keys_seen(int p, int j0, int len, int window, int sinks) {
  const int last = min(p + 7, len - 1) - j0, lo = p - window + 1 - j0;
  if (p >= len) return Groups(1, 0);
  if (sinks <= j0) return Groups(lo, last);
  return Groups(0, lo <= BT - 1 ? last : min(last, sinks - 1 - j0));
}
// f(std::integral_constant<int, n>) for n in 1..4: code for that many groups.
template <typename F>
GDNX_DEV void for_groups(int n, F f) {
  switch (n) {
    case 1: f(std::integral_constant<int, 1>()); break;
    case 2: f(std::integral_constant<int, 2>()); break;
    case 3: f(std::integral_constant<int, 3>()); break;
    case 4: f(std::integral_constant<int, 4>()); break;
  }
}

// s[a][c] = sum_{d < D} A[a][d] B[16c][d]  (D a multiple of 8), two d to an instruction
template <int DP, int NC>
GDNX_DEV void dot_tile(float (&s)[4][4], const float* A, const float* B, int D) {
  float2 t[4][NC];
#pragma unroll
  for (int a = 0; a < 4; ++a)
#pragma unroll
    for (int c = 0; c < NC; ++c) t[a][c] = make_float2(0.f, 0.f);
#pragma unroll 4
  for (int d = 0; d < D; d += 4) {
    float4 x[4], y[NC];
#pragma unroll
    for (int a = 0; a < 4; ++a) x[a] = *reinterpret_cast<const float4*>(A + a * (DP + 4) + d);
#pragma unroll
    for (int c = 0; c < NC; ++c) y[c] = *reinterpret_cast<const float4*>(B + 16 * c * (DP + 4) + d);
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        t[a][c] = fma2(make_float2(x[a].x, x[a].y), make_float2(y[c].x, y[c].y), t[a][c]);
        t[a][c] = fma2(make_float2(x[a].z, x[a].w), make_float2(y[c].z, y[c].w), t[a][c]);
      }
  }
#pragma unroll
  for (int a = 0; a < 4; ++a)
#pragma unroll
    for (int c = 0; c < NC; ++c) s[a][c] = t[a][c].x + t[a][c].y;
}

// A thread holds DP/16 columns of a row: four of each 64 (from 64 g + tx*4), then two of the last 32.
// o[a][columns] += sum_j W[a][j] X[j][columns] over the groups' j
template <int DP>
GDNX_DEV void acc_tile(float2 (&o)[4][DP / 32], const float* W, const float* X, int tx, const Groups& gr) {
#pragma unroll 2
  for (int j = 16 * gr.first; j < 16 * (gr.first + gr.n); j += 4) {
    float4 w[4];
#pragma unroll
    for (int a = 0; a < 4; ++a) w[a] = *reinterpret_cast<const float4*>(W + a * LDP + j);
#pragma unroll
    for (int jj = 0; jj < 4; ++jj) {
      const float* row = X + (j + jj) * (DP + 4);
#pragma unroll
      for (int g = 0; g < DP / 64; ++g) {
        const float4 x = *reinterpret_cast<const float4*>(row + g * 64 + tx * 4);
#pragma unroll
        for (int a = 0; a < 4; ++a) {
          const float p = jj == 0 ? w[a].x : jj == 1 ? w[a].y : jj == 2 ? w[a].z : w[a].w;
          o[a][g * 2] = fma2(make_float2(p, p), make_float2(x.x, x.y), o[a][g * 2]);
          o[a][g * 2 + 1] = fma2(make_float2(p, p), make_float2(x.z, x.w), o[a][g * 2 + 1]);
        }
      }
      if (DP % 64) {
        const float2 x = *reinterpret_cast<const float2*>(row + DP / 64 * 64 + tx * 2);
#pragma unroll
        for (int a = 0; a < 4; ++a) {
          const float p = jj == 0 ? w[a].x : jj == 1 ? w[a].y : jj == 2 ? w[a].z : w[a].w;
          o[a][DP / 32 - 1] = fma2(make_float2(p, p), x, o[a][DP / 32 - 1]);
        }
      }
    }
  }
}
template <int N>
GDNX_DEV void clear(float2 (&o)[4][N]) {
#pragma unroll
  for (int a = 0; a < 4; ++a)
#pragma unroll
    for (int d = 0; d < N; ++d) o[a][d] = make_float2(0.f, 0.f);
}
// f(first column, its values' pairs, how many columns) for each piece of a thread's columns.
template <int DP, typename F>
GDNX_DEV void for_pieces(const float2 (&o)[DP / 32], int tx, F f) {
#pragma unroll
  for (int g = 0; g < DP / 64; ++g) f(g * 64 + tx * 4, &o[g * 2], std::integral_constant<int, 4>());
  if constexpr (DP % 64) f(DP / 64 * 64 + tx * 2, &o[DP / 32 - 1], std::integral_constant<int, 2>());
}
// N values of a row, scaled.
template <int N>
GDNX_DEV void store_piece(void* dst, int dtype, int64_t at, const float2* o, float scale) {
  float* p = static_cast<float*>(dst) + at;
  if (dtype == GDNX_F32 && reinterpret_cast<uintptr_t>(p) % (4 * N) == 0) {
    if constexpr (N == 4) *reinterpret_cast<float4*>(p) = make_float4(o[0].x * scale, o[0].y * scale, o[1].x * scale, o[1].y * scale);
    else *reinterpret_cast<float2*>(p) = make_float2(o[0].x * scale, o[0].y * scale);
    return;
  }
#pragma unroll
  for (int e = 0; e < N; ++e) st_from_f32(dst, dtype, at + e, (e % 2 ? o[e / 2].y : o[e / 2].x) * scale);
}

GDNX_DEV float half_warp_max(float x) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}
GDNX_DEV float half_warp_sum(float x) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

}  // namespace
}  // namespace gdnx
