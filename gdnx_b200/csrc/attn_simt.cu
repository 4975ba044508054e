// Windowed attention on the CUDA cores: any of the three types, any strides.  All
// arithmetic is fp32, so this is the path of 32-bit inputs, and of 16-bit inputs that TMA
// cannot address.
//
// Forward, one block of 64 queries of one head, key tiles of 64 in sequence:
//   s = scale log2(e) q.k;  m' = max(m, max_j s);  p = 2^(s - m');
//   l = l 2^(m - m') + sum_j p;  o = o 2^(m - m') + p V;   y = o / l.
// Backward, with P recomputed from lse (P = exp(scale q.k - lse)) and
// delta_i = sum_d dy_id y_id (which is sum_j P_ij dP_ij):
//   dP = dy V^T;  dS = P (dP - delta);  dV = P^T dy;  dQ = scale dS K;  dK = scale dS^T Q.
// dQ has a block for each 64 queries, dK and dV one for each 64 keys, which takes the query
// heads of its key head and the query tiles in order: no atomics, sums in a fixed order.
//
// A thread holds a 4 x 4 piece of the 64 x 64 score tile and a 4 x D/16 piece of the
// accumulators.  Padding rows are loaded as zeros, so NaN in them meets no sum.
#include "attn_common.cuh"
#include "kernels.h"

namespace gdnx {
namespace {

using namespace attn;

constexpr int BT = 64;        // rows of every tile
constexpr int NT = 256;       // threads
constexpr int LDP = BT + 4;   // row stride of the weight tile (16-byte rows, conflict-free)

// Blocks run over heads, then batch rows, then tiles: those of one tile, which cost alike, side
// by side, and the tiles with most work first (the last queries; the first keys).
struct Block {
  int64_t b, h;
  int tile;
};
GDNX_DEV Block block_of(int64_t heads, int64_t B) {
  const int64_t n = blockIdx.x;
  return {n / heads % B, n % heads, (int)(n / (heads * B))};
}

template <typename T>
GDNX_DEV float to_f32(T x);
template <>
GDNX_DEV float to_f32<float>(float x) { return x; }
template <>
GDNX_DEV float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
GDNX_DEV float to_f32<__half>(__half x) { return __half2float(x); }

// Rows r0..r0+63 of head h (rows at or beyond `rows` as zeros) into dst [64][DP + 4].  Aligned
// 32-bit rows go by 16-byte asynchronous copies (landed after `wait_tiles`), others by value.
template <int DP, typename T>
GDNX_DEV void load_tile(float* dst, const gdnx_view& v, int64_t b, int64_t h, int r0, int rows, int D) {
  const T* base = reinterpret_cast<const T*>(v.ptr) + b * v.sb + h * v.sh;
  if (sizeof(T) == 4 && reinterpret_cast<uintptr_t>(base) % 16 == 0 && v.st % 4 == 0) {
#pragma unroll
    for (int k = 0; k < BT * DP / 4 / NT; ++k) {
      const int i = k * NT + threadIdx.x, r = i / (DP / 4), d = i % (DP / 4) * 4;
      const bool on = r0 + r < rows && d < D;
      const T* src = on ? base + (int64_t)(r0 + r) * v.st + d : base;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                       static_cast<uint32_t>(__cvta_generic_to_shared(dst + r * (DP + 4) + d))),
                   "l"(src), "r"(on ? 16 : 0)
                   : "memory");
    }
    return;
  }
#pragma unroll 8
  for (int i = threadIdx.x; i < BT * DP; i += NT) {
    const int r = i / DP, d = i % DP;
    float x = 0.f;
    if (r0 + r < rows && d < D) x = to_f32(base[(int64_t)(r0 + r) * v.st + d]);
    dst[r * (DP + 4) + d] = x;
  }
}
// This thread's asynchronous copies have landed (a barrier makes them everyone's).
GDNX_DEV void wait_tiles() {
  asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
}

// s[a][c] = sum_{d < D} A[ty*4+a][d] B[tx+16c][d]  (D a multiple of 8)
template <int DP>
GDNX_DEV void dot_tile(float (&s)[4][4], const float* A, const float* B, int ty, int tx, int D) {
#pragma unroll
  for (int a = 0; a < 4; ++a)
#pragma unroll
    for (int c = 0; c < 4; ++c) s[a][c] = 0.f;
#pragma unroll 4
  for (int d = 0; d < D; d += 4) {
    float4 x[4], y[4];
#pragma unroll
    for (int a = 0; a < 4; ++a) x[a] = *reinterpret_cast<const float4*>(A + (ty * 4 + a) * (DP + 4) + d);
#pragma unroll
    for (int c = 0; c < 4; ++c) y[c] = *reinterpret_cast<const float4*>(B + (tx + 16 * c) * (DP + 4) + d);
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        s[a][c] = fmaf(x[a].x, y[c].x, s[a][c]);
        s[a][c] = fmaf(x[a].y, y[c].y, s[a][c]);
        s[a][c] = fmaf(x[a].z, y[c].z, s[a][c]);
        s[a][c] = fmaf(x[a].w, y[c].w, s[a][c]);
      }
  }
}

// o[a][64 g + tx*4 ..] += sum_j W[ty*4+a][j] X[j][64 g + tx*4 ..]
template <int DP>
GDNX_DEV void acc_tile(float (&o)[4][DP / 16], const float* W, const float* X, int ty, int tx) {
#pragma unroll 2
  for (int j = 0; j < BT; j += 4) {
    float4 w[4];
#pragma unroll
    for (int a = 0; a < 4; ++a) w[a] = *reinterpret_cast<const float4*>(W + (ty * 4 + a) * LDP + j);
#pragma unroll
    for (int jj = 0; jj < 4; ++jj) {
#pragma unroll
      for (int g = 0; g < DP / 64; ++g) {
        const float4 x = *reinterpret_cast<const float4*>(X + (j + jj) * (DP + 4) + g * 64 + tx * 4);
#pragma unroll
        for (int a = 0; a < 4; ++a) {
          const float p = jj == 0 ? w[a].x : jj == 1 ? w[a].y : jj == 2 ? w[a].z : w[a].w;
          o[a][g * 4 + 0] = fmaf(p, x.x, o[a][g * 4 + 0]);
          o[a][g * 4 + 1] = fmaf(p, x.y, o[a][g * 4 + 1]);
          o[a][g * 4 + 2] = fmaf(p, x.z, o[a][g * 4 + 2]);
          o[a][g * 4 + 3] = fmaf(p, x.w, o[a][g * 4 + 3]);
        }
      }
    }
  }
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

// x in a 16-bit type and back.
GDNX_DEV float rounded(float x, int dtype) {
  return dtype == GDNX_BF16 ? __bfloat162float(__float2bfloat16_rn(x)) : __half2float(__float2half_rn(x));
}

template <int DP, typename T>
__global__ void __launch_bounds__(NT) attn_fwd_simt_kernel(const gdnx_attn_args a) {
  extern __shared__ float sm[];
  float* Q = sm;
  float* KV = Q + BT * (DP + 4);
  float* W = KV + BT * (DP + 4);
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const Block blk = block_of(a.H, a.B);
  const int i0 = ((int)((a.Tq + BT - 1) / BT) - 1 - blk.tile) * BT, D = (int)a.D;
  const int64_t h = blk.h, b = blk.b, hk = h / (a.H / a.Hk);
  const int off = (int)(a.Tk - a.Tq), len = seq_len(a, b);
  const int window = (int)a.window, sinks = (int)a.sinks;
  const float c2 = a.scale * kLog2e;
  const KeyTiles kt(i0 + off, min(i0 + BT, (int)a.Tq) - 1 + off, len, window, sinks, BT);
  load_tile<DP, T>(Q, a.q, b, h, i0, min((int)a.Tq, len - off), D);
  float o[4][DP / 16], m[4], l[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) o[r][d] = 0.f;
  }
  for (int t = 0; t < kt.count; ++t) {
    const int j0 = kt.tile(t) * BT;
    __syncthreads();
    load_tile<DP, T>(KV, a.k, b, hk, j0, len, D);
    wait_tiles();
    __syncthreads();
    float s[4][4];
    dot_tile<DP>(s, Q, KV, ty, tx, D);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int p = i0 + ty * 4 + r + off;
      float mx = m[r];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        s[r][c] = sees(p, j0 + tx + 16 * c, len, window, sinks) ? s[r][c] * c2 : -INFINITY;
        mx = fmaxf(mx, s[r][c]);
      }
      mx = half_warp_max(mx);
      const float base = mx == -INFINITY ? 0.f : mx;
      const float corr = exp2f(m[r] - base);
      float sum = 0.f;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        s[r][c] = exp2f(s[r][c] - base);
        sum += s[r][c];
        W[(ty * 4 + r) * LDP + tx + 16 * c] = s[r][c];
      }
      l[r] = l[r] * corr + half_warp_sum(sum);
      m[r] = mx;
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) o[r][d] *= corr;
    }
    __syncthreads();
    load_tile<DP, T>(KV, a.v, b, hk, j0, len, D);
    wait_tiles();
    __syncthreads();
    acc_tile<DP>(o, W, KV, ty, tx);
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int i = i0 + ty * 4 + r;
    if (i >= a.Tq) continue;
    const float inv = l[r] > 0.f ? 1.f / l[r] : 0.f;
    const int64_t row = b * a.y_sb + (int64_t)i * a.y_st + h * a.y_sh;
#pragma unroll
    for (int g = 0; g < DP / 64; ++g)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = g * 64 + tx * 4 + e;
        if (d >= D) continue;
        const float y = o[r][g * 4 + e] * inv;
        st_from_f32(a.y, a.y_dtype, row + d, y);
        if (a.y_rest) st_from_f32(a.y_rest, a.y_dtype, ((b * a.Tq + i) * a.H + h) * D + d, y - rounded(y, a.y_dtype));
      }
    if (a.lse && tx == 0)
      a.lse[(b * a.H + h) * a.Tq + i] = l[r] > 0.f ? (m[r] + log2f(l[r])) * kLn2 : -INFINITY;
  }
}

// delta[b,h,i] = sum_d dy y: one warp for each row; 0 for padding rows.
__global__ void __launch_bounds__(256) attn_delta_kernel(const gdnx_attn_bwd_args g, float* delta) {
  const gdnx_attn_args& a = g.fwd;
  const int64_t n = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  if (n >= a.B * a.Tq * a.H) return;
  const int64_t h = n % a.H, i = n / a.H % a.Tq, b = n / (a.H * a.Tq);
  const int lane = threadIdx.x % 32;
  float s = 0.f;
  if (i + a.Tk - a.Tq < seq_len(a, b)) {
    const int64_t ry = b * a.y_sb + i * a.y_st + h * a.y_sh, rd = b * g.dy.sb + i * g.dy.st + h * g.dy.sh;
    for (int d = lane; d < a.D; d += 32) {
      float y = ld_as_f32(a.y, a.y_dtype, ry + d);
      if (a.y_rest) y += ld_as_f32(a.y_rest, a.y_dtype, ((b * a.Tq + i) * a.H + h) * a.D + d);
      s = fmaf(y, ld_as_f32(g.dy.ptr, g.dy.dtype, rd + d), s);
    }
    s = warp_sum(s);
  }
  if (lane == 0) delta[(b * a.H + h) * a.Tq + i] = s;
}

// P and dS of one tile from the raw dots: p = exp(scale q.k - lse), ds = p (dp - delta).
GDNX_DEV float weight(float s, float c2, float lse2) { return exp2f(s * c2 - lse2); }

template <int DP, typename T>
__global__ void __launch_bounds__(NT) attn_dq_simt_kernel(const gdnx_attn_bwd_args g, const float* delta) {
  extern __shared__ float sm[];
  const gdnx_attn_args& a = g.fwd;
  float* Q = sm;
  float* Y = Q + BT * (DP + 4);
  float* KV = Y + BT * (DP + 4);
  float* W = KV + BT * (DP + 4);
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const Block blk = block_of(a.H, a.B);
  const int i0 = ((int)((a.Tq + BT - 1) / BT) - 1 - blk.tile) * BT, D = (int)a.D;
  const int64_t h = blk.h, b = blk.b, hk = h / (a.H / a.Hk);
  const int off = (int)(a.Tk - a.Tq), len = seq_len(a, b);
  const int window = (int)a.window, sinks = (int)a.sinks;
  const float c2 = a.scale * kLog2e;
  const KeyTiles kt(i0 + off, min(i0 + BT, (int)a.Tq) - 1 + off, len, window, sinks, BT);
  const int rows = min((int)a.Tq, len - off);
  load_tile<DP, T>(Q, a.q, b, h, i0, rows, D);
  load_tile<DP, T>(Y, g.dy, b, h, i0, rows, D);
  float o[4][DP / 16], lse2[4], dl[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int i = i0 + ty * 4 + r;
    lse2[r] = i < rows ? a.lse[(b * a.H + h) * a.Tq + i] * kLog2e : 0.f;
    dl[r] = i < rows ? delta[(b * a.H + h) * a.Tq + i] : 0.f;
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) o[r][d] = 0.f;
  }
  for (int t = 0; t < kt.count; ++t) {
    const int j0 = kt.tile(t) * BT;
    float dp[4][4], s[4][4];
    __syncthreads();
    load_tile<DP, T>(KV, a.v, b, hk, j0, len, D);
    wait_tiles();
    __syncthreads();
    dot_tile<DP>(dp, Y, KV, ty, tx, D);
    __syncthreads();
    load_tile<DP, T>(KV, a.k, b, hk, j0, len, D);
    wait_tiles();
    __syncthreads();
    dot_tile<DP>(s, Q, KV, ty, tx, D);
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int p = i0 + ty * 4 + r + off;
        const bool on = sees(p, j0 + tx + 16 * c, len, window, sinks) && !sees_one(p, window, sinks);
        W[(ty * 4 + r) * LDP + tx + 16 * c] = on ? weight(s[r][c], c2, lse2[r]) * (dp[r][c] - dl[r]) : 0.f;
      }
    __syncthreads();
    acc_tile<DP>(o, W, KV, ty, tx);
  }
  T* dq = reinterpret_cast<T*>(g.dq);
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int i = i0 + ty * 4 + r;
    if (i >= a.Tq) continue;
#pragma unroll
    for (int gg = 0; gg < DP / 64; ++gg)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = gg * 64 + tx * 4 + e;
        if (d < D) st_from_f32(dq, a.q.dtype, ((b * a.Tq + i) * a.H + h) * D + d, o[r][gg * 4 + e] * a.scale);
      }
  }
}

template <int DP, typename T>
__global__ void __launch_bounds__(NT) attn_dkv_simt_kernel(const gdnx_attn_bwd_args g, const float* delta) {
  extern __shared__ float sm[];
  const gdnx_attn_args& a = g.fwd;
  float* K = sm;
  float* V = K + BT * (DP + 4);
  float* Q = V + BT * (DP + 4);
  float* Y = Q + BT * (DP + 4);
  float* W = Y + BT * (DP + 4);  // P^T, then dS^T: [key][query]
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const Block blk = block_of(a.Hk, a.B);
  const int j0 = blk.tile * BT, D = (int)a.D;
  const int64_t hk = blk.h, b = blk.b, G = a.H / a.Hk;
  const int off = (int)(a.Tk - a.Tq), len = seq_len(a, b);
  const int window = (int)a.window, sinks = (int)a.sinks;
  const float c2 = a.scale * kLog2e;
  const int rows = min((int)a.Tq, len - off);  // queries that are not padding
  load_tile<DP, T>(K, a.k, b, hk, j0, len, D);
  load_tile<DP, T>(V, a.v, b, hk, j0, len, D);
  float dk[4][DP / 16], dv[4][DP / 16];
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) dk[r][d] = dv[r][d] = 0.f;
  // queries from position j0 on; past the window only where the tile holds sinks
  int lo = max(j0 - off, 0), hi = rows;
  if (j0 >= sinks) hi = (int)min((int64_t)rows, (int64_t)j0 + BT - 1 + window - off);
  if (j0 >= len) hi = 0;
  for (int64_t h = hk * G; h < (hk + 1) * G; ++h) {
    for (int i0 = lo / BT * BT; i0 < hi; i0 += BT) {
      __syncthreads();
      load_tile<DP, T>(Q, a.q, b, h, i0, rows, D);
      load_tile<DP, T>(Y, g.dy, b, h, i0, rows, D);
      wait_tiles();
      __syncthreads();
      float s[4][4], dp[4][4];  // [query ty*4+r][key tx+16c]
      dot_tile<DP>(s, Q, K, ty, tx, D);
      dot_tile<DP>(dp, Y, V, ty, tx, D);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = i0 + ty * 4 + r;
        const float lse2 = i < rows ? a.lse[(b * a.H + h) * a.Tq + i] * kLog2e : 0.f;
        const float dl = i < rows ? delta[(b * a.H + h) * a.Tq + i] : 0.f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float p = sees(i + off, j0 + tx + 16 * c, len, window, sinks) ? weight(s[r][c], c2, lse2) : 0.f;
          W[(tx + 16 * c) * LDP + ty * 4 + r] = p;
          s[r][c] = sees_one(i + off, window, sinks) ? 0.f : p * (dp[r][c] - dl);
        }
      }
      __syncthreads();
      acc_tile<DP>(dv, W, Y, ty, tx);
      __syncthreads();
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < 4; ++c) W[(tx + 16 * c) * LDP + ty * 4 + r] = s[r][c];
      __syncthreads();
      acc_tile<DP>(dk, W, Q, ty, tx);
    }
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int j = j0 + ty * 4 + r;
    if (j >= a.Tk) continue;
#pragma unroll
    for (int gg = 0; gg < DP / 64; ++gg)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = gg * 64 + tx * 4 + e;
        const int64_t at = ((b * a.Tk + j) * a.Hk + hk) * D + d;
        if (d < D) {
          st_from_f32(g.dk, a.k.dtype, at, dk[r][gg * 4 + e] * a.scale);
          st_from_f32(g.dv, a.k.dtype, at, dv[r][gg * 4 + e]);
        }
      }
  }
}

constexpr size_t smem_of(int dp, int tiles) { return ((size_t)tiles * BT * (dp + 4) + BT * LDP) * sizeof(float); }

dim3 blocks(int64_t T, int64_t heads, int64_t B) { return dim3((unsigned)((T + BT - 1) / BT * heads * B)); }

template <typename F>
gdnx_status run(F kernel, dim3 grid, size_t smem, cudaStream_t st, void** args) {
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess ||
      cudaLaunchKernel(reinterpret_cast<const void*>(kernel), grid, dim3(NT), args, smem, st) != cudaSuccess) {
    cudaGetLastError();
    return GDNX_ELAUNCH;
  }
  return GDNX_OK;
}

template <int DP, typename T>
gdnx_status fwd(const gdnx_attn_args& a, cudaStream_t st) {
  gdnx_attn_args arg = a;
  void* p[] = {&arg};
  return run(attn_fwd_simt_kernel<DP, T>, blocks(a.Tq, a.H, a.B),
             smem_of(DP, 2), st, p);
}

template <int DP, typename T>
gdnx_status bwd(const gdnx_attn_bwd_args& g, float* delta, cudaStream_t st) {
  gdnx_attn_bwd_args arg = g;
  void* p[] = {&arg, &delta};
  const gdnx_attn_args& a = g.fwd;
  gdnx_status s = run(attn_dq_simt_kernel<DP, T>,
                      blocks(a.Tq, a.H, a.B), smem_of(DP, 3), st, p);
  if (s != GDNX_OK) return s;
  return run(attn_dkv_simt_kernel<DP, T>, blocks(a.Tk, a.Hk, a.B),
             smem_of(DP, 4), st, p);
}

}  // namespace

gdnx_status launch_attn_fwd_simt(const gdnx_attn_args& a, cudaStream_t st) {
  const bool wide = a.D > 64;
  switch (a.q.dtype) {
    case GDNX_BF16: return wide ? fwd<128, __nv_bfloat16>(a, st) : fwd<64, __nv_bfloat16>(a, st);
    case GDNX_F16: return wide ? fwd<128, __half>(a, st) : fwd<64, __half>(a, st);
    default: return wide ? fwd<128, float>(a, st) : fwd<64, float>(a, st);
  }
}

gdnx_status launch_attn_delta(const gdnx_attn_bwd_args& g, float* delta, cudaStream_t st) {
  const int64_t rows = g.fwd.B * g.fwd.Tq * g.fwd.H;
  attn_delta_kernel<<<(unsigned)((rows + 7) / 8), 256, 0, st>>>(g, delta);
  return cudaGetLastError() == cudaSuccess ? GDNX_OK : GDNX_ELAUNCH;
}

gdnx_status launch_attn_bwd_simt(const gdnx_attn_bwd_args& g, float* delta, cudaStream_t st) {
  const bool wide = g.fwd.D > 64;
  switch (g.fwd.q.dtype) {
    case GDNX_BF16: return wide ? bwd<128, __nv_bfloat16>(g, delta, st) : bwd<64, __nv_bfloat16>(g, delta, st);
    case GDNX_F16: return wide ? bwd<128, __half>(g, delta, st) : bwd<64, __half>(g, delta, st);
    default: return wide ? bwd<128, float>(g, delta, st) : bwd<64, float>(g, delta, st);
  }
}

}  // namespace gdnx
