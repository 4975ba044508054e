// Windowed attention on the CUDA cores: any of the three types, any strides.  All
// arithmetic is fp32, so this is the path of 32-bit inputs, and of 16-bit inputs that TMA
// cannot address.
//
// Forward, one block of 32 queries of one head, key tiles of 64 in sequence:
//   s = scale log2(e) q.k;  m' = max(m, max_j s);  p = 2^(s - m');
//   l = l 2^(m - m') + sum_j p;  o = o 2^(m - m') + p V;   y = o / l.
// Backward, with P recomputed from lse (P = exp(scale q.k - lse)) and
// delta_i = sum_d dy_id y_id (which is sum_j P_ij dP_ij):
//   dP = dy V^T;  dS = P (dP - delta);  dV = P^T dy;  dQ = scale dS K;  dK = scale dS^T Q.
// dQ has a block for each 32 queries, dK and dV one for each 32 keys, which takes the query
// heads of its key head and the query tiles in order: no atomics, sums in a fixed order.
//
// A block's own tile has 32 rows, the tiles that stream past it 64.  A thread holds a 4 x 4 piece of
// the scores and a 4 x D/16 piece of the accumulators, a warp eight rows: so a warp's weights are its
// own (no barrier between the two products), and it leaves out the groups of 16 columns that none of
// its rows sees, which at the ends of the window and in the sinks' tile are most.  Several blocks of an
// SM cover each other's loads.  Products go two d to an instruction.  Padding rows are loaded as zeros,
// so NaN in them meets no sum.
//
// Measured, fp32: 3 x 1031 tokens, 8 heads over 2 of 96, window 300: 68 us; 2 x 512 tokens, 16 heads of
// 128, window 128, forward and gradients: 205 us (tiles of 64 x 64 that masked in registers only: 111 and
// 361 us).  Shared-memory reads bound it: 8 of 16 bytes feed 64 multiply-adds a thread.
#include "attn_simt.cuh"
#include "kernels.h"
#include "launch.cuh"

namespace gdnx {
namespace {

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

// Rows r0..r0+R-1 of head h (rows at or beyond `rows` as zeros) into dst [R][DP + 4].  Aligned
// 32-bit rows go by 16-byte asynchronous copies (landed after `wait_tiles`), others by value.
template <int R, int DP, typename T>
GDNX_DEV void load_tile(float* dst, const gdnx_view& v, int64_t b, int64_t h, int r0, int rows, int D) {
  const T* base = reinterpret_cast<const T*>(v.ptr) + b * v.sb + h * v.sh;
  if (sizeof(T) == 4 && reinterpret_cast<uintptr_t>(base) % 16 == 0 && v.st % 4 == 0) {
#pragma unroll
    for (int k = 0; k < R * DP / 4 / NT; ++k) {
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
  for (int i = threadIdx.x; i < R * DP; i += NT) {
    const int r = i / DP, d = i % DP;
    float x = 0.f;
    if (r0 + r < rows && d < D) x = to_f32(base[(int64_t)(r0 + r) * v.st + d]);
    dst[r * (DP + 4) + d] = x;
  }
}
// Queries of the tile at position p0 that see the keys j..j+7.
GDNX_DEV Groups queries_seeing(int j, int p0, int len, int window, int sinks) {
  if (j >= len) return Groups(1, 0);
  const int last = j < sinks ? len - 1 : (int)min((int64_t)len - 1, (int64_t)j + 6 + window);
  return Groups(j - p0, last - p0);
}

// x in a 16-bit type and back.
GDNX_DEV float rounded(float x, int dtype) {
  return dtype == GDNX_BF16 ? __bfloat162float(__float2bfloat16_rn(x)) : __half2float(__float2half_rn(x));
}

// Bytes of `own` tiles of a block, `streamed` tiles, the weights and two statistics of a streamed tile's rows.
constexpr size_t smem_of(int dp, int own, int streamed) {
  return ((size_t)(own * BR + streamed * BT) * (dp + 4) + BR * LDP + 2 * BT) * sizeof(float);
}

template <int DP, typename T>
__global__ void __launch_bounds__(NT, 3) attn_fwd_simt_kernel(const gdnx_attn_args a) {
  extern __shared__ float sm[];
  float* Q = sm;
  float* KV = Q + BR * (DP + 4);
  float* W = KV + BT * (DP + 4);
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const Block blk = block_of(a.H, a.B);
  const int i0 = ((int)((a.Tq + BR - 1) / BR) - 1 - blk.tile) * BR, D = (int)a.D;
  const int64_t h = blk.h, b = blk.b, hk = h / (a.H / a.Hk);
  const int off = (int)(a.Tk - a.Tq), len = seq_len(a, b);
  const int window = (int)a.window, sinks = (int)a.sinks;
  const float c2 = a.scale * kLog2e;
  const KeyTiles kt(i0 + off, min(i0 + BR, (int)a.Tq) - 1 + off, len, window, sinks, BT);
  load_tile<BR, DP, T>(Q, a.q, b, h, i0, min((int)a.Tq, len - off), D);
  const int pw = i0 + off + ty / 2 * 8;  // the warp's first position
  const float* q = Q + ty * 4 * (DP + 4);
  float* w = W + ty * 4 * LDP;
  float2 o[4][DP / 32];
  float m[4], l[4];
  clear(o);
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
  }
  for (int t = 0; t < kt.count; ++t) {
    const int j0 = kt.tile(t) * BT;
    const Groups gr = keys_seen(pw, j0, len, window, sinks);
    __syncthreads();
    load_tile<BT, DP, T>(KV, a.k, b, hk, j0, len, D);
    wait_tiles();
    __syncthreads();
    for_groups(gr.n, [&](auto nc) {
      constexpr int NC = decltype(nc)::value;
      const int col = 16 * gr.first + tx;
      float s[4][4];
      dot_tile<DP, NC>(s, q, KV + col * (DP + 4), D);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int p = i0 + ty * 4 + r + off;
        float mx = m[r];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          s[r][c] = sees(p, j0 + col + 16 * c, len, window, sinks) ? s[r][c] * c2 : -INFINITY;
          mx = fmaxf(mx, s[r][c]);
        }
        mx = half_warp_max(mx);
        const float base = mx == -INFINITY ? 0.f : mx;
        const float corr = exp2f(m[r] - base);
        float sum = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          s[r][c] = exp2f(s[r][c] - base);
          sum += s[r][c];
          w[r * LDP + col + 16 * c] = s[r][c];
        }
        l[r] = l[r] * corr + half_warp_sum(sum);
        m[r] = mx;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) o[r][d] = mul2(o[r][d], make_float2(corr, corr));
      }
    });
    __syncthreads();
    load_tile<BT, DP, T>(KV, a.v, b, hk, j0, len, D);
    wait_tiles();
    __syncthreads();
    acc_tile<DP>(o, w, KV, tx, gr);
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int i = i0 + ty * 4 + r;
    if (i >= a.Tq) continue;
    // every row but padding sees itself: a sum that is not positive comes of scores that are not finite
    const float none = i + off < len ? NAN : 0.f;
    const float inv = l[r] > 0.f ? 1.f / l[r] : none;
    const int64_t row = b * a.y_sb + (int64_t)i * a.y_st + h * a.y_sh;
    for_pieces<DP>(o[r], tx, [&](int d, const float2* v, auto n) {
      if (d >= D) return;
      store_piece<decltype(n)::value>(a.y, a.y_dtype, row + d, v, inv);
      if (a.y_rest)
#pragma unroll
        for (int e = 0; e < decltype(n)::value; ++e) {
          const float y = (e % 2 ? v[e / 2].y : v[e / 2].x) * inv;
          st_from_f32(a.y_rest, a.y_dtype, ((b * a.Tq + i) * a.H + h) * D + d + e, y - rounded(y, a.y_dtype));
        }
    });
    if (a.lse && tx == 0)
      a.lse[(b * a.H + h) * a.Tq + i] = l[r] > 0.f ? (m[r] + log2f(l[r])) * kLn2 : none == 0.f ? -INFINITY : none;
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
    const float *y = static_cast<const float*>(a.y) + ry, *dy = static_cast<const float*>(g.dy.ptr) + rd;
    if (a.y_dtype == GDNX_F32 && g.dy.dtype == GDNX_F32 && !a.y_rest &&
        (reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(dy)) % 16 == 0) {
      if (4 * lane < a.D) {
        const float4 u = *reinterpret_cast<const float4*>(y + 4 * lane), v = *reinterpret_cast<const float4*>(dy + 4 * lane);
        s = fmaf(u.x, v.x, fmaf(u.y, v.y, fmaf(u.z, v.z, u.w * v.w)));
      }
    } else
#pragma unroll 4
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
__global__ void __launch_bounds__(NT, 2) attn_dq_simt_kernel(const gdnx_attn_bwd_args g, const float* delta) {
  extern __shared__ float sm[];
  const gdnx_attn_args& a = g.fwd;
  float* Q = sm;
  float* Y = Q + BR * (DP + 4);
  float* K = Y + BR * (DP + 4);
  float* V = K + BT * (DP + 4);
  float* W = V + BT * (DP + 4);
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const Block blk = block_of(a.H, a.B);
  const int i0 = ((int)((a.Tq + BR - 1) / BR) - 1 - blk.tile) * BR, D = (int)a.D;
  const int64_t h = blk.h, b = blk.b, hk = h / (a.H / a.Hk);
  const int off = (int)(a.Tk - a.Tq), len = seq_len(a, b);
  const int window = (int)a.window, sinks = (int)a.sinks;
  const float c2 = a.scale * kLog2e;
  const KeyTiles kt(i0 + off, min(i0 + BR, (int)a.Tq) - 1 + off, len, window, sinks, BT);
  const int rows = min((int)a.Tq, len - off);
  load_tile<BR, DP, T>(Q, a.q, b, h, i0, rows, D);
  load_tile<BR, DP, T>(Y, g.dy, b, h, i0, rows, D);
  const int pw = i0 + off + ty / 2 * 8;  // the warp's first position
  float* w = W + ty * 4 * LDP;
  float2 o[4][DP / 32];
  float lse2[4], dl[4];
  clear(o);
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int i = i0 + ty * 4 + r;
    lse2[r] = i < rows ? a.lse[(b * a.H + h) * a.Tq + i] * kLog2e : 0.f;
    dl[r] = i < rows ? __ldcg(delta + (b * a.H + h) * a.Tq + i) : 0.f;
  }
  for (int t = 0; t < kt.count; ++t) {
    const int j0 = kt.tile(t) * BT;
    const Groups gr = keys_seen(pw, j0, len, window, sinks);
    __syncthreads();
    load_tile<BT, DP, T>(K, a.k, b, hk, j0, len, D);
    load_tile<BT, DP, T>(V, a.v, b, hk, j0, len, D);
    wait_tiles();
    __syncthreads();
    for_groups(gr.n, [&](auto nc) {
      constexpr int NC = decltype(nc)::value;
      const int col = 16 * gr.first + tx;
      float dp[4][4], s[4][4];
      dot_tile<DP, NC>(s, Q + ty * 4 * (DP + 4), K + col * (DP + 4), D);
      dot_tile<DP, NC>(dp, Y + ty * 4 * (DP + 4), V + col * (DP + 4), D);
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const int p = i0 + ty * 4 + r + off;
          const bool on = sees(p, j0 + col + 16 * c, len, window, sinks) && !sees_one(p, window, sinks);
          w[r * LDP + col + 16 * c] = on ? weight(s[r][c], c2, lse2[r]) * (dp[r][c] - dl[r]) : 0.f;
        }
    });
    __syncwarp();  // a warp's weights are its own
    acc_tile<DP>(o, w, K, tx, gr);
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int i = i0 + ty * 4 + r;
    if (i >= a.Tq) continue;
    for_pieces<DP>(o[r], tx, [&](int d, const float2* v, auto n) {
      if (d < D) store_piece<decltype(n)::value>(g.dq, a.q.dtype, ((b * a.Tq + i) * a.H + h) * D + d, v, a.scale);
    });
  }
  wait_for_earlier();
}

template <int DP, typename T>
__global__ void __launch_bounds__(NT, 2) attn_dkv_simt_kernel(const gdnx_attn_bwd_args g, const float* delta) {
  dependents_may_start();
  extern __shared__ float sm[];
  const gdnx_attn_args& a = g.fwd;
  float* K = sm;
  float* V = K + BR * (DP + 4);
  float* Q = V + BR * (DP + 4);
  float* Y = Q + BT * (DP + 4);
  float* W = Y + BT * (DP + 4);  // P^T, then dS^T: [key][query]
  float* lse = W + BR * LDP;     // of the tile's queries, in the log2 domain
  float* dl = lse + BT;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const Block blk = block_of(a.Hk, a.B);
  const int j0 = blk.tile * BR, D = (int)a.D;
  const int64_t hk = blk.h, b = blk.b, G = a.H / a.Hk;
  const int off = (int)(a.Tk - a.Tq), len = seq_len(a, b);
  const int window = (int)a.window, sinks = (int)a.sinks;
  const float c2 = a.scale * kLog2e;
  const int rows = min((int)a.Tq, len - off);  // queries that are not padding
  load_tile<BR, DP, T>(K, a.k, b, hk, j0, len, D);
  load_tile<BR, DP, T>(V, a.v, b, hk, j0, len, D);
  const int jw = j0 + ty / 2 * 8;  // the warp's first key
  float* w = W + ty * 4 * LDP;
  float2 dk[4][DP / 32], dv[4][DP / 32];
  clear(dk);
  clear(dv);
  // queries from position j0 on; past the window only where the tile holds sinks
  int lo = max(j0 - off, 0), hi = rows;
  if (j0 >= sinks) hi = (int)min((int64_t)rows, (int64_t)j0 + BR - 1 + window - off);
  if (j0 >= len) hi = 0;
  for (int64_t h = hk * G; h < (hk + 1) * G; ++h) {
    for (int i0 = lo / BT * BT; i0 < hi; i0 += BT) {
      const Groups gr = queries_seeing(jw, i0 + off, len, window, sinks);
      __syncthreads();
      load_tile<BT, DP, T>(Q, a.q, b, h, i0, rows, D);
      load_tile<BT, DP, T>(Y, g.dy, b, h, i0, rows, D);
      if (threadIdx.x < BT) {
        const int i = i0 + (int)threadIdx.x;
        const int64_t at = (b * a.H + h) * a.Tq + i;
        lse[threadIdx.x] = i < rows ? a.lse[at] * kLog2e : 0.f;
        dl[threadIdx.x] = i < rows ? delta[at] : 0.f;
      }
      wait_tiles();
      __syncthreads();
      float ds[4][4];
      for_groups(gr.n, [&](auto nc) {
        constexpr int NC = decltype(nc)::value;
        const int col = 16 * gr.first + tx;
        float s[4][4];  // [key ty*4+r][query]
        dot_tile<DP, NC>(s, K + ty * 4 * (DP + 4), Q + col * (DP + 4), D);
        dot_tile<DP, NC>(ds, V + ty * 4 * (DP + 4), Y + col * (DP + 4), D);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const int p = i0 + off + col + 16 * c;
          const float lse2 = lse[col + 16 * c], d = dl[col + 16 * c];
          const bool one = sees_one(p, window, sinks);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float x = sees(p, j0 + ty * 4 + r, len, window, sinks) ? weight(s[r][c], c2, lse2) : 0.f;
            w[r * LDP + col + 16 * c] = x;
            ds[r][c] = one ? 0.f : x * (ds[r][c] - d);
          }
        }
      });
      __syncwarp();  // a warp's weights are its own
      acc_tile<DP>(dv, w, Y, tx, gr);
      __syncwarp();
      for_groups(gr.n, [&](auto nc) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int c = 0; c < decltype(nc)::value; ++c) w[r * LDP + 16 * (gr.first + c) + tx] = ds[r][c];
      });
      __syncwarp();
      acc_tile<DP>(dk, w, Q, tx, gr);
    }
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int j = j0 + ty * 4 + r;
    if (j >= a.Tk) continue;
    const int64_t at = ((b * a.Tk + j) * a.Hk + hk) * D;
    for_pieces<DP>(dk[r], tx, [&](int d, const float2* v, auto n) {
      if (d < D) store_piece<decltype(n)::value>(g.dk, a.k.dtype, at + d, v, a.scale);
    });
    for_pieces<DP>(dv[r], tx, [&](int d, const float2* v, auto n) {
      if (d < D) store_piece<decltype(n)::value>(g.dv, a.k.dtype, at + d, v, 1.f);
    });
  }
}

dim3 blocks(int64_t T, int64_t heads, int64_t B) { return dim3((unsigned)((T + BR - 1) / BR * heads * B)); }

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
             smem_of(DP, 1, 1), st, p);
}

template <int DP, typename T>
gdnx_status bwd(const gdnx_attn_bwd_args& g, float* delta, cudaStream_t st) {
  gdnx_attn_bwd_args arg = g;
  void* p[] = {&arg, &delta};
  const gdnx_attn_args& a = g.fwd;
  constexpr size_t smem = smem_of(DP, 2, 2);
  const gdnx_status s = run(attn_dkv_simt_kernel<DP, T>, blocks(a.Tk, a.Hk, a.B), smem, st, p);
  if (s != GDNX_OK) return s;
  if (cudaFuncSetAttribute(attn_dq_simt_kernel<DP, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess ||
      launch_early(attn_dq_simt_kernel<DP, T>, blocks(a.Tq, a.H, a.B), dim3(NT), smem, st, g, delta) != cudaSuccess) {
    cudaGetLastError();
    return GDNX_ELAUNCH;
  }
  return GDNX_OK;
}

template <typename T>
gdnx_status fwd_of(const gdnx_attn_args& a, cudaStream_t st) {
  return a.D > 96 ? fwd<128, T>(a, st) : a.D > 64 ? fwd<96, T>(a, st) : fwd<64, T>(a, st);
}
template <typename T>
gdnx_status bwd_of(const gdnx_attn_bwd_args& g, float* delta, cudaStream_t st) {
  const int64_t D = g.fwd.D;
  return D > 96 ? bwd<128, T>(g, delta, st) : D > 64 ? bwd<96, T>(g, delta, st) : bwd<64, T>(g, delta, st);
}

}  // namespace

gdnx_status launch_attn_fwd_simt(const gdnx_attn_args& a, cudaStream_t st) {
  switch (a.q.dtype) {
    case GDNX_BF16: return fwd_of<__nv_bfloat16>(a, st);
    case GDNX_F16: return fwd_of<__half>(a, st);
    default: return fwd_of<float>(a, st);
  }
}

gdnx_status launch_attn_delta(const gdnx_attn_bwd_args& g, float* delta, cudaStream_t st) {
  const int64_t rows = g.fwd.B * g.fwd.Tq * g.fwd.H;
  attn_delta_kernel<<<(unsigned)((rows + 7) / 8), 256, 0, st>>>(g, delta);
  return cudaGetLastError() == cudaSuccess ? GDNX_OK : GDNX_ELAUNCH;
}

gdnx_status launch_attn_bwd_simt(const gdnx_attn_bwd_args& g, float* delta, cudaStream_t st) {
  switch (g.fwd.q.dtype) {
    case GDNX_BF16: return bwd_of<__nv_bfloat16>(g, delta, st);
    case GDNX_F16: return bwd_of<__half>(g, delta, st);
    default: return bwd_of<float>(g, delta, st);
  }
}

}  // namespace gdnx
