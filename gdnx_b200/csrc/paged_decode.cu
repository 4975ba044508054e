// Attention of one new token per sequence over a paged key/value cache of 32-bit values, on
// the CUDA cores (all arithmetic fp32).
//
//   y = sum_j softmax_j(scale q.k_j) v_j   over the visible tokens j of the slot.
// The visible tokens are walked in tiles of 64 positions, split evenly over the CTAs of one
// (sequence, key head, group of query heads); each CTA leaves its running maximum, sum and
// unnormalised output, and a second kernel joins the parts in order:
//   m = max_s m_s;  y = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s.
// The bytes of K and V bound it.  A warp reads one token's row with D / 8 lanes, eight values
// a lane, and holds the G query heads of the key head in registers, so each byte of K and V
// is read once for up to GB = 4 heads.
#include "attn_common.cuh"
#include "kernels.h"

namespace gdnx {
namespace {

using namespace attn;

constexpr int TILE = 64;      // tokens of one step of a CTA
constexpr int NT = 128;
constexpr int WARPS = NT / 32;
constexpr int GB = 4;         // query heads of one CTA
constexpr int MAX_SPLITS = 128;

// Eight consecutive values.
GDNX_DEV void load8(float (&x)[8], const float* p) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
  x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}

struct Dec {
  gdnx_paged_decode_args a;
  int splits, groups;  // parts of a sequence; CTAs of GB query heads for one key head
  float* part;         // [B, H, splits, D] unnormalised outputs
  float* stat;         // [B, H, splits, 2] maximum (log2 domain) and sum
};

GDNX_DEV int dec_length(const Dec& P, int64_t b, int& row) {
  const gdnx_cache& c = P.a.cache;
  row = P.a.rows ? P.a.rows[b] : (int)b;
  if (row < 0 || row >= c.slots) return 0;
  const int64_t n = c.lengths[row], most = c.width * c.page;
  return (int)(n < 0 ? 0 : (n > most ? most : n));
}

template <int LPK>  // lanes per key: 8 (D <= 64) or 16 (D <= 128)
__global__ void __launch_bounds__(NT) paged_decode_kernel(const Dec P) {
  constexpr int KPW = 32 / LPK;              // tokens of one pass of a warp
  constexpr int PASSES = TILE / WARPS / KPW;  // passes of a warp over its part of a tile
  __shared__ float red_o[WARPS * KPW][GB][LPK * 8];
  __shared__ float red_m[WARPS * KPW][GB], red_l[WARPS * KPW][GB];
  const gdnx_paged_decode_args& a = P.a;
  const gdnx_cache& c = a.cache;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, sub = lane / LPK, dl = lane % LPK;
  const int split = blockIdx.x, D = (int)c.D, G = (int)(a.H / c.Hk);
  const int64_t b = blockIdx.z, hk = blockIdx.y / P.groups;
  const int g0 = (int)(blockIdx.y % P.groups) * GB, ng = min(GB, G - g0);
  int row;
  const int len = dec_length(P, b, row);
  const int window = (int)a.window, sinks = (int)a.sinks, page = c.page;
  const KeyTiles kt(len - 1, len - 1, len, window, sinks, TILE);
  const int per = (kt.count + P.splits - 1) / P.splits, t0 = split * per, t1 = min(kt.count, t0 + per);
  const bool mine = dl * 8 < D;  // lanes beyond a narrow head hold zeros
  const float c2 = a.scale * kLog2e;
  float q[GB][8], o[GB][8], m[GB], l[GB];
#pragma unroll
  for (int g = 0; g < GB; ++g) {
    m[g] = -INFINITY;
    l[g] = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      o[g][e] = 0.f;
      q[g][e] = (g < ng && mine)
                    ? ld_as_f32(a.q.ptr, a.q.dtype, b * a.q.sb + (hk * G + g0 + g) * a.q.sh + dl * 8 + e) * c2
                    : 0.f;
    }
  }
  const float* kv = static_cast<const float*>(c.kv);
  const int64_t side = c.pages * c.Hk * page * D;  // one layer's keys or values
  const float* kbase = kv + a.layer * 2 * side + hk * page * D + dl * 8;
  const int32_t* table = c.table + (int64_t)row * c.width;
  for (int t = t0; t < t1; ++t) {
    const int j0 = kt.tile(t) * TILE + warp * (TILE / WARPS) + sub;
    float s[PASSES][GB];
    int64_t at[PASSES];
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int j = j0 + i * KPW;
      at[i] = -1;
      if (j < len && (len - 1 - j < window || j < sinks)) {
        const int p = table[j / page];
        if (p >= 0 && p < c.pages) at[i] = ((int64_t)p * c.Hk * page + j % page) * D;
      }
    }
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      float x[8] = {};
      if (at[i] >= 0 && mine) load8(x, kbase + at[i]);
#pragma unroll
      for (int g = 0; g < GB; ++g) {
        float d = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) d = fmaf(q[g][e], x[e], d);
#pragma unroll
        for (int sh = LPK / 2; sh > 0; sh >>= 1) d += __shfl_xor_sync(0xffffffffu, d, sh);
        s[i][g] = at[i] >= 0 ? d : -INFINITY;
      }
    }
#pragma unroll
    for (int g = 0; g < GB; ++g) {
      float mx = m[g];
#pragma unroll
      for (int i = 0; i < PASSES; ++i) mx = fmaxf(mx, s[i][g]);
      const float base = mx == -INFINITY ? 0.f : mx, corr = exp2f(m[g] - base);
      m[g] = mx;
      l[g] *= corr;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[g][e] *= corr;
#pragma unroll
      for (int i = 0; i < PASSES; ++i) {
        s[i][g] = exp2f(s[i][g] - base);
        l[g] += s[i][g];
      }
    }
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      float x[8] = {};
      if (at[i] >= 0 && mine) load8(x, kbase + side + at[i]);
#pragma unroll
      for (int g = 0; g < GB; ++g)
#pragma unroll
        for (int e = 0; e < 8; ++e) o[g][e] = fmaf(s[i][g], x[e], o[g][e]);
    }
  }
  // join the CTA's WARPS * KPW partial results
  const int part = warp * KPW + sub;
#pragma unroll
  for (int g = 0; g < GB; ++g) {
#pragma unroll
    for (int e = 0; e < 8; ++e) red_o[part][g][dl * 8 + e] = o[g][e];
    if (dl == 0) {
      red_m[part][g] = m[g];
      red_l[part][g] = l[g];
    }
  }
  __syncthreads();
  for (int x = threadIdx.x; x < ng * D; x += NT) {
    const int g = x / D, d = x % D;
    float mx = -INFINITY, sum = 0.f, y = 0.f;
#pragma unroll
    for (int k = 0; k < WARPS * KPW; ++k) mx = fmaxf(mx, red_m[k][g]);
    const float base = mx == -INFINITY ? 0.f : mx;
#pragma unroll
    for (int k = 0; k < WARPS * KPW; ++k) {
      const float w = exp2f(red_m[k][g] - base);
      sum = fmaf(w, red_l[k][g], sum);
      y = fmaf(w, red_o[k][g][d], y);
    }
    const int64_t h = hk * G + g0 + g;
    if (P.splits == 1) {
      st_from_f32(a.y, a.y_dtype, b * a.y_sb + h * a.y_sh + d, sum > 0.f ? y / sum : 0.f);
    } else {
      const int64_t at = (b * a.H + h) * P.splits + split;
      P.part[at * D + d] = y;
      if (d == 0) {
        P.stat[2 * at] = mx;
        P.stat[2 * at + 1] = sum;
      }
    }
  }
}

// One CTA for each (sequence, query head).
__global__ void __launch_bounds__(128) paged_decode_join_kernel(const Dec P) {
  const gdnx_paged_decode_args& a = P.a;
  const int64_t h = blockIdx.x % a.H, b = blockIdx.x / a.H, at = (b * a.H + h) * P.splits;
  const int D = (int)a.cache.D;
  float mx = -INFINITY, sum = 0.f, y = 0.f;
  for (int s = 0; s < P.splits; ++s) mx = fmaxf(mx, P.stat[2 * (at + s)]);
  const float base = mx == -INFINITY ? 0.f : mx;
  const int d = threadIdx.x;
  for (int s = 0; s < P.splits; ++s) {
    const float w = exp2f(P.stat[2 * (at + s)] - base);
    sum = fmaf(w, P.stat[2 * (at + s) + 1], sum);
    if (d < D) y = fmaf(w, P.part[(at + s) * D + d], y);
  }
  if (d < D) st_from_f32(a.y, a.y_dtype, b * a.y_sb + h * a.y_sh + d, sum > 0.f ? y / sum : 0.f);
}

// Parts of a sequence: about four CTAs for each SM, and at least two tiles for each part.
int split_count(const gdnx_paged_decode_args& a, int groups) {
  const gdnx_cache& c = a.cache;
  int64_t most = c.width * c.page;
  if (a.max_len > 0 && a.max_len < most) most = a.max_len;
  int64_t tiles = (most + TILE - 1) / TILE;
  const int64_t seen = (a.window + TILE - 1) / TILE + 1 + (a.sinks + TILE - 1) / TILE;
  if (seen < tiles) tiles = seen;
  const int64_t ctas = a.B * c.Hk * groups;
  int64_t s = (148 * 4 + ctas - 1) / ctas;
  if (s > (tiles + 1) / 2) s = (tiles + 1) / 2;
  return (int)(s < 1 ? 1 : s > MAX_SPLITS ? MAX_SPLITS : s);
}

int group_count(const gdnx_paged_decode_args& a) { return (int)((a.H / a.cache.Hk + GB - 1) / GB); }

}  // namespace

size_t paged_decode_workspace_bytes(const gdnx_paged_decode_args& a) {
  const int s = split_count(a, group_count(a));
  return s == 1 ? 0 : (size_t)(a.B * a.H * s * (a.cache.D + 2)) * sizeof(float);
}

gdnx_status launch_paged_decode(const gdnx_paged_decode_args& a, cudaStream_t st) {
  Dec P;
  P.a = a;
  P.groups = group_count(a);
  P.splits = split_count(a, P.groups);
  P.part = static_cast<float*>(a.workspace);
  P.stat = P.part + a.B * a.H * P.splits * a.cache.D;
  const dim3 grid((unsigned)P.splits, (unsigned)(a.cache.Hk * P.groups), (unsigned)a.B);
  if (a.cache.D > 64) paged_decode_kernel<16><<<grid, NT, 0, st>>>(P);
  else paged_decode_kernel<8><<<grid, NT, 0, st>>>(P);
  if (cudaGetLastError() != cudaSuccess) return GDNX_ELAUNCH;
  if (P.splits > 1) {
    paged_decode_join_kernel<<<(unsigned)(a.B * a.H), 128, 0, st>>>(P);
    if (cudaGetLastError() != cudaSuccess) return GDNX_ELAUNCH;
  }
  return GDNX_OK;
}

}  // namespace gdnx
