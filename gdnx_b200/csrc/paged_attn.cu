// Attention of a chunk of new tokens over a paged cache of 32-bit values, on the CUDA cores
// (all arithmetic fp32).
//
// Blocks of 32 rows (tokens times the heads of a group, paged_attn.cuh) walk key tiles of 64 as windowed attention's
// forward does (attn_simt.cuh):  s = scale log2(e) q.k;  m' = max(m, max_j s);  p = 2^(s - m');
//   l = l 2^(m - m') + sum_j p;  o = o 2^(m - m') + p V;   y = o / l.
// A tile's tokens come from up to four pages by 16-byte asynchronous copies; what lies on no page, or behind the
// sequence's last token, is zero and not seen.  The next tile's keys come under the product with the values, its values
// under the product with its keys, its page ids under both (loads and products in turn: 106 us for the case below).
//
// Measured: three chunks of up to 301 tokens and two single ones at lengths up to 1031, 8 heads over 2 of 96, window 300,
// 3 sinks: 58 to 66 us (7 us of multiply-adds at the CUDA cores' rate, which shared-memory reads hold to a quarter; start,
// join and two or three tiles a CTA are the rest); 1000 tokens after 1000 without a window: 184 us.
#include "attn_simt.cuh"
#include "paged_attn.cuh"

namespace gdnx {
namespace {

struct Simt : Shape<BR, BT, false> {
  static constexpr int OVER = 4, SMALL = 12, LEAST = 4;
};
constexpr int GRANULES = BT / 16;  // of 16 tokens: the smallest page

// Tokens j0.. of keys or values (side) into dst [BT][DP + 4], as one group of asynchronous copies.  ids: page of each
// granule, -1 where there is none.
template <int DP>
GDNX_DEV void load_paged(float* dst, const gdnx_cache& c, int64_t layer, int side, int hk, const int* ids, int j0, int len) {
  const int D = (int)c.D, mask = c.page - 1, row = c.page * D;
  const float* base = static_cast<const float*>(c.kv) + ((layer * 2 + side) * c.pages * c.Hk + hk) * row;
#pragma unroll
  for (int k = 0; k < BT * DP / 4 / NT; ++k) {
    const int i = k * NT + threadIdx.x, r = i / (DP / 4), d = i % (DP / 4) * 4;
    const int id = ids[r / 16];
    const bool on = id >= 0 && j0 + r < len && d < D;
    const float* src = on ? base + (int64_t)id * c.Hk * row + ((j0 + r) & mask) * D + d : base;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                     static_cast<uint32_t>(__cvta_generic_to_shared(dst + r * (DP + 4) + d))),
                 "l"(src), "r"(on ? 16 : 0)
                 : "memory");
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
}
// This thread's groups but the newest have landed (a barrier makes them everyone's).
GDNX_DEV void wait_but_one() { asm volatile("cp.async.wait_group 1;" ::: "memory"); }

template <int DP>
__global__ void __launch_bounds__(NT, 3) paged_attn_simt_kernel(const ChunkParams P) {
  extern __shared__ float sm[];
  __shared__ Share share;
  __shared__ long long sums[NT / 32];
  __shared__ int ids[2][GRANULES];
  const gdnx_paged_attn_args& a = P.a;
  const gdnx_cache& c = a.cache;
  float* Q = sm;
  float* K = Q + BR * (DP + 4);
  float* V = K + BT * (DP + 4);
  float* W = V + BT * (DP + 4);
  dependents_may_start();
  wait_for_earlier();
  find_share<Simt, NT>(P, share, sums);
  if (threadIdx.x == 0 && P.cut) P.joint[blockIdx.x] = {0, 0, 0, 0, -1};
  write_padding(P, threadIdx.x, NT);
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16, D = (int)c.D;
  const int window = (int)a.window, sinks = (int)a.sinks;
  const float c2 = a.scale * kLog2e;
  const float* q = Q + ty * 4 * (DP + 4);
  float* w = W + ty * 4 * LDP;
  Walk<Simt> x(P, share);
  while (x.next()) {
    const int heads = x.heads(), h0 = x.head0(), len = x.s.len(), t0 = x.x.t0, hk = x.hk();
    const auto read_ids = [&](int k) {  // of tile k, by the first threads
      if (threadIdx.x < GRANULES && k < x.tb) {
        const int64_t page = (x.x.kt.tile(k) * BT + 16 * threadIdx.x) / c.page;
        const int id = page < c.width ? c.table[(int64_t)x.s.row * c.width + page] : -1;
        ids[k & 1][threadIdx.x] = id >= 0 && id < c.pages ? id : -1;
      }
    };
    __syncthreads();  // the unit before has read its tiles
    read_ids(x.ta);
    __syncthreads();
    load_paged<DP>(K, c, a.layer, 0, hk, ids[x.ta & 1], x.x.kt.tile(x.ta) * BT, len);
    load_paged<DP>(V, c, a.layer, 1, hk, ids[x.ta & 1], x.x.kt.tile(x.ta) * BT, len);
    for (int i = threadIdx.x; i < BR * DP; i += NT) {
      const int r = i / DP, d = i % DP, t = t0 + r / P.gs, g = r % P.gs;
      float v = 0.f;
      if (r / P.gs < P.tb && g < heads && t < x.s.count && d < D)
        v = static_cast<const float*>(a.q.ptr)[(int64_t)(x.s.start + t) * a.q.st + (int64_t)(h0 + g) * a.q.sh + d];
      Q[r * (DP + 4) + d] = v;
    }
    int p[4];  // positions of this thread's rows, -1: no query
    float m[4], l[4];
    bool any[4];
    float2 o[4][DP / 32];
    clear(o);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = ty * 4 + r, t = t0 + i / P.gs;
      p[r] = i / P.gs < P.tb && i % P.gs < heads && t < x.s.count ? x.s.first + t : -1;
      m[r] = -INFINITY;
      l[r] = 0.f;
      any[r] = false;
    }
    // positions of the warp's eight rows
    const int pw = x.s.first + t0 + ty / 2 * 8 / P.gs, pz = min(x.s.first + t0 + (ty / 2 * 8 + 7) / P.gs, len - 1);
    for (int k = x.ta; k < x.tb; ++k) {
      const int j0 = x.x.kt.tile(k) * BT;
      // columns that some of the warp's rows see
      const int lo = pw - window + 1 - j0;
      const Groups gr = pw >= len ? Groups(1, 0) : sinks <= j0 ? Groups(lo, pz - j0)
                                                               : Groups(0, lo <= BT - 1 ? pz - j0 : min(pz - j0, sinks - 1 - j0));
      const int* here = ids[k & 1];
      const int next0 = k + 1 < x.tb ? x.x.kt.tile(k + 1) * BT : 0;
      wait_but_one();
      __syncthreads();  // K (and, of the first tile, Q)
      read_ids(k + 1);
      for_groups(gr.n, [&](auto nc) {
        constexpr int NC = decltype(nc)::value;
        const int col = 16 * gr.first + tx;
        float s[4][4];
        dot_tile<DP, NC>(s, q, K + col * (DP + 4), D);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float mx = m[r];
#pragma unroll
          for (int e = 0; e < NC; ++e) {
            const bool on = sees(p[r], j0 + col + 16 * e, len, window, sinks) && here[gr.first + e] >= 0;
            any[r] |= on;
            s[r][e] = on ? s[r][e] * c2 : -INFINITY;
            mx = fmaxf(mx, s[r][e]);
          }
          mx = half_warp_max(mx);
          const float base = mx == -INFINITY ? 0.f : mx;
          const float corr = exp2f(m[r] - base);
          float sum = 0.f;
#pragma unroll
          for (int e = 0; e < NC; ++e) {
            s[r][e] = exp2f(s[r][e] - base);
            sum += s[r][e];
            w[r * LDP + col + 16 * e] = s[r][e];
          }
          l[r] = l[r] * corr + half_warp_sum(sum);
          m[r] = mx;
#pragma unroll
          for (int d = 0; d < DP / 32; ++d) o[r][d] = mul2(o[r][d], make_float2(corr, corr));
        }
      });
      __syncthreads();  // K has been read, and the next tile's ids are there
      if (k + 1 < x.tb) load_paged<DP>(K, c, a.layer, 0, hk, ids[(k + 1) & 1], next0, len);
      else asm volatile("cp.async.commit_group;" ::: "memory");
      wait_but_one();
      __syncthreads();  // V
      acc_tile<DP>(o, w, V, tx, gr);
      __syncthreads();
      if (k + 1 < x.tb) load_paged<DP>(V, c, a.layer, 1, hk, ids[(k + 1) & 1], next0, len);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = ty * 4 + r;
      const uint32_t half = 0xffffu << (threadIdx.x % 32 / 16 * 16);
      const bool seen = __ballot_sync(0xffffffffu, any[r]) & half;
      if (p[r] < 0) continue;
      const float top = seen ? fmaxf(m[r], kNoScore) : -INFINITY;
      if (x.whole()) {
        const int64_t tok = x.s.start + t0 + i / P.gs, h = h0 + i % P.gs;
        const float f = scale_of(top, l[r]);
        for_pieces<DP>(o[r], tx, [&](int d, const float2* v, auto n) {
          if (d < D) store_piece<decltype(n)::value>(a.y, a.y_dtype, tok * a.y_st + h * a.y_sh + d, v, f);
        });
        if (a.lse && tx == 0) a.lse[tok * a.H + h] = lse_of(top, l[r]);
      } else {
        const int64_t at = x.part() + i;
        for_pieces<DP>(o[r], tx, [&](int d, const float2* v, auto n) {
          if (d < D) store_piece<decltype(n)::value>(P.part, GDNX_F32, at * D + d, v, 1.f);
        });
        if (tx == 0) {
          P.stat[at * 2] = top;
          P.stat[at * 2 + 1] = l[r];
        }
      }
    }
    if (threadIdx.x == 0 && x.ends_cut()) P.joint[blockIdx.x] = x.joint(share.per);
  }
}

template <int DP>
gdnx_status run(const ChunkParams& P, cudaStream_t st) {
  constexpr int smem = ((BR + 2 * BT) * (DP + 4) + BR * LDP) * (int)sizeof(float);
  static std::atomic<uint64_t> done;
  if (!allow_smem(paged_attn_simt_kernel<DP>, smem, done)) return GDNX_ELAUNCH;
  if (launch_early(paged_attn_simt_kernel<DP>, dim3((unsigned)P.grid), dim3(NT), smem, st, P) != cudaSuccess)
    return GDNX_ELAUNCH;
  return join_chunks<Simt>(P, st);
}
// As many CTAs as shared memory has room for.
ChunkParams plan(const gdnx_paged_attn_args& a) { return plan_chunks<Simt>(a, sm_count() * (a.cache.D > 96 ? 2 : 3)); }

}  // namespace

size_t paged_attn_simt_workspace_bytes(const gdnx_paged_attn_args& a) { return chunk_bytes(plan(a)); }

gdnx_status launch_paged_attn_simt(const gdnx_paged_attn_args& a, cudaStream_t st) {
  const ChunkParams P = plan(a);
  return a.cache.D > 96 ? run<128>(P, st) : a.cache.D > 64 ? run<96>(P, st) : run<64>(P, st);
}

}  // namespace gdnx
