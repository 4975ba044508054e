// Attention of one new token per sequence over a paged cache of 32-bit values, on the CUDA cores
// (all arithmetic fp32; the work of a call is cut as in paged_decode.cuh).
//
// The bytes of K and V bound it, so the loads run by themselves: one warp copies the keys and
// values of 32 tokens at a time into a ring of six stages (a head's tokens of one page are one
// contiguous run: bulk asynchronous copies), 160 KB ahead of the eight warps that use them.
// Each of these takes four of a stage's tokens, 32 / LPK at a time; LPK lanes share a token, eight
// values of its row each, and hold the unit's NH query heads and outputs for them:
//   s = c q.k (a sum over LPK lanes);  p = 2^(s - m);  l += p;  o += p v
// with the maximum m moved only where a score lies more than 8 above it (a vote of the warp).
// The groups' (m, l, o) are joined when the unit ends.
//
// Measured: 64 sequences of 4096 tokens, 16 heads over 4 of 128: 230 us, 4.7 TB/s; one of 16,384 tokens: 34 us with
// nothing in L2.  Two warps a scheduler issue in 52 % of cycles and have one ready in as many: a warp's chain of
// dot product, exponential and sums, not the loads, is what the ring waits for.
#include "paged_decode.cuh"

namespace gdnx {
namespace {

constexpr int WARPS = 8;                     // that use the loads
constexpr int NTHREADS = WARPS * 32 + 32;
constexpr int SUB = 32;                      // tokens of a stage
constexpr int STAGES = 6;
constexpr uint32_t SIDE = SUB * 128 * 4;     // bytes of a stage's keys or values, at most
constexpr float kLazy = 8.f;

template <int NH>
struct Small {
  float o[WARPS][NH][128], m[WARPS][NH], l[WARPS][NH];
  uint64_t full[STAGES], empty[STAGES];
  Range range;
  long long sums[NTHREADS / 32];
  int ok[STAGES];  // which halves of a stage's tokens lie on pages
  int abort_flag;
};

// Does the sequence's newest token see any of tokens j..j+31?
GDNX_DEV bool sub_seen(int j, int len, int64_t window, int64_t sinks) {
  return j < len && (j + SUB > (int64_t)len - window || j < sinks);
}

template <int NH>
GDNX_DEV void load_stages(const DecParams& P, Walk w, uint8_t* ring, Small<NH>& sm) {
  const gdnx_cache& c = P.a.cache;
  const int lane = threadIdx.x % 32, page = c.page, npp = TM / page, ahead = 32 / npp, D = (int)c.D;
  const int runs = page < SUB ? SUB / page : 1, tokens = SUB / runs;  // contiguous runs of a stage
  const float* kv = static_cast<const float*>(c.kv);
  uint32_t n = 0;
  while (w.next()) {
    const int hk = w.unit / P.groups;
    int ids = -1;
    for (int t = w.ta; t < w.tb; ++t) {
      const int k = (t - w.ta) % ahead;
      if (k == 0) {
        const int mine = t + lane / npp;
        ids = mine < w.tb ? page_id(P, w.seq, w.seq.kt.tile(mine), lane % npp) : -1;
      }
      for (int s = 0; s < TM / SUB; ++s) {
        const int j = w.seq.kt.tile(t) * TM + s * SUB;
        if (!sub_seen(j, w.seq.len, P.a.window, P.a.sinks)) continue;
        const uint32_t st = n % STAGES;
        if (!warp_wait(&sm.empty[st], (n / STAGES & 1) ^ 1, &sm.abort_flag)) return;
        ++n;
        // lane: side and run
        const int run = lane / 2 % 2, side = lane % 2;
        const int id = __shfl_sync(0xffffffffu, ids, (k * npp + (s * SUB + run * tokens) / page) & 31);
        const bool go = lane < 4 && run < runs && id >= 0;
        const uint32_t got = __ballot_sync(0xffffffffu, go);
        const uint32_t bar = tc::smem_u32(&sm.full[st]), bytes = (uint32_t)(tokens * D * 4);
        if (lane == 0) {
          sm.ok[st] = runs == 1 ? (got & 1 ? 3 : 0) : (int)((got & 1) | (got >> 1 & 2));
          pipe::expect_tx(bar, __popc(got) * bytes);
        }
        __syncwarp();
        if (go) {
          const int64_t row = ((((P.a.layer * 2 + side) * c.pages + id) * c.Hk + hk) * page + (j + run * tokens) % page);
          pipe::bulk_load(tc::smem_u32(ring) + st * 2 * SIDE + side * SIDE + run * tokens * D * 4, kv + row * D, bytes, bar);
        }
      }
    }
  }
}

template <int LPK, int NH>
GDNX_DEV void use_stages(const DecParams& P, Walk w, int64_t per, const uint8_t* ring, Small<NH>& sm) {
  constexpr int KPW = 32 / LPK, PASSES = SUB / WARPS / KPW;
  const gdnx_paged_decode_args& a = P.a;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, sub = lane / LPK, dl = lane % LPK, D = (int)a.cache.D;
  const int d0 = 4 * dl, d1 = 4 * (LPK + dl);  // this lane's two runs of four values
  const int window = (int)a.window, sinks = (int)a.sinks;
  const float c2 = a.scale * kLog2e;
  uint32_t n = 0;
  bool ok = true;  // a wait that gave up is told at the next vote, where all warps leave
  if (threadIdx.x == 0 && !P.whole) P.joint[blockIdx.x] = {0, 0, 0, -1};
  while (w.next()) {
    const Heads hd(P, w.unit, NH);
    float q[NH][8], o[NH][8], m[NH], l[NH];
    bool any = false;  // this lane's group saw a token
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      m[h] = -INFINITY;
      l[h] = 0.f;
      const float* row = static_cast<const float*>(a.q.ptr) + w.b * a.q.sb + (hd.h0 + h) * a.q.sh;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int d = (e < 4 ? d0 : d1 - 4) + e;
        o[h][e] = 0.f;
        q[h][e] = h < hd.n && d < D ? row[d] * c2 : 0.f;
      }
    }
    for (int t = w.ta; t < w.tb; ++t) {
      for (int s = 0; s < TM / SUB; ++s) {
        const int j0 = w.seq.kt.tile(t) * TM + s * SUB;
        if (!sub_seen(j0, w.seq.len, a.window, a.sinks)) continue;
        const uint32_t st = n % STAGES;
        ok = ok && warp_wait(&sm.full[st], n / STAGES & 1, &sm.abort_flag);
        ++n;
        if (!ok) continue;
        const int on_page = *const_cast<volatile int*>(&sm.ok[st]);
        const float* kt = reinterpret_cast<const float*>(ring + st * 2 * SIDE);
        const float* vt = reinterpret_cast<const float*>(ring + st * 2 * SIDE + SIDE);
        float x[PASSES][NH];
        bool seen[PASSES], over = false;
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
          const int r = warp * (SUB / WARPS) + i * KPW + sub, j = j0 + r;
          seen[i] = key_seen(j, w.seq.len, window, sinks) && (on_page >> (r / 16) & 1);
          any |= seen[i];
          float4 k0 = make_float4(0.f, 0.f, 0.f, 0.f), k1 = k0;
          if (seen[i] && d0 < D) k0 = *reinterpret_cast<const float4*>(kt + r * D + d0);
          if (seen[i] && d1 < D) k1 = *reinterpret_cast<const float4*>(kt + r * D + d1);
#pragma unroll
          for (int h = 0; h < NH; ++h) {
            float d = q[h][0] * k0.x;
            d = fmaf(q[h][1], k0.y, d);
            d = fmaf(q[h][2], k0.z, d);
            d = fmaf(q[h][3], k0.w, d);
            d = fmaf(q[h][4], k1.x, d);
            d = fmaf(q[h][5], k1.y, d);
            d = fmaf(q[h][6], k1.z, d);
            d = fmaf(q[h][7], k1.w, d);
#pragma unroll
            for (int z = LPK / 2; z > 0; z >>= 1) d += __shfl_xor_sync(0xffffffffu, d, z);
            x[i][h] = seen[i] ? d : -INFINITY;
            over |= x[i][h] > m[h] + kLazy;
          }
        }
        if (__any_sync(0xffffffffu, over)) {
#pragma unroll
          for (int h = 0; h < NH; ++h) {
            float top = m[h];
#pragma unroll
            for (int i = 0; i < PASSES; ++i) top = fmaxf(top, x[i][h]);
            const float corr = top == -INFINITY ? 1.f : exp2f(m[h] - top);
            m[h] = top;
            l[h] *= corr;
#pragma unroll
            for (int e = 0; e < 8; ++e) o[h][e] *= corr;
          }
        }
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
          const int r = warp * (SUB / WARPS) + i * KPW + sub;
          float4 v0 = make_float4(0.f, 0.f, 0.f, 0.f), v1 = v0;
          if (seen[i] && d0 < D) v0 = *reinterpret_cast<const float4*>(vt + r * D + d0);
          if (seen[i] && d1 < D) v1 = *reinterpret_cast<const float4*>(vt + r * D + d1);
#pragma unroll
          for (int h = 0; h < NH; ++h) {
            const float p = x[i][h] == -INFINITY ? 0.f : exp2f(x[i][h] - m[h]);
            l[h] += p;
            o[h][0] = fmaf(p, v0.x, o[h][0]);
            o[h][1] = fmaf(p, v0.y, o[h][1]);
            o[h][2] = fmaf(p, v0.z, o[h][2]);
            o[h][3] = fmaf(p, v0.w, o[h][3]);
            o[h][4] = fmaf(p, v1.x, o[h][4]);
            o[h][5] = fmaf(p, v1.y, o[h][5]);
            o[h][6] = fmaf(p, v1.z, o[h][6]);
            o[h][7] = fmaf(p, v1.w, o[h][7]);
          }
        }
        __syncwarp();
        if (lane == 0) pipe::mbar_arrive(&sm.empty[st]);
      }
    }
    // the groups of a warp, then the warps in order
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      if (any) m[h] = fmaxf(m[h], kNoScore);
      float top = m[h];
#pragma unroll
      for (int z = LPK; z < 32; z <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, z));
      const float corr = top == -INFINITY ? 0.f : exp2f(m[h] - top);
      l[h] *= corr;
#pragma unroll
      for (int z = LPK; z < 32; z <<= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], z);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        o[h][e] *= corr;
#pragma unroll
        for (int z = LPK; z < 32; z <<= 1) o[h][e] += __shfl_xor_sync(0xffffffffu, o[h][e], z);
      }
      if (sub == 0) {
        *reinterpret_cast<float4*>(&sm.o[warp][h][d0]) = make_float4(o[h][0], o[h][1], o[h][2], o[h][3]);
        *reinterpret_cast<float4*>(&sm.o[warp][h][d1]) = make_float4(o[h][4], o[h][5], o[h][6], o[h][7]);
        if (dl == 0) {
          sm.m[warp][h] = top;
          sm.l[warp][h] = l[h];
        }
      }
    }
    if (pipe::group_any(1, WARPS * 32, !ok)) return;
    const bool whole = w.whole();
    // a part that goes on in the next CTA is this CTA's last, any other its first
    const int64_t at = ((int64_t)blockIdx.x * 2 + (w.tb < w.seq.kt.count && w.ta == 0 ? 1 : 0)) * NH;
    for (int i = threadIdx.x; i < hd.n * D; i += WARPS * 32) {
      const int h = i / D, d = i % D;
      float top = -INFINITY, sum = 0.f, y = 0.f;
#pragma unroll
      for (int k = 0; k < WARPS; ++k) top = fmaxf(top, sm.m[k][h]);
      const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int k = 0; k < WARPS; ++k) {
        const float z = exp2f(sm.m[k][h] - ref);
        sum = fmaf(z, sm.l[k][h], sum);
        y = fmaf(z, sm.o[k][h][d], y);
      }
      if (whole) {
        st_from_f32(a.y, a.y_dtype, w.b * a.y_sb + (hd.h0 + h) * a.y_sh + d, sum == 0.f ? no_weights(top) : y / sum);
      } else {
        P.part[(at + h) * 128 + d] = y;
        if (d == 0) {
          P.stat[(at + h) * 2] = top;
          P.stat[(at + h) * 2 + 1] = sum;
        }
      }
    }
    if (threadIdx.x == 0 && w.ta > 0 && w.tb == w.seq.kt.count)  // the unit's last part
      P.joint[blockIdx.x] = {(int)w.b, w.unit, (int)((w.before + (int64_t)w.unit * w.seq.kt.count) / per), (int)blockIdx.x};
    if (pipe::group_any(1, WARPS * 32, !ok)) return;  // what was joined may be written again
  }
}

template <int LPK, int NH>
__global__ void __launch_bounds__(NTHREADS, 1) paged_decode_kernel(const DecParams P) {
  extern __shared__ __align__(128) uint8_t ring[];
  Small<NH>& sm = *reinterpret_cast<Small<NH>*>(ring + STAGES * 2 * SIDE);
  const int warp = threadIdx.x / 32, units = (int)P.a.cache.Hk * P.groups;
  dependents_may_start();
  if (threadIdx.x == 0) {
    sm.abort_flag = 0;
    for (int i = 0; i < STAGES; ++i) {
      tc::mbar_init(&sm.full[i], 1);
      tc::mbar_init(&sm.empty[i], WARPS);
    }
  }
  wait_for_earlier();
  find_range<NTHREADS>(P, units, sm.range, sm.sums);  // synchronises
  const Walk w(P, units, sm.range);
  if (warp < WARPS) {
    use_stages<LPK, NH>(P, w, sm.range.per, ring, sm);
  } else {
    load_stages<NH>(P, w, ring, sm);
    write_zeros(P);
    if (*const_cast<volatile int*>(&sm.abort_flag))  // let the copies in flight land
      for (uint32_t it = 0; it < (1u << 12); ++it) __nanosleep(100);
  }
  __syncthreads();
  if (threadIdx.x == 0 && sm.abort_flag && P.a.error) *P.a.error = GDNX_ETIMEOUT;
}

template <int LPK, int NH>
gdnx_status launch(const DecParams& P, cudaStream_t st) {
  constexpr int smem = (int)(STAGES * 2 * SIDE + sizeof(Small<NH>));
  const auto kernel = paged_decode_kernel<LPK, NH>;
  static std::atomic<uint64_t> done;
  if (!allow_smem(kernel, smem, done)) return GDNX_ELAUNCH;
  if (launch_early(kernel, dim3((unsigned)P.grid), dim3(NTHREADS), smem, st, P) != cudaSuccess) return GDNX_ELAUNCH;
  return join_parts<NH>(P, st);
}

// Query heads of a unit.
int heads_of(const gdnx_paged_decode_args& a) { return a.H / a.cache.Hk > 4 ? 8 : 4; }

}  // namespace

size_t paged_decode_workspace_bytes(const gdnx_paged_decode_args& a) { return plan_bytes(make_plan(a, heads_of(a))); }

gdnx_status launch_paged_decode(const gdnx_paged_decode_args& a, cudaStream_t st) {
  DecParams P;
  fill(P, a, make_plan(a, heads_of(a)));
  if (a.cache.D > 64) return heads_of(a) == 4 ? launch<16, 4>(P, st) : launch<16, 8>(P, st);
  return heads_of(a) == 4 ? launch<8, 4>(P, st) : launch<8, 8>(P, st);
}

}  // namespace gdnx
