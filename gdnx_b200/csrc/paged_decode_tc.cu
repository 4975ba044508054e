// Attention of one new token per sequence over a paged cache, on the tensor cores (16-bit
// caches).  The bytes of K and V bound it; the products only have to keep out of their way.
//
// A tile.  With the keys as rows the products are narrow and nothing is padded to 128 but the
// heads to NH:  S^T [128 keys x NH] = K Q^T,  O^T [128 dims x NH] += V^T P  (V read with its
// rows as K; of head sizes up to 64 lanes 64.. read shifted rows and are not used).  Thread j owns
// key j: p_h = 2^(c s_jh - m_h), written to shared memory as the right factor, in the cache's type (both
// factors of a product have one; a weight's rounding averages out over the keys like V's own, and the
// sums take it unrounded).  The maxima m are those of the first tile and move only when some score lies
// more than 8 above (p stays below 2^8), so a tile costs one vote and no reduction; sums stay
// in the threads until the unit ends.
//
// Measured: 64 sequences of up to 8192 tokens, 16 heads over 4 of 128, pages of 64: 94 us, 5.7 TB/s of
// the copy's 6.5; one sequence of 262,144 tokens over 2 key heads: 57 us, 4.7 TB/s (its start and the
// join take 10 us); 256 sequences whose window of 1024 is read from pages of 32: 102 us.
//
// Pages come by TMA, one box for each page and 64 dims; pages that hold nothing visible are not
// fetched.  Rows that are not visible are masked in S and zeroed in V, since what unwritten
// and released pages hold may be NaN.
#include "paged_decode.cuh"

namespace gdnx {
namespace {

constexpr int NTHREADS = 224;  // four warps of keys, one that issues products, one that loads, one for the queries
struct TcParams : DecParams {
  CUtensorMap kv;  // {D, Hk * page, L * 2 * pages}
  int vec_q;       // q's rows are 16-byte aligned
};

struct Bars {
  uint64_t full[12], empty[12], q_ready[2], q_empty[2], s_full[2], p_ready[2], pv_done[2], done;
};

template <int NH>
struct Small {
  Bars bar;
  Range range;
  long long sums[NTHREADS / 32];
  float red[4 * NH];
  uint32_t tmem_at;
  int abort_flag;
};

template <int DB, int NH>
struct Layout {
  static constexpr int SLOTS = DB == 2 ? 6 : 12;  // K and V tiles in flight
  static constexpr uint32_t TILE = DB * BLOCK_BYTES;
  static constexpr uint32_t QB = DB * NH * 128, PB = 2 * NH * 128;  // a Q tile, a P tile
  static constexpr uint32_t RING = 0, Q = SLOTS * TILE, P = Q + 2 * QB, SMALL = P + 2 * PB;
  // no static shared memory: the base is 1024-aligned
  static constexpr size_t SMEM = SMALL + sizeof(Small<NH>);
  static constexpr int TMEM = NH == 16 ? 64 : 128;  // columns: S twice, O
};

GDNX_DEV void tma_load_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t mbar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(mbar)
      : "memory");
}

template <int DB, int NH>
GDNX_DEV void run_loads(const TcParams& P, Walk w, uint32_t smem, Bars& bar, volatile int* abort_flag) {
  using Lo = Layout<DB, NH>;
  const gdnx_cache& c = P.a.cache;
  const int lane = threadIdx.x % 32, npp = TM / c.page, page = c.page;
  const int ahead = 32 / npp;  // tiles whose page ids one load of the warp covers
  const uint32_t box = (uint32_t)page * 128;
  uint32_t cnt = 0;
  while (w.next()) {
    const int hk = w.unit / P.groups;
    int ids = -1;
    for (int t = w.ta; t < w.tb; ++t) {
      const int k = (t - w.ta) % ahead;
      if (k == 0) {
        const int mine = t + lane / npp;
        ids = mine < w.tb ? page_id(P, w.seq, w.seq.kt.tile(mine), lane % npp) : -1;
      }
      const int pg = lane / DB, d = lane % DB;
      const int id = __shfl_sync(0xffffffffu, ids, (k * npp + pg) & 31);
      const bool go = pg < npp && id >= 0;
      const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, go)) * box;
#pragma unroll
      for (int side = 0; side < 2; ++side, ++cnt) {
        const uint32_t sl = cnt % Lo::SLOTS, mb = tc::smem_u32(&bar.full[sl]);
        if (!warp_wait(&bar.empty[sl], (cnt / Lo::SLOTS & 1) ^ 1, abort_flag)) return;
        if (lane == 0) pipe::expect_tx(mb, bytes);
        __syncwarp();
        if (go)
          tma_load_3d(smem + Lo::RING + sl * Lo::TILE + d * BLOCK_BYTES + pg * box, &P.kv, d * 64, hk * page,
                      (int)((P.a.layer * 2 + side) * c.pages + id), mb);
      }
    }
  }
}

template <int DB, int NH, bool BF16>
GDNX_DEV void run_products(const TcParams& P, Walk w, uint32_t smem, uint32_t tmem, Bars& bar,
                           volatile int* abort_flag) {
  using Lo = Layout<DB, NH>;
  constexpr uint32_t ID_S = idesc16(BF16, 128, NH, false, false), ID_O = idesc16(BF16, 128, NH, true, false);
  // S(t+1) goes out before P(t) is waited for, so the rows may be done with t+1 by then, and
  // they skip most of pv_done: both have a barrier for each parity of t, which cannot be lapped
  // (S(t+2) follows PV(t))
  uint32_t nt = 0, seg = 0;  // tiles and segments so far
  bool pend = false, first = false;
  const auto values = [&]() {  // O^T += V^T P of the tile before
    if (!pend) return true;
    const uint32_t t = nt - 1, vc = 2 * t + 1, sl = vc % Lo::SLOTS;
    if (!warp_wait(&bar.full[sl], vc / Lo::SLOTS & 1, abort_flag)) return false;
    if (!warp_wait(&bar.p_ready[t & 1], t / 2 & 1, abort_flag)) return false;
    tc::fence_after();
    if (elect_one()) {
      const uint64_t v = tc::smem_desc(smem + Lo::RING + sl * Lo::TILE, DB == 2 ? BLOCK_BYTES : 1024, 1024);
      const uint64_t p = tc::smem_desc(smem + Lo::P + (t & 1) * Lo::PB, 16, 1024);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        tc::mma_bf16(tmem + 2 * NH, v + k * (2048 >> 4), p + (((k / 4) * NH * 128 + (k % 4) * 32) >> 4), ID_O,
                     !first || k > 0);
      tc::commit(&bar.pv_done[t & 1]);
      tc::commit(&bar.empty[sl]);
    }
    __syncwarp();
    pend = false;
    return true;
  };
  for (; w.next(); ++seg) {
    for (int t = w.ta; t < w.tb; ++t) {
      const uint32_t kc = 2 * nt, sl = kc % Lo::SLOTS;
      if (t == w.ta) {
        // the last unit's output is read before its successor's first product by p_ready
        if (!values()) return;
        if (!warp_wait(&bar.q_ready[seg & 1], seg / 2 & 1, abort_flag)) return;
      }
      if (!warp_wait(&bar.full[sl], kc / Lo::SLOTS & 1, abort_flag)) return;
      tc::fence_after();
      if (elect_one()) {
        const uint64_t k = tc::smem_desc(smem + Lo::RING + sl * Lo::TILE, 16, 1024);
        const uint64_t q = tc::smem_desc(smem + Lo::Q + (seg & 1) * Lo::QB, 16, 1024);
#pragma unroll
        for (int x = 0; x < 4 * DB; ++x)
          tc::mma_bf16(tmem + (nt & 1) * NH, k + (((x / 4) * BLOCK_BYTES + (x % 4) * 32) >> 4),
                       q + (((x / 4) * NH * 128 + (x % 4) * 32) >> 4), ID_S, x > 0);
        tc::commit(&bar.s_full[nt & 1]);
        tc::commit(&bar.empty[sl]);
        if (t + 1 == w.tb) tc::commit(&bar.q_empty[seg & 1]);
      }
      __syncwarp();
      if (!values()) return;
      ++nt;
      pend = true;
      first = t == w.ta;
    }
  }
  values();
}

// The unit's query rows as a K-major tile of NH rows (rows beyond its heads zero), by one warp.
template <int DB, int NH>
GDNX_DEV void stage_q(const TcParams& P, const Walk& w, uint8_t* dst) {
  const gdnx_paged_decode_args& a = P.a;
  const Heads hd(P, w.unit, NH);
  const int D = (int)a.cache.D;
#pragma unroll 4
  for (int x = threadIdx.x % 32; x < NH * DB * 8; x += 32) {
    const int h = x / (DB * 8), c = x % (DB * 8);
    uint4 u = make_uint4(0, 0, 0, 0);
    if (h < hd.n && c * 8 < D) {
      const uint16_t* src = static_cast<const uint16_t*>(a.q.ptr) + w.b * a.q.sb + (hd.h0 + h) * a.q.sh + c * 8;
      if (P.vec_q) {
        u = *reinterpret_cast<const uint4*>(src);
      } else {
        u.x = src[0] | (uint32_t)src[1] << 16;
        u.y = src[2] | (uint32_t)src[3] << 16;
        u.z = src[4] | (uint32_t)src[5] << 16;
        u.w = src[6] | (uint32_t)src[7] << 16;
      }
    }
    *reinterpret_cast<uint4*>(dst + tc::sw128(h, c, NH)) = u;
  }
}

template <int DB, int NH>
GDNX_DEV void run_queries(const TcParams& P, Walk w, uint8_t* base, Bars& bar, volatile int* abort_flag) {
  using Lo = Layout<DB, NH>;
  for (uint32_t seg = 0; w.next(); ++seg) {
    if (!warp_wait(&bar.q_empty[seg & 1], (seg / 2 & 1) ^ 1, abort_flag)) return;
    stage_q<DB, NH>(P, w, base + Lo::Q + (seg & 1) * Lo::QB);
    tc::fence_async_smem();
    pipe::mbar_arrive(&bar.q_ready[seg & 1]);
  }
}

// NC columns of a thread's lane, in the widths of a tensor-memory move (4 and 8 at once).
template <int NC>
GDNX_DEV void tmem_ld(uint32_t at, float (&v)[NC]) {
#pragma unroll
  for (int i = 0; i < NC; i += 4)
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=f"(v[i]), "=f"(v[i + 1]), "=f"(v[i + 2]), "=f"(v[i + 3])
                 : "r"(at + i)
                 : "memory");
}
template <>
GDNX_DEV void tmem_ld<16>(uint32_t at, float (&v)[16]) { tc::tmem_ld16(at, v); }
template <>
GDNX_DEV void tmem_ld<32>(uint32_t at, float (&v)[32]) { tc::tmem_ld32(at, v); }
template <int NC>
GDNX_DEV void tmem_st(uint32_t at, const float (&v)[NC]) {
#pragma unroll
  for (int i = 0; i < NC; i += 4)
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};\n\ttcgen05.wait::st.sync.aligned;"
                 :
                 : "r"(at + i), "f"(v[i]), "f"(v[i + 1]), "f"(v[i + 2]), "f"(v[i + 3])
                 : "memory");
}

// NC: heads that a thread works on, the unit's rounded up (the others' columns are not used).
template <int DB, int NH, int NC, bool BF16>
GDNX_DEV void run_keys(const TcParams& P, Walk w, int64_t per, uint8_t* base, uint32_t tmem, Bars& bar, float* red,
                       volatile int* abort_flag) {
  using Lo = Layout<DB, NH>;
  const gdnx_paged_decode_args& a = P.a;
  const int r = threadIdx.x, lane = r % 32, warp = r / 32, D = (int)a.cache.D;
  const uint32_t lane_at = (uint32_t)(warp * 32) << 16;
  const float c2 = a.scale * kLog2e;
  const int window = (int)a.window, sinks = (int)a.sinks;
  uint32_t nt = 0;
  bool ok = true;  // a wait that gave up is told at the next vote, where all four warps leave
  if (r == 0 && !P.whole) P.joint[blockIdx.x] = {0, 0, 0, -1};
  while (w.next()) {
    const Heads hd(P, w.unit, NH);
    float m[NC], l[NC];
    bool any = false;  // this thread saw a key
#pragma unroll
    for (int h = 0; h < NC; ++h) {
      m[h] = -INFINITY;
      l[h] = 0.f;
    }
    for (int t = w.ta; t < w.tb; ++t, ++nt) {
      const int j0 = w.seq.kt.tile(t) * TM, j = j0 + r;
      // a released page inside the visible range is not seen either
      bool seen = key_seen(j, w.seq.len, window, sinks);
      if (seen) {
        const int p = a.cache.table[(int64_t)w.seq.row * a.cache.width + j / a.cache.page];
        seen = p >= 0 && p < a.cache.pages;
      }
      any |= seen;
      ok = ok && warp_wait(&bar.s_full[nt & 1], nt / 2 & 1, abort_flag);
      tc::fence_after();
      float s[NC];
      tmem_ld(tmem + lane_at + (nt & 1) * NH, s);
      bool over = t == w.ta || !ok;
#pragma unroll
      for (int h = 0; h < NC; ++h) {
        s[h] = seen ? s[h] * c2 : -INFINITY;
        over |= s[h] > m[h] + 8.f;
      }
      if (pipe::group_any(1, 128, over)) {
        // new maxima: of each warp's keys, then of the four warps
#pragma unroll
        for (int h = 0; h < NC; ++h) {
          float x = s[h];
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
          if (lane == 0) red[warp * NH + h] = x;
        }
        if (pipe::group_any(1, 128, !ok)) return;
        float o[NC];
        if (t > w.ta) {
          ok = warp_wait(&bar.pv_done[(nt - 1) & 1], (nt - 1) / 2 & 1, abort_flag);
          tc::fence_after();
          tmem_ld(tmem + lane_at + 2 * NH, o);
        }
#pragma unroll
        for (int h = 0; h < NC; ++h) {
          const float x = fmaxf(fmaxf(fmaxf(red[h], red[NH + h]), fmaxf(red[2 * NH + h], red[3 * NH + h])), m[h]);
          const float corr = x == -INFINITY ? 1.f : ex2(m[h] - x);
          m[h] = x;
          l[h] *= corr;
          if (t > w.ta) o[h] *= corr;
        }
        if (t > w.ta) tmem_st(tmem + lane_at + 2 * NH, o);
        if (pipe::group_any(1, 128, !ok)) return;  // and red may be written again
      }
      uint8_t* pt = base + Lo::P + (nt & 1) * Lo::PB + (r / 64) * NH * 128 + r % 8 * 2;
#pragma unroll
      for (int h = 0; h < NC; ++h) {
        const float p = ex2(s[h] - (m[h] == -INFINITY ? 0.f : m[h]));
        l[h] += p;
        *reinterpret_cast<uint16_t*>(pt + h * 128 + (((r % 64 / 8) ^ (h & 7)) << 4)) = (uint16_t)pack2<BF16>(p, 0.f);
      }
      if (__any_sync(0xffffffffu, !seen)) {
        const uint32_t vc = 2 * nt + 1, sl = vc % Lo::SLOTS;
        ok = warp_wait(&bar.full[sl], vc / Lo::SLOTS & 1, abort_flag);
        if (!seen && ok)
#pragma unroll
          for (int c = 0; c < DB * 8; ++c)  // rows begin at different pieces: no bank conflicts
            *reinterpret_cast<uint4*>(base + Lo::RING + sl * Lo::TILE + (c / 8) * BLOCK_BYTES + r * 128 + ((c ^ r) & 7) * 16) =
                make_uint4(0, 0, 0, 0);
      }
      tc::fence_async_smem();
      tc::fence_before();
      pipe::mbar_arrive(&bar.p_ready[nt & 1]);
    }
    // the unit's sums, then its output: lane d of tensor memory holds dimension d.  (Without a score above -inf
    // the sums tell whether a key was seen.)
#pragma unroll
    for (int h = 0; h < NC; ++h) {
      const float x = warp_sum(any && m[h] == -INFINITY ? l[h] + 1.f : l[h]);
      if (lane == 0) red[warp * NH + h] = x;
    }
    if (pipe::group_any(1, 128, !ok)) return;
    ok = warp_wait(&bar.pv_done[(nt - 1) & 1], (nt - 1) / 2 & 1, abort_flag);
    tc::fence_after();
    float o[NC];
    tmem_ld(tmem + lane_at + 2 * NH, o);
    const bool whole = w.whole();
    // a part that goes on in the next CTA is this CTA's last, any other its first
    const int64_t at = ((int64_t)blockIdx.x * 2 + (w.tb < w.seq.kt.count && w.ta == 0 ? 1 : 0)) * NH;
#pragma unroll
    for (int h = 0; h < NC; ++h) {
      if (h >= hd.n) continue;
      float sum = red[h] + red[NH + h] + red[2 * NH + h] + red[3 * NH + h], top = m[h];
      if (top == -INFINITY && sum > 0.f) {
        top = kNoScore;
        sum = 0.f;
      }
      if (whole) {
        if (r < D)
          st_from_f32(a.y, a.y_dtype, w.b * a.y_sb + (hd.h0 + h) * a.y_sh + r,
                      sum == 0.f ? no_weights(top) : o[h] * (1.f / sum));
      } else {
        P.part[(at + h) * 128 + r] = o[h];
        if (r == 0) {
          P.stat[(at + h) * 2] = top;
          P.stat[(at + h) * 2 + 1] = sum;
        }
      }
    }
    if (r == 0 && w.ta > 0 && w.tb == w.seq.kt.count)  // the unit's last part
      P.joint[blockIdx.x] = {(int)w.b, w.unit, (int)((w.before + (int64_t)w.unit * w.seq.kt.count) / per), (int)blockIdx.x};
    if (pipe::group_any(1, 128, !ok)) return;  // and red may be written again
  }
}

template <int DB, int NC, bool BF16>
__global__ void __launch_bounds__(NTHREADS, 1) paged_decode_tc_kernel(const __grid_constant__ TcParams P) {
  constexpr int NH = NC > 16 ? 32 : 16;
  using Lo = Layout<DB, NH>;
  extern __shared__ __align__(1024) uint8_t base[];
  Small<NH>& sm = *reinterpret_cast<Small<NH>*>(base + Lo::SMALL);
  Bars& bar = sm.bar;
  volatile int* abort_flag = &sm.abort_flag;
  const uint32_t smem = uniform(tc::smem_u32(base));
  const int warp = uniform(threadIdx.x / 32), units = (int)P.a.cache.Hk * P.groups;
  dependents_may_start();
  if (warp == 4) {
    tc::tmem_alloc(&sm.tmem_at, Lo::TMEM);
  } else if (threadIdx.x == 160) {
    *abort_flag = smem % 1024 ? 1 : 0;  // swizzled tiles need an aligned base
    for (int i = 0; i < Lo::SLOTS; ++i) {
      tc::mbar_init(&bar.full[i], 1);
      tc::mbar_init(&bar.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&bar.q_ready[i], 32);
      tc::mbar_init(&bar.q_empty[i], 1);
      tc::mbar_init(&bar.s_full[i], 1);
      tc::mbar_init(&bar.p_ready[i], 128);
      tc::mbar_init(&bar.pv_done[i], 1);
    }
    tc::mbar_init(&bar.done, 1);
  }
  tc::fence_before();
  wait_for_earlier();
  find_range<NTHREADS>(P, units, sm.range, sm.sums);  // synchronises
  tc::fence_after();
  const uint32_t tmem = uniform(sm.tmem_at);
  const Walk w(P, units, sm.range);
  if (smem % 1024) {  // never entered: the base is aligned
  } else if (warp < 4) {
    run_keys<DB, NH, NC, BF16>(P, w, sm.range.per, base, tmem, bar, sm.red, abort_flag);
  } else if (warp == 4) {
    run_products<DB, NH, BF16>(P, w, smem, tmem, bar, abort_flag);
    __syncwarp();
    if (elect_one()) tc::commit(&bar.done);  // every product issued has ended before tensor memory is freed
    tc::mbar_wait(&bar.done, 0);
  } else if (warp == 6) {
    run_queries<DB, NH>(P, w, base, bar, abort_flag);
  } else {
    run_loads<DB, NH>(P, w, smem, bar, abort_flag);
    write_zeros(P);
    if (*abort_flag)  // let the copies in flight land
      for (uint32_t it = 0; it < (1u << 12); ++it) __nanosleep(100);
  }
  __syncwarp();
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (warp == 4) tc::tmem_dealloc(tmem, Lo::TMEM);
  if (threadIdx.x == 0 && *abort_flag && P.a.error) *P.a.error = GDNX_ETIMEOUT;
}

template <int DB, int NC, bool BF16>
gdnx_status launch(const TcParams& P, cudaStream_t st) {
  constexpr int NH = NC > 16 ? 32 : 16;
  const auto kernel = paged_decode_tc_kernel<DB, NC, BF16>;
  constexpr int smem = (int)Layout<DB, NH>::SMEM;
  static std::atomic<uint64_t> done;
  if (!allow_smem(kernel, smem, done)) return GDNX_ELAUNCH;
  if (launch_early(kernel, dim3((unsigned)P.grid), dim3(NTHREADS), smem, st, P) != cudaSuccess) return GDNX_ELAUNCH;
  return join_parts<NH>(P, st);
}

template <int DB, bool BF16>
gdnx_status launch_heads(const TcParams& P, cudaStream_t st) {
  const int64_t G = P.a.H / P.a.cache.Hk;
  if (G <= 4) return launch<DB, 4, BF16>(P, st);
  if (G <= 8) return launch<DB, 8, BF16>(P, st);
  return G <= 16 ? launch<DB, 16, BF16>(P, st) : launch<DB, 32, BF16>(P, st);
}

template <bool BF16>
gdnx_status launch_type(const TcParams& P, cudaStream_t st) {
  return P.a.cache.D > 64 ? launch_heads<2, BF16>(P, st) : launch_heads<1, BF16>(P, st);
}

}  // namespace

size_t paged_decode_tc_workspace_bytes(const gdnx_paged_decode_args& a) {
  return plan_bytes(make_plan(a, a.H / a.cache.Hk > 16 ? 32 : 16));
}

gdnx_status launch_paged_decode_tc(const gdnx_paged_decode_args& a, cudaStream_t st) {
  const gdnx_cache& c = a.cache;
  const EncodeTiledFn enc = encode_fn();
  if (!enc) return GDNX_ELAUNCH;
  if (c.L * 2 * c.pages > ((int64_t)1 << 31) - 1 || c.Hk * c.page * c.D * 2 >= ((int64_t)1 << 40))
    return GDNX_EUNSUPPORTED;
  TcParams P;
  const cuuint64_t dims[3] = {(cuuint64_t)c.D, (cuuint64_t)(c.Hk * c.page), (cuuint64_t)(c.L * 2 * c.pages)};
  const cuuint64_t strides[2] = {(cuuint64_t)c.D * 2, (cuuint64_t)(c.Hk * c.page * c.D) * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)c.page, 1}, es[3] = {1, 1, 1};
  if (enc(&P.kv, c.dtype == GDNX_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, c.kv,
          dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return GDNX_EINVAL;
  fill(P, a, make_plan(a, a.H / c.Hk > 16 ? 32 : 16));
  P.vec_q = reinterpret_cast<uintptr_t>(a.q.ptr) % 16 == 0 && a.q.sb % 8 == 0 && a.q.sh % 8 == 0;
  return c.dtype == GDNX_BF16 ? launch_type<true>(P, st) : launch_type<false>(P, st);
}

}  // namespace gdnx
