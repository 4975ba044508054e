// Windowed attention, forward, on the tensor cores (16-bit inputs that TMA can address).
//
// A persistent CTA takes two blocks of 128 queries of one key head at a time ("stages":
// two query heads at the same positions where the key head serves an even number of them,
// else two consecutive blocks of one head) and walks the key tiles of 128 that either sees:
//   S_s = Q_s K^T (tcgen05, fp32 in tensor memory) -> registers, one query per thread:
//   m = max, p = 2^(c (s - m)), l += p -> P_s packed 16-bit over S_s's columns ->
//   O_s += P_s V (tcgen05, P from tensor memory, V read with its rows as K).
// While one stage's 128 threads take exponentials, the tensor cores work for the other.
// Warps 0-3 and 4-7 are the stages' rows, warp 8 issues the products, warp 9 the TMA loads
// (Q of each stage, K and V through one ring).  The product warp puts PV(t) and S(t+1) of a
// stage in one run, so S(t+1) complete means PV(t) complete and O at rest.
//
// The maximum is lazy: P is taken against the last m that O was scaled to, and O is rescaled
// only when the new maximum is more than 8 above it in log2 (P stays below 2^8, exact in
// fp32 sums and without overflow in either 16-bit type); the result does not depend on m.
// P is rounded to the inputs' type, the error of which averages out over the keys like the
// inputs' own rounding; l sums it unrounded in fp32.
#include "attn_tc.cuh"
#include "kernels.h"

namespace gdnx {
namespace {

using namespace attn;

constexpr int NTHREADS = 384;  // three warpgroups: a stage's rows each, and the warps that issue
constexpr uint32_t T_S = 0, T_O = 256;  // tensor-memory columns: S_0, S_1, then O_0, O_1

struct FwdParams {
  TileMap q, k, v;
  gdnx_attn_args a;
  int64_t items;
  int pairs, units, by_heads;  // stage pairs of a key head; blocks (or block pairs) of queries
};

// One stage of a work item: head, first row, the key tiles of its rows.
struct Stage {
  int h, i0, p0, p1, lo, hi;  // hi < 0: sees nothing
  bool valid;
};

struct Item {
  int b, hk, len, nst;  // nst: tiles that hold sinks
  Stage s[2];
  int nsink, lo, count;  // the tiles either stage sees, as one sequence
  GDNX_DEV int tile(int i) const { return i < nsink ? i : lo + i - nsink; }
  GDNX_DEV bool active(int st, int kt) const {
    const Stage& x = s[st];
    return kt <= x.hi && (kt >= x.lo || kt < nst);
  }
};

GDNX_DEV Item make_item(const FwdParams& P, int64_t n) {
  const gdnx_attn_args& a = P.a;
  Item w;
  const int Hk = (int)a.Hk, G = (int)(a.H / a.Hk), off = (int)(a.Tk - a.Tq), window = (int)a.window;
  const int pr = (int)(n % P.pairs);
  n /= P.pairs;
  w.hk = (int)(n % Hk);
  n /= Hk;
  w.b = (int)(n % a.B);
  const int u = P.units - 1 - (int)(n / a.B);  // the blocks that see most first
  w.len = seq_len(a, w.b);
  w.nst = (int)((a.sinks + TM - 1) / TM);
#pragma unroll
  for (int st = 0; st < 2; ++st) {
    Stage& x = w.s[st];
    x.h = P.by_heads ? w.hk * G + 2 * pr + st : w.hk * G + pr;
    x.i0 = (P.by_heads ? u : 2 * u + st) * TM;
    x.valid = x.i0 < a.Tq;
    x.p0 = x.i0 + off;
    x.p1 = min(x.i0 + TM, (int)a.Tq) - 1 + off;
    x.lo = max(0, x.p0 - window + 1) / TM;
    x.hi = x.valid && x.p0 < w.len ? min(x.p1, w.len - 1) / TM : -1;
  }
  w.lo = w.s[0].lo;
  w.nsink = min(w.nst, w.lo);
  w.count = w.s[0].hi < 0 ? 0 : w.nsink + max(w.s[0].hi, w.s[1].hi) - w.lo + 1;
  return w;
}

template <int DB>
struct Layout {
  static constexpr int SLOTS = DB == 2 ? 5 : 8;  // K and V tiles in flight
  static constexpr uint32_t TILE = DB * BLOCK_BYTES;
  static constexpr uint32_t Q = 0, KV = 2 * TILE, END = KV + SLOTS * TILE;
  static constexpr size_t SMEM = END + 1024;
};

struct Bars {
  uint64_t kv_full[8], kv_empty[8], q_full[2], q_empty[2], s_full[2], p_ready[2], o_full[2], fix, done;
};

// Bits lo..hi (inclusive, any integers) of the 32-bit word that holds columns 32w..32w+31.
GDNX_DEV uint32_t range_bits(int lo, int hi, int w) {
  lo = max(lo - 32 * w, 0);
  hi = min(hi - 32 * w, 31);
  return lo > hi ? 0u : (0xffffffffu >> (31 - hi)) & (0xffffffffu << lo);
}

GDNX_DEV void store8(void* y, int dtype, int64_t at, const float* x) {
  if (dtype == GDNX_F32) {
    float4* p = reinterpret_cast<float4*>(static_cast<float*>(y) + at);
    p[0] = make_float4(x[0], x[1], x[2], x[3]);
    p[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    uint4 u;
    if (dtype == GDNX_BF16) {
      u.x = pack2<true>(x[0], x[1]); u.y = pack2<true>(x[2], x[3]);
      u.z = pack2<true>(x[4], x[5]); u.w = pack2<true>(x[6], x[7]);
    } else {
      u.x = pack2<false>(x[0], x[1]); u.y = pack2<false>(x[2], x[3]);
      u.z = pack2<false>(x[4], x[5]); u.w = pack2<false>(x[6], x[7]);
    }
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(y) + at) = u;
  }
}

// The rows of one stage: scores to weights, tile after tile, and the output.
template <int DB, bool BF16>
GDNX_DEV void run_rows(const FwdParams& P, int st, uint32_t tmem, Bars& bar, volatile int* abort_flag) {
  const gdnx_attn_args& a = P.a;
  const int r = threadIdx.x % 128;
  const uint32_t lane_at = (uint32_t)(r / 32 * 32) << 16;
  const uint32_t tS = tmem + T_S + st * 128 + lane_at, tO = tmem + T_O + st * 128 + lane_at;
  const int window = (int)a.window, sinks = (int)a.sinks, D = (int)a.D;
  const float c2 = a.scale * kLog2e;
  uint32_t nS = 0, nO = 0;
  for (int64_t n = blockIdx.x; n < P.items; n += gridDim.x) {
    const Item w = make_item(P, n);
    const Stage& x = w.s[st];
    if (!x.valid) continue;
    float m = -INFINITY, l = 0.f;
    const int p = x.p0 + r;
    for (int i = 0; i < w.count; ++i) {
      const int kt = w.tile(i), j0 = kt * TM;
      if (!w.active(st, kt)) continue;
      if (!warp_wait(&bar.s_full[st], nS++ & 1, abort_flag)) return;
      tc::fence_after();
      float s[128];
      tmem_ld128(tS, s);
      // every row sees the whole tile?
      const bool whole = j0 + TM - 1 <= x.p0 && j0 + TM <= w.len &&
                         (x.p0 + TM - 1 - j0 < window || j0 + TM <= sinks);
      if (!whole) {
        const int hi = p < w.len ? min(p, w.len - 1) - j0 : -1;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t on = range_bits(p - window + 1 - j0, hi, q) | range_bits(0, min(sinks - 1 - j0, hi), q);
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (!(on >> e & 1)) s[32 * q + e] = -INFINITY;
        }
      }
      float mx[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) mx[q] = s[q];
#pragma unroll
      for (int e = 4; e < 128; e += 4)
#pragma unroll
        for (int q = 0; q < 4; ++q) mx[q] = fmaxf(mx[q], s[e + q]);
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      const bool grow = m != -INFINITY && (top - m) * c2 > 8.f;
      if (__any_sync(0xffffffffu, grow)) {
        const float corr = grow ? ex2((m - top) * c2) : 1.f;
        l *= corr;
        if (grow) m = top;
#pragma unroll
        for (int d = 0; d < 2 * DB; ++d) {
          float o[32];
          tc::tmem_ld32(tO + 32 * d, o);
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] *= corr;
          tc::tmem_st32(tO + 32 * d, o);
        }
      }
      if (m == -INFINITY) m = top;
      const float mc = m == -INFINITY ? 0.f : m * c2;
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t pk[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const float x0 = ex2(fmaf(s[64 * half + 2 * e], c2, -mc)), x1 = ex2(fmaf(s[64 * half + 2 * e + 1], c2, -mc));
          sum[0] += x0;
          sum[1] += x1;
          pk[e] = pack2<BF16>(x0, x1);
        }
        tmem_st32u(tS + 32 * half, pk);
      }
      l += sum[0] + sum[1];
      tc::fence_before();
      pipe::mbar_arrive(&bar.p_ready[st]);
    }
    if (x.hi >= 0) {
      if (!warp_wait(&bar.o_full[st], nO++ & 1, abort_flag)) return;
      tc::fence_after();
    }
    const int i = x.i0 + r;
    if (p >= w.len) l = 0.f;  // padding
    const float inv = l > 0.f ? 1.f / l : l != l ? l : 0.f;
    const int64_t at = w.b * a.y_sb + (int64_t)i * a.y_st + x.h * a.y_sh;
#pragma unroll
    for (int d = 0; d < 2 * DB; ++d) {
      float o[32];
      if (x.hi >= 0) tc::tmem_ld32(tO + 32 * d, o);
#pragma unroll
      for (int e = 0; e < 32; ++e) o[e] = l == 0.f ? 0.f : o[e] * inv;
      if (i < a.Tq) {
#pragma unroll
        for (int e = 0; e < 32; e += 8)
          if (32 * d + e < D) store8(a.y, a.y_dtype, at + 32 * d + e, o + e);
      }
    }
    if (a.lse && i < a.Tq)
      a.lse[((int64_t)w.b * a.H + x.h) * a.Tq + i] = l == 0.f ? -INFINITY : (m * c2 + log2f(l)) * kLn2;
  }
}

// One thread issues every product.  Per tile and stage: PV of the stage's previous tile (its
// weights are ready), then S of this one.
template <int DB, bool BF16>
GDNX_DEV void run_products(const FwdParams& P, uint32_t smem, uint32_t tmem, Bars& bar, volatile int* abort_flag) {
  using Lo = Layout<DB>;
  constexpr uint32_t ID_S = idesc16(BF16, 128, 128, false, false), ID_O = idesc16(BF16, 128, 64 * DB, false, true);
  uint32_t cnt = 0, nP[2] = {0, 0}, nQ[2] = {0, 0};
  bool pend[2] = {false, false}, first[2] = {false, false}, last[2] = {false, false};
  uint32_t v_of[2] = {0, 0}, old_v = 0;
  bool have_old = false;
  const auto flush = [&](int st) {  // the pending PV of a stage
    if (!pend[st]) return true;
    const uint32_t sl = v_of[st] % Lo::SLOTS;
    if (!pipe::wait_or_abort(&bar.kv_full[sl], v_of[st] / Lo::SLOTS & 1, abort_flag)) return false;
    if (!pipe::wait_or_abort(&bar.p_ready[st], nP[st]++ & 1, abort_flag)) return false;
    tc::fence_after();
    mma_px(tmem + T_O + st * 128, tmem + T_S + st * 128, smem + Lo::KV + sl * Lo::TILE, ID_O, !first[st]);
    if (last[st]) tc::commit(&bar.o_full[st]);
    pend[st] = false;
    return true;
  };
  for (int64_t n = blockIdx.x; n < P.items; n += gridDim.x) {
    const Item w = make_item(P, n);
    bool begun[2] = {false, false};
    for (int i = 0; i < w.count; ++i) {
      const int kt = w.tile(i);
      const uint32_t kc = cnt, ksl = kc % Lo::SLOTS;
      cnt += 2;
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        if (!flush(st)) return;
        if (st == 0 && !pipe::wait_or_abort(&bar.kv_full[ksl], kc / Lo::SLOTS & 1, abort_flag)) return;
        if (st == 1 && have_old) tc::commit(&bar.kv_empty[old_v % Lo::SLOTS]);
        if (!w.active(st, kt)) continue;
        if (!begun[st] && !pipe::wait_or_abort(&bar.q_full[st], nQ[st]++ & 1, abort_flag)) return;
        first[st] = !begun[st];
        begun[st] = true;
        last[st] = kt == w.s[st].hi;
        tc::fence_after();
        mma_abt<DB>(tmem + T_S + st * 128, smem + Lo::Q + st * Lo::TILE, smem + Lo::KV + ksl * Lo::TILE, ID_S);
        tc::commit(&bar.s_full[st]);
        if (last[st]) tc::commit(&bar.q_empty[st]);
        pend[st] = true;
        v_of[st] = kc + 1;
      }
      tc::commit(&bar.kv_empty[ksl]);
      old_v = kc + 1;
      have_old = true;
    }
  }
  if (!flush(0) || !flush(1)) return;
  if (have_old) tc::commit(&bar.kv_empty[old_v % Lo::SLOTS]);
}

// The warp that loads: K(0), Q, V(0), K(1), V(1), ... of each item.
template <int DB>
GDNX_DEV void run_loads(const FwdParams& P, uint8_t* base, uint32_t smem, Bars& bar, volatile int* abort_flag,
                        uint32_t& issued) {
  using Lo = Layout<DB>;
  const int lane = threadIdx.x % 32;
  uint32_t cnt = 0, nQ[2] = {0, 0}, nfix = 0;
  for (int64_t n = blockIdx.x; n < P.items; n += gridDim.x) {
    const Item w = make_item(P, n);
    for (int i = 0; i < w.count; ++i) {
      const int j0 = w.tile(i) * TM;
#pragma unroll
      for (int side = 0; side < 2; ++side, ++cnt) {
        const uint32_t sl = cnt % Lo::SLOTS, dst = smem + Lo::KV + sl * Lo::TILE;
        if (!warp_wait(&bar.kv_empty[sl], (cnt / Lo::SLOTS & 1) ^ 1, abort_flag)) return;
        // padding rows of V meet weights of 0, so they must not hold NaN
        const bool fix = side == 1 && w.len < P.a.Tk && j0 + TM > w.len;
        if (lane == 0) {
          const uint32_t mb = tc::smem_u32(fix ? &bar.fix : &bar.kv_full[sl]);
          pipe::expect_tx(mb, Lo::TILE);
          load_rows<DB>(dst, side ? P.v : P.k, j0, w.hk, w.b, mb);
        }
        if (fix) {
          if (!warp_wait(&bar.fix, nfix++ & 1, abort_flag)) return;
          for (int x = lane; x < (j0 + TM - w.len) * DB * 8; x += 32) {
            const int row = w.len - j0 + x / (DB * 8), c = x % (DB * 8);
            *reinterpret_cast<uint4*>(base + Lo::KV + sl * Lo::TILE + (c / 8) * BLOCK_BYTES + row * 128 + c % 8 * 16) =
                make_uint4(0, 0, 0, 0);
          }
          tc::fence_async_smem();
          __syncwarp();
          if (lane == 0) pipe::mbar_arrive(&bar.kv_full[sl]);
        }
        issued = cnt + 1;
        if (i == 0 && side == 0) {
#pragma unroll
          for (int st = 0; st < 2; ++st) {
            if (w.s[st].hi < 0) continue;
            if (!warp_wait(&bar.q_empty[st], (nQ[st]++ & 1) ^ 1, abort_flag)) return;
            if (lane == 0) {
              const uint32_t mb = tc::smem_u32(&bar.q_full[st]);
              pipe::expect_tx(mb, Lo::TILE);
              load_rows<DB>(smem + Lo::Q + st * Lo::TILE, P.q, w.s[st].i0, w.s[st].h, w.b, mb);
            }
          }
        }
      }
    }
  }
}

template <int DB, bool BF16>
__global__ void __launch_bounds__(NTHREADS, 1) attn_fwd_tc_kernel(const __grid_constant__ FwdParams P) {
  using Lo = Layout<DB>;
  extern __shared__ uint8_t raw[];
  __shared__ Bars bar;
  __shared__ uint32_t tmem_at;
  __shared__ int abort_flag;
  uint8_t* base = tc::align_smem(raw, 1024);
  const uint32_t smem = tc::smem_u32(base);
  const int warp = threadIdx.x / 32;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int i = 0; i < 8; ++i) {
      tc::mbar_init(&bar.kv_full[i], 1);
      tc::mbar_init(&bar.kv_empty[i], 1);
    }
    for (int s = 0; s < 2; ++s) {
      tc::mbar_init(&bar.q_full[s], 1);
      tc::mbar_init(&bar.q_empty[s], 1);
      tc::mbar_init(&bar.s_full[s], 1);
      tc::mbar_init(&bar.p_ready[s], 128);
      tc::mbar_init(&bar.o_full[s], 1);
    }
    tc::mbar_init(&bar.fix, 1);
    tc::mbar_init(&bar.done, 1);
  }
  if (warp == 8) tc::tmem_alloc(&tmem_at, 512);
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = tmem_at;
  // 384 threads start with 168 registers each: 2 x 128 x 208 + 128 x 88 is just that
  if (warp < 8) {
    regs_up<208>();
    run_rows<DB, BF16>(P, warp / 4, tmem, bar, &abort_flag);
  } else {
    regs_down<88>();
    uint32_t issued = 0;
    if (warp == 8 && threadIdx.x % 32 == 0) {
      run_products<DB, BF16>(P, smem, tmem, bar, &abort_flag);
      tc::commit(&bar.done);  // every product issued has ended before tensor memory is freed
      tc::mbar_wait(&bar.done, 0);
    }
    if (warp == 9) run_loads<DB>(P, base, smem, bar, &abort_flag, issued);
    if (warp == 9 && abort_flag && threadIdx.x % 32 == 0) {  // let the copies in flight land
      for (uint32_t c = issued > Lo::SLOTS ? issued - Lo::SLOTS : 0; c < issued; ++c)
        tc::mbar_wait(&bar.kv_full[c % Lo::SLOTS], c / Lo::SLOTS & 1, 1u << 16);
      for (uint32_t it = 0; it < (1u << 12); ++it) __nanosleep(100);
    }
  }
  __syncwarp();
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (warp == 8) tc::tmem_dealloc(tmem, 512);
  if (threadIdx.x == 0 && abort_flag && P.a.error) *P.a.error = GDNX_ETIMEOUT;
}

template <int DB, bool BF16>
gdnx_status launch(const FwdParams& P, int sms, cudaStream_t st) {
  const auto kernel = attn_fwd_tc_kernel<DB, BF16>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Layout<DB>::SMEM) != cudaSuccess) {
    cudaGetLastError();
    return GDNX_ELAUNCH;
  }
  const unsigned grid = (unsigned)(P.items < sms ? P.items : sms);
  kernel<<<grid, NTHREADS, Layout<DB>::SMEM, st>>>(P);
  return cudaGetLastError() == cudaSuccess ? GDNX_OK : GDNX_ELAUNCH;
}

}  // namespace

gdnx_status launch_attn_fwd_tc(const gdnx_attn_args& a, cudaStream_t st) {
  const int es = a.y_dtype == GDNX_F32 ? 4 : 2, vec = 16 / es;
  if (reinterpret_cast<uintptr_t>(a.y) % 16 || a.y_sb % vec || a.y_st % vec || a.y_sh % vec) return GDNX_EUNSUPPORTED;
  FwdParams P;
  if (!make_tile_map(a.q, a.B, a.Tq, a.H, a.D, &P.q) || !make_tile_map(a.k, a.B, a.Tk, a.Hk, a.D, &P.k) ||
      !make_tile_map(a.v, a.B, a.Tk, a.Hk, a.D, &P.v))
    return GDNX_EUNSUPPORTED;
  P.a = a;
  const int G = (int)(a.H / a.Hk), blocks = (int)((a.Tq + TM - 1) / TM);
  P.by_heads = G % 2 == 0;
  P.pairs = P.by_heads ? G / 2 : G;
  P.units = P.by_heads ? blocks : (blocks + 1) / 2;
  P.items = (int64_t)P.units * a.B * a.Hk * P.pairs;
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return GDNX_ELAUNCH;
  const bool bf16 = a.q.dtype == GDNX_BF16;
  if (a.D > 64) return bf16 ? launch<2, true>(P, sms, st) : launch<2, false>(P, sms, st);
  return bf16 ? launch<1, true>(P, sms, st) : launch<1, false>(P, sms, st);
}

}  // namespace gdnx
