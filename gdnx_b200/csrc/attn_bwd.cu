// Windowed attention, gradients, on the tensor cores (bfloat16 inputs that TMA can address).
//
// Two kernels recompute P from lse and write every gradient once, in a fixed order: seven
// products of a tile instead of five, against atomics (whose order would show in the bits)
// or dQ partials of T x W / 128 fp32 rows.
//   attn_dkv: 128 keys of a key head; over its query heads and the query tiles that see them
//     S^T = K Q^T, dP^T = V dY^T; P^T = exp(c S^T - lse), dS^T = P^T (dP^T - delta) packed
//     16-bit over the columns of S^T and dP^T; dV += P^T dY, dK += dS^T Q.
//   attn_dq: 128 queries of a head; over the key tiles that they see
//     S = Q K^T (two buffers), dP = dY V^T; dS over S's columns; dQ += dS K.
// Accumulators stay in tensor memory (fp32).  Warpgroups 0 to 3 own 32 of a tile's 128
// columns each (every lane's row in all), warp 16 issues the products, warp 17 the loads.
// In attn_dkv dV(t) and S(t+1) run while the rows form dS(t), dK(t) and dP(t+1) while they
// form P(t+1).
//
// A key tile that holds sinks is seen by every later query, far more than the others; its
// iterations (and all tiles' where there are few) are cut into parts that leave fp32
// partial sums, added in order when attn_dkv has ended (by the blocks of attn_dq).
//
// attn_dkv's blocks take their key tile whole, which leaves SMs idle at its end (256 tiles on 148
// SMs: two rounds).  So attn_dq starts there as they fall free and deals its items out by a
// counter: together they end evenly (2 x 4096 tokens, 16 heads over 4 of 128, window 1024: 8 % less of a whole
// step than one after the other).
//
// Measured at those sizes: a step with its forward takes 388 us in a sustained run (under the 1000 W cap), 352 to
// 358 us by itself.  Of the latter 24 us are delta's (y, what its rounding left, and dy: 4.1 TB/s), 147 us
// pass until dK, dV are done, 229 us in all.  An iteration of dK, dV takes 2850 cycles where its four products
// take 2048: the rows hold the products up between P and dS.
//
// Weights and dS are rounded to bf16 for the products, like the inputs themselves (the tensor cores take both factors
// in one type; it leaves dq, dk, dv 1.4 times as far from 64 bits as rounding the results alone would); dS of
// float16 inputs could leave float16's range, so those take the CUDA-core kernels (9.9 ms at the sizes above).
#include "attn_tc.cuh"
#include "kernels.h"
#include "launch.cuh"

namespace gdnx {
namespace {

using namespace attn;

constexpr int NTHREADS = 640;  // four warpgroups of rows, and the warps that issue
constexpr int SLOTS = 5;        // streamed tiles in flight
constexpr uint32_t STAT = TM * 4;  // bytes of one statistic of a tile's queries

struct BwdParams {
  TileMap q, k, v, dy;
  gdnx_attn_args a;
  void *dq, *dk, *dv;
  const float *lse2, *delta;  // [B,H,qpad]: minus lse in the log2 domain (-inf where padding), minus delta (0)
  float* part;                // partial dK, dV of cut tiles: [item][2][128][64 DB]
  int qtiles, ktiles, nst;    // nst: key tiles that hold sinks
  int seg_sink, seg;          // parts of such a tile and of the others
  unsigned queries;           // items of attn_dq
  unsigned* next;             // the next of them to take
};

struct Bars {
  uint64_t full[SLOTS], empty[SLOTS], res[2], res_empty[2], stat_full[2], stat_empty[2], s_full[2], dp_full, p_ready, ds_ready[2],
      dp_read, o_full, fix, done, item_full[2], item_empty[2];
};

template <int DB>
struct Layout {
  static constexpr uint32_t TILE = DB * BLOCK_BYTES;
  static constexpr uint32_t RES = 0, RING = 2 * TILE, STATS = RING + SLOTS * TILE, BARS = STATS + 4 * STAT,
                            END = BARS + 512;
  static constexpr size_t SMEM = END + 512;  // the base is 1024-aligned: there is no static shared memory
};

// D (+)= P X with P's columns in four quarters, each over the start of its 32 of 128 columns.
GDNX_DEV void mma_quarters(uint32_t d, uint32_t p, uint32_t x, uint32_t idesc, bool acc) {
  const uint64_t dx = tc::smem_desc(x, BLOCK_BYTES, 1024);
#pragma unroll
  for (int k = 0; k < 8; ++k)
    tc::mma_bf16_ts(d, p + 32 * (k / 2) + 8 * (k % 2), dx + k * (2048 >> 4), idesc, acc || k > 0);
}

// Rows r0.. of a landed tile to zero: padding rows meet weights of 0, so they must not hold NaN.
template <int DB>
GDNX_DEV void zero_rows(uint8_t* tile, int r0, int lane) {
  for (int x = lane; x < (TM - r0) * DB * 8; x += 32) {
    const int row = r0 + x / (DB * 8), c = x % (DB * 8);
    *reinterpret_cast<uint4*>(tile + (c / 8) * BLOCK_BYTES + row * 128 + c % 8 * 16) = make_uint4(0, 0, 0, 0);
  }
  tc::fence_async_smem();
  __syncwarp();
}

// A place in the ring: its slot, and how often the slot was used before.
struct Place {
  uint32_t sl, use;
};
// attn_dkv: Q and dY of its tiles in turn through all five slots.
GDNX_DEV Place keys_place(uint32_t c) { return {c % SLOTS, c / SLOTS}; }
// attn_dq: K through three slots and V through two.  K(t) stays until dQ(t), V(t) only until
// dP(t): in one ring V(t+2) would take K(t)'s slot, and its load would stand between dQ(t) and
// dP(t+2).
GDNX_DEV Place queries_place(uint32_t t, int side) {
  return side ? Place{3 + t % 2, t / 2} : Place{t % 3, t / 3};
}

// One streamed tile (whole warp): rows t0.. of head h, rows from `valid` on (in the tensor's own
// rows, below `rows`) to zero.
template <int DB>
GDNX_DEV bool stream_tile(uint8_t* base, uint32_t smem, Bars& bar, volatile int* abort_flag, Place at,
                          const TileMap& m, int t0, int64_t h, int64_t b, int valid, int64_t rows, uint32_t& nfix) {
  using Lo = Layout<DB>;
  const uint32_t sl = at.sl;
  const int lane = threadIdx.x % 32;
  if (!warp_wait(&bar.empty[sl], (at.use & 1) ^ 1, abort_flag)) return false;
  const bool fix = valid < rows && t0 + TM > valid;
  if (lane == 0) {
    const uint32_t mb = tc::smem_u32(fix ? &bar.fix : &bar.full[sl]);
    pipe::expect_tx(mb, Lo::TILE);
    load_rows<DB>(smem + Lo::RING + sl * Lo::TILE, m, t0, h, b, mb);
  }
  if (fix) {
    if (!warp_wait(&bar.fix, nfix++ & 1, abort_flag)) return false;
    zero_rows<DB>(base + Lo::RING + sl * Lo::TILE, max(0, valid - t0), lane);
    if (lane == 0) pipe::mbar_arrive(&bar.full[sl]);
  }
  return true;
}

GDNX_DEV void init_bars(Bars& bar) {
  for (int i = 0; i < SLOTS; ++i) {
    tc::mbar_init(&bar.full[i], 1);
    tc::mbar_init(&bar.empty[i], 1);
  }
  for (int i = 0; i < 2; ++i) {
    tc::mbar_init(&bar.res[i], 1);
    tc::mbar_init(&bar.res_empty[i], 1);
    tc::mbar_init(&bar.stat_full[i], 1);
    tc::mbar_init(&bar.stat_empty[i], 512);
    tc::mbar_init(&bar.s_full[i], 1);
    tc::mbar_init(&bar.ds_ready[i], 512);
    tc::mbar_init(&bar.item_full[i], 1);
    tc::mbar_init(&bar.item_empty[i], 512 + 1);
  }
  tc::mbar_init(&bar.dp_full, 1);
  tc::mbar_init(&bar.p_ready, 512);
  tc::mbar_init(&bar.dp_read, 512);
  tc::mbar_init(&bar.o_full, 1);
  tc::mbar_init(&bar.fix, 1);
  tc::mbar_init(&bar.done, 1);
}

// N accumulator values of one row, scaled, to 16-bit or fp32 memory (columns below D only).
template <bool F32, int N>
GDNX_DEV void store_row(void* dst, int64_t at, const float* o, float scale, int left) {
#pragma unroll
  for (int e = 0; e < N; e += 8) {
    if (e >= left) continue;
    if (F32) {
      float4* p = reinterpret_cast<float4*>(static_cast<float*>(dst) + at + e);
      p[0] = make_float4(o[e] * scale, o[e + 1] * scale, o[e + 2] * scale, o[e + 3] * scale);
      p[1] = make_float4(o[e + 4] * scale, o[e + 5] * scale, o[e + 6] * scale, o[e + 7] * scale);
    } else {
      uint4 u;
      u.x = tc::pack_bf16(o[e] * scale, o[e + 1] * scale);
      u.y = tc::pack_bf16(o[e + 2] * scale, o[e + 3] * scale);
      u.z = tc::pack_bf16(o[e + 4] * scale, o[e + 5] * scale);
      u.w = tc::pack_bf16(o[e + 6] * scale, o[e + 7] * scale);
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(dst) + at + e) = u;
    }
  }
}

// ------------------------------- dK and dV -----------------------------------

// One CTA's work: a key tile, and the part t0..t1-1 of its (query head, query tile) list.
struct KeyItem {
  int b, hk, kt, j0, len, seg, nseg, qlo, nq, t0, t1;
};

GDNX_DEV KeyItem key_item(const BwdParams& P) {
  const gdnx_attn_args& a = P.a;
  KeyItem w;
  const int G = (int)(a.H / a.Hk), off = (int)(a.Tk - a.Tq), bh = (int)(a.B * a.Hk);
  int n = blockIdx.x;
  const int sink_items = bh * P.nst * P.seg_sink;
  const bool sink = n < sink_items;
  if (!sink) n -= sink_items;
  w.nseg = sink ? P.seg_sink : P.seg;
  const int who = n % bh;  // key heads side by side: their queries' tiles are shared in L2
  n /= bh;
  w.seg = n % w.nseg;
  w.kt = n / w.nseg + (sink ? 0 : P.nst);
  w.b = who / (int)a.Hk;
  w.hk = who % (int)a.Hk;
  w.j0 = w.kt * TM;
  w.len = uniform(seq_len(a, w.b));
  const int rows = min((int)a.Tq, w.len - off);
  int hi = rows;
  if (w.j0 >= a.sinks) hi = (int)min((int64_t)rows, (int64_t)w.j0 + TM - 1 + a.window - off);
  w.qlo = max(w.j0 - off, 0) / TM;
  w.nq = w.j0 < w.len ? max(0, (hi + TM - 1) / TM - w.qlo) : 0;
  const int64_t all = (int64_t)G * w.nq;
  w.t0 = (int)(all * w.seg / w.nseg);
  w.t1 = (int)(all * (w.seg + 1) / w.nseg);
  return w;
}

constexpr uint32_t K_S = 0, K_DP = 128, K_DV = 256, K_DK = 384;  // tensor-memory columns

template <int DB>
GDNX_DEV void keys_rows(const BwdParams& P, const KeyItem& w, const uint8_t* base, uint32_t tmem, Bars& bar,
                        volatile int* abort_flag) {
  using Lo = Layout<DB>;
  const gdnx_attn_args& a = P.a;
  const int r = threadIdx.x % 128, part = threadIdx.x / 128;
  const uint32_t lane_at = (uint32_t)(r / 32 * 32) << 16;
  const uint32_t tS = tmem + lane_at + K_S + part * 32, tP = tmem + lane_at + K_DP + part * 32;
  const int off = (int)(a.Tk - a.Tq), window = (int)a.window, sinks = (int)a.sinks, len = w.len;
  const float c2 = a.scale * kLog2e;
  const int j = w.j0 + r;
  const int last = j >= len ? -1 : (j < sinks ? len - 1 : (int)min((int64_t)len - 1, (int64_t)j + window - 1));
  const bool none = window == 1 && sinks == 0;  // every query sees one key: dS is 0
  for (int t = w.t0; t < w.t1; ++t) {
    const uint32_t it = t - w.t0, ss = it & 1;
    const int p0 = (w.qlo + t % w.nq) * TM + off + part * 32;  // position of this quarter's first column
    const float* lse = reinterpret_cast<const float*>(base + Lo::STATS + ss * 2 * STAT) + part * 32;
    const float* del = lse + TM;
    if (!warp_wait(&bar.stat_full[ss], it / 2 & 1, abort_flag) || !warp_wait(&bar.s_full[0], it & 1, abort_flag)) return;
    tc::fence_after();
    float s[32];
    tc::tmem_ld32(tS, s);
    const bool whole = p0 >= w.j0 + TM - 1 && p0 + 32 <= len && w.j0 + TM <= len &&
                       (p0 + 31 - w.j0 < window || w.j0 + TM <= sinks);
    uint32_t on = 0xffffffffu;
    const float2 cc = make_float2(c2, c2);
#pragma unroll
    for (int e = 0; e < 32; e += 4) {  // every other pair on the FMA pipes; lse of NaN has to reach dV
      const float4 z = *reinterpret_cast<const float4*>(lse + e);
      const float2 x = fma2(make_float2(s[e], s[e + 1]), cc, make_float2(z.x, z.y));
      const float2 y = ex2_poly<true>(fma2(make_float2(s[e + 2], s[e + 3]), cc, make_float2(z.z, z.w)));
      s[e] = ex2(x.x);
      s[e + 1] = ex2(x.y);
      s[e + 2] = y.x;
      s[e + 3] = y.y;
    }
    if (!whole) {
      on = range_bits(j - p0, last - p0, 0);
#pragma unroll
      for (int e = 0; e < 32; ++e)
        if (!(on >> e & 1)) s[e] = 0.f;
      if (p0 == 0) on &= ~1u;  // position 0 sees one key
      if (none) on = 0;
    }
    uint32_t pk[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) pk[e] = tc::pack_bf16(s[2 * e], s[2 * e + 1]);
    tc::tmem_st16u(tS, pk);
    tc::fence_before();
    pipe::mbar_arrive(&bar.p_ready);
    if (!warp_wait(&bar.dp_full, it & 1, abort_flag)) return;
    tc::fence_after();
    float d[32];
    tc::tmem_ld32(tP, d);
#pragma unroll
    for (int e = 0; e < 32; e += 4) {
      const float4 z = *reinterpret_cast<const float4*>(del + e);
      const float2 x = mul2(make_float2(s[e], s[e + 1]), add2(make_float2(d[e], d[e + 1]), make_float2(z.x, z.y)));
      const float2 y = mul2(make_float2(s[e + 2], s[e + 3]), add2(make_float2(d[e + 2], d[e + 3]), make_float2(z.z, z.w)));
      s[e] = x.x;
      s[e + 1] = x.y;
      s[e + 2] = y.x;
      s[e + 3] = y.y;
    }
    if (!whole) {
#pragma unroll
      for (int e = 0; e < 32; ++e)
        if (!(on >> e & 1)) s[e] = 0.f;
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) pk[e] = tc::pack_bf16(s[2 * e], s[2 * e + 1]);
    tc::tmem_st16u(tP, pk);
    tc::fence_before();
    pipe::mbar_arrive(&bar.ds_ready[0]);
    pipe::mbar_arrive(&bar.stat_empty[ss]);
  }
  // warpgroups 0 and 1 write dV, 2 and 3 dK, half of the columns each
  if (w.t1 > w.t0) {
    if (!warp_wait(&bar.o_full, 0, abort_flag)) return;
    tc::fence_after();
  }
  const int side = part / 2;
  const uint32_t tO = tmem + lane_at + (side ? K_DK : K_DV);
  const float scale = side ? a.scale : 1.f;
#pragma unroll
  for (int d = 0; d < DB; ++d) {
    float o[32];
    const int c = 32 * (part % 2 * DB + d);
    if (w.t1 > w.t0) tc::tmem_ld32(tO + c, o);
    else
#pragma unroll
      for (int e = 0; e < 32; ++e) o[e] = 0.f;
    if (w.nseg > 1) {
      float* dst = P.part + ((int64_t)blockIdx.x * 2 + side) * TM * 64 * DB;
      store_row<true, 32>(dst, (int64_t)r * 64 * DB + c, o, scale, 32);
    } else if (j < a.Tk) {
      store_row<false, 32>(side ? P.dk : P.dv, (((int64_t)w.b * a.Tk + j) * a.Hk + w.hk) * a.D + c, o, scale, (int)a.D - c);
    }
  }
}

template <int DB>
GDNX_DEV void keys_products(const KeyItem& w, uint32_t smem, uint32_t tmem, Bars& bar, volatile int* abort_flag) {
  using Lo = Layout<DB>;
  constexpr uint32_t ID_S = idesc16(true, 128, 128, false, false), ID_O = idesc16(true, 128, 64 * DB, false, true);
  const int n = w.t1 - w.t0;
  const auto slot = [&](uint32_t c) { return smem + Lo::RING + c % SLOTS * Lo::TILE; };
  const auto landed = [&](uint32_t c) { return warp_wait(&bar.full[c % SLOTS], c / SLOTS & 1, abort_flag); };
  const auto scores = [&](int t) {
    if (!landed(2 * t)) return false;
    if (elect_one()) {
      mma_abt<DB>(tmem + K_S, smem + Lo::RES, slot(2 * t), ID_S);
      tc::commit(&bar.s_full[0]);
    }
    __syncwarp();
    return true;
  };
  const auto dprobs = [&](int t) {
    if (!landed(2 * t + 1)) return false;
    if (elect_one()) {
      mma_abt<DB>(tmem + K_DP, smem + Lo::RES + Lo::TILE, slot(2 * t + 1), ID_S);
      tc::commit(&bar.dp_full);
    }
    __syncwarp();
    return true;
  };
  if (n == 0) return;
  if (!warp_wait(&bar.res[0], 0, abort_flag) || !scores(0)) return;
  if (!warp_wait(&bar.res[1], 0, abort_flag) || !dprobs(0)) return;
  for (int t = 0; t < n; ++t) {
    if (!warp_wait(&bar.p_ready, t & 1, abort_flag)) return;
    tc::fence_after();
    if (elect_one()) {
      mma_quarters(tmem + K_DV, tmem + K_S, slot(2 * t + 1), ID_O, t > 0);
      tc::commit(&bar.empty[(2 * t + 1) % SLOTS]);
    }
    __syncwarp();
    if (t + 1 < n && !scores(t + 1)) return;
    if (!warp_wait(&bar.ds_ready[0], t & 1, abort_flag)) return;
    tc::fence_after();
    if (elect_one()) {
      mma_quarters(tmem + K_DK, tmem + K_DP, slot(2 * t), ID_O, t > 0);
      tc::commit(&bar.empty[(2 * t) % SLOTS]);
    }
    __syncwarp();
    if (t + 1 < n && !dprobs(t + 1)) return;
  }
  if (elect_one()) tc::commit(&bar.o_full);
}

template <int DB>
GDNX_DEV void keys_loads(const BwdParams& P, const KeyItem& w, uint8_t* base, uint32_t smem, Bars& bar,
                         volatile int* abort_flag) {
  using Lo = Layout<DB>;
  const gdnx_attn_args& a = P.a;
  const int lane = threadIdx.x % 32, G = (int)(a.H / a.Hk), off = (int)(a.Tk - a.Tq);
  const int rows = min((int)a.Tq, w.len - off);
  uint32_t nfix = 0;
  if (w.t1 == w.t0) return;
  if (lane == 0)
    for (int i = 0; i < 2; ++i) {
      const uint32_t mb = tc::smem_u32(&bar.res[i]);
      pipe::expect_tx(mb, Lo::TILE);
      load_rows<DB>(smem + Lo::RES + i * Lo::TILE, i ? P.v : P.k, w.j0, w.hk, w.b, mb);
    }
  for (int t = w.t0; t < w.t1; ++t) {
    const uint32_t it = t - w.t0, ss = it & 1;
    const int h = w.hk * G + t / w.nq, qt = w.qlo + t % w.nq;
    if (!stream_tile<DB>(base, smem, bar, abort_flag, keys_place(2 * it), P.q, qt * TM, h, w.b, rows, a.Tq, nfix)) return;
    if (!warp_wait(&bar.stat_empty[ss], (it / 2 & 1) ^ 1, abort_flag)) return;
    if (lane == 0) {
      const uint32_t mb = tc::smem_u32(&bar.stat_full[ss]), dst = smem + Lo::STATS + ss * 2 * STAT;
      const int64_t at = ((int64_t)w.b * a.H + h) * P.qtiles * TM + qt * TM;
      pipe::expect_tx(mb, 2 * STAT);
      pipe::bulk_load(dst, P.lse2 + at, STAT, mb);
      pipe::bulk_load(dst + STAT, P.delta + at, STAT, mb);
    }
    if (!stream_tile<DB>(base, smem, bar, abort_flag, keys_place(2 * it + 1), P.dy, qt * TM, h, w.b, rows, a.Tq, nfix)) return;
  }
}

// ---------------------------------- dQ ---------------------------------------

struct QueryItem {
  int b, h, hk, i0, p0, len;
  KeyTiles kt;
};

GDNX_DEV QueryItem query_item(const BwdParams& P, unsigned n) {
  const gdnx_attn_args& a = P.a;
  const int h = (int)(n % (unsigned)a.H);
  n /= (unsigned)a.H;
  const int b = (int)(n % (unsigned)a.B), qt = P.qtiles - 1 - (int)(n / (unsigned)a.B);  // those that see most first
  const int off = (int)(a.Tk - a.Tq), len = uniform(seq_len(a, b));
  return {b, h, h / (int)(a.H / a.Hk), qt * TM, qt * TM + off, len,
          KeyTiles(qt * TM + off, min(qt * TM + TM, (int)a.Tq) - 1 + off, len, (int)a.window, (int)a.sinks, TM)};
}

constexpr uint32_t Q_S = 0, Q_DP = 256, Q_DQ = 384;  // S has two buffers

// A persistent CTA takes item after item: tiles are counted through (T), so that the loads and
// the first products of an item run under the one before.  CTAs start as attn_dkv leaves SMs
// free, so items are dealt out by a counter: the loads take a number and pass it on through two
// places (an item is computed alike whoever takes it).
GDNX_DEV bool next_item(Bars& bar, const volatile unsigned* dealt, uint32_t k, unsigned& n, volatile int* abort_flag) {
  if (!warp_wait(&bar.item_full[k & 1], k / 2 & 1, abort_flag)) return false;
  n = dealt[k & 1];
  return true;
}

template <int DB>
GDNX_DEV void queries_rows(const BwdParams& P, uint32_t tmem, Bars& bar, const volatile unsigned* dealt,
                           volatile int* abort_flag) {
  const gdnx_attn_args& a = P.a;
  const int r = threadIdx.x % 128, part = threadIdx.x / 128;
  const uint32_t lane_at = (uint32_t)(r / 32 * 32) << 16;
  const uint32_t tS = tmem + lane_at + Q_S + part * 32, tP = tmem + lane_at + Q_DP + part * 32;
  const int window = (int)a.window, sinks = (int)a.sinks;
  const float c2 = a.scale * kLog2e;
  const float2 cc = make_float2(c2, c2);
  uint32_t T = 0, items = 0;
  for (uint32_t k = 0;; ++k) {
    unsigned n;
    if (!next_item(bar, dealt, k, n, abort_flag) || n >= P.queries) return;
    pipe::mbar_arrive(&bar.item_empty[k & 1]);
    const QueryItem w = query_item(P, n);
    const int len = w.len, p = w.p0 + r, i = w.i0 + r;
    const int64_t at = ((int64_t)w.b * a.H + w.h) * P.qtiles * TM + i;
    const float lse2 = __ldcg(P.lse2 + at), del = __ldcg(P.delta + at);
    const bool one = sees_one(p, window, sinks);
    for (int t = 0; t < w.kt.count; ++t, ++T) {
      const uint32_t buf = T & 1;
      const int j0 = w.kt.tile(t) * TM, c0 = j0 + part * 32;  // this quarter's first key
      if (!warp_wait(&bar.s_full[buf], T / 2 & 1, abort_flag)) return;
      tc::fence_after();
      float s[32];
      tc::tmem_ld32(tS + buf * 128, s);
      const bool whole = c0 + 31 <= w.p0 && w.p0 + TM <= len && (w.p0 + TM - 1 - c0 < window || c0 + 32 <= sinks);
#pragma unroll
      for (int e = 0; e < 32; e += 4) {  // every other pair on the FMA pipes
        const float2 x = fma2(make_float2(s[e], s[e + 1]), cc, make_float2(lse2, lse2));
        const float2 y = ex2_poly<false>(fma2(make_float2(s[e + 2], s[e + 3]), cc, make_float2(lse2, lse2)));  // NaN is in del
        s[e] = ex2(x.x);
        s[e + 1] = ex2(x.y);
        s[e + 2] = y.x;
        s[e + 3] = y.y;
      }
      if (!warp_wait(&bar.dp_full, T & 1, abort_flag)) return;
      tc::fence_after();
      float d[32];
      tc::tmem_ld32(tP, d);
      tc::fence_before();
      pipe::mbar_arrive(&bar.dp_read);
#pragma unroll
      for (int e = 0; e < 32; e += 2) {
        const float2 x = mul2(make_float2(s[e], s[e + 1]), add2(make_float2(d[e], d[e + 1]), make_float2(del, del)));
        s[e] = x.x;
        s[e + 1] = x.y;
      }
      if (!whole) {
        const int hi = p < len && !one ? p - c0 : -1;
        const uint32_t on = range_bits(p - window + 1 - c0, hi, 0) | range_bits(0, min(sinks - 1 - c0, hi), 0);
#pragma unroll
        for (int e = 0; e < 32; ++e)
          if (!(on >> e & 1)) s[e] = 0.f;
      }
      uint32_t pk[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) pk[e] = tc::pack_bf16(s[2 * e], s[2 * e + 1]);
      tc::tmem_st16u(tS + buf * 128, pk);
      tc::fence_before();
      pipe::mbar_arrive(&bar.ds_ready[buf]);
    }
    if (w.kt.count) {
      if (!warp_wait(&bar.o_full, items++ & 1, abort_flag)) return;
      tc::fence_after();
    }
#pragma unroll
    for (int d = 0; d < 16 * DB; d += 16) {  // each warpgroup takes a quarter of the columns
      float o[16];
      const int c = 16 * DB * part + d;
      if (w.kt.count) tc::tmem_ld16(tmem + lane_at + Q_DQ + c, o);
      else
#pragma unroll
        for (int e = 0; e < 16; ++e) o[e] = 0.f;
      if (i < a.Tq)
        store_row<false, 16>(P.dq, (((int64_t)w.b * a.Tq + i) * a.H + w.h) * a.D + c, o, a.scale, (int)a.D - c);
    }
  }
}

template <int DB>
GDNX_DEV void queries_products(const BwdParams& P, uint32_t smem, uint32_t tmem, Bars& bar,
                               const volatile unsigned* dealt, volatile int* abort_flag) {
  using Lo = Layout<DB>;
  constexpr uint32_t ID_S = idesc16(true, 128, 128, false, false), ID_O = idesc16(true, 128, 64 * DB, false, true);
  uint32_t T = 0, items = 0;  // tiles before this item; items with tiles
  const auto slot = [&](Place at) { return smem + Lo::RING + at.sl * Lo::TILE; };
  const auto landed = [&](Place at) { return warp_wait(&bar.full[at.sl], at.use & 1, abort_flag); };
  const auto scores = [&](int t, bool last) {
    const Place c = queries_place(T + t, 0);
    const uint32_t buf = (T + t) & 1;
    if (!landed(c)) return false;
    if (elect_one()) {
      mma_abt<DB>(tmem + Q_S + buf * 128, smem + Lo::RES, slot(c), ID_S);
      tc::commit(&bar.s_full[buf]);
      if (last) tc::commit(&bar.res_empty[0]);
    }
    __syncwarp();
    return true;
  };
  const auto dprobs = [&](int t, bool last) {
    const Place c = queries_place(T + t, 1);
    if (!landed(c)) return false;
    if (T + t > 0 && !warp_wait(&bar.dp_read, (T + t - 1) & 1, abort_flag)) return false;
    tc::fence_after();
    if (elect_one()) {
      mma_abt<DB>(tmem + Q_DP, smem + Lo::RES + Lo::TILE, slot(c), ID_S);
      tc::commit(&bar.dp_full);
      tc::commit(&bar.empty[c.sl]);
      if (last) tc::commit(&bar.res_empty[1]);
    }
    __syncwarp();
    return true;
  };
  for (uint32_t k = 0;; ++k) {
    unsigned it;
    if (!next_item(bar, dealt, k, it, abort_flag)) return;
    __syncwarp();  // read by every lane
    if (threadIdx.x % 32 == 0) pipe::mbar_arrive(&bar.item_empty[k & 1]);
    it = uniform(it);
    if (it >= P.queries) return;
    const int n = query_item(P, it).kt.count;
    if (n == 0) continue;
    if (!warp_wait(&bar.res[0], items & 1, abort_flag) || !scores(0, n == 1)) return;
    if (!warp_wait(&bar.res[1], items & 1, abort_flag) || !dprobs(0, n == 1)) return;
    ++items;
    if (n > 1 && !scores(1, n == 2)) return;
    for (int t = 0; t < n; ++t) {
      if (t + 1 < n && !dprobs(t + 1, t + 2 == n)) return;
      const Place c = queries_place(T + t, 0);
      const uint32_t buf = (T + t) & 1;
      if (!warp_wait(&bar.ds_ready[buf], (T + t) / 2 & 1, abort_flag)) return;
      tc::fence_after();
      if (elect_one()) {
        mma_quarters(tmem + Q_DQ, tmem + Q_S + buf * 128, slot(c), ID_O, t > 0);
        tc::commit(&bar.empty[c.sl]);
        if (t + 1 == n) tc::commit(&bar.o_full);
      }
      __syncwarp();
      if (t + 2 < n && !scores(t + 2, t + 3 == n)) return;
    }
    T += n;
  }
}

template <int DB>
GDNX_DEV void queries_loads(const BwdParams& P, uint8_t* base, uint32_t smem, Bars& bar, volatile unsigned* dealt,
                            volatile int* abort_flag) {
  using Lo = Layout<DB>;
  const gdnx_attn_args& a = P.a;
  uint32_t nfix = 0, T = 0, items = 0;
  for (uint32_t k = 0;; ++k) {
    unsigned n = 0;
    if (!warp_wait(&bar.item_empty[k & 1], (k / 2 & 1) ^ 1, abort_flag)) return;
    if (threadIdx.x % 32 == 0) {
      n = atomicAdd(P.next, 1u);
      dealt[k & 1] = n;
      pipe::mbar_arrive(&bar.item_full[k & 1]);
    }
    n = uniform(n);
    if (n >= P.queries) return;
    const QueryItem w = query_item(P, n);
    for (int t = 0; t < w.kt.count; ++t, ++T) {
      const int j0 = w.kt.tile(t) * TM;
#pragma unroll
      for (int side = 0; side < 2; ++side) {
        // K is also the right factor of dS K: its padding rows must not hold NaN
        if (!stream_tile<DB>(base, smem, bar, abort_flag, queries_place(T, side), side ? P.v : P.k, j0, w.hk, w.b,
                             side ? (int)a.Tk : w.len, a.Tk, nfix))
          return;
        if (t == 0) {  // Q beside the first K, dY beside the first V
          if (!warp_wait(&bar.res_empty[side], (items & 1) ^ 1, abort_flag)) return;
          if (threadIdx.x % 32 == 0) {
            const uint32_t mb = tc::smem_u32(&bar.res[side]);
            pipe::expect_tx(mb, Lo::TILE);
            load_rows<DB>(smem + Lo::RES + side * Lo::TILE, side ? P.dy : P.q, w.i0, w.h, w.b, mb);
          }
        }
      }
    }
    if (w.kt.count) ++items;
  }
}

// Sums of cut tiles' parts, in order: one thread for each (tile, key, four values).
template <int DB>
GDNX_DEV void join_parts(const BwdParams& P, int first, int tiles) {
  const gdnx_attn_args& a = P.a;
  const int bh = (int)(a.B * a.Hk), W = 64 * DB, nseg = first == 0 && P.nst > 0 ? P.seg_sink : P.seg;
  const int64_t item0 = first == 0 ? 0 : (int64_t)bh * P.nst * P.seg_sink;
  const int64_t all = (int64_t)tiles * bh * 2 * TM * (W / 4);
  for (int64_t x = (int64_t)blockIdx.x * NTHREADS + threadIdx.x; x < all; x += (int64_t)gridDim.x * NTHREADS) {
    const int d = (int)(x % (W / 4)) * 4, r = (int)(x / (W / 4) % TM), side = (int)(x / (W / 4 * TM) % 2);
    const int who = (int)(x / (2 * (W / 4) * TM) % bh), tile = (int)(x / ((int64_t)2 * (W / 4) * TM * bh));
    const int64_t j = (int64_t)(first + tile) * TM + r;
    if (j >= a.Tk || d >= a.D) continue;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int s = 0; s < nseg; ++s) {
      const float4 v = __ldcg(reinterpret_cast<const float4*>(
          P.part + (((item0 + ((int64_t)tile * nseg + s) * bh + who) * 2 + side) * TM + r) * W + d));
      sum = make_float4(sum.x + v.x, sum.y + v.y, sum.z + v.z, sum.w + v.w);
    }
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(side ? P.dk : P.dv) +
                              ((who / a.Hk * a.Tk + j) * a.Hk + who % a.Hk) * a.D + d) =
        make_uint2(tc::pack_bf16(sum.x, sum.y), tc::pack_bf16(sum.z, sum.w));
  }
}

// The frame of both kernels.  attn_dkv needs the statistics; attn_dq needs them too, which every CTA
// of attn_dkv has waited for before it lets attn_dq start.  attn_dq ends after attn_dkv, whose parts it
// joins.
template <int DB, bool KEYS>
__global__ void __launch_bounds__(NTHREADS, 1) attn_bwd_tc_kernel(const __grid_constant__ BwdParams P) {
  using Lo = Layout<DB>;
  extern __shared__ __align__(1024) uint8_t base[];
  Bars& bar = *reinterpret_cast<Bars*>(base + Lo::BARS);
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(base + Lo::BARS + 448);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(base + Lo::BARS + 452);
  volatile unsigned* dealt = reinterpret_cast<volatile unsigned*>(base + Lo::BARS + 456);
  static_assert(sizeof(Bars) <= 448, "barriers fit their place");
  const uint32_t smem = uniform(tc::smem_u32(base));
  const int warp = uniform(threadIdx.x / 32);
  if (threadIdx.x == 0) {
    *abort_flag = smem % 1024 ? 1 : 0;  // swizzled tiles need an aligned base
    init_bars(bar);
  }
  if (warp == 16) tc::tmem_alloc(tmem_at, 512);
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = uniform(*tmem_at);
  if (KEYS) {
    wait_for_earlier();
    dependents_may_start();
  }
  if (smem % 1024 == 0) {
    if (KEYS) {
      const KeyItem w = key_item(P);
      if (warp < 16) keys_rows<DB>(P, w, base, tmem, bar, abort_flag);
      else if (warp == 16) keys_products<DB>(w, smem, tmem, bar, abort_flag);
      else if (warp == 17) keys_loads<DB>(P, w, base, smem, bar, abort_flag);
    } else {
      if (warp < 16) queries_rows<DB>(P, tmem, bar, dealt, abort_flag);
      else if (warp == 16) queries_products<DB>(P, smem, tmem, bar, dealt, abort_flag);
      else if (warp == 17) queries_loads<DB>(P, base, smem, bar, dealt, abort_flag);
    }
  }
  if (warp == 16) {  // every product issued has ended
    __syncwarp();
    if (elect_one()) tc::commit(&bar.done);
    tc::mbar_wait(&bar.done, 0);
  }
  if (warp == 17 && *abort_flag)  // let the copies in flight land
    for (uint32_t it = 0; it < (1u << 12); ++it) __nanosleep(100);
  __syncwarp();
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (warp == 16) tc::tmem_dealloc(tmem, 512);
  if (threadIdx.x == 0 && *abort_flag && P.a.error) *P.a.error = GDNX_ETIMEOUT;
  if (!KEYS) {
    wait_for_earlier();
    if (P.nst > 0 && P.seg_sink > 1) join_parts<DB>(P, 0, P.nst);
    if (P.ktiles > P.nst && P.seg > 1) join_parts<DB>(P, P.nst, P.ktiles - P.nst);
  }
}

// Minus lse in the log2 domain and minus delta = sum_d dy y, padded to whole tiles of queries: eight lanes
// for each row.
__global__ void __launch_bounds__(256) attn_stats_kernel(const gdnx_attn_bwd_args g, float* lse2, float* delta,
                                                         unsigned* next, int qpad) {
  dependents_may_start();
  if (blockIdx.x == 0 && threadIdx.x == 0) *next = 0;
  const gdnx_attn_args& a = g.fwd;
  const int64_t n = (int64_t)blockIdx.x * 32 + threadIdx.x / 8;
  if (n >= a.B * a.H * qpad) return;  // whole groups of eight
  const int64_t h = n % a.H, i = n / a.H % qpad, b = n / a.H / qpad;  // heads side by side, as they lie in memory
  const bool on = i < a.Tq && i + a.Tk - a.Tq < seq_len(a, b);
  float s = 0.f;
  if (on) {
    const uint16_t* y = static_cast<const uint16_t*>(a.y) + b * a.y_sb + i * a.y_st + h * a.y_sh;
    const uint16_t* dy = static_cast<const uint16_t*>(g.dy.ptr) + b * g.dy.sb + i * g.dy.st + h * g.dy.sh;
#pragma unroll 2
    for (int d = threadIdx.x % 8 * 8; d < a.D; d += 64) {
      const uint4 u = *reinterpret_cast<const uint4*>(y + d), v = *reinterpret_cast<const uint4*>(dy + d);
      uint4 z = make_uint4(0, 0, 0, 0);
      if (a.y_rest) z = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.y_rest) + ((b * a.Tq + i) * a.H + h) * a.D + d);
      const uint32_t uw[4] = {u.x, u.y, u.z, u.w}, vw[4] = {v.x, v.y, v.z, v.w}, zw[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s = fmaf(__uint_as_float(uw[e] << 16) + __uint_as_float(zw[e] << 16), __uint_as_float(vw[e] << 16), s);
        s = fmaf(__uint_as_float(uw[e] & 0xffff0000u) + __uint_as_float(zw[e] & 0xffff0000u),
                 __uint_as_float(vw[e] & 0xffff0000u), s);
      }
    }
  }
  const uint32_t mask = 0xffu << (threadIdx.x % 32 / 8 * 8);
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) s += __shfl_xor_sync(mask, s, o);
  if (threadIdx.x % 8 == 0) {
    const int64_t at = (b * a.H + h) * qpad + i;
    lse2[at] = on ? -a.lse[(b * a.H + h) * a.Tq + i] * kLog2e : -INFINITY;
    delta[at] = -s;
  }
}

// How the key tiles' iterations are cut: a part is about a full SM's share of all of them, at
// least eight iterations; tiles that hold sinks are cut to the others' length, or to a quarter of an SM's
// share where that is longer: at most eight parts an SM are kept in fp32 (155 MB), however many sinks there are
// (16,384 tokens, 64 heads over 16 of 128, window 128, 2048 sinks: 104 MB and 5.1 ms of a training step; 2 GB and
// 6.6 ms cut to the others' length).
void plan(BwdParams& P) {
  const gdnx_attn_args& a = P.a;
  const int64_t G = a.H / a.Hk, bh = a.B * a.Hk;
  P.qtiles = (int)((a.Tq + TM - 1) / TM);
  P.ktiles = (int)((a.Tk + TM - 1) / TM);
  P.nst = (int)((a.sinks + TM - 1) / TM);
  P.queries = (unsigned)(P.qtiles * a.B * a.H);
  int64_t near = (a.window + TM - 1) / TM + 1;
  if (near > P.qtiles) near = P.qtiles;
  const int64_t it = G * near, it_sink = G * P.qtiles;
  const int64_t total = bh * (P.nst * it_sink + (P.ktiles - P.nst) * it);
  const int64_t sms = sm_count();
  int64_t share = (total + sms - 1) / sms;
  const int64_t quarter = (share + 3) / 4;
  if (share < 8) share = 8;
  if (share > it) share = it > 8 ? it : 8;
  const auto cut = [](int64_t n, int64_t share) {
    const int64_t s = (n + share - 1) / share;
    return (int)(s < 1 ? 1 : s > 64 ? 64 : s);
  };
  P.seg = cut(it, share);
  P.seg_sink = cut(it_sink, share > quarter ? share : quarter);
}

size_t stats_floats(const BwdParams& P) { return (size_t)P.a.B * P.a.H * P.qtiles * TM; }

int64_t items_of(const BwdParams& P) {
  return P.a.B * P.a.Hk * ((int64_t)P.nst * P.seg_sink + (int64_t)(P.ktiles - P.nst) * P.seg);
}

// Floats of partial sums: the cut tiles' items come first in the grid where only sinks are cut.
size_t part_floats(const BwdParams& P) {
  const size_t one = (size_t)2 * TM * (P.a.D > 64 ? 128 : 64);
  if (P.seg > 1) return (size_t)items_of(P) * one;
  return P.seg_sink > 1 ? (size_t)P.a.B * P.a.Hk * P.nst * P.seg_sink * one : 0;
}

template <int DB>
gdnx_status run(const gdnx_attn_bwd_args& g, BwdParams& P, cudaStream_t st) {
  const gdnx_attn_args& a = P.a;
  const auto keys = attn_bwd_tc_kernel<DB, true>;
  const auto queries = attn_bwd_tc_kernel<DB, false>;
  constexpr int smem = (int)Layout<DB>::SMEM;
  static std::atomic<uint64_t> done_keys, done_queries;
  if (!allow_smem(keys, smem, done_keys) || !allow_smem(queries, smem, done_queries)) return GDNX_ELAUNCH;
  const int64_t rows = (int64_t)stats_floats(P);
  attn_stats_kernel<<<(unsigned)((rows + 31) / 32), 256, 0, st>>>(
      g, const_cast<float*>(P.lse2), const_cast<float*>(P.delta), P.next, P.qtiles * TM);
  if (cudaGetLastError() != cudaSuccess ||
      launch_early(keys, dim3((unsigned)items_of(P)), dim3(NTHREADS), smem, st, P) != cudaSuccess)
    return GDNX_ELAUNCH;
  const int64_t joined = ((P.seg_sink > 1 ? P.nst : 0) + (P.seg > 1 ? P.ktiles - P.nst : 0)) * a.B * a.Hk;
  const int64_t work = joined * 8 > P.queries ? joined * 8 : P.queries;  // a block for some rows of a joined tile
  const unsigned sms = (unsigned)sm_count();
  if (launch_early(queries, dim3(work < sms ? (unsigned)work : sms), dim3(NTHREADS), smem, st, P) != cudaSuccess)
    return GDNX_ELAUNCH;
  return GDNX_OK;
}

}  // namespace

size_t attn_bwd_tc_workspace_bytes(const gdnx_attn_args& a) {
  BwdParams P;
  P.a = a;
  plan(P);
  return (2 * stats_floats(P) + 4 + part_floats(P)) * sizeof(float);
}

gdnx_status launch_attn_bwd_tc(const gdnx_attn_bwd_args& g, cudaStream_t st) {
  const gdnx_attn_args& a = g.fwd;
  const auto wide = [](const void* p, int64_t b, int64_t t, int64_t h) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && b % 8 == 0 && t % 8 == 0 && h % 8 == 0;
  };
  if (a.q.dtype != GDNX_BF16 || a.y_dtype != GDNX_BF16 || !wide(a.y, a.y_sb, a.y_st, a.y_sh) ||
      !wide(g.dy.ptr, g.dy.sb, g.dy.st, g.dy.sh) || !wide(g.dq, 0, 0, 0) || !wide(g.dk, 0, 0, 0) ||
      !wide(g.dv, 0, 0, 0) || !wide(g.workspace, 0, 0, 0) ||
      !wide(a.y_rest, 0, 0, 0))
    return GDNX_EUNSUPPORTED;
  BwdParams P;
  if (!make_tile_map(a.q, a.B, a.Tq, a.H, a.D, &P.q) || !make_tile_map(a.k, a.B, a.Tk, a.Hk, a.D, &P.k) ||
      !make_tile_map(a.v, a.B, a.Tk, a.Hk, a.D, &P.v) || !make_tile_map(g.dy, a.B, a.Tq, a.H, a.D, &P.dy))
    return GDNX_EUNSUPPORTED;
  P.a = a;
  P.dq = g.dq;
  P.dk = g.dk;
  P.dv = g.dv;
  plan(P);
  float* ws = static_cast<float*>(g.workspace);
  P.lse2 = ws;
  P.delta = ws + stats_floats(P);
  P.next = reinterpret_cast<unsigned*>(ws + 2 * stats_floats(P));  // 16 bytes
  P.part = ws + 2 * stats_floats(P) + 4;
  return a.D > 64 ? run<2>(g, P, st) : run<1>(g, P, st);
}

}  // namespace gdnx
