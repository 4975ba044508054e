// Windowed attention, forward, on the tensor cores (16-bit inputs that TMA can address).
//
// A persistent CTA takes two blocks of 128 queries of one key head at a time ("stages":
// two query heads at the same positions where the key head serves an even number of them,
// else two consecutive blocks of one head) and walks the key tiles of 128 that either sees:
//   S_s = Q_s K^T (tcgen05, fp32 in tensor memory) -> registers, one query per thread:
//   m = max, p = 2^(c (s - m)), l += p -> P_s packed 16-bit over S_s's columns ->
//   O_s += P_s V (tcgen05, P from tensor memory, V read with its rows as K).
// While one stage's rows take exponentials, the tensor cores work for the other.
// Warps 0-3 and 4-7 are the stages' rows, warp 8 issues the products, warp 9 the TMA loads
// (Q of each stage, K and V through one ring).  A stage's PV(t) and S(t+1) are
// issued in order, so S(t+1) complete means PV(t) complete and O at rest.  P is handed over in
// halves of 64 keys: PV(t) starts under the second half's exponentials.
//
// The exponentials are what the tensor cores wait for: 128 x 128 of them a tile take the
// special-function units as long as its two products take the tensor cores.  So an eighth of
// them goes to the FMA pipes instead (ex2_poly), scaling and sums run two to an instruction.
//
// The maximum is lazy: P is taken against the last m that O was scaled to, and O is rescaled
// only when the new maximum is more than 8 above it in log2 (P stays below 2^8, exact in
// fp32 sums and without overflow in either 16-bit type); the result does not depend on m.
// P is rounded to the inputs' type, the error of which averages out over the keys like the
// inputs' own rounding; l sums it unrounded in fp32.
//
// Items that do not fill a last round of the SMs go to a second kernel where they are at most half a
// round, which starts as the first one's blocks leave SMs free: each block of queries has a CTA to itself, the
// two stages take its key tiles in turn and stage 0 joins the two outputs, in tensor memory both.  That
// is the whole work of a single short prompt (1024 tokens, 16 heads: 23 -> 17 us; 512 tokens after 7680,
// window 4096: 68 -> 44 us), and balances long ones (8192 after 8192: 6 % less).
//
// Measured: 8 x 4096 tokens, 16 heads over 4 of 128, window 1024, 4 sinks, bf16: 322 us in a sustained run, which the
// 1000 W cap holds at 1.69 GHz (749 TFLOP/s of visible pairs, 45 % of a large matrix product's rate), 286 us for a
// call by itself; 8192 tokens after 8192, window 4096: 287 us (973 TFLOP/s), 257 us by itself.  A pair of tiles
// takes the tensor cores 2048 cycles and lasts 3350: each stage's rows take longer than the other stage's products.
// Maxima that keep NaN cost 2 us of these.
#include "attn_tc.cuh"
#include "kernels.h"
#include "launch.cuh"

namespace gdnx {
namespace {

using namespace attn;

constexpr int NTHREADS = 384;  // a warpgroup for each stage's rows, and the warps that issue
constexpr uint32_t T_S = 0, T_O = 256;  // tensor-memory columns: S_0, S_1, then O_0, O_1

struct FwdParams {
  TileMap q, k, v, y, rest;
  gdnx_attn_args a;
  int64_t items;               // pairs of blocks for the first kernel
  int split;                   // pairs that the second kernel takes, block by block
  int tma_y;                   // 16-bit outputs leave through shared memory and TMA
  int pairs, units, by_heads;  // stage pairs of a key head; blocks (or block pairs) of queries
};

// A work item: its two stages' heads and rows, and the key tiles that either sees as one
// sequence.  (Scalars and selects: an array indexed by the stage would live in memory.)
struct Item {
  int b, hk, len, off, Tq, nst;  // nst: tiles that hold sinks
  int h0, i0, di;                // stage 1: head h0 + dh or rows i0 + di
  int dh, lo0, lo1, hi0, hi1;    // a stage's window tiles; hi < 0: sees nothing
  int nsink, count;
  GDNX_DEV int head(int st) const { return st ? h0 + dh : h0; }
  GDNX_DEV int row(int st) const { return st ? i0 + di : i0; }
  GDNX_DEV bool valid(int st) const { return row(st) < Tq; }
  GDNX_DEV int lo(int st) const { return st ? lo1 : lo0; }
  GDNX_DEV int hi(int st) const { return st ? hi1 : hi0; }
  GDNX_DEV int tile(int i) const { return i < nsink ? i : lo0 + i - nsink; }
  GDNX_DEV bool active(int st, int kt) const { return kt <= hi(st) && (kt >= lo(st) || kt < nst); }
};

GDNX_DEV Item make_item(const FwdParams& P, int64_t item) {
  const gdnx_attn_args& a = P.a;
  Item w;
  const int Hk = (int)a.Hk, G = (int)a.H / Hk, B = (int)a.B, window = (int)a.window;
  // the grid's items fit 31 bits
  unsigned n = (unsigned)item;
  const int pr = (int)(n % (unsigned)P.pairs);
  n /= (unsigned)P.pairs;
  w.hk = (int)(n % (unsigned)Hk);
  n /= (unsigned)Hk;
  w.b = (int)(n % (unsigned)B);
  const int u = P.units - 1 - (int)(n / (unsigned)B);  // the blocks that see most first
  w.len = uniform(seq_len(a, w.b));
  w.off = (int)(a.Tk - a.Tq);
  w.Tq = (int)a.Tq;
  w.nst = (int)((a.sinks + TM - 1) / TM);
  w.h0 = P.by_heads ? w.hk * G + 2 * pr : w.hk * G + pr;
  w.dh = P.by_heads ? 1 : 0;
  w.i0 = (P.by_heads ? u : 2 * u) * TM;
  w.di = P.by_heads ? 0 : TM;
  const auto span = [&](int row, int& lo, int& hi) {
    const int p0 = row + w.off, p1 = min(row + TM, w.Tq) - 1 + w.off;
    lo = max(0, p0 - window + 1) / TM;
    hi = row < w.Tq && p0 < w.len ? min(p1, w.len - 1) / TM : -1;
  };
  span(w.i0, w.lo0, w.hi0);
  span(w.i0 + w.di, w.lo1, w.hi1);
  w.nsink = min(w.nst, w.lo0);
  w.count = w.hi0 < 0 ? 0 : w.nsink + max(w.hi0, w.hi1) - w.lo0 + 1;
  return w;
}

// The second kernel's item: one block of the last pairs, whose key tiles the two stages take in turn
// (tile i by stage i % 2).
GDNX_DEV Item split_item(const FwdParams& P) {
  Item w = make_item(P, P.items + blockIdx.x / 2);
  if (blockIdx.x & 1) {
    w.h0 += w.dh;
    w.i0 += w.di;
    const int p0 = w.i0 + w.off, p1 = min(w.i0 + TM, w.Tq) - 1 + w.off;
    w.lo0 = max(0, p0 - (int)P.a.window + 1) / TM;
    w.hi0 = w.i0 < w.Tq && p0 < w.len ? min(p1, w.len - 1) / TM : -1;
  }
  w.dh = w.di = 0;
  w.lo1 = w.lo0;
  w.hi1 = w.hi0;
  w.nsink = min(w.nst, w.lo0);
  w.count = w.hi0 < 0 ? 0 : w.nsink + w.hi0 - w.lo0 + 1;
  return w;
}

struct Bars {
  uint64_t kv_full[8], kv_empty[8], q_full[2], q_empty[2], s_full[2], p_ready[2][2], o_full[2], fix, done, merge;
};

struct Small {
  Bars bar;
  uint32_t tmem_at;
  int abort_flag;
};

template <int DB>
struct Layout {
  static constexpr int SLOTS = DB == 2 ? 4 : 8;  // K and V tiles in flight
  static constexpr uint32_t TILE = DB * BLOCK_BYTES;
  // Q of both stages, the ring, and for each row warp 32 rows x 64 values on their way out
  static constexpr uint32_t Q = 0, KV = 2 * TILE, OUT = KV + SLOTS * TILE, SMALL = OUT + 8 * 4096;
  static constexpr size_t SMEM = SMALL + sizeof(Small);  // no static shared memory: the base is 1024-aligned
};

// Weights of N columns: p = 2^(c2 s - mc), summed, packed 16-bit.  One pair in eight is taken on
// the FMA pipes (where masked scores give 2^-125: nothing beside a weight that counts).
template <bool BF16, int N>
GDNX_DEV void weights(const float* s, float c2, float mc, float2& sum, uint32_t* pk) {
#pragma unroll
  for (int e = 0; e < N / 2; ++e) {
    const float2 x = fma2(make_float2(s[2 * e], s[2 * e + 1]), make_float2(c2, c2), make_float2(-mc, -mc));
    const float2 p = e % 8 == 3 ? ex2_poly<false>(x) : make_float2(ex2(x.x), ex2(x.y));
    sum = add2(sum, p);
    pk[e] = pack2<BF16>(p.x, p.y);
  }
}

// 64 values less what `u` holds of them.
GDNX_DEV void subtract_row(float* o, const uint32_t* u, int dtype) {
#pragma unroll
  for (int e = 0; e < 32; ++e) {
    float2 x;
    if (dtype == GDNX_BF16) x = make_float2(__uint_as_float(u[e] << 16), __uint_as_float(u[e] & 0xffff0000u));
    else x = __half22float2(*reinterpret_cast<const __half2*>(&u[e]));
    o[2 * e] -= x.x;
    o[2 * e + 1] -= x.y;
  }
}

// A row's running state: the maximum that O and l are scaled to, and the sum.
struct Row {
  float m, l;
};

// Takes a tile's maximum into the row, rescaling O where it lies too far above the old one.
// Returns what the tile's scores (times c2) are taken against.  A score that is NaN or +inf is the tile's maximum
// whatever its column, and from then on l and O or the maximum itself say so (ex2_poly alone would not).
template <int DB>
GDNX_DEV float take_max(Row& w, float top, float c2, uint32_t tO) {
  const bool grow = w.m != -INFINITY && !((top - w.m) * c2 <= 8.f);
  if (__any_sync(0xffffffffu, grow)) {
    const float corr = grow ? ex2((w.m - top) * c2) : 1.f;
    w.l *= corr;
    if (grow) w.m = top;
#pragma unroll 1
    for (int d = 0; d < 64 * DB; d += 16) {
      float o[16];
      tc::tmem_ld16(tO + d, o);
#pragma unroll
      for (int e = 0; e < 16; ++e) o[e] *= corr;
      tc::tmem_st16u(tO + d, reinterpret_cast<const uint32_t*>(o));
    }
  }
  if (w.m == -INFINITY) w.m = top;
  return w.m == -INFINITY ? 0.f : w.m * c2;
}

// 32 values of a row as 16-bit words.
GDNX_DEV void pack_row(uint32_t* u, const float* o, int dtype) {
  if (dtype == GDNX_BF16) {
#pragma unroll
    for (int e = 0; e < 16; ++e) u[e] = pack2<true>(o[2 * e], o[2 * e + 1]);
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e) u[e] = pack2<false>(o[2 * e], o[2 * e + 1]);
  }
}

// One stage's rows, one for each thread.
template <int DB, bool BF16, bool REST, bool SPLIT>
GDNX_DEV void run_rows(const FwdParams& P, uint8_t* base, uint32_t tmem, Bars& bar, volatile int* abort_flag) {
  using Lo = Layout<DB>;
  const gdnx_attn_args& a = P.a;
  const int r = threadIdx.x % 128, lane = r % 32, warp = threadIdx.x / 32, st = warp / 4;
  const uint32_t lane_at = (uint32_t)(r / 32 * 32) << 16;
  const uint32_t tS = tmem + T_S + st * 128 + lane_at, tO = tmem + T_O + st * 128 + lane_at;
  const int window = (int)a.window, sinks = (int)a.sinks, D = (int)a.D;
  const float c2 = a.scale * kLog2e;
  uint8_t* out = base + Lo::OUT + warp * 4096;
  uint32_t nS = 0, nO = 0;
  for (int64_t n = blockIdx.x; n < (SPLIT ? gridDim.x : P.items); n += gridDim.x) {
    const Item w = SPLIT ? split_item(P) : make_item(P, n);
    if (!w.valid(st)) continue;
    const int i0 = w.row(st), head = w.head(st), p0 = i0 + w.off, p = p0 + r;
    Row row = {-INFINITY, 0.f};
    for (int i = SPLIT ? st : 0; i < w.count; i += SPLIT ? 2 : 1) {
      const int kt = w.tile(i), j0 = kt * TM;
      if (!w.active(st, kt)) continue;
      if (!warp_wait(&bar.s_full[st], nS++ & 1, abort_flag)) return;
      tc::fence_after();
      float2 sum = make_float2(0.f, 0.f);
      // does every row see the whole tile?
      if (j0 + TM - 1 <= p0 && p0 + TM <= w.len && (p0 + TM - 1 - j0 < window || j0 + TM <= sinks)) {
        float s[128], t[4];
        tmem_ld128(tS, s);
#pragma unroll
        for (int f = 0; f < 4; ++f) t[f] = s[f];
#pragma unroll
        for (int e = 4; e < 128; e += 4)
#pragma unroll
          for (int f = 0; f < 4; ++f) t[f] = max_nan(t[f], s[e + f]);
        const float mc = take_max<DB>(row, max_nan(max_nan(t[0], t[1]), max_nan(t[2], t[3])), c2, tO);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t pk[32];
          weights<BF16, 64>(s + 64 * half, c2, mc, sum, pk);
          tmem_st32u(tS + 32 * half, pk);
          tc::fence_before();
          pipe::mbar_arrive(&bar.p_ready[st][half]);
        }
      } else {
        // chunk by chunk of 32 columns: what no row of the warp sees costs nothing
        // visible columns: lo..hi, and those up to sk
        const int hi = p < w.len ? p - j0 : -1, lo = p - window + 1 - j0, sk = min(sinks - 1 - j0, hi);
        uint32_t used = 0;
        float top = -INFINITY;
#pragma unroll 1
        for (int q = 0; q < 4; ++q) {
          const uint32_t on = range_bits(lo, hi, q) | range_bits(0, sk, q);
          if (!__any_sync(0xffffffffu, on)) continue;
          used |= 1u << q;
          float s[32];
          tc::tmem_ld32(tS + 32 * q, s);
#pragma unroll
          for (int e = 0; e < 32; ++e) top = max_nan(top, on >> e & 1 ? s[e] : -INFINITY);
        }
        const float mc = take_max<DB>(row, top, c2, tO);
#pragma unroll 1
        for (int q = 0; q < 4; ++q) {
          uint32_t pk[16] = {};
          if (used >> q & 1) {
            const uint32_t on = range_bits(lo, hi, q) | range_bits(0, sk, q);
            float s[32];
            tc::tmem_ld32(tS + 32 * q, s);
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!(on >> e & 1)) s[e] = -INFINITY;
            weights<BF16, 32>(s, c2, mc, sum, pk);
          }
          tc::tmem_st16u(tS + 16 * q, pk);  // over scores that have been read
          if (q % 2) {
            tc::fence_before();
            pipe::mbar_arrive(&bar.p_ready[st][q / 2]);
          }
        }
      }
      row.l += sum.x + sum.y;
    }
    if (SPLIT ? w.count > st : w.hi(st) >= 0) {
      if (!warp_wait(&bar.o_full[st], nO++ & 1, abort_flag)) return;
      tc::fence_after();
    }
    float f0 = 1.f, f1 = 0.f;  // SPLIT: the stages' factors
    if (SPLIT) {  // stage 1 leaves its maximum and sum in its staging rows, stage 0 reads both outputs
      float2* other = reinterpret_cast<float2*>(base + Lo::OUT + 4 * 4096) + r;
      if (st == 1) {
        *other = make_float2(row.m, row.l);
        pipe::mbar_arrive(&bar.merge);
        return;
      }
      if (!warp_wait(&bar.merge, 0, abort_flag)) return;
      if (w.count > 1) {
        if (!warp_wait(&bar.o_full[1], 0, abort_flag)) return;
        tc::fence_after();
        const float2 x = *other;
        const float m = fmaxf(row.m, x.x);
        f0 = row.m == -INFINITY ? 0.f : ex2((row.m - m) * c2);
        f1 = x.x == -INFINITY ? 0.f : ex2((x.x - m) * c2);
        row.m = m;
        row.l = row.l * f0 + x.y * f1;
      }
    }
    // every row but padding sees itself: a maximum that is not finite comes of scores that are not
    const float l = p >= w.len ? 0.f : fabsf(row.m * c2) < INFINITY ? row.l : NAN;
    const int i = i0 + r, row0 = i0 + r / 32 * 32;
    const float inv = l > 0.f ? 1.f / l : l != l ? l : 0.f;
#pragma unroll 1
    for (int d = 0; d < 64 * DB; d += 64) {
      float o[64];
      if (w.hi(st) >= 0) tmem_ld64(tO + d, o);
      if (SPLIT && w.count > 1) {
        float x[64];
        tmem_ld64(tO + 128 + d, x);
#pragma unroll
        for (int e = 0; e < 64; ++e) o[e] = o[e] * f0 + x[e] * f1;
      }
#pragma unroll
      for (int e = 0; e < 64; ++e) o[e] = l == 0.f ? 0.f : o[e] * inv;
      if (P.tma_y) {
        for (int rest = 0; rest < (REST ? 2 : 1); ++rest) {  // y, and what its rounding left
          uint32_t u[32];
          pack_row(u, o, a.y_dtype);
          pack_row(u + 16, o + 32, a.y_dtype);
          if (lane == 0) pipe::bulk_wait_read();  // the store before has read the staging rows
          __syncwarp();
#pragma unroll
          for (int e = 0; e < 8; ++e)
            *reinterpret_cast<uint4*>(out + tc::sw128(lane, e, 32)) =
                make_uint4(u[4 * e], u[4 * e + 1], u[4 * e + 2], u[4 * e + 3]);
          tc::fence_async_smem();
          __syncwarp();
          if (lane == 0 && row0 < a.Tq) {
            if (rest) tma_store_4d(&P.rest.map, d, P.rest.use_h ? head : 0, row0, P.rest.use_b ? w.b : 0, tc::smem_u32(out));
            else tma_store_4d(&P.y.map, d, P.y.use_h ? head : 0, row0, P.y.use_b ? w.b : 0, tc::smem_u32(out));
            pipe::bulk_commit();
          }
          if (REST) subtract_row(o, u, a.y_dtype);
        }
      } else if (i < a.Tq) {  // fp32
        float* dst = static_cast<float*>(a.y) + w.b * a.y_sb + (int64_t)i * a.y_st + head * a.y_sh + d;
#pragma unroll
        for (int e = 0; e < 64; e += 4)
          if (d + e < D) *reinterpret_cast<float4*>(dst + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
      }
    }
    if (a.lse && i < a.Tq)
      a.lse[((int64_t)w.b * a.H + head) * a.Tq + i] = l == 0.f ? -INFINITY : (row.m * c2 + log2f(l)) * kLn2;
  }
}

// The warp that issues the products: for each tile and stage PV of the tile before, once its
// weights are there, and S of this one, in one run.  In order, S(t+1) complete means PV(t)
// complete.  All waits but the one for the weights come first.
template <int DB, bool BF16>
GDNX_DEV void run_products(const FwdParams& P, uint32_t smem, uint32_t tmem, Bars& bar, volatile int* abort_flag) {
  using Lo = Layout<DB>;
  constexpr uint32_t ID_S = idesc16(BF16, 128, 128, false, false), ID_O = idesc16(BF16, 128, 64 * DB, false, true);
  uint32_t cnt = 0, nP[2] = {0, 0}, nQ[2] = {0, 0};
  for (int64_t n = blockIdx.x; n < P.items; n += gridDim.x) {
    const Item w = make_item(P, n);
    if (w.count == 0) continue;
    bool begun[2] = {false, false}, pend[2] = {false, false}, acc[2] = {false, false}, last[2] = {false, false};
    uint32_t old = 0;      // V's slot of the tile before
    for (int i = 0; i <= w.count; ++i) {
      const bool more = i < w.count;
      // stage 1 may see the sinks' tile and not the next one: its last tile ends it, not its first gap
      const int kt = more ? w.tile(i) : 1 << 29;
      const uint32_t ksl = cnt % Lo::SLOTS, k = smem + Lo::KV + ksl * Lo::TILE, v = smem + Lo::KV + old * Lo::TILE;
      if (more && !warp_wait(&bar.kv_full[ksl], cnt / Lo::SLOTS & 1, abort_flag)) return;
      if (i > 0 && !warp_wait(&bar.kv_full[old], (cnt - 1) / Lo::SLOTS & 1, abort_flag)) return;
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        const uint32_t tS = tmem + T_S + st * 128, tO = tmem + T_O + st * 128;
        const bool on = more && w.active(st, kt);
        if (on && !begun[st] && !warp_wait(&bar.q_full[st], nQ[st]++ & 1, abort_flag)) return;
        if (pend[st]) {  // the first half's weights, then the second's
          if (!warp_wait(&bar.p_ready[st][0], nP[st] & 1, abort_flag)) return;
          tc::fence_after();
          if (elect_one()) mma_px<4>(tO, tS, v, ID_O, acc[st]);
          __syncwarp();
          if (!warp_wait(&bar.p_ready[st][1], nP[st]++ & 1, abort_flag)) return;
        }
        tc::fence_after();
        if (elect_one()) {
          if (pend[st]) {
            mma_px<4>(tO, tS + 32, v + 64 * 128, ID_O, true);
            if (last[st]) tc::commit(&bar.o_full[st]);
          }
          if (st == 1 && i > 0) tc::commit(&bar.kv_empty[old]);
          if (on) {
            mma_abt<DB>(tS, smem + Lo::Q + st * Lo::TILE, k, ID_S);
            tc::commit(&bar.s_full[st]);
            if (kt == w.hi(st)) tc::commit(&bar.q_empty[st]);
          }
          if (st == 1 && more) tc::commit(&bar.kv_empty[ksl]);
        }
        __syncwarp();
        acc[st] = acc[st] || pend[st];
        begun[st] = begun[st] || on;
        pend[st] = on;
        last[st] = kt == w.hi(st);
      }
      old = (cnt + 1) % Lo::SLOTS;
      if (more) cnt += 2;
    }
  }
}

// The same for a split item: step t holds tile 2t of stage 0 and 2t + 1 of stage 1, places 4t and
// 4t + 1 of the ring their K, the next two their V.
template <int DB, bool BF16>
GDNX_DEV void split_products(const FwdParams& P, uint32_t smem, uint32_t tmem, Bars& bar, volatile int* abort_flag) {
  using Lo = Layout<DB>;
  constexpr uint32_t ID_S = idesc16(BF16, 128, 128, false, false), ID_O = idesc16(BF16, 128, 64 * DB, false, true);
  const Item w = split_item(P);
  if (w.count == 0 || !warp_wait(&bar.q_full[0], 0, abort_flag)) return;
  for (int t = 0; t <= (w.count + 1) / 2; ++t) {
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      const uint32_t tS = tmem + T_S + st * 128, tO = tmem + T_O + st * 128;
      const bool pv = t > 0 && 2 * t - 2 + st < w.count, on = 2 * t + st < w.count;
      const uint32_t kp = 4 * t + st, vp = kp - 2u, ksl = kp % Lo::SLOTS, vsl = vp % Lo::SLOTS;
      const uint32_t k = smem + Lo::KV + ksl * Lo::TILE, v = smem + Lo::KV + vsl * Lo::TILE;
      if (on && !warp_wait(&bar.kv_full[ksl], kp / Lo::SLOTS & 1, abort_flag)) return;
      if (pv) {
        if (!warp_wait(&bar.kv_full[vsl], vp / Lo::SLOTS & 1, abort_flag)) return;
        if (!warp_wait(&bar.p_ready[st][0], (t - 1) & 1, abort_flag)) return;
        tc::fence_after();
        if (elect_one()) mma_px<4>(tO, tS, v, ID_O, t > 1);
        __syncwarp();
        if (!warp_wait(&bar.p_ready[st][1], (t - 1) & 1, abort_flag)) return;
      }
      tc::fence_after();
      if (elect_one()) {
        if (pv) {
          mma_px<4>(tO, tS + 32, v + 64 * 128, ID_O, true);
          tc::commit(&bar.kv_empty[vsl]);
          if (!on) tc::commit(&bar.o_full[st]);
        }
        if (on) {
          mma_abt<DB>(tS, smem + Lo::Q, k, ID_S);
          tc::commit(&bar.s_full[st]);
          tc::commit(&bar.kv_empty[ksl]);
        }
      }
      __syncwarp();
    }
  }
}

// One tile of K or V (whole warp), padding rows of V to zero: they meet weights of 0, so they must not hold NaN.
template <int DB>
GDNX_DEV bool load_kv(const FwdParams& P, const Item& w, int side, int j0, uint32_t place, uint8_t* base, uint32_t smem,
                      Bars& bar, volatile int* abort_flag, uint32_t& nfix) {
  using Lo = Layout<DB>;
  const int lane = threadIdx.x % 32;
  const uint32_t sl = place % Lo::SLOTS, dst = smem + Lo::KV + sl * Lo::TILE;
  if (!warp_wait(&bar.kv_empty[sl], (place / Lo::SLOTS & 1) ^ 1, abort_flag)) return false;
  const bool fix = side == 1 && w.len < P.a.Tk && j0 + TM > w.len;
  if (lane == 0) {
    const uint32_t mb = tc::smem_u32(fix ? &bar.fix : &bar.kv_full[sl]);
    pipe::expect_tx(mb, Lo::TILE);
    load_rows<DB>(dst, side ? P.v : P.k, j0, w.hk, w.b, mb);
  }
  if (fix) {
    if (!warp_wait(&bar.fix, nfix++ & 1, abort_flag)) return false;
    for (int x = lane; x < (j0 + TM - w.len) * DB * 8; x += 32) {
      const int row = w.len - j0 + x / (DB * 8), c = x % (DB * 8);
      *reinterpret_cast<uint4*>(base + Lo::KV + sl * Lo::TILE + (c / 8) * BLOCK_BYTES + row * 128 + c % 8 * 16) =
          make_uint4(0, 0, 0, 0);
    }
    tc::fence_async_smem();
    __syncwarp();
    if (lane == 0) pipe::mbar_arrive(&bar.kv_full[sl]);
  }
  return true;
}

// Loads of a split item.
template <int DB>
GDNX_DEV void split_loads(const FwdParams& P, uint8_t* base, uint32_t smem, Bars& bar, volatile int* abort_flag,
                          uint32_t& issued) {
  using Lo = Layout<DB>;
  const Item w = split_item(P);
  uint32_t nfix = 0;
  for (int t = 0; 2 * t < w.count; ++t)
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int i = 2 * t + x % 2, side = x / 2;
      if (i >= w.count) continue;
      if (!load_kv<DB>(P, w, side, w.tile(i) * TM, 4 * t + x, base, smem, bar, abort_flag, nfix)) return;
      issued = 4 * t + x + 1;
      if (t == 0 && x == 0 && threadIdx.x % 32 == 0) {
        const uint32_t mb = tc::smem_u32(&bar.q_full[0]);
        pipe::expect_tx(mb, Lo::TILE);
        load_rows<DB>(smem + Lo::Q, P.q, w.i0, w.h0, w.b, mb);
      }
    }
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
        if (!load_kv<DB>(P, w, side, j0, cnt, base, smem, bar, abort_flag, nfix)) return;
        issued = cnt + 1;
        if (i == 0 && side == 0) {
#pragma unroll
          for (int st = 0; st < 2; ++st) {
            if (w.hi(st) < 0) continue;
            if (!warp_wait(&bar.q_empty[st], (nQ[st]++ & 1) ^ 1, abort_flag)) return;
            if (lane == 0) {
              const uint32_t mb = tc::smem_u32(&bar.q_full[st]);
              pipe::expect_tx(mb, Lo::TILE);
              load_rows<DB>(smem + Lo::Q + st * Lo::TILE, P.q, w.row(st), w.head(st), w.b, mb);
            }
          }
        }
      }
    }
  }
}

template <int DB, bool BF16, bool REST, bool SPLIT>
__global__ void __launch_bounds__(NTHREADS, 1) attn_fwd_tc_kernel(const __grid_constant__ FwdParams P) {
  using Lo = Layout<DB>;
  extern __shared__ __align__(1024) uint8_t base[];
  Small& sm = *reinterpret_cast<Small*>(base + Lo::SMALL);
  Bars& bar = sm.bar;
  volatile int* abort_flag = &sm.abort_flag;
  const uint32_t smem = uniform(tc::smem_u32(base));
  const int warp = uniform(threadIdx.x / 32);
  if (!SPLIT) dependents_may_start();
  if (threadIdx.x == 0) {
    *abort_flag = smem % 1024 ? 1 : 0;  // swizzled tiles need an aligned base
    for (int i = 0; i < 8; ++i) {
      tc::mbar_init(&bar.kv_full[i], 1);
      tc::mbar_init(&bar.kv_empty[i], 1);
    }
    for (int s = 0; s < 2; ++s) {
      tc::mbar_init(&bar.q_full[s], 1);
      tc::mbar_init(&bar.q_empty[s], 1);
      tc::mbar_init(&bar.s_full[s], 1);
      tc::mbar_init(&bar.p_ready[s][0], 128);
      tc::mbar_init(&bar.p_ready[s][1], 128);
      tc::mbar_init(&bar.o_full[s], 1);
    }
    tc::mbar_init(&bar.fix, 1);
    tc::mbar_init(&bar.done, 1);
    tc::mbar_init(&bar.merge, 128);
  }
  if (warp == 8) tc::tmem_alloc(&sm.tmem_at, 512);
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = uniform(sm.tmem_at);
  if (smem % 1024) {  // never entered: the base is aligned
  } else if (warp < 8) {  // 384 threads start with 168 registers each: 2 x 128 x 224 + 128 x 56 is just that
    regs_up<224>();
    run_rows<DB, BF16, REST, SPLIT>(P, base, tmem, bar, abort_flag);
    if (threadIdx.x % 32 == 0) pipe::bulk_wait_all();
  } else {
    regs_down<56>();
    if (warp == 8) {
      if (SPLIT) split_products<DB, BF16>(P, smem, tmem, bar, abort_flag);
      else run_products<DB, BF16>(P, smem, tmem, bar, abort_flag);
      __syncwarp();
      if (elect_one()) tc::commit(&bar.done);  // every product issued has ended before tensor memory is freed
      tc::mbar_wait(&bar.done, 0);
    } else if (warp == 9) {
      uint32_t issued = 0;
      if (SPLIT) split_loads<DB>(P, base, smem, bar, abort_flag, issued);
      else run_loads<DB>(P, base, smem, bar, abort_flag, issued);
      if (*abort_flag && threadIdx.x % 32 == 0) {  // let the copies in flight land
        for (uint32_t c = issued > Lo::SLOTS ? issued - Lo::SLOTS : 0; c < issued; ++c)
          tc::mbar_wait(&bar.kv_full[c % Lo::SLOTS], c / Lo::SLOTS & 1, 1u << 16);
        for (uint32_t it = 0; it < (1u << 12); ++it) __nanosleep(100);
      }
    }
  }
  __syncwarp();
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (warp == 8) tc::tmem_dealloc(tmem, 512);
  if (threadIdx.x == 0 && *abort_flag && P.a.error) *P.a.error = GDNX_ETIMEOUT;
  if (SPLIT) wait_for_earlier();  // what follows may rely on both kernels
}

template <int DB, bool BF16, bool REST>
gdnx_status launch(const FwdParams& P, int sms, cudaStream_t st) {
  const auto whole = attn_fwd_tc_kernel<DB, BF16, REST, false>, split = attn_fwd_tc_kernel<DB, BF16, REST, true>;
  constexpr int smem = (int)Layout<DB>::SMEM;
  static std::atomic<uint64_t> done_whole, done_split;
  if (!allow_smem(whole, smem, done_whole) || !allow_smem(split, smem, done_split)) return GDNX_ELAUNCH;
  if (P.items > 0) whole<<<(unsigned)(P.items < sms ? P.items : sms), NTHREADS, smem, st>>>(P);
  if (cudaGetLastError() != cudaSuccess) return GDNX_ELAUNCH;
  if (P.split > 0 && P.items > 0)  // starts as the first kernel's blocks leave SMs free
    return launch_early(split, dim3((unsigned)(2 * P.split)), dim3(NTHREADS), smem, st, P) == cudaSuccess ? GDNX_OK : GDNX_ELAUNCH;
  if (P.split > 0) split<<<(unsigned)(2 * P.split), NTHREADS, smem, st>>>(P);
  return cudaGetLastError() == cudaSuccess ? GDNX_OK : GDNX_ELAUNCH;
}

template <int DB, bool BF16>
gdnx_status launch(const FwdParams& P, int sms, cudaStream_t st) {
  return P.a.y_rest ? launch<DB, BF16, true>(P, sms, st) : launch<DB, BF16, false>(P, sms, st);
}

}  // namespace

gdnx_status launch_attn_fwd_tc(const gdnx_attn_args& a, cudaStream_t st) {
  const int es = a.y_dtype == GDNX_F32 ? 4 : 2, vec = 16 / es;
  if (reinterpret_cast<uintptr_t>(a.y) % 16 || a.y_sb % vec || a.y_st % vec || a.y_sh % vec) return GDNX_EUNSUPPORTED;
  FwdParams P;
  if (!make_tile_map(a.q, a.B, a.Tq, a.H, a.D, &P.q) || !make_tile_map(a.k, a.B, a.Tk, a.Hk, a.D, &P.k) ||
      !make_tile_map(a.v, a.B, a.Tk, a.Hk, a.D, &P.v))
    return GDNX_EUNSUPPORTED;
  P.tma_y = a.y_dtype != GDNX_F32;
  if (P.tma_y) {
    gdnx_view y = {a.y, a.y_dtype, (int32_t)a.D, a.y_sb, a.y_st, a.y_sh, 0, 0};
    if (!make_tile_map(y, a.B, a.Tq, a.H, a.D, &P.y, 32)) return GDNX_EUNSUPPORTED;
    if (a.y_rest) {
      y = {a.y_rest, a.y_dtype, (int32_t)a.D, a.Tq * a.H * a.D, a.H * a.D, a.D, 0, 0};
      if (!make_tile_map(y, a.B, a.Tq, a.H, a.D, &P.rest, 32)) return GDNX_EUNSUPPORTED;
    }
  }
  P.a = a;
  const int G = (int)(a.H / a.Hk), blocks = (int)((a.Tq + TM - 1) / TM);
  P.by_heads = G % 2 == 0;
  P.pairs = P.by_heads ? G / 2 : G;
  P.units = P.by_heads ? blocks : (blocks + 1) / 2;
  P.items = (int64_t)P.units * a.B * a.Hk * P.pairs;
  if (P.items >= ((int64_t)1 << 31)) return GDNX_EUNSUPPORTED;
  const int sms = sm_count();
  // Pairs that do not fill a last round of the SMs: where they are at most half of them, each block has
  // an SM to itself and its keys are split over the two stages (half a pair's time instead of a whole).
  const int rest = (int)(P.items % sms);
  P.split = 2 * rest <= sms ? rest : 0;
  P.items -= P.split;
  const bool bf16 = a.q.dtype == GDNX_BF16;
  if (a.D > 64) return bf16 ? launch<2, true>(P, sms, st) : launch<2, false>(P, sms, st);
  return bf16 ? launch<1, true>(P, sms, st) : launch<1, false>(P, sms, st);
}

}  // namespace gdnx
