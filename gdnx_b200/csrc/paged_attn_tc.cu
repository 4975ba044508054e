// Attention of a chunk of new tokens over a paged cache, on the tensor cores (16-bit caches).
//
// A persistent CTA walks its share of units (paged_attn.cuh): one or two blocks of 128 rows, a row being one query head
// of one token.  Two stages, each a warpgroup with one row a thread, take turns with the tensor cores:
//   S_s = Q_s K^T (tcgen05, fp32 in tensor memory) -> registers:  m = max, p = 2^(c (s - m)), l += p ->
//   P_s packed 16-bit over S_s's columns -> O_s += P_s V (tcgen05, P from tensor memory, V read with its rows as K).
// A unit of two blocks gives each stage one, and each tile of 128 keys serves both.  A unit of one block gives its
// tiles to the two stages in turn, whose outputs stage 0 joins at the end.  The maximum is lazy and the weights are
// rounded as in windowed attention's forward (attn_fwd.cu).
//
// Keys and values come by TMA, a box for each page and 64 dims.  Pages that are not there are not fetched; rows of V
// that no query may see (those, and rows behind the last token) may hold NaN and are cleared.
// Warps 0-3 and 4-7 are the stages' rows, warp 8 issues the products, warp 9 the loads, warp 11 clears rows of V.  Warp
// 10 walks the share ahead of them all and leaves what they need of each segment in a short queue, so that none waits
// for lengths and page tables where one segment ends and the next begins; then it clears padding rows of the output.
// Warps 10 and 11 may have nothing to do for as long as a whole segment, or the whole share, takes (38 s for 2^20 tokens of
// 80 heads): the bound of their waits counts from the last tile that the loads asked for.  All other waits last some tiles,
// or the walk over sequences without tokens.
//
// The shape: a small chunk is bound by the bytes of K and V, of which 192 KB are on their way or in use, a long one by the
// rows' chain (scores out of tensor memory, maximum, exponentials), which two stages cover in part.  Products are issued
// from uniform registers (from others a tile pair took 2750 cycles of issue, and 4096 tokens after 28,672 took 1186 us
// instead of 959), K, V and Q share one pool of slots, a unit's start and end weigh six tiles in the cut (one tile: 148 and
// 246 us instead of 114 and 189 for the second and third case below).
//
// Measured: 4096 tokens after 28,672, 16 heads over 2 of 128, f16: 990 us under sustained load (1041 TFLOP/s of visible
// pairs, 74 % of a large product's rate under the power cap), 876 us for the first 40 ms after a pause (1177 TFLOP/s, 71 %
// of a product's burst rate); tensor pipes busy 59 % of cycles; 64 sequences of up to 8192 tokens with 2 to 5 new ones
// each, 16 heads over 4, bf16, pages of 64: 112 us (4.8 TB/s of the copy's 6.5); 4 chunks of up to 512 beside 60 single
// tokens over as many: 175 to 179 us (DRAM 47 %: its chunks' products and its tokens' bytes come one after the other on an
// SM); 33 tokens after 467, 4 heads of 64, pages of 16: 18 us, of which the first key tile arrives after 7 (one load after
// the other: lengths, page table, keys) and its 64 boxes of 2 KB take 5 to ask for.
#include "paged_attn.cuh"

namespace gdnx {
namespace {

using Tc = Shape<128, TM, true>;

constexpr int NTHREADS = 384;
constexpr uint32_t T_S = 0, T_O = 256;  // tensor-memory columns: S_0, S_1, then O_0, O_1

struct TcParams : ChunkParams {
  CUtensorMap kv;  // {D, Hk * page, L * 2 * pages}
  CUtensorMap q;   // {D, H, tokens}, box {64, gs, tb}
  int tma_q;       // q's layout is one that TMA can address, and heads come in whole groups
  int vec_q, vec_y;  // rows are 16-byte aligned
};

constexpr int MOST_SLOTS = 14;

struct Bars {
  uint64_t full[MOST_SLOTS], empty[MOST_SLOTS], landed[MOST_SLOTS], s_full[2], p_ready[2][2], o_full[2], done, left, joined;
  uint64_t item_full[4], item_empty[4], job_full[4], job_empty[4];
};

// What a segment asks of its stages.
struct Seg {
  int n;        // tiles
  bool pair;    // each stage has its own block
  int lo1, hi0, hi1, nst;  // block 1's first window tile, the blocks' last tiles, and how many tiles hold sinks
  int last0, last1;        // the last tile of each stage, counted from the segment's first; -1: none
  int from, nsink, lo;     // the unit's tile that the segment begins with; its tiles' numbers (KeyTiles)
  GDNX_DEV Seg(const ChunkParams& P, const Walk<Tc>& w) {
    n = w.tb - w.ta;
    pair = w.x.blocks == 2;
    nst = (int)((P.a.sinks + TM - 1) / TM);
    from = w.ta;
    nsink = w.x.kt.nsink;
    lo = w.x.kt.lo;
    if (!pair) {
      last0 = (n - 1) & ~1;
      last1 = n > 1 ? ((n - 2) | 1) : -1;
      lo1 = hi0 = hi1 = 0;
      return;
    }
    const int p = w.s.first + w.x.t0 + P.tb;  // block 1's first position
    lo1 = max(0, p - (int)P.a.window + 1) / TM;
    hi0 = (p - 1) / TM;
    hi1 = (w.s.first + min(w.x.t0 + 2 * P.tb, w.s.count) - 1) / TM;
    const KeyTiles& k = w.x.kt;
    last0 = min(w.tb - 1, k.nsink + hi0 - k.lo) - w.ta;  // block 0 has every tile up to its last
    if (last0 < 0) last0 = -1;
    int e = w.tb - 1;  // block 1: but those between the sinks and its window
    if (e >= k.nsink && k.tile(e) < lo1 && k.tile(e) >= nst) e = nst - 1 >= k.lo ? k.nsink + nst - 1 - k.lo : k.nsink - 1;
    last1 = e < w.ta ? -1 : e - w.ta;
  }
  // The same in a form that the compiler knows to be uniform: what products are issued from.
  GDNX_DEV void make_uniform() {
    n = uniform(n);
    pair = uniform((int)pair);
    lo1 = uniform(lo1);
    hi0 = uniform(hi0);
    hi1 = uniform(hi1);
    last0 = uniform(last0);
    last1 = uniform(last1);
    from = uniform(from);
    nsink = uniform(nsink);
    lo = uniform(lo);
  }
  // Number of the segment's i-th tile.
  GDNX_DEV int tile(int i) const { return from + i < nsink ? from + i : lo + from + i - nsink; }
  GDNX_DEV int last(int st) const { return st ? last1 : last0; }
  // Does stage st work on the segment's i-th tile, number kt?
  GDNX_DEV bool on(int st, int i, int kt) const {
    if (!pair) return (i & 1) == st;
    return st ? kt <= hi1 && (kt >= lo1 || kt < nst) : kt <= hi0;
  }
};

// A segment in the queue; the last has no tiles.
struct Item {
  Seg g;
  int row, start, first, count, t0;  // the chunk, and the segment's first token in it
  int hk, head0, heads;
  int part, whole;  // rows of its part; or it is a whole unit
  int ids[32];      // page ids of its first tiles, a lane's each
  GDNX_DEV int len() const { return first + count; }
};
constexpr int ITEMS = 4, JOBS = 4, MASKS = 32;

// A tile of V to be cleared, once it has landed, of the rows from `end` on and of the pages that are not there; slot < 0:
// there are no more.
struct Job {
  int slot, end;
  uint32_t there;
};

struct Small {
  Bars bar;
  Item item[ITEMS];
  Job job[JOBS];
  Share share;
  long long sums[NTHREADS / 32];
  float2 stat[128];  // stage 1's maxima and sums
  uint8_t there[MASKS];  // pages of the tiles that are there, tile after tile
  uint32_t asked;        // changes with every tile that the loads ask for
  uint32_t tmem_at;
  int abort_flag;
};

// Shared memory is slots of one tile.  The first holds the block's Q, the second a second block's; the others, and the
// second where there is one block, are the ring that K and V go round, from its first slot in every segment.
template <int DB>
struct Layout {
  static constexpr int SLOTS = DB == 2 ? 7 : 14;
  static constexpr uint32_t TILE = DB * BLOCK_BYTES, SMALL = SLOTS * TILE;
  static constexpr size_t SMEM = SMALL + sizeof(Small);  // no static shared memory: the base is 1024-aligned
  static_assert(SMEM <= 227 * 1024, "shared memory of a CTA");
};

// A place of a segment's ring: its slot behind the ring's first, and whether an odd number of rounds lies behind it.
struct Place {
  int at;
  uint32_t odd;
};

// What a role knows of the slots: a bit for each, the parity of its next use in this segment.
template <int DB>
struct Ring {
  uint32_t bits = 0;
  int first = 1, size = 1;  // of the segment's ring
  GDNX_DEV void begin(bool pair) {
    first = pair ? 2 : 1;
    size = Layout<DB>::SLOTS - first;
  }
  // The place n (at most a round) behind p.
  GDNX_DEV Place behind(Place p, int n) const {
    p.at += n;
    if (p.at >= size) {
      p.at -= size;
      p.odd ^= 1;
    }
    return p;
  }
  GDNX_DEV int slot(Place p) const { return first + p.at; }
  GDNX_DEV uint32_t parity(Place p) const { return (bits >> (first + p.at) ^ p.odd) & 1; }
  GDNX_DEV uint32_t q_parity(int b) const { return bits >> b & 1; }
  // A segment of n places and these Qs is over.
  GDNX_DEV void end(int n, bool q0, bool q1) {
    // slots before n % size have had one use more than the others
    const uint32_t all = ((1u << size) - 1) << first, more = ((1u << n % size) - 1) << first;
    bits ^= (n / size & 1 ? all : 0) ^ more ^ (q0 ? 1 : 0) ^ (q1 ? 2 : 0);
  }
};

GDNX_DEV void tma_load_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t mbar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(mbar)
      : "memory");
}

// Weights of N columns: p = 2^(c2 s - mc), summed, packed 16-bit.  One pair in eight is taken on the FMA pipes (where
// masked scores give 2^-125: nothing beside a weight that counts).
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

// A row's running state: the maximum that O and l are scaled to, the sum, whether it saw a key, and whether it is a
// query at all (another may hold anything, and rescales nothing).
struct Row {
  float m, l;
  bool any, query;
};

// Takes a tile's maximum into the row, rescaling O where it lies too far above the old one.
// Returns what the tile's scores (times c2) are taken against.  A score that is NaN or +inf is the tile's maximum
// whatever its column, and from then on l and O or the maximum itself say so (ex2_poly alone would not).
template <int DB>
GDNX_DEV float take_max(Row& w, float top, float c2, uint32_t tO) {
  const bool grow = w.query && w.m != -INFINITY && !((top - w.m) * c2 <= 8.f);
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

// Bits of a word of 32 columns (word q of a tile) on pages that are not there: bit i of `gone` is the tile's i-th page.
GDNX_DEV uint32_t gone_bits(uint32_t gone, int page, int q) {
  if (page >= 32) return gone >> (32 * q / page) & 1 ? 0xffffffffu : 0u;
  return (gone >> (2 * q) & 1 ? 0xffffu : 0u) | (gone >> (2 * q + 1) & 1 ? 0xffff0000u : 0u);
}

// One stage's rows, one for each thread.
template <int DB, bool BF16>
GDNX_DEV void run_rows(const TcParams& P, Small& sm, uint32_t tmem) {
  const gdnx_paged_attn_args& a = P.a;
  const gdnx_cache& c = a.cache;
  Bars& bar = sm.bar;
  volatile int* abort_flag = &sm.abort_flag;
  const int r = threadIdx.x % 128, lane = r % 32, warp = threadIdx.x / 32, st = warp / 4;
  const uint32_t lane_at = (uint32_t)(r / 32 * 32) << 16;
  const uint32_t tS = tmem + T_S + st * 128 + lane_at, tO = tmem + T_O + st * 128 + lane_at;
  const int window = (int)a.window, sinks = (int)a.sinks, D = (int)c.D;
  const uint32_t all_pages = (1u << TM / c.page) - 1;
  const float c2 = a.scale * kLog2e;
  const int tok = r / P.gs, head = r % P.gs;  // this thread's row
  uint32_t nS = 0, nO = 0, nj = 0, tiles = 0;
  for (uint32_t k = 0;; ++k) {
    __syncwarp();  // the segment before is done with
    if (k > 0 && lane == 0) pipe::mbar_arrive(&bar.item_empty[(k - 1) % ITEMS]);
    if (!warp_wait(&bar.item_full[k % ITEMS], k / ITEMS & 1, abort_flag)) return;
    const Item& w = sm.item[k % ITEMS];
    const Seg g = w.g;
    if (g.n == 0) return;
    const int t0 = w.t0 + (g.pair && st ? P.tb : 0), t = t0 + tok, first = w.first, count = w.count;
    const bool valid = tok < P.tb && head < w.heads && t < count;
    const int p = valid ? first + t : -1;
    const bool some = __any_sync(0xffffffffu, valid);
    const int p0 = first + t0, p1 = first + min(t0 + P.tb, count) - 1;  // of the block
    Row row = {-INFINITY, 0.f, false, valid};
    bool worked = false;
    const uint32_t from = tiles;
    tiles += g.n;
    for (int i = 0; i < g.n; ++i) {
      const int kt = g.tile(i), j0 = kt * TM;
      if (!g.on(st, i, kt)) continue;
      worked = true;
      if (!warp_wait(&bar.s_full[st], nS++ & 1, abort_flag)) return;
      tc::fence_after();
      if (!some) {  // no row of the warp is a query: what its weights are does not matter
        pipe::mbar_arrive(&bar.p_ready[st][0]);
        pipe::mbar_arrive(&bar.p_ready[st][1]);
        continue;
      }
      // the tile's pages that are not there
      const uint32_t gone = ~*const_cast<volatile uint8_t*>(&sm.there[(from + i) % MASKS]) & all_pages;
      float2 sum = make_float2(0.f, 0.f);
      float s[128], t4[4];
      tmem_ld128(tS, s);
      // does every row see the whole tile?
      if (!gone && j0 + TM - 1 <= p0 && (p1 - j0 < window || j0 + TM <= sinks)) {
        row.any = true;
      } else {
        // visible columns: lo..hi, and those up to sk
        const int hi = p - j0, lo = p - window + 1 - j0, sk = min(sinks - 1 - j0, hi);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t on = (range_bits(lo, hi, q) | range_bits(0, sk, q)) & ~gone_bits(gone, c.page, q);
          row.any |= on != 0;
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (!(on >> e & 1)) s[32 * q + e] = -INFINITY;
        }
      }
#pragma unroll
      for (int f = 0; f < 4; ++f) t4[f] = s[f];
#pragma unroll
      for (int e = 4; e < 128; e += 4)
#pragma unroll
        for (int f = 0; f < 4; ++f) t4[f] = max_nan(t4[f], s[e + f]);
      const float mc = take_max<DB>(row, max_nan(max_nan(t4[0], t4[1]), max_nan(t4[2], t4[3])), c2, tO);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t pk[32];
        weights<BF16, 64>(s + 64 * half, c2, mc, sum, pk);
        tmem_st32u(tS + 32 * half, pk);
        tc::fence_before();
        pipe::mbar_arrive(&bar.p_ready[st][half]);
      }
      row.l += sum.x + sum.y;
    }
    if (worked) {
      if (!warp_wait(&bar.o_full[st], nO++ & 1, abort_flag)) return;
      tc::fence_after();
    }
    const bool both = !g.pair && g.n > 1;  // both stages worked on the one block
    if (!g.pair) {
      if (st == 1) {
        if (!both) continue;
        // stage 1 leaves its maximum and sum, and its output until stage 0 has read it
        sm.stat[r] = make_float2(row.m, row.any ? row.l : -1.f);
        tc::fence_before();
        pipe::mbar_arrive(&bar.left);
        if (!warp_wait(&bar.joined, nj++ & 1, abort_flag)) return;
        continue;
      }
    }
    float f0 = 1.f, f1 = 0.f;  // the stages' factors
    if (both) {
      if (!warp_wait(&bar.left, nj++ & 1, abort_flag)) return;
      tc::fence_after();
      const float2 x = sm.stat[r];
      const bool other = !(x.y < 0.f);  // (NaN: it saw something)
      // a maximum that is NaN stays one
      const float m = max_nan(row.m, x.x);
      f0 = row.m == -INFINITY ? 0.f : ex2((row.m - m) * c2);
      f1 = x.x == -INFINITY ? 0.f : ex2((x.x - m) * c2);
      row.m = m;
      row.l = row.l * f0 + (other ? x.y * f1 : 0.f);
      row.any |= other;
    }
    if (!some) {
      if (both) pipe::mbar_arrive(&bar.joined);
      continue;
    }
    // the maximum in the log2 domain and the sum as the join takes them: a maximum that is not finite comes of scores
    // that are not, and shows in the sum
    const float mc = row.m * c2;
    const bool finite = fabsf(mc) < INFINITY;
    const float top = !row.any ? -INFINITY : finite ? mc : kNoScore;
    const float l = !row.any || row.m == -INFINITY ? 0.f : finite ? row.l : NAN;
    const bool whole = w.whole;
    const float f = whole ? scale_of(top, l) : 1.f;
    const int64_t row_at = (int64_t)(w.start + t) * a.y_st + (int64_t)(w.head0 + head) * a.y_sh;
    const int64_t part = (int64_t)w.part + (g.pair ? st * 128 : 0) + r;
#pragma unroll 1
    for (int d = 0; d < 64 * DB; d += 64) {
      float o[64];
      if (worked) tmem_ld64(tO + d, o);
      else
#pragma unroll
        for (int e = 0; e < 64; ++e) o[e] = 0.f;
      if (both) {
        float x[64];
        tmem_ld64(tO + 128 + d, x);
#pragma unroll
        for (int e = 0; e < 64; ++e) o[e] = o[e] * f0 + x[e] * f1;
        if (d + 64 == 64 * DB) {  // stage 1's output may be written again
          tc::fence_before();
          pipe::mbar_arrive(&bar.joined);
        }
      }
      if (!whole) {
        if (valid)
#pragma unroll
          for (int e = 0; e < 64; e += 4)
            if (d + e < D) *reinterpret_cast<float4*>(P.part + part * D + d + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        continue;
      }
#pragma unroll
      for (int e = 0; e < 64; ++e) o[e] = f == 0.f ? 0.f : o[e] * f;
      if (a.y_dtype != GDNX_F32 && P.vec_y) {
        uint32_t u[32];
        pack_row(u, o, a.y_dtype);
        pack_row(u + 16, o + 32, a.y_dtype);
        uint16_t* dst = static_cast<uint16_t*>(a.y) + row_at + d;
        if (valid)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (d + e * 8 < D) *reinterpret_cast<uint4*>(dst + e * 8) = make_uint4(u[4 * e], u[4 * e + 1], u[4 * e + 2], u[4 * e + 3]);
      } else if (valid) {
#pragma unroll
        for (int e = 0; e < 64; ++e)
          if (d + e < D) st_from_f32(a.y, a.y_dtype, row_at + d + e, o[e]);
      }
    }
    if (valid && whole && a.lse) a.lse[(int64_t)(w.start + t) * a.H + w.head0 + head] = lse_of(top, l);
    if (valid && !whole) {
      P.stat[part * 2] = top;
      P.stat[part * 2 + 1] = l;
    }
  }
}

// The warp that issues the products: for each step and stage PV of the step before, once its weights are there, and S of
// this one, in one run.  In order, S of a step complete means PV of the one before complete.  A step is a tile of two
// blocks, or two tiles of one.
template <int DB, bool BF16, bool PAIR>
GDNX_DEV bool segment_products(const Seg& g, Ring<DB>& ring, uint32_t (&nP)[2], uint32_t smem, uint32_t tmem, Bars& bar,
                               volatile int* abort_flag) {
  using Lo = Layout<DB>;
  constexpr uint32_t ID_S = idesc16(BF16, 128, 128, false, false), ID_O = idesc16(BF16, 128, 64 * DB, false, true);
  const int steps = PAIR ? g.n : (g.n + 1) / 2;
  bool begun[2] = {false, false}, pend[2] = {false, false}, acc[2] = {false, false};
  ring.begin(PAIR);
  Place now = {0, 0}, before = {0, 0};  // where the step's tiles begin, and those of the one before
  for (int s = 0; s <= steps; ++s) {
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      const uint32_t tS = tmem + T_S + st * 128, tO = tmem + T_O + st * 128;
      const int i = PAIR ? s : 2 * s + st, was = PAIR ? s - 1 : i - 2;
      const bool there = i < g.n, on = there && (!PAIR || g.on(st, i, g.tile(i)));
      const Place kp = ring.behind(now, PAIR ? 0 : st);
      const Place vp = ring.behind(before, PAIR ? 1 : was == g.n - 1 && st == 0 ? 1 : 2 + st);
      const uint32_t ksl = ring.slot(kp), vsl = ring.slot(vp), k = smem + ksl * Lo::TILE, v = smem + vsl * Lo::TILE;
      if (on) {
        if (!begun[st] && (PAIR || st == 0) && !warp_wait(&bar.full[st], ring.q_parity(st), abort_flag)) return false;
        if (!warp_wait(&bar.full[ksl], ring.parity(kp), abort_flag)) return false;
      }
      if (pend[st]) {  // the first half's weights, then the second's
        if (!warp_wait(&bar.full[vsl], ring.parity(vp), abort_flag)) return false;
        if (!warp_wait(&bar.p_ready[st][0], nP[st] & 1, abort_flag)) return false;
        tc::fence_after();
        if (elect_one()) mma_px<4>(tO, tS, v, ID_O, acc[st]);
        __syncwarp();
        if (!warp_wait(&bar.p_ready[st][1], nP[st]++ & 1, abort_flag)) return false;
      }
      tc::fence_after();
      if (elect_one()) {
        if (pend[st]) {
          mma_px<4>(tO, tS + 32, v + 64 * 128, ID_O, true);
          if (was == g.last(st)) tc::commit(&bar.o_full[st]);
        }
        // V of the step before is done with: by both stages, or by the one whose it is
        if (PAIR ? s > 0 && st == 1 : pend[st]) tc::commit(&bar.empty[vsl]);
        if (on) {
          mma_abt<DB>(tS, smem + (PAIR ? st : 0) * Lo::TILE, k, ID_S);
          tc::commit(&bar.s_full[st]);
          // the last product that reads a Q
          if (i == (PAIR ? g.last(st) : g.n - 1)) tc::commit(&bar.empty[PAIR ? st : 0]);
        }
        if (there && (!PAIR || st == 1)) tc::commit(&bar.empty[ksl]);
      }
      __syncwarp();
      acc[st] = acc[st] || pend[st];
      begun[st] = begun[st] || on;
      pend[st] = on;  // (a stage's gap between the sinks' tile and its window ends nothing)
    }
    before = now;
    now = ring.behind(now, PAIR ? 2 : 4);
  }
  ring.end(2 * g.n, g.last0 >= 0, PAIR && g.last1 >= 0);
  return true;
}

template <int DB, bool BF16>
GDNX_DEV void run_products(Small& sm, uint32_t smem, uint32_t tmem) {
  Bars& bar = sm.bar;
  volatile int* abort_flag = &sm.abort_flag;
  uint32_t nP[2] = {0, 0};
  Ring<DB> ring;
  for (uint32_t k = 0;; ++k) {
    if (!warp_wait(&bar.item_full[k % ITEMS], k / ITEMS & 1, abort_flag)) return;
    Seg g = sm.item[k % ITEMS].g;
    g.make_uniform();
    if (g.n == 0) return;
    __syncwarp();
    if (threadIdx.x % 32 == 0) pipe::mbar_arrive(&bar.item_empty[k % ITEMS]);
    if (!(g.pair ? segment_products<DB, BF16, true>(g, ring, nP, smem, tmem, bar, abort_flag)
                 : segment_products<DB, BF16, false>(g, ring, nP, smem, tmem, bar, abort_flag)))
      return;
  }
}

// What the table says of tile kt's i-th page, -1 where it says nothing.  (Checked against the pool when it is used: the
// warp that reads ahead then does not wait for what it read.)
GDNX_DEV int table_entry(const gdnx_cache& c, int row, int len, int kt, int i) {
  const int64_t x = (int64_t)kt * (TM / c.page) + i;
  return x < c.width && x * c.page < len ? c.table[(int64_t)row * c.width + x] : -1;
}

// The warp that walks the share.
GDNX_DEV void run_schedule(const TcParams& P, Small& sm) {
  Bars& bar = sm.bar;
  const int lane = threadIdx.x % 32, npp = TM / P.a.cache.page;
  if (lane == 0 && P.cut) P.joint[blockIdx.x] = {0, 0, 0, 0, -1};
  Walk<Tc> w(P, sm.share);
  for (uint32_t k = 0;; ++k) {
    const bool more = w.next();
    if (!warp_wait(&bar.item_empty[k % ITEMS], (k / ITEMS & 1) ^ 1, &sm.abort_flag, &sm.asked)) return;
    Item& x = sm.item[k % ITEMS];
    if (more) {
      const Seg g(P, w);
      const int i = lane / npp;
      x.ids[lane] = i < g.n ? table_entry(P.a.cache, w.s.row, w.s.len(), g.tile(i), lane % npp) : -1;
      if (lane == 0) {
        x.g = g;
        x.row = w.s.row;
        x.start = w.s.start;
        x.first = w.s.first;
        x.count = w.s.count;
        x.t0 = w.x.t0;
        x.hk = w.hk();
        x.head0 = w.head0();
        x.heads = w.heads();
        x.part = (int)w.part();
        x.whole = w.whole();
        if (w.ends_cut()) P.joint[blockIdx.x] = w.joint(sm.share.per);
      }
    } else if (lane == 0) {
      x.g.n = 0;
    }
    __syncwarp();
    if (lane == 0) pipe::mbar_arrive(&bar.item_full[k % ITEMS]);
    if (!more) return;
  }
}

// A segment's places in order: f(tile, side (0: K, 1: V), place), until that is false.  Two blocks: K0 V0 K1 V1 ...  One
// block: two tiles at a time, K0 K1 V0 V1 K2 K3 ...; a last odd one K V.
template <int DB, typename F>
GDNX_DEV bool for_places(const Ring<DB>& ring, const Seg& g, F f) {
  Place at = {0, 0};
  for (int x = 0; x < 2 * g.n; ++x, at = ring.behind(at, 1)) {
    const bool two = g.pair || (g.n % 2 && x >= 2 * g.n - 2);
    if (!f(two ? x / 2 : x / 4 * 2 + x % 2, two ? x % 2 : x % 4 / 2, at)) return false;
  }
  return true;
}

// The warp that loads: a segment's first K, its Q, then the tiles in their places' order.
template <int DB>
GDNX_DEV void run_loads(const TcParams& P, Small& sm, uint8_t* base, uint32_t smem) {
  using Lo = Layout<DB>;
  const gdnx_cache& c = P.a.cache;
  Bars& bar = sm.bar;
  volatile int* abort_flag = &sm.abort_flag;
  const int lane = threadIdx.x % 32, page = c.page, npp = TM / page, ahead = 32 / npp, pg = lane / DB, d = lane % DB;
  const uint32_t box = (uint32_t)page * 128, all_pages = (1u << npp) - 1;
  uint32_t tiles = 0, jobs = 0;
  const auto post = [&](const Job& j) {  // to the warp that clears
    if (!warp_wait(&bar.job_empty[jobs % JOBS], (jobs / JOBS & 1) ^ 1, abort_flag)) return false;
    if (lane == 0) {
      sm.job[jobs % JOBS] = j;
      pipe::mbar_arrive(&bar.job_full[jobs % JOBS]);
    }
    __syncwarp();
    ++jobs;
    return true;
  };
  Ring<DB> ring;
  for (uint32_t k = 0;; ++k) {
    if (!warp_wait(&bar.item_full[k % ITEMS], k / ITEMS & 1, abort_flag)) return;
    const Item& w = sm.item[k % ITEMS];
    const Seg g = w.g;
    if (g.n == 0) break;
    const int hk = w.hk, row = w.row, len = w.len();
    ring.begin(g.pair);
    // page ids of tiles from .. from + ahead - 1, a lane's each, and of those behind them
    const auto read = [&](int first) {
      const int i = first + lane / npp;
      return i < g.n ? table_entry(c, row, len, g.tile(i), lane % npp) : -1;
    };
    const auto in_pool = [&](int id) { return id < c.pages ? id : -1; };
    int from = 0, ids = in_pool(w.ids[lane]), next = ahead < g.n ? read(ahead) : -1;
    const auto load = [&](int i, int side, Place at) {
      if (i >= from + ahead) {  // (a step's two tiles lie in one reading: their number is even, or one)
        from += ahead;
        ids = in_pool(next);
        if (from + ahead < g.n) next = read(from + ahead);
      }
      const int id = __shfl_sync(0xffffffffu, ids, ((i - from) * npp + pg) & 31);
      const uint32_t there = __ballot_sync(0xffffffffu, ids >= 0) >> ((i - from) * npp) & all_pages;
      const int sl = ring.slot(at), j0 = g.tile(i) * TM;
      if (!warp_wait(&bar.empty[sl], ring.parity(at) ^ 1, abort_flag)) return false;
      // rows of V that no query may see meet weights of 0, so they must not hold NaN
      const bool clear = side == 1 && (there != all_pages || j0 + TM > len);
      const uint32_t mb = tc::smem_u32(clear ? &bar.landed[sl] : &bar.full[sl]);
      if (lane == 0) {
        if (side == 0) {
          *const_cast<volatile uint8_t*>(&sm.there[(tiles + i) % MASKS]) = (uint8_t)there;
          *const_cast<volatile uint32_t*>(&sm.asked) = tiles + i + 1;
        }
        pipe::expect_tx(mb, __popc(there) * DB * box);
      }
      __syncwarp();
      if (pg < npp && id >= 0)
        tma_load_3d(smem + sl * Lo::TILE + d * BLOCK_BYTES + pg * box, &P.kv, d * 64, hk * page,
                    (int)((P.a.layer * 2 + side) * c.pages + id), mb);
      if (clear && !post({sl, len - j0, there})) return false;
      if (side == 0 && i == 0) {
        const gdnx_view& q = P.a.q;
        for (int b = 0; b < (g.pair ? 2 : 1); ++b) {
          if (g.last(b) < 0) continue;
          if (!warp_wait(&bar.empty[b], ring.q_parity(b) ^ 1, abort_flag)) return false;
          const uint32_t to = smem + b * Lo::TILE, qb = tc::smem_u32(&bar.full[b]);
          const int t0 = w.t0 + b * P.tb, row0 = w.start + t0;
          if (P.tma_q) {
            if (lane == 0) {
              pipe::expect_tx(qb, DB * (uint32_t)(P.gs * P.tb) * 128);
#pragma unroll
              for (int e = 0; e < DB; ++e) tma_load_3d(to + e * BLOCK_BYTES, &P.q, e * 64, w.head0, row0, qb);
            }
            __syncwarp();
          } else {
            const int heads = w.heads, n = min(P.tb, w.count - t0), D = (int)c.D;
            for (int y = lane; y < 128 * DB * 8; y += 32) {
              const int r = y / (DB * 8), e = y % (DB * 8), t = r / P.gs, h = r % P.gs;
              uint4 u = make_uint4(0, 0, 0, 0);
              if (t < n && h < heads && e * 8 < D) {
                const uint16_t* src = static_cast<const uint16_t*>(q.ptr) + (int64_t)(row0 + t) * q.st + (w.head0 + h) * q.sh + e * 8;
                if (P.vec_q) {
                  u = *reinterpret_cast<const uint4*>(src);
                } else {
                  u.x = src[0] | (uint32_t)src[1] << 16;
                  u.y = src[2] | (uint32_t)src[3] << 16;
                  u.z = src[4] | (uint32_t)src[5] << 16;
                  u.w = src[6] | (uint32_t)src[7] << 16;
                }
              }
              *reinterpret_cast<uint4*>(base + b * Lo::TILE + tc::sw128(r, e, 128)) = u;
            }
            tc::fence_async_smem();
            __syncwarp();
            if (lane == 0) pipe::mbar_arrive(&bar.full[b]);
          }
        }
      }
      return true;
    };
    if (!for_places(ring, g, load)) return;
    ring.end(2 * g.n, g.last0 >= 0, g.pair && g.last1 >= 0);
    tiles += g.n;
    __syncwarp();
    if (lane == 0) pipe::mbar_arrive(&bar.item_empty[k % ITEMS]);
  }
  post({-1, 0, 0});
}

// The warp that clears rows of V.
template <int DB>
GDNX_DEV void run_clears(const TcParams& P, Small& sm, uint8_t* base) {
  using Lo = Layout<DB>;
  Bars& bar = sm.bar;
  const int lane = threadIdx.x % 32, page = P.a.cache.page, e = lane % (8 * DB);
  uint32_t bits = 0;  // a bit for each slot: the parity of its next clearing
  for (uint32_t k = 0;; ++k) {
    if (!warp_wait(&bar.job_full[k % JOBS], k / JOBS & 1, &sm.abort_flag, &sm.asked)) return;
    const Job j = sm.job[k % JOBS];
    __syncwarp();
    if (lane == 0) pipe::mbar_arrive(&bar.job_empty[k % JOBS]);
    if (j.slot < 0) return;
    if (!warp_wait(&bar.landed[j.slot], bits >> j.slot & 1, &sm.abort_flag)) return;
    bits ^= 1u << j.slot;
    for (int row = lane / (8 * DB); row < TM; row += 32 / (8 * DB)) {
      if (row < j.end && (j.there >> (row / page) & 1)) continue;
      *reinterpret_cast<uint4*>(base + j.slot * Lo::TILE + (e / 8) * BLOCK_BYTES + row * 128 + e % 8 * 16) = make_uint4(0, 0, 0, 0);
    }
    tc::fence_async_smem();
    __syncwarp();
    if (lane == 0) pipe::mbar_arrive(&bar.full[j.slot]);
  }
}

template <int DB, bool BF16>
__global__ void __launch_bounds__(NTHREADS, 1) paged_attn_tc_kernel(const __grid_constant__ TcParams P) {
  using Lo = Layout<DB>;
  extern __shared__ __align__(1024) uint8_t base[];
  Small& sm = *reinterpret_cast<Small*>(base + Lo::SMALL);
  Bars& bar = sm.bar;
  volatile int* abort_flag = &sm.abort_flag;
  const uint32_t smem = uniform(tc::smem_u32(base));
  const int warp = uniform(threadIdx.x / 32);
  dependents_may_start();
  if (threadIdx.x == 288) {
    // what is read first is looked up (and its pages' addresses) under the set-up
    if (P.a.n > 0)
      for (const int32_t* p : {P.a.starts, P.a.first, P.a.rows, (const int32_t*)P.a.cache.table})
        asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&P.kv)) : "memory");
    if (P.tma_q) asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&P.q)) : "memory");
  }
  if (threadIdx.x == 0) {
    *abort_flag = smem % 1024 ? 1 : 0;  // swizzled tiles need an aligned base
    sm.asked = 0;
    for (int i = 0; i < Lo::SLOTS; ++i) {
      tc::mbar_init(&bar.full[i], 1);
      tc::mbar_init(&bar.empty[i], 1);
      tc::mbar_init(&bar.landed[i], 1);
    }
    for (int i = 0; i < 4; ++i) {
      tc::mbar_init(&bar.item_full[i], 1);
      tc::mbar_init(&bar.item_empty[i], 10);  // eight warps of rows, the products', the loads'
      tc::mbar_init(&bar.job_full[i], 1);
      tc::mbar_init(&bar.job_empty[i], 1);
    }
    for (int s = 0; s < 2; ++s) {
      tc::mbar_init(&bar.s_full[s], 1);
      tc::mbar_init(&bar.p_ready[s][0], 128);
      tc::mbar_init(&bar.p_ready[s][1], 128);
      tc::mbar_init(&bar.o_full[s], 1);
    }
    tc::mbar_init(&bar.done, 1);
    tc::mbar_init(&bar.left, 128);
    tc::mbar_init(&bar.joined, 128);
  }
  if (warp == 8) tc::tmem_alloc(&sm.tmem_at, 512);
  tc::fence_before();
  wait_for_earlier();
  find_share<Tc, NTHREADS>(P, sm.share, sm.sums);  // synchronises
  tc::fence_after();
  const uint32_t tmem = uniform(sm.tmem_at);
  if (smem % 1024) {  // never entered: the base is aligned
  } else if (warp < 8) {  // 384 threads start with 168 registers each: 2 x 128 x 216 + 128 x 72 is just that
    regs_up<216>();
    run_rows<DB, BF16>(P, sm, tmem);
  } else {
    regs_down<72>();
    if (warp == 8) {
      run_products<DB, BF16>(sm, smem, tmem);
      __syncwarp();
      if (elect_one()) tc::commit(&bar.done);  // every product issued has ended before tensor memory is freed
      tc::mbar_wait(&bar.done, 0);
    } else if (warp == 9) {
      run_loads<DB>(P, sm, base, smem);
      if (*abort_flag)  // let the copies in flight land
        for (uint32_t it = 0; it < (1u << 12); ++it) __nanosleep(100);
    } else if (warp == 10) {
      run_schedule(P, sm);
      write_padding(P, threadIdx.x % 32, 32);
    } else {
      run_clears<DB>(P, sm, base);
    }
  }
  __syncwarp();
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (warp == 8) tc::tmem_dealloc(tmem, 512);
  if (threadIdx.x == 0 && *abort_flag && P.a.error) *P.a.error = GDNX_ETIMEOUT;
}

template <int DB, bool BF16>
gdnx_status launch(const TcParams& P, cudaStream_t st) {
  const auto kernel = paged_attn_tc_kernel<DB, BF16>;
  constexpr int smem = (int)Layout<DB>::SMEM;
  static std::atomic<uint64_t> done;
  if (!allow_smem(kernel, smem, done)) return GDNX_ELAUNCH;
  if (launch_early(kernel, dim3((unsigned)P.grid), dim3(NTHREADS), smem, st, P) != cudaSuccess) return GDNX_ELAUNCH;
  return join_chunks<Tc>(P, st);
}

ChunkParams plan(const gdnx_paged_attn_args& a) { return plan_chunks<Tc>(a, sm_count()); }

}  // namespace

size_t paged_attn_tc_workspace_bytes(const gdnx_paged_attn_args& a) { return chunk_bytes(plan(a)); }

gdnx_status launch_paged_attn_tc(const gdnx_paged_attn_args& a, cudaStream_t st) {
  const gdnx_cache& c = a.cache;
  const EncodeTiledFn enc = encode_fn();
  if (!enc) return GDNX_ELAUNCH;
  if (c.L * 2 * c.pages > ((int64_t)1 << 31) - 1 || c.Hk * c.page * c.D * 2 >= ((int64_t)1 << 40)) return GDNX_EUNSUPPORTED;
  TcParams P;
  static_cast<ChunkParams&>(P) = plan(a);
  const CUtensorMapDataType type = c.dtype == GDNX_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const cuuint32_t es[3] = {1, 1, 1};
  {
    const cuuint64_t dims[3] = {(cuuint64_t)c.D, (cuuint64_t)(c.Hk * c.page), (cuuint64_t)(c.L * 2 * c.pages)};
    const cuuint64_t strides[2] = {(cuuint64_t)c.D * 2, (cuuint64_t)(c.Hk * c.page * c.D) * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)c.page, 1};
    if (enc(&P.kv, type, 3, c.kv, dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return GDNX_EINVAL;
  }
  P.vec_q = reinterpret_cast<uintptr_t>(a.q.ptr) % 16 == 0 && a.q.st % 8 == 0 && a.q.sh % 8 == 0;
  P.vec_y = reinterpret_cast<uintptr_t>(a.y) % 16 == 0 && a.y_st % 8 == 0 && a.y_sh % 8 == 0;
  // TMA takes 16-byte strides below 2^40, none of them 0 where there is more than one; a last group of fewer heads would
  // read the next key head's
  P.tma_q = P.vec_q && P.groups == 1 && (a.q.sh > 0 || a.H == 1) && (a.q.st > 0 || a.tokens == 1) &&
            a.q.st < ((int64_t)1 << 39) && a.q.sh < ((int64_t)1 << 39);
  if (P.tma_q) {
    const cuuint64_t one = (cuuint64_t)((c.D + 7) / 8 * 16);
    const cuuint64_t dims[3] = {(cuuint64_t)c.D, (cuuint64_t)a.H, (cuuint64_t)a.tokens};
    const cuuint64_t strides[2] = {a.H > 1 ? (cuuint64_t)a.q.sh * 2 : one, a.tokens > 1 ? (cuuint64_t)a.q.st * 2 : one};
    const cuuint32_t box[3] = {64, (cuuint32_t)P.gs, (cuuint32_t)P.tb};
    if (enc(&P.q, type, 3, const_cast<void*>(a.q.ptr), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      P.tma_q = 0;
  }
  if (c.D > 64) return c.dtype == GDNX_BF16 ? launch<2, true>(P, st) : launch<2, false>(P, st);
  return c.dtype == GDNX_BF16 ? launch<1, true>(P, st) : launch<1, false>(P, st);
}

}  // namespace gdnx
