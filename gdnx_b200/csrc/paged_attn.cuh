// What the kernels of chunk attention over a paged cache share: the work of a call as one row of weights, cut evenly
// over the CTAs, and the kernel that joins the parts of a cut unit.
//
// A block of ROWS rows holds the queries of one key head (a group of at most ROWS of its query heads) at `tb` tokens in
// sequence: row r is token r / gs, head r % gs.  So a chunk of a few tokens fills a tile with its heads, and keys and
// values are read once for all of them.  A unit is one block (PAIR: two, where the chunk has them) of one sequence;
// its tiles of KEYS keys have a weight each, its start and end another.  Units are ordered by
// sequence, head group, tokens.  Every CTA finds its share of the row from the lengths by itself, without a word to
// the host: mixed batches of whole chunks and single tokens leave no SM waiting, and one token over a long cache has
// all of them.  Units of up to SMALL in weight stay whole: a few more tiles in a row take less time than a join.
#pragma once

#include "attn_tc.cuh"
#include "kernels.h"
#include "launch.cuh"

namespace gdnx {
namespace {  // one copy for each kernel file

using namespace attn;

// A unit that was cut: its parts lie in CTAs c0..c1.  c1 < 0: none.
struct Joint {
  int seq, hg, u, c0, c1;
};

struct ChunkParams {
  gdnx_paged_attn_args a;
  float* part;   // [grid][2][rows][D] unnormalised outputs of a CTA's first and last unit
  float* stat;   // [grid][2][rows][2] maximum (log2 domain) and sum
  Joint* joint;  // [grid] the cut unit that ends in a CTA
  int grid;
  int groups, gs, tb;  // groups of a key head's queries, heads of a group, tokens of a block
  int rows;            // rows of a part
  int cut;             // some unit may be cut
  int vec_join;        // four values of y lie aligned
};

// The new tokens of one sequence: rows start .. start + count - 1 of the packed tensors, at positions first ...
struct Chunk {
  int row, first, start, count;
  GDNX_DEV int len() const { return first + count; }
};

GDNX_DEV Chunk make_chunk(const gdnx_paged_attn_args& a, int64_t i) {
  const gdnx_cache& c = a.cache;
  const int total = (int)a.tokens, most = (int)(c.width * c.page);
  Chunk s;
  s.start = min(max(a.starts[i], 0), total);
  s.count = min(max(a.starts[i + 1], s.start), total) - s.start;
  s.first = a.first[i];
  s.row = a.rows[i];
  // a sequence that is no slot's, or ends beyond it, has no tokens (its rows are padding)
  if (s.row < 0 || s.row >= c.slots || s.first < 0 || s.first > most - s.count) s.count = 0;
  return s;
}

template <int ROWS_, int KEYS_, bool PAIR_>
struct Shape {
  static constexpr int ROWS = ROWS_, KEYS = KEYS_;
  static constexpr bool PAIR = PAIR_;
  // Weights: of a unit's start and end, of a tile of one block and of two, of a unit that stays whole, and of a CTA's
  // share at least, so that few tiles are not cut into less.
  static constexpr int OVER = 12, ONE = 2, TWO = 4, SMALL = 24, LEAST = 8;
};

// A unit of a sequence: its key tiles, blocks and weight.
template <class S>
struct Unit {
  KeyTiles kt;
  int t0, blocks, w;  // first token of the chunk
  GDNX_DEV Unit() : kt(), t0(0), blocks(0), w(0) {}
  GDNX_DEV Unit(const ChunkParams& P, const Chunk& s, int u) {
    const int step = S::PAIR ? 2 * P.tb : P.tb;
    t0 = u * step;
    const int n = min(step, s.count - t0);
    blocks = n > P.tb ? 2 : 1;
    kt = KeyTiles(s.first + t0, s.first + t0 + n - 1, s.len(), (int)P.a.window, (int)P.a.sinks, S::KEYS);
    w = S::OVER + (blocks == 2 ? S::TWO : S::ONE) * kt.count;
  }
};

template <class S>
GDNX_DEV int units_of(const ChunkParams& P, const Chunk& s) {
  const int step = S::PAIR ? 2 * P.tb : P.tb;
  return (s.count + step - 1) / step;
}

GDNX_DEV long long warp_sum64(long long x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}
GDNX_DEV long long warp_scan64(long long x) {  // inclusive
  const int lane = threadIdx.x % 32;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  return x;
}

// Weight of one head group of each lane's sequence; those of many units are added up by the whole warp.
template <class S>
GDNX_DEV long long chunk_weight(const ChunkParams& P, const Chunk& s) {
  const int nu = units_of<S>(P, s);
  long long w = 0;
  if (nu <= 4)
    for (int u = 0; u < nu; ++u) w += Unit<S>(P, s, u).w;
  for (uint32_t big = __ballot_sync(0xffffffffu, nu > 4); big; big &= big - 1) {
    const int src = __ffs(big) - 1, n = __shfl_sync(0xffffffffu, nu, src);
    Chunk t;
    t.row = 0;
    t.start = 0;
    t.first = __shfl_sync(0xffffffffu, s.first, src);
    t.count = __shfl_sync(0xffffffffu, s.count, src);
    long long x = 0;
    for (int u = threadIdx.x % 32; u < n; u += 32) x += Unit<S>(P, t, u).w;
    x = warp_sum64(x);
    if (threadIdx.x % 32 == src) w = x;
  }
  return w;
}

// A CTA's share t0..t1-1 of the row of weights, the unit that holds t0 and the weight before it.
struct Share {
  long long t0, t1, before, per, one;  // one: weight of a head group of the sequence
  int seq, hg, u;
};

template <class S, int THREADS>
GDNX_DEV void find_share(const ChunkParams& P, Share& out, long long* sums) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, hgs = (int)P.a.cache.Hk * P.groups;
  const int64_t n = P.a.n, run = (n + THREADS - 1) / THREADS;
  const int64_t b0 = min((int64_t)threadIdx.x * run, n), b1 = min(b0 + run, n);
  const auto weight = [&](int64_t i) {
    Chunk s = {0, 0, 0, 0};
    if (i < b1) s = make_chunk(P.a, i);
    return chunk_weight<S>(P, s);
  };
  long long mine = 0;
  for (int64_t k = 0; k < run; ++k) mine += weight(b0 + k);
  long long s = warp_scan64(mine);
  if (lane == 31) sums[warp] = s;
  if (threadIdx.x == 0) out = {0, 0, 0, 1, 1, 0, 0, 0};
  __syncthreads();
  long long before = s - mine, total = 0;
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) {
    if (i < warp) before += sums[i];
    total += sums[i];
  }
  total *= hgs;
  before *= hgs;
  long long per = (total + P.grid - 1) / P.grid;
  if (per < S::LEAST) per = S::LEAST;
  const long long t0 = min(blockIdx.x * per, total);
  // the thread whose run of sequences holds t0 finds the one (a warp votes, since weights are found by warps)
  const bool here = t0 < total && t0 >= before && t0 < before + mine * hgs;
  if (__any_sync(0xffffffffu, here)) {
    bool found = false;
    for (int64_t k = 0; k < run; ++k) {
      const long long w = (run == 1 ? mine : weight(b0 + k)) * hgs;
      if (here && !found && t0 < before + w) {
        found = true;
        out = {t0, min(t0 + per, total), before, per, w / hgs, (int)(b0 + k), 0, 0};
      }
      if (!found) before += w;
    }
  }
  __syncthreads();
  if (warp == 0 && out.t0 < out.t1) {
    const Chunk c = make_chunk(P.a, out.seq);
    const int nu = units_of<S>(P, c);
    const int hg = (int)((t0 - out.before) / out.one);
    long long at = out.before + hg * out.one;
    if (nu == 1 && lane == 0) {
      out.before = at;
      out.hg = hg;
      out.u = 0;
    }
    for (int u0 = 0; nu > 1 && u0 < nu; u0 += 32) {
      const long long w = u0 + lane < nu ? Unit<S>(P, c, u0 + lane).w : 0, in = warp_scan64(w);
      const uint32_t behind = __ballot_sync(0xffffffffu, t0 < at + in);
      if (behind) {
        const int first = __ffs(behind) - 1;
        at += __shfl_sync(0xffffffffu, in - w, first);
        if (lane == 0) {
          out.before = at;
          out.hg = hg;
          out.u = u0 + first;
        }
        break;
      }
      at += __shfl_sync(0xffffffffu, in, 31);
    }
  }
  __syncthreads();
}

// Walks the units of a share: every role sees the same sequence of segments.
template <class S>
struct Walk {
  const ChunkParams& P;
  long long t0, t1, before;
  int seq, hg, u;
  Chunk s;
  Unit<S> x;
  int ta, tb;  // segment: tiles ta..tb-1 of the unit
  bool begun;
  GDNX_DEV Walk(const ChunkParams& P_, const Share& r)
      : P(P_), t0(r.t0), t1(r.t1), before(r.before), seq(r.seq), hg(r.hg), u(r.u), s(), x(), ta(0), tb(0), begun(false) {
    if (t0 < t1) s = make_chunk(P.a, seq);
  }
  GDNX_DEV bool next() {
    if (t0 >= t1) return false;
    for (;;) {
      if (begun) {
        before += x.w;
        if (before >= t1) return false;
        if (++u >= units_of<S>(P, s)) {
          u = 0;
          if (++hg == (int)P.a.cache.Hk * P.groups) {
            hg = 0;
            do {
              if (++seq >= P.a.n) return false;
              s = make_chunk(P.a, seq);
            } while (s.count == 0);
          }
        }
      }
      begun = true;
      x = Unit<S>(P, s, u);
      if (!P.cut || x.w <= S::SMALL) {
        ta = 0;
        tb = before >= t0 ? x.kt.count : 0;
      } else {
        // tile i lies at before + OVER + i of its weights, and belongs to the share that this lies in
        const long long lo = t0 - before - S::OVER, hi = t1 - before - S::OVER;
        ta = tiles_before(lo);
        tb = tiles_before(hi);
      }
      if (ta < tb) return true;
    }
  }
  // Tiles of the unit that begin before weight z behind its start.
  GDNX_DEV int tiles_before(long long z) const {
    if (z <= 0) return 0;
    const int most = (int)min(z, (long long)x.w);  // (a tile weighs 1 or more)
    return min(x.blocks == 2 ? (most + S::TWO - 1) / S::TWO : (most + S::ONE - 1) / S::ONE, x.kt.count);
  }
  GDNX_DEV bool whole() const { return ta == 0 && tb == x.kt.count; }
  // Where this segment's part lies: one that goes on in the next CTA is this CTA's last, any other its first.
  GDNX_DEV int64_t part() const { return ((int64_t)blockIdx.x * 2 + (ta == 0 ? 1 : 0)) * P.rows; }
  GDNX_DEV int hk() const { return hg / P.groups; }
  GDNX_DEV int head0() const { return hk() * (int)(P.a.H / P.a.cache.Hk) + hg % P.groups * P.gs; }
  // Heads of this group.
  GDNX_DEV int heads() const { return min(P.gs, (int)(P.a.H / P.a.cache.Hk) - hg % P.groups * P.gs); }
  // The joint of the cut unit that ends here.
  GDNX_DEV bool ends_cut() const { return ta > 0 && tb == x.kt.count; }
  GDNX_DEV Joint joint(long long per) const { return {seq, hg, u, (int)((before + S::OVER) / per), (int)blockIdx.x}; }
};

// What stands for the maximum where something is seen but no score lies above -inf (nothing seen: -inf).
constexpr float kNoScore = -3.402823466e38f;

// Zeros (and lse -inf) for packed rows r0..r1-1, by `threads` threads of which this is the i-th.
GDNX_DEV void zero_rows(const ChunkParams& P, int64_t r0, int64_t r1, int i, int threads) {
  const gdnx_paged_attn_args& a = P.a;
  const int D = (int)a.cache.D, n = (int)a.H * D;
  for (int64_t t = r0; t < r1; ++t)
    for (int x = i; x < n; x += threads) {
      st_from_f32(a.y, a.y_dtype, t * a.y_st + x / D * a.y_sh + x % D, 0.f);
      if (a.lse && x % D == 0) a.lse[t * a.H + x / D] = -INFINITY;
    }
}
// Padding rows: those before the first sequence and behind the last, and sequences that have no tokens after all.
GDNX_DEV void write_padding(const ChunkParams& P, int i, int threads) {
  const gdnx_paged_attn_args& a = P.a;
  const int64_t begin = a.n ? min((int64_t)max(a.starts[0], 0), a.tokens) : 0;
  const int64_t end = a.n ? min((int64_t)max(a.starts[a.n], 0), a.tokens) : 0;
  for (int64_t t = blockIdx.x; t < begin; t += P.grid) zero_rows(P, t, t + 1, i, threads);
  for (int64_t t = end + blockIdx.x; t < a.tokens; t += P.grid) zero_rows(P, t, t + 1, i, threads);
  for (int64_t b = blockIdx.x; b < a.n; b += P.grid) {
    const Chunk s = make_chunk(a, b);
    if (s.count == 0) zero_rows(P, s.start, min(max(a.starts[b + 1], s.start), (int)a.tokens), i, threads);
  }
}

// A row's output and log of the sum of exponentials where its parts are (maximum, sum): 0 where nothing was seen, NaN
// where all that was seen is -inf or some score is NaN or +inf.
GDNX_DEV float scale_of(float top, float sum) { return sum > 0.f ? 1.f / sum : top == -INFINITY ? 0.f : NAN; }
GDNX_DEV float lse_of(float top, float sum) {
  return sum > 0.f ? (top + log2f(sum)) * kLn2 : top == -INFINITY ? -INFINITY : NAN;
}

// Joins a cut unit's parts, CTA after CTA: block (c, y) rows JOIN_ROWS y .. of the unit that ends in CTA c.  Eight lanes
// share a row, which keeps the work that a row needs once to an eighth of a warp (a row to a warp took 26 us where 4096
// tokens of 16 heads are cut for 148 CTAs; now 14).  Where there are many parts, all eight warps take each row, a
// run of the parts each, joined in order.
constexpr int JOIN_WARPS = 8, JOIN_ROWS = 64;

template <class S>
__global__ void __launch_bounds__(JOIN_WARPS * 32) paged_attn_join_kernel(const ChunkParams P) {
  const gdnx_paged_attn_args& a = P.a;
  __shared__ float red_m[JOIN_WARPS], red_l[JOIN_WARPS], red_o[JOIN_WARPS][128];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, D = (int)a.cache.D;
  dependents_may_start();
  wait_for_earlier();  // the parts are there
  const Joint j = P.joint[blockIdx.x];
  if (j.c1 < 0) return;
  const Chunk s = make_chunk(a, j.seq);
  const int G = (int)(a.H / a.cache.Hk), h0 = j.hg / P.groups * G + j.hg % P.groups * P.gs;
  const int heads = min(P.gs, G - j.hg % P.groups * P.gs), t0 = j.u * (S::PAIR ? 2 * P.tb : P.tb);
  const auto place = [&](int c, int r) { return ((int64_t)c * 2 + (c == j.c0)) * P.rows + r; };
  // the packed row and head of row r, or -1
  const auto query = [&](int r, int& head) {
    const int q = r % S::ROWS, tok = q / P.gs, t = t0 + r / S::ROWS * P.tb + tok;
    head = h0 + q - tok * P.gs;
    return tok < P.tb && head < h0 + heads && t < s.count ? s.start + t : -1;
  };
  const int parts = j.c1 - j.c0 + 1, r0 = blockIdx.y * JOIN_ROWS, r1 = min(r0 + JOIN_ROWS, P.rows);
  if (parts <= 8) {
    const int d0 = lane % 8 * 4;  // this lane's values: four of each 32
    for (int r = r0 + warp * 4 + lane / 8; r < r1; r += JOIN_WARPS * 4) {
      int head;
      const int64_t tok = query(r, head);
      if (tok < 0) continue;
      float m = -INFINITY, l = 0.f;
      for (int c = j.c0; c <= j.c1; ++c) m = fmaxf(m, P.stat[place(c, r) * 2]);
      const float base = m == -INFINITY ? 0.f : m;
      float4 y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int c = j.c0; c <= j.c1; ++c) {
        const int64_t at = place(c, r);
        const float2 st = *reinterpret_cast<const float2*>(P.stat + at * 2);
        const float w = exp2f(st.x - base);
        const float* x = P.part + at * D + d0;
        l = fmaf(w, st.y, l);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (d0 + 32 * e < D) {
            const float4 v = *reinterpret_cast<const float4*>(x + 32 * e);
            y[e] = make_float4(fmaf(w, v.x, y[e].x), fmaf(w, v.y, y[e].y), fmaf(w, v.z, y[e].z), fmaf(w, v.w, y[e].w));
          }
      }
      const float f = scale_of(m, l);
      const int64_t out = tok * a.y_st + head * a.y_sh + d0;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (d0 + 32 * e < D) {
          const float v[4] = {y[e].x * f, y[e].y * f, y[e].z * f, y[e].w * f};
          if (P.vec_join && a.y_dtype != GDNX_F32) {
            const bool bf = a.y_dtype == GDNX_BF16;
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.y) + out + 32 * e) =
                make_uint2(bf ? pack2<true>(v[0], v[1]) : pack2<false>(v[0], v[1]), bf ? pack2<true>(v[2], v[3]) : pack2<false>(v[2], v[3]));
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) st_from_f32(a.y, a.y_dtype, out + 32 * e + i, v[i]);
          }
        }
      if (a.lse && d0 == 0) a.lse[tok * a.H + head] = lse_of(m, l);
    }
    return;
  }
  const int run = (parts + JOIN_WARPS - 1) / JOIN_WARPS;
  const int from = min(j.c0 + warp * run, j.c1 + 1), to = min(from + run, j.c1 + 1);
  for (int r = r0; r < r1; ++r) {
    int head;
    const int64_t tok = query(r, head);
    if (tok < 0) continue;
    float m = -INFINITY, l = 0.f;
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c = from + lane; c < to; c += 32) m = fmaxf(m, P.stat[place(c, r) * 2]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll 4
    for (int c = from; c < to; ++c) {
      const int64_t at = place(c, r);
      const float w = exp2f(P.stat[at * 2] - base);
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (lane * 4 < D) x = *reinterpret_cast<const float4*>(P.part + at * D + lane * 4);
      l = fmaf(w, P.stat[at * 2 + 1], l);
      y = make_float4(fmaf(w, x.x, y.x), fmaf(w, x.y, y.y), fmaf(w, x.z, y.z), fmaf(w, x.w, y.w));
    }
    *reinterpret_cast<float4*>(&red_o[warp][lane * 4]) = y;
    if (lane == 0) {
      red_m[warp] = m;
      red_l[warp] = l;
    }
    __syncthreads();
    const int d = threadIdx.x;
    if (d < D) {
      float top = -INFINITY, sum = 0.f, v = 0.f;
#pragma unroll
      for (int i = 0; i < JOIN_WARPS; ++i) top = fmaxf(top, red_m[i]);
      const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int i = 0; i < JOIN_WARPS; ++i) {
        const float w = exp2f(red_m[i] - ref);
        sum = fmaf(w, red_l[i], sum);
        v = fmaf(w, red_o[i][d], v);
      }
      st_from_f32(a.y, a.y_dtype, tok * a.y_st + head * a.y_sh + d, v * scale_of(top, sum));
      if (a.lse && d == 0) a.lse[tok * a.H + head] = lse_of(top, sum);
    }
    __syncthreads();
  }
}

// The plan of a call with `ctas` resident CTAs.
template <class S>
ChunkParams plan_chunks(const gdnx_paged_attn_args& a, int ctas) {
  ChunkParams P = {};
  P.a = a;
  const int64_t G = a.H / a.cache.Hk;
  P.groups = (int)((G + S::ROWS - 1) / S::ROWS);
  P.gs = (int)((G + P.groups - 1) / P.groups);
  P.tb = S::ROWS / P.gs;
  P.rows = S::PAIR && a.tokens > P.tb ? 2 * S::ROWS : S::ROWS;
  int64_t most = a.cache.width * a.cache.page;
  if (a.max_len > 0 && a.max_len < most) most = a.max_len;
  int64_t tiles = (most + S::KEYS - 1) / S::KEYS;  // of a unit, at most
  const int64_t seen = (a.window + (S::PAIR ? 2 : 1) * P.tb + S::KEYS - 1) / S::KEYS + 1 + (a.sinks + S::KEYS - 1) / S::KEYS;
  if (seen < tiles) tiles = seen;
  const int64_t w = S::OVER + tiles * (P.rows > S::ROWS ? S::TWO : S::ONE);  // of a unit, at most
  P.cut = w > S::SMALL;
  // a CTA's share is LEAST in weight, or a unit
  const int64_t units = (a.tokens / P.tb + a.n) * a.cache.Hk * P.groups;
  const int64_t want = P.cut ? (units * w + S::LEAST - 1) / S::LEAST : units;
  P.grid = (int)(want < ctas ? (want > 0 ? want : 1) : ctas);
  P.vec_join = reinterpret_cast<uintptr_t>(a.y) % 8 == 0 && a.y_st % 4 == 0 && a.y_sh % 4 == 0;
  P.part = static_cast<float*>(a.workspace);
  P.stat = P.part + (size_t)P.grid * 2 * P.rows * a.cache.D;
  P.joint = reinterpret_cast<Joint*>(P.stat + (size_t)P.grid * 2 * P.rows * 2);
  return P;
}

inline size_t chunk_bytes(const ChunkParams& P) {
  return P.cut ? (size_t)P.grid * (2 * P.rows * (P.a.cache.D + 2) * sizeof(float) + sizeof(Joint)) : 0;
}

// The join behind the kernel, where units may have been cut.
template <class S>
gdnx_status join_chunks(const ChunkParams& P, cudaStream_t st) {
  if (!P.cut) return GDNX_OK;
  const cudaError_t e = launch_early(paged_attn_join_kernel<S>, dim3((unsigned)P.grid, (unsigned)((P.rows + JOIN_ROWS - 1) / JOIN_ROWS)),
                                     dim3(JOIN_WARPS * 32), 0, st, P);
  return e == cudaSuccess ? GDNX_OK : GDNX_ELAUNCH;
}

}  // namespace
}  // namespace gdnx
