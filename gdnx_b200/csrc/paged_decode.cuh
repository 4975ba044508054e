// What the decode kernels share: the work of a call as a row of tiles, cut evenly over the CTAs,
// and the kernel that joins the parts of a cut unit.
//
// A unit is one sequence and key head (and group of up to NH of its query heads); its visible
// tokens are walked in tiles of 128 positions.  All units' tiles in a row are cut evenly over the
// CTAs (one on each SM), so that mixed lengths leave none waiting: a CTA takes the end of one
// unit, whole units, the beginning of another.  Whole units are written at once; parts leave
// maximum, sum and unnormalised output, and a second kernel joins them in order.  Every CTA finds
// its range from the lengths by itself.  Where no unit can have more than four tiles, a CTA takes
// whole units and there is nothing to join.
#pragma once

#include "attn_tc.cuh"
#include "kernels.h"
#include "launch.cuh"

namespace gdnx {
namespace {  // one copy for each kernel file

using namespace attn;

constexpr int WHOLE_TILES = 4;  // units of up to so many tiles are not cut


// A unit that was cut: its parts lie in CTAs c0..c1.  c1 < 0: none.
struct Joint {
  int b, unit, c0, c1;
};

struct DecParams {
  gdnx_paged_decode_args a;
  float* part;     // [grid][2][NH][128] unnormalised outputs of a CTA's first and last unit
  float* stat;     // [grid][2][NH][2] maximum (log2 domain) and sum
  Joint* joint;    // [grid] the unit cut in several parts that ends in a CTA
  int grid, groups;
  int whole;       // no unit is cut: a CTA takes whole units
};

// The place of a CTA in the row of all tiles: its tiles t0..t1-1, the sequence b that holds t0
// and the tiles of the sequences before b.  Tiles are ordered by sequence, unit, tile.
struct Range {
  int64_t t0, t1, before, b, per;
};

// Visible tokens of one sequence.
struct Seq {
  int row, len;
  KeyTiles kt;
};

GDNX_DEV int slot_length(const gdnx_paged_decode_args& a, int64_t b, int& row) {
  const gdnx_cache& c = a.cache;
  row = a.rows ? a.rows[b] : (int)b;
  if (row < 0 || row >= c.slots) return 0;
  const int64_t n = c.lengths[row], most = c.width * c.page;
  return (int)(n < 0 ? 0 : (n > most ? most : n));
}

GDNX_DEV Seq make_seq(const gdnx_paged_decode_args& a, int64_t b) {
  int row;
  const int len = slot_length(a, b, row);
  return {row, len, KeyTiles(len - 1, len - 1, len, (int)a.window, (int)a.sinks, TM)};
}

GDNX_DEV int tiles_of(const gdnx_paged_decode_args& a, int64_t b) { return make_seq(a, b).kt.count; }

// The CTA finds its range: every thread adds up a run of sequences, and the one whose run holds
// the range's first tile walks to its sequence.  (Whole units: t0 and t1 count units.)
template <int THREADS>
GDNX_DEV void find_range(const DecParams& P, int units, Range& out, long long* sums) {
  if (P.whole) {
    if (threadIdx.x == 0) {
      const int64_t all = P.a.B * units;
      out = {all * blockIdx.x / P.grid, all * (blockIdx.x + 1) / P.grid, 0, 0, 0};
    }
    __syncthreads();
    return;
  }
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int64_t run = (P.a.B + THREADS - 1) / THREADS;
  const int64_t b0 = min((int64_t)threadIdx.x * run, P.a.B), b1 = min(b0 + run, P.a.B);
  long long mine = 0;
  for (int64_t b = b0; b < b1; ++b) mine += tiles_of(P.a, b);
  long long s = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += y;
  }
  if (lane == 31) sums[warp] = s;
  if (threadIdx.x == 0) out = {0, 0, 0, 0, 1};
  __syncthreads();
  long long before = s - mine, total = 0;
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) {
    if (i < warp) before += sums[i];
    total += sums[i];
  }
  total *= units;
  before *= units;
  const long long per = (total + P.grid - 1) / P.grid, t0 = min(blockIdx.x * per, total);
  if (t0 < total && t0 >= before && t0 < before + mine * units) {
    int64_t b = b0;
    for (; b + 1 < b1; ++b) {
      const long long n = (long long)tiles_of(P.a, b) * units;
      if (t0 < before + n) break;
      before += n;
    }
    out = {t0, min(t0 + per, total), before, b, per};
  }
  __syncthreads();
}

// Walks the units of a range: every role sees the same sequence of segments.
struct Walk {
  const DecParams& P;
  int units;
  int64_t t, t1, b, before;
  Seq seq;
  int unit, ta, tb;  // segment: tiles ta..tb-1 of `unit` of sequence b
  GDNX_DEV Walk(const DecParams& P_, int units_, const Range& r)
      : P(P_), units(units_), t(r.t0), t1(r.t1), b(r.b), before(r.before), seq(), unit(0), ta(0), tb(0) {
    if (t < t1 && !P.whole) seq = make_seq(P.a, b);
  }
  GDNX_DEV bool next() {
    if (P.whole) {
      for (; t < t1; ++t) {
        b = t / units;
        unit = (int)(t % units);
        seq = make_seq(P.a, b);
        if ((tb = seq.kt.count) == 0) continue;
        ++t;
        return true;
      }
      return false;
    }
    if (t >= t1) return false;
    while (t >= before + (int64_t)seq.kt.count * units) {
      before += (int64_t)seq.kt.count * units;
      seq = make_seq(P.a, ++b);
    }
    const int n = seq.kt.count;
    unit = (int)((t - before) / n);
    ta = (int)((t - before) % n);
    tb = (int)min((int64_t)n, ta + (t1 - t));
    t += tb - ta;
    return true;
  }
  GDNX_DEV bool whole() const { return ta == 0 && tb == seq.kt.count; }
};

GDNX_DEV bool key_seen(int j, int len, int window, int sinks) {
  return j < len && (len - 1 - j < window || j < sinks);
}

// Page ids of a tile's pages, or -1 where nothing visible is there (lane < npp).
GDNX_DEV int page_id(const DecParams& P, const Seq& s, int kt, int i) {
  const gdnx_cache& c = P.a.cache;
  const int64_t first = (int64_t)kt * TM + i * c.page;
  if (first >= s.len || !(first + c.page > (int64_t)s.len - P.a.window || first < P.a.sinks)) return -1;
  const int p = c.table[(int64_t)s.row * c.width + first / c.page];
  return p >= 0 && p < c.pages ? p : -1;
}

// What stands for the maximum where something is seen but no score lies above -inf (nothing seen: -inf).
constexpr float kNoScore = -3.402823466e38f;

// The output where the weights' sum is 0.
GDNX_DEV float no_weights(float top) { return top == -INFINITY ? 0.f : NAN; }

// Zeros for the sequences that see nothing.
GDNX_DEV void write_zeros(const DecParams& P) {
  const gdnx_paged_decode_args& a = P.a;
  const int D = (int)a.cache.D, n = (int)a.H * D;
  for (int64_t b = blockIdx.x; b < a.B; b += P.grid) {
    if (tiles_of(a, b) > 0) continue;
    for (int x = threadIdx.x % 32; x < n; x += 32)
      st_from_f32(a.y, a.y_dtype, b * a.y_sb + x / D * a.y_sh + x % D, 0.f);
  }
}

// Heads of one unit.
struct Heads {
  int h0, n;
  GDNX_DEV Heads(const DecParams& P, int unit, int NH) {
    const int G = (int)(P.a.H / P.a.cache.Hk), g = unit % P.groups;
    h0 = unit / P.groups * G + g * NH;
    n = min(NH, G - g * NH);
  }
};

// Joins a cut unit's parts, CTA after CTA: block (c, g) head g of the unit that ends in CTA c.
// Each warp sums a contiguous run of the parts; the runs are added in order.
constexpr int JOIN_WARPS = 8;

template <int NH>
__global__ void __launch_bounds__(JOIN_WARPS * 32) paged_decode_join_kernel(const DecParams P) {
  const gdnx_paged_decode_args& a = P.a;
  __shared__ float red_m[JOIN_WARPS], red_l[JOIN_WARPS], red_o[JOIN_WARPS][128];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, D = (int)a.cache.D, g = blockIdx.y;
  dependents_may_start();
  wait_for_earlier();  // the parts are there
  const Joint j = P.joint[blockIdx.x];
  if (j.c1 < 0) return;
  const Heads hd(P, j.unit, NH);
  if (g >= hd.n) return;
  const int64_t out = j.b * a.y_sb + (hd.h0 + g) * a.y_sh;
  const auto place = [&](int c) { return ((int64_t)c * 2 + (c == j.c0)) * NH + g; };
  const int parts = j.c1 - j.c0 + 1, run = (parts + JOIN_WARPS - 1) / JOIN_WARPS;
  const int r0 = j.c0 + warp * run, r1 = min(r0 + run, j.c1 + 1);
  float m = -INFINITY, l = 0.f;
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int c = r0 + lane; c < r1; c += 32) m = fmaxf(m, P.stat[place(c) * 2]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float base = m == -INFINITY ? 0.f : m;
#pragma unroll 4
  for (int c = r0; c < r1; ++c) {
    const int64_t at = place(c);
    const float w = exp2f(P.stat[at * 2] - base);
    const float4 x = *reinterpret_cast<const float4*>(P.part + at * 128 + lane * 4);
    l = fmaf(w, P.stat[at * 2 + 1], l);
    y.x = fmaf(w, x.x, y.x);
    y.y = fmaf(w, x.y, y.y);
    y.z = fmaf(w, x.z, y.z);
    y.w = fmaf(w, x.w, y.w);
  }
  *reinterpret_cast<float4*>(&red_o[warp][lane * 4]) = y;
  if (lane == 0) {
    red_m[warp] = m;
    red_l[warp] = l;
  }
  __syncthreads();
  const int d = threadIdx.x;
  if (d >= D) return;
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
  st_from_f32(a.y, a.y_dtype, out + d, sum == 0.f ? no_weights(top) : v / sum);
}

// The plan of a call with groups of `nh` query heads.
struct Plan {
  int nh, groups, grid, whole;
};

inline Plan make_plan(const gdnx_paged_decode_args& a, int nh) {
  Plan p;
  const int64_t G = a.H / a.cache.Hk, sms = sm_count();
  p.nh = nh;
  p.groups = (int)((G + nh - 1) / nh);
  int64_t most = a.cache.width * a.cache.page;
  if (a.max_len > 0 && a.max_len < most) most = a.max_len;
  int64_t n = (most + TM - 1) / TM;  // tiles of a unit, at most
  const int64_t seen = (a.window + TM - 1) / TM + 1 + (a.sinks + TM - 1) / TM;
  if (seen < n) n = seen;
  const int64_t units = a.B * a.cache.Hk * p.groups;
  // Short units are not cut: a few more tiles in a row take less time than a join.
  p.whole = n <= WHOLE_TILES;
  const int64_t ctas = p.whole ? units : units * n;
  p.grid = (int)(ctas < sms ? (ctas > 0 ? ctas : 1) : sms);
  return p;
}

inline size_t plan_bytes(const Plan& p) {
  return p.whole ? 0 : (size_t)p.grid * (2 * p.nh * (128 + 2) * sizeof(float) + sizeof(Joint));
}

inline void fill(DecParams& P, const gdnx_paged_decode_args& a, const Plan& p) {
  P.a = a;
  P.grid = p.grid;
  P.groups = p.groups;
  P.whole = p.whole;
  P.part = static_cast<float*>(a.workspace);
  P.stat = P.part + (size_t)p.grid * 2 * p.nh * 128;
  P.joint = reinterpret_cast<Joint*>(P.stat + (size_t)p.grid * 2 * p.nh * 2);
}

// The join behind a decode kernel, where units were cut.
template <int NH>
gdnx_status join_parts(const DecParams& P, cudaStream_t st) {
  if (P.whole) return GDNX_OK;
  const int64_t G = P.a.H / P.a.cache.Hk;
  const cudaError_t e = launch_early(paged_decode_join_kernel<NH>, dim3((unsigned)P.grid, (unsigned)(G < NH ? G : NH)),
                                     dim3(JOIN_WARPS * 32), 0, st, P);
  return e == cudaSuccess ? GDNX_OK : GDNX_ELAUNCH;
}

}  // namespace
}  // namespace gdnx
