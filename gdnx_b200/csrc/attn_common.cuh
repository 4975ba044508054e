// Shared pieces of the windowed-attention kernels: which keys a block of queries sees.
#pragma once

#include "common.cuh"

namespace gdnx {
namespace attn {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Query position p sees key j.  `len` is the sequence's length; keys and queries at or
// beyond it are padding.  The distance p - j is below 2^31 (sizes are checked on the host).
GDNX_DEV bool sees(int p, int j, int len, int window, int sinks) {
  return j <= p && j < len && p < len && (p - j < window || j < sinks);
}

// Position p sees one key only.  A softmax over one key has no gradient: its dS is 0, while
// dP - delta would leave the difference of two roundings.
GDNX_DEV bool sees_one(int p, int window, int sinks) { return p == 0 || (window == 1 && sinks == 0); }

GDNX_DEV int seq_len(const gdnx_attn_args& a, int64_t b) {
  if (!a.lengths) return (int)a.Tk;
  const int n = a.lengths[b];
  return n < 0 ? 0 : (n > (int)a.Tk ? (int)a.Tk : n);
}

// The key tiles (of `BK` keys) that the queries at positions p0..p1 (inclusive) see, as
// one sequence 0..count-1: first the tiles that hold sinks and lie before the window,
// then the window's own.
struct KeyTiles {
  int nsink, lo, count;
  GDNX_DEV KeyTiles() : nsink(0), lo(0), count(0) {}
  GDNX_DEV KeyTiles(int p0, int p1, int len, int window, int sinks, int BK) {
    const int last = min(p1, len - 1);
    if (p0 >= len || last < 0) {
      nsink = lo = count = 0;
      return;
    }
    const int first = max(0, p0 - window + 1);
    lo = first / BK;
    nsink = min((int)(((int64_t)sinks + BK - 1) / BK), lo);
    count = nsink + last / BK - lo + 1;
  }
  GDNX_DEV int tile(int i) const { return i < nsink ? i : lo + i - nsink; }
};

}  // namespace attn
}  // namespace gdnx
