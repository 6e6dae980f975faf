// Which keys the new tokens of a paged prompt see: plain arithmetic of the planner, in functions that a host
// compiler takes too.  Positions may be negative (a sequence shorter than its new tokens) and a window as long as
// an int, so nothing is subtracted before it is known to be the smaller one.
#pragma once
#include <cstdint>

#ifdef __CUDACC__
#define ZS_PLAN_FN __host__ __device__ __forceinline__
#else
#define ZS_PLAN_FN inline
#endif

namespace zs {
namespace paged {

// A sequence's length inside [0, cap].
ZS_PLAN_FN int length_within(int len, int cap) { return len < 0 ? 0 : len > cap ? cap : len; }

// A window that reaches over every position of a table of cap tokens is none (0).
ZS_PLAN_FN int window_within(int window, int64_t cap) { return window >= cap ? 0 : window; }

// The first key that a query at position p (or later) sees.
ZS_PLAN_FN int first_seen(int p, int window) {
  return window > 0 && p >= window ? p - window + 1 : 0;
}

// The key tiles [lo, lo + cnt) of TILE keys that `rows` queries from position p0 on see; cnt is 0 where all of
// them lie before the first position.
struct KeyTiles {
  int lo, cnt;
};
template <int TILE>
ZS_PLAN_FN KeyTiles key_tiles(int p0, int rows, int window) {
  KeyTiles k;
  k.lo = first_seen(p0, window) / TILE;
  k.cnt = rows > 0 && p0 + (rows - 1) >= 0 ? (p0 + (rows - 1)) / TILE - k.lo + 1 : 0;
  return k;
}

}  // namespace paged
}  // namespace zs
