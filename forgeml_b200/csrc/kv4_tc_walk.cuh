// Which parts of the batch a CTA of the tensor-core kernel works through, and what it
// does about those that it can no longer work on.
#pragma once

#include "kv4_attention.cuh"

namespace fml {
namespace kv4 {
namespace tc {

constexpr int kRows = 128;   // query rows of a segment
constexpr int kBlock = 128;  // positions of a block

// A part of a segment: its blocks [lo, hi) (those that its rows attend at all).
struct Part {
  int b, h, row0, rows;  // rows of the request's head: row0 .. row0 + rows - 1
  int start, kend;       // request's first position; positions that some row attends
  int lo, hi;
  bool whole;
  unsigned seg0, units;  // in the batch's order: the segment's first unit, its units
  int which;             // first or last part of the CTA's share
};
using BlockCursor = Cursor<kBlock>;
// The parts that this CTA works through, in order; every role walks alike.
struct Walk {
  bool shared;
  int row_tiles, left;
  unsigned at, begin;
  BlockCursor cur;
  __host__ __device__ __forceinline__ bool next(const Pool& p, const Problem& a, Part& o) {
    if (left == 0) return false;
    const int n = shared ? min(cur.units - cur.unit, left) : 1;
    const int rows = a.group * a.tq;
    o.b = cur.b;
    o.h = cur.seg / row_tiles;
    o.row0 = (cur.seg - o.h * row_tiles) * kRows;
    o.rows = min(kRows, rows - o.row0);
    o.start = a.start_pos[cur.b];
    o.kend = min(cur.keys, o.start + (o.row0 + o.rows - 1) / a.group + 1);
    const int blocks = (o.kend + kBlock - 1) / kBlock;
    o.lo = shared ? cur.unit : 0;
    o.hi = shared ? max(o.lo, min(cur.unit + n, blocks)) : blocks;
    o.whole = !shared || n == cur.units;
    o.units = cur.units;
    o.which = at == begin ? 0 : 1;
    o.seg0 = at - cur.unit;
    left -= n;
    at += n;
    if (shared) {
      cur.unit += n;
      if (cur.unit == cur.units) cur.next_segment(p, a);
    }
    return true;
  }
};

// The parts that begin at unit `begin` of the batch's order and end before `end`.
__host__ __device__ __forceinline__ Walk walk_from(const Pool& p, const Problem& a, int row_tiles, unsigned begin,
                                                   unsigned end) {
  Walk w;
  w.shared = true;
  w.row_tiles = row_tiles;
  w.begin = w.at = begin;
  w.left = (int)(end - begin);
  w.cur.seg = w.cur.unit = 0;
  w.cur.request(p, a, 0);
  w.cur.skip(p, a, begin);
  return w;
}
// A CTA whose wait gave up still takes the tickets that it owes (`took`: bit 0 where it
// has its first part's, bit 1 its last one's; no others are split).  A ticket word counts
// a launch's tickets and is cleaned by the last one; a replayed graph launches with the
// same number, and would begin from what a missing ticket left.  take(part, w0) returns
// the tickets of word w0 taken so far, clean(w0) makes it ready for the next launch.
template <typename Take, typename Clean>
__host__ __device__ __forceinline__ void give_up(const Pool& p, const Problem& a, const Shares& shares, int row_tiles,
                                                 unsigned cta, unsigned took, Take take, Clean clean) {
  if (cta >= shares.W) return;
  Walk walk = walk_from(p, a, row_tiles, shares.begin(cta), shares.begin(cta + 1));
  Part part;
  while (walk.next(p, a, part)) {
    if (part.whole || (took >> part.which & 1)) continue;
    const unsigned w0 = shares.holder(part.seg0, cta), w1 = shares.holder(part.seg0 + part.units - 1, cta);
    if (take(part, w0) == w1 - w0 + 1) clean(w0);
  }
}

}  // namespace tc
}  // namespace kv4
}  // namespace fml
