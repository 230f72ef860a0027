// beam_sched.h — how the kernels for several continuations of a prompt share out their
// work: integer rules that the device evaluates and host tests check.
//
// Host-compilable on purpose (plain C++, no HIP types): tests/test_beam_sched.py builds
// a host program from this header with g++.
#ifndef MI355_BEAM_SCHED_H
#define MI355_BEAM_SCHED_H

#include <stdint.h>

#include "serve_sched.h"

namespace mi355fa {

// ── shared decode: what a group reads once, and what is left to its requests ──
// Tiles of kDecTile keys that every request of a group sees whole: inside the prefix,
// of the shortest request's keys, from the longest one's window on. `least` and `most`:
// lengths of those requests of the group that have keys.
struct TileSpan {
  int t0, t1;   // tiles [t0, t1); 0, 0 where there is nothing to share
};
MI355_HD inline TileSpan shared_tiles(int prefix, int least, int most, int window, int requests) {
  if (requests < 2) return TileSpan{0, 0};
  const int lo = imax(0, most - window), hi = imin(prefix, least);
  const TileSpan s{(lo + kDecTile - 1) / kDecTile, hi / kDecTile};
  return s.t0 < s.t1 ? s : TileSpan{0, 0};
}
// The tiles that a request reads by itself: `before` of them from `first` on, the others
// from `behind` on. Its seen keys are [lo, len).
struct OwnTiles {
  int lo, len, first, before, behind, count;
};
MI355_HD inline OwnTiles own_tiles(int len, int window, TileSpan s) {
  OwnTiles o{imax(0, len - window), len, 0, 0, 0, 0};
  if (len <= 0) return o;
  o.first = o.lo / kDecTile;
  const int end = (len + kDecTile - 1) / kDecTile;
  o.before = s.t0 < s.t1 ? s.t0 - o.first : end - o.first;
  o.behind = s.t1;
  o.count = s.t0 < s.t1 ? o.before + end - s.t1 : o.before;
  return o;
}
MI355_HD inline int own_tile(const OwnTiles& o, int i) { return i < o.before ? o.first + i : o.behind + i - o.before; }

// Tiles of a group's part where all tiles of all units are `sum` and about `target` workgroups
// wanted, each of which takes as many; of a request's, which one wave of four takes. At
// most target workgroups, and one for each group's unit and each four of the requests', come of it.
MI355_HD inline int share_size(int64_t sum, int target, int least) { return imax((int)((double)sum / target) + 1, least); }
MI355_HD inline int wave_share_size(int per, int least) { return imax((per + 3) / 4, least); }
MI355_HD inline int share_count(int tiles, int per) { return (tiles + per - 1) / per; }   // 0 of no tiles
// Part p of n takes tiles [share_start(p), share_start(p + 1)).
MI355_HD inline int share_start(int tiles, int n, int p) {
  const int each = tiles / n, more = tiles - each * n;
  return p * each + imin(p, more);
}

// Place `place` of an item's parts, of heads · blocks units of n parts each: the blocks of one
// part of one head read the same tiles, and are 8 places apart, on one XCD.
struct UnitPart {
  int hk, block, part;
};
MI355_HD inline UnitPart unit_part(int place, int n, int heads, int blocks) {
  const uint32_t all = (uint32_t)(heads * n), whole = all & ~7u, x = (uint32_t)place;
  uint32_t item, block;
  if (x < whole * blocks) {
    const uint32_t eight = x >> 3;
    item = eight / blocks * 8 + (x & 7);
    block = eight % blocks;
  } else {
    const uint32_t rest = all - whole, y = x - whole * blocks;
    item = whole + y % rest;
    block = y / rest;
  }
  return {(int)(item / (uint32_t)n), (int)block, (int)(item % (uint32_t)n)};
}

}  // namespace mi355fa

#endif  // MI355_BEAM_SCHED_H
