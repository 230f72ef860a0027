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

// ── shared decode: the plan in LDS ────────────────────────────────────────────
constexpr int kShMax = 1024;   // requests, and groups
// Its words: 64 of its own, eight of each request or group (one more of the offsets), in whole 16
// bytes, since the waves' rows of V lie behind it.
constexpr int kShWords = (64 + 8 * kShMax + 1 + 3) / 4 * 4;

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

// A workgroup's steps where `sum` waves' tiles are to be read (a group's tile by a wave for each
// 32 columns, a request's own as own_weight of them) and about `target` workgroups of four waves
// wanted; a group's part of them, whose waves take `ways` tiles a step, of at least 4 tiles; and
// a wave's own tiles. At most target + 1 workgroups, and one for each group's
// unit, come of it. (At least 2, 4, 8 tiles: 4 requests of 300 keys 11.7, 11.7, 12.5 us, 21 of 4099
// keys 21.8, 19.5, 21.5.)
// An own tile costs more than a shared one: a wave waits for each unit's first. Measured, for
// weights of 1, 2, 3, 4, 6: 9 groups of 32 columns 35.4, 28.2, 31.3, 32.2, 40.2 us, one of 1020
// columns 80, 56, 48.2, 47.8, 51.9 us.
MI355_HD inline int own_weight(int columns) { return imax(columns / 32, 2); }
MI355_HD inline int share_steps(int64_t sum, int target) { return (int)((double)sum / (4.0 * target)) + 1; }
MI355_HD inline int share_size(int steps, int ways) { return imax(steps * ways, 4); }
MI355_HD inline int wave_share_size(int steps, int weight) { return imax((steps + weight - 1) / weight, 1); }
MI355_HD inline int share_count(int tiles, int per) { return (tiles + per - 1) / per; }   // 0 of no tiles
// Part p of n takes tiles [share_start(p), share_start(p + 1)).
MI355_HD inline int share_start(int tiles, int n, int p) {
  const int each = tiles / n, more = tiles - each * n;
  return p * each + imin(p, more);
}

// Where the requests' own tiles, one behind another, are cut into waves of `per`: the wave of
// tile `start`, and how many of its tiles come before.
struct WaveTile {
  int wave, before;
};
MI355_HD inline WaveTile wave_tile(int64_t start, int per) {
  int wave = (int)((double)start / per);   // (at most one off)
  int64_t before = start - (int64_t)wave * per;
  if (before < 0) --wave, before += per;
  if (before >= per) ++wave, before -= per;
  return {wave, (int)before};
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

// ── selection: parts of a row of logits ──────────────────────────────────────
constexpr int kSelThreads = 256;
constexpr int kSelCandidates = 1 << 14;   // of a search, that the join holds
constexpr int kSelMostPer = 1 << 30;

// A row's parts, of `per` tokens each but the last; wide: the steps are of `vectors` times 8 elements a
// thread. `rows` of all searches, `beams` of one, of `vocab` tokens each, the `k` best wanted.
struct SelectSplit {
  int parts, per, wide;
};
MI355_HD inline SelectSplit select_split(int64_t rows, int beams, int vocab, int k, int vectors, int cus) {
  const int small = kSelThreads * 8;
  // Parts of a row: workgroups for all CUs, four on each, but one where k is large, since the
  // join's candidates grow with both (us for one, two, four: [4 x 50 x 10007] fp32, k = 50
  // 25.8 / 34.1 / 35.7; [64 x 8 x 128000] bf16, k = 16 71 / 71 / 60); no more than the join holds
  const int64_t most = kSelCandidates / ((int64_t)beams * k), all_cus = (k > 32 ? 1 : 4) * (int64_t)cus / rows;
  const int64_t wanted = imax(1, (int)(all_cus < most ? all_cus : most));
  const int64_t steps = ((int64_t)vocab + small - 1) / small;
  SelectSplit s;
  s.wide = steps >= vectors * wanted;
  const int step = s.wide ? vectors * small : small;
  const int64_t all = ((int64_t)vocab + step - 1) / step, each = (all + wanted - 1) / wanted;
  s.per = (int)(each * step < kSelMostPer ? each * step : kSelMostPer);
  s.parts = (int)(((int64_t)vocab + s.per - 1) / s.per);
  return s;
}
// Tokens of a part, at least one; of the last part, begin + per may be 2^31 or more.
struct SelectSpan {
  int begin, end;
};
MI355_HD inline SelectSpan select_span(int part, int per, int vocab) {
  const int begin = part * per;
  return {begin, vocab - begin < per ? vocab : begin + per};
}

}  // namespace mi355fa

#endif  // MI355_BEAM_SCHED_H
