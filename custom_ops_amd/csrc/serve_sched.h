// serve_sched.h — how the serving kernels share out their work: integer rules that the
// device evaluates and host tests check.
//
// Host-compilable on purpose (plain C++, no HIP types): tests/test_serve_sched.py builds
// a host program from this header with g++.
#ifndef MI355_SERVE_SCHED_H
#define MI355_SERVE_SCHED_H

#include <limits.h>
#include <stdint.h>

#include "bits.h"

namespace mi355fa {

MI355_HD inline int imin(int a, int b) { return a < b ? a : b; }
MI355_HD inline int imax(int a, int b) { return a > b ? a : b; }

constexpr int kNoWindow = 1 << 30;   // a window that hides nothing

// ── packed attention: row blocks in classes by length ────────────────────────
// A sequence of `rows` rows and lk keys; its blocks are of 2^shift rows.
struct RowSpans {
  int causal, window, shift;   // window: kNoWindow where there is none
};
MI355_HD inline int block_count(const RowSpans& s, int rows) { return (int)(((int64_t)rows + (1 << s.shift) - 1) >> s.shift); }
// Keys that block b spans, about; the same or more for later blocks.
MI355_HD inline int block_span(const RowSpans& s, int rows, int lk, int b) {
  if (!s.causal) return s.window > lk / 2 ? lk : 2 * s.window;
  const int64_t hi = ((int64_t)(b + 1) << s.shift) + lk - rows;
  return imax(0, imin((int)(hi < lk ? hi : lk), s.window));
}
// The first block that spans more than lim (block_count where none does).
MI355_HD inline int first_over(const RowSpans& s, int rows, int lk, int lim) {
  const int n = block_count(s, rows);
  if (n == 0 || block_span(s, rows, lk, n - 1) <= lim) return n;
  if (block_span(s, rows, lk, 0) > lim) return 0;
  return imin(n, (int)((lim - ((int64_t)lk - rows)) >> s.shift));   // causal: (b + 1)·2^shift + lk − rows > lim
}
// Class `level` of `levels` holds the blocks that span more than class_floor and at most
// class_ceil, half of the class before; the last holds the rest. most: the largest span.
MI355_HD inline int class_floor(int most, int level, int levels) { return level == levels - 1 ? -1 : most >> (level + 1); }
MI355_HD inline int class_ceil(int most, int level) { return level == 0 ? INT_MAX : most >> level; }

// Workgroups of ranks [fold, 2·fold) of `ranks` take their blocks in reverse order (fold 0:
// none): the first `fold` ranks give every CU its first workgroup.
MI355_HD inline int folded(int rank, int fold, int ranks) {
  const int end = imin(2 * fold, ranks);
  return rank >= fold && rank < end ? fold + end - 1 - rank : rank;
}

// ── paged decode: parts of requests ──────────────────────────────────────────
constexpr int kDecTile = 32;   // keys per tile

struct KeySpan {
  int len, first, tile0, tiles;   // seen keys [first, len), the tiles they lie in
};
MI355_HD inline KeySpan key_span(int len, int64_t cap, int window) {
  KeySpan k;
  k.len = imax(0, (int)(len < cap ? len : cap));
  k.first = imax(0, k.len - window);
  k.tile0 = k.first / kDecTile;
  k.tiles = (k.len + kDecTile - 1) / kDecTile - k.tile0;
  return k;
}
// What a request counts for in the sum of all tiles: 2^20 at most (2^25 keys), so that
// the sum of kDecMaxScan requests stays below 2^31.
constexpr int kDecMaxScan = 1024;
MI355_HD inline int weighed(int tiles) { return imin(tiles, 1 << 20); }
// Tiles of a part, for about `target` parts of `groups` head groups each; sum: of weighed
// tiles. At most target + requests·groups parts come of it.
MI355_HD inline int part_size(int sum, int groups, int target, int least) {
  const int64_t per = ((int64_t)sum * groups + target - 1) / target;
  return (int)(per > least ? per : least);
}
MI355_HD inline int part_count(int tiles, int per) { return imax(1, (weighed(tiles) + per - 1) / per); }
// Part p of n takes tiles [part_start(p), part_start(p + 1)) of a request's.
MI355_HD inline int part_start(int tiles, int n, int p) { return (int)((int64_t)((tiles + n - 1) / n) * p < tiles ? (tiles + n - 1) / n * p : tiles); }

}  // namespace mi355fa

#endif  // MI355_SERVE_SCHED_H
