// page_ops.h — forking, compacting and copying of a cache's pages. Included by beam.hip
// inside namespace mi355fa.
//
// Which pages are in use follows from the table alone: a bit a page. The first kernel's
// workgroups each take some rows, set the bits of their pages in LDS and write their
// bitmaps down; the second's all join the bitmaps, so that each has the whole, and form
// the running count of bits from which a page's rank, and the page of a rank, follow. Few
// rows are one workgroup's, which does both.
// Bound: a launch, and the waits that follow one another. Measured in a graph: a fork of 4 rows 5.0
// us, of 512 with 512 columns and 49000 pages 14.9 (marks 5.0, the rest 10.2: two bitmaps joined,
// two running counts, a hash of the last pages); compacting 8 rows 5.1 us, 500 of 257 columns over
// 84000 pages 15.5 (marks 4.2, the rest 12.1, of which joining the bitmaps 2.9, the counts 1.6, the
// table's searches 1.8). A bit a page in LDS needs no clearing between calls, as one map in memory would.

constexpr int kPgThreads = 1024;
constexpr int kPgRows = 4096;            // rows of a fork: a bit each, and a hash of their last pages
constexpr int kPgHash = 2 * kPgRows;
constexpr int kPgColumns = 256;          // of a row, that a wave compacts at once

struct PageArgs {
  const int* table_in;
  const int* seq;
  const int* parents;    // fork: the old row of each new one; NULL: each its own
  const int* held;
  int* table;
  int* lens;
  int* src;
  int* dst;
  int* remap;
  int* free_pages;
  int* counts;
  uint32_t* maps;        // [marks][2][words]: pages of any kind; of whole ones and held
  int64_t ts;
  int n, r, cols, pages, page, n_held;
  int words;             // of a bitmap: pages / 32, up to a multiple of 4
  int marks;             // workgroups of the first kernel
};

// Row i of the new table: its old row (-1: none) and its length.
__device__ __forceinline__ int old_row(const PageArgs& a, int i, int& len) {
  const int64_t most = (int64_t)a.cols * a.page;
  const int row = a.parents ? a.parents[i] : i;
  const bool real = row >= 0 && row < a.n;
  len = real ? max(a.seq[row], 0) : 0;
  if (len > most) len = (int)most;
  return real ? row : -1;
}

// Marks of the pages of rows first, first + step, .. (a wave each) and of the held ones, for a
// fork of whole ones apart, and of a fork the new table. Bitmaps: cleared, of whole ones behind any.
template <bool FORK> __device__ __forceinline__ void mark_rows(const PageArgs& a, uint32_t* any, uint32_t* whole, int first, int step, bool held) {
  const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6);
  if (held)
    for (int i = tid; i < a.n_held; i += kPgThreads) {
      const int p = a.held[i];
      if (p >= 0 && p < a.pages) {
        atomicOr(&any[p >> 5], 1u << (p & 31));
        if (FORK) atomicOr(&whole[p >> 5], 1u << (p & 31));
      }
    }
  for (int i = first + wave; i < a.r; i += step) {
    int len;
    const int row = old_row(a, i, len);
    const int used = (int)(((int64_t)len + a.page - 1) / a.page), full = len / a.page;
    const int* from = a.table_in + (int64_t)max(row, 0) * a.ts;
    int* to = a.table + (int64_t)i * a.cols;
    for (int c0 = lane; c0 < (FORK ? a.cols : used); c0 += 256) {
      int p[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) p[e] = c0 + e * 64 < used ? from[c0 + e * 64] : -1;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int c = c0 + e * 64, x = p[e] >= 0 && p[e] < a.pages ? p[e] : -1;
        if (x >= 0) {
          atomicOr(&any[x >> 5], 1u << (x & 31));
          if (FORK && c < full) atomicOr(&whole[x >> 5], 1u << (x & 31));
        }
        if (FORK && c < a.cols) to[c] = x;
      }
    }
  }
  __syncthreads();
}

template <bool FORK>
__global__ __launch_bounds__(kPgThreads) void page_mark_kernel(const PageArgs a) {
  extern __shared__ __align__(16) uint32_t bits[];   // [2][words]
  const int tid = threadIdx.x;
  for (int i = tid; i < (FORK ? 2 : 1) * a.words; i += kPgThreads) bits[i] = 0;
  __syncthreads();
  mark_rows<FORK>(a, bits, bits + a.words, blockIdx.x * (kPgThreads / 64), gridDim.x * (kPgThreads / 64), blockIdx.x == 0);
  uint32_t* out = a.maps + (int64_t)blockIdx.x * 2 * a.words;
  for (int i = tid; i < (FORK ? 2 : 1) * a.words; i += kPgThreads) out[i] = bits[i];
}

// The bitmap of all workgroups: a thread takes 16 bytes of every so many of them, 16 asked for at once.
__device__ __forceinline__ void joined(const PageArgs& a, int which, uint32_t* bits) {
  for (int i = threadIdx.x; i < a.words; i += kPgThreads) bits[i] = 0;
  __syncthreads();
  const int quads = a.words / 4, ways = max(1, min(kPgThreads / quads, a.marks));
  for (int x = threadIdx.x; x < quads * ways; x += kPgThreads) {
    const int m0 = (int)((uint32_t)x / (uint32_t)quads), q = x - m0 * quads;
    const u32x4* from = reinterpret_cast<const u32x4*>(a.maps + (int64_t)which * a.words) + q;
    u32x4 y = {0u, 0u, 0u, 0u};
    for (int m = m0; m < a.marks; m += 16 * ways) {
      u32x4 z[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) z[e] = from[(int64_t)min(m + e * ways, a.marks - 1) * 2 * quads];   // (the last one's bits belong in all)
#pragma unroll
      for (int e = 0; e < 16; ++e) y |= z[e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (y[e]) atomicOr(&bits[q * 4 + e], y[e]);
  }
  __syncthreads();
}

// before[i]: set bits in words below i, of the first `pages` bits; returns all of them.
__device__ __forceinline__ int ranks(const uint32_t* bits, int* before, int words, int* sums) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int per = (words + kPgThreads - 1) / kPgThreads;
  int mine = 0;
  for (int e = 0; e < per; ++e) {
    const int i = tid * per + e;
    if (i < words) mine += __builtin_popcount(bits[i]);
  }
  const int incl = wave_scan(mine);
  if (lane == 63) sums[wave] = incl;
  __syncthreads();
  int run = incl - mine, all = 0;
#pragma unroll
  for (int w = 0; w < kPgThreads / 64; ++w) {
    if (w < wave) run += sums[w];
    all += sums[w];
  }
  for (int e = 0; e < per; ++e) {
    const int i = tid * per + e;
    if (i < words) {
      before[i] = run;
      run += __builtin_popcount(bits[i]);
    }
  }
  __syncthreads();
  return all;
}
// Set bits below bit p.
__device__ __forceinline__ int rank_of(const uint32_t* bits, const int* before, int p) {
  return before[p >> 5] + __builtin_popcount(bits[p >> 5] & ((1u << (p & 31)) - 1u));
}
// Where every 64th clear bit lies: the word of the (64·i)-th in start[i], and behind the last
// one the last word (a bitmap's words / 2 + 1 of them). All threads.
__device__ __forceinline__ void clear_index(const uint32_t* bits, const int* before, int words, uint16_t* start) {
  const int all = 32 * words - before[words - 1] - __builtin_popcount(bits[words - 1]);
  for (int i = threadIdx.x; i < words; i += kPgThreads) {
    const int c0 = 32 * i - before[i], c1 = c0 + 32 - __builtin_popcount(bits[i]), at = (c0 + 63) / 64;
    if (at * 64 < c1) start[at] = (uint16_t)i;   // (32 at most: one, if any)
  }
  if (threadIdx.x == 0) start[(all + 63) / 64] = (uint16_t)(words - 1);
  __syncthreads();
}
// j: in, which clear bit of [0, their number); out, its page. N at once, so that their steps wait
// for LDS together.
template <int N> __device__ __forceinline__ void clear_of(const uint32_t* bits, const int* before, const uint16_t* start, int (&j)[N]) {
  int lo[N], hi[N];   // the last word with at most j clear bits below it is of [lo, hi]
  bool more = false;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    lo[e] = start[j[e] >> 6];
    hi[e] = start[(j[e] >> 6) + 1];
    more |= lo[e] < hi[e];
  }
  while (__builtin_amdgcn_ballot_w64(more)) {
    more = false;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int mid = (lo[e] + hi[e] + 1) / 2;
      const bool up = 32 * mid - before[mid] <= j[e];
      lo[e] = up ? mid : lo[e];
      hi[e] = up || lo[e] == hi[e] ? hi[e] : mid - 1;
      more |= lo[e] < hi[e];
    }
  }
#pragma unroll
  for (int e = 0; e < N; ++e) {
  // the bit of its word by halves
    uint32_t x = ~bits[lo[e]];
    int left = j[e] - (32 * lo[e] - before[lo[e]]), at = 0;
#pragma unroll
    for (int half = 16; half; half /= 2) {
      const int low = __builtin_popcount(x & ((1u << half) - 1u));
      const bool up = left >= low;
      left -= up ? low : 0;
      at += up ? half : 0;
      x >>= up ? half : 0;
    }
    j[e] = 32 * lo[e] + at;
  }
}

// What a fork adds to the table: pages for the rows that cannot keep their last one. All
// workgroups find the same; the first writes the rows' results, each its share of the free pages.
// ONE: the only workgroup, which marks the rows itself.
template <bool ONE>
__global__ __launch_bounds__(kPgThreads) void page_fork_kernel(const PageArgs a) {
  extern __shared__ __align__(16) uint32_t bits[];   // [words] of whole pages, then of any; beside it a hash, then [words] ranks and where to look for clear bits
  __shared__ uint32_t wants[kPgRows / 32];
  __shared__ int wants_before[kPgRows / 32], sums[kPgThreads / 64];
  int* key = reinterpret_cast<int*>(bits + a.words);
  int* low = key + kPgHash;
  int* before = key;
  uint16_t* start = reinterpret_cast<uint16_t*>(before + a.words);
  uint32_t* any = ONE ? bits + a.words + 2 * kPgHash : bits;
  const int tid = threadIdx.x;
  // each row's last page, if it is partly filled (asked for first, and met behind the bitmaps)
  constexpr int E = kPgRows / kPgThreads;
  int page[E], place[E], col[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int i = e * kPgThreads + tid;
    page[e] = -1;
    place[e] = col[e] = 0;
    if (i < a.r) {
      int len;
      const int row = old_row(a, i, len);
      if (blockIdx.x == 0) a.lens[i] = len;
      if (len % a.page) {
        col[e] = len / a.page;
        page[e] = a.table_in[(int64_t)row * a.ts + col[e]];
      }
    }
  }
  for (int i = tid; i < kPgHash; i += kPgThreads) {
    key[i] = -1;
    low[i] = INT_MAX;
  }
  for (int i = tid; i < kPgRows / 32; i += kPgThreads) wants[i] = 0;
  if constexpr (ONE) {
    for (int i = tid; i < a.words; i += kPgThreads) any[i] = bits[i] = 0;
    __syncthreads();
    mark_rows<true>(a, any, bits, 0, kPgThreads / 64, true);
  } else joined(a, 1, bits);
  // the lowest row of those that have a page so
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int i = e * kPgThreads + tid;
    if (page[e] >= a.pages) page[e] = -1;
    if (page[e] >= 0) {
      uint32_t h = ((uint32_t)page[e] * 2654435761u) >> 19;   // 13 bits
      for (;;) {
        const int was = atomicCAS(&key[h], -1, page[e]);
        if (was == -1 || was == page[e]) break;
        h = (h + 1) & (kPgHash - 1);
      }
      place[e] = (int)h;
      atomicMin(&low[h], i);
    }
  }
  static_assert(kPgHash == 1 << 13, "the hash takes 13 bits");
  __syncthreads();
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int i = e * kPgThreads + tid;
    if (page[e] >= 0 && (low[place[e]] != i || (bits[page[e] >> 5] >> (page[e] & 31) & 1))) atomicOr(&wants[i >> 5], 1u << (i & 31));
  }
  __syncthreads();
  const int wanted = ranks(wants, wants_before, kPgRows / 32, sums);
  if constexpr (!ONE) joined(a, 0, any);
  const int used = ranks(any, before, a.words, sums), left = a.pages - used, taken = min(wanted, left);
  if (blockIdx.x == 0) {
    clear_index(any, before, a.words, start);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int i = e * kPgThreads + tid;
      if (i >= a.r) continue;
      int from = -1, to = -1;
      if (wants[i >> 5] >> (i & 31) & 1) {
        const int nth = rank_of(wants, wants_before, i);
        if (nth < left) {
          int x[1] = {nth};
          clear_of(any, before, start, x);
          from = page[e];
          to = x[0];
        }
        a.table[(int64_t)i * a.cols + col[e]] = to;
      }
      a.src[i] = from;
      a.dst[i] = to;
    }
    if (tid == 0) {
      a.counts[0] = left - taken;
      a.counts[1] = taken;
      a.counts[2] = wanted - taken;
    }
  }
  for (int p = blockIdx.x * kPgThreads + tid; p < a.pages; p += gridDim.x * kPgThreads) {
    if (!(any[p >> 5] >> (p & 31) & 1)) {
      const int nth = p - rank_of(any, before, p) - taken;
      if (nth >= 0) a.free_pages[nth] = p;
    }
    if (p >= left - taken) a.free_pages[p] = -1;
  }
}

// The new numbers, the moves, and the table by them; each workgroup its shares. ONE: as above.
template <bool ONE>
__global__ __launch_bounds__(kPgThreads) void page_compact_kernel(const PageArgs a) {
  extern __shared__ __align__(16) uint32_t bits[];   // [words], [words] ranks, and where to look for clear bits
  __shared__ int sums[kPgThreads / 64];
  int* before = reinterpret_cast<int*>(bits + a.words);
  constexpr int C = ONE ? 64 : kPgColumns;   // (few rows are bound by the code they fetch)
  const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6);
  // Rows of the table, C columns a wave at once; the first are asked for before others' bitmaps.
  const int chunks = (a.cols + C - 1) / C, units = a.n * chunks, step = gridDim.x * (kPgThreads / 64);
  int w = blockIdx.x * (kPgThreads / 64) + wave, p[C / 64];
  auto load = [&]() __attribute__((always_inline)) {
    if (w >= units) return;
    const int i = (int)((uint32_t)w / (uint32_t)chunks), c0 = (w - i * chunks) * C + lane;
    int len;
    old_row(a, i, len);
    const int held = (int)(((int64_t)len + a.page - 1) / a.page);
#pragma unroll
    for (int e = 0; e < C / 64; ++e) {
      const int c = c0 + e * 64;
      p[e] = c < held ? a.table_in[(int64_t)i * a.ts + c] : -1;
    }
  };
  auto next = [&]() __attribute__((always_inline)) {
    w += step;
    load();
  };
  if constexpr (ONE) {
    for (int i = tid; i < a.words; i += kPgThreads) bits[i] = 0;
    __syncthreads();
    mark_rows<false>(a, bits, nullptr, 0, kPgThreads / 64, true);
    load();   // (from the cache by now)
  } else {
    load();
    joined(a, 0, bits);
  }
  const int used = ranks(bits, before, a.words, sums);
  uint16_t* start = reinterpret_cast<uint16_t*>(before + a.words);
  clear_index(bits, before, a.words, start);
  const int stay = used < a.pages ? rank_of(bits, before, used) : used, moved = used - stay;   // pages below `used`
  // The new numbers of N pages (-1: none): those below `used` stay, the others fill the gaps there.
  auto numbers = [&](auto& p) __attribute__((always_inline)) {
    constexpr int N = sizeof(p) / sizeof(int);
    int j[N];
    bool gap = false;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      if (p[e] < 0 || p[e] >= a.pages || !(bits[p[e] >> 5] >> (p[e] & 31) & 1)) p[e] = -1;
      j[e] = p[e] < used ? 0 : rank_of(bits, before, p[e]) - stay;
      gap |= p[e] >= used;
    }
    if (!__builtin_amdgcn_ballot_w64(gap)) return;
    clear_of(bits, before, start, j);
#pragma unroll
    for (int e = 0; e < N; ++e) p[e] = p[e] < used ? p[e] : j[e];
  };
  for (int p = blockIdx.x * kPgThreads + tid; p < a.pages; p += gridDim.x * kPgThreads) {
    int x[1] = {p};
    numbers(x);
    const int to = x[0];
    a.remap[p] = to;
    if (p >= used && to >= 0) {
      const int j = rank_of(bits, before, p) - stay;
      a.src[j] = p;
      a.dst[j] = to;
    }
    if (p >= moved && p < a.pages / 2) a.src[p] = a.dst[p] = -1;
    a.free_pages[p] = p < a.pages - used ? used + p : -1;
  }
  if (blockIdx.x == 0 && tid == 0) {
    a.counts[0] = used;
    a.counts[1] = moved;
  }
  for (; w < units; next()) {
    numbers(p);
    const int i = (int)((uint32_t)w / (uint32_t)chunks), c0 = (w - i * chunks) * C + lane;
#pragma unroll
    for (int e = 0; e < C / 64; ++e) {
      const int c = c0 + e * 64;
      if (c < a.cols) a.table[(int64_t)i * a.cols + c] = p[e];
    }
  }
}

struct CopyArgs {
  uint16_t* k;
  uint16_t* v;
  const int* src;
  const int* dst;
  int64_t kp, kh, kr, vp, vh, vr;
  int n, pages, hk, page, chunks;   // chunks: 16-byte ones of a row
  int pieces, units;                // a page's 16-byte units, and pieces of kCopyUnits of them
  int dense;                        // a page's rows lie one after the other in both caches
};

// A wave copies a piece of one page of one cache: kCopyUnits 16-byte units, all loaded
// before any is stored. Bound: bytes, read and written (2000 pages of 8 heads, 64 rows of 128: 213
// us, 4.9 TB/s; 67 small ones 2.7 us).
constexpr int kCopyLoads = 4, kCopyUnits = 64 * kCopyLoads, kCopyThreads = 256;
__global__ __launch_bounds__(kCopyThreads) void page_copy_kernel(const CopyArgs a) {
  const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6);
  const int waves = gridDim.x * (kCopyThreads / 64);
  const int total = a.n * 2 * a.pieces;
  for (int64_t w = blockIdx.x * (kCopyThreads / 64) + wave; w < total; w += waves) {
    const int x = (int)w, pair = x / (2 * a.pieces), rest = x - pair * 2 * a.pieces;
    const int src = uni(a.src[pair]), dst = uni(a.dst[pair]);
    if (src < 0 || src >= a.pages || dst < 0 || dst >= a.pages) continue;
    const bool second = rest >= a.pieces;
    const int unit0 = (second ? rest - a.pieces : rest) * kCopyUnits + lane;
    uint16_t* base = second ? a.v : a.k;
    const int64_t ps = second ? a.vp : a.kp, hs = second ? a.vh : a.kh, rs = second ? a.vr : a.kr;
    const uint16_t* from = base + src * ps;
    uint16_t* to = base + dst * ps;
    u32x4 y[kCopyLoads];
    int64_t off[kCopyLoads];
#pragma unroll
    for (int i = 0; i < kCopyLoads; ++i) {
      const int u = unit0 + i * 64;
      off[i] = (int64_t)u * 8;
      if (!a.dense) {
        const int r = u / a.chunks, head = r / a.page;
        off[i] = head * hs + (r - head * a.page) * rs + (u - r * a.chunks) * 8;
      }
      if (u < a.units) y[i] = *reinterpret_cast<const u32x4*>(from + off[i]);
    }
#pragma unroll
    for (int i = 0; i < kCopyLoads; ++i)
      if (unit0 + i * 64 < a.units) *reinterpret_cast<u32x4*>(to + off[i]) = y[i];
  }
}
