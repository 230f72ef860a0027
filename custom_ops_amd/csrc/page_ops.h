// page_ops.h — forking, compacting and copying of a cache's pages. Included by beam.hip
// inside namespace mi355fa.
//
// Which pages are in use follows from the table alone: a bit a page. The first kernel's
// workgroups each take some rows, set the bits of their pages in LDS and write their
// bitmaps down; the second's all join the bitmaps, so that each has the whole, and form
// the running count of bits from which a page's rank, and the page of a rank, follow.
// Bound: the bytes of the tables, and for small ones two launches.

constexpr int kPgThreads = 1024;
constexpr int kPgRows = 4096;            // rows of a fork: a bit each, and a hash of their last pages
constexpr int kPgHash = 2 * kPgRows;

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
  int words;             // of a bitmap: pages / 32, up
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

// Rows of each workgroup: marks of their pages, and for a fork the new table.
template <bool FORK>
__global__ __launch_bounds__(kPgThreads) void page_mark_kernel(const PageArgs a) {
  extern __shared__ uint32_t bits[];   // [2][words]
  uint32_t* any = bits;
  uint32_t* whole = bits + a.words;
  const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6), wgs = gridDim.x;
  for (int i = tid; i < 2 * a.words; i += kPgThreads) bits[i] = 0;
  __syncthreads();
  if (blockIdx.x == 0)
    for (int i = tid; i < a.n_held; i += kPgThreads) {
      const int p = a.held[i];
      if (p >= 0 && p < a.pages) {
        atomicOr(&any[p >> 5], 1u << (p & 31));
        atomicOr(&whole[p >> 5], 1u << (p & 31));
      }
    }
  // a wave a row
  for (int i = blockIdx.x * (kPgThreads / 64) + wave; i < a.r; i += wgs * (kPgThreads / 64)) {
    int len;
    const int row = old_row(a, i, len);
    const int used = (int)(((int64_t)len + a.page - 1) / a.page), full = len / a.page;
    const int* from = a.table_in + (int64_t)max(row, 0) * a.ts;
    int* to = a.table + (int64_t)i * a.cols;
    for (int c = lane; c < (FORK ? a.cols : used); c += 64) {
      int p = c < used ? from[c] : -1;
      if (p >= a.pages) p = -1;
      if (p >= 0) {
        atomicOr(&any[p >> 5], 1u << (p & 31));
        if (FORK && c < full) atomicOr(&whole[p >> 5], 1u << (p & 31));
      }
      if (FORK) to[c] = p < 0 ? -1 : p;
    }
  }
  __syncthreads();
  uint32_t* out = a.maps + (int64_t)blockIdx.x * 2 * a.words;
  for (int i = tid; i < (FORK ? 2 : 1) * a.words; i += kPgThreads) out[i] = bits[i];
}

// The bitmap of all workgroups.
__device__ __forceinline__ void joined(const PageArgs& a, int which, uint32_t* bits) {
  for (int i = threadIdx.x; i < a.words; i += kPgThreads) {
    uint32_t x = 0;
#pragma unroll 8
    for (int m = 0; m < a.marks; ++m) x |= a.maps[((int64_t)m * 2 + which) * a.words + i];
    bits[i] = x;
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
// The page of the j-th clear bit (j below their number).
__device__ __forceinline__ int clear_of(const uint32_t* bits, const int* before, int words, int j) {
  int lo = 0, hi = words - 1;   // the last word with at most j clear bits below it
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (32 * mid - before[mid] <= j) lo = mid;
    else hi = mid - 1;
  }
  uint32_t x = ~bits[lo];
  for (int left = j - (32 * lo - before[lo]); left > 0; --left) x &= x - 1;
  return 32 * lo + __builtin_ctz(x);
}

// What a fork adds to the table: pages for the rows that cannot keep their last one. All
// workgroups find the same; the first writes the rows' results, each its share of the free pages.
__global__ __launch_bounds__(kPgThreads) void page_fork_kernel(const PageArgs a) {
  extern __shared__ uint32_t bits[];   // [words] of whole pages, then of any; beside it a hash, then [words] ranks
  __shared__ uint32_t wants[kPgRows / 32];
  __shared__ int wants_before[kPgRows / 32], sums[kPgThreads / 64];
  int* key = reinterpret_cast<int*>(bits + a.words);
  int* low = key + kPgHash;
  int* before = key;
  const int tid = threadIdx.x;
  for (int i = tid; i < kPgHash; i += kPgThreads) {
    key[i] = -1;
    low[i] = INT_MAX;
  }
  for (int i = tid; i < kPgRows / 32; i += kPgThreads) wants[i] = 0;
  joined(a, 1, bits);
  // each row's last page, if it is partly filled: the lowest row of those that have it so
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
        if (page[e] >= a.pages) page[e] = -1;
      }
    }
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
  joined(a, 0, bits);
  const int used = ranks(bits, before, a.words, sums), left = a.pages - used, taken = min(wanted, left);
  if (blockIdx.x == 0) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int i = e * kPgThreads + tid;
      if (i >= a.r) continue;
      int from = -1, to = -1;
      if (wants[i >> 5] >> (i & 31) & 1) {
        const int nth = rank_of(wants, wants_before, i);
        if (nth < left) {
          from = page[e];
          to = clear_of(bits, before, a.words, nth);
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
    if (!(bits[p >> 5] >> (p & 31) & 1)) {
      const int nth = p - rank_of(bits, before, p) - taken;
      if (nth >= 0) a.free_pages[nth] = p;
    }
    if (p >= left - taken) a.free_pages[p] = -1;
  }
}

// The new numbers, the moves, and the table by them; each workgroup its shares.
__global__ __launch_bounds__(kPgThreads) void page_compact_kernel(const PageArgs a) {
  extern __shared__ uint32_t bits[];   // [words], [words] ranks
  __shared__ int sums[kPgThreads / 64];
  int* before = reinterpret_cast<int*>(bits + a.words);
  const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6);
  joined(a, 0, bits);
  const int used = ranks(bits, before, a.words, sums);
  const int stay = used < a.pages ? rank_of(bits, before, used) : used, moved = used - stay;   // pages below `used`
  auto number = [&](int p) {
    if (!(bits[p >> 5] >> (p & 31) & 1)) return -1;
    return p < used ? p : clear_of(bits, before, a.words, rank_of(bits, before, p) - stay);
  };
  for (int p = blockIdx.x * kPgThreads + tid; p < a.pages; p += gridDim.x * kPgThreads) {
    const int to = number(p);
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
  for (int i = blockIdx.x * (kPgThreads / 64) + wave; i < a.n; i += gridDim.x * (kPgThreads / 64)) {
    int len;
    old_row(a, i, len);
    const int held = (int)(((int64_t)len + a.page - 1) / a.page);
    for (int c = lane; c < a.cols; c += 64) {
      const int p = c < held ? a.table_in[(int64_t)i * a.ts + c] : -1;
      a.table[(int64_t)i * a.cols + c] = p >= 0 && p < a.pages ? number(p) : -1;
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
// before any is stored. Bound: bytes, read and written.
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
