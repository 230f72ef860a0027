// paged_layout.h — page tables, slots and positions of one step from the requests'
// lengths. Included by serve.hip inside namespace mi355fa.
//
// Two running sums over the requests (new tokens, pages taken), then every table
// entry and every token on its own. Bound: the latency of one small launch, and
// for wide tables the bytes of the table.
//
//  * Every workgroup forms both sums itself, from 8 bytes a request, and keeps
//    them in LDS; so one launch does, with nothing passed between workgroups.
//  * A token finds its request by bisection of the first sum.

constexpr int kLayoutThreads = 256;

struct LayoutArgs {
  const int* seq;
  const int* fresh;
  const int* table_in;
  const int* free_pages;
  int* kv_lens;
  int* cu;
  int* positions;
  int64_t* slots;
  int* table;
  int* counts;
  int64_t ts;
  int n, cols, n_free, page, max_tokens;
};

// Exclusive sum over the workgroup's threads of a pair; total: of all.
__device__ __forceinline__ void layout_scan(int64_t& x, int64_t& y, int64_t& tx, int64_t& ty, int64_t (*red)[2]) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int64_t ix = x, iy = y;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int64_t px = __shfl_up(ix, d), py = __shfl_up(iy, d);
    if (lane >= d) { ix += px; iy += py; }
  }
  if (lane == 63) { red[wave][0] = ix; red[wave][1] = iy; }
  __syncthreads();
  int64_t bx = 0, by = 0;
  tx = ty = 0;
#pragma unroll
  for (int w = 0; w < kLayoutThreads / 64; ++w) {
    if (w < wave) { bx += red[w][0]; by += red[w][1]; }
    tx += red[w][0];
    ty += red[w][1];
  }
  x = bx + ix - x;
  y = by + iy - y;
}

__global__ __launch_bounds__(kLayoutThreads) void paged_layout_kernel(const LayoutArgs a) {
  extern __shared__ int lay[];   // [n + 1] first token, [n] first page of each request
  int* s_cu = lay;
  int* s_at = lay + a.n + 1;
  __shared__ int64_t red[kLayoutThreads / 64][2];
  __shared__ int64_t red2[kLayoutThreads / 64][2];
  const int tid = threadIdx.x;
  const bool head = blockIdx.x == 0;
  auto pages = [&](int64_t tokens) { return (tokens + a.page - 1) / a.page; };
  // each thread a run of requests
  const int per = (a.n + kLayoutThreads - 1) / kLayoutThreads;
  const int r0 = min(a.n, tid * per), r1 = min(a.n, r0 + per);
  int64_t toks = 0, grow = 0, want = 0;
  for (int r = r0; r < r1; ++r) {
    const int64_t seq = max(a.seq[r], 0), add = max(a.fresh[r], 0);
    const int64_t held = pages(seq), need = pages(seq + add);
    toks += add;
    grow += max((int64_t)0, min(need, (int64_t)a.cols) - held);
    want += need - held;
  }
  int64_t at_t = toks, at_p = grow, all_t, all_p;
  layout_scan(at_t, at_p, all_t, all_p, red);
  for (int r = r0; r < r1; ++r) {
    const int64_t seq = max(a.seq[r], 0), add = max(a.fresh[r], 0);
    const int64_t held = pages(seq), need = pages(seq + add);
    s_cu[r] = (int)min(at_t, (int64_t)INT32_MAX);
    s_at[r] = (int)min(at_p, (int64_t)INT32_MAX);
    if (head) {
      a.kv_lens[r] = (int)min(seq + add, (int64_t)INT32_MAX);
      a.cu[r] = s_cu[r];
    }
    at_t += add;
    at_p += max((int64_t)0, min(need, (int64_t)a.cols) - held);
  }
  if (tid == 0) s_cu[a.n] = (int)min(all_t, (int64_t)INT32_MAX);
  if (head) {
    int64_t x = want, y = 0, tx, ty;
    layout_scan(x, y, tx, ty, red2);
    if (tid == 0) {
      const int64_t taken = min(all_p, (int64_t)a.n_free);
      a.cu[a.n] = s_cu[a.n];
      a.counts[0] = s_cu[a.n];
      a.counts[1] = (int)taken;
      a.counts[2] = (int)min(tx - taken, (int64_t)INT32_MAX);
    }
  }
  __syncthreads();

  // entry c of request r's table
  auto entry = [&](int r, int64_t c, int64_t held, int64_t need) -> int {
    if (c >= need) return -1;
    if (c < held) return a.table_in[(int64_t)r * a.ts + c];
    const int64_t nth = s_at[r] + (c - held);
    return nth < a.n_free ? a.free_pages[nth] : -1;
  };
  const int64_t step = (int64_t)gridDim.x * kLayoutThreads;
  const int64_t me = (int64_t)blockIdx.x * kLayoutThreads + tid;
  for (int64_t x = me; x < (int64_t)a.n * a.cols; x += step) {
    const int r = (int)(x / a.cols), c = (int)(x - (int64_t)r * a.cols);
    const int64_t seq = max(a.seq[r], 0), add = max(a.fresh[r], 0);
    a.table[x] = entry(r, c, pages(seq), min(pages(seq + add), (int64_t)a.cols));
  }
  for (int64_t x = me; x < a.max_tokens; x += step) {
    int pos = 0;
    int64_t slot = -1;
    if (x < s_cu[a.n]) {
      int lo = 0, hi = a.n;   // the last request that starts at or before the token
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (s_cu[mid] <= x) lo = mid;
        else hi = mid;
      }
      const int64_t seq = max(a.seq[lo], 0), add = max(a.fresh[lo], 0);
      const int64_t p = seq + (x - s_cu[lo]);
      pos = (int)min(p, (int64_t)INT32_MAX);
      const int64_t c = p / a.page;
      const int e = c < a.cols ? entry(lo, c, pages(seq), min(pages(seq + add), (int64_t)a.cols)) : -1;
      if (e >= 0) slot = (int64_t)e * a.page + (p - c * a.page);
    }
    a.positions[x] = pos;
    a.slots[x] = slot;
  }
}
