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

// A request's tokens before and after the step, and the pages of both. (Two lengths
// below 2^31 have a sum below 2^32: 32-bit divisions do, a 64-bit one takes 100
// instructions.)
struct LayoutReq {
  uint32_t seq, add, held, want;
};
__device__ __forceinline__ LayoutReq layout_req(const LayoutArgs& a, int seq, int add) {
  auto pages = [&](uint32_t tokens) { return tokens / (uint32_t)a.page + (tokens % (uint32_t)a.page != 0); };
  LayoutReq q;
  q.seq = (uint32_t)max(seq, 0);
  q.add = (uint32_t)max(add, 0);
  q.held = pages(q.seq);
  q.want = pages(q.seq + q.add);
  return q;
}

__global__ __launch_bounds__(kLayoutThreads) void paged_layout_kernel(const LayoutArgs a) {
  extern __shared__ int lay[];   // [n + 1] first token, [n] first page of each request
  int* s_cu = lay;
  int* s_at = lay + a.n + 1;
  __shared__ int64_t red[kLayoutThreads / 64][2];
  __shared__ int64_t red2[kLayoutThreads / 64][2];
  const int tid = threadIdx.x, lane = tid & 63;
  const bool head = blockIdx.x == 0;
  auto grow_of = [&](const LayoutReq& q) { return (int)max((int64_t)0, (int64_t)min(q.want, (uint32_t)a.cols) - q.held); };
  // each thread a run of requests; their own numbers in LDS, then the sums before them
  const int per = (a.n + kLayoutThreads - 1) / kLayoutThreads;
  const int r0 = min(a.n, tid * per), r1 = min(a.n, r0 + per);
  int64_t toks = 0, grow = 0, wanted = 0;
  constexpr int J = 4;   // loads in flight
  for (int b = r0; b < r1; b += J) {
    int seq[J], add[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      seq[j] = a.seq[min(b + j, r1 - 1)];
      add[j] = a.fresh[min(b + j, r1 - 1)];
    }
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int r = b + j;
      if (r >= r1) break;
      const LayoutReq q = layout_req(a, seq[j], add[j]);
      const int g = grow_of(q);
      s_cu[r] = (int)q.add;
      s_at[r] = g;
      toks += q.add;
      grow += g;
      wanted += q.want - q.held;
      if (head) a.kv_lens[r] = (int)min(q.seq + q.add, (uint32_t)INT32_MAX);
    }
  }
  int64_t at_t = toks, at_p = grow, all_t, all_p;
  layout_scan(at_t, at_p, all_t, all_p, red);
  for (int r = r0; r < r1; ++r) {
    const int add = s_cu[r], g = s_at[r];
    s_cu[r] = (int)min(at_t, (int64_t)INT32_MAX);
    s_at[r] = (int)min(at_p, (int64_t)INT32_MAX);
    if (head) a.cu[r] = s_cu[r];
    at_t += add;
    at_p += g;
  }
  if (tid == 0) s_cu[a.n] = (int)min(all_t, (int64_t)INT32_MAX);
  if (head) {
    int64_t x = wanted, y = 0, tx, ty;
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

  // where column c of request r's table comes from: a page held, a free one, or none
  auto entry = [&](int r, uint32_t c, const LayoutReq& q) -> const int* {
    if (c >= q.want) return nullptr;
    if (c < q.held) return a.table_in + (int64_t)r * a.ts + c;
    const uint32_t nth = (uint32_t)s_at[r] + (c - q.held);
    return nth < (uint32_t)a.n_free ? a.free_pages + nth : nullptr;
  };
  // a wave a row of the table, a lane a token
  const int waves = gridDim.x * (kLayoutThreads / 64);
  if (a.cols > 0)
    for (int r = blockIdx.x * (kLayoutThreads / 64) + (tid >> 6); r < a.n; r += waves) {
      const LayoutReq q = layout_req(a, a.seq[r], a.fresh[r]);
      for (int c0 = lane; c0 < a.cols; c0 += 64 * J) {
        int e[J];
        bool ok[J];
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const int c = c0 + 64 * j;
          const int* at = c < a.cols ? entry(r, (uint32_t)c, q) : nullptr;
          ok[j] = at != nullptr;
          e[j] = *(ok[j] ? at : a.seq);   // (no load depends on a branch)
        }
#pragma unroll
        for (int j = 0; j < J; ++j)
          if (c0 + 64 * j < a.cols) a.table[(int64_t)r * a.cols + c0 + 64 * j] = ok[j] ? e[j] : -1;
      }
    }
  const int64_t step = (int64_t)gridDim.x * kLayoutThreads;
  for (int64_t x = (int64_t)blockIdx.x * kLayoutThreads + tid; x < a.max_tokens; x += step) {
    int pos = 0;
    int64_t slot = -1;
    if (x < s_cu[a.n]) {
      int lo = 0, hi = a.n;   // the last request that starts at or before the token
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (s_cu[mid] <= x) lo = mid;
        else hi = mid;
      }
      const LayoutReq q = layout_req(a, a.seq[lo], a.fresh[lo]);
      const uint32_t p = q.seq + (uint32_t)(x - s_cu[lo]);
      pos = (int)min(p, (uint32_t)INT32_MAX);
      const uint32_t c = p / (uint32_t)a.page;
      const int* at = c < (uint32_t)a.cols ? entry(lo, c, q) : nullptr;
      const int e = at ? *at : -1;
      if (e >= 0) slot = (int64_t)e * a.page + (p - c * (uint32_t)a.page);
    }
    a.positions[x] = pos;
    a.slots[x] = slot;
  }
}
