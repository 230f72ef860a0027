// shared_decode.h — attention of one new token per request over a paged cache, of which
// groups of requests share prefixes. Included by beam.hip inside namespace mi355fa.
//
// The softmax over a request's keys is that over its group's common keys joined with that
// over its own: each part gives (max, sum, Σ p·v) in fp32, and a second kernel joins
// them. The common keys are read once for all requests of a group: their heads of one KV
// head are the columns of one matrix product. Bound: the bytes of the prefixes and the
// own keys; the products where many requests share a prefix (4·d operations a key and
// column).
//
//  * The tiles of 32 keys that all requests of a group see whole are shared; what remains
//    of the prefix at its ends belongs to the requests (beam_sched.h). So no column of a
//    shared tile hides a key, and nothing of an unseen key can reach a row.
//  * A workgroup is a part: some tiles of one unit, which is a block of 16·NC columns of a
//    group's (KV head, requests), or a request's 16 heads of a KV head. Each of its 4
//    waves streams every fourth tile: Sᵀ = K·Qᵀ with 16x16x32 MFMAs, K rows straight from
//    the cache into the operand registers and used by all NC column blocks; V rows
//    through the wave's own LDS slice, read transposed once for all NC.
//  * Lengths and offsets stay on the device: every workgroup derives the same plan from
//    them and takes its part; workgroup 0 writes down for the join where parts lie.

constexpr int kShWaves = 4;
constexpr int kShThreads = 64 * kShWaves;
constexpr int kShColumns(int d) { return d == 128 ? 32 : 64; }   // of a workgroup, where groups are of more than 16
constexpr int kShMax = 2048;                   // requests, and groups
constexpr int kShItems = 2 * kShMax / kShThreads;   // groups and requests of a thread

struct SharedArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* o;
  const int* table;
  const int* lens;
  const int* cu;
  const int* prefix;
  const float* slopes;
  int* rec;        // [n_groups + b][4]: first slot, parts of a unit, and of a request its group or -1
  float* part_ml;  // [parts][16·NC][2]: max in log2 units, sum
  float* part_o;   // [parts][16·NC][D]
  int64_t q_bs, q_hs, o_bs, o_hs, kp, kh, kr, vp, vh, vr, ts;
  int b, n_groups, h, hk, ratio;
  int groups;      // 16-head groups per KV head of a request's own keys
  int pages, shift, cols, window;
  int target, least;             // parts to make, about; tiles of a part at least
  int cap;                       // scores are capped
  float u_scale, c2, bias;       // as in PackedArgs
};

// What a workgroup does.
struct Share {
  int group;       // >= 0: shared tiles of it, columns from col0 on; -1: own tiles of request b
  int b;           // the first request of the group, or the request
  int leader;      // the row that names the prefix's pages
  int hk, col0;    // KV head; first column, or first head of the request's
  int cols;        // columns there are
  int prefix;      // keys below it: of the leader's row
  int slot, lo, hi;   // where the part's results go; its tiles [lo, hi) of the unit's
  OwnTiles own;    // a group's tiles: own.first + i
  bool alone;      // the request's only part
};

// The plan. LDS: s, of kShPlan words.
constexpr int kShPlan = 5 * kShMax + 64;
__device__ __forceinline__ bool find_share(const SharedArgs& a, int columns, int w, int* s, Share& sh) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int* len_of = s;                  // [b]
  int* group_of = s + kShMax;       // [b]
  int* least_of = s + 2 * kShMax;   // [n_groups], then tiles t0
  int* most_of = s + 3 * kShMax;    // [n_groups], then tiles t1
  int* members = s + 4 * kShMax;    // [n_groups]
  int* acc = s + 5 * kShMax;        // [64]
  const int64_t span = (int64_t)a.cols << a.shift;
  const int cap = (int)span;
  for (int i = tid; i < a.b; i += kShThreads) {
    len_of[i] = min(max(a.lens[i], 0), cap);
    group_of[i] = -1;
  }
  for (int g = tid; g < a.n_groups; g += kShThreads) {
    least_of[g] = INT_MAX;
    most_of[g] = members[g] = 0;
  }
  __syncthreads();
  // a request's group: the last one that starts at or before it, if it ends behind it
  for (int g = tid; g < a.n_groups; g += kShThreads) {
    const int c = a.cu[g];
    if (c >= 0 && c < a.b) atomicMax(&group_of[c], g);
  }
  __syncthreads();
  constexpr int E = kShMax / kShThreads;
  int mine[E], top = -1;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int i = tid * E + e;
    top = max(top, i < a.b ? group_of[i] : -1);
    mine[e] = top;
  }
  const int upto = wave_max_scan(top);
  if (lane == 63) acc[wave] = upto;
  int before = __shfl_up(upto, 1);
  if (lane == 0) before = -1;
  __syncthreads();
  for (int x = 0; x < wave; ++x) before = max(before, acc[x]);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int i = tid * E + e;
    if (i < a.b) {
      int g = max(mine[e], before);
      if (g >= 0 && i >= a.cu[g + 1]) g = -1;
      group_of[i] = g;
      if (g >= 0) atomicAdd(&members[g], 1);
      if (g >= 0 && len_of[i] > 0) {
        atomicMin(&least_of[g], len_of[i]);
        atomicMax(&most_of[g], len_of[i]);
      }
    }
  }
  __syncthreads();
  for (int g = tid; g < a.n_groups; g += kShThreads) {
    const int c0 = a.cu[g], c1 = min(a.cu[g + 1], a.b);
    TileSpan t{0, 0};
    // (offsets that do not ascend: a group that lacks some of its rows shares nothing, so
    // that groups are apart and the parts fit the grid)
    if (c0 >= 0 && c0 < c1 && members[g] == c1 - c0 && most_of[g] > 0)
      t = shared_tiles(min(max(a.prefix[g], 0), cap), least_of[g], most_of[g], a.window, c1 - c0);
    least_of[g] = t.t0;
    most_of[g] = t.t1;
  }
  __syncthreads();
  // items: the groups, then the requests
  const int items = a.n_groups + a.b;
  int tiles[kShItems], units[kShItems];
  int64_t sum = 0;
#pragma unroll
  for (int e = 0; e < kShItems; ++e) {
    const int i = e * kShThreads + tid;
    tiles[e] = units[e] = 0;
    if (i < a.n_groups) {
      tiles[e] = most_of[i] - least_of[i];
      if (tiles[e] > 0) units[e] = a.hk * ((int)(((int64_t)(min(a.cu[i + 1], a.b) - a.cu[i]) * a.ratio + columns - 1) / columns));
    } else if (i < items) {
      const int b = i - a.n_groups, g = group_of[b];
      tiles[e] = own_tiles(len_of[b], a.window, g >= 0 ? TileSpan{least_of[g], most_of[g]} : TileSpan{0, 0}).count;
      units[e] = a.hk * a.groups;
    }
    sum += (int64_t)tiles[e] * units[e];
  }
#pragma unroll
  for (int x = 1; x < 64; x *= 2) sum += __shfl_xor(sum, x);
  int64_t* wide = reinterpret_cast<int64_t*>(acc);
  if (lane == 0) wide[wave] = sum;
  __syncthreads();
  sum = 0;
#pragma unroll
  for (int x = 0; x < kShWaves; ++x) sum += wide[x];
  const int per = share_size(sum, a.target, a.least);
  // the item that holds part w
  int run = 0;
#pragma unroll 1
  for (int e = 0; e * kShThreads < items; ++e) {
    int t = 0, u = 0;
#pragma unroll
    for (int x = 0; x < kShItems; ++x)
      if (x == e) {
        t = tiles[x];
        u = units[x];
      }
    const int n = share_count(t, per);
    const int incl = wave_scan(n * u);
    int* part = acc + 16 + (e & 1) * 4;   // (two sets, so that one barrier a step is enough)
    if (lane == 63) part[wave] = incl;
    __syncthreads();
    int start = run + incl - n * u;
#pragma unroll
    for (int x = 0; x < kShWaves; ++x) {
      if (x < wave) start += part[x];
      run += part[x];
    }
    const int i = e * kShThreads + tid;
    if (w == 0 && i < items) {
      int* r = a.rec + (int64_t)i * 4;
      r[0] = start;
      r[1] = n;
      r[2] = i < a.n_groups ? -1 : group_of[i - a.n_groups];
      r[3] = i < a.n_groups ? a.cu[i] : 0;
    }
    if (w >= start && w < start + n * u) {
      acc[32] = i;
      acc[33] = start;
      acc[34] = n;
      acc[35] = t;
    }
  }
  if (w >= run) return false;
  __syncthreads();
  const int item = uni(acc[32]), start = uni(acc[33]), n = uni(acc[34]), t = uni(acc[35]);
  const int unit = (w - start) / n, p = (w - start) % n;
  sh.slot = w;
  sh.lo = share_start(t, n, p);
  sh.hi = share_start(t, n, p + 1);
  if (item < a.n_groups) {
    const int c0 = uni(a.cu[item]), c1 = min(uni(a.cu[item + 1]), a.b);
    const int total = (c1 - c0) * a.ratio, blocks = (total + columns - 1) / columns;
    sh.group = item;
    sh.b = sh.leader = c0;
    sh.hk = unit / blocks;
    sh.col0 = unit % blocks * columns;
    sh.cols = min(columns, total - sh.col0);
    sh.own = OwnTiles{0, INT_MAX, uni(least_of[item]), INT_MAX, 0, 0};
    sh.prefix = INT_MAX;
    sh.alone = false;
  } else {
    const int b = item - a.n_groups, g = uni(group_of[b]);
    const TileSpan sp = g >= 0 ? TileSpan{uni(least_of[g]), uni(most_of[g])} : TileSpan{0, 0};
    sh.group = -1;
    sh.b = b;
    sh.leader = g >= 0 ? uni(a.cu[g]) : b;
    sh.prefix = g >= 0 ? min(max(uni(a.prefix[g]), 0), cap) : 0;
    sh.hk = unit / a.groups;
    sh.col0 = unit % a.groups * 16;
    sh.cols = min(16, a.ratio - sh.col0);
    sh.own = own_tiles(uni(len_of[b]), a.window, sp);
    sh.alone = n == 1 && sp.t0 == sp.t1;
  }
  return true;
}

// A part of NB blocks of 16 columns. sv: V slices of the waves. len_of: the requests' lengths in
// LDS are gone by now, so columns read their own.
template <int D, bool BF16, int NB, int NC>
__device__ __forceinline__ void share_part(kernarg<SharedArgs>& a, const Share& sh, uint8_t (*sV)[kDecTile * (D * 2 + 32)], float (*sM)[16], float (*sL)[16]) {
  typedef typename Elt<BF16>::v8 V8;
  constexpr int KD = D / 32, DB = D / 16;
  constexpr int kRow = D * 2 + 32;   // LDS bytes per V row: transposed reads of 16 rows touch all banks alike
  const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  const int page_size = 1 << a.shift;
  const int64_t span = (int64_t)a.cols << a.shift;

  // Q: B operand, column 16·n + l16, d = 8·(4·kd + g). Column c is head c % ratio of the
  // KV head's, of request c / ratio.
  V8 qreg[NB][KD];
  float bco[NB], last[NB];   // slope, and the last key of the column's request
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const int c = n * 16 + l16;
    const bool real = c < sh.cols;
    const int col = sh.col0 + (real ? c : 0);
    const int b = sh.group >= 0 ? sh.b + col / a.ratio : sh.b;
    const int h = sh.hk * a.ratio + (sh.group >= 0 ? col % a.ratio : col);
    const uint16_t* q = a.q + (int64_t)b * a.q_bs + (int64_t)h * a.q_hs + g * 8;
#pragma unroll
    for (int kd = 0; kd < KD; ++kd) {
      u32x4 x = {0u, 0u, 0u, 0u};
      if (real) x = *reinterpret_cast<const u32x4*>(q + kd * 32);
      qreg[n][kd] = bitcast<V8>(x);
    }
    bco[n] = a.slopes ? a.slopes[h] * a.bias : 0.f;
    last[n] = a.slopes ? (float)(min(max(a.lens[b], 0), (int)span) - 1) : 0.f;
  }
  const float c2 = a.c2, slack = kSlackLog2 / a.c2;
  f32x4 oacc[NB][DB];
  float m_run[NB], mlog2[NB], l_run[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
#pragma unroll
    for (int db = 0; db < DB; ++db) oacc[n][db] = f32x4{};
    m_run[n] = -INFINITY;
    mlog2[n] = l_run[n] = 0.f;
  }

  const int* tab = a.table + (int64_t)sh.b * a.ts;
  const int* lead = a.table + (int64_t)sh.leader * a.ts;
  const uint16_t* kbase = a.k + (int64_t)sh.hk * a.kh + g * 8;
  const uint16_t* vbase = a.v + (int64_t)sh.hk * a.vh + g * 8;
  const OwnTiles own = sh.own;
  const int end = sh.group >= 0 ? (int)min((int64_t)INT_MAX, span) : own.len, bound = max(end - 1, 0);
  // Page numbers of the lane's keys l16 and 16 + l16 of tile i of the unit (-1: not seen).
  // No load of the loop is conditional, or the compiler would wait for all loads in
  // flight where the paths meet: what is behind the part's end reads what is there anyway.
  auto entries = [&](int i, int (&e)[2]) __attribute__((always_inline)) {
    const int t = own_tile(own, min(i, sh.hi - 1));
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int key = t * kDecTile + r * 16 + l16;
      const int x = (key < sh.prefix ? lead : tab)[min(key, bound) >> a.shift];
      e[r] = (i < sh.hi && key >= own.lo && key < end) ? x : -1;
    }
  };
  struct Tile { u32x4 k[2][KD], v[2][KD]; bool ok[2]; };
  auto fetch = [&](int i, const int (&e)[2], Tile& x) __attribute__((always_inline)) {
    const int t = own_tile(own, min(i, sh.hi - 1));
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      x.ok[r] = e[r] >= 0 && e[r] < a.pages;
      const int64_t page = x.ok[r] ? e[r] : 0;
      const int64_t in = x.ok[r] ? (t * kDecTile + r * 16 + l16) & (page_size - 1) : 0;
      const uint16_t* kp = kbase + page * a.kp + in * a.kr;
      const uint16_t* vp = vbase + page * a.vp + in * a.vr;
#pragma unroll
      for (int kd = 0; kd < KD; ++kd) {
        x.k[r][kd] = *reinterpret_cast<const u32x4*>(kp + kd * 32);
        x.v[r][kd] = *reinterpret_cast<const u32x4*>(vp + kd * 32);
      }
    }
  };
  uint8_t* sv = sV[wave];
  auto compute = [&](int i, const Tile& x) __attribute__((always_inline)) {
    const int t = own_tile(own, i);
    const bool whole = __builtin_amdgcn_ballot_w64(x.ok[0] && x.ok[1]) == ~0ull;
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int kd = 0; kd < KD; ++kd) {
        u32x4 y = x.v[r][kd];
        if (!whole && !x.ok[r]) y = u32x4{0u, 0u, 0u, 0u};   // nothing of an unseen key's V
        *reinterpret_cast<u32x4*>(sv + (r * 16 + l16) * kRow + (kd * 4 + g) * 16) = y;
      }
    f32x4 s[NB][2];
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int r = 0; r < 2; ++r) s[n][r] = f32x4{};
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int kd = 0; kd < KD; ++kd)
#pragma unroll
        for (int n = 0; n < NB; ++n) s[n][r] = mfma16<BF16>(bitcast<V8>(x.k[r][kd]), qreg[n][kd], s[n][r]);
    // this lane: column 16·n + l16, keys 16·r + 4·g + e
    const uint64_t ok0 = __builtin_amdgcn_ballot_w64(x.ok[0]), ok1 = __builtin_amdgcn_ballot_w64(x.ok[1]);
    V8 p[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      if (a.cap) {
#pragma unroll
        for (int c = 0; c < 8; ++c) s[n][c / 4][c % 4] = __builtin_amdgcn_rcpf(-1.f - __builtin_amdgcn_exp2f(s[n][c / 4][c % 4] * a.u_scale));
      }
      if (a.slopes) {
        const float back = last[n] - (float)(t * kDecTile + 4 * g);
#pragma unroll
        for (int c = 0; c < 8; ++c) s[n][c / 4][c % 4] = __builtin_fmaf(bco[n], back - (float)(c / 4 * 16 + c % 4), s[n][c / 4][c % 4]);
      }
      if (!whole) {
#pragma unroll
        for (int c = 0; c < 8; ++c)
          s[n][c / 4][c % 4] = (((c / 4 ? ok1 : ok0) >> (4 * g + c % 4)) & 1) ? s[n][c / 4][c % 4] : -INFINITY;
      }
      float mx = -INFINITY;
#pragma unroll
      for (int c = 0; c < 8; ++c) mx = fmaxf(mx, s[n][c / 4][c % 4]);
      if (__builtin_amdgcn_ballot_w64(mx > m_run[n] + slack)) {
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const bool need = mx > m_run[n] + slack;
        const float alpha = need ? __builtin_amdgcn_exp2f((m_run[n] - mx) * c2) : 1.f;
        m_run[n] = need ? mx : m_run[n];
        mlog2[n] = m_run[n] == -INFINITY ? 0.f : m_run[n] * c2;
        l_run[n] *= alpha;
#pragma unroll
        for (int db = 0; db < DB; ++db) oacc[n][db] *= alpha;
      }
      f32x8 pf;
#pragma unroll
      for (int c = 0; c < 8; ++c) pf[c] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][c / 4][c % 4], c2, -mlog2[n]));
      // P rounded for the second product, and its sum of the rounded: normalised by their
      // own sum, the weights' errors are independent and O's about that of its own rounding
      p[n] = __builtin_convertvector(pf, V8);
      l_run[n] = psum8<BF16>(p[n], l_run[n]);
    }
    // Vᵀ: lane s of a 16-lane group reads 4 columns of row 4·g + s/4 (and 16 + that)
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      const uint8_t* at = sv + (4 * g + l16 / 4) * kRow + (db * 16 + 4 * (l16 & 3)) * 2;
      const s16x4 x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at);
      const s16x4 x1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + 16 * kRow));
      const V8 vt = bitcast<V8>(__builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
      for (int n = 0; n < NB; ++n) oacc[n][db] = mfma16<BF16>(vt, p[n], oacc[n][db]);
    }
  };

  if (sh.lo + wave < sh.hi) {
    int t = sh.lo + wave;
    int e0[2], e1[2];
    Tile x0, x1;
    entries(t, e0);
    entries(t + kShWaves, e1);
    fetch(t, e0, x0);
    for (; t + kShWaves < sh.hi; t += 2 * kShWaves) {
      entries(t + 2 * kShWaves, e0);
      fetch(t + kShWaves, e1, x1);
      compute(t, x0);
      entries(t + 3 * kShWaves, e1);
      fetch(t + 2 * kShWaves, e0, x0);
      compute(t + kShWaves, x1);
    }
    if (t < sh.hi) compute(t, x0);
  }

  // join the waves, one block of columns after the other: O in the wave's slice as fp32,
  // [16 columns][D + 2] (the slices are free)
  float* so = reinterpret_cast<float*>(sv);
  static_assert(16 * (D + 2) * 4 <= kDecTile * kRow, "O fits in the V slice");
#pragma unroll 1
  for (int n = 0; n < NB; ++n) {
    if (n * 16 >= sh.cols) break;
    if (n > 0) __syncthreads();   // the last block's slices are read
#pragma unroll
    for (int x = 0; x < NB; ++x)
      if (x == n) {
        float l = l_run[x];
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        if (lane < 16) {
          sM[wave][l16] = m_run[x] == -INFINITY ? -INFINITY : m_run[x] * c2;
          sL[wave][l16] = l;
        }
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int e = 0; e < 4; ++e) so[l16 * (D + 2) + db * 16 + 4 * g + e] = oacc[x][db][e];
      }
    __syncthreads();
    const int cols = min(16, sh.cols - n * 16);
    for (int x = tid; x < cols * D; x += kShThreads) {
      const int c = x / D, d = x % D;
      float m = sM[0][c];
#pragma unroll
      for (int w = 1; w < kShWaves; ++w) m = fmaxf(m, sM[w][c]);
      float acc = 0.f, l = 0.f;
#pragma unroll
      for (int w = 0; w < kShWaves; ++w) {
        const float f = sM[w][c] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(sM[w][c] - m);
        // a wave that saw nothing adds nothing; NaN sums stay
        l += sL[w][c] == 0.f ? 0.f : sL[w][c] * f;
        acc += sL[w][c] == 0.f ? 0.f : reinterpret_cast<const float*>(sV[w])[c * (D + 2) + d] * f;
      }
      if (sh.alone) {
        const float r = l == 0.f ? 0.f : acc / l;
        uint16_t out;
        if constexpr (BF16) out = bitcast<uint16_t>((__bf16)r);
        else out = bitcast<uint16_t>((_Float16)r);
        a.o[(int64_t)sh.b * a.o_bs + (int64_t)(sh.hk * a.ratio + sh.col0 + c) * a.o_hs + d] = out;
      } else {
        const int64_t at = (int64_t)sh.slot * (16 * NC) + n * 16 + c;
        a.part_o[at * D + d] = acc;
        if (d == 0) {
          a.part_ml[at * 2] = m;
          a.part_ml[at * 2 + 1] = l;
        }
      }
    }
  }
}

template <int D, bool BF16, int NC>
__global__ __launch_bounds__(kShThreads) __attribute__((amdgpu_waves_per_eu(NC > 1 ? 1 : 2)))
void shared_decode_kernel(const SharedArgs a) {
  constexpr int kSlice = kDecTile * (D * 2 + 32);
  constexpr int kBytes = kShWaves * kSlice > kShPlan * 4 ? kShWaves * kSlice : kShPlan * 4;
  __shared__ __align__(16) uint8_t lds[kBytes];
  __shared__ float sM[kShWaves][16], sL[kShWaves][16];
  Share sh;
  if (!find_share(a, 16 * NC, blockIdx.x, reinterpret_cast<int*>(lds), sh)) return;
  __syncthreads();   // the plan's words are read
  uint8_t (*sV)[kSlice] = reinterpret_cast<uint8_t (*)[kSlice]>(lds);
  if (NC > 1 && sh.group >= 0) share_part<D, BF16, NC, NC>(reload_kernarg(a), sh, sV, sM, sL);
  else share_part<D, BF16, 1, NC>(reload_kernarg(a), sh, sV, sM, sL);
}

// One workgroup per (request, head): its group's parts and its own, weighted by
// 2^(m_s − m). Its 256 threads are 1024 / D rows of D / 4 threads; a row takes every so
// many parts, 8 of them in flight, with a running max; the rows' sums are joined in LDS.
template <int D, bool BF16>
__device__ __forceinline__ void shared_join(const SharedArgs& a, int columns) {
  constexpr int TPR = D / 4, ROWS = 256 / TPR, J = 8;
  __shared__ float sAcc[ROWS][D], sMax[ROWS], sSum[ROWS];
  const int b = blockIdx.x / a.h, h = blockIdx.x % a.h, tid = threadIdx.x;
  const int hk = h / a.ratio, n = h - hk * a.ratio;
  const int* rec = a.rec + (int64_t)(a.n_groups + b) * 4;
  const int own_parts = uni(rec[1]), group = uni(rec[2]);
  const int own_at = uni(rec[0]) + (hk * a.groups + n / 16) * own_parts;
  int parts0 = 0, at0 = 0, col = 0;
  const int64_t span = (int64_t)a.cols << a.shift;
  if (group >= 0 && a.lens[b] > 0 && span > 0) {
    const int* r = a.rec + (int64_t)group * 4;
    parts0 = uni(r[1]);
    const int first = uni(r[3]), end = min(uni(a.cu[group + 1]), a.b);
    const int blocks = ((end - first) * a.ratio + columns - 1) / columns;
    col = (b - first) * a.ratio + n;
    at0 = uni(r[0]) + (hk * blocks + col / columns) * parts0;
    col %= columns;
  }
  const int parts = parts0 + own_parts;
  if (parts0 == 0 && own_parts == 1) return;   // written by its one part
  auto at = [&](int s) { return s < parts0 ? (int64_t)(at0 + s) * columns + col : (int64_t)(own_at + s - parts0) * columns + n % 16; };
  const int row = tid / TPR, c = tid % TPR;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  for (int s0 = row; s0 < parts; s0 += ROWS * J) {
    float ms[J], ls[J];
    f32x4 x[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int64_t i = at(min(s0 + j * ROWS, parts - 1));
      ms[j] = a.part_ml[i * 2];
      ls[j] = a.part_ml[i * 2 + 1];
      x[j] = *reinterpret_cast<const f32x4*>(a.part_o + i * D + c * 4);
    }
    float top = m;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      if (s0 + j * ROWS >= parts) ls[j] = 0.f;   // a copy of the last part
      top = fmaxf(top, ls[j] == 0.f ? -INFINITY : ms[j]);
    }
    const float old = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - top);
    l *= old;
    acc *= old;
    m = top;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      // a part that saw nothing adds nothing; NaN sums stay
      const float f = ms[j] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ms[j] - top);
      l += ls[j] == 0.f ? 0.f : ls[j] * f;
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] += ls[j] == 0.f ? 0.f : x[j][i] * f;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) sAcc[row][c * 4 + i] = acc[i];
  if (c == 0) {
    sMax[row] = m;
    sSum[row] = l;
  }
  __syncthreads();
  if (tid < D) {
    float top = sMax[0];
#pragma unroll
    for (int r = 1; r < ROWS; ++r) top = fmaxf(top, sMax[r]);
    float y = 0.f, t = 0.f;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const float f = sMax[r] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(sMax[r] - top);
      y += sSum[r] == 0.f ? 0.f : sAcc[r][tid] * f;
      t += sSum[r] == 0.f ? 0.f : sSum[r] * f;
    }
    const float r = t == 0.f ? 0.f : y / t;
    uint16_t out;
    if constexpr (BF16) out = bitcast<uint16_t>((__bf16)r);
    else out = bitcast<uint16_t>((_Float16)r);
    a.o[(int64_t)b * a.o_bs + (int64_t)h * a.o_hs + tid] = out;
  }
}

template <int D, bool BF16, int NC>
__global__ __launch_bounds__(256) void shared_join_kernel(const SharedArgs a) { shared_join<D, BF16>(a, 16 * NC); }
