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
//  * Shared tiles: a workgroup is 32·RW columns by KG groups of waves that take every
//    KG-th tile and join their sums in LDS at the end. Sᵀ = K·Qᵀ with 32x32x16 MFMAs, so
//    that a lane holds one column's scores; K and V come from the pages to LDS by DMA, of
//    128 columns (64 KB of LDS) four stages, else two, one barrier a step. The shape follows
//    from the columns a group has on average: fewer than a workgroup's are idle products,
//    more groups of waves fewer barriers a tile.
//  * Own tiles: 16 columns, the heads of one KV head; a wave by itself streams tiles of 32
//    keys, K to the operand registers, V through its own LDS slice, the next tile in flight.
//    All requests' own tiles are one sequence, cut into waves of equal length wherever that
//    falls, so that every workgroup runs at once.
//  * Lengths and offsets stay on the device: every workgroup derives the same plan from
//    them and takes its part; workgroup 0 writes down for the join where parts lie. (A plan
//    by a kernel of its own would cost a launch, 2.1 us, and the wait for it.) The grid has room
//    for a part that is not whole of each group's units, so with many groups workgroups come in
//    rounds, each of which plans: 1024 groups of one request 534 us, as paged decode 373.
// Measured in a graph, with the join: 9 groups, 67 requests of 16 heads of 128 on 4 KV
// heads, prefixes to 4099 keys, capped: 28 us (65 MB: 13.9 us); one group of 256 requests,
// 8192 keys: 48 us (74 MB, 17 GFLOP), of which plan and first loads take 8, the shared tiles
// 26 (17 % of the matrix units' time; vector and scalar work of two waves a SIMD and the
// wait for LDS and for each other fill the rest), the join 8; 4 requests, 300 keys of 64: 11.9 us;
// 128 groups of 4 requests of 32 heads on 8, prefixes to 2000 keys: 364 us (886 MB: 187 us).

constexpr int kShWaves = 4;
constexpr int kShThreads = 64 * kShWaves;

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
  int* rec;        // [n_groups + b + 1][4]: of groups the row of the first part, parts of a unit, first request;
                   // of requests the first wave, its tiles before, tiles of a unit, group or -1; last the wave's tiles
  float* part_ml;  // [rows][2]: max in log2 units, sum
  float* part_o;   // [rows][D]: `columns` rows of each group's part, then 16 of each of requests' own
  int64_t q_bs, q_hs, o_bs, o_hs, kp, kh, kr, vp, vh, vr, ts;
  int b, n_groups, h, hk, ratio;
  int groups;      // 16-head groups per KV head of a request's own keys
  int columns;     // of a group's workgroup
  int own_rows;    // first row of part_o of own tiles
  int pages, shift, cols, window;
  int target;                    // workgroups wanted
  int col_shift;                 // log2 of columns
  int cap;                       // scores are capped
  float u_scale, c2, bias;       // as in PackedArgs
};

// 4 values rounded to the type, as 8 bytes.
template <bool BF16> __device__ __forceinline__ void store4(uint16_t* to, f32x4 x) {
  typedef __attribute__((ext_vector_type(4))) __bf16 bf16x4;
  typedef __attribute__((ext_vector_type(4))) _Float16 f16x4;
  if constexpr (BF16) *reinterpret_cast<u32x2*>(to) = bitcast<u32x2>(__builtin_convertvector(x, bf16x4));
  else *reinterpret_cast<u32x2*>(to) = bitcast<u32x2>(__builtin_convertvector(x, f16x4));
}

// What a wave does.
struct Share {
  int kind;        // 0: nothing; 1: shared tiles of a group; 2: own tiles, the wave by itself
  int b;           // the first request of the group, or the request
  int leader;      // the row that names the prefix's pages
  int hk, col0;    // KV head; first column, or first head of the request's
  int cols;        // columns there are
  int prefix;      // keys below it: of the leader's row
  int row, lo, hi; // where the part's results go (rows of part_o); its tiles [lo, hi) of the unit's
  int alone;       // the request's only part
  OwnTiles own;    // a group's tiles: own.first + i
};

// The plan, by T threads (one wave, where all have little to do: no barriers). LDS: s, of
// kShWords. Units of groups have parts that take a workgroup each; behind them come the
// requests' own, four to a workgroup. What workgroup w holds is left in s[0 ..]: see share_of.
struct PlanLds {
  int *acc, *len_of, *group_of, *least_of, *most_of, *members, *prefix, *leader, *cu;
  __device__ __forceinline__ explicit PlanLds(int* s)
      : acc(s), len_of(s + 64), group_of(len_of + kShMax), least_of(group_of + kShMax), most_of(least_of + kShMax), members(most_of + kShMax),
        prefix(members + kShMax), leader(prefix + kShMax), cu(leader + kShMax) {}
};
template <int T> __device__ __forceinline__ void find_share(const SharedArgs& a, int w, int* s) {
  constexpr bool SOLO = T == 64;
  constexpr int WAVES = T / 64;
  auto meet = [&]() __attribute__((always_inline)) {
    if constexpr (SOLO) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // (a wave's LDS accesses stay in order)
    else __syncthreads();
  };
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const PlanLds l(s);
  const int cap = (int)((int64_t)a.cols << a.shift);
  for (int i = tid; i < a.b; i += T) {
    l.len_of[i] = min(max(a.lens[i], 0), cap);
    l.group_of[i] = -1;
  }
  for (int g = tid; g <= a.n_groups; g += T) {
    l.cu[g] = a.cu[g];
    if (g < a.n_groups) {
      l.prefix[g] = min(max(a.prefix[g], 0), cap);
      l.least_of[g] = INT_MAX;
      l.most_of[g] = l.members[g] = 0;
    }
  }
  if (tid < 64) l.acc[tid] = 0;
  meet();
  // a request's group: the last one that starts at or before it, if it ends behind it
  for (int g = tid; g < a.n_groups; g += T) {
    const int c = l.cu[g];
    if (c >= 0 && c < a.b) atomicMax(&l.group_of[c], g);
  }
  meet();
  const int each = (a.b + T - 1) / T, i0 = tid * each, i1 = min(i0 + each, a.b);
  int top = -1;
  for (int i = i0; i < i1; ++i) top = max(top, l.group_of[i]);
  const int upto = wave_max_scan(top);
  int before = __shfl_up(upto, 1);
  if (lane == 0) before = -1;
  if constexpr (!SOLO) {
    if (lane == 63) l.acc[32 + wave] = upto;
    meet();
    for (int x = 0; x < wave; ++x) before = max(before, l.acc[32 + x]);
  }
  for (int i = i0; i < i1; ++i) {
    before = max(before, l.group_of[i]);
    const int g = before >= 0 && i < l.cu[before + 1] ? before : -1, n = l.len_of[i];
    l.group_of[i] = g;
    if (g >= 0) atomicAdd(&l.members[g], 1);
    if (g >= 0 && n > 0) {
      atomicMin(&l.least_of[g], n);
      atomicMax(&l.most_of[g], n);
    }
  }
  meet();
  auto units_of = [&](int g) { return a.hk * (((min(l.cu[g + 1], a.b) - l.cu[g]) * a.ratio + a.columns - 1) >> a.col_shift); };
  const int own_units = a.hk * a.groups, weight = own_weight(a.columns);
  int64_t sum = 0;
  for (int g = tid; g < a.n_groups; g += T) {
    const int c0 = l.cu[g], c1 = min(l.cu[g + 1], a.b);
    TileSpan t{0, 0};
    // (offsets that do not ascend: a group that lacks some of its rows shares nothing, so
    // that groups are apart and the parts fit the grid)
    if (c0 >= 0 && c0 < c1 && l.members[g] == c1 - c0 && l.most_of[g] > 0)
      t = shared_tiles(l.prefix[g], l.least_of[g], l.most_of[g], a.window, c1 - c0);
    const bool ended = l.most_of[g] > 0 && l.len_of[c0] == 0;   // the first request, and not all
    l.leader[g] = ended ? INT_MAX : c0;
    if (ended) l.acc[36] = 1;
    l.least_of[g] = t.t0;
    l.most_of[g] = t.t1;
    if (t.t1 > t.t0) sum += (int64_t)(t.t1 - t.t0) * units_of(g) * (a.columns / 32);
  }
  meet();
  // The row that names such a group's prefix is the first that has keys or a page: an ended
  // request's may be kept for the prefix, but a fork leaves it empty.
  if (uni(l.acc[36]))
    for (int i = tid; i < a.b; i += T) {
      const int g = l.group_of[i];
      if (g >= 0 && l.len_of[l.cu[g]] == 0 && (l.len_of[i] > 0 || (uint32_t)a.table[(int64_t)i * a.ts] < (uint32_t)a.pages)) atomicMin(&l.leader[g], i);
    }
  int* counts = l.members;
  for (int b = tid; b < a.b; b += T) {
    const int g = l.group_of[b], n = own_tiles(l.len_of[b], a.window, g >= 0 ? TileSpan{l.least_of[g], l.most_of[g]} : TileSpan{0, 0}).count;
    counts[b] = n;
    sum += (int64_t)n * own_units * weight;
  }
#pragma unroll
  for (int x = 1; x < 64; x *= 2) sum += __shfl_xor(sum, x);
  if constexpr (!SOLO) {
    int64_t* wide = reinterpret_cast<int64_t*>(l.acc + 40);
    if (lane == 0) wide[wave] = sum;
    meet();
    sum = 0;
#pragma unroll
    for (int x = 0; x < WAVES; ++x) sum += wide[x];
  }
  const int steps = share_steps(sum, a.target), per = share_size(steps, kShWaves * 32 / a.columns), wave_per = wave_share_size(steps, weight);
  int turn = 0;
  // The sum over the threads before this one (and, of all, in `run`); 64 bits as two halves that cannot overflow.
  auto scan = [&](int64_t x, int64_t& run) __attribute__((always_inline)) {
    const int lo = (int)x & 0xfffff, hi = (int)(x >> 20), slo = wave_scan(lo), shi = wave_scan(hi);
    int64_t start = run + ((int64_t)(shi - hi) << 20) + (slo - lo);
    const int64_t all = ((int64_t)__builtin_amdgcn_readlane(shi, 63) << 20) + __builtin_amdgcn_readlane(slo, 63);
    if constexpr (SOLO) run += all;
    else {
      int64_t* part = reinterpret_cast<int64_t*>(l.acc + 48 + (turn++ & 1) * 8);   // (two sets, so that one barrier a step is enough)
      if (lane == 63) part[wave] = all;
      meet();
#pragma unroll
      for (int x = 0; x < WAVES; ++x) {
        if (x < wave) start += part[x];
        run += part[x];
      }
    }
    return start;
  };
  int64_t run = 0;
  for (int e = 0; e < a.n_groups; e += T) {
    const int g = e + tid;
    const bool real = g < a.n_groups;
    const int t = real ? l.most_of[g] - l.least_of[g] : 0, n = share_count(t, per), all = t > 0 ? n * units_of(g) : 0;
    const int start = (int)scan(all, run);
    if (real && w == 0) *reinterpret_cast<i32x4*>(a.rec + (int64_t)g * 4) = i32x4{start << a.col_shift, n, l.cu[g], 0};
    if (w >= start && w < start + all) {
      l.acc[0] = 1 + g;
      l.acc[1] = w - start;
      l.acc[2] = n;
      l.acc[3] = start;
    }
  }
  const int parts = (int)run;
  if (tid == 0) {
    l.acc[16] = parts;
    l.acc[17] = wave_per;
    if (w == 0) a.rec[(int64_t)(a.n_groups + a.b) * 4] = wave_per;
  }
  if (w > 0 && w < parts) return;   // (the first one goes on for the records)
  run = 0;
  for (int e = 0; e < a.b; e += T) {
    const int b = e + tid;
    const bool real = b < a.b;
    const int64_t all = real ? (int64_t)counts[b] * own_units : 0, start = scan(all, run);
    if (real && w == 0) {
      const WaveTile at = wave_tile(start, wave_per);
      *reinterpret_cast<i32x4*>(a.rec + (int64_t)(a.n_groups + b) * 4) = i32x4{at.wave, at.before, counts[b], l.group_of[b]};
    }
#pragma unroll
    for (int x = 0; x < kShWaves; ++x) {
      const int64_t from = ((int64_t)(w - parts) * kShWaves + x) * wave_per;
      if (w >= parts && from >= start && from < start + all) {
        l.acc[4 * x] = 1 + b;
        l.acc[4 * x + 1] = (int)(from - start);
      }
    }
  }
}

// A group's part, from the plan's words; all waves, before they are overwritten.
__device__ __forceinline__ Share group_share(const SharedArgs& a, int* s) {
  const PlanLds l(s);
  Share sh{};
  const int g = uni(l.acc[0]) - 1, place = uni(l.acc[1]), n = uni(l.acc[2]), start = uni(l.acc[3]);
  const int c0 = uni(l.cu[g]), c1 = min(uni(l.cu[g + 1]), a.b), total = (c1 - c0) * a.ratio, blocks = (total + a.columns - 1) >> a.col_shift;
  const int t0 = uni(l.least_of[g]), t = uni(l.most_of[g]) - t0;
  const UnitPart at = unit_part(place, n, a.hk, blocks);
  sh.kind = 1;
  sh.b = c0;
  sh.leader = uni(l.leader[g]);
  sh.hk = at.hk;
  sh.col0 = at.block * a.columns;
  sh.cols = min(a.columns, total - sh.col0);
  sh.prefix = INT_MAX;
  sh.row = (start + (at.hk * blocks + at.block) * n + at.part) << a.col_shift;
  sh.lo = share_start(t, n, at.part);
  sh.hi = share_start(t, n, at.part + 1);
  sh.own = OwnTiles{0, INT_MAX, t0, INT_MAX, 0, 0};
  return sh;
}

// A wave's own tiles: from tile `off` of request b's (all its units', one behind another) on.
struct Walk {
  int b, off, left, number;   // left: tiles; number: of the wave
};
// The tiles that follow as far as they are of one unit; false: none do.
__device__ __forceinline__ bool own_share(const SharedArgs& a, int* s, Walk& w, Share& sh) {
  const PlanLds l(s);
  if (w.b < 0 || w.left <= 0) return false;
  const int lane = threadIdx.x & 63, own_units = a.hk * a.groups;
  int count = uni(l.members[w.b]);
  if (w.off == count * own_units) {   // the next request that has some
    w.off = count = 0;
    for (int b = w.b + 1; b < a.b; b += 64) {
      const int i = min(b + lane, a.b - 1), n = l.members[i];
      const uint64_t has = __builtin_amdgcn_ballot_w64(n > 0 && b + lane < a.b);
      if (has) {
        const int first = __builtin_ctzll(has);
        w.b = b + first;
        count = __builtin_amdgcn_readlane(n, first);
        break;
      }
    }
    if (count == 0) return false;
  }
  const int unit = (int)((uint32_t)w.off / (uint32_t)count), g = uni(l.group_of[w.b]);
  const TileSpan sp = g >= 0 ? TileSpan{uni(l.least_of[g]), uni(l.most_of[g])} : TileSpan{0, 0};
  sh.kind = 2;
  sh.b = w.b;
  sh.leader = g >= 0 ? uni(l.leader[g]) : w.b;
  sh.hk = (int)((uint32_t)unit / (uint32_t)a.groups);
  sh.col0 = (unit - sh.hk * a.groups) * 16;
  sh.cols = min(16, a.ratio - sh.col0);
  sh.prefix = g >= 0 ? uni(l.prefix[g]) : 0;
  sh.row = a.own_rows + (w.number + w.b * own_units + unit) * 16;
  sh.lo = w.off - unit * count;
  sh.hi = min(count, sh.lo + w.left);
  sh.alone = sh.lo == 0 && sh.hi == count && sp.t0 == sp.t1;
  sh.own = own_tiles(uni(l.len_of[w.b]), a.window, sp);
  w.off += sh.hi - sh.lo;
  w.left -= sh.hi - sh.lo;
  return true;
}

// Own tiles: 16 columns of request sh.b, or of a group that has a bad page, streamed by W waves,
// of which this is number `wave`; sv: the wave's V slice.
template <int D, bool BF16> struct Stream {
  typedef typename Elt<BF16>::v8 V8;
  static constexpr int KD = D / 32, DB = D / 16;
  static constexpr int kRow = D * 2 + 32;   // LDS bytes per V row: transposed reads of 16 rows touch all banks alike
  static constexpr int kSlice = kDecTile * kRow;
  f32x4 oacc[DB];
  float m_run = -INFINITY, mlog2 = 0.f, l_run = 0.f;

  __device__ __forceinline__ void run(kernarg<SharedArgs>& a, const Share& sh, int col0, int cols, int wave, int W, uint8_t* sv) {
    const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
    const int page_size = 1 << a.shift;
    const int64_t span = (int64_t)a.cols << a.shift;
    // Q: B operand, column l16, d = 8·(4·kd + g). A group's column c is head c % ratio of the
    // KV head's, of request c / ratio.
    const bool mine = l16 < cols;
    const int col = col0 + (mine ? l16 : 0);
    const int b = sh.kind == 1 ? sh.b + col / a.ratio : sh.b, h = sh.hk * a.ratio + (sh.kind == 1 ? col % a.ratio : col);
    V8 qreg[KD];
    const uint16_t* q = a.q + (int64_t)b * a.q_bs + (int64_t)h * a.q_hs + g * 8;
#pragma unroll
    for (int kd = 0; kd < KD; ++kd) {
      u32x4 x = {0u, 0u, 0u, 0u};
      if (mine) x = *reinterpret_cast<const u32x4*>(q + kd * 32);
      qreg[kd] = bitcast<V8>(x);
    }
    const float bco = a.slopes ? a.slopes[h] * a.bias : 0.f;
    const float last = a.slopes ? (float)(min(max(a.lens[b], 0), (int)span) - 1) : 0.f;   // the column's last key
    const float c2 = a.c2, slack = kSlackLog2 / a.c2;
#pragma unroll
    for (int db = 0; db < DB; ++db) oacc[db] = f32x4{};
    m_run = -INFINITY;
    mlog2 = l_run = 0.f;

    const int* tab = a.table + (int64_t)sh.b * a.ts;
    const int* lead = a.table + (int64_t)sh.leader * a.ts;
    const uint16_t* kbase = a.k + (int64_t)sh.hk * a.kh + g * 8;
    const uint16_t* vbase = a.v + (int64_t)sh.hk * a.vh + g * 8;
    const OwnTiles own = sh.own;
    const int end = sh.kind == 1 ? (int)span : own.len, bound = max(end - 1, 0);
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
      f32x4 s[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        s[r] = f32x4{};
#pragma unroll
        for (int kd = 0; kd < KD; ++kd) s[r] = mfma16<BF16>(bitcast<V8>(x.k[r][kd]), qreg[kd], s[r]);
      }
      // this lane: column l16, keys 16·r + 4·g + e
      const uint64_t ok0 = __builtin_amdgcn_ballot_w64(x.ok[0]), ok1 = __builtin_amdgcn_ballot_w64(x.ok[1]);
      if (a.cap) {
#pragma unroll
        for (int c = 0; c < 8; ++c) s[c / 4][c % 4] = __builtin_amdgcn_rcpf(-1.f - __builtin_amdgcn_exp2f(s[c / 4][c % 4] * a.u_scale));
      }
      if (a.slopes) {
        const float back = last - (float)(t * kDecTile + 4 * g);
#pragma unroll
        for (int c = 0; c < 8; ++c) s[c / 4][c % 4] = __builtin_fmaf(bco, back - (float)(c / 4 * 16 + c % 4), s[c / 4][c % 4]);
      }
      if (!whole) {
#pragma unroll
        for (int c = 0; c < 8; ++c) s[c / 4][c % 4] = (((c / 4 ? ok1 : ok0) >> (4 * g + c % 4)) & 1) ? s[c / 4][c % 4] : -INFINITY;
      }
      float mx = -INFINITY;
#pragma unroll
      for (int c = 0; c < 8; ++c) mx = fmaxf(mx, s[c / 4][c % 4]);
      if (__builtin_amdgcn_ballot_w64(mx > m_run + slack)) {
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const bool need = mx > m_run + slack;
        const float alpha = need ? __builtin_amdgcn_exp2f((m_run - mx) * c2) : 1.f;
        m_run = need ? mx : m_run;
        mlog2 = m_run == -INFINITY ? 0.f : m_run * c2;
        l_run *= alpha;
#pragma unroll
        for (int db = 0; db < DB; ++db) oacc[db] *= alpha;
      }
      f32x8 pf;
#pragma unroll
      for (int c = 0; c < 8; ++c) pf[c] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[c / 4][c % 4], c2, -mlog2));
      // P rounded for the second product, and its sum of the rounded: normalised by their
      // own sum, the weights' errors are independent and O's about that of its own rounding
      const V8 p = __builtin_convertvector(pf, V8);
      l_run = psum8<BF16>(p, l_run);
      // Vᵀ: lane s of a 16-lane group reads 4 columns of row 4·g + s/4 (and 16 + that)
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        const uint8_t* at = sv + (4 * g + l16 / 4) * kRow + (db * 16 + 4 * (l16 & 3)) * 2;
        const s16x4 x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at);
        const s16x4 x1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + 16 * kRow));
        oacc[db] = mfma16<BF16>(bitcast<V8>(__builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7)), p, oacc[db]);
      }
    };

    if (sh.lo + wave < sh.hi) {
      int t = sh.lo + wave;
      int e0[2], e1[2];
      Tile x0, x1;
      entries(t, e0);
      entries(t + W, e1);
      fetch(t, e0, x0);
      for (; t + W < sh.hi; t += 2 * W) {
        entries(t + 2 * W, e0);
        fetch(t + W, e1, x1);
        compute(t, x0);
        entries(t + 3 * W, e1);
        fetch(t + 2 * W, e0, x0);
        compute(t + W, x1);
      }
      if (t < sh.hi) compute(t, x0);
    }
    l_run += __shfl_xor(l_run, 16);
    l_run += __shfl_xor(l_run, 32);
  }

  // The wave's sums as a part, or as the result.
  __device__ __forceinline__ void store(kernarg<SharedArgs>& a, const Share& sh) const {
    const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
    if (l16 >= sh.cols) return;
    if (sh.alone) {
      const float inv = l_run == 0.f ? 0.f : 1.f / l_run;
      uint16_t* o = a.o + (int64_t)sh.b * a.o_bs + (int64_t)(sh.hk * a.ratio + sh.col0 + l16) * a.o_hs;
#pragma unroll
      for (int db = 0; db < DB; ++db) store4<BF16>(o + db * 16 + 4 * g, l_run == 0.f ? f32x4{} : oacc[db] * inv);
    } else {
      const int64_t at = (int64_t)sh.row + l16;
#pragma unroll
      for (int db = 0; db < DB; ++db) *reinterpret_cast<f32x4*>(a.part_o + at * D + db * 16 + 4 * g) = oacc[db];
      if (g == 0) {
        a.part_ml[at * 2] = m_run == -INFINITY ? -INFINITY : m_run * a.c2;
        a.part_ml[at * 2 + 1] = l_run;
      }
    }
  }

  // The four waves' sums as one, of columns col0 .. of the part: each wave's O in its slice as
  // fp32, [16 columns][D + 2]. All waves; the slices are free at the end.
  __device__ __forceinline__ void join(kernarg<SharedArgs>& a, const Share& sh, int col0, int cols, uint8_t* slices, float (*sM)[16], float (*sL)[16]) const {
    const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6), l16 = lane & 15, g = lane >> 4;
    float* so = reinterpret_cast<float*>(slices + wave * kSlice);
    static_assert(16 * (D + 2) * 4 <= kSlice, "O fits in the V slice");
    if (lane < 16) {
      sM[wave][l16] = m_run == -INFINITY ? -INFINITY : m_run * a.c2;
      sL[wave][l16] = l_run;
    }
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int e = 0; e < 4; ++e) so[l16 * (D + 2) + db * 16 + 4 * g + e] = oacc[db][e];
    __syncthreads();
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
        acc += sL[w][c] == 0.f ? 0.f : reinterpret_cast<const float*>(slices + w * kSlice)[c * (D + 2) + d] * f;
      }
      const int64_t at = (int64_t)sh.row + col0 + c;
      a.part_o[at * D + d] = acc;
      if (d == 0) {
        a.part_ml[at * 2] = m;
        a.part_ml[at * 2 + 1] = l;
      }
    }
    __syncthreads();
  }
};

// Stages of the DMA, and pages whose numbers are held in LDS.
template <int KG> constexpr int kShStages() { return KG == 1 ? 4 : 2; }
constexpr int kShPages = 1024;

template <int D, int RW, int KG> constexpr int kShLds() {
  const int stages = kShStages<KG>() * 2 * KG * kDecTile * D * 2 + kShPages * 4, sums = (RW * KG * 16 * (D / 32) * 64 + RW * KG * 2 * 64 + 1) * 4,
            own = kShWords * 4 + kShWaves * kDecTile * (D * 2 + 32);
  return stages > sums ? (stages > own ? stages : own) : sums > own ? sums : own;
}

// Shared tiles: 32·RW columns by KG key groups of a tile a step. True if a page was none of
// the cache's: nothing is done then.
template <int D, bool BF16, int RW, int KG>
__device__ __forceinline__ bool group_part(kernarg<SharedArgs>& a, const Share& sh, uint8_t* lds) {
  typedef typename Elt<BF16>::v8 V8;
  static_assert(RW * KG == kShWaves, "four waves");
  constexpr int UPR = D / 8, KD = D / 16, DB = D / 32, S = kShStages<KG>();
  constexpr int kElems = kDecTile * D;              // of a K or V tile
  constexpr int R = kDecTile / RW;                  // rows that a wave brings
  constexpr int kLoads = R * UPR / 64, RPL = 64 / UPR;   // loads of K, of V; rows of one
  uint16_t* sKV = reinterpret_cast<uint16_t*>(lds);   // [stage][K, V][KG][kElems]
  const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6);
  const int rw = wave % RW, kg = wave / RW, l32 = lane & 31, g = lane >> 5;
  const int page_size = 1 << a.shift;

  // the lane's column, and Q: B operand
  const int c = rw * 32 + l32;
  const bool mine = c < sh.cols;
  const int col = sh.col0 + (mine ? c : 0);
  const int b = sh.b + col / a.ratio, h = sh.hk * a.ratio + col % a.ratio;
  const uint16_t* q = a.q + (int64_t)b * a.q_bs + (int64_t)h * a.q_hs + g * 8;
  V8 qreg[KD];
#pragma unroll
  for (int kd = 0; kd < KD; ++kd) qreg[kd] = bitcast<V8>(*reinterpret_cast<const u32x4*>(q + kd * 16));
  float bco = a.slopes ? a.slopes[h] * a.bias : 0.f;
  float last = a.slopes ? (float)(min(max(a.lens[b], 0), (int)((int64_t)a.cols << a.shift)) - 1) : 0.f;   // the column's last key
  const float c2 = a.c2, slack = kSlackLog2 / a.c2;

  // steps of KG tiles: key group kg has tile first + step·KG + kg, if it is there
  const int count = sh.hi - sh.lo, first = sh.own.first + sh.lo;
  const int steps = (count + KG - 1) / KG;
  auto there = [&](int step) { return step * KG + kg < count; };
  // The wave's rows of the LDS tiles: load i brings rows rw·R + i·RPL .., of K the keys π(row).
  // 4 rows of K are 4 keys that follow one another in a page, and RPL rows of V are so too, so
  // that their page is the same for all lanes, which add an offset of their own (of d = 64,
  // K's 8 rows are two such runs, 16 keys apart: one page where it has 32 rows, else an address each).
  const int* lead = a.table + (int64_t)sh.leader * a.ts;
  const int q4 = lane / UPR, slot = lane % UPR;
  const uint16_t* kbase = a.k + (int64_t)sh.hk * a.kh;
  const uint16_t* vbase = a.v + (int64_t)sh.hk * a.vh;
  const int most = (first + count) * kDecTile - 1;   // the part's last key
  const bool two = RPL == 8 && a.shift < 5;          // K's loads reach into two pages
  // Offsets of the lane from where the tile starts in a page (of fewer than 32 rows: from the page)
  const int in_page = page_size - 1;
  uint32_t k_off[kLoads], v_off[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int r = rw * R + i * RPL;
    k_off[i] = (uint32_t)(((key_perm(r) & in_page) + key_perm(r + q4) - key_perm(r)) * (int)a.kr + (slot ^ ((r + q4) % UPR)) * 8) * 2u;
    v_off[i] = (uint32_t)(((r & in_page) + q4) * (int)a.vr + (slot ^ v_swz<D>(q4)) * 8) * 2u;
  }
  // Page numbers in LDS, kShPages from page `held` on. (Loads of the loop's own would make it
  // wait for the DMA issued before them.) A page outside the cache is read as page 0, and all of
  // it done again at the end.
  int* pages = reinterpret_cast<int*>(lds + S * 2 * KG * kElems * 2);
  const int last_page = most >> a.shift;
  int held = (first * kDecTile) >> a.shift;
  bool bad = false;
  auto fill = [&]() {
#pragma unroll
    for (int x = 0; x < kShPages / kShThreads; ++x) {
      const int at = x * kShThreads + tid;
      if (held + x * kShThreads > last_page) break;
      const int page = lead[min(held + at, last_page)];
      const bool none = (uint32_t)page >= (uint32_t)a.pages;
      bad |= none;
      pages[at] = none ? 0 : page;
    }
    wg_barrier();
  };
  // Where a step's loads start: those of K in lanes 0 .., then V's.
  static_assert(2 * kLoads <= 64, "a lane each");
  const int of = lane < kLoads ? lane : min(lane - kLoads, kLoads - 1), of_row = rw * R + of * RPL;
  const int of_key = lane < kLoads ? key_perm(of_row) : of_row;
  const bool of_k = lane < kLoads;
  const uint64_t of_base = reinterpret_cast<uint64_t>(of_k ? kbase : vbase), of_page = (uint64_t)(of_k ? a.kp : a.vp) * 2, of_step = (uint64_t)(of_k ? a.kr : a.vr) * 2;
  auto key_of = [&](int step) { return (first + step * KG + kg) * kDecTile; };
  auto entries = [&](int step) __attribute__((always_inline)) {
    const int behind = min((first + min(step + 1, steps) * KG) * kDecTile - 1, most) >> a.shift;   // the step's last page
    if (behind - held >= kShPages) {   // (all waves come here, of step after step)
      wg_barrier();
      held = min((first + step * KG) * kDecTile, most) >> a.shift;
      fill();
    }
    // (of small pages the tile starts at 0, and the lane's key is in its offset)
    const int key0 = key_of(step), page = pages[(min(key0 + of_key, most) >> a.shift) - held];
    return of_base + (uint64_t)(uint32_t)page * of_page + (uint64_t)(uint32_t)(key0 & in_page) * of_step;
  };
  const uint32_t lds0 = lds_addr(sKV);
  auto issue = [&](int step, int st, uint64_t e) __attribute__((always_inline)) {
    if (!there(step)) return;
    const uint32_t tk = lds0 + (uint32_t)(((st * 2) * KG + kg) * kElems + rw * R * D) * 2u, tv = tk + KG * kElems * 2u;
    const uint32_t lo = low_u32(e), hi = high_u32(e);
    auto base = [&](int x) { return reinterpret_cast<const uint8_t*>(compose_u64(__builtin_amdgcn_readlane(lo, x), __builtin_amdgcn_readlane(hi, x))); };
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      if (two) {   // (its own page for each lane)
        const int r = rw * R + i * RPL, key = key_of(step) + key_perm(r + q4);
        const int x = pages[(min(key, most) >> a.shift) - held];
        gload16_lds(kbase + (int64_t)x * a.kp + (int64_t)(key & in_page) * a.kr + (slot ^ ((r + q4) % UPR)) * 8, tk + (uint32_t)(i * 64 * 16));
      } else
        gload16_lds(base(i), k_off[i], tk + (uint32_t)(i * 64 * 16));
      gload16_lds(base(kLoads + i), v_off[i], tv + (uint32_t)(i * 64 * 16));
    }
  };

  uint32_t k_rd[KD], v_rd[DB];
#pragma unroll
  for (int kd = 0; kd < KD; ++kd) k_rd[kd] = (uint32_t)(l32 * UPR + ((2 * kd + g) ^ (l32 % UPR))) * 16u;
  {
    // transposed read: lane s of a 16-lane group reads 4 columns of key row 16g + s/4
    const int s16 = lane & 15, grp = lane >> 4, r = 16 * g + s16 / 4;
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      const int d = 32 * db + 16 * (grp & 1) + 4 * (s16 & 3);
      v_rd[db] = (uint32_t)(r * D * 2 + (((d / 8) ^ v_swz<D>(r)) * 16) + (d % 8) * 2);
    }
  }
  f32x16 oacc[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) oacc[db] = f32x16{};
  float m_run = -INFINITY, mlog2 = 0.f, l_run = 0.f;

  // The tile at LDS tk, tv; base: its first key
  auto compute = [&](int base, uint32_t tk, uint32_t tv) __attribute__((always_inline)) {
    constexpr int kWin = 2;   // LDS operand reads in flight
    f32x16 s;
    {
      auto rd = [&](int i) { return bitcast<V8>(*(const lds_u32x4*)(tk + k_rd[i])); };
      V8 win[kWin];
#pragma unroll
      for (int i = 0; i < kWin; ++i) win[i] = rd(i);
#pragma unroll
      for (int i = 0; i < KD; ++i) {
        const V8 x = win[i % kWin];
        if (i + kWin < KD) win[i % kWin] = rd(i + kWin);
        s = Elt<BF16>::mfma(x, qreg[i], i == 0 ? f32x16{} : s);
      }
    }
    float u[16];   // key base + 16·g + x
#pragma unroll
    for (int x = 0; x < 16; ++x) u[x] = s[x];
    if (a.cap) {
#pragma unroll
      for (int x = 0; x < 16; ++x) u[x] = __builtin_amdgcn_rcpf(-1.f - __builtin_amdgcn_exp2f(u[x] * a.u_scale));
    }
    if (a.slopes) {
      const float back = last - (float)(base + 16 * g);
#pragma unroll
      for (int x = 0; x < 16; ++x) u[x] = __builtin_fmaf(bco, back - (float)x, u[x]);
    }
    float mx = -INFINITY;
#pragma unroll
    for (int x = 0; x < 16; ++x) mx = fmaxf(mx, u[x]);
    mx = xhalf_max(mx);
    const bool need = mx > m_run + slack;
    if (__builtin_amdgcn_ballot_w64(need)) {
      // lanes that keep their max scale by exactly 1 (also avoids -inf - -inf)
      const float alpha = need ? __builtin_amdgcn_exp2f((m_run - mx) * c2) : 1.f;
      m_run = need ? mx : m_run;
      mlog2 = m_run == -INFINITY ? 0.f : m_run * c2;
      l_run *= alpha;
#pragma unroll
      for (int db = 0; db < DB; ++db) oacc[db] *= alpha;
    }
    constexpr int N = 2 * DB;
    auto rd = [&](int i) {
      const int j = i / DB, db = i % DB;
      const int o = j * 8 * D * 2;
      const s16x4 x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(tv + v_rd[db] + o));
      const s16x4 x1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(tv + v_rd[db] + o + 4 * D * 2));
      return bitcast<V8>(__builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    V8 win[kWin];
#pragma unroll
    for (int i = 0; i < kWin; ++i) win[i] = rd(i);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      f32x8 pf;
#pragma unroll
      for (int e = 0; e < 8; ++e) pf[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(u[j * 8 + e], c2, -mlog2));
      const V8 p = __builtin_convertvector(pf, V8);
      l_run = psum8<BF16>(p, l_run);   // of the rounded P: the weights that V meets
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        const int i = j * DB + db;
        const V8 x = win[i % kWin];
        if (i + kWin < N) win[i % kWin] = rd(i + kWin);
        oacc[db] = Elt<BF16>::mfma(x, p, oacc[db]);
      }
    }
  };

  fill();
  // Q and the slopes are here (they were asked for before the pages): were it left to their first
  // use, every step would wait for all loads in flight
#pragma unroll
  for (int kd = 0; kd < KD; ++kd) {
    u32x4 x = bitcast<u32x4>(qreg[kd]);
    asm volatile("" : "+v"(x));
    qreg[kd] = bitcast<V8>(x);
  }
  asm volatile("" : "+v"(bco), "+v"(last));
  uint64_t e = entries(0);
#pragma unroll
  for (int x = 0; x < S - 1; ++x) {
    if (x < steps) issue(x, x, e);
    e = entries(x + 1);
  }
  int st = 0;
  for (int i = 0; i < steps; ++i) {
    // the wave's loads of step i have landed; with four stages, each step has one tile
    if (S > 2 && i + S - 2 < steps) wait_vmcnt<(S - 2) * 2 * kLoads>();
    else wait_vmcnt<0>();
    wg_barrier();      // all waves' have, and all have left the stage of step i − 1
    if (i + S - 1 < steps) issue(i + S - 1, st == 0 ? S - 1 : st - 1, e);
    e = entries(i + S);
    const uint32_t tk = lds0 + (uint32_t)(((st * 2) * KG + kg) * kElems) * 2u, tv = tk + KG * kElems * 2u;
    st = st + 1 == S ? 0 : st + 1;
    if (there(i)) compute(key_of(i), tk, tv);
  }
  wait_vmcnt<0>();
  l_run = xhalf_sum(l_run);
  const int64_t at = (int64_t)sh.row + c;
  // The key groups' sums of the same columns, which the same lanes hold: group x of their waves
  // forms the x-th share of the 16·DB sums, and the others hand theirs over in LDS.
  constexpr int OWN = 16 * DB / KG, kSums = KG > 1 ? RW * KG * 16 * DB * 64 : 0;
  float* sj = reinterpret_cast<float*>(lds);   // [RW][KG shares][KG][OWN][64], then [RW][KG][2][64]
  float* sml = sj + kSums;
  static_assert((kSums + RW * KG * 2 * 64 + 1) * 4 <= kShLds<D, RW, KG>(), "sums fit");
  uint32_t* flag = reinterpret_cast<uint32_t*>(sml + RW * KG * 2 * 64);
  wg_barrier();   // the stages are free
  if (tid == 0) *flag = 0;
  if constexpr (KG > 1) {
#pragma unroll
    for (int x = 0; x < KG; ++x)
      if (x != kg)
#pragma unroll
        for (int y = 0; y < OWN; ++y) sj[(((rw * KG + x) * KG + kg) * OWN + y) * 64 + lane] = oacc[(x * OWN + y) / 16][(x * OWN + y) % 16];
    sml[((rw * KG + kg) * 2) * 64 + lane] = m_run;
    sml[((rw * KG + kg) * 2 + 1) * 64 + lane] = l_run;
  }
  __syncthreads();
  if (__builtin_amdgcn_ballot_w64(bad) && lane == 0) atomicOr(flag, 1u);
  float f[KG], m = m_run;
  if constexpr (KG > 1) {
    float l = 0.f;
#pragma unroll
    for (int x = 0; x < KG; ++x) m = fmaxf(m, f[x] = sml[((rw * KG + x) * 2) * 64 + lane]);
#pragma unroll
    for (int x = 0; x < KG; ++x) {
      // a group that saw nothing has sums of 0 (or NaN, which stay)
      f[x] = f[x] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((f[x] - m) * c2);
      l += sml[((rw * KG + x) * 2 + 1) * 64 + lane] * f[x];
    }
    l_run = l;
  } else f[0] = 1.f;
#pragma unroll
  for (int x = 0; x < KG; ++x)
    if (x == kg) {
      float y[OWN];
#pragma unroll
      for (int i = 0; i < OWN; ++i) {
        y[i] = oacc[(x * OWN + i) / 16][(x * OWN + i) % 16] * f[x];
#pragma unroll
        for (int z = 0; z < KG; ++z)
          if (z != x) y[i] += sj[(((rw * KG + x) * KG + z) * OWN + i) * 64 + lane] * f[z];
      }
      if (mine)
#pragma unroll
        for (int i = 0; i < OWN; i += 4) {
          const int e = x * OWN + i;   // sum e of the lane is that of d = 32·(e / 16) + 8·(e % 16 / 4) + 4·g + e % 4
          *reinterpret_cast<f32x4*>(a.part_o + at * D + e / 16 * 32 + e % 16 / 4 * 8 + g * 4) = f32x4{y[i], y[i + 1], y[i + 2], y[i + 3]};
        }
    }
  if (mine && kg == 0 && g == 0) {
    a.part_ml[at * 2] = m == -INFINITY ? -INFINITY : m * c2;
    a.part_ml[at * 2 + 1] = l_run;
  }
  __syncthreads();
  return *flag != 0;
}

// Workgroups that a CU holds.
template <int D, int RW, int KG> constexpr int kShPerCu() { return kShLds<D, RW, KG>() <= 78 * 1024 ? 2 : 1; }

template <int D, bool BF16, int RW, int KG>
__global__ __launch_bounds__(kShThreads) __attribute__((amdgpu_waves_per_eu(kShPerCu<D, RW, KG>())))
void shared_decode_kernel(const SharedArgs a) {
  __shared__ __align__(16) uint8_t lds[kShLds<D, RW, KG>()];
  __shared__ float sM[kShWaves][16], sL[kShWaves][16];
  __shared__ Share shares[kShWaves];
  int* words = reinterpret_cast<int*>(lds);
  const int wave = uni(threadIdx.x >> 6);
  // (one wave needs no barriers: 5 of them 12.9 us a call against 13.7, 126 29.6 against 29.9, 143 31.4 against 30.9)
  if (a.n_groups + a.b <= 128) {
    if (wave == 0) find_share<64>(a, blockIdx.x, words);
  } else find_share<kShThreads>(a, blockIdx.x, words);
  __syncthreads();
  // (each way keeps its share in LDS, and reads it and the arguments again: held from here on they would spill)
  auto keep = [&](const Share& sh) __attribute__((always_inline)) {
    if (threadIdx.x % 64 == 0) shares[wave] = sh;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  };
  auto share = [&]() __attribute__((always_inline)) {
    static_assert(sizeof(Share) % 4 == 0, "words");
    struct Words { int x[sizeof(Share) / 4]; } x;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(Share) / 4); ++i) x.x[i] = uni(reinterpret_cast<const int*>(&shares[wave])[i]);
    return bitcast<Share>(x);
  };
  uint8_t* slices = lds + kShWords * 4;   // (behind the plan, which the streams go on reading)
  static_assert(kShWords * 4 % 16 == 0 && Stream<D, BF16>::kSlice % 16 == 0, "rows of V are stored 16 bytes at a time");
  const int parts = uni(words[16]), number = ((int)blockIdx.x - parts) * kShWaves + wave;
  if (number >= 0) {
    Walk at{uni(words[4 * wave]) - 1, uni(words[4 * wave + 1]), uni(words[17]), number};
    Share next{};
#pragma unroll 1
    while (own_share(a, words, at, next)) {
      keep(next);
      kernarg<SharedArgs>& z = reload_kernarg(a);
      const Share sh = share();
      Stream<D, BF16> st;
      st.run(z, sh, sh.col0, sh.cols, 0, 1, slices + wave * Stream<D, BF16>::kSlice);
      st.store(z, sh);
    }
    return;
  }
  keep(group_share(a, words));
  __syncthreads();   // the plan's words are read
  if (!group_part<D, BF16, RW, KG>(reload_kernarg(a), share(), lds)) return;
  // a page outside the cache hides its keys, which only the stream can
  __syncthreads();
#pragma unroll 1
  for (int c = 0; c < uni(shares[wave].cols); c += 16) {
    kernarg<SharedArgs>& z = reload_kernarg(a);
    const Share sh = share();
    const int cols = min(16, sh.cols - c);
    Stream<D, BF16> st;
    st.run(z, sh, sh.col0 + c, cols, wave, kShWaves, slices + wave * Stream<D, BF16>::kSlice);
    st.join(reload_kernarg(a), share(), c, cols, slices, sM, sL);
  }
}

// The parts of (request, head) bh: its group's and its own.
struct Parts {
  int shared, own;     // how many
  int at0, at1;        // rows of the first ones; steps from one to the next: columns, 16
};
__device__ __forceinline__ Parts parts_of(const SharedArgs& a, int b, int h) {
  const int hk = h / a.ratio, n = h - hk * a.ratio;
  const i32x4 rec = *reinterpret_cast<const i32x4*>(a.rec + (int64_t)(a.n_groups + b) * 4);
  const uint32_t per = a.rec[(int64_t)(a.n_groups + a.b) * 4];
  Parts p{0, 0, 0, 0};
  const int count = rec[2], group = rec[3], unit = hk * a.groups + n / 16;
  if (count > 0) {
    const uint32_t from = (uint32_t)rec[1] + (uint32_t)(unit * count), w0 = from / per, w1 = (from + (uint32_t)count - 1) / per;
    p.own = (int)(w1 - w0) + 1;
    p.at1 = a.own_rows + (rec[0] + (int)w0 + b * a.hk * a.groups + unit) * 16 + n % 16;
  }
  if (group >= 0 && a.lens[b] > 0 && a.cols > 0) {
    const int* r = a.rec + (int64_t)group * 4;
    const int first = r[2], end = min(a.cu[group + 1], a.b);
    const int blocks = ((end - first) * a.ratio + a.columns - 1) / a.columns, col = (b - first) * a.ratio + n;
    p.shared = r[1];
    p.at0 = r[0] + (hk * blocks + col / a.columns) * p.shared * a.columns + col % a.columns;
  }
  return p;
}

// One workgroup per (request, head): its group's parts and its own, weighted by
// 2^(m_s − m). Its 256 threads are 1024 / D rows of D / 4 threads; a row takes every so
// many parts, 8 of them in flight, with a running max; the rows' sums are joined in LDS.
// MANY: a wave each, four to a workgroup.
template <int D, bool BF16, bool MANY>
__global__ __launch_bounds__(256) void shared_join_kernel(const SharedArgs a) {
  constexpr int TPR = D / 4, ROWS = (MANY ? 64 : 256) / TPR, J = MANY ? 4 : 8, GROUPS = MANY ? 4 : 1;
  __shared__ float sAcc[GROUPS][ROWS][D], sMax[GROUPS][ROWS], sSum[GROUPS][ROWS];
  const int who = MANY ? uni(threadIdx.x >> 6) : 0, tid = MANY ? threadIdx.x & 63 : threadIdx.x;
  const int64_t bh = (int64_t)blockIdx.x * GROUPS + who;
  const bool real = bh < (int64_t)a.b * a.h;
  const int b = real ? (int)(bh / a.h) : 0, h = real ? (int)(bh % a.h) : 0;
  const Parts pt = parts_of(a, b, h);
  const int parts = pt.shared + pt.own;
  const bool written = !real || (pt.shared == 0 && pt.own == 1);   // by its one part
  if (!MANY && written) return;
  auto at = [&](int s) { return s < pt.shared ? (int64_t)pt.at0 + (int64_t)s * a.columns : (int64_t)pt.at1 + (int64_t)(s - pt.shared) * 16; };
  const int row = tid / TPR, c = tid % TPR;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  for (int s0 = row; s0 < (written ? 0 : parts); s0 += ROWS * J) {
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
  for (int i = 0; i < 4; ++i) sAcc[who][row][c * 4 + i] = acc[i];
  if (c == 0) {
    sMax[who][row] = m;
    sSum[who][row] = l;
  }
  __syncthreads();
  if (tid < TPR && !written) {
    float top = sMax[who][0];
#pragma unroll
    for (int r = 1; r < ROWS; ++r) top = fmaxf(top, sMax[who][r]);
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
    float t = 0.f;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const float f = sMax[who][r] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(sMax[who][r] - top);
      t += sSum[who][r] == 0.f ? 0.f : sSum[who][r] * f;
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] += sSum[who][r] == 0.f ? 0.f : sAcc[who][r][c * 4 + i] * f;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = t == 0.f ? 0.f : y[i] / t;
    store4<BF16>(a.o + (int64_t)b * a.o_bs + (int64_t)h * a.o_hs + c * 4, y);
  }
}
