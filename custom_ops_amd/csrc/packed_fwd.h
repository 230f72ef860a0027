// packed_fwd.h — attention over packed sequences, with scores that are capped by
// a tanh, biased by distance, and masked by structure (documents, causal, window,
// prefix). Included by serve.hip inside namespace mi355fa.
//
// Per sequence and head, O = softmax(f(scale·Q·Kᵀ))·V in one pass over the keys:
// running row max and sum in fp32, P rounded to the input type for the second
// product. Bound: the two products, 4·d operations per seen pair on the matrix
// core; the vector unit's exponentials (one per pair, three with a cap) run
// beside them.
//
//  * A workgroup is RW·KG waves: RW of 32 rows each, of one sequence and `pack` heads
//    of one KV head, and KG groups of them that take every KG-th key tile and join
//    their sums in LDS at the end. A wave computes Sᵀ = K·Qᵀ, so that a lane holds one
//    row's scores. No mask is read: a row's seen keys are [lo, hi) and [0, prefix), and
//    only key tiles that a border crosses compare keys with them.
//  * Key tiles that no row of the workgroup sees are not visited.
//  * Offsets stay on the device: the workgroup finds its rows by a scan over the
//    sequences, the longest blocks first, so the grid holds total_q / BM + n_seqs + 2 blocks per head, the most
//    that any split of the rows can need.
//  * K and V tiles come HBM → LDS by DMA, two stages, one barrier per tile.

struct PackedArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* o;
  const int* cu_q;
  const int* cu_k;
  const int* prefix;
  const float* slopes;
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, o_ts, o_hs;
  int tq, tk, n, h, ratio;
  int causal, window;   // window: 2^30 where there is none
  int pack;             // heads of one KV head that share a workgroup: divides ratio, 1, 2 or 4
  int bm_shift;         // log2 of a block's rows: 32·RW / pack
  int levels;           // classes of block lengths (find_block)
  int fold;             // see folded
  float u_scale;        // capped: 2·log2(e)·scale / softcap
  float tanh_lim, tanh_p[4];   // capped: scores up to which tanh is the polynomial, and its factors
  float c2;             // scores u to log2 units: scale·log2(e), capped 2·softcap·log2(e)
  float bias;           // slopes to u: −1/scale, capped −1/(2·softcap)
};

// A row block: rows m0 .. of the sequence's lq, which start at global row q0, its lk
// keys, which start at global key k0, and the prefix that all rows see.
struct RowBlock {
  int q0, lq, m0, k0, lk, pre;
};

__device__ __forceinline__ int wave_max(int x) {   // of values >= 0, over the wave's lanes
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));
  return __builtin_amdgcn_readlane(x, 63);
}

// Row block t of a head, the blocks with the most key tiles first: in a.levels classes,
// each of half the tiles of the one before, so that no long block starts last. Segment
// e = 0 .. n + 1 holds the rows from cu[e − 1] to cu[e] (0 before the first, tq behind
// the last): sequence e − 1, or rows of none, which have no keys. Offsets are held to
// 0 .. tq. All waves find the same, each for itself, 64 segments at a time; of more
// than 62 sequences (short ones, then) there is one class.
__device__ __forceinline__ bool find_block(const PackedArgs& a, int t, RowBlock& rb) {
  const int lane = threadIdx.x & 63;
  const int iters = (a.n + 2 + 63) / 64;
  struct Seg { int c0, rows, k0, lk, pre; };
  auto segment = [&](int it) __attribute__((always_inline)) {
    const int e = it * 64 + lane;
    Seg x{0, 0, 0, 0, 0};
    if (e <= a.n + 1) {
      const bool real = e >= 1 && e <= a.n;
      const int c1 = e == a.n + 1 ? a.tq : a.cu_q[e], k1 = real ? a.cu_k[e] : 0;
      const int c0 = e == 0 ? 0 : a.cu_q[e - 1], k0 = real ? a.cu_k[e - 1] : 0;
      const int pre = real && a.prefix ? a.prefix[e - 1] : 0;
      x.c0 = min(max(c0, 0), a.tq);
      x.rows = max(0, min(max(c1, 0), a.tq) - x.c0);
      x.k0 = min(max(k0, 0), a.tk);
      x.lk = real ? max(0, min(max(k1, 0), a.tk) - x.k0) : 0;
      x.pre = min(max(pre, 0), x.lk);
    }
    return x;
  };
  const RowSpans rs{a.causal, a.window, a.bm_shift};
  Seg x = segment(0);
  const int levels = iters == 1 ? a.levels : 1;
  int most = 0;
  if (levels > 1) {
    const int n = block_count(rs, x.rows);
    most = wave_max(n ? block_span(rs, x.rows, x.lk, n - 1) : 0);
  }
  int run = 0;
#pragma unroll 1
  for (int level = 0; level < levels; ++level) {
    for (int it = 0; it < iters; ++it) {
      if (iters > 1) x = segment(it);
      const int b0 = first_over(rs, x.rows, x.lk, class_floor(most, level, levels));
      const int cnt = first_over(rs, x.rows, x.lk, class_ceil(most, level)) - b0;
      const int incl = wave_scan(cnt);
      const uint64_t hit = __builtin_amdgcn_ballot_w64(run + incl > t);
      if (hit) {
        const int l = __builtin_ctzll(hit);
        const int left = run + (int)__builtin_amdgcn_readlane(incl, l) - 1 - t;   // blocks of the class behind t in its segment
        rb.m0 = ((int)__builtin_amdgcn_readlane(b0, l) + left) << a.bm_shift;
        rb.q0 = __builtin_amdgcn_readlane(x.c0, l);
        rb.lq = __builtin_amdgcn_readlane(x.rows, l);
        rb.k0 = __builtin_amdgcn_readlane(x.k0, l);
        rb.lk = __builtin_amdgcn_readlane(x.lk, l);
        rb.pre = __builtin_amdgcn_readlane(x.pre, l);
        return true;
      }
      run += __builtin_amdgcn_readlane(incl, 63);
    }
  }
  return false;
}

// Keys of a tile; and waves per SIMD: of two workgroups on a CU where their LDS allows it
template <int D, int KG> constexpr int kKeys = KG * D > 256 ? 32 : 64;
template <int D, int RW, int KG> constexpr int kWavesPerEu = RW * KG / 4 * (2 * 4 * KG * kKeys<D, KG> * D * 2 <= 160 * 1024 ? 2 : 1);

template <int D, bool BF16, bool CAP, bool BIAS, int RW, int KG>
__global__ __launch_bounds__(64 * RW * KG) __attribute__((amdgpu_waves_per_eu(kWavesPerEu<D, RW, KG>)))
void packed_fwd_kernel(const PackedArgs a) {
  typedef typename Elt<BF16>::v8 V8;
  constexpr int WAVES = RW * KG, kTile = kKeys<D, KG>, NKB = kTile / 32;
  constexpr int UPR = D / 8, KD = D / 16, DB = D / 32;
  constexpr int kElems = kTile * D, kWaveLoads = kTile * UPR / 64;   // of a K or V tile
  constexpr int kLoads = (kWaveLoads + WAVES - 1) / WAVES;
  __shared__ __align__(16) uint16_t sKV[4][KG * kElems];   // two K stages, two V stages

  // Head groups fastest, KV heads before the groups of one: workgroup i runs on XCD
  // i % 8, so a KV head's keys stay on few XCDs' L2
  RowBlock rb;
  const int groups = a.h / a.pack, hks = a.h / a.ratio;
  if (!find_block(a, folded(blockIdx.x / groups, a.fold, gridDim.x / groups), rb)) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6);
  const int rw = wave % RW, kg = wave / RW;
  const int l32 = lane & 31, g = lane >> 5;
  const int hg = blockIdx.x % groups, hk = hg % hks;
  const int h = hk * a.ratio + hg / hks * a.pack + rw % a.pack;

  const int k0 = rb.k0, lk = rb.lk, pre = rb.pre;
  const int off = lk - rb.lq;   // row r is at key position r + off
  auto hi_of = [&](int i) { return a.causal ? min(lk, i + 1) : min(lk, i + a.window); };
  auto lo_of = [&](int i) { return max(0, i - a.window + 1); };

  // key tiles that some row of the block sees: those of the prefix, then a range
  const int i0 = rb.m0 + off, i1 = min(rb.m0 + (1 << a.bm_shift), rb.lq) - 1 + off;
  const int np = (pre + kTile - 1) / kTile;
  const int hi_b = max(0, hi_of(i1)), lo_b = lo_of(i0);
  const int t0 = max(np, lo_b / kTile);
  const int t1 = lo_b < hi_b ? (hi_b + kTile - 1) / kTile : 0;
  const int cnt = np + max(0, t1 - t0);
  auto tile_at = [&](int i) { return i < np ? i : i - np + t0; };

  // this wave's rows, and this lane's
  const int w0 = rb.m0 + rw / a.pack * 32, w1 = min(w0 + 31, rb.lq - 1);
  const int row = w0 + l32;
  const bool mine = row < rb.lq;
  const int ia = row + off;
  const int hi = mine ? hi_of(ia) : 0, lo = lo_of(ia), pl = mine ? pre : 0;
  const int w_hi0 = hi_of(w0 + off), w_hi1 = hi_of(w1 + off), w_lo0 = lo_of(w0 + off), w_lo1 = lo_of(w1 + off);

  uint32_t k_off[kLoads], v_off[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int u = (i * WAVES + wave) * 64 + lane;
    const int r = u / UPR, slot = u % UPR;
    const int key = (r & ~31) + key_perm(r & 31);
    k_off[i] = (uint32_t)(key * (int)a.k_ts + (slot ^ (r % UPR)) * 8) * 2u;
    v_off[i] = (uint32_t)(r * (int)a.v_ts + (slot ^ v_swz<D>(r)) * 8) * 2u;
  }
  const uint16_t* kb = a.k + (int64_t)k0 * a.k_ts + (int64_t)hk * a.k_hs;
  const uint16_t* vb = a.v + (int64_t)k0 * a.v_ts + (int64_t)hk * a.v_hs;
  // bytes that a number of rows reach over
  auto span = [](int rows, int64_t ts) { return rows > 0 ? ((uint32_t)(rows - 1) * (uint32_t)ts + D) * 2u : 0u; };
  auto issue = [&](const uint16_t* base, int64_t ts, const uint32_t (&offs)[kLoads], int tile, uint16_t* dst) __attribute__((always_inline)) {
    const int first = tile * kTile;
    const i32x4 r = make_rsrc_words(base + (int64_t)first * ts, span(min(kTile, lk - first), ts));
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      if (kWaveLoads % WAVES == 0 || i * WAVES + wave < kWaveLoads)
        bload16_lds(r, lds_addr(dst) + (uint32_t)((i * WAVES + wave) * 64 * 16), offs[i]);
  };
  auto issue_step = [&](int i, int st) __attribute__((always_inline)) {   // tiles i·KG .. into stage st
#pragma unroll
    for (int j = 0; j < KG; ++j)
      if (i * KG + j < cnt) {
        const int tile = tile_at(i * KG + j), left = lk - tile * kTile;
        issue(kb, a.k_ts, k_off, tile, sKV[st] + j * kElems);
        issue(vb, a.v_ts, v_off, tile, sKV[2 + st] + j * kElems);
        // V rows behind the last key are 0, since they meet a P of 0. They lie outside the
        // resource (V's rows do not overlap: v_ts >= D), so the DMA brings nothing of them
        if (left < kTile)
          for (int x = left * UPR + tid; x < kTile * UPR; x += 64 * WAVES)
            reinterpret_cast<u32x4*>(sKV[2 + st] + j * kElems)[x] = u32x4{0u, 0u, 0u, 0u};
      }
  };

  issue_step(0, 0);
  V8 qreg[KD];
  {
    const rsrc_t rq = make_rsrc(a.q + (int64_t)(rb.q0 + w0) * a.q_ts + (int64_t)h * a.q_hs,
                                span(min(32, rb.lq - w0), a.q_ts));
#pragma unroll
    for (int kd = 0; kd < KD; ++kd)
      qreg[kd] = bitcast<V8>(bload16(rq, (uint32_t)(l32 * (int)a.q_ts + kd * 16 + g * 8) * 2u));
  }
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
  const float c2 = a.c2, slack = kSlackLog2 / a.c2;
  const float bco = BIAS ? a.slopes[h] * a.bias : 0.f;
  float m_run = -INFINITY, mlog2 = 0.f, l_run = 0.f;
  wait_vmcnt<0>();

  constexpr int kWin = 2;   // LDS operand reads in flight (4 and 8 measured the same)
  f32x16 s[NKB];
  auto qk = [&](int base, const uint16_t* tK) __attribute__((always_inline)) {
    // the distance bias is where the sums start from; keys that are all behind the wave's
    // rows take one operation each
    constexpr bool START = BIAS && !CAP;
    if constexpr (START) {
      const float x0 = (float)(ia - base - g * 16), bx = bco * x0;
      if (base + kTile <= w0 + off + 1) {
#pragma unroll
        for (int c = 0; c < 16 * NKB; ++c) s[c / 16][c % 16] = __builtin_fmaf(-bco, (float)(c / 16 * 32 + c % 16), bx);
      } else {
#pragma unroll
        for (int c = 0; c < 16 * NKB; ++c) s[c / 16][c % 16] = bco * __builtin_fabsf(x0 - (float)(c / 16 * 32 + c % 16));
      }
    }
    const uint8_t* k8 = reinterpret_cast<const uint8_t*>(tK);
    auto rd = [&](int i) {
      return bitcast<V8>(*reinterpret_cast<const u32x4*>(k8 + (i / KD) * 32 * D * 2 + k_rd[i % KD]));
    };
    V8 win[kWin];
#pragma unroll
    for (int i = 0; i < kWin; ++i) win[i] = rd(i);
#pragma unroll
    for (int i = 0; i < NKB * KD; ++i) {
      const V8 x = win[i % kWin];
      if (i + kWin < NKB * KD) win[i % kWin] = rd(i + kWin);
      s[i / KD] = Elt<BF16>::mfma(x, qreg[i % KD], i % KD == 0 && !START ? f32x16{} : s[i / KD]);
    }
  };
  auto softmax_pv = [&](int base, const uint16_t* tV) __attribute__((always_inline)) {
    const uint8_t* v8 = reinterpret_cast<const uint8_t*>(tV);
    // u: scores up to the factor c2. Capped: tanh z = 1 − 2 / (e^{2z} + 1), and the
    // 1 cancels in the softmax, so u = −1 / (e^{2z} + 1) with c2 = 2·softcap·log2(e).
    // Where |z| is below 1/2 it is (tanh z − 1) / 2 with tanh z / z as a polynomial in z²
    // (least squares in Chebyshev nodes, off by 6·10^-7): 5 operations of 4 cycles a score,
    // where the two transcendental ones take 16 each. The two forms differ in their last
    // bits, so no score of an unseen key may choose: the whole wave chooses together on a
    // tile that all of its rows see, each lane by the scores its row sees on the others
    // (4099 tokens in 3 documents with window and prefix: 57.6 us, of which that takes 2).
    float u[16 * NKB];   // key 32·(c / 16) + c % 16, from the lane's first
#pragma unroll
    for (int c = 0; c < 16 * NKB; ++c) u[c] = s[c / 16][c % 16];
    // Only a tile that a border crosses hides scores: a bit for each key of the lane, and
    // two operations a score (a compare with each border takes four and the scalar unit's)
    auto crossed = [&]() { return base + kTile > pre && (base + kTile > w_hi0 || base < w_lo1); };
    auto hidden_of = [&](int b) {   // of the lane's 16 keys
      const int first = base + b * 32 + g * 16;
      auto below = [&](int x) { return (1u << min(max(x - first, 0), 16)) - 1u; };   // keys before x
      return (int)~((below(hi) & ~below(lo)) | below(pl));
    };
    auto hides = [](int hidden, int i) { return (uint32_t)__builtin_amdgcn_sbfe(hidden, i, 1); };   // all ones where hidden
    if constexpr (CAP) {
      const float x0 = (float)(ia - base - g * 16);
      auto biased = [&](int c, float x) {
        return BIAS ? __builtin_fmaf(bco, __builtin_fabsf(x0 - (float)(c / 16 * 32 + c % 16)), x) : x;
      };
      bool small = false;
      if constexpr (D == 128) {   // (d = 64 has no registers for the choice at 4 waves a SIMD)
        float big = 0.f;
        if (crossed()) {
#pragma unroll
          for (int b = 0; b < NKB; ++b) {
            const int hidden = hidden_of(b);
#pragma unroll
            for (int i = 0; i < 16; ++i) big = fmaxf(big, __uint_as_float(__float_as_uint(u[b * 16 + i]) & 0x7fffffffu & ~hides(hidden, i)));
          }
          small = !(big > a.tanh_lim);
        } else {
#pragma unroll
          for (int c = 0; c < 16 * NKB; ++c) big = fmaxf(big, __builtin_fabsf(u[c]));
          small = __builtin_amdgcn_ballot_w64(big > a.tanh_lim) == 0;
        }
      }
      if (small) {
#pragma unroll
        for (int c = 0; c < 16 * NKB; ++c) {
          const float t = u[c] * u[c];
          const float p = __builtin_fmaf(__builtin_fmaf(__builtin_fmaf(a.tanh_p[3], t, a.tanh_p[2]), t, a.tanh_p[1]), t, a.tanh_p[0]);
          u[c] = biased(c, __builtin_fmaf(u[c], p, -0.5f));
        }
      } else {
#pragma unroll
        for (int c = 0; c < 16 * NKB; ++c) u[c] = biased(c, __builtin_amdgcn_rcpf(-1.f - __builtin_amdgcn_exp2f(u[c] * a.u_scale)));
      }
    }
    if (crossed()) {
#pragma unroll
      for (int b = 0; b < NKB; ++b) {
        const int hidden = hidden_of(b);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const uint32_t h = hides(hidden, i);
          float& x = u[b * 16 + i];
          x = __uint_as_float((h & 0xff800000u) | (~h & __float_as_uint(x)));
        }
      }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int c = 0; c < 16 * NKB; ++c) mx = fmaxf(mx, u[c]);
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
    {
      constexpr int N = 2 * NKB * DB;
      auto rd = [&](int i) {
        const int j = i / DB, db = i % DB;
        const int o = ((j / 2) * 32 + (j % 2) * 8) * D * 2;
        const s16x4 x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(v8 + v_rd[db] + o));
        const s16x4 x1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(v8 + v_rd[db] + o + 4 * D * 2));
        return bitcast<V8>(__builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7));
      };
      V8 win[kWin];
#pragma unroll
      for (int i = 0; i < kWin; ++i) win[i] = rd(i);
      auto pstep = [&](int j) {
        f32x8 pf;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          pf[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(u[j * 8 + e], c2, -mlog2));
        return __builtin_convertvector(pf, V8);
      };
      V8 pcur = pstep(0);
      l_run = psum8<BF16>(pcur, l_run);   // of the rounded P: the weights that V meets
#pragma unroll
      for (int j = 0; j < 2 * NKB; ++j) {
        V8 pnext;
        if (j < 2 * NKB - 1) pnext = pstep(j + 1);
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          const int i = j * DB + db;
          const V8 x = win[i % kWin];
          if (i + kWin < N) win[i % kWin] = rd(i + kWin);
          oacc[db] = Elt<BF16>::mfma(x, pcur, oacc[db]);
        }
        if (j < 2 * NKB - 1) {
          l_run = psum8<BF16>(pnext, l_run);
          pcur = pnext;
        }
      }
    }
  };
  // Step i: tiles i·KG .., one for each key group
  const int steps = (cnt + KG - 1) / KG;
  auto iter = [&](auto stc, int i) __attribute__((always_inline)) {
    constexpr int ST = decltype(stc)::value;   // i % 2
    wait_vmcnt<0>();   // the wave's loads of step i have landed
    wg_barrier();      // all waves' have, and all have left the stage of step i − 1
    issue_step(i + 1, ST ^ 1);
    if (i * KG + kg >= cnt || w0 >= rb.lq) return;
    const int base = tile_at(i * KG + kg) * kTile;
    if (base >= pre && (base >= w_hi1 || base + kTile <= w_lo0)) return;   // no row of the wave sees it
    qk(base, sKV[ST] + kg * kElems);

    softmax_pv(base, sKV[2 + ST] + kg * kElems);
  };
  int i = 0;
  for (; i + 1 < steps; i += 2) {
    iter(std::integral_constant<int, 0>{}, i);
    iter(std::integral_constant<int, 1>{}, i + 1);
  }
  if (i < steps) iter(std::integral_constant<int, 0>{}, i);

  wait_vmcnt<0>();
  wg_barrier();   // the stages are free
  l_run = xhalf_sum(l_run);
  // the key groups' sums of the same rows, in the lanes that hold them
  constexpr int kJoin = (DB * 16 + 2) * 64;   // floats of one wave
  float* sj = reinterpret_cast<float*>(sKV[0]);
  if constexpr (KG > 1) {
    static_assert(RW * (KG - 1) * kJoin * 4 <= (int)sizeof(sKV), "joined sums fit");
    if (kg > 0) {
      float* at = sj + (rw * (KG - 1) + kg - 1) * kJoin + lane;
      at[0] = m_run;
      at[64] = l_run;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e) at[(2 + db * 16 + e) * 64] = oacc[db][e];
    }
    __syncthreads();
    if (kg > 0) return;
#pragma unroll 1
    for (int k = 1; k < KG; ++k) {
      const float* at = sj + (rw * (KG - 1) + k - 1) * kJoin + lane;
      const float mk = at[0], lk2 = at[64];
      const float top = fmaxf(m_run, mk);
      // a group that saw nothing has sums of 0 (or NaN, which stay)
      const float f0 = m_run == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m_run - top) * c2);
      const float f1 = mk == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((mk - top) * c2);
      l_run = l_run * f0 + lk2 * f1;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e) oacc[db][e] = oacc[db][e] * f0 + at[(2 + db * 16 + e) * 64] * f1;
      m_run = top;
    }
  }

  kernarg<PackedArgs>& z = reload_kernarg(a);
  // O through LDS, each wave in a slice of its own (which no other wave reads), so that
  // a store instruction writes whole rows
  uint8_t* stg = KG > 1 ? reinterpret_cast<uint8_t*>(sj + rw * (KG - 1) * kJoin) : reinterpret_cast<uint8_t*>(sKV[0]) + wave * 32 * D * 2;
  static_assert(RW * 32 * D * 2 <= (int)sizeof(sKV) && 32 * D * 2 <= kJoin * 4, "staging fits");
  const float l = l_run;
  const float inv = (l == 0.f || l != l) ? 1.f : 1.f / l;
  bool odd = false;   // a value that is not finite
  constexpr int CH = D / 8, RPI = 64 / CH;
  typedef __attribute__((ext_vector_type(4))) __bf16 bf16x4;
  typedef __attribute__((ext_vector_type(4))) _Float16 f16x4;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {
      f32x4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = oacc[db][q4 * 4 + e] * inv;
        odd |= !(__builtin_fabsf(x[e]) < INFINITY);
      }
      u32x2 packed;
      if constexpr (BF16) packed = bitcast<u32x2>(__builtin_convertvector(x, bf16x4));
      else packed = bitcast<u32x2>(__builtin_convertvector(x, f16x4));
      const int c = db * 4 + q4;
      *reinterpret_cast<u32x2*>(stg + l32 * D * 2 + ((c ^ (l32 & (CH - 1))) * 16) + g * 8) = packed;
    }
  const rsrc_t ro = make_rsrc(z.o + (int64_t)(rb.q0 + w0) * z.o_ts + (int64_t)h * z.o_hs,
                              span(min(32, rb.lq - w0), z.o_ts));
  const int ch = lane % CH, r0 = lane / CH;
#pragma unroll
  for (int k = 0; k < 32 / RPI; ++k) {
    const int r = r0 + k * RPI;
    const u32x4 x = *reinterpret_cast<const u32x4*>(stg + r * D * 2 + ((ch ^ (r & (CH - 1))) * 16));
    __builtin_amdgcn_raw_buffer_store_b128(x, ro, (uint32_t)(r * (int)z.o_ts + ch * 8) * 2u, 0, 0);
  }

  // A tile that a border crosses multiplies the V of its unseen keys by a P of 0, which
  // makes NaN of what is not finite. So rows of finite weights with such values look at
  // the unseen keys of those tiles, and where one of them holds a value that is not finite
  // in a column, and no seen one a NaN, that column is formed again from the seen keys alone.
  const uint64_t odds = __builtin_amdgcn_ballot_w64(odd && mine && l < INFINITY);
  uint32_t rows = (uint32_t)(odds | odds >> 32);
  if (rows) {
    wait_vmcnt<0>();   // the rows are stored
    constexpr int C = D / 64;   // columns lane, lane + 64 of a row
    const uint16_t* kz = z.k + (int64_t)k0 * z.k_ts + (int64_t)hk * z.k_hs;
    const uint16_t* vz = z.v + (int64_t)k0 * z.v_ts + (int64_t)hk * z.v_hs;
    auto num = [](uint16_t x) {
      if constexpr (BF16) return __uint_as_float((uint32_t)x << 16);
      else return (float)bitcast<_Float16>(x);
    };
    while (rows) {
      const int r = __builtin_ctz(rows);
      rows &= rows - 1;
      const int at = w0 + r + off, r_hi = min(lk, z.causal ? at + 1 : at + z.window), r_lo = max(0, at - z.window + 1);
      auto sees = [&](int j) { return (j < r_hi && j >= r_lo) || j < pre; };
      bool out[C], unseen[C] = {}, known[C] = {}, again[C], any = false;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int d = lane + 64 * c;
        const float x = num(*reinterpret_cast<const uint16_t*>(stg + r * D * 2 + (((d / 8) ^ (r & (CH - 1))) * 16) + d % 8 * 2));
        out[c] = !(__builtin_fabsf(x) < INFINITY);
      }
      for (int t = 0; t < cnt; ++t) {
        const int base = tile_at(t) * kTile;
        if (base + kTile <= pre || (base + kTile <= r_hi && base >= r_lo)) continue;   // all seen
        for (int j = base; j < min(base + kTile, lk); ++j)
#pragma unroll
          for (int c = 0; c < C; ++c) {
            const float x = num(vz[(int64_t)j * z.v_ts + lane + 64 * c]);
            unseen[c] |= !(__builtin_fabsf(x) < INFINITY) && !sees(j);
            known[c] |= x != x && sees(j);
          }
      }
#pragma unroll
      for (int c = 0; c < C; ++c) any |= again[c] = out[c] && unseen[c] && !known[c];
      if (!__builtin_amdgcn_ballot_w64(any)) continue;
      const uint16_t* q = z.q + (int64_t)(rb.q0 + w0 + r) * z.q_ts + (int64_t)h * z.q_hs;
      const float bc = BIAS ? z.slopes[h] * z.bias : 0.f;
      float m = -INFINITY, sum = 0.f, acc[C] = {};
      for (int t = 0; t < cnt; ++t) {
        const int base = tile_at(t) * kTile, j = base + lane;   // a key each lane
        const bool seen = lane < kTile && j < lk && sees(j);
        float u = -INFINITY;
        if (seen) {
          u = 0.f;
          for (int d = 0; d < D; ++d) u = __builtin_fmaf(num(q[d]), num(kz[(int64_t)j * z.k_ts + d]), u);
          if constexpr (CAP) u = __builtin_amdgcn_rcpf(-1.f - __builtin_amdgcn_exp2f(u * z.u_scale));
          if constexpr (BIAS) u = __builtin_fmaf(bc, __builtin_fabsf((float)(at - j)), u);
        }
        float top = u;
#pragma unroll
        for (int x = 1; x < 64; x *= 2) top = fmaxf(top, __shfl_xor(top, x));
        top = fmaxf(top, m);
        if (top == -INFINITY) continue;
        const float old = __builtin_amdgcn_exp2f((m - top) * c2), w = seen ? __builtin_amdgcn_exp2f((u - top) * c2) : 0.f;
        m = top;
        sum = sum * old + w;   // of the lane's keys
#pragma unroll
        for (int c = 0; c < C; ++c) acc[c] *= old;
        for (uint64_t left = __builtin_amdgcn_ballot_w64(seen); left; left &= left - 1) {
          const int x = __builtin_ctzll(left);
          const float p = __shfl(w, x);
#pragma unroll
          for (int c = 0; c < C; ++c) acc[c] = __builtin_fmaf(p, num(vz[(int64_t)(base + x) * z.v_ts + lane + 64 * c]), acc[c]);
        }
      }
#pragma unroll
      for (int x = 1; x < 64; x *= 2) sum += __shfl_xor(sum, x);
      uint16_t* o = z.o + (int64_t)(rb.q0 + w0 + r) * z.o_ts + (int64_t)h * z.o_hs;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const float y = sum == 0.f ? 0.f : acc[c] / sum;
        if (again[c]) {
          if constexpr (BF16) o[lane + 64 * c] = bitcast<uint16_t>((__bf16)y);
          else o[lane + 64 * c] = bitcast<uint16_t>((_Float16)y);
        }
      }
    }
  }
}
