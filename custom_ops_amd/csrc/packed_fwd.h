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
//  * A workgroup serves BM = 32·WAVES rows of one sequence and one head; each
//    wave owns 32 of them and computes Sᵀ = K·Qᵀ, so that a lane holds one row's
//    scores. No mask is read: a row's seen keys are [lo, hi) and [0, prefix), and
//    only key tiles that a border crosses compare keys with them.
//  * Key tiles that no row of the workgroup sees are not visited.
//  * Offsets stay on the device: the workgroup finds its sequence by a scan over
//    cu_q, so the grid holds total_q / BM + n_seqs + 2 blocks per head, the most
//    that any split of the rows can need.
//  * K and V tiles come HBM → LDS by DMA, two stages, one barrier per tile.

constexpr int kTile = 64;   // keys per tile
constexpr float kSlackLog2 = 8.f;   // the running max moves when a score passes it by this (P <= 2^8)

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
  int blocks;           // row blocks per head in the grid
  float u_scale;        // capped: 2·log2(e)·scale / softcap
  float c2;             // scores u to log2 units: scale·log2(e), capped 2·softcap·log2(e)
  float bias;           // slopes to u: −1/scale, capped −1/(2·softcap)
};

// A row block: rows m0 .. of the sequence's lq, which start at global row q0.
struct RowBlock {
  int seq;   // -1: rows of no sequence
  int q0, lq, m0;
};

// Inclusive sum over the wave's lanes: rows of 16 by shifts, then the rows' sums.
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);   // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);   // row_bcast:15 into rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);   // row_bcast:31 into rows 2 and 3
  return x;
}

// Block t of the rows, counted from the last sequence's last rows (with a causal
// mask the longest blocks run first). Segment e = 0 .. n + 1 holds the rows from
// cu[e − 1] to cu[e] (0 before the first, tq behind the last): sequence e − 1, or
// rows of none. Offsets are held to 0 .. tq.
template <int BM>
__device__ __forceinline__ bool find_block(const PackedArgs& a, int t, RowBlock& rb) {
  const int lane = threadIdx.x & 63;
  int run = 0;
  for (int base = 0; base < a.n + 2; base += 64) {
    const int e = a.n + 1 - (base + lane);
    int c0 = 0, c1 = 0;
    if (e >= 0) {
      c0 = e == 0 ? 0 : min(max(a.cu_q[e - 1], 0), a.tq);
      c1 = e == a.n + 1 ? a.tq : min(max(a.cu_q[e], 0), a.tq);
    }
    const int cnt = c1 > c0 ? (c1 - c0 + BM - 1) / BM : 0;
    const int incl = wave_scan(cnt);
    const uint64_t hit = __builtin_amdgcn_ballot_w64(run + incl > t);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      const int es = uni(__builtin_amdgcn_readlane(e, l));
      const int ends = run + (int)__builtin_amdgcn_readlane(incl, l);
      rb.q0 = __builtin_amdgcn_readlane(c0, l);
      rb.lq = (int)__builtin_amdgcn_readlane(c1, l) - rb.q0;
      rb.m0 = (ends - 1 - t) * BM;
      rb.seq = es >= 1 && es <= a.n ? es - 1 : -1;
      return true;
    }
    run += __builtin_amdgcn_readlane(incl, 63);
  }
  return false;
}

template <int D, bool BF16, bool CAP, bool BIAS, int WAVES>
__global__ __launch_bounds__(64 * WAVES) __attribute__((amdgpu_waves_per_eu(2, 2)))
void packed_fwd_kernel(const PackedArgs a) {
  typedef typename Elt<BF16>::v8 V8;
  constexpr int BM = 32 * WAVES, UPR = D / 8, KD = D / 16, DB = D / 32;
  constexpr int kElems = kTile * D, kLoads = kTile * UPR / 64 / WAVES;
  __shared__ __align__(16) uint16_t sK[2][kElems];
  __shared__ __align__(16) uint16_t sV[2][kElems];

  const int id = xcd_remap(blockIdx.x, gridDim.x);
  const int h = id / a.blocks;
  RowBlock rb;
  if (!find_block<BM>(a, id - h * a.blocks, rb)) return;
  const int hk = h / a.ratio;
  const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6);
  const int l32 = lane & 31, g = lane >> 5;

  int k0 = 0, lk = 0, pre = 0;
  if (rb.seq >= 0) {
    k0 = uni(min(max(a.cu_k[rb.seq], 0), a.tk));
    lk = uni(min(max(a.cu_k[rb.seq + 1], k0), a.tk)) - k0;
    if (a.prefix) pre = uni(min(max(a.prefix[rb.seq], 0), lk));
  }
  const int off = lk - rb.lq;   // row r is at key position r + off
  auto hi_of = [&](int i) { return a.causal ? min(lk, i + 1) : min(lk, i + a.window); };
  auto lo_of = [&](int i) { return max(0, i - a.window + 1); };

  // key tiles that some row of the block sees: those of the prefix, then a range
  const int i0 = rb.m0 + off, i1 = min(rb.m0 + BM, rb.lq) - 1 + off;
  const int np = (pre + kTile - 1) / kTile;
  const int hi_b = max(0, hi_of(i1)), lo_b = lo_of(i0);
  const int t0 = max(np, lo_b / kTile);
  const int t1 = lo_b < hi_b ? (hi_b + kTile - 1) / kTile : 0;
  const int cnt = np + max(0, t1 - t0);
  auto tile_at = [&](int i) { return i < np ? i : i - np + t0; };

  // this wave's rows, and this lane's
  const int w0 = rb.m0 + wave * 32, w1 = min(w0 + 31, rb.lq - 1);
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
      bload16_lds(r, lds_addr(dst) + (uint32_t)((i * WAVES + wave) * 64 * 16), offs[i]);
  };

  // A tile that the sequence ends inside leaves V rows unwritten, whose P is 0:
  // they hold 0, or an earlier tile's values
  if (lk % kTile != 0) {
    for (int i = tid; i < kElems / 8; i += 64 * WAVES) {
      reinterpret_cast<u32x4*>(sV[0])[i] = u32x4{0u, 0u, 0u, 0u};
      reinterpret_cast<u32x4*>(sV[1])[i] = u32x4{0u, 0u, 0u, 0u};
    }
    __syncthreads();
  }
  if (cnt > 0) {
    issue(kb, a.k_ts, k_off, tile_at(0), sK[0]);
    issue(vb, a.v_ts, v_off, tile_at(0), sV[0]);
  }
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

  auto body = [&](int base, const uint16_t* tK, const uint16_t* tV) __attribute__((always_inline)) {
    const uint8_t* k8 = reinterpret_cast<const uint8_t*>(tK);
    const uint8_t* v8 = reinterpret_cast<const uint8_t*>(tV);
    constexpr int kWin = 2;   // LDS operand reads in flight
    f32x16 s[2] = {f32x16{}, f32x16{}};
    {
      auto rd = [&](int i) {
        return bitcast<V8>(*reinterpret_cast<const u32x4*>(k8 + (i / KD) * 32 * D * 2 + k_rd[i % KD]));
      };
      V8 win[kWin];
#pragma unroll
      for (int i = 0; i < kWin; ++i) win[i] = rd(i);
#pragma unroll
      for (int i = 0; i < 2 * KD; ++i) {
        const V8 x = win[i % kWin];
        if (i + kWin < 2 * KD) win[i % kWin] = rd(i + kWin);
        s[i / KD] = Elt<BF16>::mfma(x, qreg[i % KD], s[i / KD]);
      }
    }
    // u: scores up to the factor c2. Capped: tanh z = 1 − 2 / (e^{2z} + 1), and the
    // 1 cancels in the softmax, so u = −1 / (e^{2z} + 1) with c2 = 2·softcap·log2(e)
    if constexpr (CAP || BIAS) {
      const float x0 = (float)(ia - base - g * 16);
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float u = s[b][i];
          if constexpr (CAP) u = __builtin_amdgcn_rcpf(-1.f - __builtin_amdgcn_exp2f(u * a.u_scale));
          if constexpr (BIAS) u = __builtin_fmaf(bco, __builtin_fabsf(x0 - (float)(b * 32 + i)), u);
          s[b][i] = u;
        }
    }
    const bool full = base + kTile <= pre || (base + kTile <= w_hi0 && base >= w_lo1);
    if (!full) {
      const int h_r = hi - base - g * 16, l_r = lo - base - g * 16, p_r = pl - base - g * 16;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int c = b * 32 + i;
          const bool seen = (c < h_r && c >= l_r) || c < p_r;
          s[b][i] = seen ? s[b][i] : -INFINITY;
        }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[b][i]);
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
      constexpr int N = 4 * DB;
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
          pf[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j / 2][(j % 2) * 8 + e], c2, -mlog2));
        return __builtin_convertvector(pf, V8);
      };
      V8 pcur = pstep(0);
      l_run = psum8<BF16>(pcur, l_run);   // of the rounded P: the weights that V meets
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        V8 pnext;
        if (j < 3) pnext = pstep(j + 1);
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          const int i = j * DB + db;
          const V8 x = win[i % kWin];
          if (i + kWin < N) win[i % kWin] = rd(i + kWin);
          oacc[db] = Elt<BF16>::mfma(x, pcur, oacc[db]);
        }
        if (j < 3) {
          l_run = psum8<BF16>(pnext, l_run);
          pcur = pnext;
        }
      }
    }
  };
  auto iter = [&](auto stc, int i) __attribute__((always_inline)) {
    constexpr int ST = decltype(stc)::value;
    wait_vmcnt<0>();   // tile i has landed
    wg_barrier();      // for every wave; and all have left tile i − 1's stage
    if (i + 1 < cnt) {
      issue(kb, a.k_ts, k_off, tile_at(i + 1), sK[ST ^ 1]);
      issue(vb, a.v_ts, v_off, tile_at(i + 1), sV[ST ^ 1]);
    }
    const int base = tile_at(i) * kTile;
    // a tile that none of the wave's rows sees
    const bool dead = w0 >= rb.lq || (base >= pre && (base >= w_hi1 || base + kTile <= w_lo0));
    if (!dead) body(base, sK[ST], sV[ST]);
  };
  int i = 0;
  for (; i + 1 < cnt; i += 2) {
    iter(std::integral_constant<int, 0>{}, i);
    iter(std::integral_constant<int, 1>{}, i + 1);
  }
  if (i < cnt) iter(std::integral_constant<int, 0>{}, i);

  // O through LDS, each wave in its own slice of the stages, so that a store
  // instruction writes whole rows
  wait_vmcnt<0>();
  wg_barrier();
  uint8_t* stg = (wave < 4 ? reinterpret_cast<uint8_t*>(sK[0]) : reinterpret_cast<uint8_t*>(sV[0])) + (wave & 3) * 32 * D * 2;
  static_assert(4 * 32 * D * 2 <= 2 * kElems * 2, "staging fits");
  const float l = xhalf_sum(l_run);
  const float inv = (l == 0.f || l != l) ? 1.f : 1.f / l;
  constexpr int CH = D / 8, RPI = 64 / CH;
  typedef __attribute__((ext_vector_type(4))) __bf16 bf16x4;
  typedef __attribute__((ext_vector_type(4))) _Float16 f16x4;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {
      f32x4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = oacc[db][q4 * 4 + e] * inv;
      u32x2 packed;
      if constexpr (BF16) packed = bitcast<u32x2>(__builtin_convertvector(x, bf16x4));
      else packed = bitcast<u32x2>(__builtin_convertvector(x, f16x4));
      const int c = db * 4 + q4;
      *reinterpret_cast<u32x2*>(stg + l32 * D * 2 + ((c ^ (l32 & (CH - 1))) * 16) + g * 8) = packed;
    }
  const rsrc_t ro = make_rsrc(a.o + (int64_t)(rb.q0 + w0) * a.o_ts + (int64_t)h * a.o_hs,
                              span(min(32, rb.lq - w0), a.o_ts));
  const int ch = lane % CH, r0 = lane / CH;
#pragma unroll
  for (int k = 0; k < 32 / RPI; ++k) {
    const int r = r0 + k * RPI;
    const u32x4 x = *reinterpret_cast<const u32x4*>(stg + r * D * 2 + ((ch ^ (r & (CH - 1))) * 16));
    __builtin_amdgcn_raw_buffer_store_b128(x, ro, (uint32_t)(r * (int)a.o_ts + ch * 8) * 2u, 0, 0);
  }
}
