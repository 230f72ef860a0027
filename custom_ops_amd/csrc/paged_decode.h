// paged_decode.h — attention of one new token per request over a paged key-value
// cache. Included by serve.hip inside namespace mi355fa.
//
// The h / h_k heads that share a KV head are the columns of one 16-wide matrix
// product, so K and V are read once for all of them. Bound: the bytes of the seen
// keys; the products and exponentials of 16 heads take a few percent of the time
// that their keys take to arrive.
//
//  * Each wave runs its own stream of 32-key tiles: Sᵀ = K·Qᵀ with 16x16x32 MFMAs,
//    K rows straight from the cache into the operand registers; a lane then holds
//    4 + 4 keys of one head, which rounded are the B operand of Oᵀ += Vᵀ·Pᵀ. V rows
//    pass through the wave's own LDS slice to be read transposed. No barrier but
//    the join of the waves at the end.
//  * K and V of the next tile are in flight, in registers, while a tile computes;
//    the page numbers of the one behind it too.
//  * Sequences are split by their own lengths, which only the device knows: every
//    workgroup sums the tiles of all requests, takes the part size that makes about
//    `target` parts of them, and finds its own part by a scan. So a long sequence
//    in a ragged batch is shared by many workgroups and a short one is not split.
//    Parts (O, max, sum, fp32) of a shared sequence are joined by a second kernel.

constexpr int kDecWaves = 4;
constexpr int kDecHeads = 16;   // heads of a group per workgroup

struct DecodeArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* o;
  const int* table;
  const int* lens;
  const float* slopes;
  int* rec;        // [b][hk·groups][2]: first part, parts
  float* part_ml;  // [parts][16][2]: max in log2 units, sum
  float* part_o;   // [parts][16][D]
  int64_t q_bs, q_hs, o_bs, o_hs, kp, kh, kr, vp, vh, vr, ts;
  int b, h, hk, ratio, groups;   // groups: 16-head groups per KV head
  int pages, shift, cols, window;
  int split;       // 0: a workgroup per (request, head group)
  int target;      // parts to make, about
  int least;       // tiles of a part at least
  float u_scale, c2, bias;       // as in PackedArgs
};

template <bool BF16>
__device__ __forceinline__ f32x4 mfma16(typename Elt<BF16>::v8 a, typename Elt<BF16>::v8 b, f32x4 c) {
  if constexpr (BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ KeySpan keys_of(const DecodeArgs& a, int len) {
  return key_span(len, (int64_t)a.cols << a.shift, a.window);
}

// Part w: request, head group, place among the request's parts. All waves of the
// workgroup find the same, each for itself: two passes over the lengths, 64 at a time.
struct Part {
  int b, hg, part, parts, slot;   // slot: of part 0
  int len;                        // the request's keys
};
__device__ __forceinline__ bool find_part(const DecodeArgs& a, int w, Part& p) {
  const int hgs = a.hk * a.groups, lane = threadIdx.x & 63;
  if (!a.split) {
    p = Part{w / hgs, w % hgs, 0, 1, 0, 0};
    p.len = a.lens[p.b];
    return true;
  }
  int sum = 0;
  for (int i = lane; i < a.b; i += 64) sum += weighed(keys_of(a, a.lens[i]).tiles);
  sum = __builtin_amdgcn_readlane(wave_scan(sum), 63);
  const int per = part_size(sum, hgs, a.target, a.least);
  int run = 0;
  for (int base = 0; base < a.b; base += 64) {
    const int i = base + lane;
    const int len = i < a.b ? a.lens[i] : 0;
    const int n = i < a.b ? part_count(keys_of(a, len).tiles, per) : 0;
    const int incl = wave_scan(n * hgs);
    const uint64_t hit = __builtin_amdgcn_ballot_w64(run + incl > w);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      p.b = base + l;
      p.len = __builtin_amdgcn_readlane(len, l);
      p.parts = __builtin_amdgcn_readlane(n, l);
      const int start = run + (int)__builtin_amdgcn_readlane(incl, l) - p.parts * hgs;
      p.hg = (w - start) / p.parts;
      p.part = (w - start) % p.parts;
      p.slot = w - p.part;
      return true;
    }
    run += __builtin_amdgcn_readlane(incl, 63);
  }
  return false;
}

template <int D, bool BF16, bool CAP, bool BIAS, int WAVES>
__global__ __launch_bounds__(64 * WAVES) __attribute__((amdgpu_waves_per_eu(2)))
void paged_decode_kernel(const DecodeArgs a) {
  typedef typename Elt<BF16>::v8 V8;
  constexpr int KD = D / 32, DB = D / 16;
  constexpr int kRow = D * 2 + 32;   // LDS bytes per V row: transposed reads of 16 rows touch all banks alike
  __shared__ __align__(16) uint8_t sV[WAVES][kDecTile * kRow];
  __shared__ float sM[WAVES][kDecHeads], sL[WAVES][kDecHeads];

  Part pt;
  if (!find_part(a, blockIdx.x, pt)) return;
  const int b = pt.b, hg = pt.hg;
  const int hk = hg / a.groups, h0 = hk * a.ratio + (hg % a.groups) * kDecHeads;
  const int heads = min(kDecHeads, (hk + 1) * a.ratio - h0);
  const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6);
  const int l16 = lane & 15, g = lane >> 4;

  const int page_size = 1 << a.shift;
  const KeySpan ks = keys_of(a, pt.len);
  const int len = uni(ks.len), first = uni(ks.first), tile0 = uni(ks.tile0), tiles = uni(ks.tiles);
  // tiles of this part, this wave: t_lo + wave, + WAVES, ...
  const int t_lo = tile0 + part_start(tiles, pt.parts, pt.part), t_hi = tile0 + part_start(tiles, pt.parts, pt.part + 1);

  // Q of the wave's heads: B operand, column l16, d = 8·(4·kd + g)
  V8 qreg[KD];
#pragma unroll
  for (int kd = 0; kd < KD; ++kd) {
    u32x4 x = {0u, 0u, 0u, 0u};
    if (l16 < heads)
      x = *reinterpret_cast<const u32x4*>(a.q + (int64_t)b * a.q_bs + (int64_t)(h0 + l16) * a.q_hs + (kd * 4 + g) * 8);
    qreg[kd] = bitcast<V8>(x);
  }
  const float bco = BIAS ? a.slopes[min(h0 + l16, a.h - 1)] * a.bias : 0.f;
  const float c2 = a.c2, slack = kSlackLog2 / a.c2;
  f32x4 oacc[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) oacc[db] = f32x4{};
  float m_run = -INFINITY, mlog2 = 0.f, l_run = 0.f;

  const int* table = a.table + (int64_t)b * a.ts;
  const uint16_t* kbase = a.k + (int64_t)hk * a.kh + g * 8;
  const uint16_t* vbase = a.v + (int64_t)hk * a.vh + g * 8;
  // Page numbers of the lane's keys l16 and 16 + l16 of a tile (-1: not seen). No load
  // of the loop is conditional, or the compiler would wait for all loads in flight where
  // the paths meet: what is behind the part's end reads what is there anyway.
  const int last = max(len - 1, 0);
  auto entries = [&](int t, int (&e)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int key = t * kDecTile + r * 16 + l16;
      const int x = table[min(key, last) >> a.shift];
      e[r] = (t < t_hi && key >= first && key < len) ? x : -1;
    }
  };
  struct Tile { u32x4 k[2][KD], v[2][KD]; bool ok[2]; };
  auto fetch = [&](int t, const int (&e)[2], Tile& x) __attribute__((always_inline)) {
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
  auto compute = [&](int t, const Tile& x) __attribute__((always_inline)) {
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
    // this lane: head l16, keys 16·r + 4·g + i
    const uint64_t ok0 = __builtin_amdgcn_ballot_w64(x.ok[0]), ok1 = __builtin_amdgcn_ballot_w64(x.ok[1]);
    const float back = (float)(len - 1 - t * kDecTile - 4 * g);
    float mx = -INFINITY;
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float u = s[r][i];
        if constexpr (CAP) u = __builtin_amdgcn_rcpf(-1.f - __builtin_amdgcn_exp2f(u * a.u_scale));
        if constexpr (BIAS) u = __builtin_fmaf(bco, back - (float)(r * 16 + i), u);
        if (!whole) u = (((r ? ok1 : ok0) >> (4 * g + i)) & 1) ? u : -INFINITY;
        s[r][i] = u;
        mx = fmaxf(mx, u);
      }
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
    for (int e = 0; e < 8; ++e) pf[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e / 4][e % 4], c2, -mlog2));
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

  if (t_lo + wave < t_hi) {
    int t = t_lo + wave;
    int e0[2], e1[2];
    Tile x0, x1;
    entries(t, e0);
    entries(t + WAVES, e1);
    fetch(t, e0, x0);
    for (; t + WAVES < t_hi; t += 2 * WAVES) {
      entries(t + 2 * WAVES, e0);
      fetch(t + WAVES, e1, x1);
      compute(t, x0);
      entries(t + 3 * WAVES, e1);
      fetch(t + 2 * WAVES, e0, x0);
      compute(t + WAVES, x1);
    }
    if (t < t_hi) compute(t, x0);
  }

  // join the waves: O in its own slice as fp32, [D][16 heads] (the slices are free)
  l_run += __shfl_xor(l_run, 16);
  l_run += __shfl_xor(l_run, 32);
  if (lane < kDecHeads) {
    sM[wave][l16] = m_run == -INFINITY ? -INFINITY : m_run * c2;
    sL[wave][l16] = l_run;
  }
  float* so = reinterpret_cast<float*>(sv);   // [l16][D + 2]
  static_assert(kDecHeads * (D + 2) * 4 <= kDecTile * kRow, "O fits in the V slice");
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int i = 0; i < 4; ++i) so[l16 * (D + 2) + db * 16 + 4 * g + i] = oacc[db][i];
  __syncthreads();
  for (int x = tid; x < heads * D; x += 64 * WAVES) {
    const int n = x / D, d = x % D;
    float m = sM[0][n];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) m = fmaxf(m, sM[w][n]);
    float acc = 0.f, l = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float f = sM[w][n] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sM[w][n] - m);
      // a wave that saw nothing adds nothing; NaN sums stay
      l += sL[w][n] == 0.f ? 0.f : sL[w][n] * (sM[w][n] == -INFINITY ? 1.f : f);
      const float y = reinterpret_cast<const float*>(sV[w])[n * (D + 2) + d];
      acc += sL[w][n] == 0.f ? 0.f : y * (sM[w][n] == -INFINITY ? 1.f : f);
    }
    if (pt.parts == 1) {
      const float r = l == 0.f ? 0.f : acc / l;
      uint16_t out;
      if constexpr (BF16) out = bitcast<uint16_t>((__bf16)r);
      else out = bitcast<uint16_t>((_Float16)r);
      a.o[(int64_t)b * a.o_bs + (int64_t)(h0 + n) * a.o_hs + d] = out;
    } else {
      const int64_t at = (int64_t)(pt.slot + pt.part) * kDecHeads + n;
      a.part_o[at * D + d] = acc;
      if (d == 0) {
        a.part_ml[at * 2] = m;
        a.part_ml[at * 2 + 1] = l;
      }
    }
  }
  if (a.split && pt.part == 0 && tid == 0) {
    int* rec = a.rec + ((int64_t)b * a.hk * a.groups + hg) * 2;
    rec[0] = pt.slot;
    rec[1] = pt.parts;
  }
}

// One workgroup per (request, head): the parts, weighted by 2^(m_s − m). Its 256
// threads are 1024 / D rows of D / 4 threads; a row takes every so many parts, 8 of
// them in flight, with a running max, and the rows' sums are joined in LDS.
template <int D, bool BF16>
__global__ __launch_bounds__(256) void paged_join_kernel(const DecodeArgs a) {
  constexpr int TPR = D / 4, ROWS = 256 / TPR, J = 8;
  __shared__ float sAcc[ROWS][D], sMax[ROWS], sSum[ROWS];
  const int b = blockIdx.x / a.h, h = blockIdx.x % a.h, tid = threadIdx.x;
  const int hk = h / a.ratio, n = (h - hk * a.ratio) % kDecHeads, hg = hk * a.groups + (h - hk * a.ratio) / kDecHeads;
  const int* rec = a.rec + ((int64_t)b * a.hk * a.groups + hg) * 2;
  const int slot = uni(rec[0]), parts = uni(rec[1]);
  if (parts <= 1) return;   // written by its one part
  const float* ml = a.part_ml + ((int64_t)slot * kDecHeads + n) * 2;
  const float* po = a.part_o + ((int64_t)slot * kDecHeads + n) * D;
  const int row = tid / TPR, c = tid % TPR;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  for (int s0 = row; s0 < parts; s0 += ROWS * J) {
    float ms[J], ls[J];
    f32x4 x[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int s = min(s0 + j * ROWS, parts - 1);
      ms[j] = ml[(int64_t)s * kDecHeads * 2];
      ls[j] = ml[(int64_t)s * kDecHeads * 2 + 1];
      x[j] = *reinterpret_cast<const f32x4*>(po + (int64_t)s * kDecHeads * D + c * 4);
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
