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
//  * The length is split over workgroups; their parts (O, max, sum, fp32) are joined
//    by a second kernel.

constexpr int kDecTile = 32;    // keys per wave tile
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
  float* part_o;   // [splits][b·h][D]
  float* part_ml;  // [splits][b·h][2]: max in log2 units, sum
  int64_t q_bs, q_hs, o_bs, o_hs, kp, kh, kr, vp, vh, vr, ts;
  int b, h, hk, ratio, groups;   // groups: 16-head groups per KV head
  int pages, shift, cols, window, splits;
  float u_scale, c2, bias;       // as in PackedArgs
};

template <bool BF16>
__device__ __forceinline__ f32x4 mfma16(typename Elt<BF16>::v8 a, typename Elt<BF16>::v8 b, f32x4 c) {
  if constexpr (BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

template <int D, bool BF16, bool CAP, bool BIAS>
__global__ __launch_bounds__(64 * kDecWaves) __attribute__((amdgpu_waves_per_eu(2, 2)))
void paged_decode_kernel(const DecodeArgs a) {
  typedef typename Elt<BF16>::v8 V8;
  constexpr int KD = D / 32, DB = D / 16;
  constexpr int kRow = D * 2 + 32;   // LDS bytes per V row: transposed reads of 16 rows touch all banks alike
  __shared__ __align__(16) uint8_t sV[kDecWaves][kDecTile * kRow];
  __shared__ float sM[kDecWaves][kDecHeads], sL[kDecWaves][kDecHeads];

  const int split = blockIdx.x % a.splits;
  const int rest = blockIdx.x / a.splits;
  const int hg = rest % (a.hk * a.groups), b = rest / (a.hk * a.groups);
  const int hk = hg / a.groups, h0 = hk * a.ratio + (hg % a.groups) * kDecHeads;
  const int heads = min(kDecHeads, (hk + 1) * a.ratio - h0);
  const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6);
  const int l16 = lane & 15, g = lane >> 4;

  const int page_size = 1 << a.shift;
  const int len = uni(max(0, (int)min((int64_t)a.lens[b], (int64_t)a.cols << a.shift)));
  const int first = max(0, len - a.window);
  // tiles of this split, this wave: t_lo + wave, + kDecWaves, ...
  const int tile0 = first / kDecTile, tiles = (len + kDecTile - 1) / kDecTile - tile0;
  const int per = (tiles + a.splits - 1) / a.splits;
  const int t_lo = tile0 + min(tiles, split * per), t_hi = tile0 + min(tiles, (split + 1) * per);

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
  // page numbers of the lane's keys l16 and 16 + l16 of a tile (-1: not seen)
  auto entries = [&](int t, int (&e)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int key = t * kDecTile + r * 16 + l16;
      e[r] = (t < t_hi && key >= first && key < len) ? table[key >> a.shift] : -1;
    }
  };
  struct Tile { u32x4 k[2][KD], v[2][KD]; bool ok[2]; };
  auto fetch = [&](int t, const int (&e)[2], Tile& x) __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      x.ok[r] = e[r] >= 0 && e[r] < a.pages;
      const int64_t page = x.ok[r] ? e[r] : 0;
      const int64_t in = (t * kDecTile + r * 16 + l16) & (page_size - 1);
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

  {
    int t = t_lo + wave;
    int e0[2], e1[2];
    Tile x0, x1;
    entries(t, e0);
    entries(t + kDecWaves, e1);
    if (t < t_hi) fetch(t, e0, x0);
    for (; t < t_hi; t += 2 * kDecWaves) {
      entries(t + 2 * kDecWaves, e0);
      if (t + kDecWaves < t_hi) fetch(t + kDecWaves, e1, x1);
      compute(t, x0);
      if (t + kDecWaves < t_hi) {
        entries(t + 3 * kDecWaves, e1);
        if (t + 2 * kDecWaves < t_hi) fetch(t + 2 * kDecWaves, e0, x0);
        compute(t + kDecWaves, x1);
      }
    }
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
  for (int x = tid; x < heads * D; x += 64 * kDecWaves) {
    const int n = x / D, d = x % D;
    float m = sM[0][n];
#pragma unroll
    for (int w = 1; w < kDecWaves; ++w) m = fmaxf(m, sM[w][n]);
    float acc = 0.f, l = 0.f;
#pragma unroll
    for (int w = 0; w < kDecWaves; ++w) {
      const float f = sM[w][n] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sM[w][n] - m);
      // a wave that saw nothing adds nothing; NaN sums stay
      l += sL[w][n] == 0.f ? 0.f : sL[w][n] * (sM[w][n] == -INFINITY ? 1.f : f);
      const float y = reinterpret_cast<const float*>(sV[w])[n * (D + 2) + d];
      acc += sL[w][n] == 0.f ? 0.f : y * (sM[w][n] == -INFINITY ? 1.f : f);
    }
    if (a.splits == 1) {
      const float r = l == 0.f ? 0.f : acc / l;
      uint16_t out;
      if constexpr (BF16) out = bitcast<uint16_t>((__bf16)r);
      else out = bitcast<uint16_t>((_Float16)r);
      a.o[(int64_t)b * a.o_bs + (int64_t)(h0 + n) * a.o_hs + d] = out;
    } else {
      const int64_t bh = (int64_t)split * a.b * a.h + (int64_t)b * a.h + h0 + n;
      a.part_o[bh * D + d] = acc;
      if (d == 0) {
        a.part_ml[bh * 2] = m;
        a.part_ml[bh * 2 + 1] = l;
      }
    }
  }
}

// One workgroup per (request, head): the splits' parts, weighted by 2^(m_s − m).
template <int D, bool BF16>
__global__ __launch_bounds__(D) void paged_join_kernel(const DecodeArgs a) {
  const int bh = blockIdx.x, d = threadIdx.x;
  const int64_t n = (int64_t)a.b * a.h;
  float m = -INFINITY;
  for (int s = 0; s < a.splits; ++s) m = fmaxf(m, a.part_ml[(s * n + bh) * 2]);
  float acc = 0.f, l = 0.f;
  for (int s = 0; s < a.splits; ++s) {
    const float ms = a.part_ml[(s * n + bh) * 2], ls = a.part_ml[(s * n + bh) * 2 + 1];
    const float f = ms == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ms - m);
    l += ls == 0.f ? 0.f : ls * f;
    acc += ls == 0.f ? 0.f : a.part_o[(s * n + bh) * D + d] * f;
  }
  const float r = l == 0.f ? 0.f : acc / l;
  uint16_t out;
  if constexpr (BF16) out = bitcast<uint16_t>((__bf16)r);
  else out = bitcast<uint16_t>((_Float16)r);
  a.o[(int64_t)(bh / a.h) * a.o_bs + (int64_t)(bh % a.h) * a.o_hs + d] = out;
}
