// beam_select.h — the selection of a step of beam search: of each search's beams·vocab
// values scores[w] + x[w, v] − log Σ exp x[w, ·] the k largest. Included by beam.hip
// inside namespace mi355fa.
//
// Order is a whole-number result: two beams' candidates that differ in the 8th digit have
// to come out as the formula says, so the sum of exponentials is formed in 64 bits. The
// vector unit multiplies and adds in 64 bits as fast as in 32: an exponential is 17 such
// operations. Bound: the bytes of the logits, each read once.
//
//  * Of a row's logits only the k largest can be selected (their order is that of the
//    scores), so a workgroup that reads some of a row keeps its k largest logits beside
//    the running maximum and sum. All elements of a step are in registers; a bound below
//    the k-th largest comes from the lanes' maxima of 8 elements, by bisecting its bits
//    with ballots; the few elements above it go to a list in LDS, which is ranked by
//    counting at the end.
//  * A second kernel, a workgroup a search, joins the parts' sums and lists.

constexpr int kSelThreads = 256;
constexpr int kSelList = 1024;      // a list in LDS
constexpr int kSelMaxK = 64;
constexpr int kSelMaxBeams = 256;

struct SelectHead {
  double sum;   // Σ exp(x − max)
  float max;    // NaN: the beam has no candidates
  int n;        // candidates listed
};
struct SelectArgs {
  const void* x;
  const float* scores;
  const uint8_t* done;
  float* out_s;
  int* out_t;
  int* out_p;
  SelectHead* heads;   // [rows][parts]
  u32x2* lists;        // [rows][parts][k]: logit's ordered bits, token; descending
  int64_t gs, bs;
  int groups, beams, vocab, k, eos;
  int parts, per;      // parts of a row, tokens of one
};

// Integers in the order of the floats, the two zeros one.
__device__ __forceinline__ uint32_t ordered(float x) {
  const int b = bitcast<int>(x + 0.f);
  return (uint32_t)(b ^ ((b >> 31) & 0x7fffffff)) ^ 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t u) {
  const int b = (int)(u ^ 0x80000000u);
  return bitcast<float>(b ^ ((b >> 31) & 0x7fffffff));
}
constexpr uint32_t kLowest = 0x007fffffu;   // of −infinity

// exp of t in [−700, 0], off by 10^-12 of its value: 2^n·p(t − n·ln 2), p of degree 8 fitted
// for the least relative error on |x| <= ln(2)/2.
__device__ __forceinline__ double exp_neg(double t) {
  constexpr double kRound = 6755399441055744.0;   // 1.5·2^52: the sum's low word is the nearest integer
  const double u = __builtin_fma(t, 1.4426950408889634, kRound);
  const double r = __builtin_fma(u - kRound, -0.6931471805599453, t);
  double p = 2.4727097752539182e-05;
  p = __builtin_fma(p, r, 0.00019915434933597152);
  p = __builtin_fma(p, r, 0.0013889178972678572);
  p = __builtin_fma(p, r, 0.008333267008842798);
  p = __builtin_fma(p, r, 0.04166666421728999);
  p = __builtin_fma(p, r, 0.1666666688556212);
  p = __builtin_fma(p, r, 0.5000000000618945);
  p = __builtin_fma(p, r, 0.999999999980611);
  p = __builtin_fma(p, r, 0.9999999999997615);
  const uint64_t n = (uint64_t)low_u32(bitcast<uint64_t>(u)) << 52;
  return bitcast<double>(bitcast<uint64_t>(p) + n);
}

template <class T> struct Logits;
template <> struct Logits<float> {
  static __device__ __forceinline__ void load8(const void* x, int64_t i, float (&y)[8]) {
    struct __attribute__((packed, aligned(4))) V { u32x4 a, b; };
    const V v = *reinterpret_cast<const V*>(static_cast<const float*>(x) + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      y[e] = bitcast<float>(v.a[e]);
      y[4 + e] = bitcast<float>(v.b[e]);
    }
  }
  static __device__ __forceinline__ float load(const void* x, int64_t i) { return static_cast<const float*>(x)[i]; }
};
template <> struct Logits<__bf16> {
  static __device__ __forceinline__ void load8(const void* x, int64_t i, float (&y)[8]) {
    struct __attribute__((packed, aligned(2))) V { u32x4 a; };
    const V v = *reinterpret_cast<const V*>(static_cast<const uint16_t*>(x) + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      y[2 * e] = bitcast<float>(v.a[e] << 16);
      y[2 * e + 1] = bitcast<float>(v.a[e] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ float load(const void* x, int64_t i) { return bitcast<float>((uint32_t)static_cast<const uint16_t*>(x)[i] << 16); }
};
template <> struct Logits<_Float16> {
  static __device__ __forceinline__ void load8(const void* x, int64_t i, float (&y)[8]) {
    struct __attribute__((packed, aligned(2))) V { f16x8 a; };
    const V v = *reinterpret_cast<const V*>(static_cast<const uint16_t*>(x) + i);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = (float)v.a[e];
  }
  static __device__ __forceinline__ float load(const void* x, int64_t i) { return (float)static_cast<const _Float16*>(x)[i]; }
};

// Ranks a list of n keys (all different) and keeps the k largest, in order. All of the
// workgroup; the list is the same before and after for everybody.
__device__ __forceinline__ void keep_largest(uint64_t* list, int n, int k) {
  constexpr int E = kSelList / kSelThreads;
  uint64_t mine[E];
  int rank[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int i = e * kSelThreads + (int)threadIdx.x;
    mine[e] = i < n ? list[i] : 0;
    rank[e] = 0;
  }
  for (int j = 0; j < n; ++j) {
    const uint64_t y = list[j];
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (e * kSelThreads < n) rank[e] += y > mine[e];
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (e * kSelThreads + (int)threadIdx.x < n && rank[e] < k) list[rank[e]] = mine[e];
  __syncthreads();
}

// Σ of the threads' counts, for all of the workgroup.
__device__ __forceinline__ int count_all(int x, int* words) {
  x = __builtin_amdgcn_readlane(wave_scan(x), 63);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) words[threadIdx.x >> 6] = x;
  __syncthreads();
  int sum = 0;
#pragma unroll
  for (int w = 0; w < kSelThreads / 64; ++w) sum += words[w];
  return sum;
}

// N·8 elements of each thread at a step.
template <class T, int N>
__global__ __launch_bounds__(kSelThreads) void select_scan_kernel(const SelectArgs a) {
  constexpr int WAVES = kSelThreads / 64, STEP = kSelThreads * 8 * N;
  __shared__ uint64_t list[kSelList];   // ordered logit, then the complement of the token: the lowest first among equals
  __shared__ int words[WAVES];
  __shared__ int count;
  __shared__ uint32_t bound;
  __shared__ double sSum[WAVES];
  __shared__ float sMax[WAVES];
  const int row = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
  if (a.done && a.done[row]) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6), k = a.k;
  const int64_t base = (int64_t)(row / a.beams) * a.gs + (int64_t)(row % a.beams) * a.bs;
  const int begin = part * a.per, end = min(a.vocab, begin + a.per);
  if (tid == 0) {
    count = 0;
    bound = 0;
  }
  __syncthreads();
  double sum = 0.;
  float top = -INFINITY;   // the wave's
  bool bad = false;
  int kept = 0;
  for (int at = begin; at < end; at += STEP) {
    float x[N][8], best[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int i = at + (j * kSelThreads + tid) * 8;
      if (i + 8 <= end) Logits<T>::load8(a.x, base + i, x[j]);
      else
#pragma unroll
        for (int e = 0; e < 8; ++e) x[j][e] = i + e < end ? Logits<T>::load(a.x, base + i + e) : -INFINITY;
    }
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      best[j] = -INFINITY;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        best[j] = fmaxf(best[j], x[j][e]);
        bad |= x[j][e] != x[j][e];
      }
      most = max(most, ordered(best[j]));
    }
    const float now = unordered((uint32_t)__builtin_amdgcn_readlane(wave_max_scan((int)(most ^ 0x80000000u)), 63) ^ 0x80000000u);
    if (now > top) {
      if (top > -INFINITY) sum *= exp((double)top - (double)now);
      top = now;
    }
    if (top > -INFINITY) {
      const double m = top;
#pragma unroll
      for (int j = 0; j < N; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += exp_neg(fmax((double)x[j][e] - m, -700.));
    }
    // At least k of the wave's elements reach t, since k of the maxima of 8 do: the largest
    // such t, to 16 bits.
    uint32_t t = 0;
#pragma unroll 1
    for (int bit = 31; bit >= 16; --bit) {
      const uint32_t trial = t | 1u << bit;
      int n = 0;
#pragma unroll
      for (int j = 0; j < N; ++j) n += __builtin_popcountll(__builtin_amdgcn_ballot_w64(ordered(best[j]) >= trial));
      if (n >= k) t = trial;
    }
    if (lane == 0) atomicMax(&bound, t);
    t = max(t, bound);   // (others' bounds hold as well, seen or not)
    t = max(t, kLowest + 1);   // never −infinity
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (!__builtin_amdgcn_ballot_w64(ordered(best[j]) >= t)) continue;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (ordered(x[j][e]) >= t && x[j][e] == x[j][e]) {
          const int n = atomicAdd(&count, 1);
          if (n < kSelList) list[n] = (uint64_t)ordered(x[j][e]) << 32 | (uint32_t)~(at + (j * kSelThreads + tid) * 8 + e);
        }
      }
    }
    __syncthreads();
    int n = count;
    if (n > kSelList / 2) {
      __syncthreads();   // all have seen it
      if (n > kSelList) {
        // Too many of this step, most of them equal: exactly its k largest, by their
        // value's bits and, among those of the k-th value, by their places'
        keep_largest(list, kept, k);
        kept = min(kept, k);
        uint32_t v = 0;
        for (int bit = 31; bit >= 0; --bit) {
          const uint32_t trial = v | 1u << bit;
          int c = 0;
#pragma unroll
          for (int j = 0; j < N; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) c += ordered(x[j][e]) >= trial && x[j][e] == x[j][e];
          if (count_all(c, words) >= k) v = trial;
        }
        int above = 0;
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
          for (int e = 0; e < 8; ++e) above += ordered(x[j][e]) > v && x[j][e] == x[j][e];
        const int need = k - count_all(above, words);
        int place = 0;   // `need` of the elements of value v lie at or before it
        for (int bit = 31 - __builtin_clz(STEP); bit >= 0; --bit) {
          const int trial = place | 1 << bit;
          int c = 0;
#pragma unroll
          for (int j = 0; j < N; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) c += ordered(x[j][e]) == v && (j * kSelThreads + tid) * 8 + e < trial;
          if (count_all(c, words) < need) place = trial;
        }
        if (tid == 0) count = kept;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int i = (j * kSelThreads + tid) * 8 + e;
            const uint32_t o = ordered(x[j][e]);
            if (x[j][e] == x[j][e] && (o > v || (o == v && i <= place))) list[atomicAdd(&count, 1)] = (uint64_t)o << 32 | (uint32_t)~(at + i);
          }
        __syncthreads();
        n = count;
      }
      keep_largest(list, n, k);
      n = min(n, k);
      if (tid == 0) {
        count = n;
        if (n == k) bound = max(bound, (uint32_t)(list[k - 1] >> 32));
      }
      __syncthreads();
    }
    kept = n;
    __syncthreads();   // nobody adds before all have seen the count
  }
  const int n = kept;
  keep_largest(list, n, k);
  const int64_t slot = blockIdx.x;
  for (int i = tid; i < min(n, k); i += kSelThreads)
    a.lists[slot * k + i] = u32x2{(uint32_t)(list[i] >> 32), ~(uint32_t)list[i]};
#pragma unroll
  for (int x = 1; x < 64; x *= 2) sum += __shfl_xor(sum, x);
  const bool any_bad = __builtin_amdgcn_ballot_w64(bad) != 0;
  if (lane == 0) {
    sSum[wave] = sum;
    sMax[wave] = any_bad ? NAN : top;
  }
  __syncthreads();
  if (tid == 0) {
    float m = -INFINITY;
    bool nan = false;
    for (int w = 0; w < WAVES; ++w) {
      m = fmaxf(m, sMax[w]);
      nan |= !(sMax[w] < INFINITY);
    }
    double s = 0.;
    for (int w = 0; w < WAVES; ++w)
      if (sMax[w] > -INFINITY) s += sSum[w] * exp((double)sMax[w] - (double)m);
    a.heads[slot] = SelectHead{s, nan ? NAN : m, min(n, k)};
  }
}

// A search: the rows' parts together.
__global__ __launch_bounds__(kSelThreads) void select_join_kernel(const SelectArgs a) {
  __shared__ double base[kSelMaxBeams];    // scores[w] and the logarithm of the sum; NaN: no candidates
  __shared__ double score[kSelList];
  __shared__ uint32_t index[kSelList];
  __shared__ float run[kSelMaxBeams];
  __shared__ int count, words[kSelThreads / 64];
  __shared__ uint32_t bound;
  const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6), k = a.k, g = blockIdx.x;
  const int64_t row0 = (int64_t)g * a.beams;
  if (tid == 0) {
    count = 0;
    bound = 0;
  }
  for (int w = wave; w < a.beams; w += kSelThreads / 64) {
    const int64_t row = row0 + w;
    const float s = a.scores[row];
    const bool done = a.done && a.done[row];
    float m = -INFINITY;
    bool nan = false;
    double sum = 0.;
    if (!done) {
      for (int p = lane; p < a.parts; p += 64) {
        const float x = a.heads[row * a.parts + p].max;
        m = fmaxf(m, x);
        nan |= !(x < INFINITY);
      }
#pragma unroll
      for (int x = 1; x < 64; x *= 2) m = fmaxf(m, __shfl_xor(m, x));
      nan = __builtin_amdgcn_ballot_w64(nan) != 0 || m == -INFINITY;
      for (int p = lane; p < a.parts; p += 64) {
        const SelectHead h = a.heads[row * a.parts + p];
        if (h.max > -INFINITY) sum += h.sum * exp((double)h.max - (double)m);
      }
#pragma unroll
      for (int x = 1; x < 64; x *= 2) sum += __shfl_xor(sum, x);
    }
    if (lane == 0) {
      const bool real = s > -INFINITY && s < INFINITY && (done || !nan);
      run[w] = real ? s : NAN;
      base[w] = done ? INFINITY : (double)m + log(sum);   // (a finished beam: infinity)
    }
  }
  __syncthreads();
  // Candidate j of list i (its rows' parts in order), and its place w·vocab + v; false: there is none
  const int lists = a.beams * a.parts;
  auto candidate = [&](int i, int j, double& s, uint32_t& at) __attribute__((always_inline)) {
    const int w = i / a.parts, p = i % a.parts;
    if (run[w] != run[w]) return false;
    if (base[w] == INFINITY) {
      s = run[w];
      at = (uint32_t)w * a.vocab + a.eos;
      return p == 0 && j == 0;
    }
    const int64_t slot = (row0 + w) * a.parts + p;
    if (j >= a.heads[slot].n) return false;
    const u32x2 c = a.lists[slot * k + j];
    s = (double)run[w] + ((double)unordered(c[0]) - base[w]);
    at = (uint32_t)w * a.vocab + c[1];
    return true;
  };
  // Ranks the list and keeps the k best: the highest score, the lowest place among equals
  auto keep = [&](int n) __attribute__((always_inline)) {
    constexpr int E = kSelList / kSelThreads;
    double mine[E];
    uint32_t at[E];
    int rank[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int i = e * kSelThreads + tid;
      mine[e] = i < n ? score[i] : -INFINITY;
      at[e] = i < n ? index[i] : 0;
      rank[e] = 0;
    }
    for (int j = 0; j < n; ++j) {
      const double y = score[j];
      const uint32_t z = index[j];
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (e * kSelThreads < n) rank[e] += y > mine[e] || (y == mine[e] && z < at[e]);
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (e * kSelThreads + tid < n && rank[e] < k) {
        score[rank[e]] = mine[e];
        index[rank[e]] = at[e];
      }
    if (tid == 0) count = min(n, k);
    __syncthreads();
  };
  // Lists descend, so the candidates of rank j come after those of rank j − 1, and none
  // are left once no list has one that reaches the bound.
  for (int j = 0; j < k; ++j) {
    int some = 0;
    for (int i0 = 0; i0 < lists; i0 += kSelThreads) {
      double s = 0.;
      uint32_t at = 0;
      const int i = i0 + tid;
      const bool real = i < lists && candidate(i, j, s, at);
      if (real && ordered((float)s) >= bound) {
        const int n = atomicAdd(&count, 1);
        score[n] = s;
        index[n] = at;
        ++some;
      }
      __syncthreads();
      const int n = count;
      __syncthreads();   // all have seen it
      if (n > kSelList - kSelThreads || (j == 0 && i0 + kSelThreads >= lists && n > k)) {
        keep(n);
        if (tid == 0 && n >= k) bound = ordered((float)score[k - 1]);
        __syncthreads();
      }
    }
    if (count_all(some, words) == 0) break;
  }
  __syncthreads();
  const int n = count;
  __syncthreads();
  keep(n);
  for (int i = tid; i < k; i += kSelThreads) {
    const bool real = i < n;
    const int64_t o = (int64_t)g * k + i;
    a.out_s[o] = real ? (float)score[i] : -INFINITY;
    a.out_t[o] = real ? (int)(index[i] % (uint32_t)a.vocab) : -1;
    a.out_p[o] = real ? (int)(row0 + index[i] / (uint32_t)a.vocab) : -1;
  }
}
