// beam_select.h — the selection of a step of beam search: of each search's beams·vocab
// values scores[w] + x[w, v] − log Σ exp x[w, ·] the k largest. Included by beam.hip
// inside namespace mi355fa.
//
// Order is a whole-number result: two beams' candidates that differ in the 8th digit have
// to come out as the formula says, so the sum of exponentials is formed in 64 bits. The
// vector unit multiplies and adds in 64 bits as fast as in 32: an exponential is 15 such
// operations. Bound: the bytes of the logits, each read once; the exponentials take about
// as long.
//
//  * Of a row's logits only the k largest can be selected (their order is that of the
//    scores), so each wave that reads some of a row keeps the k largest of them beside the
//    sum, in a list of its own in LDS. A bound below the k-th largest of the first step comes
//    from the lanes' maxima, by bisecting bits with ballots; waves tell each other theirs, and
//    only elements that reach it are listed.
//  * The next step's logits are in flight while a step computes.
//  * bf16 logits of long parts are counted by value and their exponentials taken once a value.
//    (Eight logits of which one is 0, below 2^-10, 64 or more, or −infinity go one after the other.)
//  * A second kernel, a workgroup a search, joins the parts' sums and lists: all
//    candidates in registers, a bound by bisection in each wave, and the few that reach it
//    ranked by counting.
//  * Equal scores: a row's candidates stay in the order of their logits, so that what a part keeps
//    and what the join takes are the same order, which does not depend on the split.
// Measured in a graph: one search of 4 beams, 32000 tokens, bf16: 9.4 us (scan 5.5, join 4.0);
// 128000 tokens 13.0, of which the join has 1008 candidates; 4 of 50 beams, k 50, 10007 tokens,
// fp32: 26; 64 of 8, k 16, 128000 tokens, bf16: 60, of which the scan 57 for 131 MB (2.3 TB/s):
// counting and listing, not the bytes. Of that size, normal logits 63 us in bf16, 65 in fp16, 69 in
// fp32; a tenth of them −infinity 116, 66, 70; all equal 331, 216, 151 (one bin; all listed).

constexpr int kSelWave = 256;       // of a wave's
constexpr int kSelMaxK = 64;
constexpr int kSelMaxBeams = 256;
constexpr int kSelJoin = 1024;      // threads of the join, and candidates of a thread, at most
constexpr int kSelEach = 16;
static_assert(kSelJoin * kSelEach == kSelCandidates, "what the join holds");

// Σ over the wave, in all lanes.
template <int CTRL, int ROWS> __device__ __forceinline__ double dpp_add(double x) {
  const uint64_t b = bitcast<uint64_t>(x);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0u, low_u32(b), CTRL, ROWS, 0xf, false), hi = __builtin_amdgcn_update_dpp(0u, high_u32(b), CTRL, ROWS, 0xf, false);
  return x + bitcast<double>(compose_u64(lo, hi));   // (a lane without a source adds 0)
}
__device__ __forceinline__ double wave_sum(double x) {
  x = dpp_add<0x111, 0xf>(x);
  x = dpp_add<0x112, 0xf>(x);
  x = dpp_add<0x114, 0xf>(x);
  x = dpp_add<0x118, 0xf>(x);
  x = dpp_add<0x142, 0xa>(x);
  x = dpp_add<0x143, 0xc>(x);
  const uint64_t b = bitcast<uint64_t>(x);
  return bitcast<double>(compose_u64(__builtin_amdgcn_readlane(low_u32(b), 63), __builtin_amdgcn_readlane(high_u32(b), 63)));
}

template <class T> constexpr int kSelWide = sizeof(T) == 2 ? 4 : 2;   // 16-byte loads of a thread at a step of a long part: 4

// bf16 logits have few values, so a long part counts them: a bin for each of the 4096 values
// of 2^-10 up to 64 and their negatives, of which the exponentials are taken at the end;
// others at once. An exponential takes 14 operations in 64 bits, a count 5 and an addition in LDS.
template <class T, int N> constexpr bool kSelBins = std::is_same_v<T, __bf16> && N > 1;
constexpr uint32_t kBins = 4096, kBinFirst = 117u << 7;   // bits of 2^-10

struct SelectHead {
  double sum;   // 2^600·Σ exp(x − ref)
  float ref;    // −infinity: nothing there; NaN: the beam has no candidates
  int unused;
};
struct SelectArgs {
  const void* x;
  const float* scores;
  const uint8_t* done;
  float* out_s;
  int* out_t;
  int* out_p;
  SelectHead* heads;   // [rows][parts]
  u32x2* lists;        // [rows][parts][k]: logit's ordered bits (0: none), token
  int64_t gs, bs;
  int groups, beams, vocab, k, eos;
  int parts, per;      // parts of a row, tokens of one
  uint32_t row_magic;  // ceil(2^32 / (parts·k)), 0 where that is 1
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

// 2^600·exp(x − ref), x − ref in [−415, 110]: 2^n·p(y − n) with n the whole part of
// y = (x − ref)·log2(e) + 600 and p of degree 8, exactly 1 at 0, fitted for the least relative
// error on [0, 1], which is 8·10^-13.
constexpr double kExpShift = 600.;   // no term is less than 1
constexpr float kExpLow = 415.f, kExpHigh = 100.f;
__device__ __forceinline__ double exp_term(float x, double ref) {
  const double y = __builtin_fma((double)x - ref, 1.4426950408889634, kExpShift);
  const double f = __builtin_amdgcn_fract(y);
  double p = 1.8586588623567065e-06;
  p = __builtin_fma(p, f, 1.42173236346545e-05);
  p = __builtin_fma(p, f, 0.00015507427260292705);
  p = __builtin_fma(p, f, 0.0013327602242329773);
  p = __builtin_fma(p, f, 0.00961832601697772);
  p = __builtin_fma(p, f, 0.05550407297522302);
  p = __builtin_fma(p, f, 0.24022651005780424);
  p = __builtin_fma(p, f, 0.6931471804690105);
  p = __builtin_fma(p, f, 1.);
  const uint64_t bits = bitcast<uint64_t>(p);
  return bitcast<double>(compose_u64(low_u32(bits), high_u32(bits) + ((uint32_t)y << 20)));
}

// The larger one; NaN where one is NaN.
__device__ __forceinline__ float maximum(float x, float y) { return __builtin_elementwise_maximum(x, y); }

// 8 logits of a row, as loaded; behind its end −infinity.
template <class T> struct Logits;
template <> struct Logits<float> {
  struct __attribute__((packed, aligned(4))) Raw { u32x4 a, b; };
  static __device__ __forceinline__ Raw tail(const void* x, int64_t i, int n) {
    Raw r;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t* p = static_cast<const uint32_t*>(x) + i + e;
      r.a[e] = e < n ? p[0] : 0xff800000u;
      r.b[e] = e + 4 < n ? p[4] : 0xff800000u;
    }
    return r;
  }
  static __device__ __forceinline__ float value(const Raw& r, int e) { return bitcast<float>(e < 4 ? r.a[e % 4] : r.b[e % 4]); }
  static __device__ __forceinline__ float one(const void* x, int64_t i) { return static_cast<const float*>(x)[i]; }
};
struct __attribute__((packed, aligned(2))) HalfRaw { u32x4 a; };
__device__ __forceinline__ HalfRaw half_tail(const void* x, int64_t i, int n, uint32_t none) {
  HalfRaw r;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint16_t* p = static_cast<const uint16_t*>(x) + i + 2 * e;
    const uint32_t lo = 2 * e < n ? p[0] : none, hi = 2 * e + 1 < n ? p[1] : none;
    r.a[e] = lo | hi << 16;
  }
  return r;
}
template <> struct Logits<__bf16> {
  typedef HalfRaw Raw;
  static __device__ __forceinline__ Raw tail(const void* x, int64_t i, int n) { return half_tail(x, i, n, 0xff80u); }
  static __device__ __forceinline__ float one(const void* x, int64_t i) { return bitcast<float>((uint32_t)static_cast<const uint16_t*>(x)[i] << 16); }
  static __device__ __forceinline__ float value(const Raw& r, int e) { return bitcast<float>(e % 2 ? r.a[e / 2] & 0xffff0000u : r.a[e / 2] << 16); }
};
template <> struct Logits<_Float16> {
  typedef HalfRaw Raw;
  static __device__ __forceinline__ Raw tail(const void* x, int64_t i, int n) { return half_tail(x, i, n, 0xfc00u); }
  static __device__ __forceinline__ float one(const void* x, int64_t i) { return (float)static_cast<const _Float16*>(x)[i]; }
  static __device__ __forceinline__ float value(const Raw& r, int e) { return (float)bitcast<_Float16>((uint16_t)(e % 2 ? r.a[e / 2] >> 16 : r.a[e / 2])); }
};

// Lanes of m before this one.
__device__ __forceinline__ int rank_in(uint64_t m) { return __builtin_amdgcn_mbcnt_hi(high_u32(m), __builtin_amdgcn_mbcnt_lo(low_u32(m), 0)); }

// Of a wave's values v (E of each lane) the largest t that k of them reach, by its bits from
// the highest to bit `low`, or a smaller one that exactly k reach (then exact is set); 0 of fewer than k.
template <int E> __device__ __forceinline__ uint32_t bisect(const uint32_t (&v)[E], int k, int low, bool& exact) {
  uint32_t t = 0;
  exact = false;
#pragma unroll 1
  for (int bit = 30; bit >= low; bit -= 2) {   // two at a time: the counts' latency is what it takes
    int c[4];
#pragma unroll
    for (int x = 1; x < 4; ++x) {
      c[x] = 0;
      const uint32_t trial = t | (uint32_t)x << bit;
#pragma unroll
      for (int e = 0; e < E; ++e) c[x] += __builtin_popcountll(__builtin_amdgcn_ballot_w64(v[e] >= trial));
    }
    const int x = c[3] >= k ? 3 : c[2] >= k ? 2 : c[1] >= k ? 1 : 0;
    t |= (uint32_t)x << bit;
    if (c[1] == k || c[2] == k || c[3] == k) {
      // (the largest trial that k reach is one that exactly k reach)
      exact = true;
      break;
    }
  }
  return t;
}
// f(integral_constant E) with the least power of two that E·per covers n, at most 16
template <class F> __device__ __forceinline__ void by_count(int n, int per, F f) {
  if (n <= per) f(std::integral_constant<int, 1>{});
  else if (n <= 2 * per) f(std::integral_constant<int, 2>{});
  else if (n <= 4 * per) f(std::integral_constant<int, 4>{});
  else f(std::integral_constant<int, 16>{});
}

// Keeps the k largest of a wave's list of n different keys in LDS, n at most 64·E, in any
// order, and gives the k-th's upper word, or a smaller one that only those k reach (0 where there are fewer).
template <int E> __device__ __forceinline__ uint32_t keep_some(uint64_t* list, int n, int k) {
  const int lane = threadIdx.x & 63;
  uint32_t hi[E], lo[E], low[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const uint64_t x = e * 64 + lane < n ? list[e * 64 + lane] : 0;
    hi[e] = high_u32(x);
    lo[e] = low_u32(x);
  }
  bool exact;
  const uint32_t h = bisect<E>(hi, k, 0, exact);
  uint32_t l = 0;
  if (!exact) {   // equal upper words: of those the lower
    int above = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      above += __builtin_popcountll(__builtin_amdgcn_ballot_w64(hi[e] > h));
      low[e] = hi[e] == h ? lo[e] : 0;
    }
    l = bisect<E>(low, k - above, 0, exact);
  }
  int at = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const bool stays = hi[e] > h || (hi[e] == h && lo[e] >= l);
    const uint64_t m = __builtin_amdgcn_ballot_w64(stays);
    if (stays) list[at + rank_in(m)] = compose_u64(lo[e], hi[e]);
    at += __builtin_popcountll(m);
  }
  return h;
}
// Of 64 at most: by their ranks, so that they are in order.
__device__ __forceinline__ uint32_t keep_few(uint64_t* list, int n, int k) {
  const int lane = threadIdx.x & 63;
  const uint64_t x = lane < n ? list[lane] : 0;
  int rank = 0;
#pragma unroll 4
  for (int j = 0; j < n; ++j) rank += list[j] > x;
  if (lane < n && rank < k) list[rank] = x;
  const int last = __builtin_ctzll(__builtin_amdgcn_ballot_w64(lane < n && rank == k - 1));
  return (uint32_t)__builtin_amdgcn_readlane(high_u32(x), last);
}
__device__ __forceinline__ uint32_t keep_largest(uint64_t* list, int& n, int k) {
  if (n <= k) return 0;
  const uint32_t h = n <= 64 ? keep_few(list, n, k) : n <= 128 ? keep_some<2>(list, n, k) : keep_some<4>(list, n, k);
  n = k;
  return h;
}

// What k of a wave's list of n >= k reach, to 16 bits.
__device__ __forceinline__ uint32_t some_of(const uint64_t* list, int n, int k) {
  const int lane = threadIdx.x & 63;
  bool exact;
  if (n <= 64) {
    const uint32_t v[1] = {lane < n ? high_u32(list[lane]) : 0};
    return bisect<1>(v, k, 16, exact);
  }
  uint32_t v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = e * 64 + lane < n ? high_u32(list[e * 64 + lane]) : 0;
  return bisect<4>(v, k, 16, exact);
}

// N·8 elements of each thread at a step.
template <class T, int N>
__global__ __launch_bounds__(kSelThreads) __attribute__((amdgpu_waves_per_eu(4))) void select_scan_kernel(const SelectArgs a) {
  constexpr bool BINS = kSelBins<T, N>;
  typedef Logits<T> L;
  typedef typename L::Raw Raw;
  constexpr int WAVES = kSelThreads / 64, STEP = kSelThreads * 8 * N;
  __shared__ uint64_t lists[WAVES][kSelWave];   // ordered logit, then the complement of the token: the lowest first among equals
  __shared__ __align__(16) Raw some8[WAVES][8];
  __shared__ int from8[WAVES][8], counts[WAVES];
  __shared__ __align__(16) uint32_t quarter[WAVES];   // what a share of k of the wave's elements reach
  __shared__ double sSum[WAVES];
  __shared__ float sRef[WAVES];
  __shared__ uint32_t bins[BINS ? kBins : 1];
  const int row = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
  const bool done = a.done && a.done[row];
  const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6), k = a.k;
  const int64_t base = (int64_t)(row / a.beams) * a.gs + (int64_t)(row % a.beams) * a.bs;
  const T* x = static_cast<const T*>(a.x) + base;
  const SelectSpan span = select_span(part, a.per, a.vocab);
  const int begin = span.begin, end = span.end;
  // a whole step, and the last one
  auto fetch = [&](int at, Raw (&r)[N]) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < N; ++j) r[j] = *reinterpret_cast<const Raw*>(x + at + (j * kSelThreads + tid) * 8);
  };
  auto fetch_tail = [&](int at, Raw (&r)[N]) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int i = (j * kSelThreads + tid) * 8, left = end - at;   // (at + i may be 2^31 or more)
      if (i + 8 <= left) r[j] = *reinterpret_cast<const Raw*>(x + at + i);
      else r[j] = L::tail(x + at, i, left - i);
    }
  };
  Raw cur[N], next[N];
  // (before it is known whether they are needed)
  if (end - begin >= STEP) fetch(begin, cur);
  else fetch_tail(begin, cur);
  if (done) return;
  if constexpr (BINS)
    for (int i = tid; i < (int)kBins; i += kSelThreads) bins[i] = 0;
  // (waves that have whole vectors of elements: the others have nothing to tell)
  const int active = min(WAVES, max(1, (end - begin) / 512));
  if (tid < WAVES) quarter[tid] = tid < active ? 0 : ~0u;
  __syncthreads();
  // After the first step the waves go their own ways, but that each tells what its share of
  // k of its elements reach: k of the workgroup's reach the least of that.
  uint64_t* list = lists[wave];
  const int some = (k + active - 1) / active;
  auto tell = [&](uint32_t q) __attribute__((always_inline)) {
    if (lane == 0 && wave < active) *const_cast<volatile uint32_t*>(&quarter[wave]) = q;
  };
  double sum = 0.;
  float ref = -INFINITY;   // the wave's
  bool bad = false;
  int n = 0, steps = 0;       // of the wave's list; done
  uint32_t t = kLowest + 1;   // what reaches it is listed; never −infinity
  for (int at = begin;; at += STEP) {
    const int left = end - at;   // (more than 0)
    const bool whole = left >= 2 * STEP;   // the step that follows
    if (whole) fetch(at + STEP, next);
    // f(logit, token) for the thread's elements of the step, read again: for rare cases
    auto each = [&](auto f) __attribute__((always_inline)) {
#pragma unroll 1
      for (int e = 0; e < 8 * N; ++e) {
        const int i = (e / 8 * kSelThreads + tid) * 8 + e % 8;
        if (i < left) f(L::one(x + at, i), at + i);
      }
    };
    float best[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      best[j] = L::value(cur[j], 0);
#pragma unroll
      for (int e = 1; e < 8; ++e) best[j] = maximum(best[j], L::value(cur[j], e));   // (a NaN stays)
      bad |= !(best[j] < INFINITY);
    }
    float most = best[0];
#pragma unroll
    for (int j = 1; j < N; ++j) most = fmaxf(most, best[j]);
    if (__builtin_amdgcn_ballot_w64(most > ref + kExpHigh)) {   // (the sums' reference need not be their maximum)
      const float top = unordered((uint32_t)__builtin_amdgcn_readlane(wave_max_scan((int)(ordered(most) ^ 0x80000000u)), 63) ^ 0x80000000u);
      if (ref > -INFINITY) sum *= exp((double)ref - (double)top);
      ref = top;
    }
    if (at == begin) {
      // Of the wave's maxima of 8 elements, to 16 bits, so that it is found in 8 steps
      bool exact;
      uint32_t v[N];
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = best[j] == best[j] ? ordered(best[j]) : 0;
      const uint32_t q = bisect<N>(v, some, 16, exact);
      tell(q);
      __syncthreads();
    }
    const u32x4 q4 = *reinterpret_cast<const volatile u32x4*>(quarter);
    t = max(t, min(min(q4[0], q4[1]), min(q4[2], q4[3])));
    if (__builtin_fabsf(ref) < 1e6f) {
      const float low = ref - kExpLow;
      const double m = ref;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if constexpr (BINS) {
          // (a bin is 4 bytes; the sign's half of them lies kBins / 2 on)
          uint32_t to[8], most = 0;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint32_t w = cur[j].a[e / 2];
            const uint32_t size = e % 2 ? w >> 16 & 0x7fffu : w & 0x7fffu;
            to[e] = size - kBinFirst;
            most = max(most, to[e]);
            to[e] |= (e % 2 ? w >> 31 : w >> 15 & 1u) * (kBins / 2);
          }
          if (__builtin_amdgcn_ballot_w64(most >= kBins / 2) == 0) {
#pragma unroll
            for (int e = 0; e < 8; ++e) atomicAdd(&bins[to[e]], 1u);
          } else {
#pragma unroll 1
            for (int e = 0; e < 8; ++e) {
              const uint32_t w = cur[j].a[0] >> (e & 1) * 16;
              // (the words move up, so that the loop need not be unrolled)
              const uint32_t i = (w & 0x7fffu) - kBinFirst;
              if (i < kBins / 2) atomicAdd(&bins[i | (w >> 15 & 1u) * (kBins / 2)], 1u);
              else sum += exp_term(maximum(bitcast<float>(w << 16), low), m);
              if (e & 1) cur[j].a = u32x4{cur[j].a[1], cur[j].a[2], cur[j].a[3], cur[j].a[0]};
            }
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) sum += exp_term(maximum(L::value(cur[j], e), low), m);
        }
      }
    } else if (ref > -INFINITY) {   // (ref − 415 may be ref)
      each([&](float y, int) { sum += exp_term((float)fmax((double)y - (double)ref, (double)-kExpLow), 0.); });
    }
    // Threads with an element that reaches t write their 8 down, 8 threads at a time, and
    // each lane looks at one
    int hits = 0, place[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const uint64_t m = __builtin_amdgcn_ballot_w64(best[j] >= unordered(t));
      place[j] = m >> lane & 1 ? hits + rank_in(m) : -1;
      hits += __builtin_popcountll(m);
    }
    uint32_t full = 0;
    for (int p = 0; p < hits; p += 8) {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if ((uint32_t)(place[j] - p) < 8u) {
          some8[wave][place[j] - p] = cur[j];
          from8[wave][place[j] - p] = at + (j * kSelThreads + tid) * 8;
        }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // (a wave's LDS accesses stay in order)
      const int i = lane >> 3;
      const float y = L::one(&some8[wave][i], lane & 7);
      const uint32_t token = (uint32_t)from8[wave][i] + (lane & 7);
      uint64_t m = __builtin_amdgcn_ballot_w64(i < hits - p && y >= unordered(t));
      if (n > kSelWave - 64) {
        full = keep_largest(list, n, k);
        t = max(t, full);
        m = __builtin_amdgcn_ballot_w64(i < hits - p && y >= unordered(t));
      }
      if (m >> lane & 1) list[n + rank_in(m)] = compose_u64(~token, ordered(y));
      n += __builtin_popcountll(m);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    if (n >= 3 * k || full) {
      full = keep_largest(list, n, k);
      // (k of the elements up to here reach `full`, and equals come later)
      if (full) t = max(t, full + 1);
    }
    // after 1, 2, 4, .. steps: by then half of what is seen is new
    ++steps;
    if (left <= STEP) break;
    if ((steps & (steps - 1)) == 0 && n >= some) tell(some_of(list, n, some));
    if (whole) {
#pragma unroll
      for (int j = 0; j < N; ++j) cur[j] = next[j];
    } else fetch_tail(at + STEP, cur);
  }
  // the waves' lists as one
  if (n > 64) keep_largest(list, n, k);
  if (lane == 0) counts[wave] = n;
  __syncthreads();
  if (wave == 0) {
#pragma unroll
    for (int w = 1; w < WAVES; ++w) {
      const int c = counts[w];
      const uint64_t x = lane < c ? lists[w][lane] : 0;
      if (lane < c) list[n + lane] = x;
      n += c;
    }
    keep_largest(list, n, k);
    u32x2* out = a.lists + (int64_t)blockIdx.x * k;
    if (lane < k) {
      const uint64_t x = lane < n ? list[lane] : ~0ull >> 32;
      out[lane] = u32x2{high_u32(x), ~low_u32(x)};   // (0 where there is none)
    }
  }
  const int64_t slot = blockIdx.x;
  if constexpr (BINS) {
    if (lane == 0) sRef[wave] = ref;
    __syncthreads();
    float top = sRef[0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) top = fmaxf(top, sRef[w]);
    if (top > -INFINITY && top < 1e6f) {   // (beside a larger one the bins' values are nothing)
      sum = ref > -INFINITY ? sum * exp((double)ref - (double)top) : 0.;
      ref = top;
      for (int i = tid; i < (int)kBins; i += kSelThreads) {
        const uint32_t c = bins[i];
        if (__builtin_amdgcn_ballot_w64(c != 0)) {
          const float x = bitcast<float>(((i & (kBins / 2 - 1)) + kBinFirst) << 16 | (i / (kBins / 2)) << 31);
          sum = __builtin_fma((double)c, exp_term(fmaxf(x, top - kExpLow), top), sum);
        }
      }
    }
    __syncthreads();
  }
  sum = wave_sum(sum);
  const bool any_bad = __builtin_amdgcn_ballot_w64(bad) != 0;
  if (lane == 0) {
    sSum[wave] = sum;
    sRef[wave] = any_bad ? NAN : ref;
  }
  __syncthreads();
  if (wave == 0) {
    const float r = sRef[lane % WAVES];
    const double s = sSum[lane % WAVES];
    float m = r;
    bool nan = r != r;
#pragma unroll
    for (int w = 1; w < WAVES; w *= 2) m = fmaxf(m, __shfl_xor(m, w));
    nan = __builtin_amdgcn_ballot_w64(nan) != 0;
    double y = r > -INFINITY ? s * exp((double)r - (double)m) : 0.;
#pragma unroll
    for (int w = 1; w < WAVES; w *= 2) y += __shfl_xor(y, w);
    if (lane == 0) a.heads[slot] = SelectHead{y, nan ? NAN : m, 0};
  }
}

// Of a join: a score; among equal ones the lower row, then the larger logit (`tie`: row, then the
// complement of the logit's ordered bits), then the lower place. A row's are so in the order of its
// logits, by which its parts keep theirs, whatever the score's 64 bits lose of them.
struct Candidate {
  double s;
  uint64_t tie;
  uint32_t at;
};
__device__ __forceinline__ bool ahead(const Candidate& x, const Candidate& y) {
  return x.s > y.s || (x.s == y.s && (x.tie < y.tie || (x.tie == y.tie && x.at < y.at)));
}

// A search: the rows' parts together. THREADS: 1024, or 256 where each then has one candidate
// (4 waves meet at a barrier sooner than 16: 256 candidates 4.3 us, with 1024 threads 6.8).
template <int THREADS, int EACH>
__global__ __launch_bounds__(THREADS) void select_join_kernel(const SelectArgs a) {
  constexpr int WAVES = THREADS / 64, LIST = THREADS;
  __shared__ double base[kSelMaxBeams];    // logarithm of the row's sum; infinity: finished
  __shared__ float run[kSelMaxBeams];      // scores[w]; NaN: no candidates
  __shared__ double score[LIST], last[LIST];
  __shared__ uint64_t tie[LIST], tied[LIST];
  __shared__ uint32_t index[LIST], place[LIST];
  __shared__ int rank[LIST];
  __shared__ int count, left;
  __shared__ uint32_t bound;
  const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6), k = a.k, g = blockIdx.x;
  const int64_t row0 = (int64_t)g * a.beams;
  const int per_row = a.parts * k, entries = a.beams * per_row;
  const u32x2* lists = a.lists + row0 * per_row;
  u32x2 c[EACH];   // (a finished row's are not written, and not used)
#pragma unroll
  for (int e = 0; e < EACH; ++e)
    if (e == 0 || e * THREADS < entries) c[e] = lists[min(e * THREADS + tid, entries - 1)];
  if (tid == 0) {
    count = left = 0;
    bound = 0;
  }
  rank[tid] = 0;
  int width = 1;   // lanes of a row, and rows of a wave: 64 / width
  while (width < a.parts && width < 64) width *= 2;
  for (int w0 = wave * (64 / width); w0 < a.beams; w0 += WAVES * (64 / width)) {
    const int w = w0 + lane / width;
    const bool real = w < a.beams;
    const int64_t row = row0 + min(w, a.beams - 1);
    const float s = a.scores[row];
    const bool done = a.done && a.done[row];
    float m = -INFINITY;
    int nan = 0;
    double sum = 0.;
    if (real && !done)   // (a finished row's are not written)
      for (int p = lane % width; p < a.parts; p += width) {
        const SelectHead h = a.heads[row * a.parts + p];
        nan |= h.ref != h.ref;
        if (h.ref > m) {
          sum = (m > -INFINITY ? sum * exp((double)m - (double)h.ref) : 0.) + h.sum;
          m = h.ref;
        } else if (h.ref > -INFINITY) sum += h.sum * exp((double)h.ref - (double)m);
      }
    float top = m;
    for (int x = 1; x < width; x *= 2) {
      top = fmaxf(top, __shfl_xor(top, x));
      nan |= __shfl_xor(nan, x);
    }
    sum = m > -INFINITY ? sum * exp((double)m - (double)top) : 0.;
    for (int x = 1; x < width; x *= 2) sum += __shfl_xor(sum, x);
    if (real && lane % width == 0) {
      run[w] = s > -INFINITY && s < INFINITY && (done || (!nan && top > -INFINITY)) ? s : NAN;
      base[w] = done ? INFINITY : (double)top + (log(sum) - kExpShift * 0.6931471805599453);
    }
  }
  __syncthreads();
  // entry i of the rows' lists, one after the other; false: there is none
  auto valued = [&](int i, u32x2 c, Candidate& x) __attribute__((always_inline)) {
    const int w = a.row_magic ? (int)__umulhi((uint32_t)i, a.row_magic) : i;
    const float r = run[w];
    const double b = base[w];
    const bool done = b == INFINITY;
    x.s = done ? (double)r : (double)r + ((double)unordered(c[0]) - b);
    x.tie = compose_u64(~c[0], (uint32_t)w);
    x.at = (uint32_t)w * a.vocab + (done ? (uint32_t)a.eos : c[1]);
    return r == r && (done ? i == w * per_row : c[0] != 0);
  };
  auto candidate = [&](int i, Candidate& x) __attribute__((always_inline)) { return valued(i, lists[i], x); };
  uint32_t key[EACH];   // the score in 32 bits; 0: none
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    key[e] = 0;
    if (e == 0 || e * THREADS < entries) {
      const int i = e * THREADS + tid;
      Candidate x;
      if (valued(min(i, entries - 1), c[e], x) && i < entries) key[e] = ordered((float)x.s);
    }
  }
  uint32_t t = 0;
  bool exact;
  if constexpr (EACH == 1) t = bisect<1>(key, k, 12, exact);
  else
    by_count(entries, THREADS, [&](auto size) __attribute__((always_inline)) {
      constexpr int E = decltype(size)::value;
      uint32_t v[E];
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = key[e];
      t = bisect<E>(v, k, 12, exact);
    });
  if (lane == 0) atomicMax(&bound, t);
  __syncthreads();
  t = max(bound, 1u);
#pragma unroll
  for (int e = 0; e < EACH; ++e)
    if (key[e] >= t) {
      const int n = atomicAdd(&count, 1);
      if (n < LIST) {
        Candidate x;
        candidate(e * THREADS + tid, x);
        score[n] = x.s;
        tie[n] = x.tie;
        index[n] = x.at;
      }
    }
  __syncthreads();
  int n = count;
  if (n > LIST) {
    // Too many, most of them equal: one after the other
    Candidate before{INFINITY, 0, 0};
    for (int x = 0; x < k; ++x) {
      Candidate best{-INFINITY, ~0ull, ~0u};
      for (int i = tid; i < entries; i += THREADS) {
        Candidate y;
        if (candidate(i, y) && ahead(before, y) && ahead(y, best)) best = y;
      }
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const Candidate y{__shfl_xor(best.s, d), (uint64_t)__shfl_xor((unsigned long long)best.tie, d), (uint32_t)__shfl_xor(best.at, d)};
        if (ahead(y, best)) best = y;
      }
      __syncthreads();
      if (lane == 0) {
        last[wave] = best.s;
        tied[wave] = best.tie;
        place[wave] = best.at;
      }
      __syncthreads();
#pragma unroll 1
      for (int w = 0; w < WAVES; ++w) {
        const Candidate y{last[w], tied[w], place[w]};
        if (ahead(y, best)) best = y;
      }
      before = best;
      if (tid == 0) {
        score[x] = best.s;
        tie[x] = best.tie;
        index[x] = best.at;
      }
    }
    __syncthreads();
    n = k;
  }
  // many: the k-th of the list in 32 bits, and what reaches it
  uint32_t h = 0;
  if (n > 2 * k && n > 64) {
    if (wave == 0)
      by_count(n, 64, [&](auto size) __attribute__((always_inline)) {
        constexpr int E = decltype(size)::value;
        uint32_t v[E];
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = e * 64 + lane < n ? ordered((float)score[e * 64 + lane]) : 0;
        h = bisect<E>(v, k, 0, exact);
      });
    if (tid == 0) bound = h;
    __syncthreads();
    h = bound;
  }
  if (tid < n && ordered((float)score[tid]) >= h) {
    const int i = atomicAdd(&left, 1);
    last[i] = score[tid];
    tied[i] = tie[tid];
    place[i] = index[tid];
  }
  __syncthreads();
  // rank: a wave compares 64 of them with a share of all
  n = left;
  for (int i0 = 0; i0 < n; i0 += 64) {
    const int i = min(i0 + lane, n - 1);
    const Candidate x{last[i], tied[i], place[i]};
    int better = 0;
    for (int j = wave; j < n; j += WAVES) {
      const Candidate y{last[j], tied[j], place[j]};
      // (as `ahead`, without branches: 64 searches 59.9 us a call, with them 60.8)
      better += (y.s > x.s) | ((y.s == x.s) & ((y.tie < x.tie) | ((y.tie == x.tie) & (y.at < x.at))));
    }
    if (i0 + lane < n && better) atomicAdd(&rank[i], better);
  }
  __syncthreads();
  const int64_t o = (int64_t)g * k;
  if (tid < n && rank[tid] < k) {
    const int64_t i = o + rank[tid];
    const uint32_t w = place[tid] / (uint32_t)a.vocab;
    a.out_s[i] = (float)last[tid];
    a.out_t[i] = (int)(place[tid] - w * (uint32_t)a.vocab);
    a.out_p[i] = (int)(row0 + w);
  }
  if (tid >= n && tid < k) {
    a.out_s[o + tid] = -INFINITY;
    a.out_t[o + tid] = a.out_p[o + tid] = -1;
  }
}
