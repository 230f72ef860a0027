// rope_store.h — rotary positions of q and k and the write of k and v into a paged
// cache, in one pass over a projection's output. Included by serve.hip inside
// namespace mi355fa.
//
// Pair (a, b) of a head becomes (a·c − b·s, b·c + a·s), c and s amplitude times
// the cosine and sine of position·inv_freq. Bound: bytes; q, k and v are read once
// and each output is written once.
//
//  * A workgroup serves a token: its threads first form each pair's cosine and sine
//    once, for all heads. The angle is a 64-bit product, reduced
//    to half turns in 64 bits: in 32 bits position 10^6 is off by 0.06 radians.
//  * Then a thread turns 16 elements at a time: two 16-byte chunks that hold 8
//    whole pairs, chunks (j, j + rot/16) of a head, or (2j, 2j + 1) interleaved.

struct RopeArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* qo;
  uint16_t* ko;
  uint16_t* kc;
  uint16_t* vc;
  const int* positions;
  const double* inv_freq;
  const int64_t* slots;
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, qo_ts, qo_hs, ko_ts, ko_hs;
  int64_t kc_ps, kc_hs, kc_rs, vc_ps, vc_hs, vc_rs;
  int64_t num_slots;
  int t, h, hk, rot, page;
  float amplitude;
};

template <int D, bool BF16, bool INTER>
__global__ __launch_bounds__(256) void rope_store_kernel(const RopeArgs a) {
  typedef typename Elt<BF16>::v8 V8;
  constexpr int U = D / 16;   // units of two chunks per head
  __shared__ float sC[D / 2], sS[D / 2];
  const int64_t t = blockIdx.x;
  const int tid = threadIdx.x;
  if (tid < a.rot / 2) {
    constexpr double kInvPi = 0.31830988618379067154;
    const double half = (double)a.positions[t] * a.inv_freq[tid] * kInvPi;   // half turns
    float s, c;
    sincospif((float)(half - 2.0 * rint(half * 0.5)), &s, &c);
    sC[tid] = c * a.amplitude;
    sS[tid] = s * a.amplitude;
  }
  __syncthreads();
  const int heads = a.h + 2 * a.hk, units = heads * U;
  const int ru = a.rot / 16;   // units that turn
  for (int x = tid; x < units; x += 256) {
    const int head = x / U, j = x % U;
    const uint16_t* src;
    if (head < a.h) src = a.q + t * a.q_ts + head * a.q_hs;
    else if (head < a.h + a.hk) src = a.k + t * a.k_ts + (head - a.h) * a.k_hs;
    else src = a.v + t * a.v_ts + (head - a.h - a.hk) * a.v_hs;
    const bool turns = j < ru && head < a.h + a.hk;
    const int c0 = (INTER || j >= ru) ? 2 * j : j, c1 = (INTER || j >= ru) ? 2 * j + 1 : j + ru;
    u32x4 lo = *reinterpret_cast<const u32x4*>(src + c0 * 8), hi = *reinterpret_cast<const u32x4*>(src + c1 * 8);
    if (turns) {
      const f32x8 xl = __builtin_convertvector(bitcast<V8>(lo), f32x8), xh = __builtin_convertvector(bitcast<V8>(hi), f32x8);
      const float* cs = &sC[j * 8];
      const float* sn = &sS[j * 8];
      f32x8 yl, yh;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float p = INTER ? (i < 4 ? xl[2 * (i & 3)] : xh[2 * (i & 3)]) : xl[i];
        const float r = INTER ? (i < 4 ? xl[2 * (i & 3) + 1] : xh[2 * (i & 3) + 1]) : xh[i];
        const float u = p * cs[i] - r * sn[i], w = r * cs[i] + p * sn[i];
        if constexpr (INTER) {
          if (i < 4) { yl[2 * (i & 3)] = u; yl[2 * (i & 3) + 1] = w; }
          else { yh[2 * (i & 3)] = u; yh[2 * (i & 3) + 1] = w; }
        } else {
          yl[i] = u;
          yh[i] = w;
        }
      }
      lo = bitcast<u32x4>(__builtin_convertvector(yl, V8));
      hi = bitcast<u32x4>(__builtin_convertvector(yh, V8));
    }
    uint16_t* out = nullptr;
    uint16_t* row = nullptr;
    if (head < a.h) {
      out = a.qo + t * a.qo_ts + head * a.qo_hs;
    } else {
      const int64_t slot = a.slots[t];
      const bool kept = slot >= 0 && slot < a.num_slots;
      const int64_t page = kept ? slot / a.page : 0, in = kept ? slot - page * a.page : 0;
      if (head < a.h + a.hk) {
        const int hk = head - a.h;
        out = a.ko + t * a.ko_ts + hk * a.ko_hs;
        if (kept) row = a.kc + page * a.kc_ps + hk * a.kc_hs + in * a.kc_rs;
      } else if (kept) {
        row = a.vc + page * a.vc_ps + (head - a.h - a.hk) * a.vc_hs + in * a.vc_rs;
      }
    }
    if (out) {
      *reinterpret_cast<u32x4*>(out + c0 * 8) = lo;
      *reinterpret_cast<u32x4*>(out + c1 * 8) = hi;
    }
    if (row) {
      *reinterpret_cast<u32x4*>(row + c0 * 8) = lo;
      *reinterpret_cast<u32x4*>(row + c1 * 8) = hi;
    }
  }
}
