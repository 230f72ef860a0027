// gfx950.h — what the kernels of this library share: element types and MFMA
// traits, buffer resources and the LDS DMA, waits and barriers, the key order
// of score tiles, reductions over the two halves of a wave.
#ifndef MI355_FA_GFX950_H
#define MI355_FA_GFX950_H

#include <hip/hip_runtime.h>

#include <stdint.h>

#include "bits.h"

namespace mi355fa {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.4426950408889634f;

// ── element traits ───────────────────────────────────────────────────────────
template <bool BF16> struct Elt;
template <> struct Elt<true> {
  typedef bf16x8 v8;
  static __device__ __forceinline__ f32x16 mfma(v8 a, v8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct Elt<false> {
  typedef f16x8 v8;
  static __device__ __forceinline__ f32x16 mfma(v8 a, v8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};

template <typename To, typename From>
__device__ __forceinline__ To bitcast(const From& x) {
  static_assert(sizeof(To) == sizeof(From), "size mismatch");
  return __builtin_bit_cast(To, x);
}

// ── buffer resources ──────────────────────────────────────────────────────────
// Raw buffer loads/stores with 32-bit offsets: the hardware returns 0 for reads
// (and drops writes) at offsets >= num_records. Each resource is bounded to the
// valid rows of one head / one batch, so K/V rows >= Sk, Q/O rows >= Sq and mask
// rows >= mask_seqlen_q need no predicate. All variable per-lane offsets are
// passed as the VGPR offset, which is what the range check covers; the per-tile
// shift along the keys moves the resource base instead (scalar arithmetic),
// shrinking num_records by the same amount so the check is unchanged.
typedef __amdgpu_buffer_rsrc_t rsrc_t;
typedef __attribute__((address_space(3))) void lds_void;
constexpr int kRsrcFlags = 0x00020000;  // raw buffer, 32-bit data format (gfx9 family)

__device__ __forceinline__ rsrc_t make_rsrc(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, (int)bytes,
                                           kRsrcFlags);
}
__device__ __forceinline__ u32x4 bload16(rsrc_t r, uint32_t voff) {
  return __builtin_amdgcn_raw_buffer_load_b128(r, voff, 0, 0);
}
// 16 bytes per lane from the buffer straight into LDS: lane i of the wave lands
// at lds + 16·i (gfx950 LDS DMA), no VGPR staging. Issued as inline assembly so
// the compiler does not track the LDS write: it would otherwise wait for every
// DMA in flight (vmcnt(0)) before each LDS read and each workgroup barrier,
// which serialises a multi-stage pipeline. Completion is therefore the
// caller's job: wait_vmcnt for the issuing wave, then wg_barrier for the others.
typedef int i32x4 __attribute__((ext_vector_type(4)));
// The same buffer descriptor as make_rsrc, as four plain words for the asm.
__device__ __forceinline__ i32x4 make_rsrc_words(const void* base, uint32_t bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(base);
  // Uniform by construction; readfirstlane makes the compiler keep it in SGPRs.
  return i32x4{(int)__builtin_amdgcn_readfirstlane((uint32_t)a),
               (int)__builtin_amdgcn_readfirstlane((uint32_t)(a >> 32) & 0xffffu),
               (int)__builtin_amdgcn_readfirstlane(bytes), kRsrcFlags};
}
// LDS byte address of a __shared__ array (folds to a constant after inlining).
__device__ __forceinline__ uint32_t lds_addr(const uint16_t* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint16_t*)p;
}
// NT: the non-temporal hint, for data each workgroup reads exactly once in a
// launch (the replacement policy then keeps other lines; cold reads of such a
// stream run up to 10 % faster).
template <bool NT = false>
__device__ __forceinline__ void bload16_lds(i32x4 rs, uint32_t lds_byte, uint32_t voff) {
  const uint32_t m0v = __builtin_amdgcn_readfirstlane(lds_byte);
  if constexpr (NT)
    asm volatile(
        "s_mov_b32 m0, %0\n\t"
        "s_nop 0\n\t"
        "buffer_load_dwordx4 %1, %2, 0 offen nt lds"
        :
        : "s"(m0v), "v"(voff), "s"(rs)
        : "memory", "m0");
  else
    asm volatile(
        "s_mov_b32 m0, %0\n\t"
        "s_nop 0\n\t"
        "buffer_load_dwordx4 %1, %2, 0 offen lds"
        :
        : "s"(m0v), "v"(voff), "s"(rs)
        : "memory", "m0");
}

// Workgroup-id remap: the hardware hands linear id L to XCD (L % 8). Give each
// XCD a contiguous chunk of logical tile ids so neighbouring tiles share an L2.
__device__ __forceinline__ int xcd_remap(int L, int total) {
  constexpr int kXcd = 8;
  const int q = total / kXcd, r = total % kXcd;
  const int xcd = L % kXcd, local = L / kXcd;
  return (xcd < r) ? xcd * (q + 1) + local : r * (q + 1) + (xcd - r) * q + local;
}

// Row r of a 32-key block of K in LDS holds key π(r): in the 32x32 C layout of
// Sᵀ = K·Qᵀ a lane (query row, half g) then owns the 16 consecutive keys 16g ..
// 16g + 15, and the rounded probabilities of 8 of them are one B operand of
// Oᵀ += Vᵀ·Pᵀ.
__device__ __forceinline__ int key_perm(int r) {   // π within a 32-key block
  return ((r >> 2) & 1) * 16 + (r >> 3) * 4 + (r & 3);
}

// s_waitcnt vmcnt(N), other counters untouched (gfx9 encoding: vmcnt[3:0] | [15:14])
template <int N> __device__ __forceinline__ void wait_vmcnt() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (15 << 8) | ((N >> 4) << 14));
  __atomic_signal_fence(__ATOMIC_SEQ_CST);   // no LDS access moves above the wait
}

// Workgroup barrier for the LDS pipeline: this wave's LDS reads have returned
// (so no other wave's DMA can overwrite what they read) and nothing moves across.
// Unlike __syncthreads it does not wait for the LDS DMAs in flight.
__device__ __forceinline__ void wg_barrier() {
  __builtin_amdgcn_s_waitcnt(15 | (7 << 4) | (0 << 8) | (3 << 14));   // lgkmcnt(0)
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_s_barrier();
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
}

// max / sum with the lane 32 apart (the other half of the same query row)
__device__ __forceinline__ float xhalf_max(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float xhalf_sum(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Σ of the 8 rounded P values of one MFMA operand, two per dot2 (fp32 accumulate).
template <bool BF16>
__device__ __forceinline__ float psum8(typename Elt<BF16>::v8 v, float acc) {
  if constexpr (BF16) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 one = {(__bf16)1.0f, (__bf16)1.0f};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      acc = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{v[2 * i], v[2 * i + 1]}, one, acc, false);
  } else {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    const f16x2 one = {(_Float16)1.0f, (_Float16)1.0f};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      acc = __builtin_amdgcn_fdot2(f16x2{v[2 * i], v[2 * i + 1]}, one, acc, false);
  }
  return acc;
}

// readfirstlane of a value the caller knows to be uniform
__device__ __forceinline__ int uni(int x) { return (int)__builtin_amdgcn_readfirstlane((uint32_t)x); }

// The kernel's parameter struct, read again from the kernarg segment (scalar loads, behind
// an empty asm statement) where an epilogue needs it: held from the kernel's entry across
// a tile loop its fields would spill.
template <class T> using kernarg = const __attribute__((address_space(4))) T;
template <class T> __device__ __forceinline__ kernarg<T>& reload_kernarg(const T& host) {
#if defined(__HIP_DEVICE_COMPILE__)
  kernarg<T>* q = (kernarg<T>*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(q));
  return *q;
#else
  return *(kernarg<T>*)&host;   // host pass only: never runs
#endif
}

// XOR swizzle of V's 16-byte chunks by LDS row, for conflict-free transposed reads
template <int D> __device__ __forceinline__ int v_swz(int r) {
  return (D == 128) ? 4 * (r & 3) : 4 * ((r >> 1) & 1);
}

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

}  // namespace mi355fa

#endif  // MI355_FA_GFX950_H
