// Arithmetic shared by the attention kernels over a paged cache.
#pragma once

#include "common.cuh"

namespace smb {

constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kNegInf = -__builtin_huge_valf();

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two 32-bit values in one instruction.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// A row's running maximum m is raised when a score passes it by more than kGrow + kLift (base-2 units), and then to
// that score less kLift: most tiles skip the rescaling, and the weights p = 2^(score - m) stay below
// 2^(kGrow + kLift).  fp16 ends at 2^16 and loses places below 2^-14, so its weights are lifted by 2^7: they keep their
// relative precision down to 2^-21 of the row's largest (2^-14 without), and are off by 2^-32 of it at most below.
constexpr float kGrow = 8.f;

template <typename T>
struct Half2;
template <>
struct Half2<__nv_bfloat16> {
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  // 16 + nibble e (and e + 4) of w: ulp of 16.0 is 2^-3, so the nibble goes to mantissa bits 3-6
  static constexpr uint32_t kMask = 0x00780078u, kBase = 0x41804180u;
  static constexpr int kUp = 3;
  static constexpr float kMost = 3.38953138925153547590e38f;  // the largest finite number
  static constexpr float kLift = 0.f;
  static __device__ __forceinline__ uint32_t towards_zero(float x) { return __bfloat16_as_ushort(__float2bfloat16_rz(x)); }
  static __device__ __forceinline__ uint32_t dequant(uint32_t v, uint32_t s2, uint32_t z2) {
    const __nv_bfloat162 x = *reinterpret_cast<const __nv_bfloat162*>(&v);
    const uint32_t base = kBase;
    const __nv_bfloat162 d = __hsub2(x, *reinterpret_cast<const __nv_bfloat162*>(&base));
    const __nv_bfloat162 r = __hfma2(d, *reinterpret_cast<const __nv_bfloat162*>(&s2), *reinterpret_cast<const __nv_bfloat162*>(&z2));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ float lo(uint32_t v) { return __uint_as_float(v << 16); }
  static __device__ __forceinline__ float hi(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }
  static __device__ __forceinline__ bool nonfinite(uint32_t h) { return (h & 0x7f80u) == 0x7f80u; }
};
template <>
struct Half2<__half> {
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  // ulp of 16.0 is 2^-6: mantissa bits 6-9
  static constexpr uint32_t kMask = 0x03C003C0u, kBase = 0x4C004C00u;
  static constexpr int kUp = 6;
  static constexpr float kMost = 65504.f;  // the largest finite number
  static constexpr float kLift = 7.f;
  static __device__ __forceinline__ uint32_t towards_zero(float x) { return __half_as_ushort(__float2half_rz(x)); }
  static __device__ __forceinline__ uint32_t dequant(uint32_t v, uint32_t s2, uint32_t z2) {
    const __half2 x = *reinterpret_cast<const __half2*>(&v);
    const uint32_t base = kBase;
    const __half2 d = __hsub2(x, *reinterpret_cast<const __half2*>(&base));
    const __half2 r = __hfma2(d, *reinterpret_cast<const __half2*>(&s2), *reinterpret_cast<const __half2*>(&z2));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ float2 both(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
  static __device__ __forceinline__ float lo(uint32_t v) { return both(v).x; }
  static __device__ __forceinline__ float hi(uint32_t v) { return both(v).y; }
  static __device__ __forceinline__ bool nonfinite(uint32_t h) { return (h & 0x7c00u) == 0x7c00u; }
};

// Nibbles e and e + 4 of w as 16 + code, one in each half.
template <typename T, int E>
__device__ __forceinline__ uint32_t nib(uint32_t w) {
  constexpr int sh = Half2<T>::kUp - 4 * E;
  uint32_t v;
  if constexpr (sh >= 0) v = w << sh;
  else v = w >> (-sh);
  return (v & Half2<T>::kMask) | Half2<T>::kBase;
}

// The value of a code of a 4-bit group with the pair `sz` (scale, zero), as the products get it: the 16-bit
// number (in the low half) nearest code * scale + zero, which may overflow though all three are finite.
template <typename T>
__device__ __forceinline__ uint32_t value_of(uint32_t code, uint32_t sz) {
  const uint32_t v = Half2<T>::kBase | (code * 0x00010001u << Half2<T>::kUp);
  return Half2<T>::dequant(v, __byte_perm(sz, sz, 0x1010), __byte_perm(sz, sz, 0x3232)) & 0xffffu;
}

// Whether some code of such a group has a value that is not finite.  Rounding keeps the order, so the two
// ends tell (an infinite scale makes NaN of code 0).
template <typename T>
__device__ __forceinline__ bool group_overflows(uint32_t sz) {
  return Half2<T>::nonfinite(value_of<T>(0, sz)) || Half2<T>::nonfinite(value_of<T>(15, sz));
}

// Takes those values out of a group, to where a weight of 0 makes 0 of them; its finite values stay.  (A code whose value
// overflows goes to code 0, whose value is the zero: the rows that see it are infinite there already.)
template <typename T>
__device__ __forceinline__ void take_out_nonfinite(uint32_t* codes, uint32_t* sz) {
  const uint32_t pair = *sz;
  if (Half2<T>::nonfinite(pair & 0xffffu) || Half2<T>::nonfinite(pair >> 16)) {
    *sz = 0;
    return;
  }
#pragma unroll 1
  for (int e = 0; e < 32; ++e) {
    const int sh = 4 * (e & 7);
    if (Half2<T>::nonfinite(value_of<T>((codes[e >> 3] >> sh) & 15u, pair))) codes[e >> 3] &= ~(15u << sh);
  }
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool fill) {
  const int n = fill ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
}  // namespace smb
