// t5e_blocks.cuh -- device pieces shared by the block-scaled E2M1 kernels:
// real types, the block scale rules, the E2M1 conversions and the scale
// layout.
#pragma once

#include <cuda_runtime.h>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "t5e.h"

namespace t5e {
namespace blocks {

// Real element types (T5E_REAL_*): bits, conversion to F32.
template <int TYPE>
struct Real;
template <>
struct Real<T5E_REAL_F32> {
  using type = float;
  static constexpr int kBytes = 4;
};
template <>
struct Real<T5E_REAL_BF16> {
  using type = __nv_bfloat16;
  static constexpr int kBytes = 2;
};
template <>
struct Real<T5E_REAL_F16> {
  using type = __half;
  static constexpr int kBytes = 2;
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }

template <int TYPE>
__device__ __forceinline__ typename Real<TYPE>::type from_f32(float v) {
  if constexpr (TYPE == T5E_REAL_F32) return v;
  else if constexpr (TYPE == T5E_REAL_BF16) return __float2bfloat16_rn(v);
  else return __float2half_rn(v);
}

// Two elements of a packed 32-bit word (low element first).
template <int TYPE>
__device__ __forceinline__ void unpack2(uint32_t w, float& lo, float& hi) {
  if constexpr (TYPE == T5E_REAL_BF16) {
    lo = __uint_as_float(w << 16);
    hi = __uint_as_float(w & 0xFFFF0000u);
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    lo = f.x;
    hi = f.y;
  }
}

template <int TYPE>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (TYPE == T5E_REAL_BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}

// Loads of memory that the kernel before on the stream wrote.  Ordinary loads
// that stay behind the wait for that kernel: with programmatic launches it may
// still be writing while this one has begun, so the memory is not read-only for
// this kernel's whole time as non-coherent loads (__ldg, ld.global.nc) ask, and a
// compiler may move those ahead of the wait.  They take the same time (8192 x
// 8192 BF16 to UE4M3 blocks 31 to 32 us either way, back 29.3 and 29.4).
__device__ __forceinline__ uint4 load16(const void* p) {
  uint4 v;
  asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// 32 bytes of a lane in one access (32-byte aligned) or two (16-byte aligned): a
// warp whose lanes take neighbouring 32 bytes then touches whole lines.
__device__ __forceinline__ void load32(const void* p, bool wide, uint4& a, uint4& b) {
  if (wide) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w), "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w) : "l"(p));
  } else {
    a = load16(p);
    b = load16(static_cast<const uint4*>(p) + 1);
  }
}
__device__ __forceinline__ void store32(void* p, bool wide, const uint4& a, const uint4& b) {
  if (wide) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 :: "l"(p), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w) : "memory");
  } else {
    static_cast<uint4*>(p)[0] = a;
    static_cast<uint4*>(p)[1] = b;
  }
}

// Byte offset of scale b of row r in the scale tiles: 128 rows by 4 scales
// are 512 consecutive bytes, ordered so that one 16-byte line holds the four
// scales of rows r, r + 32, r + 64 and r + 96 (the order in which the tensor
// cores take them from tensor memory).  `groups` = ceil(scales per row / 4).
__device__ __forceinline__ uint64_t scale_offset(uint64_t r, uint32_t b, uint32_t groups) {
  return ((r >> 7) * groups + (b >> 2)) * 512u + (r & 31u) * 16u + ((r >> 5) & 3u) * 4u + (b & 3u);
}

// Value of a scale byte (NaN for the NaN codes; the sign bit of a UE4M3 byte
// is ignored, as by the tensor cores).
template <bool E8M0>
__device__ __forceinline__ float scale_value(uint32_t byte) {
  if constexpr (E8M0) {
    if (byte == 0xFFu) return __uint_as_float(0x7FC00000u);
    return byte == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23);
  } else {
    uint32_t h2;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"((uint16_t)(byte & 0x7Fu)));
    return __half2float(__ushort_as_half((unsigned short)(h2 & 0xFFFFu)));
  }
}

// How the elements of a tensor are multiplied and divided.
//
// General (kExact): u = F32(x * m), then u / step correctly rounded (Markstein's
// correction of the product with the correctly rounded reciprocal).  A quotient
// so rounded is an E2M1 tie only where the real one is: a tie times the step has
// at most 7 significand bits, so an F32 neighbour of it stays off the tie.
//
// Narrow (kNarrow): x has at most 11 significand bits and m is a power of two,
// so u is exact and, where it is not a tie itself, at least 2^-12 away from one:
// one product, truncated, with the nearest reciprocal is enough.  For the eight
// significands of a UE4M3 step that reciprocal is never below the real one and
// above it by less than 2^-24 of its value, so at a tie the product exceeds the
// tie by less than a unit in its last place and truncates to it.  m is part of
// the reciprocal; this holds m to 2^+-60.  With UE8M0 steps, whose products are
// exact, narrow means m = 1, for any type.
enum { kExact = 0, kNarrow = 1 };

template <int TYPE, bool E8M0>
__device__ __forceinline__ bool is_narrow(float m) {
  if constexpr (E8M0) return m == 1.f;
  const uint32_t b = __float_as_uint(m);
  return TYPE != T5E_REAL_F32 && (b & 0x007FFFFFu) == 0u && b >= (67u << 23) && b <= (187u << 23);
}

// Scale of a block from the largest magnitude `a` of its elements before the
// multiplier; returns the scale byte, and what divide() needs.
//   UE4M3: RNE of min(am / 6, 448).  am / 6 correctly rounded to F32 is a tie
//          of the 4-bit rounding only where the real quotient is (6 t has at
//          most 7 significand bits); narrow values need only the product with
//          F32(1/6), which returns t exactly for every am = 6 t.
//   UE8M0: 2^(floor(log2 am) - 2), or with `ceil` the smallest 2^e >= am / 6.
// Rounding to F32 is monotonic, so am = F32(a * m) is the largest |u|.  A block
// with a NaN or an infinity (or a product beyond F32) gets the NaN scale and a
// zero step.
//
// `inverses`: for narrow UE4M3 blocks, m / scale for every scale byte (0 for a
// zero scale and for NaN) in shared memory, see fill_inverses.
template <bool E8M0, int HOW>
__device__ __forceinline__ uint32_t block_scale(float a, float m, bool ceil, const float* inverses, float& step,
                                                float& inv) {
  const float am = a * m;
  const uint32_t bits = __float_as_uint(am);
  if constexpr (E8M0) {
    // word = floor(log2 am) - 2 + 127: the F32 exponent field less 2; F32
    // subnormals have field 0 and clamp to word 0 (2^-127), as zero does
    int w = (int)(bits >> 23) - 2;
    if (ceil && (bits & 0x7FFFFFu) > 0x400000u) w += 1;  // am > 1.5 * 2^floor(log2 am) = 6 * 2^(floor(log2 am) - 2)
    w = w < 0 ? 0 : w;
    const bool finite = bits < 0x7F800000u;
    // 2^(127 - w) without leaving F32: w = 0 gives 2^127 (w is at most 253)
    inv = finite ? __uint_as_float((uint32_t)(254 - w) << 23) : 0.f;
    step = 0.f;  // unused: products with inv are exact wherever they reach the E2M1 range
    return finite ? (uint32_t)w : 0xFFu;
  } else {
    if constexpr (HOW == kNarrow) {
      uint16_t two;
      asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(two) : "f"(0.f), "f"(am * (1.f / 6.f)));
      const uint32_t word = bits < 0x7F800000u ? (uint32_t)two : 0x7Fu;
      inv = inverses[word];
      step = 0.f;  // unused
      return word;
    } else {
      const bool finite = bits < 0x7F800000u;
      uint16_t two;
      asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(two) : "f"(0.f), "f"(__fdiv_rn(am, 6.f)));
      step = scale_value<false>(two);
      inv = finite && step > 0.f ? __frcp_rn(step) : 0.f;
      return finite ? (uint32_t)two : 0x7Fu;
    }
  }
}

// The 128 entries of block_scale's table, by the block's threads; a barrier has
// to follow.
__device__ __forceinline__ void fill_inverses(float* inverses, float m) {
  for (uint32_t i = threadIdx.x; i < 128u; i += blockDim.x) {
    const float step = scale_value<false>(i);
    inverses[i] = i == 0u || i == 0x7Fu ? 0.f : __frcp_rn(step) * m;
  }
}

template <bool E8M0, int HOW>
__device__ __forceinline__ float divide(float x, float m, float step, float inv) {
  if constexpr (E8M0) {
    return HOW == kNarrow ? x * inv : x * m * inv;
  } else if constexpr (HOW == kNarrow) {
    return __fmul_rz(x, inv);
  } else {
    const float u = x * m, y = __fmul_rn(u, inv);
    return __fmaf_rn(-__fmaf_rn(y, step, -u), inv, y);  // this order of signs keeps a negative zero
  }
}

// Eight values to eight E2M1 codes (RNE, magnitudes above 6 become 6), the first in
// the lowest nibble.
__device__ __forceinline__ uint32_t e2m1x8(const float* v) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}\n"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

// Eight E2M1 codes to their values.
__device__ __forceinline__ void from_e2m1x8(uint32_t w, float* v) {
  uint32_t h[4];
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "mov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}\n"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(w));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

// The tensor multiplier of a largest magnitude: the largest power of two m
// with a * m <= 6 * 448, held to 2^+-126; 1 where a is 0 or not finite.
// 2688 = 1.3125 * 2^11.
__device__ __forceinline__ float multiplier_of(uint32_t abs_bits) {
  if (abs_bits == 0u || abs_bits >= 0x7F800000u) return 1.f;
  int e;
  const float f = frexpf(__uint_as_float(abs_bits), &e);  // a = 2f * 2^(e - 1)
  int p = 11 - (e - 1) - (2.f * f > 1.3125f ? 1 : 0);
  p = p > 126 ? 126 : (p < -126 ? -126 : p);
  return __uint_as_float((uint32_t)(p + 127) << 23);
}

__device__ __forceinline__ void wait_for_previous_grid() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_grid_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

}  // namespace blocks
}  // namespace t5e
