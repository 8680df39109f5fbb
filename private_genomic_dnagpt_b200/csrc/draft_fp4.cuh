// draft_fp4.cuh -- rows of a 4-bit cache.
//
// A head's elements in groups of 16: each element x is a 4-bit floating-point
// number c (sign, two exponent bits, one mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4,
// 6) times the group's scale s, an 8-bit one (five exponent bits, three of
// mantissa, no sign).  A row is the groups' elements, 8 bytes each with the
// even element in a byte's low half, then the groups' scales, then zeros up to
// a multiple of four bytes: 9/16 of a byte an element.
//
// c s has at most six significant bits and lies in float16's range (s is at
// most 10240, six of it a float16; 2^-17 at the finest), so bfloat16 and float16
// hold every value of a row exactly and a product over the cache loses nothing
// on its way to the tensor cores.  An 8-bit scale without a sign has room for
// float16's exponents: it is the leading half of a float16 but for the sign,
// and decoding is one shift.
#pragma once
#include <cuda_fp4.h>

#include "draft.hpp"

namespace ckks {
namespace draft {

constexpr int kGroup4 = 16;
constexpr uint32_t kScaleTop = 0xE2;   // 10240
constexpr uint32_t kScaleNone = 0xFC;  // no number: a group that holds an infinity or a NaN

__host__ __device__ constexpr int groups4(int head_dim) { return (head_dim + kGroup4 - 1) / kGroup4; }
__host__ __device__ constexpr int row4_bytes(int head_dim) { return (9 * groups4(head_dim) + 3) / 4 * 4; }

// a cache's rows start on 4-byte boundaries
inline void check_row4(const ckks_rows& r, int batch, int heads, int rows, const char* what) {
  auto fits = [](int64_t s, int n) { return n <= 1 || s % 4 == 0; };
  if (reinterpret_cast<uintptr_t>(r.data) % 4 || !fits(r.batch, batch) || !fits(r.head, heads) || !fits(r.row, rows))
    throw Error(CKKS_EARG, std::string(what) + ": a 4-bit row does not start on a 4-byte boundary");
}

__device__ __forceinline__ __half scale4(uint32_t byte) { return __ushort_as_half((unsigned short)(byte << 7)); }

// A sixth of the group's largest magnitude, rounded to three bits of mantissa
// (to even in the middle).  The quotient rounded to 24 bits first gives the
// same result as the exact one: it can only reach a middle m of five bits from
// 6 m itself, because the float next to 6 m is off by more than half a step of m.
// (Rounded as in encode4; below 2^-18, where that need not hold, all become 0.)
__device__ __forceinline__ uint32_t scale4_of(float top) {
  constexpr float sixth = 1.0f / 6.0f;
  const float q = __fmul_rn(top, sixth), a = __fmaf_rn(__fmaf_rn(-q, 6.0f, top), sixth, q);
  const uint32_t u = __float_as_uint(a);
  const uint32_t b = min(((u + 0x7FFFFu + (u >> 20 & 1u)) >> 20) - (112u << 3), kScaleTop);
  return a < 6.103515625e-5f ? (uint32_t)__float2int_rn(a * 131072.0f) : b;  // below 2^-14: multiples of 2^-17
}

// One group: the 16 codes, and the scale from the largest magnitude (as bits).
// x / s is rounded to 24 bits, which moves no quotient onto or over
// the border between two codes (a border times s has at most seven bits, and
// the float next to it is off by more than half a step of the border).  The
// quotient is q + r e with q = x r, e = x - q s and r = 1 / s rounded: with r
// rounded correctly this is x / s rounded correctly (Markstein, "Computation
// of elementary functions on the IBM RISC System/6000 processor", 1990).
// r is one Newton step from an approximation to 2^-23, off by 2^-46 before it is
// rounded: s is a power of two times 8/8, 9/8, ..., 15/8, and the binary
// expansions of 8/9, 8/10, ..., 8/15 have periods of 2 to 12 digits, none of
// which continues a middle between two floats for 22 digits.
__device__ __forceinline__ uint2 encode4(const float* x, uint32_t top, uint32_t& scale) {
  const bool none = top >= 0x7F800000u;
  scale = scale4_of(__uint_as_float(top));
  // what is too small for any scale rounds to zeros, which keep their signs
  const float s = scale ? __half2float(scale4(scale)) : 1.0f;
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
  r = __fmaf_rn(r, __fmaf_rn(-s, r, 1.0f), r);
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float v = x[8 * h + i], q = __fmul_rn(v, r);
      t[i] = copysignf(__fmaf_rn(__fmaf_rn(-q, s, v), r, q), v);  // -0 stays
    }
    asm("{\n .reg .b8 a, b, c, d;\n cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
        " cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n mov.b32 %0, {a, b, c, d};\n}"
        : "=r"(w[h])
        : "f"(t[0]), "f"(t[1]), "f"(t[2]), "f"(t[3]), "f"(t[4]), "f"(t[5]), "f"(t[6]), "f"(t[7]));
  }
  if (none) scale = kScaleNone;
  return none ? make_uint2(0u, 0u) : make_uint2(w[0], w[1]);
}

// two elements from a byte, times the scale (in both halves), exactly
__device__ __forceinline__ __half2 decode4(uint32_t byte, __half2 scale) {
  return __hmul2(__half2(__nv_cvt_fp4x2_to_halfraw2((__nv_fp4x2_storage_t)byte, __NV_E2M1)), scale);
}
// the eight elements of a word, as pairs of T (bfloat16 or float16; exact in either)
template <typename T>
__device__ __forceinline__ void decode4_word(uint32_t word, __half2 scale, uint32_t* out) {
  uint32_t h[4];
  asm("{\n .reg .b8 a, b, c, d;\n mov.b32 {a, b, c, d}, %4;\n cvt.rn.f16x2.e2m1x2 %0, a;\n"
      " cvt.rn.f16x2.e2m1x2 %1, b;\n cvt.rn.f16x2.e2m1x2 %2, c;\n cvt.rn.f16x2.e2m1x2 %3, d;\n}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(word));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same_v<T, __nv_bfloat16>) {
      float lo, hi;  // the products as floats at once
      asm("{\n .reg .b16 a, b, s, t;\n mov.b32 {a, b}, %2;\n mov.b32 {s, t}, %3;\n fma.rn.f32.f16 %0, a, s, %4;\n"
          " fma.rn.f32.f16 %1, b, t, %4;\n}"
          : "=f"(lo), "=f"(hi)
          : "r"(h[i]), "r"(*reinterpret_cast<const uint32_t*>(&scale)), "f"(0.0f));
      const __nv_bfloat162 x = __floats2bfloat162_rn(lo, hi);
      out[i] = *reinterpret_cast<const uint32_t*>(&x);
    } else {
      const __half2 x = __hmul2(*reinterpret_cast<const __half2*>(&h[i]), scale);
      out[i] = *reinterpret_cast<const uint32_t*>(&x);
    }
  }
}
// scale byte `i` of a word, in both halves
__device__ __forceinline__ __half2 scale4_pair(uint32_t word, int i) {
  const uint32_t b = (word >> (8 * i) & 0xFFu) * 0x00800080u;
  return *reinterpret_cast<const __half2*>(&b);
}

// elements d .. d + 3 of a row (d a multiple of 4)
__device__ __forceinline__ void load_row4_4bit(float* dst, const uint8_t* row, int d, int D) {
  const __half2 s = __half2half2(scale4(row[8 * groups4(D) + d / kGroup4]));
  const float2 a = __half22float2(decode4(row[d / 2], s)), b = __half22float2(decode4(row[d / 2 + 1], s));
  dst[0] = a.x, dst[1] = a.y, dst[2] = b.x, dst[3] = b.y;
}

// attention over a 4-bit cache on the tensor cores (draft_attention4.cu): false,
// and nothing is launched, where the sizes or the caches' strides are not its
size_t attention4_tc_workspace(const Context& c, const ckks_draft_attention_args& a);
bool attention4_tc(const Context& c, const ckks_draft_attention_args& a, cudaStream_t st);

}  // namespace draft
}  // namespace ckks
