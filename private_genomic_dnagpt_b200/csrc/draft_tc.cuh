// draft_tc.cuh -- what the attention kernels on the tensor cores share: tile
// sizes, arithmetic on pairs, waits that whole warps agree on, tensor maps.
#pragma once
#include "draft.hpp"
#include "tcgen.cuh"

namespace ckks {
namespace draft {

constexpr int kM = 128, kKeys = 128, kTmemCols = 512;
constexpr uint32_t kPanel = 128 * 128;  // 128 rows x 64 elements
constexpr float kSlack = 8.0f;
// float16 weights end at 2^-24, far above the smallest ones beside a heavy key,
// so their reference point lies 2^7 below the maximum: the largest weight is
// between 2^7 and 2^15
template <typename T>
constexpr float kBelow = std::is_same_v<T, __half> ? 7.0f : 0.0f;

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same_v<T, __nv_bfloat16>) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}

// two float32 operations in one instruction
__device__ __forceinline__ unsigned long long pair_of(float2 v) {
  return (unsigned long long)__float_as_uint(v.y) << 32 | __float_as_uint(v.x);
}
__device__ __forceinline__ float2 of_pair(unsigned long long v) {
  return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(pair_of(a)), "l"(pair_of(b)), "l"(pair_of(c)));
  return of_pair(d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  unsigned long long d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(pair_of(a)), "l"(pair_of(b)));
  return of_pair(d);
}
__device__ __forceinline__ float2 sub2(float2 a, float2 b) {
  unsigned long long d;
  asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(pair_of(a)), "l"(pair_of(b)));
  return of_pair(d);
}

// any of eight 16-bit elements infinite or NaN
template <typename T>
__device__ __forceinline__ bool not_finite(uint4 v) {
  constexpr uint32_t e = std::is_same_v<T, __nv_bfloat16> ? 0x7F80u : 0x7C00u;
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  bool bad = false;
#pragma unroll
  for (int k = 0; k < 4; ++k) bad |= (w[k] & e) == e || ((w[k] >> 16) & e) == e;
  return bad;
}

__device__ __forceinline__ void group_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// The barriers above wait without limit, so warps that meet there go on or
// leave together: a wait on an mbarrier counts for the whole warp (which then
// runs the collective tensor-memory instructions or does not), and the warps'
// results are joined at a barrier that all of them reach, whatever theirs is.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity) {
  return (bool)__all_sync(0xffffffffu, mbar_wait_short(bar, parity));
}
// the same where the phase is mostly complete already: one look without a loop
__device__ __forceinline__ bool warp_wait_done(uint32_t bar, uint32_t parity) {
  return __all_sync(0xffffffffu, mbar_test(bar, parity)) || warp_wait(bar, parity);
}
// two such waits; done both, they cost one look (a look takes about 200 cycles of
// the warp that issues the products: trees of 21 over 4001 keys 29.2 -> 27.6 us)
__device__ __forceinline__ bool warp_wait_both(uint32_t a, uint32_t pa, uint32_t b, uint32_t pb) {
  uint32_t done;
  asm volatile(
      "{\n .reg .pred p, q;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      " mbarrier.try_wait.parity.shared::cta.b64 q, [%3], %4;\n and.pred p, p, q;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(done)
      : "r"(a), "r"(pa), "r"(b), "r"(pb)
      : "memory");
  return __all_sync(0xffffffffu, done) || (warp_wait(a, pa) && warp_wait(b, pb));
}
// three
__device__ __forceinline__ bool warp_wait_all(uint32_t a, uint32_t pa, uint32_t b, uint32_t pb, uint32_t c, uint32_t pc) {
  uint32_t done;
  asm volatile(
      "{\n .reg .pred p, q, r;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      " mbarrier.try_wait.parity.shared::cta.b64 q, [%3], %4;\n mbarrier.try_wait.parity.shared::cta.b64 r, [%5], %6;\n"
      " and.pred p, p, q;\n and.pred p, p, r;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(done)
      : "r"(a), "r"(pa), "r"(b), "r"(pb), "r"(c), "r"(pc)
      : "memory");
  return __all_sync(0xffffffffu, done) || (warp_wait(a, pa) && warp_wait(b, pb) && warp_wait(c, pc));
}
__device__ __forceinline__ bool group_all(int id, int threads, bool ok) {
  uint32_t all;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 p, %3, 0;\n bar.red.and.pred q, %1, %2, p;\n selp.u32 %0, 1, 0, q;\n}\n"
      : "=r"(all)
      : "r"(id), "r"(threads), "r"((uint32_t)ok)
      : "memory");
  return all != 0;
}

using EncodeTiled = decltype(&cuTensorMapEncodeTiled);
inline EncodeTiled encode_tiled() {
  static const EncodeTiled f = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &r) != cudaSuccess ||
        r != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return f;
}

// [batch][outer][inner][head_dim] in boxes of box_outer x box_inner rows of 64
// elements; what a box has outside the tensor reads as 0
inline bool tile_map(CUtensorMap* m, void* data, int dtype, int head_dim, int inner, int64_t inner_stride, int box_inner,
              int outer, int64_t outer_stride, int box_outer, int batch, int64_t batch_stride) {
  const EncodeTiled f = encode_tiled();
  if (!f) return false;
  auto bytes = [](int64_t s, int n) { return n > 1 ? (cuuint64_t)s * 2 : (cuuint64_t)16; };
  const cuuint64_t dims[4] = {(cuuint64_t)head_dim, (cuuint64_t)inner, (cuuint64_t)outer, (cuuint64_t)batch};
  const cuuint64_t strides[3] = {bytes(inner_stride, inner), bytes(outer_stride, outer), bytes(batch_stride, batch)};
  const cuuint32_t box[4] = {64, (cuuint32_t)box_inner, (cuuint32_t)box_outer, 1}, ones[4] = {1, 1, 1, 1};
  return f(m, dtype == CKKS_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, data, dims,
           strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace draft
}  // namespace ckks
