// tcgen.cuh -- the fifth-generation tensor core: tensor memory, matrix
// products issued by one thread, their completion on an mbarrier, and tiled
// copies into swizzled shared memory.
#pragma once
#include <cuda.h>

#include "bulk.cuh"

namespace ckks {

// ---- tensor memory ---------------------------------------------------------
// one warp allocates `cols` columns (a power of two from 32) and frees them
__device__ __forceinline__ void tmem_alloc(uint32_t smem_slot, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_slot), "r"(cols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}

__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols));
}

// n columns of this warp's 32 lanes, one lane per thread
__device__ __forceinline__ void tmem_load16(uint32_t addr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, "
               "%10, %11, %12, %13, %14, %15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                 "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(addr));
}
__device__ __forceinline__ void tmem_load32(uint32_t addr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, "
               "%10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, "
               "%28, %29, %30, %31}, [%32];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                 "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
                 "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
                 "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]),
                 "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
               : "r"(addr));
}
__device__ __forceinline__ void tmem_store16(uint32_t addr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, "
               "%10, %11, %12, %13, %14, %15, %16};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), 
               "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), 
               "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
               : "memory");
}
__device__ __forceinline__ void tmem_store32(uint32_t addr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, "
               "%10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, "
               "%28, %29, %30, %31, %32};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), 
               "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), 
               "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), 
               "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), 
               "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
               : "memory");
}
template <int N>
__device__ __forceinline__ void tmem_load(uint32_t addr, uint32_t* r) {
  static_assert(N == 16 || N % 32 == 0);
  if constexpr (N == 16) {
    tmem_load16(addr, r);
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 32) tmem_load32(addr + i, r + i);
  }
}
template <int N>
__device__ __forceinline__ void tmem_store(uint32_t addr, const uint32_t* r) {
  static_assert(N == 16 || N % 32 == 0);
  if constexpr (N == 16) {
    tmem_store16(addr, r);
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 32) tmem_store32(addr + i, r + i);
  }
}

__device__ __forceinline__ void tmem_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// around a barrier between threads that use tensor memory
__device__ __forceinline__ void tmem_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// ---- matrix products ---------------------------------------------------------
// Shared-memory operand in rows of 128 bytes under the 128-byte swizzle (16
// byte piece c of row r sits at piece c ^ (r % 8)), groups of eight rows 1024
// bytes apart.  K-major: rows are the M or N index, a step of 16 elements
// along K is 32 bytes.  MN-major: rows are the K index, `lead` is the distance
// of the 64-element panels along M or N.
__device__ __forceinline__ uint64_t smem_operand(uint32_t addr, uint32_t lead) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | (uint64_t)((lead >> 4) & 0x3FFFu) << 16 | (uint64_t)(1024u >> 4) << 32 |
         1ull << 46 | 2ull << 61;
}

// instruction word: 16-bit operands (bf16 or f16), float32 sums, M x N, B
// K-major or MN-major
__host__ __device__ constexpr uint32_t mma_word(bool bf16, int m, int n, bool b_mn_major) {
  return 1u << 4 | (bf16 ? 1u << 7 | 1u << 10 : 0u) | (b_mn_major ? 1u << 16 : 0u) | (uint32_t)(n >> 3) << 17 |
         (uint32_t)(m >> 4) << 24;
}

// The following are called by a whole converged warp, one lane of which issues:
// the operands are uniform registers, and in a branch that one lane takes
// alone every product spends about 90 cycles on moving them there.

// D (tensor memory) = A B (+ D), A and B in shared memory
__device__ __forceinline__ void mma_smem(uint32_t d, uint64_t a, uint64_t b, uint32_t word, bool add) {
  asm volatile(
      "{\n .reg .pred p, one;\n setp.ne.u32 p, %4, 0;\n elect.sync _|one, 0xffffffff;\n"
      " @one tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(word), "r"((uint32_t)add)
      : "memory");
}

// the same with A in tensor memory
__device__ __forceinline__ void mma_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t word, bool add) {
  asm volatile(
      "{\n .reg .pred p, one;\n setp.ne.u32 p, %4, 0;\n elect.sync _|one, 0xffffffff;\n"
      " @one tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(word), "r"((uint32_t)add)
      : "memory");
}

// one arrival on `bar` once every product that this warp issued so far is done
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile(
      "{\n .reg .pred one;\n elect.sync _|one, 0xffffffff;\n"
      " @one tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(bar)
      : "memory");
}

// ---- shared memory ------------------------------------------------------------
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// makes this thread's writes to shared memory visible to copies and products
__device__ __forceinline__ void smem_fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// mbar_wait_bounded for waits that are mostly short: the global timer, whose
// reading takes longer than such a wait, is looked at only after a few polls
__device__ __forceinline__ bool mbar_wait_short(uint32_t bar, uint32_t parity) {
#pragma unroll 1
  for (int i = 0; i < 32; ++i)
    if (mbar_test(bar, parity)) return true;
  return mbar_wait_bounded(bar, parity);
}

// a box of a 4-d tensor map at (x, y, z, w) into shared memory
__device__ __forceinline__ void tile_load(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w,
                                          uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
      : "memory");
}

__device__ __forceinline__ void tile_prefetch(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

}  // namespace ckks
