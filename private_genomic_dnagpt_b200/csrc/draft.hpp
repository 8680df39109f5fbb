// draft.hpp -- what the translation units of the drafted-decoding operators
// share: argument checks, the device guard, element conversions and the
// ancestor masks of a tree of drafted nodes.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <string>

#include "../../include/ckks_b200.h"
#include "capi_types.hpp"
#include "ckks_internal.hpp"

namespace ckks {
namespace draft {

constexpr int kMaxNodes = 64;  // a node's ancestors are the bits of one 64-bit word
constexpr int kMaxHeadDim = 256;

inline void need(bool ok, const char* msg) {
  if (!ok) throw Error(CKKS_EARG, msg);
}

template <typename F>
int guard(F&& f) {
  try {
    f();
    return CKKS_OK;
  } catch (const Error& e) {
    set_last_error(e.what());
    return e.code;
  } catch (const std::exception& e) {
    set_last_error(e.what());
    return CKKS_EARG;
  } catch (...) {
    set_last_error("unknown error");
    return CKKS_EARG;
  }
}

inline Context& context_of(ckks_ctx* x) {
  need(x && x->c, "null context");
  return *x->c;
}

// makes the context's device current for one call
struct OnDevice {
  int prev = -1;
  explicit OnDevice(const Context& c) {
    int cur = -1;
    CKKS_CUDA(cudaGetDevice(&cur));
    if (cur != c.params.device) {
      CKKS_CUDA(cudaSetDevice(c.params.device));
      prev = cur;
    }
  }
  ~OnDevice() {
    if (prev >= 0) cudaSetDevice(prev);
  }
};

inline int element_bytes(int dtype) {
  switch (dtype) {
    case CKKS_BF16:
    case CKKS_FP16:
      return 2;
    case CKKS_FP32:
      return 4;
    case CKKS_FP64:
      return 8;
  }
  throw Error(CKKS_EARG, "element type is none of CKKS_BF16, CKKS_FP16, CKKS_FP32, CKKS_FP64");
}

inline void check_rows(const ckks_rows& r, int bytes, const char* what) {
  if (!r.data) throw Error(CKKS_EARG, std::string(what) + ": null device buffer");
  if (reinterpret_cast<uintptr_t>(r.data) % bytes)
    throw Error(CKKS_EARG, std::string(what) + ": address not aligned to its elements");
  if (r.batch < 0 || r.head < 0 || r.row < 0) throw Error(CKKS_EARG, std::string(what) + ": negative stride");
}

template <typename P>
void check_ptr(const P* p, const char* what) {
  if (!p) throw Error(CKKS_EARG, std::string(what) + ": null device buffer");
  if (reinterpret_cast<uintptr_t>(p) % alignof(P))
    throw Error(CKKS_EARG, std::string(what) + ": address not aligned to its elements");
}

// whether every row starts on a 16-byte boundary and holds whole 16-byte
// pieces (wide loads; TMA asks the same of bases and strides).  A stride
// along which there is one entry is never used.
inline bool wide_rows(const ckks_rows& r, int batch, int heads, int rows, int head_dim, int bytes) {
  auto fits = [&](int64_t s, int n) { return n <= 1 || (s * bytes) % 16 == 0; };
  return reinterpret_cast<uintptr_t>(r.data) % 16 == 0 && (head_dim * bytes) % 16 == 0 && fits(r.batch, batch) &&
         fits(r.head, heads) && fits(r.row, rows);
}

// last byte + 1 of a tensor of rows
inline const char* end_of(const ckks_rows& r, int batch, int heads, int rows, int row_elems, int bytes) {
  const int64_t last = (batch - 1) * r.batch + (heads - 1) * r.head + (int64_t)(rows - 1) * r.row + row_elems;
  return static_cast<const char*>(r.data) + last * bytes;
}

// `clusters` clusters of C CTAs
template <int C, class P>
void launch_cluster(void (*kernel)(P), int clusters, int threads, cudaStream_t st, const P& params) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)clusters * C);
  cfg.blockDim = dim3(threads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  CKKS_CUDA(cudaLaunchKernelEx(&cfg, kernel, params));
}

// all CTAs of the cluster, and a value in CTA `rank`'s shared memory
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_addr(const void* p, int rank) {
  uint32_t a;
  const uint32_t own = (uint32_t)__cvta_generic_to_shared(p);
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(own), "r"(rank));
  return a;
}
__device__ __forceinline__ int cluster_read(const int* p, int rank) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(cluster_addr(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ double cluster_read(const double* p, int rank) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(cluster_addr(p, rank)) : "memory");
  return v;
}

template <typename T>
__device__ __forceinline__ float to_f32(T x) {
  if constexpr (std::is_same_v<T, __nv_bfloat16>)
    return __bfloat162float(x);
  else if constexpr (std::is_same_v<T, __half>)
    return __half2float(x);
  else
    return (float)x;
}

template <typename T>
__device__ __forceinline__ T from_f32(float x) {
  if constexpr (std::is_same_v<T, __nv_bfloat16>)
    return __float2bfloat16_rn(x);
  else if constexpr (std::is_same_v<T, __half>)
    return __float2half_rn(x);
  else
    return (T)x;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// four elements of a row from element d on, as floats; 0 behind the row's end
template <typename T>
__device__ __forceinline__ void load_row4(float* dst, const T* src, int d, int D, bool wide) {
  if (wide) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(dst) = *reinterpret_cast<const float4*>(src + d);
    } else {
      const uint2 u = *reinterpret_cast<const uint2*>(src + d);
      const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
      for (int k = 0; k < 4; ++k) dst[k] = to_f32(e[k]);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) dst[k] = d + k < D ? to_f32(src[d + k]) : 0.0f;
  }
}

// Whether a sequence's count, path and length fit; evaluated alike by every
// thread of a CTA from `count` entries of path
__device__ __forceinline__ bool fits(const int32_t* path, int count, int len, int nodes, int capacity) {
  if (count < 0 || count > nodes || len < 0 || len > capacity || count > capacity - len) return false;
  bool ok = true;
#pragma unroll 8
  for (int j = 0; j < count; ++j) ok &= (unsigned)path[j] < (unsigned)nodes;  // no read waits for another
  return ok;
}

// A list of work whose length only the device knows: sequence b has `units`
// units of entries_of(b) entries each, one after the other.  CTA i of n takes
// the entries from list_start(i) to list_start(i + 1).
__device__ __forceinline__ int list_start(int entries, int i, int n) {
  return entries / n * i + (int)((unsigned)(entries % n) * (unsigned)i / (unsigned)n);
}

// entries of one unit of every sequence, summed; by a whole warp.  `first`:
// those of sequence `lane`
template <class F>
__device__ __forceinline__ int list_sum(int batch, F entries_of, int& first) {
  const int lane = threadIdx.x & 31;
  first = lane < batch ? entries_of(lane) : 0;
  int s = first;
  for (int b = lane + 32; b < batch; b += 32) s += entries_of(b);
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

struct ListPlace {
  int b, unit, entry, entries;  // sequence, its unit, the entry within that, the unit's entries
};

// entry `w` of the list; by a whole warp
template <class F>
__device__ __forceinline__ ListPlace list_find(int batch, int units, int w, int first, F entries_of) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int b0 = 0;; b0 += 32) {
    const int t = b0 == 0 ? first : b0 + lane < batch ? entries_of(b0 + lane) : 0;
    int sum = t * units;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += y;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, before + sum > w);
    if (past || b0 + 32 >= batch) {
      const int k = past ? __ffs(past) - 1 : 31;
      const int tk = max(1, __shfl_sync(0xffffffffu, t, k));
      const int off = w - (before + __shfl_sync(0xffffffffu, sum, k) - tk * units);
      return {b0 + k, off / tk, off % tk, tk};
    }
    before += __shfl_sync(0xffffffffu, sum, 31);
  }
}

// Ancestor masks of one tree, by one warp, in two steps: the parents into
// registers, then mask[i] gets the bits of node i and of the nodes above it, 0
// where i is padding.  Six rounds of pointer doubling cover every depth up to
// 64.  `jump` is scratch of 64 ints.
struct TreeReader {
  int parent[2];
  __device__ __forceinline__ void read(const int32_t* __restrict__ parents, int n) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int k = 0; k < 2; ++k) parent[k] = lane + 32 * k < n ? parents[lane + 32 * k] : -2;
  }
  __device__ __forceinline__ void masks(uint64_t* mask, int* jump) const {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int i = lane + 32 * k;
      const bool ok = parent[k] >= -1 && parent[k] < i;  // a parent comes before its children
      mask[i] = ok ? 1ull << i : 0ull;
      jump[i] = ok ? parent[k] : -2;
    }
    __syncwarp();
#pragma unroll 1
    for (int r = 0; r < 6; ++r) {
      uint64_t m[2];
      int j[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int i = lane + 32 * k;
        const int p = jump[i];
        m[k] = mask[i] | (p >= 0 ? mask[p] : 0ull);
        j[k] = p >= 0 ? jump[p] : p;
      }
      __syncwarp();
      bool open = false;  // a walk has not reached the root yet
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        mask[lane + 32 * k] = m[k];
        jump[lane + 32 * k] = j[k];
        open |= j[k] >= 0;
      }
      __syncwarp();
      if (!__any_sync(0xffffffffu, open)) break;
    }
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (jump[lane + 32 * k] != -1) mask[lane + 32 * k] = 0ull;
    __syncwarp();
  }
};

__device__ __forceinline__ void tree_masks(const int32_t* __restrict__ parents, int n, uint64_t* mask, int* jump) {
  TreeReader t;
  t.read(parents, n);
  t.masks(mask, jump);
}

}  // namespace draft
}  // namespace ckks
