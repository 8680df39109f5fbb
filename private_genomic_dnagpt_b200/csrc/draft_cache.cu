// draft_cache.cu -- what happens to the draft model's key/value cache once
// the target has confirmed drafts: the accepted rows are appended
// (ckks_draft_commit), the attention weight they give each cached key is
// added up (ckks_draft_accumulate), and a cache that has grown past its
// budget keeps its latest and its heaviest keys (ckks_draft_evict).
#include <algorithm>
#include <cmath>

#include "draft.hpp"

namespace ckks {
namespace draft {
namespace {

// Whether a sequence's count, path and length fit; evaluated alike by every
// thread of a CTA from `count` entries of path
__device__ __forceinline__ bool fits(const int32_t* path, int count, int len, int nodes, int capacity) {
  if (count < 0 || count > nodes || len < 0 || len > capacity || count > capacity - len) return false;
  bool ok = true;
#pragma unroll 8
  for (int j = 0; j < count; ++j) ok &= (unsigned)path[j] < (unsigned)nodes;  // no read waits for another
  return ok;
}

// ---- commit --------------------------------------------------------------------
struct CommitParams {
  ckks_rows kc, vc, kn, vn;
  const int32_t* lens;
  const int32_t* path;
  const int32_t* count;
  int32_t* lens_out;
  unsigned int* refused;
  int batch, kv_heads, head_dim, nodes, capacity;
};

// CTA = (sequence, head): copies its accepted rows in pieces of V elements.  A
// few hundred KB: the launch bounds it (2.4 us for 3 rows of 12 heads, 3.2 us for
// 32 sequences of 16 heads).
template <typename T, typename V>
__global__ void __launch_bounds__(128) commit_kernel(CommitParams p) {
  const int b = blockIdx.x, h = blockIdx.y;
  const int32_t* path = p.path + (size_t)b * p.nodes;
  const int len = p.lens[b], count = p.count[b];
  const bool ok = fits(path, count, len, p.nodes, p.capacity);
  if (h == 0 && threadIdx.x == 0) {
    p.lens_out[b] = ok ? len + count : len;
    if (!ok) atomicAdd(p.refused, 1u);
  }
  if (!ok) return;
  constexpr int W = sizeof(V) / sizeof(T);
  const int per = p.head_dim / W;
  T* kc = static_cast<T*>(p.kc.data) + b * p.kc.batch + h * p.kc.head;
  T* vc = static_cast<T*>(p.vc.data) + b * p.vc.batch + h * p.vc.head;
  const T* kn = static_cast<const T*>(p.kn.data) + b * p.kn.batch + h * p.kn.head;
  const T* vn = static_cast<const T*>(p.vn.data) + b * p.vn.batch + h * p.vn.head;
  for (int i = threadIdx.x; i < count * per; i += blockDim.x) {
    const int j = i / per, d = i % per * W, node = path[j];
    *reinterpret_cast<V*>(kc + (len + j) * p.kc.row + d) = *reinterpret_cast<const V*>(kn + node * p.kn.row + d);
    *reinterpret_cast<V*>(vc + (len + j) * p.vc.row + d) = *reinterpret_cast<const V*>(vn + node * p.vn.row + d);
  }
}

// ---- accumulate -----------------------------------------------------------------
struct AccParams {
  ckks_rows q, kc, acc;
  const float* lse;
  const int32_t* lens;
  const int32_t* path;
  const int32_t* count;
  int batch, kv_heads, group, head_dim, nodes, capacity;
  float scale;
};

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kAccKeys = 128, kAccRows = 8;

// Any stride, size and alignment.  CTA = (sequence x head, 128 keys): one key
// per thread, the accepted rows in shared memory eight at a time; a key's
// weights are added in the order of the rows, so results do not depend on
// timing
template <typename T>
__global__ void __launch_bounds__(kAccKeys) accumulate_kernel(AccParams p) {
  __shared__ float sq[kAccRows][kMaxHeadDim], sl[kAccRows];
  const int b = blockIdx.x / p.kv_heads, h = blockIdx.x % p.kv_heads;
  const int32_t* path = p.path + (size_t)b * p.nodes;
  const int len = p.lens[b], count = p.count[b], D = p.head_dim;
  if (count == 0 || !fits(path, count, len, p.nodes, p.capacity)) return;
  const int total = len + count, rows = count * p.group;
  for (int base = blockIdx.y * kAccKeys; base < total; base += gridDim.y * kAccKeys) {
    const int s = base + threadIdx.x;
    float sum = 0.0f;
    for (int r0 = 0; r0 < rows; r0 += kAccRows) {
      __syncthreads();
      const int nr = min(kAccRows, rows - r0);
      for (int i = threadIdx.x; i < nr * D; i += kAccKeys) {
        const int row = r0 + i / D, node = path[row / p.group], qh = h * p.group + row % p.group;
        sq[i / D][i % D] = p.scale * kLog2e *
                           to_f32(static_cast<const T*>(p.q.data)[b * p.q.batch + qh * p.q.head + node * p.q.row + i % D]);
      }
      if (threadIdx.x < nr) {
        const int row = r0 + threadIdx.x, node = path[row / p.group], qh = h * p.group + row % p.group;
        sl[threadIdx.x] = kLog2e * p.lse[((size_t)b * p.nodes + node) * p.kv_heads * p.group + qh];
      }
      __syncthreads();
      if (s < total) {
        const T* k = static_cast<const T*>(p.kc.data) + b * p.kc.batch + h * p.kc.head + s * p.kc.row;
        float x[kAccRows];
#pragma unroll
        for (int r = 0; r < kAccRows; ++r) x[r] = 0.0f;
        for (int d = 0; d < D; ++d) {
          const float kd = to_f32(k[d]);
#pragma unroll
          for (int r = 0; r < kAccRows; ++r)
            if (r < nr) x[r] = fmaf(kd, sq[r][d], x[r]);
        }
#pragma unroll
        for (int r = 0; r < kAccRows; ++r)
          if (r < nr && s <= len + (r0 + r) / p.group) sum += exp2f(x[r] - sl[r]);
      }
    }
    if (s < total) {
      float* a = static_cast<float*>(p.acc.data) + b * p.acc.batch + h * p.acc.head + s;
      *a = s < len ? *a + sum : sum;
    }
  }
}

// Rows of whole, aligned 16-byte pieces.  The accepted rows (a few nodes times
// the query heads on a key/value head) are few, so this streams K once: a warp
// takes 16 keys at a time as the A operand of 16 x 8 matrix products.  Each
// lane copies the pieces that it will use itself into its own places of a ring
// in shared memory, ahead by the ring's steps and without any barrier: a
// larger register file for loads in flight.  The order of the products along head_dim is free as long as both operands have the same one:
// lane t of a quad reads the 16-byte pieces t, t + 4, ... of its two keys and
// uses each as two steps' elements, which the q rows in shared memory follow.
// The exponentials of a key lie in one quad, so its sum is two shuffles; a key's weights are
// added in a fixed order.
// 16 accepted rows over 65536 keys of 128 take 45.2 us, 84 % of the copy rate; 4
// over 4001 keys of 64, eight sequences, 12.1 us, where the chain of reads
// (lengths, accepted nodes, their rows) shows.
// A float32 element is three bfloat16 numbers of 8 bits each (cut, so their sum
// is the element), and a product of two elements eight of the nine products of
// these, to 2^-30 of it; sums are in 32 bits, the smaller products' apart from
// the largest ones'.  What is infinite or no number has no such parts: a score
// that is not finite is computed anew by `score_of`.
// (Two tensor-float parts and three products, to 2^-22, took 118 us where this
// takes 84: 16 rows over 30000 keys of 128, two sequences of 8 heads.)
template <typename T>
struct Pieces {
  struct Sums {
    float c[4];
    __device__ __forceinline__ float total(int e) const { return c[e]; }
  };
  __device__ __forceinline__ static void mac(Sums& s, const uint4& a, const uint4& b, const uint4& q) {
    mac(s.c, a, b, q);
  }
  // products of one pair of pieces (keys g and g + 8) with one q piece
  __device__ __forceinline__ static void mac(float* c, const uint4& a, const uint4& b, const uint4& q) {
    step(c, a.x, b.x, a.y, b.y, q.x, q.y);
    step(c, a.z, b.z, a.w, b.w, q.z, q.w);
  }
  __device__ __forceinline__ static void step(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                              uint32_t b1) {
    if constexpr (std::is_same_v<T, __nv_bfloat16>)
      asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
          : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
          : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
      asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
          : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
          : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};

template <>
struct Pieces<float> {
  struct Sums {
    float c[4], rest[4];
    __device__ __forceinline__ float total(int e) const { return c[e] + rest[e]; }
  };
  // four elements as pairs of their parts
  struct Parts {
    uint32_t p[3][2];
    __device__ __forceinline__ static uint32_t upper(float x) { return __float_as_uint(x) & 0xFFFF0000u; }
    __device__ __forceinline__ explicit Parts(const uint4& v) {
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float x = __uint_as_float(w[2 * k]), y = __uint_as_float(w[2 * k + 1]);
#pragma unroll
        for (int i = 0; i < 3; ++i) {
          p[i][k] = __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
          x -= __uint_as_float(upper(x));
          y -= __uint_as_float(upper(y));
        }
      }
    }
  };
  __device__ __forceinline__ static void mac(Sums& s, const uint4& a, const uint4& b, const uint4& q) {
    const Parts x(a), y(b), z(q);
    auto step = [&](float* c, int i, int j) {
      Pieces<__nv_bfloat16>::step(c, x.p[i][0], y.p[i][0], x.p[i][1], y.p[i][1], z.p[j][0], z.p[j][1]);
    };
    step(s.rest, 1, 2);
    step(s.rest, 2, 1);
    step(s.rest, 0, 2);
    step(s.rest, 2, 0);
    step(s.rest, 1, 1);
    step(s.rest, 0, 1);
    step(s.rest, 1, 0);
    step(s.c, 0, 0);
  }
};

// q . k in the order of the elements
template <typename T>
__device__ __noinline__ float score_of(const T* q, const T* k, int D) {
  float s = 0.0f;
  for (int d = 0; d < D; ++d) s = fmaf(to_f32(q[d]), to_f32(k[d]), s);
  return s;
}

constexpr int kStreamWarps = 8, kStreamRows = 64;  // warps of a CTA; q rows in shared memory at once

// 16-byte pieces of a key's row for each lane of its quad -> tiles of 16 keys a warp reads at once
constexpr int stream_tiles(int jc) { return jc <= 2 ? 2 : 1; }
// CTAs on an SM, and steps of the ring: 64 to 96 KB in flight in each
constexpr int stream_ctas(int jc) { return jc <= 4 ? 2 : 1; }
constexpr int stream_ring(int jc) { return jc <= 8 ? 3 : 1; }
constexpr size_t stream_ring_bytes(int jc) {
  return (size_t)stream_ring(jc) * kStreamWarps * 32 * 2 * jc * stream_tiles(jc) * 16;
}

__device__ __forceinline__ void copy16(uint4* dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src),
               "r"(real ? 16 : 0)
               : "memory");
}

// keys of sequence b that get weight: none where nothing is accepted
__device__ __forceinline__ int weighed_keys(const AccParams& p, int b) {
  const int len = p.lens[b], count = p.count[b];
  return count > 0 && fits(p.path + (size_t)b * p.nodes, count, len, p.nodes, p.capacity) ? len + count : 0;
}

// each > 0: CTA (x, y) takes `each` steps of head x from step y each on, if the
// head has that many.  Otherwise the CTAs divide the list of all heads' keys
// evenly (their number is known on the device only), in entries of one step:
// caches of unequal lengths then end together, but a CTA reads the whole
// batch's lengths first and may begin a second head.
template <typename T, int JC>
__global__ void __launch_bounds__(32 * kStreamWarps, stream_ctas(JC)) accumulate_stream_kernel(AccParams p, int each) {
  constexpr int W = 16 / sizeof(T), U = stream_tiles(JC), R = stream_ring(JC);
  constexpr int kWarpKeys = 16 * U, kStep = kStreamWarps * kWarpKeys;
  // the ring, [step][warp][piece of a key][lane], and q in the order of the
  // products, [8 rows][piece][lane]
  extern __shared__ __align__(16) uint4 s_ring[];
  uint4* const s_q = s_ring + stream_ring_bytes(JC) / 16;
  __shared__ float s_lse[kStreamRows];
  __shared__ int s_last[kStreamRows];  // the last key that a row sees; -1 for a row that is not there
  const int D = p.head_dim, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const float c2 = p.scale * kLog2e;
  auto entries_of = [&](int b) { return (weighed_keys(p, b) + kStep - 1) / kStep; };
  int w0 = 0, w1;
  ListPlace at;
  if (each > 0) {
    at.b = blockIdx.x / p.kv_heads, at.unit = blockIdx.x % p.kv_heads, at.entry = blockIdx.y * each;
    at.entries = entries_of(at.b);
    w1 = min(each, at.entries - at.entry);
  } else {
    int first;
    const int entries = list_sum(p.batch, entries_of, first) * p.kv_heads;
    w0 = list_start(entries, blockIdx.x, gridDim.x), w1 = list_start(entries, blockIdx.x + 1, gridDim.x);
    if (w0 < w1) at = list_find(p.batch, p.kv_heads, w0, first, entries_of);
  }
  if (w0 >= w1) return;
  for (int w = w0; w < w1;) {
    const int steps = min(at.entries - at.entry, w1 - w);
    const int b = at.b, h = at.unit, len = p.lens[b], count = p.count[b], total = len + count, rows = count * p.group;
    const int32_t* path = p.path + (size_t)b * p.nodes;
    const T* kc = static_cast<const T*>(p.kc.data) + b * p.kc.batch + h * p.kc.head;
    float* acc = static_cast<float*>(p.acc.data) + b * p.acc.batch + h * p.acc.head;
    for (int r0 = 0; r0 < rows; r0 += kStreamRows) {
      const int groups = (min(kStreamRows, rows - r0) + 7) / 8;
      // the lane's pieces of its keys in step i, into its places
      auto place = [&](int i, int u, int half, int j) {
        return s_ring + ((((i % R) * kStreamWarps + warp) * U + u) * 2 + half) * JC * 32 + j * 32 + lane;
      };
      auto fetch = [&](int i) {
        const int k0 = (at.entry + i) * kStep + warp * kWarpKeys + g;
        const T* key = kc + k0 * p.kc.row + t * W;
        const bool whole = i < steps && k0 + kWarpKeys - 8 < total;  // all of this lane's keys are there
#pragma unroll
        for (int u = 0; u < 2 * U; ++u, key += 8 * p.kc.row) {
          const bool there = whole || (i < steps && k0 + 8 * u < total);
#pragma unroll
          for (int j = 0; j < JC; ++j) {
            const bool real = there && (t + 4 * j) * W < D;
            copy16(place(i, u >> 1, u & 1, j), real ? key + 4 * j * W : kc, real);
          }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
#pragma unroll
      for (int i = 0; i < R; ++i) fetch(i);
      __syncthreads();
      for (int i = threadIdx.x; i < groups * JC * 32; i += 32 * kStreamWarps) {
        const int ln = i & 31, j = (i >> 5) % JC, row = r0 + (i >> 5) / JC * 8 + (ln >> 2), d = ((ln & 3) + 4 * j) * W;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (row < rows && d < D) {
          const int node = path[row / p.group], qh = h * p.group + row % p.group;
          v = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.q.data) + b * p.q.batch + qh * p.q.head +
                                              node * p.q.row + d);
        }
        s_q[i] = v;
      }
      if (threadIdx.x < kStreamRows) {
        const int row = r0 + threadIdx.x;
        // a row that is not there weighs nothing
        s_lse[threadIdx.x] = INFINITY;
        s_last[threadIdx.x] = row < rows ? len + row / p.group : -1;
        if (row < rows)
          s_lse[threadIdx.x] = kLog2e * p.lse[((size_t)b * p.nodes + path[row / p.group]) * p.kv_heads * p.group +
                                              h * p.group + row % p.group];
      }
      // the weights so far of the keys of step i whose sums this lane will write
      float soon[U][2];
      auto weights = [&](int i) {
        const int s0 = (at.entry + i) * kStep + warp * kWarpKeys + g, end = i < steps && t == 0 ? r0 > 0 ? total : len : 0;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int half = 0; half < 2; ++half)
            soon[u][half] = s0 + 16 * u + 8 * half < end ? acc[s0 + 16 * u + 8 * half] : 0.0f;
      };
      weights(0);
      __syncthreads();
      for (int i = 0; i < steps; ++i) {
        const int k0 = (at.entry + i) * kStep + warp * kWarpKeys;
        if (k0 >= total) break;
        asm volatile("cp.async.wait_group %0;" ::"n"(R - 1) : "memory");
        uint4 a[U][2][JC];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int j = 0; j < JC; ++j) a[u][half][j] = *place(i, u, half, j);
        fetch(i + R);
        float old[U][2], sum[U][2];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int half = 0; half < 2; ++half) old[u][half] = soon[u][half], sum[u][half] = 0.0f;
        weights(i + 1);
        for (int gr = 0; gr < groups; ++gr) {
          typename Pieces<T>::Sums sums[U] = {};
#pragma unroll
          for (int j = 0; j < JC; ++j) {
            const uint4 q = s_q[(gr * JC + j) * 32 + lane];
#pragma unroll
            for (int u = 0; u < U; ++u) Pieces<T>::mac(sums[u], a[u][0][j], a[u][1][j], q);
          }
          const int row = gr * 8 + 2 * t;  // the lane's two rows
          const float2 l = *reinterpret_cast<const float2*>(s_lse + row);
          const int2 last = *reinterpret_cast<const int2*>(s_last + row);
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int s = k0 + 16 * u + g;
            float c[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              c[e] = sums[u].total(e);
              if constexpr (std::is_same_v<T, float>) {
                const int key = s + (e < 2 ? 0 : 8), r = r0 + row + (e & 1);
                if (!(fabsf(c[e]) < INFINITY) && key <= (e & 1 ? last.y : last.x))
                  c[e] = score_of(static_cast<const T*>(p.q.data) + b * p.q.batch +
                                      (h * p.group + r % p.group) * p.q.head + path[r / p.group] * p.q.row,
                                  kc + key * p.kc.row, D);
              }
            }
            float e[4] = {ex2(fmaf(c[0], c2, -l.x)), ex2(fmaf(c[1], c2, -l.y)), ex2(fmaf(c[2], c2, -l.x)),
                          ex2(fmaf(c[3], c2, -l.y))};
            e[0] = s <= last.x ? e[0] : 0.0f;
            e[1] = s <= last.y ? e[1] : 0.0f;
            e[2] = s + 8 <= last.x ? e[2] : 0.0f;
            e[3] = s + 8 <= last.y ? e[3] : 0.0f;
            sum[u][0] += e[0] + e[1];
            sum[u][1] += e[2] + e[3];
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            float x = sum[u][half];
            x += __shfl_xor_sync(0xffffffffu, x, 1);
            x += __shfl_xor_sync(0xffffffffu, x, 2);
            const int s = k0 + 16 * u + g + 8 * half;
            if (t == 0 && s < total) acc[s] = old[u][half] + x;
          }
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory");  // before the ring is filled anew
    }
    w += steps;
    if (w >= w1) break;
    at.entry = 0;
    if (++at.unit == p.kv_heads) {
      at.unit = 0;
      do {
        at.entries = ++at.b < p.batch ? entries_of(at.b) : 1;
      } while (at.entries == 0);
    }
  }
}

// ---- evict ----------------------------------------------------------------------
struct EvictParams {
  ckks_rows kc, vc, acc, ko, vo, ao;
  const int32_t* lens;
  int32_t* index;
  int32_t* lens_out;
  int batch, kv_heads, head_dim, capacity, budget, recent;
};

// unsigned order of floats: larger weight, larger word; -0 equals 0, NaN is
// the smallest
__device__ __forceinline__ uint32_t order_of(float x) {
  if (isnan(x)) return 0u;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kSelThreads = 512, kSelWarps = kSelThreads / 32, kSelHeld = 16;

// exclusive prefix sums over the CTA's threads of two counts, and the sums;
// `scratch` holds 2 kSelWarps ints
__device__ __forceinline__ int2 counts_before(int gt, int eq, int* scratch, int2& all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int a = gt, b = eq;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, b, o);
    if (lane >= o) a += x, b += y;
  }
  __syncthreads();
  if (lane == 31) scratch[2 * warp] = a, scratch[2 * warp + 1] = b;
  __syncthreads();
  int2 before = make_int2(a - gt, b - eq);
  all = make_int2(0, 0);
#pragma unroll
  for (int w = 0; w < kSelWarps; ++w) {
    const int x = scratch[2 * w], y = scratch[2 * w + 1];
    if (w < warp) before.x += x, before.y += y;
    all.x += x, all.y += y;
  }
  return before;
}

// Cluster of C CTAs = (sequence, head): the rows to keep, in order.  Each CTA
// has a contiguous share of the weights in blocks of 16 for each thread; the
// first block stays in registers (a longer cache's others are read again in
// each pass), so that one read of the weights serves four passes over 8 bits
// that narrow the smallest weight kept down to its 32 bits: histograms in
// shared memory (one for every fourth lane, since most weights share their
// high bits), added across the cluster by each CTA from its neighbours'
// memory, and a suffix sum over the 256 bins by one warp.  Then the rows above
// that weight and the first of those at it are listed by prefix sums.  32 heads
// of 65536 weights take 22 us (one CTA a head took 130), 12 heads of 2100 about 8:
// four passes of barriers, not the bytes.
template <int C>
__global__ void __launch_bounds__(kSelThreads, 2) select_kernel(EvictParams p) {
  __shared__ int s_hist[4][256], s_total[256], s_scratch[2 * kSelWarps];
  __shared__ int s_digit, s_left, s_count[2];
  const unsigned rank = C > 1 ? blockIdx.x % C : 0;
  const int head = blockIdx.x / C, b = head / p.kv_heads, h = head % p.kv_heads;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int len = min(max(p.lens[b], 0), p.capacity);
  const int kept = min(len, p.budget), recent = min(p.recent, kept);
  const int older = len - recent, pick = kept - recent;
  const float* acc = static_cast<const float*>(p.acc.data) + b * p.acc.batch + h * p.acc.head;
  int32_t* index = p.index + (size_t)head * p.budget;
  const int all = C * kSelThreads, me = rank * kSelThreads + tid;  // of the cluster's threads
  if (h == 0 && me == 0) p.lens_out[b] = kept;
  for (int i = kept + me; i < p.budget; i += all) index[i] = -1;
  for (int i = me; i < recent; i += all) index[pick + i] = older + i;
  if (pick == 0 || pick == older) {  // alike in the whole cluster
    for (int i = me; i < pick; i += all) index[i] = i;
    return;
  }
  // this CTA's weights [lo, hi), whole blocks but for the last
  constexpr int kBlock = kSelThreads * kSelHeld;
  const int share = ((older + C - 1) / C + kSelHeld - 1) / kSelHeld * kSelHeld;
  const int lo = min(older, (int)rank * share), hi = min(older, lo + share), blocks = (hi - lo + kBlock - 1) / kBlock;
  const bool wide = reinterpret_cast<uintptr_t>(acc) % 16 == 0;  // lo is a multiple of 16
  auto read = [&](int block, uint32_t* u) {
    const int i0 = lo + block * kBlock + tid * kSelHeld;
    float x[kSelHeld];
    if (wide && i0 + kSelHeld <= hi) {
#pragma unroll
      for (int k = 0; k < kSelHeld; k += 4) *reinterpret_cast<float4*>(x + k) = *reinterpret_cast<const float4*>(acc + i0 + k);
    } else {
#pragma unroll
      for (int k = 0; k < kSelHeld; ++k) x[k] = i0 + k < hi ? acc[i0 + k] : 0.0f;
    }
#pragma unroll
    for (int k = 0; k < kSelHeld; ++k) u[k] = order_of(x[k]);
    return max(0, min(kSelHeld, hi - i0));  // those that are there
  };
  uint32_t held[kSelHeld];
  const int mine = read(0, held);
  uint32_t prefix = 0;
  int left = pick;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 4 * 256; i += kSelThreads) (&s_hist[0][0])[i] = 0;
    __syncthreads();
    auto add = [&](const uint32_t* u, int n) {
#pragma unroll
      for (int k = 0; k < kSelHeld; ++k)
        if (k < n && (shift == 24 || u[k] >> (shift + 8) == prefix >> (shift + 8)))
          atomicAdd(&s_hist[lane & 3][u[k] >> shift & 255], 1);
    };
    add(held, mine);
    for (int k = 1; k < blocks; ++k) {
      uint32_t u[kSelHeld];
      const int n = read(k, u);
      add(u, n);
    }
    __syncthreads();
    if (tid < 256) s_total[tid] = s_hist[0][tid] + s_hist[1][tid] + s_hist[2][tid] + s_hist[3][tid];
    if constexpr (C > 1) {
      cluster_sync();
      if (tid < 256) {
        int n = 0;
#pragma unroll
        for (int r = 0; r < C; ++r) n += cluster_read(&s_total[tid], r);
        s_hist[0][tid] = n;
      }
    } else if (tid < 256) {
      s_hist[0][tid] = s_total[tid];
    }
    __syncthreads();
    if (warp == 0) {
      // the highest digits first: lane 0 has bins 255 .. 248
      int n[8], sum = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) sum += n[k] = s_hist[0][255 - 8 * lane - k];
      int upto = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
      }
      const uint32_t past = __ballot_sync(0xffffffffu, upto >= left);
      if (lane == __ffs(past) - 1) {
        int above = upto - sum, k = 0;
        while (k < 7 && above + n[k] < left) above += n[k++];
        s_digit = 255 - 8 * lane - k;
        s_left = left - above;
      }
    }
    __syncthreads();
    prefix |= (uint32_t)s_digit << shift;
    left = s_left;
    // the neighbours have read this CTA's counts before they are written again
    if constexpr (C > 1) cluster_sync();
  }
  // `left` rows at the edge weight are kept, the first ones
  const uint32_t edge = prefix;
  auto count = [&](const uint32_t* u, int n, int& gt, int& eq) {
#pragma unroll
    for (int k = 0; k < kSelHeld; ++k) {
      gt += k < n && u[k] > edge;
      eq += k < n && u[k] == edge;
    }
  };
  int gt = 0, eq = 0;
  count(held, mine, gt, eq);
  int2 sum;
  int2 before = counts_before(gt, eq, s_scratch, sum);
  int above = 0, at_edge = 0;  // of the CTAs before this one
  if constexpr (C > 1) {
    int g2 = 0, e2 = 0;
    for (int k = 1; k < blocks; ++k) {
      uint32_t u[kSelHeld];
      const int n = read(k, u);
      count(u, n, g2, e2);
    }
    int2 more = make_int2(0, 0);
    if (blocks > 1) counts_before(g2, e2, s_scratch, more);
    if (tid == 0) s_count[0] = sum.x + more.x, s_count[1] = sum.y + more.y;
    cluster_sync();
#pragma unroll
    for (int r = 0; r < C; ++r)
      if (r < (int)rank) {
        above += cluster_read(&s_count[0], r);
        at_edge += cluster_read(&s_count[1], r);
      }
  }
  auto list = [&](const uint32_t* u, int n, int i0) {
    int bg = above + before.x, be = at_edge + before.y;
#pragma unroll
    for (int k = 0; k < kSelHeld; ++k) {
      const bool is_gt = k < n && u[k] > edge, is_eq = k < n && u[k] == edge;
      if (is_gt || (is_eq && be < left)) index[bg + min(be, left)] = i0 + k;
      bg += is_gt;
      be += is_eq;
    }
    above += sum.x;
    at_edge += sum.y;
  };
  list(held, mine, lo + tid * kSelHeld);
  for (int k = 1; k < blocks; ++k) {
    uint32_t u[kSelHeld];
    const int n = read(k, u);
    gt = eq = 0;
    count(u, n, gt, eq);
    before = counts_before(gt, eq, s_scratch, sum);
    list(u, n, lo + k * kBlock + tid * kSelHeld);
  }
  if constexpr (C > 1) cluster_sync();  // no CTA ends while another may read its counts
}

// copies the rows listed in index and their weights, rows in pieces of V
// elements, at the copy rate (537 MB in 85 us): CTA.x = (sequence
// x head), CTA.y strides over the budget
template <typename T, typename V>
__global__ void __launch_bounds__(256) gather_kernel(EvictParams p) {
  constexpr int W = sizeof(V) / sizeof(T);
  CKKS_PDL_ENTRY();
  const int b = blockIdx.x / p.kv_heads, h = blockIdx.x % p.kv_heads;
  const int kept = min(min(max(p.lens[b], 0), p.capacity), p.budget);
  const int per = p.head_dim / W;
  const int32_t* index = p.index + (size_t)blockIdx.x * p.budget;
  const T* kc = static_cast<const T*>(p.kc.data) + b * p.kc.batch + h * p.kc.head;
  const T* vc = static_cast<const T*>(p.vc.data) + b * p.vc.batch + h * p.vc.head;
  const float* acc = static_cast<const float*>(p.acc.data) + b * p.acc.batch + h * p.acc.head;
  float* ao = static_cast<float*>(p.ao.data) + b * p.ao.batch + h * p.ao.head;
  T* ko = static_cast<T*>(p.ko.data) + b * p.ko.batch + h * p.ko.head;
  T* vo = static_cast<T*>(p.vo.data) + b * p.vo.batch + h * p.vo.head;
  const long long n = (long long)kept * per;
  for (long long i = (long long)blockIdx.y * blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.y * blockDim.x) {
    const int r = (int)(i / per), d = (int)(i % per) * W, s = index[r];
    if (d == 0) ao[r] = acc[s];
    const V k = *reinterpret_cast<const V*>(kc + s * p.kc.row + d);
    const V v = *reinterpret_cast<const V*>(vc + s * p.vc.row + d);
    *reinterpret_cast<V*>(ko + r * p.ko.row + d) = k;
    *reinterpret_cast<V*>(vo + r * p.vo.row + d) = v;
  }
}

template <typename T, int JC>
void launch_stream(const Context& c, const AccParams& p, cudaStream_t st) {
  constexpr int kKeys = kStreamWarps * 16 * stream_tiles(JC);  // of one entry
  const long long heads = (long long)p.batch * p.kv_heads, steps = (p.capacity + kKeys - 1) / kKeys;
  const long long entries = heads * steps, ctas = (long long)stream_ctas(JC) * c.sms;
  // By heads: one wave when the caches are three quarters full (12 heads of 8
  // sequences over 4001 keys took 18.9 / 13.9 / 17.5 us with 3 / 4 / 6 steps
  // each).  As a list where a CTA's share is long against what the heads that
  // it begins cost, about 16 steps each: by heads / as a list, 12 heads over
  // 4001 keys 10.8 / 12.5 us with 8 sequences, over 8000 keys 30.3 / 43.7 with
  // 16, 8 wider heads over 65536 keys 61.1 / 44.4 with 2.
  const int each = (int)((3 * entries + 4 * ctas - 1) / (4 * ctas));
  const bool by_head = entries < 16 * (heads + ctas);
  const dim3 grid = by_head ? dim3((unsigned)heads, (unsigned)((steps + each - 1) / each))
                            : dim3((unsigned)std::min(entries, ctas));
  const size_t smem = stream_ring_bytes(JC) + (size_t)(std::min(kStreamRows, p.nodes * p.group) + 7) / 8 * JC * 512;
  constexpr size_t most = stream_ring_bytes(JC) + kStreamRows / 8 * JC * 512;
  static_assert(stream_ctas(JC) * (most + 2048) <= 228 << 10, "fits an SM");
  auto* k = accumulate_stream_kernel<T, JC>;
  // the most that any call asks for: calls of other sizes from other threads
  // may come between this and the launch
  CKKS_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most));
  k<<<grid, 32 * kStreamWarps, smem, st>>>(p, by_head ? each : 0);
  CKKS_CUDA(cudaGetLastError());
}

template <typename T>
void run_stream(const Context& c, const AccParams& p, cudaStream_t st) {
  const int pieces = (p.head_dim * (int)sizeof(T) / 16 + 3) / 4;
  if (pieces <= 2)
    launch_stream<T, 2>(c, p, st);
  else if (pieces <= 4)
    launch_stream<T, 4>(c, p, st);
  else if (sizeof(T) == 2 || pieces <= 8)
    launch_stream<T, 8>(c, p, st);
  else if constexpr (sizeof(T) == 4)
    launch_stream<T, 16>(c, p, st);
}

void check_cache(int dtype, int batch, int kv_heads, int head_dim, int capacity) {
  need(dtype == CKKS_BF16 || dtype == CKKS_FP16 || dtype == CKKS_FP32,
       "caches are CKKS_BF16, CKKS_FP16 or CKKS_FP32");
  need(batch >= 0 && capacity >= 0, "negative batch or capacity");
  need(kv_heads >= 1 && kv_heads <= 65535, "key/value head count out of range");
  need(head_dim >= 1 && head_dim <= kMaxHeadDim, "head_dim outside 1..256");
  need((long long)batch * kv_heads * (capacity / 128 + 1) < (1ll << 31) - 1 && capacity < (1 << 30), "sizes too large");
}

bool disjoint(const void* a0, const void* a1, const void* b0, const void* b1) { return a1 <= b0 || b1 <= a0; }

// rows as 16-byte pieces, or as single elements of a type of their size
template <typename F>
void by_piece(int bytes, bool wide, F&& f) {
  if (bytes == 2)
    wide ? f(uint16_t{}, uint4{}) : f(uint16_t{}, uint16_t{});
  else
    wide ? f(uint32_t{}, uint4{}) : f(uint32_t{}, uint32_t{});
}

}  // namespace
}  // namespace draft
}  // namespace ckks

using namespace ckks;
using namespace ckks::draft;

extern "C" int ckks_draft_commit(ckks_ctx* ctx, const ckks_draft_commit_args* args, void* stream) {
  return guard([&] {
    Context& c = context_of(ctx);
    need(args != nullptr, "null argument");
    const ckks_draft_commit_args& a = *args;
    check_cache(a.dtype, a.batch, a.kv_heads, a.head_dim, a.capacity);
    need(a.nodes >= 1 && a.nodes <= kMaxNodes, "node count outside 1..64");
    if (a.batch == 0) return;
    const int e = element_bytes(a.dtype);
    if (a.capacity) {
      check_rows(a.k_cache, e, "k_cache");
      check_rows(a.v_cache, e, "v_cache");
    }
    check_rows(a.k_new, e, "k_new");
    check_rows(a.v_new, e, "v_new");
    check_ptr(a.lens, "lens");
    check_ptr(a.path, "path");
    check_ptr(a.count, "count");
    check_ptr(a.lens_out, "lens_out");
    need(disjoint(a.lens, a.lens + a.batch, a.lens_out, a.lens_out + a.batch), "lens_out overlaps lens");
    if (a.capacity)
      for (const ckks_rows* cache : {&a.k_cache, &a.v_cache})
        for (const ckks_rows* fresh : {&a.k_new, &a.v_new})
          need(disjoint(cache->data, end_of(*cache, a.batch, a.kv_heads, a.capacity, a.head_dim, e), fresh->data,
                        end_of(*fresh, a.batch, a.kv_heads, a.nodes, a.head_dim, e)),
               "new rows overlap the cache");
    CommitParams p{a.k_cache, a.v_cache,  a.k_new,    a.v_new, a.lens,    a.path, a.count, a.lens_out,
                   c.d_faults + 1, a.batch, a.kv_heads, a.head_dim, a.nodes, a.capacity};
    const bool wide = a.capacity && wide_rows(a.k_cache, a.batch, a.kv_heads, a.capacity, a.head_dim, e) &&
                      wide_rows(a.v_cache, a.batch, a.kv_heads, a.capacity, a.head_dim, e) &&
                      wide_rows(a.k_new, a.batch, a.kv_heads, a.nodes, a.head_dim, e) &&
                      wide_rows(a.v_new, a.batch, a.kv_heads, a.nodes, a.head_dim, e);
    OnDevice dev(c);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    ProfScope ps(c, "draft_commit", 4.0 * e * a.batch * a.kv_heads * a.nodes * a.head_dim, st);
    by_piece(e, wide, [&](auto t, auto v) {
      commit_kernel<decltype(t), decltype(v)><<<dim3(a.batch, a.kv_heads), 128, 0, st>>>(p);
    });
    CKKS_CUDA(cudaGetLastError());
  });
}

extern "C" int ckks_draft_accumulate(ckks_ctx* ctx, const ckks_draft_accumulate_args* args, void* stream) {
  return guard([&] {
    Context& c = context_of(ctx);
    need(args != nullptr, "null argument");
    const ckks_draft_accumulate_args& a = *args;
    check_cache(a.dtype, a.batch, a.kv_heads, a.head_dim, a.capacity);
    need(a.nodes >= 1 && a.nodes <= kMaxNodes, "node count outside 1..64");
    need(a.q_heads >= 1 && a.q_heads % a.kv_heads == 0, "query heads are not a multiple of the key/value heads");
    need(a.reserved == 0, "reserved field is not 0");
    need(std::isfinite((float)a.scale * kLog2e), "scale is not finite");
    if (a.batch == 0 || a.capacity == 0) return;
    const int e = element_bytes(a.dtype);
    check_rows(a.q, e, "q");
    check_rows(a.k_cache, e, "k_cache");
    check_rows(a.acc, 4, "acc");
    check_ptr(a.lse, "lse");
    check_ptr(a.lens, "lens");
    check_ptr(a.path, "path");
    check_ptr(a.count, "count");
    AccParams p{a.q,     a.k_cache, a.acc,     a.lse, a.lens, a.path, a.count, a.batch, a.kv_heads, a.q_heads / a.kv_heads,
                a.head_dim, a.nodes, a.capacity, (float)a.scale};
    OnDevice dev(c);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    ProfScope ps(c, "draft_accumulate", (double)e * a.batch * a.kv_heads * a.capacity * a.head_dim, st);
    if (wide_rows(a.q, a.batch, a.q_heads, a.nodes, a.head_dim, e) &&
        wide_rows(a.k_cache, a.batch, a.kv_heads, a.capacity, a.head_dim, e)) {
      if (a.dtype == CKKS_BF16)
        run_stream<__nv_bfloat16>(c, p, st);
      else if (a.dtype == CKKS_FP16)
        run_stream<__half>(c, p, st);
      else
        run_stream<float>(c, p, st);
      return;
    }
    const dim3 grid((unsigned)(a.batch * a.kv_heads), (unsigned)std::min(65535, (a.capacity + kAccKeys - 1) / kAccKeys));
    if (a.dtype == CKKS_BF16)
      accumulate_kernel<__nv_bfloat16><<<grid, kAccKeys, 0, st>>>(p);
    else if (a.dtype == CKKS_FP16)
      accumulate_kernel<__half><<<grid, kAccKeys, 0, st>>>(p);
    else
      accumulate_kernel<float><<<grid, kAccKeys, 0, st>>>(p);
    CKKS_CUDA(cudaGetLastError());
  });
}

namespace {
void check_evict(const ckks_draft_evict_args& a) {
  check_cache(a.dtype, a.batch, a.kv_heads, a.head_dim, a.capacity);
  need(a.budget >= 1 && a.recent >= 0 && a.recent <= a.budget, "need budget >= 1 and 0 <= recent <= budget");
  need(a.out_capacity >= a.budget && a.out_capacity < (1 << 30), "output capacity below the budget");
}
}  // namespace

extern "C" long long ckks_draft_evict_workspace(ckks_ctx* ctx, const ckks_draft_evict_args* args) {
  long long n = -1;
  guard([&] {
    context_of(ctx);
    need(args != nullptr, "null argument");
    check_evict(*args);
    n = 0;
  });
  return n;
}

extern "C" int ckks_draft_evict(ckks_ctx* ctx, const ckks_draft_evict_args* args, void* stream) {
  return guard([&] {
    Context& c = context_of(ctx);
    need(args != nullptr, "null argument");
    const ckks_draft_evict_args& a = *args;
    check_evict(a);
    if (a.batch == 0) return;
    const int e = element_bytes(a.dtype);
    check_rows(a.k_out, e, "k_out");
    check_rows(a.v_out, e, "v_out");
    check_rows(a.acc_out, 4, "acc_out");
    check_ptr(a.lens, "lens");
    check_ptr(a.index, "index");
    check_ptr(a.lens_out, "lens_out");
    need(disjoint(a.lens, a.lens + a.batch, a.lens_out, a.lens_out + a.batch), "lens_out overlaps lens");
    if (a.capacity) {
      check_rows(a.k_cache, e, "k_cache");
      check_rows(a.v_cache, e, "v_cache");
      check_rows(a.acc, 4, "acc");
      const ckks_rows ins[3] = {a.k_cache, a.v_cache, a.acc}, outs[3] = {a.k_out, a.v_out, a.acc_out};
      for (int i = 0; i < 3; ++i)
        for (int o = 0; o < 3; ++o) {
          auto end = [&](const ckks_rows& r, int k, int rows) {
            ckks_rows x = r;
            if (k == 2) x.row = 1;
            return end_of(x, a.batch, a.kv_heads, rows, k == 2 ? 1 : a.head_dim, k == 2 ? 4 : e);
          };
          need(disjoint(ins[i].data, end(ins[i], i, a.capacity), outs[o].data, end(outs[o], o, a.budget)),
               "output overlaps input");
        }
    }
    EvictParams p{a.k_cache, a.v_cache, a.acc,      a.k_out,    a.v_out,    a.acc_out, a.lens, a.index,
                  a.lens_out, a.batch,  a.kv_heads, a.head_dim, a.capacity, a.budget,  a.recent};
    const bool wide = wide_rows(a.k_out, a.batch, a.kv_heads, a.budget, a.head_dim, e) &&
                      wide_rows(a.v_out, a.batch, a.kv_heads, a.budget, a.head_dim, e) &&
                      (a.capacity == 0 || (wide_rows(a.k_cache, a.batch, a.kv_heads, a.capacity, a.head_dim, e) &&
                                           wide_rows(a.v_cache, a.batch, a.kv_heads, a.capacity, a.head_dim, e)));
    OnDevice dev(c);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int heads = a.batch * a.kv_heads;
    ProfScope ps(c, "draft_evict", heads * (4.0 * a.capacity + a.budget * (4.0 * e * a.head_dim + 8.0)), st);
    // a CTA for each 4096 weights, eight at most
    if (a.capacity <= 4096)
      launch_cluster<1>(select_kernel<1>, heads, kSelThreads, st, p);
    else if (a.capacity <= 8192)
      launch_cluster<2>(select_kernel<2>, heads, kSelThreads, st, p);
    else if (a.capacity <= 16384)
      launch_cluster<4>(select_kernel<4>, heads, kSelThreads, st, p);
    else
      launch_cluster<8>(select_kernel<8>, heads, kSelThreads, st, p);
    by_piece(e, wide, [&](auto t, auto v) {
      const long long pieces = (long long)a.budget * a.head_dim * e / (long long)sizeof(v);
      const long long most = std::max(1ll, 16ll * c.sms / heads);
      const unsigned y = (unsigned)std::min({(pieces + 255) / 256, most, 65535ll});
      launch_pdl(gather_kernel<decltype(t), decltype(v)>, dim3(heads, y), dim3(256), 0, st, p);
    });
  });
}
