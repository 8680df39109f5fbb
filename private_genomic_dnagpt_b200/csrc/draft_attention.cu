// draft_attention.cu -- attention of a tree of drafted nodes over a
// key/value cache (ckks_draft_attention): the data owner's draft model reads
// its cache once for all nodes of a tree.
//
// For the rows r = (node, query head) of one key/value head,
//   s_rk = scale q_r . k_k,  out_r = sum_k exp(s_rk - m_r) v_k / l_r,
//   m_r = max_k s_rk,  l_r = sum_k exp(s_rk - m_r),  lse_r = m_r + ln l_r,
// over the cached keys k < len and the new keys of r's node and its
// ancestors.  Each cached key is read once for all rows, so the floor is the
// cache's bytes.  A sequence's keys are split over CTAs that each keep
// (m, l, sum) of their part; a second kernel joins the parts.
#include <algorithm>
#include <cmath>

#include "draft.hpp"

namespace ckks {
namespace draft {
namespace {

struct AttnParams {
  ckks_rows q, kc, vc, kn, vn, out;
  const int32_t* lens;
  const int32_t* parents;
  float* lse;
  float* part;  // [batch * kv_heads][splits][rows][head_dim + 2]
  int batch, kv_heads, group, head_dim, nodes, capacity, splits;
  float scale;
  bool wide;  // every row is whole, aligned 16-byte pieces
};

__device__ __forceinline__ int length_of(const AttnParams& p, int b) { return min(max(p.lens[b], 0), p.capacity); }

// natural exponent through the base-2 one: scores are kept times log2(e)
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// writes one finished row: node i, query head h
template <typename T>
__device__ __forceinline__ T* out_row(const AttnParams& p, int b, int node, int qh) {
  return static_cast<T*>(p.out.data) + b * p.out.batch + qh * p.out.head + node * p.out.row;
}

// ---- every type, size and stride: CUDA cores ----------------------------------
// A CTA of 128 threads takes 8 rows of one key/value head and one split of
// the keys, in tiles of 64 keys staged in shared memory as floats.  Scores:
// a thread has one key and 4 rows, so a key element from shared memory feeds
// 4 multiply-adds and the query elements are broadcasts.  Values: 16 threads
// across head_dim (4 elements each, looping over larger ones), 8 across the
// keys of the tile, each with the sums of all 8 rows in registers; the 8
// partial sums meet once, at the end.  Products and sums are in 32 bits.
constexpr int kRows = 8, kTile = 64, kThreads = 128;

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

// DC: chunks of 64 elements that cover head_dim
template <typename T, int DC>
__global__ void __launch_bounds__(kThreads) attend_kernel(AttnParams p) {
  extern __shared__ __align__(16) float sm[];
  const int D = p.head_dim, D4 = (D + 3) & ~3, KS = D4 + 4;  // row stride of the keys: 16-byte reads without conflicts
  float* sk = sm;                       // [kTile][KS]
  float* sv = sk + kTile * KS;          // [kTile][D4]
  float* sq = sv + kTile * D4;          // [kRows][D4]
  float* sp = sq + kRows * D4;          // [kTile][kRows]
  __shared__ float s_m[kRows], s_l[kRows], s_c[kRows];
  __shared__ uint64_t s_mask[kMaxNodes];
  __shared__ int s_jump[kMaxNodes];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rows = p.nodes * p.group, tiles_r = (rows + kRows - 1) / kRows;
  const int rt = blockIdx.x % tiles_r, bh = blockIdx.x / tiles_r;
  const int b = bh / p.kv_heads, h = bh % p.kv_heads;
  const int len = length_of(p, b), total = len + p.nodes;
  // this split's keys [k0, k1) of the cached and then the new ones
  const int per = ((total + p.splits - 1) / p.splits + kTile - 1) / kTile * kTile;
  const int k0 = min(total, (int)blockIdx.y * per), k1 = min(total, k0 + per);
  if (warp == 0) tree_masks(p.parents + (size_t)b * p.nodes, p.nodes, s_mask, s_jump);
  for (int i = tid; i < kRows * (D4 / 4); i += kThreads) {
    const int r = i / (D4 / 4), d = i % (D4 / 4) * 4, row = rt * kRows + r;
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    if (row < rows) {
      const T* src = static_cast<const T*>(p.q.data) + b * p.q.batch + (h * p.group + row % p.group) * p.q.head +
                     (row / p.group) * p.q.row;
      load_row4(x, src, d, D, p.wide);
    }
    for (int k = 0; k < 4; ++k) sq[r * D4 + d + k] = x[k] * (p.scale * kLog2e);
  }
  if (tid < kRows) {
    s_m[tid] = -INFINITY;
    s_l[tid] = 0.0f;
  }
  float acc[DC][kRows][4];
#pragma unroll
  for (int c = 0; c < DC; ++c)
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[c][r][e] = 0.0f;
  __syncthreads();
  const int key = tid & 63, rh = tid >> 6;  // scores: this thread's key of the tile and rows 4 rh .. 4 rh + 3
  const int dg = tid & 15, kg = tid >> 4;   // values: this thread's elements and every eighth key
  const T* kc = static_cast<const T*>(p.kc.data) + b * p.kc.batch + h * p.kc.head;
  const T* vc = static_cast<const T*>(p.vc.data) + b * p.vc.batch + h * p.vc.head;
  const T* kn = static_cast<const T*>(p.kn.data) + b * p.kn.batch + h * p.kn.head;
  const T* vn = static_cast<const T*>(p.vn.data) + b * p.vn.batch + h * p.vn.head;
  for (int t0 = k0; t0 < k1; t0 += kTile) {
    const int nk = min(kTile, k1 - t0);
    for (int i = tid; i < kTile * (D4 / 4); i += kThreads) {
      const int r = i / (D4 / 4), d = i % (D4 / 4) * 4, s = t0 + r;
      float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
      if (r < nk) {
        if (s < len) {
          load_row4(x, kc + s * p.kc.row, d, D, p.wide);
          load_row4(y, vc + s * p.vc.row, d, D, p.wide);
        } else if (s_mask[s - len]) {
          load_row4(x, kn + (s - len) * p.kn.row, d, D, p.wide);
          load_row4(y, vn + (s - len) * p.vn.row, d, D, p.wide);
        }
      }
      *reinterpret_cast<float4*>(sk + r * KS + d) = make_float4(x[0], x[1], x[2], x[3]);
      *reinterpret_cast<float4*>(sv + r * D4 + d) = make_float4(y[0], y[1], y[2], y[3]);
    }
    __syncthreads();
    {
      float s[4] = {0.f, 0.f, 0.f, 0.f};
      for (int d = 0; d < D4; d += 4) {
        const float4 k4 = *reinterpret_cast<const float4*>(sk + key * KS + d);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float4 q4 = *reinterpret_cast<const float4*>(sq + (4 * rh + r) * D4 + d);
          s[r] = fmaf(k4.x, q4.x, fmaf(k4.y, q4.y, fmaf(k4.z, q4.z, fmaf(k4.w, q4.w, s[r]))));
        }
      }
      const int at = t0 + key;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = rt * kRows + 4 * rh + r;
        const uint64_t m = row < rows ? s_mask[row / p.group] : 0ull;
        const bool sees = key < nk && m && (at < len || (m >> (at - len) & 1));
        if (!sees) s[r] = -INFINITY;
      }
      *reinterpret_cast<float4*>(sp + key * kRows + 4 * rh) = make_float4(s[0], s[1], s[2], s[3]);
    }
    __syncthreads();
    // running maximum and sum: warp w has rows 2 w and 2 w + 1
#pragma unroll
    for (int r = 2 * warp; r < 2 * warp + 2; ++r) {
      const float a = sp[lane * kRows + r], c = sp[(lane + 32) * kRows + r];
      float mx = fmaxf(a, c);
#pragma unroll
      for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      const float old = s_m[r], m = fmaxf(old, mx);
      // a row that has seen nothing yet keeps weight 0
      const float base = m == -INFINITY ? 0.0f : m;
      const float ea = exp2f(a - base), ec = exp2f(c - base), f = exp2f(old - base);
      float sum = ea + ec;
#pragma unroll
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      sp[lane * kRows + r] = ea;
      sp[(lane + 32) * kRows + r] = ec;
      if (lane == 0) {
        s_m[r] = m;
        s_l[r] = s_l[r] * f + sum;
        s_c[r] = f;
      }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const float f = s_c[r];
#pragma unroll
      for (int c = 0; c < DC; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[c][r][e] *= f;
    }
    for (int k = kg; k < nk; k += 8) {
      const float4 p0 = *reinterpret_cast<const float4*>(sp + k * kRows);
      const float4 p1 = *reinterpret_cast<const float4*>(sp + k * kRows + 4);
      const float w[kRows] = {p0.x, p0.y, p0.z, p0.w, p1.x, p1.y, p1.z, p1.w};
#pragma unroll
      for (int c = 0; c < DC; ++c) {
        const int d = c * 64 + dg * 4;
        if (d >= D4) continue;
        const float4 v4 = *reinterpret_cast<const float4*>(sv + k * D4 + d);
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          // a weight of 0 adds nothing, whatever a value that other rows see holds
          const float x = w[r];
          if (x != 0.0f) {
            acc[c][r][0] = fmaf(x, v4.x, acc[c][r][0]);
            acc[c][r][1] = fmaf(x, v4.y, acc[c][r][1]);
            acc[c][r][2] = fmaf(x, v4.z, acc[c][r][2]);
            acc[c][r][3] = fmaf(x, v4.w, acc[c][r][3]);
          }
        }
      }
    }
    __syncthreads();
  }
  // the eight key groups' sums meet in shared memory, one chunk of 64 elements at a time
  float* red = sm;  // [8][kRows][64]
#pragma unroll
  for (int c = 0; c < DC; ++c) {
#pragma unroll
    for (int r = 0; r < kRows; ++r)
      *reinterpret_cast<float4*>(red + (kg * kRows + r) * 64 + dg * 4) =
          make_float4(acc[c][r][0], acc[c][r][1], acc[c][r][2], acc[c][r][3]);
    __syncthreads();
    for (int i = tid; i < kRows * 64; i += kThreads) {
      const int r = i / 64, d = c * 64 + i % 64, row = rt * kRows + r;
      if (row >= rows || d >= D) continue;
      float x = 0.0f;
#pragma unroll
      for (int g = 0; g < 8; ++g) x += red[(g * kRows + r) * 64 + i % 64];
      if (p.splits > 1) {
        p.part[(((size_t)bh * p.splits + blockIdx.y) * rows + row) * (D + 2) + d] = x;
      } else {
        const float l = s_l[r];
        out_row<T>(p, b, row / p.group, h * p.group + row % p.group)[d] = from_f32<T>(l != 0.0f ? x / l : 0.0f);
      }
    }
    __syncthreads();
  }
  if (tid < kRows && rt * kRows + tid < rows) {
    const int row = rt * kRows + tid;
    if (p.splits > 1) {
      float* o = p.part + (((size_t)bh * p.splits + blockIdx.y) * rows + row) * (D + 2) + D;
      o[0] = s_m[tid];
      o[1] = s_l[tid];
    } else {
      p.lse[((size_t)b * p.nodes + row / p.group) * p.kv_heads * p.group + h * p.group + row % p.group] =
          s_l[tid] != 0.0f ? kLn2 * (s_m[tid] + log2f(s_l[tid])) : -INFINITY;
    }
  }
}

// joins the splits of one row: CTA = (batch x kv head, row)
template <typename T>
__global__ void __launch_bounds__(kThreads) join_kernel(AttnParams p) {
  const int rows = p.nodes * p.group, D = p.head_dim;
  const int row = blockIdx.x % rows, bh = blockIdx.x / rows;
  const int b = bh / p.kv_heads, h = bh % p.kv_heads;
  const float* part = p.part + ((size_t)bh * p.splits * rows + row) * (D + 2);
  const size_t step = (size_t)rows * (D + 2);
  float m = -INFINITY;
  for (int s = 0; s < p.splits; ++s) m = fmaxf(m, part[s * step + D]);
  const float base = m == -INFINITY ? 0.0f : m;
  float l = 0.0f;
  for (int s = 0; s < p.splits; ++s) l = fmaf(part[s * step + D + 1], exp2f(part[s * step + D] - base), l);
  const int qh = h * p.group + row % p.group, node = row / p.group;
  T* o = out_row<T>(p, b, node, qh);
  for (int d = threadIdx.x; d < D; d += kThreads) {
    float x = 0.0f;
    for (int s = 0; s < p.splits; ++s) x = fmaf(part[s * step + d], exp2f(part[s * step + D] - base), x);
    o[d] = from_f32<T>(l != 0.0f ? x / l : 0.0f);
  }
  if (threadIdx.x == 0)
    p.lse[((size_t)b * p.nodes + node) * p.kv_heads * p.group + qh] = l != 0.0f ? kLn2 * (m + log2f(l)) : -INFINITY;
}

size_t attend_smem(int D) {
  const int D4 = (D + 3) & ~3;
  const size_t run = sizeof(float) * ((size_t)kTile * (D4 + 4) + kTile * D4 + kRows * D4 + kTile * kRows);
  const size_t red = sizeof(float) * 8 * kRows * 64;
  return run > red ? run : red;
}

template <typename T, int DC>
void launch_attend(const AttnParams& p, cudaStream_t st) {
  const size_t smem = attend_smem(p.head_dim);
  auto* k = attend_kernel<T, DC>;
  CKKS_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  const int rows = p.nodes * p.group;
  const dim3 grid((unsigned)(p.batch * p.kv_heads * ((rows + kRows - 1) / kRows)), p.splits);
  k<<<grid, kThreads, smem, st>>>(p);
  CKKS_CUDA(cudaGetLastError());
}

template <typename T>
void run_attend(const AttnParams& p, cudaStream_t st) {
  switch ((p.head_dim + 63) / 64) {
    case 1: launch_attend<T, 1>(p, st); break;
    case 2: launch_attend<T, 2>(p, st); break;
    case 3: launch_attend<T, 3>(p, st); break;
    default: launch_attend<T, 4>(p, st); break;
  }
  if (p.splits > 1) {
    join_kernel<T><<<(unsigned)(p.batch * p.kv_heads * p.nodes * p.group), kThreads, 0, st>>>(p);
    CKKS_CUDA(cudaGetLastError());
  }
}

// splits of a sequence's keys: enough CTAs for four on each SM, none with
// less than two tiles of keys at the full capacity
int split_count(const Context& c, const ckks_draft_attention_args& a) {
  const long long rows = (long long)a.nodes * (a.q_heads / a.kv_heads);
  const long long ctas = (long long)a.batch * a.kv_heads * ((rows + kRows - 1) / kRows);
  const long long tiles = ((long long)a.capacity + a.nodes + kTile - 1) / kTile;
  const long long want = (4ll * c.sms + ctas - 1) / ctas, most = (tiles + 1) / 2;
  return (int)std::max(1ll, std::min({want, most, 64ll}));
}

void check_shape(const ckks_draft_attention_args& a) {
  need(a.dtype == CKKS_BF16 || a.dtype == CKKS_FP16 || a.dtype == CKKS_FP32,
       "attention takes CKKS_BF16, CKKS_FP16 or CKKS_FP32");
  need(a.batch >= 0 && a.capacity >= 0, "negative batch or capacity");
  need(a.nodes >= 1 && a.nodes <= kMaxNodes, "node count outside 1..64");
  need(a.kv_heads >= 1 && a.q_heads >= 1 && a.q_heads % a.kv_heads == 0,
       "query heads are not a multiple of the key/value heads");
  need(a.head_dim >= 1 && a.head_dim <= kMaxHeadDim, "head_dim outside 1..256");
  need((long long)a.batch * a.q_heads * a.nodes < (1ll << 31) - 1 && a.capacity < (1 << 30), "sizes too large");
}

size_t workspace_of(const Context& c, const ckks_draft_attention_args& a) {
  const int s = split_count(c, a);
  if (s == 1 || a.batch == 0) return 0;
  return sizeof(float) * (size_t)a.batch * a.q_heads * a.nodes * s * (a.head_dim + 2);
}

}  // namespace
}  // namespace draft
}  // namespace ckks

using namespace ckks;
using namespace ckks::draft;

extern "C" long long ckks_draft_attention_workspace(ckks_ctx* ctx, const ckks_draft_attention_args* a) {
  long long n = -1;
  guard([&] {
    Context& c = context_of(ctx);
    need(a != nullptr, "null argument");
    check_shape(*a);
    n = (long long)workspace_of(c, *a);
  });
  return n;
}

extern "C" int ckks_draft_attention(ckks_ctx* ctx, const ckks_draft_attention_args* args, void* stream) {
  return guard([&] {
    Context& c = context_of(ctx);
    need(args != nullptr, "null argument");
    const ckks_draft_attention_args& a = *args;
    check_shape(a);
    need(std::isfinite(a.scale), "scale is not finite");
    if (a.batch == 0) return;
    const int e = element_bytes(a.dtype);
    check_rows(a.q, e, "q");
    if (a.capacity) {
      check_rows(a.k_cache, e, "k_cache");
      check_rows(a.v_cache, e, "v_cache");
    }
    check_rows(a.k_new, e, "k_new");
    check_rows(a.v_new, e, "v_new");
    check_rows(a.out, e, "out");
    check_ptr(a.lens, "lens");
    check_ptr(a.parents, "parents");
    check_ptr(a.lse, "lse");
    const size_t ws = workspace_of(c, a);
    need(a.workspace_bytes >= ws && (ws == 0 || a.workspace), "workspace smaller than ckks_draft_attention_workspace");
    need(reinterpret_cast<uintptr_t>(a.workspace) % 16 == 0, "workspace not aligned to 16 bytes");
    AttnParams p{};
    p.q = a.q, p.kc = a.k_cache, p.vc = a.v_cache, p.kn = a.k_new, p.vn = a.v_new, p.out = a.out;
    p.lens = a.lens, p.parents = a.parents, p.lse = a.lse, p.part = static_cast<float*>(a.workspace);
    p.batch = a.batch, p.kv_heads = a.kv_heads, p.group = a.q_heads / a.kv_heads, p.head_dim = a.head_dim;
    p.nodes = a.nodes, p.capacity = a.capacity, p.scale = (float)a.scale;
    p.splits = split_count(c, a);
    p.wide = wide_rows(a.q, a.batch, a.q_heads, a.nodes, a.head_dim, e) &&
             wide_rows(a.k_new, a.batch, a.kv_heads, a.nodes, a.head_dim, e) &&
             wide_rows(a.v_new, a.batch, a.kv_heads, a.nodes, a.head_dim, e) &&
             (a.capacity == 0 || (wide_rows(a.k_cache, a.batch, a.kv_heads, a.capacity, a.head_dim, e) &&
                                  wide_rows(a.v_cache, a.batch, a.kv_heads, a.capacity, a.head_dim, e)));
    OnDevice dev(c);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const double bytes = 2.0 * e * a.batch * a.kv_heads * a.capacity * a.head_dim;
    ProfScope ps(c, "draft_attention", bytes, st);
    if (a.dtype == CKKS_BF16)
      run_attend<__nv_bfloat16>(p, st);
    else if (a.dtype == CKKS_FP16)
      run_attend<__half>(p, st);
    else
      run_attend<float>(p, st);
  });
}
