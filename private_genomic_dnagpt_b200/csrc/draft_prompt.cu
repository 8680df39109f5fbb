// draft_prompt.cu -- causal attention within packed prompts
// (ckks_draft_prompt): what the draft model evaluates before its first tree.
//
// Sequence b has the rows from start(b) to start(b + 1) of q, k and v, and for
// row i of it and each query head
//   s_j = scale q_i . k_j,  out_i = sum_j exp(s_j - m) v_j / l,
//   m = max_j s_j,  l = sum_j exp(s_j - m),  lse_i = m + ln l
// over the rows j <= i of the sequence.  A sequence of n rows costs
// 2 n (n + 1) head_dim operations a query head, 4 bytes a score if scores were
// written: they stay on the chip, and arithmetic bounds all but short prompts.
#include <algorithm>
#include <cmath>

#include "draft.hpp"

namespace ckks {
namespace draft {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct PromptParams {
  ckks_rows q, k, v, out;
  const int32_t* starts;
  float* lse;
  int batch, q_heads, group, head_dim, tokens;
  float scale;
  bool wide;
};

// start(b) is the largest of starts[0..b], each taken as 0..tokens: an order
// that decreases leaves a sequence without rows, and no row belongs to two.
// This walks 32 sequences at a time; by a whole warp.
struct Starts {
  int first, last;  // start(0), and start() behind the sequences walked so far
  __device__ __forceinline__ void begin(const PromptParams& p) {
    first = last = min(max(p.starts[0], 0), p.tokens);
  }
  // sequence b0 + lane's first row and length
  __device__ __forceinline__ int2 next(const PromptParams& p, int b0) {
    const int lane = threadIdx.x & 31, b = b0 + lane;
    int e = b < p.batch ? min(max(p.starts[b + 1], 0), p.tokens) : 0;
    e = max(e, last);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, e, o);
      if (lane >= o) e = max(e, y);
    }
    int a = __shfl_up_sync(0xffffffffu, e, 1);
    if (lane == 0) a = last;
    last = __shfl_sync(0xffffffffu, e, 31);
    return make_int2(a, e - a);
  }
};

// rows of no sequence: out 0, lse -inf; by the first `threads` of all CTAs
template <typename T>
__device__ __forceinline__ void clear_spare(const PromptParams& p, int first, int last, int threads) {
  const int spare = p.tokens - (last - first);
  for (int i = blockIdx.x; i < spare; i += gridDim.x) {
    const int t = i < first ? i : last + (i - first);
    for (int x = threadIdx.x; x < p.q_heads * p.head_dim; x += threads)
      static_cast<T*>(p.out.data)[(int64_t)t * p.out.row + x / p.head_dim * p.out.head + x % p.head_dim] = from_f32<T>(0.0f);
    for (int h = threadIdx.x; h < p.q_heads; h += threads) p.lse[(int64_t)t * p.q_heads + h] = -INFINITY;
  }
}

// ---- every type, size and stride: CUDA cores ------------------------------------
// A CTA of 16 x 16 threads takes 64 rows of one query head, the longest first,
// over tiles of 64 keys staged in shared memory as floats.  Scores: a thread
// has 4 rows x 4 keys; values: 4 rows x 4 elements of every 64.  A row's 16
// threads are half a warp, so its maximum and sum are shuffles.
constexpr int kRows = 64, kThreads = 256;

template <typename T, int DC>
__global__ void __launch_bounds__(kThreads) prompt_kernel(PromptParams p) {
  extern __shared__ __align__(16) float sm[];
  const int D = p.head_dim, D4 = (D + 3) & ~3, KS = D4 + 4, PS = kRows + 4;
  float* sq = sm;                  // [kRows][D4]
  float* sk = sq + kRows * D4;     // [kRows][KS]
  float* sv = sk + kRows * KS;     // [kRows][D4]
  float* sp = sv + kRows * D4;     // [kRows][PS]
  __shared__ int s_place[5];       // first row of the sequence, its length, first row of the tile, start(0), start(batch)
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int h = blockIdx.x % p.q_heads;
  if (tid < 32) {
    Starts s;
    s.begin(p);
    int unit = blockIdx.x / p.q_heads;
    if (tid == 0) s_place[2] = -1;
    __syncwarp();
    for (int b0 = 0; b0 < p.batch; b0 += 32) {
      const int2 at = s.next(p, b0);
      const int tiles = (at.y + kRows - 1) / kRows;
      int sum = tiles;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, sum, o);
        if ((tid & 31) >= o) sum += y;
      }
      if (unit >= sum - tiles && unit < sum) {
        s_place[0] = at.x;
        s_place[1] = at.y;
        s_place[2] = (sum - 1 - unit) * kRows;
      }
      unit -= __shfl_sync(0xffffffffu, sum, 31);
    }
    if (tid == 0) s_place[3] = s.first, s_place[4] = s.last;
  }
  __syncthreads();
  clear_spare<T>(p, s_place[3], s_place[4], kThreads);
  const int seq = s_place[0], len = s_place[1], row0 = s_place[2];
  if (row0 < 0) return;
  const T* q = static_cast<const T*>(p.q.data) + (int64_t)(seq + row0) * p.q.row + h * p.q.head;
  const T* k = static_cast<const T*>(p.k.data) + (int64_t)seq * p.k.row + h / p.group * p.k.head;
  const T* v = static_cast<const T*>(p.v.data) + (int64_t)seq * p.v.row + h / p.group * p.v.head;
  const int rows = min(kRows, len - row0);
  for (int i = tid; i < kRows * (D4 / 4); i += kThreads) {
    const int r = i / (D4 / 4), d = i % (D4 / 4) * 4;
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    if (r < rows) load_row4(x, q + (int64_t)r * p.q.row, d, D, p.wide);
#pragma unroll
    for (int e = 0; e < 4; ++e) sq[r * D4 + d + e] = x[e] * (p.scale * kLog2e);
  }
  float m[4], l[4], acc[DC][4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY, l[i] = 0.0f;
#pragma unroll
    for (int c = 0; c < DC; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[c][i][e] = 0.0f;
  }
  for (int t0 = 0; t0 < row0 + rows; t0 += kRows) {
    const int nk = min(kRows, len - t0);
    const bool last = t0 == row0;  // the tile that the causal mask cuts
    __syncthreads();
    for (int i = tid; i < kRows * (D4 / 4); i += kThreads) {
      const int r = i / (D4 / 4), d = i % (D4 / 4) * 4;
      float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
      if (r < nk) {
        load_row4(x, k + (int64_t)(t0 + r) * p.k.row, d, D, p.wide);
        load_row4(y, v + (int64_t)(t0 + r) * p.v.row, d, D, p.wide);
      }
      *reinterpret_cast<float4*>(sk + r * KS + d) = make_float4(x[0], x[1], x[2], x[3]);
      *reinterpret_cast<float4*>(sv + r * D4 + d) = make_float4(y[0], y[1], y[2], y[3]);
    }
    __syncthreads();
    float s[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[i][j] = 0.0f;
    for (int d = 0; d < D4; d += 4) {
      float4 a[4], c[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = *reinterpret_cast<const float4*>(sq + (4 * ty + i) * D4 + d);
#pragma unroll
      for (int j = 0; j < 4; ++j) c[j] = *reinterpret_cast<const float4*>(sk + (tx + 16 * j) * KS + d);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          s[i][j] = fmaf(a[i].x, c[j].x, fmaf(a[i].y, c[j].y, fmaf(a[i].z, c[j].z, fmaf(a[i].w, c[j].w, s[i][j]))));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (last)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (tx + 16 * j > 4 * ty + i) s[i][j] = -INFINITY;
      float mx = fmaxf(fmaxf(s[i][0], s[i][1]), fmaxf(s[i][2], s[i][3]));
#pragma unroll
      for (int o = 8; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      const float top = fmaxf(m[i], mx), base = top == -INFINITY ? 0.0f : top, f = exp2f(m[i] - base);
      m[i] = top;
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float e = exp2f(s[i][j] - base);
        sum += e;
        sp[(4 * ty + i) * PS + tx + 16 * j] = e;
      }
#pragma unroll
      for (int o = 8; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      l[i] = fmaf(l[i], f, sum);
#pragma unroll
      for (int c = 0; c < DC; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[c][i][e] *= f;
    }
    __syncwarp();  // a row's weights are of one half warp
    const int to = last ? rows : kRows;
    for (int j = 0; j < to; ++j) {
      float w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = sp[(4 * ty + i) * PS + j];
#pragma unroll
      for (int c = 0; c < DC; ++c) {
        const int d = 64 * c + 4 * tx;
        if (d >= D4) continue;
        const float4 y = *reinterpret_cast<const float4*>(sv + j * D4 + d);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // a value reaches the rows that see it only, whatever it holds
          if (last && j > 4 * ty + i) continue;
          acc[c][i][0] = fmaf(w[i], y.x, acc[c][i][0]);
          acc[c][i][1] = fmaf(w[i], y.y, acc[c][i][1]);
          acc[c][i][2] = fmaf(w[i], y.z, acc[c][i][2]);
          acc[c][i][3] = fmaf(w[i], y.w, acc[c][i][3]);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 4 * ty + i;
    if (r >= rows) continue;
    const float inv = l[i] != 0.0f ? 1.0f / l[i] : 0.0f;  // 0: no score is above -inf
    T* o = static_cast<T*>(p.out.data) + (int64_t)(seq + row0 + r) * p.out.row + h * p.out.head;
#pragma unroll
    for (int c = 0; c < DC; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (64 * c + 4 * tx + e < D) o[64 * c + 4 * tx + e] = from_f32<T>(acc[c][i][e] * inv);
    if (tx == 0) p.lse[(int64_t)(seq + row0 + r) * p.q_heads + h] = l[i] != 0.0f ? kLn2 * (m[i] + log2f(l[i])) : -INFINITY;
  }
}

constexpr size_t prompt_smem(int D4) { return sizeof(float) * kRows * (3 * D4 + 4 + kRows + 4); }

template <typename T, int DC>
void launch_prompt(const PromptParams& p, cudaStream_t st) {
  auto* k = prompt_kernel<T, DC>;
  static_assert(prompt_smem(64 * DC) <= 232448 - 64, "shared memory of one block");
  CKKS_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)prompt_smem(64 * DC)));
  const unsigned grid = (unsigned)(std::max(1, p.batch + p.tokens / kRows) * p.q_heads);
  k<<<grid, kThreads, prompt_smem((p.head_dim + 3) & ~3), st>>>(p);
  CKKS_CUDA(cudaGetLastError());
}

template <typename T>
void run_prompt(const PromptParams& p, cudaStream_t st) {
  switch ((p.head_dim + 63) / 64) {
    case 1: launch_prompt<T, 1>(p, st); break;
    case 2: launch_prompt<T, 2>(p, st); break;
    case 3: launch_prompt<T, 3>(p, st); break;
    default: launch_prompt<T, 4>(p, st); break;
  }
}

}  // namespace
}  // namespace draft
}  // namespace ckks

using namespace ckks;
using namespace ckks::draft;

extern "C" int ckks_draft_prompt(ckks_ctx* ctx, const ckks_draft_prompt_args* args, void* stream) {
  return guard([&] {
    Context& c = context_of(ctx);
    need(args != nullptr, "null argument");
    const ckks_draft_prompt_args& a = *args;
    need(a.dtype == CKKS_BF16 || a.dtype == CKKS_FP16 || a.dtype == CKKS_FP32,
         "attention takes CKKS_BF16, CKKS_FP16 or CKKS_FP32");
    need(a.batch >= 0 && a.batch < (1 << 24) && a.tokens >= 0 && a.tokens < (1 << 30), "batch or tokens out of range");
    need(a.kv_heads >= 1 && a.q_heads >= 1 && a.q_heads % a.kv_heads == 0,
         "query heads are not a multiple of the key/value heads");
    need(a.head_dim >= 1 && a.head_dim <= kMaxHeadDim, "head_dim outside 1..256");
    need(((long long)a.batch + a.tokens / kRows) * a.q_heads < (1ll << 31) - 1, "sizes too large");
    need(std::isfinite((float)a.scale * kLog2e), "scale is not finite");
    if (a.tokens == 0) return;
    const int e = element_bytes(a.dtype);
    check_rows(a.q, e, "q");
    check_rows(a.k, e, "k");
    check_rows(a.v, e, "v");
    check_rows(a.out, e, "out");
    check_ptr(a.starts, "starts");
    check_ptr(a.lse, "lse");
    PromptParams p{};
    p.q = a.q, p.k = a.k, p.v = a.v, p.out = a.out, p.starts = a.starts, p.lse = a.lse;
    p.batch = a.batch, p.q_heads = a.q_heads, p.group = a.q_heads / a.kv_heads, p.head_dim = a.head_dim;
    p.tokens = a.tokens, p.scale = (float)a.scale;
    p.wide = wide_rows(a.q, 1, a.q_heads, a.tokens, a.head_dim, e) &&
             wide_rows(a.k, 1, a.kv_heads, a.tokens, a.head_dim, e) &&
             wide_rows(a.v, 1, a.kv_heads, a.tokens, a.head_dim, e) &&
             wide_rows(a.out, 1, a.q_heads, a.tokens, a.head_dim, e);
    OnDevice dev(c);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    ProfScope ps(c, "draft_prompt", 2.0 * e * a.tokens * (a.q_heads + a.kv_heads) * a.head_dim, st);
    if (a.dtype == CKKS_BF16)
      run_prompt<__nv_bfloat16>(p, st);
    else if (a.dtype == CKKS_FP16)
      run_prompt<__half>(p, st);
    else
      run_prompt<float>(p, st);
  });
}
