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
#include <limits>

#include "draft_tc.cuh"

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

// a place in the list of units; walked upwards by a whole warp
struct Unit {
  int seq, len, row0, head;  // first row of the sequence, its length, the unit's first row of it, query head
};
// Of 32 sequences after the others, the units come by their place in the
// sequence, the last (and longest) ones first.
template <int ROWS>
struct Units {
  Starts starts;
  int b0 = 0, before = 0, first, len, rungs, all, level, above;  // rungs of ROWS rows; those above `level`, of all lanes
  __device__ __forceinline__ void load(const PromptParams& p) {
    const int2 at = starts.next(p, b0);
    first = at.x, len = at.y;
    rungs = (len + ROWS - 1) / ROWS;
    all = __reduce_add_sync(0xffffffffu, rungs) * p.q_heads;
    level = __reduce_max_sync(0xffffffffu, rungs) - 1;
    above = 0;
  }
  __device__ __forceinline__ void begin(const PromptParams& p) {
    starts.begin(p);
    load(p);
  }
  // unit w, no earlier than the one before; false behind the last
  __device__ __forceinline__ bool find(const PromptParams& p, int w, Unit& u) {
    while (w - before >= all) {
      if (b0 + 32 >= p.batch) return false;
      before += all;
      b0 += 32;
      load(p);
    }
    const int rung = (w - before) / p.q_heads;
    uint32_t with = __ballot_sync(0xffffffffu, rungs > level);
    while (rung >= above + __popc(with)) {
      above += __popc(with);
      --level;
      with = __ballot_sync(0xffffffffu, rungs > level);
    }
    const uint32_t lower = (1u << (threadIdx.x & 31)) - 1u;
    const bool mine = rungs > level && __popc(with & lower) == rung - above;
    const int k = __ffs(__ballot_sync(0xffffffffu, mine)) - 1;
    u.seq = __shfl_sync(0xffffffffu, first, k);
    u.len = __shfl_sync(0xffffffffu, len, k);
    u.row0 = level * ROWS;
    u.head = (w - before) % p.q_heads;
    return true;
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
// A CTA of 16 x 16 threads takes 16 RT rows of one query head, the longest
// first, over tiles of 64 keys staged in shared memory as floats.  Scores: a
// thread has RT rows x 4 keys; values: RT rows x 4 elements of every 64.  A row's
// 16 threads are half a warp, so its maximum and sum are shuffles.  Issue slots
// and reads from shared memory bound it (8 of 16 bytes for 64 multiply-adds, 12
// for 128 with RT 8): 31 TFLOP/s for one prompt of 4096 and 16 heads of 64 in
// float32, 35 for four of 2048 and 8 of 128.  Two CTAs an SM are worth more than
// the few registers that then go to memory (up to 1030 four prompts of 12 heads of 64:
// 183 us, with one CTA 225); multiply-adds in pairs took 243.  Heads of 125 to 128 ask for
// 118 KB of shared memory with 64 rows, so one CTA runs there on the registers of two.
// (These and the rules' figures below are of calls back to back; replayed in a graph the
// four prompts take 195 us.)
constexpr int kKeyTile = 64, kThreads = 256;

template <typename T, int DC, int RT>
__global__ void __launch_bounds__(kThreads, DC <= 2 && RT == 4 ? 2 : 1) prompt_kernel(PromptParams p) {
  constexpr int ROWS = 16 * RT, PS = kKeyTile + 4;
  extern __shared__ __align__(16) float sm[];
  const int D = p.head_dim, D4 = (D + 3) & ~3, KS = D4 + 4, QS = DC == 1 ? D4 : KS;
  float* sq = sm;                     // [ROWS][QS]
  float* sk = sq + ROWS * QS;         // [kKeyTile][KS]
  float* sv = sk + kKeyTile * KS;     // [kKeyTile][D4]
  float* sp = sv + kKeyTile * D4;     // [ROWS][PS]
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  // A thread has rows 4 ty to 4 ty + 3 of every 64: with rows of K's pitch the two that
  // a warp reads at once lie 16 banks apart (one prompt of 8192, 4 heads of 128, 2051 us,
  // 2086 without either; heads of 64 are faster without the pitch, 183 us for 189 in the
  // case below, as reads are not what they wait for)
  auto after = [](int i) { return i % 4 + i / 4 * 64; };
  Units<ROWS> list;
  list.begin(p);
  Unit u;
  const bool some = list.find(p, blockIdx.x, u);
  while (list.b0 + 32 < p.batch) list.b0 += 32, list.load(p);  // the rest of the starts
  clear_spare<T>(p, list.starts.first, list.starts.last, kThreads);
  if (!some) return;
  const int seq = u.seq, len = u.len, row0 = u.row0, h = u.head;
  const T* q = static_cast<const T*>(p.q.data) + (int64_t)(seq + row0) * p.q.row + h * p.q.head;
  const T* k = static_cast<const T*>(p.k.data) + (int64_t)seq * p.k.row + h / p.group * p.k.head;
  const T* v = static_cast<const T*>(p.v.data) + (int64_t)seq * p.v.row + h / p.group * p.v.head;
  const int rows = min(ROWS, len - row0);
  for (int i = tid; i < ROWS * (D4 / 4); i += kThreads) {
    const int r = i / (D4 / 4), d = i % (D4 / 4) * 4;
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    if (r < rows) load_row4(x, q + (int64_t)r * p.q.row, d, D, p.wide);
#pragma unroll
    for (int e = 0; e < 4; ++e) sq[r * QS + d + e] = x[e] * (p.scale * kLog2e);
  }
  float m[RT], l[RT], acc[DC][RT][4];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    m[i] = -INFINITY, l[i] = 0.0f;
#pragma unroll
    for (int c = 0; c < DC; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[c][i][e] = 0.0f;
  }
  for (int t0 = 0; t0 < row0 + rows; t0 += kKeyTile) {
    const int nk = min(kKeyTile, len - t0);
    const bool cut = t0 + kKeyTile - 1 > row0;  // by the causal mask
    __syncthreads();
#pragma unroll
    for (int c = 0; c < DC; ++c) {
      const int d = 64 * c + 4 * tx;
      if (d >= D4) continue;
      float x[4][4], y[4][4];  // all reads before the first write
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = ty + 16 * j;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[j][e] = y[j][e] = 0.0f;
        if (r < nk) {
          load_row4(x[j], k + (int64_t)(t0 + r) * p.k.row, d, D, p.wide);
          load_row4(y[j], v + (int64_t)(t0 + r) * p.v.row, d, D, p.wide);
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = ty + 16 * j;
        *reinterpret_cast<float4*>(sk + r * KS + d) = make_float4(x[j][0], x[j][1], x[j][2], x[j][3]);
        *reinterpret_cast<float4*>(sv + r * D4 + d) = make_float4(y[j][0], y[j][1], y[j][2], y[j][3]);
      }
    }
    __syncthreads();
    float s[RT][4];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[i][j] = 0.0f;
#pragma unroll 2
    for (int d = 0; d < D4; d += 4) {
      float4 c[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) c[j] = *reinterpret_cast<const float4*>(sk + (tx + 16 * j) * KS + d);
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        const float4 a = *reinterpret_cast<const float4*>(sq + (4 * ty + after(i)) * QS + d);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          s[i][j] = fmaf(a.x, c[j].x, fmaf(a.y, c[j].y, fmaf(a.z, c[j].z, fmaf(a.w, c[j].w, s[i][j]))));
      }
    }
    // the last key of this tile that the thread's first row sees
    const int seen = row0 + 4 * ty - t0;
    float f[RT];  // what the sums so far are scaled by
    bool moved = false;
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      if (cut)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (tx + 16 * j > seen + after(i)) s[i][j] = -INFINITY;
      float mx = fmaxf(fmaxf(s[i][0], s[i][1]), fmaxf(s[i][2], s[i][3]));
#pragma unroll
      for (int o = 8; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      const float top = fmaxf(m[i], mx), base = top == -INFINITY ? 0.0f : top;
      f[i] = ex2(m[i] - base);
      moved |= f[i] != 1.0f;
      m[i] = top;
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float e = ex2(s[i][j] - base);
        sum += e;
        sp[(4 * ty + after(i)) * PS + tx + 16 * j] = e;
      }
#pragma unroll
      for (int o = 8; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      l[i] = fmaf(l[i], f[i], sum);
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int c = 0; c < DC; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[c][i][e] *= f[i];
    }
    __syncwarp();  // a row's weights are of one half warp
    // four keys at a time; a value reaches the rows that see it only, whatever it holds
    auto values = [&](auto masked) {
#pragma unroll 1
      for (int j0 = 0; j0 < (decltype(masked)::value ? min(kKeyTile, seen + after(RT - 1) + 1) : kKeyTile); j0 += 4) {
        float4 w[RT];
#pragma unroll
        for (int i = 0; i < RT; ++i) w[i] = *reinterpret_cast<const float4*>(sp + (4 * ty + after(i)) * PS + j0);
#pragma unroll
        for (int c = 0; c < DC; ++c) {
          const int d = 64 * c + 4 * tx;
          if (d >= D4) continue;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float4 y = *reinterpret_cast<const float4*>(sv + (j0 + j) * D4 + d);
#pragma unroll
            for (int i = 0; i < RT; ++i) {
              if (decltype(masked)::value && j0 + j > seen + after(i)) continue;
              const float x = j == 0 ? w[i].x : j == 1 ? w[i].y : j == 2 ? w[i].z : w[i].w;
              acc[c][i][0] = fmaf(x, y.x, acc[c][i][0]);
              acc[c][i][1] = fmaf(x, y.y, acc[c][i][1]);
              acc[c][i][2] = fmaf(x, y.z, acc[c][i][2]);
              acc[c][i][3] = fmaf(x, y.w, acc[c][i][3]);
            }
          }
        }
      }
    };
    if (cut)
      values(std::true_type{});
    else
      values(std::false_type{});
  }
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    const int r = 4 * ty + after(i);
    if (r >= rows) continue;
    const float inv = l[i] != 0.0f ? 1.0f / l[i] : 0.0f;  // 0: no score is above -inf
    T* o = static_cast<T*>(p.out.data) + (int64_t)(seq + row0 + r) * p.out.row + h * p.out.head;
#pragma unroll
    for (int c = 0; c < DC; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (64 * c + 4 * tx + e < D) o[64 * c + 4 * tx + e] = from_f32<T>(acc[c][i][e] * inv);
    if (tx == 0)
      p.lse[(int64_t)(seq + row0 + r) * p.q_heads + h] = l[i] != 0.0f ? kLn2 * (m[i] + log2f(l[i])) : -INFINITY;
  }
}

constexpr size_t prompt_smem(int rows, int D4) {
  return sizeof(float) * (rows * (D4 + kKeyTile + 8) + kKeyTile * (2 * D4 + 4));
}

template <typename T, int DC, int RT>
void launch_prompt(const PromptParams& p, cudaStream_t st) {
  constexpr int ROWS = 16 * RT;
  auto* k = prompt_kernel<T, DC, RT>;
  static_assert(prompt_smem(ROWS, 64 * DC) <= 232448, "shared memory of one block");
  CKKS_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)prompt_smem(ROWS, 64 * DC)));
  const unsigned grid = (unsigned)(std::max(1, p.batch + p.tokens / ROWS) * p.q_heads);
  k<<<grid, kThreads, prompt_smem(ROWS, (p.head_dim + 3) & ~3), st>>>(p);
  CKKS_CUDA(cudaGetLastError());
}

template <typename T>
void run_prompt(const Context& c, const PromptParams& p, cudaStream_t st) {
  switch ((p.head_dim + 63) / 64) {
    case 1: launch_prompt<T, 1, 4>(p, st); break;
    case 2:
      // 128 rows, for fewer reads a multiply-add, where that leaves three units for two
      // SMs: one prompt of 8192, 4 heads of 128, 2096 us (2424 with 64 rows); two of
      // 1500, 12 heads of 100, 455 (489); but one of 3000, 8 heads of 128, 774 (709).
      // Heads of 64 gain little and lose on shorter prompts: one of 4096, 16 heads, 1080
      // (1116), up to 1030 four of 12, 273 (186).
      if ((long long)p.tokens / 128 * p.q_heads >= 3ll * c.sms / 2)
        launch_prompt<T, 2, 8>(p, st);
      else
        launch_prompt<T, 2, 4>(p, st);
      break;
    case 3: launch_prompt<T, 3, 4>(p, st); break;
    default: launch_prompt<T, 4, 4>(p, st); break;
  }
}

// ---- 16-bit types: tensor cores -------------------------------------------------
// A unit is 256 rows of one query head of one sequence: two groups of four
// softmax warps have 128 rows each (over 128 elements there is one group, as
// tensor memory holds one O then), a thread a row.  Keys come in tiles of 128,
// each copied once for both groups, and are worked on by halves: a group has two
// places of 64 scores in tensor memory, S = Q K^T into one while its warps turn
// the other into weights, which take their scores' place as the 16-bit A operand
// of O += P V.  One warp issues copies, one for each group its products.  The
// first group has one tile less than the second, and only a group's last tile
// is cut by the causal mask.  (One place of 128 scores a group waited for its
// products in turn with them, and one warp for both groups' products took 200
// cycles at each barrier: 623 us for the first case below, where this takes 502.)
//
// CTAs are one to an SM and take the units of the list in turns, one round
// upwards and the next one downwards.  The longest units of 32 sequences come
// first, so every CTA gets about the same (prompts up to 2001: 52 tiles at most
// where 49 is the mean, 73 with one sequence behind the other).
//
// A row's reference point m follows the maximum only when that has grown by
// more than 2^8; O is seldom rescaled.  A weight is rounded once, to the
// operands' type (half a step, as the result is), and summed in 32 bits before
// that.  Two numbers a weight, as over a cache, would be half as many products
// again; one number leaves a bfloat16 result 1.3 times as far from the exact one
// as its own rounding takes it (2.1e-3 of it against 1.6e-3).
//
// The exponential unit takes 8 cycles for a warp's 32: 2048 cycles for a pair of
// tiles, whose products take 1024 at 64 elements and 2048 at 128.  So two in
// eight of the exponentials are computed with multiply-adds: 2^x = 2^n 2^r, n
// the nearest integer, and 2^r the polynomial 1 + ... of degree 4 with the least
// largest relative error on [-1/2, 1/2] (2.9e-6, fitted to 2^r).  None, one, two, three, four
// in eight: 553, 546, 542, 566, 580 us for the first case, 525, 495, 484, 501, 530 for
// heads of 64.
//
// Measured: 8192 tokens, 32/8 heads of 128, bfloat16, 502 us (1.10 PFLOP/s, 65 % of
// a library product) in bursts; 586 us and 0.94 in calls back to back, under the power limit;
// twelve prompts up to 2001, 12 heads of 64, float16, 107 us.  Half a tile takes a
// softmax warp some 1600 cycles: 240 at the barrier of its scores, 300 for their
// maximum, 1000 for the weights (two warps share an exponential unit), and no
// stage of this chain is much shorter than the others: without exponentials,
// maxima, most products or most copies heads of 64 still take 85 % of the time.
// 103 tokens of 12 heads take 9 us: set-up, copies, two products and the write,
// one behind the other.
constexpr int kHalf = 64;  // keys of a half tile

template <int PANELS>
struct PromptShape {
  static constexpr int kGroups = PANELS <= 2 ? 2 : 1, kThreads = 32 * (5 * kGroups + 1), kUnitRows = kM * kGroups;
  static constexpr int kSlots = PANELS == 1 ? 10 : PANELS == 2 ? 5 : PANELS == 3 ? 3 : 2;
  static constexpr uint32_t kTileBytes = PANELS * kPanel;
  // Q of each group, the ring of K and V tiles, barriers, masks, one word
  static constexpr uint32_t kRing = kGroups * kTileBytes, kExtra = kRing + kSlots * kTileBytes;
  static constexpr int kBars = 2 * kSlots + 20;
  static constexpr size_t kSmem = kExtra + kBars * 8 + 6 * 4 * 4 + 16;
  // of eight pairs of exponentials, how many the multiply-adds take
  static constexpr int kPoly = PANELS <= 2 ? 2 : 0;
};

// 2^x for x >= -126; off by 2^-127 at most below, and 0 from -127 on (r is 0 there,
// and the bits of 1 less 127 exponents are those of 0): a key whose weight is nothing
// leaves nothing, however large its value
__device__ __forceinline__ float2 exp2_poly(float2 x) {
  const float2 big = make_float2(12582912.0f, 12582912.0f);  // 1.5 2^23: the sum's low bits are the nearest integer
  x.x = fmaxf(x.x, -127.0f), x.y = fmaxf(x.y, -127.0f);
  const float2 t = add2(x, big), r = sub2(x, sub2(t, big));
  auto two = [](float v) { return make_float2(v, v); };
  float2 y = fma2(r, two(0.009582852944731712f), two(0.055906426161527634f));
  y = fma2(y, r, two(0.24024099111557007f));
  y = fma2(y, r, two(0.6931241750717163f));
  y = fma2(y, r, two(1.0f));
  return make_float2(__uint_as_float(__float_as_uint(y.x) + (__float_as_uint(t.x) << 23)),
                     __uint_as_float(__float_as_uint(y.y) + (__float_as_uint(t.y) << 23)));
}

// the largest of three; a NaN wins
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// takes the elements that are not finite out of a piece of a row; whether there were any
template <typename T>
__device__ __forceinline__ bool take_out(uint4* piece) {
  constexpr uint32_t e = std::is_same_v<T, __nv_bfloat16> ? 0x7F80u : 0x7C00u;
  const uint4 v = *piece;
  if (!not_finite<T>(v)) return false;
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if ((w[k] & e) == e) w[k] &= 0xFFFF0000u;
    if ((w[k] >> 16 & e) == e) w[k] &= 0xFFFFu;
  }
  *piece = make_uint4(w[0], w[1], w[2], w[3]);
  return true;
}

// adds to a finished row what was taken out of the rows `which` (32 from `key0`
// on) that it sees: an infinity or a NaN shows whatever its weight
template <typename T>
__device__ __noinline__ void add_taken_out(const PromptParams& p, const Unit& u, uint32_t which, int key0, int row,
                                           T* out) {
  for (; which; which &= which - 1) {
    const int j = key0 + __ffs(which) - 1;
    if (j > row) break;
    const T* v = static_cast<const T*>(p.v.data) + (int64_t)(u.seq + j) * p.v.row + u.head / p.group * p.v.head;
    for (int d = 0; d < p.head_dim; ++d) {
      const float x = to_f32(v[d]);
      if (!(fabsf(x) < INFINITY)) out[d] = from_f32<T>(to_f32(out[d]) + x);
    }
  }
}

struct PromptMaps {
  CUtensorMap q, k, v;
};

template <typename T, int PANELS>
__global__ void __launch_bounds__(PromptShape<PANELS>::kThreads, 1)
    prompt_tc_kernel(const __grid_constant__ PromptParams p, const __grid_constant__ PromptMaps maps, bool negative,
                     float c, unsigned int* __restrict__ faults) {
  using S = PromptShape<PANELS>;
  constexpr int DP = 64 * PANELS, NS = S::kSlots, GR = S::kGroups, ROWS = S::kUnitRows;
  constexpr bool kBf = std::is_same_v<T, __nv_bfloat16>;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* const s_bar = reinterpret_cast<uint64_t*>(smem + S::kExtra);
  // rows of a group's last tile from which elements were taken out, of two
  // units; then the same of the first group's for the second, of two pairs
  uint32_t(*const s_out)[4] = reinterpret_cast<uint32_t(*)[4]>(s_bar + S::kBars);
  uint32_t* const s_tmem = reinterpret_cast<uint32_t*>(s_out + 6);
  const uint32_t sq = smem_addr(smem), ring = sq + S::kRing, bars = smem_addr(s_bar);
  auto full = [&](int s) { return bars + 8 * s; };
  auto empty = [&](int s) { return bars + 8 * (NS + s); };
  // of a group and a half tile
  auto s_full = [&](int g, int half) { return bars + 8 * (2 * NS + 2 * g + half); };
  auto p_ready = [&](int g, int half) { return bars + 8 * (2 * NS + 4 + 2 * g + half); };
  auto pv_done = [&](int g, int half) { return bars + 8 * (2 * NS + 8 + 2 * g + half); };
  auto q_full = [&](int g) { return bars + 8 * (2 * NS + 12 + g); };
  auto q_empty = [&](int g) { return bars + 8 * (2 * NS + 14 + g); };
  // The first group's last values are clean, in one of four units of two groups.
  // (While the second group's products wait for one, the fourth after it does
  // not get that far: its keys would lie 15 slots behind the one that they hold.)
  auto clean = [&](int pair) { return bars + 8 * (2 * NS + 16 + (pair & 3)); };
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), GR);
    }
    for (int i = 0; i < 4; ++i) mbar_init(clean(i), 4);
    for (int g = 0; g < 2; ++g) {
      for (int h = 0; h < 2; ++h) {
        mbar_init(s_full(g, h), 1);
        mbar_init(p_ready(g, h), 4);
        mbar_init(pv_done(g, h), 1);
      }
      mbar_init(q_full(g), 1);
      mbar_init(q_empty(g), 1);
    }
  }
  if (warp == 4 * GR + 1) tmem_alloc(smem_addr(s_tmem), kTmemCols);
  if (warp == 4 * GR && lane == 0) {
    tile_prefetch(&maps.q);
    tile_prefetch(&maps.k);
    tile_prefetch(&maps.v);
  }
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  const uint32_t tmem = *s_tmem;  // S of every group, then O of every group
  Units<ROWS> list;
  list.begin(p);
  Unit u;
  // round r's unit of this CTA
  auto unit_of = [&](int r) {
    return r * (int)gridDim.x + (r & 1 ? (int)gridDim.x - 1 - (int)blockIdx.x : (int)blockIdx.x);
  };
  // tiles of group g in this unit
  auto tiles_of = [&](int g) { return u.row0 + kM * g < u.len ? u.row0 / kM + g + 1 : 0; };
  bool fine = true;  // no wait gave up
  if (warp == 4 * GR) {
    // ---- copies
    int slot = 0, lap = 0, nq[2] = {0, 0}, k = 0;
    for (int r = 0; fine && list.find(p, unit_of(r), u); ++r) {
      if (lane == 0) {
        const int n = max(tiles_of(0), GR > 1 ? tiles_of(1) : 0), kv = u.head / p.group;
        auto load = [&](const CUtensorMap* m, int tile) {
          if (lap > 0 && !mbar_wait_short(empty(slot), (lap - 1) & 1)) return fine = false;
          mbar_expect_tx(full(slot), S::kTileBytes);
#pragma unroll
          for (int x = 0; x < PANELS; ++x)
            tile_load(ring + slot * S::kTileBytes + x * kPanel, m, 64 * x, u.seq + tile * kKeys, kv, 0, full(slot));
          ++k;
          if (++slot == NS) slot = 0, ++lap;
          return true;
        };
        load(&maps.k, 0);
#pragma unroll
        for (int g = 0; g < GR; ++g) {
          if (!fine || !tiles_of(g)) continue;
          if (nq[g] > 0 && !(fine = mbar_wait_short(q_empty(g), (nq[g] - 1) & 1))) continue;
          ++nq[g];
          mbar_expect_tx(q_full(g), S::kTileBytes);
#pragma unroll
          for (int x = 0; x < PANELS; ++x)
            tile_load(sq + g * S::kTileBytes + x * kPanel, &maps.q, 64 * x, u.seq + u.row0 + kM * g, u.head, 0,
                      q_full(g));
        }
        for (int t = 0; t < n && fine; ++t)
          if (load(&maps.v, t) && t + 1 < n) load(&maps.k, t + 1);
      }
      fine = __shfl_sync(0xffffffffu, fine, 0);
    }
    if (lane == 0) {
      // copies still in flight land before the CTA ends
      for (int j = k > NS ? k - NS : 0; j < k; ++j) fine = mbar_wait_short(full(j % NS), (j / NS) & 1) && fine;
#pragma unroll
      for (int g = 0; g < GR; ++g)
        if (nq[g]) fine = mbar_wait_short(q_full(g), (nq[g] - 1) & 1) && fine;
    }
  } else if (warp > 4 * GR) {
    // ---- products of group g, by the whole warp in step
    const int g = warp - (4 * GR + 1);
    constexpr uint32_t word_s = mma_word(kBf, kM, kHalf, false), word_o = mma_word(kBf, kM, DP, true);
    const uint32_t t_base = __shfl_sync(0xffffffffu, tmem, 0), t_s = t_base + 128 * g, t_o = t_base + 128 * (GR + g);
    int slot = 0, pairs = 0;
    uint32_t lap = 0, q_phase = 0, p_phase = 0;
    for (int r = 0; fine && list.find(p, unit_of(r), u); ++r) {
      const int n = __shfl_sync(0xffffffffu, tiles_of(g), 0);
      const int other = GR > 1 ? __shfl_sync(0xffffffffu, tiles_of(g ^ 1), 0) : 0, most = max(n, other);
      auto next = [&] {
        if (++slot == NS) slot = 0, lap ^= 1u;
      };
      // a tile of the other group alone: this one is done with it as soon as it is there
      auto pass = [&](int s, uint32_t l) {
        if (!warp_wait(full(s), l)) return false;
        if (lane == 0) mbar_arrive(empty(s));
        return true;
      };
      // half `h` of tile t, in slot s
      auto scores = [&](int t, int h, int s) {
        const uint32_t qb = sq + g * S::kTileBytes, kb = ring + s * S::kTileBytes + h * (kPanel / 2);
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) {
          const uint32_t off = (i / 4) * kPanel + (i % 4) * 32;
          mma_smem(t_s + kHalf * h, smem_operand(qb + off, 16), smem_operand(kb + off, 16), word_s, i > 0);
        }
        mma_commit(s_full(g, h));
        if (h == 1 && t + 1 == n) mma_commit(q_empty(g));
      };
      auto sums = [&](int t, int h, int s) {
        const uint32_t vb = ring + s * S::kTileBytes + h * (kPanel / 2);
#pragma unroll
        for (int i = 0; i < kHalf / 16; ++i)
          mma_tmem(t_o, t_s + kHalf * h + 8 * i, smem_operand(vb + 2048 * i, kPanel), word_o, i > 0 || h > 0 || t > 0);
        mma_commit(pv_done(g, h));
      };
      if (n) {
        if (!(fine = warp_wait_both(full(slot), lap, q_full(g), q_phase))) break;
        q_phase ^= 1u;
        tmem_fence_after();
        scores(0, 0, slot);
        scores(0, 1, slot);
        mma_commit(empty(slot));
      } else if (!(fine = pass(slot, lap))) {
        break;
      }
      next();
      for (int t = 0; t < most; ++t) {
        const int vs = slot;
        const uint32_t vlap = lap;
        next();
        const int ks = slot;  // of the next tile's keys
        const uint32_t klap = lap;
        if (t + 1 < most) next();
        if (t >= n) {
          if (!(fine = pass(vs, vlap) && (t + 1 == most || pass(ks, klap)))) break;
          continue;
        }
        if (GR > 1 && g == 1 && t + 2 == n && !(fine = warp_wait_done(clean(pairs), pairs >> 2 & 1))) break;
        if (t + 1 < n) {
          if (!(fine = warp_wait_all(full(vs), vlap, p_ready(g, 0), p_phase, full(ks), klap))) break;
          tmem_fence_after();
          sums(t, 0, vs);
          scores(t + 1, 0, ks);  // in the place of these weights
          if (!(fine = warp_wait_done(p_ready(g, 1), p_phase))) break;
          tmem_fence_after();
          sums(t, 1, vs);
          mma_commit(empty(vs));
          scores(t + 1, 1, ks);
          mma_commit(empty(ks));
        } else {
          if (!(fine = warp_wait_both(full(vs), vlap, p_ready(g, 0), p_phase))) break;
          tmem_fence_after();
          sums(t, 0, vs);
          if (!(fine = warp_wait_done(p_ready(g, 1), p_phase))) break;
          tmem_fence_after();
          sums(t, 1, vs);
          mma_commit(empty(vs));
          if (t + 1 < most && !(fine = pass(ks, klap))) break;
        }
        p_phase ^= 1u;
      }
      pairs += GR > 1 && n && other;
    }
  } else {
    // ---- softmax: group g, tensor-memory lane L, that is row L of the group's
    const int g = warp >> 2, quarter = warp & 3, L = quarter * 32 + lane;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const uint32_t t_s = tmem + 128 * g + lanes, t_o = tmem + 128 * (GR + g) + lanes;
    int base = 0, nu = 0, pairs = 0;  // tiles of keys and values before this unit's; units of this group, of both
    uint32_t phase = 0;               // of this group's tile
    for (int r = 0; fine && list.find(p, unit_of(r), u); ++r) {
      const int n = tiles_of(g), most = max(n, GR > 1 ? tiles_of(g ^ 1) : 0);
      const bool both = GR > 1 && n && tiles_of(g ^ 1);
      float m = -INFINITY, l = 0.0f;
#pragma unroll 1
      for (int step = 0; step < 2 * n; ++step) {
        const int h = step & 1, t = step >> 1;
        const bool last = t + 1 == n;
        if (!(fine = warp_wait(s_full(g, h), phase))) break;
        if (last && h == 0) {
          // The values of keys that only some rows of this tile see: what is
          // not finite is taken out of the product.  (The copy that had the slot
          // before was used ahead of this tile's scores, so the wait cannot take
          // its arrival for this one's.)
          const int kv = base + 2 * t + 1;
          if (!(fine = warp_wait(full(kv % NS), (kv / NS) & 1))) break;
          uint8_t* vs = smem + S::kRing + (kv % NS) * S::kTileBytes + L * 128;
          bool out = false;
#pragma unroll
          for (int i = 0; i < DP / 8; ++i)
            out |= take_out<T>(reinterpret_cast<uint4*>(vs + (i / 8) * kPanel + ((i % 8) << 4)));
          const uint32_t some = __ballot_sync(0xffffffffu, out);
          if (some) smem_fence_async();
          __syncwarp();
          if (lane == 0) {
            s_out[2 * g + (nu & 1)][quarter] = some;
            if (both && g == 0) {
              s_out[4 + (pairs & 1)][quarter] = some;
              mbar_arrive(clean(pairs));
            }
          }
        }
        tmem_fence_after();
        uint32_t x[kHalf];
        tmem_load<kHalf>(t_s + kHalf * h, x);
        tmem_wait_load();
        if (negative) {  // scores of -q
#pragma unroll
          for (int i = 0; i < kHalf; ++i) x[i] ^= 0x80000000u;
        }
        if (last) {
          const int seen = L - kHalf * h;
#pragma unroll
          for (int i = 0; i < kHalf; ++i)
            if (i > seen) x[i] = __float_as_uint(-INFINITY);
        }
        float mx4[4] = {__uint_as_float(x[0]), __uint_as_float(x[1]), __uint_as_float(x[2]), __uint_as_float(x[3])};
#pragma unroll
        for (int i = 4; i < kHalf; i += 2)
          mx4[i / 2 & 3] = max3(mx4[i / 2 & 3], __uint_as_float(x[i]), __uint_as_float(x[i + 1]));
        const float mx = max3(max3(mx4[0], mx4[1], mx4[2]), mx4[3], -INFINITY);
        float top = mx == -INFINITY ? mx : fmaf(mx, c, -kBelow<T>);
        bool bare = false;  // a row that has seen no score above -inf
        if (__any_sync(0xffffffffu, !(top <= m + kSlack) || m == -INFINITY)) {  // grown, no number, or bare
          float f = 1.0f;
          if (!(top <= m + kSlack)) {
            if (!(top < INFINITY)) top = __uint_as_float(0x7FC00000u);  // an infinite score leaves no number
            f = m == -INFINITY && top == top ? 0.0f : ex2(m - top);
            m = top;
            l *= f;
          }
          bare = __any_sync(0xffffffffu, m == -INFINITY);
          if (step > 0 && __any_sync(0xffffffffu, f != 1.0f)) {
            // the sums so far, on the new reference point, once the product before is done
            if (!(fine = warp_wait(pv_done(g, h ^ 1), h ? phase : phase ^ 1u))) break;
            tmem_fence_after();
#pragma unroll 1
            for (int i = 0; i < DP; i += 16) {
              uint32_t o[16];
              tmem_load<16>(t_o + i, o);
              tmem_wait_load();
#pragma unroll
              for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
              tmem_store<16>(t_o + i, o);
            }
          }
        }
        const float ref = m == -INFINITY ? 0.0f : m;
        // the weights take the place of their scores.  A masked score's is 0, and
        // so are those of a row that has seen none above -inf
        float2 sum[4];
        auto weights = [&](auto poly) {
#pragma unroll
          for (int i0 = 0; i0 < kHalf; i0 += 32) {
            // all exponentials of a piece before the first is used
            float2 e[16];
#pragma unroll
            for (int i = 0; i < 16; ++i)
              e[i] = fma2(make_float2(__uint_as_float(x[i0 + 2 * i]), __uint_as_float(x[i0 + 2 * i + 1])),
                          make_float2(c, c), make_float2(-ref, -ref));
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              if (i % 8 < decltype(poly)::value)
                e[i] = exp2_poly(e[i]);
              else
                e[i] = make_float2(ex2(e[i].x), ex2(e[i].y));
            }
            uint32_t w[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              sum[i & 3] = i0 == 0 && i < 4 ? e[i] : add2(sum[i & 3], e[i]);
              w[i] = pack2<T>(e[i].x, e[i].y);
            }
            tmem_store<16>(t_s + kHalf * h + i0 / 2, w);
          }
        };
        if (last || bare)
          weights(std::integral_constant<int, 0>{});
        else
          weights(std::integral_constant<int, S::kPoly>{});
        const float2 all = add2(add2(sum[0], sum[1]), add2(sum[2], sum[3]));
        l += all.x + all.y;
        tmem_wait_store();
        tmem_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_ready(g, h));
        if (h) phase ^= 1u;
      }
      if (!fine) break;
      base += 2 * most;
      if (n) {
        if (!(fine = warp_wait(pv_done(g, 1), phase ^ 1u))) break;
        tmem_fence_after();
        const int row = u.row0 + kM * g + L;
        const bool mine = row < u.len;
        const float inv = l != 0.0f ? 1.0f / l : 0.0f;
        T* const out = static_cast<T*>(p.out.data) + (int64_t)(u.seq + row) * p.out.row + u.head * p.out.head;
#pragma unroll 1
        for (int i = 0; i < DP; i += 32) {
          uint32_t o[32];
          tmem_load<32>(t_o + i, o);
          tmem_wait_load();
          if (mine) {
#pragma unroll
            for (int j = 0; j < 32; j += 8) {
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e)
                w[e] = pack2<T>(__uint_as_float(o[j + 2 * e]) * inv, __uint_as_float(o[j + 2 * e + 1]) * inv);
              if (i + j < p.head_dim) *reinterpret_cast<uint4*>(out + i + j) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
        }
        if (mine) {
          p.lse[(int64_t)(u.seq + row) * p.q_heads + u.head] = l != 0.0f ? kLn2 * (m + log2f(l)) : -INFINITY;
          const uint32_t* own = s_out[2 * g + (nu & 1)];
          const uint32_t* other = s_out[4 + (pairs & 1)];
          uint32_t any = own[0] | own[1] | own[2] | own[3];
          if (both && g == 1) any |= other[0] | other[1] | other[2] | other[3];
          if (any) {
            const int tile0 = (n - 1) * kKeys;
            if (both && g == 1)
              for (int q = 0; q < 4; ++q) add_taken_out<T>(p, u, other[q], tile0 - kKeys + 32 * q, row, out);
            for (int q = 0; q < 4; ++q) add_taken_out<T>(p, u, own[q], tile0 + 32 * q, row, out);
          }
        }
        __syncwarp();
        ++nu;
        pairs += both;
        tmem_fence_before();
      }
    }
    if (fine) clear_spare<T>(p, list.starts.first, list.starts.last, 128 * GR);
  }
  if (!fine && (warp < 4 * GR || lane == 0)) atomicAdd(faults, 1u);
  tmem_fence_before();
  __syncthreads();
  if (warp == 4 * GR + 1) {
    __syncwarp();
    tmem_free(tmem, kTmemCols);
  }
}

template <typename T, int PANELS>
void launch_prompt_tc(const Context& c, const PromptParams& p, const PromptMaps& maps, cudaStream_t st) {
  using S = PromptShape<PANELS>;
  static_assert(S::kSmem <= 232448, "shared memory of one block");
  auto* k = prompt_tc_kernel<T, PANELS>;
  CKKS_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::kSmem));
  // a scale of 0 becomes the least there is: a masked score times 0 would be no
  // number, and no finite score times 2^-149 reaches 2^-21
  const float factor = std::max(std::fabs(p.scale) * kLog2e, std::numeric_limits<float>::denorm_min());
  const long long units = (long long)std::max(1, p.batch + p.tokens / S::kUnitRows) * p.q_heads;
  k<<<(unsigned)std::min<long long>(units, c.sms), S::kThreads, S::kSmem, st>>>(p, maps, p.scale < 0.0f, factor,
                                                                               c.d_faults);
  CKKS_CUDA(cudaGetLastError());
}

template <typename T>
bool run_prompt_tc(const Context& c, int dtype, int kv_heads, const PromptParams& p, cudaStream_t st) {
  PromptMaps m;
  auto map = [&](CUtensorMap* t, const ckks_rows& r, int heads) {
    return tile_map(t, r.data, dtype, p.head_dim, p.tokens, r.row, kM, heads, r.head, 1, 1, 0);
  };
  if (!map(&m.q, p.q, p.q_heads) || !map(&m.k, p.k, kv_heads) || !map(&m.v, p.v, kv_heads)) return false;
  switch ((p.head_dim + 63) / 64) {
    case 1: launch_prompt_tc<T, 1>(c, p, m, st); break;
    case 2: launch_prompt_tc<T, 2>(c, p, m, st); break;
    case 3: launch_prompt_tc<T, 3>(c, p, m, st); break;
    default: launch_prompt_tc<T, 4>(c, p, m, st); break;
  }
  return true;
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
    need(((long long)a.batch + a.tokens / 64) * a.q_heads < (1ll << 31) - 1, "sizes too large");
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
    // strides that no tensor map holds are left to the plain kernel
    if (p.wide && a.dtype != CKKS_FP32) {
      if (a.dtype == CKKS_BF16 ? run_prompt_tc<__nv_bfloat16>(c, a.dtype, a.kv_heads, p, st)
                               : run_prompt_tc<__half>(c, a.dtype, a.kv_heads, p, st))
        return;
    }
    if (a.dtype == CKKS_BF16)
      run_prompt<__nv_bfloat16>(c, p, st);
    else if (a.dtype == CKKS_FP16)
      run_prompt<__half>(c, p, st);
    else
      run_prompt<float>(c, p, st);
  });
}
