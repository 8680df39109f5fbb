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

#include "draft_fp4.cuh"
#include "draft_tc.cuh"

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
  // The kernels that divide a list of units among their CTAs: rows of a unit,
  // keys of a tile, whether the new keys have a tile of their own, and what a
  // unit's start and end cost in tiles
  int tile_nodes, tile_rows, tile_keys, new_apart, unit_cost;
  float scale;
  bool wide;  // every row is whole, aligned 16-byte pieces
};

__device__ __forceinline__ int length_of(const AttnParams& p, int b) { return min(max(p.lens[b], 0), p.capacity); }

// tiles of a unit of sequence b
__device__ __forceinline__ int tiles_of(const AttnParams& p, int b) {
  const int len = length_of(p, b);
  return p.new_apart ? (len + p.tile_keys - 1) / p.tile_keys + 1 : (len + p.nodes + p.tile_keys - 1) / p.tile_keys;
}

// A place in the list: sequence, unit within it, tile within that (below 0:
// the unit's start) and the unit's tiles
struct Cursor {
  int b, unit, tile, tiles;
  __device__ __forceinline__ void next_unit(const AttnParams& p, int units) {
    tile = -p.unit_cost;
    if (++unit == units) {
      unit = 0;
      tiles = ++b < p.batch ? tiles_of(p, b) : 1;
    }
  }
};

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
// partial sums meet once, at the end.  Products and sums are in 32 bits.  What
// the two kernels below do not take comes here: unaligned rows, odd head sizes.
// Loads are not overlapped within a CTA (5 float32 rows over 6000 keys took it
// 87 us, against 40 below).
constexpr int kRows = 8, kTile = 64, kThreads = 128;
constexpr uint32_t kUnseen = 0x80000000u;  // -0: the weight of a key that a row does not see (others are +0 and more)

// DC: chunks of 64 elements that cover head_dim; FOUR: the caches are 4-bit rows
template <typename T, int DC, bool FOUR>
__global__ void __launch_bounds__(kThreads) attend_kernel(AttnParams p) {
  using Cached = std::conditional_t<FOUR, uint8_t, T>;
  extern __shared__ __align__(16) float sm[];
  const int D = p.head_dim, D4 = (D + 3) & ~3, KS = D4 + 4;  // row stride of the keys: 16-byte reads without conflicts
  float* sk = sm;                       // [kTile][KS]
  float* sv = sk + kTile * KS;          // [kTile][D4]
  float* sq = sv + kTile * D4;          // [kRows][D4]
  float* sp = sq + kRows * D4;          // [kTile][kRows]
  __shared__ float s_m[kRows], s_l[kRows], s_c[kRows];
  __shared__ uint64_t s_mask[kMaxNodes], s_row[kRows];  // of the nodes, and of the rows here
  __shared__ int s_jump[kMaxNodes];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rows = p.nodes * p.group, tiles_r = (rows + kRows - 1) / kRows;
  const int rt = blockIdx.x % tiles_r, bh = blockIdx.x / tiles_r;
  const int b = bh / p.kv_heads, h = bh % p.kv_heads;
  const int len = length_of(p, b), total = len + p.nodes;
  // this split's keys [k0, k1) of the cached and then the new ones
  const int per = ((total + p.splits - 1) / p.splits + kTile - 1) / kTile * kTile;
  const int k0 = min(total, (int)blockIdx.y * per), k1 = min(total, k0 + per);
  if (warp == 0) {
    tree_masks(p.parents + (size_t)b * p.nodes, p.nodes, s_mask, s_jump);
    if (lane < kRows) s_row[lane] = rt * kRows + lane < rows ? s_mask[(rt * kRows + lane) / p.group] : 0ull;
  }
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
  const Cached* kc = static_cast<const Cached*>(p.kc.data) + b * p.kc.batch + h * p.kc.head;
  const Cached* vc = static_cast<const Cached*>(p.vc.data) + b * p.vc.batch + h * p.vc.head;
  const T* kn = static_cast<const T*>(p.kn.data) + b * p.kn.batch + h * p.kn.head;
  const T* vn = static_cast<const T*>(p.vn.data) + b * p.vn.batch + h * p.vn.head;
  for (int t0 = k0; t0 < k1; t0 += kTile) {
    const int nk = min(kTile, k1 - t0);
    for (int i = tid; i < kTile * (D4 / 4); i += kThreads) {
      const int r = i / (D4 / 4), d = i % (D4 / 4) * 4, s = t0 + r;
      float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
      if (r < nk) {
        if (s < len) {
          if constexpr (FOUR) {
            load_row4_4bit(x, kc + s * p.kc.row, d, D);
            load_row4_4bit(y, vc + s * p.vc.row, d, D);
          } else {
            load_row4(x, kc + s * p.kc.row, d, D, p.wide);
            load_row4(y, vc + s * p.vc.row, d, D, p.wide);
          }
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
      auto sees = [&](int at) { return at < len || (at < k1 && (s_row[r] >> (at - len) & 1)); };
      sp[lane * kRows + r] = sees(t0 + lane) ? ea : __uint_as_float(kUnseen);
      sp[(lane + 32) * kRows + r] = sees(t0 + lane + 32) ? ec : __uint_as_float(kUnseen);
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
          // a new key's values, whatever they hold, reach the rows that see it only
          const float x = w[r];
          if (__float_as_uint(x) != kUnseen) {
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

// Adds to one finished row the new keys whose values are not finite, which
// the product left out so that they do not reach the rows that may not see
// them: what those elements add is infinite or no number, whatever the weight.
template <typename T>
__device__ __noinline__ void add_spoiled(const AttnParams& p, int b, int h, int node, int qh, unsigned long long which,
                                         float m, float inv, T* out) {
  const T* q = static_cast<const T*>(p.q.data) + b * p.q.batch + qh * p.q.head + node * p.q.row;
  for (; which; which &= which - 1) {
    const int j = __ffsll((long long)which) - 1;
    const T* k = static_cast<const T*>(p.kn.data) + b * p.kn.batch + h * p.kn.head + j * p.kn.row;
    const T* v = static_cast<const T*>(p.vn.data) + b * p.vn.batch + h * p.vn.head + j * p.vn.row;
    float s = 0.0f;
    for (int d = 0; d < p.head_dim; ++d) s = fmaf(to_f32(q[d]), to_f32(k[d]), s);
    const float w = exp2f(s * (p.scale * kLog2e) - m) * inv;
    for (int d = 0; d < p.head_dim; ++d) out[d] = from_f32<T>(fmaf(w, to_f32(v[d]), to_f32(out[d])));
  }
}

// ---- 16-bit types: tensor cores -------------------------------------------------
// The rows of one key/value head (nodes x query heads on it) are the M = 128
// rows of a tile; a unit of work is (sequence, head, 128 rows), and its keys
// are tiles of 128: ceil(len / 128) of the cache, then one with the new keys.
// (A tile holds whole nodes, so it may have a few rows less.)
// Scores S = Q K^T go to tensor memory; a thread takes the scores of its row
// into registers, keeps the running maximum and sum, and puts the weights
// back as the 16-bit A operand of O += P V, O staying in tensor memory.
//
// One CTA per SM: a thread that copies K and V into a ring of slots (tiled
// copies), a thread that issues both products, and two groups of four softmax
// warps that take the unit's tiles in turn, each with its own S and O: one
// group's products and copies run under the other's exponentials.  K of the
// next tile comes before V of this one, in the order of the products.  (Over
// 128 elements there is one group, whose scores and weights share their place.)
//
// With 64 rows or fewer the rows are repeated in the tile (COPIES times), and
// a copy weighs only its share of a tile's keys, the others' weights being 0:
// the products cost the same, and the exponentials spread over all warps.
// The copies and the two groups are parts of the softmax like any split of
// the keys; they are joined in shared memory when a unit is done.
//
// The lengths are known on the device only, so the CTAs divide the list of
// all units' tiles evenly: a CTA may finish one unit, take some whole ones
// and begin another.  A unit also counts as some tiles for its start and
// its end.  A unit that more than one CTA has part of leaves (m, l, O) in the
// workspace for the second kernel.
//
// A row's reference point m follows the maximum only when that has grown by
// more than 2^8 (the weights then stay below 2^8, 2^15 in float16, which the types hold):
// O is seldom rescaled.  l sums the weights in 32 bits.  For the second
// product each weight is two numbers of the operands' type, so that the result
// is as far from the exact one as its own rounding takes it.  With one number
// the error was 1.1 to 1.4 times that; the second costs half as many products
// again (91 us instead of 98 for the first case below, 26.9 instead of 27.8).
//
// Measured: 32 nodes x 4 heads over 65536 keys of 128 (470 MB) 98 us: 49 tiles a
// CTA at 1.55 us (1.40 with one number a weight, both at 1.65 GHz, where the
// power limit has the clock), set-up 3, the unit's end 6 and joining 10.  A
// tile is 24 products of 64 cycles and three looks at barriers in the warp
// that issues them, against 1.5 us for its bytes.  21 nodes over 4001 keys of
// 64, eight ragged sequences, 27.8 us: a tile takes that warp 1600 cycles, its
// bytes would take 1420; set-up, unit ends and joining some 9 us.  Four
// sequences over 8000 keys of 256: 8 nodes and 8 heads 59 us (floor 33), 32
// nodes x 4 heads on each of 4 heads 49 us (6560 on the CUDA cores above).
struct TileMaps {
  CUtensorMap q, kc, vc, kn, vn;
};

// Two positive weights as the sum of two pairs of the type: `hi` has their
// leading bits (cut, so that what is left is exact: one byte permutation in
// bfloat16), `lo` what is left, rounded: 16 bits of each weight in bfloat16, 22
// in float16, there in multiples of 2^-24 at the finest (2^-31 of the largest weight).
template <typename T>
__device__ __forceinline__ void split2(float2 e, uint32_t& hi, uint32_t& lo) {
  constexpr uint32_t keep = std::is_same_v<T, __nv_bfloat16> ? 0xFFFF0000u : 0xFFFFE000u;
  const uint32_t u = __float_as_uint(e.x), v = __float_as_uint(e.y);
  const float2 cut = make_float2(__uint_as_float(u & keep), __uint_as_float(v & keep)), left = sub2(e, cut);
  if constexpr (std::is_same_v<T, __nv_bfloat16>)
    hi = __byte_perm(u, v, 0x7632);
  else
    hi = pack2<T>(cut.x, cut.y);
  lo = pack2<T>(left.x, left.y);
}

// by panels of 64 elements of head_dim
template <int PANELS>
struct TcShape {
  // over 128 elements tensor memory has room for one group's O, and shared
  // memory for one Q
  static constexpr int kGroups = PANELS <= 2 ? 2 : 1, kThreads = 32 * (4 * kGroups + 2);
  static constexpr int kSlots = PANELS == 1 ? 9 : PANELS == 2 ? 5 : PANELS == 3 ? 3 : 2;
  static constexpr uint32_t kTileBytes = PANELS * kPanel;
  // A buffer for Q for each group, the next unit's arriving early; 32 floats of
  // each group's 128 rows, in which a unit's parts meet at its end (but for one
  // panel its own Q); the ring; (m, l) of one group's rows, the nodes' masks of
  // two units, barriers, two words
  static constexpr uint32_t kMeet = PANELS == 1 ? 2 * kPanel : 0;
  static constexpr uint32_t kRing = PANELS == 1 ? 4 * kPanel : kGroups * kTileBytes;
  static constexpr uint32_t kExtra = kRing + kSlots * kTileBytes;
  static constexpr int kBars = 2 * kSlots + 9;
  static constexpr size_t kSmem = kExtra + kM * sizeof(float2) + 2 * kMaxNodes * 8 + kBars * 8 + 16;
};

template <typename T, int PANELS, int COPIES>
__global__ void __launch_bounds__(TcShape<PANELS>::kThreads, 1)
    attend_tc_kernel(const __grid_constant__ AttnParams p, const __grid_constant__ TileMaps maps, bool negative, float c,
                     unsigned int* __restrict__ faults) {
  using S = TcShape<PANELS>;
  constexpr int DP = 64 * PANELS, NS = S::kSlots, KQ = kKeys / COPIES, CW = 32, GR = S::kGroups;
  constexpr bool kBf = std::is_same_v<T, __nv_bfloat16>;
  extern __shared__ __align__(1024) uint8_t smem[];
  float2* const s_ml = reinterpret_cast<float2*>(smem + S::kExtra);  // [kM]
  uint64_t* const s_mask = reinterpret_cast<uint64_t*>(s_ml + kM);
  uint64_t* const s_bar = s_mask + 2 * kMaxNodes;
  unsigned long long* const s_spoiled = reinterpret_cast<unsigned long long*>(s_bar + S::kBars);
  uint32_t* const s_tmem = reinterpret_cast<uint32_t*>(s_spoiled + 1);
  const uint32_t sq = smem_addr(smem), ring = sq + S::kRing, bars = smem_addr(s_bar);
  auto full = [&](int s) { return bars + 8 * s; };
  auto empty = [&](int s) { return bars + 8 * (NS + s); };
  auto s_full = [&](int g) { return bars + 8 * (2 * NS + g); };
  auto p_ready = [&](int g) { return bars + 8 * (2 * NS + 2 + g); };
  auto q_full = [&](int i) { return bars + 8 * (2 * NS + 4 + i); };
  auto q_empty = [&](int i) { return bars + 8 * (2 * NS + 6 + i); };
  const uint32_t o_full = bars + 8 * (2 * NS + 8);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int tiles_r = (p.nodes + p.tile_nodes - 1) / p.tile_nodes, units = p.kv_heads * tiles_r;
  const int tile_rows = p.tile_rows;
  asm volatile("griddepcontrol.launch_dependents;");
  if (tid == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    for (int g = 0; g < 2; ++g) {
      mbar_init(s_full(g), 1);
      mbar_init(p_ready(g), 4);
      mbar_init(q_full(g), 1);
      mbar_init(q_empty(g), 1);
    }
    mbar_init(o_full, 1);
    *s_spoiled = 0ull;
  }
  if (warp == 4 * GR + 1) tmem_alloc(smem_addr(s_tmem), kTmemCols);
  // this CTA's entries [w0, w1) of the list
  int first;
  auto entries_of = [&](int b) { return tiles_of(p, b) + p.unit_cost; };
  const int entries = list_sum(p.batch, entries_of, first) * units;
  const int w0 = list_start(entries, blockIdx.x, gridDim.x), w1 = list_start(entries, blockIdx.x + 1, gridDim.x);
  const ListPlace begin = list_find(p.batch, units, w0, first, entries_of);
  Cursor at = {begin.b, begin.unit, begin.entry - p.unit_cost, begin.entries - p.unit_cost};
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  const uint32_t tmem = *s_tmem;  // S of every group, then O of every group
  // the tiles of this CTA in the unit at `at`, from tile at.tile on; none
  // where the CTA has only the unit's start
  auto tiles_here = [&](int& w) {
    const int skip = max(0, min(-at.tile, w1 - w));
    at.tile += skip;
    w += skip;
    return max(0, min(at.tiles - at.tile, w1 - w));
  };
  bool fine = true;  // no wait gave up
  if (warp == 4 * GR) {
    // ---- copies
    if (lane == 0) {
      tile_prefetch(&maps.q);
      tile_prefetch(&maps.kc);
      tile_prefetch(&maps.vc);
      int k = 0, u = 0;  // tiles of keys or values and units whose copies are issued
      for (int w = w0; w < w1 && fine;) {
        const int n = tiles_here(w), h = at.unit / tiles_r;
        auto load = [&](int tile, bool value) {
          const int s = k % NS;
          if (k >= NS && !mbar_wait_short(empty(s), ((k / NS) - 1) & 1)) return fine = false;
          const bool tree = tile == at.tiles - 1;
          const CUtensorMap* m = tree ? (value ? &maps.vn : &maps.kn) : (value ? &maps.vc : &maps.kc);
          mbar_expect_tx(full(s), S::kTileBytes);
#pragma unroll
          for (int x = 0; x < PANELS; ++x)
            tile_load(ring + s * S::kTileBytes + x * kPanel, m, 64 * x, tree ? 0 : tile * kKeys, h, at.b, full(s));
          ++k;
          return true;
        };
        if (n) {
          const int i = u % GR;
          if (u >= GR && !(fine = mbar_wait_short(q_empty(i), (u / GR - 1) & 1))) break;
          ++u;
          mbar_expect_tx(q_full(i), COPIES * PANELS * tile_rows * 128);
#pragma unroll
          for (int x = 0; x < COPIES * PANELS; ++x)
            tile_load(sq + i * S::kTileBytes + (x % PANELS) * kPanel + (x / PANELS) * (kPanel / COPIES), &maps.q,
                      64 * (x % PANELS), h * p.group, at.unit % tiles_r * p.tile_nodes, at.b, q_full(i));
          load(at.tile, false);
        }
        // in the order of the products
        for (int t = 0; t < n && fine; ++t) {
          if (GR == 2 && t + 1 < n && !load(at.tile + t + 1, false)) break;
          if (load(at.tile + t, true) && GR == 1 && t + 1 < n) load(at.tile + t + 1, false);
        }
        w += n;
        at.next_unit(p, units);
      }
      // copies still in flight land before the CTA ends
      for (int j = k > NS ? k - NS : 0; j < k; ++j) fine = mbar_wait_short(full(j % NS), (j / NS) & 1) && fine;
      for (int j = u > GR ? u - GR : 0; j < u; ++j) fine = mbar_wait_short(q_full(j % GR), j / GR & 1) && fine;
    }
  } else if (warp == 4 * GR + 1) {
    // ---- products, by the whole warp in step
    constexpr uint32_t word_s = mma_word(kBf, kM, kKeys, false), word_o = mma_word(kBf, kM, DP, true);
    const uint32_t t_base = __shfl_sync(0xffffffffu, tmem, 0);
    int k = 0, u = 0;
    uint32_t phase = 0;  // bit g: parity of group g's next weights
    for (int w = w0; w < w1 && fine;) {
      const int n = __shfl_sync(0xffffffffu, tiles_here(w), 0);
      auto scores = [&](int g) {
        const int s = k % NS;
        if (!warp_wait(full(s), (k / NS) & 1)) return fine = false;
        tmem_fence_after();
        const uint32_t qb = sq + (u % GR) * S::kTileBytes, kb = ring + s * S::kTileBytes;
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) {
          const uint32_t off = (i / 4) * kPanel + (i % 4) * 32;
          mma_smem(t_base + 128 * g, smem_operand(qb + off, 16), smem_operand(kb + off, 16), word_s, i > 0);
        }
        mma_commit(s_full(g));
        mma_commit(empty(s));
        ++k;
        return true;
      };
      if (n) {
        fine = warp_wait(q_full(u % GR), u / GR & 1) && scores(0);
        for (int t = 0; t < n && fine; ++t) {
          // one group's next scores take the place of this tile's weights
          if (GR == 2 && t + 1 < n && !scores((t + 1) & 1)) break;
          const int g = t % GR, s = k % NS;
          if (!(fine = warp_wait_both(full(s), (k / NS) & 1, p_ready(g), phase >> g & 1))) break;
          phase ^= 1u << g;
          tmem_fence_after();
          const uint32_t vb = ring + s * S::kTileBytes;
#pragma unroll
          for (int i = 0; i < kKeys / 16; ++i) {
            const uint64_t v = smem_operand(vb + 2048 * i, kPanel);
            mma_tmem(t_base + 128 * (GR + g), t_base + 128 * g + 16 * i, v, word_o, i > 0 || t >= GR);
            mma_tmem(t_base + 128 * (GR + g), t_base + 128 * g + 16 * i + 8, v, word_o, true);
          }
          mma_commit(empty(s));
          ++k;
          if (GR == 1 && t + 1 < n && !scores(0)) break;
        }
        if (fine) mma_commit(o_full);
        ++u;
      }
      w += n;
      at.next_unit(p, units);
    }
  } else {
    // ---- softmax: group g, tensor-memory lane L, that is row `row` of the
    // unit's rows and part `part` of every tile's keys
    const int g = warp >> 2, quarter = warp & 3, L = quarter * 32 + lane;
    const int part = COPIES == 4 ? quarter : COPIES == 2 ? quarter >> 1 : 0;
    const int r0 = COPIES == 4 ? lane : COPIES == 2 ? L & 63 : L;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const uint32_t t_s = tmem + 128 * g + lanes, t_o = tmem + 128 * (GR + g) + lanes;
    int k = 0, u = 0;  // k: tiles of keys and values before this unit's
    uint32_t phase = 0;
    // The parents of the next unit's nodes are read before this unit's tiles
    // and become masks at its end: a read among the copies' traffic takes
    // thousands of cycles.
    TreeReader reader;
    if (warp == 0 && w0 < w1) {
      reader.read(p.parents + (size_t)at.b * p.nodes, p.nodes);
      reader.masks(s_mask, reinterpret_cast<int*>(s_ml));
    }
    for (int w = w0; w < w1 && fine;) {
      const int n = tiles_here(w);
      if (n == 0) break;  // only a unit's start is left
      const int b = at.b, h = at.unit / tiles_r, node0 = at.unit % tiles_r * p.tile_nodes;
      const int here = min(p.tile_nodes, p.nodes - node0) * p.group;  // rows of this unit
      const bool mine = r0 < here;
      const int node = mine ? node0 + r0 / p.group : 0, qh = h * p.group + (mine ? r0 % p.group : 0);
      uint64_t* const masks = s_mask + (u & 1) * kMaxNodes;
      Cursor then = at;
      then.next_unit(p, units);
      const bool more = w + n < w1;
      if (warp == 0 && more) reader.read(p.parents + (size_t)then.b * p.nodes, p.nodes);
      group_sync(1, 128 * GR);
      const uint64_t mask = mine ? masks[node] : 0ull;
      const int len = length_of(p, b);
      float m = -INFINITY, l = 0.0f;
#pragma unroll 1
      for (int t = g; t < n; t += GR) {
        const int tile = at.tile + t;
        const bool tree = tile == at.tiles - 1;
        const int nk = tree ? p.nodes : min(kKeys, len - tile * kKeys);
        if (!(fine = warp_wait(s_full(g), phase))) break;
        phase ^= 1u;
        if (tree || nk < kKeys) {
          // the values of keys that no row sees are taken out of the product,
          // and those of new keys that are not finite, which only some see.  (The
          // copy that had the slot before was used ahead of this tile's scores,
          // so the wait cannot take its arrival for this one's.)
          const int kv = k + (GR == 2 && t + 1 < n ? 2 * t + 2 : 2 * t + 1);
          if (!(fine = warp_wait(full(kv % NS), (kv / NS) & 1))) break;
          uint8_t* vs = smem + S::kRing + (kv % NS) * S::kTileBytes;
          for (int r = tree ? L : nk + L; r < (tree ? p.nodes : kKeys); r += kM) {
            bool out = !tree || masks[r] == 0ull;
            if (!out) {
#pragma unroll
              for (int i = 0; i < DP / 8; ++i)
                out |= not_finite<T>(*reinterpret_cast<const uint4*>(vs + (i / 8) * kPanel + r * 128 +
                                                                     (((i % 8) ^ (r & 7)) << 4)));
              if (out) atomicOr(s_spoiled, 1ull << r);
            }
            if (out)
#pragma unroll
              for (int i = 0; i < DP / 8; ++i)
                *reinterpret_cast<uint4*>(vs + (i / 8) * kPanel + r * 128 + ((i % 8) << 4)) = make_uint4(0, 0, 0, 0);
          }
          smem_fence_async();
        }
        tmem_fence_after();
        uint32_t x[KQ];
        tmem_load<KQ>(t_s + part * KQ, x);
        tmem_wait_load();
        if (negative) {  // scores of -q
#pragma unroll
          for (int i = 0; i < KQ; ++i) x[i] ^= 0x80000000u;
        }
        if (tree) {
          const uint64_t seen = part * KQ < kMaxNodes ? mask >> (part * KQ) : 0ull;
#pragma unroll
          for (int i = 0; i < KQ; ++i)
            if (i >= kMaxNodes || !(seen >> (i & 63) & 1)) x[i] = __float_as_uint(-INFINITY);
        } else if (nk < kKeys) {
#pragma unroll
          for (int i = 0; i < KQ; ++i)
            if (part * KQ + i >= nk) x[i] = __float_as_uint(-INFINITY);
        }
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < KQ; ++i) mx4[i & 3] = fmaxf(mx4[i & 3], __uint_as_float(x[i]));
        const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
        const float top = mx == -INFINITY ? mx : fmaf(mx, c, -kBelow<T>);
        float f = 1.0f;
        if (top > m + kSlack || m == -INFINITY) {
          f = m == -INFINITY ? 0.0f : ex2(m - top);
          m = top;
          l *= f;
        }
        if (t >= GR && __any_sync(0xffffffffu, f != 1.0f)) {
          // the sums so far, on the new reference point
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
        const float ref = m == -INFINITY ? 0.0f : m;
        // 16 keys' weights take the place of their scores: 8 columns of pairs
        // rounded to the type and 8 of what that left
        float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int i0 = 0; i0 < KQ; i0 += 16) {
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            const float2 s2 = fma2(make_float2(__uint_as_float(x[i0 + i]), __uint_as_float(x[i0 + i + 1])),
                                   make_float2(c, c), make_float2(-ref, -ref));
            const float2 e = make_float2(ex2(s2.x), ex2(s2.y));
            sum = add2(sum, e);
            split2<T>(e, w[i / 2], w[i / 2 + 8]);
          }
          tmem_store<16>(t_s + part * KQ + i0, w);
        }
        l += sum.x + sum.y;
        if constexpr (COPIES > 1) {
          uint32_t zero[KQ];
#pragma unroll
          for (int i = 0; i < KQ; ++i) zero[i] = 0u;
#pragma unroll
          for (int i = 0; i < COPIES; ++i)
            if (i != part) tmem_store<KQ>(t_s + i * KQ, zero);
        }
        tmem_wait_store();
        tmem_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_ready(g));
      }
      fine = fine && warp_wait(o_full, u & 1);
      tmem_fence_after();
      // join the parts of each row: reference point and sum first
      // [GR][kM][CW], 16-byte pieces swizzled; before that the second group's (m, l)
      float4* const buf = reinterpret_cast<float4*>(smem + (PANELS == 1 ? S::kMeet : (u % GR) * S::kTileBytes));
      float2* const ml[2] = {s_ml, reinterpret_cast<float2*>(buf)};
      ml[g][L] = make_float2(m, l);
      if (!(fine = group_all(1, 128 * GR, fine))) break;
      float top = -INFINITY, total = 0.0f;
#pragma unroll
      for (int i = 0; i < GR * COPIES; ++i) top = fmaxf(top, ml[i % GR][i / GR * (kM / COPIES) + r0].x);
      const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
      for (int i = 0; i < GR * COPIES; ++i) {
        const float2 e = ml[i % GR][i / GR * (kM / COPIES) + r0];
        total = fmaf(e.y, ex2(e.x - ref), total);
      }
      const float f = ex2(m - ref);
      const bool some = g < n;  // a group without a tile has no sums
      const bool whole = at.tile == 0 && n == at.tiles, seen = mask != 0ull;  // a padding node's row is empty
      const float inv = total != 0.0f && seen ? 1.0f / total : 0.0f;
      const unsigned long long spoiled = *s_spoiled;
      // part of a unit: slot 1 holds a unit's beginning, slot 0 what follows
      float* const keep = p.part + (size_t)(2 * blockIdx.x + (at.tile == 0 ? 1 : 0)) * tile_rows * (DP + 4);
      const bool leads = g == 0 && part == 0 && mine;  // one thread of each row
      group_sync(1, 128 * GR);
      // every row's factor, 0 for one that sees nothing, in the place of its first part's m
      if (leads) s_ml[r0] = make_float2(whole ? inv : 1.0f, seen || !whole ? 1.0f : 0.0f);
      auto place = [&](int gg, int ll, int piece) { return (gg * kM + ll) * (CW / 4) + (piece ^ (ll & 7)); };
#pragma unroll 1
      for (int i = 0; i < DP; i += CW) {
        uint32_t o[CW];
        tmem_load<CW>(t_o + i, o);
        tmem_wait_load();
#pragma unroll
        for (int j = 0; j < CW / 4; ++j) {
          float4 e;
          e.x = some ? __uint_as_float(o[4 * j]) * f : 0.0f;
          e.y = some ? __uint_as_float(o[4 * j + 1]) * f : 0.0f;
          e.z = some ? __uint_as_float(o[4 * j + 2]) * f : 0.0f;
          e.w = some ? __uint_as_float(o[4 * j + 3]) * f : 0.0f;
          buf[place(g, L, j)] = e;
        }
        group_sync(1, 128 * GR);
        // neighbouring threads take neighbouring pieces of a row
        for (int x = tid; x < here * (CW / 4); x += 128 * GR) {
          const int r = x / (CW / 4), j = x % (CW / 4), d = i + 4 * j;
          float4 e = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
          for (int q = 0; q < GR * COPIES; ++q) {
            const float4 y = buf[place(q % GR, q / GR * (kM / COPIES) + r, j)];
            e.x += y.x, e.y += y.y, e.z += y.z, e.w += y.w;
          }
          if (!whole) {
            *reinterpret_cast<float4*>(keep + r * (DP + 4) + d) = e;
          } else if (d < p.head_dim) {
            const float2 k2 = s_ml[r];
            if (k2.y == 0.0f) e = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            T* dst = out_row<T>(p, b, node0 + r / p.group, h * p.group + r % p.group) + d;
            *reinterpret_cast<uint2*>(dst) =
                make_uint2(pack2<T>(e.x * k2.x, e.y * k2.x), pack2<T>(e.z * k2.x, e.w * k2.x));
          }
        }
        group_sync(1, 128 * GR);
      }
      if (leads) {
        if (whole) {
          if (spoiled & mask)
            add_spoiled<T>(p, b, h, node, qh, spoiled & mask, top, inv, out_row<T>(p, b, node, qh));
          p.lse[((size_t)b * p.nodes + node) * p.kv_heads * p.group + qh] =
              total != 0.0f && seen ? kLn2 * (top + log2f(total)) : -INFINITY;
        } else {
          *reinterpret_cast<float4*>(keep + r0 * (DP + 4) + DP) =
              make_float4(top, total, __uint_as_float((uint32_t)spoiled), __uint_as_float((uint32_t)(spoiled >> 32)));
        }
      }
      if (tid == 0) {
        *s_spoiled = 0ull;
        if constexpr (PANELS > 1) smem_fence_async();  // the copy of a later Q follows the sums that met here
        mbar_arrive(q_empty(u % GR));
      }
      ++u;
      if (warp == 0 && more) reader.masks(s_mask + (u & 1) * kMaxNodes, reinterpret_cast<int*>(s_ml));
      tmem_fence_before();
      k += 2 * n;
      w += n;
      at = then;
    }
  }
  if (!fine && (warp < 4 * GR || lane == 0)) atomicAdd(faults, 1u);
  tmem_fence_before();
  __syncthreads();
  if (warp == 4 * GR + 1) {
    __syncwarp();
    tmem_free(tmem, kTmemCols);
  }
}

// Eight warps meet after waits of which one lane's, in warp `starved`, can only
// run out: seen[w] is 1 where warp w went on and 2 where it left.
__global__ void group_wait_probe_kernel(int starved, int* __restrict__ seen, unsigned int* __restrict__ faults) {
  __shared__ alignas(8) uint64_t s_bar[2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t bars = smem_addr(s_bar);
  if (threadIdx.x == 0) {
    mbar_init(bars, 1);
    mbar_init(bars + 8, 1);
  }
  __syncthreads();
  if (threadIdx.x == 0) mbar_arrive(bars);
  const bool ok = group_all(1, blockDim.x, warp_wait(bars + (warp == starved && lane == 5 ? 8 : 0), 0));
  if (lane == 0) {
    seen[warp] = ok ? 1 : 2;
    if (!ok) atomicAdd(faults, 1u);
  }
}

// joins the parts of the units that several CTAs share; a warp per row
template <typename T, int PANELS>
__global__ void __launch_bounds__(256) join_list_kernel(const __grid_constant__ AttnParams p, int ctas) {
  constexpr int DP = 64 * PANELS;
  __shared__ uint64_t s_mask[8][kMaxNodes];
  __shared__ int s_jump[8][kMaxNodes];
  const int rows = p.nodes * p.group;
  const int tile_rows = p.tile_rows, tiles_r = (rows + tile_rows - 1) / tile_rows, units = p.kv_heads * tiles_r;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per = (rows + 7) / 8;  // CTAs of a (sequence, head)
  const int bh = blockIdx.x / per, row = blockIdx.x % per * 8 + warp;
  const int b = bh / p.kv_heads, h = bh % p.kv_heads;
  if (row >= rows) {
    CKKS_PDL_ENTRY();
    return;
  }
  const int unit = h * tiles_r + row / tile_rows, r = row % tile_rows;
  // the reads that wait for nothing first: this kernel is a chain of them
  TreeReader reader;
  reader.read(p.parents + (size_t)b * p.nodes, p.nodes);
  // this unit's tiles [u0, u1) of the list, and the CTAs that have the first
  // and the last: CTA i begins at list_start(i), so w is CTA
  // floor((ctas (w + 1) - 1) / entries)'s
  int before = 0, all = 0;
  for (int i = lane; i < p.batch; i += 32) {
    const int t = tiles_of(p, i) + p.unit_cost;
    all += t;
    if (i < b) before += t;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    all += __shfl_xor_sync(0xffffffffu, all, o);
    before += __shfl_xor_sync(0xffffffffu, before, o);
  }
  const int tiles = tiles_of(p, b);
  const long long W = (long long)all * units;
  const long long u0 = (long long)before * units + unit * (tiles + p.unit_cost) + p.unit_cost;
  const int c0 = (int)((ctas * (u0 + 1) - 1) / W), c1 = (int)((ctas * (u0 + tiles) - 1) / W);
  if (c0 == c1) {
    CKKS_PDL_ENTRY();
    return;
  }
  const int node = row / p.group, qh = h * p.group + row % p.group;
  CKKS_PDL_ENTRY();  // what is read above no kernel of this call writes
  auto part = [&](int i) { return p.part + ((size_t)(2 * i + (i == c0 ? 1 : 0)) * tile_rows + r) * (DP + 4); };
  // with fewer entries than CTAs some have none and wrote nothing
  auto idle = [&](int i) { return W < ctas && list_start((int)W, i, ctas) == list_start((int)W, i + 1, ctas); };
  // A lane has the (m, l) of one part; more than 32 parts (one sequence over a
  // whole wave) come in rounds on a growing reference point.  The parts'
  // sums are read eight at a time, so that a row waits for memory twice.
  float m = -INFINITY, l = 0.0f, x[2 * PANELS];
  unsigned long long spoiled = 0ull;
#pragma unroll
  for (int j = 0; j < 2 * PANELS; ++j) x[j] = 0.0f;
  for (int i0 = c0; i0 <= c1; i0 += 32) {
    const int mine = i0 + lane, n = min(32, c1 - i0 + 1);
    const bool real = mine <= c1 && !idle(mine);
    const float4 e = real ? *reinterpret_cast<const float4*>(part(mine) + DP) : make_float4(-INFINITY, 0.f, 0.f, 0.f);
    const uint32_t there = __ballot_sync(0xffffffffu, real);
    if (i0 == c0) reader.masks(s_mask[warp], s_jump[warp]);  // while the read above is on its way
    float top = e.x;
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    spoiled |= (unsigned long long)__reduce_or_sync(0xffffffffu, __float_as_uint(e.z)) |
               (unsigned long long)__reduce_or_sync(0xffffffffu, __float_as_uint(e.w)) << 32;
    const float up = fmaxf(m, top), ref = up == -INFINITY ? 0.0f : up, old = exp2f(m - ref), f = exp2f(e.x - ref);
    float sum = e.y * f;
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    l = fmaf(l, old, sum);
    m = up;
#pragma unroll
    for (int j = 0; j < 2 * PANELS; ++j) x[j] *= old;
    for (int i = 0; i < n; i += 8) {
      float y[8][2 * PANELS];
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const bool is = i + q < 32 && (there >> ((i + q) & 31) & 1);
        const float* o = part(i0 + i + q);
#pragma unroll
        for (int j = 0; j < 2 * PANELS; ++j) y[q][j] = is ? o[lane + 32 * j] : 0.0f;
      }
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const float fq = __shfl_sync(0xffffffffu, f, (i + q) & 31);
#pragma unroll
        for (int j = 0; j < 2 * PANELS; ++j) x[j] = fmaf(y[q][j], fq, x[j]);
      }
    }
  }
  const uint64_t mask = s_mask[warp][node];
  const bool seen = mask != 0ull;
  const float inv = l != 0.0f && seen ? 1.0f / l : 0.0f;
  T* o = out_row<T>(p, b, node, qh);
#pragma unroll
  for (int j = 0; j < 2 * PANELS; ++j)
    if (lane + 32 * j < p.head_dim) o[lane + 32 * j] = from_f32<T>(seen ? x[j] * inv : 0.0f);
  __syncwarp();
  if (lane == 0) {
    if (spoiled & mask) add_spoiled<T>(p, b, h, node, qh, spoiled & mask, m, inv, o);
    p.lse[((size_t)b * p.nodes + node) * p.kv_heads * p.group + qh] =
        l != 0.0f && seen ? kLn2 * (m + log2f(l)) : -INFINITY;
  }
}

// ---- float32: CUDA cores --------------------------------------------------------
// A unit is (sequence, head, RT rows); the CTAs divide the list of all units'
// key tiles evenly, as above.  A tile of KT keys (the cached and then the new
// ones) and its values arrive in one of two stages by asynchronous copies
// while the other is worked on; three CTAs share an SM for heads of up to 64
// elements (71 to 75 KB each), two for wider ones (56 to 76 KB).
// Scores: a thread has one key and RPT rows, so an element of K from shared
// memory feeds RPT multiply-adds and those of q are broadcasts.  Values: 16
// threads across each 64 elements, eight across the tile's keys, each with the
// sums of all RT rows in registers, which meet when the unit is done.  The
// products are plain float32 multiply-adds: a 32-bit cache is kept for its
// accuracy.  Bound by issue slots: 5 rows over 6000 keys of 64 take 40.2 us
// (3.0 TB/s, 1.34 instructions a cycle from 12 warps an SM).
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_close() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <int RT, int DC>
struct F32Shape {
  static constexpr int KT = DC == 1 ? 64 : DC == 2 ? 32 : 16, DP = 64 * DC;
  static constexpr int KS = DP + 4;                  // stride of K's rows: reads without conflicts
  static constexpr int kStage = KT * KS + KT * DP;  // floats
  static constexpr int kCtas = DC == 1 ? 3 : 2;  // on an SM
  static constexpr size_t kSmem = sizeof(float) * (2 * kStage + RT * DP + KT * RT + 3 * RT) + (kMaxNodes + RT) * 8;
  static_assert(kCtas * (kSmem + 1024) <= 228 << 10, "the CTAs that a launch counts on fit an SM");
  static_assert(KT * RT >= kMaxNodes, "the masks' scratch fits the scores' place");
  static_assert(sizeof(float) * 8 * RT * 64 <= sizeof(float) * 2 * kStage, "a unit's sums meet in the stages");
};

template <int RT, int DC>
__global__ void __launch_bounds__(kThreads, F32Shape<RT, DC>::kCtas) attend_f32_kernel(const __grid_constant__ AttnParams p) {
  using S = F32Shape<RT, DC>;
  constexpr int KT = S::KT, DP = S::DP, KS = S::KS, KG = kThreads / KT, RPT = RT / KG;  // row groups, rows of a thread
  extern __shared__ __align__(16) float sm[];
  float* const sq = sm + 2 * S::kStage;  // [RT][DP]
  float* const sp = sq + RT * DP;        // [KT][RT]
  float* const s_m = sp + KT * RT;       // running maximum, sum and this tile's factor of each row
  float* const s_l = s_m + RT;
  float* const s_c = s_l + RT;
  uint64_t* const s_mask = reinterpret_cast<uint64_t*>(s_c + RT);
  uint64_t* const s_row = s_mask + kMaxNodes;  // the masks of a unit's rows
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rows = p.nodes * p.group, tiles_r = (rows + RT - 1) / RT, units = p.kv_heads * tiles_r, D = p.head_dim;
  asm volatile("griddepcontrol.launch_dependents;");
  int first;
  auto entries_of = [&](int b) { return tiles_of(p, b) + p.unit_cost; };
  const int entries = list_sum(p.batch, entries_of, first) * units;
  const int w0 = list_start(entries, blockIdx.x, gridDim.x), w1 = list_start(entries, blockIdx.x + 1, gridDim.x);
  if (w0 >= w1) return;
  const ListPlace begin = list_find(p.batch, units, w0, first, entries_of);
  Cursor at = {begin.b, begin.unit, begin.entry - p.unit_cost, begin.entries - p.unit_cost};
  const int key = tid % KT, rg = tid / KT;  // scores: this thread's key of the tile and rows RPT rg ..
  const int dg = tid & 15, kg = tid >> 4;   // values: this thread's elements and every eighth key
  int masks_of = -1;
  for (int w = w0; w < w1;) {
    const int skip = max(0, min(-at.tile, w1 - w));
    at.tile += skip;
    w += skip;
    const int n = max(0, min(at.tiles - at.tile, w1 - w));
    if (n == 0) break;  // only a unit's start is left
    const int b = at.b, h = at.unit / tiles_r, row0 = at.unit % tiles_r * RT;
    const int len = length_of(p, b), total = len + p.nodes;
    const float* kc = static_cast<const float*>(p.kc.data) + b * p.kc.batch + h * p.kc.head;
    const float* vc = static_cast<const float*>(p.vc.data) + b * p.vc.batch + h * p.vc.head;
    const float* kn = static_cast<const float*>(p.kn.data) + b * p.kn.batch + h * p.kn.head;
    const float* vn = static_cast<const float*>(p.vn.data) + b * p.vn.batch + h * p.vn.head;
    // a thread copies the same elements of every RS-th key
    constexpr int kAcross = DC == 1 ? 16 : DC == 2 ? 32 : 64, RS = kThreads / kAcross;
    static_assert(KT % RS == 0 && 4 * kAcross >= DP, "whole rounds of whole rows");
    const int cr = tid / kAcross, cd = tid % kAcross * 4;
    auto load = [&](int t, int stage) {
      const int t0 = (at.tile + t) * KT;
      uint32_t k_at = smem_addr(sm + stage * S::kStage) + 4 * (cr * KS + cd);
      uint32_t v_at = smem_addr(sm + stage * S::kStage + KT * KS) + 4 * (cr * DP + cd);
      if (cd >= DP) {
        // 192 elements: a quarter of the threads has none
      } else if (t0 + KT <= len) {
        const float *k = kc + (t0 + cr) * p.kc.row + cd, *v = vc + (t0 + cr) * p.vc.row + cd;
        const bool real = cd < D;
        if (!real) k = kc, v = vc;
#pragma unroll
        for (int r = 0; r < KT; r += RS, k_at += 4 * RS * KS, v_at += 4 * RS * DP) {
          copy16(k_at, k, real);
          copy16(v_at, v, real);
          if (real) k += RS * p.kc.row, v += RS * p.vc.row;
        }
      } else {
        for (int r = 0; r < KT; r += RS, k_at += 4 * RS * KS, v_at += 4 * RS * DP) {
          const int s = t0 + cr + r;
          const bool cached = s < len, real = cd < D && s < total && (cached || s_mask[s - len] != 0ull);
          const float *k = static_cast<const float*>(p.q.data), *v = k;  // not read where nothing is there
          if (real) {
            k = (cached ? kc + s * p.kc.row : kn + (s - len) * p.kn.row) + cd;
            v = (cached ? vc + s * p.vc.row : vn + (s - len) * p.vn.row) + cd;
          }
          copy16(k_at, k, real);
          copy16(v_at, v, real);
        }
      }
      copies_close();
    };
    if (masks_of != b && warp == 0) tree_masks(p.parents + (size_t)b * p.nodes, p.nodes, s_mask, reinterpret_cast<int*>(sp));
    masks_of = b;
    if (tid < RT) s_m[tid] = -INFINITY, s_l[tid] = 0.0f;
    __syncthreads();
    if (tid < RT) s_row[tid] = row0 + tid < rows ? s_mask[(row0 + tid) / p.group] : 0ull;  // used behind a barrier
    load(0, 0);
    for (int i = tid; i < RT * (DP / 4); i += kThreads) {
      const int r = i / (DP / 4), d = i % (DP / 4) * 4, row = row0 + r;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (row < rows && d < D)
        x = *reinterpret_cast<const float4*>(static_cast<const float*>(p.q.data) + b * p.q.batch +
                                             (h * p.group + row % p.group) * p.q.head + (row / p.group) * p.q.row + d);
      const float c = p.scale * kLog2e;
      *reinterpret_cast<float4*>(sq + r * DP + d) = make_float4(x.x * c, x.y * c, x.z * c, x.w * c);
    }
    float acc[DC][RT][4];
#pragma unroll
    for (int c = 0; c < DC; ++c)
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[c][r][e] = 0.0f;
    for (int t = 0; t < n; ++t) {
      const int t0 = (at.tile + t) * KT, nk = min(KT, total - t0);
      if (t + 1 < n) {
        load(t + 1, (t + 1) & 1);
        copies_wait<1>();
      } else {
        copies_wait<0>();
      }
      __syncthreads();
      const float* sk = sm + (t & 1) * S::kStage;
      const float* sv = sk + KT * KS;
      {
        float x[RPT];
#pragma unroll
        for (int r = 0; r < RPT; ++r) x[r] = 0.0f;
#pragma unroll 8
        for (int d = 0; d < DP; d += 4) {
          const float4 k4 = *reinterpret_cast<const float4*>(sk + key * KS + d);
#pragma unroll
          for (int r = 0; r < RPT; ++r) {
            const float4 q4 = *reinterpret_cast<const float4*>(sq + (RPT * rg + r) * DP + d);
            x[r] = fmaf(k4.x, q4.x, fmaf(k4.y, q4.y, fmaf(k4.z, q4.z, fmaf(k4.w, q4.w, x[r]))));
          }
        }
        const int s = t0 + key;
        if (t0 + KT > len) {
#pragma unroll
          for (int r = 0; r < RPT; ++r) {
            const uint64_t m = s_row[RPT * rg + r];
            if (!(key < nk && m && (s < len || (m >> (s - len) & 1)))) x[r] = -INFINITY;
          }
        }
#pragma unroll
        for (int r = 0; r < RPT; ++r) sp[key * RT + RPT * rg + r] = x[r];
      }
      __syncthreads();
      // running maximum and sum: a warp has RT / 4 rows
#pragma unroll
      for (int j = 0; j < RT / 4; ++j) {
        const int r = warp * (RT / 4) + j;
        constexpr int KL = (KT + 31) / 32;
        float x[KL];
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < KL; ++i) {
          x[i] = lane + 32 * i < KT ? sp[(lane + 32 * i) * RT + r] : -INFINITY;
          mx = fmaxf(mx, x[i]);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float old = s_m[r], m = fmaxf(old, mx), base = m == -INFINITY ? 0.0f : m;
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < KL; ++i) {
          const int at = t0 + lane + 32 * i;
          x[i] = exp2f(x[i] - base);
          sum += x[i];
          if (at >= len && !(at < total && (s_row[r] >> (at - len) & 1))) x[i] = __uint_as_float(kUnseen);
          if (lane + 32 * i < KT) sp[(lane + 32 * i) * RT + r] = x[i];
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) {
          const float f = exp2f(old - base);
          s_m[r] = m;
          s_l[r] = s_l[r] * f + sum;
          s_c[r] = f;
        }
      }
      __syncthreads();
      bool same = true;
#pragma unroll
      for (int r = 0; r < RT; ++r) same = same && s_c[r] == 1.0f;
      if (!same) {
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const float f = s_c[r];
#pragma unroll
          for (int c = 0; c < DC; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[c][r][e] *= f;
        }
      }
      auto values = [&](auto apart) {
#pragma unroll
        for (int i = 0; i < KT / 8; ++i) {
          const int k = kg + 8 * i;
          float x[RT];
#pragma unroll
          for (int r = 0; r < RT; r += 4)
            *reinterpret_cast<float4*>(x + r) = *reinterpret_cast<const float4*>(sp + k * RT + r);
#pragma unroll
          for (int c = 0; c < DC; ++c) {
            const float4 v4 = *reinterpret_cast<const float4*>(sv + k * DP + c * 64 + dg * 4);
#pragma unroll
            for (int r = 0; r < RT; ++r)
              if (!decltype(apart)::value || __float_as_uint(x[r]) != kUnseen) {
                acc[c][r][0] = fmaf(x[r], v4.x, acc[c][r][0]);
                acc[c][r][1] = fmaf(x[r], v4.y, acc[c][r][1]);
                acc[c][r][2] = fmaf(x[r], v4.z, acc[c][r][2]);
                acc[c][r][3] = fmaf(x[r], v4.w, acc[c][r][3]);
              }
          }
        }
      };
      // a new key's values, whatever they hold, reach the rows that see it only
      if (t0 + KT > len)
        values(std::true_type{});
      else
        values(std::false_type{});
      __syncthreads();
    }
    // the eight key groups' sums meet in the stages, 64 elements at a time
    const bool whole = at.tile == 0 && n == at.tiles;
    if (whole && tid < RT && row0 + tid < rows && s_mask[(row0 + tid) / p.group] == 0ull) s_l[tid] = 0.0f;  // padding
    float* const keep = p.part + (size_t)(2 * blockIdx.x + (at.tile == 0 ? 1 : 0)) * RT * (DP + 4);
#pragma unroll
    for (int c = 0; c < DC; ++c) {
#pragma unroll
      for (int r = 0; r < RT; ++r)
        *reinterpret_cast<float4*>(sm + (kg * RT + r) * 64 + dg * 4) =
            make_float4(acc[c][r][0], acc[c][r][1], acc[c][r][2], acc[c][r][3]);
      __syncthreads();
      for (int i = tid; i < RT * 64; i += kThreads) {
        const int r = i / 64, d = c * 64 + i % 64, row = row0 + r;
        if (row >= rows) continue;
        float x = 0.0f;
#pragma unroll
        for (int g = 0; g < 8; ++g) x += sm[(g * RT + r) * 64 + i % 64];
        if (!whole) {
          keep[r * (DP + 4) + d] = x;
        } else if (d < D) {
          const float l = s_l[r];
          out_row<float>(p, b, row / p.group, h * p.group + row % p.group)[d] = l != 0.0f ? x / l : 0.0f;
        }
      }
      __syncthreads();
    }
    if (tid < RT && row0 + tid < rows) {
      const int row = row0 + tid;
      if (whole)
        p.lse[((size_t)b * p.nodes + row / p.group) * p.kv_heads * p.group + h * p.group + row % p.group] =
            s_l[tid] != 0.0f ? kLn2 * (s_m[tid] + log2f(s_l[tid])) : -INFINITY;
      else
        *reinterpret_cast<float4*>(keep + tid * (DP + 4) + DP) = make_float4(s_m[tid], s_l[tid], 0.0f, 0.0f);
    }
    __syncthreads();
    w += n;
    at.next_unit(p, units);
  }
}

size_t attend_smem(int D) {
  const int D4 = (D + 3) & ~3;
  const size_t run = sizeof(float) * ((size_t)kTile * (D4 + 4) + kTile * D4 + kRows * D4 + kTile * kRows);
  const size_t red = sizeof(float) * 8 * kRows * 64;
  return run > red ? run : red;
}

template <typename T, int DC, bool FOUR>
void launch_attend(const AttnParams& p, cudaStream_t st) {
  const size_t smem = attend_smem(p.head_dim);
  auto* k = attend_kernel<T, DC, FOUR>;
  // the most that any call asks for: calls of other sizes from other threads
  // may come between this and the launch
  CKKS_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)attend_smem(64 * DC)));
  const int rows = p.nodes * p.group;
  const dim3 grid((unsigned)(p.batch * p.kv_heads * ((rows + kRows - 1) / kRows)), p.splits);
  k<<<grid, kThreads, smem, st>>>(p);
  CKKS_CUDA(cudaGetLastError());
}

template <typename T, bool FOUR>
void run_attend(const AttnParams& p, cudaStream_t st) {
  switch ((p.head_dim + 63) / 64) {
    case 1: launch_attend<T, 1, FOUR>(p, st); break;
    case 2: launch_attend<T, 2, FOUR>(p, st); break;
    case 3: launch_attend<T, 3, FOUR>(p, st); break;
    default: launch_attend<T, 4, FOUR>(p, st); break;
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
  need((long long)a.batch * a.q_heads * a.nodes < (1ll << 31) - 1 && a.capacity < (1 << 30) &&
           (long long)a.batch * a.q_heads * (a.capacity / 128 + 4) < (1ll << 31) - 1,
       "sizes too large");
}

bool tc_sizes(const ckks_draft_attention_args& a) {
  return a.dtype != CKKS_FP32 && a.head_dim % 8 == 0 && a.q_heads / a.kv_heads <= kM;
}

// nodes whose rows a tile of the tensor-core kernel holds
int tile_nodes(const ckks_draft_attention_args& a) { return std::min(a.nodes, kM / (a.q_heads / a.kv_heads)); }

// how a kernel divides its list of units
struct Division {
  int tile_rows, tile_keys, new_apart, unit_cost, ctas;
  bool alone;   // no unit is shared
  bool listed;  // the list of full caches has fewer than 2^31 - 1 entries
};

// `per_sm` CTAs on each SM, but no fewer than four tiles of keys each at the
// full capacity (a shorter part is all start-up), and one for each unit where
// there are fewer units than that
Division divide(const Context& c, const ckks_draft_attention_args& a, Division d, int per_sm) {
  const long long rows = (long long)a.nodes * (a.q_heads / a.kv_heads);
  const long long units = (long long)a.batch * a.kv_heads * ((rows + d.tile_rows - 1) / d.tile_rows);
  const long long tiles = units * ((a.capacity + d.tile_keys - 1) / d.tile_keys + 1);
  // the kernels count the list's entries in 32 bits
  const long long keys = (long long)a.capacity + (d.new_apart ? 0 : a.nodes);
  d.listed = units * ((keys + d.tile_keys - 1) / d.tile_keys + (d.new_apart ? 1 : 0) + d.unit_cost) < (1ll << 31) - 1;
  d.ctas = (int)std::max(1ll, std::min((long long)per_sm * c.sms, std::max(tiles / 4, units)));
  d.alone = a.batch == 1 && d.ctas == units;  // one sequence and a CTA for each unit
  return d;
}

// What a unit's start and end cost, in tiles of its keys; wider heads have
// longer tiles.  Measured with 2 / 4 / 6 / 10 tiles (us): heads of 64, 21 rows over
// 4001 keys, eight ragged sequences of 12: 36.3 / 27.6 / 28.2 / 29.8; 128 rows over
// 65536, two of 8: 78.0 / 75.7 / 75.5 / 75.5.  Heads of 128, 128 rows over 65536:
// 104 / 102 / 100 / 98.3, over 2000, eight of 8: 48.3 / 39.0 / 37.4 / 38.2; 16 rows over
// 4001, eight of 12: 49 / 39 / 38.4 / 45.  Heads of 256, 8 rows over 8000, four of 8:
// 60.0 / 61.0 / 60.3 / 64.5, over 32000: 99 / 100 / 102 / 101; of 192, 16 rows over
// 3000: 27.3 / 30.1 / 29.3 / 31.3.
Division tc_division(const Context& c, const ckks_draft_attention_args& a) {
  const int rows = tile_nodes(a) * (a.q_heads / a.kv_heads);
  return divide(c, a, Division{rows, kKeys, 1, a.head_dim <= 64 ? 4 : a.head_dim <= 128 ? 6 : 2, 0, false, false}, 1);
}

bool f32_sizes(const ckks_draft_attention_args& a) { return a.dtype == CKKS_FP32 && a.head_dim % 4 == 0; }

// 16 rows in a unit where there are more than 8: K and V come from memory or
// L2 once for all of them.  Wide heads have no registers for that.
int f32_rows(const ckks_draft_attention_args& a) {
  return a.head_dim <= 128 && a.nodes * (a.q_heads / a.kv_heads) > 8 ? 16 : 8;
}

Division f32_division(const Context& c, const ckks_draft_attention_args& a) {
  const int dc = (a.head_dim + 63) / 64;
  return divide(c, a, Division{f32_rows(a), dc == 1 ? 64 : dc == 2 ? 32 : 16, 0, 1, 0, false, false}, dc == 1 ? 3 : 2);
}

size_t division_floats(const ckks_draft_attention_args& a, const Division& d) {
  return d.alone ? 0 : (size_t)2 * d.ctas * d.tile_rows * ((a.head_dim + 63) / 64 * 64 + 4);
}

// which of the kernels that divide a list takes these sizes; a list whose
// entries 32 bits do not hold is left to the plain kernel, which has none
bool takes_tc(const Context& c, const ckks_draft_attention_args& a) { return tc_sizes(a) && tc_division(c, a).listed; }
bool takes_f32(const Context& c, const ckks_draft_attention_args& a) {
  return f32_sizes(a) && f32_division(c, a).listed;
}

size_t workspace_of(const Context& c, const ckks_draft_attention_args& a) {
  if (a.batch == 0) return 0;
  // the tensors' strides decide which kernel runs
  const int s = split_count(c, a);
  size_t n = s == 1 ? 0 : (size_t)a.batch * a.q_heads * a.nodes * s * (a.head_dim + 2);
  if (takes_tc(c, a)) n = std::max(n, division_floats(a, tc_division(c, a)));
  if (takes_f32(c, a)) n = std::max(n, division_floats(a, f32_division(c, a)));
  return sizeof(float) * n;
}

// over a 4-bit cache
size_t workspace4_of(const Context& c, const ckks_draft_attention_args& a) {
  if (a.batch == 0) return 0;
  const int s = split_count(c, a);
  // the caches' strides decide which kernel runs
  const size_t plain = s == 1 ? 0 : sizeof(float) * (size_t)a.batch * a.q_heads * a.nodes * s * (a.head_dim + 2);
  return std::max(plain, attention4_tc_workspace(c, a));
}

AttnParams with(AttnParams p, const Division& d) {
  p.tile_rows = d.tile_rows, p.tile_keys = d.tile_keys, p.new_apart = d.new_apart, p.unit_cost = d.unit_cost;
  return p;
}

template <typename T, int PANELS>
void join_division(const AttnParams& p, const Division& d, cudaStream_t st) {
  if (d.alone) return;
  const int rows = p.nodes * p.group;
  const dim3 grid((unsigned)(p.batch * p.kv_heads * ((rows + 7) / 8)));
  launch_pdl(join_list_kernel<T, PANELS>, grid, dim3(256), 0, st, p, d.ctas);
}

template <int RT, int DC>
void launch_f32(const AttnParams& p, const Division& d, cudaStream_t st) {
  using S = F32Shape<RT, DC>;
  auto* k = attend_f32_kernel<RT, DC>;
  CKKS_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::kSmem));
  k<<<d.ctas, kThreads, S::kSmem, st>>>(p);
  CKKS_CUDA(cudaGetLastError());
  join_division<float, DC>(p, d, st);
}

void run_f32(const Context& c, const ckks_draft_attention_args& a, const AttnParams& base, cudaStream_t st) {
  const Division d = f32_division(c, a);
  const AttnParams p = with(base, d);
  const bool many = d.tile_rows == 16;
  switch ((a.head_dim + 63) / 64) {
    case 1: many ? launch_f32<16, 1>(p, d, st) : launch_f32<8, 1>(p, d, st); break;
    case 2: many ? launch_f32<16, 2>(p, d, st) : launch_f32<8, 2>(p, d, st); break;
    case 3: launch_f32<8, 3>(p, d, st); break;
    default: launch_f32<8, 4>(p, d, st); break;
  }
}

template <typename T, int PANELS, int COPIES>
void launch_tc(const Context& c, const AttnParams& p, const TileMaps& maps, const Division& d, cudaStream_t st) {
  using S = TcShape<PANELS>;
  static_assert(S::kSmem <= 232448, "shared memory of one block");
  auto* k = attend_tc_kernel<T, PANELS, COPIES>;
  CKKS_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::kSmem));
  // a scale of 0 becomes one that changes no weight: a masked score times 0 would be no number
  const float factor = std::max(std::fabs(p.scale) * kLog2e, 1e-30f);
  k<<<d.ctas, S::kThreads, S::kSmem, st>>>(p, maps, p.scale < 0.0f, factor, c.d_faults);
  CKKS_CUDA(cudaGetLastError());
  join_division<T, PANELS>(p, d, st);
}

template <typename T, int PANELS>
void launch_tc(const Context& c, const ckks_draft_attention_args& a, const AttnParams& base, const TileMaps& maps,
               cudaStream_t st) {
  const Division d = tc_division(c, a);
  const AttnParams p = with(base, d);
  const int rows = p.nodes * p.group;
  if (rows <= 32)
    launch_tc<T, PANELS, 4>(c, p, maps, d, st);
  else if (rows <= 64)
    launch_tc<T, PANELS, 2>(c, p, maps, d, st);
  else
    launch_tc<T, PANELS, 1>(c, p, maps, d, st);
}

template <typename T>
bool run_tc(const Context& c, const ckks_draft_attention_args& a, const AttnParams& p, cudaStream_t st) {
  TileMaps m;
  // keys and values: 128 rows of one head
  auto rows_map = [&](CUtensorMap* t, const ckks_rows& r, int rows) {
    return tile_map(t, r.data, a.dtype, a.head_dim, rows, r.row, kKeys, a.kv_heads, r.head, 1, a.batch, r.batch);
  };
  // queries: the heads on one key/value head, of a tile's nodes
  if (!tile_map(&m.q, a.q.data, a.dtype, a.head_dim, a.q_heads, a.q.head, p.group, a.nodes, a.q.row, p.tile_nodes,
                a.batch, a.q.batch) ||
      !rows_map(&m.kn, a.k_new, a.nodes) || !rows_map(&m.vn, a.v_new, a.nodes))
    return false;
  if (a.capacity == 0) {
    m.kc = m.kn, m.vc = m.vn;  // not read
  } else if (!rows_map(&m.kc, a.k_cache, a.capacity) || !rows_map(&m.vc, a.v_cache, a.capacity)) {
    return false;
  }
  switch ((a.head_dim + 63) / 64) {
    case 1: launch_tc<T, 1>(c, a, p, m, st); break;
    case 2: launch_tc<T, 2>(c, a, p, m, st); break;
    case 3: launch_tc<T, 3>(c, a, p, m, st); break;
    default: launch_tc<T, 4>(c, a, p, m, st); break;
  }
  return true;
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

namespace {
// FOUR: the caches are 4-bit rows, strides in bytes
template <bool FOUR>
int run(ckks_ctx* ctx, const ckks_draft_attention_args* args, void* stream) {
  return guard([&] {
    Context& c = context_of(ctx);
    need(args != nullptr, "null argument");
    const ckks_draft_attention_args& a = *args;
    check_shape(a);
    need(a.reserved == 0, "reserved field is not 0");
    need(std::isfinite((float)a.scale * kLog2e), "scale is not finite");
    if (a.batch == 0) return;
    const int e = element_bytes(a.dtype);
    check_rows(a.q, e, "q");
    if (a.capacity) {
      check_rows(a.k_cache, FOUR ? 1 : e, "k_cache");
      check_rows(a.v_cache, FOUR ? 1 : e, "v_cache");
      if constexpr (FOUR) {
        check_row4(a.k_cache, a.batch, a.kv_heads, a.capacity, "k_cache");
        check_row4(a.v_cache, a.batch, a.kv_heads, a.capacity, "v_cache");
      }
    }
    check_rows(a.k_new, e, "k_new");
    check_rows(a.v_new, e, "v_new");
    check_rows(a.out, e, "out");
    check_ptr(a.lens, "lens");
    check_ptr(a.parents, "parents");
    check_ptr(a.lse, "lse");
    const size_t ws = FOUR ? workspace4_of(c, a) : workspace_of(c, a);
    need(a.workspace_bytes >= ws && (ws == 0 || a.workspace),
         FOUR ? "workspace smaller than ckks_draft_attention4_workspace" : "workspace smaller than ckks_draft_attention_workspace");
    need(reinterpret_cast<uintptr_t>(a.workspace) % 16 == 0, "workspace not aligned to 16 bytes");
    AttnParams p{};
    p.q = a.q, p.kc = a.k_cache, p.vc = a.v_cache, p.kn = a.k_new, p.vn = a.v_new, p.out = a.out;
    p.lens = a.lens, p.parents = a.parents, p.lse = a.lse, p.part = static_cast<float*>(a.workspace);
    p.batch = a.batch, p.kv_heads = a.kv_heads, p.group = a.q_heads / a.kv_heads, p.head_dim = a.head_dim;
    p.nodes = a.nodes, p.capacity = a.capacity, p.scale = (float)a.scale;
    p.splits = split_count(c, a), p.tile_nodes = tile_nodes(a);
    p.wide = wide_rows(a.q, a.batch, a.q_heads, a.nodes, a.head_dim, e) &&
             wide_rows(a.out, a.batch, a.q_heads, a.nodes, a.head_dim, e) &&
             wide_rows(a.k_new, a.batch, a.kv_heads, a.nodes, a.head_dim, e) &&
             wide_rows(a.v_new, a.batch, a.kv_heads, a.nodes, a.head_dim, e);
    if (!FOUR && a.capacity)
      p.wide = p.wide && wide_rows(a.k_cache, a.batch, a.kv_heads, a.capacity, a.head_dim, e) &&
               wide_rows(a.v_cache, a.batch, a.kv_heads, a.capacity, a.head_dim, e);
    OnDevice dev(c);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const double bytes = 2.0 * a.batch * a.kv_heads * a.capacity * (FOUR ? row4_bytes(a.head_dim) : e * a.head_dim);
    ProfScope ps(c, FOUR ? "draft_attention4" : "draft_attention", bytes, st);
    if constexpr (FOUR) {
      if (attention4_tc(c, a, st)) return;
    } else {
      // strides that no tensor map holds are left to the plain kernel
      if (p.wide && takes_tc(c, a)) {
        if (a.dtype == CKKS_BF16 ? run_tc<__nv_bfloat16>(c, a, p, st) : run_tc<__half>(c, a, p, st)) return;
      }
      if (p.wide && takes_f32(c, a)) {
        run_f32(c, a, p, st);
        return;
      }
    }
    if (a.dtype == CKKS_BF16)
      run_attend<__nv_bfloat16, FOUR>(p, st);
    else if (a.dtype == CKKS_FP16)
      run_attend<__half, FOUR>(p, st);
    else
      run_attend<float, FOUR>(p, st);
  });
}
}  // namespace

extern "C" int ckks_draft_attention(ckks_ctx* ctx, const ckks_draft_attention_args* args, void* stream) {
  return run<false>(ctx, args, stream);
}

extern "C" long long ckks_draft_attention4_workspace(ckks_ctx* ctx, const ckks_draft_attention_args* a) {
  long long n = -1;
  guard([&] {
    Context& c = context_of(ctx);
    need(a != nullptr, "null argument");
    check_shape(*a);
    n = (long long)workspace4_of(c, *a);
  });
  return n;
}

extern "C" int ckks_draft_attention4(ckks_ctx* ctx, const ckks_draft_attention_args* args, void* stream) {
  return run<true>(ctx, args, stream);
}

extern "C" int ckks_selftest_group_wait(ckks_ctx* ctx, int starved) {
  return guard([&] {
    Context& c = context_of(ctx);
    constexpr int kWarps = 8;
    int seen[kWarps] = {};
    OnDevice dev(c);
    int* d = (int*)c.alloc(sizeof(seen));
    CKKS_CUDA(cudaMemsetAsync(d, 0, sizeof(seen), c.stream));
    group_wait_probe_kernel<<<1, 32 * kWarps, 0, c.stream>>>(starved, d, c.d_faults);
    CKKS_CUDA(cudaGetLastError());
    CKKS_CUDA(cudaMemcpyAsync(seen, d, sizeof(seen), cudaMemcpyDeviceToHost, c.stream));
    CKKS_CUDA(cudaStreamSynchronize(c.stream));
    c.release(d);
    const unsigned int faults = take_device_faults(c);
    for (int w = 1; w < kWarps; ++w)
      if (seen[w] != seen[0]) throw Error(CKKS_ESTATE, "warps that met after a wait did not go on or leave together");
    if (seen[0] != 1 || faults) throw Error(CKKS_ECUDA, "bounded wait of a group of warps gave up");
  });
}
