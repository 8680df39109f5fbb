// draft_attention4.cu -- attention of a tree of drafted nodes over a 4-bit
// cache on the tensor cores (what ckks_draft_attention4 does with 16-bit rows
// and contiguous caches; draft_attention.cu has the rest).
//
// For the rows r = (node, query head) of one key/value head over the cached
// keys k < len, with the codes' values K and V (draft_fp4.cuh):
//   S^T = K Q^T,  P^T = 2^(c_r S^T - m_r),  O^T += V^T P,  l_r = sum_k P_rk.
// Few rows read many keys, so the keys are the 128 rows of the first product
// and the elements of V those of the second: their cost grows with the rows
// (4 cycles a row and 128 keys of 128), and not with 128 rows whatever there are.
//
// One CTA per SM.  A thread copies tiles of 128 keys as they are (9/16 of a
// byte an element); four warps decode K, a thread a key, into tensor memory as
// the first product's A operand, four decode V into shared memory as the
// second's; a warp for each product issues it; a group of four warps for every
// 16 rows, a thread a key, turns scores into weights.  Every step has two
// buffers, so that each works on another tile.
//
// The first product's operands have the queries' type, the second's are
// float16: either type holds the caches' values exactly, so every product of
// a query's element and a key's is exact, however far apart the elements of a
// row lie (a group of small keys may meet the large ones: rounding a bfloat16
// row to float16 would lose its small elements).  A weight
// has float16's 11 bits.  A row's reference point m lies 2^7 below the maximum
// when it is set, and is set anew where a score passes it by more than 2^8 more: weights
// end at 2^15.  Sums are in 32 bits.
//
// The lengths are known on the device only, so the CTAs divide the list of all
// units' tiles evenly, a unit being (sequence, head, up to 64 rows).  Each
// leaves (m, l, O) of its part of a unit in the workspace, and a second kernel,
// a warp or eight a row, joins them with the new keys of the row's ancestors, which it
// takes on the CUDA cores while the first kernel still runs.
//
// Measured: one node over four sequences of 65536 to 40960 keys, 32/8 heads of 128,
// bfloat16, 93 us (245 MB, 2.6 TB/s, 40 % of the copy rate; in a replayed graph 91, with
// float16 queries 84; 1326 on the CUDA cores); trees of 21 over 4001 keys, eight ragged
// sequences of 12 heads of 64, 29 us; trees of 16 over 32768 and 24576 keys, 64 rows on each
// of 8 heads, 53 us.  A tile takes about 1670 cycles with 16 rows of 128 and float16 queries,
// start and end included, where its bytes take 710: decoding V (1100 of a warp's cycles), the
// softmax warps (1000) and the two products (560, and their looks at barriers) are all near
// that, issue slots are half used and so is shared memory.  K in bfloat16 goes through floats
// and takes 8 % more.  Two sets of softmax warps that take the tiles in turns, twice as many
// warps for V, K's warps decoding some of V, and 8-byte reads of the rows all left 85 us
// where they were or at 88 to 101; with 64 rows the softmax warps' chain bounds it (2700 cycles).
#include <algorithm>
#include <cmath>

#include "draft_fp4.cuh"
#include "draft_tc.cuh"

namespace ckks {
namespace draft {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kUnset = -3.0e38f;  // reference point of a row that has seen no key

struct Params4 {
  ckks_rows q, kc, vc, kn, vn, out;
  const int32_t* lens;
  const int32_t* parents;
  float* lse;
  float* part;  // [units + CTAs][N][DP + 4]
  int batch, kv_heads, group, head_dim, nodes, capacity;
  int rows, tiles_r, unit_cost, ctas, row_bytes;  // rows of a unit, units of a (sequence, head), ...
  float scale;
};

__device__ __forceinline__ int length_of(const Params4& p, int b) { return min(max(p.lens[b], 0), p.capacity); }
// entries of a unit of sequence b in the list: its tiles, and what its start and end cost
__device__ __forceinline__ int entries_of(const Params4& p, int b) {
  const int t = (length_of(p, b) + kKeys - 1) / kKeys;
  return t ? t + p.unit_cost : 0;
}

// A part of a unit: the tiles [tile, tile + n) of sequence b's unit `unit`
struct Piece {
  int b, unit, tile, n;
};

// The pieces of one CTA, in their order; by a whole warp
struct Pieces4 {
  int w, w1, b, unit, entry, entries, units;
  __device__ __forceinline__ void begin(const Params4& p, int& all) {
    units = p.kv_heads * p.tiles_r;
    auto of = [&](int i) { return entries_of(p, i); };
    int first;
    all = list_sum(p.batch, of, first) * units;
    const int ctas = min((int)gridDim.x, all), i = blockIdx.x;
    w = w1 = 0;
    if (i >= ctas) return;
    w = list_start(all, i, ctas), w1 = list_start(all, i + 1, ctas);
    const ListPlace at = list_find(p.batch, units, w, first, of);
    b = at.b, unit = at.unit, entry = at.entry, entries = at.entries;
  }
  // false behind the last piece; a piece may have no tiles (n = 0)
  __device__ __forceinline__ bool next(const Params4& p, Piece& x) {
    if (w >= w1) return false;
    const int here = min(entries - entry, w1 - w);
    const int skip = max(0, min(p.unit_cost - entry, here));
    x = {b, unit, max(0, entry - p.unit_cost), here - skip};
    w += here;
    entry = 0;
    if (w < w1 && ++unit == units) {
      unit = 0;
      do entries = entries_of(p, ++b);
      while (entries == 0);  // w1 lies behind no sequence without keys
    }
    return true;
  }
};

// by panels of 64 elements of head_dim (1, 2 or 4) and rows of a unit
template <int PANELS, int N>
struct Shape4 {
  static constexpr int DP = 64 * PANELS;
  static constexpr int kBlocks = PANELS <= 2 ? 1 : 2;    // of 128 elements, in the second product
  static constexpr int kCols = 16, kGroups = N / kCols;  // rows that a softmax thread has; groups of four softmax warps
  static constexpr int kWarps = 4 * kGroups + 11, kThreads = 32 * kWarps;
  static constexpr int kRowMost = row4_bytes(DP);
  static constexpr uint32_t kRaw = (kKeys * kRowMost + 16 + 127) / 128 * 128;  // one tile of K or V as it is
  static constexpr int kSlots = PANELS == 1 ? 6 : PANELS == 2 ? 4 : 2;
  static constexpr uint32_t kValues = kBlocks * 2 * kPanel;                    // one decoded tile of V
  static constexpr int kValueBufs = PANELS <= 2 ? 2 : 1;
  static constexpr uint32_t kQ = PANELS * N * 128;
  static constexpr uint32_t kP = kPanel;                                       // 128 keys x up to 64 rows
  static constexpr uint32_t kAtQ = kValueBufs * kValues, kAtP = kAtQ + (kQ + 1023) / 1024 * 1024, kAtRaw = kAtP + 2 * kP;
  static constexpr uint32_t kAtRows = kAtRaw + 2 * kSlots * kRaw;              // float2 [2][N], float [5][N]
  static constexpr uint32_t kAtBars = kAtRows + N * (2 * 8 + 5 * 4);
  static constexpr int kBars = 2 * kSlots + 12;
  static constexpr size_t kSmem = kAtBars + kBars * 8 + 16;
  // tensor memory: K twice, S twice, O
  static constexpr int kColS = DP, kColO = DP + 2 * N;
  static_assert(kColO + kBlocks * N <= kTmemCols);
};

// the sum over a warp of 16 columns: lane x gets column x / 2
__device__ __forceinline__ float warp_columns(float* v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 16, n = 16; o > 1; o >>= 1) {
    // halves of the columns go to the lanes whose bit is clear and set
    const bool up = lane & o;
    n /= 2;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float give = up ? v[i] : v[i + n], keep = up ? v[i + n] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
    }
  }
  return v[0] + __shfl_xor_sync(0xffffffffu, v[0], 1);
}

// monotone integers of floats, for the largest of a warp
__device__ __forceinline__ int ordered(float x) {
  const int i = __float_as_int(x);
  return i ^ (i >> 31 & 0x7FFFFFFF);
}
__device__ __forceinline__ float unordered(int i) { return __int_as_float(i ^ (i >> 31 & 0x7FFFFFFF)); }

// T: of the queries
template <typename T, int PANELS, int N>
__global__ void __launch_bounds__(Shape4<PANELS, N>::kThreads, 1)
    attend4_kernel(const __grid_constant__ Params4 p, unsigned int* __restrict__ faults) {
  using S = Shape4<PANELS, N>;
  constexpr int DP = S::DP, NS = S::kSlots, GR = S::kGroups, C = S::kCols, VB = S::kValueBufs;
  constexpr bool kBf = std::is_same_v<T, __nv_bfloat16>;
  constexpr int kWarpK = 4 * GR, kWarpV = kWarpK + 4, kWarpCopy = kWarpV + 4, kWarpQk = kWarpCopy + 1, kWarpPv = kWarpQk + 1;
  extern __shared__ __align__(1024) uint8_t smem[];
  float2* const s_row = reinterpret_cast<float2*>(smem + S::kAtRows);      // [2][N] factor and reference point
  float* const s_max = reinterpret_cast<float*>(s_row + 2 * N);            // [4][N]
  float* const s_fac = s_max + 4 * N;                                      // [N]
  uint64_t* const s_bar = reinterpret_cast<uint64_t*>(smem + S::kAtBars);
  uint32_t* const s_tmem = reinterpret_cast<uint32_t*>(s_bar + S::kBars);
  const uint32_t base = smem_addr(smem), bars = smem_addr(s_bar);
  auto raw_full = [&](int s) { return bars + 8 * s; };
  auto raw_empty = [&](int s) { return bars + 8 * (NS + s); };
  auto k_ready = [&](int i) { return bars + 8 * (2 * NS + i); };
  auto s_full = [&](int i) { return bars + 8 * (2 * NS + 2 + i); };
  auto v_ready = [&](int i) { return bars + 8 * (2 * NS + 4 + i); };
  auto p_ready = [&](int i) { return bars + 8 * (2 * NS + 6 + i); };
  auto pv_done = [&](int i) { return bars + 8 * (2 * NS + 8 + i); };
  auto v_free = [&](int i) { return bars + 8 * (2 * NS + 8 + (VB == 2 ? i : 2)); };
  const uint32_t q_ready = bars + 8 * (2 * NS + 11);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  asm volatile("griddepcontrol.launch_dependents;");
  if (tid == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(raw_full(s), 1);
      mbar_init(raw_empty(s), 8);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(k_ready(i), 4);
      mbar_init(s_full(i), 1);
      mbar_init(v_ready(i), 4);
      mbar_init(p_ready(i), 4 * GR);
      mbar_init(pv_done(i), 1);
    }
    mbar_init(bars + 8 * (2 * NS + 10), 1);
    mbar_init(q_ready, 4 * GR);
  }
  if (warp == kWarpQk) tmem_alloc(smem_addr(s_tmem), kTmemCols);
  // the panel that a head of up to 64 elements has none for stays 0
  if constexpr (PANELS == 1)
    for (int i = tid; i < (int)(S::kValueBufs * kPanel / 16); i += S::kThreads)
      reinterpret_cast<uint4*>(smem + i / (kPanel / 16) * S::kValues + kPanel)[i % (kPanel / 16)] = make_uint4(0, 0, 0, 0);
  smem_fence_async();
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  const uint32_t tmem = *s_tmem;
  Pieces4 list;
  int all;
  list.begin(p, all);
  Piece x = {0, 0, 0, 0};
  bool fine = true;  // no wait gave up
  const int G = groups4(p.head_dim), R = p.row_bytes;
  auto source = [&](const ckks_rows& r, int tile) {
    return static_cast<const uint8_t*>(r.data) + x.b * r.batch + x.unit / p.tiles_r * r.head + (int64_t)tile * (kKeys * R);
  };
  if (warp == kWarpCopy) {
    // ---- copies.  A tile may start on any 4-byte boundary; the copy takes the
    // aligned 16-byte pieces that hold its bytes (all of them in the tensor's own
    // 16-byte pieces of memory).
    int slot = 0, lap = 0, k = 0;
    while (fine && list.next(p, x)) {
      if (lane == 0) {
        const int len = length_of(p, x.b);
        for (int t = x.tile; t < x.tile + x.n && fine; ++t) {
          if (lap > 0 && !(fine = mbar_wait_short(raw_empty(slot), (lap - 1) & 1))) break;
          const uint32_t bytes = min(kKeys, len - t * kKeys) * R;
          const uint8_t* from[2] = {source(p.kc, t), source(p.vc, t)};
          uint32_t size[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t off = (uint32_t)reinterpret_cast<uintptr_t>(from[i]) & 15u;
            from[i] -= off;
            size[i] = (off + bytes + 15u) & ~15u;
          }
          mbar_expect_tx(raw_full(slot), size[0] + size[1]);
#pragma unroll
          for (int i = 0; i < 2; ++i)
            bulk_load(base + S::kAtRaw + (2 * slot + i) * S::kRaw, from[i], size[i], raw_full(slot));
          ++k;
          if (++slot == NS) slot = 0, ++lap;
        }
      }
      fine = __shfl_sync(0xffffffffu, fine, 0);
    }
    // copies still in flight land before the CTA ends
    if (lane == 0)
      for (int j = k > NS ? k - NS : 0; j < k; ++j) fine = mbar_wait_short(raw_full(j % NS), (j / NS) & 1) && fine;
  } else if (warp >= kWarpK && warp < kWarpCopy) {
    // ---- decoding, a thread a key: K into tensor memory, V into shared memory
    const bool value = warp >= kWarpV;
    const int key = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    int slot = 0, i = 0;
    uint32_t lap = 0;
    while (fine && list.next(p, x)) {
      const int len = length_of(p, x.b);
      for (int t = x.tile; t < x.tile + x.n; ++t, ++i) {
        const uint32_t off = (uint32_t)reinterpret_cast<uintptr_t>(source(value ? p.vc : p.kc, t)) & 15u;
        // (what this tile takes the place of is used)
        const int back = value ? VB : 2;
        const uint32_t used = value ? v_free(VB == 2 ? i & 1 : 0) : s_full(i & 1);
        if (!(fine = i < back ? warp_wait_done(raw_full(slot), lap)
                              : warp_wait_both(raw_full(slot), lap, used, (i / back - 1) & 1)))
          break;
        const uint32_t* const row = reinterpret_cast<const uint32_t*>(smem + S::kAtRaw + (2 * slot + (value ? 1 : 0)) * S::kRaw +
                                                                      off + key * R);
        // the row's groups four at a time: 8 words of codes and one of scales
        struct Quad {
          uint32_t code[8], scale;
        };
        auto read = [&](int g) {
          Quad y;
#pragma unroll
          for (int j = 0; j < 8; ++j) y.code[j] = g + j / 2 < G ? row[2 * g + j] : 0u;
          y.scale = g < G ? row[2 * G + g / 4] : 0u;
          return y;
        };
        const bool there = t * kKeys + key < len;
        const int buf = i & 1;
        if (!value) {
          tmem_fence_after();
          // 16 columns a store, and the next words read ahead of it (one node over 65536
          // bfloat16 keys 91 us, with 32 columns 94)
          Quad y = read(0);
#pragma unroll
          for (int g = 0; g < 4 * PANELS; g += 4) {
#pragma unroll
            for (int i0 = 0; i0 < 8; i0 += 4) {
              uint32_t w[16];
#pragma unroll
              for (int j = 0; j < 4; ++j) decode4_word<T>(y.code[i0 + j], scale4_pair(y.scale, (i0 + j) / 2), w + 4 * j);
              if (i0 && g + 4 < 4 * PANELS) y = read(g + 4);
              tmem_store<16>(tmem + lanes + buf * (DP / 2) + 8 * g + 4 * i0, w);
            }
          }
          tmem_wait_store();
          tmem_fence_before();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(raw_empty(slot));
            mbar_arrive(k_ready(buf));
          }
        } else {
          const int vb = VB == 2 ? buf : 0;
          uint8_t* const to = smem + vb * S::kValues + key * 128;
#pragma unroll
          for (int g = 0; g < 4 * PANELS; g += 4) {
            Quad y = read(g);
            if (!there) y.scale = 0u;  // a key that no row sees: zeros
            uint8_t* const panel = to + (g / 4) * kPanel;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              uint32_t w[4];
              decode4_word<__half>(y.code[j], scale4_pair(y.scale, j / 2), w);
              *reinterpret_cast<uint4*>(panel + ((j ^ (key & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
          smem_fence_async();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(raw_empty(slot));
            mbar_arrive(v_ready(vb));
          }
        }
        if (++slot == NS) slot = 0, lap ^= 1u;
      }
    }
  } else if (warp == kWarpQk) {
    // ---- the scores' products, by the whole warp in step
    constexpr uint32_t word = mma_word(kBf, kM, N, false);
    const uint32_t t_base = __shfl_sync(0xffffffffu, tmem, 0);
    int i = 0;
    uint32_t units = 0;
    while (fine && list.next(p, x)) {
      const int n = __shfl_sync(0xffffffffu, x.n, 0);
      if (!n) continue;
      if (!(fine = warp_wait(q_ready, units & 1))) break;
      ++units;
      for (int t = 0; t < n; ++t, ++i) {
        const int buf = i & 1;
        // (the scores that this buffer had are read)
        if (!(fine = i < 2 ? warp_wait(k_ready(buf), 0)
                           : warp_wait_both(k_ready(buf), (i / 2) & 1, p_ready(buf), (i / 2 - 1) & 1)))
          break;
        tmem_fence_after();
#pragma unroll
        for (int s = 0; s < DP / 16; ++s)
          mma_tmem(t_base + S::kColS + buf * N, t_base + buf * (DP / 2) + 8 * s,
                   smem_operand(base + S::kAtQ + (s / 4) * (N * 128) + (s % 4) * 32, 16), word, s > 0);
        mma_commit(s_full(buf));
      }
    }
  } else if (warp == kWarpPv) {
    // ---- the sums' products, by the whole warp in step
    constexpr uint32_t word = mma_word(false, kM, N, true) | 1u << 15;  // A is as the values lie
    const uint32_t t_base = __shfl_sync(0xffffffffu, tmem, 0);
    int i = 0;
    while (fine && list.next(p, x)) {
      const int n = __shfl_sync(0xffffffffu, x.n, 0);
      for (int t = 0; t < n; ++t, ++i) {
        const int buf = i & 1, vb = VB == 2 ? buf : 0;
        if (!(fine = warp_wait_both(v_ready(vb), (i / VB) & 1, p_ready(buf), (i / 2) & 1))) break;
        tmem_fence_after();
#pragma unroll
        for (int m = 0; m < S::kBlocks; ++m)
#pragma unroll
          for (int s = 0; s < kKeys / 16; ++s)
            mma_smem(t_base + S::kColO + m * N, smem_operand(base + vb * S::kValues + m * 2 * kPanel + 2048 * s, kPanel),
                     smem_operand(base + S::kAtP + buf * S::kP + 2048 * s, kPanel), word, s > 0 || t > 0);
        mma_commit(pv_done(buf));
        if constexpr (VB == 1) mma_commit(v_free(0));
      }
    }
  } else {
    // ---- softmax: group g has rows C g .. C g + C - 1, a thread key L of a tile
    const int g = warp >> 2, quarter = warp & 3, L = quarter * 32 + lane, r0 = C * g, id = 1 + g;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const int rows = p.nodes * p.group;
    int i = 0, units = 0;
    // Queries of a piece, a warp a row.  A bfloat16 row whose largest element is
    // above 2^101 or below 2^-60 is scaled to there, so that the sums stay within a
    // float's range; what that costs lies 2^226 below the largest.
    auto queries = [&](const Piece& y) {
      const int h = y.unit / p.tiles_r, first = y.unit % p.tiles_r * N;
      float2* const row_of = s_row + (units & 1) * N;
#pragma unroll 2
      for (int r = r0 + quarter; r < r0 + C; r += 4) {
        const int row = first + r;
        const bool real = row < rows;
        const T* const q = static_cast<const T*>(p.q.data) + y.b * p.q.batch + (h * p.group + row % p.group) * p.q.head +
                           (int64_t)(row / p.group) * p.q.row;
        float v[2 * PANELS];
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < 2 * PANELS; ++j) {
          const int d = 2 * lane + 64 * (j / 2) + (j & 1);
          v[j] = real && d < p.head_dim ? to_f32(q[d]) : 0.0f;
          const uint32_t u = __float_as_uint(v[j]) & 0x7FFFFFFFu;
          top = max(top, u < 0x7F800000u ? u : 0u);
        }
        int e = 0;  // the row is scaled by 2^-e
        if constexpr (kBf) {
          const int high = (int)(__reduce_max_sync(0xffffffffu, top) >> 23) - 127;
          e = high > 100 ? high - 100 : high < -60 ? high + 60 : 0;
        }
        const float down = __int_as_float((127 - e) << 23);
#pragma unroll
        for (int j = 0; j < PANELS; ++j)
          *reinterpret_cast<uint32_t*>(smem + S::kAtQ + j * (N * 128) + r * 128 + (((lane / 4) ^ (r & 7)) << 4) +
                                       (lane % 4) * 4) = pack2<T>(v[2 * j] * down, v[2 * j + 1] * down);
        if (lane == 0) row_of[r] = make_float2(p.scale * kLog2e * __int_as_float((127 + e) << 23), kUnset);
      }
      smem_fence_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_ready);
    };
    bool have = list.next(p, x);
    while (have && x.n == 0) have = list.next(p, x);
    if (have) queries(x);
    while (have) {
      const int len = length_of(p, x.b), n = x.n;
      float2* const row_of = s_row + (units & 1) * N + r0;
      float l[C];
#pragma unroll
      for (int r = 0; r < C; ++r) l[r] = 0.0f;
      // every warp's rows are there, whatever the waits before gave
      if (!(fine = group_all(id, 128, fine))) break;
#pragma unroll 1
      for (int t = 0; t < n; ++t, ++i) {
        const int buf = i & 1, seen = len - (x.tile + t) * kKeys;
        const bool there = L < seen;
        const uint32_t t_s = tmem + lanes + S::kColS + buf * N + r0;
        float z[C];
        // scores against their rows' reference points
        auto scores = [&] {
          tmem_load<C>(t_s, reinterpret_cast<uint32_t*>(z));
          tmem_wait_load();
#pragma unroll
          for (int r = 0; r < C; r += 2) {
            const float4 f = *reinterpret_cast<const float4*>(row_of + r);
            z[r] = fmaf(z[r], f.x, -f.y);
            z[r + 1] = fmaf(z[r + 1], f.z, -f.w);
          }
          if (seen < kKeys) {
#pragma unroll
            for (int r = 0; r < C; ++r) z[r] = there ? z[r] : -INFINITY;
          }
        };
        fine = fine && warp_wait_done(s_full(buf), (i / 2) & 1);
        bool above = false;
        if (fine) {
          tmem_fence_after();
          scores();
          float top[2] = {z[0], z[1]};
#pragma unroll
          for (int r = 2; r < C; ++r) top[r & 1] = fmaxf(top[r & 1], z[r]);
          above = fmaxf(top[0], top[1]) > kSlack + kBelow<__half>;
        }
        // one warp's score above its row's reference point, or a wait that gave up, concerns all
        if (!group_all(id, 128, fine && !above)) {
          if (!(fine = group_all(id, 128, fine))) break;
          tmem_load<C>(t_s, reinterpret_cast<uint32_t*>(z));
          tmem_wait_load();
#pragma unroll
          for (int r = 0; r < C; ++r) {
            const int best = __reduce_max_sync(0xffffffffu, ordered(there ? z[r] * row_of[r].x : -INFINITY));
            if (lane == 0) s_max[quarter * N + r0 + r] = unordered(best);
          }
          // sums so far are on the old points until the last product is done
          if (t > 0) fine = warp_wait(pv_done(buf ^ 1), ((i - 1) / 2) & 1);
          if (!(fine = group_all(id, 128, fine))) break;
          if (L < C) {
            float best = s_max[r0 + L];
            bool nan = best != best;
#pragma unroll
            for (int q = 1; q < 4; ++q) {
              const float o = s_max[q * N + r0 + L];
              nan |= o != o;
              best = fmaxf(best, o);
            }
            if (nan) best = __int_as_float(0x7FC00000);
            const float2 f = row_of[L];
            // (a point that is no number stays)
            const bool set = f.y == f.y && !(best <= f.y + (kSlack + kBelow<__half>)) && best != -INFINITY;
            const float to = set ? best - kBelow<__half> : f.y;
            s_fac[r0 + L] = set ? ex2(f.y - to) : 1.0f;
            row_of[L].y = to;
          }
          group_sync(id, 128);
          if (t > 0) tmem_fence_after();
#pragma unroll
          for (int m = 0; m < (t > 0 ? S::kBlocks : 0); ++m) {
            float o[C];
            tmem_load<C>(tmem + lanes + S::kColO + m * N + r0, reinterpret_cast<uint32_t*>(o));
            tmem_wait_load();
#pragma unroll
            for (int r = 0; r < C; ++r) o[r] *= s_fac[r0 + r];
            tmem_store<C>(tmem + lanes + S::kColO + m * N + r0, reinterpret_cast<const uint32_t*>(o));
          }
          tmem_wait_store();
#pragma unroll
          for (int r = 0; r < C; ++r) l[r] *= s_fac[r0 + r];
          scores();
          group_sync(id, 128);  // s_max and s_fac are read
        }
        uint32_t w[C / 2];
#pragma unroll
        for (int r = 0; r < C; r += 2) {
          const float2 e = make_float2(ex2(z[r]), ex2(z[r + 1]));
          l[r] += e.x, l[r + 1] += e.y;
          w[r / 2] = pack2<__half>(e.x, e.y);
        }
        // the product that read this buffer is done
        if (i >= 2) fine = warp_wait_done(pv_done(buf), (i / 2 - 1) & 1);
        if (fine) {
          uint8_t* const to = smem + S::kAtP + buf * S::kP + L * 128;
#pragma unroll
          for (int j = 0; j < C / 8; ++j)
            *reinterpret_cast<uint4*>(to + (((r0 / 8 + j) ^ (L & 7)) << 4)) =
                make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
        }
        smem_fence_async();
        tmem_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_ready(buf));
      }
      if (!(fine = group_all(id, 128, fine))) break;
      // the next piece's queries may come: every product over this one's is done
      const Piece done = x;
      const int last = i - 1;
      do have = list.next(p, x);
      while (have && x.n == 0);
      ++units;
      if (have) queries(x);
      // this piece's sums: l over the keys of all warps, O as it is
      const float mine = warp_columns(l);
      if (!(lane & 1)) s_max[quarter * N + r0 + (lane >> 1)] = mine;
      fine = warp_wait(pv_done(last & 1), (last / 2) & 1);
      if (!(fine = group_all(id, 128, fine))) break;
      tmem_fence_after();
      float* const keep = p.part + ((int64_t)done.b * list.units + done.unit + blockIdx.x) * (N * (DP + 4));
#pragma unroll
      for (int m = 0; m < S::kBlocks; ++m) {
        float o[C];
        tmem_load<C>(tmem + lanes + S::kColO + m * N + r0, reinterpret_cast<uint32_t*>(o));
        tmem_wait_load();
        if (128 * m + L < DP)
#pragma unroll
          for (int r = 0; r < C; ++r) keep[(r0 + r) * (DP + 4) + 128 * m + L] = o[r];
      }
      if (L < C)
        *reinterpret_cast<float2*>(keep + (r0 + L) * (DP + 4) + DP) =
            make_float2(row_of[L].y, (s_max[r0 + L] + s_max[N + r0 + L]) + (s_max[2 * N + r0 + L] + s_max[3 * N + r0 + L]));
      tmem_fence_before();
    }
  }
  if (!fine && (warp < kWarpK || lane == 0)) atomicAdd(faults, 1u);
  tmem_fence_before();
  __syncthreads();
  if (warp == kWarpQk) {
    __syncwarp();
    tmem_free(tmem, kTmemCols);
  }
}

// Joins the parts of a row over the cache and adds its new keys; W warps a row,
// which take the parts in turns.  What does not wait for the first kernel comes
// first.
template <typename T, int PANELS, int W>
__global__ void __launch_bounds__(256) join4_kernel(const __grid_constant__ Params4 p) {
  constexpr int DP = 64 * PANELS;
  __shared__ uint64_t s_mask[8][kMaxNodes];
  __shared__ int s_jump[8][kMaxNodes];
  __shared__ float s_sum[W > 1 ? 8 : 1][W > 1 ? DP + 2 : 1];
  const int rows = p.nodes * p.group, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, N = p.rows;
  const int per = (rows * W + 7) / 8, bh = blockIdx.x / per, row = (blockIdx.x % per * 8 + warp) / W, turn = warp % W;
  const int b = bh / p.kv_heads, h = bh % p.kv_heads;
  if (row >= rows) {
    CKKS_PDL_ENTRY();
    return;
  }
  tree_masks(p.parents + (size_t)b * p.nodes, p.nodes, s_mask[warp], s_jump[warp]);
  const int node = row / p.group, qh = h * p.group + row % p.group;
  const uint64_t mask = s_mask[warp][node];
  T* const out = static_cast<T*>(p.out.data) + b * p.out.batch + qh * p.out.head + (int64_t)node * p.out.row;
  float* const lse = p.lse + ((size_t)b * p.nodes + node) * p.kv_heads * p.group + qh;
  // the new keys: lane x has elements x, x + 32, ...
  float q[2 * PANELS], acc[2 * PANELS], m = -INFINITY, l = 0.0f;
  const T* const q_row = static_cast<const T*>(p.q.data) + b * p.q.batch + qh * p.q.head + (int64_t)node * p.q.row;
  const T* const kn = static_cast<const T*>(p.kn.data) + b * p.kn.batch + h * p.kn.head;
  const T* const vn = static_cast<const T*>(p.vn.data) + b * p.vn.batch + h * p.vn.head;
#pragma unroll
  for (int j = 0; j < 2 * PANELS; ++j) {
    const int d = lane + 32 * j;
    q[j] = mask && d < p.head_dim ? to_f32(q_row[d]) : 0.0f;
    acc[j] = 0.0f;
  }
  for (uint64_t left = turn == 0 ? mask : 0ull; left;) {
    // four keys at a time, so that their reads wait together
    int key[4];
    float s[4], v[4][2 * PANELS];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      key[i] = left ? __ffsll((long long)left) - 1 : -1;
      left &= left - 1;
      s[i] = 0.0f;
#pragma unroll
      for (int j = 0; j < 2 * PANELS; ++j) {
        const int d = lane + 32 * j;
        const bool is = key[i] >= 0 && d < p.head_dim;
        s[i] = fmaf(q[j], is ? to_f32(kn[(int64_t)key[i] * p.kn.row + d]) : 0.0f, s[i]);
        v[i][j] = is ? to_f32(vn[(int64_t)key[i] * p.vn.row + d]) : 0.0f;
      }
    }
    float top = m;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int o = 16; o; o >>= 1) s[i] += __shfl_xor_sync(0xffffffffu, s[i], o);
      s[i] = key[i] >= 0 ? s[i] * (p.scale * kLog2e) : -INFINITY;
      top = fmaxf(top, s[i]);
    }
    const float ref = top == -INFINITY ? 0.0f : top, f = exp2f(m - ref);
    m = top;
    l *= f;
#pragma unroll
    for (int j = 0; j < 2 * PANELS; ++j) acc[j] *= f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (key[i] < 0) continue;
      const float w = exp2f(s[i] - ref);
      l += w;
#pragma unroll
      for (int j = 0; j < 2 * PANELS; ++j) acc[j] = fmaf(w, v[i][j], acc[j]);
    }
  }
  // this row's unit: its tiles [u0, u0 + tiles) of the list, and the CTAs that
  // have the first and the last: CTA i begins at list_start(i), so entry w is
  // CTA floor((ctas (w + 1) - 1) / entries)'s
  const int units = p.kv_heads * p.tiles_r, unit = h * p.tiles_r + row / N;
  int before = 0, all = 0;
  for (int i = lane; i < p.batch; i += 32) {
    const int t = entries_of(p, i);
    all += t;
    if (i < b) before += t;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    all += __shfl_xor_sync(0xffffffffu, all, o);
    before += __shfl_xor_sync(0xffffffffu, before, o);
  }
  const int entries = entries_of(p, b);
  CKKS_PDL_ENTRY();  // what is read above no kernel of this call writes
  if (entries) {
    const long long list = (long long)all * units, ctas = min((long long)p.ctas, list);
    const long long u0 = (long long)before * units + (long long)unit * entries + p.unit_cost;
    const int c0 = (int)((ctas * (u0 + 1) - 1) / list), c1 = (int)((ctas * (u0 + entries - p.unit_cost) - 1) / list);
    const float* const part = p.part + ((int64_t)(b * units + unit) * N + row % N) * (DP + 4);
    // Parts read at once, so that a row seldom waits for memory twice: with 8 warps 20,
    // which is a turn of every SM's part (one node of 4/1 heads over 65536 keys 13.6 us, 15.7
    // with 8, 16.7 with 4), as far as the registers go; with one 12 (trees of 16 over
    // 32768 and 24576 keys 52.8, with 8 54.7).
    constexpr int kAtOnce = W > 1 && PANELS < 4 ? 20 : 12;
    for (int c = c0 + turn; c <= c1; c += kAtOnce * W) {
      float2 ml[kAtOnce];
      float y[kAtOnce][2 * PANELS];
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const bool is = c + W * i <= c1;
        const float* const o = part + (int64_t)(c + W * i) * (N * (DP + 4));
        ml[i] = is ? *reinterpret_cast<const float2*>(o + DP) : make_float2(-INFINITY, 0.0f);
#pragma unroll
        for (int j = 0; j < 2 * PANELS; ++j) y[i][j] = is ? o[lane + 32 * j] : 0.0f;
      }
      float top = m;
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) top = fmaxf(top, ml[i].x);
      const float ref = top == -INFINITY ? 0.0f : top, f = exp2f(m - ref);
      m = top;
      l *= f;
#pragma unroll
      for (int j = 0; j < 2 * PANELS; ++j) acc[j] *= f;
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const float w = exp2f(ml[i].x - ref);
        l = fmaf(ml[i].y, w, l);
#pragma unroll
        for (int j = 0; j < 2 * PANELS; ++j) acc[j] = fmaf(y[i][j], w, acc[j]);
      }
    }
  }
  if constexpr (W > 1) {
    static_assert(W == 8, "a CTA has one row");
#pragma unroll
    for (int j = 0; j < 2 * PANELS; ++j) s_sum[warp][lane + 32 * j] = acc[j];
    if (lane == 0) s_sum[warp][DP] = m, s_sum[warp][DP + 1] = l;
    __syncthreads();
    if (warp) return;
    for (int i = 1; i < W; ++i) {
      const float o = s_sum[i][DP], top = fmaxf(m, o), ref = top == -INFINITY ? 0.0f : top;
      const float f = exp2f(m - ref), w = exp2f(o - ref);
      m = top;
      l = fmaf(s_sum[i][DP + 1], w, l * f);
#pragma unroll
      for (int j = 0; j < 2 * PANELS; ++j) acc[j] = fmaf(s_sum[i][lane + 32 * j], w, acc[j] * f);
    }
  }
  const float inv = l != 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
  for (int j = 0; j < 2 * PANELS; ++j)
    if (lane + 32 * j < p.head_dim) out[lane + 32 * j] = from_f32<T>(mask ? acc[j] * inv : 0.0f);
  if (lane == 0) *lse = mask && l != 0.0f ? kLn2 * (m + log2f(l)) : -INFINITY;
}

struct Plan4 {
  int rows, tiles_r, ctas;  // rows of a unit, units of a (sequence, head)
  long long units;
  bool listed;  // the list has fewer than 2^31 entries
};

// What a unit's start costs in the list, in tiles: its query rows are scaled and
// laid out and its sums left.  With 1, 3 and 6: trees of 21 over 4001 keys, eight ragged
// sequences of 12 heads of 64, 35.7, 27.2 and 26.9 us; one node of 16/4 heads over
// 16 sequences of 1500 to 3000 keys 20.8, 20.0 and 20.9; one node over 65536 to 40960 keys,
// four sequences of 32/8 heads of 128, 92.3, 90.9 and 91.6.
constexpr int kUnitCost = 3;

Plan4 plan4(const Context& c, const ckks_draft_attention_args& a) {
  const int rows = a.nodes * (a.q_heads / a.kv_heads);
  Plan4 d;
  // The fewest of 16, 32 and 64 rows that hold a (sequence, head)'s, and 64 at a time beyond:
  // one node over 65536 to 40960 keys (4 rows) takes 91 us with 16 rows, 101 with 32 and 138
  // with 64; trees of 21 (21 rows) 27.2 with 32 and 35.9 with 64.
  d.rows = rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
  d.tiles_r = (rows + d.rows - 1) / d.rows;
  d.units = (long long)a.batch * a.kv_heads * d.tiles_r;
  const long long tiles = (a.capacity + kKeys - 1) / kKeys;
  d.listed = d.units * (tiles + kUnitCost) < (1ll << 31) - 1;
  // Two tiles of the longest sequence a CTA, if there are SMs for it: chains of 5 over 1000 keys
  // of 12 heads take 10.6 us, 12.4 with four and 10.0 with one; 8 nodes of 8/2 heads over
  // 20000 keys 18.0, 15.0 and 18.0.
  d.ctas = (int)std::max(1ll, std::min<long long>(c.sms, d.units * std::max(1ll, tiles / 2)));
  return d;
}

template <typename T, int PANELS>
void launch_join4(const ckks_draft_attention_args& a, const Params4& p, cudaStream_t st) {
  const long long heads = (long long)a.batch * a.kv_heads, rows = (long long)a.nodes * p.group;
  // Many parts a unit go to eight warps a row, few to one: 8 nodes of 8/2 heads over
  // 20000 keys, 74 parts, take 18 us with eight and 29 with one, 16 nodes of 12 heads
  // over 8000 keys, 12.3 parts, 16 and 18; trees of 16 over 32768 and 24576 keys,
  // 9 parts and 512 rows, 62 and 55.
  if (p.ctas > 12 * heads * p.tiles_r)
    launch_pdl(join4_kernel<T, PANELS, 8>, dim3((unsigned)(heads * rows)), dim3(256), 0, st, p);
  else
    launch_pdl(join4_kernel<T, PANELS, 1>, dim3((unsigned)(heads * ((rows + 7) / 8))), dim3(256), 0, st, p);
}

template <typename T, int PANELS, int N>
void launch4(const Context& c, const ckks_draft_attention_args& a, const Params4& p, cudaStream_t st) {
  using S = Shape4<PANELS, N>;
  static_assert(S::kSmem <= 232448, "shared memory of one block");
  auto* k = attend4_kernel<T, PANELS, N>;
  CKKS_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::kSmem));
  k<<<p.ctas, S::kThreads, S::kSmem, st>>>(p, c.d_faults);
  CKKS_CUDA(cudaGetLastError());
  launch_join4<T, PANELS>(a, p, st);
}

template <typename T, int PANELS>
void launch4(const Context& c, const ckks_draft_attention_args& a, const Params4& p, cudaStream_t st) {
  if (p.rows == 16)
    launch4<T, PANELS, 16>(c, a, p, st);
  else if (p.rows == 32)
    launch4<T, PANELS, 32>(c, a, p, st);
  else
    launch4<T, PANELS, 64>(c, a, p, st);
}

template <typename T>
void launch4(const Context& c, const ckks_draft_attention_args& a, const Params4& p, int panels, cudaStream_t st) {
  switch (panels) {
    case 1: launch4<T, 1>(c, a, p, st); break;
    case 2: launch4<T, 2>(c, a, p, st); break;
    default: launch4<T, 4>(c, a, p, st); break;
  }
}

int panels4(int head_dim) { return head_dim <= 64 ? 1 : head_dim <= 128 ? 2 : 4; }

}  // namespace

size_t attention4_tc_workspace(const Context& c, const ckks_draft_attention_args& a) {
  const Plan4 d = plan4(c, a);
  if (a.dtype == CKKS_FP32 || !d.listed) return 0;
  return sizeof(float) * (size_t)(d.units + d.ctas) * d.rows * (64 * panels4(a.head_dim) + 4);
}

bool attention4_tc(const Context& c, const ckks_draft_attention_args& a, cudaStream_t st) {
  const Plan4 d = plan4(c, a);
  const int R = row4_bytes(a.head_dim);
  if (a.dtype == CKKS_FP32 || !d.listed) return false;
  // a head's rows one behind the other
  if (a.capacity > 1 && (a.k_cache.row != R || a.v_cache.row != R)) return false;
  Params4 p{};
  p.q = a.q, p.kc = a.k_cache, p.vc = a.v_cache, p.kn = a.k_new, p.vn = a.v_new, p.out = a.out;
  p.lens = a.lens, p.parents = a.parents, p.lse = a.lse, p.part = static_cast<float*>(a.workspace);
  p.batch = a.batch, p.kv_heads = a.kv_heads, p.group = a.q_heads / a.kv_heads, p.head_dim = a.head_dim;
  p.nodes = a.nodes, p.capacity = a.capacity, p.scale = (float)a.scale;
  p.rows = d.rows, p.tiles_r = d.tiles_r, p.unit_cost = kUnitCost, p.ctas = d.ctas, p.row_bytes = R;
  if (a.dtype == CKKS_BF16)
    launch4<__nv_bfloat16>(c, a, p, panels4(a.head_dim), st);
  else
    launch4<__half>(c, a, p, panels4(a.head_dim), st);
  return true;
}

}  // namespace draft
}  // namespace ckks
