// draft_fill.cu -- rows written to the draft model's key/value cache and read
// back: packed prompts appended to a plain or a 4-bit cache (ckks_draft_fill,
// ckks_draft_fill4), accepted nodes to a 4-bit one (ckks_draft_commit4), and
// a 4-bit cache's values (ckks_draft_read4).  Each element is read once and
// written once.  The launch bounds the short ones (103 rows of 12 heads written
// and read back, three calls, 14 us).  40500 rows of 8 heads of 128 take 51 us to
// write (213 MB, 4.2 TB/s: about 15 instructions an element, two thirds of them
// the exact quotient, its scale and unpacking) and 39 to read back (156 MB,
// 4.0 TB/s: memory latency, two groups in flight a thread).
#include <algorithm>

#include "draft_fp4.cuh"

namespace ckks {
namespace draft {
namespace {

// Group g's elements as floats, 0 behind the row's end, and the bits of their
// largest magnitude
template <typename T, bool WIDE>
__device__ __forceinline__ uint32_t load_group(float* x, const T* row, int g, int D) {
  const int d = g * kGroup4;
  uint32_t top = 0;
  if constexpr (WIDE && sizeof(T) == 2) {  // whole, aligned 16-byte pieces
    uint4 u[2];
    u[0] = __ldg(reinterpret_cast<const uint4*>(row + d));
    u[1] = d + 8 < D ? __ldg(reinterpret_cast<const uint4*>(row + d) + 1) : make_uint4(0, 0, 0, 0);
    const T* e = reinterpret_cast<const T*>(u);
#pragma unroll
    for (int k = 0; k < kGroup4; ++k) x[k] = to_f32(e[k]);
    // two magnitudes a word, as integers
    const uint32_t m = 0x7FFF7FFFu;
    uint32_t w = 0;
#pragma unroll
    for (int k = 0; k < 2; ++k)
      w = __vmaxu2(w, __vmaxu2(__vmaxu2(u[k].x & m, u[k].y & m), __vmaxu2(u[k].z & m, u[k].w & m)));
    const unsigned short b = (unsigned short)max(w & 0xFFFFu, w >> 16);
    top = __float_as_uint(to_f32(*reinterpret_cast<const T*>(&b)));
  } else {
    if constexpr (WIDE) {
#pragma unroll
      for (int i = 0; i < kGroup4; i += 4) {
        const float4 u = d + i < D ? __ldg(reinterpret_cast<const float4*>(row + d + i)) : make_float4(0, 0, 0, 0);
        x[i] = u.x, x[i + 1] = u.y, x[i + 2] = u.z, x[i + 3] = u.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kGroup4; ++i) x[i] = d + i < D ? to_f32(row[d + i]) : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < kGroup4; ++i) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
  }
  return top;
}

// group g of a 4-bit row of G; the row is 4-byte aligned
__device__ __forceinline__ void store_group(uint8_t* row, const float* x, uint32_t top, int g, int G) {
  uint32_t scale;
  const uint2 code = encode4(x, top, scale);
  uint32_t* c = reinterpret_cast<uint32_t*>(row) + 2 * g;
  c[0] = code.x, c[1] = code.y;
  row[8 * G + g] = (uint8_t)scale;
  if (g == G - 1)
    for (int i = 9 * G; i & 3; ++i) row[i] = 0;
}

// Threads over the groups (or pieces) of a row's heads, `per` of them, several
// rows at a time: f(head-and-group, first row, rows between a thread's)
template <class F>
__device__ __forceinline__ void over_rows(int threads, int per, F f) {
  const int at = per < threads ? threads / per : 1, c0 = per < threads ? threadIdx.x % per : threadIdx.x;
  const int r0 = per < threads ? threadIdx.x / per : 0;
  if (r0 < at)
    for (int c = c0; c < per; c += threads) f(c, r0, at);
}

// ---- packed rows ----------------------------------------------------------------
// Sequence b has the rows from start(b) to start(b + 1), where start(b) is the
// largest of starts[0..b], each taken as 0..tokens: an order that decreases
// leaves a sequence without rows, and no row belongs to two.
struct FillParams {
  ckks_rows kc, vc, k, v;
  const int32_t* starts;
  const int32_t* lens;
  int32_t* lens_out;
  unsigned int* refused;
  int batch, kv_heads, head_dim, tokens, capacity;
  int rows;  // of a chunk
};

constexpr int kFillThreads = 256;

// One warp of a CTA walks the starts; the CTA takes a chunk of rows, keys and
// values in turn.
template <typename T, typename V, bool FOUR, bool WIDE>
__global__ void __launch_bounds__(kFillThreads) fill_kernel(FillParams p) {
  __shared__ int s_place[4];  // sequence, its first row here, rows, first slot (or -1: the sequence does not fit)
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int chunk = blockIdx.x, carry = 0, found = 0;
    for (int b0 = 0; b0 < p.batch && !found; b0 += 32) {
      const int b = b0 + lane;
      int e = b < p.batch ? min(max(p.starts[b + 1], 0), p.tokens) : 0;
      if (b0 == 0) carry = min(max(p.starts[0], 0), p.tokens);
      e = max(e, carry);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, e, o);
        if (lane >= o) e = max(e, y);
      }
      int a = __shfl_up_sync(0xffffffffu, e, 1);
      if (lane == 0) a = carry;
      carry = __shfl_sync(0xffffffffu, e, 31);
      const int rows = b < p.batch ? e - a : 0;
      const int mine = b < p.batch ? max(1, (rows + p.rows - 1) / p.rows) : 0;  // one chunk at least: it has the length
      int sum = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += y;
      }
      const bool here = chunk >= sum - mine && chunk < sum;
      if (here) {
        const int first = (chunk - (sum - mine)) * p.rows;
        const int len = p.lens[b];
        const bool ok = len >= 0 && len <= p.capacity && rows <= p.capacity - len;
        s_place[0] = b;
        s_place[1] = a + first;
        s_place[2] = min(p.rows, rows - first);
        s_place[3] = ok ? len + first : -1;
        if (first == 0) {
          p.lens_out[b] = ok ? len + rows : len;
          if (!ok) atomicAdd(p.refused, 1u);
        }
      }
      found = __any_sync(0xffffffffu, here);
      chunk -= __shfl_sync(0xffffffffu, sum, 31);
    }
    if (!found && lane == 0) s_place[3] = -1;
  }
  __syncthreads();
  if (s_place[3] < 0) return;
  const int b = s_place[0], row0 = s_place[1], rows = s_place[2], slot0 = s_place[3], H = p.kv_heads;
  if constexpr (FOUR) {
    const int G = groups4(p.head_dim);
    over_rows(kFillThreads, H * G, [&](int c, int r0, int at) {
      const int h = c / G, g = c % G;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const ckks_rows& from = w ? p.v : p.k;
        const ckks_rows& to = w ? p.vc : p.kc;
        const T* src = static_cast<const T*>(from.data) + (int64_t)(row0 + r0) * from.row + h * from.head;
        uint8_t* dst = static_cast<uint8_t*>(to.data) + b * to.batch + h * to.head + (int64_t)(slot0 + r0) * to.row;
        const int64_t step = at * from.row, to_step = at * to.row;
#pragma unroll 2
        for (int r = r0; r < rows; r += at, src += step, dst += to_step) {
          float x[kGroup4];
          const uint32_t top = load_group<T, WIDE>(x, src, g, p.head_dim);
          store_group(dst, x, top, g, G);
        }
      }
    });
  } else {
    constexpr int W = sizeof(V) / sizeof(T);
    const int D = p.head_dim / W;
    over_rows(kFillThreads, H * D, [&](int c, int r0, int at) {
      const int h = c / D, d = c % D * W;
      for (int w = 0; w < 2; ++w) {
        const ckks_rows& from = w ? p.v : p.k;
        const ckks_rows& to = w ? p.vc : p.kc;
        const T* src = static_cast<const T*>(from.data) + (int64_t)(row0 + r0) * from.row + h * from.head + d;
        T* dst = static_cast<T*>(to.data) + b * to.batch + h * to.head + (int64_t)(slot0 + r0) * to.row + d;
        for (int r = r0; r < rows; r += at, src += at * from.row, dst += at * to.row)
          *reinterpret_cast<V*>(dst) = *reinterpret_cast<const V*>(src);
      }
    });
  }
}

// ---- accepted nodes ---------------------------------------------------------------
struct Commit4Params {
  ckks_rows kc, vc, kn, vn;
  const int32_t* lens;
  const int32_t* path;
  const int32_t* count;
  int32_t* lens_out;
  unsigned int* refused;
  int batch, kv_heads, head_dim, nodes, capacity;
};

// CTA = (sequence, head)
template <typename T, bool WIDE>
__global__ void __launch_bounds__(128) commit4_kernel(Commit4Params p) {
  const int b = blockIdx.x, h = blockIdx.y;
  const int32_t* path = p.path + (size_t)b * p.nodes;
  const int len = p.lens[b], count = p.count[b];
  const bool ok = fits(path, count, len, p.nodes, p.capacity);
  if (h == 0 && threadIdx.x == 0) {
    p.lens_out[b] = ok ? len + count : len;
    if (!ok) atomicAdd(p.refused, 1u);
  }
  if (!ok) return;
  const int G = groups4(p.head_dim);
  over_rows(128, G, [&](int g, int r0, int at) {
    for (int w = 0; w < 2; ++w) {
      const ckks_rows& from = w ? p.vn : p.kn;
      const ckks_rows& to = w ? p.vc : p.kc;
      for (int r = r0; r < count; r += at) {
        float x[kGroup4];
        const uint32_t top = load_group<T, WIDE>(
            x, static_cast<const T*>(from.data) + b * from.batch + h * from.head + path[r] * from.row, g, p.head_dim);
        store_group(static_cast<uint8_t*>(to.data) + b * to.batch + h * to.head + (int64_t)(len + r) * to.row, x, top, g, G);
      }
    }
  });
}

// ---- reading back -------------------------------------------------------------------
struct ReadParams {
  ckks_rows cache, out;
  const int32_t* lens;
  int batch, kv_heads, head_dim, capacity;
  int rows;  // of a chunk
};

constexpr int kReadRows = 32;  // the least

// CTA = (chunk of rows, head, sequence); a thread takes groups of 16 elements
template <typename T, bool WIDE>
__global__ void __launch_bounds__(256) read4_kernel(ReadParams p) {
  const int r0 = blockIdx.x * p.rows, rows = min(p.rows, p.capacity - r0), h = blockIdx.y, D = p.head_dim, G = groups4(D);
  for (int b = blockIdx.z; b < p.batch; b += gridDim.z) {
    const int len = min(max(__ldg(p.lens + b), 0), p.capacity);
    const uint8_t* in = static_cast<const uint8_t*>(p.cache.data) + b * p.cache.batch + h * p.cache.head;
    T* out = static_cast<T*>(p.out.data) + b * p.out.batch + h * p.out.head;
    over_rows(256, G, [&](int g, int first, int at) {
      const int d0 = kGroup4 * g, held = len - r0;
      const uint8_t* row = in + (int64_t)(r0 + first) * p.cache.row;
      T* dst = out + (int64_t)(r0 + first) * p.out.row + d0;
      const int64_t step = at * p.cache.row, out_step = at * p.out.row;
#pragma unroll 2
      for (int i = first; i < rows; i += at, row += step, dst += out_step) {
        uint32_t y[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (i < held) {
          const uint32_t* c = reinterpret_cast<const uint32_t*>(row) + 2 * g;
          const uint32_t a = __ldg(c), b = __ldg(c + 1);
          const __half2 s = scale4_pair(__ldg(row + 8 * G + g), 0);
          decode4_word<__half>(a, s, y);
          decode4_word<__half>(b, s, y + 4);
        }
        if constexpr (WIDE && std::is_same_v<T, __half>) {
          *reinterpret_cast<uint4*>(dst) = make_uint4(y[0], y[1], y[2], y[3]);
          if (d0 + 8 < D) *reinterpret_cast<uint4*>(dst + 8) = make_uint4(y[4], y[5], y[6], y[7]);
        } else {
          alignas(16) T x[kGroup4];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&y[k]));
            if constexpr (std::is_same_v<T, __nv_bfloat16>)
              *reinterpret_cast<__nv_bfloat162*>(x + 2 * k) = __floats2bfloat162_rn(f.x, f.y);
            else
              x[2 * k] = from_f32<T>(f.x), x[2 * k + 1] = from_f32<T>(f.y);
          }
          if constexpr (WIDE) {
            constexpr int W = 16 / sizeof(T);
#pragma unroll
            for (int k = 0; k < kGroup4; k += W)
              if (d0 + k < D) *reinterpret_cast<uint4*>(dst + k) = *reinterpret_cast<const uint4*>(x + k);
          } else {
#pragma unroll
            for (int k = 0; k < kGroup4; ++k)
              if (d0 + k < D) dst[k] = x[k];
          }
        }
      }
    });
  }
}

void check_sizes(int dtype, int batch, int kv_heads, int head_dim, int capacity) {
  need(dtype == CKKS_BF16 || dtype == CKKS_FP16 || dtype == CKKS_FP32, "rows are CKKS_BF16, CKKS_FP16 or CKKS_FP32");
  need(batch >= 0 && capacity >= 0 && capacity < (1 << 30), "batch or capacity out of range");
  need(kv_heads >= 1 && kv_heads <= 65535, "head count outside 1..65535");
  need(head_dim >= 1 && head_dim <= kMaxHeadDim, "head_dim outside 1..256");
  need((long long)batch * kv_heads * (capacity / kReadRows + 1) < (1ll << 31) - 1, "sizes too large");
}

bool apart(const void* a, const void* a_end, const void* b, const void* b_end) {
  return reinterpret_cast<uintptr_t>(a_end) <= reinterpret_cast<uintptr_t>(b) ||
         reinterpret_cast<uintptr_t>(b_end) <= reinterpret_cast<uintptr_t>(a);
}

template <class F>
void by_type(int dtype, F f) {
  if (dtype == CKKS_BF16)
    f(__nv_bfloat16{});
  else if (dtype == CKKS_FP16)
    f(__half{});
  else
    f(float{});
}

// a call's k and v, and the caches they go to, do not overlap
void check_apart(const ckks_rows& cache, int batch, int heads, int capacity, int row, int e, const ckks_rows& fresh,
                 int fresh_batch, int fresh_rows, int head_dim, int fe) {
  if (capacity && fresh_rows)
    need(apart(cache.data, end_of(cache, batch, heads, capacity, row, e), fresh.data,
               end_of(fresh, fresh_batch, heads, fresh_rows, head_dim, fe)),
         "new rows overlap the cache");
}

int run_fill(ckks_ctx* ctx, const ckks_draft_fill_args* args, void* stream, bool four) {
  return guard([&] {
    Context& c = context_of(ctx);
    need(args != nullptr, "null argument");
    const ckks_draft_fill_args& a = *args;
    check_sizes(a.dtype, a.batch, a.kv_heads, a.head_dim, a.capacity);
    need(a.tokens >= 0 && a.tokens < (1 << 30), "token count out of range");
    need((long long)a.batch + a.tokens / 4 < (1ll << 31) - 1, "sizes too large");
    if (a.batch == 0) return;
    const int e = element_bytes(a.dtype), R = four ? row4_bytes(a.head_dim) : a.head_dim;
    if (a.capacity)
      for (const ckks_rows* r : {&a.k_cache, &a.v_cache}) {
        check_rows(*r, four ? 1 : e, r == &a.k_cache ? "k_cache" : "v_cache");
        if (four) check_row4(*r, a.batch, a.kv_heads, a.capacity, r == &a.k_cache ? "k_cache" : "v_cache");
      }
    if (a.tokens) {
      check_rows(a.k, e, "k");
      check_rows(a.v, e, "v");
    }
    check_ptr(a.starts, "starts");
    check_ptr(a.lens, "lens");
    check_ptr(a.lens_out, "lens_out");
    need(apart(a.lens, a.lens + a.batch, a.lens_out, a.lens_out + a.batch), "lens_out overlaps lens");
    need(apart(a.starts, a.starts + a.batch + 1, a.lens_out, a.lens_out + a.batch), "lens_out overlaps starts");
    for (const ckks_rows* cache : {&a.k_cache, &a.v_cache})
      for (const ckks_rows* fresh : {&a.k, &a.v})
        check_apart(*cache, a.batch, a.kv_heads, a.capacity, R, four ? 1 : e, *fresh, 1, a.tokens, a.head_dim, e);
    // Chunks of 16 rows (40500 rows of 8 heads of 128 and their reading back take
    // 135.8, 131.9 and 131.9 us in chunks of 8, 16 and 64), down to 4 where that
    // leaves SMs without work: a chunk's rows come one behind the other
    const int rows = std::clamp(a.tokens / (8 * c.sms), 4, 16);
    const FillParams p{a.k_cache, a.v_cache,    a.k,     a.v,        a.starts,   a.lens,  a.lens_out,
                       c.d_faults + 1, a.batch, a.kv_heads, a.head_dim, a.tokens, a.capacity, rows};
    bool wide = wide_rows(a.k, 1, a.kv_heads, a.tokens, a.head_dim, e) &&
                wide_rows(a.v, 1, a.kv_heads, a.tokens, a.head_dim, e);
    if (!four)
      wide = wide && wide_rows(a.k_cache, a.batch, a.kv_heads, a.capacity, a.head_dim, e) &&
             wide_rows(a.v_cache, a.batch, a.kv_heads, a.capacity, a.head_dim, e);
    OnDevice dev(c);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    ProfScope ps(c, four ? "draft_fill4" : "draft_fill", 2.0 * a.tokens * a.kv_heads * (a.head_dim * e + R * (four ? 1 : e)),
                 st);
    // every sequence has a chunk at least, and a part of one at most
    const unsigned grid = (unsigned)(a.batch + a.tokens / rows);
    by_type(a.dtype, [&](auto t) {
      using T = decltype(t);
      if (four && wide)
        fill_kernel<T, T, true, true><<<grid, kFillThreads, 0, st>>>(p);
      else if (four)
        fill_kernel<T, T, true, false><<<grid, kFillThreads, 0, st>>>(p);
      else if (wide)
        fill_kernel<T, uint4, false, true><<<grid, kFillThreads, 0, st>>>(p);
      else
        fill_kernel<T, T, false, false><<<grid, kFillThreads, 0, st>>>(p);
    });
    CKKS_CUDA(cudaGetLastError());
  });
}

}  // namespace
}  // namespace draft
}  // namespace ckks

using namespace ckks;
using namespace ckks::draft;

extern "C" int ckks_draft_row4_bytes(int head_dim) {
  int n = -1;
  guard([&] {
    need(head_dim >= 1 && head_dim <= kMaxHeadDim, "head_dim outside 1..256");
    n = row4_bytes(head_dim);
  });
  return n;
}

extern "C" int ckks_draft_fill(ckks_ctx* ctx, const ckks_draft_fill_args* args, void* stream) {
  return run_fill(ctx, args, stream, false);
}

extern "C" int ckks_draft_fill4(ckks_ctx* ctx, const ckks_draft_fill_args* args, void* stream) {
  return run_fill(ctx, args, stream, true);
}

extern "C" int ckks_draft_commit4(ckks_ctx* ctx, const ckks_draft_commit_args* args, void* stream) {
  return guard([&] {
    Context& c = context_of(ctx);
    need(args != nullptr, "null argument");
    const ckks_draft_commit_args& a = *args;
    check_sizes(a.dtype, a.batch, a.kv_heads, a.head_dim, a.capacity);
    need(a.nodes >= 1 && a.nodes <= kMaxNodes, "node count outside 1..64");
    if (a.batch == 0) return;
    const int e = element_bytes(a.dtype), R = row4_bytes(a.head_dim);
    if (a.capacity) {
      check_rows(a.k_cache, 1, "k_cache");
      check_rows(a.v_cache, 1, "v_cache");
      check_row4(a.k_cache, a.batch, a.kv_heads, a.capacity, "k_cache");
      check_row4(a.v_cache, a.batch, a.kv_heads, a.capacity, "v_cache");
    }
    check_rows(a.k_new, e, "k_new");
    check_rows(a.v_new, e, "v_new");
    check_ptr(a.lens, "lens");
    check_ptr(a.path, "path");
    check_ptr(a.count, "count");
    check_ptr(a.lens_out, "lens_out");
    need(apart(a.lens, a.lens + a.batch, a.lens_out, a.lens_out + a.batch), "lens_out overlaps lens");
    for (const ckks_rows* cache : {&a.k_cache, &a.v_cache})
      for (const ckks_rows* fresh : {&a.k_new, &a.v_new})
        check_apart(*cache, a.batch, a.kv_heads, a.capacity, R, 1, *fresh, a.batch, a.nodes, a.head_dim, e);
    const Commit4Params p{a.k_cache, a.v_cache,    a.k_new, a.v_new,    a.lens,     a.path,  a.count,
                          a.lens_out, c.d_faults + 1, a.batch, a.kv_heads, a.head_dim, a.nodes, a.capacity};
    const bool wide = wide_rows(a.k_new, a.batch, a.kv_heads, a.nodes, a.head_dim, e) &&
                      wide_rows(a.v_new, a.batch, a.kv_heads, a.nodes, a.head_dim, e);
    OnDevice dev(c);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    ProfScope ps(c, "draft_commit4", 2.0 * a.batch * a.kv_heads * a.nodes * (a.head_dim * e + R), st);
    by_type(a.dtype, [&](auto t) {
      using T = decltype(t);
      if (wide)
        commit4_kernel<T, true><<<dim3(a.batch, a.kv_heads), 128, 0, st>>>(p);
      else
        commit4_kernel<T, false><<<dim3(a.batch, a.kv_heads), 128, 0, st>>>(p);
    });
    CKKS_CUDA(cudaGetLastError());
  });
}

extern "C" int ckks_draft_read4(ckks_ctx* ctx, const ckks_draft_read4_args* args, void* stream) {
  return guard([&] {
    Context& c = context_of(ctx);
    need(args != nullptr, "null argument");
    const ckks_draft_read4_args& a = *args;
    check_sizes(a.dtype, a.batch, a.kv_heads, a.head_dim, a.capacity);
    need(a.reserved == 0, "reserved field is not 0");
    if (a.batch == 0 || a.capacity == 0) return;
    const int e = element_bytes(a.dtype), R = row4_bytes(a.head_dim);
    check_rows(a.cache, 1, "cache");
    check_row4(a.cache, a.batch, a.kv_heads, a.capacity, "cache");
    check_rows(a.out, e, "out");
    check_ptr(a.lens, "lens");
    need(apart(a.cache.data, end_of(a.cache, a.batch, a.kv_heads, a.capacity, R, 1), a.out.data,
               end_of(a.out, a.batch, a.kv_heads, a.capacity, a.head_dim, e)),
         "out overlaps the cache");
    // Chunks of 128 rows (131.2 us in the example above, 134.7 and 132.9 with 64 and
    // 224), fewer where that leaves SMs without work
    const long long all = (long long)a.batch * a.kv_heads * a.capacity;
    const int rows = (int)std::clamp<long long>(all / (8 * c.sms) / kReadRows * kReadRows, kReadRows, 4 * kReadRows);
    const ReadParams p{a.cache, a.out, a.lens, a.batch, a.kv_heads, a.head_dim, a.capacity, rows};
    const bool wide = wide_rows(a.out, a.batch, a.kv_heads, a.capacity, a.head_dim, e);
    OnDevice dev(c);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    ProfScope ps(c, "draft_read4", (double)a.batch * a.kv_heads * a.capacity * (a.head_dim * e + R), st);
    const dim3 grid((unsigned)((a.capacity + rows - 1) / rows), (unsigned)a.kv_heads, (unsigned)std::min(a.batch, 65535));
    by_type(a.dtype, [&](auto t) {
      using T = decltype(t);
      if (wide)
        read4_kernel<T, true><<<grid, 256, 0, st>>>(p);
      else
        read4_kernel<T, false><<<grid, 256, 0, st>>>(p);
    });
    CKKS_CUDA(cudaGetLastError());
  });
}
