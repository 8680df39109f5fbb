// draft_verify.cu -- acceptance of drafted tokens against the target's
// probabilities from given random numbers, and the token that follows them
// (ckks_draft_verify).
//
// With children c drawn from the draft's row q, child c with token x is kept
// when u_c q(x) < p(x), and each child refused replaces the target's row p by
// max(p - q, 0) / Z, Z = sum max(p - q, 0): the tokens kept, and the one drawn
// from what p is at the end, are distributed as the target's.  After any
// number of refusals p is max(p0 - a q, 0) / S for the row p0 given, with
// a = 0, S = 1 at first, and a refusal makes of them
//   a' = a + S,  S' = sum max(p0 - a' q, 0)
// (max(p - q, 0) = max(max(p0 - a q, 0) - S q, 0) / S), so a refusal is one
// multiply-add for each entry, however many came before.
//
// Only the rows of the nodes at which a child is refused, or the walk ends,
// are needed whole; every other node takes two values.  All of it is in
// float64: a token is decided by comparing a running sum over the vocabulary
// with u times the whole one.
#include <algorithm>

#include "draft.hpp"

namespace ckks {
namespace draft {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;

struct VerifyParams {
  ckks_rows target, draft;
  const int32_t* tokens;
  const int32_t* parents;
  const double* uniforms;
  int32_t* path;
  int32_t* count;
  int32_t* token;
  int batch, nodes, vocab;
};

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
  for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// a probability; what is not above 0 (NaN among it) is 0
__device__ __forceinline__ double weight(float x) { return (double)fmaxf(x, 0.0f); }
__device__ __forceinline__ double weight(double x) { return x > 0.0 ? x : 0.0; }

// what is left of p(x), times S: max(p - a q, 0).  The comparison looks at the
// sign bit: float64 instructions are the scarce ones here
__device__ __forceinline__ double left_of(double p, double q, double a) {
  const double r = fma(-a, q, p);
  return __double2hiint(r) < 0 ? 0.0 : r;
}

// A cluster of C CTAs per sequence, each with a contiguous share of the
// vocabulary and each warp with a contiguous part of that; a thread keeps the
// first kHeld of its entries of the row at hand in registers, so refusals at
// one node and the last draw read the row once (larger vocabularies read the
// rest again, from L2).  Every CTA walks the tree alike: the walk needs p and
// q at the drafts' tokens only, which the threads fetch for all nodes at once,
// each in its parent's row.  Sums add the CTAs' parts in their order.
// Bound by the slowest sequence's chain: each refusal is a row from HBM, two
// conversions, a multiply-add and an add in float64 for each entry, and a
// cluster barrier, 3 to 4 us; 64 trees of 31 over 32003 entries take 20.0 us, one
// chain of 5 over 4103 7.2 us.  (One CTA a sequence took 61 us.)
template <typename TT, typename TD, int C>
__global__ void __launch_bounds__(kThreads, sizeof(TT) + sizeof(TD) == 8 ? 2 : 1) verify_kernel(VerifyParams p) {
  constexpr int kHeld = sizeof(TT) + sizeof(TD) == 8 ? 16 : 8;
  __shared__ double s_p[kMaxNodes], s_q[kMaxNodes], s_u[kMaxNodes + 1], s_sum[kWarps], s_part[2];
  __shared__ int s_parent[kMaxNodes], s_last[kWarps], s_tail;
  const int b = blockIdx.x / C, rank = C > 1 ? blockIdx.x % C : 0;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const TT* target = static_cast<const TT*>(p.target.data) + b * p.target.batch;
  const TD* draft = static_cast<const TD*>(p.draft.data) + b * p.draft.batch;
  const int n = p.nodes, V = p.vocab;
  if (tid < n) {
    const int x = p.tokens[(size_t)b * n + tid];
    int par = p.parents[(size_t)b * n + tid];
    if (par < -1 || par >= tid) par = -2;
    s_parent[tid] = par;
    const bool known = par >= -1 && x >= 0 && x < V;
    s_p[tid] = known ? weight(target[(par + 1) * p.target.row + x]) : 0.0;
    s_q[tid] = known ? weight(draft[(par + 1) * p.draft.row + x]) : 0.0;
  }
  if (tid >= kThreads - 128 && tid - (kThreads - 128) <= n)
    s_u[tid - (kThreads - 128)] = p.uniforms[(size_t)b * (n + 1) + tid - (kThreads - 128)];
  // this warp's entries [x0, x1)
  const int share = (V + C - 1) / C, lo = min(V, rank * share), hi = min(V, lo + share);
  const int part = (share + kWarps - 1) / kWarps, x0 = min(hi, lo + warp * part), x1 = min(hi, x0 + part);
  __syncthreads();
  TT hp[kHeld];
  TD hq[kHeld];
  int row = -2, at = -1, kept = 0, flip = 0;
  auto hold = [&] {
    if (row == at) return;
    row = at;
    const TT* t = target + (at + 1) * p.target.row;
    const TD* q = draft + (at + 1) * p.draft.row;
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
      const int x = x0 + 32 * k + lane;
      hp[k] = x < x1 ? t[x] : (TT)0;
      hq[k] = x < x1 ? q[x] : (TD)0;
    }
  };
  // f(x, what is left of p(x)) for this thread's entries
  auto each = [&](double a, auto&& f) {
#pragma unroll
    for (int k = 0; k < kHeld; ++k) f(x0 + 32 * k + lane, left_of(weight(hp[k]), weight(hq[k]), a));
    const TT* t = target + (at + 1) * p.target.row;
    const TD* q = draft + (at + 1) * p.draft.row;
    for (int x = x0 + 32 * kHeld + lane; x < x1; x += 32 * 8) {
      TT tp[8];
      TD tq[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        tp[k] = x + 32 * k < x1 ? t[x + 32 * k] : (TT)0;
        tq[k] = x + 32 * k < x1 ? q[x + 32 * k] : (TD)0;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) f(x + 32 * k, left_of(weight(tp[k]), weight(tq[k]), a));
    }
  };
  // sums over the warp, the CTA (s_sum[warp] holds the warps') and the cluster
  auto sum_all = [&](double a, double* before) {
    double s = 0.0;
    each(a, [&](int, double r) { s += r; });
    s = warp_sum(s);
    __syncthreads();
    if (lane == 0) s_sum[warp] = s;
    __syncthreads();
    s = 0.0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) s += s_sum[w];
    if (before) *before = 0.0;
    if constexpr (C > 1) {
      // two places in turn: a CTA may be one sum ahead of one that still reads
      flip ^= 1;
      if (tid == 0) s_part[flip] = s;
      cluster_sync();
      double all = 0.0;
#pragma unroll
      for (int r = 0; r < C; ++r) {
        if (before && r == rank) *before = all;
        all += cluster_read(&s_part[flip], r);
      }
      s = all;
    }
    return s;
  };
  double a = 0.0, S = 1.0;
  for (int i = 0; i < n; ++i) {
    if (s_parent[i] != at) continue;
    if (s_u[i] * s_q[i] < left_of(s_p[i], s_q[i], a) / S) {
      if (tid == 0 && rank == 0) p.path[(size_t)b * n + kept] = i;
      ++kept;
      at = i;
      a = 0.0, S = 1.0;
      continue;
    }
    hold();
    const double z = sum_all(a + S, nullptr);
    if (z > 0.0) a += S, S = z;
  }
  if (rank == 0) {
    if (tid >= kept && tid < n) p.path[(size_t)b * n + tid] = -1;
    if (tid == 0) p.count[b] = kept;
  }
  // the next token, from p as it stands: the CTA, the warp in it and the
  // entry at which the running sum passes u times the whole one
  hold();
  double before;
  const double goal = s_u[n] * sum_all(a, &before);
  int last = -1;  // the last entry above 0, for a goal that rounding put at the whole sum
  each(a, [&](int x, double r) {
    if (x < x1 && r > 0.0) last = x;
  });
  last = __reduce_max_sync(0xffffffffu, last);
  if (lane == 0) s_last[warp] = last;
  __syncthreads();
  double run = before;
  int hit = -1, tail = -1;
  double start = 0.0;
  for (int w = 0; w < kWarps; ++w) {
    tail = max(tail, s_last[w]);
    const double next = run + s_sum[w];
    if (hit < 0 && next > goal) hit = w, start = run;
    run = next;
  }
  // of the CTAs that pass the goal the first is the one
  bool mine = hit >= 0, none = !mine;
  if constexpr (C > 1) {
    flip ^= 1;
    if (tid == 0) s_part[flip] = hit >= 0 ? 1.0 : 0.0, s_tail = tail;
    cluster_sync();
#pragma unroll
    for (int r = 0; r < C; ++r) {
      const bool theirs = cluster_read(&s_part[flip], r) != 0.0;
      if (r < rank && theirs) mine = false;
      none = none && !theirs;
      tail = max(tail, cluster_read(&s_tail, r));
    }
  }
  if (none) {
    if (tid == 0 && rank == 0) p.token[b] = max(tail, 0);
  } else if (mine) {
    // the warps cut the part of the warp that passed the goal into theirs,
    // and the one that passes it there walks its few entries
    const TT* t = target + (at + 1) * p.target.row;
    const TD* q = draft + (at + 1) * p.draft.row;
    const int h0 = min(hi, lo + hit * part), h1 = min(hi, h0 + part), cut = (h1 - h0 + kWarps - 1) / kWarps;
    const int y0 = min(h1, h0 + warp * cut), y1 = min(h1, y0 + cut);
    double s = 0.0;
    last = -1;
    for (int x = y0 + lane; x < y1; x += 32) {
      const double r = left_of(weight(t[x]), weight(q[x]), a);
      s += r;
      if (r > 0.0) last = x;
    }
    s = warp_sum(s);
    last = __reduce_max_sync(0xffffffffu, last);
    __syncthreads();
    if (lane == 0) s_sum[warp] = s, s_last[warp] = last;
    __syncthreads();
    double base = start;
    hit = tail = -1;
    for (int w = 0; w < kWarps && hit < 0; ++w) {
      tail = max(tail, s_last[w]);
      if (base + s_sum[w] > goal)
        hit = w;
      else
        base += s_sum[w];
    }
    if (warp == max(hit, 0)) {
      int found = -1;
      for (int x = y0; hit >= 0 && x < y1 && found < 0; x += 32) {
        const double own = x + lane < y1 ? left_of(weight(t[x + lane]), weight(q[x + lane]), a) : 0.0;
        double v = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double y = __shfl_up_sync(0xffffffffu, v, o);
          if (lane >= o) v += y;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, own > 0.0 && base + v > goal);
        if (past) found = x + __ffs(past) - 1;
        base += __shfl_sync(0xffffffffu, v, 31);
      }
      // another order of the same sum may end just below the goal
      if (lane == 0) p.token[b] = found >= 0 ? found : tail;
    }
  }
  if constexpr (C > 1) cluster_sync();  // no CTA ends while another may read its parts
}

template <typename TT, typename TD>
void run_verify(const Context& c, const VerifyParams& p, cudaStream_t st) {
  // as many CTAs as the SMs take at once (two on each), none with less than
  // 1024 entries
  const int most = std::min(2 * c.sms / std::max(1, p.batch), p.vocab / 1024);
  if (most >= 8)
    launch_cluster<8>(verify_kernel<TT, TD, 8>, p.batch, kThreads, st, p);
  else if (most >= 4)
    launch_cluster<4>(verify_kernel<TT, TD, 4>, p.batch, kThreads, st, p);
  else if (most >= 2)
    launch_cluster<2>(verify_kernel<TT, TD, 2>, p.batch, kThreads, st, p);
  else
    launch_cluster<1>(verify_kernel<TT, TD, 1>, p.batch, kThreads, st, p);
}

void check_rows2(const ckks_rows& r, int dtype, const char* what) {
  need(dtype == CKKS_FP32 || dtype == CKKS_FP64, "probabilities are CKKS_FP32 or CKKS_FP64");
  check_rows(r, element_bytes(dtype), what);
}

}  // namespace
}  // namespace draft
}  // namespace ckks

using namespace ckks;
using namespace ckks::draft;

extern "C" int ckks_draft_verify(ckks_ctx* ctx, const ckks_draft_verify_args* args, void* stream) {
  return guard([&] {
    Context& c = context_of(ctx);
    need(args != nullptr, "null argument");
    const ckks_draft_verify_args& a = *args;
    need(a.reserved == 0, "reserved field is not 0");
    need(a.batch >= 0, "negative batch");
    need(a.nodes >= 1 && a.nodes <= kMaxNodes, "node count outside 1..64");
    need(a.vocab >= 1 && a.vocab < (1 << 30), "vocabulary size out of range");
    if (a.batch == 0) return;
    check_rows2(a.target, a.target_dtype, "target");
    check_rows2(a.draft, a.draft_dtype, "draft");
    check_ptr(a.tokens, "tokens");
    check_ptr(a.parents, "parents");
    check_ptr(a.uniforms, "uniforms");
    check_ptr(a.path, "path");
    check_ptr(a.count, "count");
    check_ptr(a.token, "token");
    VerifyParams p{a.target, a.draft, a.tokens, a.parents, a.uniforms, a.path, a.count, a.token, a.batch, a.nodes,
                   a.vocab};
    OnDevice dev(c);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    ProfScope ps(c, "draft_verify",
                 (double)a.batch * a.vocab * (element_bytes(a.target_dtype) + element_bytes(a.draft_dtype)), st);
    const bool td = a.target_dtype == CKKS_FP64, dd = a.draft_dtype == CKKS_FP64;
    if (td && dd)
      run_verify<double, double>(c, p, st);
    else if (td)
      run_verify<double, float>(c, p, st);
    else if (dd)
      run_verify<float, double>(c, p, st);
    else
      run_verify<float, float>(c, p, st);
  });
}
