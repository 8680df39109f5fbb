// draft_verify.cu -- acceptance of drafted tokens against the target's
// probabilities from given random numbers, and the token that follows them
// (ckks_draft_verify).
//
// With children c drawn from the draft's row q, child c with token x is kept
// when u_c q(x) < p(x), and each child refused replaces the target's row p by
// max(p - q, 0) / Z, Z = sum max(p - q, 0): the tokens kept, and the one drawn
// from what p is at the end, are distributed as the target's.  Only the rows
// of the last node reached are needed whole; every other node takes two
// values.  All sums are in float64: a token is decided by comparing a running
// sum over the vocabulary with u times the whole one.
#include "draft.hpp"

namespace ckks {
namespace draft {
namespace {

constexpr int kThreads = 1024, kWarps = kThreads / 32;

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

// p(x) after the refusals so far: `refused` normalisers in z
__device__ __forceinline__ double remaining(double t, double q, const double* z, int refused) {
  double r = t > 0.0 ? t : 0.0;
  const double d = q > 0.0 ? q : 0.0;
  for (int k = 0; k < refused; ++k) {
    r -= d;
    r = r > 0.0 ? r / z[k] : 0.0;
  }
  return r;
}

// One CTA per sequence.  The walk needs p and q at the drafts' tokens only,
// which the threads fetch for all nodes at once, each in its parent's row; a
// refusal costs one pass over that row for Z.  The last token is found by
// descending radix 32: the warps sum 32 pieces of the row, the piece in which
// the running sum passes u Z is cut into 32 again, down to single entries.
template <typename TT, typename TD>
__global__ void __launch_bounds__(kThreads) verify_kernel(VerifyParams p) {
  __shared__ double s_p[kMaxNodes], s_q[kMaxNodes], s_u[kMaxNodes + 1], s_z[kMaxNodes], s_sum[kWarps];
  __shared__ int s_parent[kMaxNodes];
  __shared__ int s_last[kWarps];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const TT* target = static_cast<const TT*>(p.target.data) + b * p.target.batch;
  const TD* draft = static_cast<const TD*>(p.draft.data) + b * p.draft.batch;
  const int n = p.nodes, V = p.vocab;
  if (tid < n) {
    const int x = p.tokens[(size_t)b * n + tid];
    int par = p.parents[(size_t)b * n + tid];
    if (par < -1 || par >= tid) par = -2;
    s_parent[tid] = par;
    const bool known = par >= -1 && x >= 0 && x < V;
    s_p[tid] = known ? (double)target[(par + 1) * p.target.row + x] : 0.0;
    s_q[tid] = known ? (double)draft[(par + 1) * p.draft.row + x] : 0.0;
  }
  if (tid <= n) s_u[tid] = p.uniforms[(size_t)b * (n + 1) + tid];
  __syncthreads();
  int at = -1, kept = 0, refused = 0;
  for (int i = 0; i < n; ++i) {
    if (s_parent[i] != at) continue;
    const TT* t = target + (at + 1) * p.target.row;
    const TD* q = draft + (at + 1) * p.draft.row;
    const double px = remaining(s_p[i], s_q[i], s_z, refused), qx = s_q[i] > 0.0 ? s_q[i] : 0.0;
    if (s_u[i] * qx < px) {
      if (tid == 0) p.path[(size_t)b * n + kept] = i;
      ++kept;
      at = i;
      refused = 0;
      __syncthreads();  // s_z is written anew
      continue;
    }
    // the refused child's normaliser
    double z = 0.0;
    for (int x = tid; x < V; x += kThreads) {
      const double d = q[x] > 0 ? (double)q[x] : 0.0;
      const double r = remaining((double)t[x], d, s_z, refused) - d;
      z += r > 0.0 ? r : 0.0;
    }
    z = warp_sum(z);
    if (lane == 0) s_sum[warp] = z;
    __syncthreads();
    z = 0.0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) z += s_sum[w];
    if (z > 0.0) {
      if (tid == 0) s_z[refused] = z;
      ++refused;
    }
    __syncthreads();
  }
  if (tid >= kept && tid < n) p.path[(size_t)b * n + tid] = -1;
  if (tid == 0) p.count[b] = kept;
  // the next token, from p as it stands
  const TT* t = target + (at + 1) * p.target.row;
  const TD* q = draft + (at + 1) * p.draft.row;
  auto value = [&](int x) { return remaining((double)t[x], refused ? (double)q[x] : 0.0, s_z, refused); };
  int lo = 0, size = V;  // the piece searched
  double before = 0.0, goal = -1.0;
  int last = 0;  // the last entry above 0, for a goal that rounding put at the whole sum
  while (true) {
    const int piece = (size + kWarps - 1) / kWarps;
    const int w0 = lo + min(size, warp * piece), w1 = lo + min(size, (warp + 1) * piece);
    double s = 0.0;
    int mine = -1;
    for (int x = w0 + lane; x < w1; x += 32) {
      const double v = value(x);
      s += v;
      if (v > 0.0) mine = x;
    }
    s = warp_sum(s);
    mine = __reduce_max_sync(0xffffffffu, mine);
    if (lane == 0) {
      s_sum[warp] = s;
      s_last[warp] = mine;
    }
    __syncthreads();
    if (goal < 0.0) {
      double all = 0.0;
      for (int w = 0; w < kWarps; ++w) {
        all += s_sum[w];
        if (s_last[w] >= 0) last = s_last[w];
      }
      goal = s_u[n] * all;
    }
    // the first piece that passes the goal, else none
    int hit = -1;
    double run = before;
    for (int w = 0; w < kWarps; ++w) {
      const double next = run + s_sum[w];
      if (next > goal) {
        hit = w;
        break;
      }
      run = next;
    }
    __syncthreads();
    if (hit < 0) {
      lo = last;
      break;
    }
    before = run;
    lo += min(size, hit * piece);
    if (piece == 1) break;
    size = min(piece, V - lo);
  }
  if (tid == 0) p.token[b] = lo;
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
      verify_kernel<double, double><<<a.batch, kThreads, 0, st>>>(p);
    else if (td)
      verify_kernel<double, float><<<a.batch, kThreads, 0, st>>>(p);
    else if (dd)
      verify_kernel<float, double><<<a.batch, kThreads, 0, st>>>(p);
    else
      verify_kernel<float, float><<<a.batch, kThreads, 0, st>>>(p);
    CKKS_CUDA(cudaGetLastError());
  });
}
