// torch_draft.cpp -- the drafted-decoding operators on torch tensors: checks
// the arguments, allocates the outputs, and calls the C entry points of
// include/ckks_b200.h on torch's current stream.  A decode step makes a few
// of these calls for each layer, most of them shorter than the interpreter
// takes to look at their arguments, so this is compiled (drafting.py holds
// the documentation).
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <cmath>
#include <optional>
#include <tuple>

#include "../../include/ckks_b200.h"

namespace {

using at::Tensor;

// the context and its device; index -1 stands for the CPU, whose tensors pass
// the checks and reach the entry points' own
struct Call {
  ckks_ctx* ctx;
  int device;
  bool grad = at::GradMode::is_enabled();
  bool forward_grad = c10::AutogradState::get_tls_state().get_fw_grad_mode();
  void* stream() const { return device < 0 ? nullptr : (void*)c10::cuda::getCurrentCUDAStream(device).stream(); }
  void done(int rc) const {
    if (rc == CKKS_OK) return;
    const pybind11::object type = pybind11::module::import("private_genomic_dnagpt_b200").attr("CKKSError");
    PyErr_SetObject(type.ptr(), type(rc, ckks_last_error()).ptr());
    throw pybind11::error_already_set();
  }
};

int type_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return CKKS_BF16;
    case at::kHalf: return CKKS_FP16;
    case at::kFloat: return CKKS_FP32;
    case at::kDouble: return CKKS_FP64;
    default: return -1;
  }
}

int cache_type(const Tensor& t, const char* name) {
  const int code = type_code(t);
  TORCH_CHECK_VALUE(code >= 0 && code != CKKS_FP64, name, ": expected bfloat16, float16 or float32, got ", t.dtype());
  return code;
}

// a size in an argument struct
int32_t size32(int64_t n, const char* what) {
  TORCH_CHECK_VALUE(n <= INT32_MAX, what, ": ", n, " is more than the entry points take");
  return (int32_t)n;
}

void four(const Tensor& t, const char* name) { TORCH_CHECK_VALUE(t.dim() == 4, name, ": expected four dimensions"); }

void check(const Call& c, const Tensor& t, const char* name, at::IntArrayRef shape, at::ScalarType type) {
  TORCH_CHECK_VALUE(t.sizes() == shape, name, ": expected the shape ", shape, ", got ", t.sizes());
  TORCH_CHECK_VALUE(t.scalar_type() == type, name, ": expected ", type, ", got ", t.scalar_type());
  TORCH_CHECK_VALUE(c.device < 0 ? t.is_cpu() : t.is_cuda() && t.get_device() == c.device, name,
                    ": expected a tensor of the context's device, cuda:", c.device, ", got ", t.device());
  TORCH_CHECK_VALUE(!(c.grad && t.requires_grad()), name,
                    ": requires a gradient, which this operator does not have (call it under torch.no_grad)");
  TORCH_CHECK_VALUE(!(c.forward_grad && t._fw_grad(/*level=*/0).defined()), name,
                    ": carries a forward-mode gradient, which this operator does not have");
  TORCH_CHECK_VALUE(!t.is_neg(), name, ": a view whose memory holds the negated values (resolve_neg makes a copy)");
}

// a tensor of rows: any strides, the last dimension contiguous
void check_rows(const Call& c, const Tensor& t, const char* name, at::IntArrayRef shape, at::ScalarType type) {
  check(c, t, name, shape, type);
  TORCH_CHECK_VALUE(t.stride(-1) == 1 || shape.back() <= 1 || t.numel() == 0, name,
                    ": its last dimension must be contiguous");
}

template <typename P>
P* small(const Call& c, const Tensor& t, const char* name, at::IntArrayRef shape, at::ScalarType type) {
  check(c, t, name, shape, type);
  TORCH_CHECK_VALUE(t.is_contiguous(), name, ": must be contiguous");
  return static_cast<P*>(t.data_ptr());
}

// refuses a tensor whose elements share memory along an expanded dimension
void check_written(const Tensor& t, const char* name) {
  for (int64_t i = 0; i < t.dim(); ++i)
    TORCH_CHECK_VALUE(t.size(i) <= 1 || t.stride(i) != 0, name, ": is written, but some of its elements share memory");
}

ckks_rows by_head(const Tensor& t) { return {t.data_ptr(), t.stride(0), t.stride(1), t.dim() > 3 ? t.stride(2) : 0}; }
ckks_rows by_node(const Tensor& t) { return {t.data_ptr(), t.stride(0), t.stride(2), t.stride(1)}; }

template <typename A>
Tensor workspace(const Call& c, long long bytes, A& a, const Tensor& like) {
  if (bytes < 0) c.done(CKKS_EARG);
  Tensor t;
  if (bytes > 0) {
    t = at::empty({(int64_t)bytes}, like.options().dtype(at::kByte));
    a.workspace = t.data_ptr();
    a.workspace_bytes = (size_t)bytes;
  }
  return t;
}

double scale_of(std::optional<double> scale, int64_t d) { return scale ? *scale : 1.0 / std::sqrt((double)d); }

std::tuple<Tensor, Tensor> attention(uintptr_t ctx, int device, const Tensor& q, const Tensor& k_cache,
                                     const Tensor& v_cache, const Tensor& lens, const Tensor& k_new,
                                     const Tensor& v_new, const Tensor& parents, std::optional<double> scale) {
  const Call c{(ckks_ctx*)ctx, device};
  four(q, "q");
  four(k_cache, "k_cache");
  const int64_t b = q.size(0), n = q.size(1), hq = q.size(2), d = q.size(3), hk = k_cache.size(1), cap = k_cache.size(2);
  const auto t = q.scalar_type();
  const int code = cache_type(q, "q");
  check_rows(c, q, "q", {b, n, hq, d}, t);
  check_rows(c, k_cache, "k_cache", {b, hk, cap, d}, t);
  check_rows(c, v_cache, "v_cache", {b, hk, cap, d}, t);
  check_rows(c, k_new, "k_new", {b, n, hk, d}, t);
  check_rows(c, v_new, "v_new", {b, n, hk, d}, t);
  ckks_draft_attention_args a{};
  a.lens = small<const int32_t>(c, lens, "lens", {b}, at::kInt);
  a.parents = small<const int32_t>(c, parents, "parents", {b, n}, at::kInt);
  Tensor out = at::empty({b, n, hq, d}, q.options()), lse = at::empty({b, n, hq}, q.options().dtype(at::kFloat));
  if (b == 0) return {out, lse};
  a.dtype = code, a.batch = size32(b, "batch"), a.q_heads = size32(hq, "query heads");
  a.kv_heads = size32(hk, "key/value heads"), a.head_dim = size32(d, "head size"), a.nodes = size32(n, "nodes");
  a.capacity = size32(cap, "capacity"), a.scale = scale_of(scale, d);
  a.q = by_node(q), a.k_cache = by_head(k_cache), a.v_cache = by_head(v_cache);
  a.k_new = by_node(k_new), a.v_new = by_node(v_new), a.out = by_node(out);
  a.lse = lse.data_ptr<float>();
  const Tensor ws = workspace(c, ckks_draft_attention_workspace(c.ctx, &a), a, q);
  c.done(ckks_draft_attention(c.ctx, &a, c.stream()));
  return {out, lse};
}

std::tuple<Tensor, Tensor, Tensor> verify(uintptr_t ctx, int device, const Tensor& target, const Tensor& draft,
                                          const Tensor& tokens, const Tensor& parents, const Tensor& uniforms) {
  const Call c{(ckks_ctx*)ctx, device};
  TORCH_CHECK_VALUE(target.dim() == 3 && target.size(1) >= 1, "target: expected [batch, nodes + 1, vocabulary]");
  const int64_t b = target.size(0), n = target.size(1) - 1, v = target.size(2);
  ckks_draft_verify_args a{};
  const auto probabilities = [&](const Tensor& t, const char* name, int32_t& code) {
    code = type_code(t);
    TORCH_CHECK_VALUE(code == CKKS_FP32 || code == CKKS_FP64, name, ": expected float32 or float64, got ", t.dtype());
    check_rows(c, t, name, {b, n + 1, v}, t.scalar_type());
    return ckks_rows{t.data_ptr(), t.stride(0), 0, t.stride(1)};
  };
  a.target = probabilities(target, "target", a.target_dtype);
  a.draft = probabilities(draft, "draft", a.draft_dtype);
  a.tokens = small<const int32_t>(c, tokens, "tokens", {b, n}, at::kInt);
  a.parents = small<const int32_t>(c, parents, "parents", {b, n}, at::kInt);
  a.uniforms = small<const double>(c, uniforms, "uniforms", {b, n + 1}, at::kDouble);
  Tensor path = at::empty({b, n}, tokens.options()), count = at::empty({b}, tokens.options()),
         token = at::empty({b}, tokens.options());
  if (b) {
    a.batch = size32(b, "batch"), a.nodes = size32(n, "nodes"), a.vocab = size32(v, "vocabulary");
    a.path = path.data_ptr<int32_t>(), a.count = count.data_ptr<int32_t>(), a.token = token.data_ptr<int32_t>();
    c.done(ckks_draft_verify(c.ctx, &a, c.stream()));
  }
  return {path, count, token};
}

Tensor commit(uintptr_t ctx, int device, const Tensor& k_cache, const Tensor& v_cache, const Tensor& lens,
              const Tensor& k_new, const Tensor& v_new, const Tensor& path, const Tensor& count) {
  const Call c{(ckks_ctx*)ctx, device};
  four(k_cache, "k_cache");
  four(k_new, "k_new");
  const int64_t b = k_cache.size(0), hk = k_cache.size(1), cap = k_cache.size(2), d = k_cache.size(3), n = k_new.size(1);
  const auto t = k_cache.scalar_type();
  ckks_draft_commit_args a{};
  a.dtype = cache_type(k_cache, "k_cache");
  check_rows(c, k_cache, "k_cache", {b, hk, cap, d}, t);
  check_rows(c, v_cache, "v_cache", {b, hk, cap, d}, t);
  check_written(k_cache, "k_cache");
  check_written(v_cache, "v_cache");
  check_rows(c, k_new, "k_new", {b, n, hk, d}, t);
  check_rows(c, v_new, "v_new", {b, n, hk, d}, t);
  a.lens = small<const int32_t>(c, lens, "lens", {b}, at::kInt);
  a.path = small<const int32_t>(c, path, "path", {b, n}, at::kInt);
  a.count = small<const int32_t>(c, count, "count", {b}, at::kInt);
  Tensor out = at::empty({b}, lens.options());
  if (b) {
    a.batch = size32(b, "batch"), a.kv_heads = size32(hk, "key/value heads"), a.head_dim = size32(d, "head size");
    a.nodes = size32(n, "nodes"), a.capacity = size32(cap, "capacity");
    a.k_cache = by_head(k_cache), a.v_cache = by_head(v_cache), a.k_new = by_node(k_new), a.v_new = by_node(v_new);
    a.lens_out = out.data_ptr<int32_t>();
    c.done(ckks_draft_commit(c.ctx, &a, c.stream()));
  }
  return out;
}

Tensor accumulate(uintptr_t ctx, int device, const Tensor& q, const Tensor& lse, const Tensor& k_cache,
                  const Tensor& lens, const Tensor& path, const Tensor& count, Tensor acc, std::optional<double> scale) {
  const Call c{(ckks_ctx*)ctx, device};
  four(q, "q");
  four(k_cache, "k_cache");
  const int64_t b = q.size(0), n = q.size(1), hq = q.size(2), d = q.size(3), hk = k_cache.size(1), cap = k_cache.size(2);
  ckks_draft_accumulate_args a{};
  a.dtype = cache_type(q, "q");
  check_rows(c, q, "q", {b, n, hq, d}, q.scalar_type());
  check_rows(c, k_cache, "k_cache", {b, hk, cap, d}, q.scalar_type());
  a.lse = small<const float>(c, lse, "lse", {b, n, hq}, at::kFloat);
  a.lens = small<const int32_t>(c, lens, "lens", {b}, at::kInt);
  a.path = small<const int32_t>(c, path, "path", {b, n}, at::kInt);
  a.count = small<const int32_t>(c, count, "count", {b}, at::kInt);
  check_rows(c, acc, "acc", {b, hk, cap}, at::kFloat);
  check_written(acc, "acc");
  if (b && cap) {
    a.batch = size32(b, "batch"), a.q_heads = size32(hq, "query heads"), a.kv_heads = size32(hk, "key/value heads");
    a.head_dim = size32(d, "head size"), a.nodes = size32(n, "nodes"), a.capacity = size32(cap, "capacity");
    a.scale = scale_of(scale, d);
    a.q = by_node(q), a.k_cache = by_head(k_cache), a.acc = by_head(acc);
    c.done(ckks_draft_accumulate(c.ctx, &a, c.stream()));
  }
  return acc;
}

using Caches = std::tuple<Tensor, Tensor, Tensor>;

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> evict(uintptr_t ctx, int device, const Tensor& k_cache,
                                                         const Tensor& v_cache, const Tensor& acc, const Tensor& lens,
                                                         int64_t budget, int64_t recent, std::optional<Caches> out) {
  const Call c{(ckks_ctx*)ctx, device};
  four(k_cache, "k_cache");
  const int64_t b = k_cache.size(0), hk = k_cache.size(1), cap = k_cache.size(2), d = k_cache.size(3);
  const auto t = k_cache.scalar_type();
  ckks_draft_evict_args a{};
  a.dtype = cache_type(k_cache, "k_cache");
  check_rows(c, k_cache, "k_cache", {b, hk, cap, d}, t);
  check_rows(c, v_cache, "v_cache", {b, hk, cap, d}, t);
  check_rows(c, acc, "acc", {b, hk, cap}, at::kFloat);
  a.lens = small<const int32_t>(c, lens, "lens", {b}, at::kInt);
  TORCH_CHECK_VALUE(budget >= 1 && budget < (1 << 30) && recent >= 0 && recent <= budget,
                    "budget: need budget >= 1 and 0 <= recent <= budget, got ", budget, " and ", recent);
  if (!out)
    out = Caches{at::zeros({b, hk, budget, d}, k_cache.options()), at::zeros({b, hk, budget, d}, k_cache.options()),
                 at::zeros({b, hk, budget}, acc.options())};
  Tensor k2 = std::get<0>(*out), v2 = std::get<1>(*out), a2 = std::get<2>(*out);
  four(k2, "out");
  const int64_t rows = k2.size(2);
  TORCH_CHECK_VALUE(rows >= budget, "out: ", rows, " rows are fewer than the budget of ", budget);
  check_rows(c, k2, "out", {b, hk, rows, d}, t);
  check_rows(c, v2, "out", {b, hk, rows, d}, t);
  check_rows(c, a2, "out", {b, hk, rows}, at::kFloat);
  for (const Tensor* x : {&k2, &v2, &a2}) check_written(*x, "out");
  Tensor index = at::empty({b, hk, budget}, lens.options()), lens_out = at::empty({b}, lens.options());
  if (b) {
    a.batch = size32(b, "batch"), a.kv_heads = size32(hk, "key/value heads"), a.head_dim = size32(d, "head size");
    a.capacity = size32(cap, "capacity"), a.out_capacity = size32(rows, "out"), a.budget = budget, a.recent = recent;
    a.k_cache = by_head(k_cache), a.v_cache = by_head(v_cache), a.acc = by_head(acc);
    a.k_out = by_head(k2), a.v_out = by_head(v2), a.acc_out = by_head(a2);
    a.index = index.data_ptr<int32_t>(), a.lens_out = lens_out.data_ptr<int32_t>();
    const Tensor ws = workspace(c, ckks_draft_evict_workspace(c.ctx, &a), a, k_cache);
    c.done(ckks_draft_evict(c.ctx, &a, c.stream()));
  }
  return {k2, v2, a2, index, lens_out};
}

}  // namespace

PYBIND11_MODULE(_draft, m) {
  m.def("attention", &attention);
  m.def("verify", &verify);
  m.def("commit", &commit);
  m.def("accumulate", &accumulate);
  m.def("evict", &evict);
}
