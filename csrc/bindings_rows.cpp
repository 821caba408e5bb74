// Bindings of the launchers that move rows by key and of the distillation kernels, with their gradients.  Outputs are made and graphs
// recorded here: these operators also run on a few rows, where the calls around a kernel take longer than the kernel (measured: a
// forward and backward pass on 24 rows took 86 us with graphs recorded in Python).
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include "api.h"

namespace {
inline cudaStream_t cur_stream() {
  (void)cudaGetLastError();      // (a status that another library left is not this launch's)
  return at::cuda::getCurrentCUDAStream().stream();
}
inline void check(int rc, const char* what) {
  TORCH_CHECK(rc == 0, what, " failed with code ", rc, " (", rc > 0 ? cudaGetErrorString(static_cast<cudaError_t>(rc)) : "argument check", ")");
}
inline int code_of(at::ScalarType t, const char* what) {
  switch (t) {
    case at::kBFloat16: return 0;
    case at::kHalf: return 1;
    case at::kFloat: return 2;
    default: TORCH_CHECK_TYPE(false, what, ": bf16, fp16 or fp32, got ", t);
  }
}
inline int code_of(const torch::Tensor& t, const char* what) { return code_of(t.scalar_type(), what); }
inline void same_device(const torch::Tensor& t, const torch::Tensor& as, const char* what) {
  TORCH_CHECK_VALUE(t.device() == as.device(), what, " is on ", t.device(), ", expected ", as.device());
}
inline int wide_ids(const torch::Tensor& t, const char* what) {
  TORCH_CHECK_TYPE(t.scalar_type() == at::kLong || t.scalar_type() == at::kInt, what, ": int64 or int32 ids, got ", t.scalar_type());
  TORCH_CHECK_VALUE(t.is_contiguous(), what, ": contiguous ids");
  return t.scalar_type() == at::kLong;
}
inline torch::Tensor dense(const torch::Tensor& t, const char* what) {      // a matrix whose rows are dense, at any distance
  TORCH_CHECK_VALUE(t.dim() == 2, what, ": a matrix");
  return t.stride(1) == 1 && t.stride(0) >= 0 ? t : t.contiguous();
}
inline int as_int(int64_t v, const char* what) {
  TORCH_CHECK_VALUE(v >= 0 && v <= (1ll << 30), what, ": ", v, " is out of range");
  return static_cast<int>(v);
}
// Integers (or, for workspaces, whatever lies in them) in one allocation, and tensors on parts of it: an allocation costs as much as a
// launch, and a few rows take six of these.
inline torch::Tensor ints(int64_t n, const torch::Tensor& like) { return at::empty({n > 0 ? n : 1}, like.options().dtype(at::kInt)); }
inline torch::Tensor part_of(const torch::Tensor& all, int64_t offset, at::IntArrayRef shape) {
  auto t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(), all.dtype());
  t.unsafeGetTensorImpl()->set_storage_offset(offset);
  t.unsafeGetTensorImpl()->set_sizes_contiguous(shape);
  return t;
}
// the device's status word, where ids outside a whole table are to be noted
inline int* status(const c10::optional<torch::Tensor>& err, const torch::Tensor& as) {
  if (!err.has_value()) return nullptr;
  same_device(*err, as, "the status word");
  TORCH_CHECK_VALUE(err->scalar_type() == at::kInt && err->numel() >= 1, "the status word is an int32");
  return err->data_ptr<int>();
}
inline bool recorded(const torch::Tensor& t) { return t.requires_grad() && at::GradMode::is_enabled(); }

using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;
using Maybe = c10::optional<torch::Tensor>;

// Gradients are not differentiated again: where a graph of the backward pass is recorded, a second pass through it is refused.
variable_list once(variable_list grads, const variable_list& incoming) {
  if (!at::GradMode::is_enabled()) return grads;
  bool live = false;
  for (const auto& g : incoming) live |= g.defined() && g.requires_grad();
  if (!live) return grads;
  variable_list out = grads;
  auto error = std::make_shared<torch::autograd::DelayedError>("this operator is differentiable once", static_cast<int64_t>(grads.size()));
  for (auto& g : grads)
    if (g.defined()) g = g.detach().set_requires_grad(true);
  auto wrapped = (*error)(std::move(grads));
  for (size_t i = 0; i < out.size(); ++i)
    if (out[i].defined()) out[i] = wrapped[i];
  return out;
}

// ----------------------------------------------------------------------------- experts' rows

// (dest [T, k], source [cap], tile_expert [cap / align] or None, bounds [E + 1])
py::tuple expert_layout(torch::Tensor ids, int64_t experts, int64_t align, const Maybe& err) {
  const c10::cuda::CUDAGuard guard(ids.device());
  ids = ids.contiguous();
  const int wide = wide_ids(ids, "expert_layout");
  TORCH_CHECK_VALUE(experts >= 1 && experts <= 2048, "expert_layout: 1 to 2048 experts, got ", experts);
  TORCH_CHECK_VALUE(align >= 1 && align <= 65536, "expert_layout: align must lie in 1 .. 65536, got ", align);
  const int n = as_int(ids.numel(), "expert_layout: rows");
  const int64_t full = std::min<int64_t>(n, experts), tiles = full + (n - full) / align, cap = align == 1 ? n : tiles * align;
  as_int(cap, "expert_layout: buffer rows");
  const int counters = rb_sort_counters(n, static_cast<int>(experts));
  const auto all = ints(n + cap + (align > 1 ? tiles : 0) + experts + 1 + (counters > 1 ? counters : 0), ids);
  int* p = all.data_ptr<int>();
  const int64_t at_source = n, at_bounds = at_source + cap, at_tiles = at_bounds + experts + 1, at_hist = at_tiles + (align > 1 ? tiles : 0);
  check(rb_expert_layout(ids.data_ptr(), wide, n, static_cast<int>(experts), static_cast<int>(align), static_cast<int>(cap), p, p + at_source,
                         align > 1 ? p + at_tiles : nullptr, p + at_bounds, counters > 1 ? p + at_hist : nullptr, status(err, ids), cur_stream()),
        "rb_expert_layout");
  return py::make_tuple(part_of(all, 0, ids.sizes()), part_of(all, at_source, {cap}), align > 1 ? py::cast(part_of(all, at_tiles, {tiles})) : py::none(),
                        part_of(all, at_bounds, {experts + 1}));
}

torch::Tensor scatter_rows(const torch::Tensor& in, const torch::Tensor& source, const torch::Tensor& dest, const char* what) {
  const c10::cuda::CUDAGuard guard(in.device());
  const auto x = dense(in, what);
  same_device(source, x, "expert_dispatch: the layout");
  auto out = at::empty({source.numel(), x.size(1)}, x.options());
  check(rb_expert_dispatch(x.data_ptr(), x.stride(0), source.data_ptr<int>(), dest.data_ptr<int>(), out.data_ptr(), as_int(source.numel(), what),
                           as_int(dest.size(0), what), as_int(dest.size(1), what), as_int(x.size(1), what), code_of(x, what), cur_stream()),
        "rb_expert_dispatch");
  return out;
}

torch::Tensor gather_rows(const torch::Tensor& in, const torch::Tensor& dest, const Maybe& weight, bool fp32, const char* what) {
  const c10::cuda::CUDAGuard guard(in.device());
  const auto y = dense(in, what);
  same_device(dest, y, "expert_combine: the layout");
  if (weight.has_value()) same_device(*weight, y, "expert_combine: weights");
  auto out = at::empty({dest.size(0), y.size(1)}, fp32 ? y.options().dtype(at::kFloat) : y.options());
  check(rb_expert_combine(y.data_ptr(), y.stride(0), dest.data_ptr<int>(), weight.has_value() ? weight->data_ptr<float>() : nullptr, out.data_ptr(),
                          as_int(dest.size(0), what), as_int(dest.size(1), what), as_int(y.size(1), what), code_of(y, what), fp32, cur_stream()),
        "rb_expert_combine");
  return out;
}

struct Dispatch : Function<Dispatch> {
  static torch::Tensor forward(AutogradContext* ctx, const torch::Tensor& x, const torch::Tensor& dest, const torch::Tensor& source) {
    ctx->save_for_backward({dest});
    return scatter_rows(x, source, dest, "expert_dispatch");
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto saved = ctx->get_saved_variables();
    return once({gather_rows(g[0], saved[0], c10::nullopt, false, "expert_dispatch"), torch::Tensor(), torch::Tensor()}, g);
  }
};
torch::Tensor expert_dispatch(const torch::Tensor& x, const torch::Tensor& dest, const torch::Tensor& source) {
  return recorded(x) ? Dispatch::apply(x, dest, source) : scatter_rows(x, source, dest, "expert_dispatch");
}

struct Combine : Function<Combine> {
  static torch::Tensor forward(AutogradContext* ctx, const torch::Tensor& y, const Maybe& weight, const torch::Tensor& dest, const torch::Tensor& source,
                               bool fp32) {
    Maybe w;
    if (weight.has_value()) w = weight->to(at::kFloat).contiguous();
    // (fixed weights learn nothing from the rows: these are not kept)
    ctx->save_for_backward({w.has_value() && weight->requires_grad() ? y : torch::Tensor(), w.has_value() ? *w : torch::Tensor(), dest, source});
    ctx->saved_data["columns"] = y.size(1);
    ctx->saved_data["type"] = static_cast<int64_t>(y.scalar_type());
    ctx->saved_data["weight_type"] = static_cast<int64_t>(weight.has_value() ? weight->scalar_type() : at::kFloat);
    return gather_rows(y, dest, w, fp32, "expert_combine");
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto saved = ctx->get_saved_variables();
    const auto &w = saved[1], &dest = saved[2], &source = saved[3];
    const c10::cuda::CUDAGuard guard(g[0].device());
    if (!w.defined()) {      // (copies: one rounding)
      const auto d = g[0].to(static_cast<at::ScalarType>(ctx->saved_data["type"].toInt()));
      return once({scatter_rows(d, source, dest, "expert_combine"), torch::Tensor(), torch::Tensor(), torch::Tensor(), torch::Tensor()}, g);
    }
    const auto type = static_cast<at::ScalarType>(ctx->saved_data["type"].toInt());
    const auto d = dense(g[0], "expert_combine");
    const bool fp32 = d.scalar_type() == at::kFloat;
    TORCH_CHECK_VALUE(fp32 || d.scalar_type() == type, "expert_combine: a gradient in ", type, " or float32, got ", d.scalar_type());
    const int64_t cols = ctx->saved_data["columns"].toInt();
    torch::Tensor y, d_y, d_w;      // what is asked for
    if (ctx->needs_input_grad(0)) d_y = at::empty({source.numel(), cols}, d.options().dtype(type));
    if (saved[0].defined() && ctx->needs_input_grad(1)) y = dense(saved[0], "expert_combine"), d_w = at::empty_like(w);
    check(rb_expert_combine_bwd(d.data_ptr(), d.stride(0), y.defined() ? y.data_ptr() : nullptr, y.defined() ? y.stride(0) : 0, source.data_ptr<int>(),
                                dest.data_ptr<int>(), w.data_ptr<float>(), d_y.defined() ? d_y.data_ptr() : nullptr,
                                d_w.defined() ? d_w.data_ptr<float>() : nullptr, as_int(source.numel(), "expert_combine"),
                                as_int(dest.size(0), "expert_combine"), as_int(dest.size(1), "expert_combine"), as_int(cols, "expert_combine"),
                                code_of(type, "expert_combine"), fp32, cur_stream()),
          "rb_expert_combine_bwd");
    if (d_w.defined()) d_w = d_w.to(static_cast<at::ScalarType>(ctx->saved_data["weight_type"].toInt()));
    return once({d_y, d_w, torch::Tensor(), torch::Tensor(), torch::Tensor()}, g);
  }
};
torch::Tensor expert_combine(const torch::Tensor& y, const Maybe& weight, const torch::Tensor& dest, const torch::Tensor& source, bool fp32) {
  if (recorded(y) || (weight.has_value() && recorded(*weight))) return Combine::apply(y, weight, dest, source, fp32);
  if (!weight.has_value()) return gather_rows(y, dest, weight, fp32, "expert_combine");
  return gather_rows(y, dest, weight->to(at::kFloat).contiguous(), fp32, "expert_combine");
}

// ----------------------------------------------------------------------------- embedding

torch::Tensor look_up(const torch::Tensor& weight, const torch::Tensor& ids, double scale, int64_t start, const Maybe& err) {
  const c10::cuda::CUDAGuard guard(weight.device());
  const auto table = dense(weight, "embedding");
  const int wide = wide_ids(ids, "embedding");
  same_device(ids, table, "embedding: tokens");
  auto shape = ids.sizes().vec();
  shape.push_back(table.size(1));
  auto out = at::empty(shape, table.options());
  check(rb_embedding(ids.data_ptr(), wide, start, table.data_ptr(), table.stride(0), as_int(table.size(0), "embedding: table rows"), out.data_ptr(),
                     as_int(ids.numel(), "embedding: tokens"), as_int(table.size(1), "embedding: columns"), static_cast<float>(scale),
                     code_of(table, "embedding"), status(err, table), cur_stream()),
        "rb_embedding");
  return out;
}

// The gradient is a new matrix in the rows' type, or is added to `main_grad` (fp32), which then stands for it.
struct Embedding : Function<Embedding> {
  static torch::Tensor forward(AutogradContext* ctx, const torch::Tensor& weight, const torch::Tensor& ids, double scale, int64_t start,
                               const Maybe& main_grad, const Maybe& err) {
    ctx->save_for_backward({ids});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["start"] = start;
    ctx->saved_data["rows"] = weight.size(0);
    ctx->saved_data["main_grad"] = main_grad;
    return look_up(weight, ids, scale, start, err);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto saved = ctx->get_saved_variables();
    const auto& ids = saved[0];
    const auto into = ctx->saved_data["main_grad"].toOptional<torch::Tensor>();
    const int64_t rows = ctx->saved_data["rows"].toInt();
    const c10::cuda::CUDAGuard guard(g[0].device());
    const auto dy = dense(g[0].reshape({ids.numel(), g[0].size(-1)}), "embedding");
    const int n = as_int(ids.numel(), "embedding: tokens"), V = as_int(rows, "embedding: table rows"), cols = as_int(dy.size(1), "embedding: columns");
    auto out = into.has_value() ? *into : at::empty({rows, cols}, dy.options());
    // two buffers of (key, row), partial sums of runs (32-byte vectors), the runs over several chunks, counters
    const int64_t chunks = (n + 31) / 32, at_part = (4ll * n + 7) / 8 * 8, at_open = at_part + (chunks > 1 ? chunks * 2 * cols : 0);
    const int64_t at_hist = at_open + 2 + chunks;
    const auto work = ints(at_hist + rb_sort_counters(n, rb_embedding_bwd_bins(V)), dy);
    int* p = work.data_ptr<int>();
    check(rb_embedding_bwd(ids.data_ptr(), ids.scalar_type() == at::kLong, ctx->saved_data["start"].toInt(), dy.data_ptr(), dy.stride(0), out.data_ptr(),
                           into.has_value(), reinterpret_cast<int2*>(p), p + at_hist, reinterpret_cast<float*>(p + at_part), p + at_open, n, V, cols,
                           static_cast<float>(ctx->saved_data["scale"].toDouble()), code_of(dy, "embedding"), cur_stream()),
          "rb_embedding_bwd");
    variable_list d(6);
    if (!into.has_value()) d[0] = out;
    return once(d, g);
  }
};
torch::Tensor embedding(const torch::Tensor& weight, const torch::Tensor& tokens, double scale, int64_t start, const Maybe& main_grad, const Maybe& err) {
  if (main_grad.has_value()) {
    same_device(*main_grad, weight, "embedding: main_grad");
    TORCH_CHECK_VALUE(main_grad->scalar_type() == at::kFloat && main_grad->is_contiguous() && main_grad->sizes() == weight.sizes(),
                      "embedding: main_grad is a dense fp32 matrix of the table's shape");
  }
  const auto ids = tokens.contiguous();
  return recorded(weight) ? Embedding::apply(weight, ids, scale, start, main_grad, err) : look_up(weight, ids, scale, start, err);
}

// ----------------------------------------------------------------------------- distillation from top ids

struct Distilled {
  torch::Tensor loss, kept, log_probs;      // kept: statistics [R, 4], sums of parts (a workspace), slopes of the ids [R, K]
};
inline int64_t slopes_at(const torch::Tensor& z, const torch::Tensor& ids) {
  return z.size(0) * (4 + 4 * rb_topk_distill_parts(z.size(0), static_cast<int>(z.size(1)), static_cast<int>(ids.size(1)), static_cast<int>(z.element_size())));
}

Distilled distill_rows(const torch::Tensor& z, const torch::Tensor& ids, const torch::Tensor& teacher, int64_t kl, int64_t norm, double alpha, double clamp,
                       double inv_temp, bool log_probs) {
  const c10::cuda::CUDAGuard guard(z.device());
  same_device(ids, z, "topk_distill: ids");
  same_device(teacher, z, "topk_distill: teacher");
  TORCH_CHECK_TYPE(ids.scalar_type() == at::kLong && teacher.scalar_type() == at::kFloat, "topk_distill: int64 ids, fp32 teacher log-probs");
  TORCH_CHECK_VALUE(ids.dim() == 2 && ids.is_contiguous() && teacher.is_contiguous() && teacher.sizes() == ids.sizes() && ids.size(0) == z.size(0),
                    "topk_distill: ids and teacher log-probs are dense [rows, K]");
  TORCH_CHECK_VALUE(ids.size(1) <= 1024, "topk_distill: up to 1024 ids per row, got ", ids.size(1));
  TORCH_CHECK_VALUE(z.size(1) >= 1 && z.size(1) <= (1 << 24), "topk_distill: 1 to 2^24 tokens in the vocabulary, got ", z.size(1));
  const auto f32 = z.options().dtype(at::kFloat);
  const int64_t R = z.size(0), K = ids.size(1), slopes = slopes_at(z, ids);
  const int code = code_of(z, "topk_distill");
  Distilled d{at::empty({R}, f32), at::empty({slopes + R * K}, f32), torch::Tensor()};
  float* kept = d.kept.data_ptr<float>();
  if (log_probs) d.log_probs = at::empty({R, K}, f32);
  check(rb_topk_distill(z.data_ptr(), z.stride(0), reinterpret_cast<const long long*>(ids.data_ptr<int64_t>()), teacher.data_ptr<float>(),
                        d.loss.data_ptr<float>(), kept + slopes, kept, log_probs ? d.log_probs.data_ptr<float>() : nullptr,
                        reinterpret_cast<double2*>(kept + 4 * R), R, static_cast<int>(z.size(1)), static_cast<int>(K), static_cast<int>(kl),
                        static_cast<int>(norm), alpha, clamp, inv_temp, code, cur_stream()),
        "rb_topk_distill");
  return d;
}

// d logits, into `out` (a dense matrix of the logits' type, or of bf16 for fp32 logits)
void distill_rows_bwd(const torch::Tensor& z, const torch::Tensor& ids, const torch::Tensor& kept, const torch::Tensor& g, double inv_temp,
                      const torch::Tensor& out) {
  const c10::cuda::CUDAGuard guard(z.device());
  TORCH_CHECK_VALUE(out.is_contiguous() && out.sizes() == z.sizes(), "topk_distill: a dense gradient of the logits' shape");
  const int64_t slopes = slopes_at(z, ids);
  TORCH_CHECK_VALUE(g.scalar_type() == at::kFloat && g.is_contiguous() && g.numel() == z.size(0) && ids.is_contiguous() && ids.size(0) == z.size(0) &&
                        kept.scalar_type() == at::kFloat && kept.is_contiguous() && kept.numel() == slopes + ids.numel(),
                    "topk_distill: gradient or kept values of another shape");
  check(rb_topk_distill_bwd(z.data_ptr(), z.stride(0), reinterpret_cast<const long long*>(ids.data_ptr<int64_t>()), kept.data_ptr<float>() + slopes,
                            kept.data_ptr<float>(), g.data_ptr<float>(), out.data_ptr(), z.size(0), as_int(z.size(1), "topk_distill: vocabulary"),
                            static_cast<int>(ids.size(1)), inv_temp, code_of(z, "topk_distill"), code_of(out, "topk_distill"),
                            cur_stream()),
        "rb_topk_distill_bwd");
}

struct TopkDistill : Function<TopkDistill> {
  static variable_list forward(AutogradContext* ctx, const torch::Tensor& z, const torch::Tensor& ids, const torch::Tensor& teacher, int64_t kl, int64_t norm,
                               double alpha, double clamp, double inv_temp, bool log_probs) {
    const auto d = distill_rows(z, ids, teacher, kl, norm, alpha, clamp, inv_temp, log_probs);
    ctx->save_for_backward({z, ids, d.kept});
    ctx->saved_data["inv_temp"] = inv_temp;
    if (!log_probs) return {d.loss};
    ctx->mark_non_differentiable({d.log_probs});
    return {d.loss, d.log_probs};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto saved = ctx->get_saved_variables();
    const c10::cuda::CUDAGuard guard(saved[0].device());
    auto out = at::empty({saved[0].size(0), saved[0].size(1)}, saved[0].options());
    distill_rows_bwd(saved[0], saved[1], saved[2], g[0].to(at::kFloat).contiguous(), ctx->saved_data["inv_temp"].toDouble(), out);
    variable_list d(9);
    d[0] = out;
    return once(d, g);
  }
};
py::object topk_distill(const torch::Tensor& logits, const torch::Tensor& ids, const torch::Tensor& teacher, int64_t kl, int64_t norm, double alpha,
                        double clamp, double inv_temp, bool log_probs) {
  const auto z = dense(logits, "topk_distill"), i = ids.contiguous(), t = teacher.detach().to(at::kFloat).contiguous();
  if (recorded(z)) {
    const auto out = TopkDistill::apply(z, i, t, kl, norm, alpha, clamp, inv_temp, log_probs);
    return log_probs ? py::object(py::make_tuple(out[0], out[1])) : py::cast(out[0]);
  }
  const auto d = distill_rows(z, i, t, kl, norm, alpha, clamp, inv_temp, log_probs);
  return log_probs ? py::object(py::make_tuple(d.loss, d.log_probs)) : py::cast(d.loss);
}
py::tuple topk_distill_rows(const torch::Tensor& z, const torch::Tensor& ids, const torch::Tensor& teacher, int64_t kl, int64_t norm, double alpha,
                            double clamp, double inv_temp) {
  const auto d = distill_rows(z, ids, teacher, kl, norm, alpha, clamp, inv_temp, false);
  return py::make_tuple(d.loss, d.kept);
}
}  // namespace

void register_rows(pybind11::module_& m) {
  m.def("expert_layout", &expert_layout, py::arg("ids"), py::arg("experts"), py::arg("align"), py::arg("err") = py::none());
  m.def("expert_dispatch", &expert_dispatch);
  m.def("expert_combine", &expert_combine);
  m.def("embedding", &embedding, py::arg("weight"), py::arg("tokens"), py::arg("scale"), py::arg("start"), py::arg("main_grad"),
        py::arg("err") = py::none());
  m.def("topk_distill", &topk_distill);
  m.def("topk_distill_rows", &topk_distill_rows);
  m.def("topk_distill_rows_bwd", &distill_rows_bwd);
}
