// The functions of the extension module for rows that are learned: embedding lookup and gradient, rows by expert, their products, dropout, plain
// (graph_sampling_b200.ops) and as autograd functions (graph_sampling_b200.gs.nn).
//
// A backward pass runs on a thread of the autograd engine that does not hold the GIL, so everything below the Python functions
// throws C++ exceptions, and the Python functions translate.  Scratch comes from torch's allocator on the current stream, call
// by call: calls on several streams, and captured ones, share nothing but the context's error counters.
#include <ATen/Functions.h>
#include <ATen/core/CachingHostAllocator.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/grad_mode.h>
#include <torch/csrc/autograd/variable.h>

#include <initializer_list>
#include <limits>
#include <optional>
#include <unordered_set>
#include <utility>

#include "native.h"

namespace {

using namespace native;
using torch::autograd::AutogradContext;
using torch::autograd::tensor_list;
using torch::autograd::variable_list;

struct BadArgument : std::runtime_error {
  using std::runtime_error::runtime_error;
};
struct Failed : std::runtime_error {  // a call of the C ABI
  int status;
  std::string where, detail;
  Failed(int st, const char* w, const char* d)
      : std::runtime_error(std::string(w) + ": " + gsb_status_string(st) + " " + d), status(st), where(w), detail(d) {}
};
void refuse_unless(bool ok, const char* what) {
  if (!ok) throw BadArgument(what);
}
void refuse_unless(bool ok, const char* name, const char* what) {
  if (!ok) throw BadArgument(std::string(name) + what);
}
void done(gsb_ctx* ctx, int st, const char* where) {
  if (st != GSB_OK) throw Failed(st, where, gsb_last_error_message(ctx));
}

int dtype_of(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return GSB_F32;
    case at::kHalf: return GSB_F16;
    case at::kBFloat16: return GSB_BF16;
    default: throw BadArgument(std::string(name) + " must be float32, float16 or bfloat16");
  }
}

// The tensor itself, or a copy where its memory holds the negative of its values (the imaginary part of a conjugate).
Tensor as_stored(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }

// A matrix whose rows are runs of memory, at any distance from each other; a copy where they are not.
struct Rows {
  Tensor t;
  int dtype;
  int64_t n, width, stride;
  const void* data() const { return t.const_data_ptr(); }
};
Rows rows_of(const Tensor& t, const char* name, bool pinned_too = false) {
  Rows r;
  r.dtype = dtype_of(t, name);
  refuse_unless(t.dim() == 2, name, " must have two dimensions");
  r.t = as_stored(t);
  refuse_unless(r.t.is_cuda() || (pinned_too && r.t.is_pinned()), name,
                pinned_too ? " must live on the GPU or in pinned host memory" : " must be a CUDA tensor");
  r.n = t.size(0);
  r.width = t.size(1);
  if (r.width > 1 && r.t.stride(1) != 1) {
    refuse_unless(t.is_cuda(), name, ": rows of a pinned host tensor must be contiguous");
    r.t = r.t.contiguous();
  }
  r.stride = r.n > 1 ? r.t.stride(0) : r.width;
  return r;
}
Tensor ids_of(const Tensor& t, const char* name) {
  refuse_unless(t.scalar_type() == at::kLong, name, " must be int64");
  refuse_unless(t.is_cuda(), name, " must be a CUDA tensor");
  return as_stored(t).contiguous();
}
void same_device(const Tensor& a, const Tensor& b) {
  refuse_unless(a.device() == b.device(), "tensors of one call must live on the same device");
}
const int64_t* ids_ptr(const Tensor& t) { return static_cast<const int64_t*>(t.const_data_ptr()); }
void* data(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
Tensor fresh(at::IntArrayRef shape, at::ScalarType dtype, c10::Device dev) {
  return at::detail::empty_cuda(shape, dtype, dev, c10::nullopt);
}
Tensor scratch(int64_t bytes, const char* where, c10::Device dev) {
  if (bytes < 0) throw Failed((int)bytes, where, "");
  return fresh({bytes}, at::kByte, dev);
}
std::vector<int64_t> with_width(at::IntArrayRef shape, int64_t width) {
  std::vector<int64_t> s(shape.begin(), shape.end());
  s.push_back(width);
  return s;
}

struct Padding {
  bool given = false;
  int64_t id = 0;
};

// ---- the operators ---------------------------------------------------------------------------------------------------------
Tensor lookup(gsb_ctx* ctx, const Tensor& table_, const Tensor& ids_, double scale, Padding pad) {
  const Rows table = rows_of(table_, "table", true);
  const Tensor ids = ids_of(ids_, "ids");
  if (table.t.is_cuda()) same_device(table.t, ids);
  const c10::cuda::CUDAGuard guard(ids.device());
  Tensor out = fresh(with_width(ids.sizes(), table.width), table.t.scalar_type(), ids.device());
  if (out.numel() == 0) return out;
  done(ctx, gsb_embedding_lookup(ctx, stream(), table.data(), table.dtype, table.n, table.width, table.stride, ids_ptr(ids),
                                 ids.numel(), (float)scale, pad.given, pad.id, data(out)),
       "gsb_embedding_lookup");
  // memory of the host allocator is not given to another tensor before the kernel has read it (a captured one's has to outlive the graph)
  if (!table.t.is_cuda() && c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None)
    at::getHostAllocator(at::kCUDA)->record_event(const_cast<void*>(table.data()), table.t.storage().data_ptr().get_context(),
                                                  c10::cuda::getCurrentCUDAStream().unwrap());
  return out;
}

// The operands of a gradient: one row of `grad` per id.
struct GradOperands {
  Rows grad;
  Tensor ids;
  int out_dtype;
  at::ScalarType out_type;
};
GradOperands grad_operands(const Tensor& grad_, const Tensor& ids_, std::optional<at::ScalarType> dtype) {
  GradOperands g;
  const int given = dtype_of(grad_, "grad");
  refuse_unless(grad_.dim() == ids_.dim() + 1 && grad_.sizes().slice(0, ids_.dim()) == ids_.sizes(),
                "grad must have the shape of ids and one more dimension");
  g.out_type = dtype.value_or(grad_.scalar_type());
  refuse_unless(g.out_type == grad_.scalar_type() || g.out_type == at::kFloat, "the result's dtype is that of grad, or float32");
  g.out_dtype = g.out_type == at::kFloat ? GSB_F32 : given;
  g.ids = ids_of(ids_, "ids");
  refuse_unless(grad_.is_cuda(), "grad must be a CUDA tensor");
  same_device(grad_, g.ids);
  g.grad = rows_of(grad_.reshape({g.ids.numel(), grad_.size(-1)}), "grad");
  return g;
}

Tensor dense_grad(gsb_ctx* ctx, const Tensor& grad_, const Tensor& ids_, int64_t num_rows, double scale, Padding pad,
                  std::optional<at::ScalarType> dtype) {
  refuse_unless(num_rows >= 0, "num_rows must not be negative");
  const GradOperands g = grad_operands(grad_, ids_, dtype);
  const c10::Device dev = g.ids.device();
  const c10::cuda::CUDAGuard guard(dev);
  Tensor out = fresh({num_rows, g.grad.width}, g.out_type, dev);
  const int64_t n = g.ids.numel();
  if (g.grad.width == 0) return out;
  Tensor work = scratch(gsb_embedding_grad_workspace(n, num_rows, g.grad.width), "gsb_embedding_grad", dev);
  done(ctx, gsb_embedding_grad(ctx, stream(), g.grad.data(), g.grad.dtype, g.grad.width, g.grad.stride, ids_ptr(g.ids), n, num_rows,
                               (float)scale, pad.given, pad.id, data(out), g.out_dtype, data(work), work.numel()),
       "gsb_embedding_grad");
  return out;
}

// (row ids, rows), trimmed to their number; or, without waiting for that, (row ids, rows, number).
std::vector<Tensor> grad_rows(gsb_ctx* ctx, const Tensor& grad_, const Tensor& ids_, int64_t num_rows, double scale, Padding pad,
                              std::optional<at::ScalarType> dtype, bool sync) {
  refuse_unless(num_rows >= 0, "num_rows must not be negative");
  const GradOperands g = grad_operands(grad_, ids_, dtype);
  refuse_unless(g.grad.width > 0, "rows must hold at least one value");
  const c10::Device dev = g.ids.device();
  const c10::cuda::CUDAGuard guard(dev);
  const int64_t n = g.ids.numel(), width = g.grad.width;
  Tensor row_ids = empty(n, dev), rows = fresh({n, width}, g.out_type, dev), count = empty(1, dev);
  Tensor work = scratch(gsb_embedding_grad_workspace(n, num_rows, width), "gsb_embedding_grad_rows", dev);
  int64_t found = 0;
  done(ctx, gsb_embedding_grad_rows(ctx, stream(), g.grad.data(), g.grad.dtype, width, g.grad.stride, ids_ptr(g.ids), n, num_rows,
                                    (float)scale, pad.given, pad.id, static_cast<int64_t*>(data(row_ids)), data(rows), g.out_dtype,
                                    static_cast<int64_t*>(data(count)), data(work), work.numel(), sync ? &found : nullptr),
       "gsb_embedding_grad_rows");
  if (!sync) return {row_ids, rows, count};
  if (found < 0 || found > n) throw Failed(GSB_ERR_CUDA, "gsb_embedding_grad_rows", "a number of rows that cannot be");
  trim(row_ids, found);
  rows.unsafeGetTensorImpl()->set_sizes_contiguous({found, width});
  return {row_ids, rows};
}

std::vector<Tensor> order(gsb_ctx* ctx, const Tensor& experts_, int64_t num_experts) {
  refuse_unless(num_experts >= 1 && num_experts <= GSB_MAX_EXPERTS, "num_experts must be between 1 and 65536");
  const Tensor experts = ids_of(experts_, "expert_ids");
  const c10::Device dev = experts.device();
  const c10::cuda::CUDAGuard guard(dev);
  const int64_t n = experts.numel();
  Tensor offsets = empty(num_experts + 1, dev), source = empty(n, dev), place = fresh(experts.sizes(), at::kLong, dev);
  Tensor work = scratch(gsb_expert_order_workspace(n, num_experts), "gsb_expert_order", dev);
  done(ctx, gsb_expert_order(ctx, stream(), ids_ptr(experts), n, num_experts, static_cast<int64_t*>(data(offsets)),
                             static_cast<int64_t*>(data(source)), static_cast<int64_t*>(data(place)), data(work), work.numel()),
       "gsb_expert_order");
  return {offsets, source, place};
}

struct Places {
  Tensor t;
  int64_t tokens, per_token;
};
Places places_of(const Tensor& t) {
  refuse_unless(t.dim() == 1 || t.dim() == 2, "place must have the shape [tokens] or [tokens, per token]");
  const int64_t per_token = t.dim() == 2 ? t.size(1) : 1;
  refuse_unless(per_token >= 1, "place must hold at least one slot per token");
  return {ids_of(t, "place"), t.size(0), per_token};
}
struct WeightsOf {
  Tensor t;
  int dtype = GSB_F32;
  const void* data() const { return t.defined() ? t.const_data_ptr() : nullptr; }
};
WeightsOf weights_of(const Tensor& w, const Tensor& place, const Rows& rows) {
  WeightsOf r;
  if (!w.defined()) return r;
  r.dtype = dtype_of(w, "weights");
  refuse_unless(r.dtype == rows.dtype || r.dtype == GSB_F32, "weights must be float32 or of the rows' dtype");
  refuse_unless(w.sizes() == place.sizes(), "weights must have the shape of place");
  refuse_unless(w.is_cuda(), "weights must be a CUDA tensor");
  same_device(w, rows.t);
  r.t = as_stored(w).contiguous();
  return r;
}

Tensor spread(gsb_ctx* ctx, const Tensor& x_, const Tensor& place_, const Tensor& weights_) {
  const Rows x = rows_of(x_, "x");
  const Places place = places_of(place_);
  refuse_unless(x.n == place.tokens, "x must have one row per token of place");
  same_device(x.t, place.t);
  const WeightsOf w = weights_of(weights_, place_, x);
  const c10::cuda::CUDAGuard guard(x.t.device());
  Tensor rows = fresh({place.t.numel(), x.width}, x.t.scalar_type(), x.t.device());
  if (rows.numel() == 0) return rows;
  done(ctx, gsb_expert_spread(ctx, stream(), x.data(), x.dtype, place.tokens, place.per_token, x.width, x.stride, ids_ptr(place.t),
                              w.data(), w.dtype, data(rows)),
       "gsb_expert_spread");
  return rows;
}

Tensor combine(gsb_ctx* ctx, const Tensor& rows_, const Tensor& place_, const Tensor& weights_) {
  const Rows rows = rows_of(rows_, "rows");
  const Places place = places_of(place_);
  refuse_unless(rows.n <= place.t.numel(), "there are more rows than slots in place");
  same_device(rows.t, place.t);
  const WeightsOf w = weights_of(weights_, place_, rows);
  const c10::cuda::CUDAGuard guard(rows.t.device());
  Tensor out = fresh({place.tokens, rows.width}, rows.t.scalar_type(), rows.t.device());
  if (out.numel() == 0) return out;
  done(ctx, gsb_expert_combine(ctx, stream(), rows.data(), rows.dtype, rows.n, place.tokens, place.per_token, rows.width,
                               rows.stride, ids_ptr(place.t), w.data(), w.dtype, data(out)),
       "gsb_expert_combine");
  return out;
}

// Gradients of combine for the rows and for the weights (undefined where there are none, or not wanted).
std::pair<Tensor, Tensor> combine_grad(gsb_ctx* ctx, const Tensor& grad_, const Tensor& rows_, const Tensor& place_,
                                       const Tensor& weights_, bool for_rows, bool for_weights) {
  const Rows grad = rows_of(grad_, "grad"), rows = rows_of(rows_, "rows");
  const Places place = places_of(place_);
  refuse_unless(grad.dtype == rows.dtype && grad.width == rows.width && grad.n == place.tokens,
                "grad must have one row per token of place, of the rows' width and dtype");
  refuse_unless(rows.n <= place.t.numel(), "there are more rows than slots in place");
  same_device(grad.t, place.t);
  same_device(rows.t, place.t);
  const WeightsOf w = weights_of(weights_, place_, rows);
  const c10::Device dev = rows.t.device();
  const c10::cuda::CUDAGuard guard(dev);
  Tensor grad_rows, grad_weights;
  if (for_rows) grad_rows = fresh({rows.n, rows.width}, rows.t.scalar_type(), dev);
  if (for_weights && w.t.defined()) grad_weights = fresh(place_.sizes(), w.t.scalar_type(), dev);
  if (rows.width == 0) {
    if (grad_weights.defined()) grad_weights.zero_();
    return {grad_rows, grad_weights};
  }
  if (grad_rows.defined() || grad_weights.defined())
    done(ctx, gsb_expert_combine_grad(ctx, stream(), grad.data(), grad.dtype, place.tokens, place.per_token, grad.width,
                                      grad.stride, rows.data(), rows.n, rows.stride, ids_ptr(place.t), w.data(), w.dtype,
                                      data(grad_rows), data(grad_weights)),
         "gsb_expert_combine_grad");
  return {grad_rows, grad_weights};
}

// One matrix per expert, its rows or its columns runs of memory; a copy where neither are.
struct Matrices {
  Tensor t;
  int64_t experts, k, n;
};
Matrices matrices_of(const Tensor& w, const Rows& rows) {
  refuse_unless(dtype_of(w, "weights") == rows.dtype, "weights must have the rows' dtype");
  refuse_unless(w.dim() == 3, "weights must have the shape [experts, k, n]");
  refuse_unless(w.size(0) >= 1 && w.size(0) <= GSB_MAX_EXPERTS, "weights must hold between 1 and 65536 experts");
  refuse_unless(w.size(1) == rows.width, "weights must have as many rows each as the rows have values");
  refuse_unless(w.is_cuda(), "weights must be a CUDA tensor");
  same_device(w, rows.t);
  Tensor t = as_stored(w);
  if (!(t.size(1) <= 1 || t.stride(1) == 1) && !(t.size(2) <= 1 || t.stride(2) == 1)) t = t.contiguous();
  return {t, w.size(0), w.size(1), w.size(2)};
}
Tensor offsets_of(const Tensor& t, int64_t experts, const Tensor& beside) {
  const Tensor offsets = ids_of(t, "offsets");
  refuse_unless(t.dim() == 1 && t.numel() >= 2, "offsets must hold one entry per expert and one more");
  refuse_unless(experts < 0 || t.numel() == experts + 1, "offsets must hold one entry per expert and one more");
  refuse_unless(t.numel() - 1 <= GSB_MAX_EXPERTS, "offsets must be of at most 65536 experts");
  same_device(offsets, beside);
  return offsets;
}

Tensor product(gsb_ctx* ctx, const Tensor& rows_, const Tensor& weights_, const Tensor& offsets_) {
  const Rows rows = rows_of(rows_, "rows");
  const Matrices w = matrices_of(weights_, rows);
  const Tensor offsets = offsets_of(offsets_, w.experts, rows.t);
  const c10::Device dev = rows.t.device();
  const c10::cuda::CUDAGuard guard(dev);
  Tensor out = fresh({rows.n, w.n}, rows.t.scalar_type(), dev);
  if (out.numel() == 0) return out;
  if (w.k == 0) return out.zero_();
  const void* matrices = w.t.const_data_ptr();
  const int64_t of_expert = w.t.stride(0), of_k = w.t.stride(1), of_n = w.t.stride(2);
  Tensor work = scratch(gsb_expert_product_workspace(rows.data(), rows.dtype, rows.n, w.k, rows.stride, matrices, of_expert, of_k, of_n, w.n, w.experts),
                        "gsb_expert_product", dev);
  done(ctx, gsb_expert_product(ctx, stream(), rows.data(), rows.dtype, rows.n, w.k, rows.stride, matrices, of_expert, of_k, of_n, w.n, ids_ptr(offsets),
                               w.experts, data(out), data(work), work.numel()),
       "gsb_expert_product");
  return out;
}

Tensor product_grad(gsb_ctx* ctx, const Tensor& rows_, const Tensor& grad_, const Tensor& offsets_) {
  const Rows rows = rows_of(rows_, "rows"), grad = rows_of(grad_, "grad");
  refuse_unless(grad.dtype == rows.dtype && grad.n == rows.n, "grad must have as many rows as rows, of the same dtype");
  same_device(grad.t, rows.t);
  const Tensor offsets = offsets_of(offsets_, -1, rows.t);
  const int64_t experts = offsets.numel() - 1;
  const c10::Device dev = rows.t.device();
  const c10::cuda::CUDAGuard guard(dev);
  Tensor out = fresh({experts, rows.width, grad.width}, rows.t.scalar_type(), dev);
  if (out.numel() == 0) return out;
  Tensor work = scratch(gsb_expert_product_grad_workspace(rows.data(), rows.dtype, rows.n, rows.width, rows.stride, grad.data(), grad.width,
                                                          grad.stride, experts),
                        "gsb_expert_product_grad", dev);
  done(ctx, gsb_expert_product_grad(ctx, stream(), rows.data(), rows.dtype, rows.n, rows.width, rows.stride, grad.data(), grad.width, grad.stride,
                                    ids_ptr(offsets), experts, data(out), data(work), work.numel()),
       "gsb_expert_product_grad");
  return out;
}

// ---- 8 bits
constexpr int64_t kLine = 16;  // bytes that a row in 8 bits begins on
int64_t in_lines(int64_t width) { return (width + kLine - 1) / kLine * kLine; }
std::pair<Tensor, Tensor> quantize(gsb_ctx* ctx, const Tensor& x_) {
  dtype_of(x_, "x");
  refuse_unless(x_.dim() >= 1, "x must have at least one dimension");
  refuse_unless(x_.is_cuda(), "x must be a CUDA tensor");
  const auto shape = x_.sizes().slice(0, x_.dim() - 1);
  const int64_t width = x_.size(-1);
  const c10::cuda::CUDAGuard guard(x_.device());
  const Rows x = rows_of(x_.reshape({c10::multiply_integers(shape), width}), "x");
  Tensor values = fresh(with_width(shape, in_lines(width)), at::kChar, x.t.device()).narrow(-1, 0, width);
  Tensor scales = fresh(shape, at::kFloat, x.t.device());
  if (x.n == 0) return {values, scales};
  if (width == 0) return {values, scales.zero_()};
  done(ctx, gsb_quantize_rows(ctx, stream(), x.data(), x.dtype, x.n, width, x.stride, static_cast<int8_t*>(data(values)), in_lines(width),
                              static_cast<float*>(data(scales))),
       "gsb_quantize_rows");
  return {values, scales};
}

// Rows in 8 bits that begin on 16-byte boundaries; a copy where they do not.
Tensor bytes_of(const Tensor& t_, const char* name, int64_t dim) {
  refuse_unless(t_.scalar_type() == at::kChar, name, " must be int8");
  refuse_unless(t_.dim() == dim, name, dim == 2 ? " must have two dimensions" : " must have the shape [experts, n, k]");
  refuse_unless(t_.is_cuda(), name, " must be a CUDA tensor");
  const Tensor t = as_stored(t_);
  bool good = (t.size(-1) <= 1 || t.stride(-1) == 1) && reinterpret_cast<uintptr_t>(t.const_data_ptr()) % kLine == 0;
  for (int64_t d = 0; d + 1 < dim; ++d) good = good && (t.size(d) <= 1 || (t.stride(d) % kLine == 0 && t.stride(d) >= t.size(-1)));
  if (good || t.numel() == 0) return t;
  Tensor copy = fresh(with_width(t.sizes().slice(0, dim - 1), in_lines(t.size(-1))), at::kChar, t.device()).narrow(-1, 0, t.size(-1));
  copy.copy_(t);
  return copy;
}
// Distance between neighbours of a dimension; where there is one alone, what it would be.
int64_t step_of(const Tensor& t, int64_t d, int64_t alone) { return t.size(d) > 1 ? t.stride(d) : alone; }
Tensor scales_of(const Tensor& t, const char* name, const Tensor& of) {
  refuse_unless(t.scalar_type() == at::kFloat, name, " must be float32");
  refuse_unless(t.sizes() == of.sizes().slice(0, of.dim() - 1), name, " must hold one value per row");
  refuse_unless(t.is_cuda(), name, " must be a CUDA tensor");
  same_device(t, of);
  return as_stored(t).contiguous();
}

Tensor product_int8(gsb_ctx* ctx, const Tensor& values_, const Tensor& scales_, const Tensor& weight_values_, const Tensor& weight_scales_,
                    const Tensor& offsets_, at::ScalarType type) {
  refuse_unless(type == at::kFloat || type == at::kHalf || type == at::kBFloat16, "the result's dtype is float32, float16 or bfloat16");
  const Tensor values = bytes_of(values_, "values", 2), w = bytes_of(weight_values_, "weight_values", 3);
  same_device(values, w);
  const int64_t n = values.size(0), k = values.size(1), experts = w.size(0), width = w.size(1);
  refuse_unless(w.size(2) == k, "weight_values must have as many values in a row as values");
  refuse_unless(k <= GSB_MAX_INT8_ROW_LEN, "rows in 8 bits must hold at most 131071 values");
  refuse_unless(experts >= 1 && experts <= GSB_MAX_EXPERTS, "weight_values must hold between 1 and 65536 experts");
  const Tensor scales = scales_of(scales_, "scales", values), weight_scales = scales_of(weight_scales_, "weight_scales", w);
  const Tensor offsets = offsets_of(offsets_, experts, values);
  const c10::cuda::CUDAGuard guard(values.device());
  Tensor out = fresh({n, width}, type, values.device());
  if (out.numel() == 0) return out;
  if (k == 0) return out.zero_();
  const int64_t of_n = step_of(w, 1, in_lines(k)), of_expert = step_of(w, 0, of_n * width);
  done(ctx, gsb_expert_product_int8(ctx, stream(), static_cast<const int8_t*>(values.const_data_ptr()), n, k, step_of(values, 0, in_lines(k)),
                                    static_cast<const float*>(scales.const_data_ptr()), static_cast<const int8_t*>(w.const_data_ptr()), of_expert, of_n,
                                    static_cast<const float*>(weight_scales.const_data_ptr()), width, ids_ptr(offsets), experts, data(out),
                                    dtype_of(out, "out")),
       "gsb_expert_product_int8");
  return out;
}

// ---- dropout
struct Seed {
  uint64_t number = 0;
  Tensor on_device;  // where defined, read in the place of the number
};
Tensor drop(gsb_ctx* ctx, const Tensor& x_, double p, const Seed& seed) {
  const int dtype = dtype_of(x_, "x");
  refuse_unless(x_.is_cuda(), "x must be a CUDA tensor");
  refuse_unless(p >= 0.0 && p <= 1.0, "p must be between 0 and 1");
  if (seed.on_device.defined()) {
    refuse_unless(seed.on_device.scalar_type() == at::kLong && seed.on_device.numel() == 1, "a seed that is a tensor must hold one int64");
    refuse_unless(seed.on_device.is_cuda(), "a seed that is a tensor must be a CUDA tensor");
    refuse_unless(!seed.on_device.is_neg(), "a seed that is a tensor must not be a negated view");
    same_device(seed.on_device, x_);
  }
  const c10::cuda::CUDAGuard guard(x_.device());
  Tensor x = as_stored(x_);
  int64_t rows = 1, width = x.numel(), stride = x.numel();
  if (!x.is_contiguous()) {  // rows at one distance are read in place
    if (x.dim() == 2 && x.stride(1) == 1) {
      rows = x.size(0);
      width = x.size(1);
      stride = x.stride(0);
    } else {
      x = x.contiguous();
    }
  }
  Tensor out = fresh(x.sizes(), x.scalar_type(), x.device());
  if (out.numel() == 0) return out;
  done(ctx, gsb_dropout(ctx, stream(), x.const_data_ptr(), dtype, rows, width, stride, p, seed.number,
                        seed.on_device.defined() ? static_cast<const uint64_t*>(seed.on_device.const_data_ptr()) : nullptr, data(out)),
       "gsb_dropout");
  return out;
}

// ---- autograd --------------------------------------------------------------------------------------------------------------
gsb_ctx* kept(int64_t handle) { return reinterpret_cast<gsb_ctx*>(handle); }
int64_t keep(gsb_ctx* ctx) { return reinterpret_cast<int64_t>(ctx); }

// Gradients that are differentiated again say that they cannot be, instead of passing for constants, whatever they are
// differentiated for: the node that says so stands between them and all that they were made of.
tensor_list only_once(tensor_list grads, std::initializer_list<Tensor> made_of) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list given;
  for (const Tensor& g : grads)
    if (g.defined()) given.push_back(g.detach().requires_grad_(true));
  given.insert(given.end(), made_of.begin(), made_of.end());
  const auto count = (int)given.size();
  auto error = std::make_shared<torch::autograd::DelayedError>("this gradient cannot be differentiated again", count);
  variable_list marked = (*error)(std::move(given));
  size_t next = 0;
  for (Tensor& g : grads)
    if (g.defined()) g = marked[next++];
  return grads;
}

// While an eager graph of a leaf is alive, a captured backward pass would add to the leaf's gradient through that graph's node,
// on the stream that it was made on, which ends the capture, and with it the process.  Said here, where it can still be helped.
bool capturing() { return c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None; }
[[noreturn]] void refuse_capture(const char* whose) {
  throw std::runtime_error(std::string("a graph of ") + whose +
                           " made outside the capture, on another stream, is still alive: drop its outputs before capturing");
}
void refuse_foreign_accumulator(const Tensor& leaf) {
  if (!leaf.defined() || !leaf.requires_grad() || leaf.grad_fn() || !leaf.is_cuda() || !capturing()) return;
  const auto node = torch::autograd::impl::try_get_grad_accumulator(leaf);
  if (!node) return;
  const auto of_node = node->stream();
  if (of_node && *of_node != c10::cuda::getCurrentCUDAStream(leaf.get_device()).unwrap()) refuse_capture("this leaf");
}

// Whether behind an operand there is, by operations of the capture alone, a leaf whose node belongs to the default stream, which cannot
// join a capture.  Only a captured backward pass would meet it, and refuses there.
bool foreign_leaf_behind(const Tensor& t) {
  if (!t.defined() || !t.requires_grad() || !t.grad_fn() || !t.is_cuda() || !capturing()) return false;
  const auto here = c10::cuda::getCurrentCUDAStream(t.get_device()).unwrap();
  const auto never = c10::cuda::getDefaultCUDAStream(t.get_device()).unwrap();
  std::vector<torch::autograd::Node*> left{t.grad_fn().get()};
  std::unordered_set<torch::autograd::Node*> seen(left.begin(), left.end());
  while (!left.empty()) {
    torch::autograd::Node* const node = left.back();
    left.pop_back();
    const auto of_node = node->stream();
    if (dynamic_cast<torch::autograd::AccumulateGrad*>(node)) {
      if (of_node && *of_node == never) return true;
    } else if (!of_node || *of_node == here) {
      for (const auto& edge : node->next_edges())
        if (edge.function && seen.insert(edge.function.get()).second) left.push_back(edge.function.get());
    }
  }
  return false;
}
void refuse_foreign_leaf(AutogradContext* a) {
  if (a->saved_data.count("foreign") != 0 && capturing()) refuse_capture("a leaf behind this operand");
}

// The kernels read memory and know nothing of forward-mode tangents: a result without one would pass for a constant.
void refuse_tangents(const char* name, const Tensor& t) {
  if (t.defined() && t._fw_grad(0).defined())
    throw std::runtime_error(std::string(name) + " carries a forward-mode tangent; only reverse-mode gradients are implemented");
}

struct EmbeddingFunction : torch::autograd::Function<EmbeddingFunction> {
  static Tensor forward(AutogradContext* a, const Tensor& table, const Tensor& ids, int64_t handle, double scale, bool padded,
                        int64_t padding, bool sparse, bool foreign) {
    a->save_for_backward({ids});
    a->set_materialize_grads(false);
    a->saved_data["handle"] = handle;
    if (foreign) a->saved_data["foreign"] = true;
    a->saved_data["scale"] = scale;
    a->saved_data["padded"] = padded;
    a->saved_data["padding"] = padding;
    a->saved_data["sparse"] = sparse;
    a->saved_data["rows"] = table.size(0);
    return lookup(kept(handle), table, ids, scale, {padded, padding});
  }
  static tensor_list backward(AutogradContext* a, tensor_list grads) {
    tensor_list out(8);
    if (!grads[0].defined()) return out;
    refuse_tangents("grad", grads[0]);
    refuse_foreign_leaf(a);
    gsb_ctx* ctx = kept(a->saved_data["handle"].toInt());
    const Tensor ids = a->get_saved_variables()[0];
    const Padding pad{a->saved_data["padded"].toBool(), a->saved_data["padding"].toInt()};
    const double scale = a->saved_data["scale"].toDouble();
    const int64_t rows = a->saved_data["rows"].toInt();
    {
      const at::NoGradGuard no_grad;
      if (a->saved_data["sparse"].toBool()) {
        const std::vector<Tensor> r = grad_rows(ctx, grads[0], ids, rows, scale, pad, std::nullopt, true);
        out[0] = at::_sparse_coo_tensor_unsafe(r[0].unsqueeze(0), r[1], {rows, r[1].size(1)}, r[1].options().layout(at::kSparse), true);
      } else {
        out[0] = dense_grad(ctx, grads[0], ids, rows, scale, pad, std::nullopt);
      }
    }
    return only_once(std::move(out), {grads[0]});
  }
};

struct DispatchFunction : torch::autograd::Function<DispatchFunction> {
  static Tensor forward(AutogradContext* a, const Tensor& x, const Tensor& place, int64_t handle, bool foreign) {
    a->save_for_backward({place});
    a->set_materialize_grads(false);
    a->saved_data["handle"] = handle;
    if (foreign) a->saved_data["foreign"] = true;
    return spread(kept(handle), x, place, Tensor());
  }
  static tensor_list backward(AutogradContext* a, tensor_list grads) {
    tensor_list out(4);
    if (!grads[0].defined()) return out;
    refuse_tangents("grad", grads[0]);
    refuse_foreign_leaf(a);
    {
      const at::NoGradGuard no_grad;
      out[0] = combine(kept(a->saved_data["handle"].toInt()), grads[0], a->get_saved_variables()[0], Tensor());
    }
    return only_once(std::move(out), {grads[0]});
  }
};

// Without weights (autograd functions take defined tensors only).
struct GatherFunction : torch::autograd::Function<GatherFunction> {
  static Tensor forward(AutogradContext* a, const Tensor& rows, const Tensor& place, int64_t handle, bool foreign) {
    a->save_for_backward({place});
    a->set_materialize_grads(false);
    a->saved_data["handle"] = handle;
    if (foreign) a->saved_data["foreign"] = true;
    a->saved_data["rows"] = rows.size(0);
    return combine(kept(handle), rows, place, Tensor());
  }
  static tensor_list backward(AutogradContext* a, tensor_list grads) {
    tensor_list out(4);
    if (!grads[0].defined()) return out;
    refuse_tangents("grad", grads[0]);
    refuse_foreign_leaf(a);
    const Tensor place = a->get_saved_variables()[0];
    {
      const at::NoGradGuard no_grad;
      out[0] = spread(kept(a->saved_data["handle"].toInt()), grads[0], place, Tensor()).narrow(0, 0, a->saved_data["rows"].toInt());
    }
    return only_once(std::move(out), {grads[0]});
  }
};

struct CombineFunction : torch::autograd::Function<CombineFunction> {
  static Tensor forward(AutogradContext* a, const Tensor& rows, const Tensor& place, const Tensor& weights, int64_t handle, bool foreign) {
    a->save_for_backward({rows, place, weights});
    a->set_materialize_grads(false);
    a->saved_data["handle"] = handle;
    if (foreign) a->saved_data["foreign"] = true;
    return combine(kept(handle), rows, place, weights);
  }
  static tensor_list backward(AutogradContext* a, tensor_list grads) {
    tensor_list out(5);
    if (!grads[0].defined()) return out;
    refuse_tangents("grad", grads[0]);
    refuse_foreign_leaf(a);
    const auto saved = a->get_saved_variables();
    {
      const at::NoGradGuard no_grad;
      std::tie(out[0], out[2]) = combine_grad(kept(a->saved_data["handle"].toInt()), grads[0], saved[0], saved[1], saved[2],
                                              a->needs_input_grad(0), a->needs_input_grad(2));
    }
    return only_once(std::move(out), {grads[0], saved[0], saved[2]});
  }
};

struct ProductFunction : torch::autograd::Function<ProductFunction> {
  static Tensor forward(AutogradContext* a, const Tensor& rows, const Tensor& weights, const Tensor& offsets, int64_t handle, bool foreign) {
    a->save_for_backward({rows, weights, offsets});
    a->set_materialize_grads(false);
    a->saved_data["handle"] = handle;
    if (foreign) a->saved_data["foreign"] = true;
    return product(kept(handle), rows, weights, offsets);
  }
  static tensor_list backward(AutogradContext* a, tensor_list grads) {
    tensor_list out(5);
    if (!grads[0].defined()) return out;
    refuse_tangents("grad", grads[0]);
    refuse_foreign_leaf(a);
    const auto saved = a->get_saved_variables();
    {
      const at::NoGradGuard no_grad;
      gsb_ctx* ctx = kept(a->saved_data["handle"].toInt());
      if (a->needs_input_grad(0)) out[0] = product(ctx, grads[0], saved[1].transpose(1, 2), saved[2]);
      if (a->needs_input_grad(1)) out[1] = product_grad(ctx, saved[0], grads[0], saved[2]);
    }
    return only_once(std::move(out), {grads[0], saved[0], saved[1]});
  }
};

// Two kinds of seed: a number, which is remembered, and a tensor, which is saved (autograd notices when it is changed in place).
struct DropoutFunction : torch::autograd::Function<DropoutFunction> {
  static Tensor forward(AutogradContext* a, const Tensor& x, double p, int64_t number, const std::optional<Tensor>& on_device, int64_t handle,
                        bool foreign) {
    a->set_materialize_grads(false);
    a->saved_data["handle"] = handle;
    if (foreign) a->saved_data["foreign"] = true;
    a->saved_data["p"] = p;
    a->saved_data["number"] = number;
    if (on_device) a->save_for_backward({*on_device});
    return drop(kept(handle), x, p, {(uint64_t)number, on_device.value_or(Tensor())});
  }
  static tensor_list backward(AutogradContext* a, tensor_list grads) {
    tensor_list out(6);
    if (!grads[0].defined()) return out;
    refuse_tangents("grad", grads[0]);
    refuse_foreign_leaf(a);
    const auto saved = a->get_saved_variables();
    {
      const at::NoGradGuard no_grad;
      out[0] = drop(kept(a->saved_data["handle"].toInt()), grads[0], a->saved_data["p"].toDouble(),
                    {(uint64_t)a->saved_data["number"].toInt(), saved.empty() ? Tensor() : saved[0]});
    }
    return only_once(std::move(out), {grads[0]});
  }
};

bool follows(const Tensor& t) { return t.defined() && t.requires_grad() && at::GradMode::is_enabled(); }

// ---- the Python functions ----------------------------------------------------------------------------------------------------
const Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) type_error(std::string(name) + " must be a tensor");
  return THPVariable_Unpack(o);
}
Tensor tensor_or_none(PyObject* o, const char* name) { return o == Py_None ? Tensor() : tensor(o, name); }
double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw PyErrorSet();
  return v;
}
Padding padding(PyObject* o) {
  if (o == Py_None) return {};
  return {true, integer(o)};
}
std::optional<at::ScalarType> dtype_or_none(PyObject* o) {
  if (o == Py_None) return std::nullopt;
  if (!THPDtype_Check(o)) type_error("dtype must be a torch.dtype");
  return reinterpret_cast<THPDtype*>(o)->scalar_type;
}

// Runs `f` without the GIL and turns what it throws into Python exceptions.
template <class F>
auto without_gil(F f) {
  try {
    NoGil free;
    return f();
  } catch (const BadArgument& e) {
    type_error(e.what());
  } catch (const Failed& e) {
    if (PyObject* o = PyObject_CallFunction(g_error, "iss", e.status, e.where.c_str(), e.detail.c_str())) {
      PyErr_SetObject(g_error, o);
      Py_DECREF(o);
    }
    throw PyErrorSet();
  }
}

FUNCTION(embedding_lookup, 5) {  // (ctx, table, ids, scale, padding id | None) -> rows
  gsb_ctx* ctx = context(a[0]);
  const Tensor &table = tensor(a[1], "table"), &ids = tensor(a[2], "ids");
  const double scale = number(a[3]);
  const Padding pad = padding(a[4]);
  return wrap(without_gil([&] {
    const at::NoGradGuard no_grad;
    return lookup(ctx, table, ids, scale, pad);
  }));
}

FUNCTION(embedding_grad, 7) {  // (ctx, grad, ids, num_rows, scale, padding id | None, dtype | None) -> gradient of the table
  gsb_ctx* ctx = context(a[0]);
  const Tensor &grad = tensor(a[1], "grad"), &ids = tensor(a[2], "ids");
  const int64_t rows = integer(a[3]);
  const double scale = number(a[4]);
  const Padding pad = padding(a[5]);
  const auto dtype = dtype_or_none(a[6]);
  return wrap(without_gil([&] {
    const at::NoGradGuard no_grad;
    return dense_grad(ctx, grad, ids, rows, scale, pad, dtype);
  }));
}

// (ctx, grad, ids, num_rows, scale, padding id | None, dtype | None, sync) -> (row ids, rows) or (row ids, rows, number)
FUNCTION(embedding_grad_rows, 8) {
  gsb_ctx* ctx = context(a[0]);
  const Tensor &grad = tensor(a[1], "grad"), &ids = tensor(a[2], "ids");
  const int64_t rows = integer(a[3]);
  const double scale = number(a[4]);
  const Padding pad = padding(a[5]);
  const auto dtype = dtype_or_none(a[6]);
  const bool sync = truth(a[7]);
  std::vector<Tensor> r = without_gil([&] {
    const at::NoGradGuard no_grad;
    return grad_rows(ctx, grad, ids, rows, scale, pad, dtype, sync);
  });
  if (sync) return tuple_of(wrap(std::move(r[0])), wrap(std::move(r[1])));
  return tuple_of(wrap(std::move(r[0])), wrap(std::move(r[1])), wrap(std::move(r[2])));
}

FUNCTION(expert_order, 3) {  // (ctx, expert ids, number of experts) -> (offsets, source, place)
  gsb_ctx* ctx = context(a[0]);
  const Tensor& experts = tensor(a[1], "expert_ids");
  const int64_t number_of = integer(a[2]);
  std::vector<Tensor> r = without_gil([&] { return order(ctx, experts, number_of); });
  return tuple_of(wrap(std::move(r[0])), wrap(std::move(r[1])), wrap(std::move(r[2])));
}

FUNCTION(expert_dispatch, 4) {  // (ctx, x, place, weights | None) -> rows
  gsb_ctx* ctx = context(a[0]);
  const Tensor &x = tensor(a[1], "x"), &place = tensor(a[2], "place");
  const Tensor weights = tensor_or_none(a[3], "weights");
  return wrap(without_gil([&] {
    const at::NoGradGuard no_grad;
    return spread(ctx, x, place, weights);
  }));
}

FUNCTION(expert_combine, 4) {  // (ctx, rows, place, weights | None) -> out
  gsb_ctx* ctx = context(a[0]);
  const Tensor &rows = tensor(a[1], "rows"), &place = tensor(a[2], "place");
  const Tensor weights = tensor_or_none(a[3], "weights");
  return wrap(without_gil([&] {
    const at::NoGradGuard no_grad;
    return combine(ctx, rows, place, weights);
  }));
}

FUNCTION(expert_combine_grad, 5) {  // (ctx, grad, rows, place, weights | None) -> (gradient of rows, of weights | None)
  gsb_ctx* ctx = context(a[0]);
  const Tensor &grad = tensor(a[1], "grad"), &rows = tensor(a[2], "rows"), &place = tensor(a[3], "place");
  const Tensor weights = tensor_or_none(a[4], "weights");
  auto r = without_gil([&] {
    const at::NoGradGuard no_grad;
    return combine_grad(ctx, grad, rows, place, weights, true, true);
  });
  return tuple_of(wrap(std::move(r.first)), wrap(std::move(r.second)));
}

FUNCTION(nn_embedding, 6) {  // (ctx, table, ids, scale, padding id | None, sparse gradient) -> rows
  gsb_ctx* ctx = context(a[0]);
  const Tensor &table = tensor(a[1], "table"), &ids = tensor(a[2], "ids");
  const double scale = number(a[3]);
  const Padding pad = padding(a[4]);
  const bool sparse = truth(a[5]);
  return wrap(without_gil([&] {
    refuse_tangents("table", table);
    if (!follows(table)) return lookup(ctx, table, ids, scale, pad);
    rows_of(table, "table");
    refuse_foreign_accumulator(table);
    return EmbeddingFunction::apply(table, ids, keep(ctx), scale, pad.given, pad.id, sparse, foreign_leaf_behind(table));
  }));
}

FUNCTION(nn_dispatch, 3) {  // (ctx, x, place) -> rows
  gsb_ctx* ctx = context(a[0]);
  const Tensor &x = tensor(a[1], "x"), &place = tensor(a[2], "place");
  return wrap(without_gil([&] {
    refuse_tangents("x", x);
    if (!follows(x)) return spread(ctx, x, place, Tensor());
    refuse_foreign_accumulator(x);
    return DispatchFunction::apply(x, place, keep(ctx), foreign_leaf_behind(x));
  }));
}

FUNCTION(nn_combine, 4) {  // (ctx, rows, place, weights | None) -> out
  gsb_ctx* ctx = context(a[0]);
  const Tensor &rows = tensor(a[1], "rows"), &place = tensor(a[2], "place");
  const Tensor weights = tensor_or_none(a[3], "weights");
  return wrap(without_gil([&] {
    refuse_tangents("rows", rows);
    refuse_tangents("weights", weights);
    if (!follows(rows) && !follows(weights)) return combine(ctx, rows, place, weights);
    refuse_foreign_accumulator(rows);
    refuse_foreign_accumulator(weights);
    const bool foreign = foreign_leaf_behind(rows) || foreign_leaf_behind(weights);
    if (!weights.defined()) return GatherFunction::apply(rows, place, keep(ctx), foreign);
    return CombineFunction::apply(rows, place, weights, keep(ctx), foreign);
  }));
}

FUNCTION(expert_product, 4) {  // (ctx, rows, weights, offsets) -> out
  gsb_ctx* ctx = context(a[0]);
  const Tensor &rows = tensor(a[1], "rows"), &weights = tensor(a[2], "weights"), &offsets = tensor(a[3], "offsets");
  return wrap(without_gil([&] {
    const at::NoGradGuard no_grad;
    return product(ctx, rows, weights, offsets);
  }));
}

FUNCTION(expert_product_grad, 4) {  // (ctx, rows, grad, offsets) -> gradient of the weights
  gsb_ctx* ctx = context(a[0]);
  const Tensor &rows = tensor(a[1], "rows"), &grad = tensor(a[2], "grad"), &offsets = tensor(a[3], "offsets");
  return wrap(without_gil([&] {
    const at::NoGradGuard no_grad;
    return product_grad(ctx, rows, grad, offsets);
  }));
}

FUNCTION(quantize_rows, 2) {  // (ctx, x) -> (values, scales)
  gsb_ctx* ctx = context(a[0]);
  const Tensor& x = tensor(a[1], "x");
  auto r = without_gil([&] {
    const at::NoGradGuard no_grad;
    return quantize(ctx, x);
  });
  return tuple_of(wrap(std::move(r.first)), wrap(std::move(r.second)));
}

FUNCTION(expert_product_int8, 7) {  // (ctx, values, scales, weight values, weight scales, offsets, dtype) -> out
  gsb_ctx* ctx = context(a[0]);
  const Tensor &values = tensor(a[1], "values"), &scales = tensor(a[2], "scales"), &weight_values = tensor(a[3], "weight_values");
  const Tensor &weight_scales = tensor(a[4], "weight_scales"), &offsets = tensor(a[5], "offsets");
  const auto dtype = dtype_or_none(a[6]);
  if (!dtype) type_error("dtype must be a torch.dtype");
  return wrap(without_gil([&] {
    const at::NoGradGuard no_grad;
    return product_int8(ctx, values, scales, weight_values, weight_scales, offsets, *dtype);
  }));
}

FUNCTION(dropout, 5) {  // (ctx, x, p, seed, seed on the device | None) -> out
  gsb_ctx* ctx = context(a[0]);
  const Tensor& x = tensor(a[1], "x");
  const double p = number(a[2]);
  const Seed seed{unsigned_integer(a[3]), tensor_or_none(a[4], "seed")};
  return wrap(without_gil([&] {
    const at::NoGradGuard no_grad;
    return drop(ctx, x, p, seed);
  }));
}

FUNCTION(nn_product, 4) {  // (ctx, rows, weights, offsets) -> out
  gsb_ctx* ctx = context(a[0]);
  const Tensor &rows = tensor(a[1], "rows"), &weights = tensor(a[2], "weights"), &offsets = tensor(a[3], "offsets");
  return wrap(without_gil([&] {
    refuse_tangents("rows", rows);
    refuse_tangents("weights", weights);
    if (!follows(rows) && !follows(weights)) return product(ctx, rows, weights, offsets);
    refuse_foreign_accumulator(rows);
    refuse_foreign_accumulator(weights);
    return ProductFunction::apply(rows, weights, offsets, keep(ctx), foreign_leaf_behind(rows) || foreign_leaf_behind(weights));
  }));
}

FUNCTION(nn_dropout, 5) {  // (ctx, x, p, seed, seed on the device | None) -> out
  gsb_ctx* ctx = context(a[0]);
  const Tensor& x = tensor(a[1], "x");
  const double p = number(a[2]);
  const Seed seed{unsigned_integer(a[3]), tensor_or_none(a[4], "seed")};
  return wrap(without_gil([&] {
    refuse_tangents("x", x);
    if (!follows(x)) return drop(ctx, x, p, seed);
    refuse_foreign_accumulator(x);
    return DropoutFunction::apply(x, p, (int64_t)seed.number, seed.on_device.defined() ? std::optional<Tensor>(seed.on_device) : std::nullopt, keep(ctx),
                                  foreign_leaf_behind(x));
  }));
}

}  // namespace

PyMethodDef native::row_methods[] = {ENTRY(embedding_lookup), ENTRY(embedding_grad), ENTRY(embedding_grad_rows),
                                     ENTRY(expert_order),     ENTRY(expert_dispatch), ENTRY(expert_combine),
                                     ENTRY(expert_combine_grad), ENTRY(nn_embedding), ENTRY(nn_dispatch),
                                     ENTRY(nn_combine),       ENTRY(expert_product), ENTRY(expert_product_grad),
                                     ENTRY(quantize_rows),    ENTRY(expert_product_int8), ENTRY(dropout),
                                     ENTRY(nn_product),       ENTRY(nn_dropout), {nullptr, nullptr, 0, nullptr}};
