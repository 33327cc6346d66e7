// lq_torch.cpp -- the calls whose host time counts, bound to torch in C++:
// AdapterBank's forward and backward pass and GradClipper's call.  They check
// their arguments, allocate and call the C entry points of lq_sm100.h, as the
// other modules do from Python through ctypes.  A decode step's adapters take
// some 5 us on the device; the same calls took 11 us in Python, and a training
// step 50 us more, most of it in Python on the autograd engine's thread.
#include <torch/extension.h>

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "../../include/lq_sm100.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

std::string name_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return "float32";
    case at::kHalf: return "float16";
    case at::kBFloat16: return "bfloat16";
    default: return c10::toString(t);
  }
}
int code_of(at::ScalarType t) { return t == at::kFloat ? LQ_F32 : t == at::kHalf ? LQ_F16 : LQ_BF16; }

void check(int status) {
  if (status == LQ_OK) return;
  const std::string m = lq_last_error();
  TORCH_CHECK_VALUE(status != LQ_EINVAL && status != LQ_ERANGE, m);
  TORCH_CHECK_TYPE(status != LQ_EDTYPE, m);
  TORCH_CHECK(false, m, " (status ", status, ")");
}

bool on16(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }

// Elements from row to row of x [..., width], or -1 where the kernels cannot
// read its rows as they lie: values side by side, one stride over all leading
// dimensions, rows on 16 bytes.
int64_t row_stride(const Tensor& x) {
  const int64_t width = x.size(-1);
  if (x.is_contiguous()) return on16(x) || x.numel() == 0 ? width : -1;
  if (x.numel() == 0 || x.stride(-1) != 1 || !on16(x)) return -1;
  int64_t rows = 1, stride = -1;
  for (int64_t d = x.dim() - 2; d >= 0; --d) {
    if (x.size(d) == 1) continue;
    if (stride < 0) stride = x.stride(d);
    else if (x.stride(d) != rows * stride) return -1;
    rows *= x.size(d);
  }
  return stride < 0 ? width : stride % 8 == 0 ? stride : -1;
}
// x as rows that the kernels can read, laid out anew if need be
Tensor rows_of(const Tensor& x, int64_t& stride) {
  stride = row_stride(x);
  if (stride >= 0) return x;
  stride = x.size(-1);
  return x.clone(at::MemoryFormat::Contiguous);
}

// t side by side and on 16 bytes
Tensor whole(const Tensor& t) { return t.is_contiguous() && on16(t) ? t : t.clone(at::MemoryFormat::Contiguous); }

// Whether the rows of y (ys apart, N wide) can be written where the rows of x are
// read: none is another token's row of x.  A token's own row is read before it
// is written.
bool rows_apart(const Tensor& x, int64_t xs, int64_t K, const Tensor& y, int64_t ys, int64_t N, int64_t tokens) {
  const int64_t at_x = reinterpret_cast<intptr_t>(x.data_ptr()) / 2, at_y = reinterpret_cast<intptr_t>(y.data_ptr()) / 2;
  if (tokens <= 1 || at_x + (tokens - 1) * xs + K <= at_y || at_y + (tokens - 1) * ys + N <= at_x) return true;
  if (xs != ys || xs < K) return false;
  const int64_t d = at_y - at_x, c = (d % xs + xs) % xs;  // the columns of x's rows that y begins at
  return c + N <= xs && (c >= K || c == d);
}

struct Call {
  lq_adapter_bank bank;
  lq_adapter_form form;
  Tensor a, b, s, x, low, out;
};

Call run(const Tensor& x, const Tensor& lora_a, const Tensor& lora_b, const Tensor& scaling, const OptTensor& base,
         const Tensor& plan, int64_t tokens, int64_t num_adapters, bool keep, bool in_place) {
  TORCH_CHECK(x.is_cuda(), "AdapterBank: expected a CUDA tensor, got device ", x.device(), " (llm_quant_b200 has no CPU implementation)");
  const auto type = x.scalar_type();
  TORCH_CHECK_TYPE(type == at::kHalf || type == at::kBFloat16, "AdapterBank: unsupported dtype ", name_of(type), " (float16, bfloat16)");
  TORCH_CHECK(lora_a.dim() == 3 && lora_b.dim() == 3 && lora_a.size(0) == lora_b.size(0) && lora_a.size(1) == lora_b.size(1) &&
                  scaling.dim() == 1 && scaling.size(0) == lora_a.size(0),
              "AdapterBank: lora_A ", lora_a.sizes(), ", lora_B ", lora_b.sizes(), " and scaling ", scaling.sizes(), " do not go together");
  const int64_t L = lora_a.size(0), R = lora_a.size(1), K = lora_a.size(2), N = lora_b.size(2);
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) == K && x.numel() == tokens * K, "AdapterBank: x ", x.sizes(), " is not ", tokens,
              " tokens of ", K, " features");
  TORCH_CHECK_VALUE(num_adapters == L, "AdapterBank: a batch for ", num_adapters, " adapters, a bank of ", L);
  TORCH_CHECK(lora_a.device() == x.device() && lora_b.device() == x.device() && scaling.device() == x.device() &&
                  plan.device() == x.device(),
              "AdapterBank: x on ", x.device(), ", the bank on ", lora_a.device(), ", the batch on ", plan.device());
  TORCH_CHECK_TYPE(lora_a.scalar_type() == lora_b.scalar_type() && scaling.scalar_type() == at::kFloat, "AdapterBank: lora_A is ",
                   name_of(lora_a.scalar_type()), ", lora_B ", name_of(lora_b.scalar_type()), ", scaling ",
                   name_of(scaling.scalar_type()), " (expected float32)");
  TORCH_CHECK_TYPE(lora_a.scalar_type() == type || lora_a.scalar_type() == at::kFloat, "AdapterBank: parameters in ",
                   name_of(lora_a.scalar_type()), " for activations in ", name_of(type), " (theirs or float32)");
  at::DimVector shape(x.sizes().begin(), x.sizes().end());
  shape.back() = N;
  if (base)
    TORCH_CHECK(base->scalar_type() == type && base->device() == x.device() && base->sizes() == at::IntArrayRef(shape),
                "AdapterBank: base ", base->sizes(), " ", name_of(base->scalar_type()), " on ", base->device(), " for x ", x.sizes(),
                " ", name_of(type), " on ", x.device());
  Call c;
  c.form = {tokens, K, N, N, keep};
  c.x = rows_of(x, c.form.x_stride);
  Tensor from;
  if (in_place) {
    const int64_t stride = row_stride(*base);
    TORCH_CHECK_VALUE(stride >= 0 && (tokens <= 1 || stride >= N), "AdapterBank.add_: y ", base->sizes(), " with strides ",
                      base->strides(), " must be rows on 16 bytes");
    TORCH_CHECK_VALUE(rows_apart(c.x, c.form.x_stride, K, *base, stride, N, tokens),
                      "AdapterBank.add_: rows of y overlap other tokens' rows of x");
    c.form.base_stride = c.form.out_stride = stride;
    from = c.out = *base;
  } else {
    if (base) from = rows_of(*base, c.form.base_stride);
    c.out = at::empty(shape, x.options().requires_grad(false));
  }
  const auto ready = [&](const Tensor& t) { return whole(t.scalar_type() == type ? t : t.to(type)); };
  c.a = ready(lora_a), c.b = ready(lora_b), c.s = scaling.contiguous();
  c.bank = {c.a.data_ptr(), c.b.data_ptr(), c.s.data_ptr<float>(), L, R, K, N, code_of(type)};
  if (tokens == 0) return c;
  const size_t low = lq_adapter_low_bytes(&c.bank, &c.form);
  if (low) c.low = at::empty({(int64_t)low}, plan.options());
  check(lq_adapter_forward(&c.bank, &c.form, plan.data_ptr(), c.x.data_ptr(), from.defined() ? from.data_ptr() : nullptr,
                           c.out.data_ptr(), low ? c.low.data_ptr() : nullptr, low, at::cuda::getCurrentCUDAStream()));
  return c;
}

// base + each token's adapter of x, with the gradients of x, lora_A, lora_B and base
struct Adapters : torch::autograd::Function<Adapters> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& lora_a, const Tensor& lora_b,
                        const OptTensor& base, const Tensor& scaling, const Tensor& plan, int64_t tokens, int64_t num_adapters) {
    TORCH_CHECK(!plan.is_inference(), "AdapterBank: a batch that was made in inference mode cannot be used with gradients");
    Call c = run(x, lora_a, lora_b, scaling, base, plan, tokens, num_adapters, true, false);
    // the weights as the call rounded them; all of these raise if they were changed since
    ctx->save_for_backward({c.x, c.a, c.b, scaling, c.low});
    // not the plan: saved-tensor hooks may bring back copies, and its status word is read where it lies
    ctx->saved_data["plan"] = plan;
    std::vector<int64_t> form = {static_cast<int64_t>(plan._version()), num_adapters, static_cast<int64_t>(lora_a.scalar_type()),
                                 base.has_value()};
    form.insert(form.end(), x.sizes().begin(), x.sizes().end());
    ctx->saved_data["form"] = std::move(form);
    return c.out;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "AdapterBank: gradients of gradients are not computed");
    torch::autograd::variable_list out(8);
    Tensor dy = grads[0];
    if (!dy.defined()) return out;
    const bool want[3] = {ctx->needs_input_grad(0), ctx->needs_input_grad(1), ctx->needs_input_grad(2)};
    const auto kept = ctx->saved_data["form"].toIntVector();  // the plan's version, adapters, the parameters' type, base, x's shape
    const at::IntArrayRef shape = at::IntArrayRef(kept).slice(4);
    if (kept[3]) out[3] = dy;
    if (!want[0] && !want[1] && !want[2]) return out;
    const auto saved = ctx->get_saved_variables();
    const Tensor plan = ctx->saved_data["plan"].toTensor();
    TORCH_CHECK(static_cast<int64_t>(plan._version()) == kept[0],
                "AdapterBank: the batch that gradients are computed for has been modified by an inplace operation "
                "(AdapterBatch.update) since the forward call");
    const auto type = static_cast<at::ScalarType>(kept[2]);
    // A hook may have laid them out anew, but what they hold has to be the same.
    const int64_t L = kept[1], R = saved[1].dim() == 3 ? saved[1].size(1) : 0;
    const int64_t sizes[2][3] = {{L, R, shape.back()}, {L, R, dy.size(-1)}};
    TORCH_CHECK(saved[0].sizes() == shape && saved[1].sizes() == at::IntArrayRef(sizes[0], 3) &&
                    saved[2].sizes() == at::IntArrayRef(sizes[1], 3) && saved[3].sizes() == at::IntArrayRef(L),
                "AdapterBank: saved tensors came back with other shapes");
    for (const Tensor& t : saved)
      if (t.defined())
        TORCH_CHECK(t.device() == plan.device(), "AdapterBank: a saved tensor came back on ", t.device(), ", not on ", plan.device());
    for (int i = 0; i < 3; ++i)
      TORCH_CHECK(saved[i].scalar_type() == dy.scalar_type(), "AdapterBank: a saved tensor came back in ", name_of(saved[i].scalar_type()));
    TORCH_CHECK(saved[3].scalar_type() == at::kFloat && (!saved[4].defined() || saved[4].scalar_type() == at::kByte),
                "AdapterBank: saved tensors came back in other types");
    const c10::cuda::CUDAGuard guard(plan.device());
    lq_adapter_form form = {saved[0].numel() / shape.back(), 0, 0, 0, 1};
    const Tensor x = rows_of(saved[0], form.x_stride), a = whole(saved[1]), b = whole(saved[2]), s = saved[3].contiguous();
    const Tensor low = saved[4].defined() ? whole(saved[4]) : Tensor();
    const lq_adapter_bank bank = {a.data_ptr(), b.data_ptr(), s.data_ptr<float>(), a.size(0), a.size(1), a.size(2), b.size(2),
                                  code_of(x.scalar_type())};
    const int64_t n = form.n;
    const Tensor d = rows_of(dy, form.out_stride);
    if (want[0]) out[0] = at::empty(shape, x.options());
    if (want[1]) out[1] = at::empty(a.sizes(), x.options().dtype(type));
    if (want[2]) out[2] = at::empty(b.sizes(), x.options().dtype(type));
    const size_t bytes = lq_adapter_backward_workspace_bytes(&bank, n);
    const Tensor ws = at::empty({(int64_t)bytes}, plan.options());
    const auto at = [](const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
    check(lq_adapter_backward(&bank, &form, plan.data_ptr(), x.data_ptr(), d.data_ptr(), at(low), low.defined() ? low.numel() : 0,
                              at(out[0]), at(out[1]), at(out[2]), code_of(type), ws.data_ptr(), bytes,
                              at::cuda::getCurrentCUDAStream()));
    return out;
  }
};

// A tangent of forward mode would be lost without a word.
void no_tangents(std::initializer_list<const Tensor*> tensors) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor* t : tensors)
    TORCH_CHECK(!t || !t->defined() || !t->_fw_grad(0).defined(), "AdapterBank: forward-mode derivatives are not computed");
}

Tensor adapters_forward(const Tensor& x, const Tensor& lora_a, const Tensor& lora_b, const Tensor& scaling, const OptTensor& base,
                        const Tensor& plan, int64_t tokens, int64_t num_adapters) {
  no_tangents({&x, &lora_a, &lora_b, &scaling, base ? &*base : nullptr});
  const c10::OptionalDeviceGuard guard(x.is_cuda() ? std::make_optional(x.device()) : std::nullopt);
  if (at::GradMode::is_enabled() &&
      (x.requires_grad() || lora_a.requires_grad() || lora_b.requires_grad() || (base && base->requires_grad())))
    return Adapters::apply(x, lora_a, lora_b, base, scaling, plan, tokens, num_adapters);
  return run(x, lora_a, lora_b, scaling, base, plan, tokens, num_adapters, false, false).out;
}

void adapters_add_(const Tensor& y, const Tensor& x, const Tensor& lora_a, const Tensor& lora_b, const Tensor& scaling,
                   const Tensor& plan, int64_t tokens, int64_t num_adapters) {
  no_tangents({&y, &x, &lora_a, &lora_b, &scaling});
  TORCH_CHECK(!at::GradMode::is_enabled() ||
                  !(x.requires_grad() || y.requires_grad() || lora_a.requires_grad() || lora_b.requires_grad()),
              "AdapterBank.add_: no gradient is computed here (use forward, or torch.no_grad())");
  const c10::OptionalDeviceGuard guard(x.is_cuda() ? std::make_optional(x.device()) : std::nullopt);
  run(x, lora_a, lora_b, scaling, y, plan, tokens, num_adapters, false, true);
  if (!y.is_inference()) y.unsafeGetTensorImpl()->bump_version();
}

// The tensors of a GradClipper, which has checked them, as the entry point takes them
class Clipper {
 public:
  Clipper(std::vector<Tensor> in, std::optional<std::vector<Tensor>> out, std::vector<Tensor> written)
      : in_(std::move(in)), out_(std::move(out)), written_(std::move(written)) {
    for (const Tensor& t : in_) from_.push_back(t.data_ptr()), n_.push_back(t.numel()), type_.push_back(code_of(t.scalar_type()));
    if (out_)
      for (const Tensor& t : *out_) to_.push_back(t.data_ptr());
    bytes_ = lq_clip_workspace_bytes(in_.size());
  }
  Tensor clip(double max_norm) const {
    for (size_t i = 0; i < in_.size(); ++i) {
      stays(in_[i], from_[i], i);
      if (out_) stays((*out_)[i], to_[i], i);
    }
    const c10::cuda::CUDAGuard guard(in_[0].device());
    const auto options = at::TensorOptions().device(in_[0].device());
    const Tensor norm = at::empty({}, options.dtype(at::kFloat)), ws = at::empty({(int64_t)bytes_}, options.dtype(at::kByte));
    check(lq_clip_grad_norm(from_.data(), out_ ? to_.data() : nullptr, n_.data(), type_.data(), in_.size(), max_norm,
                            norm.data_ptr<float>(), ws.data_ptr(), bytes_, at::cuda::getCurrentCUDAStream()));
    for (const Tensor& t : written_) t.unsafeGetTensorImpl()->bump_version();
    return norm;
  }

 private:
  // A storage that was resized has other memory, for its aliases too.
  static void stays(const Tensor& t, const void* at, size_t i) {
    TORCH_CHECK(t.numel() == 0 || (t.const_data_ptr() == at && t.storage().nbytes() >= (t.storage_offset() + t.numel()) * t.itemsize()),
                "GradClipper: the storage of tensor ", i, " was resized since the clipper was made");
  }
  std::vector<Tensor> in_;
  std::optional<std::vector<Tensor>> out_;
  std::vector<Tensor> written_;  // whose versions go up: one of those that share a buffer
  std::vector<const void*> from_;
  std::vector<void*> to_;
  std::vector<int64_t> n_;
  std::vector<int> type_;
  size_t bytes_ = 0;
};

}  // namespace

PYBIND11_MODULE(lq_torch, m) {
  m.attr("torch_version") = TORCH_VERSION;
  m.def("adapters_forward", &adapters_forward);
  m.def("adapters_add_", &adapters_add_);
  pybind11::class_<Clipper>(m, "Clipper")
      .def(pybind11::init<std::vector<Tensor>, std::optional<std::vector<Tensor>>, std::vector<Tensor>>())
      .def("clip", &Clipper::clip);
}
