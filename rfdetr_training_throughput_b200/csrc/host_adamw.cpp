// adamw_step: checks of the tensor lists and the table that rfm_adamw takes.
#include <algorithm>

#include "host_adamw.h"

namespace rfm_host {
namespace {

int64_t scales_of(int64_t numel) { return (numel + RFM_MOMENT_BLOCK - 1) / RFM_MOMENT_BLOCK; }

void check_list(const char* name, const TensorRefs& list, at::ScalarType type, const at::Device& device,
                const TensorRefs& like, bool scales) {
  RFM_REQUIRE(list.size() == like.size(), name, " has ", list.size(), " tensors, params has ", like.size());
  for (size_t i = 0; i < list.size(); ++i) {
    const Tensor& t = *list[i];
    const int64_t n = scales ? scales_of(like[i]->numel()) : like[i]->numel();
    RFM_REQUIRE(t.defined() && t.scalar_type() == type && t.device() == device && t.numel() == n &&
                    t.layout() == at::kStrided && t.is_contiguous(),
                name, " must hold contiguous ", type, " tensors on the params' device; number ", i, " needs ", n,
                " elements and is ", t.defined() ? t.toString() : std::string("undefined"), " with ",
                t.defined() ? t.numel() : 0, t.defined() && !t.is_contiguous() ? ", not contiguous" : "");
  }
}

struct Span {
  uintptr_t first, past;  // bytes
};

Span span_of(const Tensor& t) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(t.data_ptr());
  return {at, at + static_cast<uintptr_t>(t.numel()) * t.element_size()};
}

// Spans of a list's tensors that hold something; `hull` is around them all and
// `rising` whether each lies behind the one before.
struct Spans {
  std::vector<Span> all;
  Span hull{~uintptr_t(0), 0};
  bool rising = true;

  explicit Spans(const TensorRefs& list) {
    all.reserve(list.size());
    for (const Tensor* t : list) {
      const Span s = span_of(*t);
      if (s.first == s.past) continue;
      rising = rising && (all.empty() || all.back().past <= s.first);
      hull.first = std::min(hull.first, s.first);
      hull.past = std::max(hull.past, s.past);
      all.push_back(s);
    }
  }
};

bool apart(const Span& a, const Span& b) { return a.past <= b.first || b.past <= a.first; }

// Whether no written byte is written twice, and no gradient lies in one.  Lists
// of tensors that follow each other in memory, away from the other lists, need
// no sorting.
void check_memory(const std::vector<Spans>& written, const Spans& grads) {
  bool plain = true;
  for (size_t i = 0; i < written.size() && plain; ++i) {
    plain = written[i].rising && (written[i].all.empty() || grads.all.empty() || apart(written[i].hull, grads.hull));
    for (size_t j = 0; j < i && plain; ++j) {
      plain = written[i].all.empty() || written[j].all.empty() || apart(written[i].hull, written[j].hull);
    }
  }
  if (plain) return;
  std::vector<Span> all;
  for (const Spans& s : written) all.insert(all.end(), s.all.begin(), s.all.end());
  std::sort(all.begin(), all.end(), [](const Span& a, const Span& b) { return a.first < b.first; });
  for (size_t i = 1; i < all.size(); ++i) {
    RFM_REQUIRE(all[i].first >= all[i - 1].past,
                "a tensor is given twice: params, moments and scales must not share memory");
  }
  for (const Span& g : grads.all) {
    // the first written span that ends behind the gradient's start
    const auto it = std::upper_bound(all.begin(), all.end(), g.first,
                                     [](uintptr_t at, const Span& w) { return at < w.past; });
    RFM_REQUIRE(it == all.end() || it->first >= g.past,
                "gradients must not share memory with params, moments or scales");
  }
}

// A scalar that kernels of the call read lies in nothing that they write.
void check_apart(const std::vector<Spans>& written, const Tensor& scalar) {
  const Span read = span_of(scalar);
  for (const Spans& list : written) {
    if (list.all.empty() || apart(list.hull, read)) continue;
    for (const Span& s : list.all) {
      RFM_REQUIRE(apart(s, read), "step, lr and grad_scale must not share memory with params, moments or scales");
    }
  }
}

void bump_versions(const TensorRefs& list) {
  for (const Tensor* t : list) t->unsafeGetTensorImpl()->bump_version();
}

void* scalar_pointer(const char* name, const Tensor& t, at::ScalarType type, const at::Device& device) {
  RFM_REQUIRE(t.scalar_type() == type && t.numel() == 1 && t.device() == device, name, " must be one ", type,
              " element on the params' device");
  return t.data_ptr();
}

}  // namespace

void adamw_step(const TensorRefs& params, const TensorRefs& grads, const TensorRefs& exp_avg,
                const TensorRefs& exp_avg_sq, const std::optional<TensorRefs>& exp_avg_scale,
                const std::optional<TensorRefs>& exp_avg_sq_scale, int64_t step, const MaybeTensor& device_step,
                double lr, const MaybeTensor& device_lr, double beta1, double beta2, double eps, double weight_decay,
                const MaybeTensor& grad_scale) {
  refuse_traced("adamw_step");
  RFM_REQUIRE(device_step.has_value() || step >= 1, "step counts from 1, got ", step);
  RFM_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0 && eps >= 0.0 && lr >= 0.0 &&
                  weight_decay >= 0.0,
              "betas must be in [0, 1), eps, lr and weight_decay not negative");
  if (params.empty()) {
    RFM_REQUIRE(grads.empty() && exp_avg.empty() && exp_avg_sq.empty(), "params is empty, the other lists are not");
    return;
  }
  RFM_REQUIRE(params[0]->defined() && params[0]->is_cuda(), "params must be CUDA tensors (adamw_step has no CPU path)");
  const at::Device device = params[0]->device();
  const at::ScalarType type = params[0]->scalar_type();
  RFM_REQUIRE(dtype_code(type) >= 0, "params must be float32, bfloat16 or float16, got ", type);
  const bool eight = exp_avg_scale.has_value();
  check_list("params", params, type, device, params, false);
  check_list("grads", grads, type, device, params, false);
  check_list("exp_avg", exp_avg, eight ? at::kChar : at::kFloat, device, params, false);
  check_list("exp_avg_sq", exp_avg_sq, eight ? at::kByte : at::kFloat, device, params, false);
  std::vector<Spans> written{Spans(params), Spans(exp_avg), Spans(exp_avg_sq)};
  if (eight) {
    check_list("scales", *exp_avg_scale, at::kFloat, device, params, true);
    check_list("scales", *exp_avg_sq_scale, at::kFloat, device, params, true);
    written.emplace_back(*exp_avg_scale);
    written.emplace_back(*exp_avg_sq_scale);
  }
  check_memory(written, Spans(grads));
  for (const MaybeTensor* scalar : {&device_step, &device_lr, &grad_scale}) {
    if (scalar->has_value()) check_apart(written, **scalar);
  }
  const size_t count = params.size();
  std::vector<rfm_adamw_tensor> table(count);
  for (size_t i = 0; i < count; ++i) {
    rfm_adamw_tensor& t = table[i];
    t = rfm_adamw_tensor{};
    t.param = params[i]->data_ptr();
    t.grad = grads[i]->data_ptr();
    t.exp_avg = exp_avg[i]->data_ptr();
    t.exp_avg_sq = exp_avg_sq[i]->data_ptr();
    if (eight) {
      t.exp_avg_scale = static_cast<float*>((*exp_avg_scale)[i]->data_ptr());
      t.exp_avg_sq_scale = static_cast<float*>((*exp_avg_sq_scale)[i]->data_ptr());
    }
    t.numel = params[i]->numel();
  }
  void* at_step = device_step ? scalar_pointer("step", *device_step, at::kLong, device) : nullptr;
  void* at_lr = device_lr ? scalar_pointer("lr", *device_lr, at::kFloat, device) : nullptr;
  void* at_scale = grad_scale ? scalar_pointer("grad_scale", *grad_scale, at::kFloat, device) : nullptr;
  // The in-place updates count as writes for autograd's saved tensors.  Before the launch: a tensor that may
  // not be written (of inference mode, outside it) raises here.
  bump_versions(params);
  bump_versions(exp_avg);
  bump_versions(exp_avg_sq);
  if (eight) {
    bump_versions(*exp_avg_scale);
    bump_versions(*exp_avg_sq_scale);
  }
  const c10::cuda::CUDAGuard guard(device);
  Tensor work;
  if (at_step != nullptr || at_lr != nullptr) work = at::empty({4}, params[0]->options().dtype(at::kFloat));
  check_call("rfm_adamw",
             rfm_adamw(table.data(), static_cast<int>(count), dtype_code(type), eight ? 8 : 32, lr, beta1, beta2, eps,
                       weight_decay, step, static_cast<const float*>(at_lr), static_cast<const int64_t*>(at_step),
                       static_cast<const float*>(at_scale), data_or_null(work), current_stream(device)));
}

std::tuple<Tensor, Tensor> dequantize_moments(const Tensor& exp_avg, const Tensor& exp_avg_sq,
                                              const Tensor& exp_avg_scale, const Tensor& exp_avg_sq_scale) {
  refuse_traced("dequantize_moments");
  RFM_REQUIRE(exp_avg.is_cuda(), "exp_avg must be a CUDA tensor (dequantize_moments has no CPU path)");
  const at::Device device = exp_avg.device();
  const TensorRefs like{&exp_avg};
  check_list("exp_avg", {&exp_avg}, at::kChar, device, like, false);
  check_list("exp_avg_sq", {&exp_avg_sq}, at::kByte, device, like, false);
  check_list("scales", {&exp_avg_scale}, at::kFloat, device, like, true);
  check_list("scales", {&exp_avg_sq_scale}, at::kFloat, device, like, true);
  const c10::cuda::CUDAGuard guard(device);
  const auto options = exp_avg.options().dtype(at::kFloat);
  Tensor m = at::empty(exp_avg.sizes(), options), v = at::empty(exp_avg.sizes(), options);
  check_call("rfm_adamw_moments",
             rfm_adamw_moments(exp_avg.data_ptr(), exp_avg_sq.data_ptr(), exp_avg_scale.data_ptr<float>(),
                               exp_avg_sq_scale.data_ptr<float>(), exp_avg.numel(), m.data_ptr<float>(),
                               v.data_ptr<float>(), current_stream(device)));
  return {m, v};
}

}  // namespace rfm_host
