// The optimiser's step on lists of tensors (see host_adamw.cpp).
#pragma once

#include <tuple>
#include <vector>

#include "host_common.h"

namespace rfm_host {

// Tensors that somebody else holds.
using TensorRefs = std::vector<const Tensor*>;

void adamw_step(const TensorRefs& params, const TensorRefs& grads, const TensorRefs& exp_avg,
                const TensorRefs& exp_avg_sq, const std::optional<TensorRefs>& exp_avg_scale,
                const std::optional<TensorRefs>& exp_avg_sq_scale, int64_t step, const MaybeTensor& device_step,
                double lr, const MaybeTensor& device_lr, double beta1, double beta2, double eps, double weight_decay,
                const MaybeTensor& grad_scale);

std::tuple<Tensor, Tensor> dequantize_moments(const Tensor& exp_avg, const Tensor& exp_avg_sq,
                                              const Tensor& exp_avg_scale, const Tensor& exp_avg_sq_scale);

}  // namespace rfm_host
