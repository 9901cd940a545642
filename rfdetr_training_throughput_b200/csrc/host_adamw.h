// The optimiser's step on lists of tensors (see host_adamw.cpp).
#pragma once

#include <tuple>
#include <vector>

#include "host_common.h"

namespace rfm_host {

using TensorList = std::vector<Tensor>;

void adamw_step(const TensorList& params, const TensorList& grads, const TensorList& exp_avg,
                const TensorList& exp_avg_sq, const std::optional<TensorList>& exp_avg_scale,
                const std::optional<TensorList>& exp_avg_sq_scale, int64_t step, const MaybeTensor& device_step,
                double lr, const MaybeTensor& device_lr, double beta1, double beta2, double eps, double weight_decay,
                const MaybeTensor& grad_scale);

std::tuple<Tensor, Tensor> dequantize_moments(const Tensor& exp_avg, const Tensor& exp_avg_sq,
                                              const Tensor& exp_avg_scale, const Tensor& exp_avg_sq_scale);

}  // namespace rfm_host
