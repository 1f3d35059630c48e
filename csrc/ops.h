// Host entry points that live outside ps_kernels.hip; bound there.
#pragma once

#include <ATen/ATen.h>

#include <string>

// row_cache.hip
void cache_write(at::Tensor cache, at::Tensor values,
                 c10::optional<at::Tensor> slots, const std::string& fmt,
                 bool unique);
at::Tensor cache_read(at::Tensor cache, int64_t dim,
                      c10::optional<at::Tensor> slots, const std::string& fmt,
                      at::ScalarType dtype);

// muon.hip
at::Tensor orthogonalize(at::Tensor x, int64_t steps, double a, double b,
                         double c, double eps);
void apply_muon(at::Tensor table, at::Tensor momentum, at::Tensor rows,
                bool sorted_unique, at::Tensor grads, double lr,
                double mu, bool nesterov, double weight_decay, int64_t steps,
                int64_t matrix_rows, double a, double b, double c,
                double eps);
