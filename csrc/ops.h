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
