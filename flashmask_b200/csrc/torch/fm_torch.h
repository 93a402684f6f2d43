// What the sources of the native host share.
#pragma once

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include "flashmask_b200.h"

namespace fm_host {

using at::Tensor;

// A failed library call as the exception its status stands for.
void check(int rc, const char* what);
// AssertionError with `msg` unless ok.
void require(bool ok, const char* msg);
// FM_DTYPE_* of a 16-bit tensor; TypeError otherwise.
int dtype_code(const Tensor& t);
// t with its rows contiguous and no dimension of several elements with stride 0.
Tensor rows(const Tensor& t);
void strides(int64_t* out, const Tensor& t);
// fp32 [Hq] on q's device; undefined stays undefined.
Tensor sink_fp32(const Tensor& sink, const Tensor& q);
// flashmask_attention: (out, lse).
std::pair<Tensor, Tensor> attention(const Tensor& q, const Tensor& k, const Tensor& v, const std::optional<Tensor>& idx,
                                    const std::optional<Tensor>& sink, std::optional<double> scale, bool causal,
                                    int deterministic);
// The operators around attention (fm_torch_cache.cpp).
void register_cache(pybind11::module_& m);

}  // namespace fm_host
