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
// Arguments of a call without the launch tables: inputs, output, LSE; and its mask.
fm_attn_args base_args(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& out, const Tensor& lse, bool causal,
                       double scale, const Tensor& sink32);
void set_mask(fm_attn_args* a, const Tensor& idx, const Tensor& minmax, int tile_m, int tile_n);
// The per-K-tile reductions of a mask.
Tensor scan_mask(const Tensor& idx, int Sq, bool causal, int tile_m, int tile_n, void* stream);
// The operators around attention (fm_torch_cache.cpp).
void register_cache(pybind11::module_& m);

}  // namespace fm_host
