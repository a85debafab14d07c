// binding_utils.h -- what both files of the PyTorch binding use.
#pragma once

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>
#include <torch/library.h>

#include "sm120norm_b200.h"

namespace sm120n_binding {

inline int dtype_code(const torch::Tensor& t) {
  switch (t.scalar_type()) {
    case torch::kFloat32: return SM120N_F32;
    case torch::kFloat16: return SM120N_F16;
    case torch::kBFloat16: return SM120N_BF16;
    default: return -1;
  }
}

inline void* current_stream() {
  return static_cast<void*>(c10::cuda::getCurrentCUDAStream().stream());
}

inline bool is_fp8_storage(const torch::Tensor& t) {
  return t.scalar_type() == torch::kFloat8_e4m3fn || t.scalar_type() == torch::kByte;
}

// [tokens, heads, head_dim] with adjacent heads and elements; any token stride.
inline void check_head_rows(const torch::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.dim() == 3, name, " must have shape [tokens, heads, head_dim]");
  TORCH_CHECK(t.size(2) <= 1 || t.stride(2) == 1, name, " must have unit element stride");
  TORCH_CHECK(t.size(1) <= 1 || t.stride(1) == t.size(2), name,
              " heads must be adjacent (head stride == head_dim)");
}

inline int64_t token_stride(const torch::Tensor& t) {
  return t.size(0) <= 1 ? t.size(1) * t.size(2) : t.stride(0);
}

// Q, K and their optional caches as the generalised Q/K norm operators take
// them; everything but the positions.
void fill_qk_cache_args(sm120n_qk_cache_args& a, const torch::Tensor& query,
                        const torch::Tensor& key, const c10::optional<torch::Tensor>& value,
                        const torch::Tensor& query_weight, const torch::Tensor& key_weight,
                        const torch::Tensor& cos_sin_cache,
                        const c10::optional<torch::Tensor>& key_cache,
                        const c10::optional<torch::Tensor>& value_cache,
                        const c10::optional<torch::Tensor>& slot_mapping,
                        const c10::optional<torch::Tensor>& k_scale,
                        const c10::optional<torch::Tensor>& v_scale, bool is_neox,
                        c10::string_view kv_cache_layout, double epsilon);

// The serving operators as functions of the extension module.
void define_serving(pybind11::module_& m);

}  // namespace sm120n_binding
