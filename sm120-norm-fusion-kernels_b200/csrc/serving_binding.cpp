// serving_binding.cpp -- the serving operators (include/sm120norm_b200_serving.h)
// as torch.ops.sm120_norm_ext.*. Tensor checks here, size checks and launch
// behind the C ABI, on the tensors' device and the current PyTorch stream; no
// host synchronisation. Only paged_decode_attention allocates: its workspace,
// anew for every call, so that no two calls or graphs share one.
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>

#include "binding_utils.h"
#include "sm120norm_b200_serving.h"

using namespace sm120n_binding;

namespace {

void raise_if_failed(int status) {
  TORCH_CHECK(status == SM120N_OK, sm120s_last_error());
}

// A contiguous one-dimensional CUDA tensor of `count` elements (any number if negative).
void check_vector(const torch::Tensor& t, c10::ScalarType type, int64_t count,
                  const c10::Device& device, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.is_contiguous() && t.dim() == 1 && t.scalar_type() == type, name,
              " must be a contiguous one-dimensional CUDA ", c10::toString(type), " tensor");
  TORCH_CHECK(count < 0 || t.numel() == count, name, " must have ", count, " entries (got ",
              t.numel(), ")");
  TORCH_CHECK(t.device() == device, "all tensors must be on the same CUDA device");
}

void check_table(const torch::Tensor& table, int64_t rows, const c10::Device& device) {
  TORCH_CHECK(table.is_cuda() && table.dim() == 2 && table.scalar_type() == torch::kInt &&
                  (table.size(1) <= 1 || table.stride(1) == 1),
              "block_table must be a CUDA int32 tensor [requests, blocks] with adjacent entries");
  TORCH_CHECK(table.size(0) == rows, "block_table must have one row per request");
  TORCH_CHECK(table.device() == device, "all tensors must be on the same CUDA device");
}

int64_t table_stride(const torch::Tensor& table) {
  return table.size(0) <= 1 ? table.size(1) : table.stride(0);
}

// The pool's count after the call: `out`, or in place.
int32_t* count_after(const torch::Tensor& count, const c10::optional<torch::Tensor>& out,
                     const c10::Device& device) {
  if (!out.has_value()) return count.data_ptr<int32_t>();
  check_vector(*out, torch::kInt, 1, device, "free_count_out");
  return out->data_ptr<int32_t>();
}

double default_scale(c10::optional<double> scale, int64_t head_dim) {
  return scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(head_dim));
}

void check_one_float(const torch::Tensor& t, const c10::Device& device) {
  TORCH_CHECK(t.is_cuda() && t.scalar_type() == torch::kFloat32 && t.numel() == 1 &&
                  t.device() == device,
              "k_scale and v_scale must be one-element CUDA float32 tensors");
}

}  // namespace

void b200_plan_step(torch::Tensor context_lens, torch::Tensor query_lens, torch::Tensor block_table,
                    torch::Tensor free_blocks, torch::Tensor free_count, int64_t block_size,
                    torch::Tensor query_start, torch::Tensor seq_lens, torch::Tensor positions,
                    torch::Tensor slot_mapping, c10::optional<torch::Tensor> free_count_out,
                    c10::optional<torch::Tensor> row_positions,
                    c10::optional<torch::Tensor> row_slots, c10::optional<torch::Tensor> row_lens) {
  const auto device = context_lens.device();
  const int64_t requests = context_lens.numel();
  check_vector(context_lens, torch::kInt, -1, device, "context_lens");
  check_vector(query_lens, torch::kInt, requests, device, "query_lens");
  check_table(block_table, requests, device);
  check_vector(free_blocks, torch::kInt, -1, device, "free_blocks");
  check_vector(free_count, torch::kInt, 1, device, "free_count");
  check_vector(query_start, torch::kInt, requests + 1, device, "query_start");
  check_vector(seq_lens, torch::kInt, requests, device, "seq_lens");
  check_vector(positions, torch::kInt64, -1, device, "positions");
  check_vector(slot_mapping, torch::kInt, positions.numel(), device, "slot_mapping");
  if (row_positions.has_value()) {
    check_vector(*row_positions, torch::kInt64, requests, device, "row_positions");
  }
  if (row_slots.has_value()) check_vector(*row_slots, torch::kInt, requests, device, "row_slots");
  if (row_lens.has_value()) check_vector(*row_lens, torch::kInt, requests, device, "row_lens");
  c10::cuda::CUDAGuard guard(device);
  raise_if_failed(sm120s_plan_step_rows(
      context_lens.data_ptr<int32_t>(), query_lens.data_ptr<int32_t>(),
      block_table.data_ptr<int32_t>(), table_stride(block_table), free_blocks.data_ptr<int32_t>(),
      free_count.data_ptr<int32_t>(), count_after(free_count, free_count_out, device),
      query_start.data_ptr<int32_t>(), seq_lens.data_ptr<int32_t>(), positions.data_ptr<int64_t>(),
      slot_mapping.data_ptr<int32_t>(),
      row_positions.has_value() ? row_positions->data_ptr<int64_t>() : nullptr,
      row_slots.has_value() ? row_slots->data_ptr<int32_t>() : nullptr,
      row_lens.has_value() ? row_lens->data_ptr<int32_t>() : nullptr, requests, block_table.size(1),
      free_blocks.numel(), block_size, positions.numel(), current_stream()));
}

void b200_release_blocks(torch::Tensor seq_lens, torch::Tensor finished, torch::Tensor block_table,
                         torch::Tensor free_blocks, torch::Tensor free_count, int64_t block_size,
                         int64_t shared_blocks, c10::optional<torch::Tensor> free_count_out) {
  const auto device = seq_lens.device();
  const int64_t requests = seq_lens.numel();
  check_vector(seq_lens, torch::kInt, -1, device, "seq_lens");
  check_vector(finished, torch::kBool, requests, device, "finished");
  check_table(block_table, requests, device);
  check_vector(free_blocks, torch::kInt, -1, device, "free_blocks");
  check_vector(free_count, torch::kInt, 1, device, "free_count");
  c10::cuda::CUDAGuard guard(device);
  raise_if_failed(sm120s_release_blocks(
      seq_lens.data_ptr<int32_t>(), reinterpret_cast<const uint8_t*>(finished.data_ptr<bool>()),
      block_table.data_ptr<int32_t>(), table_stride(block_table), free_blocks.data_ptr<int32_t>(),
      free_count.data_ptr<int32_t>(), count_after(free_count, free_count_out, device), requests,
      block_table.size(1), free_blocks.numel(), block_size, shared_blocks, current_stream()));
}

void b200_qk_norm_mrope_cache(torch::Tensor query, torch::Tensor key,
                              c10::optional<torch::Tensor> value, torch::Tensor query_weight,
                              torch::Tensor key_weight, torch::Tensor positions,
                              torch::Tensor cos_sin_cache, at::IntArrayRef sections,
                              c10::optional<torch::Tensor> key_cache,
                              c10::optional<torch::Tensor> value_cache,
                              c10::optional<torch::Tensor> slot_mapping,
                              c10::optional<torch::Tensor> k_scale,
                              c10::optional<torch::Tensor> v_scale, bool is_neox,
                              bool interleaved_sections, c10::string_view kv_cache_layout,
                              double epsilon, c10::optional<torch::Tensor> query_out,
                              c10::optional<torch::Tensor> key_out) {
  TORCH_CHECK(positions.is_cuda() && positions.scalar_type() == torch::kInt64 &&
                  positions.dim() == 2 && (positions.size(1) <= 1 || positions.stride(1) == 1),
              "positions must be a CUDA int64 tensor [axes, tokens] with adjacent tokens");
  TORCH_CHECK(positions.size(1) == query.size(0), "positions must have one column per token");
  TORCH_CHECK(positions.device() == query.device(), "all tensors must be on the same CUDA device");
  TORCH_CHECK(static_cast<int64_t>(sections.size()) == positions.size(0),
              "sections must have one entry per axis of positions");
  TORCH_CHECK(sections.size() >= 1 && sections.size() <= SM120S_MAX_ROPE_AXES,
              "positions must have 1 to ", SM120S_MAX_ROPE_AXES, " axes");
  sm120n_qk_cache_args a{};
  fill_qk_cache_args(a, query, key, value, query_weight, key_weight, cos_sin_cache, key_cache,
                     value_cache, slot_mapping, k_scale, v_scale, is_neox, kv_cache_layout,
                     epsilon);
  a.positions = positions.data_ptr<int64_t>();
  sm120s_mrope_args m{};
  m.struct_size = sizeof(m);
  m.axes = static_cast<int32_t>(sections.size());
  for (size_t i = 0; i < sections.size(); ++i) {
    TORCH_CHECK(sections[i] >= 0 && sections[i] <= 128, "sections must be in [0, 128]");
    m.sections[i] = static_cast<int32_t>(sections[i]);
  }
  m.interleaved_sections = interleaved_sections;
  m.position_axis_stride = positions.size(0) <= 1 ? positions.size(1) : positions.stride(0);
  auto place = [&](const c10::optional<torch::Tensor>& out, const torch::Tensor& in,
                   const char* name, void** pointer, int64_t* stride) {
    if (!out.has_value()) return;
    check_head_rows(*out, name);
    TORCH_CHECK(out->sizes() == in.sizes() && out->scalar_type() == in.scalar_type(), name,
                " must have its input's shape and dtype");
    TORCH_CHECK(out->device() == in.device(), "all tensors must be on the same CUDA device");
    *pointer = out->data_ptr();
    *stride = token_stride(*out);
  };
  place(query_out, query, "query_out", &m.query_out, &m.query_out_token_stride);
  place(key_out, key, "key_out", &m.key_out, &m.key_out_token_stride);
  c10::cuda::CUDAGuard guard(query.device());
  raise_if_failed(sm120s_qk_norm_mrope_cache(&a, &m, current_stream()));
}

void b200_prompt_attention(torch::Tensor out, torch::Tensor query, torch::Tensor key,
                           torch::Tensor value, torch::Tensor query_start,
                           c10::optional<double> scale) {
  check_head_rows(out, "out");
  check_head_rows(query, "query");
  check_head_rows(key, "key");
  check_head_rows(value, "value");
  const auto device = query.device();
  TORCH_CHECK(key.size(0) == query.size(0) && key.size(2) == query.size(2) &&
                  value.sizes() == key.sizes(),
              "key and value must be [tokens, key_heads, head_dim] for query's tokens and head_dim");
  TORCH_CHECK(out.sizes() == query.sizes(), "out shape must match query");
  TORCH_CHECK(out.scalar_type() == query.scalar_type() && key.scalar_type() == query.scalar_type() &&
                  value.scalar_type() == query.scalar_type(),
              "out, query, key and value dtypes must match");
  TORCH_CHECK(out.device() == device && key.device() == device && value.device() == device,
              "all tensors must be on the same CUDA device");
  check_vector(query_start, torch::kInt, -1, device, "query_start");
  TORCH_CHECK(query_start.numel() >= 1, "query_start must have one entry per sequence and one more");
  sm120s_prompt_args a{};
  a.struct_size = sizeof(a);
  a.dtype = dtype_code(query);
  a.tokens = query.size(0);
  a.sequences = query_start.numel() - 1;
  a.query_heads = query.size(1);
  a.key_heads = key.size(1);
  a.head_dim = query.size(2);
  a.query = query.data_ptr();
  a.query_token_stride = token_stride(query);
  a.key = key.data_ptr();
  a.key_token_stride = token_stride(key);
  a.value = value.data_ptr();
  a.value_token_stride = token_stride(value);
  a.out = out.data_ptr();
  a.out_token_stride = token_stride(out);
  a.query_start = query_start.data_ptr<int32_t>();
  a.scale = static_cast<float>(default_scale(scale, query.size(2)));
  c10::cuda::CUDAGuard guard(device);
  raise_if_failed(sm120s_prompt_attention(&a, current_stream()));
}

void b200_paged_decode_attention(torch::Tensor out, torch::Tensor query, torch::Tensor key_cache,
                                 torch::Tensor value_cache, torch::Tensor block_table,
                                 torch::Tensor seq_lens,
                                 c10::optional<torch::Tensor> prefix_blocks,
                                 c10::optional<torch::Tensor> k_scale,
                                 c10::optional<torch::Tensor> v_scale,
                                 c10::string_view kv_cache_layout, c10::optional<double> scale) {
  check_head_rows(out, "out");
  check_head_rows(query, "query");
  const auto device = query.device();
  TORCH_CHECK(out.sizes() == query.sizes() && out.scalar_type() == query.scalar_type(),
              "out must have query's shape and dtype");
  const bool nhd = kv_cache_layout == "NHD";
  TORCH_CHECK(nhd || kv_cache_layout == "HND", "kv_cache_layout must be \"NHD\" or \"HND\"");
  const auto& kc = key_cache;
  const auto& vc = value_cache;
  TORCH_CHECK(kc.is_cuda() && vc.is_cuda() && kc.dim() == 4 && vc.sizes() == kc.sizes() &&
                  vc.strides() == kc.strides() && vc.scalar_type() == kc.scalar_type(),
              "key_cache and value_cache must be 4-D CUDA tensors of one shape, stride "
              "and dtype");
  const int64_t head_axis = nhd ? 2 : 1;
  const int64_t slot_axis = nhd ? 1 : 2;
  TORCH_CHECK(kc.size(3) == query.size(2),
              nhd ? "NHD caches must be [blocks, block_size, key_heads, head_dim]"
                  : "HND caches must be [blocks, key_heads, block_size, head_dim]");
  TORCH_CHECK(kc.stride(3) == 1, "KV caches must have unit element stride");
  const bool fp8 = is_fp8_storage(kc);
  TORCH_CHECK(fp8 || kc.scalar_type() == query.scalar_type(),
              "KV caches must use the activation dtype or fp8 e4m3 (float8_e4m3fn / uint8)");
  TORCH_CHECK(out.device() == device && kc.device() == device && vc.device() == device,
              "all tensors must be on the same CUDA device");
  check_table(block_table, query.size(0), device);
  check_vector(seq_lens, torch::kInt, query.size(0), device, "seq_lens");
  sm120s_decode_args a{};
  a.struct_size = sizeof(a);
  a.dtype = dtype_code(query);
  a.cache_dtype = fp8 ? SM120N_CACHE_FP8_E4M3 : SM120N_CACHE_AUTO;
  a.batch = query.size(0);
  a.query_heads = query.size(1);
  a.key_heads = kc.size(head_axis);
  a.head_dim = query.size(2);
  a.query = query.data_ptr();
  a.query_token_stride = token_stride(query);
  a.out = out.data_ptr();
  a.out_token_stride = token_stride(out);
  a.key_cache = kc.data_ptr();
  a.value_cache = vc.data_ptr();
  a.num_blocks = kc.size(0);
  a.block_size = kc.size(slot_axis);
  a.cache_block_stride = kc.size(0) <= 1 ? 0 : kc.stride(0);
  a.cache_slot_stride = kc.size(slot_axis) <= 1 ? 0 : kc.stride(slot_axis);
  a.cache_head_stride = kc.size(head_axis) <= 1 ? 0 : kc.stride(head_axis);
  if (fp8) {
    TORCH_CHECK(k_scale.has_value() && v_scale.has_value(), "fp8 caches need k_scale and v_scale");
    check_one_float(*k_scale, device);
    check_one_float(*v_scale, device);
    a.k_scale = k_scale->data_ptr<float>();
    a.v_scale = v_scale->data_ptr<float>();
  }
  a.block_table = block_table.data_ptr<int32_t>();
  a.table_width = block_table.size(1);
  a.table_stride = table_stride(block_table);
  a.seq_lens = seq_lens.data_ptr<int32_t>();
  if (prefix_blocks.has_value() && prefix_blocks->numel() > 0) {
    check_vector(*prefix_blocks, torch::kInt, -1, device, "prefix_blocks");
    a.prefix_blocks = prefix_blocks->data_ptr<int32_t>();
    a.prefix_blocks_count = prefix_blocks->numel();
  }
  a.scale = static_cast<float>(default_scale(scale, query.size(2)));
  c10::cuda::CUDAGuard guard(device);
  size_t bytes = 0;
  raise_if_failed(sm120s_paged_decode_workspace(&a, &bytes));
  const auto workspace = at::empty({static_cast<int64_t>(bytes)},
                                   query.options().dtype(torch::kByte));
  a.workspace = workspace.data_ptr();
  a.workspace_bytes = bytes;
  raise_if_failed(sm120s_paged_decode_attention(&a, current_stream()));
}

TORCH_LIBRARY_FRAGMENT(sm120_norm_ext, m) {
  m.def(
      "plan_step_(Tensor(a!) context_lens, Tensor query_lens, Tensor(b!) block_table, "
      "Tensor free_blocks, Tensor(c!) free_count, int block_size, Tensor(d!) query_start, "
      "Tensor(e!) seq_lens, Tensor(f!) positions, Tensor(g!) slot_mapping, "
      "Tensor(h!)? free_count_out=None, Tensor(i!)? row_positions=None, "
      "Tensor(j!)? row_slots=None, Tensor(k!)? row_lens=None) -> ()");
  m.def(
      "release_blocks_(Tensor seq_lens, Tensor finished, Tensor block_table, "
      "Tensor(a!) free_blocks, Tensor(b!) free_count, int block_size, int shared_blocks=0, "
      "Tensor(c!)? free_count_out=None) -> ()");
  m.def(
      "qk_norm_mrope_cache_(Tensor(a!) query, Tensor(b!) key, Tensor? value, "
      "Tensor query_weight, Tensor key_weight, Tensor positions, Tensor cos_sin_cache, "
      "int[] sections, Tensor(c!)? key_cache=None, Tensor(d!)? value_cache=None, "
      "Tensor? slot_mapping=None, Tensor? k_scale=None, Tensor? v_scale=None, "
      "bool is_neox=True, bool interleaved_sections=False, str kv_cache_layout=\"NHD\", "
      "float epsilon=1e-6, Tensor(e!)? query_out=None, Tensor(f!)? key_out=None) -> ()");
  m.def(
      "prompt_attention(Tensor(a!) out, Tensor query, Tensor key, Tensor value, "
      "Tensor query_start, float? scale=None) -> ()");
  m.def(
      "paged_decode_attention(Tensor(a!) out, Tensor query, Tensor key_cache, "
      "Tensor value_cache, Tensor block_table, Tensor seq_lens, Tensor? prefix_blocks=None, "
      "Tensor? k_scale=None, Tensor? v_scale=None, str kv_cache_layout=\"NHD\", "
      "float? scale=None) -> ()");
}

TORCH_LIBRARY_IMPL(sm120_norm_ext, CUDA, m) {
  m.impl("plan_step_", &b200_plan_step);
  m.impl("release_blocks_", &b200_release_blocks);
  m.impl("qk_norm_mrope_cache_", &b200_qk_norm_mrope_cache);
  m.impl("prompt_attention", &b200_prompt_attention);
  m.impl("paged_decode_attention", &b200_paged_decode_attention);
}

namespace {

// nothing_looks_on(*args): true where no dispatch mode, function mode or function
// transform is active and every tensor among the arguments is a plain one, so that
// a call may go past the dispatcher unseen. (Asked from Python this took 0.5 us.)
PyObject* nothing_looks_on(PyObject*, PyObject* const* args, Py_ssize_t count) {
  if (c10::impl::TorchDispatchModeTLS::any_modes_set() || at::impl::torch_function_mode_enabled() ||
      c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode)) {
    Py_RETURN_FALSE;
  }
  for (Py_ssize_t i = 0; i < count; ++i) {
    if (!THPVariable_CheckExact(args[i]) &&
        PyObject_TypeCheck(args[i], reinterpret_cast<PyTypeObject*>(THPVariableClass))) {
      Py_RETURN_FALSE;
    }
  }
  Py_RETURN_TRUE;
}

PyMethodDef g_nothing_looks_on = {
    "nothing_looks_on", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&nothing_looks_on)),
    METH_FASTCALL, "Whether a call with these arguments may go past the dispatcher"};

}  // namespace

// The same functions on the extension module: a call through it costs the host
// about half of one through the dispatcher, which is most of a small step.
void sm120n_binding::define_serving(pybind11::module_& m) {
  using OptionalTensor = c10::optional<torch::Tensor>;
  m.attr("nothing_looks_on") =
      pybind11::reinterpret_steal<pybind11::object>(PyCFunction_New(&g_nothing_looks_on, nullptr));
  m.def("plan_step_", &b200_plan_step, "Block tables, positions and slot maps of a step (CUDA)");
  m.def("release_blocks_", &b200_release_blocks, "Blocks of finished requests back to the pool (CUDA)");
  m.def("qk_norm_mrope_cache_",
        [](torch::Tensor query, torch::Tensor key, OptionalTensor value, torch::Tensor query_weight,
           torch::Tensor key_weight, torch::Tensor positions, torch::Tensor cos_sin_cache,
           std::vector<int64_t> sections, OptionalTensor key_cache, OptionalTensor value_cache,
           OptionalTensor slot_mapping, OptionalTensor k_scale, OptionalTensor v_scale,
           bool is_neox, bool interleaved_sections, const std::string& kv_cache_layout,
           double epsilon, OptionalTensor query_out, OptionalTensor key_out) {
          b200_qk_norm_mrope_cache(query, key, value, query_weight, key_weight, positions,
                                   cos_sin_cache, sections, key_cache, value_cache, slot_mapping,
                                   k_scale, v_scale, is_neox, interleaved_sections,
                                   kv_cache_layout, epsilon, query_out, key_out);
        },
        "Q/K norm + rotation by positions with several axes + KV store (CUDA)");
  m.def("prompt_attention", &b200_prompt_attention, "Causal attention of packed prompts (CUDA)");
  m.def("paged_decode_attention",
        [](torch::Tensor out, torch::Tensor query, torch::Tensor key_cache,
           torch::Tensor value_cache, torch::Tensor block_table, torch::Tensor seq_lens,
           OptionalTensor prefix_blocks, OptionalTensor k_scale, OptionalTensor v_scale,
           const std::string& kv_cache_layout, c10::optional<double> scale) {
          b200_paged_decode_attention(out, query, key_cache, value_cache, block_table, seq_lens,
                                      prefix_blocks, k_scale, v_scale, kv_cache_layout, scale);
        },
        "Attention of one token per request over a paged cache (CUDA)");
}
