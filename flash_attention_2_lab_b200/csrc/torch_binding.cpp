// PyTorch extension module `flash_attention_cuda`: the drop-in boundary.
//
// Exposes the reference's production entry point
//   tensorcore_attention_forward_production_128x128(query, key, value, causal)
// (reference csrc/bindings.cpp:63-68, :136-140) with the same argument
// meaning, the same input checks and error messages
// (csrc/tensorcore_attention.cu:2731-2823, :3035-3038), the same output
// allocation (empty_like(query), :2991) and the same stream (the current
// stream of query's device, :3084-3087). The arithmetic runs in the sm_100a
// kernel behind the C ABI in include/fa_sm100.h; this file holds no device
// code and has no fallback.
//
// The reference's older noncausal entry points (bindings.cpp:112-134) are
// kept with their own divisibility checks and routed to the same kernel.
// `attention_forward` is the general form: any sequence length, different
// query/key lengths, optional scale.

#include <torch/csrc/autograd/graph_task.h>
#include <torch/extension.h>
#include <unordered_set>
#include <vector>

#include <ATen/cuda/CUDAGraphsUtils.cuh>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <cmath>
#include <optional>

#include "fa_sm100.h"

namespace {

constexpr int64_t kHeadDimension = 64;

// Checks of validate_tensorcore_attention_inputs<kKeyTileSize>
// (reference csrc/tensorcore_attention.cu:2731-2823), same order and text.
void validate_inputs(const torch::Tensor& query, const torch::Tensor& key,
                     const torch::Tensor& value, int64_t key_tile) {
  TORCH_CHECK(query.is_cuda(), "query must be a CUDA tensor");
  TORCH_CHECK(key.is_cuda(), "key must be a CUDA tensor");
  TORCH_CHECK(value.is_cuda(), "value must be a CUDA tensor");
  TORCH_CHECK(query.device() == key.device() && query.device() == value.device(),
              "query, key, and value must be on the same device");
  TORCH_CHECK(query.scalar_type() == at::kHalf, "query must have dtype torch.float16");
  TORCH_CHECK(key.scalar_type() == at::kHalf, "key must have dtype torch.float16");
  TORCH_CHECK(value.scalar_type() == at::kHalf, "value must have dtype torch.float16");
  TORCH_CHECK(query.dim() == 4, "query must have shape [B, H, N, D]");
  TORCH_CHECK(key.dim() == 4, "key must have shape [B, H, N, D]");
  TORCH_CHECK(value.dim() == 4, "value must have shape [B, H, N, D]");
  TORCH_CHECK(query.sizes() == key.sizes(), "query and key must have identical shapes");
  TORCH_CHECK(query.sizes() == value.sizes(), "query and value must have identical shapes");
  TORCH_CHECK(query.is_contiguous(), "query must be contiguous");
  TORCH_CHECK(key.is_contiguous(), "key must be contiguous");
  TORCH_CHECK(value.is_contiguous(), "value must be contiguous");
  TORCH_CHECK(query.size(3) == kHeadDimension, "head dimension must equal 64");
  TORCH_CHECK(query.size(2) % key_tile == 0, "sequence length must be divisible by ", key_tile);
}

void check_status(int rc) {
  TORCH_CHECK(rc == FA_OK, "fa_fwd_sm100 failed (", rc, "): ", fa_last_error());
}

torch::Tensor run_fixed(const torch::Tensor& query, const torch::Tensor& key,
                        const torch::Tensor& value, bool causal, int64_t key_tile,
                        bool grid_y_check) {
  validate_inputs(query, key, value, key_tile);
  const c10::cuda::CUDAGuard device_guard(query.device());
  torch::Tensor output = torch::empty_like(query);
  const int64_t batch = query.size(0), heads = query.size(1), seq = query.size(2);
  if (batch == 0 || heads == 0 || seq == 0) return output;
  if (grid_y_check) {
    // The reference grid puts batch*heads on grid.y (:3035-3038); the
    // persistent kernel has no such limit, but the drop-in keeps the check.
    TORCH_CHECK(batch * heads <= 65535, "batch * heads exceeds CUDA grid.y limit");
  }
  const float scale = 1.0f / std::sqrt(static_cast<float>(kHeadDimension));
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(query.get_device()).stream();
  check_status(fa_fwd_sm100(query.data_ptr(), key.data_ptr(), value.data_ptr(),
                            output.data_ptr(), batch, heads, seq, causal ? 1 : 0, scale, stream));
  return output;
}

}  // namespace

torch::Tensor tensorcore_attention_forward_production_128x128(torch::Tensor query,
                                                              torch::Tensor key,
                                                              torch::Tensor value, bool causal) {
  return run_fixed(query, key, value, causal, 128, true);
}

torch::Tensor tensorcore_attention_forward(torch::Tensor query, torch::Tensor key,
                                           torch::Tensor value) {
  return run_fixed(query, key, value, false, 16, true);
}

torch::Tensor tensorcore_attention_forward_bc32(torch::Tensor query, torch::Tensor key,
                                                torch::Tensor value) {
  return run_fixed(query, key, value, false, 32, true);
}

torch::Tensor tensorcore_attention_forward_bc32_raw_pv(torch::Tensor query, torch::Tensor key,
                                                       torch::Tensor value) {
  return run_fixed(query, key, value, false, 32, true);
}

torch::Tensor tensorcore_attention_forward_bc32_raw_qk_raw_pv(torch::Tensor query,
                                                              torch::Tensor key,
                                                              torch::Tensor value) {
  return run_fixed(query, key, value, false, 32, true);
}

// General form: q [B,H,Nq,64], k/v [B,H,Nk,64], any Nq, Nk >= 1.
torch::Tensor attention_forward(torch::Tensor query, torch::Tensor key, torch::Tensor value,
                                bool causal, std::optional<double> scale) {
  TORCH_CHECK(query.is_cuda(), "query must be a CUDA tensor");
  TORCH_CHECK(key.is_cuda(), "key must be a CUDA tensor");
  TORCH_CHECK(value.is_cuda(), "value must be a CUDA tensor");
  TORCH_CHECK(query.device() == key.device() && query.device() == value.device(),
              "query, key, and value must be on the same device");
  TORCH_CHECK(query.scalar_type() == at::kHalf && key.scalar_type() == at::kHalf &&
                  value.scalar_type() == at::kHalf,
              "query, key and value must have dtype torch.float16");
  TORCH_CHECK(query.dim() == 4 && key.dim() == 4 && value.dim() == 4,
              "query, key and value must have shape [B, H, N, D]");
  TORCH_CHECK(query.size(0) == key.size(0) && query.size(0) == value.size(0),
              "query, key, and value must have the same batch size");
  TORCH_CHECK(query.size(1) == key.size(1) && query.size(1) == value.size(1),
              "query, key, and value must have the same number of heads");
  TORCH_CHECK(key.sizes() == value.sizes(), "key and value must have identical shapes");
  TORCH_CHECK(query.size(3) == kHeadDimension && key.size(3) == kHeadDimension,
              "head dimension must equal 64");
  TORCH_CHECK(query.is_contiguous() && key.is_contiguous() && value.is_contiguous(),
              "query, key and value must be contiguous");
  const c10::cuda::CUDAGuard device_guard(query.device());
  torch::Tensor output = torch::empty_like(query);
  const int64_t batch = query.size(0), heads = query.size(1);
  const int64_t nq = query.size(2), nk = key.size(2);
  if (batch == 0 || heads == 0 || nq == 0) return output;
  TORCH_CHECK(nk > 0, "key length must be positive when there are queries");
  const float s = scale.has_value() ? static_cast<float>(*scale)
                                    : 1.0f / std::sqrt(static_cast<float>(kHeadDimension));
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(query.get_device()).stream();
  check_status(fa_fwd_sm100_varlen(query.data_ptr(), key.data_ptr(), value.data_ptr(),
                                   output.data_ptr(), batch, heads, nq, nk, causal ? 1 : 0, s,
                                   stream));
  return output;
}

namespace {

// Tensors shaped like query [B, H, Nq, 64] (query, output, grad_output) and
// like key [B, H, Nk, 64] (key, value).
void check_training_inputs(const std::vector<std::pair<const char*, const torch::Tensor*>>& qs,
                           const std::vector<std::pair<const char*, const torch::Tensor*>>& ks) {
  const torch::Tensor& ref = *qs.front().second;
  TORCH_CHECK(ref.dim() == 4, "query must have shape [B, H, N, D]");
  TORCH_CHECK(ref.size(3) == kHeadDimension, "head dimension must equal 64");
  auto common = [&](const char* name, const torch::Tensor& t) {
    TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(t.device() == ref.device(), name, " must be on the same device as query");
    TORCH_CHECK(t.scalar_type() == at::kHalf, name, " must have dtype torch.float16");
    TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
  };
  for (const auto& nt : qs) {
    common(nt.first, *nt.second);
    TORCH_CHECK(nt.second->sizes() == ref.sizes(), nt.first, " must have the shape of query");
  }
  const torch::Tensor& kref = *ks.front().second;
  for (const auto& nt : ks) {
    const torch::Tensor& t = *nt.second;
    common(nt.first, t);
    TORCH_CHECK(t.dim() == 4 && t.size(0) == ref.size(0) && t.size(1) == ref.size(1) &&
                    t.size(3) == kHeadDimension,
                nt.first, " must have shape [B, H, N_kv, 64] with query's B and H");
    TORCH_CHECK(t.sizes() == kref.sizes(), nt.first, " must have the shape of key");
  }
}

}  // namespace

// Forward that also returns the row log-sum-exp [B, H, Nq] (fp32) for the
// backward; key length may differ from the query length.  No counterpart in
// the reference.
std::vector<torch::Tensor> attention_forward_lse(torch::Tensor query, torch::Tensor key,
                                                 torch::Tensor value, bool causal,
                                                 std::optional<double> scale) {
  check_training_inputs({{"query", &query}}, {{"key", &key}, {"value", &value}});
  const c10::cuda::CUDAGuard device_guard(query.device());
  torch::Tensor output = torch::empty_like(query);
  torch::Tensor lse = torch::empty({query.size(0), query.size(1), query.size(2)},
                                   query.options().dtype(at::kFloat));
  const int64_t batch = query.size(0), heads = query.size(1), nq = query.size(2),
                nk = key.size(2);
  if (batch == 0 || heads == 0 || nq == 0) return {output, lse};
  const float s = scale.has_value() ? static_cast<float>(*scale)
                                    : 1.0f / std::sqrt(static_cast<float>(kHeadDimension));
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(query.get_device()).stream();
  check_status(fa_fwd_sm100_lse(query.data_ptr(), key.data_ptr(), value.data_ptr(),
                                output.data_ptr(), lse.data_ptr<float>(), batch, heads, nq, nk,
                                causal ? 1 : 0, s, stream));
  return {output, lse};
}

// Backward of attention_forward_lse: (dq, dk, dv).  No counterpart in the
// reference.
std::vector<torch::Tensor> attention_backward(torch::Tensor query, torch::Tensor key,
                                              torch::Tensor value, torch::Tensor output,
                                              torch::Tensor grad_output, torch::Tensor lse,
                                              bool causal, std::optional<double> scale) {
  check_training_inputs({{"query", &query}, {"output", &output}, {"grad_output", &grad_output}},
                        {{"key", &key}, {"value", &value}});
  TORCH_CHECK(lse.is_cuda() && lse.device() == query.device(), "lse must be on query's device");
  TORCH_CHECK(lse.scalar_type() == at::kFloat && lse.is_contiguous() && lse.dim() == 3 &&
                  lse.size(0) == query.size(0) && lse.size(1) == query.size(1) &&
                  lse.size(2) == query.size(2),
              "lse must be a contiguous float32 tensor of shape [B, H, N_q]");
  const c10::cuda::CUDAGuard device_guard(query.device());
  torch::Tensor dq = torch::empty_like(query), dk = torch::empty_like(key),
                dv = torch::empty_like(value);
  const int64_t batch = query.size(0), heads = query.size(1), nq = query.size(2),
                nk = key.size(2);
  if (batch == 0 || heads == 0 || (nq == 0 && nk == 0)) return {dq, dk, dv};
  const float s = scale.has_value() ? static_cast<float>(*scale)
                                    : 1.0f / std::sqrt(static_cast<float>(kHeadDimension));
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(query.get_device()).stream();
  check_status(fa_bwd_sm100_varlen(query.data_ptr(), key.data_ptr(), value.data_ptr(),
                                   output.data_ptr(), grad_output.data_ptr(),
                                   lse.data_ptr<float>(), dq.data_ptr(), dk.data_ptr(),
                                   dv.data_ptr(), batch, heads, nq, nk, causal ? 1 : 0, s,
                                   stream));
  return {dq, dk, dv};
}

namespace {

// A new CUDA tensor without a trip through the dispatcher (0.5 us each, which a
// decoding step's calls of a few microseconds notice); modes that watch the
// dispatcher do not see it, the allocator's own records do.
torch::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const torch::Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}

int element_type(const torch::Tensor& t) {
  return t.scalar_type() == at::kHalf ? FA_FP16 : t.scalar_type() == at::kBFloat16 ? FA_BF16 : FA_FP32;
}

void check_rc(int rc, const char* what) {
  TORCH_CHECK(rc == FA_OK, what, " failed (", rc, "): ", fa_last_error());
}

// Tells autograd that a call has changed a tensor's values in place.
void changed(const torch::Tensor& t) {
  if (t.defined() && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// The last check of each of the calls below, so that the others need no GPU.
void check_device(const torch::Tensor& ref, const char* name,
                  std::initializer_list<std::pair<const char*, const torch::Tensor*>> others) {
  TORCH_CHECK(ref.is_cuda(), name, " must be a CUDA tensor");
  for (const auto& o : others)
    TORCH_CHECK(!o.second->defined() || o.second->device() == ref.device(), o.first,
                " must be on the device of ", name);
}

}  // namespace

namespace {

// Rotary positions of query [B, H, N, D] and key [B, H_k, N, D] (or undefined):
// contiguous results of the same shapes.
std::vector<torch::Tensor> turn(const torch::Tensor& query, const torch::Tensor& key,
                                const torch::Tensor& positions, const torch::Tensor& frequencies,
                                bool interleaved, double factor, bool inverse) {
  const torch::Tensor* sides[2] = {&query, &key};
  const char* names[2] = {"query", "key"};
  TORCH_CHECK(query.dim() == 4, "query must have shape [B, H, N, D]");
  const int64_t batch = query.size(0), tokens = query.size(2), dim = query.size(3);
  for (int i = 0; i < (key.defined() ? 2 : 1); ++i) {
    const torch::Tensor& t = *sides[i];
    TORCH_CHECK(t.dim() == 4, names[i], " must have shape [B, H, N, D]");
    TORCH_CHECK(t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16 ||
                    t.scalar_type() == at::kFloat,
                names[i], " must have dtype float16, bfloat16 or float32");
    TORCH_CHECK(t.size(3) == 1 || t.stride(3) == 1, names[i], " must have dense rows (last stride 1)");
  }
  if (key.defined()) {
    TORCH_CHECK(key.size(0) == batch && key.size(2) == tokens && key.size(3) == dim,
                "query and key must agree in batch, tokens and head dimension");
    TORCH_CHECK(key.scalar_type() == query.scalar_type(), "query and key must have the same dtype");
  }
  TORCH_CHECK(positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong,
              "positions must have dtype int32 or int64");
  const bool shared = positions.dim() == 1;
  TORCH_CHECK((shared && positions.size(0) == tokens) ||
                  (positions.dim() == 2 && positions.size(0) == batch && positions.size(1) == tokens),
              "positions must have shape [N] or [B, N]");
  TORCH_CHECK(frequencies.scalar_type() == at::kDouble && frequencies.dim() == 1 &&
                  frequencies.is_contiguous(),
              "frequencies must be a contiguous one-dimensional float64 tensor");
  TORCH_CHECK(frequencies.size(0) >= 1 && 2 * frequencies.size(0) <= dim,
              "frequencies must have 1 to D / 2 elements");
  check_device(query, "query",
               {{"key", &key}, {"positions", &positions}, {"frequencies", &frequencies}});
  const c10::cuda::CUDAGuard device_guard(query.device());
  std::vector<torch::Tensor> out;
  fa_rotary_tensor args[2] = {};
  for (int i = 0; i < (key.defined() ? 2 : 1); ++i) {
    const torch::Tensor& t = *sides[i];
    out.push_back(fresh(t.sizes(), t.scalar_type(), t));
    args[i] = {t.data_ptr(), out[i].data_ptr(), t.size(1), t.stride(0), t.stride(1), t.stride(2)};
  }
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(query.get_device()).stream();
  check_rc(fa_rotary_sm100(&args[0], key.defined() ? &args[1] : nullptr, positions.data_ptr(),
                           positions.scalar_type() == at::kLong ? 64 : 32,
                           shared ? 0 : positions.stride(0), positions.stride(shared ? 0 : 1),
                           frequencies.data_ptr<double>(), batch, tokens, dim,
                           2 * frequencies.size(0), interleaved ? 1 : 0, element_type(query),
                           static_cast<float>(factor), inverse ? 1 : 0, stream),
           "fa_rotary_sm100");
  return out;
}

std::vector<torch::Tensor> turn_differentiably(const torch::Tensor& query, const torch::Tensor& key,
                                               const torch::Tensor& positions,
                                               const torch::Tensor& frequencies, bool interleaved,
                                               double factor, bool inverse);

// In a captured backward pass the engine has the stream of every node that it
// reaches wait for the one before.  A stream of its own joins the capture that way
// and comes back at the end of the pass; the default stream cannot, nor one of
// another capture, and the attempt breaks this capture in a way that the process may
// not survive.  The gradient node of a leaf is of the stream on which the first
// eager graph that still holds it was made.
void check_captured_nodes() {
  if (at::cuda::currentStreamCaptureStatusMayInitCtx() == at::cuda::CaptureStatus::None) return;
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long here = 0, there = 0;
  C10_CUDA_CHECK(cudaStreamGetCaptureInfo(at::cuda::getCurrentCUDAStream().stream(), &status, &here));
  // the nodes that other calls of this pass have looked at are not looked at again
  thread_local int pass = -1;
  thread_local std::unordered_set<torch::autograd::Node*> seen;
  if (pass != torch::autograd::get_current_graph_task_id()) {
    pass = torch::autograd::get_current_graph_task_id();
    seen.clear();
  }
  // a pass that was asked for some tensors' gradients runs the nodes on the way to them
  const auto* run = torch::autograd::get_current_graph_task_exec_info();
  auto runs = [&](torch::autograd::Node* node) {
    if (run == nullptr || run->empty()) return true;
    const auto at = run->find(node);
    return at != run->end() && at->second.should_execute();
  };
  const auto self = torch::autograd::get_current_node();
  std::vector<torch::autograd::Node*> todo;
  if (seen.insert(self.get()).second) todo.push_back(self.get());
  while (!todo.empty()) {
    torch::autograd::Node* node = todo.back();
    todo.pop_back();
    const auto stream = node->stream();
    if (stream.has_value() && stream->device_type() == c10::DeviceType::CUDA) {
      const cudaStream_t s = c10::cuda::CUDAStream(*stream).stream();
      const bool is_default = s == nullptr || s == cudaStreamLegacy;
      status = cudaStreamCaptureStatusNone;
      if (!is_default) C10_CUDA_CHECK(cudaStreamGetCaptureInfo(s, &status, &there));
      TORCH_CHECK(!is_default && (status == cudaStreamCaptureStatusNone ||
                                  (status == cudaStreamCaptureStatusActive && there == here)),
                  "a captured backward pass reaches a tensor whose gradient node an eager graph on "
                  "the default stream, or another capture, made and still holds: drop that graph "
                  "before the capture");
    }
    for (const auto& edge : node->next_edges())
      if (edge.function && runs(edge.function.get()) && seen.insert(edge.function.get()).second)
        todo.push_back(edge.function.get());
  }
}

// A rotation's transpose turns the other way.  The nodes live in C++: one in
// Python costs a short sequence's step more than its kernels take.  One is for
// query and key, one for a query alone, as an input of a node has to be there.
template <typename Node>
struct RotaryNode : public torch::autograd::Function<Node> {
  static torch::autograd::variable_list run(torch::autograd::AutogradContext* ctx,
                                            const torch::Tensor& query, const torch::Tensor& key,
                                            const torch::Tensor& positions,
                                            const torch::Tensor& frequencies, bool interleaved,
                                            double factor, bool inverse) {
    std::vector<torch::Tensor> out = turn(query, key, positions, frequencies, interleaved, factor, inverse);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({positions, frequencies});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["factor"] = factor;
    ctx->saved_data["inverse"] = inverse;
    torch::autograd::variable_list fixed;
    if (!query.requires_grad()) fixed.push_back(out[0]);
    if (key.defined() && !key.requires_grad()) fixed.push_back(out[1]);
    ctx->mark_non_differentiable(fixed);
    return out;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    check_captured_nodes();
    const auto saved = ctx->get_saved_variables();
    torch::autograd::variable_list result(grads.size() + 5);
    std::vector<torch::Tensor> present;
    std::vector<int> at;
    for (int i = 0; i < static_cast<int>(grads.size()); ++i) {
      if (!grads[i].defined() || !ctx->needs_input_grad(i)) continue;
      // an expanded gradient has no dense rows
      const bool dense = grads[i].size(3) <= 1 || grads[i].stride(3) == 1;
      present.push_back(dense ? grads[i] : grads[i].contiguous());
      at.push_back(i);
    }
    if (present.empty()) return result;
    const auto turned = turn_differentiably(
        present[0], present.size() == 2 ? present[1] : torch::Tensor(), saved[0], saved[1],
        ctx->saved_data["interleaved"].toBool(), ctx->saved_data["factor"].toDouble(),
        !ctx->saved_data["inverse"].toBool());
    for (size_t i = 0; i < at.size(); ++i) result[at[i]] = turned[i];
    return result;
  }
};

struct RotaryBoth : public RotaryNode<RotaryBoth> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx,
                                                const torch::Tensor& query, const torch::Tensor& key,
                                                const torch::Tensor& positions,
                                                const torch::Tensor& frequencies, bool interleaved,
                                                double factor, bool inverse) {
    return run(ctx, query, key, positions, frequencies, interleaved, factor, inverse);
  }
};

struct RotaryOne : public RotaryNode<RotaryOne> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx,
                                                const torch::Tensor& query,
                                                const torch::Tensor& positions,
                                                const torch::Tensor& frequencies, bool interleaved,
                                                double factor, bool inverse) {
    return run(ctx, query, torch::Tensor(), positions, frequencies, interleaved, factor, inverse);
  }
};

std::vector<torch::Tensor> turn_differentiably(const torch::Tensor& query, const torch::Tensor& key,
                                               const torch::Tensor& positions,
                                               const torch::Tensor& frequencies, bool interleaved,
                                               double factor, bool inverse) {
  if (at::GradMode::is_enabled() && (query.requires_grad() || (key.defined() && key.requires_grad())))
    return key.defined()
               ? RotaryBoth::apply(query, key, positions, frequencies, interleaved, factor, inverse)
               : RotaryOne::apply(query, positions, frequencies, interleaved, factor, inverse);
  return turn(query, key, positions, frequencies, interleaved, factor, inverse);
}

}  // namespace

// (query', key'), key' None without a key; differentiable in both.  No
// counterpart in the reference.
std::tuple<torch::Tensor, std::optional<torch::Tensor>> rotary(
    torch::Tensor query, std::optional<torch::Tensor> key, torch::Tensor positions,
    torch::Tensor frequencies, bool interleaved, double factor, bool inverse) {
  // a tangent would be lost without a word where no gradient is asked for
  TORCH_CHECK(!query._fw_grad(0).defined() && !(key.has_value() && key->_fw_grad(0).defined()),
              "apply_rotary has no forward mode");
  const auto out = turn_differentiably(query, key.value_or(torch::Tensor()), positions, frequencies,
                                       interleaved, factor, inverse);
  return {out[0], out.size() == 2 ? std::optional<torch::Tensor>(out[1]) : std::nullopt};
}

namespace {

void check_int32(const torch::Tensor& t, const char* name, std::vector<int64_t> sizes,
                 const char* shape) {
  TORCH_CHECK(t.scalar_type() == at::kInt, name, " must have dtype torch.int32");
  TORCH_CHECK(t.sizes() == at::IntArrayRef(sizes), name, " must have shape ", shape);
}

// Pages, table and lengths of a cache; v_pages may be undefined where a call
// reads keys only.
fa_paged_cache paged_cache(const torch::Tensor& k_pages, const torch::Tensor& v_pages,
                           const torch::Tensor& block_table, const torch::Tensor& lengths) {
  TORCH_CHECK(k_pages.dim() == 4, "k_pages must have shape [pages, H_kv, page_size, D]");
  TORCH_CHECK(k_pages.scalar_type() == at::kHalf || k_pages.scalar_type() == at::kBFloat16,
              "k_pages must have dtype torch.float16 or torch.bfloat16");
  TORCH_CHECK(k_pages.is_contiguous(), "k_pages must be contiguous");
  TORCH_CHECK(k_pages.size(3) == 64 || k_pages.size(3) == 128, "head dimension must be 64 or 128");
  TORCH_CHECK(k_pages.size(2) >= 16 && k_pages.size(2) % 16 == 0,
              "page size must be a positive multiple of 16");
  if (v_pages.defined()) {
    TORCH_CHECK(v_pages.sizes() == k_pages.sizes(), "k_pages and v_pages must have identical shapes");
    TORCH_CHECK(v_pages.scalar_type() == k_pages.scalar_type(),
                "k_pages and v_pages must have the same dtype");
    TORCH_CHECK(v_pages.is_contiguous(), "v_pages must be contiguous");
  }
  TORCH_CHECK(block_table.scalar_type() == at::kInt, "block_table must have dtype torch.int32");
  TORCH_CHECK(block_table.dim() == 2, "block_table must have shape [B, pages of a sequence]");
  TORCH_CHECK(block_table.size(1) <= 1 || block_table.stride(1) == 1,
              "block_table must have dense rows (last stride 1)");
  check_int32(lengths, "lengths", {block_table.size(0)}, "[B]");
  TORCH_CHECK(lengths.is_contiguous(), "lengths must be contiguous");
  return {k_pages.data_ptr(),
          v_pages.defined() ? v_pages.data_ptr() : nullptr,
          block_table.data_ptr<int>(),
          lengths.data_ptr<int>(),
          block_table.stride(0),
          block_table.size(0),
          k_pages.size(1),
          k_pages.size(0),
          k_pages.size(2),
          block_table.size(1),
          k_pages.size(3)};
}

// Per-slot values of a cache: [B, H_kv, pages of a sequence * page_size].
void check_slots(const torch::Tensor& t, const char* name, at::ScalarType type,
                 const fa_paged_cache& c) {
  TORCH_CHECK(t.scalar_type() == type, name, " must have dtype ",
              type == at::kFloat ? "torch.float32" : "torch.int32");
  TORCH_CHECK(t.dim() == 3 && t.size(0) == c.batch && t.size(1) == c.kv_heads &&
                  t.size(2) == c.max_pages * c.page_size,
              name, " must have shape [B, H_kv, slots of a sequence]");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}

// A tensor [B, H, N, D] as rows that the kernels can load 16 bytes at a time:
// itself, or a copy where its strides or address do not allow that.
struct Rows {
  torch::Tensor held;
  fa_rows rows;
};

Rows aligned_rows(const torch::Tensor& t) {
  auto fits = [](const torch::Tensor& x) {
    bool ok = x.stride(3) == 1 && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0;
    for (int i = 0; i < 3; ++i) ok = ok && (x.size(i) <= 1 || x.stride(i) % 8 == 0);
    return ok;
  };
  Rows r;
  r.held = fits(t) ? t : t.clone(at::MemoryFormat::Contiguous);
  auto stride = [&](int i) { return r.held.size(i) <= 1 ? int64_t{0} : r.held.stride(i); };
  r.rows = {r.held.data_ptr(), stride(0), stride(1), stride(2)};
  return r;
}

void check_rows(const torch::Tensor& t, const char* name, const torch::Tensor& k_pages, int64_t batch,
                int64_t heads, int64_t rows, const char* shape) {
  TORCH_CHECK(t.scalar_type() == k_pages.scalar_type(), name, " must have the dtype of k_pages");
  TORCH_CHECK(t.dim() == 4 && t.size(0) == batch && (heads < 0 || t.size(1) == heads) &&
                  (rows < 0 || t.size(2) == rows) && t.size(3) == k_pages.size(3),
              name, " must have shape ", shape);
}

void check_queries(const torch::Tensor& query, const torch::Tensor& k_pages, int64_t batch) {
  check_rows(query, "query", k_pages, batch, -1, -1, "[B, H, T, D] with the cache's B and D");
  TORCH_CHECK(query.size(1) == 0 || (k_pages.size(1) > 0 && query.size(1) % k_pages.size(1) == 0),
              "query heads must be a multiple of the cache's heads");
}

float scale_of(std::optional<double> scale, const torch::Tensor& k_pages) {
  return scale.has_value() ? static_cast<float>(*scale)
                           : 1.0f / std::sqrt(static_cast<float>(k_pages.size(3)));
}

const torch::Tensor& or_undefined(const std::optional<torch::Tensor>& t) {
  static const torch::Tensor none;
  return t.has_value() ? *t : none;
}

template <typename V>
V* data_or_null(const torch::Tensor& t) {
  return t.defined() ? t.data_ptr<V>() : nullptr;
}

torch::Tensor workspace_on(const torch::Tensor& ref, int64_t bytes, const char* what) {
  TORCH_CHECK(bytes >= 0, what, " failed: ", fa_last_error());
  return fresh({bytes > 0 ? bytes : 1}, at::kByte, ref);
}

}  // namespace

// Appends rows to a paged cache; returns the new lengths.  No counterpart in
// the reference.
torch::Tensor append_to_cache(torch::Tensor key, torch::Tensor value, torch::Tensor k_pages,
                              torch::Tensor v_pages, torch::Tensor block_table,
                              torch::Tensor lengths, std::optional<torch::Tensor> path_,
                              std::optional<torch::Tensor> counts_,
                              std::optional<torch::Tensor> weights_,
                              std::optional<torch::Tensor> positions_,
                              std::optional<torch::Tensor> new_positions_) {
  const torch::Tensor &path = or_undefined(path_), &counts = or_undefined(counts_),
                      &weights = or_undefined(weights_), &positions = or_undefined(positions_),
                      &new_positions = or_undefined(new_positions_);
  const fa_paged_cache cache = paged_cache(k_pages, v_pages, block_table, lengths);
  check_rows(key, "key", k_pages, cache.batch, cache.kv_heads, -1,
             "[B, H_kv, N, D] with the cache's B, H_kv and D");
  check_rows(value, "value", k_pages, cache.batch, cache.kv_heads, key.size(2), "that of key");
  const int64_t rows = key.size(2);
  if (path.defined()) check_int32(path, "path", {cache.batch, rows}, "[B, N]");
  if (counts.defined()) check_int32(counts, "counts", {cache.batch}, "[B]");
  if (weights.defined()) check_slots(weights, "weights", at::kFloat, cache);
  if (positions.defined()) check_slots(positions, "positions", at::kInt, cache);
  TORCH_CHECK(positions.defined() == new_positions.defined(),
              "positions and new_positions go together");
  if (new_positions.defined()) check_int32(new_positions, "new_positions", {cache.batch, rows}, "[B, N]");
  for (const torch::Tensor* t : {&path, &counts, &new_positions})
    TORCH_CHECK(!t->defined() || t->is_contiguous(), "path, counts and new_positions must be contiguous");
  check_device(k_pages, "k_pages",
               {{"v_pages", &v_pages}, {"block_table", &block_table}, {"lengths", &lengths},
                {"key", &key}, {"value", &value}, {"path", &path}, {"counts", &counts},
                {"weights", &weights}, {"positions", &positions}, {"new_positions", &new_positions}});
  const c10::cuda::CUDAGuard device_guard(k_pages.device());
  torch::Tensor out = fresh(lengths.sizes(), at::kInt, lengths);
  if (cache.batch == 0) return out;
  const Rows k = aligned_rows(key), v = aligned_rows(value);
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(k_pages.get_device()).stream();
  check_rc(fa_cache_append_sm100(&cache, &k.rows, &v.rows, rows, data_or_null<int>(path),
                                 data_or_null<int>(counts), data_or_null<float>(weights),
                                 data_or_null<int>(positions), data_or_null<int>(new_positions),
                                 out.data_ptr<int>(), stream),
           "fa_cache_append_sm100");
  changed(k_pages);
  changed(v_pages);
  changed(weights);
  changed(positions);
  return out;
}

// Evicts by weight: (weights, positions, lengths) of the smaller cache; the
// pages change in place.  No counterpart in the reference.
std::vector<torch::Tensor> evict_from_cache(torch::Tensor k_pages, torch::Tensor v_pages,
                                            torch::Tensor block_table, torch::Tensor lengths,
                                            torch::Tensor weights, torch::Tensor positions,
                                            int64_t budget, int64_t recent, int64_t sinks) {
  const fa_paged_cache cache = paged_cache(k_pages, v_pages, block_table, lengths);
  check_slots(weights, "weights", at::kFloat, cache);
  check_slots(positions, "positions", at::kInt, cache);
  TORCH_CHECK(budget >= 1, "budget must be positive");
  TORCH_CHECK(recent >= 0 && sinks >= 0 && recent <= budget && sinks <= budget - recent,
              "recent and sinks must not be negative, and the budget must hold both");
  check_device(k_pages, "k_pages",
               {{"v_pages", &v_pages}, {"block_table", &block_table}, {"lengths", &lengths},
                {"weights", &weights}, {"positions", &positions}});
  const c10::cuda::CUDAGuard device_guard(k_pages.device());
  torch::Tensor new_weights = fresh(weights.sizes(), at::kFloat, weights),
                new_positions = fresh(positions.sizes(), at::kInt, positions),
                new_lengths = fresh(lengths.sizes(), at::kInt, lengths);
  std::vector<torch::Tensor> out = {new_weights, new_positions, new_lengths};
  if (cache.batch == 0) return out;
  auto aligned = [](const torch::Tensor& t) {
    return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 ? t : t.clone();
  };
  weights = aligned(weights);
  positions = aligned(positions);
  const int64_t bytes = fa_cache_evict_workspace(&cache, budget);
  torch::Tensor ws = workspace_on(k_pages, bytes, "fa_cache_evict_workspace");
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(k_pages.get_device()).stream();
  check_rc(fa_cache_evict_sm100(&cache, weights.data_ptr<float>(), positions.data_ptr<int>(),
                                new_weights.data_ptr<float>(), new_positions.data_ptr<int>(),
                                new_lengths.data_ptr<int>(), budget, recent, sinks, ws.data_ptr(),
                                bytes, stream),
           "fa_cache_evict_sm100");
  changed(k_pages);
  changed(v_pages);
  return out;
}

// Attention of a tree's queries over a cache and the tree: (out, lse).  No
// counterpart in the reference.
std::vector<torch::Tensor> tree_attention(torch::Tensor query, torch::Tensor k_pages,
                                          torch::Tensor v_pages, torch::Tensor block_table,
                                          torch::Tensor lengths,
                                          std::optional<torch::Tensor> k_tree_,
                                          std::optional<torch::Tensor> v_tree_,
                                          std::optional<torch::Tensor> tree_mask_,
                                          std::optional<torch::Tensor> tree_sizes_,
                                          std::optional<double> scale) {
  const torch::Tensor &k_tree = or_undefined(k_tree_), &v_tree = or_undefined(v_tree_),
                      &mask = or_undefined(tree_mask_), &sizes = or_undefined(tree_sizes_);
  const fa_paged_cache cache = paged_cache(k_pages, v_pages, block_table, lengths);
  check_queries(query, k_pages, cache.batch);
  const int64_t batch = cache.batch, heads = query.size(1), tokens = query.size(2);
  TORCH_CHECK(k_tree.defined() == v_tree.defined(), "k_tree and v_tree go together");
  if (k_tree.defined()) {
    check_rows(k_tree, "k_tree", k_pages, batch, cache.kv_heads, tokens, "[B, H_kv, T, D]");
    check_rows(v_tree, "v_tree", k_pages, batch, cache.kv_heads, tokens, "[B, H_kv, T, D]");
  }
  if (mask.defined()) {
    TORCH_CHECK(k_tree.defined(), "tree_mask needs k_tree and v_tree");
    TORCH_CHECK(mask.scalar_type() == at::kBool, "tree_mask must have dtype torch.bool");
    TORCH_CHECK((mask.dim() == 2 || (mask.dim() == 3 && mask.size(0) == batch)) &&
                    mask.size(-1) == tokens && mask.size(-2) == tokens,
                "tree_mask must have shape [T, T] or [B, T, T]");
    TORCH_CHECK(tokens <= 1 || mask.stride(-1) == 1, "tree_mask must have dense rows (last stride 1)");
  }
  if (sizes.defined()) {
    check_int32(sizes, "tree_sizes", {batch}, "[B]");
    TORCH_CHECK(sizes.is_contiguous(), "tree_sizes must be contiguous");
  }
  check_device(query, "query",
               {{"k_pages", &k_pages}, {"v_pages", &v_pages}, {"block_table", &block_table},
                {"lengths", &lengths}, {"k_tree", &k_tree}, {"v_tree", &v_tree},
                {"tree_mask", &mask}, {"tree_sizes", &sizes}});
  const c10::cuda::CUDAGuard device_guard(query.device());
  torch::Tensor out = fresh({batch, heads, tokens, query.size(3)}, query.scalar_type(), query);
  torch::Tensor lse = fresh({batch, heads, tokens}, at::kFloat, query);
  if (batch == 0 || heads == 0 || tokens == 0) return {out, lse};
  const Rows q = aligned_rows(query);
  Rows kt, vt;
  if (k_tree.defined()) {
    kt = aligned_rows(k_tree);
    vt = aligned_rows(v_tree);
  }
  const int64_t bytes = fa_tree_attention_workspace(&cache, heads, tokens, k_tree.defined() ? 1 : 0);
  torch::Tensor ws = workspace_on(query, bytes, "fa_tree_attention_workspace");
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(query.get_device()).stream();
  check_rc(fa_tree_attention_sm100(
               &cache, &q.rows, heads, tokens, k_tree.defined() ? &kt.rows : nullptr,
               k_tree.defined() ? &vt.rows : nullptr,
               mask.defined() ? static_cast<const unsigned char*>(mask.data_ptr()) : nullptr,
               mask.defined() && mask.dim() == 3 ? mask.stride(0) : 0,
               mask.defined() ? mask.stride(-2) : 0, data_or_null<int>(sizes), element_type(query),
               scale_of(scale, k_pages), out.data_ptr(), lse.data_ptr<float>(), ws.data_ptr(), bytes,
               stream),
           "fa_tree_attention_sm100");
  return {out, lse};
}

// Adds the attention weight of the cached slots to `weights`, in place.  No
// counterpart in the reference.
torch::Tensor accumulate_attention_weight(torch::Tensor weights, torch::Tensor query,
                                          torch::Tensor k_pages, torch::Tensor block_table,
                                          torch::Tensor lengths, torch::Tensor lse,
                                          std::optional<double> scale) {
  const fa_paged_cache cache = paged_cache(k_pages, torch::Tensor(), block_table, lengths);
  check_slots(weights, "weights", at::kFloat, cache);
  check_queries(query, k_pages, cache.batch);
  TORCH_CHECK(lse.scalar_type() == at::kFloat && lse.dim() == 3 && lse.size(0) == query.size(0) &&
                  lse.size(1) == query.size(1) && lse.size(2) == query.size(2) && lse.is_contiguous(),
              "lse must be a contiguous float32 tensor of shape [B, H, T]");
  check_device(query, "query",
               {{"weights", &weights}, {"k_pages", &k_pages}, {"block_table", &block_table},
                {"lengths", &lengths}, {"lse", &lse}});
  const c10::cuda::CUDAGuard device_guard(query.device());
  if (query.numel() == 0 || weights.numel() == 0) return weights;
  const Rows q = aligned_rows(query);
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(query.get_device()).stream();
  check_rc(fa_attention_weight_sm100(&cache, &q.rows, query.size(1), query.size(2),
                                     lse.data_ptr<float>(), weights.data_ptr<float>(),
                                     element_type(query), scale_of(scale, k_pages), stream),
           "fa_attention_weight_sm100");
  changed(weights);
  return weights;
}

PYBIND11_MODULE(TORCH_EXTENSION_NAME, module) {
  module.def("append_to_cache", &append_to_cache, "Rows into a paged cache (sm_100a)", py::arg("key"),
             py::arg("value"), py::arg("k_pages"), py::arg("v_pages"), py::arg("block_table"),
             py::arg("lengths"), py::arg("path") = py::none(), py::arg("counts") = py::none(),
             py::arg("weights") = py::none(), py::arg("positions") = py::none(),
             py::arg("new_positions") = py::none());
  module.def("evict_from_cache", &evict_from_cache, "Eviction by attention weight (sm_100a)",
             py::arg("k_pages"), py::arg("v_pages"), py::arg("block_table"), py::arg("lengths"),
             py::arg("weights"), py::arg("positions"), py::arg("budget"), py::arg("recent") = 0,
             py::arg("sinks") = 0);
  module.def("tree_attention", &tree_attention, "Attention of a tree over a paged cache (sm_100a)",
             py::arg("query"), py::arg("k_pages"), py::arg("v_pages"), py::arg("block_table"),
             py::arg("lengths"), py::arg("k_tree") = py::none(), py::arg("v_tree") = py::none(),
             py::arg("tree_mask") = py::none(), py::arg("tree_sizes") = py::none(),
             py::arg("scale") = py::none());
  module.def("accumulate_attention_weight", &accumulate_attention_weight,
             "Attention weight of cached keys, added in place (sm_100a)", py::arg("weights"),
             py::arg("query"), py::arg("k_pages"), py::arg("block_table"), py::arg("lengths"),
             py::arg("lse"), py::arg("scale") = py::none());
  module.def("rotary", &rotary, "Rotary positions of queries and keys (sm_100a)", py::arg("query"),
             py::arg("key"), py::arg("positions"), py::arg("frequencies"),
             py::arg("interleaved") = false, py::arg("factor") = 1.0, py::arg("inverse") = false);
  module.def("attention_forward_lse", &attention_forward_lse,
             "Attention forward returning (output, row log-sum-exp) (sm_100a)",
             py::arg("query"), py::arg("key"), py::arg("value"), py::arg("causal") = false,
             py::arg("scale") = py::none());
  module.def("attention_backward", &attention_backward,
             "Attention backward: (dq, dk, dv) (sm_100a)", py::arg("query"), py::arg("key"),
             py::arg("value"), py::arg("output"), py::arg("grad_output"), py::arg("lse"),
             py::arg("causal") = false, py::arg("scale") = py::none());
  module.def("tensorcore_attention_forward_production_128x128",
             &tensorcore_attention_forward_production_128x128, "Production kernel",
             py::arg("query"), py::arg("key"), py::arg("value"), py::arg("causal"));
  module.def("tensorcore_attention_forward", &tensorcore_attention_forward,
             "Fused FP16 Tensor Core attention forward pass");
  module.def("tensorcore_attention_forward_bc32", &tensorcore_attention_forward_bc32,
             "Fused FP16 Tensor core attention forward with Bc=32");
  module.def("tensorcore_attention_forward_bc32_raw_pv", &tensorcore_attention_forward_bc32_raw_pv,
             "Fused FP16 Tensor Core attention with raw MMA PV");
  module.def("tensorcore_attention_forward_bc32_raw_qk_raw_pv",
             &tensorcore_attention_forward_bc32_raw_qk_raw_pv,
             "Fused FP16 Tensor Core attention with raw MMA QK");
  module.def("attention_forward", &attention_forward,
             "Attention forward, any sequence lengths (sm_100a)", py::arg("query"),
             py::arg("key"), py::arg("value"), py::arg("causal") = false,
             py::arg("scale") = py::none());
}
