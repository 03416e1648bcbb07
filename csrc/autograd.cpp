// Differentiable entry points of the shared-key attention operators: torch.ops.dlgm.latent_attention and
// torch.ops.dlgm.prefix_attention on GPU tensors. One operator call each way -- the forward and the backward of a small
// layer are a handful of kernels of some 10 us, less than a Python-side autograd function takes to launch them (a 2 x 128
// token layer: 239 us a training pass that way). The forward and backward operators go through the dispatcher, so
// whatever observes operators (the stream audit) sees them with their arguments.
#include <torch/all.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime.h>

using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;
using OptTensor = c10::optional<at::Tensor>;

// gemm_lt.hip
int64_t dlgm_gemm_lt(at::Tensor out, const at::Tensor& a, const at::Tensor& b, double beta, int64_t algo_index);
// transpose.hip
at::Tensor dlgm_transpose(const at::Tensor& x, const OptTensor& out, const OptTensor& rows);
// shared_attn.hip
std::tuple<at::Tensor, at::Tensor> dlgm_latent_attn_fwd(const at::Tensor& q, const at::Tensor& kv,
                                                        const at::Tensor& k_rope, double softmax_scale, bool causal,
                                                        const OptTensor& lens);
std::tuple<at::Tensor, at::Tensor, at::Tensor> dlgm_latent_attn_bwd(const at::Tensor& dout, const at::Tensor& q,
                                                                    const at::Tensor& kv, const at::Tensor& k_rope,
                                                                    const at::Tensor& out, const at::Tensor& lse,
                                                                    double softmax_scale, bool causal,
                                                                    const OptTensor& lens);

namespace {

void check_latent(const at::Tensor& q, const at::Tensor& c, const at::Tensor& k_rope, const at::Tensor& w_kv) {
  const char* op = "latent_attention";
  TORCH_CHECK(q.dim() == 4 && c.dim() == 3 && k_rope.dim() == 3 && w_kv.dim() == 2, op,
              ": q [B, S, H, nope + rope], c [B, S, r], k_rope [B, S, rope] and w_kv [H (nope + value), r] expected");
  for (const auto* t : {&c, &k_rope, &w_kv})
    TORCH_CHECK(t->device() == q.device() && t->scalar_type() == q.scalar_type(), op,
                ": all tensors must share q's device and type");
  TORCH_CHECK(q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf, op, ": bf16 or fp16 tensors expected");
  const int64_t B = q.size(0), S = q.size(1), H = q.size(2), r = w_kv.size(1);
  TORCH_CHECK(c.size(0) == B && c.size(1) == S && c.size(2) == r && k_rope.size(0) == B && k_rope.size(1) == S, op,
              ": c and k_rope must have q's batch and length, c the columns of w_kv");
  TORCH_CHECK(H > 0 && w_kv.size(0) % H == 0 && w_kv.size(0) / H > q.size(3) - k_rope.size(2), op,
              ": w_kv must have nope + value rows per head");
  TORCH_CHECK(r > 0 && r % 8 == 0, op, ": the latent size must be a positive multiple of 8, got ", r);
}

// c, w_kv as GEMM operands: rows of r values, copied only where the library's vector loads could not read them in place
at::Tensor flat(const at::Tensor& t, int64_t cols) {
  const auto x = t.reshape({-1, cols});
  const bool aligned = reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0;
  if (aligned && x.stride(1) == 1 && x.stride(0) % 8 == 0 && x.stride(0) >= cols) return x;
  return x.clone(at::MemoryFormat::Contiguous);
}

// A gradient as the kernels read it: contiguous from a 16-byte address on. Autograd may hand on a slice of a larger one
// (out was concatenated behind something), contiguous from any element on.
at::Tensor rows16(const at::Tensor& t) {
  const auto x = t.contiguous();
  return reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0 ? x : x.clone();
}

// kv = c w_kv^T by one dense GEMM, then the attention. kv is stored in the 16-bit type, rounded once from the product's fp32:
// its rows are operands of the matrix units, which take no more, and twice the bytes would be read by every tile of queries
std::tuple<at::Tensor, at::Tensor, at::Tensor> latent_attention_fwd(const at::Tensor& q, const at::Tensor& c,
                                                                    const at::Tensor& k_rope, const at::Tensor& w_kv,
                                                                    double softmax_scale, bool causal,
                                                                    const OptTensor& lens) {
  check_latent(q, c, k_rope, w_kv);
  const c10::DeviceGuard guard(q.device());
  const int64_t r = w_kv.size(1), n = w_kv.size(0);
  auto kv = at::empty({q.size(0), q.size(1), q.size(2), n / q.size(2)}, q.options());
  if (kv.numel() > 0) dlgm_gemm_lt(kv.view({-1, n}), flat(c, r), flat(w_kv, r).t(), 0.0, -1);
  auto [out, lse] = dlgm_latent_attn_fwd(q, kv, k_rope, softmax_scale, causal, lens);
  return {out, lse, kv};
}

// (dq, dc, dk_rope, dw_kv). dkv, the operand of both GEMMs, is rounded to the 16-bit type for the same reason
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> latent_attention_bwd(
    const at::Tensor& dout, const at::Tensor& q, const at::Tensor& c, const at::Tensor& k_rope, const at::Tensor& w_kv,
    const at::Tensor& kv, const at::Tensor& out, const at::Tensor& lse, double softmax_scale, bool causal,
    const OptTensor& lens) {
  check_latent(q, c, k_rope, w_kv);
  const c10::DeviceGuard guard(q.device());
  const int64_t r = w_kv.size(1), n = w_kv.size(0);
  auto [dq, dkv, dkr] = dlgm_latent_attn_bwd(rows16(dout), q, kv, k_rope, out, lse, softmax_scale, causal, lens);
  auto dc = at::empty(c.sizes(), c.options()), dw = at::empty(w_kv.sizes(), w_kv.options());
  if (dkv.numel() == 0) return {dq, dc.zero_(), dkr, dw.zero_()};
  const auto d2 = dkv.view({-1, n});
  dlgm_gemm_lt(dc.view({-1, r}), d2, flat(w_kv, r), 0.0, -1);
  // dw = dkv^T c reduces over the rows of both. The library runs it at some 1.0 PFLOP/s as it lies and at 1.27 with c's
  // columns contiguous; transposing c costs its bytes at 4.5 TB/s and a launch, so large products transpose (8192 tokens,
  // 32 x 256 columns, r 512: 102 -> 82 us)
  const auto c2 = flat(c, r);
  const double flops = 2.0 * n * (double)c2.numel();
  const bool turn = c2.size(0) % 8 == 0 && flops * (1 / 1.0e15 - 1 / 1.27e15) > 4.0 * c2.numel() / 4.5e12 + 8e-6;
  dlgm_gemm_lt(dw, d2.t(), turn ? dlgm_transpose(c2, c10::nullopt, c10::nullopt).t() : c2, 0.0, -1);
  return {dq, dc, dkr, dw};
}

template <typename F>
auto op(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}

// A backward that is captured while an eager graph of the same leaves is alive: the leaves' accumulation was then recorded
// on the default stream, which torch's engine would make wait for this node's gradients. The default stream cannot join a
// capture, and the engine ends the process over it; raised here instead, before a kernel is launched.
void check_capture(const char* op) {
  const hipStream_t stream = c10::hip::getCurrentHIPStream();
  const auto node = torch::autograd::get_current_node();
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (stream == nullptr || !node || hipStreamIsCapturing(stream, &status) != hipSuccess ||
      status != hipStreamCaptureStatusActive)
    return;
  for (const auto& edge : node->next_edges()) {
    if (!edge.is_valid()) continue;
    const auto next = edge.function->stream();
    TORCH_CHECK(!next || c10::hip::HIPStream(c10::hip::HIPStream::UNCHECKED, *next).stream() != nullptr, op,
                ": this backward is captured into a graph, but a graph recorded on the default stream holds the same inputs; "
                "release it (its outputs) first, or record it on the capture's stream");
  }
}

// Gradients recorded for a second differentiation (create_graph) with regard to the inputs raise an error there: no kernel
// has a second derivative. `all`: as many entries as the forward has arguments, the gradients first.
variable_list once(variable_list grads, const Variable& dout, const variable_list& saved, size_t all) {
  const size_t n = grads.size();
  if (at::GradMode::is_enabled()) {
    grads.push_back(dout);
    grads.insert(grads.end(), saved.begin(), saved.begin() + n);  // the inputs, in their order
    const auto inputs = static_cast<int64_t>(grads.size());
    grads = (*std::make_shared<torch::autograd::DelayedError>(
        "a gradient of latent_attention or prefix_attention cannot be differentiated again", inputs))(std::move(grads));
    grads.resize(n);
  }
  grads.resize(all);
  return grads;
}

struct LatentAttention : public torch::autograd::Function<LatentAttention> {
  static at::Tensor forward(AutogradContext* ctx, const Variable& q, const Variable& c, const Variable& k_rope,
                            const Variable& w_kv, double softmax_scale, bool causal, const OptTensor& lens) {
    at::AutoDispatchBelowADInplaceOrView below;
    static auto fwd = op<decltype(latent_attention_fwd)>("dlgm::latent_attention_fwd");
    auto [out, lse, kv] = fwd.call(q, c, k_rope, w_kv, softmax_scale, causal, lens);
    ctx->save_for_backward({q, c, k_rope, w_kv, kv, out, lse, lens.value_or(at::Tensor())});
    ctx->saved_data["scale"] = softmax_scale;
    ctx->saved_data["causal"] = causal;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list dout) {
    check_capture("latent_attention");
    const auto s = ctx->get_saved_variables();
    at::AutoDispatchBelowADInplaceOrView below;
    static auto bwd = op<decltype(latent_attention_bwd)>("dlgm::latent_attention_bwd");
    auto [dq, dc, dkr, dw] =
        bwd.call(dout[0], s[0], s[1], s[2], s[3], s[4], s[5], s[6], ctx->saved_data["scale"].toDouble(),
                 ctx->saved_data["causal"].toBool(), s[7].defined() ? OptTensor(s[7]) : c10::nullopt);
    return once({dq, dc, dkr, dw}, dout[0], s, 7);
  }
};

using PrefixFwd = std::tuple<at::Tensor, at::Tensor>(const at::Tensor&, const at::Tensor&, const at::Tensor&,
                                                     const at::Tensor&, const at::Tensor&, double, bool,
                                                     const OptTensor&, const OptTensor&);
using PrefixBwd = std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor>(
    const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
    const at::Tensor&, const at::Tensor&, double, bool, const OptTensor&, const OptTensor&);

struct PrefixAttention : public torch::autograd::Function<PrefixAttention> {
  static at::Tensor forward(AutogradContext* ctx, const Variable& q, const Variable& k, const Variable& v,
                            const Variable& prefix_k, const Variable& prefix_v, double softmax_scale, bool causal,
                            const OptTensor& lens, const OptTensor& prefix_lens) {
    at::AutoDispatchBelowADInplaceOrView below;
    static auto fwd = op<PrefixFwd>("dlgm::prefix_attn_fwd");
    auto [out, lse] = fwd.call(q, k, v, prefix_k, prefix_v, softmax_scale, causal, lens, prefix_lens);
    ctx->save_for_backward({q, k, v, prefix_k, prefix_v, out, lse, lens.value_or(at::Tensor()),
                            prefix_lens.value_or(at::Tensor())});
    ctx->saved_data["scale"] = softmax_scale;
    ctx->saved_data["causal"] = causal;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list dout) {
    check_capture("prefix_attention");
    const auto s = ctx->get_saved_variables();
    at::AutoDispatchBelowADInplaceOrView below;
    static auto bwd = op<PrefixBwd>("dlgm::prefix_attn_bwd");
    auto [dq, dk, dv, dpk, dpv] =
        bwd.call(rows16(dout[0]), s[0], s[1], s[2], s[3], s[4], s[5], s[6], ctx->saved_data["scale"].toDouble(),
                 ctx->saved_data["causal"].toBool(), s[7].defined() ? OptTensor(s[7]) : c10::nullopt,
                 s[8].defined() ? OptTensor(s[8]) : c10::nullopt);
    return once({dq, dk, dv, dpk, dpv}, dout[0], s, 9);
  }
};

at::Tensor latent_attention(const at::Tensor& q, const at::Tensor& c, const at::Tensor& k_rope, const at::Tensor& w_kv,
                            double softmax_scale, bool causal, const OptTensor& lens) {
  return LatentAttention::apply(q, c, k_rope, w_kv, softmax_scale, causal, lens);
}

at::Tensor prefix_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& prefix_k,
                            const at::Tensor& prefix_v, double softmax_scale, bool causal, const OptTensor& lens,
                            const OptTensor& prefix_lens) {
  return PrefixAttention::apply(q, k, v, prefix_k, prefix_v, softmax_scale, causal, lens, prefix_lens);
}

// without a gradient to record (torch.no_grad goes through the autograd key all the same, inference mode does not)
at::Tensor latent_attention_plain(const at::Tensor& q, const at::Tensor& c, const at::Tensor& k_rope,
                                  const at::Tensor& w_kv, double softmax_scale, bool causal, const OptTensor& lens) {
  return std::get<0>(latent_attention_fwd(q, c, k_rope, w_kv, softmax_scale, causal, lens));
}

at::Tensor prefix_attention_plain(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                  const at::Tensor& prefix_k, const at::Tensor& prefix_v, double softmax_scale,
                                  bool causal, const OptTensor& lens, const OptTensor& prefix_lens) {
  static auto fwd = op<PrefixFwd>("dlgm::prefix_attn_fwd");
  return std::get<0>(fwd.call(q, k, v, prefix_k, prefix_v, softmax_scale, causal, lens, prefix_lens));
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(dlgm, m) {
  m.def("latent_attention_fwd(Tensor q, Tensor c, Tensor k_rope, Tensor w_kv, float softmax_scale, bool causal, Tensor? lens=None) -> (Tensor, Tensor, Tensor)");
  m.def("latent_attention_bwd(Tensor dout, Tensor q, Tensor c, Tensor k_rope, Tensor w_kv, Tensor kv, Tensor out, Tensor lse, float softmax_scale, bool causal, Tensor? lens=None) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("latent_attention(Tensor q, Tensor c, Tensor k_rope, Tensor w_kv, float softmax_scale, bool causal, Tensor? lens=None) -> Tensor");
  m.def("prefix_attention(Tensor q, Tensor k, Tensor v, Tensor prefix_k, Tensor prefix_v, float softmax_scale, bool causal, Tensor? lens=None, Tensor? prefix_lens=None) -> Tensor");
}

TORCH_LIBRARY_IMPL(dlgm, CUDA, m) {
  m.impl("latent_attention_fwd", &latent_attention_fwd);
  m.impl("latent_attention_bwd", &latent_attention_bwd);
  m.impl("latent_attention", &latent_attention_plain);
  m.impl("prefix_attention", &prefix_attention_plain);
}

TORCH_LIBRARY_IMPL(dlgm, AutogradCUDA, m) {
  m.impl("latent_attention", &latent_attention);
  m.impl("prefix_attention", &prefix_attention);
}
