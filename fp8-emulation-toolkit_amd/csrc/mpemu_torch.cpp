// mpemu_torch.cpp -- the thin PyTorch-ROCm extension over the C ABI (include/fpemu_hip.h): the operator boundary's
// two hot calls, FPEmuOp.apply (reference mpemu/pytquant/hip/fpemu.py:43-71 -> hip/fpemu_impl.cpp:27-37) and
// quantize_tensor's per-tensor "max" branch (reference qutils.py:282-287), with the argument checks, the output
// allocation, the stream / workspace lookup and the straight-through autograd node done in C++ instead of Python +
// ctypes.  Per-call host time is what the hooked models of BASELINE configs 3 / 4 are bound by (73 casts per
// BERT-base forward, ~640 per ResNet-50 step).  No arithmetic lives here: every number comes out of libfpemu_hip.so.
//
// torch supplies device memory (empty_like through the caching allocator), the current HIP stream and autograd;
// nothing else.  There is no CPU path: a CPU tensor raises.
#include <torch/extension.h>

// torch-ROCm presents HIP devices as device type "cuda": the masquerading guard / stream types are the ones to use
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include <algorithm>
#include <cmath>
#include <mutex>
#include <numeric>
#include <unordered_map>
#include <unordered_set>
#include <vector>

#include "../../include/fpemu_hip.h"

namespace {

int dtype_id(const at::Tensor &t) {
  switch (t.scalar_type()) {
    case at::kFloat: return FPEMU_F32;
    case at::kHalf: return FPEMU_F16;
    case at::kBFloat16: return FPEMU_BF16;
    case at::kDouble: return FPEMU_F64;   // plain casts only (fpemu_cast); the library refuses it elsewhere
    default:
      TORCH_CHECK_TYPE(false, "fpemu: unsupported tensor dtype ", t.scalar_type(), " (float32, float64, float16, bfloat16 only)");
  }
}

void require_device(const at::Tensor &t, const char *what) {
  TORCH_CHECK(t.is_cuda(), "fpemu: ", what, " must live on a ROCm device (got ", t.device(), "); this build has no CPU path");
  TORCH_CHECK(t.is_contiguous(), "fpemu: ", what, " must be contiguous");  // hip/fpemu_impl.cpp:23-25
}

void check(int rc) {
  if (rc == 0) return;
  const char *msg = fpemu_last_error();
  if (rc < 0 && rc != FPEMU_EUNSUPPORTED) TORCH_CHECK_VALUE(false, msg);
  TORCH_CHECK(false, rc > 0 ? "HIP error: " : "", msg);
}

// Scratch of the per-tensor path: one 257-word buffer per (device, stream), as in _binding._stream_workspace.
// Never cached while the stream is capturing (the buffer would belong to that graph's pool).
std::mutex g_ws_mutex;
std::unordered_map<uint64_t, at::Tensor> g_ws;
constexpr int64_t kWsWords = 257;

at::Tensor stream_workspace(const at::Tensor &like, const c10::hip::HIPStreamMasqueradingAsCUDA &stream) {
  const uint64_t key = ((uint64_t)(uint8_t)like.get_device() << 56) ^ (uint64_t)(uintptr_t)stream.stream();
  {
    std::lock_guard<std::mutex> lock(g_ws_mutex);
    auto it = g_ws.find(key);
    if (it != g_ws.end()) return it->second;
  }
  at::Tensor ws = at::empty({kWsWords}, like.options().dtype(at::kInt));
  hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(stream.stream(), &st) == hipSuccess && st == hipStreamCaptureStatusNone) {
    std::lock_guard<std::mutex> lock(g_ws_mutex);
    g_ws.emplace(key, ws);
  }
  return ws;
}

at::Tensor cast_impl(const at::Tensor &input, bool inplace, int64_t fmt, int64_t rmode, double scale, uint64_t seed,
                     uint64_t offset) {
  TORCH_CHECK(input.is_cuda(), "fpemu: input must live on a ROCm device (got ", input.device(), "); this build has no CPU path");
  at::Tensor src = input.contiguous();
  at::Tensor dst = inplace ? src : at::empty_like(src);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(src.device());
  const auto stream = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(src.get_device());
  check(fpemu_cast(src.data_ptr(), dst.data_ptr(), (uint64_t)src.numel(), dtype_id(src), (int)fmt, (int)rmode, (float)scale,
                   seed, offset, 0, (void *)stream.stream()));
  if (inplace && !src.is_same(input)) input.copy_(src);  // a non-contiguous tensor cast "in place"
  return inplace ? input : dst;
}

at::Tensor quantize_per_tensor_impl(const at::Tensor &input, bool inplace, int64_t fmt, int64_t rmode, double flt_max,
                                    bool clamp, uint64_t seed, uint64_t offset, const c10::optional<at::Tensor> &ws_opt) {
  TORCH_CHECK(input.is_cuda(), "fpemu: input must live on a ROCm device (got ", input.device(), "); this build has no CPU path");
  at::Tensor src = input.contiguous();
  at::Tensor dst = inplace ? src : at::empty_like(src);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(src.device());
  const auto stream = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(src.get_device());
  // an override workspace that lives on another device is ignored, as _binding._stream_workspace does (a graph
  // captured for one GPU must not stop tensors on a second one from being quantised)
  const bool use_override = ws_opt.has_value() && ws_opt->defined() && ws_opt->is_cuda() &&
                            ws_opt->get_device() == src.get_device();
  at::Tensor ws = use_override ? *ws_opt : stream_workspace(src, stream);
  TORCH_CHECK(ws.is_cuda() && ws.scalar_type() == at::kInt && ws.numel() >= 1 && ws.is_contiguous(),
              "fpemu: workspace must be a contiguous int32 tensor");
  check(fpemu_quantize_per_tensor_ws(src.data_ptr(), dst.data_ptr(), (uint64_t)src.numel(), dtype_id(src), (int)fmt,
                                     (int)rmode, (float)flt_max, clamp ? 1 : 0, (uint32_t *)ws.data_ptr(),
                                     (uint64_t)ws.numel(), seed, offset, (void *)stream.stream()));
  if (inplace && !src.is_same(input)) input.copy_(src);
  return inplace ? input : dst;
}

// quantize_tensor's per-channel / fine-grained "max" branches (reference qutils.py:289-337: a Python loop of per-row
// casts that never goes through autograd): one launch of the rows kernel over the [rows, numel / rows] view.
// offset: first of the `rows` consecutive call offsets a loop of per-row casts would draw (stochastic modes).
at::Tensor quantize_rows(const at::Tensor &input, bool inplace, int64_t fmt, int64_t rmode, double flt_max, int64_t rows,
                         bool clamp, uint64_t seed, uint64_t offset) {
  TORCH_CHECK(input.is_cuda(), "fpemu: input must live on a ROCm device (got ", input.device(), "); this build has no CPU path");
  TORCH_CHECK(rows > 0 && input.numel() % rows == 0, "fpemu: ", input.numel(), " elements do not split into ", rows, " rows");
  at::Tensor src = input.contiguous();
  at::Tensor dst = inplace ? src : at::empty_like(src);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(src.device());
  const auto stream = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(src.get_device());
  check(fpemu_quantize_rows(src.data_ptr(), dst.data_ptr(), (uint64_t)rows, (uint64_t)(src.numel() / rows), dtype_id(src),
                            (int)fmt, (int)rmode, (float)flt_max, clamp ? 1 : 0, seed, offset, (void *)stream.stream()));
  if (inplace && !src.is_same(input)) input.copy_(src);
  return inplace ? input : dst;
}

// Straight-through estimator (reference pytquant/cpp/fpemu.py:68-71): the gradient passes unchanged.
struct CastSTE : public torch::autograd::Function<CastSTE> {
  static at::Tensor forward(torch::autograd::AutogradContext *ctx, const at::Tensor &input, bool inplace, int64_t fmt,
                            int64_t rmode, double scale, int64_t seed, int64_t offset) {
    at::Tensor out = cast_impl(input, inplace, fmt, rmode, scale, (uint64_t)seed, (uint64_t)offset);
    if (inplace) ctx->mark_dirty({input});
    return out;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *, torch::autograd::variable_list grads) {
    return {grads[0], at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

struct QuantizeSTE : public torch::autograd::Function<QuantizeSTE> {
  static at::Tensor forward(torch::autograd::AutogradContext *ctx, const at::Tensor &input, bool inplace, int64_t fmt,
                            int64_t rmode, double flt_max, bool clamp, int64_t seed, int64_t offset,
                            const c10::optional<at::Tensor> &ws) {
    at::Tensor out = quantize_per_tensor_impl(input, inplace, fmt, rmode, flt_max, clamp, (uint64_t)seed, (uint64_t)offset, ws);
    if (inplace) ctx->mark_dirty({input});
    return out;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *, torch::autograd::variable_list grads) {
    return {grads[0], at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(),
            at::Tensor()};
  }
};

bool needs_graph(const at::Tensor &t) { return at::GradMode::is_enabled() && t.requires_grad(); }

// FPEmuOp.apply(tensor, mode, inplace, scale) for a dense tensor and a plain cast (no block norm)
at::Tensor fpemu_op(const at::Tensor &input, bool inplace, int64_t fmt, int64_t rmode, double scale, uint64_t seed,
                    uint64_t offset) {
  if (needs_graph(input)) return CastSTE::apply(input, inplace, fmt, rmode, scale, (int64_t)seed, (int64_t)offset);
  return cast_impl(input, inplace, fmt, rmode, scale, seed, offset);
}

// quantize_tensor's per-tensor "max" branch: amax -> device-side scale -> cast, no host sync
at::Tensor quantize_per_tensor(const at::Tensor &input, bool inplace, int64_t fmt, int64_t rmode, double flt_max, bool clamp,
                               uint64_t seed, uint64_t offset, const c10::optional<at::Tensor> &ws) {
  if (needs_graph(input))
    return QuantizeSTE::apply(input, inplace, fmt, rmode, flt_max, clamp, (int64_t)seed, (int64_t)offset, ws);
  return quantize_per_tensor_impl(input, inplace, fmt, rmode, flt_max, clamp, seed, offset, ws);
}

// ---- operators of a language model's training step (mpemu.functional, which checks types, shapes and devices) -----------

at::Tensor scratch(uint64_t bytes, const at::Tensor &like) {
  return at::empty({(int64_t)(bytes < 16 ? 16 : bytes)}, like.options().dtype(at::kByte));
}

struct OnStream {   // the tensor's device made current, and torch's current stream there
  const c10::hip::HIPGuardMasqueradingAsCUDA guard;
  void *stream;
  explicit OnStream(const at::Tensor &t)
      : guard(t.device()), stream((void *)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.get_device()).stream()) {}
};

// Their gradients are raw kernels: a second derivative would silently be missing, so it is refused.
void once_only(const char *who) {
  TORCH_CHECK(!at::GradMode::is_enabled(), who, ": differentiable once (create_graph is not supported)");
}

// Nor do they carry forward-mode derivatives: a dual tensor's result would come out without its tangent, whatever the grad
// mode and requires_grad say.  Refused before the kernels read its address, in the backward pass too.
void reverse_only(const char *who, at::ArrayRef<at::Tensor> ts) {
  for (const at::Tensor &t : ts)
    TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(/*level=*/0).defined(), who,
                                ": forward-mode derivatives are not supported (a dual tensor came in)");
}

// A leaf that an eager autograd graph still holds has its accumulation node on the eager stream.  A backward pass captured
// into a HIP graph would make the capture wait for that stream, which ends the process when the capture ends: such a
// forward is refused.  Looked for while a capture runs only: every accumulation node behind the inputs.
void refuse_live_leaves(const char *who, std::initializer_list<at::Tensor> inputs, void *raw) {
  hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing((hipStream_t)raw, &st) != hipSuccess || st == hipStreamCaptureStatusNone) return;
  using torch::autograd::Node;
  std::unordered_set<Node *> seen;
  std::vector<std::shared_ptr<Node>> todo;
  for (const at::Tensor &t : inputs) {
    if (!t.requires_grad()) continue;
    todo.push_back(t.grad_fn() ? t.grad_fn() : torch::autograd::impl::try_get_grad_accumulator(t));
  }
  while (!todo.empty()) {
    const std::shared_ptr<Node> node = todo.back();
    todo.pop_back();
    if (!node || !seen.insert(node.get()).second) continue;
    const auto on = node->stream();
    if (node->num_outputs() == 0 && on.has_value()) {
      const c10::Stream now = c10::impl::VirtualGuardImpl(on->device_type()).getStream(on->device());
      TORCH_CHECK(*on == now, who, ": an eager autograd graph of the same leaves is still alive; drop its outputs (losses) before "
                  "a backward pass is captured");
    }
    for (const auto &edge : node->next_edges()) todo.push_back(edge.function);
  }
}

std::tuple<at::Tensor, at::Tensor> group_rows(const at::Tensor &ids_in, int64_t groups) {
  at::Tensor ids = ids_in.contiguous();
  const OnStream on(ids);
  const uint64_t n = (uint64_t)ids.numel();
  at::Tensor order = at::empty({(int64_t)n}, ids.options().dtype(at::kInt));
  at::Tensor offsets = at::empty({groups + 1}, ids.options().dtype(at::kInt));
  at::Tensor ws = scratch(fpemu_group_rows_workspace_bytes(n, (uint64_t)groups), ids);
  check(fpemu_group_rows(ids.data_ptr(), (int)ids.element_size(), n, (uint64_t)groups, (int32_t *)order.data_ptr(),
                         (int32_t *)offsets.data_ptr(), ws.data_ptr(), (uint64_t)ws.numel(), on.stream));
  return {order, offsets};
}

at::Tensor embedding_impl(const at::Tensor &ids, const at::Tensor &weight_in, double scale) {
  at::Tensor weight = weight_in.contiguous();
  const OnStream on(weight);
  std::vector<int64_t> shape = ids.sizes().vec();
  shape.push_back(weight.size(1));
  at::Tensor out = at::empty(shape, weight.options());
  check(fpemu_embedding(weight.data_ptr(), ids.data_ptr(), (int)ids.element_size(), out.data_ptr(), (uint64_t)ids.numel(),
                        (uint64_t)weight.size(0), (uint64_t)weight.size(1), dtype_id(weight), (float)scale, on.stream));
  return out;
}

struct EmbeddingOp : public torch::autograd::Function<EmbeddingOp> {
  static at::Tensor forward(torch::autograd::AutogradContext *ctx, const at::Tensor &ids, const at::Tensor &weight, double scale,
                            int64_t padding) {
    ctx->save_for_backward({ids});
    ctx->saved_data["entries"] = weight.size(0);
    ctx->saved_data["width"] = weight.size(1);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    return embedding_impl(ids, weight, scale);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
    once_only("embedding");
    reverse_only("embedding", grads[0]);
    const at::Tensor ids = ctx->get_saved_variables()[0];
    const at::Tensor dout = grads[0].contiguous();
    const OnStream on(dout);
    const int64_t entries = ctx->saved_data["entries"].toInt(), width = ctx->saved_data["width"].toInt();
    at::Tensor dweight = at::empty({entries, width}, dout.options());
    const uint64_t n = (uint64_t)ids.numel();
    at::Tensor ws = scratch(fpemu_embedding_grad_workspace_bytes(n, (uint64_t)entries, (uint64_t)width), dout);
    check(fpemu_embedding_grad(dout.data_ptr(), ids.data_ptr(), (int)ids.element_size(), dweight.data_ptr(), n,
                               (uint64_t)entries, (uint64_t)width, dtype_id(dout), (float)ctx->saved_data["scale"].toDouble(),
                               ctx->saved_data["padding"].toInt(), ws.data_ptr(), (uint64_t)ws.numel(), on.stream));
    return {at::Tensor(), dweight, at::Tensor(), at::Tensor()};
  }
};

at::Tensor embedding(const at::Tensor &ids_in, const at::Tensor &weight, double scale, int64_t padding) {
  reverse_only("embedding", weight);
  const at::Tensor ids = ids_in.contiguous();
  if (needs_graph(weight)) {
    { const OnStream on(weight); refuse_live_leaves("embedding", {weight}, on.stream); }
    return EmbeddingOp::apply(ids, weight, scale, padding);
  }
  return embedding_impl(ids, weight, scale);
}

at::Tensor grouped_impl(const at::Tensor &x, const at::Tensor &w, const at::Tensor &offsets, bool trans) {
  const OnStream on(x);
  const int64_t N = trans ? w.size(1) : w.size(2), K = trans ? w.size(2) : w.size(1);
  at::Tensor y = at::empty({x.size(0), N}, x.options());
  check(fpemu_grouped_gemm(y.data_ptr(), x.data_ptr(), w.data_ptr(), (const int32_t *)offsets.data_ptr(), x.size(0), N, K,
                           w.size(0), dtype_id(x), trans ? 1 : 0, on.stream));
  return y;
}

struct GroupedOp : public torch::autograd::Function<GroupedOp> {
  static at::Tensor forward(torch::autograd::AutogradContext *ctx, const at::Tensor &x, const at::Tensor &w, const at::Tensor &offsets,
                            bool trans) {
    ctx->save_for_backward({x, w, offsets});
    ctx->saved_data["trans"] = trans;
    return grouped_impl(x, w, offsets, trans);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
    once_only("grouped_mm");
    reverse_only("grouped_mm", grads[0]);
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &x = saved[0], &w = saved[1], &offsets = saved[2];
    const bool trans = ctx->saved_data["trans"].toBool();
    const at::Tensor dy = grads[0].contiguous();
    at::Tensor dx, dw;
    if (ctx->needs_input_grad(0)) dx = grouped_impl(dy, w, offsets, !trans);
    if (ctx->needs_input_grad(1)) {
      const OnStream on(x);
      dw = at::empty(w.sizes(), w.options());
      const at::Tensor &a = trans ? dy : x, &b = trans ? x : dy;
      check(fpemu_grouped_gemm_wgrad(dw.data_ptr(), a.data_ptr(), b.data_ptr(), (const int32_t *)offsets.data_ptr(), x.size(0),
                                     w.size(1), w.size(2), w.size(0), dtype_id(x), on.stream));
    }
    return {dx, dw, at::Tensor(), at::Tensor()};
  }
};

at::Tensor grouped_mm(const at::Tensor &x_in, const at::Tensor &weight, const at::Tensor &offsets) {
  reverse_only("grouped_mm", {x_in, weight});
  // contiguous() and transpose() are differentiable steps outside the node: its operands are what the kernels read
  const at::Tensor x = x_in.contiguous();
  at::Tensor w = weight;
  bool trans = false;
  if (!weight.is_contiguous()) {
    w = weight.transpose(1, 2);
    trans = w.is_contiguous();
    if (!trans) w = weight.contiguous();
  }
  if (needs_graph(x) || needs_graph(w)) {
    { const OnStream on(x); refuse_live_leaves("grouped_mm", {x, w}, on.stream); }
    return GroupedOp::apply(x, w, offsets, trans);
  }
  return grouped_impl(x, w, offsets, trans);
}

// What _gradients() of mpemu.functional checks, here for the whole list at once.
void check_grads(const char *who, const std::vector<at::Tensor> &ts, const char *what) {
  reverse_only(who, ts);
  for (const at::Tensor &t : ts) {
    TORCH_CHECK_TYPE(!t.is_sparse(), who, ": sparse gradients are not supported");
    const auto k = t.scalar_type();
    TORCH_CHECK_TYPE(k == at::kFloat || k == at::kHalf || k == at::kBFloat16, who, ": ", what,
                     " must be a float32, float16 or bfloat16 tensor");
    TORCH_CHECK(t.is_cuda(), who, ": tensors must live on a ROCm device (got ", t.device(), "); this build has no CPU path");
    TORCH_CHECK_VALUE(t.device() == ts[0].device(), who, ": tensors on different devices (", ts[0].device(), ", ", t.device(), ")");
  }
}

// the elements of a gradient as one run of memory, in whatever order: itself where it is one, else a copy
std::vector<at::Tensor> dense_list(const std::vector<at::Tensor> &ts) {
  std::vector<at::Tensor> d;
  d.reserve(ts.size());
  for (const at::Tensor &t : ts) d.push_back(t.is_non_overlapping_and_dense() ? t : t.contiguous());
  return d;
}

std::vector<fpemu_grad_t> grad_table(const std::vector<at::Tensor> &in, const std::vector<at::Tensor> &out) {
  std::vector<fpemu_grad_t> tab(in.size());
  for (size_t i = 0; i < in.size(); i++)
    tab[i] = {in[i].data_ptr(), out[i].data_ptr(), (uint64_t)in[i].numel(), (int32_t)dtype_id(in[i]), (int32_t)dtype_id(out[i])};
  return tab;
}

// Do tensors share bytes?  An element's bytes lie at sum stride * index + byte; two sets of such places meet where one linear
// equation has a solution within bounds.  Strides nest in practice, so the search below takes a few steps; one that takes more
// than kSearch counts as "yes".
struct Places {
  struct Term { int64_t step, most; };   // step * (0 .. most)
  static constexpr int kSearch = 20000;
  std::vector<Term> terms;
  std::vector<int64_t> reach, common;    // of the terms from k on: their largest sum, their steps' common divisor
  int left = kSearch;

  void add(int64_t step, int64_t most) {
    if (most <= 0) return;
    for (Term &t : terms)
      if (t.step == step) { t.most += most; return; }
    terms.push_back({step, most});
  }
  bool contain(int64_t target) {
    std::sort(terms.begin(), terms.end(), [](const Term &a, const Term &b) { return a.step > b.step; });
    reach.assign(terms.size() + 1, 0);
    common.assign(terms.size() + 1, 0);
    for (size_t k = terms.size(); k-- > 0;) {
      reach[k] = reach[k + 1] + terms[k].step * terms[k].most;
      common[k] = std::gcd(common[k + 1], terms[k].step);
    }
    return search(0, target);
  }
  bool search(size_t k, int64_t target) {
    if (target < 0 || target > reach[k]) return false;
    if (k == terms.size()) return true;
    if (target % common[k]) return false;
    const int64_t step = terms[k].step, over = target - reach[k + 1];
    const int64_t lo = over > 0 ? (over + step - 1) / step : 0, hi = std::min(terms[k].most, target / step);
    for (int64_t x = hi; x >= lo; x--) {
      if (--left < 0 || search(k + 1, target - x * step)) return true;
    }
    return false;
  }
};

// bytes from a tensor's first to behind its last element
int64_t extent(const at::Tensor &t) {
  if (t.is_non_overlapping_and_dense()) return t.numel() * (int64_t)t.element_size();
  int64_t last = 0;
  for (int64_t d = 0; d < t.dim(); d++) last += (t.size(d) - 1) * t.stride(d);
  return (last + 1) * (int64_t)t.element_size();
}

bool share_memory(const at::Tensor &a, const at::Tensor &b) {   // both with elements, extents that meet
  if (a.is_non_overlapping_and_dense() && b.is_non_overlapping_and_dense()) return true;
  Places p;
  const at::Tensor *const both[] = {&a, &b};
  for (const at::Tensor *t : both) {
    for (int64_t d = 0; d < t->dim(); d++)
      if (t->stride(d) > 0) p.add(t->stride(d) * (int64_t)t->element_size(), t->size(d) - 1);
    p.add(1, (int64_t)t->element_size() - 1);
  }
  return p.contain((int64_t)((uintptr_t)b.data_ptr() - (uintptr_t)a.data_ptr()) + extent(b) - 1);   // b's indices backwards
}

bool shares_with_itself(const at::Tensor &t) {
  if (t.is_non_overlapping_and_dense()) return false;
  const int64_t es = (int64_t)t.element_size();
  for (int64_t first = 0; first < t.dim(); first++) {   // two elements whose indices differ from this dimension on
    if (t.size(first) < 2) continue;
    if (t.stride(first) == 0) return true;
    Places p;
    int64_t target = es - 1 - t.stride(first) * es;
    p.add(t.stride(first) * es, t.size(first) - 2);
    p.add(1, 2 * (es - 1));
    for (int64_t d = first + 1; d < t.dim(); d++) {
      if (t.stride(d) == 0) continue;   // its own turn comes
      p.add(t.stride(d) * es, 2 * (t.size(d) - 1));
      target += t.stride(d) * es * (t.size(d) - 1);
    }
    if (p.contain(target)) return true;
  }
  return false;
}

// true where an output shares memory with another entry's gradient or output, or a gradient's elements with each other
bool overlap(const std::vector<at::Tensor> &grads, const std::vector<at::Tensor> &outs) {
  struct Span { uintptr_t lo, hi; const at::Tensor *t; bool out; };
  std::vector<Span> spans;
  spans.reserve(2 * grads.size());
  const bool in_place = &grads == &outs;
  for (size_t i = 0; i < grads.size(); i++) {
    const at::Tensor &o = outs[i], &g = grads[i];
    if (o.numel() == 0) continue;
    if (shares_with_itself(o)) return true;
    const uintptr_t lo = (uintptr_t)o.data_ptr();
    spans.push_back({lo, lo + (uintptr_t)extent(o), &o, true});
    if (in_place) continue;
    const uintptr_t in = (uintptr_t)g.data_ptr();
    if (in != lo || g.scalar_type() != o.scalar_type()) spans.push_back({in, in + (uintptr_t)extent(g), &g, false});
  }
  std::sort(spans.begin(), spans.end(), [](const Span &a, const Span &b) { return a.lo < b.lo || (a.lo == b.lo && a.hi < b.hi); });
  std::vector<const Span *> open;   // spans before this one that reach over its beginning
  uintptr_t top = 0;
  for (const Span &s : spans) {
    if (s.lo >= top) open.clear();
    for (const Span *o : open)
      if (o->hi > s.lo && (o->out || s.out) && share_memory(*o->t, *s.t)) return true;
    open.push_back(&s);
    top = std::max(top, s.hi);
  }
  return false;
}

at::Tensor norm_of(const std::vector<fpemu_grad_t> &tab, int64_t order, const at::Tensor &sum, at::Tensor *norm, const OnStream &on) {
  const uint64_t bytes = fpemu_grad_norm_workspace_bytes(tab.size());
  at::Tensor ws = at::empty({(int64_t)(bytes / 8)}, sum.options());
  check(fpemu_grad_norm_multi(tab.data(), tab.size(), (int)order, (double *)sum.data_ptr(),
                              norm ? (float *)norm->data_ptr() : nullptr, ws.data_ptr(), bytes, on.stream));
  return ws;
}

at::Tensor grad_norm(const std::vector<at::Tensor> &grads, int64_t order) {
  check_grads("grad_norm", grads, "a gradient");
  const std::vector<at::Tensor> dense = dense_list(grads);
  const OnStream on(grads[0]);
  at::Tensor sum = at::empty({1}, grads[0].options().dtype(at::kDouble));
  at::Tensor norm = at::empty({}, grads[0].options().dtype(at::kFloat));
  norm_of(grad_table(dense, dense), order, sum, &norm, on);
  return norm;
}

at::Tensor clip_grads(const std::vector<at::Tensor> &grads, const c10::optional<std::vector<at::Tensor>> &outs_or_none, double max_norm,
                      int64_t order, bool finite_only) {
  at::NoGradGuard no_grad;
  check_grads("clip_grads_", grads, "a gradient");
  const std::vector<at::Tensor> &outs = outs_or_none.has_value() ? *outs_or_none : grads;
  if (outs_or_none.has_value()) {
    TORCH_CHECK_VALUE(outs.size() == grads.size(), "clip_grads_: ", grads.size(), " gradients but ", outs.size(), " outputs");
    check_grads("clip_grads_", outs, "an output");
    for (size_t i = 0; i < grads.size(); i++)
      TORCH_CHECK_VALUE(outs[i].sizes() == grads[i].sizes() && outs[i].strides() == grads[i].strides() && outs[i].device() == grads[i].device() &&
                            (outs[i].scalar_type() == grads[i].scalar_type() || outs[i].scalar_type() == at::kFloat),
                        "clip_grads_: an output needs its gradient's shape, strides and device, and its type or float32");
  }
  TORCH_CHECK_VALUE(!overlap(grads, outs), "clip_grads_: a gradient or output shares memory with another output (or with itself)");
  const std::vector<at::Tensor> dense = dense_list(grads);
  std::vector<at::Tensor> to;
  to.reserve(grads.size());
  for (size_t i = 0; i < grads.size(); i++) {
    const bool copied = !dense[i].is_same(grads[i]), in_place = outs[i].is_same(grads[i]);
    TORCH_CHECK_VALUE(!copied || in_place, "clip_grads_: out needs gradients that fill their memory without gaps");
    to.push_back(in_place ? dense[i] : outs[i]);
  }
  const std::vector<fpemu_grad_t> tab = grad_table(dense, to);
  const OnStream on(grads[0]);
  at::Tensor sum = at::empty({1}, grads[0].options().dtype(at::kDouble));
  at::Tensor norm = at::empty({}, grads[0].options().dtype(at::kFloat));
  norm_of(tab, order, sum, finite_only ? &norm : nullptr, on);
  if (finite_only) {
    const float value = norm.item<float>();
    TORCH_CHECK(std::isfinite(value), "clip_grads_: the norm of the gradients is ", value);
  }
  check(fpemu_clip_multi(tab.data(), tab.size(), (int)order, (const double *)sum.data_ptr(), (float)max_norm,
                         (float *)norm.data_ptr(), on.stream));
  for (size_t i = 0; i < grads.size(); i++) {
    if (!dense[i].is_same(grads[i])) grads[i].copy_(dense[i]);
    else if (!outs[i].is_inference()) torch::autograd::impl::bump_version(outs[i]);   // written through its address
  }
  return norm;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "thin PyTorch-ROCm front of libfpemu_hip.so (no arithmetic here)";
  m.def("abi_version", []() { return fpemu_abi_version(); });
  m.def("fpemu_op", &fpemu_op, py::arg("input"), py::arg("inplace"), py::arg("fmt"), py::arg("rmode"), py::arg("scale"),
        py::arg("seed"), py::arg("offset"));
  m.def("quantize_per_tensor", &quantize_per_tensor, py::arg("input"), py::arg("inplace"), py::arg("fmt"), py::arg("rmode"),
        py::arg("flt_max"), py::arg("clamp"), py::arg("seed"), py::arg("offset"), py::arg("workspace") = py::none());
  m.def("quantize_rows", &quantize_rows, py::arg("input"), py::arg("inplace"), py::arg("fmt"), py::arg("rmode"),
        py::arg("flt_max"), py::arg("rows"), py::arg("clamp"), py::arg("seed"), py::arg("offset"));
  m.def("group_rows", &group_rows, py::arg("ids"), py::arg("groups"));
  m.def("embedding", &embedding, py::arg("ids"), py::arg("weight"), py::arg("scale"), py::arg("padding"));
  m.def("grouped_mm", &grouped_mm, py::arg("x"), py::arg("weight"), py::arg("offsets"));
  m.def("grad_norm", &grad_norm, py::arg("grads"), py::arg("order"));
  m.def("overlap", &overlap, py::arg("grads"), py::arg("outs"));
  m.def("clip_grads", &clip_grads, py::arg("grads"), py::arg("outs").none(true), py::arg("max_norm"), py::arg("order"),
        py::arg("finite_only"));
}
