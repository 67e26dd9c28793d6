// The scaled embedding as a node of torch's autograd graph (module _autograd).
//
//   out = scale * W[tokens]             EmbeddingBackward:      g  -> g_W
//   g_W = scale * sums of g's rows      EmbeddingGradBackward:  gg -> the lookup in gg, padding_idx left out
//
// The host's part of a training call is most of it where the tokens are few: with
// the node and the calls in Python 64 tokens took 103 us forward and backward, 57 us
// so (torch's embedding and product 79 us, whose nodes are compiled too).
//
// Where launches are being counted or timed (set_watched), the backward is the Python
// function that reports them.
#include <atomic>

#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/extension.h>

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include "spk.h"

namespace {

using at::Tensor;
namespace ag = torch::autograd;

std::atomic<PyObject*> watched{nullptr};  // the Python backward, or null

int code_of(at::ScalarType t) {
  TORCH_CHECK(t == at::kFloat || t == at::kHalf || t == at::kBFloat16, "embedding takes fp32, fp16 and bf16");
  return t == at::kFloat ? SPK_F32 : t == at::kHalf ? SPK_F16 : SPK_BF16;
}

void check(int rc, const char* name) {
  TORCH_CHECK(rc == SPK_OK, name, " failed (", spk_status_string(rc), "): ", spk_last_error());
}

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

// what a gradient is taken of
struct Lookup {
  int64_t V = 0, padding_idx = -1;
  double scale = 1.0;
  at::ScalarType w_type = at::kFloat;
};

// More than data at a pointer: a batch of vmapped tensors, a tangent.
bool followed(const Tensor& t) { return !t.has_storage() || t._fw_grad(0).defined(); }

Tensor inside(const Tensor& tokens, int64_t V) { return tokens.ge(0).logical_and(tokens.lt(V)); }

// g_W by the sorted positions of `plan`
Tensor sum_rows(const Tensor& g, const Tensor& tokens, const Tensor& plan, const Lookup& of) {
  const int64_t n = tokens.numel(), D = g.size(-1);
  if (PyObject* f = watched.load(); f && n > 0) {
    py::gil_scoped_acquire gil;
    return py::cast<Tensor>(py::reinterpret_borrow<py::object>(f)(g, plan, of.V, of.scale, of.padding_idx, of.w_type));
  }
  at::NoGradGuard no_grad;
  const c10::cuda::CUDAGuard guard(g.device());
  const auto options = plan.options();
  if (n == 0) return at::zeros({of.V, D}, options.dtype(of.w_type));
  const Tensor rows = g.contiguous();
  Tensor gw = at::empty({of.V, D}, options.dtype(of.w_type));
  const int64_t bytes = spk_embedding_bwd_workspace_bytes(n, of.V, D);
  const Tensor workspace = at::empty({bytes}, options);
  check(spk_embedding_bwd(nullptr, rows.const_data_ptr(), code_of(rows.scalar_type()), (float)of.scale, of.padding_idx,
                          n, of.V, D, gw.mutable_data_ptr(), code_of(of.w_type), plan.mutable_data_ptr(), plan.numel(),
                          workspace.mutable_data_ptr(), bytes, stream_of(rows)),
        "spk_embedding_bwd");
  return gw;
}

// the same in torch's operations, which follow g
Tensor sum_rows_composed(const Tensor& g, const Tensor& tokens, const Lookup& of) {
  const Tensor used = inside(tokens, of.V);
  const Tensor rows = at::where(used.unsqueeze(-1), g.to(at::kFloat), 0.0);
  const Tensor gw = at::embedding_dense_backward(rows, at::where(used, tokens, 0), of.V, of.padding_idx, false);
  return (gw * of.scale).to(of.w_type);
}

std::tuple<Tensor, Tensor> embedding(const Tensor& weight, const Tensor& tokens, double scale, int64_t padding_idx,
                                     at::ScalarType out_type, int64_t bad_ever);

struct EmbeddingGradBackward : ag::Node {
  ag::SavedVariable tokens_;
  Lookup of;
  at::ScalarType g_type = at::kFloat;
  ag::variable_list apply(ag::variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    const Tensor& gg = grads[0];
    if (!gg.defined()) return {Tensor()};
    Tensor tokens = tokens_.unpack();
    if (of.padding_idx >= 0) tokens = at::where(tokens.eq(of.padding_idx), -1, tokens);
    if (followed(gg)) {
      const Tensor used = inside(tokens, of.V);
      const Tensor rows = at::embedding(gg.to(at::kFloat), at::where(used, tokens, 0));
      return {at::where(used.unsqueeze(-1), rows * of.scale, 0.0).to(g_type)};
    }
    return {std::get<0>(embedding(gg, tokens, of.scale, -1, g_type, 0))};
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    tokens_.reset_data();
  }
  std::string name() const override { return "EmbeddingGradBackward"; }
};

struct EmbeddingBackward : ag::Node {
  ag::SavedVariable tokens_, plan_;
  Lookup of;
  ag::variable_list apply(ag::variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    const Tensor& g = grads[0];
    if (!g.defined()) return {Tensor()};
    const Tensor tokens = tokens_.unpack(), plan = plan_.unpack();
    if (followed(g)) return {sum_rows_composed(g, tokens, of)};
    Tensor gw = sum_rows(g, tokens, plan, of);
    if (at::GradMode::is_enabled() && g.requires_grad()) {
      auto node = std::shared_ptr<EmbeddingGradBackward>(new EmbeddingGradBackward(), ag::deleteNode);
      node->set_next_edges(ag::collect_next_edges(g));
      node->tokens_ = ag::SavedVariable(tokens, false);
      node->of = of;
      node->g_type = g.scalar_type();
      ag::set_history(gw, node);
    }
    return {gw};
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    tokens_.reset_data();
    plan_.reset_data();
  }
  std::string name() const override { return "EmbeddingBackward"; }
};

// out, looked up with `plan` and without autograd, becomes the result of the node
Tensor attach(Tensor out, const Tensor& weight, const Tensor& tokens, const Tensor& plan, double scale,
              int64_t padding_idx) {
  auto node = std::shared_ptr<EmbeddingBackward>(new EmbeddingBackward(), ag::deleteNode);
  node->set_next_edges(ag::collect_next_edges(weight));
  node->tokens_ = ag::SavedVariable(tokens, false);
  node->plan_ = ag::SavedVariable(plan, false);
  node->of = Lookup{weight.size(0), padding_idx, scale, weight.scalar_type()};
  ag::set_history(out, node);
  return out;
}

// (out, bad) of checked arguments: weight [V, D], tokens contiguous int64, one CUDA device
std::tuple<Tensor, Tensor> embedding(const Tensor& weight, const Tensor& tokens, double scale, int64_t padding_idx,
                                     at::ScalarType out_type, int64_t bad_ever) {
  TORCH_CHECK(weight.is_cuda() && tokens.is_cuda() && weight.has_storage() && tokens.has_storage(),
              "embedding takes CUDA tensors with data");
  const c10::cuda::CUDAGuard guard(weight.device());
  const bool train = at::GradMode::is_enabled() && weight.requires_grad();
  const int64_t n = tokens.numel(), V = weight.size(0), D = weight.size(1);
  Tensor out, bad, plan;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    const auto options = weight.options();
    at::DimVector sizes(tokens.sizes());
    sizes.push_back(D);
    out = at::empty(sizes, options.dtype(out_type));
    if (train) plan = at::empty({spk_embedding_plan_bytes(n)}, options.dtype(at::kByte));
    if (n == 0) {
      bad = at::zeros({1}, options.dtype(at::kInt));
    } else {
      bad = at::empty({1}, options.dtype(at::kInt));
      const bool in_place = weight.is_contiguous() || (weight.stride(1) == 1 && weight.stride(0) >= D);
      const Tensor w = in_place ? weight : weight.contiguous();
      check(spk_embedding_fwd_watched(tokens.const_data_ptr<int64_t>(), w.const_data_ptr(), code_of(w.scalar_type()),
                                      w.is_contiguous() ? D : w.stride(0), (float)scale, n, V, D,
                                      out.mutable_data_ptr(), code_of(out_type), bad.mutable_data_ptr<int>(),
                                      reinterpret_cast<int*>(bad_ever), padding_idx,
                                      train ? plan.mutable_data_ptr() : nullptr, train ? plan.numel() : 0,
                                      stream_of(w)),
            "spk_embedding_fwd_watched");
    }
  }
  if (train) attach(out, weight, tokens, plan, scale, padding_idx);
  return {out, bad};
}

// f: the backward that reports its launches, or None.  Kept for good: a node of another thread may be at it.
void set_watched(const py::object& f) {
  watched.store(f.is_none() ? nullptr : f.inc_ref().ptr());
}

}  // namespace

PYBIND11_MODULE(_autograd, m) {
  m.def("embedding", &embedding, py::call_guard<py::gil_scoped_release>());
  m.def("attach", &attach);
  m.def("set_watched", &set_watched);
}
