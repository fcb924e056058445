// torch-tensor entry points of the operators over a vocabulary: a teacher's top
// log-probabilities, the distillation loss on them, and the embedding with its
// gradient.  As in cache_bindings.cpp, each checks its arguments completely,
// whatever device they are on, then launches on the current stream of their
// device; for CPU tensors it returns None and the caller computes on the host.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <pybind11/pybind11.h>
#include <torch/extension.h>

#include <climits>
#include <cmath>
#include <optional>
#include <tuple>

#include "kernels.h"
#include "op_checks.hpp"
#include "turbol/common.hpp"

namespace py = pybind11;
using namespace turbol::checks;

namespace {

constexpr int64_t kMaxVocab = 1 << 20;
constexpr int64_t kMaxList = 256;
constexpr int64_t kMaxTokens = 1 << 30, kMaxColumns = 1 << 24;  // of an embedding

// [R, V] rows with a contiguous last dimension.
int rows2(const at::Tensor& t, const char* op, const char* m) {
  chk(t.dim() == 2 && (t.size(1) <= 1 || t.stride(1) == 1) && t.size(0) <= INT_MAX, op, m);
  return type_of(t, op);
}
// Whether a [R, V] view to be written names each element once.
bool rows2_distinct(const at::Tensor& t) { return t.size(0) <= 1 || t.numel() == 0 || t.stride(0) >= t.size(1); }

void vocab_of(const at::Tensor& logits, const char* op) {
  chk(logits.size(1) >= 1 && logits.size(1) <= kMaxVocab, op, "a vocabulary of 1 to 2^20");
}
void temperature_of(double t, const char* op) {
  chk(t >= 1e-6 && t <= 1e6, op, "a temperature from 1e-6 to 1e6");
}

using TopK = std::optional<std::tuple<at::Tensor, at::Tensor, at::Tensor>>;

TopK topk_logprobs(const at::Tensor& logits, int64_t k, double temperature) {
  const char* op = "topk_logprobs";
  TbTopkLogprobsArgs a{};
  a.dtype = rows2(logits, op, "logits are [R, V] with a contiguous last dimension");
  vocab_of(logits, op);
  chk(k >= 1 && k <= kMaxList && k <= logits.size(1), op, "k from 1 to 256 and to the vocabulary");
  temperature_of(temperature, op);
  no_grad({&logits}, op);
  if (!logits.is_cuda()) return std::nullopt;
  c10::DeviceGuard guard(logits.device());
  const int64_t R = logits.size(0);
  at::Tensor logp = at::empty({R, k}, logits.options().dtype(at::kFloat));
  at::Tensor ids = at::empty({R, k}, logits.options().dtype(at::kInt));
  at::Tensor lse = at::empty({R}, logp.options());
  if (R > 0) {
    a.logits = logits.data_ptr();
    a.ld = logits.stride(0);
    a.R = static_cast<int>(R);
    a.V = static_cast<int>(logits.size(1));
    a.k = static_cast<int>(k);
    a.temperature = temperature;
    a.logp = logp.data_ptr<float>();
    a.ids = ids.data_ptr<int>();
    a.lse = lse.data_ptr<float>();
    cuda_ok(tb_topk_logprobs(&a, turbol::StreamFor(logits)), op);
  }
  return std::make_tuple(logp, ids, lse);
}

int distill_kind(const std::string& kind, bool rest, const char* op) {
  chk(kind == "forward" || kind == "reverse", op, "kind is 'forward' or 'reverse'");
  chk(rest || kind == "forward", op, "kind 'reverse' needs rest=True");
  return kind == "reverse" ? TB_DISTILL_REVERSE : rest ? TB_DISTILL_FORWARD_REST : TB_DISTILL_FORWARD;
}

void per_row(const Opt& t, int64_t R, at::ScalarType type, const at::Device& dev, const char* op, const char* m) {
  if (!t) return;
  chk(t->scalar_type() == type && t->dim() == 1 && t->size(0) == R && t->is_contiguous(), op, m);
  chk(t->device() == dev, op, "all tensors on one device");
}

// Checks everything that the loss and its gradient share, and fills the arguments.
TbDistillArgs distill_args(const at::Tensor& logits, const at::Tensor& ids, const at::Tensor& logprobs, const Opt& weight,
                           const Opt& target, const Opt& target_weight, int kind, double temperature, const Opt& error,
                           const char* op) {
  TbDistillArgs a{};
  a.dtype = rows2(logits, op, "logits are [R, V] with a contiguous last dimension");
  vocab_of(logits, op);
  const int64_t R = logits.size(0);
  const at::Device dev = logits.device();
  chk(ids.scalar_type() == at::kInt && ids.dim() == 2 && ids.size(0) == R && ids.is_contiguous(), op,
      "ids are a contiguous int32 [R, K]");
  chk(ids.size(1) >= 1 && ids.size(1) <= kMaxList, op, "a list of 1 to 256 ids");
  chk(logprobs.scalar_type() == at::kFloat && logprobs.sizes() == ids.sizes() && logprobs.is_contiguous(), op,
      "logprobs are a contiguous fp32 [R, K]");
  chk(ids.device() == dev && logprobs.device() == dev, op, "all tensors on one device");
  no_grad({&logprobs}, op, "the teacher's list");
  per_row(weight, R, at::kFloat, dev, op, "weight is a contiguous fp32 [R]");
  per_row(target, R, at::kInt, dev, op, "target is a contiguous int32 [R]");
  per_row(target_weight, R, at::kFloat, dev, op, "target_weight is a contiguous fp32 [R]");
  chk(target || !target_weight, op, "target_weight needs target");
  if (weight) no_grad({&*weight}, op, "weight");
  if (target_weight) no_grad({&*target_weight}, op, "target_weight");
  temperature_of(temperature, op);
  a.logits = logits.const_data_ptr();
  a.ld = logits.stride(0);
  a.ids = ids.data_ptr<int>();
  a.logp = logprobs.data_ptr<float>();
  a.weight = weight ? weight->data_ptr<float>() : nullptr;
  a.target = target ? target->data_ptr<int>() : nullptr;
  a.target_weight = target_weight ? target_weight->data_ptr<float>() : nullptr;
  a.R = static_cast<int>(R);
  a.V = static_cast<int>(logits.size(1));
  a.K = static_cast<int>(ids.size(1));
  a.kind = kind;
  a.temperature = temperature;
  a.err = error_of(error, dev, op);
  return a;
}

// A new gradient: rows as far past a 16-byte boundary as those of logits, so that both are
// walked in the same vectors.
at::Tensor grad_like(const at::Tensor& logits) {
  const int64_t R = logits.size(0), V = logits.size(1), e = 16 / logits.element_size();
  const int64_t more = R > 1 ? ((logits.stride(0) - V) % e + e) % e : 0;
  const int64_t first = static_cast<int64_t>(reinterpret_cast<uintptr_t>(logits.const_data_ptr()) & 15) / logits.element_size();
  if (R == 0 || (more == 0 && first == 0)) return at::empty({R, V}, logits.options());
  return at::empty({first + R * (V + more)}, logits.options()).as_strided({R, V}, {V + more, 1}, first);
}

using LossAndGrad = std::optional<std::tuple<at::Tensor, at::Tensor>>;

LossAndGrad distill_loss_grad(const at::Tensor& logits, const at::Tensor& ids, const at::Tensor& logprobs,
                              const Opt& weight, const std::string& kind, bool rest, double temperature,
                              const Opt& target, const Opt& target_weight, const Opt& out_, const Opt& error,
                              const Opt& kl) {
  const char* op = "distill_loss_grad";
  TbDistillArgs a = distill_args(logits, ids, logprobs, weight, target, target_weight, distill_kind(kind, rest, op),
                                 temperature, error, op);
  no_grad({&logits}, op);
  if (out_) {
    rows2(*out_, op, "out is [R, V] with a contiguous last dimension");
    chk(out_->sizes() == logits.sizes() && out_->scalar_type() == logits.scalar_type(), op,
        "out has logits' shape and type");
    chk(out_->device() == logits.device(), op, "all tensors on one device");
    chk(rows2_distinct(*out_), op, "out has overlapping rows");
    no_grad({&*out_}, op);
    chk(same_view(logits, *out_) || apart(logits, *out_), op, "out is logits itself or does not overlap them");
    for (const at::Tensor* t : {&ids, &logprobs}) chk(apart(*out_, *t), op, "out overlaps an input");
    for (const Opt* t : {&weight, &target, &target_weight, &error})
      chk(!*t || apart(*out_, **t), op, "out overlaps an input");
  }
  if (kl) {
    per_row(kl, a.R, at::kFloat, logits.device(), op, "kl is a contiguous fp32 [R]");
    no_grad({&*kl}, op, "kl");
    for (const at::Tensor* t : {&logits, &ids, &logprobs}) chk(apart(*kl, *t), op, "kl overlaps another tensor");
    for (const Opt* t : {&weight, &target, &target_weight, &out_, &error})
      chk(!*t || apart(*kl, **t), op, "kl overlaps another tensor");
  }
  if (!logits.is_cuda()) return std::nullopt;
  c10::DeviceGuard guard(logits.device());
  at::Tensor loss = at::empty({a.R}, logprobs.options());
  at::Tensor grad = out_ ? *out_ : grad_like(logits);
  if (a.R > 0) {
    a.grad = grad.data_ptr();
    a.ld_grad = grad.stride(0);
    a.loss = loss.data_ptr<float>();
    a.kl = kl ? kl->data_ptr<float>() : nullptr;
    cuda_ok(tb_distill(&a, turbol::StreamFor(logits)), op);
    if (out_) written({&*out_});
    if (kl) written({&*kl});
  }
  return std::make_tuple(loss, grad);
}

// The loss alone; with `stats` ([R, TB_DISTILL_STATS]) what a backward pass needs.
at::Tensor loss_of(TbDistillArgs& a, const at::Tensor& logits, const at::Tensor& logprobs, at::Tensor* stats) {
  c10::DeviceGuard guard(logits.device());
  at::Tensor loss = at::empty({a.R}, logprobs.options());
  if (stats) *stats = at::empty({a.R, TB_DISTILL_STATS}, logprobs.options());
  if (a.R == 0) return loss;
  a.loss = loss.data_ptr<float>();
  if (stats) a.stats = stats->data_ptr<float>();
  cuda_ok(tb_distill(&a, turbol::StreamFor(logits)), "distill_loss");
  return loss;
}

Opt distill_loss(const at::Tensor& logits, const at::Tensor& ids, const at::Tensor& logprobs, const Opt& weight,
                 const std::string& kind, bool rest, double temperature, const Opt& target, const Opt& target_weight,
                 const Opt& error) {
  const char* op = "distill_loss";
  TbDistillArgs a = distill_args(logits, ids, logprobs, weight, target, target_weight, distill_kind(kind, rest, op),
                                 temperature, error, op);
  if (is_dual(logits)) no_grad({&logits}, op);
  if (!logits.is_cuda()) return std::nullopt;
  return loss_of(a, logits, logprobs, nullptr);
}

// The differentiable form (CUDA tensors).  The forward pass keeps a few numbers per
// row; the backward pass reads the logits again.
struct DistillFunction : torch::autograd::Function<DistillFunction> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& ids,
                            const at::Tensor& logprobs, const Opt& weight, int64_t kind, double temperature,
                            const Opt& target, const Opt& target_weight, const Opt& error) {
    TbDistillArgs a = distill_args(logits, ids, logprobs, weight, target, target_weight, static_cast<int>(kind),
                                   temperature, error, "distill_loss");
    at::Tensor stats;
    at::Tensor loss = loss_of(a, logits, logprobs, &stats);
    auto keep = [](const Opt& t) { return t ? *t : at::Tensor(); };
    ctx->save_for_backward({logits, ids, logprobs, keep(weight), keep(target), keep(target_weight), stats});
    ctx->saved_data["kind"] = kind;
    ctx->saved_data["temperature"] = temperature;
    return loss;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 const torch::autograd::variable_list& grads) {
    torch::autograd::variable_list out(9);
    if (!grads[0].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const at::Tensor& logits = saved[0];
    if (at::GradMode::is_enabled())
      throw std::invalid_argument("distill_loss: no second derivative (create_graph)");
    auto opt = [](const at::Tensor& t) { return t.defined() ? Opt(t) : Opt(); };
    TbDistillArgs a = distill_args(logits, saved[1], saved[2], opt(saved[3]), opt(saved[4]), opt(saved[5]),
                                   static_cast<int>(ctx->saved_data["kind"].toInt()),
                                   ctx->saved_data["temperature"].toDouble(), std::nullopt, "distill_loss");
    c10::DeviceGuard guard(logits.device());
    const at::Tensor g = grads[0].contiguous();  // (a sum's gradient is broadcast)
    at::Tensor d = grad_like(logits);
    if (a.R > 0) {
      a.grad = d.data_ptr();
      a.ld_grad = d.stride(0);
      a.stats = saved[6].data_ptr<float>();
      a.dloss = g.data_ptr<float>();
      cuda_ok(tb_distill(&a, turbol::StreamFor(logits)), "distill_loss (backward)");
    }
    out[0] = d;
    return out;
  }
};

at::Tensor distill_loss_autograd(const at::Tensor& logits, const at::Tensor& ids, const at::Tensor& logprobs,
                                 const Opt& weight, const std::string& kind, bool rest, double temperature,
                                 const Opt& target, const Opt& target_weight, const Opt& error) {
  const char* op = "distill_loss";
  chk(logits.is_cuda(), op, "CUDA tensors");
  if (is_dual(logits)) no_grad({&logits}, op);
  // (inside the node gradients are off)
  no_grad({&logprobs}, op, "the teacher's list");
  if (weight) no_grad({&*weight}, op, "weight");
  if (target_weight) no_grad({&*target_weight}, op, "target_weight");
  return DistillFunction::apply(logits, ids, logprobs, weight, static_cast<int64_t>(distill_kind(kind, rest, op)),
                                temperature, target, target_weight, error);
}

// ------------------------------------------------------------------ embedding
int ids_of(const at::Tensor& ids, const char* op) {
  chk((ids.scalar_type() == at::kInt || ids.scalar_type() == at::kLong) && ids.is_contiguous() &&
          ids.numel() <= kMaxTokens,
      op, "ids are contiguous int32 or int64, at most 2^30");
  return ids.scalar_type() == at::kLong;
}
void scale_of(double scale, const char* op) {
  chk(std::isfinite(static_cast<float>(scale)), op, "a scale that is finite in fp32");
}
std::vector<int64_t> rows_shape(const at::Tensor& ids, int64_t H) {
  std::vector<int64_t> s = ids.sizes().vec();
  s.push_back(H);
  return s;
}

Opt embedding(const at::Tensor& ids, const at::Tensor& weight, double scale, const Opt& out_, const Opt& error,
              bool first_row) {
  const char* op = "embedding";
  TbEmbeddingArgs a{};
  a.ids64 = ids_of(ids, op);
  a.dtype = rows2(weight, op, "weight is [V, H] with a contiguous last dimension");
  chk(weight.size(0) >= 1 && weight.size(1) >= 1 && weight.size(1) <= kMaxColumns, op,
      "at least one row, and 1 to 2^24 columns");
  scale_of(scale, op);
  const at::Device dev = weight.device();
  chk(ids.device() == dev, op, "all tensors on one device");
  if (is_dual(weight)) no_grad({&weight}, op);
  if (first_row) no_grad({&weight}, op, "first_row=True");  // (the gradient leaves such ids out)
  const std::vector<int64_t> shape = rows_shape(ids, weight.size(1));
  if (out_) {
    chk(out_->sizes() == at::IntArrayRef(shape) && out_->scalar_type() == weight.scalar_type() && out_->is_contiguous(),
        op, "out is contiguous, with ids' shape and the rows' length, and weight's type");
    chk(out_->device() == dev, op, "all tensors on one device");
    no_grad({&*out_, &weight}, op, "out=");
    for (const at::Tensor* t : {&ids, &weight}) chk(apart(*out_, *t), op, "out overlaps an input");
    chk(!error || apart(*out_, *error), op, "out overlaps an input");
  }
  a.err = error_of(error, dev, op);
  if (!weight.is_cuda()) return std::nullopt;
  c10::DeviceGuard guard(dev);
  at::Tensor out = out_ ? *out_ : at::empty(shape, weight.options());
  if (out.numel() == 0) return out;
  a.ids = ids.data_ptr();
  a.weight = weight.data_ptr();
  a.ld_w = weight.stride(0);
  a.out = out.data_ptr();
  a.ld_out = weight.size(1);
  a.N = static_cast<int>(ids.numel());
  a.H = static_cast<int>(weight.size(1));
  a.V = static_cast<int>(weight.size(0));
  a.scale = static_cast<float>(scale);
  a.first_row = first_row;
  cuda_ok(tb_embedding(&a, turbol::StreamFor(weight)), op);
  if (out_) written({&*out_});
  return out;
}

// dy as [N, H] rows with a contiguous last dimension (a broadcast gradient is copied).
at::Tensor flat_rows(const at::Tensor& dy, int64_t N, int64_t H) {
  at::Tensor d = dy.reshape({N, H});
  return H <= 1 || d.stride(1) == 1 ? d : d.contiguous();
}

bool embedding_grad(const at::Tensor& ids, const at::Tensor& dy, const at::Tensor& grad, double scale, bool accumulate,
                    const Opt& error) {
  const char* op = "embedding_grad";
  TbEmbeddingGradArgs a{};
  a.ids64 = ids_of(ids, op);
  a.grad_dtype = rows2(grad, op, "grad is [V, H] with a contiguous last dimension");
  chk(grad.size(0) >= 1 && grad.size(1) >= 1 && grad.size(1) <= kMaxColumns, op,
      "at least one row, and 1 to 2^24 columns");
  const int64_t H = grad.size(1), N = ids.numel();
  a.dtype = type_of(dy, op);
  chk(dy.sizes() == at::IntArrayRef(rows_shape(ids, H)), op, "dy has ids' shape and grad's row length");
  scale_of(scale, op);
  const at::Device dev = grad.device();
  for (const at::Tensor* t : {&ids, &dy}) {
    chk(t->device() == dev, op, "all tensors on one device");
    chk(apart(grad, *t), op, "grad overlaps an input");
  }
  chk(rows2_distinct(grad), op, "grad has overlapping rows");
  no_grad({&dy, &grad}, op);
  a.err = error_of(error, dev, op);
  chk(!error || apart(grad, *error), op, "grad overlaps an input");
  if (!grad.is_cuda()) return false;
  if (N == 0 && accumulate) return true;
  c10::DeviceGuard guard(dev);
  const at::Tensor d = flat_rows(dy, N, H);
  a.ids = ids.data_ptr();
  a.dy = d.data_ptr();
  a.ld_dy = d.stride(0);
  a.grad = grad.data_ptr();
  a.ld_grad = grad.stride(0);
  a.N = static_cast<int>(N);
  a.H = static_cast<int>(H);
  a.V = static_cast<int>(grad.size(0));
  a.scale = static_cast<float>(scale);
  a.zero = !accumulate;
  // from the caching allocator on the current stream (inside a capture: from the
  // graph's own pool), so calls on other streams and graphs never share it
  at::Tensor ws;
  const size_t bytes = tb_embedding_grad_ws_bytes(a.N, a.H, a.V);
  if (bytes > 0) {
    ws = at::empty({static_cast<int64_t>(bytes)}, grad.options().dtype(at::kByte));
    a.ws = ws.data_ptr();
  }
  cuda_ok(tb_embedding_grad(&a, turbol::StreamFor(grad)), op);
  written({&grad});
  return true;
}

at::Tensor embedding_apply(const at::Tensor& ids, const at::Tensor& weight, double scale, const Opt& error);

// The gradient as a differentiable function of dy (its own gradient is a lookup).
struct EmbeddingGradFunction : torch::autograd::Function<EmbeddingGradFunction> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& dy, const at::Tensor& ids,
                            int64_t V, double scale) {
    at::Tensor grad = at::empty({V, dy.size(-1)}, dy.options());
    embedding_grad(ids, dy, grad, scale, /*accumulate=*/false, std::nullopt);
    ctx->save_for_backward({ids});
    ctx->saved_data["scale"] = scale;
    return grad;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 const torch::autograd::variable_list& grads) {
    at::Tensor d;
    if (grads[0].defined()) {
      const at::Tensor g = grads[0].stride(1) == 1 ? grads[0] : grads[0].contiguous();
      d = embedding_apply(ctx->get_saved_variables()[0], g, ctx->saved_data["scale"].toDouble(), std::nullopt);
    }
    return {d, at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

struct EmbeddingFunction : torch::autograd::Function<EmbeddingFunction> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& weight, const at::Tensor& ids,
                            double scale, const Opt& error) {
    at::Tensor out = *embedding(ids, weight, scale, std::nullopt, error, /*first_row=*/false);
    ctx->save_for_backward({ids});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["V"] = weight.size(0);
    return out;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 const torch::autograd::variable_list& grads) {
    at::Tensor d;
    if (grads[0].defined())
      d = EmbeddingGradFunction::apply(grads[0], ctx->get_saved_variables()[0], ctx->saved_data["V"].toInt(),
                                       ctx->saved_data["scale"].toDouble());
    return {d, at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

at::Tensor embedding_apply(const at::Tensor& ids, const at::Tensor& weight, double scale, const Opt& error) {
  return EmbeddingFunction::apply(weight, ids, scale, error);
}

at::Tensor embedding_autograd(const at::Tensor& ids, const at::Tensor& weight, double scale, const Opt& error) {
  chk(weight.is_cuda(), "embedding", "CUDA tensors");
  if (is_dual(weight)) no_grad({&weight}, "embedding");
  return embedding_apply(ids, weight, scale, error);
}

}  // namespace

void register_vocab_ops(py::module_& m) {
  m.def("topk_logprobs", &topk_logprobs, py::arg("logits"), py::arg("k"), py::arg("temperature") = 1.0,
        "(log-probabilities, ids, log-sum-exps) of the k largest logits of each row; None for CPU tensors, after the "
        "checks");
  m.def("distill_loss_grad", &distill_loss_grad, py::arg("logits"), py::arg("ids"), py::arg("logprobs"),
        py::arg("weight") = py::none(), py::arg("kind") = "forward", py::arg("rest") = true,
        py::arg("temperature") = 1.0, py::arg("target") = py::none(), py::arg("target_weight") = py::none(),
        py::arg("out") = py::none(), py::arg("error") = py::none(), py::arg("kl") = py::none(),
        "distillation loss of each row and its gradient");
  m.def("distill_loss", &distill_loss, py::arg("logits"), py::arg("ids"), py::arg("logprobs"),
        py::arg("weight") = py::none(), py::arg("kind") = "forward", py::arg("rest") = true,
        py::arg("temperature") = 1.0, py::arg("target") = py::none(), py::arg("target_weight") = py::none(),
        py::arg("error") = py::none(), "distillation loss of each row");
  m.def("distill_loss_autograd", &distill_loss_autograd, py::arg("logits"), py::arg("ids"), py::arg("logprobs"),
        py::arg("weight") = py::none(), py::arg("kind") = "forward", py::arg("rest") = true,
        py::arg("temperature") = 1.0, py::arg("target") = py::none(), py::arg("target_weight") = py::none(),
        py::arg("error") = py::none(), "the same, differentiable in logits (CUDA tensors)");
  m.def("embedding", &embedding, py::arg("ids"), py::arg("weight"), py::arg("scale") = 1.0,
        py::arg("out") = py::none(), py::arg("error") = py::none(), py::arg("first_row") = false, "scale * weight[ids]");
  m.def("embedding_grad", &embedding_grad, py::arg("ids"), py::arg("dy"), py::arg("grad"), py::arg("scale") = 1.0,
        py::arg("accumulate") = true, py::arg("error") = py::none(),
        "adds scale * dy to the rows of grad that ids name, in token order");
  m.def("embedding_autograd", &embedding_autograd, py::arg("ids"), py::arg("weight"), py::arg("scale") = 1.0,
        py::arg("error") = py::none(), "embedding, differentiable in weight (CUDA tensors)");
}
