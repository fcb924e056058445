// torch-tensor entry points of the general rotary positions and the 8-bit
// paged KV cache.  Each checks its arguments completely, whatever device they
// are on, then launches on the current stream of their device and returns its
// result (a new tensor where no output was given); for CPU tensors it returns
// None and the caller computes on the host.  The CPU-only build has them too, for
// the checks.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <pybind11/pybind11.h>
#include <torch/extension.h>

#include <climits>
#include <cmath>
#include <optional>

#include "kernels.h"
#include "op_checks.hpp"
#include "turbol/common.hpp"

namespace py = pybind11;
using namespace turbol::checks;

namespace {

// [T, H, D] rows with a contiguous last dimension.
void rows3(const at::Tensor& t, const char* op, const char* m) {
  chk(t.dim() == 3 && (t.size(2) <= 1 || t.stride(2) == 1) && t.size(0) <= INT_MAX, op, m);
  chk(t.size(2) == 0 || t.size(1) <= INT_MAX / t.size(2), op, "at most 2^31 - 1 elements per row");
}

// Whether two [T, H, D] views share no element: disjoint ranges, or column
// slices of rows with the same stride.
bool columns_apart(const at::Tensor& a, const at::Tensor& b) {
  if (apart(a, b)) return true;
  if (a.element_size() != b.element_size() || a.stride(0) != b.stride(0)) return false;
  const int64_t e = a.element_size(), row = a.stride(0) * e;
  const int64_t wa = ((a.size(1) - 1) * a.stride(1) + a.size(2)) * e, wb = ((b.size(1) - 1) * b.stride(1) + b.size(2)) * e;
  if (row <= 0) return false;
  int64_t d = static_cast<int64_t>(range_of(b).lo - range_of(a).lo);
  d %= row;
  if (d < 0) d += row;
  return d >= wa && d + wb <= row;
}
// Whether a [T, H, D] view to be written names each element once.
bool rows_distinct(const at::Tensor& t) {
  if (t.numel() == 0) return true;
  int64_t n0 = t.size(0), s0 = t.stride(0), n1 = t.size(1), s1 = t.stride(1);
  if (n0 == 1) return n1 == 1 || s1 >= t.size(2);
  if (n1 == 1) return s0 >= t.size(2);
  if (s0 < s1) {
    std::swap(n0, n1);
    std::swap(s0, s1);
  }
  return s1 >= t.size(2) && s0 >= (n1 - 1) * s1 + t.size(2);
}
// The table's dimensions: R / 2 pairs for max_pos positions.
void table_of(const at::Tensor& t, int64_t D, const char* op) {
  chk(t.scalar_type() == at::kFloat && t.dim() == 3 && t.size(2) == 2 && t.is_contiguous() && t.size(0) >= 1 &&
          t.size(0) <= INT_MAX && t.size(1) >= 1 && 2 * t.size(1) <= D,
      op, "table is a contiguous fp32 [max_pos, R / 2, 2] with 1 <= R / 2 <= D / 2");
  chk(reinterpret_cast<uintptr_t>(t.data_ptr()) % 8 == 0, op, "table is 8-byte aligned");
  no_grad({&t}, op, "the table");
}

Opt rotary(const at::Tensor& x, const at::Tensor& pos, const at::Tensor& table, const Opt& out_, bool interleaved,
           bool transpose, const Opt& error) {
  const char* op = "rotary";
  rows3(x, op, "x is [T, H, D] with a contiguous last dimension");
  const int dt = type_of(x, op);
  chk(x.size(2) % 2 == 0 && x.size(2) <= INT_MAX, op, "an even head dimension");
  index1(pos, x.size(0), op, "pos is a contiguous int32 [T]");
  table_of(table, x.size(2), op);
  const at::Device dev = x.device();
  chk(pos.device() == dev && table.device() == dev, op, "all tensors on one device");
  if (out_) {
    rows3(*out_, op, "out is [T, H, D] with a contiguous last dimension");
    chk(out_->sizes() == x.sizes() && out_->scalar_type() == x.scalar_type(), op, "out has x's shape and type");
    chk(out_->device() == dev, op, "all tensors on one device");
    chk(rows_distinct(*out_), op, "out has overlapping rows");
    chk(!is_dual(x) && !is_dual(*out_), op, "out= has no forward-mode derivative");
    chk(same_view(x, *out_) || columns_apart(x, *out_), op, "out is x itself or does not overlap it");
    for (const at::Tensor* t : {&pos, &table}) chk(apart(*out_, *t), op, "out overlaps an input");
  }
  int* err = error_of(error, dev, op);
  if (!x.is_cuda()) return std::nullopt;
  c10::DeviceGuard guard(dev);
  at::Tensor out = out_ ? *out_ : at::empty(x.sizes(), x.options());
  if (x.numel() == 0) return out;
  TbRotaryArgs a{};
  a.x = x.data_ptr();
  a.y = out.data_ptr();
  a.pos = pos.data_ptr<int>();
  a.table = table.data_ptr<float>();
  a.T = static_cast<int>(x.size(0));
  a.H = static_cast<int>(x.size(1));
  a.D = static_cast<int>(x.size(2));
  a.R = static_cast<int>(2 * table.size(1));
  a.max_pos = static_cast<int>(table.size(0));
  a.xs_t = x.stride(0);
  a.xs_h = x.stride(1);
  a.ys_t = out.stride(0);
  a.ys_h = out.stride(1);
  a.dtype = dt;
  a.interleaved = interleaved;
  a.transpose = transpose;
  a.err = err;
  cuda_ok(tb_rotary(&a, turbol::StreamFor(x)), op);
  if (out_) written({&*out_});
  if (is_dual(x)) {  // the rotation is linear: the tangent turns like x
    at::Tensor t = x._fw_grad(0);
    if (t._is_zerotensor() || t.stride(2) != 1) t = at::empty(x.sizes(), x.options()).copy_(t);
    out._set_fw_grad(*rotary(t, pos, table, std::nullopt, interleaved, transpose, error), 0, /*is_inplace_op=*/false);
  }
  return out;
}

// The differentiable form (CUDA tensors): the gradient of a rotation is the
// rotation by the negative angles (times the table's factor), itself
// differentiable.
struct RotaryFunction : torch::autograd::Function<RotaryFunction> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& pos,
                            const at::Tensor& table, bool interleaved, bool transpose, const Opt& error) {
    at::Tensor out = *rotary(x, pos, table, std::nullopt, interleaved, transpose, error);
    ctx->save_for_backward({pos, table});
    ctx->saved_data["how"] = (interleaved ? 1 : 0) | (transpose ? 2 : 0);
    if (error) ctx->saved_data["error"] = *error;
    return out;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 const torch::autograd::variable_list& grads) {
    at::Tensor dx;
    if (grads[0].defined()) {
      const auto saved = ctx->get_saved_variables();
      const int64_t how = ctx->saved_data["how"].toInt();
      Opt error;
      if (ctx->saved_data.count("error")) error = ctx->saved_data["error"].toTensor();
      const at::Tensor dy = grads[0].stride(2) == 1 ? grads[0] : grads[0].contiguous();  // a broadcast gradient
      dx = RotaryFunction::apply(dy, saved[0], saved[1], (how & 1) != 0, (how & 2) == 0, error);
    }
    return {dx, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

at::Tensor rotary_grad(const at::Tensor& x, const at::Tensor& pos, const at::Tensor& table, bool interleaved,
                       bool transpose, const Opt& error) {
  chk(x.is_cuda(), "rotary_grad", "CUDA tensors");
  no_grad({&table}, "rotary", "the table");  // (inside the node gradients are off)
  return RotaryFunction::apply(x, pos, table, interleaved, transpose, error);
}

TbQuantCache cache_of(const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& ks, const at::Tensor& vs,
                      const at::Tensor& block_table, const char* op) {
  chk(kc.scalar_type() == at::kFloat8_e4m3fn && vc.scalar_type() == at::kFloat8_e4m3fn && kc.dim() == 4 &&
          kc.sizes() == vc.sizes() && kc.is_contiguous() && vc.is_contiguous(),
      op, "kc and vc are contiguous float8_e4m3fn [num_blocks, Hk, block_size, D]");
  chk(ks.scalar_type() == at::kFloat && vs.scalar_type() == at::kFloat && ks.dim() == 3 && ks.sizes() == vs.sizes() &&
          ks.is_contiguous() && vs.is_contiguous() && ks.sizes() == kc.sizes().slice(0, 3),
      op, "ks and vs are contiguous fp32 [num_blocks, Hk, block_size]");
  no_grad({&kc, &vc, &ks, &vs}, op, "the cache");
  const int64_t D = kc.size(3);
  chk(D == 64 || D == 128 || D == 256, op, "head dimension 64, 128 or 256");
  chk(kc.size(1) >= 1 && kc.size(2) >= 1, op, "at least one KV head and one slot per block");
  chk(kc.size(1) <= INT_MAX / D && kc.size(2) <= INT_MAX, op, "at most 2^31 - 1 elements per token, slots per block");
  chk(kc.size(0) * kc.size(1) * kc.size(2) <= INT_MAX, op, "at most 2^31 - 1 rows (blocks x heads x slots)");
  chk(block_table.scalar_type() == at::kInt && block_table.dim() == 2 && block_table.is_contiguous() &&
          block_table.size(0) <= INT_MAX && block_table.size(1) <= INT_MAX / kc.size(2),
      op, "block_table is a contiguous int32 [num_seqs, max_blocks]");
  for (const at::Tensor* t : {&vc, &ks, &vs, &block_table})
    chk(t->device() == kc.device(), op, "all tensors on one device");
  for (const at::Tensor* t : {&kc, &vc, &ks, &vs})
    chk(reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0, op, "the cache tensors are 16-byte aligned");
  TbQuantCache c{};
  c.kc = kc.data_ptr();
  c.vc = vc.data_ptr();
  c.ks = ks.data_ptr<float>();
  c.vs = vs.data_ptr<float>();
  c.block_table = block_table.data_ptr<int>();
  c.num_seqs = static_cast<int>(block_table.size(0));
  c.max_blocks = static_cast<int>(block_table.size(1));
  c.num_blocks = static_cast<int>(kc.size(0));
  c.Hk = static_cast<int>(kc.size(1));
  c.bs = static_cast<int>(kc.size(2));
  c.D = static_cast<int>(D);
  return c;
}

Opt kv_quant_write(const at::Tensor& k, const at::Tensor& v, const at::Tensor& seq, const at::Tensor& pos,
                   const at::Tensor& block_table, const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& ks, const at::Tensor& vs,
                   const Opt& q_, const Opt& q_out_, const Opt& table_, bool interleaved, const Opt& error) {
  const char* op = "kv_quant_write";
  TbKvQuantWriteArgs a{};
  a.cache = cache_of(kc, vc, ks, vs, block_table, op);
  const at::Device dev = kc.device();
  rows3(k, op, "k is [T, Hk, D] with a contiguous last dimension");
  rows3(v, op, "v is [T, Hk, D] with a contiguous last dimension");
  a.rot.dtype = type_of(k, op);
  chk(k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type(), op, "k and v have the same shape and type");
  no_grad({&k, &v}, op);
  chk(k.size(1) == a.cache.Hk && k.size(2) == a.cache.D, op, "k has the cache's heads and head dimension");
  const int64_t T = k.size(0);
  index1(seq, T, op, "seq_of_token is a contiguous int32 [T]");
  index1(pos, T, op, "pos is a contiguous int32 [T]");
  for (const at::Tensor* t : {&k, &v, &seq, &pos}) chk(t->device() == dev, op, "all tensors on one device");
  const Range caches[4] = {range_of(kc), range_of(vc), range_of(ks), range_of(vs)};
  for (int i = 0; i < 4; ++i)
    for (int j = i + 1; j < 4; ++j) chk(apart(caches[i], caches[j]), op, "the cache tensors overlap");
  for (const at::Tensor* t : {&k, &v, &seq, &pos, &block_table})
    chk(apart_from_all(range_of(*t), caches), op, "an input overlaps the cache");
  a.rot.err = error_of(error, dev, op);
  if (table_) {
    const at::Tensor& table = *table_;
    table_of(table, a.cache.D, op);
    chk(table.size(1) % 4 == 0, op, "a multiple of 8 rotated dimensions");
    chk(table.device() == dev, op, "all tensors on one device");
    a.rot.table = table.data_ptr<float>();
    a.rot.R = static_cast<int>(2 * table.size(1));
    a.rot.max_pos = static_cast<int>(table.size(0));
    a.rot.interleaved = interleaved;
  }
  chk(q_ || !q_out_, op, "q_out needs q");
  if (q_) {
    chk(table_.has_value(), op, "q needs a table");
    rows3(*q_, op, "q is [T, Hq, D] with a contiguous last dimension");
    chk(q_->size(0) == T && q_->size(2) == a.cache.D && q_->scalar_type() == k.scalar_type(), op,
        "q has k's rows, head dimension and type");
    chk(q_->device() == dev, op, "all tensors on one device");
    chk(apart_from_all(range_of(*q_), caches), op, "q overlaps the cache");
    no_grad({&*q_}, op);
  }
  if (q_out_) {
    rows3(*q_out_, op, "q_out is [T, Hq, D] with a contiguous last dimension");
    chk(q_out_->sizes() == q_->sizes() && q_out_->scalar_type() == q_->scalar_type(), op,
        "q_out has q's shape and type");
    chk(q_out_->device() == dev, op, "all tensors on one device");
    chk(rows_distinct(*q_out_), op, "q_out has overlapping rows");
    no_grad({&*q_out_}, op);
    chk(same_view(*q_, *q_out_) || columns_apart(*q_, *q_out_), op, "q_out is q itself or does not overlap it");
    chk(columns_apart(*q_out_, k) && columns_apart(*q_out_, v), op, "q_out overlaps k or v");
    const Range out = range_of(*q_out_);
    chk(apart_from_all(out, caches), op, "q_out overlaps the cache");
    for (const at::Tensor* t : {&seq, &pos, &block_table, &*table_})
      chk(apart(out, range_of(*t)), op, "q_out overlaps an input");
  }
  if (!kc.is_cuda()) return std::nullopt;
  c10::DeviceGuard guard(dev);
  Opt q_out = q_out_;
  if (q_ && !q_out) q_out = at::empty(q_->sizes(), q_->options());
  if (T == 0) return q_out;
  if (q_) {
    a.rot.x = q_->data_ptr();
    a.rot.y = q_out->data_ptr();
    a.rot.H = static_cast<int>(q_->size(1));
    a.rot.xs_t = q_->stride(0);
    a.rot.xs_h = q_->stride(1);
    a.rot.ys_t = q_out->stride(0);
    a.rot.ys_h = q_out->stride(1);
  }
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.ks_t = k.stride(0);
  a.ks_h = k.stride(1);
  a.vs_t = v.stride(0);
  a.vs_h = v.stride(1);
  a.seq = seq.data_ptr<int>();
  a.pos = pos.data_ptr<int>();
  a.T = static_cast<int>(T);
  cuda_ok(tb_kv_quant_write(&a, turbol::StreamFor(kc)), op);
  written({&kc, &vc, &ks, &vs});
  if (q_out_) written({&*q_out_});
  return q_out;
}

bool kv_quant_read(const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& ks, const at::Tensor& vs,
                   const at::Tensor& seq, const at::Tensor& pos, const at::Tensor& block_table, const at::Tensor& k_out,
                   const at::Tensor& v_out, const Opt& error) {
  const char* op = "kv_quant_read";
  TbKvQuantReadArgs a{};
  a.cache = cache_of(kc, vc, ks, vs, block_table, op);
  const at::Device dev = kc.device();
  rows3(k_out, op, "out is [T, Hk, D] with a contiguous last dimension");
  rows3(v_out, op, "out is [T, Hk, D] with a contiguous last dimension");
  a.dtype = type_of(k_out, op);
  chk(k_out.sizes() == v_out.sizes() && k_out.scalar_type() == v_out.scalar_type(), op,
      "the two outputs have the same shape and type");
  chk(k_out.size(1) == a.cache.Hk && k_out.size(2) == a.cache.D, op, "out has the cache's heads and head dimension");
  const int64_t T = k_out.size(0);
  index1(seq, T, op, "seq_of_token is a contiguous int32 [T]");
  index1(pos, T, op, "pos is a contiguous int32 [T]");
  for (const at::Tensor* t : {&k_out, &v_out, &seq, &pos}) chk(t->device() == dev, op, "all tensors on one device");
  chk(rows_distinct(k_out) && rows_distinct(v_out), op, "out has overlapping rows");
  no_grad({&k_out, &v_out}, op);
  chk(columns_apart(k_out, v_out), op, "the two outputs overlap");
  const Range outs[2] = {range_of(k_out), range_of(v_out)};
  for (const at::Tensor* t : {&kc, &vc, &ks, &vs, &seq, &pos, &block_table})
    chk(apart_from_all(range_of(*t), outs), op, "out overlaps an input");
  a.err = error_of(error, dev, op);
  if (!kc.is_cuda()) return false;
  if (T == 0) return true;
  c10::DeviceGuard guard(dev);
  a.k = k_out.data_ptr();
  a.v = v_out.data_ptr();
  a.ks_t = k_out.stride(0);
  a.ks_h = k_out.stride(1);
  a.vs_t = v_out.stride(0);
  a.vs_h = v_out.stride(1);
  a.seq = seq.data_ptr<int>();
  a.pos = pos.data_ptr<int>();
  a.T = static_cast<int>(T);
  cuda_ok(tb_kv_quant_read(&a, turbol::StreamFor(kc)), op);
  written({&k_out, &v_out});
  return true;
}

Opt decode_attention_quant(const at::Tensor& q, const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& ks,
                            const at::Tensor& vs, const at::Tensor& block_table, const at::Tensor& ctx_len,
                           const Opt& out_, std::optional<double> scale_, const Opt& error) {
  const char* op = "decode_attention_quant";
  TbDecodeAttnQuantArgs a{};
  a.cache = cache_of(kc, vc, ks, vs, block_table, op);
  const at::Device dev = kc.device();
  rows3(q, op, "q is [B, Hq, D] with a contiguous last dimension");
  a.dtype = type_of(q, op);
  chk(a.dtype != TB_F32, op, "bf16 or fp16 q");
  chk(q.size(2) == a.cache.D, op, "q has the cache's head dimension");
  no_grad({&q}, op);
  chk(q.size(1) >= 1 && q.size(1) % a.cache.Hk == 0, op, "the query heads are a multiple of the KV heads");
  const int64_t B = q.size(0);
  chk(block_table.size(0) == B, op, "one block_table row per sequence");
  chk(B * q.size(1) <= INT_MAX, op, "at most 2^31 - 1 query rows");
  index1(ctx_len, B, op, "ctx_len is a contiguous int32 [B]");
  for (const at::Tensor* t : {&q, &ctx_len}) chk(t->device() == dev, op, "all tensors on one device");
  if (out_) {
    rows3(*out_, op, "out is [B, Hq, D] with a contiguous last dimension");
    chk(out_->sizes() == q.sizes() && out_->scalar_type() == q.scalar_type(), op, "out has q's shape and type");
    chk(out_->device() == dev, op, "all tensors on one device");
    chk(rows_distinct(*out_), op, "out has overlapping rows");
    chk(columns_apart(*out_, q), op, "out overlaps q");
    no_grad({&*out_}, op);
    const Range out = range_of(*out_);
    for (const at::Tensor* t : {&kc, &vc, &ks, &vs, &ctx_len, &block_table})
      chk(apart(out, range_of(*t)), op, "out overlaps an input");
  }
  const double scale = scale_ ? *scale_ : 1.0 / std::sqrt(static_cast<double>(a.cache.D));
  chk(std::isfinite(static_cast<float>(scale * M_LOG2E)), op, "a scale that is finite in fp32, times log2(e) too");
  a.err = error_of(error, dev, op);
  if (!kc.is_cuda()) return std::nullopt;
  c10::DeviceGuard guard(dev);
  at::Tensor ws, out = out_ ? *out_ : at::empty(q.sizes(), q.options());
  if (B == 0) return out;
  a.q = q.data_ptr();
  a.out = out.data_ptr();
  a.qs_b = q.stride(0);
  a.qs_h = q.stride(1);
  a.os_b = out.stride(0);
  a.os_h = out.stride(1);
  a.ctx_len = ctx_len.data_ptr<int>();
  a.B = static_cast<int>(B);
  a.Hq = static_cast<int>(q.size(1));
  a.scale = static_cast<float>(scale);
  // from the caching allocator on the current stream (inside a capture: from
  // the graph's own pool), so calls on other streams and graphs never share it
  a.ws_bytes = tb_decode_attention_quant_ws_bytes(a.B, a.Hq, a.cache.Hk, a.cache.D, a.cache.max_blocks * a.cache.bs);
  if (a.ws_bytes > 0) {
    ws = at::empty({static_cast<int64_t>((a.ws_bytes + 3) / 4)}, ks.options());
    a.ws = ws.data_ptr<float>();
  }
  cuda_ok(tb_decode_attention_quant(&a, turbol::StreamFor(kc)), op);
  if (out_) written({&*out_});
  return out;
}

}  // namespace

void register_cache_ops(py::module_& m) {
  m.def("rotary", &rotary, py::arg("x"), py::arg("pos"), py::arg("table"), py::arg("out") = py::none(),
        py::arg("interleaved") = false, py::arg("transpose") = false, py::arg("error") = py::none(),
        "rotary positions of x [T, H, D] (general form); None for CPU tensors, after the checks");
  m.def("rotary_grad", &rotary_grad, py::arg("x"), py::arg("pos"), py::arg("table"), py::arg("interleaved") = false,
        py::arg("transpose") = false, py::arg("error") = py::none(), "the same, differentiable in x (CUDA tensors)");
  m.def("kv_quant_write", &kv_quant_write, py::arg("k"), py::arg("v"), py::arg("seq_of_token"), py::arg("pos"),
        py::arg("block_table"), py::arg("kc"), py::arg("vc"), py::arg("ks"), py::arg("vs"), py::arg("q") = py::none(),
        py::arg("q_out") = py::none(), py::arg("table") = py::none(), py::arg("interleaved") = false,
        py::arg("error") = py::none(),
        "quantises K and V rows into the 8-bit paged cache (with a table: rotates q and k first)");
  m.def("kv_quant_read", &kv_quant_read, py::arg("kc"), py::arg("vc"), py::arg("ks"), py::arg("vs"),
        py::arg("seq_of_token"), py::arg("pos"), py::arg("block_table"), py::arg("k_out"), py::arg("v_out"),
        py::arg("error") = py::none(), "reads rows of the 8-bit paged cache back");
  m.def("decode_attention_quant", &decode_attention_quant, py::arg("q"), py::arg("kc"), py::arg("vc"), py::arg("ks"),
        py::arg("vs"), py::arg("block_table"), py::arg("ctx_len"), py::arg("out") = py::none(),
        py::arg("scale") = py::none(), py::arg("error") = py::none(), "attention of one token per sequence over the 8-bit paged cache");
}
