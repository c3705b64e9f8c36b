// PyTorch bindings of the operators that take bf16, fp16 and fp32 (rotary positions, block norms,
// distillation).  Their autograd nodes live here rather than in Python: a backward pass then runs
// without the interpreter, which a small training step would otherwise wait for.
// Every function checks devices, dtypes and layouts and enqueues on the current stream.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/extension.h>

#include <vector>

#include "kernels.h"

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

cudaStream_t cur_stream() { return at::cuda::getCurrentCUDAStream().stream(); }

void check_cuda(const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), "mmf: ", name, " must be a CUDA tensor");
}

bool wants_grad(std::initializer_list<const OptTensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const OptTensor* t : ts)
    if (t->has_value() && (*t)->requires_grad()) return true;
  return false;
}

void refuse_second_order(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), "mmf: ", what, " has no second derivatives (create_graph=True)");
}

const void* ptr(const OptTensor& t) { return t.has_value() ? t->data_ptr() : nullptr; }

mmf::DType dtype_of(const Tensor& t, const char* name) {
  const auto d = t.scalar_type();
  TORCH_CHECK(d == torch::kBFloat16 || d == torch::kFloat16 || d == torch::kFloat32, "mmf: ", name,
              " must be bf16, fp16 or fp32");
  return d == torch::kBFloat16 ? mmf::DType::BF16 : d == torch::kFloat16 ? mmf::DType::F16 : mmf::DType::F32;
}

// Rotary positions of q and k, [batch, seq, heads, head_dim] or [tokens, heads, head_dim]: the new
// (contiguous) tensors, or q and k themselves.
std::vector<Tensor> rotary_raw(const Tensor& q, const OptTensor& k, const OptTensor& positions, const Tensor& turns,
                           int64_t rotary_dim, bool interleaved, double magnitude, bool inverse, bool in_place) {
  check_cuda(q, "q");
  const c10::cuda::CUDAGuard guard(q.device());
  const bool pair = k.has_value();
  mmf::RotaryArgs a{};
  a.dtype = dtype_of(q, "q");
  const int64_t es = q.element_size(), nd = q.dim();
  TORCH_CHECK(nd == 3 || nd == 4, "mmf: rotary takes [batch, seq, heads, head_dim] or [tokens, heads, head_dim]");
  const int64_t B = nd == 4 ? q.size(0) : 1, T = q.size(nd - 3), D = q.size(nd - 1);
  TORCH_CHECK(B * T <= 0x7fffffff, "mmf: rotary: too many tokens");
  TORCH_CHECK(rotary_dim >= 2 && rotary_dim % 2 == 0 && rotary_dim <= D && D % 2 == 0 && D <= 256,
              "mmf: rotary: head_dim and rotary_dim must be even, rotary_dim <= head_dim <= 256");
  TORCH_CHECK(turns.device() == q.device() && turns.scalar_type() == torch::kInt64 && turns.is_contiguous() &&
                  turns.numel() == rotary_dim / 2, "mmf: rotary: turns must be int64 [rotary_dim / 2] on q's device");
  if (pair)
    TORCH_CHECK(k->device() == q.device() && k->scalar_type() == q.scalar_type() && k->dim() == nd &&
                    k->sizes().slice(0, nd - 2) == q.sizes().slice(0, nd - 2) && k->size(nd - 1) == D,
                "mmf: rotary: q and k must agree in batch, seq, head_dim, dtype and device");
  // strides for batch, seq and head (0 along dimensions of one element, whose stride is not used)
  auto strides = [&](const Tensor& t, int64_t* s) {
    s[0] = (nd == 4 && t.size(0) > 1) ? t.stride(0) : 0;
    s[1] = t.size(nd - 3) > 1 ? t.stride(nd - 3) : 0;
    s[2] = t.size(nd - 2) > 1 ? t.stride(nd - 2) : 0;
  };
  auto input = [&](Tensor t, int64_t* s) {
    strides(t, s);
    bool ok = t.numel() == 0 || t.stride(nd - 1) == 1;
    if (interleaved)  // a pair is one access
      ok = ok && reinterpret_cast<uintptr_t>(t.data_ptr()) % (2 * es) == 0 && s[0] % 2 == 0 && s[1] % 2 == 0 &&
           s[2] % 2 == 0;
    if (!ok) {
      TORCH_CHECK(!in_place, "mmf: rotary: in place needs contiguous heads that start on a pair's boundary");
      t = t.clone(at::MemoryFormat::Contiguous);
      strides(t, s);
    }
    return t;
  };
  Tensor qi = input(q, a.q_in_s), ki, qo, ko;
  if (pair) ki = input(*k, a.k_in_s);
  if (in_place) {
    qo = qi;
    ko = ki;
  } else {
    qo = torch::empty(q.sizes(), q.options());
    if (pair) ko = torch::empty(k->sizes(), k->options());
  }
  strides(qo, a.q_out_s);
  if (pair) strides(ko, a.k_out_s);
  a.q_in = qi.data_ptr();
  a.q_out = qo.data_ptr();
  a.k_in = pair ? ki.data_ptr() : nullptr;
  a.k_out = pair ? ko.data_ptr() : nullptr;
  a.batch = static_cast<uint32_t>(B);
  a.seq = static_cast<uint32_t>(T);
  a.q_heads = static_cast<int>(q.size(nd - 2));
  a.k_heads = pair ? static_cast<int>(k->size(nd - 2)) : 0;
  a.head_dim = static_cast<int>(D);
  a.rotary_dim = static_cast<int>(rotary_dim);
  a.turns = reinterpret_cast<const uint64_t*>(turns.data_ptr<int64_t>());
  if (positions.has_value()) {
    const Tensor& p = *positions;
    const bool p32 = p.scalar_type() == torch::kInt32;
    TORCH_CHECK(p.device() == q.device() && (p32 || p.scalar_type() == torch::kInt64),
                "mmf: rotary: positions must be int64 or int32 on q's device");
    const int64_t pd = p.dim();
    TORCH_CHECK(pd >= 1 && pd <= nd - 2 && (p.size(pd - 1) == T || p.size(pd - 1) == 1) &&
                    (pd == 1 || p.size(0) == B || p.size(0) == 1),
                "mmf: rotary: positions must broadcast over batch and seq");
    a.positions = p.data_ptr();
    a.positions_32 = p32;
    a.pos_stride_t = p.size(pd - 1) > 1 ? p.stride(pd - 1) : 0;
    a.pos_stride_b = (pd == 2 && p.size(0) > 1) ? p.stride(0) : 0;
  }
  a.magnitude = static_cast<float>(magnitude);
  a.inverse = inverse;
  a.interleaved = interleaved;
  a.in_place = in_place;
  mmf::rotary(a, cur_stream());
  if (pair) return {qo, ko};
  return {qo};
}

class RotaryFn : public torch::autograd::Function<RotaryFn> {
 public:
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const OptTensor& k, const OptTensor& positions,
                               const Tensor& turns, int64_t rotary_dim, bool interleaved, double magnitude) {
    at::AutoDispatchBelowADInplaceOrView guard;
    ctx->save_for_backward({turns, positions.value_or(Tensor())});
    ctx->saved_data["rotary_dim"] = rotary_dim;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["magnitude"] = magnitude;
    return rotary_raw(q, k, positions, turns, rotary_dim, interleaved, magnitude, false, false);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    refuse_second_order("rotary");
    const auto saved = ctx->get_saved_variables();
    const OptTensor positions = saved[1].defined() ? OptTensor(saved[1]) : OptTensor();
    const auto out = rotary_raw(g[0], g.size() > 1 ? OptTensor(g[1]) : OptTensor(), positions, saved[0],
                                ctx->saved_data["rotary_dim"].toInt(), ctx->saved_data["interleaved"].toBool(),
                                ctx->saved_data["magnitude"].toDouble(), true, false);
    return {out[0], out.size() > 1 ? out[1] : Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

std::vector<Tensor> rotary(const Tensor& q, const OptTensor& k, const OptTensor& positions, const Tensor& turns,
                           int64_t rotary_dim, bool interleaved, double magnitude, bool in_place) {
  const OptTensor oq(q);
  if (!wants_grad({&oq, &k})) return rotary_raw(q, k, positions, turns, rotary_dim, interleaved, magnitude, false, in_place);
  TORCH_CHECK(!in_place, "mmf: rotary: in place is for tensors outside autograd");
  return RotaryFn::apply(q, k, positions, turns, rotary_dim, interleaved, magnitude);
}

// ------------------------------------ block norms -----------------------------------------
struct NormConf {
  int64_t rows_per_gate;
  bool layer;
  double eps, residual_scale, branch_scale;
};

void check_like(const OptTensor& t, const Tensor& x, int64_t n, const char* name) {
  if (!t.has_value()) return;
  TORCH_CHECK(t->device() == x.device() && t->scalar_type() == x.scalar_type() && t->is_contiguous() && t->numel() == n,
              "mmf: block_norm: ", name, " must be contiguous, of x's device and dtype, with ", n, " values");
}

// {h} or {h, n}; stat_y, stat_h: filled where the backward needs them
variable_list block_norm_raw(const Tensor& x, const Tensor& y, const OptTensor& pw, const OptTensor& pb,
                             const OptTensor& gate, const OptTensor& nw, const OptTensor& nb, const NormConf& c,
                             Tensor* stat_y, Tensor* stat_h) {
  check_cuda(x, "x");
  const c10::cuda::CUDAGuard guard(x.device());
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1 && x.is_contiguous(), "mmf: block_norm: x must be contiguous [..., cols]");
  const int64_t cols = x.size(-1), rows = x.numel() / cols;
  mmf::BlockNormArgs a{};
  a.dtype = dtype_of(x, "x");
  check_like(y, x, x.numel(), "y");
  check_like(pw, x, cols, "post_weight");
  check_like(pb, x, cols, "post_bias");
  check_like(nw, x, cols, "pre_weight");
  check_like(nb, x, cols, "pre_bias");
  TORCH_CHECK(c.rows_per_gate >= 1 && (!gate.has_value() || rows % c.rows_per_gate == 0), "mmf: block_norm: gate rows");
  if (rows > 0) check_like(gate, x, rows / c.rows_per_gate * cols, "gate");
  Tensor h = torch::empty_like(x), n;
  if (nw.has_value()) n = torch::empty_like(x);
  const auto f32 = x.options().dtype(torch::kFloat32);
  if (stat_y && pw.has_value()) *stat_y = torch::empty({rows, c.layer ? 2 : 1}, f32);
  if (stat_h && nw.has_value()) *stat_h = torch::empty({rows, c.layer ? 2 : 1}, f32);
  a.x = x.data_ptr();
  a.y = y.data_ptr();
  a.post_w = ptr(pw);
  a.post_b = ptr(pb);
  a.gate = ptr(gate);
  a.pre_w = ptr(nw);
  a.pre_b = ptr(nb);
  a.h = h.data_ptr();
  a.n = n.defined() ? n.data_ptr() : nullptr;
  a.stat_y = stat_y && stat_y->defined() ? stat_y->data_ptr<float>() : nullptr;
  a.stat_h = stat_h && stat_h->defined() ? stat_h->data_ptr<float>() : nullptr;
  a.rows = rows;
  a.rows_per_gate = c.rows_per_gate;
  a.cols = static_cast<int>(cols);
  a.eps = static_cast<float>(c.eps);
  a.residual_scale = static_cast<float>(c.residual_scale);
  a.branch_scale = static_cast<float>(c.branch_scale);
  a.layer = c.layer;
  TORCH_CHECK(cols <= 8192, "mmf: block_norm: rows of up to 8192 values are supported, got ", cols);
  mmf::block_norm_fwd(a, cur_stream());
  if (n.defined()) return {h, n};
  return {h};
}

class BlockNormFn : public torch::autograd::Function<BlockNormFn> {
 public:
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& y, const OptTensor& pw,
                               const OptTensor& pb, const OptTensor& gate, const OptTensor& nw, const OptTensor& nb,
                               int64_t rows_per_gate, bool layer, double eps, double residual_scale,
                               double branch_scale) {
    at::AutoDispatchBelowADInplaceOrView guard;
    Tensor stat_y, stat_h;
    auto out = block_norm_raw(x, y, pw, pb, gate, nw, nb, {rows_per_gate, layer, eps, residual_scale, branch_scale},
                              &stat_y, &stat_h);
    // y only comes back through its norm or the gate, h only through its norm
    const bool keep_y = pw.has_value() || gate.has_value();
    ctx->save_for_backward({keep_y ? y : Tensor(), nw.has_value() ? out[0] : Tensor(), pw.value_or(Tensor()),
                            pb.value_or(Tensor()), gate.value_or(Tensor()), nw.value_or(Tensor()), stat_y, stat_h});
    auto& d = ctx->saved_data;
    d["rows_per_gate"] = rows_per_gate;
    d["layer"] = layer;
    d["rs"] = residual_scale;
    d["bs"] = branch_scale;
    auto need = [](const OptTensor& t) { return t.has_value() && t->requires_grad(); };
    d["need"] = static_cast<int64_t>(x.requires_grad() | y.requires_grad() << 1 | need(pw) << 2 | need(pb) << 3 |
                                     need(gate) << 4 | need(nw) << 5 | need(nb) << 6);
    ctx->set_materialize_grads(false);
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) {
    refuse_second_order("block_norm");
    auto saved = ctx->get_saved_variables();
    const Tensor &y = saved[0], &h = saved[1], &pw = saved[2], &pb = saved[3], &gate = saved[4], &nw = saved[5];
    auto& d = ctx->saved_data;
    const int64_t need = d["need"].toInt();
    variable_list out(12);
    Tensor dh = g[0].defined() ? g[0].contiguous() : Tensor();
    Tensor dn = g.size() > 1 && g[1].defined() ? g[1].contiguous() : Tensor();
    if (!dh.defined() && !dn.defined()) return out;
    const Tensor& like = dh.defined() ? dh : dn;
    const c10::cuda::CUDAGuard guard(like.device());
    mmf::BlockNormBwdArgs a{};
    a.dtype = dtype_of(like, "gradient");
    a.cols = static_cast<int>(like.size(-1));
    a.rows = like.numel() / a.cols;
    a.rows_per_gate = d["rows_per_gate"].toInt();
    a.residual_scale = static_cast<float>(d["rs"].toDouble());
    a.branch_scale = static_cast<float>(d["bs"].toDouble());
    a.layer = d["layer"].toBool();
    auto p = [](const Tensor& t) -> const void* { return t.defined() ? t.data_ptr() : nullptr; };
    auto want = [&](int i, bool there, const Tensor& shape) -> void* {
      if (!(need >> i & 1) || !there) return nullptr;
      // without rows nothing is launched, and the sums over rows are zero
      out[i] = a.rows ? torch::empty_like(shape, at::MemoryFormat::Contiguous)
                      : torch::zeros_like(shape, at::MemoryFormat::Contiguous);
      return out[i].data_ptr();
    };
    a.dh = p(dh);
    a.dn = p(dn);
    a.h = p(h);
    a.y = p(y);
    a.post_w = p(pw);
    a.post_b = p(pb);
    a.gate = p(gate);
    a.pre_w = dn.defined() ? p(nw) : nullptr;  // n was not used: its norm takes no part
    a.stat_y = saved[6].defined() ? saved[6].data_ptr<float>() : nullptr;
    a.stat_h = saved[7].defined() ? saved[7].data_ptr<float>() : nullptr;
    a.dx = want(0, true, like);
    a.dy = want(1, true, like);
    a.dpost_w = want(2, true, pw);
    a.dpost_b = want(3, true, pw);
    a.dgate = want(4, true, gate);
    a.dpre_w = want(5, dn.defined(), nw);
    a.dpre_b = want(6, dn.defined(), nw);
    Tensor parts = torch::empty({mmf::block_norm_bwd_parts(a)}, like.options().dtype(torch::kFloat32));
    a.parts = parts.data_ptr<float>();
    mmf::block_norm_bwd(a, cur_stream());
    return out;
  }
};

std::vector<Tensor> block_norm(const Tensor& x, const Tensor& y, const OptTensor& pw, const OptTensor& pb,
                               const OptTensor& gate, const OptTensor& nw, const OptTensor& nb, int64_t rows_per_gate,
                               bool layer, double eps, double residual_scale, double branch_scale) {
  const OptTensor ox(x), oy(y);
  if (!wants_grad({&ox, &oy, &pw, &pb, &gate, &nw, &nb}))
    return block_norm_raw(x, y, pw, pb, gate, nw, nb, {rows_per_gate, layer, eps, residual_scale, branch_scale}, nullptr,
                          nullptr);
  return BlockNormFn::apply(x, y, pw, pb, gate, nw, nb, rows_per_gate, layer, eps, residual_scale, branch_scale);
}

}  // namespace

void register_lm_ops(pybind11::module_& m) {
  m.def("rotary", &rotary);
  m.def("block_norm", &block_norm);
}
