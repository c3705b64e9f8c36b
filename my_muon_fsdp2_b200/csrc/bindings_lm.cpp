// PyTorch bindings of the operators that take bf16, fp16 and fp32 (rotary positions, block norms,
// distillation).  Their autograd nodes live here rather than in Python: a backward pass then runs
// without the interpreter, which a small training step would otherwise wait for.
// Every function checks devices, dtypes, shapes and layouts and enqueues on the current stream.  The
// checks of a user's call are made here, in 1 us rather than the interpreter's 4 to 6, of which a
// single token's call would feel every one; what is refused here is named by the Python function's own check.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/extension.h>

#include <algorithm>
#include <string>
#include <vector>

#include "kernels.h"

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

cudaStream_t cur_stream() { return at::cuda::getCurrentCUDAStream().stream(); }

// Numbers go into messages as text: where the C++ runtime is linked in statically a stream of the shared
// libraries' runtime formats none (it faults for want of its locale).
std::string num(int64_t n) { return std::to_string(n); }

void check_cuda(const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), "mmf: ", name, " must be a CUDA tensor");
}

bool wants_grad(std::initializer_list<const OptTensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const OptTensor* t : ts)
    if (t->has_value() && (*t)->requires_grad()) return true;
  return false;
}

// Wrappers (a DTensor outside its module's forward, say) have a device and a shape but no memory: their null
// pointers would read as a missing weight, or fault.
void check_memory(const char* what, std::initializer_list<const OptTensor*> ts) {
  for (const OptTensor* t : ts)
    TORCH_CHECK(!t->has_value() || !(*t)->defined() || (*t)->numel() == 0 || (*t)->data_ptr() != nullptr, "mmf: ", what,
                " takes tensors that have memory of their own (of a DTensor, its local tensor)");
}

// A tangent of forward-mode differentiation does not show in requires_grad: without this it would be lost.
void refuse_forward_mode(const char* what, std::initializer_list<const OptTensor*> ts) {
  for (const OptTensor* t : ts)
    TORCH_CHECK(!t->has_value() || !(*t)->defined() || !(*t)->_fw_grad(/*level=*/0).defined(), "mmf: ", what,
                " has no forward-mode derivatives");
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

py::object pair_or_one(const std::vector<Tensor>& out, bool pair) {
  return pair ? py::object(py::make_tuple(out[0], out[1])) : py::cast(out[0]);
}

py::object rotary(const Tensor& q, const OptTensor& k, const OptTensor& positions, const Tensor& turns, int64_t head_dim,
                  int64_t rotary_dim, bool interleaved, double magnitude, bool in_place) {
  const bool pair = k.has_value();
  TORCH_CHECK(q.dim() >= 3 && q.size(-1) == head_dim, "mmf: rotary: q must be [..., heads, ", num(head_dim), "]");
  const OptTensor oq(q);
  check_memory("rotary", {&oq, &k, &positions});
  refuse_forward_mode("rotary", {&oq, &k});
  const bool grad = wants_grad({&oq, &k});
  if (in_place) {
    TORCH_CHECK(!grad, "mmf: rotary: in place is for tensors outside autograd");
    auto own = [](const Tensor& t) {
      bool ok = t.dim() == 0 || t.stride(-1) == 1;
      for (int64_t i = 0; i < t.dim(); ++i) ok = ok && (t.size(i) <= 1 || t.stride(i) != 0);
      return ok;
    };
    TORCH_CHECK(own(q) && (!pair || own(*k)) && (!pair || q.numel() == 0 || q.data_ptr() != k->data_ptr()),
                "mmf: rotary: in place needs contiguous heads in memory of their own");
  }
  if (!grad) {
    const auto out = rotary_raw(q, k, positions, turns, rotary_dim, interleaved, magnitude, false, in_place);
    // a backward pass that kept q or k has to see that they have changed (a refused call leaves them as they were)
    if (in_place && !q.is_inference()) q.unsafeGetTensorImpl()->bump_version();
    if (in_place && pair && !k->is_inference()) k->unsafeGetTensorImpl()->bump_version();
    return pair_or_one(out, pair);
  }
  return pair_or_one(RotaryFn::apply(q, k, positions, turns, rotary_dim, interleaved, magnitude), pair);
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
              "mmf: block_norm: ", name, " must be contiguous, of x's device and dtype, with ", num(n), " values");
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
  TORCH_CHECK(cols <= 8192, "mmf: block_norm: rows of up to 8192 values are supported, got ", num(cols));
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
    // the backward forms h again from x and y for its norm; y comes back through its own norm and the gate
    const bool keep_y = pw.has_value() || gate.has_value() || nw.has_value();
    ctx->save_for_backward({keep_y ? y : Tensor(), nw.has_value() ? x : Tensor(), pw.value_or(Tensor()),
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
    const Tensor &y = saved[0], &x = saved[1], &pw = saved[2], &pb = saved[3], &gate = saved[4], &nw = saved[5];
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
    a.x = p(x);
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

// How many consecutive rows of x share a row of the gate: the gate's leading dimensions are x's up to
// some dimension, and 1 (or missing altogether) from there on.
int64_t rows_per_gate(const OptTensor& gate, const Tensor& x) {
  if (!gate.has_value()) return 1;
  const auto own = gate->sizes(), all = x.sizes();
  const bool one = own.size() == 1;
  TORCH_CHECK((one || own.size() == all.size()) && !own.empty() && own.back() == all.back(),
              "mmf: block_norm: the gate must be [dim] or of x's dimensions");
  const size_t lead = all.size() - 1;
  size_t i = one ? 0 : lead;
  while (i > 0 && own[i - 1] == 1) --i;
  int64_t shared = 1;
  for (size_t j = 0; j < lead; ++j) {
    TORCH_CHECK(j >= i || own[j] == all[j], "mmf: block_norm: the gate's leading dimensions must be x's, then ones");
    if (j >= i) shared *= all[j];
  }
  return std::max<int64_t>(1, shared);
}

OptTensor dense(const OptTensor& t) { return t.has_value() ? OptTensor(t->contiguous()) : t; }

py::object block_norm(const Tensor& x, const Tensor& y, const OptTensor& pw, const OptTensor& pb, const OptTensor& gate,
                      const OptTensor& nw, const OptTensor& nb, bool layer, double eps, double residual_scale,
                      double branch_scale) {
  const OptTensor ox(x), oy(y);
  check_memory("block_norm", {&ox, &oy, &pw, &pb, &gate, &nw, &nb});
  TORCH_CHECK(x.dim() >= 1 && x.sizes() == y.sizes(), "mmf: block_norm: x must be [..., dim] and y of its shape");
  for (const OptTensor* t : {&pw, &pb, &nw, &nb})
    TORCH_CHECK(!t->has_value() || (*t)->dim() == 1, "mmf: block_norm: weights and biases must be [dim]");
  TORCH_CHECK(!(pb.has_value() && !(layer && pw.has_value())) && !(nb.has_value() && !(layer && nw.has_value())),
              "mmf: block_norm: a bias needs its weight and the layer norm");
  const int64_t shared = rows_per_gate(gate, x);
  refuse_forward_mode("block_norm", {&ox, &oy, &pw, &pb, &gate, &nw, &nb});
  const Tensor xc = x.contiguous(), yc = y.contiguous();
  const OptTensor pwc = dense(pw), pbc = dense(pb), gc = dense(gate), nwc = dense(nw), nbc = dense(nb);
  if (!wants_grad({&ox, &oy, &pw, &pb, &gate, &nw, &nb}))
    return pair_or_one(block_norm_raw(xc, yc, pwc, pbc, gc, nwc, nbc, {shared, layer, eps, residual_scale, branch_scale},
                                      nullptr, nullptr), nw.has_value());
  return pair_or_one(BlockNormFn::apply(xc, yc, pwc, pbc, gc, nwc, nbc, shared, layer, eps, residual_scale, branch_scale),
                     nw.has_value());
}

// ------------------------------------ distillation ----------------------------------------
struct DistillConf {
  double tau, alpha;
  int64_t ignore_index;
};

// Checks the teacher's slots and the targets of `rows` rows and puts them into the arguments.
mmf::DistillArgs distill_args(const Tensor& like, int64_t rows, int64_t vocab, const Tensor& ids, const Tensor& teacher,
                              const OptTensor& targets, const DistillConf& c) {
  check_cuda(like, "logits");
  mmf::DistillArgs a{};
  const auto it = ids.scalar_type();
  TORCH_CHECK(ids.device() == like.device() && ids.dim() == 2 && ids.size(0) == rows && ids.is_contiguous() &&
                  (it == torch::kInt64 || it == torch::kInt32),
              "mmf: distill: ids must be contiguous int64 or int32 [rows, top] on the logits' device");
  TORCH_CHECK(teacher.device() == like.device() && teacher.is_contiguous() && teacher.sizes() == ids.sizes(),
              "mmf: distill: the teacher's logits must be contiguous, of the ids' shape, on the logits' device");
  TORCH_CHECK(ids.size(1) >= 1 && ids.size(1) <= mmf::distill_max_top(), "mmf: distill: 1 to ", num(mmf::distill_max_top()),
              " slots a row are supported");
  a.dtype = dtype_of(like, "logits");
  TORCH_CHECK(vocab >= 1 && vocab <= mmf::distill_max_vocab(a.dtype), "mmf: distill: a vocabulary of up to ",
              num(mmf::distill_max_vocab(a.dtype)), " values of this dtype is supported");
  if (targets.has_value())
    TORCH_CHECK(targets->device() == like.device() && targets->scalar_type() == torch::kInt64 &&
                    targets->is_contiguous() && targets->numel() == rows,
                "mmf: distill: targets must be contiguous int64 [rows] on the logits' device");
  a.ids = ids.data_ptr();
  a.ids_32 = it == torch::kInt32;
  a.teacher = teacher.data_ptr();
  a.teacher_dtype = dtype_of(teacher, "teacher logits");
  a.rows = rows;
  a.vocab = static_cast<int>(vocab);
  a.top = static_cast<int>(ids.size(1));
  a.tau = static_cast<float>(c.tau);
  a.alpha = static_cast<float>(c.alpha);
  // without a weight of their own the targets are not looked at, so that none is recorded as bad either
  a.targets = targets.has_value() && a.alpha < 1.f ? targets->data_ptr<int64_t>() : nullptr;
  a.ignore_index = c.ignore_index;
  return a;
}

void put_logits(mmf::DistillArgs& a, const Tensor& logits) {
  TORCH_CHECK(logits.dim() == 2 && (logits.numel() == 0 || logits.size(1) == 1 || logits.stride(1) == 1),
              "mmf: distill: logits must be [rows, vocab] with unit column stride");
  a.logits = logits.data_ptr();
  a.ld = logits.size(0) > 1 ? logits.stride(0) : 0;
}

// A gradient of the logits whose rows lie as the logits' rows do against 16-byte boundaries (the
// kernels move both through the same vectors): (the whole buffer, the rows in it).
std::pair<Tensor, Tensor> grad_like(const Tensor& logits) {
  const int64_t es = logits.element_size(), v = 16 / es, rows = logits.size(0), vocab = logits.size(1);
  const int64_t ld = rows > 1 ? logits.stride(0) : 0;
  const int64_t ld_g = vocab + ((ld - vocab) % v + v) % v;
  const int64_t off = static_cast<int64_t>(reinterpret_cast<uintptr_t>(logits.data_ptr()) % 16) / es;
  Tensor flat = torch::empty({off + rows * ld_g}, logits.options());
  return {flat, flat.as_strided({rows, vocab}, {ld_g, 1}, off)};
}

// int32 [2]: rows with a slot, rows with a target (where targets have a weight)
Tensor distill_count(const Tensor& like, int64_t vocab, const Tensor& ids, const Tensor& teacher,
                     const OptTensor& targets, int64_t ignore_index, double alpha) {
  const c10::cuda::CUDAGuard guard(like.device());
  const auto a = distill_args(like, ids.size(0), vocab, ids, teacher, targets, {1.0, alpha, ignore_index});
  Tensor counts = torch::empty({2}, like.options().dtype(torch::kInt32));
  mmf::distill_count(a, counts.data_ptr<int>(), cur_stream());
  return counts;
}

// Overwrites the logits [rows, vocab] with their gradient (unless that is not wanted); the loss of each row
// goes to `loss`.
void distill_rows_(const Tensor& logits, const Tensor& ids, const Tensor& teacher, const OptTensor& targets, double tau,
                   double alpha, int64_t ignore_index, const Tensor& counts, const Tensor& loss, bool gradient) {
  const c10::cuda::CUDAGuard guard(logits.device());
  auto a = distill_args(logits, logits.size(0), logits.size(1), ids, teacher, targets, {tau, alpha, ignore_index});
  put_logits(a, logits);
  TORCH_CHECK(counts.device() == logits.device() && counts.scalar_type() == torch::kInt32 && counts.numel() == 2,
              "mmf: distill: counts must be int32 [2]");
  TORCH_CHECK(loss.device() == logits.device() && loss.scalar_type() == torch::kFloat32 && loss.is_contiguous() &&
                  loss.numel() == a.rows, "mmf: distill: loss must be contiguous fp32 [rows]");
  a.grad = gradient ? logits.data_ptr() : nullptr;
  a.grad_ld = a.ld;
  a.counts = counts.data_ptr<int>();
  a.loss = loss.data_ptr<float>();
  mmf::distill_rows(a, cur_stream());
}

Tensor distill_sum(const Tensor& loss) {
  check_cuda(loss, "loss");
  TORCH_CHECK(loss.scalar_type() == torch::kFloat32 && loss.is_contiguous(), "mmf: distill: loss must be contiguous fp32");
  const c10::cuda::CUDAGuard guard(loss.device());
  Tensor out = torch::empty({}, loss.options());
  mmf::distill_sum(loss.data_ptr<float>(), loss.numel(), out.data_ptr<float>(), cur_stream());
  return out;
}

// x *= s, s a one-element fp32 CUDA tensor read on the device; nothing is moved when it is 1
void distill_scale_(const Tensor& x, const Tensor& s) {
  check_cuda(x, "x");
  TORCH_CHECK(x.is_contiguous() && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0 && s.device() == x.device() &&
                  s.scalar_type() == torch::kFloat32 && s.numel() == 1,
              "mmf: distill_scale_ takes a contiguous x on a 16-byte boundary and a one-element fp32 scale");
  const c10::cuda::CUDAGuard guard(x.device());
  mmf::distill_scale(x.data_ptr(), s.data_ptr<float>(), x.numel(), dtype_of(x, "x"), cur_stream());
}

// Whether the gradient is formed in the forward pass (one reading of the logits for both), to be
// multiplied by the incoming gradient when that is not 1: where there is one such factor, for types
// whose range does not need it beforehand.  fp16 gradients of a mean underflow without their loss
// scale, and a factor for each row would cost a second pass as a rule: both form it in the backward
// pass, from the logits and four kept values a row.  4096 x 128256 bf16, forward and backward: 434 us
// formed in the forward where the incoming gradient is 1, 770 where it is not, 601 formed in the backward.
// A factor that is no power of two rounds a bf16 gradient a second time: at most a step of the type instead
// of half of one, kept for the pass over the logits that it saves where the factor is 1.
bool grad_in_forward(const Tensor& logits, bool mean) { return mean && logits.scalar_type() != torch::kFloat16; }

Tensor distill_forward(const Tensor& logits, const Tensor& ids, const Tensor& teacher, const OptTensor& targets,
                       const DistillConf& c, bool mean, const Tensor& grad, const Tensor& stats,
                       Tensor* counts_kept = nullptr) {
  auto a = distill_args(logits, logits.size(0), logits.size(1), ids, teacher, targets, c);
  put_logits(a, logits);
  if (grad.defined()) {
    a.grad = grad.data_ptr();
    a.grad_ld = grad.stride(0);
  }
  if (stats.defined()) a.stats = stats.data_ptr<float>();
  Tensor loss = torch::empty({a.rows}, logits.options().dtype(torch::kFloat32));
  a.loss = loss.data_ptr<float>();
  Tensor counts;
  if (mean) {
    counts = distill_count(logits, a.vocab, ids, teacher, targets, c.ignore_index, c.alpha);
    a.counts = counts.data_ptr<int>();
    a.behind_count = true;
    if (counts_kept) *counts_kept = counts;
  }
  mmf::distill_rows(a, cur_stream());
  return mean ? distill_sum(loss) : loss;
}

class DistillFn : public torch::autograd::Function<DistillFn> {
 public:
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& ids, const Tensor& teacher,
                        const OptTensor& targets, double tau, double alpha, int64_t ignore_index, bool mean) {
    at::AutoDispatchBelowADInplaceOrView below;
    const c10::cuda::CUDAGuard guard(logits.device());
    const DistillConf c{tau, alpha, ignore_index};
    auto& d = ctx->saved_data;
    if (grad_in_forward(logits, mean)) {
      auto [flat, grad] = grad_like(logits);
      d["flat"] = flat;
      d["grad"] = grad;
      return distill_forward(logits, ids, teacher, targets, c, mean, grad, Tensor());
    }
    Tensor stats = torch::empty({logits.size(0), 4}, logits.options().dtype(torch::kFloat32));
    Tensor counts;
    Tensor loss = distill_forward(logits, ids, teacher, targets, c, mean, Tensor(), stats, &counts);
    ctx->save_for_backward({logits, ids, teacher, targets.value_or(Tensor()), stats, counts});
    d["tau"] = tau;
    d["alpha"] = alpha;
    d["ignore"] = ignore_index;
    d["mean"] = mean;
    return loss;
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) {
    refuse_second_order("distill");
    auto& d = ctx->saved_data;
    variable_list out(8);
    Tensor up = g[0].to(torch::kFloat32).contiguous();
    const c10::cuda::CUDAGuard guard(up.device());
    if (!d.count("tau")) {  // formed in the forward
      TORCH_CHECK(d.count("grad"), "mmf: distill: this loss keeps its gradient for one backward pass; its graph cannot "
                                   "be gone through a second time");
      distill_scale_(d["flat"].toTensor(), up);
      out[0] = d["grad"].toTensor();
      d.clear();
      return out;
    }
    const auto s = ctx->get_saved_variables();  // taken once: a checkpoint hands each out a single time
    const Tensor& logits = s[0];
    const bool mean = d["mean"].toBool();
    const OptTensor targets = s[3].defined() ? OptTensor(s[3]) : OptTensor();
    auto a = distill_args(logits, logits.size(0), logits.size(1), s[1], s[2], targets,
                          {d["tau"].toDouble(), d["alpha"].toDouble(), d["ignore"].toInt()});
    put_logits(a, logits);
    if (mean) a.counts = s[5].data_ptr<int>();
    out[0] = grad_like(logits).second;
    a.grad = out[0].data_ptr();
    a.grad_ld = out[0].stride(0);
    a.stats = s[4].data_ptr<float>();
    a.upstream = up.data_ptr<float>();
    a.upstream_rows = !mean;
    mmf::distill_grad(a, cur_stream());
    return out;
  }
};

// logits [..., vocab], ids and teacher [..., top], targets [...]
Tensor distill(const Tensor& logits, const Tensor& ids, const Tensor& teacher, const OptTensor& targets, double tau,
               double alpha, int64_t ignore_index, bool mean) {
  const OptTensor given(logits), slots(ids), of(teacher);
  check_memory("distill", {&given, &slots, &of, &targets});
  const int64_t lead = logits.dim() - 1;
  TORCH_CHECK(lead >= 0 && ids.dim() == lead + 1 && ids.sizes().slice(0, lead) == logits.sizes().slice(0, lead) &&
                  teacher.sizes() == ids.sizes() && (!targets.has_value() || targets->sizes() == logits.sizes().slice(0, lead)),
              "mmf: distill: the teacher's slots and the targets must have the logits' leading dimensions");
  TORCH_CHECK(!(at::GradMode::is_enabled() && teacher.requires_grad()), "mmf: distill: the teacher takes no gradient");
  refuse_forward_mode("distill", {&given, &of});
  TORCH_CHECK(tau >= 1e-3 && tau <= 1e3 && alpha >= 0 && alpha <= 1 && (alpha == 1 || targets.has_value()),
              "mmf: distill: temperature, alpha or targets out of range");
  const int64_t vocab = logits.size(-1), top = ids.size(-1);
  TORCH_CHECK(vocab >= 1 && top >= 1, "mmf: distill: an empty vocabulary, or no slot");
  int64_t rows = 1;
  for (int64_t i = 0; i < lead; ++i) rows *= logits.size(i);
  Tensor z = lead == 1 ? logits : logits.reshape({rows, vocab});
  if (z.stride(1) != 1 && vocab > 1) z = z.contiguous();
  const Tensor i = (lead == 1 ? ids : ids.reshape({rows, top})).contiguous();
  const Tensor t = (lead == 1 ? teacher : teacher.reshape({rows, top})).contiguous();
  const OptTensor y = targets.has_value() ? OptTensor((lead == 1 ? *targets : targets->reshape({rows})).contiguous()) : targets;
  const OptTensor ol(z);
  Tensor loss;
  if (wants_grad({&ol})) {
    loss = DistillFn::apply(z, i, t, y, tau, alpha, ignore_index, mean);
  } else {
    const c10::cuda::CUDAGuard guard(z.device());
    loss = distill_forward(z, i, t, y, {tau, alpha, ignore_index}, mean, Tensor(), Tensor());
  }
  return mean || lead == 1 ? loss : loss.reshape(logits.sizes().slice(0, lead));
}

}  // namespace

void register_lm_ops(pybind11::module_& m) {
  m.def("rotary", &rotary);
  m.def("block_norm", &block_norm);
  m.def("distill", &distill);
  m.def("distill_count", &distill_count, py::arg("like"), py::arg("vocab"), py::arg("ids"), py::arg("teacher"),
        py::arg("targets"), py::arg("ignore_index"), py::arg("alpha") = 0.0);
  m.def("distill_rows_", &distill_rows_, py::arg("logits"), py::arg("ids"), py::arg("teacher"), py::arg("targets"),
        py::arg("tau"), py::arg("alpha"), py::arg("ignore_index"), py::arg("counts"), py::arg("loss"),
        py::arg("gradient") = true);
  m.def("distill_sum", &distill_sum);
  m.def("distill_scale_", &distill_scale_);
}
