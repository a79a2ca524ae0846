// The fine-tuning operators as autograd nodes: what the Python layer calls after it has checked the arguments. A node's
// backward runs in C++ on the engine's thread, without the interpreter: for the smaller calls the host's time is the
// operator's time (a training call of a few microseconds on the GPU took 105 to 145 us as Python Functions over
// ctypes). The kernels are libmeep2b's, through its C ABI; buffers come from torch's allocator on the current stream.
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/extension.h>

#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/meep2b.h"

namespace {

using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

// The exceptions the ctypes layer raises for the same statuses.
void check(int status, const char* what) {
  if (status == MEEP2B_OK) return;
  const std::string text = std::string(what) + ": " + meep2b_status_string(status);
  switch (status) {
    case MEEP2B_ERR_SHAPE:
    case MEEP2B_ERR_ALIGN: TORCH_CHECK_VALUE(false, text); break;
    case MEEP2B_ERR_DTYPE: TORCH_CHECK_TYPE(false, text); break;
    case MEEP2B_ERR_UNSUPPORTED: TORCH_CHECK_NOT_IMPLEMENTED(false, text); break;
    default: TORCH_CHECK(false, text);
  }
}

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

bool aligned(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0; }

template <typename T>
T* data(const Tensor& t) {
  return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}

int32_t dtype_of(const Tensor& t) { return t.scalar_type() == at::kBFloat16 ? MEEP2B_BF16 : MEEP2B_F32; }

bool wants(const Tensor& t) { return at::GradMode::is_enabled() && t.requires_grad(); }

// The nodes know the backward direction alone: a tangent of forward-mode differentiation would be lost without a word.
void refuse_tangents(const char* name, at::ArrayRef<Tensor> inputs) {
  for (const Tensor& t : inputs)
    TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), name, " has no forward-mode derivative");
}

Tensor dense(const Tensor& t) { return t.clone(at::MemoryFormat::Contiguous); }

// The results of a backward pass that was asked to be differentiable itself: an error if they are.
variable_list once(variable_list grads, const char* name) {
  if (!at::GradMode::is_enabled()) return grads;
  for (Tensor& g : grads)
    if (g.defined()) g = g.detach().set_requires_grad(true);  // so that the error below becomes their history
  auto refuse = std::make_shared<torch::autograd::DelayedError>(
      std::string(name) + " is not differentiable twice", static_cast<int64_t>(grads.size()));
  return (*refuse)(std::move(grads));
}

template <typename N>
std::shared_ptr<N> make_node(torch::autograd::edge_list edges) {
  auto node = std::shared_ptr<N>(new N(), torch::autograd::deleteNode);
  node->set_next_edges(std::move(edges));
  return node;
}

// ------------------------------------------------------------------------------------------------ heads

// (B, T, heads, dim) that 16-byte loads can address: itself, or a copy.
Tensor heads(const Tensor& t) {
  const int64_t vec = 16 / t.element_size();
  const auto s = t.strides();
  return s[3] == 1 && s[0] % vec == 0 && s[1] % vec == 0 && s[2] % vec == 0 && aligned(t) ? t : dense(t);
}

// The type the norm weights are read in: the heads' own where both have it, else float32, which holds every other.
at::ScalarType weight_type(const Tensor& x, const Tensor& wq, const Tensor& wk) {
  return wq.scalar_type() == x.scalar_type() && wk.scalar_type() == x.scalar_type() ? x.scalar_type() : at::kFloat;
}

Tensor vector_as(const Tensor& w, at::ScalarType type) {
  Tensor v = w.scalar_type() == type ? w : w.to(type);
  return v.is_contiguous() && aligned(v) ? v : dense(v);
}

struct HeadsCall {
  Tensor q, k, wq, wk, cos, sin, positions;
  meep2b_head_norm args = {};

  HeadsCall(const Tensor& q_, const Tensor& k_, const Tensor& wq_, const Tensor& wk_, const Tensor& cos_,
            const Tensor& sin_, const Tensor& positions_, double eps)
      : q(heads(q_)), k(heads(k_)), wq(vector_as(wq_, weight_type(q_, wq_, wk_))),
        wk(vector_as(wk_, weight_type(q_, wq_, wk_))), cos(cos_), sin(sin_), positions(positions_) {
    args.q = data<void>(q), args.k = data<void>(k);
    args.batch = q.size(0), args.length = q.size(1);
    args.q_heads = static_cast<int32_t>(q.size(2)), args.kv_heads = static_cast<int32_t>(k.size(2));
    args.dim = static_cast<int32_t>(q.size(3)), args.half = static_cast<int32_t>(cos.size(1));
    for (int i = 0; i < 3; ++i) args.q_stride[i] = q.stride(i), args.k_stride[i] = k.stride(i);
    args.dtype = dtype_of(q), args.angle_dtype = dtype_of(cos);
    args.weight_f32 = wq.scalar_type() == at::kFloat;
    args.q_weight = data<void>(wq), args.k_weight = data<void>(wk);
    args.cos = data<void>(cos), args.sin = data<void>(sin);
    args.ld_cos = cos.stride(0), args.ld_sin = sin.stride(0), args.angles = cos.size(0);
    args.positions = data<int64_t>(positions);
    args.eps = static_cast<float>(eps);
  }
};

struct QkNormRopeBackward : torch::autograd::Node {
  SavedVariable q, k, wq, wk, cos, sin, positions;
  double eps = 0.0;

  std::string name() const override { return "QkNormRopeBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (auto* s : {&q, &k, &wq, &wk, &cos, &sin, &positions}) s->reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list out(4);
    if (!grads[0].defined() && !grads[1].defined()) return out;
    const Tensor wq_ = wq.unpack(), wk_ = wk.unpack();
    HeadsCall c(q.unpack(), k.unpack(), wq_, wk_, cos.unpack(), sin.unpack(), positions.unpack(), eps);
    const Tensor dy = grads[0].defined() ? heads(grads[0]) : at::zeros(c.q.sizes(), c.q.options());
    const Tensor dz = grads[1].defined() ? heads(grads[1]) : at::zeros(c.k.sizes(), c.k.options());
    out[0] = at::empty(c.q.sizes(), c.q.options());
    out[1] = at::empty(c.k.sizes(), c.k.options());
    c.args.q_out = data<void>(out[0]), c.args.k_out = data<void>(out[1]);
    c.args.dq_out = data<void>(dy), c.args.dk_out = data<void>(dz);
    for (int i = 0; i < 3; ++i) c.args.dq_out_stride[i] = dy.stride(i), c.args.dk_out_stride[i] = dz.stride(i);
    Tensor partial;
    if (task_should_compute_output(2) || task_should_compute_output(3)) {
      out[2] = at::empty(c.wq.sizes(), c.wq.options());
      out[3] = at::empty(c.wk.sizes(), c.wk.options());
      partial = at::empty({meep2b_head_norm_partials() * c.q.size(3)}, c.q.options().dtype(at::kFloat));
      c.args.dq_weight = data<void>(out[2]), c.args.dk_weight = data<void>(out[3]);
      c.args.partial = data<float>(partial);
    }
    check(meep2b_head_norm_rotate_backward(&c.args, stream_of(c.q)), "meep2b_head_norm_rotate_backward");
    if (out[2].defined()) {
      if (wq_.scalar_type() != out[2].scalar_type()) out[2] = out[2].to(wq_.scalar_type());
      if (wk_.scalar_type() != out[3].scalar_type()) out[3] = out[3].to(wk_.scalar_type());
    }
    return once(std::move(out), "qk_norm_rope");
  }
};

std::tuple<Tensor, Tensor> qk_norm_rope(const Tensor& q, const Tensor& k, const Tensor& wq, const Tensor& wk,
                                        const Tensor& cos_, const Tensor& sin_, const std::optional<Tensor>& positions,
                                        double eps) {
  refuse_tangents("qk_norm_rope", {q, k, wq, wk, cos_, sin_});
  const Tensor cos = cos_.detach(), sin = sin_.detach();
  const c10::cuda::CUDAGuard guard(q.device());
  const bool graph = wants(q) || wants(k) || wants(wq) || wants(wk);
  const Tensor pos = positions.value_or(Tensor());
  Tensor q_out, k_out;
  {
    const at::NoGradGuard none;
    HeadsCall c(q, k, wq, wk, cos, sin, pos, eps);
    q_out = at::empty(q.sizes(), c.q.options()), k_out = at::empty(k.sizes(), c.k.options());
    c.args.q_out = data<void>(q_out), c.args.k_out = data<void>(k_out);
    check(meep2b_head_norm_rotate(&c.args, stream_of(c.q)), "meep2b_head_norm_rotate");
  }
  if (graph) {
    auto node = make_node<QkNormRopeBackward>(torch::autograd::collect_next_edges(q, k, wq, wk));
    node->q = SavedVariable(q, false), node->k = SavedVariable(k, false);
    node->wq = SavedVariable(wq, false), node->wk = SavedVariable(wk, false);
    node->cos = SavedVariable(cos, false), node->sin = SavedVariable(sin, false);
    node->positions = SavedVariable(pos, false);
    node->eps = eps;
    torch::autograd::set_history(q_out, node);
    torch::autograd::set_history(k_out, node);
  }
  return {q_out, k_out};
}

// ------------------------------------------------------------------------------------------------ balance

struct BalanceCall {
  std::vector<Tensor> rows;
  std::vector<const void*> table;
  meep2b_balance args = {};

  // float32 words of the kernel's sums
  static int64_t words(int64_t experts) {
    return static_cast<int64_t>(meep2b_balance_workspace_bytes(static_cast<int32_t>(experts)) / sizeof(float));
  }
  // work: the kernel's sums, then the coefficients that the backward pass reads
  BalanceCall(const std::vector<Tensor>& logits, int64_t top_k, const Tensor& mask, const Tensor& work) {
    rows.reserve(logits.size()), table.reserve(logits.size());
    for (const Tensor& x : logits) {
      rows.push_back(x.is_contiguous() ? x : dense(x));
      table.push_back(data<void>(rows.back()));
    }
    args.logits = table.data();
    args.layers = static_cast<int32_t>(rows.size()), args.experts = static_cast<int32_t>(rows[0].size(1));
    args.tokens = rows[0].size(0), args.top_k = static_cast<int32_t>(top_k), args.dtype = dtype_of(rows[0]);
    args.mask = data<uint8_t>(mask);
    args.workspace = data<void>(work);
    args.coef = data<float>(work) + words(args.experts);
  }
};

struct BalanceLossBackward : torch::autograd::Node {
  std::vector<SavedVariable> logits;
  SavedVariable mask, work;
  int64_t top_k = 0;

  std::string name() const override { return "BalanceLossBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (auto& s : logits) s.reset_data();
    mask.reset_data(), work.reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list out(logits.size());
    if (!grads[0].defined()) return out;
    std::vector<Tensor> each;
    each.reserve(logits.size());
    for (auto& s : logits) each.push_back(s.unpack());
    const Tensor work_ = work.unpack(), mask_ = mask.unpack();
    BalanceCall c(each, top_k, mask_, work_);
    const Tensor upstream = grads[0].to(at::kFloat);
    // one allocation for all layers: the gradients are its slices
    std::vector<int64_t> sizes = {static_cast<int64_t>(each.size()), c.rows[0].size(0), c.rows[0].size(1)};
    if (each.size() == 1) out[0] = at::empty(c.rows[0].sizes(), c.rows[0].options());
    else out = at::empty(sizes, c.rows[0].options()).unbind(0);
    std::vector<void*> outs;
    outs.reserve(out.size());
    for (const Tensor& x : out) outs.push_back(data<void>(x));
    c.args.grads = outs.data(), c.args.upstream = data<float>(upstream);
    check(meep2b_balance_loss_backward(&c.args, stream_of(c.rows[0])), "meep2b_balance_loss_backward");
    return once(std::move(out), "balance_loss");
  }
};

std::tuple<Tensor, Tensor> balance_loss(const std::vector<Tensor>& logits, int64_t top_k,
                                        const std::optional<Tensor>& mask, const std::vector<Tensor>& index) {
  refuse_tangents("balance_loss", logits);
  const Tensor& first = logits[0];
  const c10::cuda::CUDAGuard guard(first.device());
  bool graph = false;
  for (const Tensor& x : logits) graph = graph || wants(x);
  const int64_t layers = static_cast<int64_t>(logits.size()), experts = first.size(1);
  const auto f32 = first.options().dtype(at::kFloat);
  Tensor loss, counts, work;
  const Tensor mask_ = mask.value_or(Tensor());
  {
    const at::NoGradGuard none;
    work = at::empty({BalanceCall::words(experts) + experts}, f32);
    loss = at::empty({}, f32);
    const auto i64 = first.options().dtype(at::kLong);
    counts = layers == 1 ? at::empty({experts}, i64) : at::empty({layers, experts}, i64);
    BalanceCall c(logits, top_k, mask_, work);
    std::vector<const int64_t*> ids;
    ids.reserve(index.size());
    for (const Tensor& i : index) ids.push_back(data<int64_t>(i));
    c.args.index = ids.empty() ? nullptr : ids.data();
    c.args.counts = data<int64_t>(counts), c.args.loss = data<float>(loss);
    check(meep2b_balance_loss(&c.args, stream_of(first)), "meep2b_balance_loss");
  }
  if (graph) {
    auto node = make_node<BalanceLossBackward>(torch::autograd::collect_next_edges(logits));
    node->logits.reserve(logits.size());
    for (const Tensor& x : logits) node->logits.emplace_back(x, false);
    node->mask = SavedVariable(mask_, false), node->work = SavedVariable(work, false);
    node->top_k = top_k;
    torch::autograd::set_history(loss, node);
  }
  return {loss, counts};
}

// ------------------------------------------------------------------------------------------------ vocabulary loss

// Rows that TMA and 16-byte loads can address: the tensor itself, or a copy.
Tensor rows_of(const Tensor& t) {
  return t.stride(1) == 1 && t.stride(0) % 8 == 0 && t.stride(0) >= t.size(1) && aligned(t) ? t : dense(t);
}

struct Plan {
  int64_t rows_pad = 0, piece_cols = 0;
  int32_t planes = 0;
};

// One buffer of parts that each start on 256 bytes.
struct Parts {
  std::vector<int64_t> at;
  int64_t end = 0;
  int add(int64_t bytes) {
    at.push_back(end);
    end += (bytes + 255) & ~int64_t(255);
    return static_cast<int>(at.size()) - 1;
  }
  Tensor take(const Tensor& like) { return at::empty({end}, like.options().dtype(at::kByte)); }
};

// kept: what the passes keep of every row: state (8), flags (rows_pad / 256), source, slot and target, the row values.
meep2b_linear_ce ce_args(const Tensor& weight, const Tensor& targets, int64_t ignore, int64_t reduction,
                         const Plan& plan, const Tensor& kept) {
  meep2b_linear_ce a = {};
  a.tokens = targets.numel(), a.hidden_size = weight.size(1);
  a.weight = data<void>(weight), a.vocab = weight.size(0), a.ld_weight = weight.stride(0);
  a.targets = data<int64_t>(targets), a.ignore_index = ignore, a.reduction = static_cast<int32_t>(reduction);
  a.planes = plan.planes, a.rows_pad = plan.rows_pad, a.piece_cols = plan.piece_cols;
  a.state = data<int32_t>(kept);
  a.flags = a.state + 8;
  a.source = a.flags + plan.rows_pad / 256;
  a.slot = a.source + plan.rows_pad;
  a.target = a.slot + plan.rows_pad;
  a.row_values = reinterpret_cast<float*>(a.target + plan.rows_pad);
  return a;
}

struct LinearCrossEntropyBackward : torch::autograd::Node {
  SavedVariable weight, targets, kept, last;  // last: the copied rows with a trained head, else the gradient's planes
  Plan plan;
  int64_t ignore = 0, reduction = 0;
  bool trained = false;

  std::string name() const override { return "LinearCrossEntropyBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (auto* s : {&weight, &targets, &kept, &last}) s->reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list out(2);
    if (!grads[0].defined()) return out;
    const Tensor w = rows_of(weight.unpack()), t = targets.unpack(), kept_ = kept.unpack(), last_ = last.unpack();
    const Tensor upstream = grads[0].to(at::kFloat).contiguous();
    const bool hidden = task_should_compute_output(0), head = trained && task_should_compute_output(1);
    const int64_t size = w.size(1);
    meep2b_linear_ce a = ce_args(w, t, ignore, reduction, plan, kept_);
    a.upstream = data<float>(upstream);
    if (hidden) out[0] = at::empty({t.numel(), size}, w.options()), a.d_hidden = data<void>(out[0]);
    Tensor scratch;
    if (trained) {  // the planes are computed here, with or without the head's gradient
      if (head) out[1] = at::empty({w.size(0), size}, w.options()), a.d_weight = data<void>(out[1]);
      Parts parts;
      const int piece = parts.add(2 * plan.rows_pad * plan.piece_cols);
      const int acc = parts.add(hidden ? 4 * int64_t(plan.planes) * plan.rows_pad * size : 0);
      scratch = parts.take(w);
      a.compact = data<void>(last_);
      a.piece = data<uint8_t>(scratch) + parts.at[piece];
      if (hidden) a.acc = reinterpret_cast<float*>(data<uint8_t>(scratch) + parts.at[acc]);
    } else {
      a.acc = data<float>(last_);
    }
    if (hidden || head) check(meep2b_linear_ce_backward(&a, stream_of(w)), "meep2b_linear_ce_backward");
    return once(std::move(out), "linear_cross_entropy");
  }
};

Tensor linear_cross_entropy(const Tensor& hidden, const Tensor& weight, const Tensor& targets, int64_t ignore,
                            int64_t reduction, int64_t piece_cols, int64_t planes) {
  refuse_tangents("linear_cross_entropy", {hidden, weight});
  const c10::cuda::CUDAGuard guard(hidden.device());
  const bool trained = wants(weight), accumulate = wants(hidden) && !trained;
  Plan plan;
  const int64_t size = weight.size(1), vocab = weight.size(0);
  check(meep2b_linear_ce_plan(targets.numel(), size, vocab, &plan.rows_pad, &plan.piece_cols, &plan.planes),
        "meep2b_linear_ce_plan");
  if (piece_cols > 0) plan.piece_cols = piece_cols;
  if (planes > 0) plan.planes = static_cast<int32_t>(planes);
  Tensor loss, kept, rows, acc;
  {
    const at::NoGradGuard none;
    const Tensor h = rows_of(hidden), w = rows_of(weight);
    const auto f32 = h.options().dtype(at::kFloat);
    kept = at::empty({8 + plan.rows_pad / 256 + 8 * plan.rows_pad}, h.options().dtype(at::kInt));
    loss = reduction == MEEP2B_REDUCE_NONE ? at::empty({targets.numel()}, f32) : at::empty({}, f32);
    if (trained) rows = at::empty({plan.rows_pad, size}, h.options());
    if (accumulate) acc = at::empty({plan.planes, plan.rows_pad, size}, f32);
    meep2b_linear_ce a = ce_args(w, targets, ignore, reduction, plan, kept);
    Parts parts;
    const int part = parts.add(4 * 2 * ((vocab + 255) / 256) * plan.rows_pad), row_loss = parts.add(4 * plan.rows_pad);
    const int compact = parts.add(trained ? 0 : 2 * plan.rows_pad * size);
    const int piece = parts.add(accumulate ? 2 * plan.rows_pad * plan.piece_cols : 0);
    const Tensor scratch = parts.take(h);
    uint8_t* const base = data<uint8_t>(scratch);
    a.hidden = data<void>(h), a.ld_hidden = h.stride(0);
    a.compact = trained ? data<void>(rows) : base + parts.at[compact];
    a.part = reinterpret_cast<float*>(base + parts.at[part]);
    a.row_loss = reinterpret_cast<float*>(base + parts.at[row_loss]);
    a.loss = data<float>(loss);
    if (accumulate) a.acc = data<float>(acc), a.piece = base + parts.at[piece];
    else a.piece_cols = 0;
    check(meep2b_linear_ce_forward(&a, stream_of(h)), "meep2b_linear_ce_forward");
  }
  if (trained || accumulate) {
    auto node = make_node<LinearCrossEntropyBackward>(torch::autograd::collect_next_edges(hidden, weight));
    node->weight = SavedVariable(weight, false), node->targets = SavedVariable(targets, false);
    node->kept = SavedVariable(kept, false), node->last = SavedVariable(trained ? rows : acc, false);
    node->plan = plan, node->ignore = ignore, node->reduction = reduction, node->trained = trained;
    torch::autograd::set_history(loss, node);
  }
  return loss;
}

}  // namespace

PYBIND11_MODULE(_native, m) {
  m.attr("built_for") = MEEP2B_NATIVE_TAG;
  // without the interpreter's lock, as ctypes calls: a full launch queue blocks no other thread
  m.def("qk_norm_rope", &qk_norm_rope, py::call_guard<py::gil_scoped_release>());
  m.def("balance_loss", &balance_loss, py::call_guard<py::gil_scoped_release>());
  m.def("linear_cross_entropy", &linear_cross_entropy, py::call_guard<py::gil_scoped_release>());
}
