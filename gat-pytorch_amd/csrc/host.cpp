// Host side of the graph-transformer operators: torch autograd nodes over libgatx's C-ABI, as the
// Python module gatx._host. A small call of one of them is host-bound, and its backward runs on the
// autograd engine's own thread: nodes in C++ need neither the interpreter nor its lock there (a
// Cora distillation step with Python nodes took 108 us around 17 us of kernels).
// Everything is allocated from torch's allocator and launched on the device's current stream;
// libgatx.so is loaded by gatx/_lib.py before this module and resolves its symbols.
#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>

#include <unordered_set>

#include "../../include/gatx.h"

namespace {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
using Opt = std::optional<Tensor>;

void run(int rc, const char* what) {
  TORCH_CHECK(rc == 0, "gatx ", what, " failed (code ", rc, "): ", gatx_last_error());
}
gatx_stream_t stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}
int code(at::ScalarType t) {
  return t == at::kFloat ? GATX_F32 : t == at::kBFloat16 ? GATX_BF16 : t == at::kHalf ? GATX_F16 : -1;
}
Tensor of(const Opt& t) { return t ? *t : Tensor(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* fptr(const Tensor& t) { return (float*)ptr(t); }
Tensor f32(const Tensor& t) { return t.defined() && t.scalar_type() != at::kFloat ? t.to(at::kFloat) : t; }
Tensor packed(const Tensor& t) { return t.defined() ? t.contiguous() : t; }
Tensor floats(const Tensor& like, at::IntArrayRef size) {
  return at::empty(size, like.options().dtype(at::kFloat));
}
Tensor bytes(const Tensor& like, size_t n) {
  return at::empty({(int64_t)n}, like.options().dtype(at::kByte));
}

// The second derivative is refused when it is asked for, not when the first is (create_graph may be
// on for other parts of the graph).
variable_list once(variable_list&& grads, const char* what) {
  if (!at::GradMode::is_enabled()) return std::move(grads);
  variable_list out;
  for (auto& g : grads) out.push_back(g.defined() ? g.detach().set_requires_grad(true) : g);
  torch::autograd::DelayedError error(std::string("gatx: ") + what + " has no second derivative",
                                      (int64_t)out.size());
  return error.apply(std::move(out));
}

// Forward-mode derivatives would be dropped without a word.
template <typename... In>
void no_tangents(const char* what, const In&... inputs) {
  for (const Tensor* t : {&inputs...})
    TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), "gatx: ", what,
                                " has no forward-mode derivative");
}

// A captured backward into a leaf that an eager graph on the default stream still holds would make
// that stream, which cannot take part in a capture, wait for the captured one: the capture breaks
// on the engine's thread, where nothing can be caught, and the process ends. So it is looked for before
// the first launch, over everything this backward goes on to (a leaf can be behind the cast of a 16-bit
// parameter, a view, any operation); leaves whose gradients nobody asks for do not count.
void check_capture(Node& node, const char* what) {
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  std::vector<Node*> todo = {&node};
  std::unordered_set<Node*> seen = {&node};
  while (!todo.empty()) {
    Node* at = todo.back();
    todo.pop_back();
    for (size_t i = 0; i < at->num_outputs(); ++i) {
      if (!at->task_should_compute_output(i)) continue;
      Node* next = at->next_edge(i).function.get();
      if (!next || !seen.insert(next).second) continue;
      todo.push_back(next);
      if (next->num_outputs() != 0) continue;
      const auto stream = next->stream();
      TORCH_CHECK(!stream || stream->id() != 0, "gatx: ", what,   // (0: the default stream)
                  ": the captured backward reaches a leaf of an autograd graph that is alive on the "
                  "default stream; drop that graph's results, or run the eager steps on the capture's "
                  "stream");
    }
  }
}

template <typename N, typename... In>
std::shared_ptr<N> node_for(const In&... inputs) {
  std::shared_ptr<N> n(new N(), torch::autograd::deleteNode);
  n->set_next_edges(torch::autograd::collect_next_edges(inputs...));
  return n;
}

// ------------------------------------------------------------------ norms
struct Rows {
  Tensor t;        // undefined: none
  int64_t ld = 0;
};
// rows x columns, in place where only the rows are strided.
Rows rows_of(const Tensor& x) {
  if (!x.defined()) return {};
  Tensor t = x.dim() == 2 ? x : x.reshape({-1, x.size(-1)});
  if (t.size(1) > 1 && t.stride(1) != 1) t = t.contiguous();
  return {t, t.size(0) > 1 ? t.stride(0) : t.size(1)};
}

void check_norm(const char* what, const Tensor& x,
                std::initializer_list<std::pair<const char*, Tensor>> vectors,
                std::initializer_list<std::pair<const char*, Tensor>> rows) {
  TORCH_CHECK(code(x.scalar_type()) >= 0, "gatx: ", what,
              " takes float32, bfloat16 or float16, got ", x.scalar_type());
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= 8192, "gatx: ", what,
                    ": 1 to 8192 columns, got ", x.sizes());
  for (auto& [name, t] : vectors) {
    if (!t.defined()) continue;
    TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == x.size(-1) && t.is_floating_point(), "gatx: ",
                      what, ": ", name, " is a vector of ", x.size(-1), ", got ", t.sizes(), " ",
                      t.scalar_type());
    TORCH_CHECK(t.device() == x.device(), "gatx: ", what, ": ", name, " is on ", t.device(),
                ", the rows on ", x.device());
  }
  for (auto& [name, t] : rows) {
    if (!t.defined()) continue;
    TORCH_CHECK_VALUE(t.sizes() == x.sizes() && t.scalar_type() == x.scalar_type(), "gatx: ", what,
                      ": ", name, " is ", x.sizes(), " ", x.scalar_type(), ", got ", t.sizes(), " ",
                      t.scalar_type());
    TORCH_CHECK(t.device() == x.device(), "gatx: ", what, ": ", name, " is on ", t.device(),
                ", the rows on ", x.device());
  }
  TORCH_CHECK(x.is_cuda(), "gatx: ", what, " needs HIP tensors (no CPU path)");
}

struct BlockNormBackward : public Node {
  SavedVariable h, weight, resid, gate, scale, next_weight;
  Tensor rstd_h, rstd_y;
  bool gate_rows = false, after = false;

  std::string name() const override { return "BlockNormBackward"; }
  void release_variables() override {
    for (auto* v : {&h, &weight, &resid, &gate, &scale, &next_weight}) v->reset_data();
    rstd_h.reset();
    rstd_y.reset();
  }
  variable_list apply(variable_list&& go) override {
    std::lock_guard<std::mutex> lock(mutex_);
    check_capture(*this, "block norm");
    const Tensor x = h.unpack(), w = weight.unpack(), r = resid.unpack(), g = gate.unpack(),
                 sc = scale.unpack(), nw = next_weight.unpack();
    variable_list out(6);
    {
      at::NoGradGuard no_grad;
      const Tensor gy = after ? go[0] : Tensor(), gn = !after ? go[0] : go.size() > 1 ? go[1] : Tensor();
      if (!gy.defined() && !gn.defined()) return out;
      const c10::DeviceGuard guard(x.device());
      const Rows hr = rows_of(x), rr = rows_of(r), gr = gate_rows ? rows_of(g) : Rows{packed(g), 0},
                 gyr = rows_of(gy), gnr = rows_of(gn);
      const Tensor wp = packed(w), sp = packed(sc), np = packed(nw);
      const int64_t n = hr.t.size(0), D = hr.t.size(1);
      auto rows = [&](int i) {
        return task_should_compute_output(i) ? at::empty(x.sizes(), x.options()) : Tensor();
      };
      auto cols = [&](int i) { return task_should_compute_output(i) ? floats(x, {D}) : Tensor(); };
      out[0] = rows(0);
      out[1] = cols(1);
      out[2] = rows(2);
      out[3] = gate_rows ? rows(3) : cols(3);
      out[4] = cols(4);
      // nothing reaches next_weight but through next
      if (gn.defined()) out[5] = cols(5);
      const size_t wb = gatx_block_norm_backward_workspace_bytes(n, D);
      const Tensor ws = bytes(x, wb);
      run(gatx_block_norm_backward(code(x.scalar_type()), n, D, ptr(hr.t), hr.ld, fptr(wp),
                                   ptr(rr.t), rr.ld, ptr(gr.t), gate_rows, gr.ld, fptr(sp),
                                   fptr(np), fptr(rstd_h), fptr(rstd_y), ptr(gyr.t), gyr.ld,
                                   ptr(gnr.t), gnr.ld, ptr(out[0]), ptr(out[2]), ptr(out[3]),
                                   fptr(out[1]), fptr(out[4]), fptr(out[5]), ptr(ws), wb,
                                   stream_of(x)),
          "block_norm_backward");
    }
    return once(std::move(out), "block norm");
  }
};

// (y, next); weight undefined: the norm before a block alone.
std::pair<Tensor, Tensor> block_norm(const Tensor& h, Tensor weight, const Tensor& resid, Tensor gate,
                                     Tensor scale, Tensor next_weight, bool gate_rows, double eps) {
  const c10::DeviceGuard guard(h.device());
  no_tangents("block norm", h, weight, resid, gate, scale, next_weight);
  weight = f32(weight);
  scale = f32(scale);
  next_weight = f32(next_weight);
  if (!gate_rows) gate = f32(gate);
  const bool grad = torch::autograd::compute_requires_grad(h, weight, resid, gate, scale, next_weight);
  Tensor y, next, rstd_h, rstd_y;
  {
    at::NoGradGuard no_grad;
    const Rows hr = rows_of(h), rr = rows_of(resid),
               gr = gate_rows ? rows_of(gate) : Rows{packed(gate), 0};
    const Tensor wp = packed(weight), sp = packed(scale), np = packed(next_weight);
    const int64_t n = hr.t.size(0), D = hr.t.size(1);
    if (weight.defined()) {
      y = at::empty(h.sizes(), h.options());
      if (grad) rstd_h = floats(h, {n});
    }
    if (next_weight.defined()) {
      next = at::empty(h.sizes(), h.options());
      if (grad) rstd_y = floats(h, {n});
    }
    run(gatx_block_norm(code(h.scalar_type()), n, D, ptr(hr.t), hr.ld, fptr(wp), ptr(rr.t), rr.ld,
                        ptr(gr.t), gate_rows, gr.ld, fptr(sp), fptr(np), (float)eps, ptr(y),
                        ptr(next), fptr(rstd_h), fptr(rstd_y), stream_of(h)),
        "block_norm");
  }
  if (grad) {
    auto n = node_for<BlockNormBackward>(h, weight, resid, gate, scale, next_weight);
    n->h = SavedVariable(h, false);
    n->weight = SavedVariable(weight, false);
    n->resid = SavedVariable(resid, false);
    n->gate = SavedVariable(gate, false);
    n->scale = SavedVariable(scale, false);
    n->next_weight = SavedVariable(next_weight, false);
    n->rstd_h = rstd_h;
    n->rstd_y = rstd_y;
    n->gate_rows = gate_rows;
    n->after = y.defined();
    if (y.defined()) torch::autograd::set_history(y, n);
    if (next.defined()) torch::autograd::set_history(next, n);
  }
  return {y, next};
}

Tensor norm_before(const Tensor& x, const Tensor& weight, double eps) {
  check_norm("norm_before", x, {{"weight", weight}}, {});
  return block_norm(x, {}, {}, {}, {}, weight, false, eps).second;
}

py::object norm_after(const Tensor& h, const Tensor& weight, const Opt& resid_, const Opt& gate_,
                      const Opt& scale_, const Opt& next_weight_, double eps) {
  const Tensor resid = of(resid_), gate = of(gate_), scale = of(scale_), next_weight = of(next_weight_);
  const bool gate_rows = gate.defined() && gate.dim() != 1;   // (one row's gate is a parameter's)
  check_norm("norm_after", h,
             {{"weight", weight}, {"scale", scale}, {"next_weight", next_weight},
              {"gate", gate_rows ? Tensor() : gate}},
             {{"resid", resid}, {"gate", gate_rows ? gate : Tensor()}});
  auto [y, next] = block_norm(h, weight, resid, gate, scale, next_weight, gate_rows, eps);
  if (!next.defined()) return py::cast(y);
  return py::make_tuple(y, next);
}

// ------------------------------------------------------------------ distillation
struct TopKDistillationBackward : public Node {
  SavedVariable logits, teacher, index;
  Tensor stat;   // the rows' statistics, then their number
  double temperature = 1.0;
  char reduction = 'm';

  std::string name() const override { return "TopKDistillationBackward"; }
  void release_variables() override {
    for (auto* v : {&logits, &teacher, &index}) v->reset_data();
    stat.reset();
  }
  variable_list apply(variable_list&& go) override;
};

struct Distill {
  Tensor x, teacher, index;
  int64_t n, C, ld;
  Distill(const Tensor& logits, const Tensor& t, const Tensor& i)
      : x(logits), teacher(t.contiguous()), index(i.contiguous()) {
    n = x.size(0);
    C = x.size(1);
    if (C > 1 && x.stride(1) != 1) x = x.contiguous();
    ld = n > 1 ? x.stride(0) : C;
  }
  bool wide() const { return index.scalar_type() == at::kLong; }
};

variable_list TopKDistillationBackward::apply(variable_list&& go) {
  std::lock_guard<std::mutex> lock(mutex_);
  check_capture(*this, "topk_distillation");
  const Tensor x = logits.unpack(), t = teacher.unpack(), i = index.unpack();
  variable_list out(1);
  if (!go[0].defined()) return out;
  {
    at::NoGradGuard no_grad;
    const c10::DeviceGuard guard(x.device());
    const Distill d(x, t, i);
    const Tensor g = go[0].to(at::kFloat).contiguous();
    out[0] = at::empty({d.n, d.C}, x.options());
    const float* st = fptr(stat);
    run(gatx_topk_distill_backward(code(x.scalar_type()), ptr(d.x), d.n, d.C, d.ld,
                                   code(t.scalar_type()), ptr(d.teacher), ptr(d.index), d.wide(),
                                   (int)t.size(1), (float)temperature, st, fptr(g),
                                   reduction == 'n', reduction == 'm' ? st + 4 * d.n : nullptr,
                                   ptr(out[0]), stream_of(x)),
        "topk_distill_backward");
  }
  return once(std::move(out), "topk_distillation");
}

Tensor topk_distillation(const Tensor& logits, const Tensor& teacher, const Tensor& index,
                         double temperature, const std::string& reduction) {
  const char* me = "gatx: topk_distillation";
  for (auto& [name, t] : {std::pair<const char*, const Tensor&>{"logits", logits},
                          {"teacher_logits", teacher}, {"teacher_index", index}}) {
    TORCH_CHECK(t.device() == logits.device(), me, ": ", name, " is on ", t.device(),
                ", logits on ", logits.device());
    TORCH_CHECK_VALUE(t.dim() == 2, me, ": ", name, " has two dimensions, got ", t.sizes());
  }
  TORCH_CHECK(code(logits.scalar_type()) >= 0 && code(teacher.scalar_type()) >= 0, me,
              " takes float32, bfloat16 or float16 logits, got ", logits.scalar_type(), " and ",
              teacher.scalar_type());
  TORCH_CHECK(index.scalar_type() == at::kLong || index.scalar_type() == at::kInt, me,
              ": teacher_index must be int64 or int32, got ", index.scalar_type());
  TORCH_CHECK_VALUE(teacher.sizes() == index.sizes() && logits.size(0) == index.size(0) &&
                        logits.size(1) >= 1 && index.size(1) >= 1 && index.size(1) <= 1024,
                    me, ": (rows, classes) logits and (rows, K <= 1024) teacher logits and classes, "
                    "got ", logits.sizes(), ", ", teacher.sizes(), ", ", index.sizes());
  TORCH_CHECK(!teacher.requires_grad(), me, " does not differentiate the teacher; pass "
              "teacher_logits.detach()");
  // (T^2 and 1 / T stay float32 numbers)
  TORCH_CHECK_VALUE(temperature >= 1e-18 && temperature <= 1e18, me,
                    ": temperature must be positive (1e-18 to 1e18), got ", temperature);
  TORCH_CHECK_VALUE(reduction == "mean" || reduction == "sum" || reduction == "none", me,
                    ": reduction '", reduction, "' is not mean, sum or none");
  TORCH_CHECK(logits.is_cuda(), me, " needs HIP tensors (no CPU path)");
  const c10::DeviceGuard guard(logits.device());
  no_tangents("topk_distillation", logits, teacher);
  const bool grad = torch::autograd::compute_requires_grad(logits), none = reduction == "none";
  Tensor loss, stat;
  {
    at::NoGradGuard no_grad;
    const Distill d(logits, teacher, index);
    loss = none ? floats(logits, {d.n}) : floats(logits, {});
    const size_t wb = none ? 0 : gatx_topk_distill_workspace_bytes(d.n);
    // the rows' statistics and their number, for the backward, and the workspace behind them
    stat = bytes(logits, 16 * d.n + 16 + wb);
    float* st = fptr(stat);
    run(gatx_topk_distill(code(logits.scalar_type()), ptr(d.x), d.n, d.C, d.ld,
                          code(teacher.scalar_type()), ptr(d.teacher), ptr(d.index), d.wide(),
                          (int)index.size(1), (float)temperature, none ? fptr(loss) : nullptr,
                          none ? nullptr : fptr(loss), reduction == "mean",
                          none ? nullptr : st + 4 * d.n, grad ? st : nullptr, st + 4 * d.n + 4, wb,
                          stream_of(logits)),
        "topk_distill");
  }
  if (grad) {
    auto n = node_for<TopKDistillationBackward>(logits);
    n->logits = SavedVariable(logits, false);
    n->teacher = SavedVariable(teacher, false);
    n->index = SavedVariable(index, false);
    n->stat = stat;
    n->temperature = temperature;
    n->reduction = reduction[0];
    torch::autograd::set_history(loss, n);
  }
  return loss;
}

// ------------------------------------------------------------------ attention
// (rows, heads, ...) with each row's heads packed: in place where only the rows are strided.
Rows heads_of(const Tensor& x) {
  int64_t want = 1;
  for (int64_t i = x.dim() - 1; i >= 1; --i) {
    if (x.size(i) != 1 && x.stride(i) != want) {
      const Tensor t = x.contiguous();
      return {t, t.stride(0)};
    }
    want *= x.size(i);
  }
  return {x, x.size(0) > 1 ? x.stride(0) : want};
}
// q, k, v in the kernels' layout (whole 8-element chunks, 16-byte aligned rows); one launch packs
// those that are not yet. Undefined: none.
std::array<Rows, 3> chunked(const Tensor& q, const Tensor& k, const Tensor& v, int H, int d, int dv) {
  const Tensor* in[3] = {&q, &k, &v};
  const int width[3] = {d, d, dv}, groups[3] = {2 * H, 2 * H, H};
  std::array<Rows, 3> out, from;   // (from: a source's copy lives until the launch)
  const void* src[3] = {};
  void* dst[3] = {};
  int64_t ld[3] = {}, n[3] = {};
  Tensor any;
  for (int i = 0; i < 3; ++i) {
    if (!in[i]->defined()) continue;
    const Rows& r = from[i] = heads_of(*in[i]);
    if (width[i] % 8 == 0 && (uintptr_t)r.t.data_ptr() % 16 == 0 &&
        r.ld * r.t.element_size() % 16 == 0) {
      out[i] = r;
      continue;
    }
    any = r.t;
    n[i] = r.t.size(0);
    src[i] = r.t.data_ptr();
    ld[i] = r.ld;
    out[i].t = at::empty({n[i], groups[i], (width[i] + 7) / 8 * 8}, r.t.options());
    out[i].ld = out[i].t.stride(0);
    dst[i] = out[i].t.data_ptr();
  }
  if (any.defined())
    run(gatx_diff_attention_pack(code(any.scalar_type()), n[0], std::max(n[1], n[2]), H, d, dv,
                                 src[0], ld[0], dst[0], src[1], ld[1], dst[1], src[2], ld[2],
                                 dst[2], stream_of(any)),
        "diff_attention_pack");
  return out;
}

// The same where nothing is gathered from q later: its rows stay as they are, and in the serving form
// those of k and v where they can. *dtype gets the flags.
std::array<Rows, 3> chunked_keys(const Tensor& q, const Tensor& k, const Tensor& v, int H, int d,
                                 int dv, bool serving, int* dtype) {
  std::array<Rows, 3> out;
  if (serving && d >= 8 && dv >= 8) {
    out = {Rows(), heads_of(k), heads_of(v)};
    *dtype |= GATX_KV_UNPACKED;
  } else {
    out = chunked({}, k, v, H, d, dv);
  }
  out[0] = heads_of(q);
  *dtype |= GATX_Q_UNPACKED;
  return out;
}

// A graph's CSR (gatx.Graph) as the calls need it.
struct Csr {
  Tensor rowptr, col, rowidx;
  int64_t num_nodes = 0, edges = 0;   // edges: the allocation's bound
};
// A plan of long rows' pieces: (edges a piece, entries, their number, the plan's bound), and the rows by
// length (none: as they are).
using Plan = std::tuple<int64_t, Opt, Opt, int64_t, Opt>;
struct Hubs {
  int edges = 0;
  Tensor hubs, count, order;
  int64_t bound = 0;
  Hubs() = default;
  explicit Hubs(const Plan& p)
      : edges((int)std::get<0>(p)), hubs(of(std::get<1>(p))), count(of(std::get<2>(p))),
        order(of(std::get<4>(p))), bound(std::get<3>(p)) {}
};
const int32_t* ints(const Tensor& t) { return (const int32_t*)ptr(t); }

struct DiffAttentionBackward : public Node {
  SavedVariable q, k, v, lam, bias;
  std::array<Rows, 3> copies;   // of q, k, v in the kernels' layout, where they were not in it
  Tensor bucket, S, stat, srowptr, scol, seid;
  Csr csr;
  Hubs hubs, src_hubs;
  double scale = 1.0;

  std::string name() const override { return "DiffAttentionBackward"; }
  void release_variables() override {
    for (auto* s : {&q, &k, &v, &lam, &bias}) s->reset_data();
    for (auto& r : copies) r.t.reset();
    for (auto* t : {&bucket, &S, &stat, &srowptr, &scol, &seid, &csr.rowptr, &csr.col, &csr.rowidx,
                    &hubs.hubs, &hubs.count, &hubs.order, &src_hubs.hubs, &src_hubs.count,
                    &src_hubs.order})
      t->reset();
  }
  variable_list apply(variable_list&& go) override {
    std::lock_guard<std::mutex> lock(mutex_);
    check_capture(*this, "diff_attention");
    // (unpack also checks that nothing was changed in place since the forward)
    const Tensor qt = q.unpack(), kt = k.unpack(), vt = v.unpack(), lt = lam.unpack(),
                 bt = bias.unpack();
    variable_list out(5);
    if (!go[0].defined()) return out;
    {
      at::NoGradGuard no_grad;
      const c10::DeviceGuard guard(qt.device());
      const int H = (int)qt.size(1), d = (int)qt.size(3), dv = (int)vt.size(2);
      const Rows g = chunked({}, {}, go[0], H, d, dv)[2];
      std::array<Rows, 3> rows = copies;
      for (int i = 0; i < 3; ++i)
        if (!rows[i].t.defined()) rows[i] = heads_of(i == 0 ? qt : i == 1 ? kt : vt);
      auto like = [&](int i, const Tensor& t) {
        return task_should_compute_output(i) ? at::empty(t.sizes(), t.options()) : Tensor();
      };
      out[0] = like(0, qt);
      out[1] = like(1, kt);
      out[2] = like(2, vt);
      out[3] = like(3, lt);
      if (bt.defined()) out[4] = like(4, bt);
      const int nb = out[4].defined() ? (int)bt.size(0) : 0;
      // either direction may be without a plan (no rows that long); both are of one length
      const int pieces_of = hubs.edges ? hubs.edges : src_hubs.edges;
      TORCH_CHECK(!src_hubs.edges || src_hubs.edges == pieces_of,
                  "gatx: diff_attention: the plans of long rows differ in their pieces' length");
      const int64_t sb = src_hubs.bound;
      const size_t wb = gatx_diff_attention_backward_workspace_bytes(csr.num_nodes, csr.edges, H, d,
                                                                     dv, nb, hubs.bound, sb);
      const Tensor ws = bytes(qt, wb), lp = packed(lt);
      run(gatx_diff_attention_backward(
              code(qt.scalar_type()), ptr(rows[0].t), rows[0].ld, ptr(rows[1].t), rows[1].ld,
              ptr(rows[2].t), rows[2].ld, ptr(g.t), g.ld, H, d, dv, ints(csr.rowptr), ints(csr.col),
              ints(srowptr), ints(scol), ints(seid), csr.edges, csr.num_nodes, (float)scale,
              fptr(lp), (const uint8_t*)ptr(bucket), nb, fptr(S), fptr(stat), ptr(out[0]),
              ptr(out[1]), ptr(out[2]), fptr(out[3]), fptr(out[4]), pieces_of, ints(hubs.hubs),
              ints(hubs.count), hubs.bound, ints(src_hubs.hubs), ints(src_hubs.count), sb, ptr(ws),
              wb, ints(hubs.order), ints(src_hubs.order), stream_of(qt)),
          "diff_attention_backward");
    }
    return once(std::move(out), "diff_attention");
  }
};

// The positions' bucket of every edge (gatx/attention.py checked the arguments).
Tensor relative_buckets(const Csr& csr, const Tensor& positions, int64_t exact,
                        const std::vector<int64_t>& bounds, bool bidirectional, const Tensor& nodes) {
  const Tensor bucket = bytes(positions, std::max<int64_t>(csr.edges, 1)), pos = positions.contiguous();
  run(gatx_relative_buckets(ints(csr.rowptr), ints(csr.col), ints(csr.rowidx), csr.edges,
                            csr.num_nodes, (const int64_t*)ptr(nodes),
                            nodes.defined() ? nodes.numel() : 0, ptr(pos),
                            pos.scalar_type() == at::kLong, (int)exact, bounds.data(),
                            (int)bounds.size(), bidirectional, (uint8_t*)ptr(bucket),
                            stream_of(positions)),
      "relative_buckets");
  return bucket;
}

Tensor diff_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lam_,
                      const Opt& bias_, const Opt& positions_, int64_t exact,
                      const std::vector<int64_t>& bounds, bool bidirectional, double scale,
                      const Tensor& rowptr, const Tensor& col, const Tensor& rowidx,
                      int64_t num_nodes, int64_t edges, const Plan& plan, const Opt& srowptr,
                      const Opt& scol, const Opt& seid, const Plan& src_plan) {
  const c10::DeviceGuard guard(q.device());
  const Tensor lam = f32(lam_), bias = f32(of(bias_));
  no_tangents("diff_attention", q, k, v, lam, bias);
  const bool grad = torch::autograd::compute_requires_grad(q, k, v, lam, bias);
  const int H = (int)q.size(1), d = (int)q.size(3), dv = (int)v.size(2);
  const Csr csr{rowptr, col, rowidx, num_nodes, edges};
  const Hubs hubs(plan);
  Tensor out, S, stat, bucket;
  std::array<Rows, 3> rows;
  {
    at::NoGradGuard no_grad;
    if (bias.defined())
      bucket = relative_buckets(csr, *positions_, exact, bounds, bidirectional, {});
    int dtype = code(q.scalar_type());
    rows = grad ? chunked(q, k, v, H, d, dv) : chunked_keys(q, k, v, H, d, dv, false, &dtype);
    out = at::empty({num_nodes, H, dv}, q.options());
    S = floats(q, {H, std::max<int64_t>(edges, 1), 2});
    stat = floats(q, {H, num_nodes, 4});
    const size_t pb = gatx_diff_attention_part_bytes(hubs.bound, H, (dv + 7) / 8 * 8);
    const Tensor part = bytes(q, pb), lp = packed(lam), bp = packed(bias);
    run(gatx_diff_attention(dtype, ptr(rows[0].t), rows[0].ld, ptr(rows[1].t),
                            rows[1].ld, ptr(rows[2].t), rows[2].ld, H, d, dv, ints(rowptr),
                            ints(col), edges, num_nodes, num_nodes, nullptr, 1, (float)scale,
                            fptr(lp), fptr(bp), (const uint8_t*)ptr(bucket), ptr(out), fptr(S),
                            fptr(stat), hubs.edges, ints(hubs.hubs), ints(hubs.count), hubs.bound,
                            ptr(part), pb, ints(hubs.order), stream_of(q)),
        "diff_attention");
  }
  if (grad) {
    auto n = node_for<DiffAttentionBackward>(q, k, v, lam, bias);
    n->q = SavedVariable(q, false);
    n->k = SavedVariable(k, false);
    n->v = SavedVariable(v, false);
    n->lam = SavedVariable(lam, false);
    n->bias = SavedVariable(bias, false);
    const Tensor* in[3] = {&q, &k, &v};
    for (int i = 0; i < 3; ++i)
      if (!rows[i].t.is_same(*in[i])) n->copies[i] = rows[i];
    n->bucket = bucket;
    n->S = S;
    n->stat = stat;
    n->srowptr = of(srowptr);
    n->scol = of(scol);
    n->seid = of(seid);
    n->csr = csr;
    n->hubs = hubs;
    n->src_hubs = Hubs(src_plan);
    n->scale = scale;
    torch::autograd::set_history(out, n);
  }
  return out;
}

Tensor diff_attention_nodes(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lam_,
                            const Opt& bias_, const Opt& positions_, int64_t exact,
                            const std::vector<int64_t>& bounds, bool bidirectional, double scale,
                            const Tensor& rowptr, const Tensor& col, const Tensor& rowidx,
                            int64_t num_nodes, int64_t edges, const Tensor& nodes_, int64_t pieces) {
  const c10::DeviceGuard guard(q.device());
  at::NoGradGuard no_grad;
  const Tensor lam = f32(lam_).contiguous(), bias = packed(f32(of(bias_)));
  no_tangents("diff_attention", q, k, v, lam, bias);
  const Tensor nodes = nodes_.to(at::kLong).contiguous();
  const int H = (int)q.size(1), d = (int)q.size(3), dv = (int)v.size(2);
  const int64_t M = nodes.numel();
  const Csr csr{rowptr, col, rowidx, num_nodes, edges};
  Tensor bucket;
  if (bias.defined())
    bucket = relative_buckets(csr, *positions_, exact, bounds, bidirectional, nodes);
  int dtype = code(q.scalar_type());
  const auto rows = chunked_keys(q, k, v, H, d, dv, true, &dtype);
  const Tensor out = at::empty({M, H, dv}, q.options());
  const size_t pb = gatx_diff_attention_part_bytes(pieces > 1 ? M * pieces : 0, H, (dv + 7) / 8 * 8);
  const Tensor part = bytes(q, pb);
  run(gatx_diff_attention(dtype, ptr(rows[0].t), rows[0].ld, ptr(rows[1].t),
                          rows[1].ld, ptr(rows[2].t), rows[2].ld, H, d, dv, ints(rowptr), ints(col),
                          edges, M, num_nodes, (const int64_t*)ptr(nodes), (int)pieces,
                          (float)scale, fptr(lam), fptr(bias), (const uint8_t*)ptr(bucket), ptr(out),
                          nullptr, nullptr, 0, nullptr, nullptr, 0, ptr(part), pb, nullptr,
                          stream_of(q)),
      "diff_attention");
  return out;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("norm_before", &norm_before);
  m.def("norm_after", &norm_after);
  m.def("topk_distillation", &topk_distillation);
  m.def("diff_attention", &diff_attention);
  m.def("diff_attention_nodes", &diff_attention_nodes);
}
