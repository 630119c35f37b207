// text_nodes.cpp — C++ autograd nodes of the text encoder's operators over the C-ABI (include/irx.h): packed attention and the
// root-mean-square norm with the residual's addition. The same calls in the same order as the Python nodes (attention.py, dense.py); what
// they save is the interpreter: a small norm's forward + backward is 150 us of host time through torch.autograd.Function, 76 here, of which
// 51 are the autograd engine's call (50 for torch's own layer norm).
#include <c10/core/impl/VirtualGuardImpl.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/extension.h>

#include "torch_nodes.h"

#include <unordered_map>
#include <unordered_set>

namespace irxn {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef c10::optional<Tensor> OptTensor;
typedef long long ll;

// The autograd engine makes an accumulator's stream wait for the backward that feeds it, and the accumulator keeps the stream of the first
// graph that used the leaf for as long as any such graph lives. Inside a capture that wait would draw a stream that is not being captured
// into it: the runtime ends the process when the capture ends.
static bool is_foreign(torch::autograd::Node& accumulator, const Tensor& leaf) {
  const auto s = accumulator.stream();
  return s.has_value() && *s != c10::impl::VirtualGuardImpl(leaf.device().type()).getStream(leaf.device());
}

// The first of `leaves` whose gradient accumulator lives on another stream than the current one of its device, or -1.
static int64_t foreign_leaf(const std::vector<OptTensor>& leaves) {
  for (size_t i = 0; i < leaves.size(); ++i) {
    const auto& t = leaves[i];
    if (!t.has_value() || !t->defined() || !t->requires_grad() || !t->is_leaf()) continue;
    const auto acc = torch::autograd::impl::try_get_grad_accumulator(*t);
    if (acc && is_foreign(*acc, *t)) return (int64_t)i;
  }
  return -1;
}

// Inside a node's backward: the accumulators that this pass will feed right behind it, or behind copies and views of a leaf (an operator
// pads and copies what its kernels cannot read in place), each with the number of the input that leads to it.
static std::vector<std::pair<int64_t, torch::autograd::AccumulateGrad*>> accumulators_behind() {
  using torch::autograd::Node;
  static const std::unordered_set<std::string> kept = {
      "CloneBackward0", "ConstantPadNdBackward0", "ToCopyBackward0", "AliasBackward0", "ViewBackward0", "UnsafeViewBackward0", "ReshapeAliasBackward0",
      "AsStridedBackward0", "TransposeBackward0", "TBackward0", "PermuteBackward0", "UnsqueezeBackward0", "SqueezeBackward0", "SqueezeBackward1",
      "SqueezeBackward2", "ExpandBackward0", "SliceBackward0", "SelectBackward0", "SplitBackward0", "SplitWithSizesBackward0", "UnbindBackward0"};
  std::vector<std::pair<int64_t, torch::autograd::AccumulateGrad*>> out;
  const auto node = torch::autograd::get_current_node();
  if (!node) return out;
  const auto* exec = torch::autograd::get_current_graph_task_exec_info();     // empty: everything runs
  auto runs = [&](Node* n) {
    if (!exec || exec->empty()) return true;
    const auto it = exec->find(n);
    return it != exec->end() && it->second.should_execute();
  };
  for (size_t i = 0; i < node->num_outputs(); ++i) {
    Node* n = node->next_edge(i).function.get();
    while (n && runs(n)) {
      if (auto* acc = dynamic_cast<torch::autograd::AccumulateGrad*>(n)) {
        out.emplace_back((int64_t)i, acc);
        break;
      }
      if (n->num_outputs() != 1 || !kept.count(n->name())) break;
      n = n->next_edge(0).function.get();
    }
  }
  return out;
}
static std::vector<Tensor> leaves_behind() {
  std::vector<Tensor> out;
  for (const auto& a : accumulators_behind()) out.push_back(a.second->variable);
  return out;
}
// The first input that leads to an accumulator of another stream, or -1.
static int64_t foreign_behind() {
  for (const auto& a : accumulators_behind())
    if (is_foreign(*a.second, a.second->variable)) return a.first;
  return -1;
}

namespace {

typedef size_t (*attn_fwd_ws_fn)(int, int, int, int, int, int, int, int);
typedef int (*attn_fwd_fn)(const void*, ll, ll, const void*, ll, ll, const void*, ll, ll, const int32_t*, const int32_t*, int, int, int, int, int, int,
                           int, float, int, const void*, int, const int32_t*, int, int, void*, void*, float*, void*, size_t, void*);
typedef size_t (*attn_bwd_ws_fn)(int, int, int, int, int, int, int, int);
typedef int (*attn_bwd_fn)(const void*, ll, ll, const void*, ll, ll, const void*, ll, ll, const void*, ll, ll, const void*, const void*, const float*,
                           const int32_t*, const int32_t*, int, int, int, int, int, int, int, float, int, const void*, int, const int32_t*, int, int,
                           void*, void*, void*, void*, void*, size_t, void*);
typedef int (*rms_fwd_fn)(const void*, const void*, const void*, int, ll, int, int, float, void*, void*, float*, void*);
typedef size_t (*rms_bwd_ws_fn)(ll, int, int);
typedef int (*rms_bwd_fn)(const void*, const void*, const void*, const void*, int, const float*, ll, int, int, void*, void*, void*, size_t, void*);
typedef int (*capturing_fn)(void*);

struct Api {
  attn_fwd_ws_fn attn_fwd_ws = nullptr;
  attn_fwd_fn attn_fwd = nullptr;
  attn_bwd_ws_fn attn_bwd_ws = nullptr;
  attn_bwd_fn attn_bwd = nullptr;
  rms_fwd_fn rms_fwd = nullptr;
  rms_bwd_ws_fn rms_bwd_ws = nullptr;
  rms_bwd_fn rms_bwd = nullptr;
  capturing_fn capturing = nullptr;
} g_text;

inline int type_of(const Tensor& t) { return t.scalar_type() == at::kFloat ? 0 : t.scalar_type() == at::kBFloat16 ? 1 : 2; }
inline Tensor bytes(size_t n, const Tensor& like) { return at::empty({(int64_t)n}, like.options().dtype(at::kByte)); }

// rows and heads are read in place from any strides that keep 16-byte alignment
inline Tensor rows(const Tensor& t) {
  const int64_t e = t.element_size();
  if (t.stride(2) == 1 && t.stride(0) * e % 16 == 0 && t.stride(0) * e < (1 << 24) && t.stride(1) * e % 16 == 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0) return t;
  return t.clone(at::MemoryFormat::Contiguous);
}

// the second derivative is not there: say so when somebody asks for it, not before
inline variable_list once(variable_list g, const char* who) {
  if (!at::GradMode::is_enabled()) return g;
  auto err = std::make_shared<torch::autograd::DelayedError>(std::string(who) + " is differentiable once", (int)g.size());
  variable_list in;
  for (auto& t : g) {
    if (t.defined()) t.set_requires_grad(true);
    in.push_back(t);
  }
  return (*err)(std::move(in));
}

inline void refuse(int64_t input, const char* who) {
  if (input >= 0)
    throw std::runtime_error(std::string(who) + ": a backward pass cannot be captured while an eager graph of the same leaves lives (input " +
                             std::to_string(input) + " was used on another stream): drop that graph's outputs first, or run the warm-up on the "
                             "capture's stream");
}
inline void refuse_foreign(const std::vector<OptTensor>& leaves, const char* who) { refuse(foreign_leaf(leaves), who); }
inline void refuse_foreign_behind(const char* who) { refuse(foreign_behind(), who); }

struct Attn {
  Tensor q, k, v, table, cu_q, cu_k, map;
  double scale;
  bool causal;
  int batch() const { return (int)cu_q.size(0) - 1; }
  int far() const { return table.defined() ? (int)(map.size(0) - 1) / 2 : -1; }
};

// stats, rest: what the backward needs of the forward (NULL: no backward)
Tensor attn_forward(const Attn& a, Tensor* stats, Tensor* rest, void* stream) {
  const Tensor &q = a.q, &k = a.k;
  const int tq = (int)q.size(0), heads = (int)q.size(1), dim = (int)q.size(2), tk = (int)k.size(0), kv = (int)k.size(1);
  Tensor out = at::empty({tq, heads, dim}, q.options());
  if (stats) *stats = at::empty({heads, tq, 2}, q.options().dtype(at::kFloat));
  if (rest && q.scalar_type() != at::kFloat) *rest = at::empty_like(out);
  const size_t n = g_text.attn_fwd_ws(tq, tk, a.batch(), heads, kv, dim, type_of(q), a.table.defined() + 2 * a.causal);
  const Tensor ws = n ? bytes(n, q) : Tensor();
  const bool b = a.table.defined();
  check(g_text.attn_fwd(q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1), a.v.data_ptr(), a.v.stride(0), a.v.stride(1),
                        a.cu_q.data_ptr<int32_t>(), a.cu_k.data_ptr<int32_t>(), a.batch(), tq, tk, heads, kv, dim, type_of(q), (float)a.scale, a.causal,
                        b ? a.table.data_ptr() : nullptr, b ? a.table.scalar_type() == at::kFloat : 1, b ? a.map.data_ptr<int32_t>() : nullptr,
                        b ? (int)a.table.size(0) : 0, b ? a.far() : 0, out.data_ptr(), rest && rest->defined() ? rest->data_ptr() : nullptr,
                        stats ? stats->data_ptr<float>() : nullptr,
                        n ? ws.data_ptr() : nullptr, n, stream),
        "irx_attn_packed_fwd");
  return out;
}

struct AttnNode : public torch::autograd::Function<AttnNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& table, const Tensor& cu_q,
                        const Tensor& cu_k, const OptTensor& map, bool causal, double scale, int64_t stream) {
    Attn a{q, k, v, table.has_value() ? *table : Tensor(), cu_q, cu_k, map.has_value() ? *map : Tensor(), scale, causal};
    Tensor stats, rest, out = attn_forward(a, &stats, &rest, (void*)stream);
    ctx->save_for_backward({q, k, v, a.table, cu_q, cu_k, a.map, out, stats, rest});
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["stream"] = stream;                   // (the engine replays the node on its forward stream)
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grad_out) {
    const auto s = ctx->get_saved_variables();
    Attn a{s[0], s[1], s[2], s[3], s[4], s[5], s[6], ctx->saved_data["scale"].toDouble(), ctx->saved_data["causal"].toBool()};
    const Tensor &q = a.q, &k = a.k, &out = s[7], &stats = s[8], &rest = s[9];
    void* stream = (void*)ctx->saved_data["stream"].toInt();
    if (g_text.capturing(stream)) refuse_foreign_behind("attention_packed");
    const Tensor dout = rows(grad_out[0]);
    const int tq = (int)q.size(0), heads = (int)q.size(1), dim = (int)q.size(2), tk = (int)k.size(0), kv = (int)k.size(1);
    Tensor dq = at::empty({tq, heads, dim}, q.options()), dk = at::empty({tk, kv, dim}, q.options()), dv = at::empty({tk, kv, dim}, q.options());
    const bool b = a.table.defined();
    Tensor dt;
    if (b) dt = tq ? at::empty_like(a.table) : at::zeros_like(a.table);
    const size_t n = g_text.attn_bwd_ws(tq, tk, a.batch(), heads, kv, dim, type_of(q), a.far());
    const Tensor ws = bytes(n ? n : 16, q);
    check(g_text.attn_bwd(q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1), a.v.data_ptr(), a.v.stride(0), a.v.stride(1),
                          dout.data_ptr(), dout.stride(0), dout.stride(1), out.data_ptr(), rest.defined() ? rest.data_ptr() : nullptr, stats.data_ptr<float>(), a.cu_q.data_ptr<int32_t>(),
                          a.cu_k.data_ptr<int32_t>(), a.batch(), tq, tk, heads, kv, dim, type_of(q), (float)a.scale, a.causal,
                          b ? a.table.data_ptr() : nullptr, b ? a.table.scalar_type() == at::kFloat : 1, b ? a.map.data_ptr<int32_t>() : nullptr,
                          b ? (int)a.table.size(0) : 0, b ? a.far() : 0, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), b ? dt.data_ptr() : nullptr,
                          ws.data_ptr(), n, stream),
          "irx_attn_packed_bwd");
    variable_list g = once({dq, dk, dv, dt}, "attention_packed");
    g.resize(10);
    return g;
  }
};

// q, k, v, table, offsets and map as attention_packed has checked them
Tensor attention(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, const OptTensor& table_in, const Tensor& cu_q, const Tensor& cu_k,
                 const OptTensor& map, bool causal, double scale, int64_t stream) {
  const Tensor q = rows(q_in), k = rows(k_in), v = rows(v_in);           // (a copy of a leaf leads back to it: the leaves themselves are asked)
  const OptTensor table = table_in.has_value() ? OptTensor(table_in->contiguous()) : table_in;
  if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad() || (table.has_value() && table->requires_grad()))) {
    if (g_text.capturing((void*)stream)) refuse_foreign({q_in, k_in, v_in, table_in}, "attention_packed");
    return AttnNode::apply(q, k, v, table, cu_q, cu_k, map, causal, scale, stream);
  }
  return attn_forward(Attn{q, k, v, table.has_value() ? *table : Tensor(), cu_q, cu_k, map.has_value() ? *map : Tensor(), scale, causal}, nullptr, nullptr, (void*)stream);
}

void rms_forward(const Tensor& x, const Tensor& r, const Tensor& w, double eps, Tensor* y, Tensor* h, Tensor* rstd, void* stream) {
  *y = at::empty_like(x);
  if (r.defined()) *h = at::empty_like(x);
  const int64_t cols = x.size(-1), rows = x.numel() / cols;
  if (rstd) *rstd = at::empty({rows}, x.options().dtype(at::kFloat));
  check(g_text.rms_fwd(x.data_ptr(), r.defined() ? r.data_ptr() : nullptr, w.data_ptr(), w.scalar_type() == at::kFloat, rows, (int)cols, type_of(x),
                       (float)eps, y->data_ptr(), h->defined() ? h->data_ptr() : nullptr, rstd ? rstd->data_ptr<float>() : nullptr, stream),
        "irx_rms_norm_fwd");
}

struct RmsNode : public torch::autograd::Function<RmsNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& r_o, const Tensor& w, double eps, int64_t stream) {
    const Tensor r = r_o.has_value() ? *r_o : Tensor();
    Tensor y, h, rstd;
    rms_forward(x, r, w, eps, &y, &h, &rstd, (void*)stream);
    ctx->save_for_backward({h.defined() ? h : x, w, rstd});              // (x and the residual are not read again)
    ctx->saved_data["residual"] = r.defined();
    ctx->saved_data["stream"] = stream;
    ctx->set_materialize_grads(false);
    if (h.defined()) return {y, h};
    return {y};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grad_out) {
    variable_list g(5);
    const auto s = ctx->get_saved_variables();
    const Tensor &h = s[0], &w = s[1], &rstd = s[2];
    const Tensor dh = grad_out.size() > 1 && grad_out[1].defined() ? grad_out[1].contiguous() : Tensor();
    if (!grad_out[0].defined() && !dh.defined()) return g;
    void* stream = (void*)ctx->saved_data["stream"].toInt();
    if (g_text.capturing(stream)) refuse_foreign_behind("rms_norm_residual");
    const Tensor dy = grad_out[0].defined() ? grad_out[0].contiguous() : at::zeros_like(h);
    Tensor dx = at::empty_like(h), dw = at::empty_like(w);
    const int64_t cols = h.size(-1), rows = h.numel() / cols;
    const size_t n = g_text.rms_bwd_ws(rows, (int)cols, type_of(h));
    const Tensor ws = bytes(n, h);
    check(g_text.rms_bwd(dy.data_ptr(), dh.defined() ? dh.data_ptr() : nullptr, h.data_ptr(), w.data_ptr(), w.scalar_type() == at::kFloat, rstd.data_ptr<float>(),
                         rows, (int)cols, type_of(h), dx.data_ptr(), dw.data_ptr(), ws.data_ptr(), n, stream),
          "irx_rms_norm_bwd");
    variable_list d = once({dx, dw}, "rms_norm_residual");
    g[0] = d[0];
    if (ctx->saved_data["residual"].toBool()) g[1] = d[0];
    g[2] = d[1];
    return g;
  }
};

// x, residual (..., C) contiguous, weight (C,) contiguous, as rms_norm_residual has checked them -> [y, h] or [y]
std::vector<Tensor> rms_norm(const Tensor& x, const OptTensor& r, const Tensor& w, double eps, int64_t stream) {
  if (at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad() || (r.has_value() && r->requires_grad()))) {
    if (g_text.capturing((void*)stream)) refuse_foreign({x, r, w}, "rms_norm_residual");
    return RmsNode::apply(x, r, w, eps, stream);
  }
  Tensor y, h;
  rms_forward(x, r.has_value() ? *r : Tensor(), w, eps, &y, &h, nullptr, (void*)stream);
  if (h.defined()) return {y, h};
  return {y};
}

// The addresses of the gradients of `params` to out (an array of pointers), for the copy that sums their norm. False, with `out` in no
// certain state, if one of them is no dense contiguous float32 tensor of its own size on the device, or if one of `filled` (parameters whose
// gradient a producer has delivered already) has a gradient besides: the caller then goes through them one by one.
bool grad_addresses(const std::vector<Tensor>& params, const std::vector<Tensor>& filled, int64_t device, int64_t counts, int64_t out) {
  const unsigned long long* n = (const unsigned long long*)counts;
  void** at = (void**)out;
  for (const Tensor& p : filled)
    if (p.grad().defined()) return false;
  for (size_t i = 0; i < params.size(); ++i) {
    const Tensor& g = params[i].grad();
    if (!g.defined() || g.layout() != at::kStrided || g.scalar_type() != at::kFloat || !g.is_cuda() || g.get_device() != device ||
        (unsigned long long)g.numel() != n[i] || !g.is_contiguous())
      return false;
    at[i] = g.data_ptr();
  }
  return true;
}

void bind_text(const std::unordered_map<std::string, int64_t>& p) {
  auto get = [&](const char* n) {
    const auto it = p.find(n);
    if (it == p.end() || it->second == 0) throw std::runtime_error(std::string("_irx_nodes: missing entry point ") + n);
    return (void*)it->second;
  };
  g_text.attn_fwd_ws = (attn_fwd_ws_fn)get("irx_attn_packed_fwd_workspace_bytes");
  g_text.attn_fwd = (attn_fwd_fn)get("irx_attn_packed_fwd");
  g_text.attn_bwd_ws = (attn_bwd_ws_fn)get("irx_attn_packed_bwd_workspace_bytes");
  g_text.attn_bwd = (attn_bwd_fn)get("irx_attn_packed_bwd");
  g_text.rms_fwd = (rms_fwd_fn)get("irx_rms_norm_fwd");
  g_text.rms_bwd_ws = (rms_bwd_ws_fn)get("irx_rms_norm_bwd_workspace_bytes");
  g_text.rms_bwd = (rms_bwd_fn)get("irx_rms_norm_bwd");
  g_text.capturing = (capturing_fn)get("irx_stream_capturing");
}

}  // namespace

void register_text(pybind11::module& m) {
  m.def("foreign_leaf", &foreign_leaf);
  m.def("foreign_behind", &foreign_behind);
  m.def("leaves_behind", &leaves_behind);
  m.def("bind_text", &bind_text);
  m.def("attention", &attention);
  m.def("rms_norm", &rms_norm);
  m.def("grad_addresses", &grad_addresses);
}

}  // namespace irxn
