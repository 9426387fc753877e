// features.cpp — the torch side of the node-feature operators: argument checks,
// output and workspace allocation, autograd nodes, around the C entry points of
// include/lanczos_b200.h.
//
// Compiled, where the rest of the package is bound with ctypes, because these
// operators are called many times a step on small inputs: through ctypes and
// Python autograd functions, layer norm forward and backward of 16 rows took
// 125 us of host time.  The autograd nodes are plain Nodes with saved variables,
// which cost a few us less a pass than torch::autograd::Function's.
// gpu_eigsh/features.py has the documentation.
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/extension.h>

#include "../../../include/lanczos_b200.h"

namespace {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

constexpr int64_t kMaxRows = 2147483646;   // 2^31 - 2

int code_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return LG_F32;
    case at::kDouble: return LG_F64;
    case at::kHalf: return LG_F16;
    case at::kBFloat16: return LG_BF16;
    default: return -1;
  }
}

at::ScalarType acc_of(at::ScalarType t) { return t == at::kDouble ? at::kDouble : at::kFloat; }

std::string name_of(at::ScalarType t) {   // as torch prints it
  switch (t) {
    case at::kFloat: return "torch.float32";
    case at::kDouble: return "torch.float64";
    case at::kHalf: return "torch.float16";
    case at::kBFloat16: return "torch.bfloat16";
    default: return c10::toString(t);
  }
}

int check_features(const char* name, const Tensor& t) {
  TORCH_CHECK_TYPE(t.is_cuda() && t.layout() == at::kStrided, name, " must be a CUDA tensor");
  const int code = code_of(t.scalar_type());
  TORCH_CHECK_TYPE(code >= 0, name, " must be float32, float64, float16 or bfloat16, got ", name_of(t.scalar_type()));
  return code;
}

void check_device(const char* name, const Tensor& t, const char* other_name, const Tensor& other) {
  TORCH_CHECK_VALUE(t.device() == other.device(), name, " is on ", t.device(), ", ", other_name, " on ", other.device());
}

// A failure of the library (RuntimeError, with the text of a LanczosError).
void check_status(int rc) {
  if (rc >= 0) return;
  char text[1024] = {0};
  lg_last_error(text, sizeof(text));
  TORCH_CHECK(false, lg_status_string(rc), " (", rc, "): ", text);
}

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

// Forward-mode derivatives would be lost without a word.
void check_forward_mode(const char* what, std::initializer_list<Tensor> inputs) {
  for (const Tensor& t : inputs)
    TORCH_CHECK_NOT_IMPLEMENTED(!torch::autograd::isFwGradDefined(t), what, " has no forward-mode derivative");
}

// t with its values in memory: not behind a pending negation (the imaginary part of
// a conjugate), and not a zero tensor without storage.
Tensor plain(const Tensor& t) {
  if (t._is_zerotensor()) return at::zeros(t.sizes(), t.options());
  return t.is_neg() ? t.resolve_neg() : t;
}

// t as rows of `dim` values with unit stride along the row; copied only where the
// strides do not allow that.
struct Rows {
  Tensor t;
  int64_t ld;
};
Rows as_rows(const Tensor& given, int64_t dim) {
  const Tensor t = plain(given);
  Tensor r = t.dim() == 2 ? t : t.reshape({-1, dim});
  const int64_t n = r.size(0);
  // (and rows 4 GiB apart and more, which the edge kernels do not address)
  if ((dim > 1 && r.stride(1) != 1) ||
      (n > 1 && (r.stride(0) < dim || r.stride(0) >= (int64_t)(1LL << 32) / (int64_t)r.element_size())))
    r = r.contiguous();
  return {r, n > 1 ? r.stride(0) : dim};
}

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

Tensor bytes(size_t n, const Tensor& like) {
  return at::empty({(int64_t)n}, like.options().dtype(at::kByte));
}

bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }

// A node over the inputs; it has a gradient for each, also for undefined ones.
template <typename N, typename... Ts> std::shared_ptr<N> node_of(const Ts&... inputs) {
  std::shared_ptr<N> node(new N(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(inputs...));
  return node;
}

// Gradients that are not differentiable themselves: where a graph of the backward
// pass is made, they lead to an error.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list defined;
  for (auto& g : grads)
    if (g.defined()) defined.push_back(g);
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that was marked with @once_differentiable", (int64_t)defined.size());
  variable_list inputs;
  for (auto& g : defined) {
    Tensor v = g.detach();
    v.requires_grad_(true);
    inputs.push_back(v);
  }
  variable_list outs = (*error)(std::move(inputs));
  size_t k = 0;
  for (auto& g : grads)
    if (g.defined()) g = outs[k++];
  return grads;
}

// ---------------------------------------------------------------------------
// Embedding lookup
// ---------------------------------------------------------------------------
struct LookupArgs {
  int mode = LG_SCALE_NONE;
  double value = 1.0;
  bool has_pad = false;
  int64_t pad = 0;
};

Tensor gather(const Tensor& table, const Tensor& column, const Tensor& ids, const LookupArgs& a) {
  std::vector<int64_t> shape(ids.sizes().begin(), ids.sizes().end());
  const int64_t rows = table.size(0), dim = table.size(1), n = ids.numel();
  shape.push_back(dim);
  Tensor out = at::empty(shape, table.options());
  if (n) {
    const c10::cuda::CUDAGuard guard(table.device());
    const Rows t = as_rows(table, dim);
    check_status(lg_rows_gather(rows, (int)dim, code_of(table.scalar_type()), t.t.data_ptr(), t.ld, n, ids.data_ptr(),
                                ids.scalar_type() == at::kLong, a.mode, ptr(column), a.value, a.has_pad, a.pad,
                                out.data_ptr(), stream_of(table)));
  }
  return out;
}

struct LookupBackward : public Node {
  SavedVariable table, column, ids;   // the table only for the scale's gradient
  LookupArgs args;
  int64_t rows = 0, dim = 0;
  at::TensorOptions options;

  std::string name() const override { return "EmbeddingLookupBackward"; }
  void release_variables() override {
    table.reset_data();
    column.reset_data();
    ids.reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    variable_list out(2);
    if (!grads[0].defined()) return out;
    const Tensor c = column.unpack(), at = ids.unpack();
    const int64_t n = at.numel();
    const int code = code_of(options.dtype().toScalarType());
    const bool want_table = task_should_compute_output(0), want_scale = c.defined() && task_should_compute_output(1);
    const c10::cuda::CUDAGuard guard(options.device());
    if (want_table) out[0] = n ? at::empty({rows, dim}, options) : at::zeros({rows, dim}, options);
    if (want_scale) out[1] = n ? at::empty({dim}, c.options()) : at::zeros({dim}, c.options());
    if (n && (want_table || want_scale)) {
      const Rows g = as_rows(grads[0], dim);
      Rows t = {Tensor(), dim};
      if (want_scale) t = as_rows(table.unpack(), dim);
      const size_t nb = lg_rows_scatter_workspace_bytes(rows, (int)dim, code, n, want_scale);
      const Tensor ws = bytes(nb, at);
      check_status(lg_rows_scatter(rows, (int)dim, code, ptr(t.t), t.ld, n, at.data_ptr(), at.scalar_type() == at::kLong,
                                   args.mode, ptr(c), args.value, args.has_pad, args.pad, g.t.data_ptr(), g.ld, ptr(out[0]),
                                   ptr(out[1]), ws.data_ptr(), nb, stream_of(at)));
    }
    return once(std::move(out));
  }
};

Tensor embedding_lookup(const Tensor& table, const Tensor& ids, const std::optional<Tensor>& scale, double value,
                        bool has_value, std::optional<int64_t> padding) {
  check_features("table", table);
  TORCH_CHECK_VALUE(table.dim() == 2 && table.size(0) >= 1 && table.size(1) >= 1, "table must be (rows, dim), got shape ",
                    table.sizes());
  TORCH_CHECK_TYPE(ids.is_cuda() && (ids.scalar_type() == at::kInt || ids.scalar_type() == at::kLong),
                   "ids must be an int32 or int64 CUDA tensor");
  check_device("ids", ids, "table", table);
  const int64_t dim = table.size(1);
  TORCH_CHECK_VALUE(table.size(0) <= kMaxRows && ids.numel() <= kMaxRows && dim <= (1 << 20),
                    "at most 2^31 - 2 rows and ids, and 2^20 columns");
  LookupArgs a;
  Tensor column;
  if (scale.has_value()) {
    const auto want = acc_of(table.scalar_type());
    TORCH_CHECK_TYPE(scale->scalar_type() == want, "scale must be ", name_of(want), " for a ",
                     name_of(table.scalar_type()), " table, got ", name_of(scale->scalar_type()));
    TORCH_CHECK_VALUE(scale->dim() == 1 && scale->size(0) == dim, "scale must have shape (", dim, ",), got ", scale->sizes());
    check_device("scale", *scale, "table", table);
    a.mode = LG_SCALE_COLUMN;
    column = plain(*scale).contiguous();
  } else if (has_value) {
    a.mode = LG_SCALE_VALUE;
    a.value = value;
  }
  a.has_pad = padding.has_value();
  a.pad = padding.value_or(0);
  const Tensor at = plain(ids).contiguous();
  check_forward_mode("embedding_lookup", {table, column});
  const bool differentiate = at::GradMode::is_enabled() && (wants_grad(table) || wants_grad(column));
  Tensor out;
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    out = gather(table, column, at, a);
  }
  if (differentiate) {
    auto node = node_of<LookupBackward>(table, column);
    if (wants_grad(column)) node->table = SavedVariable(table, false);
    node->rows = table.size(0);
    node->dim = dim;
    node->options = table.options();
    node->column = SavedVariable(column, false);
    node->ids = SavedVariable(at, false);
    node->args = a;
    torch::autograd::set_history(out, node);
  }
  return out;
}

// ---------------------------------------------------------------------------
// Layer norm
// ---------------------------------------------------------------------------
int param_code(const Tensor& x, const Tensor& w, const Tensor& b) {
  return code_of(w.defined() ? w.scalar_type() : b.defined() ? b.scalar_type() : x.scalar_type());
}

Tensor norm_forward(const Tensor& x, const Tensor& w, const Tensor& b, double eps, Tensor* stats) {
  const int64_t dim = x.size(-1), rows = x.numel() / dim;
  const c10::cuda::CUDAGuard guard(x.device());
  Tensor y = at::empty(x.sizes(), x.options());
  const auto acc = acc_of(x.scalar_type());
  char* mean = nullptr;
  char* rstd = nullptr;
  if (stats) {
    *stats = at::empty({2, rows}, x.options().dtype(acc));
    mean = static_cast<char*>(stats->data_ptr());
    rstd = mean + rows * (acc == at::kDouble ? 8 : 4);
  }
  if (rows) {
    const Rows t = as_rows(x, dim);
    check_status(lg_layer_norm_forward(rows, (int)dim, code_of(x.scalar_type()), t.t.data_ptr(), t.ld, param_code(x, w, b),
                                       ptr(w), ptr(b), eps, y.data_ptr(), mean, rstd, stream_of(x)));
  }
  return y;
}

struct LayerNormBackward : public Node {
  SavedVariable x, weight, stats;
  at::ScalarType params = at::kFloat;

  std::string name() const override { return "LayerNormBackward"; }
  void release_variables() override {
    x.reset_data();
    weight.reset_data();
    stats.reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    variable_list out(3);
    if (!grads[0].defined()) return out;
    const Tensor v = x.unpack(), w = weight.unpack(), s = stats.unpack();
    const int64_t dim = v.size(-1), rows = v.numel() / dim;
    const c10::cuda::CUDAGuard guard(v.device());
    const auto popt = v.options().dtype(params);
    Tensor &dx = out[0], &dw = out[1], &db = out[2];
    if (task_should_compute_output(0)) dx = at::empty(v.sizes(), v.options());
    if (task_should_compute_output(1)) dw = rows ? at::empty({dim}, popt) : at::zeros({dim}, popt);
    if (task_should_compute_output(2)) db = rows ? at::empty({dim}, popt) : at::zeros({dim}, popt);
    if (rows && (dx.defined() || dw.defined() || db.defined())) {
      const Rows t = as_rows(v, dim), g = as_rows(grads[0], dim);
      const int code = code_of(v.scalar_type());
      const size_t nb = lg_layer_norm_workspace_bytes(rows, (int)dim, code);
      const Tensor ws = bytes(nb, v);
      const char* mean = static_cast<const char*>(s.data_ptr());
      check_status(lg_layer_norm_backward(rows, (int)dim, code, t.t.data_ptr(), t.ld, g.t.data_ptr(), g.ld, code_of(params),
                                          ptr(w), mean, mean + rows * s.element_size(), ptr(dx), ptr(dw), ptr(db), ptr(ws),
                                          nb, stream_of(v)));
    }
    return once(std::move(out));
  }
};

Tensor layer_norm(const Tensor& x, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias, double eps) {
  check_features("x", x);
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "x must have a last dimension of at least 1, got shape ", x.sizes());
  const int64_t dim = x.size(-1);
  TORCH_CHECK_VALUE(x.numel() / dim <= kMaxRows && dim <= (1 << 24), "at most 2^31 - 2 rows and 2^24 columns");
  TORCH_CHECK_VALUE(eps >= 0.0 && eps < std::numeric_limits<double>::infinity(),
                    "eps must be finite and not negative, got ", eps);
  const auto xt = x.scalar_type();
  const bool half = xt == at::kHalf || xt == at::kBFloat16;
  Tensor w, b;
  for (int k = 0; k < 2; ++k) {
    const auto& p = k ? bias : weight;
    if (!p.has_value()) continue;
    const char* name = k ? "bias" : "weight";
    TORCH_CHECK_TYPE(p->is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK_TYPE(p->scalar_type() == xt || (half && p->scalar_type() == at::kFloat), name, " must be ", name_of(xt),
                     half ? " or torch.float32" : "", ", got ", name_of(p->scalar_type()));
    TORCH_CHECK_VALUE(p->dim() == 1 && p->size(0) == dim, name, " must have shape (", dim, ",), got ", p->sizes());
    check_device(name, *p, "x", x);
    (k ? b : w) = plain(*p).contiguous();
  }
  TORCH_CHECK_TYPE(!w.defined() || !b.defined() || w.scalar_type() == b.scalar_type(),
                   "weight and bias must have the same type");
  check_forward_mode("layer_norm", {x, w, b});
  const bool differentiate = at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(w) || wants_grad(b));
  Tensor out, stats;
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    out = norm_forward(x, w, b, eps, differentiate ? &stats : nullptr);
  }
  if (differentiate) {
    auto node = node_of<LayerNormBackward>(x, w, b);
    node->x = SavedVariable(x, false);
    node->weight = SavedVariable(w, false);
    node->stats = SavedVariable(stats, false);
    node->params = w.defined() ? w.scalar_type() : b.defined() ? b.scalar_type() : xt;
    torch::autograd::set_history(out, node);
  }
  return out;
}

// ---------------------------------------------------------------------------
// Edge distances
// ---------------------------------------------------------------------------
// The lists of lg_edge_graph and those of its long vertices; shared by every call
// (and every pending backward pass) that uses them.
struct EdgeGraph : torch::CustomClassHolder {
  int64_t n = 0, m = 0, nlong = 0, nchunks = 0;
  Tensor ends, rowptr, lists;                                  // lists: other, then eid
  Tensor long_row, long_first, chunk_row, chunk_first;
  at::Device device = at::Device(at::kCPU);
  void* built_on = nullptr;

  // Makes the lists known to the current stream when it is not the one they were
  // allocated on.
  void use() const {
    const auto cur = c10::cuda::getCurrentCUDAStream(device.index());
    if (cur.stream() == built_on) return;
    for (const Tensor* t : {&ends, &rowptr, &lists, &long_row, &long_first, &chunk_row, &chunk_first})
      if (t->defined()) t->record_stream(cur);
  }
  const int* other() const { return lists.data_ptr<int>(); }
  const int* eid() const { return lists.data_ptr<int>() + 2 * m; }
};

c10::intrusive_ptr<EdgeGraph> edge_graph(const Tensor& given, int64_t n) {
  TORCH_CHECK_TYPE(given.is_cuda(), "idx must be a CUDA tensor");
  TORCH_CHECK_TYPE(given.scalar_type() == at::kLong || given.scalar_type() == at::kInt,
                   "idx must be int64 or int32, got ", name_of(given.scalar_type()));
  TORCH_CHECK_VALUE(given.dim() == 2 && given.size(0) == 2, "idx must be (2, M), got shape ", given.sizes());
  auto g = c10::make_intrusive<EdgeGraph>();
  const int64_t m = given.size(1);
  TORCH_CHECK_VALUE(n >= 1 && n <= kMaxRows && m <= (2147483647 - LG_EDGE_CHUNK) / 2,
                    "n must be at least 1; at most 2^31 - 2 vertices and 2^30 - 65 edges");
  g->n = n;
  g->m = m;
  g->device = given.device();
  if (m == 0) return g;
  const c10::cuda::CUDAGuard guard(given.device());
  g->built_on = stream_of(given);
  const Tensor idx = plain(given).to(at::kLong).contiguous();
  const auto i32 = idx.options().dtype(at::kInt);
  g->ends = at::empty({2 * m}, i32);
  g->rowptr = at::empty({n + 1}, i32);
  g->lists = at::empty({4 * m}, i32);
  Tensor found = at::empty({2}, i32);   // a bad index; the longest list
  const size_t nb = lg_edge_graph_workspace_bytes(n, m);
  const Tensor ws = bytes(nb, idx);
  check_status(lg_edge_graph(n, m, reinterpret_cast<const long long*>(idx.data_ptr<int64_t>()), g->ends.data_ptr<int>(),
                             g->rowptr.data_ptr<int>(), g->lists.data_ptr<int>(), g->lists.data_ptr<int>() + 2 * m,
                             found.data_ptr<int>(), ws.data_ptr(), nb, stream_of(idx)));
  const Tensor degree = g->rowptr.slice(0, 1) - g->rowptr.slice(0, 0, n);
  found.slice(0, 1).copy_(degree.max().reshape({1}));
  const Tensor host = found.cpu();
  TORCH_CHECK_VALUE(host.data_ptr<int>()[0] == 0, "edge index out of range [0, n)");
  if (host.data_ptr<int>()[1] <= LG_EDGE_CHUNK) return g;
  // the vertices with long lists, and the chunks of their lists
  const Tensor row = at::nonzero(degree > LG_EDGE_CHUNK).reshape({-1});
  const Tensor count = at::floor_divide(degree.index_select(0, row).to(at::kLong) + (LG_EDGE_CHUNK - 1), LG_EDGE_CHUNK);
  const Tensor first = at::cumsum(count, 0) - count;
  const Tensor which = at::repeat_interleave(count);
  const Tensor begin = g->rowptr.index_select(0, row).to(at::kLong).index_select(0, which) +
                       (at::arange(which.numel(), row.options()) - first.index_select(0, which)) * LG_EDGE_CHUNK;
  g->nlong = row.numel();
  g->nchunks = which.numel();
  g->long_row = row.to(at::kInt);
  g->long_first = first.to(at::kInt);
  g->chunk_row = row.index_select(0, which).to(at::kInt);
  g->chunk_first = begin.to(at::kInt);
  return g;
}

Tensor edge_forward(const Tensor& x, const EdgeGraph& g) {
  const c10::cuda::CUDAGuard guard(x.device());
  Tensor out = at::empty({g.m}, x.options().dtype(acc_of(x.scalar_type())));
  if (g.m) {
    g.use();
    const Rows t = as_rows(x, x.size(1));
    const int dim = (int)x.size(1), code = code_of(x.scalar_type());
    const size_t nb = lg_edge_sqdist_workspace_bytes(g.n, g.m, dim, code, t.t.data_ptr(), t.ld);
    const Tensor ws = nb ? bytes(nb, x) : Tensor();
    check_status(lg_edge_sqdist(g.n, g.m, dim, code, g.ends.data_ptr<int>(), t.t.data_ptr(), t.ld, out.data_ptr(),
                                ptr(ws), nb, stream_of(x)));
  }
  return out;
}

struct EdgeDistBackward : public Node {
  SavedVariable x;
  c10::intrusive_ptr<EdgeGraph> graph;

  std::string name() const override { return "EdgeDistancesBackward"; }
  void release_variables() override { x.reset_data(); }
  variable_list apply(variable_list&& grads) override {
    if (!grads[0].defined()) return variable_list(1);
    const Tensor v = x.unpack();
    const EdgeGraph& e = *graph;
    const int64_t dim = v.size(1);
    const c10::cuda::CUDAGuard guard(v.device());
    Tensor dx = e.m ? at::empty({e.n, dim}, v.options()) : at::zeros({e.n, dim}, v.options());
    if (e.m) {
      e.use();
      const Rows t = as_rows(v, dim);
      const Tensor g = plain(grads[0]).contiguous();
      const int code = code_of(v.scalar_type());
      const size_t nb = lg_edge_sqdist_grad_workspace_bytes(e.n, e.m, (int)dim, code, t.t.data_ptr(), t.ld,
                                                             e.nlong ? (int)e.nchunks : 0);
      const Tensor ws = nb ? bytes(nb, v) : Tensor();
      auto list = [](const Tensor& l) { return l.defined() ? l.data_ptr<int>() : nullptr; };
      check_status(lg_edge_sqdist_grad(e.n, e.m, (int)dim, code, e.rowptr.data_ptr<int>(), e.other(), e.eid(),
                                       (int)e.nlong, list(e.long_row), list(e.long_first), (int)e.nchunks,
                                       list(e.chunk_row), list(e.chunk_first), t.t.data_ptr(), t.ld, g.data_ptr(),
                                       dx.data_ptr(), ptr(ws), nb, stream_of(v)));
    }
    return once({dx});
  }
};

Tensor edge_sqdist(const Tensor& x, const c10::intrusive_ptr<EdgeGraph>& g) {
  check_features("x", x);
  TORCH_CHECK_VALUE(x.dim() == 2 && x.size(0) == g->n && x.size(1) >= 1 && x.size(1) <= (1 << 20), "x must be (", g->n,
                    ", dim), got shape ", x.sizes());
  TORCH_CHECK_VALUE(x.device() == g->device, "x is on ", x.device(), ", the edges on ", g->device);
  check_forward_mode("EdgeDistances", {x});
  const bool differentiate = at::GradMode::is_enabled() && wants_grad(x);
  Tensor out;
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    out = edge_forward(x, *g);
  }
  if (differentiate) {
    auto node = node_of<EdgeDistBackward>(x);
    node->x = SavedVariable(x, false);
    node->graph = g;
    torch::autograd::set_history(out, node);
  }
  return out;
}

}  // namespace

TORCH_LIBRARY(gpu_eigsh, m) { m.class_<EdgeGraph>("EdgeGraph"); }

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("embedding_lookup", &embedding_lookup, py::call_guard<py::gil_scoped_release>());
  m.def("layer_norm", &layer_norm, py::call_guard<py::gil_scoped_release>());
  py::class_<EdgeGraph, c10::intrusive_ptr<EdgeGraph>>(m, "EdgeGraph")
      .def_readonly("n", &EdgeGraph::n)
      .def_readonly("m", &EdgeGraph::m);
  m.def("edge_graph", &edge_graph, py::call_guard<py::gil_scoped_release>());
  m.def("edge_sqdist", &edge_sqdist, py::call_guard<py::gil_scoped_release>());
}
