// torch_ops.cpp — the training operators (nphm_amd/train_ops.py) as seen from PyTorch: checks of arguments, outputs and workspaces, the
// autograd nodes.  The kernels are those of libnphm_amd.so, reached through the C entries that nphm_torch_bind hands over (whichever
// build of that library the process has loaded).  In C++ because a layer of a few hundred rows takes 20 us on the card, and
// the same node written in Python took 130 on the host (its backward pass runs in a thread of autograd's own and waits for the
// interpreter there); a list of 500 gradients took 280 to look through.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/library.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <initializer_list>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/nphm_amd.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Entries {
  decltype(&nphm_last_error) last_error;
  decltype(&nphm_rows_lookup) rows_lookup;
  decltype(&nphm_rows_grad_workspace_bytes) rows_grad_ws;
  decltype(&nphm_rows_grad) rows_grad;
  decltype(&nphm_rows_entries) rows_entries;
  decltype(&nphm_rows_merge) rows_merge;
  decltype(&nphm_rows_renorm) rows_renorm;
  decltype(&nphm_clip_workspace_bytes) clip_ws;
  decltype(&nphm_clip_grads) clip;
  decltype(&nphm_layer16_forward_workspace_bytes) forward_ws;
  decltype(&nphm_layer16_forward) forward;
  decltype(&nphm_layer16_backward_workspace_bytes) backward_ws;
  decltype(&nphm_layer16_backward) backward;
};
Entries lib{};

void bound() { TORCH_CHECK(lib.last_error, "nphm: the kernels' library is not bound (nphm_amd._lib.load_torch does it)"); }
void check(int rc, const char* what) { TORCH_CHECK(rc == 0, "nphm: ", what, " failed (", rc, "): ", lib.last_error()); }

int code_of(at::ScalarType t) { return t == at::kFloat ? 0 : t == at::kBFloat16 ? 1 : t == at::kHalf ? 2 : -1; }
void on_gpu(const char* what, const Tensor& t) {
  TORCH_CHECK_TYPE(t.is_cuda(), what, ": a tensor on a ROCm device (these operators have no CPU form)");
}
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
// Forward-mode derivatives: none is computed, and none may be lost without a word.  (A tensor is asked only inside a level, where alone it
// can have a tangent: 500 gradients and their outputs took 15 us to ask.)
bool in_forward_mode() { return torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr; }
void no_tangent(const char* what, const Tensor& t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(/*level=*/0).defined(), what, ": no forward-mode derivative (torch.autograd.forward_ad)");
}
void no_tangent(const char* what, std::initializer_list<const Tensor*> all) {
  if (in_forward_mode())
    for (const Tensor* t : all) no_tangent(what, *t);
}
// (address 0 and no tensor where nothing is needed)
Tensor workspace(size_t bytes, const Tensor& like) { return bytes ? at::empty({int64_t(bytes)}, like.options().dtype(at::kByte)) : Tensor(); }
void* at_of(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
const void* const_of(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
// a gradient that is not differentiable itself: asked for with create_graph it carries a node that says so
variable_list once(variable_list grads, const char* what) {
  if (!at::GradMode::is_enabled()) return grads;
  for (Tensor& g : grads)
    if (g.defined()) g = g.detach().set_requires_grad(true);
  auto node = std::make_shared<torch::autograd::DelayedError>(std::string(what) + ": its gradients are not differentiable", int64_t(grads.size()));
  return (*node)(std::move(grads));
}

// A captured backward pass whose gradients go to a leaf of which a graph of eager calls is alive: autograd adds them on the stream of those calls,
// and the default stream cannot be made to wait for a capture (the process may end by it).  Refused while nothing has happened yet.
void check_leaves(const char* what) {
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  const auto node = torch::autograd::get_current_node();
  if (!node) return;
  for (const auto& edge : node->next_edges()) {
    if (!dynamic_cast<torch::autograd::AccumulateGrad*>(edge.function.get())) continue;
    const auto stream = edge.function->stream();
    TORCH_CHECK(!stream || stream->id() != 0, "nphm: ", what, ": a backward pass is captured for a tensor of which a graph of eager calls is alive "
                "(drop its outputs first, or capture on tensors of the graph's own)");
  }
}

// ---- rows of a table -----------------------------------------------------------------------------------------------------------

void check_rows(const char* what, const Tensor& rows, const Tensor& idx, double scale) {
  bound();
  on_gpu(what, rows);
  no_tangent(what, {&rows});
  TORCH_CHECK_TYPE(code_of(rows.scalar_type()) >= 0, what, ": rows of fp32, bf16 or fp16, not ", rows.scalar_type());
  TORCH_CHECK_TYPE(idx.scalar_type() == at::kLong || idx.scalar_type() == at::kInt, what, ": idx is an int32 or int64 tensor");
  TORCH_CHECK_VALUE(idx.device() == rows.device(), what, ": idx is on ", idx.device(), ", the rows on ", rows.device());
  TORCH_CHECK_VALUE(std::isfinite(scale), what, ": scale ", scale);
}
void check_table(const char* what, const Tensor& table) {
  TORCH_CHECK_VALUE(table.dim() == 2 && table.numel() > 0, what, ": a table [rows, width], not ", table.sizes());
}
int64_t padding_of(const char* what, std::optional<int64_t> padding, int64_t rows) {
  if (!padding) return -1;
  TORCH_CHECK_VALUE(-rows <= *padding && *padding < rows, what, ": padding_idx ", *padding, " is no row of ", rows);
  return *padding < 0 ? *padding + rows : *padding;
}
// rows contiguous, at least a row apart (a copy where they are not) -> elements between them
int64_t row_strided(Tensor& t) {
  if (!t.is_contiguous() && (t.stride(1) != 1 || t.stride(0) < t.size(1))) t = t.contiguous();
  return t.is_contiguous() ? t.size(1) : t.stride(0);
}
int bits_of(const Tensor& idx) { return idx.scalar_type() == at::kLong ? 64 : 32; }

Tensor lookup(Tensor table, const Tensor& idx, double scale) {
  const c10::DeviceGuard guard(table.device());
  const int64_t ld = row_strided(table);
  const Tensor i = idx.contiguous();
  auto sizes = idx.sizes().vec();
  sizes.push_back(table.size(1));
  Tensor out = at::empty(sizes, table.options());
  check(lib.rows_lookup(const_of(table), table.size(0), table.size(1), ld, code_of(table.scalar_type()), const_of(i), bits_of(i), i.numel(),
                        float(scale), at_of(out), stream_of(table)), "nphm_rows_lookup");
  return out;
}

Tensor rows_grad(const Tensor& grad, const Tensor& idx, int64_t rows, double scale, std::optional<int64_t> padding) {
  const char* what = "lookup_rows_grad";
  check_rows(what, grad, idx, scale);
  TORCH_CHECK_VALUE(grad.dim() >= 1 && grad.sizes().slice(0, grad.dim() - 1) == idx.sizes(), what, ": grad ", grad.sizes(), " does not fit idx ",
                    idx.sizes());
  const int64_t D = grad.size(-1), count = idx.numel();
  TORCH_CHECK_VALUE(rows >= 1 && D >= 1, what, ": an empty table");
  const int64_t pad = padding_of(what, padding, rows);
  const at::NoGradGuard no_grad;
  const c10::DeviceGuard guard(grad.device());
  Tensor g = grad.dim() == 2 ? grad : grad.reshape({-1, D});
  const int64_t ld = row_strided(g);
  const Tensor i = idx.contiguous();
  const int code = code_of(grad.scalar_type());
  const size_t need = lib.rows_grad_ws(rows, D, count, code);
  Tensor out = at::empty({rows, D}, grad.options()), ws = workspace(need, grad);
  check(lib.rows_grad(const_of(g), count, D, ld, code, const_of(i), bits_of(i), rows, pad, float(scale), at_of(out), at_of(ws), need,
                      stream_of(grad)), "nphm_rows_grad");
  return out;
}

// what the gradient of a lookup is: dense; an entry for every index, which is row 0 and zeros where it must not count; the same with
// padding left on its own row (a module's: an optimiser that steps every row it finds named then moves no row by it)
enum { GRAD_DENSE = 0, GRAD_ENTRIES = 1, GRAD_ENTRIES_PADDED = 2 };

struct LookupNode : torch::autograd::Function<LookupNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& table, const Tensor& idx, double scale, int64_t padding, int64_t sparse) {
    ctx->save_for_backward({idx});
    ctx->saved_data["meta"] = std::vector<int64_t>{table.size(0), padding, sparse};
    ctx->saved_data["scale"] = scale;
    return lookup(table, idx, scale);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor idx = ctx->get_saved_variables()[0], &g = grads[0];
    const auto meta = ctx->saved_data["meta"].toIntVector();
    const int64_t rows = meta[0], padding = meta[1];
    const double scale = ctx->saved_data["scale"].toDouble();
    Tensor out;
    no_tangent("lookup_rows", {&g});
    check_leaves("lookup_rows");
    if (meta[2] == GRAD_DENSE) {
      out = rows_grad(g, idx, rows, scale, padding < 0 ? std::nullopt : std::optional<int64_t>(padding));
    } else {
      // an entry an index, as nn.Embedding(sparse=True) leaves it; an entry that must not count names a row that exists and adds zeros
      const at::NoGradGuard no_grad;
      const c10::DeviceGuard guard(g.device());
      const Tensor i = idx.contiguous();
      const int64_t count = i.numel(), D = g.size(-1);
      Tensor g2 = g.dim() == 2 ? g : g.reshape({count, D});
      const int64_t ld = row_strided(g2);
      Tensor index = at::empty({1, count}, i.options().dtype(at::kLong)), values = at::empty({count, D}, g.options());
      check(lib.rows_entries(const_of(g2), count, D, ld, code_of(g.scalar_type()), const_of(i), bits_of(i), rows, padding, float(scale),
                             static_cast<int64_t*>(at_of(index)), at_of(values), stream_of(g)), "nphm_rows_entries");
      if (meta[2] == GRAD_ENTRIES_PADDED && padding >= 0) index.view({count}).masked_fill_(i.view({count}).eq(padding), padding);
      out = at::_sparse_coo_tensor_unsafe(index, values, {rows, D}, values.options().layout(at::kSparse));
    }
    return once({out, Tensor(), Tensor(), Tensor(), Tensor()}, "lookup_rows");
  }
};

Tensor lookup_rows(const Tensor& table, const Tensor& idx, double scale, std::optional<int64_t> padding_idx, int64_t sparse) {
  const char* what = "lookup_rows";
  check_rows(what, table, idx, scale);
  check_table(what, table);
  const int64_t padding = padding_of(what, padding_idx, table.size(0));
  if (table.requires_grad() && at::GradMode::is_enabled()) return LookupNode::apply(table, idx, scale, padding, sparse);
  return lookup(table, idx, scale);
}

void renorm_rows(const Tensor& table, const Tensor& idx, double max_norm) {
  const char* what = "renorm_rows_";
  check_rows(what, table, idx, 1.0);
  check_table(what, table);
  const int64_t V = table.size(0), D = table.size(1);
  TORCH_CHECK_VALUE((D == 1 || table.stride(1) == 1) && (V == 1 || table.stride(0) >= D), what, ": a table with contiguous rows");
  TORCH_CHECK_VALUE(max_norm >= 0, what, ": max_norm ", max_norm);
  const c10::DeviceGuard guard(table.device());
  const Tensor i = idx.contiguous();
  Tensor flags = at::empty({V}, table.options().dtype(at::kByte).requires_grad(false));
  check(lib.rows_renorm(at_of(table), V, D, std::max(table.stride(0), D), code_of(table.scalar_type()), const_of(i), bits_of(i), i.numel(),
                        float(max_norm), at_of(flags), stream_of(table)), "nphm_rows_renorm");
  written(table);
}

// ---- dense layer in 16 bits ------------------------------------------------------------------------------------------------------

Tensor rows_of(const Tensor& t) { return (t.dim() == 2 ? t : t.reshape({-1, t.size(-1)})).contiguous(); }

std::tuple<Tensor, Tensor> layer_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& residual, int64_t act, double beta,
                                         bool keep) {
  const c10::DeviceGuard guard(x.device());
  const Tensor w = weight.contiguous();
  const int64_t N = w.size(0), K = w.size(1), M = x.numel() / K;
  auto sizes = x.sizes().vec();
  sizes.back() = N;
  Tensor y = at::empty(sizes, x.options()), z;
  if (keep && act) z = at::empty({M, N}, x.options());
  if (M) {
    const Tensor x2 = rows_of(x), b = bias.defined() ? bias.contiguous() : bias, r = residual.defined() ? residual.contiguous() : residual;
    const size_t need = lib.forward_ws(const_of(x2), const_of(w), M, N, K);
    Tensor ws = workspace(need, x);
    check(lib.forward(const_of(x2), const_of(w), const_of(b), const_of(r), at_of(y), at_of(z), M, N, K, code_of(x.scalar_type()), int(act), float(beta),
                      at_of(ws), need, stream_of(x)), "nphm_layer16_forward");
  }
  return {y, z};
}

struct LayerNode : torch::autograd::Function<LayerNode> {
  // asked: the inputs that ask for a gradient, one bit each (x, weight, bias, residual).  x is kept for weight's gradient, weight for x's, z for
  // the first three.
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias,
                        const std::optional<Tensor>& residual, int64_t act, double beta, int64_t asked) {
    auto [y, z] = layer_forward(x, weight, bias.value_or(Tensor()), residual.value_or(Tensor()), act, beta, (asked & 7) != 0);
    ctx->save_for_backward({asked & 2 ? x : Tensor(), asked & 1 ? weight : Tensor(), z});
    const int64_t there = 3 | (bias && bias->defined() ? 4 : 0) | (residual && residual->defined() ? 8 : 0);
    ctx->saved_data["meta"] = std::vector<int64_t>{act, asked, there, weight.size(0), weight.size(1)};
    ctx->saved_data["sizes"] = x.sizes().vec();
    ctx->saved_data["beta"] = beta;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1], &z = saved[2], &g = grads[0];
    const auto meta = ctx->saved_data["meta"].toIntVector(), sizes = ctx->saved_data["sizes"].toIntVector();
    const int64_t act = meta[0], N = meta[3], K = meta[4];
    const double beta = ctx->saved_data["beta"].toDouble();
    // of those that asked, the ones that this pass is for (an edge for every tensor there is)
    int64_t asked = 0;
    for (int64_t bit = 1, edge = 0; bit <= 8; bit *= 2)
      if (meta[2] & bit) asked |= ctx->needs_input_grad(size_t(edge++)) ? meta[1] & bit : 0;
    variable_list out(7);                                            // (one for each argument of forward)
    no_tangent("linear_act", {&g});
    check_leaves("linear_act");
    {
      const at::NoGradGuard no_grad;
      const c10::DeviceGuard guard(g.device());
      const int64_t M = g.numel() / N;
      auto made = [&](int64_t bit, at::IntArrayRef shape) {
        if (!(asked & bit)) return Tensor();
        return M ? at::empty(shape, g.options()) : at::zeros(shape, g.options());
      };
      const Tensor dx = made(1, sizes), dw = made(2, {N, K}), db = made(4, {N});
      if (M && (asked & 7)) {
        const Tensor g2 = rows_of(g), x2 = asked & 2 ? rows_of(x) : Tensor(), w = asked & 1 ? weight.contiguous() : Tensor();
        const size_t need = lib.backward_ws(const_of(g2), const_of(x2), const_of(w), M, N, K, int(act));
        const Tensor ws = workspace(need, g);
        check(lib.backward(const_of(g2), const_of(x2), const_of(w), const_of(z), at_of(dx), at_of(dw), at_of(db), M, N, K, code_of(g.scalar_type()),
                           int(act), float(beta), at_of(ws), need, stream_of(g)), "nphm_layer16_backward");
      }
      out[0] = dx;
      out[1] = dw;
      out[2] = db;
      if (asked & 8) out[3] = g;
    }
    return once(std::move(out), "linear_act");
  }
};

Tensor linear_act(const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias_, const std::optional<Tensor>& residual_, int64_t act,
                  double beta) {
  const char* what = "linear_act";
  bound();
  const Tensor bias = bias_.value_or(Tensor()), residual = residual_.value_or(Tensor());
  on_gpu(what, x);
  on_gpu(what, weight);
  no_tangent(what, {&x, &weight, &bias, &residual});
  TORCH_CHECK_TYPE(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf, what, ": bf16 or fp16 tensors, not ", x.scalar_type());
  TORCH_CHECK_VALUE(x.dim() >= 1 && weight.dim() == 2 && x.size(-1) == weight.size(1) && weight.numel() > 0, what, ": x ", x.sizes(),
                    " does not fit weight ", weight.sizes());
  const int64_t N = weight.size(0);
  TORCH_CHECK_VALUE(!bias.defined() || (bias.dim() == 1 && bias.size(0) == N), what, ": bias has the shape (", N, ",)");
  if (residual.defined())
    TORCH_CHECK_VALUE(residual.dim() == x.dim() && residual.size(-1) == N
                          && residual.sizes().slice(0, x.dim() - 1) == x.sizes().slice(0, x.dim() - 1), what, ": residual has the shape of the result");
  int64_t asked = x.requires_grad() ? 1 : 0;
  int bit = 2;
  for (const Tensor* t : {&weight, &bias, &residual}) {
    if (t->defined()) {
      TORCH_CHECK_TYPE(t->scalar_type() == x.scalar_type() && t->device() == x.device(), what, ": all tensors on one device, of one type");
      if (t->requires_grad()) asked |= bit;
    }
    bit *= 2;
  }
  TORCH_CHECK_VALUE(act != 4 || (std::isfinite(beta) && beta > 0), what, ": Softplus takes a positive beta, not ", beta);
  if (asked && at::GradMode::is_enabled()) return LayerNode::apply(x, weight, bias_, residual_, act, beta, asked);
  return std::get<0>(layer_forward(x, weight, bias, residual, act, beta, false));
}

// ---- global gradient norm ----------------------------------------------------------------------------------------------------------

// the tensors of a Python list (of the caller's own: it keeps them alive)
std::vector<const Tensor*> tensors_of(const std::string& what, PyObject* list) {
  TORCH_CHECK_TYPE(PyList_Check(list), what, ": a list of tensors");
  std::vector<const Tensor*> all(size_t(PyList_GET_SIZE(list)));
  for (size_t i = 0; i < all.size(); ++i) {
    PyObject* item = PyList_GET_ITEM(list, Py_ssize_t(i));
    TORCH_CHECK_TYPE(THPVariable_Check(item), what, ": tensors, not ", Py_TYPE(item)->tp_name);
    all[i] = &THPVariable_Unpack(item);
  }
  return all;
}

// whether two elements of a tensor lie in one place, or cannot be told apart simply: sorted by stride, each dimension has to step over
// all that the ones below it reach (views of a dense tensor do; expanded and unfolded ones do not)
bool meets_itself(const Tensor& t) {
  if (t.is_contiguous() || t.numel() < 2) return false;
  std::vector<std::pair<int64_t, int64_t>> dims;
  for (int64_t d = 0; d < t.dim(); ++d)
    if (t.size(d) > 1) dims.emplace_back(t.stride(d), t.size(d));
  std::sort(dims.begin(), dims.end());
  int64_t reach = 0;
  for (const auto& [stride, size] : dims) {
    if (stride <= reach) return true;
    reach += stride * (size - 1);
  }
  return false;
}

// the bytes of a tensor: from its first on, dimensions of more than one place as (stride, places), a single byte the smallest
struct Places {
  uintptr_t first, end;
  std::vector<std::pair<int64_t, int64_t>> dims;
  explicit Places(const Tensor& t) : first(reinterpret_cast<uintptr_t>(t.const_data_ptr())) {
    const int64_t e = int64_t(t.element_size());
    int64_t reach = e - 1;
    if (t.is_non_overlapping_and_dense()) {                          // (whatever the order of its dimensions)
      reach = t.numel() * e - 1;
      dims.emplace_back(1, t.numel() * e);
    } else {
      dims.emplace_back(1, e);
      for (int64_t d = 0; d < t.dim(); ++d)
        if (t.size(d) > 1 && t.stride(d)) dims.emplace_back(t.stride(d) * e, t.size(d)), reach += t.stride(d) * e * (t.size(d) - 1);
    }
    end = t.numel() ? first + uintptr_t(reach) + 1 : first;
  }
  bool apart(const Places& o) const { return first == end || o.first == o.end || end <= o.first || o.end <= first; }
};

// Whether two tensors share a byte: a.first + sum x_i s_i = b.first + sum y_j t_j, 0 <= x_i, y_j < their places.  Dimensions of one stride
// are one unknown with a range; from the largest stride down, only values from which the smaller ones reach the rest are tried
// (one or two each for views of one buffer).  Strides that have nothing to do with each other could take long: they count as
// meeting after 100 000 tries.
bool share(const Places& a, const Places& b) {
  if (a.apart(b)) return false;
  struct Term { int64_t stride, lo, hi; };
  std::vector<Term> terms;
  auto add = [&](int64_t stride, int64_t lo, int64_t hi) {
    for (Term& t : terms)
      if (t.stride == stride) { t.lo += lo; t.hi += hi; return; }
    terms.push_back({stride, lo, hi});
  };
  for (const auto& [stride, places] : a.dims) add(stride, 0, places - 1);
  for (const auto& [stride, places] : b.dims) add(stride, 1 - places, 0);
  std::sort(terms.begin(), terms.end(), [](const Term& x, const Term& y) { return x.stride > y.stride; });
  std::vector<int64_t> low(terms.size() + 1), high(terms.size() + 1);          // what the terms from i on reach
  for (size_t i = terms.size(); i-- > 0;) {
    low[i] = low[i + 1] + terms[i].lo * terms[i].stride;
    high[i] = high[i + 1] + terms[i].hi * terms[i].stride;
  }
  int tries = 100000;
  auto down = [](int64_t v, int64_t s) { return v >= 0 ? v / s : -((-v + s - 1) / s); };
  auto reaches = [&](auto&& self, size_t i, int64_t rest) -> bool {
    if (rest < low[i] || rest > high[i]) return false;
    if (i == terms.size() || --tries < 0) return true;
    const Term& t = terms[i];
    const int64_t from = std::max(t.lo, -down(high[i + 1] - rest, t.stride)), to = std::min(t.hi, down(rest - low[i + 1], t.stride));
    for (int64_t x = from; x <= to; ++x)
      if (self(self, i + 1, rest - x * t.stride)) return true;
    return false;
  };
  return reaches(reaches, 0, int64_t(b.first) - int64_t(a.first));
}

// -> norm; `out` None: the norm alone, the list itself: in place.  out[i] may be grads[i].
Tensor clip(const std::string& what, PyObject* grad_list, PyObject* out_list, int kind, double limit) {
  bound();
  const std::vector<const Tensor*> grads = tensors_of(what, grad_list),
                                   out = out_list == Py_None ? std::vector<const Tensor*>{} : out_list == grad_list ? grads : tensors_of(what, out_list);
  const size_t n = grads.size();
  const bool writes = !out.empty(), in_place = out_list == grad_list, forward_mode = in_forward_mode();
  TORCH_CHECK_VALUE(n && (!writes || out.size() == n), what, ": ", n, " gradients, ", out.size(), " tensors in out");
  const at::NoGradGuard no_grad;
  const at::Device device = grads[0]->device();
  for (const Tensor* g : grads) {
    TORCH_CHECK_TYPE(g->is_cuda() && g->layout() == at::kStrided, what, ": dense tensors on a ROCm device (these operators have no CPU form)");
    TORCH_CHECK_TYPE(code_of(g->scalar_type()) >= 0, what, ": fp32, bf16 or fp16 gradients, not ", g->scalar_type());
    TORCH_CHECK_VALUE(g->device() == device, what, ": gradients on ", device, " and ", g->device(), ": one call takes one device's");
  }
  const c10::DeviceGuard guard(device);
  std::vector<const void*> from(n);
  std::vector<void*> to(writes ? n : 0);
  std::vector<int64_t> counts(n);
  std::vector<int> codes(n);
  std::vector<Tensor> held;                                          // copies that the launches read or write
  std::vector<std::pair<Tensor, Tensor>> back;
  std::vector<size_t> copied;
  for (size_t i = 0; i < n; ++i) {
    const Tensor *g = grads[i], *o = writes ? out[i] : g;
    TORCH_CHECK_VALUE(in_place || (o->numel() == g->numel() && o->scalar_type() == g->scalar_type() && o->device() == device && o->layout() == at::kStrided),
                      what, ": out has a tensor of the size, type and device of each gradient");
    if (forward_mode) {
      no_tangent(what.c_str(), *g);
      no_tangent(what.c_str(), *o);
    }
    counts[i] = g->numel();
    codes[i] = code_of(g->scalar_type());
    // any order of dimensions will do, if it is the same on both sides and leaves no gap
    if (!(g->is_contiguous() && (in_place || o->is_contiguous()))
        && !(g->is_non_overlapping_and_dense() && g->sizes() == o->sizes() && g->strides() == o->strides())) {
      held.push_back(g->contiguous());
      copied.push_back(i);
      from[i] = held.back().const_data_ptr();
      if (!writes) continue;
      TORCH_CHECK(!meets_itself(*o), "nphm: ", what, ": a tensor to be written has several elements in one place");
      back.emplace_back(*o, at::empty_like(held.back()));
      to[i] = back.back().second.mutable_data_ptr();
      continue;
    }
    from[i] = g->const_data_ptr();
    if (writes) to[i] = o->mutable_data_ptr();
  }
  // tensors of which the launches see copies, or whose results come from a copy, against all others; those whose own memory is handed to the C
  // entry are compared with each other behind it
  if (!held.empty() && writes) {
    std::vector<Places> read, wrote;
    for (size_t i = 0; i < n; ++i) {
      read.emplace_back(*grads[i]);
      wrote.emplace_back(*out[i]);
    }
    for (const size_t i : copied)
      for (size_t k = 0; k < n; ++k)
        TORCH_CHECK(k == i || !(share(wrote[i], wrote[k]) || (!in_place && (share(wrote[i], read[k]) || share(read[i], wrote[k])))), "nphm: ", what,
                    ": two of the tensors share memory");
  }
  const size_t need = lib.clip_ws(counts.data(), int(n));
  const Tensor ws = workspace(need, *grads[0]), norm = at::empty({}, grads[0]->options().dtype(at::kFloat).requires_grad(false));
  void* const stream = stream_of(*grads[0]);
  PyThreadState* const python = PyEval_SaveThread();                 // (no exception leaves a C entry)
  const int rc = lib.clip(from.data(), writes ? to.data() : nullptr, counts.data(), codes.data(), int(n), kind, limit,
                          static_cast<float*>(norm.mutable_data_ptr()), at_of(ws), need, stream);
  PyEval_RestoreThread(python);
  check(rc, "nphm_clip_grads");
  for (auto& [o, flat] : back) o.copy_(flat.view(o.sizes()));
  for (const Tensor* o : out) written(*o);
  return norm;
}

// the duplicates of an uncoalesced row gradient folded, in place: the sum at a row's first entry, zeros at the others
void merge_rows(const Tensor& index, const Tensor& values, int64_t rows) {
  bound();
  const at::NoGradGuard no_grad;
  const c10::DeviceGuard guard(values.device());
  if (values.numel() == 0) return;
  const Tensor i = index.contiguous(), flat = values.reshape({values.size(0), -1}).contiguous();
  const int code = code_of(values.scalar_type());
  const size_t need = lib.rows_grad_ws(rows, flat.size(1), flat.size(0), code);
  Tensor out = at::empty_like(flat), ws = workspace(need, flat);
  check(lib.rows_merge(const_of(flat), flat.size(0), flat.size(1), code, const_of(i), bits_of(i), rows, at_of(out), at_of(ws), need, stream_of(values)),
        "nphm_rows_merge");
  values.copy_(out.view(values.sizes()));
}

}  // namespace

// the C entries, in the order of `Entries`
extern "C" __attribute__((visibility("default"))) int nphm_torch_bind(void* const* entries, int n) {
  if (n != int(sizeof(Entries) / sizeof(void*))) return -1;
  memcpy(&lib, entries, sizeof(Entries));
  return 0;
}

// clip for Python: through the dispatcher 500 tensors in two lists took 60 us to hand over, 10 so.  A new reference to the norm, or null with the
// exception set.
extern "C" __attribute__((visibility("default"))) PyObject* nphm_torch_clip(PyObject* grads, PyObject* out, int kind, double limit, const char* what) {
  HANDLE_TH_ERRORS
  return THPVariable_Wrap(clip(what, grads, out, kind, limit));
  END_HANDLE_TH_ERRORS
}

TORCH_LIBRARY(nphm_amd, m) {
  m.def("lookup_rows(Tensor table, Tensor idx, float scale, int? padding_idx, int sparse) -> Tensor", &lookup_rows);
  m.def("lookup_rows_grad(Tensor grad, Tensor idx, int num_rows, float scale, int? padding_idx) -> Tensor", &rows_grad);
  m.def("renorm_rows_(Tensor(a!) table, Tensor idx, float max_norm) -> ()", &renorm_rows);
  m.def("linear_act(Tensor x, Tensor weight, Tensor? bias, Tensor? residual, int act, float beta) -> Tensor", &linear_act);
  m.def("merge_rows_(Tensor index, Tensor(a!) values, int rows) -> ()", &merge_rows);
}
