// Host path of an encoder block's operators beside attention (group norm with its activation, rotary positions): argument checks, results,
// workspaces, autograd nodes and launches, in one native call per operation.
#include "mvr_torch_operators.h"

namespace {

// ---- group norm -----------------------------------------------------------------------------------------

struct Norm {
  int64_t groups;
  double eps;
  int activation;
};

mvr_group_norm describe(const Norm& s, const at::Tensor& x, const at::Tensor& weight, const at::Tensor& bias) {
  mvr_group_norm a = {};
  a.dtype = head_code(x.scalar_type());
  a.parameter_dtype = weight.defined() ? head_code(weight.scalar_type()) : bias.defined() ? head_code(bias.scalar_type()) : a.dtype;
  a.activation = s.activation;
  a.eps = (float)s.eps;
  a.C = x.size(-1);
  a.N = x.size(0);
  a.S = 1;
  for (int64_t i = 1; i + 1 < x.dim(); ++i) a.S *= x.size(i);
  a.groups = s.groups;
  a.x = data_or_null(x);
  a.weight = data_or_null(weight);
  a.bias = data_or_null(bias);
  return a;
}

at::Tensor norm_workspace(const mvr_group_norm& a, bool backward, const at::Tensor& like) {
  int64_t bytes = 0;
  check(mvr_group_norm_workspace(&a, backward, &bytes));
  return bytes > 0 ? at::empty({bytes}, like.options().dtype(at::kByte).requires_grad(false)) : at::Tensor();
}

struct GroupNormBackward : public torch::autograd::Node {
  Norm s;
  SavedVariable x, weight, bias, statistics;

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list result(3);
    const at::Tensor x0 = x.unpack(), w0 = weight.unpack(), b0 = bias.unpack(), st = statistics.unpack();
    if (!grads[0].defined()) return result;
    {
      at::NoGradGuard no_grad;
      c10::cuda::CUDAGuard guard(x0.device());
      check_like(grads[0], x0);
      const at::Tensor xc = x0.contiguous(), g = grads[0].contiguous(), w = w0.defined() ? w0.contiguous() : w0, b = b0.defined() ? b0.contiguous() : b0;
      mvr_group_norm a = describe(s, xc, w, b);
      const at::Tensor gx = at::empty(xc.sizes(), xc.options().requires_grad(false));
      a.grad_out = data_or_null(g);
      a.grad_x = data_or_null(gx);
      a.mean = (float*)data_or_null(st);
      a.rstd = a.mean ? a.mean + a.N * a.groups : nullptr;
      a.mean_rest = a.mean ? a.rstd + a.N * a.groups : nullptr;
      result[0] = gx;
      if (w0.defined() && task_should_compute_output(1)) {
        result[1] = at::empty(w0.sizes(), w0.options().requires_grad(false));
        a.grad_weight = data_or_null(result[1]);
      }
      if (b0.defined() && task_should_compute_output(2)) {
        result[2] = at::empty(b0.sizes(), b0.options().requires_grad(false));
        a.grad_bias = data_or_null(result[2]);
      }
      const at::Tensor ws = norm_workspace(a, true, gx);
      check(mvr_group_norm_backward(&a, ws.defined() ? ws.data_ptr() : nullptr, ws.defined() ? ws.numel() : 0, stream_of(gx)));
    }
    variable_list from = {grads[0], x0, w0, b0};
    once_differentiable("group_norm", result, from);
    if (!task_should_compute_output(0)) result[0] = at::Tensor();
    return result;
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* t : {&x, &weight, &bias, &statistics}) t->reset_data();
  }
  std::string name() const override { return "GroupNormActivationBackward"; }
};

at::Tensor group_norm(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& bias, const Norm& s) {
  const char* what = "group_norm";
  check_type(what, x);
  TORCH_CHECK(x.dim() >= 2, what, ": expected (images, ..., channels)");
  const int64_t C = x.size(-1);
  TORCH_CHECK(C >= 1, what, ": there must be a channel at least");
  TORCH_CHECK(s.groups >= 1 && C % s.groups == 0, what, ": groups (", s.groups, ") must divide the channels (", C, ")");
  TORCH_CHECK(std::isfinite(s.eps) && s.eps >= 0 && std::isfinite((float)s.eps), what, ": eps must be finite and not negative");
  for (const at::Tensor* t : {&weight, &bias}) {
    if (!t->defined()) continue;
    const char* name = t == &weight ? "weight" : "bias";
    TORCH_CHECK(t->device() == x.device(), "expected all tensors to be on the same CUDA device");
    TORCH_CHECK(t->dim() == 1 && t->size(0) == C, what, ": ", name, " must have one element per channel");
    TORCH_CHECK(t->scalar_type() == x.scalar_type() || t->scalar_type() == at::kFloat, what, ": ", name, " must be of the input's type or float32");
  }
  TORCH_CHECK(!weight.defined() || !bias.defined() || weight.scalar_type() == bias.scalar_type(), what, ": weight and bias must be of the same type");
  check_cuda(what, x);
  for (const at::Tensor* t : {&x, &weight, &bias}) check_tangent(what, *t);
  const bool graph = torch::autograd::compute_requires_grad(x, weight, bias);
  at::Tensor out, statistics;
  {
    at::NoGradGuard no_grad;
    c10::cuda::CUDAGuard guard(x.device());
    const at::Tensor xc = x.contiguous(), w = weight.defined() ? weight.contiguous() : weight, b = bias.defined() ? bias.contiguous() : bias;
    mvr_group_norm a = describe(s, xc, w, b);
    out = at::empty(xc.sizes(), xc.options().requires_grad(false));
    statistics = at::empty({3, a.N, s.groups}, out.options().dtype(at::kFloat));
    a.out = data_or_null(out);
    a.mean = (float*)data_or_null(statistics);
    a.rstd = a.mean ? a.mean + a.N * s.groups : nullptr;
    a.mean_rest = a.mean ? a.rstd + a.N * s.groups : nullptr;
    const at::Tensor ws = norm_workspace(a, false, out);
    check(mvr_group_norm_forward(&a, ws.defined() ? ws.data_ptr() : nullptr, ws.defined() ? ws.numel() : 0, stream_of(out)));
  }
  if (graph) {
    auto node = std::shared_ptr<GroupNormBackward>(new GroupNormBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x, weight, bias));
    node->s = s;
    node->x = SavedVariable(x, false);
    node->weight = SavedVariable(weight, false);
    node->bias = SavedVariable(bias, false);
    node->statistics = SavedVariable(statistics, false);
    torch::autograd::set_history(out, node);
  }
  return out;
}

// ---- rotary positions -----------------------------------------------------------------------------------

struct Rotary {
  int axes = 0;
  int64_t sections[MVR_MAX_AXES] = {};
  double base;
  bool interleaved;
};

int position_code(at::ScalarType t) { return t == at::kFloat ? MVR_INDEX_F32 : t == at::kInt ? MVR_INDEX_I32 : t == at::kLong ? MVR_INDEX_I64 : -1; }

// Both tensors turned (or turned back); an undefined one is left out.
void turn(const Rotary& s, const at::Tensor (&x)[2], const at::Tensor& positions, bool inverse, at::Tensor (&out)[2]) {
  at::NoGradGuard no_grad;
  const at::Tensor& like = x[0].defined() ? x[0] : x[1];
  c10::cuda::CUDAGuard guard(like.device());
  mvr_rotary a = {};
  a.dtype = head_code(like.scalar_type());
  a.interleaved = s.interleaved;
  a.inverse = inverse;
  a.axes = s.axes;
  for (int i = 0; i < s.axes; ++i) a.sections[i] = s.sections[i];
  a.base = s.base;
  a.N = like.size(0);
  a.L = like.size(1);
  a.D = like.size(3);
  a.positions = data_or_null(positions);
  a.position_dtype = position_code(positions.scalar_type());
  for (int k = 0; k < 3; ++k) a.position_strides[k] = positions.stride(k);
  at::Tensor rows[2];
  int to = 0;
  for (int i = 0; i < 2; ++i) {
    if (!x[i].defined()) continue;
    // (the kernel's rows are of consecutive elements, and 32-bit strides apart)
    const bool good = (x[i].size(3) <= 1 || x[i].stride(3) == 1) && x[i].stride(1) <= INT32_MAX && x[i].stride(2) <= INT32_MAX;
    rows[i] = good ? x[i] : x[i].contiguous();
    out[i] = at::empty(x[i].sizes(), x[i].options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous));
    a.heads[to] = x[i].size(2);
    a.x[to] = data_or_null(rows[i]);
    a.out[to] = data_or_null(out[i]);
    for (int k = 0; k < 3; ++k) a.strides[to][k] = rows[i].stride(k);
    ++to;
  }
  check(mvr_rotary_positions(&a, stream_of(like)));
}

struct RotaryBackward : public torch::autograd::Node {
  Rotary s;
  SavedVariable positions;
  at::ScalarType type;

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list result(grads.size());
    const at::Tensor at = positions.unpack();
    at::Tensor from[2], to[2];
    bool any = false;
    for (size_t i = 0; i < grads.size(); ++i) {
      if (!grads[i].defined() || !task_should_compute_output(i)) continue;
      TORCH_CHECK(grads[i].scalar_type() == type, "expected scalar type torch.", type_name(type), " but found torch.", type_name(grads[i].scalar_type()));
      from[i] = grads[i];
      any = true;
    }
    if (!any) return result;
    turn(s, from, at, true, to);
    for (size_t i = 0; i < grads.size(); ++i) result[i] = to[i];
    once_differentiable("rotary_positions", result, grads);
    return result;
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    positions.reset_data();
  }
  std::string name() const override { return "RotaryPositionsBackward"; }
};

void rotary_positions(const at::Tensor& query, const at::Tensor& key, const at::Tensor& positions, Rotary s, bool default_sections, at::Tensor (&out)[2]) {
  const char* what = "rotary_positions";
  check_type(what, query);
  TORCH_CHECK(query.dim() == 4, what, ": expected query (images, states, heads, dim)");
  const int64_t N = query.size(0), L = query.size(1), D = query.size(3);
  TORCH_CHECK(query.size(2) >= 1 && D >= 1, what, ": heads and head size must not be 0");
  if (key.defined()) {
    check_like(key, query);
    TORCH_CHECK(key.dim() == 4 && key.size(0) == N && key.size(1) == L && key.size(2) >= 1 && key.size(3) == D, what,
                ": key must be (images, states, heads, dim) of the query's images, states and head size");
  }
  TORCH_CHECK(positions.device() == query.device(), "expected all tensors to be on the same CUDA device");
  TORCH_CHECK(positions.dim() == 3 && positions.size(0) == N && positions.size(1) == L, what, ": positions must be (images, states, axes)");
  TORCH_CHECK(position_code(positions.scalar_type()) >= 0, what, ": positions must be float32, int32 or int64");
  TORCH_CHECK(!positions.requires_grad(), what, ": there is no gradient of positions");
  const int64_t axes = positions.size(2);
  TORCH_CHECK(axes >= 1 && axes <= MVR_MAX_AXES, what, ": positions must have 1 to ", MVR_MAX_AXES, " axes, but have ", axes);
  if (default_sections) {
    s.axes = (int)axes;
    for (int64_t i = 0; i < axes; ++i) s.sections[i] = D / 2 / axes + (i < D / 2 % axes ? 1 : 0);
  }
  TORCH_CHECK(s.axes == axes, what, ": sections must have one element per axis");
  int64_t pairs = 0;
  for (int i = 0; i < s.axes; ++i) {
    TORCH_CHECK(s.sections[i] >= 0 && s.sections[i] <= D, what, ": sections must be numbers of pairs, together at most half of the head size");
    pairs += s.sections[i];
  }
  TORCH_CHECK(2 * pairs <= D, what, ": sections must be numbers of pairs, together at most half of the head size");
  TORCH_CHECK(pairs <= 256, what, ": at most 256 pairs of columns can be turned");
  TORCH_CHECK(std::isfinite(s.base) && s.base >= 1, what, ": base must be finite and at least 1");
  check_cuda(what, query);
  check_tangent(what, query);
  if (key.defined()) check_tangent(what, key);
  const at::Tensor x[2] = {query, key};
  turn(s, x, positions, false, out);
  if (!torch::autograd::compute_requires_grad(query, key)) return;
  auto node = std::shared_ptr<RotaryBackward>(new RotaryBackward(), torch::autograd::deleteNode);
  node->set_next_edges(key.defined() ? torch::autograd::collect_next_edges(query, key) : torch::autograd::collect_next_edges(query));
  node->s = s;
  node->type = query.scalar_type();
  node->positions = SavedVariable(positions, false);
  variable_list outputs = {out[0]};
  if (key.defined()) outputs.push_back(out[1]);
  torch::autograd::set_history(outputs, node);
}

// ---- Python ---------------------------------------------------------------------------------------------

// group_norm(x, groups, weight, bias, eps, activation)
PyObject* py_group_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 6);
  const at::Tensor& x = tensor_arg(a[0], "x");
  Norm s;
  s.groups = whole_arg(a[1], "groups");
  const at::Tensor weight = optional_tensor(a[2], "weight"), bias = optional_tensor(a[3], "bias");
  s.eps = number_arg(a[4]);
  s.activation = (int)whole_arg(a[5], "activation");
  at::Tensor out;
  {
    pybind11::gil_scoped_release nogil;
    out = group_norm(x, weight, bias, s);
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// rotary_positions(query, key or None, positions, sections or None, base, interleaved) -> turned query, or (query, key)
PyObject* py_rotary_positions(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 6);
  const at::Tensor& query = tensor_arg(a[0], "query");
  const at::Tensor key = optional_tensor(a[1], "key"), positions = tensor_arg(a[2], "positions");
  Rotary s;
  if (a[3] != Py_None) {
    PyObject* list = PySequence_Fast(a[3], "sections must be a sequence of whole numbers");
    if (!list) throw python_error();
    const Py_ssize_t count = PySequence_Fast_GET_SIZE(list);
    s.axes = (int)std::min<Py_ssize_t>(count, MVR_MAX_AXES + 1);
    try {
      for (Py_ssize_t i = 0; i < count && i < MVR_MAX_AXES; ++i) s.sections[i] = whole_arg(PySequence_Fast_GET_ITEM(list, i), "sections");
    } catch (...) {
      Py_DECREF(list);
      throw;
    }
    Py_DECREF(list);
  }
  s.base = number_arg(a[4]);
  const int interleaved = PyObject_IsTrue(a[5]);
  if (interleaved < 0) throw python_error();
  s.interleaved = interleaved != 0;
  at::Tensor out[2];
  {
    pybind11::gil_scoped_release nogil;
    rotary_positions(query, key, positions, s, a[3] == Py_None, out);
  }
  if (!key.defined()) return THPVariable_Wrap(std::move(out[0]));
  PyObject* both = PyTuple_New(2);
  if (!both) throw python_error();
  PyTuple_SET_ITEM(both, 0, THPVariable_Wrap(std::move(out[0])));
  PyTuple_SET_ITEM(both, 1, THPVariable_Wrap(std::move(out[1])));
  return both;
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {{"group_norm", FAST(py_group_norm), nullptr}, {"rotary_positions", FAST(py_rotary_positions), nullptr}, {nullptr, nullptr, 0, nullptr}};

}  // namespace

namespace mvr_host {
PyMethodDef* encoder_methods() { return methods; }
}  // namespace mvr_host
