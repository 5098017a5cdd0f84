// Host path of the operators behind the roi modules (attention to an encoder's states or in a window, dropout, log-probabilities of labels):
// argument checks, results, workspaces, autograd nodes and launches, in one native call per operation.
#include "mvr_torch_operators.h"

namespace {

// ---- attention ------------------------------------------------------------------------------------------

struct Attention {
  at::Tensor index, lengths, mask;  // or undefined
  double scale;
  bool in_window = false;           // ops.window_attention: a window instead of index and mask
  mvr_window window = {};           // without the address of `offsets`
  at::Tensor offsets;               // or undefined
  at::Tensor rest;                  // what the rounding of the result left, or undefined
  const char* name() const { return in_window ? "window_attention" : "cross_attention"; }
};

// A tensor of rows of D consecutive elements: the tensor itself, or a copy where its rows are apart in themselves or start where the
// tensor-core kernels cannot read them (16 bytes; states, which TMA reads, may not overlap either).
at::Tensor rows_of(const at::Tensor& t, bool states) {
  bool good = t.size(3) <= 1 || t.stride(3) == 1;
  if (good && t.numel() > 0 && t.scalar_type() != at::kFloat && t.size(3) % 8 == 0) {
    good = (uintptr_t)t.data_ptr() % 16 == 0;
    for (int i = 0; i < 3; ++i)
      if (t.size(i) > 1) good = good && t.stride(i) % 8 == 0 && (!states || t.stride(i) > 0);
  }
  return good ? t : t.contiguous();
}

// Half types with a head size that is no multiple of 8, which TMA cannot read: in calls of some size the operands are copied with zeros
// behind, which changes no product.  (Forward and backward, 33 columns, 4 heads: 16 x 49 rows over 4096 states 458 us, in the kernels
// of float arithmetic 883 us; 2 x 16 rows over 256 states, where the copies' launches count, 429 and 88 us.)
int64_t padded_size(const Attention& s, const at::Tensor& q, const at::Tensor& k) {
  const int64_t D = q.size(3), padded = (D + 7) / 8 * 8;
  if (q.scalar_type() == at::kFloat || D == padded || padded > 128) return D;
  double states = (double)k.size(1);
  // (a few tokens over long sequences: copying all of their states would cost more than the products with those in the window)
  if (s.in_window && q.size(1) < k.size(1) / 4) return D;
  if (s.in_window) states = std::min(states, (double)s.window.before + (double)s.window.after + 1 + (double)s.window.sinks);
  const double scores = (double)q.size(0) * q.size(1) * q.size(2) * states;
  return scores >= 1 << 22 ? padded : D;
}
at::Tensor padded(const at::Tensor& t, int64_t D) { return t.size(3) == D ? t : at::constant_pad_nd(t, {0, D - t.size(3)}); }
at::Tensor narrowed(const at::Tensor& t, int64_t D) { return t.size(3) == D ? t : t.narrow(3, 0, D).contiguous(); }

void set_strides(int64_t (&to)[3], const at::Tensor& t) {
  for (int i = 0; i < 3; ++i) to[i] = t.stride(i);
}

mvr_attention describe(const Attention& s, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v) {
  mvr_attention a = {};
  a.dtype = head_code(q.scalar_type());
  a.R = q.size(0); a.T = q.size(1); a.Hq = q.size(2); a.D = q.size(3);
  a.N = k.size(0); a.L = k.size(1); a.Hk = k.size(2);
  a.q = data_or_null(q); a.k = data_or_null(k); a.v = data_or_null(v);
  set_strides(a.q_strides, q);
  set_strides(a.k_strides, k);
  set_strides(a.v_strides, v);
  if (s.index.defined()) {
    a.has_index = 1;
    a.index = data_or_null(s.index);
    a.index_type = index_code(s.index.scalar_type());
    a.index_stride = s.index.stride(0);
  }
  if (s.lengths.defined()) {
    a.lengths = data_or_null(s.lengths);
    a.lengths_64 = s.lengths.scalar_type() == at::kLong;
  }
  if (s.mask.defined()) a.mask = (const unsigned char*)data_or_null(s.mask);
  a.scale = (float)s.scale;
  return a;
}

mvr_window window_of(const Attention& s) {
  mvr_window w = s.window;
  if (s.offsets.defined()) {
    w.offsets = data_or_null(s.offsets);
    w.offsets_64 = s.offsets.scalar_type() == at::kLong;
  }
  if (s.rest.defined()) w.rest = data_or_null(s.rest);
  return w;
}

at::Tensor workspace_of(const Attention& s, const mvr_attention& a, bool backward, const at::Tensor& like) {
  int64_t bytes = 0;
  check(s.in_window ? mvr_window_attention_workspace(&a, &s.window, backward, &bytes) : mvr_attention_workspace(&a, backward, &bytes));
  return bytes > 0 ? at::empty({bytes}, like.options().dtype(at::kByte).requires_grad(false)) : at::Tensor();
}

struct AttentionBackward : public torch::autograd::Node {
  Attention s;
  SavedVariable q, k, v, out, lse, index, lengths, mask, offsets, rest;

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list result(3);
    const at::Tensor q0 = q.unpack(), k0 = k.unpack(), v0 = v.unpack(), o = out.unpack(shared_from_this()), l = lse.unpack();
    Attention args = s;
    args.index = index.unpack();
    args.lengths = lengths.unpack();
    args.mask = mask.unpack();
    args.offsets = offsets.unpack();
    args.rest = rest.unpack();
    if (!grads[0].defined()) return result;
    {
      at::NoGradGuard no_grad;
      c10::cuda::CUDAGuard guard(q0.device());
      const int64_t D = q0.size(3), wide = padded_size(args, q0, k0);
      const at::Tensor qc = rows_of(padded(q0, wide), false), kc = rows_of(padded(k0, wide), true), vc = rows_of(padded(v0, wide), true),
                       oc = padded(o, wide);
      check_like(grads[0], q0);
      const at::Tensor g = rows_of(padded(grads[0], wide), false);
      mvr_attention a = describe(args, qc, kc, vc);
      const at::Tensor gq = at::empty(qc.sizes(), q0.options().requires_grad(false)), gk = at::empty(kc.sizes(), gq.options()),
                       gv = at::empty(kc.sizes(), gq.options());
      a.out = data_or_null(oc);
      a.lse = (float*)data_or_null(l);
      a.grad_out = data_or_null(g);
      set_strides(a.g_strides, g);
      a.grad_q = data_or_null(gq);
      a.grad_k = data_or_null(gk);
      a.grad_v = data_or_null(gv);
      const at::Tensor ws = workspace_of(args, a, true, gq);
      void* workspace = ws.defined() ? ws.data_ptr() : nullptr;
      const int64_t bytes = ws.defined() ? ws.numel() : 0;
      int* status = mvr_host::status_of(gq.device().index());
      const mvr_window w = window_of(args);
      check(args.in_window ? mvr_window_attention_backward(&a, &w, workspace, bytes, status, stream_of(gq))
                           : mvr_attention_backward(&a, workspace, bytes, status, stream_of(gq)));
      result = {narrowed(gq, D), narrowed(gk, D), narrowed(gv, D)};
    }
    once_differentiable(s.name(), result, {grads[0], q0, k0, v0});
    for (int i = 0; i < 3; ++i)
      if (!task_should_compute_output(i)) result[i] = at::Tensor();
    return result;
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* t : {&q, &k, &v, &out, &lse, &index, &lengths, &mask, &offsets, &rest}) t->reset_data();
  }
  std::string name() const override { return s.in_window ? "WindowAttentionBackward" : "CrossAttentionBackward"; }
};

at::Tensor attention(const at::Tensor& query, const at::Tensor& key, const at::Tensor& value, Attention s, bool default_scale) {
  const char* what = s.name();
  check_type(what, query);
  check_like(key, query);
  check_like(value, query);
  const char *regions = s.in_window ? "sequence" : "region", *images = s.in_window ? "sequence" : "image";
  TORCH_CHECK(query.dim() == 4 && key.dim() == 4, what, ": expected query (", regions, "s, tokens, heads, dim) and key (", images, "s, states, heads, dim)");
  TORCH_CHECK(value.sizes() == key.sizes(), what, ": key and value must have the same shape");
  TORCH_CHECK(key.size(3) == query.size(3), what, ": query and key must have the same head size");
  TORCH_CHECK(query.size(3) >= 1 && query.size(2) >= 1 && key.size(2) >= 1, what, ": heads and head size must not be 0");
  const int64_t R = query.size(0), N = key.size(0), L = key.size(1);
  if (s.index.defined()) {
    TORCH_CHECK(s.index.device() == query.device(), "expected all tensors to be on the same CUDA device");
    TORCH_CHECK(s.index.dim() == 1 && s.index.size(0) == R, what, ": batch_index must have one element per region");
    TORCH_CHECK(index_code(s.index.scalar_type()) >= 0, what, ": batch_index cannot be of type ", type_name(s.index.scalar_type()));
  } else {
    TORCH_CHECK(!s.in_window || R == N, what, ": query and key must be of the same sequences, but there are ", R, " and ", N);
    TORCH_CHECK(R == N, what, ": without batch_index there must be one region per image, but there are ", R, " and ", N);
  }
  if (s.lengths.defined()) {
    TORCH_CHECK(s.lengths.device() == query.device(), "expected all tensors to be on the same CUDA device");
    TORCH_CHECK(s.lengths.dim() == 1 && s.lengths.size(0) == N, what, ": lengths must have one element per ", images);
    TORCH_CHECK(s.lengths.scalar_type() == at::kInt || s.lengths.scalar_type() == at::kLong, what, ": lengths must be int32 or int64");
  }
  if (s.offsets.defined()) {
    TORCH_CHECK(s.offsets.device() == query.device(), "expected all tensors to be on the same CUDA device");
    TORCH_CHECK(s.offsets.dim() == 1 && s.offsets.size(0) == N, what, ": offsets must have one element per sequence");
    TORCH_CHECK(s.offsets.scalar_type() == at::kInt || s.offsets.scalar_type() == at::kLong, what, ": offsets must be int32 or int64");
  }
  TORCH_CHECK(s.window.before >= 0 && s.window.after >= 0 && s.window.sinks >= 0, what, ": before, after and sinks must not be negative");
  if (s.mask.defined()) {
    TORCH_CHECK(s.mask.device() == query.device(), "expected all tensors to be on the same CUDA device");
    TORCH_CHECK(s.mask.dim() == 2 && s.mask.size(0) == N && s.mask.size(1) == L, what, ": mask must be (images, states)");
    TORCH_CHECK(s.mask.scalar_type() == at::kBool, what, ": mask must be bool (true: the state is read)");
  }
  if (default_scale) s.scale = 1.0 / std::sqrt((double)query.size(3));
  TORCH_CHECK(std::isfinite((float)(s.scale * 1.4426950408889634)), what, ": scale must be finite (in float32, in powers of two)");
  TORCH_CHECK(query.size(3) <= 256, mvr_strerror(MVR_ERR_HEAD_SIZE));
  TORCH_CHECK(query.size(2) % key.size(2) == 0, mvr_strerror(MVR_ERR_HEADS));
  check_cuda(what, query);
  for (const at::Tensor* t : {&query, &key, &value}) check_tangent(what, *t);
  const bool graph = torch::autograd::compute_requires_grad(query, key, value);
  at::Tensor out, lse;
  {
    at::NoGradGuard no_grad;
    c10::cuda::CUDAGuard guard(query.device());
    if (s.lengths.defined()) s.lengths = s.lengths.contiguous();
    if (s.mask.defined()) s.mask = s.mask.contiguous();
    if (s.offsets.defined()) s.offsets = s.offsets.contiguous();
    const int64_t D = query.size(3), wide = padded_size(s, query, key);
    const at::Tensor q = rows_of(padded(query, wide), false), k = rows_of(padded(key, wide), true), v = rows_of(padded(value, wide), true);
    mvr_attention a = describe(s, q, k, v);
    const at::Tensor ws = workspace_of(s, a, false, q);
    out = at::empty(q.sizes(), query.options().requires_grad(false));
    if (graph) lse = at::empty({R, query.size(1), query.size(2)}, out.options().dtype(at::kFloat));
    // (a token with few states has slopes that are differences of near numbers: with the result as it is rounded they lose up to three times as
    // much as the rounding of a gradient)
    if (graph && s.in_window && query.scalar_type() != at::kFloat) s.rest = at::empty(q.sizes(), out.options().dtype(at::kBFloat16));
    a.out = data_or_null(out);
    a.lse = (float*)data_or_null(lse);
    void* workspace = ws.defined() ? ws.data_ptr() : nullptr;
    const int64_t bytes = ws.defined() ? ws.numel() : 0;
    int* status = mvr_host::status_of(query.device().index());
    const mvr_window w = window_of(s);
    check(s.in_window ? mvr_window_attention_forward(&a, &w, workspace, bytes, status, stream_of(query))
                      : mvr_attention_forward(&a, workspace, bytes, status, stream_of(query)));
    out = narrowed(out, D);
  }
  if (graph) {
    auto node = std::shared_ptr<AttentionBackward>(new AttentionBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(query, key, value));
    node->s.scale = s.scale;
    node->s.in_window = s.in_window;
    node->s.window = s.window;
    node->offsets = SavedVariable(s.offsets, false);
    node->rest = SavedVariable(s.rest, false);
    node->q = SavedVariable(query, false);
    node->k = SavedVariable(key, false);
    node->v = SavedVariable(value, false);
    node->lse = SavedVariable(lse, false);
    node->index = SavedVariable(s.index, false);
    node->lengths = SavedVariable(s.lengths, false);
    node->mask = SavedVariable(s.mask, false);
    torch::autograd::set_history(out, node);
    node->out = SavedVariable(out, true);
  }
  return out;
}

// ---- dropout --------------------------------------------------------------------------------------------

struct DropoutSeed {
  uint64_t value = 0, offset = 0;
  at::Tensor tensor;  // or undefined
};

at::Tensor drop(const at::Tensor& x, const at::Tensor& residual, double p, const DropoutSeed& seed) {
  at::NoGradGuard no_grad;
  c10::cuda::CUDAGuard guard(x.device());
  const at::Tensor xc = x.contiguous(), rc = residual.defined() ? residual.contiguous() : residual;
  at::Tensor out = at::empty(x.sizes(), x.options().requires_grad(false));
  check(mvr_dropout(xc.data_ptr(), data_or_null(rc), out.data_ptr(), head_code(x.scalar_type()), x.numel(), p, seed.value,
                    seed.tensor.defined() ? (const uint64_t*)seed.tensor.data_ptr() : nullptr, seed.offset, stream_of(x)));
  return out;
}

struct DropoutBackward : public torch::autograd::Node {
  double p;
  DropoutSeed seed;
  SavedVariable seed_tensor;
  at::ScalarType type;

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list result(2);
    if (!grads[0].defined()) return result;
    if (task_should_compute_output(0)) {
      TORCH_CHECK(grads[0].scalar_type() == type, "expected scalar type torch.", type_name(type), " but found torch.",
                  type_name(grads[0].scalar_type()));
      DropoutSeed from = seed;
      from.tensor = seed_tensor.unpack();
      variable_list gx = {drop(grads[0], at::Tensor(), p, from)};
      once_differentiable("dropout", gx, {grads[0]});
      result[0] = gx[0];
    }
    if (task_should_compute_output(1)) result[1] = grads[0];
    return result;
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    seed_tensor.reset_data();
  }
  std::string name() const override { return "CounterDropoutBackward"; }
};

at::Tensor dropout(const at::Tensor& x, double p, const DropoutSeed& seed, const at::Tensor& residual) {
  const char* what = "dropout";
  check_type(what, x);
  TORCH_CHECK_VALUE(p >= 0.0 && p <= 1.0, "dropout probability has to be between 0 and 1, but got ", p);
  if (residual.defined()) {
    check_like(residual, x);
    TORCH_CHECK(residual.sizes() == x.sizes(), what, ": x and residual must have the same shape");
  }
  if (seed.tensor.defined()) {
    TORCH_CHECK(seed.tensor.device() == x.device(), "expected all tensors to be on the same CUDA device");
    TORCH_CHECK(seed.tensor.scalar_type() == at::kLong && seed.tensor.numel() == 1, what, ": a seed tensor must hold one int64");
  }
  check_cuda(what, x);
  check_tangent(what, x);
  check_tangent(what, residual);
  at::Tensor out = drop(x, residual, p, seed);
  if (torch::autograd::compute_requires_grad(x, residual)) {
    auto node = std::shared_ptr<DropoutBackward>(new DropoutBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x, residual));
    node->p = p;
    node->type = x.scalar_type();
    node->seed.value = seed.value;
    node->seed.offset = seed.offset;
    node->seed_tensor = SavedVariable(seed.tensor, false);
    torch::autograd::set_history(out, node);
  }
  return out;
}

// ---- log-probabilities of labels --------------------------------------------------------------------------

// How scores (N, K, *space) lie in memory: positions consecutive (classes apart), or classes consecutive (rows).
struct ScoreLayout {
  bool rows;
  int64_t batch, space, batch_stride, class_stride;
};

at::Tensor classes_last(const at::Tensor& t) {
  std::vector<int64_t> order = {0};
  for (int64_t i = 2; i < t.dim(); ++i) order.push_back(i);
  order.push_back(1);
  return t.permute(order);
}

bool layout_of(const at::Tensor& x, ScoreLayout& o) {
  int64_t space = 1;
  bool packed = true;  // the positions of one class are consecutive
  for (int64_t i = x.dim() - 1; i >= 2; --i) {
    packed &= x.size(i) == 1 || x.stride(i) == space;
    space *= x.size(i);
  }
  const int64_t N = x.size(0), K = x.size(1);
  if (x.numel() == 0) {
    o = {false, N, space, 0, 0};
    return true;
  }
  if (space == 1 && (K == 1 || x.stride(1) == 1)) {
    o = {true, N, 1, x.stride(0), 1};
    return true;
  }
  if (x.dim() > 2 && space > 1 && classes_last(x).is_contiguous()) {
    o = {true, N * space, 1, K, 1};
    return true;
  }
  if (space > 1 && packed) {
    o = {false, N, space, x.stride(0), x.stride(1)};
    return true;
  }
  return false;
}

// A new tensor (N, K, *space), laid out as `layout` says.
at::Tensor scores_like(const at::Tensor& x, int64_t K, const ScoreLayout& layout, at::ScalarType type) {
  std::vector<int64_t> size = x.sizes().vec();
  const at::TensorOptions options = x.options().dtype(type).requires_grad(false);
  if (!layout.rows || x.dim() == 2) {
    size[1] = K;
    return at::empty(size, options);
  }
  size.erase(size.begin() + 1);
  size.push_back(K);
  std::vector<int64_t> order = {0, x.dim() - 1};
  for (int64_t i = 1; i + 1 < x.dim(); ++i) order.push_back(i);
  return at::empty(size, options).permute(order);
}

struct LabelLogProbsBackward : public torch::autograd::Node {
  SavedVariable logits, labels, lse, entropy;  // lse: (2, ...), its float and what that leaves of it

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list result(1);
    const at::Tensor x0 = logits.unpack(), y = labels.unpack(), l = lse.unpack(), h = entropy.unpack(shared_from_this());
    if (!grads[0].defined() && !grads[1].defined()) return result;
    {
      at::NoGradGuard no_grad;
      c10::cuda::CUDAGuard guard(x0.device());
      ScoreLayout in;
      at::Tensor x = x0;
      if (!layout_of(x, in)) {
        x = x.contiguous();
        layout_of(x, in);
      }
      at::Tensor g[2];
      for (int i = 0; i < 2; ++i)
        if (grads[i].defined()) {
          TORCH_CHECK(grads[i].scalar_type() == at::kFloat, "expected scalar type torch.float32 but found torch.",
                      type_name(grads[i].scalar_type()));
          g[i] = grads[i].contiguous();
        }
      const int64_t K = x.size(1);
      at::Tensor gx = scores_like(x, K, in, x.scalar_type());
      const int64_t positions = in.rows ? K : gx.stride(0), classes = in.rows ? 1 : in.space;
      const float* lse0 = (const float*)data_or_null(l);
      check(mvr_label_log_probs_backward_rest(data_or_null(x), head_code(x.scalar_type()), data_or_null(y),
                                              mvr_host::label_type(y.scalar_type()), lse0, lse0 ? lse0 + y.numel() : nullptr,
                                              (const float*)data_or_null(h), (const float*)data_or_null(g[0]),
                                              (const float*)data_or_null(g[1]), data_or_null(gx), in.batch, K, in.space,
                                              in.batch_stride, in.class_stride, positions, classes, stream_of(x)));
      result[0] = gx;
    }
    once_differentiable("label_log_probs", result, {grads[0], grads[1], x0});
    return result;
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* t : {&logits, &labels, &lse, &entropy}) t->reset_data();
  }
  std::string name() const override { return "LabelLogProbsBackward"; }
};

struct LabelLogProbs {
  at::Tensor log_prob, entropy, top_value, top_label;
};

LabelLogProbs label_log_probs(const at::Tensor& logits, const at::Tensor& labels, int64_t top) {
  const char* what = "label_log_probs";
  check_type(what, logits);
  TORCH_CHECK(logits.dim() >= 2, what, ": expected class scores (N, classes, ...)");
  TORCH_CHECK(labels.device() == logits.device(), "expected all tensors to be on the same CUDA device");
  TORCH_CHECK(mvr_host::label_type(labels.scalar_type()) >= 0, "\"", what, "\" not implemented for labels of type '",
              type_name(labels.scalar_type()), "'");
  const int64_t N = logits.size(0), K = logits.size(1);
  // (N, ...) or, as label fields are, (N, 1, ...)
  const bool field = labels.dim() == logits.dim();
  TORCH_CHECK((field && labels.size(0) == N && labels.size(1) == 1 && labels.sizes().slice(2) == logits.sizes().slice(2)) ||
                  (labels.dim() == logits.dim() - 1 && labels.size(0) == N && labels.sizes().slice(1) == logits.sizes().slice(2)),
              what, ": labels must be (N, ...) or (N, 1, ...) for scores (N, classes, ...)");
  TORCH_CHECK(K >= 1, what, ": there must be a class at least");
  TORCH_CHECK(top >= 0 && top <= MVR_MAX_TOP && top <= K, what, ": top must be between 0 and ", MVR_MAX_TOP,
              ", and at most the number of classes, but is ", top);
  check_cuda(what, logits);
  check_tangent(what, logits);
  const bool graph = torch::autograd::compute_requires_grad(logits);
  LabelLogProbs r;
  at::Tensor y, lse;
  {
    at::NoGradGuard no_grad;
    c10::cuda::CUDAGuard guard(logits.device());
    ScoreLayout in;
    at::Tensor x = logits;
    if (!layout_of(x, in)) {
      x = x.contiguous();
      layout_of(x, in);
    }
    y = labels.contiguous();
    const at::TensorOptions f = logits.options().dtype(at::kFloat).requires_grad(false);
    r.log_prob = at::empty(labels.sizes(), f);
    r.entropy = at::empty(labels.sizes(), f);
    if (graph) lse = at::empty({2, labels.numel()}, f);
    if (top > 0) {
      r.top_value = scores_like(x, top, in, at::kFloat);
      r.top_label = scores_like(x, top, in, at::kInt);
    }
    const void *scores = data_or_null(x), *given = data_or_null(y);
    const int type = head_code(x.scalar_type()), label_type = mvr_host::label_type(y.scalar_type());
    float *log_prob = (float*)data_or_null(r.log_prob), *entropy = (float*)data_or_null(r.entropy),
          *top_value = (float*)data_or_null(r.top_value);
    int32_t* top_label = (int32_t*)data_or_null(r.top_label);
    float* lse0 = (float*)data_or_null(lse);
    check(graph ? mvr_label_log_probs_forward_rest(scores, type, given, label_type, log_prob, entropy, lse0,
                                                   lse0 ? lse0 + labels.numel() : nullptr, top_value, top_label, in.batch, K, in.space,
                                                   in.batch_stride, in.class_stride, (int)top, stream_of(x))
                : mvr_label_log_probs_forward(scores, type, given, label_type, log_prob, entropy, nullptr, top_value, top_label, in.batch, K,
                                              in.space, in.batch_stride, in.class_stride, (int)top, stream_of(x)));
  }
  if (graph) {
    auto node = std::shared_ptr<LabelLogProbsBackward>(new LabelLogProbsBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(logits));
    node->logits = SavedVariable(logits, false);
    node->labels = SavedVariable(y, false);
    node->lse = SavedVariable(lse, false);
    torch::autograd::set_history({r.log_prob, r.entropy}, node);
    node->entropy = SavedVariable(r.entropy, true);
  }
  return r;
}

// ---- Python ---------------------------------------------------------------------------------------------

// A whole number of 64 bits; negative ones stand for their two's complement.
uint64_t word_arg(PyObject* o, const char* name) {
  PyObject* index = PyNumber_Index(o);
  if (!index) throw python_error();
  int overflow = 0;
  const long long v = PyLong_AsLongLongAndOverflow(index, &overflow);
  uint64_t word = (uint64_t)v;
  if (overflow > 0) {
    word = PyLong_AsUnsignedLongLong(index);
    if (PyErr_Occurred()) overflow = -1;
  }
  Py_DECREF(index);
  if (overflow < 0) {
    PyErr_Clear();
    PyErr_Format(PyExc_ValueError, "%s must fit 64 bits", name);
    throw python_error();
  }
  if (PyErr_Occurred()) throw python_error();
  return word;
}

// cross_attention(query, key, value, batch_index, lengths, mask, scale)
PyObject* py_cross_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 7);
  const at::Tensor &q = tensor_arg(a[0], "query"), &k = tensor_arg(a[1], "key"), &v = tensor_arg(a[2], "value");
  Attention s;
  s.index = optional_tensor(a[3], "batch_index");
  s.lengths = optional_tensor(a[4], "lengths");
  s.mask = optional_tensor(a[5], "mask");
  s.scale = a[6] == Py_None ? 0.0 : number_arg(a[6]);
  at::Tensor out;
  {
    pybind11::gil_scoped_release nogil;
    out = attention(q, k, v, s, a[6] == Py_None);
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// window_attention(query, key, value, before, after, sinks, offsets, lengths, scale, rounded_weights)
PyObject* py_window_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 10);
  const at::Tensor &q = tensor_arg(a[0], "query"), &k = tensor_arg(a[1], "key"), &v = tensor_arg(a[2], "value");
  Attention s;
  s.in_window = true;
  s.window.before = whole_arg(a[3], "before");
  s.window.after = whole_arg(a[4], "after");
  s.window.sinks = whole_arg(a[5], "sinks");
  if (THPVariable_Check(a[6])) s.offsets = THPVariable_Unpack(a[6]);
  else if (a[6] != Py_None) s.window.offset = whole_arg(a[6], "offsets");
  s.lengths = optional_tensor(a[7], "lengths");
  s.scale = a[8] == Py_None ? 0.0 : number_arg(a[8]);
  const int rounded = PyObject_IsTrue(a[9]);
  if (rounded < 0) throw python_error();
  s.window.rounded_weights = rounded;
  at::Tensor out;
  {
    pybind11::gil_scoped_release nogil;
    out = attention(q, k, v, s, a[8] == Py_None);
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// dropout(x, p, seed, offset, residual)
PyObject* py_dropout(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 5);
  const at::Tensor& x = tensor_arg(a[0], "x");
  const double p = number_arg(a[1]);
  DropoutSeed seed;
  if (THPVariable_Check(a[2])) seed.tensor = THPVariable_Unpack(a[2]);
  else seed.value = word_arg(a[2], "seed");
  seed.offset = word_arg(a[3], "offset");
  const at::Tensor residual = optional_tensor(a[4], "residual");
  at::Tensor out;
  {
    pybind11::gil_scoped_release nogil;
    out = dropout(x, p, seed, residual);
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// label_log_probs(logits, labels, top) -> (log_prob, entropy, top_log_prob or None, top_label or None)
PyObject* py_label_log_probs(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 3);
  const at::Tensor &logits = tensor_arg(a[0], "logits"), &labels = tensor_arg(a[1], "labels");
  const long long top = PyLong_AsLongLong(a[2]);
  if (top == -1 && PyErr_Occurred()) throw python_error();
  LabelLogProbs r;
  {
    pybind11::gil_scoped_release nogil;
    r = label_log_probs(logits, labels, top);
  }
  PyObject* all = PyTuple_New(4);
  if (!all) throw python_error();
  const at::Tensor* parts[4] = {&r.log_prob, &r.entropy, &r.top_value, &r.top_label};
  for (int i = 0; i < 4; ++i) {
    if (parts[i]->defined()) {
      PyTuple_SET_ITEM(all, i, THPVariable_Wrap(*parts[i]));
    } else {
      Py_INCREF(Py_None);
      PyTuple_SET_ITEM(all, i, Py_None);
    }
  }
  return all;
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {{"cross_attention", FAST(py_cross_attention), nullptr},
                         {"window_attention", FAST(py_window_attention), nullptr},
                         {"dropout", FAST(py_dropout), nullptr},
                         {"label_log_probs", FAST(py_label_log_probs), nullptr},
                         {nullptr, nullptr, 0, nullptr}};

}  // namespace

namespace mvr_host {
PyMethodDef* head_methods() { return methods; }
}  // namespace mvr_host
