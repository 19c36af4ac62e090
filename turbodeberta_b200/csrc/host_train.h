// Host side of the training path's operators (part of host_ops.cpp): argument checks, outputs, launches and the autograd nodes.
// The nodes are native because a short text's kernels take a few microseconds each, and a node in Python ten times that.
#pragma once

// As the kernels take them: `rows` rows of contiguous elements.  A copy only where the last dimension is not contiguous or the
// leading ones do not collapse into one stride.
struct Rows {
  Tensor t;
  int64_t rows, cols, stride;
  Rows() : rows(0), cols(0), stride(0) {}
  explicit Rows(const Tensor& x) {
    cols = x.size(-1);
    rows = cols ? x.numel() / cols : 0;
    t = x.reshape({rows, cols});
    if (cols > 1 && t.stride(1) != 1) t = t.contiguous();
    stride = rows > 1 ? t.stride(0) : cols;
  }
  const void* ptr() const { return t.defined() ? t.data_ptr() : nullptr; }
};

void check_rc(int rc) { TORCH_CHECK(rc == 0, "libtdb_b200: ", tdb_last_error()); }

void refuse_second_derivative(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), "turbodeberta_b200: ", what, " has no second derivative (create_graph=True)");
}

void check_probability(double p) {
  if (!(p >= 0.0 && p <= 1.0)) throw py::value_error("dropout probability has to be between 0 and 1, but got " + std::to_string(p));
}
// The share of 65536 numbers that drop an element, and what the others are multiplied by.
tdb::Dropout dropout_of(double p, const OptTensor& seed, int64_t seed_value, int64_t offset) {
  tdb::Dropout d{};
  d.drop = (uint32_t)std::floor(p * 65536.0 + 0.5);
  d.scale = d.drop < 65536 ? (float)(65536.0 / (65536.0 - d.drop)) : 0.f;
  d.seed = seed ? seed->data_ptr<int64_t>() : nullptr;
  d.seed_value = seed_value;
  d.offset = offset;
  return d;
}
void check_seed(const OptTensor& seed, const Tensor& x) {
  if (!seed) return;
  if (seed->scalar_type() != at::kLong || seed->numel() != 1) throw py::value_error("seed must be an int or an int64 tensor of one element");
  device_of({&x, &*seed});
}

Tensor run_dropout(const Tensor& x, const tdb::Dropout& d) {
  c10::cuda::CUDAGuard guard(x.device());
  const Tensor in = x.contiguous();
  Tensor y = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
  check_rc(tdb_dropout(in.data_ptr(), y.data_ptr(), in.numel(), dtype_code(x), &d, c10::cuda::getCurrentCUDAStream().stream()));
  return y;
}

class DropoutNode : public torch::autograd::Function<DropoutNode> {
 public:
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const OptTensor& seed, int64_t seed_value, int64_t offset, double p) {
    at::AutoDispatchBelowAutograd below;
    ctx->save_for_backward({seed ? *seed : Tensor()});
    ctx->saved_data["value"] = seed_value;
    ctx->saved_data["offset"] = offset;
    ctx->saved_data["p"] = p;
    return run_dropout(x, dropout_of(p, seed, seed_value, offset));
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list dy) {
    refuse_second_derivative("dropout");
    const Tensor seed = ctx->get_saved_variables()[0];
    const auto d = dropout_of(ctx->saved_data["p"].toDouble(), seed.defined() ? OptTensor(seed) : std::nullopt, ctx->saved_data["value"].toInt(),
                              ctx->saved_data["offset"].toInt());
    return {run_dropout(dy[0], d), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor dropout(const Tensor& x, double p, const OptTensor& seed, int64_t seed_value, int64_t offset) {
  dtype_code(x);
  check_probability(p);
  check_seed(seed, x);
  device_of({&x});
  const auto d = dropout_of(p, seed, seed_value, offset);
  if (at::GradMode::is_enabled() && x.requires_grad()) return DropoutNode::apply(x, seed, seed_value, offset, p);
  return run_dropout(x, d);
}

// ---------------------------------------------------------------------------------------------------------------- LayerNorm
struct NormCall {
  Rows x, res, dy;
  Tensor w, b;
  tdb::Norm n{};
  NormCall(const Tensor& x_, const OptTensor& res_, const Tensor& w_, const OptTensor& b_, double eps, const tdb::Dropout& d)
      : x(x_), w(w_.contiguous()) {
    if (res_) res = Rows(*res_);
    if (b_) b = b_->contiguous();
    n.x = x.ptr(); n.x_stride = x.stride; n.rows = x.rows; n.cols = (int)x.cols;
    n.res = res.ptr(); n.res_stride = res.stride;
    n.w = w.data_ptr(); n.b = b.defined() ? b.data_ptr() : nullptr; n.w_dtype = dtype_code(w);
    n.eps = (float)eps; n.drop = d;
  }
};

std::pair<Tensor, Tensor> run_norm(const Tensor& x, const OptTensor& res, const Tensor& w, const Tensor& b, double eps, const tdb::Dropout& d, bool keep) {
  c10::cuda::CUDAGuard guard(x.device());
  NormCall c(x, res, w, b, eps, d);
  Tensor y = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous)), stats;
  c.n.y = y.data_ptr();
  if (keep) {
    stats = at::empty({c.n.rows, 2}, x.options().dtype(at::kFloat));
    c.n.stats = stats.data_ptr<float>();
  }
  check_rc(tdb_norm_forward(&c.n, dtype_code(x), c10::cuda::getCurrentCUDAStream().stream()));
  return {y, stats};
}

class NormNode : public torch::autograd::Function<NormNode> {
 public:
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const OptTensor& res, const Tensor& w, const Tensor& b, double eps,
                        double p, const OptTensor& seed, int64_t seed_value, int64_t offset) {
    at::AutoDispatchBelowAutograd below;
    auto [y, stats] = run_norm(x, res, w, b, eps, dropout_of(p, seed, seed_value, offset), true);
    ctx->save_for_backward({x, res ? *res : Tensor(), w, stats, seed ? *seed : Tensor()});
    ctx->saved_data["p"] = p;
    ctx->saved_data["value"] = seed_value;
    ctx->saved_data["offset"] = offset;
    return y;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    refuse_second_derivative("layer_norm");
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &res = saved[1], &w = saved[2], &stats = saved[3], &seed = saved[4];
    const bool need_x = ctx->needs_input_grad(0), need_res = res.defined() && ctx->needs_input_grad(1);
    const bool need_w = ctx->needs_input_grad(res.defined() ? 2 : 1), need_b = ctx->needs_input_grad(res.defined() ? 3 : 2);
    c10::cuda::CUDAGuard guard(x.device());
    const auto d = dropout_of(ctx->saved_data["p"].toDouble(), seed.defined() ? OptTensor(seed) : std::nullopt, ctx->saved_data["value"].toInt(),
                              ctx->saved_data["offset"].toInt());
    NormCall c(x, res.defined() ? OptTensor(res) : std::nullopt, w, std::nullopt, 0.0, d);
    c.dy = Rows(grads[0]);
    c.n.dy = c.dy.ptr();
    c.n.dy_stride = c.dy.stride;
    c.n.stats = stats.data_ptr<float>();
    const auto like = x.options().memory_format(at::MemoryFormat::Contiguous);
    Tensor dx, dres, dw, db, partial;
    if (!res.defined()) {
      if (need_x) dx = at::empty(x.sizes(), like);
    } else if (d.drop == 0) {                       // the sum's gradient is both summands': one tensor, as an addition gives it
      if (need_x || need_res) dx = dres = at::empty(x.sizes(), like);
    } else {
      if (need_x) dx = at::empty(x.sizes(), like);
      if (need_res) dres = at::empty(x.sizes(), like);
    }
    if (dx.defined()) c.n.dx = dx.data_ptr();
    if (dres.defined()) c.n.dres = dres.data_ptr();
    if (need_w || need_b) {
      if (c.n.rows == 0) {
        dw = at::zeros_like(w);
        db = at::zeros_like(w);
      } else {
        dw = at::empty(w.sizes(), w.options());
        db = at::empty(w.sizes(), w.options());
        partial = at::empty({tdb_norm_partial_floats(c.n.rows, c.n.cols)}, x.options().dtype(at::kFloat));
        c.n.partial = partial.data_ptr<float>();
      }
      c.n.dw = dw.data_ptr();
      c.n.db = db.data_ptr();
    }
    check_rc(tdb_norm_backward(&c.n, dtype_code(x), c10::cuda::getCurrentCUDAStream().stream()));
    const Tensor none;
    return {need_x ? dx : none, need_res ? dres : none, need_w ? dw : none, need_b ? db : none, none, none, none, none, none};
  }
};

// LayerNorm(x), or of dropout(x) + res.
Tensor norm(const Tensor& x, const OptTensor& res, const Tensor& w, const Tensor& b, double eps, double p, const OptTensor& seed, int64_t seed_value, int64_t offset) {
  const int code = dtype_code(x);
  if (x.dim() < 1) throw py::value_error("x must have at least one dimension");
  const int64_t cols = x.size(-1);
  if (cols < 1 || cols > 16384) throw py::value_error("the last dimension has to be between 1 and 16384, but is " + std::to_string(cols));
  for (const Tensor* t : {&w, &b})
    if (t->dim() != 1 || t->size(0) != cols) throw py::value_error("weight and bias must be vectors of the last dimension's size");
  if (w.scalar_type() != b.scalar_type() || (dtype_code(w) != code && dtype_code(w) != TDB_DTYPE_F32))
    throw py::value_error("weight and bias must share a dtype: that of x, or float32");
  if (res && (res->sizes() != x.sizes() || res->scalar_type() != x.scalar_type())) throw py::value_error("residual must have the shape and the dtype of x");
  if (!(eps >= 0.0) || !std::isfinite(eps)) throw py::value_error("eps has to be a finite number that is not negative");
  check_probability(p);
  check_seed(seed, x);
  device_of({&x, res ? &*res : nullptr, &w, &b});
  const auto d = dropout_of(p, seed, seed_value, offset);
  if (at::GradMode::is_enabled() && (x.requires_grad() || (res && res->requires_grad()) || w.requires_grad() || b.requires_grad()))
    return NormNode::apply(x, res, w, b, eps, p, seed, seed_value, offset);
  return run_norm(x, res, w, b, eps, d, false).first;
}
