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
    stride = cols;
    if (x.is_contiguous()) {                         // no view for what is read through its pointer anyway
      t = x;
      return;
    }
    t = x.reshape({rows, cols});
    if (cols > 1 && t.stride(1) != 1) t = t.contiguous();
    if (rows > 1) stride = t.stride(0);
  }
  const void* ptr() const { return t.defined() ? t.data_ptr() : nullptr; }
};

void check_rc(int rc) { TORCH_CHECK(rc == 0, "libtdb_b200: ", tdb_last_error()); }

void refuse_second_derivative(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), "turbodeberta_b200: ", what, " has no second derivative (create_graph=True)");
}

// A tangent (torch.autograd.forward_ad) would be lost without a word: it is no reason for autograd to record a node.  Undefined tensors have none.
void refuse_tangents(const char* what, std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors)
    TORCH_CHECK(!t || !t->_fw_grad(0).defined(), "turbodeberta_b200: ", what, " has no forward-mode derivative");
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
  if (d.drop == 0) return x.clone(at::MemoryFormat::Contiguous);
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
    refuse_tangents("dropout", {&dy[0]});
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
  refuse_tangents("dropout", {&x});
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
    refuse_tangents("layer_norm", {&grads[0]});
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
  refuse_tangents("layer_norm", {&x, res ? &*res : nullptr, &w, &b});
  const auto d = dropout_of(p, seed, seed_value, offset);
  if (at::GradMode::is_enabled() && (x.requires_grad() || (res && res->requires_grad()) || w.requires_grad() || b.requires_grad()))
    return NormNode::apply(x, res, w, b, eps, p, seed, seed_value, offset);
  return run_norm(x, res, w, b, eps, d, false).first;
}

// ----------------------------------------------------------------------------------------------------- projections with adapters
// Where the product kernels of a device report, calls and recorded graphs alike: words that no call owns, since nothing but a wait that gave up is
// ever written there.  They are the host's and zero before the first launch, also where that is being captured.
std::atomic<int32_t*> g_standing[MAX_DEV];
int32_t* standing_words(int dev) { return g_standing[dev].load(); }
int32_t* make_standing_words(int dev) {
  TORCH_CHECK(dev >= 0 && dev < MAX_DEV, "turbodeberta_b200: up to ", MAX_DEV, " devices are supported");
  if (int32_t* w = standing_words(dev)) return w;
  static std::mutex mu;
  std::lock_guard<std::mutex> lock(mu);
  if (int32_t* w = standing_words(dev)) return w;
  int32_t* w = nullptr;
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;         // nothing that a capture of this thread would have to record
  cuda_ok(cudaThreadExchangeStreamCaptureMode(&mode), "capture mode");
  const cudaError_t e = cudaHostAlloc(reinterpret_cast<void**>(&w), SLOT_WORDS * sizeof(int32_t), cudaHostAllocMapped | cudaHostAllocPortable);
  cuda_ok(cudaThreadExchangeStreamCaptureMode(&mode), "capture mode");
  cuda_ok(e, "cudaHostAlloc(status words)");
  std::fill_n(w, SLOT_WORDS, 0);
  g_standing[dev] = w;
  return w;
}

// Behind a launch that reports there.  Each stream that used them since the last check is listed once; a captured launch need not be, since a check looks
// at the words in any case.
void list_standing(int dev, c10::cuda::CUDAStream stream) {
  if (at::cuda::currentStreamCaptureStatusMayInitCtx() != at::cuda::CaptureStatus::None) return;
  StatusPool& p = g_pools[dev];
  std::lock_guard<std::mutex> lock(p.mu);
  for (auto& t : p.pending)
    if (t.slot == STANDING && t.mark.stream() == stream.stream()) { t.mark.renew(); return; }
  p.pending.push_back({STANDING, Mark(stream), true});
}

struct LoraCall {
  Rows x, dy;
  bool tensor_cores;                                 // decided by types and sizes alone: forward and backward agree
  Tensor w, bias, a, b, scaling, ids;
  tdb::Lora l{};
  LoraCall(const Tensor& x_, const Tensor& w_, const OptTensor& bias_, const Tensor& a_, const Tensor& b_, const OptTensor& scaling_, double scaling_value, const OptTensor& ids_)
      : x(x_), w(rows_of_16_bytes(w_)), a(rows_of_16_bytes(a_)), b(rows_of_16_bytes(b_)) {
    l.rows = x.rows; l.cols = (int)x.cols;
    l.features = (int)w.size(0); l.rank = (int)a.size(1); l.n = (int)a.size(0); l.dtype = dtype_code(x_);
    tensor_cores = tdb_lora_umma_applies(&l);
    fit(x);
    l.x = x.ptr(); l.x_stride = x.stride;
    l.w = w.data_ptr(); l.a = a.data_ptr(); l.b = b.data_ptr();
    if (bias_) { bias = rows_of_16_bytes(*bias_); l.bias = bias.data_ptr(); }
    l.scaling_value = (float)scaling_value;
    if (scaling_) { scaling = scaling_->contiguous(); l.scaling = scaling.data_ptr<float>(); }
    l.rows_per_id = 1;
    if (ids_) {
      ids = ids_->contiguous();
      l.ids = ids.data_ptr(); l.id_bytes = (int)ids.element_size();
      if (ids.numel()) l.rows_per_id = l.rows / ids.numel();
    }
  }
  void set_dy(const Tensor& g) {
    dy = Rows(g);
    fit(dy);
    l.dy = dy.ptr();
    l.dy_stride = dy.stride;
  }
  // Rows that the tensor-core kernels can address.
  void fit(Rows& r) const {
    if (tensor_cores && r.rows && (misaligned(r.t) || r.stride % 8 || r.stride < r.cols)) {
      r.t = rows_of_16_bytes(r.t);
      r.stride = r.cols;
    }
  }
  Tensor floats(at::IntArrayRef sizes) const { return at::empty(sizes, w.options().dtype(at::kFloat)); }
  // The product alone, in fp32, under autocast too.
  Tensor product(const Tensor& rows, const Tensor& right) const {
    const c10::impl::ExcludeDispatchKeyGuard no_autocast(c10::autocast_dispatch_keyset);
    const Tensor left = rows.dim() == 2 ? rows : rows.reshape({l.rows, rows.size(-1)});
    return l.dtype == TDB_DTYPE_F32 ? at::mm(left, right) : at::mm(left, right, at::kFloat);
  }
};

// The inner values of the rows: bf16 [rows, inner] from the tensor cores, else fp32 [rows, rank].  f: the factors, for the former.
Tensor lora_shrink(const LoraCall& c, bool back, const Tensor& f, cudaStream_t stream) {
  Tensor h;
  if (c.tensor_cores) {
    h = at::empty({c.l.rows, tdb_lora_inner(&c.l)}, c.w.options());
    check_rc(tdb_lora_umma_shrink(&c.l, back, f.data_ptr(), h.data_ptr(), stream));
  } else {
    h = c.floats({c.l.rows, c.l.rank});
    check_rc(tdb_lora_shrink(&c.l, back, h.data_ptr<float>(), stream));
  }
  return h;
}
// y or dx, in `shape`, from the rows and their inner values.  Never a view: autograd would let nobody change a node's output in place.
Tensor lora_product(const LoraCall& c, bool back, const Tensor& f, const Tensor& h, at::IntArrayRef shape, c10::cuda::CUDAStream stream) {
  if (c.tensor_cores) {
    Tensor y = at::empty(shape, c.w.options());
    if (!back && tdb_lora_skinny_applies(&c.l)) {
      check_rc(tdb_lora_skinny(&c.l, h.data_ptr(), y.data_ptr(), stream.stream()));
      return y;
    }
    const int dev = c.w.get_device();
    check_rc(tdb_lora_umma_product(&c.l, back, f.data_ptr(), h.data_ptr(), y.data_ptr(), make_standing_words(dev), stream.stream()));
    list_standing(dev, stream);
    return y;
  }
  const Tensor base = back ? c.product(c.dy.t, c.w) : c.product(c.x.t, c.w.t());
  Tensor y = c.l.dtype == TDB_DTYPE_F32 ? at::_unsafe_view(base, shape) : at::empty(shape, c.w.options());
  check_rc(tdb_lora_expand(&c.l, back, base.data_ptr<float>(), h.data_ptr<float>(), y.data_ptr(), stream.stream()));
  return y;
}
// y; the rows' inner values, from which the gradient of b is made; and the rows' order by adapter, where the kernels go by it.
std::tuple<Tensor, Tensor, Tensor> run_lora(LoraCall& c, at::IntArrayRef shape, bool train) {
  const c10::cuda::CUDAStream stream = c10::cuda::getCurrentCUDAStream();
  if (c.l.rows == 0) return {at::empty(shape, c.w.options()), Tensor(), Tensor()};
  Tensor plan;
  const int64_t words = c.tensor_cores && !train ? 0 : tdb_lora_plan_words(&c.l, c.tensor_cores);
  if (words) {
    plan = at::empty({words}, c.w.options().dtype(at::kInt));
    check_rc(tdb_lora_plan(&c.l, plan.data_ptr<int32_t>(), stream.stream()));
    c.l.plan = plan.data_ptr<int32_t>();
  }
  const Tensor h = lora_shrink(c, false, c.a, stream);
  return {lora_product(c, false, c.b, h, shape, stream), h, plan};
}

// (gradient of a, gradient of b), where u and h are given.
std::pair<Tensor, Tensor> lora_gradients(const LoraCall& c, const Tensor& u, const Tensor& h, cudaStream_t stream) {
  const int factors = c.tensor_cores ? tdb_lora_umma_gather_factors(&c.l) : 16;
  tdb::LoraGradients g{};
  Tensor da, db, part;
  const int64_t of_a = (int64_t)c.l.n * c.l.rank * c.l.cols, of_b = (int64_t)c.l.n * c.l.rank * c.l.features;
  if (u.defined()) { g.u = u.data_ptr(); g.shares_a = tdb_lora_gather_shares(&c.l, 0, factors); da = at::empty(c.a.sizes(), c.a.options()); g.da = da.data_ptr(); }
  if (h.defined()) { g.h = h.data_ptr(); g.shares_b = tdb_lora_gather_shares(&c.l, 1, factors); db = at::empty(c.b.sizes(), c.b.options()); g.db = db.data_ptr(); }
  part = c.floats({g.shares_a * of_a + g.shares_b * of_b});
  if (u.defined()) g.part_a = part.data_ptr<float>();
  if (h.defined()) g.part_b = part.data_ptr<float>() + g.shares_a * of_a;
  check_rc(c.tensor_cores ? tdb_lora_umma_gather(&c.l, &g, stream) : tdb_lora_gather(&c.l, &g, stream));
  check_rc(tdb_lora_gather_sum(&c.l, &g, stream));
  return {da, db};
}

class LoraNode : public torch::autograd::Function<LoraNode> {
 public:
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& bias, const Tensor& a, const Tensor& b,
                        const OptTensor& scaling, double scaling_value, const OptTensor& ids, std::vector<int64_t> shape) {
    at::AutoDispatchBelowAutograd below;
    c10::cuda::CUDAGuard guard(x.device());
    LoraCall c(x, w, bias, a, b, scaling, scaling_value, ids);
    auto [y, h, plan] = run_lora(c, shape, a.requires_grad() || b.requires_grad());
    ctx->save_for_backward({x, w, a, b, scaling ? *scaling : Tensor(), ids ? *ids : Tensor(), b.requires_grad() ? h : Tensor(), plan});
    ctx->saved_data["scaling"] = scaling_value;
    ctx->saved_data["bias"] = bias.has_value();
    return y;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    refuse_second_derivative("lora_linear");
    refuse_tangents("lora_linear", {&grads[0]});
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &a = saved[2], &b = saved[3], &scaling = saved[4], &ids = saved[5], &h = saved[6], &plan = saved[7];
    const int at = ctx->saved_data["bias"].toBool() ? 3 : 2;
    const bool need_x = ctx->needs_input_grad(0), need_a = ctx->needs_input_grad(at), need_b = ctx->needs_input_grad(at + 1);
    c10::cuda::CUDAGuard guard(x.device());
    const c10::cuda::CUDAStream stream = c10::cuda::getCurrentCUDAStream();
    LoraCall c(x, w, std::nullopt, a, b, scaling.defined() ? OptTensor(scaling) : std::nullopt, ctx->saved_data["scaling"].toDouble(),
               ids.defined() ? OptTensor(ids) : std::nullopt);
    c.set_dy(grads[0]);
    if (plan.defined()) c.l.plan = plan.data_ptr<int32_t>();
    Tensor dx, da, db, u;
    if (c.l.rows == 0) {
      if (need_x) dx = at::empty(x.sizes(), x.options());
    } else if (need_x || need_a) {
      Tensor a_turned, b_turned;
      if (c.tensor_cores) {
        const int64_t of_a = need_x ? a.numel() : 0;
        const Tensor both = at::empty({of_a + b.numel()}, a.options());
        if (need_x) a_turned = both.narrow(0, 0, of_a);
        b_turned = both.narrow(0, of_a, b.numel());
        check_rc(tdb_lora_turn(&c.l, need_x ? a_turned.data_ptr() : nullptr, b_turned.data_ptr(), stream));
      }
      // the product may start beside the kernel in front of it, which therefore is the one that makes u
      u = lora_shrink(c, true, b_turned, stream);
      if (need_x) dx = lora_product(c, true, a_turned, u, x.sizes(), stream);
    }
    if (c.l.rows == 0) {
      if (need_a) da = at::zeros_like(a);
      if (need_b) db = at::zeros_like(b);
    } else if (need_a || need_b) {
      std::tie(da, db) = lora_gradients(c, need_a ? u : Tensor(), need_b ? h : Tensor(), stream);
    }
    const Tensor none;
    return {dx, none, none, da, db, none, none, none, none};
  }
};

Tensor lora_linear(const Tensor& x, const Tensor& w, const OptTensor& bias, const Tensor& a, const Tensor& b, const OptTensor& scaling, double scaling_value,
                   const OptTensor& ids) {
  dtype_code(x);
  if (x.dim() < 1 || w.dim() != 2 || x.size(-1) != w.size(1)) throw py::value_error("x [..., in] and weight [out, in] do not fit together");
  const int64_t K = w.size(1), N = w.size(0);
  if (K < 1 || N < 1) throw py::value_error("weight must not be empty");
  if (a.dim() != 3 || b.dim() != 3 || a.size(0) < 1 || a.size(1) < 1 || a.size(2) != K || b.size(0) != a.size(0) || b.size(1) != N || b.size(2) != a.size(1))
    throw py::value_error("lora_a must be [adapters, rank, in] and lora_b [adapters, out, rank]");
  if (a.size(1) > 256) throw py::value_error("rank " + std::to_string(a.size(1)) + ": up to 256 is supported");
  if (a.size(0) > 4095) throw py::value_error(std::to_string(a.size(0)) + " adapters: up to 4095 in one call are supported");
  int_size(K); int_size(N);
  if (bias && (bias->dim() != 1 || bias->size(0) != N)) throw py::value_error("bias must be a vector of the weight's rows");
  for (const Tensor* t : {&w, bias ? &*bias : &w, &a, &b})
    if (t->scalar_type() != x.scalar_type()) throw py::value_error("x, weight, bias, lora_a and lora_b must share a dtype");
  if (scaling && (scaling->scalar_type() != at::kFloat || scaling->dim() != 1 || scaling->size(0) != a.size(0)))
    throw py::value_error("scaling must be a number or a float32 vector with one entry per adapter");
  if (!ids && a.size(0) != 1) throw py::value_error("adapter_ids may be left out with a single adapter only");
  if (ids) {
    if (ids->scalar_type() != at::kInt && ids->scalar_type() != at::kLong) throw py::value_error("adapter_ids must be int32 or int64");
    const auto lead = x.sizes().slice(0, x.dim() - 1);
    const bool rows = ids->sizes() == lead, first = lead.size() > 1 && ids->dim() == 1 && ids->size(0) == lead[0];
    if (!rows && !first) throw py::value_error("adapter_ids must have the shape of x without its last dimension, or one entry for each entry of x's first");
  }
  device_of({&x, &w, bias ? &*bias : nullptr, &a, &b, scaling ? &*scaling : nullptr, ids ? &*ids : nullptr});
  refuse_tangents("lora_linear", {&x, &w, bias ? &*bias : nullptr, &a, &b, scaling ? &*scaling : nullptr});
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = N;
  if (at::GradMode::is_enabled()) {
    if (w.requires_grad() || (bias && bias->requires_grad()) || (scaling && scaling->requires_grad()))
      throw std::runtime_error("turbodeberta_b200: lora_linear trains the adapters and what is in front of them; weight, bias and scaling are frozen and must not require a gradient");
    if (x.requires_grad() || a.requires_grad() || b.requires_grad()) return LoraNode::apply(x, w, bias, a, b, scaling, scaling_value, ids, shape);
  }
  c10::cuda::CUDAGuard guard(x.device());
  LoraCall c(x, w, bias, a, b, scaling, scaling_value, ids);
  return std::get<0>(run_lora(c, shape, false));
}
