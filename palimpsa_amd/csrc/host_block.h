// Native host path of the operators around the recurrences: norms, dropout, short convolution, selective scan, feed-forward block.  Part of
// host_ext.cpp, whose helpers it uses and whose rule it follows: a function serves the plain call (types that the kernels read, everything on
// the current device, no tracer or mode listening) and returns None for any other before it does anything; the Python route then
// converts, or raises the error that the call deserves.  It saves what that route takes in Python: 10 to 15 us of a forward, 50 of a
// forward and backward whose kernels take 30.
#pragma once

namespace block {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

bool rows_type(at::ScalarType t) { return t == at::kBFloat16 || t == at::kFloat; }
int32_t pal_type(at::ScalarType t) { return t == at::kBFloat16 ? PAL_DTYPE_BF16 : PAL_DTYPE_F32; }
at::TensorOptions as(const Tensor& t, at::ScalarType st) { return t.options().dtype(st).requires_grad(false); }

// on the device, of the type, a plain strided tensor (whatever its strides)
bool there(const Tensor& t, const c10::Device& dev, at::ScalarType st) {
  return t.defined() && t.device() == dev && t.scalar_type() == st && t.layout() == at::kStrided && !t.unsafeGetTensorImpl()->is_python_dispatch();
}
bool packed(const Tensor& t, const c10::Device& dev, at::ScalarType st) { return there(t, dev, st) && t.is_contiguous(); }
bool param_ok(const Tensor& t, const c10::Device& dev) { return t.defined() && rows_type(t.scalar_type()) && packed(t, dev, t.scalar_type()); }

// distances between batch rows and tokens of [B, T, inner ..] whose inner dims are packed; false: the tensor has to be copied
bool token_strides(const Tensor& t, int inner, int64_t& batch, int64_t& token) {
  int64_t row = 1;
  for (int64_t d = t.dim() - 1; d >= t.dim() - inner; --d) {
    if (t.size(d) != 1 && t.stride(d) != row) return false;
    row *= t.size(d);
  }
  token = t.size(1) > 1 ? t.stride(1) : row;
  batch = t.size(0) > 1 ? t.stride(0) : token * t.size(1);
  return token >= row && batch >= 0;
}

// A gradient that is differentiated again: the kernels have no such formula, and their results would pass for constants.
variable_list once(variable_list gr) {
  if (!at::GradMode::is_enabled()) return gr;
  auto refuse = std::make_shared<torch::autograd::DelayedError>("the gradients of this operator cannot be differentiated again", (int)gr.size());
  return (*refuse)(std::move(gr));
}

bool observed_or_dual(std::initializer_list<const Tensor*> ts) {
  if (!unobserved()) return true;
  for (const Tensor* t : ts)
    if (t->defined() && t->_fw_grad(/*level=*/0).defined()) return true;
  return false;
}
bool any_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
Tensor workspace(const Tensor& like, size_t bytes) { return at::empty({(int64_t)std::max<size_t>(bytes, 16)}, as(like, at::kByte)); }
py::object opt(const Tensor& t) { return t.defined() ? py::cast(t) : py::none(); }
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
// applies a node and carries a Python exception out of it
template <typename F>
py::object applied(F f) {
  try {
    return f();
  } catch (python_error& e) {
    e.restore();
    throw py::error_already_set();
  }
}

// ------------------------------------------------------------------------------------------------------ residual norm
// distance between the rows of [.., D] if there is one distance
bool row_stride(const Tensor& t, int64_t& stride) {
  const int64_t D = t.size(-1);
  if (t.stride(-1) != 1 && D != 1) return false;
  int64_t span = 0;
  stride = D;
  for (int64_t d = t.dim() - 2; d >= 0; --d) {
    if (t.size(d) == 1) continue;
    if (!span) {
      if (t.stride(d) < D) return false;
      stride = t.stride(d);
      span = stride * t.size(d);
    } else if (t.stride(d) == span) {
      span *= t.size(d);
    } else {
      return false;
    }
  }
  return true;
}

constexpr int64_t kMaxNormRow = 16384;

struct NormCall {
  bool ok = false;
  at::ScalarType rows, res;
  PalNormDims d{};
  NormCall(const Tensor& x, const Tensor& r, const Tensor& w, double eps, bool res_fp32, int64_t group) {
    if (!x.defined() || x.device().type() != at::kCUDA || x.device().index() != c10::hip::current_device() || x.dim() < 1 || x.numel() == 0) return;
    const c10::Device dev = x.device();
    rows = x.scalar_type();
    if (!rows_type(rows) || !there(x, dev, rows) || !param_ok(w, dev) || w.dim() != 1 || w.size(0) != x.size(-1)) return;
    res = res_fp32 || rows == at::kFloat || (r.defined() && r.scalar_type() != at::kBFloat16) ? at::kFloat : at::kBFloat16;
    if (r.defined() && (!there(r, dev, res) || r.sizes() != x.sizes())) return;
    if (!row_stride(x, d.x_stride)) return;
    d.res_stride = x.size(-1);
    if (r.defined() && !row_stride(r, d.res_stride)) return;
    if (x.size(-1) > kMaxNormRow || !(eps >= 0)) return;
    d.dim = (int32_t)x.size(-1);
    d.rows = x.numel() / d.dim;
    d.dtype = pal_type(rows); d.res_dtype = pal_type(res); d.weight_dtype = pal_type(w.scalar_type());
    d.group = (int32_t)group; d.eps = (float)eps;
    ok = true;
  }
  int run(const Tensor& x, const Tensor& r, const Tensor& w, Tensor& res_out, Tensor& y, Tensor& scales) const {
    PalNormTensors t{};
    t.x = ptr(x); t.residual = ptr(r); t.weight = ptr(w);
    t.residual_out = res_out.mutable_data_ptr(); t.y = y.mutable_data_ptr(); t.scales = fptr(scales);
    NoGil off;
    return abi.residual_norm_fwd(&d, &t, stream_of(x.device()));
  }
};

struct NormNode : torch::autograd::Function<NormNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptT& r_, const Tensor& w, double eps, bool res_fp32) {
    const Tensor r = r_.value_or(Tensor());
    NormCall c(x, r, w, eps, res_fp32, 0);
    Tensor y = at::empty(x.sizes(), as(x, c.rows)), s = at::empty(x.sizes(), as(x, c.res)), none;
    const int rc = c.run(x, r, w, s, y, none);
    if (rc) fail(rc, "pal_residual_norm_fwd");
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({s, w});
    ctx->saved_data["rows"] = (int64_t)c.rows;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["has_res"] = r.defined();
    return {y, s};
  }
  static variable_list backward(AutogradContext* ctx, variable_list gr) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &s = saved[0], &w = saved[1], none;
    if (!gr[0].defined() && !gr[1].defined()) return {none, none, none, none, none};
    const c10::DeviceGuard guard(s.device());
    const auto rows = (at::ScalarType)ctx->saved_data["rows"].toInt();
    const bool has_res = ctx->saved_data["has_res"].toBool();
    TORCH_CHECK_VALUE(s.dim() >= 1 && s.numel() > 0 && rows_type(s.scalar_type()) && packed(s, s.device(), s.scalar_type()) &&
                          param_ok(w, s.device()) && w.dim() == 1 && w.size(0) == s.size(-1) && (rows == at::kBFloat16 || s.scalar_type() == at::kFloat),
                      "residual_rms_norm backward: a saved tensor came back in another shape, dtype, layout or device");
    PalNormDims d{};
    d.dim = (int32_t)s.size(-1);
    d.rows = s.numel() / d.dim;
    d.x_stride = d.res_stride = d.dim;
    d.dtype = pal_type(rows); d.res_dtype = pal_type(s.scalar_type()); d.weight_dtype = pal_type(w.scalar_type());
    d.eps = (float)ctx->saved_data["eps"].toDouble();
    const Tensor dy = gr[0].defined() ? gr[0].to(rows).contiguous() : Tensor(), ds = gr[1].defined() ? gr[1].to(s.scalar_type()).contiguous() : Tensor();
    const bool two = rows != s.scalar_type();
    Tensor dx = at::empty(s.sizes(), as(s, rows)), dr = two ? at::empty(s.sizes(), as(s, s.scalar_type())) : dx;
    Tensor dw = at::empty(w.sizes(), as(s, at::kFloat));
    PalNormTensors t{};
    t.weight = ptr(w); t.residual_out = (void*)ptr(s);
    PalNormGrads g{};
    g.dy = ptr(dy); g.dresidual_out = ptr(ds); g.dx = dx.mutable_data_ptr(); g.dresidual = two ? dr.mutable_data_ptr() : nullptr; g.dweight = fptr(dw);
    const size_t bytes = abi.residual_norm_bwd_workspace_bytes(&d);
    Tensor ws = workspace(s, bytes);
    int rc;
    { NoGil off; rc = abi.residual_norm_bwd(&d, &t, &g, ws.mutable_data_ptr(), bytes, stream_of(s.device())); }
    if (rc) fail(rc, "pal_residual_norm_bwd");
    if (w.scalar_type() != at::kFloat) dw = dw.to(w.scalar_type());
    return once({dx, has_res ? dr : none, dw, none, none});
  }
};

// (y, residual stream), or None
py::object residual_norm(const Tensor& x, const OptT& r_, const Tensor& w, double eps, bool res_fp32) {
  const Tensor r = r_.value_or(Tensor());
  if (observed_or_dual({&x, &r, &w})) return py::none();
  const NormCall c(x, r, w, eps, res_fp32, 0);
  if (!c.ok) return py::none();
  if (any_grad({&x, &r, &w}))
    return applied([&] {
      auto o = NormNode::apply(x, r_, w, eps, res_fp32);
      return py::make_tuple(o[0], o[1]);
    });
  Tensor y = at::empty(x.sizes(), as(x, c.rows)), s = at::empty(x.sizes(), as(x, c.res)), none;
  if (c.run(x, r, w, s, y, none)) return py::none();   // nothing was launched: the Python route says what is wrong
  return py::make_tuple(y, s);
}
// (rows in 8 bits, scales, residual stream), or None; group 0: one scale a row
py::object residual_norm_fp8(const Tensor& x, const OptT& r_, const Tensor& w, double eps, bool res_fp32, int64_t group) {
  const Tensor r = r_.value_or(Tensor());
  if (observed_or_dual({&x, &r, &w}) || any_grad({&x, &r, &w}) || group < 0 || group > 256) return py::none();
  const NormCall c(x, r, w, eps, res_fp32, group);
  if (!c.ok || (group && x.size(-1) % group)) return py::none();
  auto shape = x.sizes().vec();
  Tensor q = at::empty(x.sizes(), as(x, at::kFloat8_e4m3fn)), s = at::empty(x.sizes(), as(x, c.res));
  shape.back() = group ? shape.back() / group : 1;
  Tensor scales = at::empty(shape, as(x, at::kFloat));
  if (c.run(x, r, w, s, q, scales)) return py::none();
  return py::make_tuple(q, scales, s);
}

// -------------------------------------------------------------------------------------------------- short convolution
struct ConvCall {
  bool ok = false;
  at::ScalarType rows;
  int64_t B, T, D, W, N;
  PalConvDims d{};
  ConvCall(const Tensor& x, const Tensor& w, const Tensor& b, bool silu, const Tensor& init, const Tensor& cu, const Tensor& table) {
    if (!x.defined() || x.device().type() != at::kCUDA || x.device().index() != c10::hip::current_device() || x.dim() != 3 || x.numel() == 0) return;
    const c10::Device dev = x.device();
    rows = x.scalar_type();
    if (!rows_type(rows) || !there(x, dev, rows) || !param_ok(w, dev)) return;
    B = x.size(0); T = x.size(1); D = x.size(2);
    if (!(w.dim() == 2 || (w.dim() == 3 && w.size(1) == 1)) || w.size(0) != D) return;
    W = w.size(-1);
    if (W < 2 || W > PAL_CONV_MAX_WIDTH || D > 1 << 20 || B * T > (int64_t)1 << 30) return;
    if (b.defined() && (!packed(b, dev, w.scalar_type()) || b.dim() != 1 || b.size(0) != D)) return;
    if (!token_strides(x, 1, d.x_batch_stride, d.x_token_stride)) return;
    N = B;
    if (cu.defined()) {
      if (B != 1 || !packed(cu, dev, at::kInt) || !packed(table, dev, at::kInt) || cu.dim() != 1 || cu.numel() < 2 || table.numel() % 4) return;
      N = cu.numel() - 1;
      if (N > INT32_MAX || table.numel() / 4 > INT32_MAX) return;
      d.flags |= PAL_FLAG_VARLEN;
      d.total_chunks = (int32_t)(table.numel() / 4);
    }
    if (init.defined()) {
      if (!packed(init, dev, rows) || init.dim() != 3 || init.size(0) != N || init.size(1) != D || init.size(2) != W) return;
      d.flags |= PAL_FLAG_HAS_INIT;
    }
    d.batch = (int32_t)B; d.seq_len = (int32_t)T; d.n_seqs = (int32_t)N; d.channels = (int32_t)D; d.width = (int32_t)W;
    d.dtype = pal_type(rows); d.weight_dtype = pal_type(w.scalar_type()); d.silu = silu;
    ok = true;
  }
  static void fill(PalConvTensors& t, const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& init, const Tensor& cu, const Tensor& table) {
    t.x = ptr(x); t.weight = ptr(w); t.bias = ptr(b); t.init = ptr(init);
    t.cu_seqlens = (const int32_t*)ptr(cu); t.chunk_table = (const int32_t*)ptr(table);
  }
  int run(const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& init, const Tensor& cu, const Tensor& table, Tensor& y, Tensor& fin) {
    PalConvTensors t{};
    fill(t, x, w, b, init, cu, table);
    t.y = y.mutable_data_ptr();
    if (fin.defined()) {
      t.final_ = fin.mutable_data_ptr();
      d.flags |= PAL_FLAG_STORE_FINAL;
    }
    NoGil off;
    return abi.short_conv_fwd(&d, &t, stream_of(x.device()));
  }
};

struct ConvNode : torch::autograd::Function<ConvNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptT& b_, bool silu, const OptT& init_, bool final_state,
                               const OptT& cu_, const OptT& table_) {
    const Tensor b = b_.value_or(Tensor()), init = init_.value_or(Tensor()), cu = cu_.value_or(Tensor()), table = table_.value_or(Tensor());
    ConvCall c(x, w, b, silu, init, cu, table);
    Tensor y = at::empty(x.sizes(), as(x, c.rows)), fin;
    if (final_state) fin = at::empty({c.N, c.D, c.W}, as(x, c.rows));
    const int rc = c.run(x, w, b, init, cu, table, y, fin);
    if (rc) fail(rc, "pal_short_conv_fwd");
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, w, b, init, cu, table});
    ctx->saved_data["silu"] = silu;
    ctx->saved_data["init_grad"] = init.defined() && init.requires_grad();
    variable_list o{y};
    if (final_state) o.push_back(fin);
    return o;
  }
  static variable_list backward(AutogradContext* ctx, variable_list gr) {
    const auto s = ctx->get_saved_variables();
    const Tensor &x = s[0], &w = s[1], &b = s[2], &init = s[3], &cu = s[4], &table = s[5], none;
    const c10::DeviceGuard guard(x.device());
    ConvCall c(x, w, b, ctx->saved_data["silu"].toBool(), init, cu, table);
    TORCH_CHECK_VALUE(c.ok, "short_conv backward: a saved tensor came back in another shape, dtype, layout or device");
    const Tensor dy = gr[0].defined() ? gr[0].to(c.rows).contiguous() : at::zeros(x.sizes(), as(x, c.rows));
    const Tensor df = gr.size() > 1 && gr[1].defined() ? gr[1].to(c.rows).contiguous() : Tensor();
    Tensor dx = at::empty(x.sizes(), as(x, c.rows)), dw = at::empty(w.sizes(), as(x, at::kFloat)), db, di;
    if (b.defined()) db = at::empty(b.sizes(), as(x, at::kFloat));
    if (ctx->saved_data["init_grad"].toBool()) di = at::empty(init.sizes(), as(x, c.rows));
    PalConvTensors t{};
    ConvCall::fill(t, x, w, b, init, cu, table);
    t.y = dx.mutable_data_ptr();   // not touched
    PalConvGrads g{};
    g.dy = ptr(dy); g.d_final = ptr(df); g.dx = dx.mutable_data_ptr(); g.dweight = fptr(dw); g.dbias = fptr(db);
    g.d_init = di.defined() ? di.mutable_data_ptr() : nullptr;
    const size_t bytes = abi.short_conv_bwd_workspace_bytes(&c.d);
    Tensor ws = workspace(x, bytes);
    int rc;
    { NoGil off; rc = abi.short_conv_bwd(&c.d, &t, &g, ws.mutable_data_ptr(), bytes, stream_of(x.device())); }
    if (rc) fail(rc, "pal_short_conv_bwd");
    if (w.scalar_type() != at::kFloat) {
      dw = dw.to(w.scalar_type());
      if (db.defined()) db = db.to(w.scalar_type());
    }
    return once({dx, dw, db, none, di, none, none, none});
  }
};

// (y, final state | None), or None
py::object short_conv(const Tensor& x, const Tensor& w, const OptT& b_, bool silu, const OptT& init_, bool final_state, const OptT& cu_, const OptT& table_) {
  const Tensor b = b_.value_or(Tensor()), init = init_.value_or(Tensor()), cu = cu_.value_or(Tensor()), table = table_.value_or(Tensor());
  if (observed_or_dual({&x, &w, &b, &init}) || cu.defined() != table.defined()) return py::none();
  ConvCall c(x, w, b, silu, init, cu, table);
  if (!c.ok) return py::none();
  if (any_grad({&x, &w, &b, &init}))
    return applied([&] {
      auto o = ConvNode::apply(x, w, b_, silu, init_, final_state, cu_, table_);
      return py::make_tuple(o[0], final_state ? py::cast(o[1]) : py::none());
    });
  Tensor y = at::empty(x.sizes(), as(x, c.rows)), fin;
  if (final_state) fin = at::empty({c.N, c.D, c.W}, as(x, c.rows));
  if (c.run(x, w, b, init, cu, table, y, fin)) return py::none();
  return py::make_tuple(y, opt(fin));
}
// y, the state written in place; or None
py::object short_conv_step(const Tensor& x, const Tensor& state, const Tensor& w, const OptT& b_, bool silu) {
  const Tensor b = b_.value_or(Tensor()), none;
  if (observed_or_dual({&x, &state, &w, &b}) || any_grad({&x, &state, &w, &b}) || !x.defined() || (x.dim() != 2 && x.dim() != 3)) return py::none();
  const Tensor x3 = x.dim() == 2 ? x.unsqueeze(1) : x;
  ConvCall c(x3, w, b, silu, none, none, none);
  if (!c.ok || !packed(state, x.device(), c.rows) || state.dim() != 3 || state.size(0) != c.B || state.size(1) != c.D || state.size(2) != c.W) return py::none();
  Tensor y = at::empty(x.sizes(), as(x, c.rows));
  PalConvTensors t{};
  ConvCall::fill(t, x3, w, b, none, none, none);
  t.y = y.mutable_data_ptr();
  t.final_ = state.mutable_data_ptr();
  int rc;
  { NoGil off; rc = abi.short_conv_step(&c.d, &t, stream_of(x.device())); }
  if (rc) return py::none();
  written(state);
  return py::cast(y);
}

// ----------------------------------------------------------------------------------------------------- selective scan
struct ScanIn {
  Tensor u, delta, A, B, C, D, z, bias, init, cu;
};
struct ScanCall {
  bool ok = false;
  at::ScalarType rows;
  int64_t bt, T, ch, N, G, seqs;
  PalScanDims d{};
  ScanCall(const ScanIn& i, bool softplus) {
    const Tensor& u = i.u;
    if (!u.defined() || u.device().type() != at::kCUDA || u.device().index() != c10::hip::current_device() || u.dim() != 3 || u.numel() == 0) return;
    const c10::Device dev = u.device();
    rows = u.scalar_type();
    if (!rows_type(rows) || !there(u, dev, rows) || !there(i.delta, dev, rows) || !there(i.B, dev, rows) || !there(i.C, dev, rows)) return;
    bt = u.size(0); T = u.size(1); ch = u.size(2);
    if (!packed(i.A, dev, at::kFloat) || i.A.dim() != 2 || i.A.size(0) != ch) return;
    N = i.A.size(1);
    if (i.delta.sizes() != u.sizes() || (i.z.defined() && (!there(i.z, dev, rows) || i.z.sizes() != u.sizes()))) return;
    if ((i.B.dim() != 3 && i.B.dim() != 4) || i.C.sizes() != i.B.sizes() || i.B.size(0) != bt || i.B.size(1) != T || i.B.size(-1) != N) return;
    G = i.B.dim() == 4 ? i.B.size(2) : 1;
    if (G < 1 || ch % G) return;
    for (const Tensor* t : {&i.D, &i.bias})
      if (t->defined() && (!packed(*t, dev, at::kFloat) || t->dim() != 1 || t->size(0) != ch)) return;
    const int inner = (int)i.B.dim() - 2;
    if (!token_strides(u, 1, d.u_batch, d.u_token) || !token_strides(i.delta, 1, d.delta_batch, d.delta_token) ||
        (i.z.defined() && !token_strides(i.z, 1, d.z_batch, d.z_token)) || !token_strides(i.B, inner, d.B_batch, d.B_token) ||
        !token_strides(i.C, inner, d.C_batch, d.C_token))
      return;
    for (int64_t s : {d.u_token, d.delta_token, d.z_token, d.B_token, d.C_token})
      if (s >= 1 << 24) return;
    seqs = bt;
    if (i.cu.defined()) {
      if (bt != 1 || !packed(i.cu, dev, at::kInt) || i.cu.dim() != 1 || i.cu.numel() < 2) return;
      seqs = i.cu.numel() - 1;
      d.flags |= PAL_FLAG_VARLEN;
    }
    if (i.init.defined()) {
      if (!packed(i.init, dev, at::kFloat) || i.init.dim() != 3 || i.init.size(0) != seqs || i.init.size(1) != ch || i.init.size(2) != N) return;
      d.flags |= PAL_FLAG_HAS_INIT;
    }
    if (bt > 65535 || bt * T > (int64_t)1 << 30 || ch >= 1 << 24 || seqs > INT32_MAX || N < 1 || N > PAL_SCAN_MAX_STATE) return;
    if ((uintptr_t)ptr(i.A) % 16 || (uintptr_t)ptr(i.init) % 16) return;
    d.batch = (int32_t)bt; d.seq_len = (int32_t)T; d.n_seqs = (int32_t)seqs; d.channels = (int32_t)ch; d.state = (int32_t)N; d.groups = (int32_t)G;
    d.dtype = pal_type(rows); d.softplus = softplus;
    ok = true;
  }
  static PalScanTensors fill(const ScanIn& i) {
    PalScanTensors t{};
    t.u = ptr(i.u); t.delta = ptr(i.delta); t.A = (const float*)ptr(i.A); t.B = ptr(i.B); t.C = ptr(i.C); t.D = (const float*)ptr(i.D); t.z = ptr(i.z);
    t.delta_bias = (const float*)ptr(i.bias); t.init = (const float*)ptr(i.init); t.cu_seqlens = (const int32_t*)ptr(i.cu);
    return t;
  }
  int run(const ScanIn& i, Tensor& y, float* fin, float* kept) {
    PalScanTensors t = fill(i);
    t.y = y.mutable_data_ptr();
    t.final_ = fin;
    t.checkpoints = kept;
    PalScanDims dd = d;
    if (fin) dd.flags |= PAL_FLAG_STORE_FINAL;
    const size_t bytes = abi.scan_fwd_workspace_bytes(&dd);
    Tensor ws;
    if (bytes) ws = workspace(i.u, bytes);
    NoGil off;
    return abi.scan_fwd(&dd, &t, bytes ? ws.mutable_data_ptr() : nullptr, bytes, stream_of(i.u.device()));
  }
};

struct ScanNode : torch::autograd::Function<ScanNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& u, const Tensor& delta, const Tensor& A, const Tensor& B, const Tensor& C, const OptT& D,
                               const OptT& z, const OptT& bias, const OptT& init, const OptT& cu, bool softplus, bool final_state) {
    const Tensor none;
    const ScanIn i{u, delta, A, B, C, D.value_or(none), z.value_or(none), bias.value_or(none), init.value_or(none), cu.value_or(none)};
    ScanCall c(i, softplus);
    Tensor y = at::empty(u.sizes(), as(u, c.rows)), fin;
    if (final_state) fin = at::empty({c.seqs, c.ch, c.N}, as(u, at::kFloat));
    Tensor kept = at::empty({(int64_t)std::max<size_t>(abi.scan_checkpoint_bytes(&c.d) / 4, 4)}, as(u, at::kFloat));
    const int rc = c.run(i, y, fptr(fin), fptr(kept));
    if (rc) fail(rc, "pal_scan_fwd");
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({u, delta, A, B, C, i.D, i.z, i.bias, i.init, i.cu, kept});
    ctx->saved_data["softplus"] = softplus;
    ctx->saved_data["init_grad"] = i.init.defined() && i.init.requires_grad();
    variable_list o{y};
    if (final_state) o.push_back(fin);
    return o;
  }
  static variable_list backward(AutogradContext* ctx, variable_list gr) {
    const auto s = ctx->get_saved_variables();
    const ScanIn i{s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], s[8], s[9]};
    const Tensor& kept = s[10];
    const Tensor none;
    const c10::DeviceGuard guard(i.u.device());
    ScanCall c(i, ctx->saved_data["softplus"].toBool());
    TORCH_CHECK_VALUE(c.ok && packed(kept, i.u.device(), at::kFloat) && kept.numel() == (int64_t)std::max<size_t>(abi.scan_checkpoint_bytes(&c.d) / 4, 4),
                      "selective_scan backward: a saved tensor came back in another shape, dtype, layout or device");
    const Tensor dy = gr[0].defined() ? gr[0].to(c.rows).contiguous() : at::zeros(i.u.sizes(), as(i.u, c.rows));
    Tensor df = gr.size() > 1 && gr[1].defined() ? gr[1].to(at::kFloat).contiguous() : Tensor();
    if (df.defined() && (uintptr_t)ptr(df) % 16) df = df.clone();
    auto like = [&](const Tensor& t) { return t.defined() ? at::empty(t.sizes(), as(t, t.scalar_type())) : Tensor(); };
    Tensor du = like(i.u), dd = like(i.delta), dA = like(i.A), dB = like(i.B), dC = like(i.C), dD = like(i.D), dz = like(i.z), db = like(i.bias), di;
    if (ctx->saved_data["init_grad"].toBool()) di = like(i.init);
    PalScanTensors t = ScanCall::fill(i);
    t.checkpoints = (float*)ptr(kept);
    PalScanGrads g{};
    auto out = [](Tensor& x) { return x.defined() ? x.mutable_data_ptr() : nullptr; };
    g.dy = ptr(dy); g.d_final = (const float*)ptr(df); g.du = out(du); g.ddelta = out(dd); g.dA = fptr(dA); g.dB = out(dB); g.dC = out(dC); g.dD = fptr(dD);
    g.dz = out(dz); g.ddelta_bias = fptr(db); g.d_init = fptr(di);
    const size_t bytes = abi.scan_bwd_workspace_bytes(&c.d);
    Tensor ws = workspace(i.u, bytes);
    int rc;
    { NoGil off; rc = abi.scan_bwd(&c.d, &t, &g, ws.mutable_data_ptr(), bytes, stream_of(i.u.device())); }
    if (rc) fail(rc, "pal_scan_bwd");
    return once({du, dd, dA, dB, dC, dD, dz, db, di, none, none, none});
  }
};

// (y, final state | None), or None; B, C [B, T, N] or [B, T, G, N]
py::object selective_scan(const Tensor& u, const Tensor& delta, const Tensor& A, const Tensor& B, const Tensor& C, const OptT& D, const OptT& z,
                          const OptT& bias, bool softplus, const OptT& init, bool final_state, const OptT& cu) {
  const Tensor none;
  const ScanIn i{u, delta, A, B, C, D.value_or(none), z.value_or(none), bias.value_or(none), init.value_or(none), cu.value_or(none)};
  if (observed_or_dual({&u, &delta, &A, &B, &C, &i.D, &i.z, &i.bias, &i.init})) return py::none();
  ScanCall c(i, softplus);
  if (!c.ok) return py::none();
  if (any_grad({&u, &delta, &A, &B, &C, &i.D, &i.z, &i.bias, &i.init}))
    return applied([&] {
      auto o = ScanNode::apply(u, delta, A, B, C, D, z, bias, init, cu, softplus, final_state);
      return py::make_tuple(o[0], final_state ? py::cast(o[1]) : py::none());
    });
  Tensor y = at::empty(u.sizes(), as(u, c.rows)), fin;
  if (final_state) fin = at::empty({c.seqs, c.ch, c.N}, as(u, at::kFloat));
  if (c.run(i, y, fptr(fin), nullptr)) return py::none();
  return py::make_tuple(y, opt(fin));
}
// y, the state written in place; or None.  u [B, D] with B, C [B, N] or [B, G, N], or all with a dim of tokens behind the first
py::object selective_scan_step(const Tensor& u, const Tensor& state, const Tensor& delta, const Tensor& A, const Tensor& B, const Tensor& C, const OptT& D,
                               const OptT& z, const OptT& bias, bool softplus) {
  const Tensor none;
  if (!u.defined() || (u.dim() != 2 && u.dim() != 3)) return py::none();
  const bool one = u.dim() == 2;
  auto up = [&](const Tensor& t) { return one && t.defined() && t.dim() >= 2 ? t.unsqueeze(1) : t; };
  const ScanIn i{up(u), up(delta), A, up(B), up(C), D.value_or(none), up(z.value_or(none)), bias.value_or(none), state, none};
  if (observed_or_dual({&u, &state, &delta, &A, &B, &C, &i.D, &i.z, &i.bias}) || any_grad({&u, &state, &delta, &A, &B, &C, &i.D, &i.z, &i.bias})) return py::none();
  ScanCall c(i, softplus);
  if (!c.ok) return py::none();
  Tensor y = at::empty(u.sizes(), as(u, c.rows));
  if (c.run(i, y, (float*)state.mutable_data_ptr(), nullptr)) return py::none();
  written(state);
  return py::cast(y);
}

// ------------------------------------------------------------------------------------------- dropout and layer norm
// a seed on the device: one int64 number
bool seed_ok(const Tensor& t, const c10::Device& dev) { return !t.defined() || (there(t, dev, at::kLong) && t.numel() == 1); }
PalDropout drop_of(double p, int64_t seed, const Tensor& seed_t, int64_t site) {
  return PalDropout{p, seed, (const int64_t*)ptr(seed_t), (uint32_t)site};
}

bool dropout_plain(const Tensor& x, const Tensor& seed_t, int64_t& stride) {
  if (!x.defined() || x.device().type() != at::kCUDA || x.device().index() != c10::hip::current_device() || x.dim() < 1 || x.numel() == 0) return false;
  return rows_type(x.scalar_type()) && there(x, x.device(), x.scalar_type()) && seed_ok(seed_t, x.device()) && row_stride(x, stride) && x.size(-1) <= 1 << 30;
}
int dropout_run(const Tensor& x, int64_t stride, double p, int64_t seed, const Tensor& seed_t, int64_t site, Tensor& y) {
  const PalDropout d = drop_of(p, seed, seed_t, site);
  const int64_t D = x.size(-1), rows = x.numel() / D;
  void* out = y.mutable_data_ptr();
  NoGil off;
  return abi.dropout(&d, ptr(x), out, rows, D, stride, pal_type(x.scalar_type()), stream_of(x.device()));
}
struct DropoutNode : torch::autograd::Function<DropoutNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, double p, int64_t seed, const OptT& seed_, int64_t site) {
    const Tensor seed_t = seed_.value_or(Tensor());
    int64_t stride;
    dropout_plain(x, seed_t, stride);
    Tensor y = at::empty(x.sizes(), as(x, x.scalar_type()));
    const int rc = dropout_run(x, stride, p, seed, seed_t, site, y);
    if (rc) fail(rc, "pal_dropout");
    ctx->save_for_backward({seed_t});
    ctx->saved_data["p"] = p;
    ctx->saved_data["seed"] = seed;
    ctx->saved_data["site"] = site;
    ctx->saved_data["type"] = (int64_t)x.scalar_type();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list gr) {
    const Tensor seed_t = ctx->get_saved_variables()[0], none;
    const c10::DeviceGuard guard(gr[0].device());
    const auto type = (at::ScalarType)ctx->saved_data["type"].toInt();
    Tensor dy = gr[0].to(type);
    int64_t stride;
    if (!dropout_plain(dy, seed_t, stride)) dy = dy.contiguous();
    TORCH_CHECK_VALUE(dropout_plain(dy, seed_t, stride), "dropout backward: the seed came back in another shape, dtype or device");
    Tensor dx = at::empty(dy.sizes(), as(dy, type));
    const int rc = dropout_run(dy, stride, ctx->saved_data["p"].toDouble(), ctx->saved_data["seed"].toInt(), seed_t, ctx->saved_data["site"].toInt(), dx);
    if (rc) fail(rc, "pal_dropout");
    return once({dx, none, none, none, none});
  }
};
// y, or None
py::object dropout(const Tensor& x, double p, int64_t seed, const OptT& seed_, int64_t site) {
  const Tensor seed_t = seed_.value_or(Tensor());
  if (observed_or_dual({&x})) return py::none();
  int64_t stride;
  if (!dropout_plain(x, seed_t, stride)) return py::none();
  if (any_grad({&x})) return applied([&] { return py::cast(DropoutNode::apply(x, p, seed, seed_, site)); });
  Tensor y = at::empty(x.sizes(), as(x, x.scalar_type()));
  if (dropout_run(x, stride, p, seed, seed_t, site, y)) return py::none();
  return py::cast(y);
}

struct LayerNormCall {
  bool ok = false;
  at::ScalarType rows, res;
  PalLayerNormDims d{};
  LayerNormCall(const Tensor& x, const Tensor& r, const Tensor& w, const Tensor& b, double eps, bool res_fp32, bool handed_on) {
    if (!x.defined() || x.device().type() != at::kCUDA || x.device().index() != c10::hip::current_device() || x.dim() < 1 || x.numel() == 0) return;
    const c10::Device dev = x.device();
    rows = x.scalar_type();
    if (!rows_type(rows) || !there(x, dev, rows) || !param_ok(w, dev) || w.dim() != 1 || w.size(0) != x.size(-1)) return;
    if (b.defined() && (!packed(b, dev, w.scalar_type()) || b.sizes() != w.sizes())) return;
    res = !handed_on ? rows : res_fp32 || rows == at::kFloat || (r.defined() && r.scalar_type() != at::kBFloat16) ? at::kFloat : at::kBFloat16;
    if (r.defined() && (!there(r, dev, res) || r.sizes() != x.sizes())) return;
    if (!row_stride(x, d.x_stride)) return;
    d.res_stride = x.size(-1);
    if (r.defined() && !row_stride(r, d.res_stride)) return;
    if (x.size(-1) > kMaxNormRow || !(eps >= 0)) return;
    d.dim = (int32_t)x.size(-1);
    d.rows = x.numel() / d.dim;
    d.dtype = pal_type(rows); d.res_dtype = pal_type(res); d.weight_dtype = pal_type(w.scalar_type());
    d.eps = (float)eps;
    ok = true;
  }
  int run(const Tensor& x, const Tensor& r, const Tensor& w, const Tensor& b, Tensor& s, Tensor& y, Tensor& stats) const {
    PalLayerNormTensors t{};
    t.x = ptr(x); t.residual = ptr(r); t.weight = ptr(w); t.bias = ptr(b);
    t.residual_out = s.defined() ? s.mutable_data_ptr() : nullptr; t.y = y.mutable_data_ptr(); t.stats = fptr(stats);
    NoGil off;
    return abi.layer_norm_fwd(&d, &t, stream_of(x.device()));
  }
};

struct LayerNormNode : torch::autograd::Function<LayerNormNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptT& r_, const Tensor& w, const OptT& b_, double eps, bool res_fp32, bool handed_on,
                               double p, int64_t seed, const OptT& seed_, int64_t site) {
    const Tensor r = r_.value_or(Tensor()), b = b_.value_or(Tensor()), seed_t = seed_.value_or(Tensor());
    LayerNormCall c(x, r, w, b, eps, res_fp32, handed_on);
    c.d.drop = drop_of(p, seed, seed_t, site);
    Tensor y = at::empty(x.sizes(), as(x, c.rows)), s, stats = at::empty({c.d.rows, 2}, as(x, at::kFloat));
    if (handed_on) s = at::empty(x.sizes(), as(x, c.res));
    const int rc = c.run(x, r, w, b, s, y, stats);
    if (rc) fail(rc, "pal_layer_norm_fwd");
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({handed_on ? s : x, w, stats, seed_t});
    ctx->saved_data["rows"] = (int64_t)c.rows;
    ctx->saved_data["handed_on"] = handed_on;
    ctx->saved_data["has_res"] = r.defined();
    ctx->saved_data["has_bias"] = b.defined();
    ctx->saved_data["p"] = p;
    ctx->saved_data["seed"] = seed;
    ctx->saved_data["site"] = site;
    variable_list o{y};
    if (handed_on) o.push_back(s);
    return o;
  }
  static variable_list backward(AutogradContext* ctx, variable_list gr) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &s = saved[0], &w = saved[1], &stats = saved[2], &seed_t = saved[3], none;
    if (!gr[0].defined() && (gr.size() < 2 || !gr[1].defined())) return variable_list(11);
    const c10::DeviceGuard guard(s.device());
    const auto rows = (at::ScalarType)ctx->saved_data["rows"].toInt();
    const bool handed_on = ctx->saved_data["handed_on"].toBool(), has_res = ctx->saved_data["has_res"].toBool(), has_bias = ctx->saved_data["has_bias"].toBool();
    const double p = ctx->saved_data["p"].toDouble();
    PalLayerNormDims d{};
    TORCH_CHECK_VALUE(s.dim() >= 1 && s.numel() > 0 && rows_type(s.scalar_type()) && there(s, s.device(), s.scalar_type()) && row_stride(s, d.x_stride) &&
                          (!handed_on || s.is_contiguous()) && (handed_on || s.scalar_type() == rows) && param_ok(w, s.device()) && w.dim() == 1 &&
                          w.size(0) == s.size(-1) && (rows == at::kBFloat16 || s.scalar_type() == at::kFloat) && packed(stats, s.device(), at::kFloat) &&
                          stats.numel() == 2 * (s.numel() / s.size(-1)) && seed_ok(seed_t, s.device()) && (!gr[0].defined() || gr[0].sizes() == s.sizes()) &&
                          (gr.size() < 2 || !gr[1].defined() || gr[1].sizes() == s.sizes()),
                      "layer_norm backward: a saved tensor came back in another shape, dtype, layout or device");
    d.dim = (int32_t)s.size(-1);
    d.rows = s.numel() / d.dim;
    d.res_stride = d.dim;
    d.dtype = pal_type(rows); d.res_dtype = pal_type(s.scalar_type()); d.weight_dtype = pal_type(w.scalar_type());
    d.drop = drop_of(p, ctx->saved_data["seed"].toInt(), seed_t, ctx->saved_data["site"].toInt());
    const Tensor dy = gr[0].defined() ? gr[0].to(rows).contiguous() : Tensor();
    const Tensor dr = gr.size() > 1 && gr[1].defined() ? gr[1].to(s.scalar_type()).contiguous() : Tensor();
    const bool apart = has_res && (p > 0.0 || rows != s.scalar_type());
    Tensor dx = at::empty(s.sizes(), as(s, rows)), ds, dw = at::empty(w.sizes(), as(s, at::kFloat)), db;
    if (apart) ds = at::empty(s.sizes(), as(s, s.scalar_type()));
    if (has_bias) db = at::empty(w.sizes(), as(s, at::kFloat));
    PalLayerNormTensors t{};
    t.weight = ptr(w); t.bias = has_bias ? ptr(w) : nullptr; t.stats = (float*)ptr(stats);
    if (handed_on) t.residual_out = (void*)ptr(s);
    else t.x = ptr(s);
    PalLayerNormGrads g{};
    g.dy = ptr(dy); g.dresidual_out = ptr(dr); g.dx = dx.mutable_data_ptr(); g.dresidual = ds.defined() ? ds.mutable_data_ptr() : nullptr;
    g.dweight = fptr(dw); g.dbias = fptr(db);
    const size_t bytes = abi.layer_norm_bwd_workspace_bytes(&d);
    Tensor ws = workspace(s, bytes);
    int rc;
    { NoGil off; rc = abi.layer_norm_bwd(&d, &t, &g, ws.mutable_data_ptr(), bytes, stream_of(s.device())); }
    if (rc) fail(rc, "pal_layer_norm_bwd");
    if (w.scalar_type() != at::kFloat) {
      dw = dw.to(w.scalar_type());
      if (db.defined()) db = db.to(w.scalar_type());
    }
    return once({dx, has_res ? (apart ? ds : dx) : none, dw, db, none, none, none, none, none, none, none});
  }
};

// (y,) or (y, residual stream), or None
py::object layer_norm(const Tensor& x, const OptT& r_, const Tensor& w, const OptT& b_, double eps, bool res_fp32, bool handed_on, double p, int64_t seed,
                      const OptT& seed_, int64_t site) {
  const Tensor r = r_.value_or(Tensor()), b = b_.value_or(Tensor()), seed_t = seed_.value_or(Tensor());
  if (observed_or_dual({&x, &r, &w, &b})) return py::none();
  LayerNormCall c(x, r, w, b, eps, res_fp32, handed_on);
  if (!c.ok || !seed_ok(seed_t, x.device())) return py::none();
  if (any_grad({&x, &r, &w, &b}))
    return applied([&] {
      auto o = LayerNormNode::apply(x, r_, w, b_, eps, res_fp32, handed_on, p, seed, seed_, site);
      return handed_on ? py::make_tuple(o[0], o[1]) : py::make_tuple(o[0]);
    });
  c.d.drop = drop_of(p, seed, seed_t, site);
  Tensor y = at::empty(x.sizes(), as(x, c.rows)), s, none;
  if (handed_on) s = at::empty(x.sizes(), as(x, c.res));
  if (c.run(x, r, w, b, s, y, none)) return py::none();   // nothing was launched: the Python route says what is wrong
  return handed_on ? py::make_tuple(y, s) : py::make_tuple(y);
}

// --------------------------------------------------------------------------------------------- gated feed-forward block
// Matrices that the kernels cannot read or write where they lie (dims that are no multiple of eight, addresses or strides off 16 bytes): copies of
// them in one buffer, made by one launch, and results taken out of it by another.
struct MlpCopies {
  PalMatrixCopy in[5], out[5];
  int n_in = 0, n_out = 0;
  size_t bytes = 0;
  const size_t es;
  Tensor buffer;
  explicit MlpCopies(size_t es) : es(es) {}
  static int64_t up8(int64_t n) { return (n + 7) / 8 * 8; }
  // (places are offsets until the buffer is there)
  void add(bool result, const void* p, int64_t ld, int64_t rows, int64_t cols, bool pad_rows) {
    const int64_t r8 = pad_rows ? up8(rows) : rows, c8 = up8(cols);
    if (result) out[n_out++] = PalMatrixCopy{(const void*)bytes, (void*)p, c8, ld, rows, cols, rows, cols};
    else in[n_in++] = PalMatrixCopy{p, (void*)bytes, ld, c8, rows, cols, r8, c8};
    bytes += ((size_t)(r8 * c8) * es + 255) & ~(size_t)255;
  }
  int make(const Tensor& like, int32_t dtype) {
    if (!bytes) return 0;
    buffer = workspace(like, bytes);
    char* base = (char*)buffer.mutable_data_ptr();
    for (int i = 0; i < n_in; ++i) in[i].dst = base + (size_t)in[i].dst;
    for (int i = 0; i < n_out; ++i) out[i].src = base + (size_t)out[i].src;
    return n_in ? abi.copy_matrices(in, n_in, dtype, stream_of(like.device())) : 0;
  }
  int take(const Tensor& like, int32_t dtype) { return n_out ? abi.copy_matrices(out, n_out, dtype, stream_of(like.device())) : 0; }
};

struct MlpCall {
  bool ok = false;
  at::ScalarType type;
  PalMlpDims d{};                    // multiples of eight
  int64_t D, F, Do, x_ld;            // as they are
  bool copied[4];                    // x, w_gate, w_up, w_down
  MlpCall(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, int64_t act) {
    if (!x.defined() || x.device().type() != at::kCUDA || x.device().index() != c10::hip::current_device() || x.dim() < 1 || x.numel() == 0) return;
    const c10::Device dev = x.device();
    type = x.scalar_type();
    if (!rows_type(type) || !there(x, dev, type)) return;
    for (const Tensor* w : {&wg, &wu, &wd})
      if (!packed(*w, dev, type) || w->dim() != 2) return;
    D = x.size(-1);
    F = wg.size(0);
    Do = wd.size(0);
    const int64_t rows = x.numel() / D;
    if (wg.size(1) != D || wu.sizes() != wg.sizes() || wd.size(1) != F) return;
    if (!F || !Do || D > 1 << 20 || F > 1 << 20 || Do > 1 << 20 || rows > 1 << 30) return;
    if (!row_stride(x, x_ld)) return;
    const Tensor* t[] = {&x, &wg, &wu, &wd};
    for (int i = 0; i < 4; ++i) copied[i] = (uintptr_t)ptr(*t[i]) % 16 || (i == 0 ? D % 8 || x_ld % 8 || x_ld > 1 << 20 : odd(i));
    d.rows = rows;
    d.x_stride = copied[0] ? MlpCopies::up8(D) : x_ld;
    d.dim = (int32_t)MlpCopies::up8(D); d.hidden = (int32_t)MlpCopies::up8(F); d.out_dim = (int32_t)MlpCopies::up8(Do);
    d.dtype = pal_type(type); d.activation = (int32_t)act;
    d.hidden_pad = d.hidden - (int32_t)F;
    ok = true;
  }
  // rows and columns of x (0), of the weights
  int64_t high(int i) const { return i == 0 ? d.rows : i < 3 ? F : Do; }
  int64_t wide(int i) const { return i == 0 || i < 3 ? D : F; }
  bool odd(int i) const { return wide(i) % 8 || (i && high(i) % 8); }
  size_t es() const { return type == at::kFloat ? 4 : 2; }
  Tensor out(const Tensor& x) const {
    auto shape = x.sizes().vec();
    shape.back() = Do;
    return at::empty(shape, as(x, type));
  }
  // operands, copied if need be; their copies are the first ones
  void operands(MlpCopies& c, const Tensor* const* t) const {
    for (int i = 0; i < 4; ++i)
      if (copied[i]) c.add(false, ptr(*t[i]), i == 0 ? x_ld : wide(i), high(i), wide(i), i != 0);
  }
  PalMlpTensors fill(const MlpCopies& c, const Tensor* const* t) const {
    const void* p[4];
    for (int i = 0, n = 0; i < 4; ++i) p[i] = copied[i] ? c.in[n++].dst : ptr(*t[i]);
    PalMlpTensors r{};
    r.x = p[0]; r.w_gate = p[1]; r.w_up = p[2]; r.w_down = p[3];
    return r;
  }
  int run(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, Tensor& y, Tensor& kept) const {
    const Tensor* t[] = {&x, &wg, &wu, &wd};
    MlpCopies c(es());
    operands(c, t);
    if (Do % 8) c.add(true, y.mutable_data_ptr(), Do, d.rows, Do, false);
    if (int rc = c.make(x, d.dtype)) return rc;
    PalMlpTensors r = fill(c, t);
    r.y = Do % 8 ? (void*)c.out[0].src : y.mutable_data_ptr();
    r.kept = kept.defined() ? kept.mutable_data_ptr() : nullptr;
    const size_t bytes = abi.gated_mlp_fwd_workspace_bytes(&d, kept.defined());
    Tensor ws = workspace(x, bytes);
    NoGil off;
    const int rc = abi.gated_mlp_fwd(&d, &r, ws.mutable_data_ptr(), bytes, stream_of(x.device()));
    return rc ? rc : c.take(x, d.dtype);
  }
};

struct MlpNode : torch::autograd::Function<MlpNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, int64_t act) {
    MlpCall c(x, wg, wu, wd, act);
    Tensor y = c.out(x), kept = workspace(x, abi.gated_mlp_kept_bytes(&c.d));
    const int rc = c.run(x, wg, wu, wd, y, kept);
    if (rc) fail(rc, "pal_gated_mlp_fwd");
    ctx->save_for_backward({x, wg, wu, wd, kept});
    ctx->saved_data["act"] = act;
    for (int i = 0; i < 4; ++i) {
      const Tensor* t[] = {&x, &wg, &wu, &wd};
      ctx->saved_data[std::string("need") + (char)('0' + i)] = t[i]->requires_grad();
    }
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list gr) {
    const auto s = ctx->get_saved_variables();
    const Tensor &x = s[0], &kept = s[4], none;
    const c10::DeviceGuard guard(x.device());
    MlpCall c(x, s[1], s[2], s[3], ctx->saved_data["act"].toInt());
    // (dy has the shape of y, whatever came back)
    TORCH_CHECK_VALUE(c.ok && packed(kept, x.device(), at::kByte) && kept.numel() == (int64_t)abi.gated_mlp_kept_bytes(&c.d) &&
                          gr[0].sizes().slice(0, gr[0].dim() - 1) == x.sizes().slice(0, x.dim() - 1) && gr[0].size(-1) == c.Do,
                      "gated_mlp backward: a saved tensor came back in another shape, dtype, layout or device");
    const Tensor dy = gr[0].to(c.type).contiguous();
    const Tensor* t[] = {&x, &s[1], &s[2], &s[3]};
    MlpCopies m(c.es());
    c.operands(m, t);
    const bool dy_copied = c.Do % 8 || (uintptr_t)ptr(dy) % 16;
    if (dy_copied) m.add(false, ptr(dy), c.Do, c.d.rows, c.Do, false);
    Tensor out[4];
    void* to[4] = {};
    for (int i = 0; i < 4; ++i) {
      if (!ctx->saved_data[std::string("need") + (char)('0' + i)].toBool()) continue;
      out[i] = at::empty(s[i].sizes(), as(x, c.type));
      to[i] = out[i].mutable_data_ptr();
      if (c.odd(i)) m.add(true, to[i], c.wide(i), c.high(i), c.wide(i), i != 0);
    }
    int rc = m.make(x, c.d.dtype);
    if (rc) fail(rc, "pal_copy_matrices");
    PalMlpTensors r = c.fill(m, t);
    r.kept = (void*)ptr(kept);
    for (int i = 0, n = 0; i < 4; ++i)
      if (to[i] && c.odd(i)) to[i] = (void*)m.out[n++].src;
    PalMlpGrads g{dy_copied ? m.in[m.n_in - 1].dst : ptr(dy), to[0], to[1], to[2], to[3]};
    const size_t bytes = abi.gated_mlp_bwd_workspace_bytes(&c.d, &g);
    Tensor ws = workspace(x, bytes);
    {
      NoGil off;
      rc = abi.gated_mlp_bwd(&c.d, &r, &g, ws.mutable_data_ptr(), bytes, stream_of(x.device()));
      if (!rc) rc = m.take(x, c.d.dtype);
    }
    if (rc) fail(rc, "pal_gated_mlp_bwd");
    return once({out[0], out[1], out[2], out[3], none});
  }
};

// y, or None
py::object gated_mlp(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, int64_t act) {
  if (observed_or_dual({&x, &wg, &wu, &wd})) return py::none();
  const MlpCall c(x, wg, wu, wd, act);
  if (!c.ok) return py::none();
  if (any_grad({&x, &wg, &wu, &wd})) return applied([&] { return py::cast(MlpNode::apply(x, wg, wu, wd, act)); });
  Tensor y = c.out(x), none;
  if (c.run(x, wg, wu, wd, y, none)) return py::none();
  return py::cast(y);
}

}  // namespace block
