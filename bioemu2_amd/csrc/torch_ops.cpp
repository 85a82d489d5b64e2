// The trainable operators as torch ops (torch.ops.bioemu_mi355x.{layer_norm, relative_position, attention}): argument
// checks, output and workspace allocation, the C ABI's calls and the gradients.
//
// These run in C++ because a training step's backward pass runs in autograd's own thread: the same glue in Python took
// 60 to 130 us a step of host time there and back (a step of the smallest sizes computes for 15), and 40 to 70 here.
// Each op has a form with what its backward pass reads (`*_train`) and a backward op of its own, all reached through the
// dispatcher, so that tracing, fake tensors and modes see them.  Gradients are first order.
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include "../../include/bioemu2_mi355x.h"

namespace {

using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

void check_rc(int rc, const char* what) {
  if (rc == 0) return;
  TORCH_CHECK_VALUE(rc != BIOEMU_ERR_INVALID_ARG && rc != BIOEMU_ERR_UNSUPPORTED, what, ": ", bioemu_last_error(),
                    " (code ", rc, ")");
  TORCH_CHECK(false, what, ": ", bioemu_last_error(), " (code ", rc, ")");
}

hipStream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* ptr(const optional<Tensor>& t) { return t && t->defined() ? t->data_ptr() : nullptr; }
optional<Tensor> maybe(const Tensor& t) { return t.defined() ? optional<Tensor>(t) : std::nullopt; }
Tensor or_undefined(const optional<Tensor>& t) { return t ? *t : Tensor(); }
Tensor none_like(const Tensor& t) { return at::empty({0}, t.options()); }
Tensor bytes(int64_t n, const Tensor& like) { return at::empty({n}, like.options().dtype(at::kByte)); }

bool is_float(const Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat; }
bool is_f32(const Tensor& t) { return t.scalar_type() == at::kFloat; }
bool is_bf16(const Tensor& t) { return t.scalar_type() == at::kBFloat16; }

void check_activation(const Tensor& t, const char* what) {
  TORCH_CHECK_VALUE(is_float(t), what, ": expected fp32 or bf16, got ", t.scalar_type());
}
void check_shape(const Tensor& t, const char* what, at::IntArrayRef shape, const Tensor& like) {
  TORCH_CHECK_VALUE(t.sizes() == shape, what, ": expected shape ", shape, ", got ", t.sizes());
  TORCH_CHECK_VALUE(t.device() == like.device(), what, ": tensor on ", t.device(), ", expected ", like.device());
}
// A parameter of fp32 or bf16, contiguous.
Tensor parameter(const Tensor& t, const char* what, at::IntArrayRef shape, const Tensor& like) {
  check_activation(t, what);
  check_shape(t, what, shape, like);
  return t.contiguous();
}
Tensor whole_numbers(const Tensor& t, const char* what, at::ScalarType type, at::IntArrayRef shape, const Tensor& like) {
  TORCH_CHECK_VALUE(t.scalar_type() == type, what, ": expected dtype ", type, ", got ", t.scalar_type());
  check_shape(t, what, shape, like);
  return t.contiguous();
}
optional<Tensor> whole_numbers(const optional<Tensor>& t, const char* what, at::IntArrayRef shape, const Tensor& like) {
  return t ? optional<Tensor>(whole_numbers(*t, what, at::kInt, shape, like)) : std::nullopt;
}

// Typed handle of one of the ops below, through the dispatcher.
template <class F>
c10::TypedOperatorHandle<F> handle(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}

bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }
bool wants_grad(const optional<Tensor>& t) { return t && wants_grad(*t); }

// Forward-mode derivatives are refused: below autograd a tangent would be dropped without a word.
bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }
bool has_tangent(const optional<Tensor>& t) { return t && has_tangent(*t); }
template <class... T>
void check_no_tangents(const char* what, const T&... inputs) {
  TORCH_CHECK_NOT_IMPLEMENTED(!(has_tangent(inputs) || ...), what, ": no forward-mode derivative");
}

// ---------------------------------------------------------------------------
// LayerNorm
// ---------------------------------------------------------------------------
// x with the stride of its rows (of the last dimension, neighbouring values adjacent): itself where its strides allow,
// a copy else.
std::pair<Tensor, int64_t> as_rows(const Tensor& x) {
  const int64_t n = x.dim(), c = x.size(-1);
  if (x.is_contiguous()) return {x, c};
  if (x.stride(-1) == 1 || c == 1) {
    int64_t stride = -1, rows = 1;   // rows collapsed so far, and the stride of the innermost of them
    for (int64_t d = n - 2; d >= 0; --d) {
      if (x.size(d) == 1) continue;
      if (stride < 0)
        stride = x.stride(d);
      else if (x.stride(d) != stride * rows)
        return {x.contiguous(), c};
      rows *= x.size(d);
    }
    if (stride < 0) stride = c;
    return {x, stride};
  }
  return {x.contiguous(), c};
}

void check_rows(const Tensor& x) {
  TORCH_CHECK_VALUE(x.dim() > 0 && x.sym_size(-1) > 0, "layer_norm: x must have a last dimension, got ", x.sym_sizes());
}

struct NormParams {
  Tensor w, b;
  int bf16 = 0;
};
NormParams norm_params(const Tensor& x, const optional<Tensor>& w, const optional<Tensor>& b) {
  check_activation(x, "layer_norm x");
  check_rows(x);
  const int64_t c[1] = {x.size(-1)};
  NormParams p;
  if (w) p.w = parameter(*w, "layer_norm weight", c, x);
  if (b) p.b = parameter(*b, "layer_norm bias", c, x);
  TORCH_CHECK_VALUE(!w || !b || w->scalar_type() == b->scalar_type(), "layer_norm: weight is ",
                    w ? w->scalar_type() : at::kFloat, ", bias ", b ? b->scalar_type() : at::kFloat);
  p.bf16 = (w && is_bf16(*w)) || (b && is_bf16(*b));
  return p;
}

std::pair<Tensor, Tensor> norm_run(const Tensor& x, const optional<Tensor>& w, const optional<Tensor>& b, double eps,
                                   bool train) {
  const NormParams p = norm_params(x, w, b);
  const c10::OptionalDeviceGuard guard(x.device());
  const auto [src, stride] = as_rows(x);
  const int64_t c = x.size(-1), rows = x.numel() / c;
  Tensor y = at::empty(x.sizes(), x.options()), stats;
  if (train) stats = at::empty({rows, 2}, x.options().dtype(at::kFloat));
  check_rc(bioemu_layer_norm_fwd(src.data_ptr(), ptr(p.w), ptr(p.b), y.data_ptr(), static_cast<float*>(ptr(stats)), rows,
                                 c, stride, (float)eps, is_f32(x), p.bf16, stream_of(x)),
           "bioemu_layer_norm_fwd");
  return {y, stats};
}

Tensor layer_norm_cuda(const Tensor& x, const optional<Tensor>& w, const optional<Tensor>& b, double eps) {
  return norm_run(x, w, b, eps, false).first;
}
std::tuple<Tensor, Tensor> layer_norm_train_cuda(const Tensor& x, const optional<Tensor>& w, const optional<Tensor>& b,
                                                 double eps) {
  auto [y, stats] = norm_run(x, w, b, eps, true);
  return {y, stats};
}
at::ScalarType norm_grad_type(const optional<Tensor>& w, bool bias_bf16) {
  return w ? w->scalar_type() : (bias_bf16 ? at::kBFloat16 : at::kFloat);
}
// dx, dweight and dbias; empty where not wanted
std::tuple<Tensor, Tensor, Tensor> layer_norm_backward_cuda(const Tensor& x, const Tensor& dy, const Tensor& stats,
                                                            const optional<Tensor>& w, bool want_x, bool want_w,
                                                            bool want_b, bool bias_bf16) {
  const c10::OptionalDeviceGuard guard(x.device());
  check_rows(x);
  const int64_t c = x.size(-1), rows = x.numel() / c;
  check_activation(x, "layer_norm x");
  TORCH_CHECK_VALUE(dy.scalar_type() == x.scalar_type() && dy.sizes() == x.sizes(), "layer_norm_backward: dy is ",
                    dy.scalar_type(), " ", dy.sizes());
  const int64_t sshape[2] = {rows, 2}, cshape[1] = {c};
  check_shape(stats, "layer_norm stats", sshape, x);
  const Tensor weight = w ? parameter(*w, "layer_norm weight", cshape, x) : Tensor();
  const at::ScalarType wt = norm_grad_type(w, bias_bf16);
  const auto popt = x.options().dtype(wt);
  Tensor dx = want_x ? at::empty(x.sizes(), x.options()) : none_like(x);
  if (rows == 0) return {dx, at::zeros({want_w ? c : 0}, popt), at::zeros({want_b ? c : 0}, popt)};
  Tensor dw = at::empty({want_w ? c : 0}, popt), db = at::empty({want_b ? c : 0}, popt), ws;
  const auto [src, stride] = as_rows(x);
  const auto [dsrc, dstride] = as_rows(dy);
  const int64_t need = want_w || want_b ? (int64_t)bioemu_layer_norm_bwd_workspace_bytes(rows, c) : 0;
  if (need) ws = bytes(need, x);
  check_rc(bioemu_layer_norm_bwd(src.data_ptr(), dsrc.data_ptr(), stats.data_ptr<float>(), ptr(weight),
                                 want_x ? dx.data_ptr() : nullptr, want_w ? dw.data_ptr() : nullptr,
                                 want_b ? db.data_ptr() : nullptr, ptr(ws), need, rows, c, stride, dstride, is_f32(x),
                                 wt == at::kBFloat16, stream_of(x)),
           "bioemu_layer_norm_bwd");
  return {dx, dw, db};
}

Tensor layer_norm_meta(const Tensor& x, const optional<Tensor>&, const optional<Tensor>&, double) {
  check_rows(x);
  return at::empty_symint(x.sym_sizes(), x.options());
}
std::tuple<Tensor, Tensor> layer_norm_train_meta(const Tensor& x, const optional<Tensor>&, const optional<Tensor>&,
                                                 double) {
  check_rows(x);   // rows are counted by division
  return {at::empty_symint(x.sym_sizes(), x.options()),
          at::empty_symint({x.sym_numel() / x.sym_size(-1), 2}, x.options().dtype(at::kFloat))};
}
std::tuple<Tensor, Tensor, Tensor> layer_norm_backward_meta(const Tensor& x, const Tensor&, const Tensor&,
                                                            const optional<Tensor>& w, bool want_x, bool want_w,
                                                            bool want_b, bool bias_bf16) {
  check_rows(x);
  const auto popt = x.options().dtype(norm_grad_type(w, bias_bf16));
  const c10::SymInt c = x.sym_size(-1), none = 0;
  return {want_x ? at::empty_symint(x.sym_sizes(), x.options()) : none_like(x),
          at::empty_symint({want_w ? c : none}, popt), at::empty_symint({want_b ? c : none}, popt)};
}

struct LayerNormFn : Function<LayerNormFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const optional<Tensor>& w, const optional<Tensor>& b,
                        double eps) {
    at::AutoDispatchBelowADInplaceOrView below;
    static auto op = handle<decltype(layer_norm_train_cuda)>("bioemu_mi355x::layer_norm_train");
    auto [y, stats] = op.call(x, w, b, eps);
    ctx->save_for_backward({x, or_undefined(w), stats});
    ctx->saved_data["has_b"] = b.has_value();
    ctx->saved_data["bias_bf16"] = b && is_bf16(*b);
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto saved = ctx->get_saved_variables();
    const bool has_w = saved[1].defined(), has_b = ctx->saved_data["has_b"].toBool();
    const bool need_x = ctx->needs_input_grad(0), need_w = has_w && ctx->needs_input_grad(1),
               need_b = has_b && ctx->needs_input_grad(1 + has_w);   // edges are of the tensors that are there
    static auto op = handle<decltype(layer_norm_backward_cuda)>("bioemu_mi355x::layer_norm_backward");
    auto [dx, dw, db] = op.call(saved[0], g[0], saved[2], maybe(saved[1]), need_x, need_w, need_b,
                                ctx->saved_data["bias_bf16"].toBool());
    return {need_x ? dx : Tensor(), need_w ? dw : Tensor(), need_b ? db : Tensor(), Tensor()};
  }
};

Tensor layer_norm_autograd(const Tensor& x, const optional<Tensor>& w, const optional<Tensor>& b, double eps) {
  check_no_tangents("layer_norm", x, w, b);
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(w) || wants_grad(b)))
    return LayerNormFn::apply(x, w, b, eps);
  at::AutoDispatchBelowADInplaceOrView below;
  static auto op = handle<decltype(layer_norm_cuda)>("bioemu_mi355x::layer_norm");
  return op.call(x, w, b, eps);
}

// ---------------------------------------------------------------------------
// Relative positions
// ---------------------------------------------------------------------------
struct Pairs {
  Tensor buckets, positions;
  optional<Tensor> chains;
  int64_t B, N, radius;
};
Pairs check_pairs(const Tensor& buckets, const Tensor& positions, const optional<Tensor>& chains, const Tensor& like) {
  TORCH_CHECK_VALUE(positions.dim() == 2, "relative_position: positions must be [B, N], got ", positions.sizes());
  TORCH_CHECK_VALUE(buckets.dim() == 1 && buckets.numel() % 2 == 1,
                    "relative_position: buckets must be [2 * radius + 1], got ", buckets.sizes());
  return {whole_numbers(buckets, "relative_position buckets", at::kByte, buckets.sizes(), like),
          whole_numbers(positions, "relative_position positions", at::kInt, positions.sizes(), like),
          whole_numbers(chains, "relative_position chains", positions.sizes(), like), positions.size(0),
          positions.size(1), buckets.numel() / 2};
}

Tensor relative_position_cuda(const Tensor& table, const optional<Tensor>& z, const Tensor& buckets,
                              const Tensor& positions, const optional<Tensor>& chains, at::ScalarType dtype) {
  TORCH_CHECK_VALUE(table.dim() == 2, "relative_position: table must be [num_buckets, C], got ", table.sizes());
  TORCH_CHECK_VALUE(dtype == at::kFloat || dtype == at::kBFloat16, "relative_position: expected fp32 or bf16, got ",
                    dtype);
  const c10::OptionalDeviceGuard guard(table.device());
  const Pairs p = check_pairs(buckets, positions, chains, table);
  const Tensor t = parameter(table, "relative_position table", table.sizes(), table);
  const int64_t C = t.size(1), shape[4] = {p.B, p.N, p.N, C};
  Tensor zc;
  if (z) {
    TORCH_CHECK_VALUE(z->scalar_type() == dtype, "relative_position: dtype ", dtype, ", z is ", z->scalar_type());
    check_shape(*z, "relative_position z", shape, table);
    // the kernel's 16-byte pieces; rows of other widths are read by values, at any address
    zc = z->is_contiguous() && (C * z->element_size()) % 16 == 0 && reinterpret_cast<uintptr_t>(z->data_ptr()) % 16 != 0
             ? z->clone()
             : z->contiguous();
  }
  Tensor out = at::empty(shape, t.options().dtype(dtype));
  check_rc(bioemu_relpos_fwd(t.data_ptr(), p.buckets.data_ptr<uint8_t>(), p.positions.data_ptr<int>(),
                             static_cast<int*>(ptr(p.chains)), ptr(zc), out.data_ptr(), p.B, p.N, C, p.radius,
                             t.size(0), dtype == at::kFloat, is_bf16(t), stream_of(t)),
           "bioemu_relpos_fwd");
  return out;
}
Tensor relative_position_backward_cuda(const Tensor& dout, const Tensor& buckets, const Tensor& positions,
                                       const optional<Tensor>& chains, int64_t num_buckets, at::ScalarType dtype) {
  check_activation(dout, "relative_position_backward dout");
  const c10::OptionalDeviceGuard guard(dout.device());
  const Pairs p = check_pairs(buckets, positions, chains, dout);
  TORCH_CHECK_VALUE(dout.dim() == 4, "relative_position_backward: dout must be [B, N, N, C], got ", dout.sizes());
  const int64_t C = dout.size(3), shape[4] = {p.B, p.N, p.N, C};
  check_shape(dout, "relative_position_backward dout", shape, dout);
  const auto opt = dout.options().dtype(dtype);
  if (dout.numel() == 0) return at::zeros({num_buckets, C}, opt);
  const Tensor d = dout.contiguous();
  Tensor dtable = at::empty({num_buckets, C}, opt);
  const int64_t need = (int64_t)bioemu_relpos_bwd_workspace_bytes(p.B, p.N, C, num_buckets);
  const Tensor ws = bytes(need, dout);
  check_rc(bioemu_relpos_bwd(d.data_ptr(), p.buckets.data_ptr<uint8_t>(), p.positions.data_ptr<int>(),
                             static_cast<int*>(ptr(p.chains)), dtable.data_ptr(), ws.data_ptr(), need, p.B, p.N, C,
                             p.radius, num_buckets, is_f32(d), dtype == at::kBFloat16, stream_of(d)),
           "bioemu_relpos_bwd");
  return dtable;
}

Tensor relative_position_meta(const Tensor& table, const optional<Tensor>&, const Tensor&, const Tensor& positions,
                              const optional<Tensor>&, at::ScalarType dtype) {
  const auto B = positions.sym_size(0), N = positions.sym_size(1);
  return at::empty_symint({B, N, N, table.sym_size(1)}, table.options().dtype(dtype));
}
Tensor relative_position_backward_meta(const Tensor& dout, const Tensor&, const Tensor&, const optional<Tensor>&,
                                       int64_t num_buckets, at::ScalarType dtype) {
  return at::empty_symint({num_buckets, dout.sym_size(3)}, dout.options().dtype(dtype));
}

struct RelativePositionFn : Function<RelativePositionFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& table, const optional<Tensor>& z, const Tensor& buckets,
                        const Tensor& positions, const optional<Tensor>& chains, at::ScalarType dtype) {
    at::AutoDispatchBelowADInplaceOrView below;
    static auto op = handle<decltype(relative_position_cuda)>("bioemu_mi355x::relative_position");
    ctx->save_for_backward({buckets, positions, or_undefined(chains)});
    ctx->saved_data["has_z"] = z.has_value();
    ctx->saved_data["num_buckets"] = table.size(0);
    ctx->saved_data["dtype"] = (int64_t)table.scalar_type();
    return op.call(table, z, buckets, positions, chains, dtype);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto saved = ctx->get_saved_variables();
    const bool has_z = ctx->saved_data["has_z"].toBool();
    Tensor dtable;
    static auto op = handle<decltype(relative_position_backward_cuda)>("bioemu_mi355x::relative_position_backward");
    if (ctx->needs_input_grad(0))
      dtable = op.call(g[0], saved[0], saved[1], maybe(saved[2]), ctx->saved_data["num_buckets"].toInt(),
                       (at::ScalarType)ctx->saved_data["dtype"].toInt());
    return {dtable, has_z && ctx->needs_input_grad(1) ? g[0] : Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor relative_position_autograd(const Tensor& table, const optional<Tensor>& z, const Tensor& buckets,
                                  const Tensor& positions, const optional<Tensor>& chains, at::ScalarType dtype) {
  check_no_tangents("relative_position", table, z);
  if (at::GradMode::is_enabled() && (wants_grad(table) || wants_grad(z)))
    return RelativePositionFn::apply(table, z, buckets, positions, chains, dtype);
  at::AutoDispatchBelowADInplaceOrView below;
  static auto op = handle<decltype(relative_position_cuda)>("bioemu_mi355x::relative_position");
  return op.call(table, z, buckets, positions, chains, dtype);
}

// ---------------------------------------------------------------------------
// Attention
// ---------------------------------------------------------------------------
// [B, N, H, D] with adjacent values of a head, rows at 16-byte addresses and at least a head apart: t where it is so, a
// copy else.
Tensor heads(const Tensor& t) {
  const int64_t per = 16 / t.element_size();
  const bool rows = t.size(1) <= 1 || (t.stride(1) >= t.size(3) && t.stride(1) <= (int64_t(1) << 23) &&
                                       t.stride(1) % per == 0);
  if (t.stride(3) == 1 && rows && t.stride(0) % per == 0 && t.stride(2) % per == 0 &&
      reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0)
    return t;
  return t.clone(at::MemoryFormat::Contiguous);
}

// The optional arguments, and the C ABI's structure over all of them.
struct AttentionCall {
  Tensor q, k, v, table, buckets;
  optional<Tensor> q_seg, k_seg, prefix, lengths;
  bioemu_attention_args args{};

  AttentionCall(const Tensor& q_, const Tensor& k_, const Tensor& v_, const optional<Tensor>& table_,
                const optional<Tensor>& buckets_, const optional<Tensor>& q_seg_, const optional<Tensor>& k_seg_,
                const optional<Tensor>& prefix_, const optional<Tensor>& lengths_, double scale, double cap,
                bool causal) {
    check_activation(q_, "attention q");
    TORCH_CHECK_VALUE(q_.dim() == 4 && k_.dim() == 4 && k_.sizes() == v_.sizes() && k_.size(0) == q_.size(0) &&
                          k_.size(3) == q_.size(3),
                      "attention: q ", q_.sizes(), ", k ", k_.sizes(), ", v ", v_.sizes());
    TORCH_CHECK_VALUE(k_.scalar_type() == q_.scalar_type() && v_.scalar_type() == q_.scalar_type(), "attention: q is ",
                      q_.scalar_type(), ", k ", k_.scalar_type(), ", v ", v_.scalar_type());
    TORCH_CHECK_VALUE(k_.device() == q_.device() && v_.device() == q_.device(), "attention: q on ", q_.device(),
                      ", k on ", k_.device(), ", v on ", v_.device());
    TORCH_CHECK_VALUE(q_seg_.has_value() == k_seg_.has_value(),
                      "attention: segments of queries and of keys come together");
    const int64_t B = q_.size(0), Nq = q_.size(1), H = q_.size(2), Nk = k_.size(1);
    const int64_t bq[2] = {B, Nq}, bk[2] = {B, Nk}, b1[1] = {B};
    q_seg = whole_numbers(q_seg_, "attention segments", bq, q_);
    k_seg = whole_numbers(k_seg_, "attention key segments", bk, q_);
    prefix = whole_numbers(prefix_, "attention prefix", b1, q_);
    lengths = whole_numbers(lengths_, "attention cache_lengths", b1, q_);
    TORCH_CHECK_VALUE(table_.has_value() == buckets_.has_value() && (!table_ || table_->dim() == 2),
                      "attention: a bias table [num_buckets, H] comes with its buckets");
    if (table_) {
      TORCH_CHECK_VALUE(buckets_->dim() == 1 && buckets_->numel() % 2 == 1,
                        "attention: buckets must be [2 * radius + 1], got ", buckets_->sizes());
      buckets = whole_numbers(*buckets_, "attention buckets", at::kByte, buckets_->sizes(), q_);
      const int64_t shape[2] = {table_->size(0), H};
      table = parameter(*table_, "attention bias table", shape, q_);
      args.bias_table = table.data_ptr();
      args.bias_buckets = buckets.data_ptr<uint8_t>();
      args.radius = buckets.numel() / 2;
      args.num_buckets = table.size(0);
      args.table_bf16 = is_bf16(table);
    }
    q = heads(q_);
    k = heads(k_);
    v = heads(v_);
    args.q = q.data_ptr();
    args.k = k.data_ptr();
    args.v = v.data_ptr();
    for (int i = 0; i < 3; ++i) {
      args.q_stride[i] = q.stride(i);
      args.k_stride[i] = k.stride(i);
      args.v_stride[i] = v.stride(i);
    }
    args.q_segments = static_cast<int*>(ptr(q_seg));
    args.k_segments = static_cast<int*>(ptr(k_seg));
    args.prefix = static_cast<int*>(ptr(prefix));
    args.lengths = static_cast<int*>(ptr(lengths));
    args.B = B;
    args.Nq = Nq;
    args.Nk = Nk;
    args.H = H;
    args.Hk = k.size(2);
    args.D = q.size(3);
    args.scale = (float)scale;
    args.cap = (float)cap;
    TORCH_CHECK_VALUE(cap == 0 || args.cap > 0, "attention: cap ", cap);
    args.causal = causal;
    args.f32 = is_f32(q);
  }
};

#define ATTENTION_PARAMS                                                                                            \
  const Tensor &q, const Tensor &k, const Tensor &v, const optional<Tensor>&table, const optional<Tensor>&buckets,  \
      const optional<Tensor>&q_seg, const optional<Tensor>&k_seg, const optional<Tensor>&prefix,                    \
      const optional<Tensor>&lengths, double scale, double cap, bool causal
#define ATTENTION_ARGS q, k, v, table, buckets, q_seg, k_seg, prefix, lengths, scale, cap, causal

// o, and for training what its rounding took off (empty in fp32) and the rows' log-sums
std::tuple<Tensor, Tensor, Tensor> attention_run(ATTENTION_PARAMS, bool train) {
  const c10::OptionalDeviceGuard guard(q.device());
  const AttentionCall c(ATTENTION_ARGS);
  Tensor out = at::empty(q.sizes(), q.options()), lo, lse, ws;
  if (train) {
    lo = is_f32(q) ? none_like(q) : at::empty(q.sizes(), q.options());
    lse = at::empty({2, q.size(0), q.size(2), q.size(1)}, q.options().dtype(at::kFloat));
  }
  const int64_t need = (int64_t)bioemu_attention_workspace_bytes(&c.args);
  if (need) ws = bytes(need, q);
  check_rc(bioemu_attention_fwd(&c.args, out.data_ptr(), train && !is_f32(q) ? lo.data_ptr() : nullptr,
                                static_cast<float*>(ptr(lse)), ptr(ws), need, stream_of(q)),
           "bioemu_attention_fwd");
  return {out, lo, lse};
}
Tensor attention_cuda(ATTENTION_PARAMS) { return std::get<0>(attention_run(ATTENTION_ARGS, false)); }
std::tuple<Tensor, Tensor, Tensor> attention_train_cuda(ATTENTION_PARAMS) {
  return attention_run(ATTENTION_ARGS, true);
}
// dq, dk, dv and the table's gradient (empty where not wanted)
std::tuple<Tensor, Tensor, Tensor, Tensor> attention_backward_cuda(const Tensor& out, const Tensor& lo,
                                                                   const Tensor& lse, const Tensor& dout,
                                                                   ATTENTION_PARAMS,
                                                                   bool want_table) {
  const c10::OptionalDeviceGuard guard(q.device());
  const AttentionCall c(ATTENTION_ARGS);
  TORCH_CHECK_VALUE(dout.scalar_type() == q.scalar_type() && dout.sizes() == q.sizes() &&
                        out.scalar_type() == q.scalar_type() && out.sizes() == q.sizes(),
                    "attention_backward: out ", out.sizes(), ", dout ", dout.sizes(), " of q ", q.sizes());
  const int64_t lshape[4] = {2, q.size(0), q.size(2), q.size(1)};
  check_shape(lse, "attention_backward lse", lshape, q);
  if (!is_f32(q)) check_shape(lo, "attention_backward lo", q.sizes(), q);
  want_table = want_table && table;
  const auto fresh = [](const Tensor& t) { return at::empty(t.sizes(), t.options()); };
  if (q.size(0) == 0 || q.size(1) == 0)
    return {fresh(q), at::zeros(k.sizes(), k.options()), at::zeros(v.sizes(), v.options()),
            want_table ? at::zeros(table->sizes(), table->options()) : none_like(q)};
  Tensor dq = fresh(q), dk = fresh(k), dv = fresh(v), dtable = want_table ? fresh(c.table) : none_like(q);
  const Tensor o = out.contiguous(), ol = lo.contiguous(), d = heads(dout), l = lse.contiguous();
  const int64_t need = (int64_t)bioemu_attention_bwd_workspace_bytes(&c.args, want_table);
  const Tensor ws = bytes(need, q);
  const int64_t ds[3] = {d.stride(0), d.stride(1), d.stride(2)};
  check_rc(bioemu_attention_bwd(&c.args, o.data_ptr(), is_f32(q) ? nullptr : ol.data_ptr(), l.data_ptr<float>(),
                                d.data_ptr(), ds, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                                want_table ? dtable.data_ptr() : nullptr, ws.data_ptr(), need, stream_of(q)),
           "bioemu_attention_bwd");
  return {dq, dk, dv, dtable};
}

Tensor attention_meta(ATTENTION_PARAMS) { return at::empty_symint(q.sym_sizes(), q.options()); }
std::tuple<Tensor, Tensor, Tensor> attention_train_meta(ATTENTION_PARAMS) {
  return {at::empty_symint(q.sym_sizes(), q.options()),
          is_f32(q) ? none_like(q) : at::empty_symint(q.sym_sizes(), q.options()),
          at::empty_symint({2, q.sym_size(0), q.sym_size(2), q.sym_size(1)}, q.options().dtype(at::kFloat))};
}
std::tuple<Tensor, Tensor, Tensor, Tensor> attention_backward_meta(const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                                                                   ATTENTION_PARAMS, bool want_table) {
  const auto fresh = [](const Tensor& t) { return at::empty_symint(t.sym_sizes(), t.options()); };
  return {fresh(q), fresh(k), fresh(v), want_table && table ? fresh(*table) : none_like(q)};
}

struct AttentionFn : Function<AttentionFn> {
  static Tensor forward(AutogradContext* ctx, ATTENTION_PARAMS) {
    at::AutoDispatchBelowADInplaceOrView below;
    static auto op = handle<decltype(attention_train_cuda)>("bioemu_mi355x::attention_train");
    auto [out, lo, lse] = op.call(ATTENTION_ARGS);
    ctx->save_for_backward({q, k, v, or_undefined(table), or_undefined(buckets), or_undefined(q_seg),
                            or_undefined(k_seg), or_undefined(prefix), or_undefined(lengths), out, lo, lse});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["cap"] = cap;
    ctx->saved_data["causal"] = causal;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto s = ctx->get_saved_variables();
    const bool need_table = s[3].defined() && ctx->needs_input_grad(3);
    static auto op = handle<decltype(attention_backward_cuda)>("bioemu_mi355x::attention_backward");
    auto [dq, dk, dv, dtable] =
        op.call(s[9], s[10], s[11], g[0], s[0], s[1], s[2], maybe(s[3]), maybe(s[4]), maybe(s[5]), maybe(s[6]), maybe(s[7]),
                maybe(s[8]), ctx->saved_data["scale"].toDouble(), ctx->saved_data["cap"].toDouble(),
                ctx->saved_data["causal"].toBool(), need_table);
    variable_list grads(12);
    if (ctx->needs_input_grad(0)) grads[0] = dq;
    if (ctx->needs_input_grad(1)) grads[1] = dk;
    if (ctx->needs_input_grad(2)) grads[2] = dv;
    if (need_table) grads[3] = dtable;
    return grads;
  }
};

Tensor attention_autograd(ATTENTION_PARAMS) {
  check_no_tangents("attention", q, k, v, table);
  if (at::GradMode::is_enabled() && (wants_grad(q) || wants_grad(k) || wants_grad(v) || wants_grad(table)))
    return AttentionFn::apply(ATTENTION_ARGS);
  at::AutoDispatchBelowADInplaceOrView below;
  static auto op = handle<decltype(attention_cuda)>("bioemu_mi355x::attention");
  return op.call(ATTENTION_ARGS);
}

#define ATTENTION_SCHEMA                                                                                            \
  "Tensor q, Tensor k, Tensor v, Tensor? table, Tensor? buckets, Tensor? q_segments, Tensor? k_segments, "          \
  "Tensor? prefix, Tensor? lengths, float scale, float cap, bool causal"

}  // namespace

TORCH_LIBRARY_FRAGMENT(bioemu_mi355x, m) {
  m.def("layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps) -> Tensor");
  m.def("layer_norm_train(Tensor x, Tensor? weight, Tensor? bias, float eps) -> (Tensor, Tensor)");
  m.def("layer_norm_backward(Tensor x, Tensor dy, Tensor stats, Tensor? weight, bool want_x, bool want_weight, "
        "bool want_bias, bool bias_bf16) -> (Tensor, Tensor, Tensor)");
  m.def("relative_position(Tensor table, Tensor? z, Tensor buckets, Tensor positions, Tensor? chains, "
        "ScalarType dtype) -> Tensor");
  m.def("relative_position_backward(Tensor dout, Tensor buckets, Tensor positions, Tensor? chains, int num_buckets, "
        "ScalarType dtype) -> Tensor");
  m.def("attention(" ATTENTION_SCHEMA ") -> Tensor");
  m.def("attention_train(" ATTENTION_SCHEMA ") -> (Tensor, Tensor, Tensor)");
  m.def("attention_backward(Tensor out, Tensor out_lo, Tensor lse, Tensor dout, " ATTENTION_SCHEMA
        ", bool want_table) -> (Tensor, Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(bioemu_mi355x, CUDA, m) {
  m.impl("layer_norm", &layer_norm_cuda);
  m.impl("layer_norm_train", &layer_norm_train_cuda);
  m.impl("layer_norm_backward", &layer_norm_backward_cuda);
  m.impl("relative_position", &relative_position_cuda);
  m.impl("relative_position_backward", &relative_position_backward_cuda);
  m.impl("attention", &attention_cuda);
  m.impl("attention_train", &attention_train_cuda);
  m.impl("attention_backward", &attention_backward_cuda);
}

TORCH_LIBRARY_IMPL(bioemu_mi355x, Meta, m) {
  m.impl("layer_norm", &layer_norm_meta);
  m.impl("layer_norm_train", &layer_norm_train_meta);
  m.impl("layer_norm_backward", &layer_norm_backward_meta);
  m.impl("relative_position", &relative_position_meta);
  m.impl("relative_position_backward", &relative_position_backward_meta);
  m.impl("attention", &attention_meta);
  m.impl("attention_train", &attention_train_meta);
  m.impl("attention_backward", &attention_backward_meta);
}

TORCH_LIBRARY_IMPL(bioemu_mi355x, Autograd, m) {
  m.impl("layer_norm", &layer_norm_autograd);
  m.impl("relative_position", &relative_position_autograd);
  m.impl("attention", &attention_autograd);
  // a gradient of a gradient raises
  for (const char* name : {"layer_norm_train", "layer_norm_backward", "relative_position_backward", "attention_train",
                           "attention_backward"})
    m.impl(name, torch::autograd::autogradNotImplementedFallback());
}
