// torch binding of the operators that come with gradients or are called for
// single tokens: argument checks, allocations and the C ABI call in compiled
// code, and their autograd functions (a Python autograd.Function and ctypes
// call cost several times the kernels' own time there).  The other entry
// points are bound by ctypes.  The library's functions are handed over by
// address, so that INT8_HYBRID_MOE_LIB decides here too.
#include <torch/extension.h>
#include <torch/version.h>

#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>

#include <initializer_list>
#include <optional>
#include <string>
#include <tuple>
#include <unordered_map>

#include "i8moe.h"

namespace {

using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Library {
  decltype(&i8moe_last_error) last_error;
  decltype(&i8moe_route_workspace_size) route_workspace_size;
  decltype(&i8moe_moe_permute_metadata) moe_permute_metadata;
  decltype(&i8moe_moe_scatter_rows) moe_scatter_rows;
  decltype(&i8moe_moe_unpermute_rows) moe_unpermute_rows;
  decltype(&i8moe_moe_permute_backward) moe_permute_backward;
  decltype(&i8moe_moe_unpermute_backward) moe_unpermute_backward;
  decltype(&i8moe_rms_norm) rms_norm;
  decltype(&i8moe_rms_norm_backward_workspace_size) rms_norm_backward_workspace_size;
  decltype(&i8moe_rms_norm_backward) rms_norm_backward;
  decltype(&i8moe_int4_grouped_mv) int4_grouped_mv;
} lib{};

void bind(const std::unordered_map<std::string, uintptr_t>& address) {
#define I8_BIND(name) \
  lib.name = reinterpret_cast<decltype(lib.name)>(address.at("i8moe_" #name))
  I8_BIND(last_error);
  I8_BIND(route_workspace_size);
  I8_BIND(moe_permute_metadata);
  I8_BIND(moe_scatter_rows);
  I8_BIND(moe_unpermute_rows);
  I8_BIND(moe_permute_backward);
  I8_BIND(moe_unpermute_backward);
  I8_BIND(rms_norm);
  I8_BIND(rms_norm_backward_workspace_size);
  I8_BIND(rms_norm_backward);
  I8_BIND(int4_grouped_mv);
#undef I8_BIND
}

void check(int rc, const char* what) { TORCH_CHECK(rc == 0, what, ": ", lib.last_error()); }

bool float_type(const Tensor& t) {
  return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf ||
         t.scalar_type() == at::kFloat;
}

int type_of(const Tensor& t) {
  return t.scalar_type() == at::kBFloat16 ? I8MOE_BF16
         : t.scalar_type() == at::kHalf   ? I8MOE_FP16
                                          : I8MOE_FP32;
}

i8moe_stream_t stream_of(const Tensor& t) {
  return at::cuda::getCurrentCUDAStream(t.get_device()).stream();
}

// Past the dispatcher: half a microsecond less per tensor.
Tensor empty(at::IntArrayRef size, const Tensor& like, at::ScalarType type) {
  return Tensor(at::detail::empty_cuda(size, type, like.device(), std::nullopt));
}

// A gradient function of these operators runs once: their gradients are no
// differentiable operators.
void once(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what, " is differentiable once (no create_graph)");
}

// These operators go past the dispatcher and would leave out the tangents of
// forward-mode differentiation.
void no_tangents(const char* what, std::initializer_list<Tensor> inputs) {
  for (const Tensor& t : inputs)
    TORCH_CHECK(!t.defined() || !t._fw_grad(0).defined(), what, " has no forward-mode derivative");
}

// Inside a graph's capture: a leaf whose gradient node lives on in an eager
// graph brings that graph's stream into the captured backward pass, which ends
// the process there.  Refused here instead.
void check_capture(const char* what, std::initializer_list<Tensor> inputs) {
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
  for (const Tensor& t : inputs) {
    if (!t.defined() || !t.requires_grad() || !t.is_leaf()) continue;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(t);
    if (!node) continue;
    const auto stream = node->stream();
    TORCH_CHECK(!stream || *stream == at::cuda::getCurrentCUDAStream(t.get_device()).unwrap(), what,
                ": an eager graph of the same leaves is alive; drop its outputs before capturing");
  }
}

// ------------------------------------------------------------------- norm

// `t` as [rows, K]: a view where its strides allow one, else a copy.
Tensor rows_of(const Tensor& t) {
  Tensor r = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
  return r.size(1) == 1 || r.stride(1) == 1 ? r : r.contiguous();
}

void check_norm(const char* what, const Tensor& x, const Tensor& weight, double eps,
                const optional<Tensor>& residual) {
  TORCH_CHECK(x.is_cuda(), what, ": x must be a CUDA tensor");
  TORCH_CHECK(float_type(x), what, ": x must be bfloat16, float16 or float32");
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1, what, ": x must have shape [..., K] with K >= 1");
  TORCH_CHECK(weight.device() == x.device(), what, ": weight must be on x's device");
  TORCH_CHECK(weight.scalar_type() == x.scalar_type() || weight.scalar_type() == at::kFloat, what,
              ": weight must have x's dtype or float32");
  TORCH_CHECK(weight.dim() == 1 && weight.size(0) == x.size(-1), what,
              ": weight must have shape [K]");
  TORCH_CHECK(eps >= 0 && eps < 3e38, what, ": eps must be finite and not negative");
  no_tangents(what, {x, weight, residual ? *residual : Tensor()});
  if (residual) {
    TORCH_CHECK(residual->device() == x.device(), what, ": residual must be on x's device");
    TORCH_CHECK(residual->scalar_type() == x.scalar_type(), what,
                ": residual must have x's dtype");
    TORCH_CHECK(residual->sizes() == x.sizes(), what, ": residual must have x's shape");
  }
}

// Launches the norm; returns the residual stream (undefined without one).
Tensor norm_forward(const Tensor& x, const Tensor& weight, double eps,
                    const optional<Tensor>& residual, Tensor* y, Tensor* rstd, Tensor* q,
                    Tensor* scale) {
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor xr = rows_of(x), w = weight.contiguous();
  Tensor rr, h;
  if (residual) {
    rr = rows_of(*residual);
    h = empty(x.sizes(), x, x.scalar_type());
  }
  check(lib.rms_norm(xr.data_ptr(), xr.stride(0), residual ? rr.data_ptr() : nullptr,
                     residual ? rr.stride(0) : 0, type_of(x), w.data_ptr(), type_of(w), xr.size(0),
                     xr.size(1), static_cast<float>(eps), residual ? h.data_ptr() : nullptr,
                     y ? y->data_ptr() : nullptr,
                     rstd ? static_cast<float*>(rstd->data_ptr()) : nullptr,
                     q ? static_cast<int8_t*>(q->data_ptr()) : nullptr,
                     scale ? static_cast<float*>(scale->data_ptr()) : nullptr, stream_of(x)),
        "rms_norm");
  return h;
}

std::tuple<Tensor, optional<Tensor>> rms_norm_backward(
    const Tensor& dy, const Tensor& x, const Tensor& weight, const Tensor& rstd,
    const optional<Tensor>& residual, const optional<Tensor>& residual_grad, bool weight_grad) {
  const char* what = "rms_norm_backward";
  check_norm(what, x, weight, 0.0, residual);
  auto like_x = [&](const Tensor& t) {
    return t.sizes() == x.sizes() && t.scalar_type() == x.scalar_type() && t.device() == x.device();
  };
  TORCH_CHECK(like_x(dy), what, ": dy must have x's shape, dtype and device");
  TORCH_CHECK(!residual_grad || like_x(*residual_grad), what,
              ": residual_grad must have x's shape, dtype and device");
  TORCH_CHECK(rstd.scalar_type() == at::kFloat && rstd.is_contiguous() &&
                  rstd.device() == x.device() && rstd.numel() == x.numel() / x.size(-1),
              what, ": rstd must be float32 [rows] on x's device");
  no_tangents(what, {dy, rstd, residual_grad ? *residual_grad : Tensor()});
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor xr = rows_of(x), gr = rows_of(dy), w = weight.contiguous();
  Tensor rr, hr;
  if (residual) rr = rows_of(*residual);
  if (residual_grad) hr = rows_of(*residual_grad);
  Tensor dx = empty(x.sizes(), x, x.scalar_type());
  optional<Tensor> dw;
  Tensor workspace;
  size_t bytes = 0;
  if (weight_grad) {
    dw = empty(weight.sizes(), x, weight.scalar_type());
    bytes = lib.rms_norm_backward_workspace_size(xr.size(0), xr.size(1));
    workspace = empty({static_cast<int64_t>(bytes)}, x, at::kByte);
  }
  check(lib.rms_norm_backward(gr.data_ptr(), gr.stride(0), residual_grad ? hr.data_ptr() : nullptr,
                              residual_grad ? hr.stride(0) : 0, xr.data_ptr(), xr.stride(0),
                              residual ? rr.data_ptr() : nullptr, residual ? rr.stride(0) : 0,
                              type_of(x), w.data_ptr(), type_of(w),
                              static_cast<const float*>(rstd.data_ptr()), xr.size(0), xr.size(1),
                              dx.data_ptr(), dw ? dw->data_ptr() : nullptr,
                              dw ? workspace.data_ptr() : nullptr, bytes, stream_of(x)),
        what);
  return {dx, dw};
}

optional<Tensor> some(const Tensor& t) { return t.defined() ? optional<Tensor>(t) : std::nullopt; }

struct RmsNorm : torch::autograd::Function<RmsNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight,
                               double eps, const optional<Tensor>& residual) {
    Tensor y = empty(x.sizes(), x, x.scalar_type());
    Tensor rstd = empty({x.numel() / x.size(-1)}, x, at::kFloat);
    const Tensor h = norm_forward(x, weight, eps, residual, &y, &rstd, nullptr, nullptr);
    ctx->save_for_backward({x, weight, rstd, residual ? *residual : Tensor()});
    ctx->set_materialize_grads(false);
    return residual ? variable_list{y, h} : variable_list{y};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("rms_norm");
    const Tensor dh = grads.size() > 1 ? grads[1] : Tensor();
    const bool two = grads.size() > 1;
    if (!grads[0].defined())  // y was not used: only the residual stream's gradient passes
      return {dh, Tensor(), Tensor(), two ? dh : Tensor()};
    const variable_list saved = ctx->get_saved_variables();
    const auto [dx, dw] =
        rms_norm_backward(grads[0], saved[0], saved[1], saved[2], some(saved[3]), some(dh),
                          ctx->needs_input_grad(1));
    return {dx, dw ? *dw : Tensor(), Tensor(), two ? dx : Tensor()};
  }
};

py::object rms_norm(const Tensor& x, const Tensor& weight, double eps,
                    const optional<Tensor>& residual) {
  check_norm("rms_norm", x, weight, eps, residual);
  if (at::GradMode::is_enabled() &&
      (x.requires_grad() || weight.requires_grad() || (residual && residual->requires_grad()))) {
    check_capture("rms_norm", {x, weight, residual ? *residual : Tensor()});
    const variable_list out = RmsNorm::apply(x, weight, eps, residual);
    return residual ? py::cast(std::make_tuple(out[0], out[1])) : py::cast(out[0]);
  }
  Tensor y = empty(x.sizes(), x, x.scalar_type());
  const Tensor h = norm_forward(x, weight, eps, residual, &y, nullptr, nullptr, nullptr);
  return residual ? py::cast(std::make_tuple(y, h)) : py::cast(y);
}

std::tuple<Tensor, Tensor, optional<Tensor>, optional<Tensor>> rms_norm_quant_int8(
    const Tensor& x, const Tensor& weight, double eps, const optional<Tensor>& residual,
    bool return_norm) {
  const char* what = "rms_norm_quant_int8";
  check_norm(what, x, weight, eps, residual);
  TORCH_CHECK(!(at::GradMode::is_enabled() &&
                (x.requires_grad() || weight.requires_grad() ||
                 (residual && residual->requires_grad()))),
              what, " has no gradient: call it under torch.no_grad()");
  Tensor q = empty(x.sizes(), x, at::kChar);
  Tensor scale = empty(x.sizes().slice(0, x.dim() - 1), x, at::kFloat);
  optional<Tensor> y, h;
  if (return_norm) y = empty(x.sizes(), x, x.scalar_type());
  const Tensor sum =
      norm_forward(x, weight, eps, residual, y ? &*y : nullptr, nullptr, &q, &scale);
  if (residual) h = sum;
  return {q, scale, y, h};
}

// ---------------------------------------------------------- sort and return

void check_rows(const char* what, const char* name, const Tensor& t) {
  TORCH_CHECK(t.is_cuda() && t.dim() == 2, what, ": ", name,
              " must be a CUDA tensor [rows, hidden]");
  TORCH_CHECK(float_type(t), what, ": ", name, " must be bfloat16, float16 or float32");
  TORCH_CHECK(t.size(1) * t.element_size() % 16 == 0, what,
              ": hidden row must be a multiple of 16 bytes");
}

void check_maps(const char* what, const Tensor& inv, const optional<Tensor>& eft, int64_t rows,
                const Tensor& like) {
  TORCH_CHECK(inv.scalar_type() == at::kInt && inv.is_contiguous() &&
                  inv.device() == like.device() && inv.numel() == rows,
              what, ": inv_permuted_idx must be contiguous int32 with n_token * topk elements");
  if (eft)
    TORCH_CHECK(eft->scalar_type() == at::kLong && eft->is_contiguous() &&
                    eft->device() == like.device() && eft->dim() == 1 && eft->numel() >= 1,
                what, ": expert_first_token_offset must be contiguous int64 [n_local_expert + 1]");
}

// `t` contiguous and 16-byte aligned, copied when it is not.
Tensor aligned(const Tensor& t) {
  Tensor c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0 ? c : c.clone();
}

const int32_t* ints(const Tensor& t) { return static_cast<const int32_t*>(t.data_ptr()); }

const int64_t* offsets(const optional<Tensor>& eft) {
  return eft ? static_cast<const int64_t*>(eft->data_ptr()) : nullptr;
}

int64_t experts(const optional<Tensor>& eft) { return eft ? eft->numel() - 1 : 0; }

Tensor moe_permute_backward(const Tensor& permuted_grad, const Tensor& inv,
                            const optional<Tensor>& eft, int64_t n_token, int64_t topk) {
  const char* what = "moe_permute_backward";
  check_rows(what, "permuted_grad", permuted_grad);
  TORCH_CHECK(n_token >= 0 && topk >= 1 && permuted_grad.size(0) == n_token * topk, what,
              ": permuted_grad must have n_token * topk rows");
  check_maps(what, inv, eft, n_token * topk, permuted_grad);
  no_tangents(what, {permuted_grad});
  const c10::cuda::CUDAGuard guard(permuted_grad.device());
  const Tensor g = aligned(permuted_grad);
  Tensor out = empty({n_token, g.size(1)}, g, g.scalar_type());
  check(lib.moe_permute_backward(g.data_ptr(), type_of(g), ints(inv), offsets(eft), experts(eft),
                                 n_token, topk, g.size(1), out.data_ptr(), stream_of(g)),
        what);
  return out;
}

std::tuple<Tensor, Tensor> moe_unpermute_backward(const Tensor& out_grad, const Tensor& rows,
                                                  const Tensor& weights, const Tensor& inv,
                                                  const optional<Tensor>& eft) {
  const char* what = "moe_unpermute_backward";
  check_rows(what, "permuted_hidden_states", rows);
  TORCH_CHECK(weights.dim() == 2 && weights.scalar_type() == at::kFloat &&
                  weights.device() == rows.device(),
              what, ": topk_weights must be float32 [n_token, topk]");
  const int64_t n_token = weights.size(0), topk = weights.size(1);
  TORCH_CHECK(topk >= 1 && rows.size(0) == n_token * topk, what,
              ": permuted_hidden_states must have n_token * topk rows");
  TORCH_CHECK(out_grad.dim() == 2 && out_grad.size(0) == n_token &&
                  out_grad.size(1) == rows.size(1) &&
                  out_grad.scalar_type() == rows.scalar_type() &&
                  out_grad.device() == rows.device(),
              what, ": out_grad must be [n_token, hidden] of permuted_hidden_states' dtype");
  check_maps(what, inv, eft, n_token * topk, rows);
  no_tangents(what, {out_grad, rows, weights});
  const c10::cuda::CUDAGuard guard(rows.device());
  const Tensor g = aligned(out_grad), y = aligned(rows), w = weights.contiguous();
  Tensor dy = empty(y.sizes(), y, y.scalar_type()), dw = empty(w.sizes(), w, at::kFloat);
  check(lib.moe_unpermute_backward(g.data_ptr(), y.data_ptr(), type_of(y),
                                   static_cast<const float*>(w.data_ptr()), ints(inv),
                                   offsets(eft), experts(eft), n_token, topk, y.size(1),
                                   dy.data_ptr(), static_cast<float*>(dw.data_ptr()),
                                   stream_of(y)),
        what);
  return {dy, dw};
}

struct SortRows : torch::autograd::Function<SortRows> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& ids,
                               const optional<Tensor>& emap, int64_t n_expert, int64_t n_local) {
    const c10::cuda::CUDAGuard guard(x.device());
    const int64_t n_token = ids.size(0), topk = ids.size(1), n = n_token * topk;
    Tensor eft = empty({n_local + 1}, x, at::kLong), inv = empty({n}, x, at::kInt);
    Tensor pidx = empty({n}, x, at::kInt), rows = empty({n, x.size(1)}, x, x.scalar_type());
    const size_t bytes = lib.route_workspace_size(n, n_expert);
    Tensor workspace = empty({static_cast<int64_t>(bytes)}, x, at::kByte);
    check(lib.moe_permute_metadata(
              ints(ids), nullptr, emap ? ints(*emap) : nullptr, n_token, topk, n_expert, n_local,
              static_cast<int64_t*>(eft.data_ptr()), static_cast<int32_t*>(inv.data_ptr()),
              static_cast<int32_t*>(pidx.data_ptr()), workspace.data_ptr(), bytes, stream_of(x)),
          "moe_permute_train");
    check(lib.moe_scatter_rows(x.data_ptr(), type_of(x), ints(inv),
                               static_cast<const int64_t*>(eft.data_ptr()), n_local, n_token, topk,
                               x.size(1), rows.data_ptr(), stream_of(x)),
          "moe_permute_train");
    ctx->save_for_backward({eft, inv});
    ctx->saved_data["n_token"] = n_token;
    ctx->saved_data["topk"] = topk;
    ctx->mark_non_differentiable({eft, inv, pidx});
    ctx->set_materialize_grads(false);
    return {rows, eft, inv, pidx};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("moe_permute_train");
    Tensor dx;
    if (grads[0].defined()) {
      const variable_list saved = ctx->get_saved_variables();
      dx = moe_permute_backward(grads[0], saved[1], saved[0], ctx->saved_data["n_token"].toInt(),
                                ctx->saved_data["topk"].toInt());
    }
    return {dx, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

struct ReturnRows : torch::autograd::Function<ReturnRows> {
  static Tensor forward(AutogradContext* ctx, const Tensor& rows, const Tensor& weights,
                        const Tensor& inv, const optional<Tensor>& eft) {
    const c10::cuda::CUDAGuard guard(rows.device());
    Tensor out = empty({weights.size(0), rows.size(1)}, rows, rows.scalar_type());
    check(lib.moe_unpermute_rows(rows.data_ptr(), rows.size(0), type_of(rows),
                                 static_cast<const float*>(weights.data_ptr()), ints(inv),
                                 offsets(eft), experts(eft), weights.size(0), weights.size(1),
                                 rows.size(1), out.data_ptr(), stream_of(rows)),
          "moe_unpermute_train");
    ctx->save_for_backward({rows, weights, inv, eft ? *eft : Tensor()});
    ctx->set_materialize_grads(false);
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("moe_unpermute_train");
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const variable_list saved = ctx->get_saved_variables();
    const auto [dy, dw] =
        moe_unpermute_backward(grads[0], saved[0], saved[1], saved[2], some(saved[3]));
    return {ctx->needs_input_grad(0) ? dy : Tensor(), ctx->needs_input_grad(1) ? dw : Tensor(),
            Tensor(), Tensor()};
  }
};

std::tuple<Tensor, Tensor, Tensor, Tensor> moe_permute_train(const Tensor& x, const Tensor& ids,
                                                             int64_t n_expert, int64_t n_local,
                                                             const optional<Tensor>& emap) {
  const char* what = "moe_permute_train";
  check_rows(what, "hidden_states", x);
  TORCH_CHECK(ids.dim() == 2 && ids.size(0) == x.size(0) && ids.size(1) >= 1 &&
                  ids.device() == x.device(),
              what, ": topk_ids must have shape [n_token, topk] on hidden_states' device");
  TORCH_CHECK(at::isIntegralType(ids.scalar_type(), false), what, ": topk_ids must be integers");
  if (n_local == -1) n_local = n_expert;
  TORCH_CHECK(n_expert >= 1 && n_expert <= 2048 && n_local >= 0 && n_local <= n_expert, what,
              ": n_expert must be in [1, 2048] and n_local_expert in [0, n_expert]");
  if (emap)
    TORCH_CHECK(emap->scalar_type() == at::kInt && emap->is_contiguous() &&
                    emap->device() == x.device() && emap->dim() == 1 && emap->size(0) == n_expert,
                what,
                ": expert_map must be contiguous int32 [n_expert] on hidden_states' device");
  no_tangents(what, {x});
  if (at::GradMode::is_enabled()) check_capture(what, {x});
  const variable_list out =
      SortRows::apply(aligned(x), ids.to(at::kInt).contiguous(), emap, n_expert, n_local);
  return {out[0], out[1], out[2], out[3]};
}

Tensor moe_unpermute_train(const Tensor& rows, const Tensor& weights, const Tensor& inv,
                           const optional<Tensor>& eft) {
  const char* what = "moe_unpermute_train";
  check_rows(what, "permuted_hidden_states", rows);
  TORCH_CHECK(weights.dim() == 2 && weights.size(1) >= 1 && weights.device() == rows.device() &&
                  rows.size(0) == weights.numel(),
              what,
              ": permuted_hidden_states must have one row per element of topk_weights "
              "[n_token, topk]");
  check_maps(what, inv, eft, weights.numel(), rows);
  no_tangents(what, {rows, weights});
  if (at::GradMode::is_enabled()) check_capture(what, {rows, weights});
  return ReturnRows::apply(aligned(rows), weights.to(at::kFloat).contiguous(), inv, eft);
}

// ---------------------------------------------------------- 4-bit products

// Whether the contiguous `out` has bytes of a row of x (rows of stride(0) >=
// size(1) elements); torch's own check gives up on rows with gaps.
bool rows_meet(const Tensor& x, const Tensor& out) {
  if (x.numel() == 0 || out.numel() == 0) return false;
  const int64_t row = x.size(1) * x.element_size(), step = x.stride(0) * x.element_size();
  const auto start = reinterpret_cast<intptr_t>(x.data_ptr());
  const int64_t o0 = reinterpret_cast<intptr_t>(out.data_ptr()) - start;
  const int64_t o1 = o0 + out.numel() * out.element_size();
  if (o1 <= 0) return false;
  // the first row that ends behind out's start
  const int64_t r = o0 < row || step == 0 ? 0 : (o0 - row) / step + 1;
  return r < x.size(0) && r * step < o1 && r * step + row > o0;
}

Tensor int4_grouped_mv(const Tensor& x_in, const Tensor& packed, const Tensor& scale,
                       const Tensor& eo, int64_t group, const optional<Tensor>& pidx, int64_t topk,
                       bool silu, const optional<Tensor>& out_in) {
  const char* what = "int4_grouped_mv";
  TORCH_CHECK(x_in.is_cuda() && x_in.dim() == 2, what, ": x must be a CUDA tensor [rows, K]");
  TORCH_CHECK(x_in.scalar_type() == at::kBFloat16 || x_in.scalar_type() == at::kHalf, what,
              ": x must be bfloat16 or float16");
  const auto device = x_in.device();
  TORCH_CHECK(packed.scalar_type() == at::kByte && packed.dim() == 3 && packed.is_contiguous() &&
                  packed.device() == device,
              what, ": w_packed must be contiguous uint8 [E, N, K/2] on x's device");
  const int64_t E = packed.size(0), N = packed.size(1), K = 2 * packed.size(2);
  TORCH_CHECK(group == 32 || group == 64 || group == 128, what,
              ": group_size must be 32, 64 or 128");
  TORCH_CHECK(x_in.size(1) == K, what, ": x.shape[1] must be twice w_packed.shape[2]");
  TORCH_CHECK(K >= 32 && K % 32 == 0, what, ": K must be positive and divisible by 32");
  TORCH_CHECK(scale.scalar_type() == x_in.scalar_type(), what, ": w_scale must have x's dtype");
  TORCH_CHECK(scale.dim() == 3 && scale.size(0) == E && scale.size(1) == N &&
                  scale.size(2) == (K + group - 1) / group && scale.is_contiguous() &&
                  scale.device() == device,
              what, ": w_scale must be contiguous [E, N, ceil(K / group_size)] on x's device");
  TORCH_CHECK(eo.scalar_type() == at::kInt && eo.dim() == 1 && eo.size(0) == E + 1 &&
                  eo.is_contiguous() && eo.device() == device,
              what, ": expert_offsets must be contiguous int32 [E + 1] on x's device");
  TORCH_CHECK(!silu || N % 2 == 0, what, ": N must be even with silu");
  int64_t rows = x_in.size(0);
  if (pidx) {
    TORCH_CHECK(pidx->scalar_type() == at::kInt && pidx->dim() == 1 && pidx->is_contiguous() &&
                    pidx->device() == device,
                what, ": permuted_idx must be contiguous int32 [rows] on x's device");
    TORCH_CHECK(topk >= 1, what, ": topk must be positive");
    rows = pidx->size(0);
  }
  TORCH_CHECK(!(at::GradMode::is_enabled() && (x_in.requires_grad() || scale.requires_grad())),
              what, " has no gradient: call it under torch.no_grad()");
  no_tangents(what, {x_in, scale});
  const c10::cuda::CUDAGuard guard(device);
  const int64_t n_out = silu ? N / 2 : N;
  Tensor out;
  if (out_in) {
    out = *out_in;
    TORCH_CHECK(out.scalar_type() == x_in.scalar_type() && out.dim() == 2 && out.size(0) == rows &&
                    out.size(1) == n_out && out.is_contiguous() && out.device() == device,
                what,
                ": out must be contiguous [rows, N (N/2 with silu)] of x's dtype on x's device");
    for (const Tensor& t : {x_in, packed, scale, eo, pidx ? *pidx : eo}) at::assert_no_overlap(out, t);
  } else {
    out = empty({rows, n_out}, x_in, x_in.scalar_type());
  }
  const bool in_place =
      x_in.stride(1) == 1 &&
      (x_in.size(0) < 2 || (x_in.stride(0) % 8 == 0 && x_in.stride(0) >= K)) &&
      reinterpret_cast<uintptr_t>(x_in.data_ptr()) % 16 == 0;
  const Tensor x = in_place ? x_in : aligned(x_in);
  TORCH_CHECK(!out_in || !rows_meet(x, out), what,
              ": x and out refer to a single memory location in some elements");
  check(lib.int4_grouped_mv(x.data_ptr(), x.size(0) < 2 ? K : x.stride(0), x.size(0), type_of(x),
                            pidx ? ints(*pidx) : nullptr, topk,
                            static_cast<const uint8_t*>(packed.data_ptr()), scale.data_ptr(), group,
                            ints(eo), E, rows, N, K, silu ? 1 : 0, out.data_ptr(), stream_of(x)),
        what);
  return out;
}

}  // namespace

PYBIND11_MODULE(_torch_ops, m) {
  m.attr("torch_version") = TORCH_VERSION;
  m.def("bind", &bind);
  m.def("rms_norm", &rms_norm);
  m.def("rms_norm_quant_int8", &rms_norm_quant_int8);
  m.def("rms_norm_backward", &rms_norm_backward);
  m.def("moe_permute_train", &moe_permute_train);
  m.def("moe_unpermute_train", &moe_unpermute_train);
  m.def("moe_permute_backward", &moe_permute_backward);
  m.def("moe_unpermute_backward", &moe_unpermute_backward);
  m.def("int4_grouped_mv", &int4_grouped_mv);
}
