// Host path of the group norm (include/mvm_group_norm.h).  Part of
// torch_ext.cpp's one translation unit.
#pragma once

#include "mvm_group_norm.h"
#include "torch_seq.h"

namespace {

// (N, ..., C) as rows of contiguous channels, a stride apart; a copy only where the layout has no such view
Tensor as_channel_rows(const Tensor& t) {
  const Tensor r = t.reshape({-1, t.size(-1)});
  return r.size(1) > 1 && r.stride(1) != 1 ? r.contiguous() : r;
}

struct GroupNormFn : Function<GroupNormFn> {
  static mvm_group_norm_desc desc(const Tensor& x, const Tensor& rows, const Tensor& zrows, int64_t groups, double eps,
                                  bool silu) {
    mvm_group_norm_desc d{};
    d.batch = x.size(0);
    d.positions = rows.size(0) / std::max<int64_t>(1, x.size(0));
    d.channels = x.size(-1);
    d.groups = groups;
    d.x_stride = row_stride(rows);
    d.z_stride = zrows.defined() ? row_stride(zrows) : 0;
    d.eps = static_cast<float>(eps);
    d.dtype = type_code(x.scalar_type());
    d.silu = silu;
    return d;
  }
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& w_, const OptTensor& b_,
                               const OptTensor& z_, int64_t groups, double eps, bool silu) {
    const Tensor w = w_.value_or(Tensor()), b = b_.value_or(Tensor()), z = z_.value_or(Tensor());
    if (!is_act(x.scalar_type()))
      bad_value(std::string("x must be float32 or bfloat16; got ") + c10::toString(x.scalar_type()));
    if (x.dim() < 2) bad_value("x must be (N, ..., C); got " + shape_str(x));
    const int64_t C = x.size(-1);
    if (groups < 1 || C < 1 || C % groups != 0)
      bad_value("groups=" + std::to_string(groups) + " must divide x's " + std::to_string(C) + " channels");
    for (const Tensor* t : {&w, &b})
      if (t->defined() && t->sizes() != at::IntArrayRef({C}))
        bad_value("weight and bias must be (" + std::to_string(C) + ",); got " + shape_str(*t));
    if (z.defined() && (z.sizes() != x.sizes() || z.scalar_type() != x.scalar_type()))
      bad_value("z must have x's shape " + shape_str(x) + " and type; got " + shape_str(z) + " of " +
                c10::toString(z.scalar_type()));
    if (!(eps >= 0)) bad_value("eps must be >= 0");
    check_device({&x, &w, &b, &z});
    c10::OptionalDeviceGuard guard(x.device());
    Tensor y = empty_like_opts(x.sizes(), x, x.scalar_type());
    Tensor stats = empty_like_opts({x.size(0), groups, 2}, x);
    if (y.numel() > 0) {
      const Tensor rows = as_channel_rows(x), zrows = z.defined() ? as_channel_rows(z) : z, wf = f32(w), bf = f32(b);
      const auto d = desc(x, rows, zrows, groups, eps, silu);
      const int64_t nbytes = check(mvm_group_norm_workspace_bytes(&d, 0));
      const Tensor ws = workspace(nbytes, x);
      check(mvm_group_norm_fwd(&d, vp(rows), fp(wf), fp(bf), vp(zrows), vpm(y), fpm(stats), ws.mutable_data_ptr(),
                               static_cast<size_t>(nbytes), stream_of(x)));
    }
    ctx->save_for_backward({x, w, b, z, stats});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["silu"] = silu;
    return {y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    return in_backward([&] { return once_differentiable(grads(ctx, g), g, "the group norm"); });
  }
  static variable_list grads(AutogradContext* ctx, const variable_list& g) {
    at::NoGradGuard no_grad;
    const auto sv = ctx->get_saved_variables();
    const Tensor &x = sv[0], &w = sv[1], &b = sv[2], &z = sv[3];
    c10::OptionalDeviceGuard guard(x.device());
    check_captured_edges(x, "the group norm");
    const Tensor dy = g[0].to(x.scalar_type()).contiguous();
    Tensor dx = empty_like_opts(x.sizes(), x, x.scalar_type()), dw, db, dz;
    if (w.defined()) dw = empty_like_opts(w.sizes(), x);
    if (b.defined()) db = empty_like_opts(b.sizes(), x);
    if (z.defined()) dz = empty_like_opts(z.sizes(), z, z.scalar_type());
    if (dx.numel() > 0) {
      const Tensor rows = as_channel_rows(x), zrows = z.defined() ? as_channel_rows(z) : z, wf = f32(w), bf = f32(b);
      const auto d = desc(x, rows, zrows, ctx->saved_data["groups"].toInt(), ctx->saved_data["eps"].toDouble(),
                          ctx->saved_data["silu"].toBool());
      const int64_t nbytes = check(mvm_group_norm_workspace_bytes(&d, 1));
      const Tensor ws = workspace(nbytes, x);
      check(mvm_group_norm_bwd(&d, vp(rows), fp(wf), fp(bf), vp(zrows), fp(sv[4]), vp(dy), vpm(dx), fpm(dw), fpm(db),
                               vpm(dz), ws.mutable_data_ptr(), static_cast<size_t>(nbytes), stream_of(x)));
    } else {
      for (Tensor* t : {&dw, &db})
        if (t->defined()) t->zero_();
    }
    return {dx, w.defined() ? dw.to(w.scalar_type()) : dw, b.defined() ? db.to(b.scalar_type()) : db, dz, Tensor(),
            Tensor(), Tensor()};
  }
};

Tensor group_norm(const Tensor& x, int64_t groups, const OptTensor& w, const OptTensor& b, double eps, bool silu,
                  const OptTensor& z) {
  return guarded([&] { return GroupNormFn::apply(x, w, b, z, groups, eps, silu)[0]; });
}

}  // namespace
