// Host path of the gated delta rule (include/mvm_delta.h): the autograd Function
// of the packed form, and the calls that advance a cache of states in place.
// Part of torch_ext.cpp's one translation unit.
#pragma once

#include "mvm_delta.h"
#include "torch_seq.h"

namespace {

struct DeltaFlags {
  std::optional<double> scale;
  bool l2;
  int64_t max_len, split_len;
};

// operands as the kernels take them, with their descriptor
struct DeltaArgs {
  Tensor q, k, v, g, beta;
  Seqs seqs;
  mvm_delta_desc d{};
};

// (T, H, D) rows with a contiguous last dimension; a copy only where the layout has no such view
Tensor as_heads(const Tensor& t) {
  Tensor r = t.dim() == 4 ? t.reshape({t.size(0) * t.size(1), t.size(2), t.size(3)}) : t;
  return r.size(2) > 1 && r.stride(2) != 1 ? r.contiguous() : r;
}
// (a single row's, or head's, stride is never walked)
int64_t token_stride(const Tensor& r) { return r.size(0) > 1 ? r.stride(0) : r.size(1) * r.size(2); }
int64_t head_stride(const Tensor& r) { return r.size(1) > 1 ? r.stride(1) : r.size(2); }

DeltaArgs delta_args(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta,
                     const Tensor& off, bool step, const DeltaFlags& fl) {
  const auto t = q.scalar_type();
  if (!is_act(t)) bad_value(std::string("q must be float32 or bfloat16; got ") + c10::toString(t));
  const bool rows = step || off.defined();
  if (q.dim() != (rows ? 3 : 4))
    bad_value(std::string("q must be ") + (step ? "(S, H, D), one token for each sequence" : rows ? "(T, H, D) with offsets" : "(B, L, H, D) without offsets") +
              "; got " + shape_str(q));
  if (k.sizes() != q.sizes()) bad_value("k must have q's shape " + shape_str(q) + "; got " + shape_str(k));
  if (v.dim() != q.dim() || v.sizes().slice(0, q.dim() - 2) != q.sizes().slice(0, q.dim() - 2))
    bad_value("v must be q's rows of (value heads, D); got " + shape_str(v) + " for q " + shape_str(q));
  const int64_t hk = q.size(-2), hv = v.size(-2), dk = q.size(-1), dv = v.size(-1);
  if (hk < 1 || hv < 1 || hv % hk != 0)
    bad_value("v's heads must be a multiple of q's and k's; got " + std::to_string(hv) + " and " + std::to_string(hk));
  if (dk < 1 || dk > MVM_DELTA_MAX_DK || dv < 1 || dv > MVM_DELTA_MAX_DV)
    bad_value("head sizes of 1.." + std::to_string(MVM_DELTA_MAX_DK) + " (q, k) and 1.." +
              std::to_string(MVM_DELTA_MAX_DV) + " (v) are supported; got " + std::to_string(dk) + " and " +
              std::to_string(dv));
  const auto per_head = v.sizes().slice(0, v.dim() - 1);
  if (g.sizes() != per_head || beta.sizes() != per_head)
    bad_value("g and beta must be v's rows of value heads; got " + shape_str(g) + ", " + shape_str(beta) + " for v " +
              shape_str(v));
  if (k.scalar_type() != t || v.scalar_type() != t)
    bad_value(std::string("k and v must have q's type ") + c10::toString(t));
  if (!g.is_floating_point() || (beta.scalar_type() != t && beta.scalar_type() != at::kFloat))
    bad_value(std::string("g must be floating and beta float32 or of q's type ") + c10::toString(t));
  if (off.defined() && (off.scalar_type() != at::kInt || off.dim() != 1 || off.size(0) < 1 || !off.is_contiguous()))
    bad_value("offsets must be a contiguous int32 tensor of S + 1 elements; got " + shape_str(off));
  check_device({&q, &k, &v, &g, &beta, &off});
  DeltaArgs a;
  if (off.defined())
    a.seqs = {q.size(0), off.size(0) - 1, 0, 0, off};
  else if (step)
    a.seqs = {q.size(0), q.size(0), 1, 0, Tensor()};
  else
    a.seqs = {q.size(0) * q.size(1), q.size(0), q.size(1), 0, Tensor()};
  a.q = as_heads(q);
  a.k = as_heads(k);
  a.v = as_heads(v);
  a.g = as_rows(g.to(at::kFloat));
  a.beta = as_rows(beta);
  a.d.key_heads = hk;
  a.d.value_heads = hv;
  a.d.dk = dk;
  a.d.dv = dv;
  a.d.q_stride = token_stride(a.q);
  a.d.q_stride_head = head_stride(a.q);
  a.d.k_stride = token_stride(a.k);
  a.d.k_stride_head = head_stride(a.k);
  a.d.v_stride = token_stride(a.v);
  a.d.v_stride_head = head_stride(a.v);
  a.d.g_stride = row_stride(a.g);
  a.d.beta_stride = row_stride(a.beta);
  a.d.max_len = fl.max_len;
  a.d.scale = static_cast<float>(fl.scale.value_or(1.0 / std::sqrt(static_cast<double>(dk))));
  a.d.dtype = type_code(t);
  a.d.beta_dtype = type_code(beta.scalar_type());
  a.d.qk_l2norm = fl.l2;
  a.d.split_len = static_cast<int32_t>(fl.split_len);
  return a;
}

// o in v's shape; ckpt is allocated when asked for
Tensor delta_launch(const DeltaArgs& a, at::IntArrayRef shape, const Tensor& h0, const Tensor& h1, Tensor* ckpt) {
  c10::OptionalDeviceGuard guard(a.q.device());
  Tensor o = empty_like_opts(shape, a.q, a.q.scalar_type());
  if (ckpt != nullptr) *ckpt = empty_like_opts({check(mvm_delta_ckpt_elems(&a.d))}, a.q);
  const int64_t nbytes = check(mvm_delta_workspace_bytes(&a.d, 0));
  const Tensor ws = workspace(nbytes, a.q);
  check(mvm_delta_fwd(&a.d, vp(a.q), vp(a.k), vp(a.v), fp(a.g), vp(a.beta), fp(h0), fpm(h1), vpm(o),
                      ckpt != nullptr ? fpm(*ckpt) : nullptr, ws.mutable_data_ptr(), static_cast<size_t>(nbytes),
                      stream_of(a.q)));
  return o;
}

// The states' rows of a call's operands
std::vector<int64_t> delta_rows(const DeltaArgs& a, int64_t rows) {
  return {rows, a.d.value_heads, a.d.dk, a.d.dv};
}

struct DeltaFn : Function<DeltaFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                               const Tensor& g, const Tensor& beta, const OptTensor& h0_, const OptTensor& off_,
                               std::optional<double> scale, bool l2, int64_t max_len, int64_t split_len, bool needs) {
    const Tensor h0 = h0_.value_or(Tensor()), off = off_.value_or(Tensor());
    DeltaArgs a = delta_args(q, k, v, g, beta, off, false, {scale, l2, max_len, split_len});
    const auto rows = delta_rows(a, a.seqs.nseq);
    if (h0.defined() && h0.sizes() != rows)
      bad_value("initial_states must be (" + std::to_string(rows[0]) + ", " + std::to_string(rows[1]) + ", " +
                std::to_string(rows[2]) + ", " + std::to_string(rows[3]) + "); got " + shape_str(h0));
    if (h0.defined()) check_device({&q, &h0});
    a.d.seq = seq_desc(a.seqs, a.seqs.nseq, Tensor(), Tensor());
    Tensor h1 = empty_like_opts(rows, q), ckpt;
    Tensor o = delta_launch(a, v.sizes(), f32(h0), h1, needs ? &ckpt : nullptr);
    ctx->set_materialize_grads(false);
    ctx->saved_data["scale"] = static_cast<double>(a.d.scale);
    ctx->saved_data["flags"] =
        std::vector<int64_t>{l2, max_len, split_len, h0.defined() ? static_cast<int64_t>(h0.scalar_type()) : -1};
    if (needs) ctx->save_for_backward({q, k, v, g, beta, ckpt, off});
    return {o, h1};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    return in_backward([&] { return grads(ctx, g); });
  }
  static variable_list grads(AutogradContext* ctx, const variable_list& go) {
    const auto sv = ctx->get_saved_variables();
    const auto fl = ctx->saved_data["flags"].toIntVector();
    variable_list out(12);
    if (!go[0].defined() && !go[1].defined()) return out;
    {
      at::NoGradGuard no_grad;
      const Tensor &q = sv[0], &k = sv[1], &v = sv[2], &g = sv[3], &beta = sv[4];
      DeltaArgs a = delta_args(q, k, v, g, beta, sv[6], false,
                               {ctx->saved_data["scale"].toDouble(), fl[0] != 0, fl[1], fl[2]});
      a.d.seq = seq_desc(a.seqs, a.seqs.nseq, Tensor(), Tensor());
      c10::OptionalDeviceGuard guard(q.device());
      check_captured_edges(q, "the gated delta rule");
      const Tensor d_o = go[0].defined() ? go[0].to(v.scalar_type()).contiguous() : at::zeros(v.sizes(), a.v.options());
      const Tensor dh1 = f32(go[1]);
      const auto like = [&](const Tensor& t) { return empty_like_opts(t.sizes(), t, t.scalar_type()); };
      Tensor dq = like(q), dk = like(k), dv = like(v), dg = empty_like_opts(g.sizes(), q), db = like(beta), dh0;
      if (fl[3] >= 0) dh0 = empty_like_opts(delta_rows(a, a.seqs.nseq), q);
      const int64_t nbytes = check(mvm_delta_workspace_bytes(&a.d, 1));
      const Tensor ws = workspace(nbytes, q);
      check(mvm_delta_bwd(&a.d, vp(a.q), vp(a.k), vp(a.v), fp(a.g), vp(a.beta), fp(sv[5]), vp(d_o), fp(dh1), vpm(dq),
                          vpm(dk), vpm(dv), fpm(dg), vpm(db), fpm(dh0), ws.mutable_data_ptr(),
                          static_cast<size_t>(nbytes), stream_of(q)));
      out[0] = dq; out[1] = dk; out[2] = dv; out[3] = dg.to(g.scalar_type()); out[4] = db;
      if (fl[3] >= 0) out[5] = dh0.to(static_cast<at::ScalarType>(fl[3]));
    }
    return once_differentiable(std::move(out), go, "the gated delta rule");
  }
};

std::pair<Tensor, Tensor> delta(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g,
                                const Tensor& beta, const OptTensor& h0, const OptTensor& off,
                                std::optional<double> scale, bool l2, int64_t max_len, int64_t split_len) {
  return guarded([&]() -> std::pair<Tensor, Tensor> {
    bool needs = h0.has_value() && h0->requires_grad();
    for (const Tensor* t : {&q, &k, &v, &g, &beta}) needs = needs || t->requires_grad();
    const auto out = DeltaFn::apply(q, k, v, g, beta, h0, off, scale, l2, max_len, split_len,
                                    needs && at::GradMode::is_enabled());
    return {out[0], out[1]};
  });
}

void check_delta_cache(const DeltaArgs& a, const Tensor& states, const Tensor& slots, const Tensor& fresh) {
  const auto rows = delta_rows(a, 0);
  if (states.dim() != 4 || states.sizes().slice(1) != at::IntArrayRef(rows).slice(1) ||
      states.scalar_type() != at::kFloat || !states.is_contiguous())
    bad_value("states must be a contiguous float32 (rows, " + std::to_string(rows[1]) + ", " + std::to_string(rows[2]) +
              ", " + std::to_string(rows[3]) + ") tensor; got " + shape_str(states) + " of " +
              c10::toString(states.scalar_type()));
  check_cache(a.seqs, states.flatten(2), {rows[1], rows[2] * rows[3]}, at::kFloat, slots, fresh);
}

Tensor delta_prefill(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta,
                     const Tensor& states, const OptTensor& off_, const OptTensor& slots_, const OptTensor& fresh_,
                     std::optional<double> scale, bool l2, int64_t max_len, int64_t split_len) {
  return guarded([&] {
    at::NoGradGuard no_grad;
    const Tensor off = off_.value_or(Tensor()), slots = slots_.value_or(Tensor()), fresh = fresh_.value_or(Tensor());
    DeltaArgs a = delta_args(q, k, v, g, beta, off, false, {scale, l2, max_len, split_len});
    check_delta_cache(a, states, slots, fresh);
    check_device({&q, &states, &slots, &fresh});
    a.d.seq = seq_desc(a.seqs, states.size(0), slots, fresh);
    const Tensor o = delta_launch(a, v.sizes(), states, states, nullptr);
    wrote(states);
    return o;
  });
}

Tensor delta_step(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta,
                  const Tensor& states, const OptTensor& slots_, std::optional<double> scale, bool l2) {
  return guarded([&] {
    at::NoGradGuard no_grad;
    const Tensor slots = slots_.value_or(Tensor());
    DeltaArgs a = delta_args(q, k, v, g, beta, Tensor(), true, {scale, l2, 0, 0});
    check_delta_cache(a, states, slots, Tensor());
    check_device({&q, &states, &slots});
    a.d.seq = seq_desc(a.seqs, states.size(0), slots, Tensor());
    c10::OptionalDeviceGuard guard(q.device());
    Tensor o = empty_like_opts(v.sizes(), q, q.scalar_type());
    check(mvm_delta_step(&a.d, vp(a.q), vp(a.k), vp(a.v), fp(a.g), vp(a.beta), fpm(states), vpm(o), stream_of(q)));
    wrote(states);
    return o;
  });
}

}  // namespace
