// Host path of the packed and served scan and conv (include/mvm_seq.h): the
// autograd Functions of the packed forms, and the calls that advance a cache of
// states in place.  Part of torch_ext.cpp's one translation unit.
#pragma once

#include "mvm_conv.h"
#include "mvm_seq.h"
#include "torch_host.h"

namespace {

// ---------------------------------------------------------------- sequences

bool is_act(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16; }
int32_t type_code(at::ScalarType t) { return t == at::kBFloat16 ? MVM_BF16 : MVM_F32; }

// (T, cols) or (B, L, cols) as rows of contiguous columns; a copy only where
// the layout has no such view
Tensor as_rows(const Tensor& t) {
  Tensor r = t.dim() == 3 ? t.reshape({t.size(0) * t.size(1), t.size(2)}) : t;
  return r.size(1) > 1 && r.stride(1) != 1 ? r.contiguous() : r;
}
// (a single row's stride is never walked)
int64_t row_stride(const Tensor& r) { return r.size(0) > 1 ? r.stride(0) : r.size(1); }

// The cut into sequences of an x of (T, D) with offsets (S + 1) or (B, L, D)
// without, or (S, D) in a step
struct Seqs {
  int64_t tokens, nseq, seqlen, dim;
  Tensor off;
};
Seqs seqs_of(const char* name, const Tensor& x, const Tensor& off) {
  if (!is_act(x.scalar_type()))
    bad_value(std::string(name) + " must be float32 or bfloat16; got " + c10::toString(x.scalar_type()));
  if (off.defined()) {
    if (x.dim() != 2) bad_value(std::string(name) + " must be (T, D) with offsets; got " + shape_str(x));
    if (off.scalar_type() != at::kInt || off.dim() != 1 || off.size(0) < 1 || !off.is_contiguous())
      bad_value("offsets must be a contiguous int32 tensor of S + 1 elements; got " + shape_str(off));
    return {x.size(0), off.size(0) - 1, 0, x.size(1), off};
  }
  if (x.dim() != 3) bad_value(std::string(name) + " must be (B, L, D) without offsets; got " + shape_str(x));
  return {x.size(0) * x.size(1), x.size(0), x.size(1), x.size(2), off};
}
Seqs step_seqs(const char* name, const Tensor& x) {
  if (!is_act(x.scalar_type()))
    bad_value(std::string(name) + " must be float32 or bfloat16; got " + c10::toString(x.scalar_type()));
  if (x.dim() != 2) bad_value(std::string(name) + " must be (S, D), one token for each sequence; got " + shape_str(x));
  return {x.size(0), x.size(0), 1, x.size(1), Tensor()};
}

mvm_seq_desc seq_desc(const Seqs& q, int64_t state_rows, const Tensor& slots, const Tensor& fresh) {
  mvm_seq_desc d{};
  d.tokens = q.tokens; d.nseq = q.nseq; d.seqlen = q.seqlen; d.dim = q.dim;
  d.state_rows = state_rows;
  d.offsets = q.off.defined() ? static_cast<const int32_t*>(q.off.const_data_ptr()) : nullptr;
  d.slots = slots.defined() ? static_cast<const int32_t*>(slots.const_data_ptr()) : nullptr;
  d.fresh = fresh.defined() ? static_cast<const uint8_t*>(fresh.const_data_ptr()) : nullptr;
  return d;
}

// A cache that a call advances: checked, since it cannot be copied
void check_cache(const Seqs& q, const Tensor& states, at::IntArrayRef row, at::ScalarType type, const Tensor& slots,
                 const Tensor& fresh) {
  if (states.dim() != 3 || states.sizes().slice(1) != row || states.scalar_type() != type || !states.is_contiguous())
    bad_value("states must be a contiguous (rows, " + std::to_string(row[0]) + ", " + std::to_string(row[1]) +
              ") tensor of " + c10::toString(type) + "; got " + shape_str(states) + " of " +
              c10::toString(states.scalar_type()));
  if (states.requires_grad()) bad_value("states is advanced in place and must not require a gradient");
  if (slots.defined() && (slots.scalar_type() != at::kInt || slots.dim() != 1 || slots.size(0) != q.nseq ||
                          !slots.is_contiguous()))
    bad_value("slots must be a contiguous int32 tensor of " + std::to_string(q.nseq) + " elements; got " +
              shape_str(slots));
  if (!slots.defined() && states.size(0) < q.nseq)
    bad_value("states has " + std::to_string(states.size(0)) + " rows for " + std::to_string(q.nseq) + " sequences");
  if (fresh.defined() && (fresh.scalar_type() != at::kBool || fresh.dim() != 1 || fresh.size(0) != q.nseq ||
                          !fresh.is_contiguous()))
    bad_value("fresh must be a contiguous bool tensor of " + std::to_string(q.nseq) + " elements; got " +
              shape_str(fresh));
}
void wrote(const Tensor& states) {
  if (!states.is_inference()) states.unsafeGetTensorImpl()->bump_version();
}

Tensor f32(const Tensor& t) { return t.defined() ? t.to(at::kFloat).contiguous() : t; }
const void* vp(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* vpm(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
OptTensor maybe(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }

// --------------------------------------------------------------------- scan

struct SeqScanFlags {
  bool softplus, a_is_log;
  int64_t max_len, chunk_len;
};

// operands as the kernels take them, with their descriptor
struct SeqScanArgs {
  Tensor u, delta, A, Bm, Cm, Dv, z, dbias;
  mvm_seq_scan_desc d{};
};
SeqScanArgs scan_args(const Seqs& q, const Tensor& u, const Tensor& delta, const Tensor& A, const Tensor& Bm,
                      const Tensor& Cm, const Tensor& Dv, const Tensor& z, const Tensor& dbias,
                      const SeqScanFlags& fl) {
  if (delta.sizes() != u.sizes() || (z.defined() && z.sizes() != u.sizes()))
    bad_value("delta and z must have u's shape " + shape_str(u) + "; got " + shape_str(delta) +
              (z.defined() ? " and " + shape_str(z) : ""));
  if (A.dim() != 2 || A.size(0) != q.dim)
    bad_value("A must be (D=" + std::to_string(q.dim) + ", N); got " + shape_str(A));
  const int64_t N = A.size(1);
  if (N < 1 || N > MVM_MAX_DSTATE)
    bad_value("d_state=" + std::to_string(N) + " unsupported (1.." + std::to_string(MVM_MAX_DSTATE) + ")");
  auto bc = u.sizes().vec();
  bc.back() = N;
  if (Bm.sizes() != bc || Cm.sizes() != bc)
    bad_value("B and C must be u's rows of N=" + std::to_string(N) + " states; got " + shape_str(Bm) + ", " +
              shape_str(Cm));
  if (Dv.sizes() != at::IntArrayRef({q.dim}) || (dbias.defined() && dbias.sizes() != at::IntArrayRef({q.dim})))
    bad_value("D and delta_bias must be (D=" + std::to_string(q.dim) + ",)");
  const auto t = u.scalar_type();
  if (Bm.scalar_type() != t || Cm.scalar_type() != t || (z.defined() && z.scalar_type() != t))
    bad_value(std::string("B, C and z must have u's type ") + c10::toString(t));
  if (delta.scalar_type() != t && delta.scalar_type() != at::kFloat)
    bad_value(std::string("delta must be float32 or have u's type ") + c10::toString(t));
  check_device({&u, &delta, &A, &Bm, &Cm, &Dv, &z, &dbias, &q.off});
  SeqScanArgs a;
  a.u = as_rows(u);
  a.delta = as_rows(delta);
  a.Bm = as_rows(Bm);
  a.Cm = as_rows(Cm);
  if (row_stride(a.Bm) != row_stride(a.Cm)) {
    a.Bm = a.Bm.contiguous();
    a.Cm = a.Cm.contiguous();
  }
  if (z.defined()) a.z = as_rows(z);
  a.A = f32(A);
  a.Dv = f32(Dv);
  a.dbias = f32(dbias);
  a.d.dstate = N;
  a.d.u_stride = row_stride(a.u);
  a.d.delta_stride = row_stride(a.delta);
  a.d.bc_stride = row_stride(a.Bm);
  a.d.y_stride = q.dim;
  a.d.z_stride = a.z.defined() ? row_stride(a.z) : 0;
  a.d.dtype = type_code(t);
  a.d.delta_dtype = type_code(delta.scalar_type());
  a.d.delta_softplus = fl.softplus;
  a.d.a_is_log = fl.a_is_log;
  a.d.max_len = fl.max_len;
  a.d.chunk_len = static_cast<int32_t>(fl.chunk_len);
  return a;
}

// y in u's shape; ckpt is allocated when asked for
Tensor scan_launch(const SeqScanArgs& a, at::IntArrayRef shape, const Tensor& h0, const Tensor& h1, Tensor* ckpt) {
  c10::OptionalDeviceGuard guard(a.u.device());
  Tensor y = empty_like_opts(shape, a.u, a.u.scalar_type());
  if (ckpt != nullptr) *ckpt = empty_like_opts({check(mvm_seq_scan_ckpt_elems(&a.d))}, a.u);
  const int64_t nbytes = check(mvm_seq_scan_workspace_bytes(&a.d, 0));
  const Tensor ws = workspace(nbytes, a.u);
  check(mvm_seq_scan_fwd(&a.d, vp(a.u), vp(a.delta), fp(a.dbias), fp(a.A), vp(a.Bm), vp(a.Cm), fp(a.Dv), vp(a.z),
                         fp(h0), fpm(h1), vpm(y), ckpt != nullptr ? fpm(*ckpt) : nullptr, ws.mutable_data_ptr(),
                         static_cast<size_t>(nbytes), stream_of(a.u)));
  return y;
}

struct SeqScanFn : Function<SeqScanFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& u, const Tensor& delta, const Tensor& A,
                               const Tensor& Bm, const Tensor& Cm, const Tensor& Dv, const OptTensor& z_,
                               const OptTensor& dbias_, const OptTensor& h0_, const OptTensor& off_, bool softplus,
                               bool a_is_log, int64_t max_len, int64_t chunk_len, bool needs) {
    const Tensor z = z_.value_or(Tensor()), dbias = dbias_.value_or(Tensor()), h0 = h0_.value_or(Tensor()),
                 off = off_.value_or(Tensor());
    const Seqs q = seqs_of("u", u, off);
    SeqScanArgs a = scan_args(q, u, delta, A, Bm, Cm, Dv, z, dbias, {softplus, a_is_log, max_len, chunk_len});
    const std::vector<int64_t> rows = {q.nseq, q.dim, A.size(1)};
    if (h0.defined() && h0.sizes() != rows)
      bad_value("initial_states must be (" + std::to_string(rows[0]) + ", " + std::to_string(rows[1]) + ", " +
                std::to_string(rows[2]) + "); got " + shape_str(h0));
    if (h0.defined()) check_device({&u, &h0});
    a.d.seq = seq_desc(q, q.nseq, Tensor(), Tensor());
    Tensor h1 = empty_like_opts(rows, u), ckpt;
    Tensor y = scan_launch(a, u.sizes(), f32(h0), h1, needs ? &ckpt : nullptr);
    ctx->set_materialize_grads(false);
    ctx->saved_data["flags"] = std::vector<int64_t>{softplus, a_is_log, max_len, chunk_len,
                                                    h0.defined() ? static_cast<int64_t>(h0.scalar_type()) : -1};
    if (needs) ctx->save_for_backward({u, delta, A, Bm, Cm, Dv, z, dbias, ckpt, off});
    return {y, h1};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    return in_backward([&] { return grads(ctx, g); });
  }
  static variable_list grads(AutogradContext* ctx, const variable_list& g) {
    const auto sv = ctx->get_saved_variables();
    const auto fl = ctx->saved_data["flags"].toIntVector();
    variable_list out(15);
    if (!g[0].defined() && !g[1].defined()) return out;
    {
      at::NoGradGuard no_grad;
      const Tensor &u = sv[0], &delta = sv[1], &A = sv[2], &z = sv[6], &dbias = sv[7], &off = sv[9];
      const Seqs q = seqs_of("u", u, off);
      SeqScanArgs a = scan_args(q, u, delta, A, sv[3], sv[4], sv[5], z, dbias,
                                {fl[0] != 0, fl[1] != 0, fl[2], fl[3]});
      a.d.seq = seq_desc(q, q.nseq, Tensor(), Tensor());
      c10::OptionalDeviceGuard guard(u.device());
      const Tensor dy = g[0].defined() ? g[0].to(u.scalar_type()).contiguous() : at::zeros(u.sizes(), a.u.options());
      const Tensor dh1 = f32(g[1]);
      const auto like = [&](const Tensor& t) { return empty_like_opts(t.sizes(), t, t.scalar_type()); };
      Tensor du = like(u), dd = like(delta), dB = like(sv[3]), dC = like(sv[4]), dz, ddb, dh0;
      Tensor dA = empty_like_opts(A.sizes(), u), dD = empty_like_opts({q.dim}, u);
      if (z.defined()) dz = like(z);
      if (dbias.defined()) ddb = empty_like_opts({q.dim}, u);
      if (fl[4] >= 0) dh0 = empty_like_opts({q.nseq, q.dim, A.size(1)}, u);
      const int64_t nbytes = check(mvm_seq_scan_workspace_bytes(&a.d, 1));
      const Tensor ws = workspace(nbytes, u);
      check(mvm_seq_scan_bwd(&a.d, vp(a.u), vp(a.delta), fp(a.dbias), fp(a.A), vp(a.Bm), vp(a.Cm), fp(a.Dv), vp(a.z),
                             fp(sv[8]), vp(dy), fp(dh1), vpm(du), vpm(dd), fpm(ddb), fpm(dA), vpm(dB), vpm(dC),
                             fpm(dD), vpm(dz), fpm(dh0), ws.mutable_data_ptr(), static_cast<size_t>(nbytes),
                             stream_of(u)));
      out[0] = du; out[1] = dd; out[2] = dA.to(A.scalar_type()); out[3] = dB; out[4] = dC;
      out[5] = dD.to(sv[5].scalar_type());
      out[6] = dz;
      if (dbias.defined()) out[7] = ddb.to(dbias.scalar_type());
      if (fl[4] >= 0) out[8] = dh0.to(static_cast<at::ScalarType>(fl[4]));
    }
    return once_differentiable(std::move(out), g, "the packed selective scan");
  }
};

std::pair<Tensor, Tensor> seq_scan(const Tensor& u, const Tensor& delta, const Tensor& A, const Tensor& Bm,
                                   const Tensor& Cm, const Tensor& Dv, const OptTensor& z, const OptTensor& dbias,
                                   const OptTensor& h0, const OptTensor& off, bool softplus, bool a_is_log,
                                   int64_t max_len, int64_t chunk_len) {
  return guarded([&]() -> std::pair<Tensor, Tensor> {
    bool needs = false;
    for (const Tensor* t : {&u, &delta, &A, &Bm, &Cm, &Dv}) needs = needs || t->requires_grad();
    for (const OptTensor* t : {&z, &dbias, &h0}) needs = needs || (t->has_value() && (*t)->requires_grad());
    const auto out = SeqScanFn::apply(u, delta, A, Bm, Cm, Dv, z, dbias, h0, off, softplus, a_is_log, max_len,
                                      chunk_len, needs && at::GradMode::is_enabled());
    return {out[0], out[1]};
  });
}

Tensor seq_scan_prefill(const Tensor& u, const Tensor& delta, const Tensor& A, const Tensor& Bm, const Tensor& Cm,
                        const Tensor& Dv, const Tensor& states, const OptTensor& off_, const OptTensor& slots_,
                        const OptTensor& fresh_, const OptTensor& z, const OptTensor& dbias, bool softplus,
                        bool a_is_log, int64_t max_len, int64_t chunk_len) {
  return guarded([&] {
    at::NoGradGuard no_grad;
    const Tensor off = off_.value_or(Tensor()), slots = slots_.value_or(Tensor()), fresh = fresh_.value_or(Tensor());
    const Seqs q = seqs_of("u", u, off);
    SeqScanArgs a = scan_args(q, u, delta, A, Bm, Cm, Dv, z.value_or(Tensor()), dbias.value_or(Tensor()),
                              {softplus, a_is_log, max_len, chunk_len});
    check_cache(q, states, {q.dim, A.size(1)}, at::kFloat, slots, fresh);
    check_device({&u, &states, &slots, &fresh});
    a.d.seq = seq_desc(q, states.size(0), slots, fresh);
    const Tensor y = scan_launch(a, u.sizes(), states, states, nullptr);
    wrote(states);
    return y;
  });
}

Tensor seq_scan_step(const Tensor& u, const Tensor& delta, const Tensor& A, const Tensor& Bm, const Tensor& Cm,
                     const Tensor& Dv, const Tensor& states, const OptTensor& slots_, const OptTensor& z,
                     const OptTensor& dbias, bool softplus, bool a_is_log) {
  return guarded([&] {
    at::NoGradGuard no_grad;
    const Tensor slots = slots_.value_or(Tensor());
    const Seqs q = step_seqs("u", u);
    SeqScanArgs a = scan_args(q, u, delta, A, Bm, Cm, Dv, z.value_or(Tensor()), dbias.value_or(Tensor()),
                              {softplus, a_is_log, 0, 0});
    check_cache(q, states, {q.dim, A.size(1)}, at::kFloat, slots, Tensor());
    check_device({&u, &states, &slots});
    a.d.seq = seq_desc(q, states.size(0), slots, Tensor());
    c10::OptionalDeviceGuard guard(u.device());
    Tensor y = empty_like_opts(u.sizes(), u, u.scalar_type());
    check(mvm_seq_scan_step(&a.d, vp(a.u), vp(a.delta), fp(a.dbias), fp(a.A), vp(a.Bm), vp(a.Cm), fp(a.Dv), vp(a.z),
                            fpm(states), vpm(y), stream_of(u)));
    wrote(states);
    return y;
  });
}

// --------------------------------------------------------------------- conv

struct SeqConvArgs {
  Tensor x, w, b;
  mvm_seq_conv_desc d{};
};
SeqConvArgs conv_args(const Seqs& q, const Tensor& x, const Tensor& w, const Tensor& b) {
  if (w.dim() != 2 || w.size(0) != q.dim || w.size(1) < 1 || w.size(1) > MVM_CONV_MAX_KWIDTH)
    bad_value("weight must be (D=" + std::to_string(q.dim) + ", d_conv) with d_conv 1.." +
              std::to_string(MVM_CONV_MAX_KWIDTH) + "; got " + shape_str(w));
  if (b.defined() && b.sizes() != at::IntArrayRef({q.dim}))
    bad_value("bias must be (D=" + std::to_string(q.dim) + ",); got " + shape_str(b));
  check_device({&x, &w, &b, &q.off});
  SeqConvArgs a;
  a.x = as_rows(x);
  a.w = f32(w);
  a.b = f32(b);
  a.d.kwidth = w.size(1);
  a.d.x_stride = row_stride(a.x);
  a.d.y_stride = q.dim;
  a.d.dtype = type_code(x.scalar_type());
  return a;
}

struct SeqConvFn : Function<SeqConvFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& b_,
                               const OptTensor& c0_, const OptTensor& off_) {
    const Tensor b = b_.value_or(Tensor()), c0 = c0_.value_or(Tensor()), off = off_.value_or(Tensor());
    const Seqs q = seqs_of("x", x, off);
    SeqConvArgs a = conv_args(q, x, w, b);
    const std::vector<int64_t> rows = {q.nseq, w.size(1) - 1, q.dim};
    if (c0.defined() && (c0.sizes() != rows || c0.scalar_type() != x.scalar_type()))
      bad_value("initial_states must be (" + std::to_string(rows[0]) + ", " + std::to_string(rows[1]) + ", " +
                std::to_string(rows[2]) + ") of x's type; got " + shape_str(c0) + " of " +
                c10::toString(c0.scalar_type()));
    if (c0.defined()) check_device({&x, &c0});
    a.d.seq = seq_desc(q, q.nseq, Tensor(), Tensor());
    c10::OptionalDeviceGuard guard(x.device());
    Tensor y = empty_like_opts(x.sizes(), x, x.scalar_type()), c1 = empty_like_opts(rows, x, x.scalar_type());
    const Tensor c0c = c0.defined() ? c0.contiguous() : c0;
    check(mvm_seq_conv_fwd(&a.d, vp(a.x), fp(a.w), fp(a.b), vp(c0c), vpm(c1), vpm(y), stream_of(x)));
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, w, b, c0, off});
    return {y, c1};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    return in_backward([&] { return grads(ctx, g); });
  }
  static variable_list grads(AutogradContext* ctx, const variable_list& g) {
    const auto sv = ctx->get_saved_variables();
    variable_list out(5);
    if (!g[0].defined() && !g[1].defined()) return out;
    {
      at::NoGradGuard no_grad;
      const Tensor &x = sv[0], &w = sv[1], &b = sv[2], &off = sv[4];
      const Seqs q = seqs_of("x", x, off);
      SeqConvArgs a = conv_args(q, x, w, b);
      a.d.seq = seq_desc(q, q.nseq, Tensor(), Tensor());
      c10::OptionalDeviceGuard guard(x.device());
      const auto t = x.scalar_type();
      const Tensor dy = g[0].defined() ? g[0].to(t).contiguous() : at::zeros(x.sizes(), a.x.options());
      const Tensor dc1 = g[1].defined() ? g[1].to(t).contiguous() : Tensor();
      const Tensor c0 = sv[3].defined() ? sv[3].contiguous() : sv[3];
      Tensor dx = empty_like_opts(x.sizes(), x, t), dw = empty_like_opts(w.sizes(), x), db, dc0;
      if (b.defined()) db = empty_like_opts(b.sizes(), x);
      if (c0.defined()) dc0 = empty_like_opts(c0.sizes(), x, t);
      const int64_t nbytes = check(mvm_seq_conv_workspace_bytes(&a.d));
      const Tensor ws = workspace(nbytes, x);
      check(mvm_seq_conv_bwd(&a.d, vp(a.x), fp(a.w), fp(a.b), vp(c0), vp(dy), vp(dc1), vpm(dx), fpm(dw), fpm(db),
                             vpm(dc0), ws.mutable_data_ptr(), static_cast<size_t>(nbytes), stream_of(x)));
      out[0] = dx;
      out[1] = dw.to(w.scalar_type());
      if (b.defined()) out[2] = db.to(b.scalar_type());
      out[3] = dc0;
    }
    return once_differentiable(std::move(out), g, "the packed causal conv");
  }
};

std::pair<Tensor, Tensor> seq_conv(const Tensor& x, const Tensor& w, const OptTensor& b, const OptTensor& c0,
                                   const OptTensor& off) {
  return guarded([&]() -> std::pair<Tensor, Tensor> {
    const auto out = SeqConvFn::apply(x, w, b, c0, off);
    return {out[0], out[1]};
  });
}

Tensor seq_conv_prefill(const Tensor& x, const Tensor& w, const OptTensor& b, const Tensor& states,
                        const OptTensor& off_, const OptTensor& slots_, const OptTensor& fresh_) {
  return guarded([&] {
    at::NoGradGuard no_grad;
    const Tensor off = off_.value_or(Tensor()), slots = slots_.value_or(Tensor()), fresh = fresh_.value_or(Tensor());
    const Seqs q = seqs_of("x", x, off);
    SeqConvArgs a = conv_args(q, x, w, b.value_or(Tensor()));
    check_cache(q, states, {w.size(1) - 1, q.dim}, x.scalar_type(), slots, fresh);
    check_device({&x, &states, &slots, &fresh});
    a.d.seq = seq_desc(q, states.size(0), slots, fresh);
    c10::OptionalDeviceGuard guard(x.device());
    Tensor y = empty_like_opts(x.sizes(), x, x.scalar_type());
    check(mvm_seq_conv_fwd(&a.d, vp(a.x), fp(a.w), fp(a.b), vp(states), vpm(states), vpm(y), stream_of(x)));
    wrote(states);
    return y;
  });
}

Tensor seq_conv_step(const Tensor& x, const Tensor& w, const OptTensor& b, const Tensor& states,
                     const OptTensor& slots_) {
  return guarded([&] {
    at::NoGradGuard no_grad;
    const Tensor slots = slots_.value_or(Tensor());
    const Seqs q = step_seqs("x", x);
    SeqConvArgs a = conv_args(q, x, w, b.value_or(Tensor()));
    check_cache(q, states, {w.size(1) - 1, q.dim}, x.scalar_type(), slots, Tensor());
    check_device({&x, &states, &slots});
    a.d.seq = seq_desc(q, states.size(0), slots, Tensor());
    c10::OptionalDeviceGuard guard(x.device());
    Tensor y = empty_like_opts(x.sizes(), x, x.scalar_type());
    check(mvm_seq_conv_step(&a.d, vp(a.x), fp(a.w), fp(a.b), vpm(states), vpm(y), stream_of(x)));
    wrote(states);
    return y;
  });
}

}  // namespace
