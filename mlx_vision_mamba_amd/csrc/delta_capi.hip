// C ABI of the gated delta rule (include/mvm_delta.h): validation, the split of
// the time axis, and of the caller's workspace.
#include <algorithm>
#include <initializer_list>

#include "delta_kernels.h"
#include "mvm_delta.h"
#include "mvm_scan.h"
#include "status.h"

namespace {

using mvm::fail;
using mvm::hip_status;
using mvm::ok;

constexpr int64_t kMaxTokens = INT32_MAX - 64;
constexpr int64_t kMaxBlocks = (int64_t{1} << 32) / 256 - 8;  // 2^32 threads a launch
constexpr int64_t kMaxHeads = 1 << 20;
constexpr size_t kAlign = 256;

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
size_t align_up(size_t x) { return (x + kAlign - 1) / kAlign * kAlign; }

int check_seq(const mvm_seq_desc& q) {
  if (q.tokens < 0 || q.nseq < 0 || q.seqlen < 0 || q.state_rows < 0)
    return fail(MVM_ERR_INVALID_ARG, "negative size (tokens=%lld nseq=%lld seqlen=%lld state_rows=%lld)",
                (long long)q.tokens, (long long)q.nseq, (long long)q.seqlen, (long long)q.state_rows);
  if (q.dim != 0) return fail(MVM_ERR_INVALID_ARG, "seq.dim=%lld must be 0", (long long)q.dim);
  if (q.tokens > kMaxTokens || q.nseq > kMaxTokens || q.state_rows > kMaxTokens)
    return fail(MVM_ERR_UNSUPPORTED, "tokens, nseq and state_rows must be at most %lld", (long long)kMaxTokens);
  // (seqlen <= tokens where there are sequences, so the product cannot overflow)
  if (q.offsets == nullptr && (q.nseq > 0 ? q.seqlen > q.tokens || q.nseq * q.seqlen != q.tokens : q.tokens != 0))
    return fail(MVM_ERR_INVALID_ARG, "without offsets tokens=%lld must be nseq=%lld * seqlen=%lld",
                (long long)q.tokens, (long long)q.nseq, (long long)q.seqlen);
  if (q.slots == nullptr && q.state_rows < q.nseq)
    return fail(MVM_ERR_INVALID_ARG, "state_rows=%lld < nseq=%lld without slots", (long long)q.state_rows,
                (long long)q.nseq);
  return MVM_OK;
}

int check_stride(const char* name, int64_t stride) {
  if (stride < 0) return fail(MVM_ERR_INVALID_ARG, "%s=%lld is negative", name, (long long)stride);
  if (stride > (INT32_MAX >> 2))
    return fail(MVM_ERR_UNSUPPORTED, "%s=%lld: strides of at most %d values", name, (long long)stride, INT32_MAX >> 2);
  return MVM_OK;
}

// The parts of the time axis.  Whole sequences leave compute units idle where
// there are few of them and heads; parts cost a pass for their ends and
// transitions, of twice the columns, and their joining, one after the other.  The
// cheapest cut by a model in units of a main pass's chunk (5.5-7 us, 128 x 128
// heads of bfloat16): a workgroup a compute unit, so passes take whole rounds of
// them; a chunk of the parts' pass takes 0.7, a part's joining 0.2 to 0.75.
// Measured on MI355X with 12 such heads, us forward whole / in parts: one
// sequence of 32768 tokens 3122 / 588, of 8192 793 / 218; 6 of 2730 333 / 317; 16
// of 512 96 / 162.
constexpr int64_t kUnits = 256;

void pick_parts(const mvm_delta_desc* d, mvm::DeltaGeom& g) {
  const int64_t T = d->seq.tokens, S = std::max<int64_t>(1, d->seq.nseq);
  int64_t longest = d->seq.offsets == nullptr ? d->seq.seqlen : T;
  if (d->max_len > 0) longest = std::min(longest, d->max_len);
  int64_t len = d->split_len;
  if (len == 0) {
    const int dkp = mvm::delta_dkp(g.DK);
    const int64_t vcb = mvm::delta_col_blocks(g.DV, g.waves), tcb = mvm::delta_col_blocks(dkp, g.waves);
    const int64_t C = mvm::kDeltaChunk, chunks = ceil_div(longest, C);
    const double join = dkp == 128 ? 0.75 : (dkp == 64 ? 0.3 : 0.2);
    // a tenth in favour of whole sequences: less memory, fewer launches
    double best = 0.9 * std::max<int64_t>(chunks, ceil_div((T / C + S / 2) * g.HV * vcb, kUnits));
    len = longest;
    for (int64_t n = 2; n <= std::min<int64_t>(chunks, 128); ++n) {
      const int64_t lc = ceil_div(chunks, n), parts = T / (lc * C) + (S + 1) / 2;
      const double cost = static_cast<double>(lc) * ceil_div(parts * g.HV * vcb, kUnits) +
                          0.7 * lc * ceil_div(std::max<int64_t>(1, parts - S) * g.HV * (vcb + tcb), kUnits) + join * n + 2;
      if (cost < best) best = cost, len = lc * C;
    }
  }
  // Whole sequences: one part whatever max_len says
  g.parts = len < longest ? static_cast<int32_t>(ceil_div(longest, len)) : 1;
  g.part = mvm::seq_cut(g.parts > 1 ? len : std::max<int64_t>(mvm::kDeltaChunk, T + 1));
}

// Waves of a workgroup of the passes along time: eight share a chunk's operands where the state has columns for them
// and the card is full of them (bfloat16, 8191 tokens in 23 prompts of 12 heads of 128 x 128: 134 us, 141 by four; but 2048
// tokens of 4 heads 100, and 91 by four, whose chunks take less long).  Float32 operands are three parts, of which
// eight waves' registers spill (16384 tokens of 12 heads: 568 us forward, 354 by four).
int pick_waves(const mvm_delta_desc* d, const mvm::DeltaGeom& g) {
  const int64_t items = (d->seq.tokens / mvm::kDeltaChunk + d->seq.nseq) * g.HV;
  return d->dtype == MVM_BF16 && g.DV > 64 && items >= 512 ? 8 : 4;
}

mvm::DeltaGeom geom(const mvm_delta_desc* d) {
  mvm::DeltaGeom g{};
  g.q.T = static_cast<int32_t>(d->seq.tokens);
  g.q.S = static_cast<int32_t>(d->seq.nseq);
  g.q.M = static_cast<int32_t>(d->seq.state_rows);
  g.q.L = static_cast<int32_t>(d->seq.seqlen);
  g.q.off = d->seq.offsets;
  g.q.slots = d->seq.slots;
  g.q.fresh = d->seq.fresh;
  g.HK = static_cast<int32_t>(d->key_heads);
  g.HV = static_cast<int32_t>(d->value_heads);
  g.group = g.HV / g.HK;
  g.DK = static_cast<int32_t>(d->dk);
  g.DV = static_cast<int32_t>(d->dv);
  g.qs = d->q_stride;
  g.qh = d->q_stride_head;
  g.ks = d->k_stride;
  g.kh = d->k_stride_head;
  g.vs = d->v_stride;
  g.vh = d->v_stride_head;
  g.gs = d->g_stride;
  g.bs = d->beta_stride;
  g.scale = d->scale;
  g.l2 = d->qk_l2norm;
  g.beta_f32 = d->beta_dtype == MVM_F32;
  g.cut = mvm::seq_cut(mvm::kDeltaChunk);
  g.waves = pick_waves(d, g);
  pick_parts(d, g);
  return g;
}

// Which rows are accessed 16 bytes at a time.
bool fits(const void* p, int64_t row, int64_t head) {
  return ((static_cast<int64_t>(reinterpret_cast<uintptr_t>(p)) | row | head) & 15) == 0;
}
bool wide(const mvm::DeltaGeom& g, const mvm::DeltaIn& in, int dtype, std::initializer_list<const void*> outs) {
  const int64_t e = dtype == MVM_F32 ? 4 : 2;
  bool ok = g.DK * e % 16 == 0 && fits(in.q, g.qs * e, g.qh * e) && fits(in.k, g.ks * e, g.kh * e) &&
            fits(in.v, g.vs * e, g.vh * e);
  for (const void* p : outs) ok = ok && fits(p, g.DV * e, 0);
  return ok;
}

int check_delta(const mvm_delta_desc* d) {
  if (d == nullptr) return fail(MVM_ERR_INVALID_ARG, "desc is NULL");
  int rc = check_seq(d->seq);
  if (rc != MVM_OK) return rc;
  if (d->key_heads < 1 || d->value_heads < 1 || d->value_heads % d->key_heads != 0)
    return fail(MVM_ERR_INVALID_ARG, "value_heads=%lld must be a multiple of key_heads=%lld", (long long)d->value_heads,
                (long long)d->key_heads);
  if (d->value_heads > kMaxHeads)
    return fail(MVM_ERR_UNSUPPORTED, "value_heads=%lld: at most %lld", (long long)d->value_heads, (long long)kMaxHeads);
  if (d->dk < 1 || d->dk > MVM_DELTA_MAX_DK || d->dv < 1 || d->dv > MVM_DELTA_MAX_DV)
    return fail(MVM_ERR_UNSUPPORTED, "dk=%lld, dv=%lld unsupported (1..%d, 1..%d)", (long long)d->dk, (long long)d->dv,
                MVM_DELTA_MAX_DK, MVM_DELTA_MAX_DV);
  if (d->dtype != MVM_F32 && d->dtype != MVM_BF16)
    return fail(MVM_ERR_UNSUPPORTED, "dtype=%d unsupported", d->dtype);
  if (d->beta_dtype != MVM_F32 && d->beta_dtype != d->dtype)
    return fail(MVM_ERR_UNSUPPORTED, "beta_dtype=%d must be MVM_F32 or dtype", d->beta_dtype);
  if (d->reserved != 0) return fail(MVM_ERR_INVALID_ARG, "reserved must be 0");
  if (d->qk_l2norm != 0 && d->qk_l2norm != 1)
    return fail(MVM_ERR_INVALID_ARG, "qk_l2norm=%d must be 0 or 1", d->qk_l2norm);
  if (d->max_len < 0) return fail(MVM_ERR_INVALID_ARG, "max_len=%lld is negative", (long long)d->max_len);
  if (d->split_len < 0 || d->split_len % mvm::kDeltaChunk != 0)
    return fail(MVM_ERR_INVALID_ARG, "split_len=%d must be 0 or a multiple of %d", d->split_len, mvm::kDeltaChunk);
  if ((rc = check_stride("q_stride", d->q_stride)) || (rc = check_stride("q_stride_head", d->q_stride_head)) ||
      (rc = check_stride("k_stride", d->k_stride)) || (rc = check_stride("k_stride_head", d->k_stride_head)) ||
      (rc = check_stride("v_stride", d->v_stride)) || (rc = check_stride("v_stride_head", d->v_stride_head)) ||
      (rc = check_stride("g_stride", d->g_stride)) || (rc = check_stride("beta_stride", d->beta_stride)))
    return rc;
  if (d->v_stride > mvm::kDeltaMaxStride || d->value_heads * d->dv > mvm::kDeltaMaxStride)
    return fail(MVM_ERR_UNSUPPORTED, "v_stride=%lld and value_heads * dv: at most %lld", (long long)d->v_stride,
                (long long)mvm::kDeltaMaxStride);
  // the largest launch: a chunk of every part, head and block of 16 columns
  const int64_t slots = d->seq.tokens / mvm::kDeltaChunk + d->seq.nseq + 1;
  if (slots > kMaxBlocks / (d->value_heads + 8) / ceil_div(std::max(d->dk, d->dv), 16))
    return fail(MVM_ERR_UNSUPPORTED, "tokens=%lld, nseq=%lld and value_heads=%lld are too many for one launch",
                (long long)d->seq.tokens, (long long)d->seq.nseq, (long long)d->value_heads);
  return MVM_OK;
}

// What a training forward leaves: the chunks' initial states, the rows d_t, and (DeltaWork) their triangles and scalars.
struct Ckpt {
  size_t s0, vt, tri, dec, gam, total;
};
Ckpt ckpt_of(const mvm::DeltaGeom& g) {
  const size_t items = static_cast<size_t>(mvm::chunk_slots(g.q, g.cut)) * g.HV;
  const size_t tiles = items * static_cast<size_t>(mvm::delta_col_tiles(g)) * 256 * 4;
  Ckpt c;
  c.s0 = align_up(tiles * (mvm::delta_dkp(g.DK) / 16));
  c.vt = align_up(tiles * 4);
  c.tri = align_up(items * mvm::kTriBytes);
  c.dec = align_up(items * mvm::kDeltaChunk * 16);
  c.gam = align_up(items * 4);
  c.total = c.s0 + c.vt + c.tri + c.dec + c.gam;
  return c;
}

struct Ws {
  size_t tri = 0, dec = 0, gam = 0, trans = 0, carry = 0, x = 0, dend = 0, total = 0;
};
Ws ws_of(const mvm::DeltaGeom& g, bool backward) {
  Ws w;
  const Ckpt c = ckpt_of(g);
  if (backward) {
    w.x = c.vt;
    w.dend = c.s0;
  } else {
    w.tri = c.tri;
    w.dec = c.dec;
    w.gam = c.gam;
  }
  if (g.parts > 1) {
    const size_t parts = static_cast<size_t>(mvm::chunk_slots(g.q, g.part)) * g.HV, dkp = mvm::delta_dkp(g.DK);
    w.trans = align_up(parts * dkp * dkp * 4);
    w.carry = align_up(parts * static_cast<size_t>(mvm::delta_col_tiles(g)) * 16 * dkp * 4);
  }
  w.total = w.tri + w.dec + w.gam + w.trans + w.carry + w.x + w.dend;
  return w;
}

struct Take {
  char* at;
  float* operator()(size_t n) {
    float* p = n > 0 ? reinterpret_cast<float*>(at) : nullptr;
    at += n;
    return p;
  }
};

void take_ckpt(const mvm::DeltaGeom& g, const float* ckpt, float*& s0, float*& vt, mvm::DeltaWork& w) {
  const Ckpt c = ckpt_of(g);
  Take take{reinterpret_cast<char*>(const_cast<float*>(ckpt))};
  s0 = take(c.s0);
  vt = take(c.vt);
  w.tri = take(c.tri);
  w.dec = take(c.dec);
  w.gam = take(c.gam);
}

int check_ws(const char* what, const void* ws, size_t have, size_t need) {
  if (need > 0 && (ws == nullptr || have < need))
    return fail(MVM_ERR_WORKSPACE, "%s: workspace %zu bytes < %zu needed", what, have, need);
  if (need > 0 && (reinterpret_cast<uintptr_t>(ws) & (kAlign - 1)) != 0)
    return fail(MVM_ERR_WORKSPACE, "%s: workspace must be %zu-byte aligned", what, kAlign);
  return MVM_OK;
}
int check_ckpt(const char* what, const float* ckpt) {
  if ((reinterpret_cast<uintptr_t>(ckpt) & 15u) != 0)
    return fail(MVM_ERR_INVALID_ARG, "%s: ckpt must be 16-byte aligned", what);
  return MVM_OK;
}

bool missing(const mvm::DeltaIn& in) { return !in.q || !in.k || !in.v || !in.g || !in.beta; }

}  // namespace

extern "C" {

int mvm_delta_validate(const mvm_delta_desc* desc) {
  const int rc = check_delta(desc);
  return rc == MVM_OK ? ok() : rc;
}

int64_t mvm_delta_ckpt_elems(const mvm_delta_desc* desc) {
  const int rc = check_delta(desc);
  if (rc != MVM_OK) return rc;
  return static_cast<int64_t>(ckpt_of(geom(desc)).total / sizeof(float));
}

int64_t mvm_delta_workspace_bytes(const mvm_delta_desc* desc, int which) {
  const int rc = check_delta(desc);
  if (rc != MVM_OK) return rc;
  if (which != 0 && which != 1) return fail(MVM_ERR_INVALID_ARG, "which=%d must be 0 or 1", which);
  return static_cast<int64_t>(ws_of(geom(desc), which == 1).total);
}

int mvm_delta_fwd(const mvm_delta_desc* desc, const void* q, const void* k, const void* v, const float* g,
                  const void* beta, const float* h0, float* h1, void* o, float* ckpt, void* workspace,
                  size_t workspace_bytes, void* stream) {
  int rc = check_delta(desc);
  if (rc != MVM_OK) return rc;
  mvm::DeltaGeom gm = geom(desc);
  if (gm.q.T == 0 && gm.q.S == 0) return ok();
  const mvm::DeltaIn in{q, k, v, g, beta};
  if (gm.q.T > 0 && (missing(in) || !o)) return fail(MVM_ERR_INVALID_ARG, "mvm_delta_fwd: NULL pointer");
  if ((rc = check_ckpt("mvm_delta_fwd", ckpt)) != MVM_OK) return rc;
  const Ws w = ws_of(gm, false);
  if ((rc = check_ws("mvm_delta_fwd", workspace, workspace_bytes, w.total)) != MVM_OK) return rc;
  gm.vec = wide(gm, in, desc->dtype, {o});
  Take take{static_cast<char*>(workspace)};
  mvm::DeltaWork b{};
  b.tri = take(w.tri);
  b.dec = take(w.dec);
  b.gam = take(w.gam);
  b.trans = take(w.trans);
  b.carry = take(w.carry);
  float *s0 = nullptr, *vt = nullptr;
  if (ckpt != nullptr) take_ckpt(gm, ckpt, s0, vt, b);
  return hip_status(mvm::launch_delta_fwd(gm, in, b, h0, h1, o, s0, vt, desc->dtype, static_cast<hipStream_t>(stream)),
                    "mvm_delta_fwd launch");
}

int mvm_delta_bwd(const mvm_delta_desc* desc, const void* q, const void* k, const void* v, const float* g,
                  const void* beta, const float* ckpt, const void* d_o, const float* dh1, void* dq, void* dk, void* dv,
                  float* dg, void* dbeta, float* dh0, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_delta(desc);
  if (rc != MVM_OK) return rc;
  if (desc->seq.slots != nullptr || desc->seq.fresh != nullptr)
    return fail(MVM_ERR_INVALID_ARG, "a backward takes neither slots nor fresh");
  mvm::DeltaGeom gm = geom(desc);
  if (gm.q.T == 0 && gm.q.S == 0) return ok();
  const mvm::DeltaIn in{q, k, v, g, beta};
  if (gm.q.T > 0 && (missing(in) || !ckpt || !d_o || !dq || !dk || !dv || !dg || !dbeta))
    return fail(MVM_ERR_INVALID_ARG, "mvm_delta_bwd: NULL pointer");
  if ((rc = check_ckpt("mvm_delta_bwd", ckpt)) != MVM_OK) return rc;
  const Ws w = ws_of(gm, true);
  if ((rc = check_ws("mvm_delta_bwd", workspace, workspace_bytes, w.total)) != MVM_OK) return rc;
  gm.vec = wide(gm, in, desc->dtype, {d_o, dv}) && fits(dq, 0, 0) && fits(dk, 0, 0);
  Take take{static_cast<char*>(workspace)};
  mvm::DeltaWork b{};
  b.trans = take(w.trans);
  b.carry = take(w.carry);
  mvm::DeltaBwd r{};
  float *s0 = nullptr, *vt = nullptr;
  if (ckpt != nullptr) take_ckpt(gm, ckpt, s0, vt, b);
  r.s0 = s0;
  r.vt = vt;
  r.d_o = d_o; r.dh1 = dh1; r.dh0 = dh0;
  r.x = take(w.x);
  r.dend = take(w.dend);
  r.dq = dq; r.dk = dk; r.dv = dv; r.dg = dg; r.dbeta = dbeta;
  return hip_status(mvm::launch_delta_bwd(gm, in, b, r, desc->dtype, static_cast<hipStream_t>(stream)),
                    "mvm_delta_bwd launch");
}

int mvm_delta_step(const mvm_delta_desc* desc, const void* q, const void* k, const void* v, const float* g,
                   const void* beta, float* states, void* o, void* stream) {
  int rc = check_delta(desc);
  if (rc != MVM_OK) return rc;
  const mvm_seq_desc& s = desc->seq;
  if (s.offsets != nullptr || s.tokens != s.nseq || (s.nseq > 0 && s.seqlen != 1))
    return fail(MVM_ERR_INVALID_ARG, "a step takes one token for each sequence (tokens == nseq, seqlen 1, no offsets)");
  mvm::DeltaGeom gm = geom(desc);
  if (gm.q.S == 0) return ok();
  const mvm::DeltaIn in{q, k, v, g, beta};
  if (missing(in) || !states || !o) return fail(MVM_ERR_INVALID_ARG, "mvm_delta_step: NULL pointer");
  return hip_status(mvm::launch_delta_step(gm, in, states, o, desc->dtype, static_cast<hipStream_t>(stream)),
                    "mvm_delta_step launch");
}

}  // extern "C"
