// C ABI of the packed and served forms (include/mvm_seq.h): validation, the
// cut into time chunks, and the split of the caller's workspace.
#include <algorithm>

#include "mvm_conv.h"
#include "mvm_scan.h"
#include "mvm_seq.h"
#include "seq_kernels.h"
#include "status.h"

namespace {

using mvm::fail;
using mvm::hip_status;
using mvm::ok;

// positions are int32, and formed up to a chunk's tile past the last
constexpr int64_t kMaxTokens = INT32_MAX - 64;
constexpr int64_t kMaxThreads = (int64_t{1} << 32) - 1024;  // of one launch

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
constexpr size_t kAlign = 256;
size_t align_up(size_t x) { return (x + kAlign - 1) / kAlign * kAlign; }

int check_seq(const mvm_seq_desc& q) {
  if (q.tokens < 0 || q.nseq < 0 || q.seqlen < 0 || q.dim < 0 || q.state_rows < 0)
    return fail(MVM_ERR_INVALID_ARG, "negative size (tokens=%lld nseq=%lld seqlen=%lld dim=%lld state_rows=%lld)",
                (long long)q.tokens, (long long)q.nseq, (long long)q.seqlen, (long long)q.dim,
                (long long)q.state_rows);
  if (q.tokens > kMaxTokens || q.nseq > kMaxTokens || q.state_rows > kMaxTokens || q.dim > (kMaxTokens >> 2))
    return fail(MVM_ERR_UNSUPPORTED, "tokens, nseq and state_rows must be at most %lld, dim %lld",
                (long long)kMaxTokens, (long long)(kMaxTokens >> 2));
  // (seqlen <= tokens where there are sequences, so the product cannot overflow)
  if (q.offsets == nullptr && (q.nseq > 0 ? q.seqlen > q.tokens || q.nseq * q.seqlen != q.tokens : q.tokens != 0))
    return fail(MVM_ERR_INVALID_ARG, "without offsets tokens=%lld must be nseq=%lld * seqlen=%lld",
                (long long)q.tokens, (long long)q.nseq, (long long)q.seqlen);
  if (q.slots == nullptr && q.state_rows < q.nseq)
    return fail(MVM_ERR_INVALID_ARG, "state_rows=%lld < nseq=%lld without slots", (long long)q.state_rows,
                (long long)q.nseq);
  return MVM_OK;
}

int check_rows(const char* name, int64_t stride, int64_t tokens, int64_t cols, bool written) {
  if (stride > (INT32_MAX >> 2))
    return fail(MVM_ERR_UNSUPPORTED, "%s=%lld: strides of at most %d values", name, (long long)stride, INT32_MAX >> 2);
  if (stride < 0 || (written && tokens > 1 && stride < cols))
    return fail(MVM_ERR_INVALID_ARG, "%s=%lld: rows of %lld values %s", name, (long long)stride, (long long)cols,
                written ? "must not overlap" : "need a stride >= 0");
  return MVM_OK;
}

int check_scan_fields(const mvm_seq_scan_desc* d) {
  if (d == nullptr) return fail(MVM_ERR_INVALID_ARG, "desc is NULL");
  int rc = check_seq(d->seq);
  if (rc != MVM_OK) return rc;
  if (d->dstate < 1 || d->dstate > MVM_MAX_DSTATE)
    return fail(MVM_ERR_UNSUPPORTED, "dstate=%lld unsupported (1..%d)", (long long)d->dstate, MVM_MAX_DSTATE);
  if (d->dtype != MVM_F32 && d->dtype != MVM_BF16)
    return fail(MVM_ERR_UNSUPPORTED, "dtype=%d unsupported", d->dtype);
  if (d->delta_dtype != MVM_F32 && d->delta_dtype != d->dtype)
    return fail(MVM_ERR_UNSUPPORTED, "delta_dtype=%d must be MVM_F32 or dtype", d->delta_dtype);
  if (d->reserved != 0) return fail(MVM_ERR_INVALID_ARG, "reserved must be 0");
  if (d->max_len < 0) return fail(MVM_ERR_INVALID_ARG, "max_len=%lld is negative", (long long)d->max_len);
  if (d->chunk_len != 0 && (d->chunk_len < 16 || (d->chunk_len & (d->chunk_len - 1)) != 0))
    return fail(MVM_ERR_INVALID_ARG, "chunk_len=%d must be 0 or a power of two >= 16", d->chunk_len);
  const int64_t t = d->seq.tokens, c = d->seq.dim;
  if ((rc = check_rows("u_stride", d->u_stride, t, c, false)) || (rc = check_rows("delta_stride", d->delta_stride, t, c, false)) ||
      (rc = check_rows("bc_stride", d->bc_stride, t, d->dstate, false)) ||
      (rc = check_rows("z_stride", d->z_stride, t, c, false)) || (rc = check_rows("y_stride", d->y_stride, t, c, true)))
    return rc;
  return MVM_OK;
}

int check_threads(const mvm_seq_desc& q, int64_t blocks, int64_t threads) {
  if (threads > 0 && blocks > kMaxThreads / threads)
    return fail(MVM_ERR_UNSUPPORTED, "tokens=%lld, nseq=%lld and dim=%lld are too many for one launch",
                (long long)q.tokens, (long long)q.nseq, (long long)q.dim);
  return MVM_OK;
}

mvm::SeqGeom seq_geom(const mvm_seq_desc& q) {
  mvm::SeqGeom g;
  g.T = static_cast<int32_t>(q.tokens);
  g.S = static_cast<int32_t>(q.nseq);
  g.M = static_cast<int32_t>(q.state_rows);
  g.L = static_cast<int32_t>(q.seqlen);
  g.D = q.dim;
  g.off = q.offsets;
  g.slots = q.slots;
  g.fresh = q.fresh;
  return g;
}

// The cut into time chunks.  A wave is 64 channels of one chunk; chunks let
// one sequence use more waves, but need an aggregate pass before the main one,
// which repeats most of the recurrence, and their joining.  Waves are placed
// when the launch starts, so a pass takes as long as the SIMDs with the most of
// them: the cut is the cheapest of those that just fit 1/4, 1/2, 1, 2, .. waves
// on each of the card's 1024 SIMDs (from `waves` on, what fits at once, in
// rounds), and of whole sequences, by a model in cycles at 2.36 GHz.  It is
// fitted to times of 14 packings of 1 to 60 sequences at 4 to 28 lengths each on
// MI355X (5 % off on average), where its choices take 0.1 % longer than the best
// length forward and 1.6 % backward.
struct Cost {
  int waves;
  int64_t start, placed;         // the launches and first loads, and for one wave a SIMD
  int64_t work;                  // a token of a SIMD's share of all tokens and waves
  int64_t token[4], whole[4];    // one token of chunks, of whole sequences, on a SIMD of 1, 2, .. waves
  int64_t whole_start;
};
constexpr Cost kFwdCost = {4, 8000, 11500, 0, {1910, 2210, 2520, 2910}, {1280, 1540, 1900, 2270}, 3000};
constexpr Cost kBwdCost = {3, 32000, 5800, 1000, {2600, 2940, 3400}, {2300, 3250, 5600}, 20000};
constexpr int64_t kSimds = 1024;
constexpr int64_t kFold = 1060;        // the main pass joins one chunk before its own
constexpr int64_t kCarry = 9000;       // a carry pass,
constexpr int64_t kCarryRound = 3000;  // its rounds of 128 chunks,
constexpr int64_t kCarryWave = 12;     // and its traffic for one wave's aggregate

void pick_chunk(const mvm_seq_scan_desc* d, const Cost& k, mvm::SeqScanGeom& g) {
  const int64_t T = d->seq.tokens, S = d->seq.nseq, ncb = std::max<int64_t>(1, ceil_div(d->seq.dim, 64));
  int64_t longest = d->seq.offsets == nullptr ? d->seq.seqlen : T;
  if (d->max_len > 0) longest = std::min(longest, d->max_len);
  // (a sequence's last chunk is half a chunk on average)
  const auto waves_of = [&](int64_t len) { return ncb * ceil_div(T + (S - 1) * len / 2, len); };
  const auto join = [&](int64_t waves, int64_t nth, bool fold) {
    return fold ? (nth - 1) * kFold * std::max(waves, kSimds) / kSimds
                : kCarry + ceil_div(nth, 128) * kCarryRound + waves * kCarryWave;
  };
  const int64_t share = T * ncb / kSimds;
  const auto cost = [&](int64_t len) {
    // slots of no chunk take their places too
    const int64_t waves = waves_of(len), nth = ceil_div(longest, len), placed = ncb * ((T - 1) / len + S);
    const int64_t n = std::max<int64_t>(1, ceil_div(placed, kSimds));
    const int64_t token = n <= k.waves ? k.token[n - 1] : k.token[k.waves - 1] * n / k.waves;
    return k.start + k.placed * placed / kSimds + k.work * share + len * token +
           std::min(join(waves, nth, true), join(waves, nth, false));
  };
  int64_t len = d->chunk_len;
  if (len == 0) {
    // whole sequences: the longest, or all the work where it comes in rounds
    const int64_t n = std::max<int64_t>(1, ceil_div(ncb * S, kSimds));
    int64_t best = k.whole_start + (n <= k.waves ? longest * k.whole[n - 1]
                                                 : std::max(longest * k.whole[0],
                                                            (share + longest / 2) * k.whole[k.waves - 1] / k.waves));
    len = longest;
    for (int64_t quarters = 1; quarters <= 16 * k.waves;
         quarters += quarters < 4 || quarters >= 4 * k.waves ? quarters : 4) {
      const int64_t chunks = quarters * (kSimds / 4) / ncb - S;  // beside each sequence's first
      if (chunks < 0) continue;
      const int64_t n = std::max<int64_t>(1, ceil_div(ceil_div(T, chunks + 1), mvm::kSeqTile)) * mvm::kSeqTile;
      if (n >= longest) continue;
      const int64_t c = cost(n);
      if (c < best) best = c, len = n;
    }
  }
  g.multi = len < longest;
  // Whole sequences: one chunk whatever max_len says
  if (!g.multi) len = std::max<int64_t>(16, T + 1);
  const int64_t nth = ceil_div(longest, len), waves = waves_of(len);
  g.cut = mvm::seq_cut(len);
  g.fold = g.multi && join(waves, nth, true) <= join(waves, nth, false);
  g.max_chunks = g.multi ? static_cast<int32_t>(nth) : 1;
}

mvm::SeqScanGeom scan_geom(const mvm_seq_scan_desc* d, bool backward) {
  mvm::SeqScanGeom g;
  g.q = seq_geom(d->seq);
  g.us = d->u_stride;
  g.ds = d->delta_stride;
  g.bs = d->bc_stride;
  g.ys = d->y_stride;
  g.zs = d->z_stride;
  g.N = static_cast<int32_t>(d->dstate);
  g.a_log = d->a_is_log != 0;
  g.softplus = d->delta_softplus != 0;
  pick_chunk(d, backward ? kBwdCost : kFwdCost, g);
  return g;
}

// Everything that a call of either direction would be refused for.
int check_scan(const mvm_seq_scan_desc* d) {
  int rc = check_scan_fields(d);
  if (rc == MVM_OK) rc = check_threads(d->seq, d->seq.tokens, ceil_div(d->seq.dim, 64));
  for (int backward = 0; rc == MVM_OK && backward < 2; ++backward) {
    const mvm::SeqScanGeom g = scan_geom(d, backward != 0);
    const int64_t carry = g.multi ? ceil_div(g.q.D, 16) * g.q.S : 0;
    if ((rc = check_threads(d->seq, mvm::chunk_slots(g.q, g.cut), ceil_div(g.q.D, 64) * 64)) == MVM_OK &&
        (rc = check_threads(d->seq, carry, 64 * mvm::carry_waves(g))) == MVM_OK)
      rc = check_threads(d->seq, g.q.D, 18 * 16);  // the reduction's workgroups of 64 columns
  }
  return rc;
}

int64_t ckpt_elems(const mvm_seq_scan_desc* d) {
  return ((d->seq.tokens >> mvm::kSeqTileShift) + d->seq.nseq + 1) * d->seq.dim * 16;
}

struct ScanWs {
  size_t agg_h = 0, agg_s = 0, bc = 0, part = 0, part_bc = 0, total = 0;
};
ScanWs scan_ws(const mvm_seq_scan_desc* d, const mvm::SeqScanGeom& g, bool backward) {
  ScanWs w;
  const size_t slots = static_cast<size_t>(mvm::chunk_slots(g.q, g.cut)), D = static_cast<size_t>(g.q.D);
  const size_t T = static_cast<size_t>(g.q.T);
  if (g.multi) {
    w.agg_h = align_up(slots * D * 16 * sizeof(float));
    w.agg_s = align_up(slots * D * sizeof(float));
  }
  if (d->dtype != MVM_F32 || d->dstate != 16) w.bc = align_up(T * 32 * sizeof(float));
  if (backward) {
    w.part = align_up(slots * D * 18 * sizeof(float));
    w.part_bc = align_up(static_cast<size_t>(ceil_div(g.q.D, 64)) * T * 32 * sizeof(float));
  }
  w.total = w.agg_h + w.agg_s + w.bc + w.part + w.part_bc;
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

int check_ws(const char* what, const void* ws, size_t have, size_t need) {
  if (need > 0 && (ws == nullptr || have < need))
    return fail(MVM_ERR_WORKSPACE, "%s: workspace %zu bytes < %zu needed", what, have, need);
  if (need > 0 && (reinterpret_cast<uintptr_t>(ws) & (kAlign - 1)) != 0)
    return fail(MVM_ERR_WORKSPACE, "%s: workspace must be %zu-byte aligned", what, kAlign);
  return MVM_OK;
}

// (accessed 16 bytes at a time)
int check_ckpt(const char* what, const float* ckpt) {
  if ((reinterpret_cast<uintptr_t>(ckpt) & 15u) != 0)
    return fail(MVM_ERR_INVALID_ARG, "%s: ckpt must be 16-byte aligned", what);
  return MVM_OK;
}

// Operands that are read wherever there are tokens.
bool missing(const mvm::SeqScanIn& in) { return !in.u || !in.delta || !in.A || !in.Bm || !in.Cm || !in.Dv; }

int check_conv(const mvm_seq_conv_desc* d) {
  if (d == nullptr) return fail(MVM_ERR_INVALID_ARG, "desc is NULL");
  int rc = check_seq(d->seq);
  if (rc != MVM_OK) return rc;
  if (d->kwidth < 1 || d->kwidth > MVM_CONV_MAX_KWIDTH)
    return fail(MVM_ERR_UNSUPPORTED, "kwidth=%lld unsupported (1..%d)", (long long)d->kwidth, MVM_CONV_MAX_KWIDTH);
  if (d->dtype != MVM_F32 && d->dtype != MVM_BF16)
    return fail(MVM_ERR_UNSUPPORTED, "dtype=%d unsupported", d->dtype);
  if (d->reserved != 0) return fail(MVM_ERR_INVALID_ARG, "reserved must be 0");
  const int64_t t = d->seq.tokens, c = d->seq.dim;
  if ((rc = check_rows("x_stride", d->x_stride, t, c, false)) || (rc = check_rows("y_stride", d->y_stride, t, c, true)))
    return rc;
  return check_threads(d->seq, t / mvm::conv_cut(4).len + d->seq.nseq + 1, ceil_div(c, 64) * 256);
}

mvm::SeqConvGeom conv_geom(const mvm_seq_conv_desc* d) {
  mvm::SeqConvGeom g;
  g.q = seq_geom(d->seq);
  g.xs = d->x_stride;
  g.ys = d->y_stride;
  g.kc = static_cast<int32_t>(d->kwidth);
  // waves with 16 bytes a lane (backward: two channels) at the longer runs.
  // MI355X, forward: 392 tokens of 1536 bf16 channels 6.4 us by runs of 8, 5.1
  // by 4; 12000 tokens 19.5 and 21.0
  const int64_t lanes = d->dtype == MVM_F32 ? 4 : 8, t = d->seq.tokens;
  // (a run is at least the window's earlier positions)
  g.fwd_pos = d->kwidth > 5 || ceil_div(d->seq.dim, 64 * lanes) * (t / 8) >= 1536 ? 8 : 4;
  g.bwd_pos = ceil_div(d->seq.dim, 128) * (t / 16) >= 1536 ? 16 : 8;
  return g;
}

int check_step(const mvm_seq_desc& q) {
  if (q.offsets != nullptr || q.tokens != q.nseq || (q.nseq > 0 && q.seqlen != 1))
    return fail(MVM_ERR_INVALID_ARG, "a step takes one token for each sequence (tokens == nseq, seqlen 1, no offsets)");
  return MVM_OK;
}

int check_plain(const mvm_seq_desc& q) {
  if (q.slots != nullptr || q.fresh != nullptr)
    return fail(MVM_ERR_INVALID_ARG, "a backward takes neither slots nor fresh");
  return MVM_OK;
}

}  // namespace

extern "C" {

int mvm_seq_scan_validate(const mvm_seq_scan_desc* desc) {
  const int rc = check_scan(desc);
  return rc == MVM_OK ? ok() : rc;
}

int64_t mvm_seq_scan_ckpt_elems(const mvm_seq_scan_desc* desc) {
  const int rc = check_scan(desc);
  return rc == MVM_OK ? ckpt_elems(desc) : rc;
}

int64_t mvm_seq_scan_workspace_bytes(const mvm_seq_scan_desc* desc, int which) {
  const int rc = check_scan(desc);
  if (rc != MVM_OK) return rc;
  if (which != 0 && which != 1) return fail(MVM_ERR_INVALID_ARG, "which=%d must be 0 or 1", which);
  return static_cast<int64_t>(scan_ws(desc, scan_geom(desc, which == 1), which == 1).total);
}

int mvm_seq_scan_fwd(const mvm_seq_scan_desc* desc, const void* u, const void* delta, const float* delta_bias,
                     const float* A, const void* Bm, const void* Cm, const float* Dv, const void* z, const float* h0,
                     float* h1, void* y, float* ckpt, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_scan(desc);
  if (rc != MVM_OK) return rc;
  const mvm::SeqScanGeom g = scan_geom(desc, false);
  if (g.q.D == 0 || (g.q.T == 0 && g.q.S == 0)) return ok();
  const mvm::SeqScanIn in{u, delta, delta_bias, A, Bm, Cm, Dv, z};
  if (!A || !Dv || (g.q.T > 0 && (missing(in) || !y)))
    return fail(MVM_ERR_INVALID_ARG, "mvm_seq_scan_fwd: NULL pointer");
  if ((rc = check_ckpt("mvm_seq_scan_fwd", ckpt)) != MVM_OK) return rc;
  const ScanWs w = scan_ws(desc, g, false);
  if ((rc = check_ws("mvm_seq_scan_fwd", workspace, workspace_bytes, w.total)) != MVM_OK) return rc;
  Take take{static_cast<char*>(workspace)};
  mvm::SeqScanFwd b{h0, h1, y, ckpt, take(w.agg_h), take(w.agg_s), take(w.bc)};
  if (mvm::seq_bc_in_place(g, in, desc->dtype)) b.bc = nullptr;
  return hip_status(mvm::launch_seq_scan_fwd(g, in, b, desc->dtype, desc->delta_dtype, static_cast<hipStream_t>(stream)),
                    "mvm_seq_scan_fwd launch");
}

int mvm_seq_scan_bwd(const mvm_seq_scan_desc* desc, const void* u, const void* delta, const float* delta_bias,
                     const float* A, const void* Bm, const void* Cm, const float* Dv, const void* z, const float* ckpt,
                     const void* dy, const float* dh1, void* du, void* ddelta, float* ddelta_bias, float* dA, void* dB,
                     void* dC, float* dD, void* dz, float* dh0, void* workspace, size_t workspace_bytes,
                     void* stream) {
  int rc = check_scan(desc);
  if (rc != MVM_OK || (rc = check_plain(desc->seq)) != MVM_OK) return rc;
  const mvm::SeqScanGeom g = scan_geom(desc, true);
  const mvm::SeqScanIn in{u, delta, delta_bias, A, Bm, Cm, Dv, z};
  if (g.q.D == 0) {  // (dB and dC are sums over no channels)
    if (g.q.T > 0 && (!dB || !dC)) return fail(MVM_ERR_INVALID_ARG, "mvm_seq_scan_bwd: NULL pointer");
    mvm::SeqScanBwd b{};
    b.dB = dB; b.dC = dC;
    return hip_status(mvm::launch_seq_scan_bwd(g, in, b, desc->dtype, desc->delta_dtype,
                                               static_cast<hipStream_t>(stream)),
                      "mvm_seq_scan_bwd launch");
  }
  if (!A || !Dv || !dA || !dD ||
      (g.q.T > 0 && (missing(in) || !ckpt || !dy || !du || !ddelta || !dB || !dC || (z != nullptr) != (dz != nullptr))))
    return fail(MVM_ERR_INVALID_ARG, "mvm_seq_scan_bwd: NULL pointer");
  if ((rc = check_ckpt("mvm_seq_scan_bwd", ckpt)) != MVM_OK) return rc;
  const ScanWs w = scan_ws(desc, g, true);
  if ((rc = check_ws("mvm_seq_scan_bwd", workspace, workspace_bytes, w.total)) != MVM_OK) return rc;
  Take take{static_cast<char*>(workspace)};
  mvm::SeqScanBwd b{};
  b.ckpt = ckpt; b.dy = dy; b.dh1 = dh1; b.du = du; b.ddelta = ddelta; b.ddbias = ddelta_bias; b.dA = dA;
  b.dB = dB; b.dC = dC; b.dD = dD; b.dz = dz; b.dh0 = dh0;
  b.agg_h = take(w.agg_h);
  b.agg_s = take(w.agg_s);
  b.bc = take(w.bc);
  if (mvm::seq_bc_in_place(g, in, desc->dtype)) b.bc = nullptr;
  b.part = take(w.part);
  b.part_bc = take(w.part_bc);
  return hip_status(mvm::launch_seq_scan_bwd(g, in, b, desc->dtype, desc->delta_dtype, static_cast<hipStream_t>(stream)),
                    "mvm_seq_scan_bwd launch");
}

int mvm_seq_scan_step(const mvm_seq_scan_desc* desc, const void* u, const void* delta, const float* delta_bias,
                      const float* A, const void* Bm, const void* Cm, const float* Dv, const void* z, float* states,
                      void* y, void* stream) {
  int rc = check_scan(desc);
  if (rc != MVM_OK || (rc = check_step(desc->seq)) != MVM_OK) return rc;
  const mvm::SeqScanGeom g = scan_geom(desc, false);
  if ((rc = check_threads(desc->seq, g.q.S, ceil_div(g.q.D, 64) * 256)) != MVM_OK) return rc;
  if (g.q.D == 0 || g.q.S == 0) return ok();
  const mvm::SeqScanIn in{u, delta, delta_bias, A, Bm, Cm, Dv, z};
  if (missing(in) || !states || !y) return fail(MVM_ERR_INVALID_ARG, "mvm_seq_scan_step: NULL pointer");
  return hip_status(mvm::launch_seq_scan_step(g, in, states, y, desc->dtype, desc->delta_dtype,
                                              static_cast<hipStream_t>(stream)),
                    "mvm_seq_scan_step launch");
}

int mvm_seq_conv_validate(const mvm_seq_conv_desc* desc) {
  const int rc = check_conv(desc);
  return rc == MVM_OK ? ok() : rc;
}

int64_t mvm_seq_conv_workspace_bytes(const mvm_seq_conv_desc* desc) {
  const int rc = check_conv(desc);
  if (rc != MVM_OK) return rc;
  return static_cast<int64_t>(align_up(sizeof(float) * mvm::seq_conv_partial_floats(conv_geom(desc))));
}

int mvm_seq_conv_fwd(const mvm_seq_conv_desc* desc, const void* x, const float* w, const float* bias, const void* c0,
                     void* c1, void* y, void* stream) {
  const int rc = check_conv(desc);
  if (rc != MVM_OK) return rc;
  const mvm::SeqConvGeom g = conv_geom(desc);
  if (g.q.D == 0 || (g.q.T == 0 && g.q.S == 0)) return ok();
  if (!w || (g.q.T > 0 && (!x || !y))) return fail(MVM_ERR_INVALID_ARG, "mvm_seq_conv_fwd: NULL pointer");
  return hip_status(mvm::launch_seq_conv_fwd(g, x, w, bias, c0, c1, y, desc->dtype, static_cast<hipStream_t>(stream)),
                    "mvm_seq_conv_fwd launch");
}

int mvm_seq_conv_bwd(const mvm_seq_conv_desc* desc, const void* x, const float* w, const float* bias, const void* c0,
                     const void* dy, const void* dc1, void* dx, float* dw, float* dbias, void* dc0, void* workspace,
                     size_t workspace_bytes, void* stream) {
  int rc = check_conv(desc);
  if (rc != MVM_OK || (rc = check_plain(desc->seq)) != MVM_OK) return rc;
  const mvm::SeqConvGeom g = conv_geom(desc);
  if (g.q.D == 0) return ok();
  if (!w || !dw || (g.q.T > 0 && (!x || !dy || !dx)))
    return fail(MVM_ERR_INVALID_ARG, "mvm_seq_conv_bwd: NULL pointer");
  const size_t need = align_up(sizeof(float) * mvm::seq_conv_partial_floats(g));
  if ((rc = check_ws("mvm_seq_conv_bwd", workspace, workspace_bytes, need)) != MVM_OK) return rc;
  return hip_status(mvm::launch_seq_conv_bwd(g, x, w, bias, c0, dy, dc1, dx, dw, dbias, dc0,
                                             static_cast<float*>(workspace), desc->dtype,
                                             static_cast<hipStream_t>(stream)),
                    "mvm_seq_conv_bwd launch");
}

int mvm_seq_conv_step(const mvm_seq_conv_desc* desc, const void* x, const float* w, const float* bias, void* states,
                      void* y, void* stream) {
  int rc = check_conv(desc);
  if (rc != MVM_OK || (rc = check_step(desc->seq)) != MVM_OK) return rc;
  const mvm::SeqConvGeom g = conv_geom(desc);
  if (g.q.D == 0 || g.q.S == 0) return ok();
  if (!x || !w || !y || (!states && g.kc > 1)) return fail(MVM_ERR_INVALID_ARG, "mvm_seq_conv_step: NULL pointer");
  return hip_status(mvm::launch_seq_conv_step(g, x, w, bias, states, y, desc->dtype, static_cast<hipStream_t>(stream)),
                    "mvm_seq_conv_step launch");
}

}  // extern "C"
