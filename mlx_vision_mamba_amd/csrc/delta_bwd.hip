// Gradients of the gated delta rule, by chunks of 64 tokens (delta_fwd.hip has
// the forward's equations; dO' = scale dO, D: rows d_t, E: the gradient of the
// chunk's final state S').
//
// Along time, from the last chunk to the first (delta_bwd_kernel):
//   dD = P' dO + diag(e^(Gc - G)) K E
//   X  = T' dD
//   dS = e^Gc E + Q' diag(e^G) dO' - K' diag(beta e^G) X
// the same chain of products as the forward's, with a wave keeping 16 columns
// of E in registers.  It leaves X and every chunk's E.
//
// Then every chunk and key head by itself (delta_grads_kernel), with M_ij =
// exp(G_i - G_j):
//   dv_i    = beta_i X_i
//   u_i     = -e^(G_i) S X_i - sum_{j < i} M_ij (X_i . D_j) k_j
//   dbeta_i = X_i . v_i + k_i . u_i
//   dq_i    = scale (e^(G_i) S dO_i + sum_{j <= i} M_ij (dO_i . D_j) k_j)
//   dk_i    = beta_i u_i + e^(Gc - G_i) E D_i - sum_{j > i} M_ji beta_j (X_j . D_i) k_j
//             + scale sum_{j >= i} M_ji (dO_j . D_i) q_j
//   dG_i    = q_i . dq_i - k_i . dk_i + 2 beta_i k_i . u_i
//   dg_t    = sum_{i >= t} dG_i + sum_i e^(Gc - G_i) k_i . E D_i + e^Gc <S, E>
// where dG collects, for each factor exp(G_i), the gradients' own products, and
// the last two terms are those of the factor exp(Gc).  All products are formed
// with the token as the result's column: then the small triangles are B
// operands as they come out, a token's scalars are a lane's, and a lane holds
// four consecutive values of dq and dk.
#include "delta_common.h"

namespace mvm {
namespace {

struct BwdArgs {
  DeltaGeom g;
  DeltaIn in;
  DeltaWork w;
  DeltaBwd b;
  uint32_t vcb, ncb, nslots;  // column blocks of the values, and of the launch
};

// AGG: a part's gradient of its initial state from zero, and (column blocks
// from a.vcb on) its transition: what the identity becomes where dO is zero.
template <typename T, int DKP, int NW, bool VEC, bool AGG>
__global__ void __launch_bounds__(64 * NW)
delta_bwd_kernel(BwdArgs a) {
  constexpr int P = kRawParts<T>, KT = DKP / 16, KS = DKP / 32, NT = 64 * NW;
  __shared__ __attribute__((aligned(16))) Tile<kC, DKP, P> sK, sQ;
  __shared__ uint4 sTri[StageTri<3, NT>::kCount];
  __shared__ __attribute__((aligned(16))) float sDec[4][kC];
  const DeltaGeom& g = a.g;
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_id(), m = lane & 15, grp = lane >> 4;
  const DeltaPos p = delta_pos(a.ncb, a.nslots, static_cast<uint32_t>(g.HV));
  if (!p.ok) return;
  const int h = p.h, hk = h / g.group;
  const bool trans = AGG && p.cb >= static_cast<int32_t>(a.vcb);
  const int col0 = ((trans ? p.cb - static_cast<int32_t>(a.vcb) : p.cb) * NW + wave) * 16, col = col0 + m;
  const bool live = trans ? col < DKP : col < g.DV;
  const int at_col = col0 < g.DV ? col0 : 0;  // (waves without columns address the first)
  const SeqChunk part = seq_chunk(g.q, p.slot, g.part, lane);
  if (part.t0 < 0 || part.seq >= g.q.S || (AGG && part.t0 == part.start)) return;  // (nothing precedes a first part)
  const int64_t cells = static_cast<int64_t>(g.DK) * g.DV;
  const int64_t at_h = (static_cast<int64_t>(part.seq) * g.HV + h) * cells + at_col;
  const int64_t at_part = (static_cast<int64_t>(p.slot) * g.HV + h) * cells + at_col;
  f32x4 E[KT];
  if (trans) {
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) E[t][r] = 16 * t + 4 * grp + r == col ? 1.f : 0.f;
  } else {
    const float* src = AGG ? nullptr : a.w.carry != nullptr ? a.w.carry + at_part : a.b.dh1 != nullptr ? a.b.dh1 + at_h : nullptr;
    load_state<KT>(E, src, g.DV, src != nullptr ? g.DK : 0, m, grp, live);
  }
  const T* kp = static_cast<const T*>(a.in.k) + hk * g.kh;
  const T* qp = static_cast<const T*>(a.in.q) + hk * g.qh;
  const int64_t orow = static_cast<int64_t>(g.HV) * g.DV, ocol = static_cast<int64_t>(h) * g.DV + at_col;
  const T* dop = static_cast<const T*>(a.b.d_o) + ocol;
  const bool vlive = live && !trans;
  const int32_t slot0 = cut_div(g.cut, part.start) + part.seq + (part.t0 - part.start) / kC;
  const int32_t chunks = (part.t1 - part.t0 + kC - 1) / kC;
  StageRows<T, DKP, NT> rK, rQ;
  StageTri<3, NT> rT;
  float rDec;
  float rGam;
  Cols<T> rO;
  const auto load = [&](int32_t i) {
    const int32_t t0 = part.t0 + i * kC;
    const int n = part.t1 - t0 < kC ? part.t1 - t0 : kC;
    const int64_t at = static_cast<int64_t>(slot0 + i) * g.HV + h;
    rK.template load<VEC>(kp + t0 * g.ks, g.ks, n, g.DK, tid);
    rQ.template load<VEC>(qp + t0 * g.qs, g.qs, n, g.DK, tid);
    rT.load(reinterpret_cast<const uint4*>(a.w.tri) + at * kTriFragments, tid);
    if (tid < 4 * kC) rDec = a.w.dec[at * (4 * kC) + tid];
    rGam = a.w.gam[at];
  };
  const auto load_o = [&](int32_t i) {
    const int32_t t0 = part.t0 + i * kC;
    rO.load(dop + t0 * orow, orow, m, grp, part.t1 - t0 < kC ? part.t1 - t0 : kC, vlive);
  };
  if (chunks > 0) load(chunks - 1), load_o(chunks - 1);
  for (int32_t nth = chunks - 1; nth >= 0; --nth) {
    const int32_t t0 = part.t0 + nth * kC;
    const int n = part.t1 - t0 < kC ? part.t1 - t0 : kC;
    const int64_t at = static_cast<int64_t>(slot0 + nth) * g.HV + h;
    __syncthreads();
    rK.put(sK, n, g.DK, tid);
    rQ.put(sQ, n, g.DK, tid);
    rT.put(sTri, tid);
    if (tid < 4 * kC) sDec[0][tid] = rDec;
    const float gam = rGam;
    if (nth > 0) load(nth - 1);
    if constexpr (!AGG) store_state<KT>(a.b.dend + at * cells + at_col, g.DV, g.DK, E, m, grp, live);
    __syncthreads();
    f32x4 D[4], X[4], O[4];
#pragma unroll
    for (int rt = 0; rt < 4; ++rt) D[rt] = X[rt] = f32x4{0.f, 0.f, 0.f, 0.f};
    Frag<P> fk[2][4];
    const auto rows = [&](int ks) {
#pragma unroll
      for (int rt = 0; rt < 4; ++rt) fk[ks & 1][rt] = sK.rows(16 * rt + m, 32 * ks + 4 * grp);
    };
    Frag<3> ft[2][2];
    const auto tri = [&](int which, int rt) {
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
        if (tri_frag<true>(rt, ks) >= 0) ft[rt & 1][ks] = tri_at<3>(sTri, which, tri_frag<true>(rt, ks), lane);
    };
    f32x4 up[4];
    rows(0);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      if (ks + 1 < KS)
        rows(ks + 1);
      else
#pragma unroll
        for (int rt = 0; rt < 4; ++rt) up[rt] = dec_at(sDec, kDecUp, rt, grp);
      const Frag<3> ef = split_tiles<3>(E[2 * ks], E[2 * ks + 1]);
#pragma unroll
      for (int rt = 0; rt < 4; ++rt) D[rt] = mma<3>(fk[ks & 1][rt], ef, D[rt]);
      phase();
    }
    tri(1, 0);
    tri(1, 1);
#pragma unroll
    for (int rt = 0; rt < 4; ++rt) {
      O[rt] = rO.tile(rt, grp, n, vlive);
      D[rt] *= up[rt];
    }
    if (nth > 0) load_o(nth - 1);
    {
      const Frag<P> of[2] = {split_tiles<P>(O[0], O[1]), split_tiles<P>(O[2], O[3])};
      phase();
#pragma unroll
      for (int rt = 0; rt < 4; ++rt) {
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
          if (tri_frag<true>(rt, ks) >= 0) D[rt] = mma<3>(ft[rt & 1][ks], of[ks], D[rt]);
        phase();
        tri(rt < 2 ? 1 : 0, rt < 2 ? rt + 2 : rt - 2);
      }
    }
    f32x4 dx[4], dout[4];
    {
      const Frag<3> df[2] = {split_tiles<3>(D[0], D[1]), split_tiles<3>(D[2], D[3])};
#pragma unroll
      for (int rt = 0; rt < 4; ++rt) {
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
          if (tri_frag<true>(rt, ks) >= 0) X[rt] = mma<3>(ft[rt & 1][ks], df[ks], X[rt]);
        phase();
        if (rt < 2) tri(0, rt + 2);
        dx[rt] = dec_at(sDec, kDecBetaKey, rt, grp);
        dout[rt] = dec_at(sDec, kDecOut, rt, grp);
      }
    }
    if constexpr (!AGG) store_cols<float>(a.b.x + t0 * orow + ocol, orow, X, m, grp, n, live);
    Frag<P> fc[2][2], fd[2][2];
    const auto keys = [&](int t) {
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        fc[t & 1][ks] = sK.cols(16 * t, 32 * ks + 4 * grp, m);
        fd[t & 1][ks] = sQ.cols(16 * t, 32 * ks + 4 * grp, m);
      }
    };
    keys(0);
#pragma unroll
    for (int rt = 0; rt < 4; ++rt) {
      X[rt] *= -dx[rt];
      O[rt] *= dout[rt];
    }
    const Frag<3> xf[2] = {split_tiles<3>(X[0], X[1]), split_tiles<3>(X[2], X[3])};
    const Frag<3> of[2] = {split_tiles<3>(O[0], O[1]), split_tiles<3>(O[2], O[3])};
    phase();
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      if (t + 1 < KT) keys(t + 1);
      E[t] *= gam;
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        E[t] = mma<3>(fc[t & 1][ks], xf[ks], E[t]);
        E[t] = mma<3>(fd[t & 1][ks], of[ks], E[t]);
      }
      phase();
    }
  }
  if (AGG && trans)
    store_state<KT>(a.w.trans + (static_cast<int64_t>(p.slot) * g.HV + h) * (DKP * DKP) + col0, DKP, DKP, E, m, grp, live);
  else if (AGG)
    store_state<KT>(a.w.carry + at_part, g.DV, g.DK, E, m, grp, live);
  else if (a.b.dh0 != nullptr && part.t0 == part.start)
    store_state<KT>(a.b.dh0 + at_h, g.DV, g.DK, E, m, grp, live);
}

// Zeros in the gradients of the rows that belong to no sequence.
template <typename T>
__device__ void zero_rows(const BwdArgs& a, int32_t t0, int32_t t1, int hk, int tid) {
  const DeltaGeom& g = a.g;
  for (int32_t t = t0; t < t1; ++t) {
    for (int c = tid; c < g.DK; c += 256) {
      const int64_t i = (static_cast<int64_t>(t) * g.HK + hk) * g.DK + c;
      static_cast<T*>(a.b.dq)[i] = from_f32<T>(0.f);
      static_cast<T*>(a.b.dk)[i] = from_f32<T>(0.f);
    }
    for (int c = tid; c < g.group * g.DV; c += 256)
      static_cast<T*>(a.b.dv)[(static_cast<int64_t>(t) * g.HV + hk * g.group) * g.DV + c] = from_f32<T>(0.f);
    for (int c = tid; c < g.group; c += 256) {
      const int64_t i = static_cast<int64_t>(t) * g.HV + hk * g.group + c;
      a.b.dg[i] = 0.f;
      if (g.beta_f32)
        static_cast<float*>(a.b.dbeta)[i] = 0.f;
      else
        static_cast<T*>(a.b.dbeta)[i] = from_f32<T>(0.f);
    }
  }
}

template <typename T, int DKP, bool VEC>
__global__ void __launch_bounds__(256)
delta_grads_kernel(BwdArgs a) {
  constexpr int P = kRawParts<T>, KT = DKP / 16;
  struct Rows {  // 32 columns of the values' side
    Tile<kC, 32, 3> X, D;
    Tile<kC, 32, P> O;
    Tile<DKP, 32, 3> S, E;
  };
  struct Keys {
    Tile<kC, DKP, P> K, Q;
  };
  __shared__ __attribute__((aligned(16))) union { Rows r; Keys k; } sm;
  __shared__ double sG[kC], sDG[kC];
  __shared__ float sBeta[kC], sRk[kC], sRq[kC], sXv[kC], sSum[4][2];
  const DeltaGeom& g = a.g;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, m = lane & 15, grp = lane >> 4;
  const uint32_t slot = blockIdx.x / static_cast<uint32_t>(g.HK);
  const int hk = static_cast<int>(blockIdx.x - slot * static_cast<uint32_t>(g.HK));
  const SeqChunk c = seq_chunk(g.q, static_cast<int32_t>(slot), g.cut, lane);
  if (c.t0 < 0 || c.t1 == c.t0) return;
  if (c.seq >= g.q.S) return zero_rows<T>(a, c.t0, c.t1, hk, tid);
  const int n = c.t1 - c.t0;
  const int64_t orow = static_cast<int64_t>(g.HV) * g.DV, cells = static_cast<int64_t>(g.DK) * g.DV;
  const bool vec4 = g.DV % 4 == 0;
  const f32x4 z4 = {0.f, 0.f, 0.f, 0.f};
  const int ti = 16 * wave + m;  // this lane's token
  f32x4 sumQ[KT], sumK[KT];
#pragma unroll
  for (int t = 0; t < KT; ++t) sumQ[t] = sumK[t] = z4;
  for (int hg = 0; hg < g.group; ++hg) {
    const int h = hk * g.group + hg;
    const int64_t at = static_cast<int64_t>(slot) * g.HV + h;
    __syncthreads();
    const double G = log_decay(g, a.in.g, c.t0, n, h, lane);
    if (wave == 0) {
      sG[lane] = G;
      sBeta[lane] = lane < n ? load_beta<T>(g, a.in.beta, c.t0 + lane, h) : 0.f;
    }
    const double Gc = __shfl(G, 63);
    f32x4 accQ[KT], accU[KT], accK[KT];
#pragma unroll
    for (int t = 0; t < KT; ++t) accQ[t] = accU[t] = accK[t] = z4;
    // rows j of a tile, column the lane's token i: D_j . dO_i and D_j . X_i for j <= i, X_j . D_i and dO_j . D_i
    // for j >= i
    f32x4 DO[4], DX[4], XD[4], OD[4];
#pragma unroll
    for (int jt = 0; jt < 4; ++jt) DO[jt] = DX[jt] = XD[jt] = OD[jt] = z4;
    float xv = 0.f, se = 0.f;
    const int row = tid >> 2, cc = (tid & 3) * 8;
    const bool in_row = row < n;
    const int64_t vat = (c.t0 + (in_row ? row : 0)) * orow + static_cast<int64_t>(h) * g.DV;
    const float brow = in_row ? load_beta<T>(g, a.in.beta, c.t0 + row, h) : 0.f;
    const T* vrow = static_cast<const T*>(a.in.v) + (c.t0 + static_cast<int64_t>(in_row ? row : 0)) * g.vs + h * g.vh;
    for (int kb = 0; kb < g.DV; kb += 32) {
      __syncthreads();
      {
        const int lim = in_row ? g.DV : 0;
        float x[8], v[8];
        load8f(x, a.b.x + vat, kb + cc, lim, vec4);
        load8f(v, vrow, kb + cc, lim, g.v_vec);
        sm.r.X.put(row, cc, split8<3>(x));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          xv = fmaf(x[i], v[i], xv);
          x[i] *= brow;
        }
        store8(static_cast<T*>(a.b.dv) + vat, kb + cc, lim, a.b.o_vec, x);
        load8f(v, a.b.vt + vat, kb + cc, lim, vec4);
        sm.r.D.put(row, cc, split8<3>(v));
        sm.r.O.put(row, cc, load8(static_cast<const T*>(a.b.d_o) + vat, kb + cc, lim, a.b.o_vec));
      }
#pragma unroll
      for (int i = 0; i < DKP / 64 + (DKP < 64); ++i) {
        const int d = row + 64 * i;
        if (DKP < 64 && d >= DKP) break;
        const int lim = d < g.DK ? g.DV : 0;
        const int64_t sat = at * cells + static_cast<int64_t>(d < g.DK ? d : 0) * g.DV;
        float s[8], e[8];
        load8f(s, a.b.s0 + sat, kb + cc, lim, vec4);
        load8f(e, a.b.dend + sat, kb + cc, lim, vec4);
#pragma unroll
        for (int j = 0; j < 8; ++j) se = fmaf(s[j], e[j], se);
        sm.r.S.put(d, cc, split8<3>(s));
        sm.r.E.put(d, cc, split8<3>(e));
      }
      __syncthreads();
      const int k0 = 8 * grp;
      const Frag<3> bX = sm.r.X.rows_plain(ti, k0), bD = sm.r.D.rows_plain(ti, k0);
      const Frag<P> bO = sm.r.O.rows_plain(ti, k0);
#pragma unroll
      for (int jt = 0; jt < 4; ++jt) {
        if (jt <= wave) {
          const Frag<3> f = sm.r.D.rows_plain(16 * jt + m, k0);
          DO[jt] = mma<3>(f, bO, DO[jt]);
          DX[jt] = mma<3>(f, bX, DX[jt]);
        }
        if (jt >= wave) {
          XD[jt] = mma<3>(sm.r.X.rows_plain(16 * jt + m, k0), bD, XD[jt]);
          OD[jt] = mma<3>(sm.r.O.rows_plain(16 * jt + m, k0), bD, OD[jt]);
        }
      }
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        const Frag<3> f = sm.r.S.rows_plain(16 * t + m, k0);
        accQ[t] = mma<3>(f, bO, accQ[t]);
        accU[t] = mma<3>(f, bX, accU[t]);
        accK[t] = mma<3>(sm.r.E.rows_plain(16 * t + m, k0), bD, accK[t]);
      }
    }
    xv += __shfl_xor(xv, 1);
    xv += __shfl_xor(xv, 2);
    if ((tid & 3) == 0) sXv[row] = xv;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) se += __shfl_xor(se, o);
    __syncthreads();
    {
      StageRows<T, DKP, 256> rK, rQ;
      rK.template load<VEC>(static_cast<const T*>(a.in.k) + c.t0 * g.ks + hk * g.kh, g.ks, n, g.DK, tid);
      rQ.template load<VEC>(static_cast<const T*>(a.in.q) + c.t0 * g.qs + hk * g.qh, g.qs, n, g.DK, tid);
      rK.put(sm.k.K, n, g.DK, tid);
      rQ.put(sm.k.Q, n, g.DK, tid);
    }
    __syncthreads();
    {
      float nk = 0.f, nq = 0.f;
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        const f32x4 x = sm.k.K.get4(ti, 16 * t + 4 * grp), y = sm.k.Q.get4(ti, 16 * t + 4 * grp);
#pragma unroll
        for (int r = 0; r < 4; ++r) nk = fmaf(x[r], x[r], nk), nq = fmaf(y[r], y[r], nq);
      }
      nk = sum_g(nk);
      nq = sum_g(nq);
      if (grp == 0) {
        sRk[ti] = g.l2 ? 1.f / sqrtf(nk + kL2Eps) : 1.f;
        sRq[ti] = g.l2 ? 1.f / sqrtf(nq + kL2Eps) : 1.f;
      }
    }
    __syncthreads();
    const double Gi = sG[ti];
    const float eG = exp_diff(Gi), eR = exp_diff(Gc - Gi), bi = sBeta[ti], rk = sRk[ti], rq = sRq[ti];
    float kh = 0.f;
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      accQ[t] *= g.scale * eG;
      accU[t] *= -eG;
      accK[t] *= eR;
      const f32x4 x = sm.k.K.get4(ti, 16 * t + 4 * grp);
#pragma unroll
      for (int r = 0; r < 4; ++r) kh = fmaf(accK[t][r], x[r], kh);
    }
#pragma unroll
    for (int jt = 0; jt < 4; ++jt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int j = 16 * jt + 4 * grp + r;
        const double Gj = sG[j];
        const float lo = j <= ti ? exp_diff(Gi - Gj) : 0.f, hi = j >= ti ? exp_diff(Gj - Gi) : 0.f;
        DO[jt][r] *= j <= ti ? g.scale * sRk[j] * lo : 0.f;
        DX[jt][r] *= j < ti ? -sRk[j] * lo : 0.f;
        XD[jt][r] *= j > ti ? -sBeta[j] * sRk[j] * hi : 0.f;
        OD[jt][r] *= j >= ti ? g.scale * sRq[j] * hi : 0.f;
      }
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const int j0 = 32 * ks + 4 * grp;
      if (2 * ks <= wave) {
        const Frag<3> f1 = split_tiles<3>(DO[2 * ks], DO[2 * ks + 1]), f2 = split_tiles<3>(DX[2 * ks], DX[2 * ks + 1]);
#pragma unroll
        for (int t = 0; t < KT; ++t) {
          const Frag<P> k = sm.k.K.cols(16 * t, j0, m);
          accQ[t] = mma<3>(k, f1, accQ[t]);
          accU[t] = mma<3>(k, f2, accU[t]);
        }
      }
      if (2 * ks + 1 >= wave) {
        const Frag<3> f1 = split_tiles<3>(XD[2 * ks], XD[2 * ks + 1]), f2 = split_tiles<3>(OD[2 * ks], OD[2 * ks + 1]);
#pragma unroll
        for (int t = 0; t < KT; ++t) {
          accK[t] = mma<3>(sm.k.K.cols(16 * t, j0, m), f1, accK[t]);
          accK[t] = mma<3>(sm.k.Q.cols(16 * t, j0, m), f2, accK[t]);
        }
      }
    }
    float ku = 0.f, qd = 0.f, kd = 0.f;
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      const f32x4 x = sm.k.K.get4(ti, 16 * t + 4 * grp), y = sm.k.Q.get4(ti, 16 * t + 4 * grp);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        ku = fmaf(accU[t][r], x[r], ku);
        accK[t][r] = fmaf(bi, accU[t][r], accK[t][r]);
        kd = fmaf(accK[t][r], x[r], kd);
        qd = fmaf(accQ[t][r], y[r], qd);
      }
      sumQ[t] += accQ[t];
      sumK[t] += accK[t];
    }
    ku = sum_g(ku) * rk;
    kd = sum_g(kd) * rk;
    qd = sum_g(qd) * rq;
    kh = sum_g(kh) * rk;
    if (grp == 0) {
      sDG[ti] = static_cast<double>(qd) - kd + 2.f * bi * ku;
      if (ti < n) {
        const float db = sXv[ti] + ku;
        const int64_t i = (c.t0 + static_cast<int64_t>(ti)) * g.HV + h;
        if (g.beta_f32)
          static_cast<float*>(a.b.dbeta)[i] = db;
        else
          static_cast<T*>(a.b.dbeta)[i] = from_f32<T>(db);
      }
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) kh += __shfl_xor(kh, o);
    if (lane == 0) {
      sSum[wave][0] = se;
      sSum[wave][1] = kh;
    }
    __syncthreads();
    if (wave == 0) {
      double s = sDG[63 - lane];
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const double v = __shfl_up(s, o);
        if (lane >= o) s += v;
      }
      const double all = static_cast<double>(exp_diff(Gc)) * ((sSum[0][0] + sSum[1][0]) + (sSum[2][0] + sSum[3][0])) +
                         ((sSum[0][1] + sSum[1][1]) + (sSum[2][1] + sSum[3][1]));
      if (63 - lane < n) a.b.dg[(c.t0 + 63 - lane) * static_cast<int64_t>(g.HV) + h] = static_cast<float>(s + all);
    }
  }
  // (the keys of the last head are still in LDS)
  float qd = 0.f, kd = 0.f;
  const float rk = sRk[ti], rq = sRq[ti];
  if (g.l2) {
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      const f32x4 x = sm.k.K.get4(ti, 16 * t + 4 * grp), y = sm.k.Q.get4(ti, 16 * t + 4 * grp);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        kd = fmaf(sumK[t][r], x[r], kd);
        qd = fmaf(sumQ[t][r], y[r], qd);
      }
    }
    kd = sum_g(kd) * rk * rk;
    qd = sum_g(qd) * rq * rq;
  }
  if (ti >= n) return;
  const int64_t out = ((c.t0 + static_cast<int64_t>(ti)) * g.HK + hk) * g.DK;
#pragma unroll
  for (int t = 0; t < KT; ++t) {
    const f32x4 x = sm.k.K.get4(ti, 16 * t + 4 * grp), y = sm.k.Q.get4(ti, 16 * t + 4 * grp);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int d = 16 * t + 4 * grp + r;
      if (d < g.DK) {
        static_cast<T*>(a.b.dk)[out + d] = from_f32<T>(rk * fmaf(-kd, x[r], sumK[t][r]));
        static_cast<T*>(a.b.dq)[out + d] = from_f32<T>(rq * fmaf(-qd, y[r], sumQ[t][r]));
      }
    }
  }
}

}  // namespace

hipError_t launch_delta_bwd(const DeltaGeom& g, const DeltaIn& in, const DeltaWork& w, const DeltaBwd& b, int dtype,
                            hipStream_t s) {
  // (rows that are read value by value: more registers, so four waves)
  const int nw = g.qk_vec ? delta_waves(g.DV) : 4;
  const uint32_t vcb = delta_col_blocks(g.DV, nw);
  BwdArgs a{g, in, w, b, vcb, vcb, static_cast<uint32_t>(chunk_slots(g.q, g.part))};
  hipError_t e = launch_delta_prep(g, in, w, true, dtype, s);
  if (e != hipSuccess) return e;
  const auto run = [&](auto t, auto dkp, auto waves, auto vec) {
    using T = decltype(t);
    constexpr int DKP = decltype(dkp)::value, NW = decltype(waves)::value;
    constexpr bool VEC = decltype(vec)::value;
    hipError_t e;
    if (g.parts > 1) {
      a.ncb = vcb + delta_col_blocks(DKP, NW);
      hipLaunchKernelGGL((delta_bwd_kernel<T, DKP, NW, VEC, true>),
                         dim3(static_cast<unsigned>(delta_blocks(a.ncb, a.nslots, g.HV))), dim3(64 * NW), 0, s, a);
      if ((e = hipGetLastError()) != hipSuccess || (e = launch_delta_carry<true>(g, w, b.dh1, s)) != hipSuccess) return e;
      a.ncb = vcb;
    }
    hipLaunchKernelGGL((delta_bwd_kernel<T, DKP, NW, VEC, false>),
                       dim3(static_cast<unsigned>(delta_blocks(a.ncb, a.nslots, g.HV))), dim3(64 * NW), 0, s, a);
    e = hipGetLastError();
    if (e != hipSuccess || g.q.T == 0) return e;
    hipLaunchKernelGGL((delta_grads_kernel<T, DKP, VEC>), dim3(static_cast<unsigned>(chunk_slots(g.q, g.cut) * g.HK)),
                       dim3(256), 0, s, a);
    return hipGetLastError();
  };
  return delta_dispatch(dtype, g.DK, [&](auto t, auto dkp) {
    using Four = std::integral_constant<int, 4>;
    if (!g.qk_vec) return run(t, dkp, Four{}, std::false_type{});
    return nw == 8 ? run(t, dkp, std::integral_constant<int, 8>{}, std::true_type{}) : run(t, dkp, Four{}, std::true_type{});
  });
}

}  // namespace mvm
