// Gradients of the gated delta rule, by chunks of 64 tokens (delta_fwd.hip has
// the forward's equations; dO' = scale dO, D: rows d_t, E: the gradient of the
// chunk's final state S').
//
// Along time, from the last chunk to the first (delta_bwd_kernel):
//   dD = P' dO + diag(e^(Gc - G)) K E
//   X  = T' dD
//   dS = e^Gc E + Q' diag(e^G) dO' - K' diag(beta e^G) X
// the same chain of products as the forward's, with a wave keeping 16 columns
// of E in registers.  It leaves X and every chunk's E.  (16384 tokens of 12 heads of
// 128 x 128 in bfloat16: 136 us, as bound as the forward's.)
//
// Then every chunk and key head by itself (delta_grads_kernel), with M_ij =
// exp(G_i - G_j):
//   dv_i    = beta_i X_i
//   u_i     = -e^(G_i) S X_i - sum_{j < i} M_ij (X_i . D_j) k_j
//   dbeta_i = X_i . v_i + k_i . u_i
//   dq_i    = scale (e^(G_i) S dO_i + sum_{j <= i} M_ij (dO_i . D_j) k_j)
//   dk_i    = beta_i u_i + e^(Gc - G_i) E D_i - sum_{j > i} M_ji beta_j (X_j . D_i) k_j
//             + scale sum_{j >= i} M_ji (dO_j . D_i) q_j
//   dg_t    = e^Gc <S, E> + sum_{i < t} e^(Gc - G_i) k_i . E D_i
//             + sum_{i >= t} e^(G_i) (scale q_i . S dO_i - beta_i k_i . S X_i)
//             + sum_{j < t <= i} M_ij (scale (dO_i . D_j) (q_i . k_j) - beta_i (X_i . D_j) (k_i . k_j))
// where each product of dg_t has exp(g_t) as a factor, and its sums add, so
// that a gate that lets little through keeps its gradient's digits.  (The same
// sums as differences of q . dq, k . dk and k . u hold products without that
// factor, of which only the rounding is left: 1e-3 of dg at g = -8.)  All
// products are formed with the token as the result's column: then the small
// triangles are B operands as they come out, a token's scalars are a lane's,
// and a lane holds four consecutive values of dq and dk.
#include "delta_common.h"

namespace mvm {
namespace {

struct BwdArgs {
  DeltaGeom g;
  DeltaIn in;
  DeltaWork w;
  DeltaBwd b;
  int64_t col_tiles;
  uint32_t vcb, ncb, nslots;  // column blocks of the values, and of the launch
};

// AGG: a part's gradient of its initial state from zero, and (column blocks
// from a.vcb on) its transition: what the identity becomes where dO is zero.
template <typename T, int DKP, int NW, bool VEC, bool AGG>
__global__ void __launch_bounds__(64 * NW)
delta_bwd_kernel(BwdArgs a) {
  constexpr int P = kRawParts<T>, KT = DKP / 16, KS = DKP / 32, NT = 64 * NW;
  __shared__ __attribute__((aligned(16))) Tile<kC, DKP, P> sK, sQ;
  constexpr bool OLDS = P == 1;  // (as V in the forward)
  __shared__ __attribute__((aligned(16))) Tile<OLDS ? kC : 1, 16 * NW, 1> sO;
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
  const int64_t at_part = ((static_cast<int64_t>(p.slot) * g.HV + h) * a.col_tiles + col0 / 16) * (KT * 256);
  const bool tiles = !trans && col0 < g.DV;
  f32x4 E[KT];
  if (trans) {
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) E[t][r] = 16 * t + 4 * grp + r == col ? 1.f : 0.f;
  } else if (!AGG && a.w.carry != nullptr) {
#pragma unroll
    for (int t = 0; t < KT; ++t)
      E[t] = tiles ? reinterpret_cast<const f32x4*>(a.w.carry + at_part)[64 * t + lane] : f32x4{0.f, 0.f, 0.f, 0.f};
  } else {
    const int32_t on = !AGG && a.b.dh1 != nullptr;
    load_state<KT>(E, a.b.dh1 + on * at_h, g.DV, on * g.DK, m, grp, live);
  }
  const T* kp = static_cast<const T*>(a.in.k) + hk * g.kh;
  const T* qp = static_cast<const T*>(a.in.q) + hk * g.qh;
  const int64_t orow = static_cast<int64_t>(g.HV) * g.DV;
  const int vcol0 = trans ? 0 : p.cb * NW * 16;
  const T* dop = static_cast<const T*>(a.b.d_o) + static_cast<int64_t>(h) * g.DV + (OLDS ? vcol0 : at_col);
  const bool vlive = live && !trans;
  const int32_t slot0 = cut_div(g.cut, part.start) + part.seq + (part.t0 - part.start) / kC;
  const int32_t chunks = (part.t1 - part.t0 + kC - 1) / kC;
  StageRows<T, DKP, NT> rK, rQ;
  StageTri<3, NT> rT;
  float rDec;
  float rGam;
  Cols<T> rO;
  StageRows<T, 16 * NW, NT> rOt;
  // (a few at a time, as in the forward)
  constexpr int kLoads = 8;
  const auto load = [&](int32_t i, int which) {
    const int32_t t0 = part.t0 + i * kC;
    const int n = part.t1 - t0 < kC ? part.t1 - t0 : kC;
    const int64_t at = static_cast<int64_t>(slot0 + i) * g.HV + h;
    switch (which) {
      case 0: rK.template load<VEC>(kp + t0 * g.ks, g.ks, n, g.DK, tid); break;
      case 1: rQ.template load<VEC>(qp + t0 * g.qs, g.qs, n, g.DK, tid); break;
      case 2:
        if constexpr (OLDS) rOt.template load<VEC>(dop + t0 * orow, orow, n, trans ? 0 : g.DV - vcol0, tid);
        break;
      case 3:
        if (tid < 4 * kC) rDec = a.w.dec[at * (4 * kC) + tid];
        rGam = a.w.gam[at];
        break;
      default: rT.load(reinterpret_cast<const uint4*>(a.w.tri) + at * kTriFragments, tid, which - 4, which - 3); break;
    }
  };
  const auto load_o = [&](int32_t i) {
    const int32_t t0 = part.t0 + i * kC;
    rO.load(dop + t0 * orow, orow, m, grp, part.t1 - t0 < kC ? part.t1 - t0 : kC, vlive);
  };
  if (chunks > 0) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) load(chunks - 1, i);
    if constexpr (!OLDS) load_o(chunks - 1);
  }
  for (int32_t nth = chunks - 1; nth >= 0; --nth) {
    const int32_t t0 = part.t0 + nth * kC;
    const int n = part.t1 - t0 < kC ? part.t1 - t0 : kC;
    const int64_t at = static_cast<int64_t>(slot0 + nth) * g.HV + h;
    __syncthreads();
    rK.put(sK, n, g.DK, tid);
    rQ.put(sQ, n, g.DK, tid);
    if constexpr (OLDS) rOt.put(sO, n, trans ? 0 : g.DV - vcol0, tid);
    rT.put(sTri, tid);
    if (tid < 4 * kC) sDec[0][tid] = rDec;
    const float gam = rGam;
    const int32_t ahead = nth > 0 ? nth - 1 : 0;
    const int64_t at_tile = (at * a.col_tiles + col0 / 16) * 256;
    if constexpr (!AGG)
      if (col0 < g.DV) store_tiles<KT>(a.b.dend + at_tile * KT, E, lane);
    __syncthreads();
    f32x4 D[4], X[4], O[4];
#pragma unroll
    for (int rt = 0; rt < 4; ++rt) D[rt] = X[rt] = f32x4{0.f, 0.f, 0.f, 0.f};
    Frag<P> fk[2][4];
    const auto rows = [&](int ks) {
#pragma unroll
      for (int rt = 0; rt < 4; ++rt) fk[ks & 1][rt] = sK.rows(16 * rt + m, ks, grp);
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
      mma_n<3>(fk[ks & 1], ef, D);
#pragma unroll
      for (int i = 4 * ks / KS; i < 4 * (ks + 1) / KS; ++i) load(ahead, i);
      phase();
    }
    Frag<3> f1[4], f0[2];
    tri_tiles_t<0>(f1, sTri, 1, 1, m, grp);
#pragma unroll
    for (int rt = 0; rt < 4; ++rt) {
      if constexpr (OLDS)
        O[rt] = sO.col4(16 * wave, 16 * rt + 4 * grp, m);
      else
        O[rt] = rO.tile(rt, grp, n, vlive);
      D[rt] *= up[rt];
    }
    if constexpr (!OLDS) load_o(ahead);
    {
      const Frag<P> of[2] = {split_tiles<P>(O[0], O[1]), split_tiles<P>(O[2], O[3])};
      phase();
      tri_tiles_t<0>(f0, sTri, 1, 0, m, grp);
      mma_n<3>(f1, of[1], D);
      phase();
      tri_tiles_t<0>(f1, sTri, 0, 1, m, grp);
      mma_n<3>(f0, of[0], D);
      load(ahead, 4);
      phase();
    }
    f32x4 dx[4], dout[4];
    {
      const Frag<3> df[2] = {split_tiles<3>(D[0], D[1]), split_tiles<3>(D[2], D[3])};
      tri_tiles_t<0>(f0, sTri, 0, 0, m, grp);
      mma_n<3>(f1, df[1], X);
      load(ahead, 5);
      phase();
#pragma unroll
      for (int rt = 0; rt < 4; ++rt) {
        dx[rt] = dec_at(sDec, kDecBeta, rt, grp) * dec_at(sDec, kDecKey, rt, grp);
        dout[rt] = dec_at(sDec, kDecOut, rt, grp);
      }
      mma_n<3>(f0, df[0], X);
    }
    constexpr int KG = KT < 4 ? KT : 4;  // row tiles of the state at a time
    Frag<P> fc[2][KG];
    const auto keys = [&](int i) {  // K's and Q's columns, of the chunk's first and second half, in turn
      const int t0 = i / 4 * KG, ks = i / 2 % 2;
#pragma unroll
      for (int j = 0; j < KG; ++j) fc[i & 1][j] = (i % 2 ? sQ : sK).cols(16 * (t0 + j), 32 * ks + 4 * grp, m);
    };
    keys(0);
    if constexpr (!AGG)
      if (col0 < g.DV) store_tiles<4>(a.b.x + at_tile * 4, X, lane);
#pragma unroll
    for (int rt = 0; rt < 4; ++rt) {
      X[rt] *= -dx[rt];
      O[rt] *= dout[rt];
    }
    const Frag<3> xf[2] = {split_tiles<3>(X[0], X[1]), split_tiles<3>(X[2], X[3])};
    const Frag<3> of[2] = {split_tiles<3>(O[0], O[1]), split_tiles<3>(O[2], O[3])};
#pragma unroll
    for (int t = 0; t < KT; ++t) E[t] *= gam;
    load(ahead, 6);
    load(ahead, 7);
    phase();
#pragma unroll
    for (int i = 0; i < 4 * (KT / KG); ++i) {
      if (i + 1 < 4 * (KT / KG)) keys(i + 1);
      mma_n<3>(fc[i & 1], i % 2 ? of[i / 2 % 2] : xf[i / 2 % 2], E + i / 4 * KG);
      phase();
    }
  }
  if (AGG && trans) {
    if (col0 < DKP) store_tiles<KT>(a.w.trans + ((static_cast<int64_t>(p.slot) * g.HV + h) * KT + col0 / 16) * (KT * 256), E, lane);
  } else if (AGG) {
    if (tiles) store_tiles<KT>(a.w.carry + at_part, E, lane);
  }
  else if (a.b.dh0 != nullptr && part.t0 == part.start)
    store_state<KT>(a.b.dh0 + at_h, g.DV, g.DK, E, m, grp, live);
}

// Zeros in the gradients of the rows that belong to no sequence.
template <typename T>
__device__ void zero_rows(const BwdArgs& a, int32_t t0, int32_t t1, int hk, int tid, int nt) {
  const DeltaGeom& g = a.g;
  for (int32_t t = t0; t < t1; ++t) {
    for (int c = tid; c < g.DK; c += nt) {
      const int64_t i = (static_cast<int64_t>(t) * g.HK + hk) * g.DK + c;
      static_cast<T*>(a.b.dq)[i] = from_f32<T>(0.f);
      static_cast<T*>(a.b.dk)[i] = from_f32<T>(0.f);
    }
    for (int c = tid; c < g.group * g.DV; c += nt)
      static_cast<T*>(a.b.dv)[(static_cast<int64_t>(t) * g.HV + hk * g.group) * g.DV + c] = from_f32<T>(0.f);
    for (int c = tid; c < g.group; c += nt) {
      const int64_t i = static_cast<int64_t>(t) * g.HV + hk * g.group + c;
      a.b.dg[i] = 0.f;
      if (g.beta_f32)
        static_cast<float*>(a.b.dbeta)[i] = 0.f;
      else
        static_cast<T*>(a.b.dbeta)[i] = from_f32<T>(0.f);
    }
  }
}

// The sum over the 16 lanes of a row
__device__ __forceinline__ float row_sum(float x) {
  x += dpp<kRowRor8>(x);
  x += dpp<kRowRor4>(x);
  x += dpp<0x122>(x);
  return x + dpp<0x121>(x);
}

// x of a pair's even and odd row of 16 lanes, and of a wave's lower and upper half (both results through one 64-bit
// value, as in scan_common.h)
struct Halves {
  float lo, hi;
};
__device__ __forceinline__ Halves halves(uint64_t w) {
  return {__uint_as_float(static_cast<uint32_t>(w)), __uint_as_float(static_cast<uint32_t>(w >> 32))};
}
__device__ __forceinline__ Halves rows_of_pair(float x) {
  const uint32_t u = __float_as_uint(x);
  return halves(__builtin_bit_cast(uint64_t, __builtin_amdgcn_permlane16_swap(u, u, false, false)));
}
__device__ __forceinline__ Halves halves_of_wave(float x) {
  const uint32_t u = __float_as_uint(x);
  return halves(__builtin_bit_cast(uint64_t, __builtin_amdgcn_permlane32_swap(u, u, false, false)));
}

// W: of one token i (the lane's column) and the tile's rows j, zero from j = i on.  Adds to `before`, the sum over the
// tiles before, and returns for each row's number t the sum of W over j < t, where t <= i, over the tile's tokens.
__device__ __forceinline__ f32x4 pairs_across(const f32x4& W, float& before, int j0, int ti, int m, int grp) {
  const float s0 = W[0], s1 = s0 + W[1], s2 = s1 + W[2];
  const Halves p = rows_of_pair(s2 + W[3]), q = halves_of_wave(p.lo + p.hi);
  const float b = before + ((grp & 1 ? p.lo : 0.f) + (grp & 2 ? q.lo : 0.f));
  before += q.lo + q.hi;
  const f32x4 pre = {b, b + s0, b + s1, b + s2};
  f32x4 f;
#pragma unroll
  for (int r = 0; r < 4; ++r) f[r] = row_sum(j0 + r <= ti ? pre[r] : 0.f);
  return f;
}

// Eight waves a chunk and key head: a wave has 16 tokens and half of the keys' columns; the small triangles of its
// tokens are formed by both waves.  GROUPED: more than one value head a key head.
// Bound by waits and issue: 16384 tokens of 12 heads of 128 x 128 in bfloat16 take 416 us, MFMA busy 21 %, and two waves
// a SIMD that wait 46 % of their cycles; their 256 registers leave no room for a second workgroup.  With keys shared, and
// in float32, heads of more than 64 key values spill 116 to 340 bytes a lane, nearly all of it once a head, outside the
// loop over the values' columns.
template <typename T, int DKP, bool VEC, bool GROUPED>
__global__ void __launch_bounds__(512)
delta_grads_kernel(BwdArgs a) {
  constexpr int P = kRawParts<T>, KT = DKP / 16, KH = KT / 2, NT = 512;
  struct Rows {  // 32 columns of the values' side, rows the columns; dO: rows the tokens
    Tile<32, kC, 3> X, D;
    Tile<32, DKP, 3> S, E;
    Tile<kC, 32, P> O;
  };
  struct Keys {
    Tile<kC, DKP, P> K, Q;
  };
  __shared__ __attribute__((aligned(16))) union { Rows r; Keys k; } sm;
  __shared__ __attribute__((aligned(16))) double sG[kC];
  __shared__ __attribute__((aligned(16))) float sBeta[kC], sRk[kC], sRq[kC];
  __shared__ float sSe[8];
  __shared__ float sDot[5][2][kC];  // k . u | k . E D | of the factor exp(G_i) | with qk_l2norm: k . dk | q . dq
  __shared__ float sPair[8][kC];
  const DeltaGeom& g = a.g;
  int tid = threadIdx.x, lane = tid & 63, m = lane & 15, grp = lane >> 4;
  const int wave = wave_id(), tw = wave & 3, half = wave >> 2, d0 = half * KH * 16;  // token tile, first key column
  const uint32_t slot = blockIdx.x / static_cast<uint32_t>(g.HK);
  const int hk = static_cast<int>(blockIdx.x - slot * static_cast<uint32_t>(g.HK));
  const SeqChunk c = seq_chunk(g.q, static_cast<int32_t>(slot), g.cut, lane);
  if (c.t0 < 0 || c.t1 == c.t0) return;
  if (c.seq >= g.q.S) return zero_rows<T>(a, c.t0, c.t1, hk, tid, NT);
  const int n = c.t1 - c.t0;
  const int64_t orow = static_cast<int64_t>(g.HV) * g.DV;
  const f32x4 z4 = {0.f, 0.f, 0.f, 0.f};
  int ti = 16 * tw + m;  // this lane's token
  bool mine = ti < n;
  int64_t row_t = c.t0 + (mine ? ti : 0);
  f32x4 sumQ[GROUPED ? KH : 1], sumK[GROUPED ? KH : 1];
#pragma unroll
  for (int t = 0; t < (GROUPED ? KH : 1); ++t) sumQ[t] = sumK[t] = z4;
  f32x4 accQ[KH], accU[KH], accK[KH];
  float rk = 1.f, rq = 1.f;
  for (int hg = 0; hg < (GROUPED ? g.group : 1); ++hg) {
    const int h = hk * g.group + hg;
    const int64_t at = static_cast<int64_t>(slot) * g.HV + h;
    if constexpr (GROUPED) {  // addresses are formed anew: kept over the heads, they would spill
      asm volatile("" : "+v"(tid));
      lane = tid & 63, m = lane & 15, grp = lane >> 4;
      ti = 16 * tw + m;
      mine = ti < n;
      row_t = c.t0 + (mine ? ti : 0);
    }
    __syncthreads();
    const double G = log_decay(g, a.in.g, c.t0, n, h, lane);
    // (gates below the least one have no part in the outputs)
    const uint64_t below = __ballot(lane < n && a.in.g[(c.t0 + static_cast<int64_t>(lane)) * g.gs + h] < kMinLogDecay);
    if (wave == 0) {
      sG[lane] = G;
      sBeta[lane] = lane < n ? load_beta<T>(g, a.in.beta, c.t0 + lane, h) : 0.f;
    }
    const double Gc = __shfl(G, 63);
#pragma unroll
    for (int t = 0; t < KH; ++t) accQ[t] = accU[t] = accK[t] = z4;
    // Rows j of a tile, column the lane's token i: D_j . dO_i and D_j . X_i for tiles up to the wave's own, dO_j .
    // D_i and X_j . D_i behind it; of its own tile both.
    f32x4 UO[4], UX[4], ownO = z4, ownX = z4;
#pragma unroll
    for (int jt = 0; jt < 4; ++jt) UO[jt] = UX[jt] = z4;
    float xv = 0.f, se = 0.f;
    const float btok = mine ? load_beta<T>(g, a.in.beta, row_t, h) : 0.f;
    const T* vrow = static_cast<const T*>(a.in.v) + row_t * g.vs + h * g.vh;
    T* dvrow = static_cast<T*>(a.b.dv) + row_t * orow + static_cast<int64_t>(h) * g.DV;
    const T* dorow = static_cast<const T*>(a.b.d_o) + static_cast<int64_t>(c.t0) * orow + static_cast<int64_t>(h) * g.DV;
    // the next block's operands, on their way while this one's are at work
    constexpr int kState = (2 * KT * 64 + NT - 1) / NT;  // 16-byte pieces of two column tiles of a state
    f32x4 rX, rD, rS[kState], rE[kState], rV[2];
    StageRows<T, 32, NT> rO;
    StageRows<T, DKP, NT> rK, rQ;
    const auto load = [&](int kb, int which) {
      const int64_t ct = at * a.col_tiles + kb / 16;
      const bool two = kb + 16 < g.DV;  // (the second column tile exists)
      if (which == 0) {
        const int64_t x = (ct + (two ? tid >> 8 : 0)) * (4 * 256) + (tid & 255) * 4;
        rX = *reinterpret_cast<const f32x4*>(a.b.x + x);
        rD = *reinterpret_cast<const f32x4*>(a.b.vt + x);
      } else if (which == 1 || which == 2) {
#pragma unroll
        for (int i = 0; i < kState; ++i) {
          const int j = (tid + NT * i) % (2 * KT * 64);
          const int64_t y = (ct + (two ? j / (64 * KT) : 0)) * (KT * 256) + j % (64 * KT) * 4;
          (which == 1 ? rS : rE)[i] = *reinterpret_cast<const f32x4*>((which == 1 ? a.b.s0 : a.b.dend) + y);
        }
      } else {
        rO.template load<VEC>(dorow + kb, orow, n, g.DV - kb, tid);
        if (half == 0)
#pragma unroll
          for (int i = 0; i < 2; ++i) rV[i] = load4(vrow, kb + 16 * i + 4 * grp, mine ? g.DV : 0, VEC);
      }
    };
#pragma unroll
    for (int i = 0; i < 4; ++i) load(0, i);
    // (the last block apart: its registers are others)
    const auto block = [&](int kb, auto last_block) {
      constexpr bool more = !decltype(last_block)::value;
      const bool two = kb + 16 < g.DV;
      __syncthreads();
      {
        const bool on = tid < 256 || two;
        const int t = tid >> 6 & 3;
        sm.r.X.put4(16 * (tid >> 8) + m, 16 * t + 4 * grp, on ? rX : z4);
        sm.r.D.put4(16 * (tid >> 8) + m, 16 * t + 4 * grp, on ? rD : z4);
      }
#pragma unroll
      for (int i = 0; i < kState; ++i) {
        const int j = tid + NT * i, ct = j / (64 * KT), t = j / 64 % KT;
        if (j < 2 * KT * 64) {
          const f32x4 s = ct == 0 || two ? rS[i] : z4, e = ct == 0 || two ? rE[i] : z4;
#pragma unroll
          for (int r = 0; r < 4; ++r) se = fmaf(s[r], e[r], se);
          sm.r.S.put4(16 * ct + m, 16 * t + 4 * grp, s);
          sm.r.E.put4(16 * ct + m, 16 * t + 4 * grp, e);
        }
        phase();
      }
      rO.put(sm.r.O, n, g.DV - kb, tid);
      const f32x4 v0 = rV[0], v1 = rV[1];
      __syncthreads();
      // (a few loads between the phases: more at once hold up the wave that issues them; in the last block, q and k)
      const int k0 = 4 * grp;
      const Frag<3> bX = sm.r.X.cols(16 * tw, k0, m), bD = sm.r.D.cols(16 * tw, k0, m);
      const Frag<P> bO = sm.r.O.rows(ti, 0, grp);
      if (half == 0) {  // dv, and X . v
        f32x4 x0 = z4, x1 = z4;
#pragma unroll
        for (int p = 2; p >= 0; --p) {
          x0 += f32x4{__uint_as_float(bX.p[p].x << 16), __uint_as_float(bX.p[p].x & 0xffff0000u),
                      __uint_as_float(bX.p[p].y << 16), __uint_as_float(bX.p[p].y & 0xffff0000u)};
          x1 += f32x4{__uint_as_float(bX.p[p].z << 16), __uint_as_float(bX.p[p].z & 0xffff0000u),
                      __uint_as_float(bX.p[p].w << 16), __uint_as_float(bX.p[p].w & 0xffff0000u)};
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) xv = fmaf(x0[r], v0[r], fmaf(x1[r], v1[r], xv));
        if (mine) {
          Quad<T> q;
#pragma unroll
          for (int r = 0; r < 4; ++r) x0[r] *= btok, x1[r] *= btok;
          q.set(x0);
          q.store(dvrow, kb + 4 * grp, g.DV, VEC);
          q.set(x1);
          q.store(dvrow, kb + 16 + 4 * grp, g.DV, VEC);
        }
      }
      phase();
#pragma unroll
      for (int jt = 0; jt < 4; ++jt) {
        if (jt <= tw) {
          const Frag<3> f = sm.r.D.cols(16 * jt, k0, m);
          UO[jt] = mma<3>(f, bO, UO[jt]);
          UX[jt] = mma<3>(f, bX, UX[jt]);
        }
        if (jt >= tw) {
          const Frag<3> fx = sm.r.X.cols(16 * jt, k0, m);
          const Frag<P> fo = sm.r.O.rows(16 * jt + m, 0, grp);
          if (jt == tw) {
            ownX = mma<3>(fx, bD, ownX);
            ownO = mma<3>(fo, bD, ownO);
          } else {
            UX[jt] = mma<3>(fx, bD, UX[jt]);
            UO[jt] = mma<3>(fo, bD, UO[jt]);
          }
        }
        if constexpr (more) {
          load(kb + 32, jt);
        } else if (jt == 0) {
          rK.template load<VEC>(static_cast<const T*>(a.in.k) + c.t0 * g.ks + hk * g.kh, g.ks, n, g.DK, tid);
        } else if (jt == 2) {
          rQ.template load<VEC>(static_cast<const T*>(a.in.q) + c.t0 * g.qs + hk * g.qh, g.qs, n, g.DK, tid);
        }
        phase();
      }
      phase();
      constexpr int TG = KH < 2 ? KH : 2;
#pragma unroll
      for (int t = 0; t < KH; t += TG) {
        Frag<3> f[TG], e[TG];
#pragma unroll
        for (int i = 0; i < TG; ++i) {
          f[i] = sm.r.S.cols(d0 + 16 * (t + i), k0, m);
          e[i] = sm.r.E.cols(d0 + 16 * (t + i), k0, m);
        }
        mma_n<3>(f, bO, accQ + t);
        mma_n<3>(f, bX, accU + t);
        mma_n<3>(e, bD, accK + t);
        phase();
      }
    };
    int kb = 0;
    for (; kb + 32 < g.DV; kb += 32) block(kb, std::false_type{});
    block(kb, std::true_type{});
    xv = sum_g(xv);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) se += __shfl_xor(se, o);
    __syncthreads();
    rK.put(sm.k.K, n, g.DK, tid);
    rQ.put(sm.k.Q, n, g.DK, tid);
    if (lane == 0) sSe[wave] = se;
    __syncthreads();
    {
      float nk = 0.f, nq = 0.f;
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        const f32x4 x = sm.k.K.get4(ti, 16 * t + 4 * grp), y = sm.k.Q.get4(ti, 16 * t + 4 * grp);
#pragma unroll
        for (int r = 0; r < 4; ++r) nk = fmaf(x[r], x[r], nk), nq = fmaf(y[r], y[r], nq);
        phase();
      }
      nk = sum_g(nk);
      nq = sum_g(nq);
      rk = g.l2 ? 1.f / sqrtf(nk + kL2Eps) : 1.f;
      rq = g.l2 ? 1.f / sqrtf(nq + kL2Eps) : 1.f;
      if (grp == 0 && half == 0) {
        sRk[ti] = rk;
        sRq[ti] = rq;
      }
    }
    __syncthreads();
    const double Gi = sG[ti];
    const float eG = exp_diff(Gi), eR = exp_diff(Gc - Gi), bi = sBeta[ti];
    float kh = 0.f, us = 0.f, qs = 0.f;
#pragma unroll
    for (int t = 0; t < KH; ++t) {
      accQ[t] *= g.scale * eG;
      accU[t] *= -eG;
      accK[t] *= eR;
      const f32x4 x = sm.k.K.get4(ti, d0 + 16 * t + 4 * grp), y = sm.k.Q.get4(ti, d0 + 16 * t + 4 * grp);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        kh = fmaf(accK[t][r], x[r], kh);
        us = fmaf(accU[t][r], x[r], us);
        qs = fmaf(accQ[t][r], y[r], qs);
      }
      phase();
    }
    // The decay between two tokens, from the earlier to the later, on all pairs; and dg's sums over them, of which the
    // waves of the first half take those of q and k, the second half's those of k and k
    {
      const float own = half == 0 ? g.scale * rq : -bi * rk;
      float before = 0.f;
#pragma unroll
      for (int jt = 0; jt < 4; ++jt) {
        const int j0 = 16 * jt + 4 * grp;
        f32x4 e;
#pragma unroll
        for (int r = 0; r < 4; ++r) e[r] = exp_diff(j0 + r <= ti ? Gi - sG[j0 + r] : sG[j0 + r] - Gi);
        UO[jt] *= e;
        UX[jt] *= e;
        if (jt == tw) {
          ownO *= e;
          ownX *= e;
        }
        phase();
        if (jt <= tw) {
          f32x4 W = z4;
          int row = ti;  // (read anew for every tile: kept over them, the token's operands would spill)
          asm volatile("" : "+v"(row));
#pragma unroll
          for (int s = 0; s < DKP / 32; ++s) {
            W = mma<3>(sm.k.K.rows(16 * jt + m, s, grp), (half == 0 ? sm.k.Q : sm.k.K).rows(row, s, grp), W);
            if constexpr (P == 3) phase();
          }
          const f32x4 rkj = *reinterpret_cast<const f32x4*>(&sRk[j0]);
#pragma unroll
          for (int r = 0; r < 4; ++r) W[r] = j0 + r < ti ? W[r] * own * rkj[r] * (half == 0 ? UO : UX)[jt][r] : 0.f;
          const f32x4 f = pairs_across(W, before, j0, ti, m, grp);
          if (m < 4) sPair[wave][j0 + m] = m == 0 ? f[0] : m == 1 ? f[1] : m == 2 ? f[2] : f[3];
        }
        phase();
      }
    }
    constexpr int KG = (P == 3 || GROUPED) && KH > 2 ? 2 : KH;  // column tiles whose operands are held at a time
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      f32x4 DO[2], DX[2], XD[2], OD[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int jt = 2 * ks + i, j0 = 16 * jt + 4 * grp;
        const f32x4 rkj = *reinterpret_cast<const f32x4*>(&sRk[j0]), rqj = *reinterpret_cast<const f32x4*>(&sRq[j0]),
                    bj = *reinterpret_cast<const f32x4*>(&sBeta[j0]);
        const f32x4 uo = jt == tw ? ownO : UO[jt], ux = jt == tw ? ownX : UX[jt];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int j = j0 + r;
          DO[i][r] = j <= ti ? g.scale * rkj[r] * UO[jt][r] : 0.f;
          DX[i][r] = j < ti ? -rkj[r] * UX[jt][r] : 0.f;
          XD[i][r] = j > ti ? -bj[r] * rkj[r] * ux[r] : 0.f;
          OD[i][r] = j >= ti ? g.scale * rqj[r] * uo[r] : 0.f;
        }
        phase();
      }
      const int j0 = 32 * ks + 4 * grp;
      if (2 * ks <= tw) {
        const Frag<3> f1 = split_tiles<3>(DO[0], DO[1]), f2 = split_tiles<3>(DX[0], DX[1]);
#pragma unroll
        for (int t = 0; t < KH; t += KG) {
          Frag<P> k[KG];
#pragma unroll
          for (int i = 0; i < KG; ++i) k[i] = sm.k.K.cols(d0 + 16 * (t + i), j0, m);
          mma_n<3>(k, f1, accQ + t);
          mma_n<3>(k, f2, accU + t);
          if constexpr (KG < KH) phase();
        }
      }
      phase();
      if (2 * ks + 1 >= tw) {
        const Frag<3> f1 = split_tiles<3>(XD[0], XD[1]), f2 = split_tiles<3>(OD[0], OD[1]);
#pragma unroll
        for (int t = 0; t < KH; t += KG) {
          Frag<P> k[KG];
#pragma unroll
          for (int i = 0; i < KG; ++i) k[i] = sm.k.K.cols(d0 + 16 * (t + i), j0, m);
          mma_n<3>(k, f1, accK + t);
#pragma unroll
          for (int i = 0; i < KG; ++i) k[i] = sm.k.Q.cols(d0 + 16 * (t + i), j0, m);
          mma_n<3>(k, f2, accK + t);
          if constexpr (KG < KH) phase();
        }
      }
      phase();
    }
    float ku = 0.f, qd = 0.f, kd = 0.f;
#pragma unroll
    for (int t = 0; t < KH; ++t) {
      const f32x4 x = sm.k.K.get4(ti, d0 + 16 * t + 4 * grp), y = sm.k.Q.get4(ti, d0 + 16 * t + 4 * grp);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        ku = fmaf(accU[t][r], x[r], ku);
        accK[t][r] = fmaf(bi, accU[t][r], accK[t][r]);
        if constexpr (!GROUPED) {
          kd = fmaf(accK[t][r], x[r], kd);
          qd = fmaf(accQ[t][r], y[r], qd);
        }
      }
      if constexpr (GROUPED) {
        sumQ[t] += accQ[t];
        sumK[t] += accK[t];
      }
      phase();
    }
    ku = sum_g(ku) * rk;
    kh = sum_g(kh) * rk;
    us = sum_g(us) * rk;
    qs = sum_g(qs) * rq;
    if constexpr (!GROUPED) {
      kd = sum_g(kd) * rk;
      qd = sum_g(qd) * rq;
    }
    if (grp == 0) {
      sDot[0][half][ti] = ku;
      sDot[1][half][ti] = kh;
      sDot[2][half][ti] = fmaf(bi, us, qs);
      if constexpr (!GROUPED) {
        sDot[3][half][ti] = kd;
        sDot[4][half][ti] = qd;
      }
    }
    __syncthreads();
    if (wave == 0) {  // lane = token
      const auto both = [&](int which, int t) { return sDot[which][0][t] + sDot[which][1][t]; };
      const double to = __shfl_up(wave_scan(both(1, lane)), 1), from = __shfl(wave_scan(both(2, 63 - lane)), 63 - lane);
      double sums = 0.0, s = 0.0;
#pragma unroll
      for (int i = 0; i < 8; ++i) sums += sSe[i];
#pragma unroll
      for (int i = 0; i < 8; ++i) s += (i & 3) >= lane / 16 ? sPair[i][lane] : 0.f;  // (waves of tokens behind it)
      s += from + (lane > 0 ? to : 0.0) + static_cast<double>(exp_diff(Gc)) * sums;
      if (lane < n) a.b.dg[(c.t0 + static_cast<int64_t>(lane)) * g.HV + h] = below >> lane & 1 ? 0.f : static_cast<float>(s);
    }
    if (half == 0 && grp == 0 && mine) {
      const float db = xv + ku + sDot[0][1][ti];
      const int64_t i = row_t * g.HV + h;
      if (g.beta_f32)
        static_cast<float*>(a.b.dbeta)[i] = db;
      else
        static_cast<T*>(a.b.dbeta)[i] = from_f32<T>(db);
    }
  }
  // (the keys of the last head are still in LDS)
  const auto gq = [&](int t) -> const f32x4& {
    if constexpr (GROUPED) return sumQ[t];
    else return accQ[t];
  };
  const auto gk = [&](int t) -> const f32x4& {
    if constexpr (GROUPED) return sumK[t];
    else return accK[t];
  };
  float qd = 0.f, kd = 0.f;
  if (g.l2) {
    if constexpr (GROUPED) {
#pragma unroll
      for (int t = 0; t < KH; ++t) {
        const f32x4 x = sm.k.K.get4(ti, d0 + 16 * t + 4 * grp), y = sm.k.Q.get4(ti, d0 + 16 * t + 4 * grp);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          kd = fmaf(gk(t)[r], x[r], kd);
          qd = fmaf(gq(t)[r], y[r], qd);
        }
      }
      kd = sum_g(kd) * rk;
      qd = sum_g(qd) * rq;
      __syncthreads();
      if (grp == 0) {
        sDot[3][half][ti] = kd;
        sDot[4][half][ti] = qd;
      }
      __syncthreads();
    }
    kd = (sDot[3][0][ti] + sDot[3][1][ti]) * rk;
    qd = (sDot[4][0][ti] + sDot[4][1][ti]) * rq;
  }
  if (!mine) return;
  const int64_t out = (row_t * g.HK + hk) * g.DK;
#pragma unroll
  for (int t = 0; t < KH; ++t) {
    const int d = d0 + 16 * t + 4 * grp;
    const f32x4 x = sm.k.K.get4(ti, d), y = sm.k.Q.get4(ti, d);
    Quad<T> q;
    q.set((gk(t) - x * kd) * rk);
    q.store(static_cast<T*>(a.b.dk) + out, d, g.DK, VEC);
    q.set((gq(t) - y * qd) * rq);
    q.store(static_cast<T*>(a.b.dq) + out, d, g.DK, VEC);
  }
}

}  // namespace

hipError_t launch_delta_bwd(const DeltaGeom& g, const DeltaIn& in, const DeltaWork& w, const DeltaBwd& b, int dtype,
                            hipStream_t s) {
  // (rows that are read value by value: more registers, so four waves)
  const int nw = g.vec ? g.waves : 4;
  const uint32_t vcb = delta_col_blocks(g.DV, nw);
  BwdArgs a{g, in, w, b, delta_col_tiles(g), vcb, vcb, static_cast<uint32_t>(chunk_slots(g.q, g.part))};
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
    const dim3 grid(static_cast<unsigned>(chunk_slots(g.q, g.cut) * g.HK));
    if (g.group > 1)
      hipLaunchKernelGGL((delta_grads_kernel<T, DKP, VEC, true>), grid, dim3(512), 0, s, a);
    else
      hipLaunchKernelGGL((delta_grads_kernel<T, DKP, VEC, false>), grid, dim3(512), 0, s, a);
    return hipGetLastError();
  };
  return delta_dispatch(dtype, g.DK, [&](auto t, auto dkp) {
    using Four = std::integral_constant<int, 4>;
    if (!g.vec) return run(t, dkp, Four{}, std::false_type{});
    if constexpr (sizeof(t) == 2)
      if (nw == 8) return run(t, dkp, std::integral_constant<int, 8>{}, std::true_type{});
    return run(t, dkp, Four{}, std::true_type{});
  });
}

}  // namespace mvm
