// The gated delta rule's chunks by themselves: for 64 tokens and a value head
//   A_ij = beta_i (k_i . k_j) exp(G_i - G_j), i > j,    T = (I + A)^-1,
//   P_ij = scale (q_i . k_j) exp(G_i - G_j), i >= j     (G: log decays summed)
// and the tokens' scalars, for the passes along time (delta_fwd.hip,
// delta_bwd.hip), which take T and P as ready A operands: their bf16 parts in
// the order in which the lanes load them (the backward pass: of T' and P').
//
// A workgroup of four waves takes one chunk and head.  T: the four 16 x 16
// blocks on the diagonal by substitution, a column a lane (a series in powers
// of A would cancel: they grow like binomials where keys repeat), those below
// by products of blocks, T_ij = -T_ii sum_k A_ik T_kj, in the float32 matrix
// instructions, a block column a wave.
#include "delta_common.h"

namespace mvm {
namespace {

constexpr int kLda = kC + 4;

__device__ __forceinline__ f32x4 mma_f32(const f32x4& a, const f32x4& b, f32x4 c) {
  // summed index 4g + s in step s: a result tile is the B operand as it is
#pragma unroll
  for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[s], b[s], c, 0, 0, 0);
  return c;
}

template <typename T, int DKP, bool BWD>
__global__ void __launch_bounds__(256)
delta_prep_kernel(DeltaGeom g, DeltaIn in, DeltaWork w) {
  constexpr int P = kRawParts<T>;
  __shared__ __attribute__((aligned(16))) Tile<kC, DKP, P> sK, sQ;
  __shared__ __attribute__((aligned(16))) float sA[kC][kLda], sT[kC][kLda];
  __shared__ double sG[kC];
  __shared__ float sBeta[kC], sRk[kC], sRq[kC];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, m = lane & 15, grp = lane >> 4;
  const uint32_t slot = blockIdx.x / static_cast<uint32_t>(g.HV);
  const int h = static_cast<int>(blockIdx.x - slot * static_cast<uint32_t>(g.HV)), hk = h / g.group;
  const SeqChunk c = seq_chunk(g.q, static_cast<int32_t>(slot), g.cut, lane);
  if (c.seq >= g.q.S || c.t0 < 0 || c.t1 == c.t0) return;
  const int n = c.t1 - c.t0;
  stage_rows<T, DKP>(sK, static_cast<const T*>(in.k) + c.t0 * g.ks + hk * g.kh, g.ks, n, g.DK, g.qk_vec, tid, 256);
  stage_rows<T, DKP>(sQ, static_cast<const T*>(in.q) + c.t0 * g.qs + hk * g.qh, g.qs, n, g.DK, g.qk_vec, tid, 256);
  const double G = log_decay(g, in.g, c.t0, n, h, lane);
  const float beta = lane < n ? load_beta<T>(g, in.beta, c.t0 + lane, h) : 0.f;
  if (wave == 0) {
    sG[lane] = G;
    sBeta[lane] = beta;
  }
  __syncthreads();
  {
    float nk = 0.f, nq = 0.f;
#pragma unroll
    for (int t = 0; t < DKP / 16; ++t) {
      const f32x4 a = sK.get4(16 * wave + m, 16 * t + 4 * grp), b = sQ.get4(16 * wave + m, 16 * t + 4 * grp);
#pragma unroll
      for (int r = 0; r < 4; ++r) nk = fmaf(a[r], a[r], nk), nq = fmaf(b[r], b[r], nq);
    }
    nk = sum_g(nk);
    nq = sum_g(nq);
    if (grp == 0) {
      sRk[16 * wave + m] = g.l2 ? 1.f / sqrtf(nk + kL2Eps) : 1.f;
      sRq[16 * wave + m] = g.l2 ? 1.f / sqrtf(nq + kL2Eps) : 1.f;
    }
  }
  __syncthreads();
  const int64_t at = static_cast<int64_t>(slot) * g.HV + h;
  const double Gc = __shfl(G, 63);
  if (wave == 0) {
    const float eG = exp_diff(G), eR = exp_diff(Gc - G);
    reinterpret_cast<float4*>(w.dec)[at * kC + lane] =
        make_float4(sRk[lane] * eG, sRk[lane] * eR, g.scale * sRq[lane] * eG, beta);
    if (lane == 0) w.gam[at] = exp_diff(Gc);
  }
  // row tile `wave` of K K' and Q K'
  f32x4 kk[4], qk[4];
#pragma unroll
  for (int ct = 0; ct < 4; ++ct) kk[ct] = qk[ct] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int ks = 0; ks < DKP / 32; ++ks) {
    const int k0 = 32 * ks + 8 * grp;
    const Frag<P> a = sK.rows_plain(16 * wave + m, k0), aq = sQ.rows_plain(16 * wave + m, k0);
#pragma unroll
    for (int ct = 0; ct < 4; ++ct)
      if (ct <= wave) {
        const Frag<P> b = sK.rows_plain(16 * ct + m, k0);
        kk[ct] = mma<3>(a, b, kk[ct]);
        qk[ct] = mma<3>(aq, b, qk[ct]);
      }
  }
#pragma unroll
  for (int ct = 0; ct < 4; ++ct) {
    const int j = 16 * ct + m;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = 16 * wave + 4 * grp + r;
      const float e = j <= i ? exp_diff(sG[i] - sG[j]) * sRk[j] : 0.f;
      sA[i][j] = j < i ? sBeta[i] * sRk[i] * e * kk[ct][r] : 0.f;
      qk[ct][r] = j <= i ? g.scale * sRq[i] * e * qk[ct][r] : 0.f;
    }
  }
  __syncthreads();
  {  // the diagonal block, column m
    float t[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float s = i == m ? 1.f : 0.f;
#pragma unroll
      for (int j = 0; j < i; ++j) s = fmaf(-sA[16 * wave + i][16 * wave + j], t[j], s);
      t[i] = s;
    }
    if (grp == 0)
#pragma unroll
      for (int i = 0; i < 16; ++i) sT[16 * wave + i][16 * wave + m] = t[i];
    for (int ct = wave + 1; ct < 4; ++ct)
      *reinterpret_cast<float4*>(&sT[16 * wave + m][16 * ct + 4 * grp]) = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  __syncthreads();
  {  // block column `wave`
    f32x4 X[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i == wave)
#pragma unroll
        for (int r = 0; r < 4; ++r) X[i][r] = sT[16 * i + 4 * grp + r][16 * i + m];
      if (i > wave) {
        f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < i; ++k)
          if (k >= wave) s = mma_f32(*reinterpret_cast<const f32x4*>(&sA[16 * i + m][16 * k + 4 * grp]), X[k], s);
        const f32x4 z = {0.f, 0.f, 0.f, 0.f};
        X[i] = -mma_f32(*reinterpret_cast<const f32x4*>(&sT[16 * i + m][16 * i + 4 * grp]), s, z);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i > wave)
#pragma unroll
        for (int r = 0; r < 4; ++r) sT[16 * i + 4 * grp + r][16 * wave + m] = X[i][r];
  }
  __syncthreads();
#pragma unroll
  for (int ct = 0; ct < 4; ++ct)
#pragma unroll
    for (int r = 0; r < 4; ++r) sA[16 * wave + 4 * grp + r][16 * ct + m] = qk[ct][r];
  __syncthreads();
  uint4* out = reinterpret_cast<uint4*>(w.tri) + at * (2 * kTriFrags * kTriParts * 64);
  for (int f = wave; f < 2 * kTriFrags; f += 4) {
    const float(*src)[kLda] = f < kTriFrags ? sT : sA;
    const int i = f % kTriFrags;
    const int rt = BWD ? (i < 4 ? i >> 1 : i - 2) : (i < 2 ? i : (i + 2) >> 1);
    const int ks = BWD ? (i < 4 ? i & 1 : 1) : (i < 2 ? 0 : i & 1);
    const int row = 16 * rt + m, k0 = 32 * ks + 4 * grp;
    f32x4 a, b;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      a[r] = BWD ? src[k0 + r][row] : src[row][k0 + r];
      b[r] = BWD ? src[k0 + 16 + r][row] : src[row][k0 + 16 + r];
    }
    const Frag<kTriParts> fr = split_tiles<kTriParts>(a, b);
#pragma unroll
    for (int p = 0; p < kTriParts; ++p) out[(f * kTriParts + p) * 64 + lane] = fr.p[p];
  }
}

}  // namespace

hipError_t launch_delta_prep(const DeltaGeom& g, const DeltaIn& in, const DeltaWork& w, bool backward, int dtype,
                             hipStream_t s) {
  if (g.q.T == 0) return hipSuccess;
  const dim3 grid(static_cast<unsigned>(chunk_slots(g.q, g.cut) * g.HV));
  return delta_dispatch(dtype, g.DK, [&](auto t, auto dkp) {
    using T = decltype(t);
    constexpr int DKP = decltype(dkp)::value;
    if (backward)
      hipLaunchKernelGGL((delta_prep_kernel<T, DKP, true>), grid, dim3(256), 0, s, g, in, w);
    else
      hipLaunchKernelGGL((delta_prep_kernel<T, DKP, false>), grid, dim3(256), 0, s, g, in, w);
    return hipGetLastError();
  });
}

}  // namespace mvm
