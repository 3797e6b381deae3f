// The gated delta rule's chunks by themselves: for 64 tokens and a value head
//   A_ij = beta_i (k_i . k_j) exp(G_i - G_j), i > j,    T = (I + A)^-1,
//   P_ij = scale (q_i . k_j) exp(G_i - G_j), i >= j     (G: log decays summed)
// and the tokens' scalars, for the passes along time (delta_fwd.hip,
// delta_bwd.hip), which take T and P as ready A operands: their bf16 parts in
// the order in which the lanes load them.
//
// A workgroup of four waves takes one chunk and head, a wave 16 rows of both
// triangles.  A result tile is, as the lanes hold it, an A operand of its
// transpose: so K Q' and the inverse of I + A' are formed, and nothing is
// transposed.  The inverse: the four 16 x 16 blocks on the diagonal by
// substitution, a column a lane (a series in powers of A would cancel: they grow
// like binomials where keys repeat), the others by products of blocks, with M =
// T': M_iw = -M_ii sum_k A'_ik M_kw, in the float32 matrix instructions, a block
// column a wave, chained in registers.
//
// Bound by waits: every workgroup is one chain of loads, products, substitution
// and stores (32768 tokens of 12 heads of 128 in bfloat16: 132 us, of which 228 MB
// of fragments written would take 47 at a copy's rate; MFMA busy 7 %).
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

template <typename T, int DKP>
__global__ void __launch_bounds__(256)
delta_prep_kernel(DeltaGeom g, DeltaIn in, DeltaWork w) {
  constexpr int P = kRawParts<T>;
  // A', and the inverses of its diagonal blocks
  __shared__ __attribute__((aligned(16))) float sA[kC][kLda], sD[4][16][20];
  __shared__ double sG[kC];
  __shared__ float sBeta[kC], sRk[kC], sRq[kC];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, m = lane & 15, grp = lane >> 4;
  const uint32_t slot = blockIdx.x / static_cast<uint32_t>(g.HV);
  const int h = static_cast<int>(blockIdx.x - slot * static_cast<uint32_t>(g.HV)), hk = h / g.group;
  const SeqChunk c = seq_chunk(g.q, static_cast<int32_t>(slot), g.cut, lane);
  if (c.seq >= g.q.S || c.t0 < 0 || c.t1 == c.t0) return;
  const int n = c.t1 - c.t0;
  const T* kp = static_cast<const T*>(in.k) + c.t0 * g.ks + hk * g.kh;
  const T* qp = static_cast<const T*>(in.q) + c.t0 * g.qs + hk * g.qh;
  // Tiles of K K' and K Q': rows jt, the keys up to the wave's tokens, which are the columns.
  f32x4 kk[4], qk[4], qq = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int jt = 0; jt < 4; ++jt) kk[jt] = qk[jt] = qq;
  const int own = 16 * wave + m;
#pragma unroll
  for (int ks = 0; ks < DKP / 32; ++ks) {
    const int k0 = 32 * ks + 8 * grp;
    const auto frag = [&](const T* p, int64_t stride, int row) {
      return row_frag<T>(p + (row < n ? row : 0) * stride, k0, g.DK, g.vec, row < n);
    };
    const Frag<P> bk = frag(kp, g.ks, own), bq = frag(qp, g.qs, own);
    qq = mma<3>(bq, bq, qq);
#pragma unroll
    for (int jt = 0; jt < 4; ++jt)
      if (jt <= wave) {
        const Frag<P> ak = jt == wave ? bk : frag(kp, g.ks, 16 * jt + m);
        kk[jt] = mma<3>(ak, bk, kk[jt]);
        qk[jt] = mma<3>(ak, bq, qk[jt]);
      }
  }
  const double G = log_decay(g, in.g, c.t0, n, h, lane);
  if (wave == 0) {
    sG[lane] = G;
    sBeta[lane] = lane < n ? load_beta<T>(g, in.beta, c.t0 + lane, h) : 0.f;
  }
  // the squared norms lie on the diagonal tiles' diagonals
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (m == 4 * grp + r) {
      float nk = 0.f;
#pragma unroll
      for (int jt = 0; jt < 4; ++jt) nk = jt == wave ? kk[jt][r] : nk;
      sRk[own] = g.l2 ? 1.f / sqrtf(nk + kL2Eps) : 1.f;
      sRq[own] = g.l2 ? 1.f / sqrtf(qq[r] + kL2Eps) : 1.f;
    }
  __syncthreads();
  const int64_t at = static_cast<int64_t>(slot) * g.HV + h;
  if (wave == 0) {
    const double Gc = __shfl(G, 63);
    const float eG = exp_diff(G), eR = exp_diff(Gc - G);
    float* dec = w.dec + at * (4 * kC) + lane;
    dec[kDecKey * kC] = sRk[lane] * eG;
    dec[kDecUp * kC] = sRk[lane] * eR;
    dec[kDecOut * kC] = g.scale * sRq[lane] * eG;
    dec[kDecBeta * kC] = sBeta[lane];
    if (lane == 0) w.gam[at] = exp_diff(Gc);
  }
  const double Gown = sG[own];
  const float bown = sBeta[own] * sRk[own], qown = g.scale * sRq[own];
#pragma unroll
  for (int jt = 0; jt < 4; ++jt)
    if (jt <= wave) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int j = 16 * jt + 4 * grp + r;
        const float e = j <= own ? exp_diff(Gown - sG[j]) * sRk[j] : 0.f;
        sA[j][own] = j < own ? e * kk[jt][r] * bown : 0.f;
        qk[jt][r] *= e * qown;
      }
    }
  // (a wave's own diagonal block: its own writes)
  float t[16];
#pragma unroll
  for (int x = 0; x < 16; ++x) {
    const int i = 15 - x;
    float s = i == m ? 1.f : 0.f;
#pragma unroll
    for (int y = 0; y < 16; ++y)
      if (y > i) s = fmaf(-sA[16 * wave + i][16 * wave + y], t[y], s);
    t[i] = s;
  }
  if (grp == 0)
#pragma unroll
    for (int i = 0; i < 16; ++i) sD[wave][i][m] = t[i];
  __syncthreads();
  f32x4 X[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const float v = grp == 0 ? t[r] : grp == 1 ? t[4 + r] : grp == 2 ? t[8 + r] : t[12 + r];
#pragma unroll
    for (int i = 0; i < 4; ++i) X[i][r] = i == wave ? v : 0.f;
  }
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const int i = 3 - x;
    if (i < wave) {
      f32x4 s = {0.f, 0.f, 0.f, 0.f};
      const f32x4 z = s;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (k > i && k <= wave)
          s = mma_f32(*reinterpret_cast<const f32x4*>(&sA[16 * i + m][16 * k + 4 * grp]), X[k], s);
      X[i] = -mma_f32(*reinterpret_cast<const f32x4*>(&sD[i][m][4 * grp]), s, z);
    }
  }
  uint4* out = reinterpret_cast<uint4*>(w.tri) + at * kTriFragments + tri_lane(m, grp);
#pragma unroll
  for (int ks = 0; ks < 2; ++ks)
    if (2 * ks <= wave) {
      const int f = wave < 2 ? wave : 2 * wave - 2 + ks;
      const Frag<kTriParts> a = split_tiles<kTriParts>(X[2 * ks], X[2 * ks + 1]),
                            b = split_tiles<kTriParts>(qk[2 * ks], qk[2 * ks + 1]);
#pragma unroll
      for (int p = 0; p < kTriParts; ++p) {
        out[tri_index(0, p, f)] = a.p[p];
        out[tri_index(1, p, f)] = b.p[p];
      }
    }
}

}  // namespace

hipError_t launch_delta_prep(const DeltaGeom& g, const DeltaIn& in, const DeltaWork& w, int dtype, hipStream_t s) {
  if (g.q.T == 0) return hipSuccess;
  const dim3 grid(static_cast<unsigned>(chunk_slots(g.q, g.cut) * g.HV));
  return delta_dispatch(dtype, g.DK, [&](auto t, auto dkp) {
    hipLaunchKernelGGL((delta_prep_kernel<decltype(t), decltype(dkp)::value>), grid, dim3(256), 0, s, g, in, w);
    return hipGetLastError();
  });
}

}  // namespace mvm
