// The gated delta rule's single tokens: every sequence's states (dk x dv values
// a head) are read, advanced and written once, which is all the time a full
// batch takes; few sequences are bound by latency.
//
// One pass needs S^T k before it can write and S'^T q after: with
//   S' = a S + k d',  d = beta (v - a S^T k),  o = scale (a S^T q + (q . k) d)
// both sums are over the old state, so it is read once, held in registers and
// written back.  A workgroup takes a head's columns V CL at a time: CL lanes a
// row, V columns each, 256 / CL rows side by side.  512 sequences of 12 heads of
// 128 x 128 move 812 MB in 190 us, 4.3 TB/s (a large copy: 4.84); loads and stores
// that pass the caches by took 206.
#include "delta_common.h"

namespace mvm {
namespace {

__device__ __forceinline__ float wave_total(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

template <typename T, int DKP, int CL, int V>
__global__ void __launch_bounds__(256)
delta_step_kernel(DeltaGeom g, DeltaIn in, uint32_t ncb, float* __restrict__ states, T* __restrict__ o) {
  constexpr int RG = 256 / CL, RP = DKP / RG;  // rows side by side, and of a thread
  static_assert(RP >= 1, "every thread has a row");
  __shared__ float sSum[4][2][CL * V];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, cl = tid % CL, rg = tid / CL;
  const uint32_t item = blockIdx.x / ncb;
  const int32_t cb = static_cast<int32_t>(blockIdx.x - item * ncb);
  const int32_t i = static_cast<int32_t>(item / static_cast<uint32_t>(g.HV));
  const int h = static_cast<int>(item - static_cast<uint32_t>(i) * g.HV), hk = h / g.group;
  const int32_t row = seq_slot(g.q, i);
  const int c0 = (cb * CL + cl) * V;
  T* op = o + (static_cast<int64_t>(i) * g.HV + h) * g.DV;
  if (row < 0) {
    if (rg == 0)
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (c0 + j < g.DV) op[c0 + j] = from_f32<T>(0.f);
    return;
  }
  const T* kp = static_cast<const T*>(in.k) + i * g.ks + hk * g.kh;
  const T* qp = static_cast<const T*>(in.q) + i * g.qs + hk * g.qh;
  const T* vp = static_cast<const T*>(in.v) + i * g.vs + h * g.vh;
  float* sp = states + (static_cast<int64_t>(row) * g.HV + h) * g.DK * static_cast<int64_t>(g.DV);
  const bool zero = __builtin_amdgcn_readfirstlane(seq_fresh(g.q, i) ? 1 : 0) != 0, in_c = c0 < g.DV;  // (DV is a multiple of V)
  Pack<float, V> S[RP];
  float kd[RP], qd[RP];
#pragma unroll
  for (int r = 0; r < RP; ++r) {
    const int d = rg + r * RG;
    const bool ok = d < g.DK;
    S[r] = load_pack<float, V>(sp + static_cast<int64_t>(ok ? d : 0) * g.DV + (in_c ? c0 : 0));
    kd[r] = ok ? to_f32(kp[d]) : 0.f;
    qd[r] = ok ? to_f32(qp[d]) : 0.f;
  }
  float vv[V];
#pragma unroll
  for (int j = 0; j < V; ++j) vv[j] = in_c ? to_f32(vp[c0 + j]) : 0.f;
  // a lane's two rows of k and q, for the sums over all of them
  float kk = 0.f, qq = 0.f, qk = 0.f;
#pragma unroll
  for (int b = 0; b < DKP; b += 64) {
    const int d = b + lane;
    const float kf = d < g.DK ? to_f32(kp[d]) : 0.f, qf = d < g.DK ? to_f32(qp[d]) : 0.f;
    kk = fmaf(kf, kf, kk);
    qq = fmaf(qf, qf, qq);
    qk = fmaf(qf, kf, qk);
  }
  qk = wave_total(qk);
  float rk = 1.f, rq = 1.f;
  if (g.l2) {
    rk = 1.f / sqrtf(wave_total(kk) + kL2Eps);
    rq = 1.f / sqrtf(wave_total(qq) + kL2Eps);
  }
  const float gv = in.g[i * g.gs + h];
  const float al = expf(gv < kMinLogDecay ? kMinLogDecay : gv), beta = load_beta<T>(g, in.beta, i, h);
  float sk[V], sq[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    sk[j] = sq[j] = 0.f;
#pragma unroll
    for (int r = 0; r < RP; ++r) {
      // (rows past dk and a fresh sequence's hold anything)
      S[r].v[j] = zero || rg + r * RG >= g.DK ? 0.f : S[r].v[j];
      sk[j] = fmaf(kd[r], S[r].v[j], sk[j]);
      sq[j] = fmaf(qd[r], S[r].v[j], sq[j]);
    }
#pragma unroll
    for (int b = CL; b < 64; b <<= 1) {
      sk[j] += __shfl_xor(sk[j], b);
      sq[j] += __shfl_xor(sq[j], b);
    }
    if (lane < CL) {
      sSum[wave][0][cl * V + j] = sk[j];
      sSum[wave][1][cl * V + j] = sq[j];
    }
  }
  __syncthreads();
  if (!in_c) return;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int c = cl * V + j;
    const float a = (sSum[0][0][c] + sSum[1][0][c]) + (sSum[2][0][c] + sSum[3][0][c]);
    const float b = (sSum[0][1][c] + sSum[1][1][c]) + (sSum[2][1][c] + sSum[3][1][c]);
    const float d = beta * fmaf(-al * rk, a, vv[j]);
    if (rg == 0) op[c0 + j] = from_f32<T>(g.scale * rq * fmaf(al, b, qk * rk * d));
#pragma unroll
    for (int r = 0; r < RP; ++r) S[r].v[j] = fmaf(al, S[r].v[j], kd[r] * rk * d);
  }
#pragma unroll
  for (int r = 0; r < RP; ++r)
    if (rg + r * RG < g.DK) store_pack(sp + static_cast<int64_t>(rg + r * RG) * g.DV + c0, S[r]);
}

}  // namespace

hipError_t launch_delta_step(const DeltaGeom& g, const DeltaIn& in, float* states, void* o, int dtype, hipStream_t s) {
  const bool vec = g.DV % 4 == 0 && (reinterpret_cast<uintptr_t>(states) & 15) == 0;
  const int64_t heads = static_cast<int64_t>(g.q.S) * g.HV;
  return delta_dispatch(dtype, g.DK, [&](auto t, auto dkp) {
    using T = decltype(t);
    constexpr int DKP = decltype(dkp)::value;
    const auto launch = [&](auto kernel, int cols) {
      const uint32_t ncb = static_cast<uint32_t>((g.DV + cols - 1) / cols);
      hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(heads * ncb)), dim3(256), 0, s, g, in, ncb, states,
                         static_cast<T*>(o));
      return hipGetLastError();
    };
    if (!vec) return launch(delta_step_kernel<T, DKP, 32, 1>, 32);
    // Fewer heads than compute units: more workgroups, of 32 columns (12 heads of 128 x 128 6.2 us, 6.8 by 64 and 9.3 by
    // 128).  Else 64 (6144 of them 188 us, 194 by 32, 198 by 128, which leaves registers for three waves a SIMD), and
    // 128 where the state's rows are few and long (1000 heads of 40 x 100: 9.3 us, 13.7 by 64, 19 by 32).
    if (heads < 256) return launch(delta_step_kernel<T, DKP, 8, 4>, 32);
    if constexpr (DKP <= 64)
      if (g.DV > 64) return launch(delta_step_kernel<T, DKP, 32, 4>, 128);
    return launch(delta_step_kernel<T, DKP, 16, 4>, 64);
  });
}

}  // namespace mvm
