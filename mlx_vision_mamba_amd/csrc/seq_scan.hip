// Selective scan of packed sequences with states, forward, backward and one
// token, for gfx950.
//
//   h_t[n] = exp(delta_t A[n]) h_{t-1}[n] + delta_t u_t B_t[n]
//   y_t    = (sum_n C_t[n] h_t[n] + D u_t) * z_t sigmoid(z_t)
//
// A lane holds one channel with its 16 states in registers, a wave 64
// channels of one chunk of one sequence.  Everything that belongs to a
// (token, channel), the softplus and the gate among it, is computed once, and
// the sum over the states needs no other lane.  B and C are the same for the
// whole wave: they come through scalar loads and enter the vector
// instructions as scalar operands.  Each (token, channel, state) is then two
// multiplications, an exponential and two fused multiply-adds.
//
// Long sequences are cut into chunks: a first pass runs each chunk from a
// zero state for its end state, a small pass joins those in order (the decay
// over a chunk is one exponential of the summed delta), the main pass runs
// each chunk from its carry.
#include "mvm_scan.h"
#include "seq_common.h"

namespace mvm {

namespace {

constexpr int kWave = 64;
constexpr float kMaxA2 = 3.4028234e38f;

// A log2(e) of one channel's states 4q .. 4q + 3, 0 past N and for channels
// that do not exist.  Kept finite, so that a delta of zero always means no
// decay.
__device__ __forceinline__ void load_a2(float (&a)[4], const float* A, int64_t row, int q, int N, bool valid,
                                        int a_log) {
  load_ax4(a, A, row, q, N, valid, a_log);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float v = a[j] * kLog2e;
    a[j] = v < -kMaxA2 ? -kMaxA2 : (v > kMaxA2 ? kMaxA2 : v);
  }
}

// States 4q .. 4q + 3 of a channel of a state tensor (rows, D, N).
__device__ __forceinline__ void load_state4(float (&h)[4], const float* p, int64_t row, int64_t D, int64_t d, int q,
                                            int N, bool valid) {
  const float* at = p + (row * D + d) * N;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int n = 4 * q + j;
    const float v = at[n < N ? n : 0];
    h[j] = valid && n < N ? v : 0.f;
  }
}
__device__ __forceinline__ void store_state4(const float (&h)[4], float* p, int64_t row, int64_t D, int64_t d, int q,
                                             int N, bool valid) {
  float* at = p + (row * D + d) * N;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (valid && 4 * q + j < N) at[4 * q + j] = h[j];
}

// Rows of B | C for the kernels: the tensors themselves (rows of `st` values
// of T), or the float32 copy (rows of 32: B at 0, C at 16).  Wave-uniform row
// addresses through the constant address space: scalar loads.
template <typename T>
struct BcRows;
template <>
struct BcRows<float> {
  const float *B, *C;
  int64_t st;
  template <int N4>
  __device__ __forceinline__ static void get(float (&x)[N4], const float* p) {
    const const_f32* q = (const const_f32*)p;
#pragma unroll
    for (int n = 0; n < N4; ++n) x[n] = q[n];
  }
  template <int N4>
  __device__ __forceinline__ void b(float (&x)[N4], int32_t t, int n0) const { get(x, B + t * st + n0); }
  template <int N4>
  __device__ __forceinline__ void c(float (&x)[N4], int32_t t, int n0) const { get(x, C + t * st + n0); }
};
template <>
struct BcRows<bf16_t> {
  const bf16_t *B, *C;
  int64_t st;
  template <int N4>
  __device__ __forceinline__ static void get(float (&x)[N4], const bf16_t* p) {
    const const_u32* q = (const const_u32*)p;
#pragma unroll
    for (int n = 0; n < N4 / 2; ++n) {
      const uint32_t w = q[n];
      x[2 * n] = __uint_as_float(w << 16);
      x[2 * n + 1] = __uint_as_float(w & 0xffff0000u);
    }
  }
  template <int N4>
  __device__ __forceinline__ void b(float (&x)[N4], int32_t t, int n0) const { get(x, B + t * st + n0); }
  template <int N4>
  __device__ __forceinline__ void c(float (&x)[N4], int32_t t, int n0) const { get(x, C + t * st + n0); }
};

// kSeqTile rows of a channel-indexed tensor from row t on; rows past the
// chunk read its last one.
template <typename T>
__device__ __forceinline__ void load_tile(T (&v)[kSeqTile], const T* p, int64_t st, int32_t t, int32_t t1, int64_t d) {
#pragma unroll
  for (int i = 0; i < kSeqTile; ++i) {
    const int32_t r = t + i < t1 ? t + i : t1 - 1;
    v[i] = (p + r * st)[d];
  }
}

// ------------------------------------------------------------------ forward

struct FwdPtrs {
  const float* dbias;
  const float* A;
  const float* Dv;
  const float* h0;
  float* h1;
  float* ckpt;
  float* agg_h;
  float* agg_s;
};

// AGG: the end state of each chunk but a sequence's last from a zero state,
// and the sum of delta over it.  Otherwise the main pass.
template <typename T, typename DT, typename BT, bool AGG>
__global__ void __launch_bounds__(kWave)
seq_scan_fwd_kernel(SeqScanGeom g, FwdPtrs p, BcRows<BT> bc, uint32_t ncb, const T* __restrict__ u,
                    const DT* __restrict__ delta, const T* __restrict__ z, T* __restrict__ y) {
  const int lane = threadIdx.x;
  const BlockPos pos = block_pos(ncb);
  const SeqChunk c = seq_chunk(g.q, pos.slot, g.shift, lane);
  if (c.t0 < 0) return;
  const int64_t D = g.q.D;
  const int64_t d = static_cast<int64_t>(pos.cb) * kWave + lane;
  const bool valid = d < D;
  const int64_t dc = valid ? d : 0;
  if (c.seq == g.q.S) {  // rows of no sequence
    if constexpr (!AGG) {
      if (valid)
        for (int32_t t = c.t0; t < c.t1; ++t) y[t * g.ys + d] = from_f32<T>(0.f);
    }
    return;
  }
  if (AGG && c.t1 == c.end) return;
  float a2[16], h[16];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    float v[4];
    load_a2(v, p.A, dc * g.N, q, g.N, valid, g.a_log);
#pragma unroll
    for (int j = 0; j < 4; ++j) a2[4 * q + j] = v[j];
  }
  const int32_t row = seq_slot(g.q, c.seq);
  if (AGG) {
#pragma unroll
    for (int n = 0; n < 16; ++n) h[n] = 0.f;
  } else if (g.multi) {
    const float* at = p.agg_h + (static_cast<int64_t>(c.slot) * 4 * D + dc) * 4;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const Pack<float, 4> v = load_pack<float, 4>(at + q * 4 * D);
#pragma unroll
      for (int j = 0; j < 4; ++j) h[4 * q + j] = v.v[j];
    }
  } else {
    const bool any = p.h0 != nullptr && row >= 0 && !seq_fresh(g.q, c.seq);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float v[4] = {0.f, 0.f, 0.f, 0.f};
      if (any) load_state4(v, p.h0, row, D, dc, q, g.N, valid);
#pragma unroll
      for (int j = 0; j < 4; ++j) h[4 * q + j] = v[j];
    }
  }
  const float bias = p.dbias ? p.dbias[dc] : 0.f;
  const float Dd = AGG ? 0.f : p.Dv[dc];
  const bool soft = g.softplus != 0, gate = !AGG && z != nullptr;
  float sum_dl = 0.f;
  T nu[kSeqTile], nz[kSeqTile];
  DT nd[kSeqTile];
  auto fetch = [&](int32_t t) {
    load_tile(nu, u, g.us, t, c.t1, dc);
    load_tile(nd, delta, g.ds, t, c.t1, dc);
    if (gate) load_tile(nz, z, g.zs, t, c.t1, dc);
  };
  if (c.t0 < c.t1) fetch(c.t0);
  for (int32_t t = c.t0; t < c.t1; t += kSeqTile) {
    float du[kSeqTile], dl[kSeqTile], uf[kSeqTile], gz[kSeqTile];
#pragma unroll
    for (int i = 0; i < kSeqTile; ++i) {
      uf[i] = to_f32(nu[i]);
      dl[i] = to_f32(nd[i]) + bias;
      gz[i] = gate ? to_f32(nz[i]) : 1.f;
    }
    if (t + kSeqTile < c.t1) fetch(t + kSeqTile);
    if (soft) {
#pragma unroll
      for (int i = 0; i < kSeqTile; ++i) dl[i] = softplus_f(dl[i]);
    }
    if (gate) {
#pragma unroll
      for (int i = 0; i < kSeqTile; ++i) gz[i] *= sigmoid_f(gz[i]);
    }
#pragma unroll
    for (int i = 0; i < kSeqTile; ++i) du[i] = dl[i] * uf[i];
    if (!AGG && p.ckpt != nullptr) {
      const int64_t ck = (c.start >> kSeqTileShift) + c.seq + ((t - c.start) >> kSeqTileShift);
      float* at = p.ckpt + (ck * 4 * D + dc) * 4;
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (valid) store_pack(at + q * 4 * D, Pack<float, 4>{h[4 * q], h[4 * q + 1], h[4 * q + 2], h[4 * q + 3]});
    }
    auto step = [&](int i) {
      float Bv[16], acc[4] = {0.f, 0.f, 0.f, 0.f};
      bc.b(Bv, t + i, 0);
#pragma unroll
      for (int n = 0; n < 16; ++n) h[n] = fmaf(fast_exp2(dl[i] * a2[n]), h[n], du[i] * Bv[n]);
      if constexpr (AGG) {
        sum_dl += dl[i];
      } else {
        float Cv[16];
        bc.c(Cv, t + i, 0);
#pragma unroll
        for (int n = 0; n < 16; ++n) acc[n & 3] = fmaf(h[n], Cv[n], acc[n & 3]);
        const float r = fmaf(Dd, uf[i], (acc[0] + acc[1]) + (acc[2] + acc[3]));
        if (valid) (y + (t + i) * g.ys)[d] = from_f32<T>(r * gz[i]);
      }
    };
    if (t + kSeqTile <= c.t1) {
#pragma unroll
      for (int i = 0; i < kSeqTile; ++i) step(i);
    } else {
#pragma unroll
      for (int i = 0; i < kSeqTile; ++i)
        if (t + i < c.t1) step(i);
    }
  }
  if constexpr (AGG) {
    if (valid) {
      float* at = p.agg_h + (static_cast<int64_t>(c.slot) * 4 * D + d) * 4;
#pragma unroll
      for (int q = 0; q < 4; ++q)
        store_pack(at + q * 4 * D, Pack<float, 4>{h[4 * q], h[4 * q + 1], h[4 * q + 2], h[4 * q + 3]});
      p.agg_s[c.slot * D + d] = sum_dl;
    }
  } else if (c.t1 == c.end && p.h1 != nullptr && row >= 0) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float v[4] = {h[4 * q], h[4 * q + 1], h[4 * q + 2], h[4 * q + 3]};
      store_state4(v, p.h1, row, D, dc, q, g.N, valid);
    }
  }
}

// Carries over the chunks of one sequence, in order (REV: from its end): the
// aggregates are replaced by what enters each chunk.  A thread is one
// (channel, four states); the loads of several chunks are in flight together.
template <bool REV>
__global__ void __launch_bounds__(256)
seq_carry_kernel(SeqScanGeom g, uint32_t ncb, const float* __restrict__ A, const float* __restrict__ enter,
                 float* __restrict__ agg_h, const float* __restrict__ agg_s) {
  const BlockPos pos = block_pos(ncb);
  const int32_t seq = pos.slot, q = threadIdx.x >> 6;
  const int64_t D = g.q.D, d = static_cast<int64_t>(pos.cb) * kWave + (threadIdx.x & 63);
  if (d >= D) return;
  const int32_t start = seq_off_u(g.q, seq), next = seq_off_u(g.q, seq + 1);
  const int64_t len = next > start ? next - start : 0;
  const int32_t n = static_cast<int32_t>((len + (int64_t{1} << g.shift) - 1) >> g.shift);
  const int32_t row = seq_slot(g.q, seq);
  float a2[4], h[4] = {0.f, 0.f, 0.f, 0.f};
  load_a2(a2, A, d * g.N, q, g.N, true, g.a_log);
  if (enter != nullptr && row >= 0 && !seq_fresh(g.q, seq)) load_state4(h, enter, row, D, d, q, g.N, true);
  const int64_t base = (start >> g.shift) + seq;
  auto at = [&](int32_t j) {  // j-th chunk in the carry's order
    return base + (REV ? n - 1 - j : j);
  };
  for (int32_t j0 = 0; j0 < n; j0 += kCarryBatch) {
    Pack<float, 4> v[kCarryBatch];
    float s[kCarryBatch];
#pragma unroll
    for (int i = 0; i < kCarryBatch; ++i) {
      // the last chunk in order has no aggregate: nothing follows it
      const int64_t slot = at(j0 + i < n ? j0 + i : n - 1);
      v[i] = load_pack<float, 4>(agg_h + ((slot * 4 + q) * D + d) * 4);
      s[i] = agg_s[slot * D + d];
    }
#pragma unroll
    for (int i = 0; i < kCarryBatch; ++i) {
      if (j0 + i >= n) break;
      store_pack(agg_h + ((at(j0 + i) * 4 + q) * D + d) * 4, Pack<float, 4>{h[0], h[1], h[2], h[3]});
#pragma unroll
      for (int j = 0; j < 4; ++j) h[j] = fmaf(fast_exp2(a2[j] * s[i]), h[j], v[i].v[j]);
    }
  }
  // an empty sequence's one chunk
  if (n == 0) store_pack(agg_h + ((base * 4 + q) * D + d) * 4, Pack<float, 4>{h[0], h[1], h[2], h[3]});
}

// Float32 copies of B | C in rows of 32, zero past N.
template <typename T>
__global__ void __launch_bounds__(256)
seq_bc_kernel(int32_t T_, int32_t N, int64_t st, const T* __restrict__ Bm, const T* __restrict__ Cm,
              float* __restrict__ out) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t t = i >> 5;
  const int n = static_cast<int>(i & 15);
  if (t >= T_) return;
  const T* src = (i & 16) ? Cm : Bm;
  out[i] = n < N ? to_f32(src[t * st + n]) : 0.f;
}

// ----------------------------------------------------------------- backward
//
//   dr_t = dy_t silu(z_t),  dh_t = C_t dr_t + c_{t+1},  c_t = exp(delta_t A) dh_t
//   dB_t = sum_d dh_t delta_t u_t,  dC_t = sum_d dr_t h_t,
//   ddelta_t = sum_n dh_t (A exp(delta_t A) h_{t-1} + B_t u_t),
//   du_t = delta_t sum_n dh_t B_t + D dr_t,  dA = sum_t dh_t delta_t exp(delta_t A) h_{t-1}
//
// with c past a sequence's end the final state's gradient, and c_first the
// initial state's.  The same three passes as forward, in the other direction.

struct BwdPtrs {
  const float* dbias;
  const float* A;
  const float* Dv;
  const float* dh1;
  float* dh0;
  const float* ckpt;
  float* agg_h;
  float* agg_s;
  float* part;
  float* part_bc;
};

// The adjoint that leaves each chunk but a sequence's first to its front, from
// zero, and the sum of delta.
template <typename T, typename DT, typename BT>
__global__ void __launch_bounds__(kWave)
seq_scan_bwd_agg_kernel(SeqScanGeom g, BwdPtrs p, BcRows<BT> bc, uint32_t ncb, const DT* __restrict__ delta,
                        const T* __restrict__ z, const T* __restrict__ dy) {
  const int lane = threadIdx.x;
  const BlockPos pos = block_pos(ncb);
  const SeqChunk c = seq_chunk(g.q, pos.slot, g.shift, lane);
  if (c.t0 <= c.start || c.seq == g.q.S) return;
  const int64_t D = g.q.D;
  const int64_t d = static_cast<int64_t>(pos.cb) * kWave + lane;
  const bool valid = d < D;
  const int64_t dc = valid ? d : 0;
  float a2[16], h[16];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    float v[4];
    load_a2(v, p.A, dc * g.N, q, g.N, valid, g.a_log);
#pragma unroll
    for (int j = 0; j < 4; ++j) a2[4 * q + j] = v[j];
  }
#pragma unroll
  for (int n = 0; n < 16; ++n) h[n] = 0.f;
  const float bias = p.dbias ? p.dbias[dc] : 0.f;
  const bool soft = g.softplus != 0, gate = z != nullptr;
  float sum_dl = 0.f;
  T ny[kSeqTile], nz[kSeqTile];
  DT nd[kSeqTile];
  auto fetch = [&](int32_t t) {
    load_tile(ny, dy, g.ys, t, c.t1, dc);
    load_tile(nd, delta, g.ds, t, c.t1, dc);
    if (gate) load_tile(nz, z, g.zs, t, c.t1, dc);
  };
  const int32_t last = c.t0 + ((c.t1 - 1 - c.t0) & ~(kSeqTile - 1));
  fetch(last);
  for (int32_t t = last; t >= c.t0; t -= kSeqTile) {
    float dl[kSeqTile], dr[kSeqTile], zf[kSeqTile];
#pragma unroll
    for (int i = 0; i < kSeqTile; ++i) {
      dl[i] = to_f32(nd[i]) + bias;
      dr[i] = to_f32(ny[i]);
      zf[i] = gate ? to_f32(nz[i]) : 0.f;
    }
    if (t > c.t0) fetch(t - kSeqTile);
    if (soft) {
#pragma unroll
      for (int i = 0; i < kSeqTile; ++i) dl[i] = softplus_f(dl[i]);
    }
    if (gate) {
#pragma unroll
      for (int i = 0; i < kSeqTile; ++i) dr[i] *= zf[i] * sigmoid_f(zf[i]);
    }
    auto step = [&](int i) {
      float Cv[16];
      bc.c(Cv, t + i, 0);
#pragma unroll
      for (int n = 0; n < 16; ++n) h[n] = fast_exp2(dl[i] * a2[n]) * fmaf(Cv[n], dr[i], h[n]);
      sum_dl += dl[i];
    };
    if (t + kSeqTile <= c.t1) {
#pragma unroll
      for (int i = kSeqTile - 1; i >= 0; --i) step(i);
    } else {
#pragma unroll
      for (int i = kSeqTile - 1; i >= 0; --i)
        if (t + i < c.t1) step(i);
    }
  }
  if (valid) {
    float* at = p.agg_h + (static_cast<int64_t>(c.slot) * 4 * D + d) * 4;
#pragma unroll
    for (int q = 0; q < 4; ++q)
      store_pack(at + q * 4 * D, Pack<float, 4>{h[4 * q], h[4 * q + 1], h[4 * q + 2], h[4 * q + 3]});
    p.agg_s[c.slot * D + d] = sum_dl;
  }
}

// v[0..15] summed over the wave's 64 lanes: the sum of v[k] is in the lanes
// with (lane >> 2) == k.  17 additions for 16 sums: each level halves the
// values that a lane holds by trading with a lane across bit 5, 4, 3 or 2.
__device__ __forceinline__ float wave_sums16(const float (&v)[16], int lane) {
  float a[8], b[4], e[2];
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] = pair_reduce32(v[i], v[i + 8]);
#pragma unroll
  for (int i = 0; i < 4; ++i) b[i] = pair_reduce16(a[i], a[i + 4]);
  const bool hi8 = (lane & 8) != 0, hi4 = (lane & 4) != 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float keep = hi8 ? b[i + 2] : b[i], give = hi8 ? b[i] : b[i + 2];
    e[i] = keep + dpp<kRowRor8>(give);
  }
  // a row rotation by 4 would pair lanes across bit 3; mirroring a half row
  // (lane ^ 7) pairs across bit 2 within it
  const float keep = hi4 ? e[1] : e[0], give = hi4 ? e[0] : e[1];
  float s = keep + dpp<0x141>(give);
  s += dpp<kQuadXor1>(s);
  s += dpp<kQuadXor2>(s);
  return s;
}

// The main pass.  Per tile of 8 tokens the states are taken four at a time
// (an inner loop that is not unrolled): the tile is run forward from its
// checkpoint with the states and decays kept in registers, then backward.
// What a state carries from tile to tile (its adjoint and dA) waits in LDS.
template <typename T, typename DT, typename BT>
__global__ void __launch_bounds__(kWave)
seq_scan_bwd_kernel(SeqScanGeom g, BwdPtrs p, BcRows<BT> bc, uint32_t ncb, const T* __restrict__ u,
                    const DT* __restrict__ delta, const T* __restrict__ z, const T* __restrict__ dy,
                    T* __restrict__ du_out, DT* __restrict__ dd_out, T* __restrict__ dz_out) {
  __shared__ Pack<float, 4> sA2[4][kWave], sC[4][kWave], sDA[4][kWave];
  __shared__ float sBC[16][17];  // [token | 8 for dC][state]
  const int lane = threadIdx.x;
  const BlockPos pos = block_pos(ncb);
  const SeqChunk c = seq_chunk(g.q, pos.slot, g.shift, lane);
  const int64_t D = g.q.D;
  const int64_t d = static_cast<int64_t>(pos.cb) * kWave + lane;
  const bool valid = d < D;
  const int64_t dc = valid ? d : 0;
  float* part = p.part + (static_cast<int64_t>(pos.slot) * 18) * D + d;
  if (c.t0 < 0 || c.seq == g.q.S) {
    if (valid)
      for (int i = 0; i < 18; ++i) part[i * D] = 0.f;
    for (int32_t t = c.t0; t < c.t1; ++t) {  // (c.t1 == c.t0 without a chunk)
      if (valid) {
        du_out[t * D + d] = from_f32<T>(0.f);
        dd_out[t * D + d] = from_f32<DT>(0.f);
        if (dz_out) dz_out[t * D + d] = from_f32<T>(0.f);
      }
      if (lane < 32) p.part_bc[(static_cast<int64_t>(pos.cb) * g.q.T + t) * 32 + lane] = 0.f;
    }
    return;
  }
  const int32_t row = seq_slot(g.q, c.seq);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    float a2[4], h[4] = {0.f, 0.f, 0.f, 0.f};
    load_a2(a2, p.A, dc * g.N, q, g.N, valid, g.a_log);
    if (g.multi) {
      const Pack<float, 4> v = load_pack<float, 4>(p.agg_h + ((static_cast<int64_t>(c.slot) * 4 + q) * D + dc) * 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) h[j] = v.v[j];
    } else if (p.dh1 != nullptr) {
      load_state4(h, p.dh1, row, D, dc, q, g.N, valid);
    }
    sA2[q][lane] = Pack<float, 4>{a2[0], a2[1], a2[2], a2[3]};
    sC[q][lane] = Pack<float, 4>{h[0], h[1], h[2], h[3]};
    sDA[q][lane] = Pack<float, 4>{0.f, 0.f, 0.f, 0.f};
  }
  const float bias = p.dbias ? p.dbias[dc] : 0.f;
  const float Dd = valid ? p.Dv[dc] : 0.f;
  const bool soft = g.softplus != 0, gate = z != nullptr;
  float dD = 0.f, ddb = 0.f;
  T nu[kSeqTile], ny[kSeqTile], nz[kSeqTile];
  DT nd[kSeqTile];
  auto fetch = [&](int32_t t) {
    load_tile(nu, u, g.us, t, c.t1, dc);
    load_tile(nd, delta, g.ds, t, c.t1, dc);
    load_tile(ny, dy, g.ys, t, c.t1, dc);
    if (gate) load_tile(nz, z, g.zs, t, c.t1, dc);
  };
  const int64_t ck0 = (c.start >> kSeqTileShift) + c.seq;
  const int32_t last = c.t0 + ((c.t1 - 1 - c.t0) & ~(kSeqTile - 1));
  if (c.t0 < c.t1) fetch(last);
  for (int32_t t = last; c.t0 < c.t1 && t >= c.t0; t -= kSeqTile) {
    float uf[kSeqTile], raw[kSeqTile], dl[kSeqTile], du[kSeqTile], dr[kSeqTile], yf[kSeqTile], zf[kSeqTile];
    float qs[kSeqTile], ws[kSeqTile], rs[kSeqTile];
#pragma unroll
    for (int i = 0; i < kSeqTile; ++i) {
      // rows past the chunk: nothing decays, enters or leaves
      const bool in = valid && t + i < c.t1;
      uf[i] = in ? to_f32(nu[i]) : 0.f;
      raw[i] = to_f32(nd[i]) + bias;
      yf[i] = in ? to_f32(ny[i]) : 0.f;
      zf[i] = gate ? to_f32(nz[i]) : 0.f;
      dl[i] = raw[i];
      dr[i] = yf[i];
      qs[i] = ws[i] = rs[i] = 0.f;
    }
    if (t > c.t0) fetch(t - kSeqTile);
    if (soft) {
#pragma unroll
      for (int i = 0; i < kSeqTile; ++i) dl[i] = softplus_f(dl[i]);
    }
    if (gate) {
#pragma unroll
      for (int i = 0; i < kSeqTile; ++i) dr[i] *= zf[i] * sigmoid_f(zf[i]);
    }
#pragma unroll
    for (int i = 0; i < kSeqTile; ++i) {
      dl[i] = valid && t + i < c.t1 ? dl[i] : 0.f;
      du[i] = dl[i] * uf[i];
    }
    const float* ck = p.ckpt + ((ck0 + ((t - c.start) >> kSeqTileShift)) * 4 * D + dc) * 4;
#pragma unroll 1
    for (int q = 0; q < 4; ++q) {
      const Pack<float, 4> hs = load_pack<float, 4>(ck + q * 4 * D), a2 = sA2[q][lane];
      Pack<float, 4> cs = sC[q][lane], da = sDA[q][lane];
      float Bv[kSeqTile][4], Cv[kSeqTile][4];
#pragma unroll
      for (int i = 0; i < kSeqTile; ++i) {
        const int32_t r = t + i < c.t1 ? t + i : c.t1 - 1;
        bc.b(Bv[i], r, 4 * q);
        bc.c(Cv[i], r, 4 * q);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float h = valid ? hs.v[j] : 0.f;
        float a[kSeqTile], ah[kSeqTile], hh[kSeqTile];
#pragma unroll
        for (int i = 0; i < kSeqTile; ++i) {
          a[i] = fast_exp2(dl[i] * a2.v[j]);
          ah[i] = a[i] * h;
          h = hh[i] = fmaf(du[i], Bv[i][j], ah[i]);
          rs[i] = fmaf(h, Cv[i][j], rs[i]);
        }
        float v[16];  // the terms of dB of the 8 tokens, then those of dC
#pragma unroll
        for (int i = kSeqTile - 1; i >= 0; --i) {
          const float dh = fmaf(Cv[i][j], dr[i], cs.v[j]);
          qs[i] = fmaf(dh, Bv[i][j], qs[i]);
          v[i] = dh * du[i];
          v[8 + i] = dr[i] * hh[i];
          const float w = dh * ah[i];
          da.v[j] = fmaf(w, dl[i], da.v[j]);
          ws[i] = fmaf(w, a2.v[j], ws[i]);
          cs.v[j] = dh * a[i];
        }
        const float s = wave_sums16(v, lane);
        if ((lane & 3) == 0) sBC[lane >> 2][4 * q + j] = s;
      }
      sC[q][lane] = cs;
      sDA[q][lane] = da;
    }
    __syncthreads();
    // rows t .. t + 7 of 32 values: dB at 0, dC at 16
    float* out = p.part_bc + (static_cast<int64_t>(pos.cb) * g.q.T + t) * 32;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = k * 2 + (lane >> 5), n = lane & 31;
      if (t + i < c.t1) out[i * 32 + n] = sBC[i + ((n >> 4) << 3)][n & 15];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSeqTile; ++i) {
      if (valid && t + i < c.t1) {
        const int64_t at = static_cast<int64_t>(t + i) * D + d;
        dD = fmaf(dr[i], uf[i], dD);
        du_out[at] = from_f32<T>(fmaf(qs[i], dl[i], Dd * dr[i]));
        float dd = fmaf(ws[i], kLn2, qs[i] * uf[i]);
        if (soft) dd *= sigmoid_f(raw[i]);
        ddb += dd;
        dd_out[at] = from_f32<DT>(dd);
        if (gate) {
          const float sg = sigmoid_f(zf[i]);
          dz_out[at] = from_f32<T>(yf[i] * fmaf(Dd, uf[i], rs[i]) * sg * fmaf(zf[i], 1.f - sg, 1.f));
        }
      }
    }
  }
  if (!valid) return;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const Pack<float, 4> da = sDA[q][lane], cs = sC[q][lane];
#pragma unroll
    for (int j = 0; j < 4; ++j) part[(4 * q + j) * D] = da.v[j];
    if (c.t0 == c.start && p.dh0 != nullptr) store_state4(cs.v, p.dh0, row, D, d, q, g.N, true);
  }
  part[16 * D] = dD;
  part[17 * D] = ddb;
}

// dA, dD and ddelta_bias: the chunks' sums, added in order.
__global__ void __launch_bounds__(1024)
seq_reduce_params_kernel(int64_t D, int32_t N, int64_t nparts, int a_log, const float* __restrict__ A,
                         const float* __restrict__ part, float* __restrict__ dA, float* __restrict__ dD,
                         float* __restrict__ ddb) {
  sum_columns(part, nparts, 18 * D, [&](int64_t col, float s) {
    const int64_t k = col / D, d = col - k * D;
    if (k < N)
      dA[d * N + k] = a_log ? s * -expf(A[d * N + k]) : s;  // of A_log: A' = A
    else if (k == 16)
      dD[d] = s;
    else if (k == 17 && ddb != nullptr)
      ddb[d] = s;
  });
}

// dB and dC: the channel blocks' sums, added in order.
template <typename T>
__global__ void __launch_bounds__(256)
seq_reduce_bc_kernel(int32_t rows, int32_t N, int32_t ncb, const float* __restrict__ part, T* __restrict__ dB,
                     T* __restrict__ dC) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t total = static_cast<int64_t>(rows) * 32;
  if (i >= total) return;
  float s = 0.f;
  for (int32_t k0 = 0; k0 < ncb; k0 += 8) {
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = part[(k0 + k < ncb ? k0 + k : 0) * total + i];
#pragma unroll
    for (int k = 0; k < 8; ++k) s += k0 + k < ncb ? v[k] : 0.f;
  }
  const int n = static_cast<int>(i & 15);
  if (n < N) ((i & 16) ? dC : dB)[(i >> 5) * N + n] = from_f32<T>(s);
}

// --------------------------------------------------------------- one token

// Lane 4c + q holds states 4q .. 4q + 3 of channel c: a wave reads 16
// channels' states, 1 KB, at once.  Bound by the states' traffic.  VEC: the
// states are read four at a time (N a multiple of 4).
template <typename T, typename DT, bool VEC>
__global__ void __launch_bounds__(256)
seq_scan_step_kernel(SeqScanGeom g, uint32_t ncb, const T* __restrict__ u, const DT* __restrict__ delta,
                     const float* __restrict__ dbias, const float* __restrict__ A, const T* __restrict__ Bm,
                     const T* __restrict__ Cm, const float* __restrict__ Dv, const T* __restrict__ z,
                     float* __restrict__ states, T* __restrict__ y) {
  const BlockPos pos = block_pos(ncb);
  const int q = threadIdx.x & 3, N = g.N;
  const int64_t D = g.q.D, d = static_cast<int64_t>(pos.cb) * 64 + (threadIdx.x >> 2);
  const bool valid = d < D;
  const int64_t dc = valid ? d : 0;
  const int32_t i = pos.slot;
  const int32_t row = seq_slot(g.q, i);
  T* yr = y + i * g.ys;
  if (row < 0) {
    if (valid && q == 0) yr[d] = from_f32<T>(0.f);
    return;
  }
  const bool fresh = seq_fresh(g.q, i), mine = valid && 4 * q < N;
  float* at = states + (row * D + dc) * N + (mine ? 4 * q : 0);
  float h[4], a2[4], b[4], c[4];
  if constexpr (VEC) {
    const Pack<float, 4> v = load_pack<float, 4>(at);
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = v.v[j];
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = at[mine && 4 * q + j < N ? j : 0];
  }
  const float uf = to_f32(u[i * g.us + dc]), zf = z ? to_f32(z[i * g.zs + dc]) : 0.f;
  float dl = to_f32(delta[i * g.ds + dc]) + (dbias ? dbias[dc] : 0.f);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int n = 4 * q + j < N ? 4 * q + j : 0;
    b[j] = to_f32(Bm[i * g.bs + n]);
    c[j] = to_f32(Cm[i * g.bs + n]);
  }
  load_a2(a2, A, dc * N, q, N, valid, g.a_log);
  if (g.softplus) dl = softplus_f(dl);
  const float du = dl * uf;
  float r = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const bool in = 4 * q + j < N;
    h[j] = fmaf(fast_exp2(dl * a2[j]), fresh ? 0.f : h[j], du * b[j]);
    r = in ? fmaf(h[j], c[j], r) : r;
  }
  if (mine) {
    if constexpr (VEC) {
      store_pack(at, Pack<float, 4>{h[0], h[1], h[2], h[3]});
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (4 * q + j < N) at[j] = h[j];
    }
  }
  r = sum_groups(r);
  r = fmaf(Dv[dc], uf, r);
  if (z) r *= zf * sigmoid_f(zf);
  if (valid && q == 0) yr[d] = from_f32<T>(r);
}

// ----------------------------------------------------------------- launches

uint32_t blocks_of(int64_t D) { return static_cast<uint32_t>((D + kWave - 1) / kWave); }

template <typename T>
hipError_t copy_bc(const SeqScanGeom& g, const SeqScanIn& in, float* out, hipStream_t s) {
  const int64_t n = static_cast<int64_t>(g.q.T) * 32;
  if (n == 0) return hipSuccess;
  hipLaunchKernelGGL(seq_bc_kernel<T>, dim3(static_cast<unsigned>((n + 255) / 256)), dim3(256), 0, s, g.q.T, g.N, g.bs,
                     static_cast<const T*>(in.Bm), static_cast<const T*>(in.Cm), out);
  return hipGetLastError();
}

template <typename T, typename DT, typename BT>
hipError_t fwd_t(const SeqScanGeom& g, const SeqScanIn& in, const SeqScanFwd& b, BcRows<BT> bc, hipStream_t s) {
  const uint32_t ncb = blocks_of(g.q.D);
  const dim3 grid(static_cast<unsigned>(chunk_slots(g.q, g.shift) * ncb));
  const FwdPtrs p{in.dbias, in.A, in.Dv, b.h0, b.h1, b.ckpt, b.agg_h, b.agg_s};
  const T* u = static_cast<const T*>(in.u);
  const DT* delta = static_cast<const DT*>(in.delta);
  const T* z = static_cast<const T*>(in.z);
  T* y = static_cast<T*>(b.y);
  if (g.multi) {
    hipLaunchKernelGGL((seq_scan_fwd_kernel<T, DT, BT, true>), grid, dim3(kWave), 0, s, g, p, bc, ncb, u, delta, z, y);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (g.q.S > 0) {
      hipLaunchKernelGGL(seq_carry_kernel<false>, dim3(ncb * static_cast<unsigned>(g.q.S)), dim3(256), 0, s, g, ncb,
                         in.A, b.h0, b.agg_h, b.agg_s);
      e = hipGetLastError();
      if (e != hipSuccess) return e;
    }
  }
  hipLaunchKernelGGL((seq_scan_fwd_kernel<T, DT, BT, false>), grid, dim3(kWave), 0, s, g, p, bc, ncb, u, delta, z, y);
  return hipGetLastError();
}

template <typename T, typename DT, typename BT>
hipError_t bwd_t(const SeqScanGeom& g, const SeqScanIn& in, const SeqScanBwd& b, BcRows<BT> bc, hipStream_t s) {
  const uint32_t ncb = blocks_of(g.q.D);
  const int64_t slots = chunk_slots(g.q, g.shift);
  const dim3 grid(static_cast<unsigned>(slots * ncb));
  const BwdPtrs p{in.dbias, in.A, in.Dv, b.dh1, b.dh0, b.ckpt, b.agg_h, b.agg_s, b.part, b.part_bc};
  const T* u = static_cast<const T*>(in.u);
  const DT* delta = static_cast<const DT*>(in.delta);
  const T* z = static_cast<const T*>(in.z);
  const T* dy = static_cast<const T*>(b.dy);
  hipError_t e;
  if (g.multi) {
    hipLaunchKernelGGL((seq_scan_bwd_agg_kernel<T, DT, BT>), grid, dim3(kWave), 0, s, g, p, bc, ncb, delta, z, dy);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    if (g.q.S > 0) {
      hipLaunchKernelGGL(seq_carry_kernel<true>, dim3(ncb * static_cast<unsigned>(g.q.S)), dim3(256), 0, s, g, ncb,
                         in.A, b.dh1, b.agg_h, b.agg_s);
      if ((e = hipGetLastError()) != hipSuccess) return e;
    }
  }
  hipLaunchKernelGGL((seq_scan_bwd_kernel<T, DT, BT>), grid, dim3(kWave), 0, s, g, p, bc, ncb, u, delta, z, dy,
                     static_cast<T*>(b.du), static_cast<DT*>(b.ddelta), static_cast<T*>(b.dz));
  if ((e = hipGetLastError()) != hipSuccess) return e;
  hipLaunchKernelGGL(seq_reduce_params_kernel, dim3(static_cast<unsigned>((18 * g.q.D + 63) / 64)), dim3(1024), 0, s,
                     g.q.D, g.N, slots, g.a_log, in.A, b.part, b.dA, b.dD, b.ddbias);
  if ((e = hipGetLastError()) != hipSuccess) return e;
  const int64_t n = static_cast<int64_t>(g.q.T) * 32;
  if (n == 0) return hipSuccess;
  hipLaunchKernelGGL(seq_reduce_bc_kernel<T>, dim3(static_cast<unsigned>((n + 255) / 256)), dim3(256), 0, s, g.q.T,
                     g.N, static_cast<int32_t>(ncb), b.part_bc, static_cast<T*>(b.dB), static_cast<T*>(b.dC));
  return hipGetLastError();
}

// B and C as the kernels read them: in place, or from the float32 copy made here
template <typename T, typename DT, typename Buf, typename F>
hipError_t with_bc(const SeqScanGeom& g, const SeqScanIn& in, const Buf& b, F&& f, hipStream_t s) {
  if (b.bc == nullptr)
    return f(BcRows<T>{static_cast<const T*>(in.Bm), static_cast<const T*>(in.Cm), g.bs});
  const hipError_t e = copy_bc<T>(g, in, b.bc, s);
  return e != hipSuccess ? e : f(BcRows<float>{b.bc, b.bc + 16, 32});
}

template <typename T, typename DT>
hipError_t step_t(const SeqScanGeom& g, const SeqScanIn& in, float* states, void* y, hipStream_t s) {
  const uint32_t ncb = static_cast<uint32_t>((g.q.D + 63) / 64);
  const dim3 grid(ncb * static_cast<unsigned>(g.q.S));
  const bool vec = g.N % 4 == 0 && (reinterpret_cast<uintptr_t>(states) & 15) == 0;
  auto run = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, g, ncb, static_cast<const T*>(in.u),
                       static_cast<const DT*>(in.delta), in.dbias, in.A, static_cast<const T*>(in.Bm),
                       static_cast<const T*>(in.Cm), in.Dv, static_cast<const T*>(in.z), states, static_cast<T*>(y));
    return hipGetLastError();
  };
  return vec ? run(seq_scan_step_kernel<T, DT, true>) : run(seq_scan_step_kernel<T, DT, false>);
}

// f<T, DT>(): T the activations' type, DT delta's
template <typename F>
hipError_t by_types(int dtype, int delta_dtype, F&& f) {
  if (dtype == MVM_F32) return f(float{}, float{});
  return delta_dtype == MVM_F32 ? f(bf16_t{}, float{}) : f(bf16_t{}, bf16_t{});
}

}  // namespace

bool seq_bc_in_place(const SeqScanGeom& g, const SeqScanIn& in, int dtype) {
  if (g.N != 16) return false;
  if (dtype == MVM_F32) return true;
  return g.bs % 2 == 0 && ((reinterpret_cast<uintptr_t>(in.Bm) | reinterpret_cast<uintptr_t>(in.Cm)) & 3) == 0;
}

hipError_t launch_seq_scan_fwd(const SeqScanGeom& g, const SeqScanIn& in, const SeqScanFwd& b, int dtype,
                               int delta_dtype, hipStream_t s) {
  return by_types(dtype, delta_dtype, [&](auto t, auto dt) {
    using T = decltype(t);
    using DT = decltype(dt);
    return with_bc<T, DT>(g, in, b, [&](auto bc) { return fwd_t<T, DT>(g, in, b, bc, s); }, s);
  });
}

hipError_t launch_seq_scan_bwd(const SeqScanGeom& g, const SeqScanIn& in, const SeqScanBwd& b, int dtype,
                               int delta_dtype, hipStream_t s) {
  return by_types(dtype, delta_dtype, [&](auto t, auto dt) {
    using T = decltype(t);
    using DT = decltype(dt);
    return with_bc<T, DT>(g, in, b, [&](auto bc) { return bwd_t<T, DT>(g, in, b, bc, s); }, s);
  });
}

hipError_t launch_seq_scan_step(const SeqScanGeom& g, const SeqScanIn& in, float* states, void* y, int dtype,
                                int delta_dtype, hipStream_t s) {
  return by_types(dtype, delta_dtype, [&](auto t, auto dt) {
    return step_t<decltype(t), decltype(dt)>(g, in, states, y, s);
  });
}

}  // namespace mvm
