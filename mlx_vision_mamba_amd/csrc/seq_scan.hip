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
#include <algorithm>

#include "mvm_scan.h"
#include "seq_common.h"

namespace mvm {

namespace {

constexpr int kWave = 64;
constexpr float kMaxA2 = 3.4028234e38f;
constexpr float kLog2eLow = 1.925963e-8f;  // log2(e) - kLog2e

// A log2(e) of one channel's states from n0 on, 0 past N.  Kept finite, so
// that a delta of zero always means no decay.  A = -exp(A_log) by the
// exponential unit: the rounding error of A_log log2(e) is put back by its
// first-order term (2 ulp of A; the routine of the maths library costs 20
// instructions a state, as much as 4 tokens of the scan).
template <int COUNT>
__device__ __forceinline__ void load_a2(float (&a)[COUNT], const float* A, int64_t row, int n0, int N, int a_log) {
#pragma unroll
  for (int j = 0; j < COUNT; ++j) a[j] = A[row + state_col(n0 + j, N)];
  if (a_log) {
#pragma unroll
    for (int j = 0; j < COUNT; ++j) {
      const float x = a[j] > 88.f ? 88.f : (a[j] < -128.f ? -128.f : a[j]);  // (NaN stays)
      const float hi = x * kLog2e, lo = fmaf(x, kLog2eLow, fmaf(x, kLog2e, -hi));
      const float e = fast_exp2(hi);
      a[j] = -fmaf(e * kLn2, lo, e);
    }
  }
#pragma unroll
  for (int j = 0; j < COUNT; ++j) {
    const float x = a[j] * kLog2e;
    a[j] = n0 + j < N ? (x < -kMaxA2 ? -kMaxA2 : (x > kMaxA2 ? kMaxA2 : x)) : 0.f;
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
// addresses through the constant address space: scalar loads.  A kernel asks
// for N4 values as they lie (Raw) and takes them apart where it needs them.
template <typename T>
struct BcRows;
template <>
struct BcRows<float> {
  const float *B, *C;
  int64_t st;
  template <int N4>
  struct Raw {
    float w[N4];
    __device__ __forceinline__ void load(uint64_t at) {
      const const_f32* q = (const const_f32*)at;
#pragma unroll
      for (int n = 0; n < N4; ++n) w[n] = q[n];
    }
    __device__ __forceinline__ float operator[](int n) const { return w[n]; }
  };
};
template <>
struct BcRows<bf16_t> {
  const bf16_t *B, *C;
  int64_t st;
  template <int N4>
  struct Raw {
    uint32_t w[N4 / 2];
    __device__ __forceinline__ void load(uint64_t at) {
      const const_u32* q = (const const_u32*)at;
#pragma unroll
      for (int n = 0; n < N4 / 2; ++n) w[n] = q[n];
    }
    __device__ __forceinline__ float operator[](int n) const {
      return __uint_as_float((n & 1) ? w[n / 2] & 0xffff0000u : w[n / 2] << 16);
    }
  };
};

// A row of a tensor as a wave walks along it: a wave-uniform address that
// moves by whole rows.  The empty asm keeps each step's sum in the scalar unit
// where it stands: left to itself the compiler forms the addresses of all rows
// of a tile at once, and has no scalar registers for them.
struct RowPtr {
  uint64_t at;
  uint32_t st;  // bytes (below 2^31: checked on the host)
  template <typename T>
  __device__ __forceinline__ void set(const T* p, int64_t row, int64_t stride) {
    st = static_cast<uint32_t>(stride * static_cast<int64_t>(sizeof(T)));
    at = reinterpret_cast<uint64_t>(p) + row * st;
  }
  __device__ __forceinline__ void next(bool go = true) {
    at += go ? st : 0u;
    asm volatile("" : "+s"(at));
  }
  __device__ __forceinline__ void prev(bool go) {
    at -= go ? st : 0u;
    asm volatile("" : "+s"(at));
  }
  template <typename T>
  __device__ __forceinline__ const T* global() const {
    return (const T*)(const __attribute__((address_space(1))) T*)at;
  }
  template <typename T>
  __device__ __forceinline__ T load(uint32_t lane) const {
    return global<T>()[lane];
  }
  template <typename T>
  __device__ __forceinline__ void store(uint32_t lane, float v) const {
    const_cast<T*>(global<T>())[lane] = from_f32<T>(v);
  }
};

// The next kSeqTile rows, from row t on; rows past the chunk read its last one.
template <typename T>
__device__ __forceinline__ void load_next(T (&v)[kSeqTile], RowPtr& p, int32_t t, int32_t t1, uint32_t lane) {
#pragma unroll
  for (int i = 0; i < kSeqTile; ++i) {
    v[i] = p.load<T>(lane);
    p.next(t + i + 1 < t1);
  }
}
// The kSeqTile rows from row t on, last one first: p is at row t + 7, or at
// the chunk's last, and comes to rest at row t - 1 (t0 at the least).
template <typename T>
__device__ __forceinline__ void load_prev(T (&v)[kSeqTile], RowPtr& p, int32_t t, int32_t t0, int32_t t1,
                                          uint32_t lane) {
#pragma unroll
  for (int i = kSeqTile - 1; i >= 0; --i) {
    v[i] = p.load<T>(lane);
    p.prev(t + i < t1 && t + i > t0);
  }
}
// The first `rows` of the next kSeqTile rows.
template <typename T>
__device__ __forceinline__ void store_next(RowPtr& p, int32_t rows, uint32_t lane, const float (&v)[kSeqTile]) {
  if (rows >= kSeqTile) {
#pragma unroll
    for (int i = 0; i < kSeqTile; ++i) {
      p.store<T>(lane, v[i]);
      p.next();
    }
  } else {
#pragma unroll
    for (int i = 0; i < kSeqTile; ++i)
      if (i < rows) {
        p.store<T>(lane, v[i]);
        p.next();
      }
  }
}

// A SIMD issues for its oldest wave first, so of the waves that start together
// the first would end early and the last run alone, at half the rate.  A wave
// lowers its priority when half, a quarter and an eighth of its chunk are left:
// those behind catch up.
struct Pace {
  int32_t left, next, level;
  __device__ __forceinline__ explicit Pace(int32_t len) : left(len), next(len >> 1), level(3) {
    __builtin_amdgcn_s_setprio(3);
  }
  __device__ __forceinline__ void tile() {
    if (left <= next) {
      next >>= 1;
      --level;
      if (level == 2) __builtin_amdgcn_s_setprio(2);
      else if (level == 1) __builtin_amdgcn_s_setprio(1);
      else __builtin_amdgcn_s_setprio(0);
    }
    left -= kSeqTile;
  }
};

// The wave's share of a launch: workgroups of four waves, numbered over
// (slot, block of 64 channels) with the channel blocks innermost.
struct WavePos {
  int32_t cb, slot;
};
__device__ __forceinline__ WavePos wave_pos(uint32_t ncb) {
  const uint32_t w = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  return {static_cast<int32_t>(w % ncb), static_cast<int32_t>(w / ncb)};
}

// A kernel's one argument, read again where it is used: what only the end of a
// chunk needs would otherwise hold scalar registers through the main loop.
template <typename Args>
__device__ __forceinline__ const __attribute__((address_space(4))) Args& late_args() {
  uint64_t at = (uint64_t)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(at));
  return *(const __attribute__((address_space(4))) Args*)at;
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
template <typename T, typename DT, typename BT>
struct FwdArgs {
  SeqScanGeom g;
  FwdPtrs p;
  BcRows<BT> bc;
  uint32_t ncb;
  const T* u;
  const DT* delta;
  const T* z;
  T* y;
};

// AGG: the end state of each chunk but a sequence's last from a zero state,
// and the sum of delta over it.  Otherwise the main pass.
template <typename T, typename DT, typename BT, bool AGG>
__global__ void __launch_bounds__(256, AGG ? 5 : 4)
seq_scan_fwd_kernel(FwdArgs<T, DT, BT> args) {
  const SeqScanGeom& g = args.g;
  const FwdPtrs& p = args.p;
  const BcRows<BT>& bc = args.bc;
  const uint32_t lane = threadIdx.x & 63;
  const WavePos pos = wave_pos(args.ncb);
  const SeqChunk c = seq_chunk(g.q, pos.slot, g.cut, lane);
  const int64_t D = g.q.D, d0 = static_cast<int64_t>(pos.cb) * kWave, d = d0 + lane;
  // (lanes past the last channel take no further part: nothing below crosses lanes)
  if (c.t0 < 0 || d >= D) return;
  if (c.seq == g.q.S) {  // rows of no sequence
    if constexpr (!AGG)
      for (int32_t t = c.t0; t < c.t1; ++t) args.y[t * g.ys + d] = from_f32<T>(0.f);
    return;
  }
  if (AGG && c.t1 == c.end) return;
  float a2[16], h[16];
  load_a2(a2, p.A, d * g.N, 0, g.N, g.a_log);
  const int32_t row = seq_slot(g.q, c.seq);
  if (AGG) {
#pragma unroll
    for (int n = 0; n < 16; ++n) h[n] = 0.f;
  } else if (g.multi) {
    const float* at = p.agg_h + (static_cast<int64_t>(c.slot) * 4 * D + d) * 4;
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
      if (any) load_state4(v, p.h0, row, D, d, q, g.N, true);
#pragma unroll
      for (int j = 0; j < 4; ++j) h[4 * q + j] = v[j];
    }
  }
  const float bias = p.dbias ? p.dbias[d] : 0.f;
  const float Dd = AGG ? 0.f : p.Dv[d];
  const bool soft = g.softplus != 0, gate = !AGG && args.z != nullptr;
  RowPtr pu, pd, pz, py, pb, pc;
  pu.set(args.u + d0, c.t0, g.us);
  pd.set(args.delta + d0, c.t0, g.ds);
  if (gate) pz.set(args.z + d0, c.t0, g.zs);
  py.set(args.y + d0, c.t0, g.ys);
  pb.set(bc.B, c.t0, bc.st);
  pc.set(bc.C, c.t0, bc.st);
  float sum_dl = 0.f;
  T nu[kSeqTile], nz[kSeqTile];
  DT nd[kSeqTile];
  auto fetch = [&](int32_t t) {
    load_next(nu, pu, t, c.t1, lane);
    load_next(nd, pd, t, c.t1, lane);
    if (gate) load_next(nz, pz, t, c.t1, lane);
  };
  if (c.t0 < c.t1) fetch(c.t0);
  Pace pace(c.t1 - c.t0);
  for (int32_t t = c.t0; t < c.t1; t += kSeqTile) {
    pace.tile();
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
    if (t + kSeqTile > c.t1) {  // positions past the chunk: nothing decays or enters
#pragma unroll
      for (int i = 0; i < kSeqTile; ++i) dl[i] = t + i < c.t1 ? dl[i] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < kSeqTile; ++i) du[i] = dl[i] * uf[i];
    if (!AGG && p.ckpt != nullptr) {
      const int64_t ck = (c.start >> kSeqTileShift) + c.seq + ((t - c.start) >> kSeqTileShift);
      float* at = p.ckpt + (ck * 4 * D + d) * 4;
#pragma unroll
      for (int q = 0; q < 4; ++q)
        store_pack(at + q * 4 * D, Pack<float, 4>{h[4 * q], h[4 * q + 1], h[4 * q + 2], h[4 * q + 3]});
    }
    float out[kSeqTile];
#pragma unroll
    for (int i = 0; i < kSeqTile; ++i) {
      // B and C are on their way while the decays are formed
      float a[16];
      typename BcRows<BT>::template Raw<16> Bv, Cv;
      Bv.load(pb.at);
      pb.next(t + i + 1 < c.t1);
      if constexpr (!AGG) {
        Cv.load(pc.at);
        pc.next(t + i + 1 < c.t1);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < 16; ++n) a[n] = fast_exp2(dl[i] * a2[n]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < 16; ++n) h[n] = fmaf(a[n], h[n], du[i] * Bv[n]);
      if constexpr (AGG) {
        sum_dl += dl[i];
      } else {
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int n = 0; n < 16; ++n) acc[n & 3] = fmaf(h[n], Cv[n], acc[n & 3]);
        const float r = fmaf(Dd, uf[i], (acc[0] + acc[1]) + (acc[2] + acc[3]));
        out[i] = r * gz[i];
      }
    }
    if constexpr (!AGG) {
      store_next<T>(py, c.t1 - t, lane, out);
    }
  }
  const auto& late = late_args<FwdArgs<T, DT, BT>>();
  if constexpr (AGG) {
    float* at = late.p.agg_h + (static_cast<int64_t>(c.slot) * 4 * D + d) * 4;
#pragma unroll
    for (int q = 0; q < 4; ++q)
      store_pack(at + q * 4 * D, Pack<float, 4>{h[4 * q], h[4 * q + 1], h[4 * q + 2], h[4 * q + 3]});
    late.p.agg_s[c.slot * D + d] = sum_dl;
  } else if (c.t1 == c.end && late.p.h1 != nullptr && row >= 0) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float v[4] = {h[4 * q], h[4 * q + 1], h[4 * q + 2], h[4 * q + 3]};
      store_state4(v, late.p.h1, row, D, d, q, late.g.N, true);
    }
  }
}

// Carries over the chunks of one sequence, in order (REV: from its end): the
// aggregates are replaced by what enters each chunk.  A wave is 16 channels
// (lane & 15) x 4 groups of states and takes kCarryRun consecutive chunks in
// registers, one round of loads; the waves' own aggregates are joined through
// LDS, and the workgroup goes on with the next kCarryRun * (its waves) chunks.
template <bool REV>
__global__ void __launch_bounds__(1024)
seq_carry_kernel(SeqScanGeom g, uint32_t ncb, const float* __restrict__ A, const float* __restrict__ enter,
                 float* __restrict__ agg_h, const float* __restrict__ agg_s) {
  __shared__ Pack<float, 4> sE[16][64];
  __shared__ float sS[16][64];
  const int lane = threadIdx.x & 63, q = lane >> 4;
  const int32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6;
  const BlockPos pos = block_pos(ncb);
  const int32_t seq = pos.slot;
  const int64_t D = g.q.D, d = static_cast<int64_t>(pos.cb) * 16 + (lane & 15);
  const int64_t dc = d < D ? d : D - 1;
  const int32_t start = seq_off_u(g.q, seq), next = seq_off_u(g.q, seq + 1);
  const int32_t len = next > start ? next - start : 0;
  const int32_t n = cut_div(g.cut, len) + (cut_div(g.cut, len) * static_cast<int64_t>(g.cut.len) < len ? 1 : 0);
  const int32_t row = seq_slot(g.q, seq);
  float a2[4], h[4] = {0.f, 0.f, 0.f, 0.f};
  load_a2(a2, A, dc * g.N, 4 * q, g.N, g.a_log);
  if (enter != nullptr && row >= 0 && !seq_fresh(g.q, seq)) load_state4(h, enter, row, D, dc, q, g.N, true);
  const int64_t base = static_cast<int64_t>(cut_div(g.cut, start)) + seq;
  auto slot_of = [&](int32_t j) { return base + (REV ? n - 1 - j : j); };  // j-th chunk in the carry's order
  auto put = [&](int64_t slot) {
    if (d < D) store_pack(agg_h + ((slot * 4 + q) * D + d) * 4, Pack<float, 4>{h[0], h[1], h[2], h[3]});
  };
  if (n == 0) {  // an empty sequence's one chunk
    if (wave == 0) put(base);
    return;
  }
  for (int32_t j0 = 0; j0 < n; j0 += nw * kCarryRun) {
    const int32_t j = j0 + wave * kCarryRun;
    Pack<float, 4> v[kCarryRun];
    float s[kCarryRun];
#pragma unroll
    for (int i = 0; i < kCarryRun; ++i) {
      // (the last chunk in order has no aggregate, and nothing follows it)
      const int64_t slot = slot_of(j + i < n ? j + i : n - 1);
      v[i] = load_pack<float, 4>(agg_h + ((slot * 4 + q) * D + dc) * 4);
      s[i] = agg_s[slot * D + dc];
    }
    float e[4] = {0.f, 0.f, 0.f, 0.f}, sum = 0.f;
#pragma unroll
    for (int i = 0; i < kCarryRun; ++i) {
      if (j + i < n - 1) {
#pragma unroll
        for (int k = 0; k < 4; ++k) e[k] = fmaf(fast_exp2(a2[k] * s[i]), e[k], v[i].v[k]);
        sum += s[i];
      }
    }
    if (nw > 1) {
      if (j0 > 0) __syncthreads();
      sE[wave][lane] = Pack<float, 4>{e[0], e[1], e[2], e[3]};
      sS[wave][lane] = sum;
      __syncthreads();
      // every wave folds the runs before its own; the rest after its stores
      for (int32_t w = 0; w < wave; ++w) {
        const Pack<float, 4> x = sE[w][lane];
        const float sw = sS[w][lane];
#pragma unroll
        for (int k = 0; k < 4; ++k) h[k] = fmaf(fast_exp2(a2[k] * sw), h[k], x.v[k]);
      }
    }
    float after[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) after[k] = fmaf(fast_exp2(a2[k] * sum), h[k], e[k]);
#pragma unroll
    for (int i = 0; i < kCarryRun; ++i) {
      if (j + i < n) {
        put(slot_of(j + i));
#pragma unroll
        for (int k = 0; k < 4; ++k) h[k] = fmaf(fast_exp2(a2[k] * s[i]), h[k], v[i].v[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) h[k] = after[k];
    for (int32_t w = wave + 1; w < nw; ++w) {
      const Pack<float, 4> x = sE[w][lane];
      const float sw = sS[w][lane];
#pragma unroll
      for (int k = 0; k < 4; ++k) h[k] = fmaf(fast_exp2(a2[k] * sw), h[k], x.v[k]);
    }
  }
}

// Float32 copies of B | C in rows of 32, zero past N.
template <typename T>
__global__ void __launch_bounds__(256)
seq_bc_kernel(int32_t T_, int32_t N, int64_t st, const T* __restrict__ Bm, const T* __restrict__ Cm,
              float* __restrict__ out) {
  const int n = threadIdx.x & 15;
  const T* src = (threadIdx.x & 16) ? Cm : Bm;
  const int64_t total = static_cast<int64_t>(T_) * 32, step = static_cast<int64_t>(gridDim.x) * 256;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total; i += step)
    out[i] = n < N ? to_f32(src[(i >> 5) * st + n]) : 0.f;
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
template <typename T, typename DT, typename BT>
struct BwdArgs {
  SeqScanGeom g;
  BwdPtrs p;
  BcRows<BT> bc;
  uint32_t ncb, nslots;
  const T* u;
  const DT* delta;
  const T* z;
  const T* dy;
  T* du;
  DT* ddelta;
  T* dz;
};

// The adjoint that leaves each chunk but a sequence's first to its front, from
// zero, and the sum of delta.
template <typename T, typename DT, typename BT>
__global__ void __launch_bounds__(256, 4)
seq_scan_bwd_agg_kernel(BwdArgs<T, DT, BT> args) {
  const SeqScanGeom& g = args.g;
  const BwdPtrs& p = args.p;
  const BcRows<BT>& bc = args.bc;
  const uint32_t lane = threadIdx.x & 63;
  const WavePos pos = wave_pos(args.ncb);
  const SeqChunk c = seq_chunk(g.q, pos.slot, g.cut, lane);
  const int64_t D = g.q.D, d0 = static_cast<int64_t>(pos.cb) * kWave, d = d0 + lane;
  if (c.t0 <= c.start || c.seq == g.q.S || d >= D) return;
  float a2[16], h[16];
  load_a2(a2, p.A, d * g.N, 0, g.N, g.a_log);
#pragma unroll
  for (int n = 0; n < 16; ++n) h[n] = 0.f;
  const float bias = p.dbias ? p.dbias[d] : 0.f;
  const bool soft = g.softplus != 0, gate = args.z != nullptr;
  RowPtr py, pd, pz, pc;
  py.set(args.dy + d0, c.t1 - 1, g.ys);
  pd.set(args.delta + d0, c.t1 - 1, g.ds);
  if (gate) pz.set(args.z + d0, c.t1 - 1, g.zs);
  pc.set(bc.C, c.t1 - 1, bc.st);
  float sum_dl = 0.f;
  T ny[kSeqTile], nz[kSeqTile];
  DT nd[kSeqTile];
  auto fetch = [&](int32_t t) {
    load_prev(ny, py, t, c.t0, c.t1, lane);
    load_prev(nd, pd, t, c.t0, c.t1, lane);
    if (gate) load_prev(nz, pz, t, c.t0, c.t1, lane);
  };
  const int32_t last = c.t0 + ((c.t1 - 1 - c.t0) & ~(kSeqTile - 1));
  fetch(last);
  Pace pace(c.t1 - c.t0);
  for (int32_t t = last; t >= c.t0; t -= kSeqTile) {
    pace.tile();
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
    if (t + kSeqTile > c.t1) {  // positions past the chunk: nothing decays or enters
#pragma unroll
      for (int i = 0; i < kSeqTile; ++i) {
        dl[i] = t + i < c.t1 ? dl[i] : 0.f;
        dr[i] = t + i < c.t1 ? dr[i] : 0.f;
      }
    }
#pragma unroll
    for (int i = kSeqTile - 1; i >= 0; --i) {
      float a[16];
      typename BcRows<BT>::template Raw<16> Cv;
      Cv.load(pc.at);
      pc.prev(t + i < c.t1 && t + i > c.t0);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < 16; ++n) a[n] = fast_exp2(dl[i] * a2[n]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < 16; ++n) h[n] = a[n] * fmaf(Cv[n], dr[i], h[n]);
      sum_dl += dl[i];
    }
  }
  const auto& late = late_args<BwdArgs<T, DT, BT>>();
  float* at = late.p.agg_h + (static_cast<int64_t>(c.slot) * 4 * D + d) * 4;
#pragma unroll
  for (int q = 0; q < 4; ++q)
    store_pack(at + q * 4 * D, Pack<float, 4>{h[4 * q], h[4 * q + 1], h[4 * q + 2], h[4 * q + 3]});
  late.p.agg_s[c.slot * D + d] = sum_dl;
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
// All of a wave's LDS is its own: no barrier.
struct BwdLds {
  Pack<float, 4> a2[4][kWave], c[4][kWave], da[4][kWave];
  float bc[16][17];  // [token | 8 for dC][state]
};

template <typename T, typename DT, typename BT>
__global__ void __launch_bounds__(256, 3)
seq_scan_bwd_kernel(BwdArgs<T, DT, BT> args) {
  __shared__ BwdLds lds[4];
  const SeqScanGeom& g = args.g;
  const BwdPtrs& p = args.p;
  const BcRows<BT>& bc = args.bc;
  const uint32_t lane = threadIdx.x & 63;
  const WavePos pos = wave_pos(args.ncb);
  if (static_cast<uint32_t>(pos.slot) >= args.nslots) return;
  BwdLds& s = lds[__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)];
  const SeqChunk c = seq_chunk(g.q, pos.slot, g.cut, lane);
  const int64_t D = g.q.D, d0 = static_cast<int64_t>(pos.cb) * kWave, d = d0 + lane;
  const bool valid = d < D;
  // (lanes past the last channel read the last one, and add zeros)
  const uint32_t lc = valid ? lane : static_cast<uint32_t>(D - 1 - d0);
  const int64_t dc = d0 + lc;
  if (c.t0 < 0 || c.seq == g.q.S) {
    if (valid)
      for (int i = 0; i < 18; ++i) p.part[(static_cast<int64_t>(pos.slot) * 18 + i) * D + d] = 0.f;
    for (int32_t t = c.t0; t < c.t1; ++t) {  // (c.t1 == c.t0 without a chunk)
      if (valid) {
        args.du[t * D + d] = from_f32<T>(0.f);
        args.ddelta[t * D + d] = from_f32<DT>(0.f);
        if (args.dz) args.dz[t * D + d] = from_f32<T>(0.f);
      }
      if (lane < 32) p.part_bc[(static_cast<int64_t>(pos.cb) * g.q.T + t) * 32 + lane] = 0.f;
    }
    return;
  }
  const int32_t row = seq_slot(g.q, c.seq);
  float a2[16];
  load_a2(a2, p.A, dc * g.N, 0, g.N, g.a_log);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    float h[4] = {0.f, 0.f, 0.f, 0.f};
    if (g.multi) {
      const Pack<float, 4> v = load_pack<float, 4>(p.agg_h + ((static_cast<int64_t>(c.slot) * 4 + q) * D + dc) * 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) h[j] = v.v[j];
    } else if (p.dh1 != nullptr) {
      load_state4(h, p.dh1, row, D, dc, q, g.N, true);
    }
    if (!valid) {
#pragma unroll
      for (int j = 0; j < 4; ++j) h[j] = 0.f;
    }
    s.a2[q][lane] = Pack<float, 4>{a2[4 * q], a2[4 * q + 1], a2[4 * q + 2], a2[4 * q + 3]};
    s.c[q][lane] = Pack<float, 4>{h[0], h[1], h[2], h[3]};
    s.da[q][lane] = Pack<float, 4>{0.f, 0.f, 0.f, 0.f};
  }
  const float bias = p.dbias ? p.dbias[dc] : 0.f;
  const float Dd = p.Dv[dc];
  const bool soft = g.softplus != 0, gate = args.z != nullptr, all_valid = d0 + kWave <= D;
  RowPtr pu, pd, py, pz;
  pu.set(args.u + d0, c.t1 - 1, g.us);
  pd.set(args.delta + d0, c.t1 - 1, g.ds);
  py.set(args.dy + d0, c.t1 - 1, g.ys);
  if (gate) pz.set(args.z + d0, c.t1 - 1, g.zs);
  float dD = 0.f, ddb = 0.f;
  T nu[kSeqTile], ny[kSeqTile], nz[kSeqTile];
  DT nd[kSeqTile];
  auto fetch = [&](int32_t t) {
    load_prev(nu, pu, t, c.t0, c.t1, lc);
    load_prev(nd, pd, t, c.t0, c.t1, lc);
    load_prev(ny, py, t, c.t0, c.t1, lc);
    if (gate) load_prev(nz, pz, t, c.t0, c.t1, lc);
  };
  const int64_t ck0 = (c.start >> kSeqTileShift) + c.seq;
  const int32_t last = c.t0 + ((c.t1 - 1 - c.t0) & ~(kSeqTile - 1));
  Pace pace(c.t1 - c.t0);
  for (int32_t t = last; c.t0 < c.t1 && t >= c.t0; t -= kSeqTile) {
    pace.tile();
    float dl[kSeqTile], du[kSeqTile], dr[kSeqTile], qs[kSeqTile], ws[kSeqTile], rs[kSeqTile];
    float us[kSeqTile], sg[kSeqTile], gz[kSeqTile];  // for the outputs
    fetch(t);
#pragma unroll
    for (int i = 0; i < kSeqTile; ++i) {
      us[i] = to_f32(nu[i]);
      dl[i] = to_f32(nd[i]) + bias;
      dr[i] = to_f32(ny[i]);
      sg[i] = 1.f;
      gz[i] = qs[i] = ws[i] = 0.f;
    }
    if (soft) {
#pragma unroll
      for (int i = 0; i < kSeqTile; ++i) softplus_sigmoid(dl[i], dl[i], sg[i]);
    }
    if (gate) {
#pragma unroll
      for (int i = 0; i < kSeqTile; ++i) {
        const float zf = to_f32(nz[i]), sz = sigmoid_f(zf), ys = dr[i] * sz;
        dr[i] = ys * zf;
        gz[i] = ys * fmaf(zf, 1.f - sz, 1.f);  // dy times the derivative of silu(z)
      }
    }
    if (t + kSeqTile > c.t1 || !all_valid) {
      // positions past the chunk, channels that do not exist: nothing decays,
      // enters or leaves
#pragma unroll
      for (int i = 0; i < kSeqTile; ++i) {
        const bool in = valid && t + i < c.t1;
        dl[i] = in ? dl[i] : 0.f;
        us[i] = in ? us[i] : 0.f;
        dr[i] = in ? dr[i] : 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < kSeqTile; ++i) {
      dD = fmaf(dr[i], us[i], dD);
      rs[i] = Dd * us[i];
      du[i] = dl[i] * us[i];
    }
    const float* ck = p.ckpt + ((ck0 + ((t - c.start) >> kSeqTileShift)) * 4 * D + dc) * 4;
    Pack<float, 4> hs = load_pack<float, 4>(ck);
#pragma unroll 1
    for (int q = 0; q < 4; ++q) {
      const Pack<float, 4> a2 = s.a2[q][lane];
      Pack<float, 4> cs = s.c[q][lane], da = s.da[q][lane], h4 = hs;
      if (q < 3) hs = load_pack<float, 4>(ck + (q + 1) * 4 * D);
      typename BcRows<BT>::template Raw<2> Bv[kSeqTile], Cv[kSeqTile];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        __builtin_amdgcn_sched_barrier(0);
        if (j % 2 == 0) {  // two states at a time: what the scalar registers hold
          RowPtr pb, pc;
          pb.set(bc.B + 4 * q + j, t, bc.st);
          pc.set(bc.C + 4 * q + j, t, bc.st);
#pragma unroll
          for (int i = 0; i < kSeqTile; ++i) {
            Bv[i].load(pb.at);
            Cv[i].load(pc.at);
            pb.next(t + i + 1 < c.t1);
            pc.next(t + i + 1 < c.t1);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        float h = h4.v[j];
        float a[kSeqTile], ah[kSeqTile], v[16];  // v: the terms of dB of the 8 tokens, then those of dC
#pragma unroll
        for (int i = 0; i < kSeqTile; ++i) {
          a[i] = fast_exp2(dl[i] * a2.v[j]);
          ah[i] = a[i] * h;
          h = fmaf(du[i], Bv[i][j & 1], ah[i]);
          rs[i] = fmaf(h, Cv[i][j & 1], rs[i]);
          v[8 + i] = dr[i] * h;
        }
#pragma unroll
        for (int i = kSeqTile - 1; i >= 0; --i) {
          const float dh = fmaf(Cv[i][j & 1], dr[i], cs.v[j]);
          qs[i] = fmaf(dh, Bv[i][j & 1], qs[i]);
          v[i] = dh * du[i];
          const float w = dh * ah[i];
          da.v[j] = fmaf(w, dl[i], da.v[j]);
          ws[i] = fmaf(w, a2.v[j], ws[i]);
          cs.v[j] = dh * a[i];
        }
        s.bc[lane >> 2][4 * q + j] = wave_sums16(v, lane);  // (four lanes, one value)
      }
      s.c[q][lane] = cs;
      s.da[q][lane] = da;
    }
    const auto& late = late_args<BwdArgs<T, DT, BT>>();
    __builtin_amdgcn_wave_barrier();
    // rows t .. t + 7 of 32 values: dB at 0, dC at 16
    float* out = late.p.part_bc + (static_cast<int64_t>(pos.cb) * g.q.T + t) * 32;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = k * 2 + (lane >> 5), n = lane & 31;
      const float v = s.bc[i + ((n >> 4) << 3)][n & 15];
      if (t + i < c.t1) out[i * 32 + n] = v;
    }
    __builtin_amdgcn_wave_barrier();
    const int32_t rows = c.t1 - t < kSeqTile ? c.t1 - t : kSeqTile;
#pragma unroll
    for (int i = 0; i < kSeqTile; ++i) {
      const float dd = fmaf(ws[i], kLn2, qs[i] * us[i]) * sg[i];
      ddb += i < rows ? dd : 0.f;
      ws[i] = dd;
      qs[i] = fmaf(qs[i], dl[i], Dd * dr[i]);
      rs[i] *= gz[i];
    }
    if (valid) {
      RowPtr o;
      o.set(late.du + d0, t, D);
      store_next<T>(o, rows, lane, qs);
      o.set(late.ddelta + d0, t, D);
      store_next<DT>(o, rows, lane, ws);
      if (gate) {
        o.set(late.dz + d0, t, D);
        store_next<T>(o, rows, lane, rs);
      }
    }
  }
  if (!valid) return;
  const auto& late = late_args<BwdArgs<T, DT, BT>>();
  float* part = late.p.part + static_cast<int64_t>(c.slot) * 18 * D + d;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const Pack<float, 4> da = s.da[q][lane], cs = s.c[q][lane];
#pragma unroll
    for (int j = 0; j < 4; ++j) part[(4 * q + j) * D] = da.v[j];
    if (c.t0 == c.start && late.p.dh0 != nullptr) store_state4(cs.v, late.p.dh0, row, D, d, q, late.g.N, true);
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
  const int64_t total = static_cast<int64_t>(rows) * 32, step = static_cast<int64_t>(gridDim.x) * 256;
  const int n = threadIdx.x & 15;
  T* out = (threadIdx.x & 16) ? dC : dB;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total; i += step) {
    float s = 0.f;
    for (int32_t k0 = 0; k0 < ncb; k0 += 8) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = part[(k0 + k < ncb ? k0 + k : 0) * total + i];
#pragma unroll
      for (int k = 0; k < 8; ++k) s += k0 + k < ncb ? v[k] : 0.f;
    }
    if (n < N) out[(i >> 5) * N + n] = from_f32<T>(s);
  }
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
  load_a2(a2, A, dc * N, 4 * q, N, g.a_log);
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
dim3 wave_grid(int64_t slots, uint32_t ncb) { return dim3(static_cast<unsigned>((slots * ncb + 3) / 4)); }
// workgroups of 256 over n elements that a kernel walks in steps of the grid
dim3 strided_grid(int64_t n) { return dim3(static_cast<unsigned>(std::min<int64_t>((n + 255) / 256, 1 << 20))); }

template <bool REV>
hipError_t carry(const SeqScanGeom& g, const float* A, const float* enter, float* agg_h, const float* agg_s,
                 hipStream_t s) {
  if (g.q.S == 0) return hipSuccess;
  const uint32_t ncb = static_cast<uint32_t>((g.q.D + 15) / 16);
  hipLaunchKernelGGL(seq_carry_kernel<REV>, dim3(ncb * static_cast<unsigned>(g.q.S)),
                     dim3(64 * carry_waves(g)), 0, s, g, ncb, A, enter, agg_h, agg_s);
  return hipGetLastError();
}

template <typename T>
hipError_t copy_bc(const SeqScanGeom& g, const SeqScanIn& in, float* out, hipStream_t s) {
  const int64_t n = static_cast<int64_t>(g.q.T) * 32;
  if (n == 0) return hipSuccess;
  hipLaunchKernelGGL(seq_bc_kernel<T>, strided_grid(n), dim3(256), 0, s, g.q.T, g.N, g.bs,
                     static_cast<const T*>(in.Bm), static_cast<const T*>(in.Cm), out);
  return hipGetLastError();
}

template <typename T, typename DT, typename BT>
hipError_t fwd_t(const SeqScanGeom& g, const SeqScanIn& in, const SeqScanFwd& b, BcRows<BT> bc, hipStream_t s) {
  const uint32_t ncb = blocks_of(g.q.D);
  const dim3 grid = wave_grid(chunk_slots(g.q, g.cut), ncb);
  const FwdArgs<T, DT, BT> args{g, {in.dbias, in.A, in.Dv, b.h0, b.h1, b.ckpt, b.agg_h, b.agg_s}, bc, ncb,
                                static_cast<const T*>(in.u), static_cast<const DT*>(in.delta),
                                static_cast<const T*>(in.z), static_cast<T*>(b.y)};
  if (g.multi) {
    hipLaunchKernelGGL((seq_scan_fwd_kernel<T, DT, BT, true>), grid, dim3(256), 0, s, args);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || (e = carry<false>(g, in.A, b.h0, b.agg_h, b.agg_s, s)) != hipSuccess) return e;
  }
  hipLaunchKernelGGL((seq_scan_fwd_kernel<T, DT, BT, false>), grid, dim3(256), 0, s, args);
  return hipGetLastError();
}

template <typename T, typename DT, typename BT>
hipError_t bwd_t(const SeqScanGeom& g, const SeqScanIn& in, const SeqScanBwd& b, BcRows<BT> bc, hipStream_t s) {
  const uint32_t ncb = blocks_of(g.q.D);
  const int64_t slots = chunk_slots(g.q, g.cut);
  const dim3 grid = wave_grid(slots, ncb);
  const BwdArgs<T, DT, BT> args{g, {in.dbias, in.A, in.Dv, b.dh1, b.dh0, b.ckpt, b.agg_h, b.agg_s, b.part, b.part_bc},
                                bc, ncb, static_cast<uint32_t>(slots), static_cast<const T*>(in.u),
                                static_cast<const DT*>(in.delta), static_cast<const T*>(in.z),
                                static_cast<const T*>(b.dy), static_cast<T*>(b.du), static_cast<DT*>(b.ddelta),
                                static_cast<T*>(b.dz)};
  hipError_t e;
  if (g.multi) {
    hipLaunchKernelGGL((seq_scan_bwd_agg_kernel<T, DT, BT>), grid, dim3(256), 0, s, args);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    if ((e = carry<true>(g, in.A, b.dh1, b.agg_h, b.agg_s, s)) != hipSuccess) return e;
  }
  hipLaunchKernelGGL((seq_scan_bwd_kernel<T, DT, BT>), grid, dim3(256), 0, s, args);
  if ((e = hipGetLastError()) != hipSuccess) return e;
  hipLaunchKernelGGL(seq_reduce_params_kernel, dim3(static_cast<unsigned>((18 * g.q.D + 63) / 64)), dim3(1024), 0, s,
                     g.q.D, g.N, slots, g.a_log, in.A, b.part, b.dA, b.dD, b.ddbias);
  if ((e = hipGetLastError()) != hipSuccess) return e;
  const int64_t n = static_cast<int64_t>(g.q.T) * 32;
  if (n == 0) return hipSuccess;
  hipLaunchKernelGGL(seq_reduce_bc_kernel<T>, strided_grid(n), dim3(256), 0, s, g.q.T,
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
