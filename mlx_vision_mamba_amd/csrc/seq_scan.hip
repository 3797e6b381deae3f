// Selective scan of packed sequences with states, forward and one token, for
// gfx950.
//
//   h_t[n] = exp(delta_t A[n]) h_{t-1}[n] + delta_t u_t B_t[n]
//   y_t    = (sum_n C_t[n] h_t[n] + D u_t) * z_t sigmoid(z_t)
//
// A lane holds one channel with its states in registers, a wave 64
// channels of one chunk of one sequence.  Everything that belongs to a
// (token, channel), the softplus and the gate among it, is computed once, and
// the sum over the states needs no other lane.  Each (token, channel, state)
// is then two multiplications, an exponential and two fused multiply-adds.
//
// Long sequences are cut into chunks: a first pass runs each chunk from a
// zero state for its end state, those are joined in order (the decay over a
// chunk is one exponential of the summed delta), the main pass runs each chunk
// from its carry.
//
// Bound by VALU issue.  On MI355X, 32768 bf16 tokens of 1536 channels with gate
// and softplus: aggregate pass 123 us, carry 16, main pass 171, the VALU busy
// 97 % of both passes (85 and 116 instructions a token and wave; 80 of
// the main pass's are the recurrence, the 16 exponentials among them count
// twice).  Four waves a SIMD; what kept it from that rate were row addresses
// held (and spilled) for whole tiles, and the issue order (Pace).
//
// B and C are the same for a whole wave and come through scalar loads, as
// scalar operands.  Through LDS instead (a tile at a time) both passes took
// 5 % longer.
#include "seq_scan_pass.h"

namespace mvm {

namespace {

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
  float zeros[kZeroRow];
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
// and the sum of delta over it.  Otherwise the main pass.  NS: the states that a
// lane holds, 8 where there are no more (16384 bf16 tokens of 1536 channels, 8
// states: 138 us, 178 by 16).
template <typename T, typename DT, typename BT, bool AGG, int NS>
__global__ void __launch_bounds__(256, 4)
seq_scan_fwd_kernel(FwdArgs<T, DT, BT> args) {
  const SeqScanGeom& g = args.g;
  const FwdPtrs& p = args.p;
  const uint32_t lane = threadIdx.x & 63;
  const WavePos pos = wave_pos(args.ncb);
  const SeqChunk c = seq_chunk(g.q, pos.slot, g.cut, lane);
  const int64_t D = g.q.D, d0 = static_cast<int64_t>(pos.cb) * kWave;
  if (c.t0 < 0) return;
  // (lanes past the last channel compute the last one's values, and store none)
  const bool valid = d0 + lane < D;
  const uint32_t lc = valid ? lane : static_cast<uint32_t>(D - 1 - d0);
  const int64_t d = d0 + lc;
  if (c.seq == g.q.S) {  // rows of no sequence
    if (!AGG && valid)
      for (int32_t t = c.t0; t < c.t1; ++t) args.y[t * g.ys + d] = from_f32<T>(0.f);
    return;
  }
  if (AGG && c.t1 == c.end) {
    // Where the main pass folds the chunks, the place of the last one's
    // aggregate takes the state that the sequence starts from: its own row may
    // hold the final state before each chunk of the main pass has read it.
    if (g.fold && valid) {
      const int32_t row = seq_slot(g.q, c.seq);
      float h[NS];
#pragma unroll
      for (int n = 0; n < NS; ++n) h[n] = 0.f;
      if (p.h0 != nullptr && row >= 0 && !seq_fresh(g.q, c.seq)) load_states(h, p.h0, row * D + d, 0, g.N, g.h_vec);
      store_agg(h, p.agg_h, c.slot, D, d);
    }
    return;
  }
  const bool soft = g.softplus != 0, gate = !AGG && args.z != nullptr;
  // Everything that a chunk starts from is asked for before any of it is used
  RowPtr pu, pd, pz, py, pb, pc;
  pu.set(args.u + d0, c.t0, g.us);
  pd.set(args.delta + d0, c.t0, g.ds);
  if (gate) pz.set(args.z + d0, c.t0, g.zs);
  py.set(args.y + d0, c.t0, g.ys);
  pb.set(args.bc.B, c.t0, args.bc.st);
  pc.set(args.bc.C, c.t0, args.bc.st);
  T nu[kSeqTile], nz[kSeqTile];
  DT nd[kSeqTile];
  auto fetch = [&](int32_t t) {
    load_next(nd, pd, t, c.t1, lc);
    load_next(nu, pu, t, c.t1, lc);
    if (gate) load_next(nz, pz, t, c.t1, lc);
  };
  StateRows<1> rows;
  if constexpr (!AGG) rows.load(g.q, c.seq, p.A);
  if (c.t0 < c.t1) fetch(c.t0);
  const float bias = p.dbias ? p.dbias[d] : 0.f;
  const float Dd = AGG ? 0.f : p.Dv[d];
  float a2[NS], h[NS];
#pragma unroll
  for (int n = 0; n < NS; ++n) h[n] = 0.f;
  if constexpr (!AGG) {
    if (g.multi)
      load_agg(h, p.agg_h, g.fold ? last_slot(g.cut, c) : c.slot, D, d);
    else if (p.h0 != nullptr && rows.row[0] >= 0)
      load_states(h, p.h0, rows.row[0] * D + d, 0, g.N, g.h_vec);
  }
  load_a2(a2, p.A, d, 0, g);
  if constexpr (!AGG) {
    rows.settle(g.q);
    if (!g.multi) {
#pragma unroll
      for (int n = 0; n < NS; ++n) h[n] = rows.fresh[0] != 0 ? 0.f : h[n];
    }
  }
  if constexpr (!AGG) {
    if (g.multi && g.fold) {
      const int64_t first = cut_div(g.cut, c.start) + c.seq;
      fold_chunks<1>(h, a2, p.agg_h, p.agg_s, first, static_cast<int32_t>(c.slot - first), D, d);
    }
  }
  float sum_dl = 0.f;
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
      for (int i = 0; i < kSeqTile; ++i) {
        dl[i] = t + i < c.t1 ? dl[i] : 0.f;
        uf[i] = t + i < c.t1 ? uf[i] : 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < kSeqTile; ++i) du[i] = dl[i] * uf[i];
    if (!AGG && p.ckpt != nullptr && valid)
      store_agg(h, p.ckpt, (c.start >> kSeqTileShift) + c.seq + ((t - c.start) >> kSeqTileShift), D, d);
    float out[kSeqTile];
    const int32_t left = c.t1 - t;
#pragma unroll
    for (int i = 0; i < kSeqTile; ++i) {
      // B and C are on their way while the decays are formed
      float a[NS];
      typename BcRows<BT>::template Raw<NS> Bv, Cv;
      Bv.load(pb.at);
      if constexpr (!AGG) Cv.load(pc.at);
      if constexpr (AGG) {  // (whole tiles only)
        pb.next(i + 1 < left);
      } else {
        pb.next_or(i + 1 < left, zero_row());
        pc.next(i + 1 < left);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < NS; ++n) a[n] = fast_exp2(dl[i] * a2[n]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < NS; ++n) h[n] = fmaf(a[n], h[n], du[i] * Bv[n]);
      if constexpr (AGG) {
        sum_dl += dl[i];
      } else {
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int n = 0; n < NS; ++n) acc[n & 3] = fmaf(h[n], Cv[n], acc[n & 3]);
        out[i] = fmaf(Dd, uf[i], (acc[0] + acc[1]) + (acc[2] + acc[3])) * gz[i];
        pin(out[i]);
      }
    }
    if constexpr (!AGG) {
      if (valid) store_next<T>(py, c.t1 - t, lane, out);
      py.at += static_cast<uint64_t>(kSeqTile) * py.st;
    }
  }
  if (!valid) return;
  const auto& late = late_args<FwdArgs<T, DT, BT>>();
  if constexpr (AGG) {
    store_agg(h, late.p.agg_h, c.slot, D, d);
    late.p.agg_s[c.slot * D + d] = sum_dl;
  } else if (c.t1 == c.end && late.p.h1 != nullptr && rows.row[0] >= 0) {
    store_states(h, late.p.h1, rows.row[0] * D + d, 0, late.g.N, late.g.h_vec);
  }
}

// Carries over the chunks of one sequence, in order (REV: from its end): the
// aggregates are replaced by what enters each chunk.  A wave is 16 channels
// (lane & 15) x 4 groups of states and takes kCarryRun consecutive chunks in
// registers, one round of loads; the waves' own aggregates are joined through
// LDS, and the workgroup goes on with the next kCarryRun * (its waves) chunks.
// MI355X, 164 chunks of 1536 channels: 15-17 us (96 chunk after chunk).
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
  StateRows<1> rows;
  rows.load(g.q, seq, A);
  const int64_t base = static_cast<int64_t>(cut_div(g.cut, start)) + seq;
  // (groups of states that there are none of carry along what lies there)
  auto slot_of = [&](int32_t j) { return base + (REV ? n - 1 - j : j); };  // j-th chunk in the carry's order
  // (waves that no run falls to only meet the others at the barrier)
  const bool idle = wave > 0 && wave * kCarryRun >= n;
  Pack<float, 4> v[kCarryRun];
  float s[kCarryRun];
  auto fetch = [&](int32_t j) {
#pragma unroll
    for (int i = 0; i < kCarryRun; ++i) {
      // (the last chunk in order has no aggregate, and nothing follows it)
      const int64_t slot = slot_of(j + i < n ? j + i : n - 1);
      v[i] = load_pack<float, 4>(agg_h + ((slot * 4 + q) * D + dc) * 4);
      s[i] = agg_s[slot * D + dc];
    }
  };
  // The first round's aggregates, the initial state and A in flight together
  float a2[4] = {0.f, 0.f, 0.f, 0.f}, h[4] = {0.f, 0.f, 0.f, 0.f};
  if (!idle && n > 0) fetch(wave * kCarryRun);
  if (!idle && enter != nullptr && rows.row[0] >= 0) load_states(h, enter, rows.row[0] * D + dc, 4 * q, g.N, g.h_vec);
  if (!idle) load_a2(a2, A, dc, 4 * q, g);
  rows.settle(g.q);
#pragma unroll
  for (int k = 0; k < 4; ++k) h[k] = rows.fresh[0] != 0 ? 0.f : h[k];
  auto put = [&](int64_t slot) {
    if (d < D) store_pack(agg_h + ((slot * 4 + q) * D + d) * 4, Pack<float, 4>{h[0], h[1], h[2], h[3]});
  };
  if (n == 0) {  // an empty sequence's one chunk
    if (wave == 0) put(base);
    return;
  }
  for (int32_t j0 = 0; j0 < n; j0 += nw * kCarryRun) {
    if (idle) {  // (n fits the waves: this is the only round)
      __syncthreads();
      return;
    }
    const int32_t j = j0 + wave * kCarryRun;
    if (j0 > 0) fetch(j);
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
    for (int32_t w = wave + 1; w < nw && j0 + nw * kCarryRun < n; ++w) {
      const Pack<float, 4> x = sE[w][lane];
      const float sw = sS[w][lane];
#pragma unroll
      for (int k = 0; k < 4; ++k) h[k] = fmaf(fast_exp2(a2[k] * sw), h[k], x.v[k]);
    }
  }
}

// --------------------------------------------------------------- one token

// Lane G c + q holds states 4q .. 4q + 3 of channel c: a wave reads 64 / G
// channels' states, 1 KB, at once.  Bound by the states' traffic, as long as
// little else is asked for beside it: a wave keeps its channels' A, D and bias
// for R sequences, and has all their loads in flight together.  VEC: states,
// and B and C, are read four at a time (N a multiple of 4, aligned rows).
// MI355X, 1024 sequences of 1536 channels, bf16: 44.4 us, 4.8 TB/s (a large copy
// reaches 4.9); 5 us more while the gate's loads stood in branches, 10 more at one
// sequence a wave.  One or two lanes a channel for up to 4 or 8 states: 2048
// sequences 28 us (N 4) and 48 (N 8), against 50 and 65 by four lanes, some of
// them idle.  Single values (N 13): 85 us, 2.1 TB/s.
template <typename T, typename DT, bool VEC, int R, int G>
__global__ void __launch_bounds__(256)
seq_scan_step_kernel(SeqScanGeom g, uint32_t ncb, const T* __restrict__ u, const DT* __restrict__ delta,
                     const float* __restrict__ dbias, const float* __restrict__ A, const T* __restrict__ Bm,
                     const T* __restrict__ Cm, const float* __restrict__ Dv, const T* __restrict__ z,
                     float* __restrict__ states, T* __restrict__ y) {
  const BlockPos pos = block_pos(ncb);
  const int q = threadIdx.x & (G - 1), N = g.N;
  const int64_t D = g.q.D, d = static_cast<int64_t>(pos.cb) * (256 / G) + threadIdx.x / G;
  const bool valid = d < D, mine = valid && 4 * q < N;
  const int64_t dc = valid ? d : D - 1;
  const int n0 = 4 * q < N ? 4 * q : 0;
  const int32_t i0 = pos.slot * R;
  float* at[R];
  Pack<float, 4> h[R];
  Pack<T, 4> b[R], c[R];
  T uv[R], zv[R];
  DT dv[R];
  StateRows<R> rows;
  rows.load(g.q, i0, u);
  const int32_t(&row)[R] = rows.row;
  // (read without a gate too: a load in a branch would be waited for there)
  const T* zp = z ? z : u;
  const int64_t zs = z ? g.zs : g.us;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int32_t i = i0 + r < g.q.S ? i0 + r : g.q.S - 1;
    at[r] = states + (static_cast<int64_t>(row[r] < 0 ? 0 : row[r]) * D + dc) * N + n0;
    if (row[r] >= 0) {
      if constexpr (VEC) {
        h[r] = load_pack<float, 4>(at[r]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) h[r].v[j] = at[r][n0 + j < N ? j : 0];
      }
    }
    uv[r] = u[i * g.us + dc];
    dv[r] = delta[i * g.ds + dc];
    zv[r] = zp[i * zs + dc];
    if constexpr (VEC) {
      b[r] = load_pack<T, 4>(Bm + i * g.bs + n0);
      c[r] = load_pack<T, 4>(Cm + i * g.bs + n0);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = state_col(n0 + j, N);
        b[r].v[j] = Bm[i * g.bs + n];
        c[r].v[j] = Cm[i * g.bs + n];
      }
    }
  }
  const float bias = dbias ? dbias[dc] : 0.f, Dd = Dv[dc];
  float a2[4], zf[R];
  load_a2(a2, A, dc, 4 * q, g);
  rows.settle(g.q);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    zf[r] = to_f32(zv[r]);
    pin(zf[r]);
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (i0 + r >= g.q.S) break;
    T* yr = y + (i0 + r) * g.ys;
    if (row[r] < 0) {
      if (valid && q == 0) yr[d] = from_f32<T>(0.f);
      continue;
    }
    const bool fresh = rows.fresh[r] != 0;
    const float uf = to_f32(uv[r]);
    float dl = to_f32(dv[r]) + bias, sum = 0.f;
    if (g.softplus) dl = softplus_f(dl);
    const float du = dl * uf;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      h[r].v[j] = fmaf(fast_exp2(dl * a2[j]), fresh ? 0.f : h[r].v[j], du * to_f32(b[r].v[j]));
      sum = 4 * q + j < N ? fmaf(h[r].v[j], to_f32(c[r].v[j]), sum) : sum;
    }
    if (mine) {
      if constexpr (VEC) {
        store_pack(at[r], h[r]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (4 * q + j < N) at[r][j] = h[r].v[j];
      }
    }
    if constexpr (G > 1) sum += dpp<kQuadXor1>(sum);
    if constexpr (G > 2) sum += dpp<kQuadXor2>(sum);
    float out = fmaf(Dd, uf, sum);
    if (z) out *= zf[r] * sigmoid_f(zf[r]);
    if (valid && q == 0) yr[d] = from_f32<T>(out);
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

// ----------------------------------------------------------------- launches

template <typename T, typename DT, typename BT, int NS>
hipError_t fwd_n(SeqScanGeom g, const SeqScanIn& in, const SeqScanFwd& b, BcRows<BT> bc, hipStream_t s) {
  const uint32_t ncb = blocks_of(g.q.D);
  const dim3 grid = wave_grid(chunk_slots(g.q, g.cut), ncb);
  set_vec(g, in.A, b.h0, b.h1);
  const FwdArgs<T, DT, BT> args{{}, g, {in.dbias, in.A, in.Dv, b.h0, b.h1, b.ckpt, b.agg_h, b.agg_s}, bc, ncb,
                                static_cast<const T*>(in.u), static_cast<const DT*>(in.delta),
                                static_cast<const T*>(in.z), static_cast<T*>(b.y)};
  if (g.multi) {
    hipLaunchKernelGGL((seq_scan_fwd_kernel<T, DT, BT, true, NS>), grid, dim3(256), 0, s, args);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (!g.fold && (e = launch_carry<false>(g, in.A, b.h0, b.agg_h, b.agg_s, s)) != hipSuccess) return e;
  }
  hipLaunchKernelGGL((seq_scan_fwd_kernel<T, DT, BT, false, NS>), grid, dim3(256), 0, s, args);
  return hipGetLastError();
}

template <typename T, typename DT, typename BT>
hipError_t fwd_t(const SeqScanGeom& g, const SeqScanIn& in, const SeqScanFwd& b, BcRows<BT> bc, hipStream_t s) {
  if constexpr (std::is_same_v<BT, float>) {  // (B and C lie as they are only for 16 states)
    if (g.N <= 8) return fwd_n<T, DT, BT, 8>(g, in, b, bc, s);
  }
  return fwd_n<T, DT, BT, 16>(g, in, b, bc, s);
}

constexpr int kStepRows = 4;

template <typename T, typename DT>
hipError_t step_t(SeqScanGeom g, const SeqScanIn& in, float* states, void* y, hipStream_t s) {
  set_vec(g, in.A, states, nullptr);
  const bool bc = (reinterpret_cast<uintptr_t>(in.Bm) | reinterpret_cast<uintptr_t>(in.Cm) |
                   static_cast<uintptr_t>(g.bs) * sizeof(T)) % (4 * sizeof(T)) == 0;
  auto launch = [&](auto kernel, uint32_t ncb, int R) {
    const dim3 grid(ncb * static_cast<unsigned>((g.q.S + R - 1) / R));
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, g, ncb, static_cast<const T*>(in.u),
                       static_cast<const DT*>(in.delta), in.dbias, in.A, static_cast<const T*>(in.Bm),
                       static_cast<const T*>(in.Cm), in.Dv, static_cast<const T*>(in.z), states, static_cast<T*>(y));
    return hipGetLastError();
  };
  const auto blocks = [&](int G) { return static_cast<uint32_t>((g.q.D * G + 255) / 256); };
  if (!g.h_vec || !bc) return launch(seq_scan_step_kernel<T, DT, false, 1, 4>, blocks(4), 1);
  // four sequences a wave once that leaves each SIMD two waves.  MI355X, 1536 bf16
  // channels: 64 sequences 6.4 us by four, 6.1 by one; 128 7.8 and 8.8; 512 24.6
  // and 30.0; 2048 89 and 109
  auto run = [&](auto groups) {
    constexpr int G = decltype(groups)::value;
    const uint32_t ncb = blocks(G);
    return static_cast<int64_t>(g.q.S) * ncb >= 2 * 1024
               ? launch(seq_scan_step_kernel<T, DT, true, kStepRows, G>, ncb, kStepRows)
               : launch(seq_scan_step_kernel<T, DT, true, 1, G>, ncb, 1);
  };
  return g.N <= 4 ? run(std::integral_constant<int, 1>{})
                  : (g.N <= 8 ? run(std::integral_constant<int, 2>{}) : run(std::integral_constant<int, 4>{}));
}

}  // namespace

template <bool REV>
hipError_t launch_carry(const SeqScanGeom& g, const float* A, const float* enter, float* agg_h, const float* agg_s,
                        hipStream_t s) {
  if (g.q.S == 0) return hipSuccess;
  const uint32_t ncb = static_cast<uint32_t>((g.q.D + 15) / 16);
  hipLaunchKernelGGL(seq_carry_kernel<REV>, dim3(ncb * static_cast<unsigned>(g.q.S)), dim3(64 * carry_waves(g)), 0, s,
                     g, ncb, A, enter, agg_h, agg_s);
  return hipGetLastError();
}
template hipError_t launch_carry<false>(const SeqScanGeom&, const float*, const float*, float*, const float*, hipStream_t);
template hipError_t launch_carry<true>(const SeqScanGeom&, const float*, const float*, float*, const float*, hipStream_t);

template <typename T>
hipError_t launch_bc(const SeqScanGeom& g, const SeqScanIn& in, float* out, hipStream_t s) {
  const int64_t n = static_cast<int64_t>(g.q.T) * 32;
  if (n == 0) return hipSuccess;
  hipLaunchKernelGGL(seq_bc_kernel<T>, strided_grid(n), dim3(256), 0, s, g.q.T, g.N, g.bs,
                     static_cast<const T*>(in.Bm), static_cast<const T*>(in.Cm), out);
  return hipGetLastError();
}
template hipError_t launch_bc<float>(const SeqScanGeom&, const SeqScanIn&, float*, hipStream_t);
template hipError_t launch_bc<bf16_t>(const SeqScanGeom&, const SeqScanIn&, float*, hipStream_t);

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
    return with_bc<T>(g, in, b.bc, [&](auto bc) { return fwd_t<T, DT>(g, in, b, bc, s); }, s);
  });
}

hipError_t launch_seq_scan_step(const SeqScanGeom& g, const SeqScanIn& in, float* states, void* y, int dtype,
                                int delta_dtype, hipStream_t s) {
  return by_types(dtype, delta_dtype, [&](auto t, auto dt) {
    return step_t<decltype(t), decltype(dt)>(g, in, states, y, s);
  });
}

}  // namespace mvm
