// Backward of the packed selective scan for gfx950 (the forward's formulas and
// cut into chunks: seq_scan.hip).
//
//   dr_t = dy_t silu(z_t),  dh_t = C_t dr_t + c_{t+1},  c_t = exp(delta_t A) dh_t
//   dB_t = sum_d dh_t delta_t u_t,  dC_t = sum_d dr_t h_t,
//   ddelta_t = sum_n dh_t (A exp(delta_t A) h_{t-1} + B_t u_t),
//   du_t = delta_t sum_n dh_t B_t + D dr_t,  dA = sum_t dh_t delta_t exp(delta_t A) h_{t-1}
//
// with c past a sequence's end the final state's gradient, and c_first the
// initial state's.  The same passes as forward, in the other direction.
//
// Bound by VALU issue.  On MI355X, 16384 bf16 tokens of 1536 channels: aggregate
// pass 78 us, carry 12, main pass 259 (VALU busy 93 %), reductions 14.  The main
// pass issues 346 VALU instructions a token and wave: 13 a state for the
// recurrence and its gradients, 4.4 for the sums of dB and dC over the wave's
// channels.  Three waves a SIMD at 168 VGPRs; one at 275 took 2.2 times as long,
// and two with the next tile's loads ahead no less than three.
#include "seq_scan_pass.h"

namespace mvm {

namespace {

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
  float zeros[kZeroRow];
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
  const uint32_t lane = threadIdx.x & 63;
  const WavePos pos = wave_pos(args.ncb);
  const SeqChunk c = seq_chunk(g.q, pos.slot, g.cut, lane);
  const int64_t D = g.q.D, d0 = static_cast<int64_t>(pos.cb) * kWave;
  if (c.t0 <= c.start || c.seq == g.q.S) return;
  const bool valid = d0 + lane < D;
  const uint32_t lc = valid ? lane : static_cast<uint32_t>(D - 1 - d0);
  const int64_t d = d0 + lc;
  const bool soft = g.softplus != 0, gate = args.z != nullptr;
  RowPtr py, pd, pz, pc;
  pc.set(args.bc.C, c.t1 - 1, args.bc.st);
  py.set(args.dy + d0, c.t1 - 1, g.ys);
  pd.set(args.delta + d0, c.t1 - 1, g.ds);
  if (gate) pz.set(args.z + d0, c.t1 - 1, g.zs);
  T ny[kSeqTile], nz[kSeqTile];
  DT nd[kSeqTile];
  auto fetch = [&](int32_t t) {
    load_prev(nd, pd, t, c.t1, lc);
    load_prev(ny, py, t, c.t1, lc);
    if (gate) load_prev(nz, pz, t, c.t1, lc);
  };
  const int32_t last = c.t0 + ((c.t1 - 1 - c.t0) & ~(kSeqTile - 1));
  fetch(last);
  const float bias = p.dbias ? p.dbias[d] : 0.f;
  float a2[16], h[16];
  load_a2(a2, p.A, d, 0, g);
#pragma unroll
  for (int n = 0; n < 16; ++n) h[n] = 0.f;
  float sum_dl = 0.f;
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
      Cv.load(t + i < c.t1 ? pc.at : zero_row());
      pc.prev(t + i < c.t1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < 16; ++n) a[n] = fast_exp2(dl[i] * a2[n]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < 16; ++n) h[n] = a[n] * fmaf(Cv[n], dr[i], h[n]);
      sum_dl += dl[i];
    }
  }
  if (!valid) return;
  const auto& late = late_args<BwdArgs<T, DT, BT>>();
  store_agg(h, late.p.agg_h, c.slot, D, d);
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
// (an inner loop that is not unrolled, and ends with the states there are:
// 16384 bf16 tokens of 1536 channels, forward and backward: 546 us with 16, 418
// with 8, 370 with 4): the tile is run forward from its
// checkpoint with the states and decays kept in registers, then backward.
// What a state carries from tile to tile (its adjoint and dA) waits in LDS, and
// the tile's B and C, from where all lanes read them.  All of a wave's LDS is
// its own: no barrier.
struct BwdLds {
  Pack<float, 4> a2[4][kWave], c[4][kWave], da[4][kWave];
  // per state B of the 8 tokens, C of the 8; replaced, once the state is done,
  // by the tile's sums for dB and dC
  Pack<float, 4> bc[16][4];
};

template <typename T, typename DT, typename BT>
__global__ void __launch_bounds__(256, 3)
seq_scan_bwd_kernel(BwdArgs<T, DT, BT> args) {
  __shared__ BwdLds lds[4];
  const SeqScanGeom& g = args.g;
  const BwdPtrs& p = args.p;
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
  const bool soft = g.softplus != 0, gate = args.z != nullptr, all_valid = d0 + kWave <= D;
  RowPtr pu, pd, py, pz;
  pu.set(args.u + d0, c.t1 - 1, g.us);
  pd.set(args.delta + d0, c.t1 - 1, g.ds);
  py.set(args.dy + d0, c.t1 - 1, g.ys);
  if (gate) pz.set(args.z + d0, c.t1 - 1, g.zs);
  T nu[kSeqTile], ny[kSeqTile], nz[kSeqTile];
  DT nd[kSeqTile];
  BcTile<BT> nbc;
  auto fetch = [&](int32_t t, int32_t end) {
    nbc.fetch(args.bc.B, args.bc.C, args.bc.st, t, end, 16, lane);
    load_prev(nd, pd, t, end, lc);
    load_prev(nu, pu, t, end, lc);
    load_prev(ny, py, t, end, lc);
    if (gate) load_prev(nz, pz, t, end, lc);
  };
  const int32_t row = seq_slot(g.q, c.seq);
  {
    float a2[16], h[16];
#pragma unroll
    for (int n = 0; n < 16; ++n) h[n] = 0.f;
    if (g.multi && !g.fold)
      load_agg(h, p.agg_h, c.slot, D, dc);
    else if (p.dh1 != nullptr)
      load_states(h, p.dh1, row * D + dc, 0, g.N, g.h_vec);
    load_a2(a2, p.A, dc, 0, g);
    if (g.multi && g.fold) {
      const int32_t end = last_slot(g.cut, c);
      fold_chunks<-1>(h, a2, p.agg_h, p.agg_s, end, end - c.slot, D, dc);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      s.a2[q][lane] = Pack<float, 4>{a2[4 * q], a2[4 * q + 1], a2[4 * q + 2], a2[4 * q + 3]};
      s.c[q][lane] = valid ? Pack<float, 4>{h[4 * q], h[4 * q + 1], h[4 * q + 2], h[4 * q + 3]}
                           : Pack<float, 4>{0.f, 0.f, 0.f, 0.f};
      s.da[q][lane] = Pack<float, 4>{0.f, 0.f, 0.f, 0.f};
    }
  }
  const float bias = p.dbias ? p.dbias[dc] : 0.f;
  const float Dd = p.Dv[dc];
  float dD = 0.f, ddb = 0.f;
  const int64_t ck0 = (c.start >> kSeqTileShift) + c.seq;
  Pace pace(c.t1 - c.t0);
  // 8 tokens from t on; of a chunk's last tile, which is taken first, maybe fewer:
  // a copy of the code with masks (which in every tile would be one instruction
  // in 13 a state; a branch inside, or two copies of the states' loop alone,
  // spill 16 to 190 registers)
  auto tile = [&](int32_t t, auto whole) {
    constexpr bool kWhole = decltype(whole)::value;
    const int32_t end = kWhole ? t + kSeqTile : c.t1;
    pace.tile();
    float dl[kSeqTile], du[kSeqTile], dr[kSeqTile], qs[kSeqTile], ws[kSeqTile], rs[kSeqTile];
    float us[kSeqTile], sg[kSeqTile], gz[kSeqTile];  // for the outputs
    fetch(t, end);
    lds_order();
#pragma unroll
    for (int j = 0; j < 4; ++j)
      reinterpret_cast<float*>(s.bc)[(4 * (lane & 3) + j) * 16 + 2 * (lane & 4) + (lane >> 3)] =
          nbc.value(j, 16, lane, t, end);
    lds_order();
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
    if (!kWhole || !all_valid) {
      // positions past the chunk, channels that do not exist: nothing decays,
      // enters or leaves
#pragma unroll
      for (int i = 0; i < kSeqTile; ++i) {
        const bool in = valid && (kWhole || t + i < end);
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
    const int32_t states = late_args<BwdArgs<T, DT, BT>>().g.N;
#pragma unroll 1
    for (int q = 0; q < 4; ++q) {
      if (4 * q >= states) break;  // (those past the last one have no part in anything)
      const Pack<float, 4> a2 = s.a2[q][lane];
      Pack<float, 4> cs = s.c[q][lane], da = s.da[q][lane], h4 = hs;
      if (q < 3) hs = load_pack<float, 4>(ck + (q + 1) * 4 * D);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        __builtin_amdgcn_sched_barrier(0);
        float Bv[kSeqTile], Cv[kSeqTile];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const Pack<float, 4> bk = s.bc[4 * q + j][k], ck4 = s.bc[4 * q + j][2 + k];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            Bv[4 * k + i] = bk.v[i];
            Cv[4 * k + i] = ck4.v[i];
          }
        }
        float h = valid ? h4.v[j] : 0.f;
        float a[kSeqTile], ah[kSeqTile], v[16];  // v: the terms of dB of the 8 tokens, then those of dC
#pragma unroll
        for (int i = 0; i < kSeqTile; ++i) {
          a[i] = fast_exp2(dl[i] * a2.v[j]);
          ah[i] = a[i] * h;
          h = fmaf(du[i], Bv[i], ah[i]);
          rs[i] = fmaf(h, Cv[i], rs[i]);
          v[8 + i] = dr[i] * h;
        }
#pragma unroll
        for (int i = kSeqTile - 1; i >= 0; --i) {
          const float dh = fmaf(Cv[i], dr[i], cs.v[j]);
          qs[i] = fmaf(dh, Bv[i], qs[i]);
          v[i] = dh * du[i];
          float w = dh * ah[i];
          // (past the chunk delta is zero, and either factor may be infinite)
          if constexpr (!kWhole) w = t + i < end ? w : 0.f;
          da.v[j] = fmaf(w, dl[i], da.v[j]);
          ws[i] = fmaf(w, a2.v[j], ws[i]);
          cs.v[j] = dh * a[i];
        }
        reinterpret_cast<float*>(s.bc[4 * q + j])[lane >> 2] = wave_sums16(v, lane);  // (four lanes, one value)
      }
      s.c[q][lane] = cs;
      s.da[q][lane] = da;
    }
    const auto& late = late_args<BwdArgs<T, DT, BT>>();
    lds_order();
    // rows t .. t + 7 of 32 values: dB at 0, dC at 16
    float* out = late.p.part_bc + (static_cast<int64_t>(pos.cb) * g.q.T + t) * 32;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = k * 2 + (lane >> 5), n = lane & 31;
      const float v = reinterpret_cast<const float*>(s.bc)[(n & 15) * 16 + (n >> 4) * 8 + i];
      if (kWhole || t + i < end) out[i * 32 + n] = v;
    }
    lds_order();
    const int32_t rows = end - t;
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
  };
  int32_t t = c.t0 + ((c.t1 - 1 - c.t0) & ~(kSeqTile - 1));
  if (c.t0 < c.t1 && t + kSeqTile > c.t1) {
    tile(t, std::false_type{});
    t -= kSeqTile;
  }
  for (; c.t0 < c.t1 && t >= c.t0; t -= kSeqTile) tile(t, std::true_type{});
  if (!valid) return;
  const auto& late = late_args<BwdArgs<T, DT, BT>>();
  float* part = late.p.part + static_cast<int64_t>(c.slot) * 18 * D + d;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const Pack<float, 4> da = s.da[q][lane], cs = s.c[q][lane];
#pragma unroll
    for (int j = 0; j < 4; ++j) part[(4 * q + j) * D] = da.v[j];
    if (c.t0 == c.start && late.p.dh0 != nullptr) store_states(cs.v, late.p.dh0, row * D + d, 4 * q, late.g.N, late.g.h_vec);
  }
  part[16 * D] = dD;
  part[17 * D] = ddb;
}

// The first `pblocks` workgroups: dA, dD and ddelta_bias, the chunks' sums added
// in order.  The others: dB and dC, the channel blocks' sums added in order.
template <typename T>
struct ReduceArgs {
  int64_t D, nparts;
  int32_t N, a_log, rows, ncb;
  uint32_t pblocks;
  const float *A, *part, *part_bc;
  float *dA, *dD, *ddb;
  T *dB, *dC;
};
template <typename T>
__global__ void __launch_bounds__(1024)
seq_reduce_kernel(ReduceArgs<T> r) {
  if (blockIdx.x < r.pblocks) {
    sum_columns(r.part, r.nparts, 18 * r.D, [&](int64_t col, float s) {
      const int64_t k = col / r.D, d = col - k * r.D;
      if (k < r.N)
        r.dA[d * r.N + k] = r.a_log ? s * -expf(r.A[d * r.N + k]) : s;  // of A_log: A' = A
      else if (k == 16)
        r.dD[d] = s;
      else if (k == 17 && r.ddb != nullptr)
        r.ddb[d] = s;
    });
    return;
  }
  const int64_t total = static_cast<int64_t>(r.rows) * 32;
  const int64_t step = static_cast<int64_t>(gridDim.x - r.pblocks) * 1024;
  const int n = threadIdx.x & 15;
  T* out = (threadIdx.x & 16) ? r.dC : r.dB;
  for (int64_t i = static_cast<int64_t>(blockIdx.x - r.pblocks) * 1024 + threadIdx.x; i < total; i += step) {
    float s = 0.f;
    for (int32_t k0 = 0; k0 < r.ncb; k0 += 8) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = r.part_bc[(k0 + k < r.ncb ? k0 + k : 0) * total + i];
#pragma unroll
      for (int k = 0; k < 8; ++k) s += k0 + k < r.ncb ? v[k] : 0.f;
    }
    if (n < r.N) out[(i >> 5) * r.N + n] = from_f32<T>(s);
  }
}

// ----------------------------------------------------------------- launches

// (without channels just zeros for dB and dC)
template <typename T>
hipError_t launch_reduce(const SeqScanGeom& g, const SeqScanIn& in, const SeqScanBwd& b, int64_t slots, hipStream_t s) {
  const uint32_t pblocks = static_cast<uint32_t>((18 * g.q.D + 63) / 64);
  const int64_t bblocks = std::min<int64_t>((static_cast<int64_t>(g.q.T) * 32 + 1023) / 1024, 1 << 18);
  if (pblocks + bblocks == 0) return hipSuccess;
  const ReduceArgs<T> red{g.q.D, slots, g.N, g.a_log, g.q.T, static_cast<int32_t>(blocks_of(g.q.D)), pblocks, in.A,
                          b.part, b.part_bc, b.dA, b.dD, b.ddbias, static_cast<T*>(b.dB), static_cast<T*>(b.dC)};
  hipLaunchKernelGGL(seq_reduce_kernel<T>, dim3(pblocks + static_cast<unsigned>(bblocks)), dim3(1024), 0, s, red);
  return hipGetLastError();
}

template <typename T, typename DT, typename BT>
hipError_t bwd_t(SeqScanGeom g, const SeqScanIn& in, const SeqScanBwd& b, BcRows<BT> bc, hipStream_t s) {
  set_vec(g, in.A, b.dh1, b.dh0);
  const uint32_t ncb = blocks_of(g.q.D);
  const int64_t slots = chunk_slots(g.q, g.cut);
  const dim3 grid = wave_grid(slots, ncb);
  const BwdArgs<T, DT, BT> args{{}, g, {in.dbias, in.A, in.Dv, b.dh1, b.dh0, b.ckpt, b.agg_h, b.agg_s, b.part, b.part_bc},
                            bc, ncb, static_cast<uint32_t>(slots), static_cast<const T*>(in.u),
                            static_cast<const DT*>(in.delta), static_cast<const T*>(in.z),
                            static_cast<const T*>(b.dy), static_cast<T*>(b.du), static_cast<DT*>(b.ddelta),
                            static_cast<T*>(b.dz)};
  hipError_t e;
  if (g.multi) {
    hipLaunchKernelGGL((seq_scan_bwd_agg_kernel<T, DT, BT>), grid, dim3(256), 0, s, args);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    if (!g.fold && (e = launch_carry<true>(g, in.A, b.dh1, b.agg_h, b.agg_s, s)) != hipSuccess) return e;
  }
  hipLaunchKernelGGL((seq_scan_bwd_kernel<T, DT, BT>), grid, dim3(256), 0, s, args);
  if ((e = hipGetLastError()) != hipSuccess) return e;
  return launch_reduce<T>(g, in, b, slots, s);
}

}  // namespace

hipError_t launch_seq_scan_bwd(const SeqScanGeom& g, const SeqScanIn& in, const SeqScanBwd& b, int dtype,
                               int delta_dtype, hipStream_t s) {
  return by_types(dtype, delta_dtype, [&](auto t, auto dt) {
    using T = decltype(t);
    using DT = decltype(dt);
    if (g.q.D == 0) return launch_reduce<T>(g, in, b, 0, s);
    return with_bc<T>(g, in, b.bc, [&](auto bc) { return bwd_t<T, DT>(g, in, b, bc, s); }, s);
  });
}

}  // namespace mvm
