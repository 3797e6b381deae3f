// The gated delta rule along time, by chunks of 64 tokens:
//   R  = diag(beta) (V - diag(e^G) K S)
//   D  = T R                                   (rows d_t)
//   O  = scale diag(e^G) Q S + P D             (formed as O', whose lanes hold
//                                               four columns of a token)
//   S' = e^Gc S + K' diag(e^(Gc - G)) D        (Gc: G of the last token)
// (with T and P of delta_prep.hip).  The columns of S are independent: a wave
// keeps 16 of them in registers, as result tiles whose rows are the keys'
// index, for the whole sequence, and the waves of a workgroup share the chunk's A
// operands in LDS: four of them, or eight (delta_capi.hip has the rule).
//
// Where sequences and heads are too few to fill the card, the sequences are cut
// into parts (delta_capi.hip decides): one pass leaves every part's end state
// from zero and its transition M (S' = M S + e), a second one joins them, and
// the main pass starts each part from its own state.
//
// Bound by the chain of products of a chunk, 5.5-7 us for bfloat16 heads of 128 x
// 128: 32768 tokens of 12 heads take 190 us in the main pass, MFMA busy 42 % with
// two waves a SIMD, which wait to issue 41 % of their cycles.  Operands are read a
// phase ahead and the next chunk's loads are spread over the phases: all at its
// start took a quarter longer.
#include "delta_common.h"

namespace mvm {
namespace {

struct FwdArgs {
  DeltaGeom g;
  DeltaIn in;
  DeltaWork w;
  const float* h0;
  float* h1;
  void* o;
  float* s0;
  float* vt;
  int64_t col_tiles;
  uint32_t vcb, ncb, nslots;  // column blocks of the values, and of the launch
};

// AGG: a part's end state from zero, and (column blocks from a.vcb on) its
// transition: what the identity becomes where V is zero.
template <typename T, int DKP, int NW, bool VEC, bool SAVE, bool AGG>
__global__ void __launch_bounds__(64 * NW)
delta_fwd_kernel(FwdArgs a) {
  constexpr int P = kRawParts<T>, KT = DKP / 16, KS = DKP / 32, NT = 64 * NW;
  constexpr int PP = AGG ? 0 : kTriParts;
  __shared__ __attribute__((aligned(16))) Tile<kC, DKP, P> sK;
  __shared__ __attribute__((aligned(16))) Tile<AGG ? 1 : kC, DKP, P> sQ;
  // float32 values go straight to the registers: with them the tiles would not fit
  constexpr bool VLDS = P == 1;
  __shared__ __attribute__((aligned(16))) Tile<VLDS ? kC : 1, 16 * NW, 1> sV;
  __shared__ uint4 sTri[StageTri<PP, NT>::kCount];
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
  if (part.t0 < 0) return;
  if (AGG && (part.seq >= g.q.S || part.t1 == part.end)) return;  // (nothing follows a last part)
  const int64_t orow = static_cast<int64_t>(g.HV) * g.DV, ocol = static_cast<int64_t>(h) * g.DV + at_col;
  const bool wlive = live && !trans;
  if (part.seq >= g.q.S) {  // rows of no sequence
    if (live)
      for (int32_t t = part.t0 + grp; t < part.t1; t += 4) static_cast<T*>(a.o)[t * orow + ocol + m] = from_f32<T>(0.f);
    return;
  }
  const int32_t row = seq_slot(g.q, part.seq);
  const int64_t cells = static_cast<int64_t>(g.DK) * g.DV, at_h = static_cast<int64_t>(h) * cells + at_col;
  const int64_t at_part = ((static_cast<int64_t>(p.slot) * g.HV + h) * a.col_tiles + col0 / 16) * (KT * 256);
  const bool tiles = !trans && col0 < g.DV;  // (this wave's column tile exists)
  f32x4 S[KT];
  if (trans) {
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) S[t][r] = 16 * t + 4 * grp + r == col ? 1.f : 0.f;
  } else if (!AGG && a.w.carry != nullptr) {
#pragma unroll
    for (int t = 0; t < KT; ++t)
      S[t] = tiles ? reinterpret_cast<const f32x4*>(a.w.carry + at_part)[64 * t + lane] : f32x4{0.f, 0.f, 0.f, 0.f};
  } else {
    const int32_t on = AGG ? 0 : seq_starts(g.q, part.seq, row, a.h0);
    load_state<KT>(S, a.h0 + on * (row * (g.HV * cells) + at_h), g.DV, on * g.DK, m, grp, live);
  }
  const T* kp = static_cast<const T*>(a.in.k) + hk * g.kh;
  const T* qp = static_cast<const T*>(a.in.q) + hk * g.qh;
  const int vcol0 = trans ? 0 : p.cb * NW * 16;  // the workgroup's columns of v
  const T* vp = static_cast<const T*>(a.in.v) + h * g.vh + (VLDS ? vcol0 : at_col);
  const int32_t slot0 = cut_div(g.cut, part.start) + part.seq + (part.t0 - part.start) / kC;
  const int32_t chunks = (part.t1 - part.t0 + kC - 1) / kC;
  // the next chunk's operands, on their way while this one's are at work
  StageRows<T, DKP, NT> rK, rQ;
  StageTri<PP, NT> rT;
  float rDec;
  float rGam;
  Cols<T> rV;
  StageRows<T, 16 * NW, NT> rVt;
  // Loads of chunk i, a few at a time between the phases of the products: all at once they hold up the wave that
  // issues them, and all waves at the next barrier, for as long as the memory pipeline takes them.
  constexpr int kLoads = 8;
  const auto load = [&](int32_t i, int which) {
    const int32_t t0 = part.t0 + i * kC;
    const int n = part.t1 - t0 < kC ? part.t1 - t0 : kC;
    const int64_t at = static_cast<int64_t>(slot0 + i) * g.HV + h;
    switch (which) {
      case 0: rK.template load<VEC>(kp + t0 * g.ks, g.ks, n, g.DK, tid); break;
      case 1:
        if constexpr (!AGG) rQ.template load<VEC>(qp + t0 * g.qs, g.qs, n, g.DK, tid);
        break;
      case 2:
        if constexpr (VLDS) rVt.template load<VEC>(vp + t0 * g.vs, g.vs, n, trans ? 0 : g.DV - vcol0, tid);
        break;
      case 3:
        if (tid < 4 * kC) rDec = a.w.dec[at * (4 * kC) + tid];
        rGam = a.w.gam[at];
        break;
      default: rT.load(reinterpret_cast<const uint4*>(a.w.tri) + at * kTriFragments, tid, which - 4, which - 3); break;
    }
  };
  const auto load_v = [&](int32_t i) {
    const int32_t t0 = part.t0 + i * kC;
    rV.load(vp + t0 * g.vs, g.vs, m, grp, part.t1 - t0 < kC ? part.t1 - t0 : kC, wlive);
  };
  Quad<T> out[4];
  const auto store = [&](int32_t t0, int n) {
#pragma unroll
    for (int rt = 0; rt < 4; ++rt)
      if (16 * rt + m < n)
        out[rt].store(static_cast<T*>(a.o) + (t0 + 16 * rt + m) * orow + static_cast<int64_t>(h) * g.DV, col0 + 4 * grp, g.DV, VEC);
  };
  if (chunks > 0) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) load(0, i);
    if constexpr (!VLDS) load_v(0);
  }
  for (int32_t nth = 0; nth < chunks; ++nth) {
    const int32_t t0 = part.t0 + nth * kC;
    const int n = part.t1 - t0 < kC ? part.t1 - t0 : kC;
    const int64_t at = static_cast<int64_t>(slot0 + nth) * g.HV + h;
    __syncthreads();
    rK.put(sK, n, g.DK, tid);
    if constexpr (!AGG) rQ.put(sQ, n, g.DK, tid);
    if constexpr (VLDS) rVt.put(sV, n, trans ? 0 : g.DV - vcol0, tid);
    rT.put(sTri, tid);
    if (tid < 4 * kC) sDec[0][tid] = rDec;
    const float gam = rGam;
    // The last chunk's outputs go out here: the wait for the loads above is one for all earlier memory accesses,
    // and stores right before it would be waited for.
    if constexpr (!AGG)
      if (nth > 0) store(t0 - kC, kC);
    // (past the last chunk: the last one again, so that no branch parts the phases)
    const int32_t ahead = nth + 1 < chunks ? nth + 1 : nth;
    const int64_t at_tile = (at * a.col_tiles + col0 / 16) * 256;
    if constexpr (SAVE)
      if (col0 < g.DV) store_tiles<KT>(a.s0 + at_tile * KT, S, lane);
    __syncthreads();
    f32x4 R[4], O[4], D[4];
#pragma unroll
    for (int rt = 0; rt < 4; ++rt) R[rt] = O[rt] = D[rt] = f32x4{0.f, 0.f, 0.f, 0.f};
    Frag<P> fk[2][4], fq[2][AGG ? 1 : 4];
    const auto rows = [&](int ks) {
#pragma unroll
      for (int rt = 0; rt < 4; ++rt) {
        fk[ks & 1][rt] = sK.rows(16 * rt + m, ks, grp);
        if constexpr (!AGG) fq[ks & 1][rt] = sQ.rows(16 * rt + m, ks, grp);
      }
    };
    f32x4 dk[4], beta[4];
    rows(0);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      if (ks + 1 < KS)
        rows(ks + 1);
      else
#pragma unroll
        for (int rt = 0; rt < 4; ++rt) {
          dk[rt] = dec_at(sDec, kDecKey, rt, grp);
          beta[rt] = dec_at(sDec, kDecBeta, rt, grp);
        }
      const Frag<3> sf = split_tiles<3>(S[2 * ks], S[2 * ks + 1]);
      mma_n<3>(fk[ks & 1], sf, R);
      if constexpr (!AGG) mma_t<3>(sf, fq[ks & 1], O);
#pragma unroll
      for (int i = 4 * ks / KS; i < 4 * (ks + 1) / KS; ++i) load(ahead, i);
      phase();
    }
    Frag<3> t0f[4], t1f[2];
    tri_tiles<0>(t0f, sTri, 0, 0, m, grp);
#pragma unroll
    for (int rt = 0; rt < 4; ++rt) {
      f32x4 V;
      if constexpr (VLDS)
        V = sV.col4(16 * wave, 16 * rt + 4 * grp, m);
      else
        V = rV.tile(rt, grp, n, wlive);
      R[rt] = beta[rt] * (V - dk[rt] * R[rt]);
    }
    if constexpr (!VLDS) load_v(ahead);
    const Frag<3> rf[2] = {split_tiles<3>(R[0], R[1]), split_tiles<3>(R[2], R[3])};
    phase();
    tri_tiles<2>(t1f, sTri, 0, 1, m, grp);
    mma_n<3>(t0f, rf[0], D);
    load(ahead, 4);
    phase();
    Frag<3> p0f[4], p1f[2];
    float dout[4];  // (the outputs' tiles have the token in the column)
    if constexpr (!AGG) {
      tri_tiles<0>(p0f, sTri, 1, 0, m, grp);
#pragma unroll
      for (int rt = 0; rt < 4; ++rt) dout[rt] = sDec[kDecOut][16 * rt + m];
    }
    mma_n<3>(t1f, rf[1], D + 2);
    load(ahead, 5);
    phase();
    if constexpr (SAVE)
      if (col0 < g.DV) store_tiles<4>(a.vt + at_tile * 4, D, lane);
    f32x4 up[4];
#pragma unroll
    for (int rt = 0; rt < 4; ++rt) up[rt] = dec_at(sDec, kDecUp, rt, grp);
    if constexpr (!AGG) {
      const Frag<3> df[2] = {split_tiles<3>(D[0], D[1]), split_tiles<3>(D[2], D[3])};
#pragma unroll
      for (int rt = 0; rt < 4; ++rt) O[rt] *= dout[rt];
      tri_tiles<2>(p1f, sTri, 1, 1, m, grp);
      mma_t<3>(df[0], p0f, O);
      phase();
      mma_t<3>(df[1], p1f, O + 2);
    }
    constexpr int KG = KT < 4 ? KT : 4;  // row tiles of the state at a time
    Frag<P> fc[2][KG];
    const auto keys = [&](int t0, int ks) {
#pragma unroll
      for (int i = 0; i < KG; ++i) fc[ks][i] = sK.cols(16 * (t0 + i), 32 * ks + 4 * grp, m);
    };
    keys(0, 0);
#pragma unroll
    for (int rt = 0; rt < 4; ++rt) D[rt] *= up[rt];
    const Frag<3> uf[2] = {split_tiles<3>(D[0], D[1]), split_tiles<3>(D[2], D[3])};
#pragma unroll
    for (int t = 0; t < KT; ++t) S[t] *= gam;
    load(ahead, 6);
    load(ahead, 7);
    phase();
#pragma unroll
    for (int t = 0; t < KT; t += KG)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        if (ks == 0)
          keys(t, 1);
        else if (t + KG < KT)
          keys(t + KG, 0);
        mma_n<3>(fc[ks], uf[ks], S + t);
        phase();
      }
    if constexpr (!AGG)
#pragma unroll
      for (int rt = 0; rt < 4; ++rt) out[rt].set(O[rt]);
  }
  if constexpr (!AGG)
    if (chunks > 0) store(part.t0 + (chunks - 1) * kC, part.t1 - part.t0 - (chunks - 1) * kC);
  if (AGG && trans) {
    if (col0 < DKP) store_tiles<KT>(a.w.trans + ((static_cast<int64_t>(p.slot) * g.HV + h) * KT + col0 / 16) * (KT * 256), S, lane);
  } else if (AGG) {
    if (tiles) store_tiles<KT>(a.w.carry + at_part, S, lane);
  }
  else if (a.h1 != nullptr && row >= 0 && part.t1 == part.end)
    store_state<KT>(a.h1 + row * (g.HV * cells) + at_h, g.DV, g.DK, S, m, grp, live);
}

// Joins the parts of a sequence: carry holds each part's end state from zero (REV: the gradient of its initial
// state) and gets its initial state (of its final one), S' = M S + e with the parts' transitions M.  The parts come
// one after the other: four waves have 16 columns of S each, share M in LDS, and load the next part's while they
// work.  (Every wave loading and splitting M for itself took 13.5 us a part, this 5.3: 128 x 128.)
template <int DKP, bool REV>
__global__ void __launch_bounds__(256)
delta_carry_kernel(DeltaGeom g, DeltaWork w, const float* __restrict__ enter, uint32_t ncb, int64_t col_tiles) {
  constexpr int KT = DKP / 16, KS = DKP / 32, kItems = KT * KT * 64 / 256;
  __shared__ __attribute__((aligned(16))) Tile<DKP, DKP, 3> sM;  // rows: M's columns
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_id(), m = lane & 15, grp = lane >> 4;
  const uint32_t item = blockIdx.x / ncb;
  const int32_t seq = static_cast<int32_t>(item / static_cast<uint32_t>(g.HV));
  const int h = static_cast<int>(item - static_cast<uint32_t>(seq) * g.HV);
  const int col0 = static_cast<int>(blockIdx.x - item * ncb) * 64 + 16 * wave;
  const bool tiles = col0 < g.DV, live = col0 + m < g.DV;
  const int32_t start = seq_off_u(g.q, seq), next = seq_off_u(g.q, seq + 1), end = next < start ? start : next;
  const int32_t slot0 = cut_div(g.part, start) + seq, parts = end > start ? cut_div(g.part, end - start - 1) + 1 : 1;
  const int32_t row = REV ? seq : seq_slot(g.q, seq);
  const int64_t cells = static_cast<int64_t>(g.DK) * g.DV;
  f32x4 S[KT], E[KT], rM[kItems];
  {
    const int32_t on = REV ? enter != nullptr : seq_starts(g.q, seq, row, enter);
    load_state<KT>(S, enter + on * ((row * static_cast<int64_t>(g.HV) + h) * cells + (tiles ? col0 : 0)), g.DV,
                   on * g.DK, m, grp, live);
  }
  const auto at_part = [&](int32_t i) { return static_cast<int64_t>(slot0 + (REV ? parts - 1 - i : i)) * g.HV + h; };
  const auto load = [&](int32_t i) {
    const f32x4* M = reinterpret_cast<const f32x4*>(w.trans + at_part(i) * (KT * KT * 256));
#pragma unroll
    for (int j = 0; j < kItems; ++j) rM[j] = M[tid + 256 * j];
  };
  if (parts > 1) load(0);
  for (int32_t i = 0; i < parts; ++i) {
    f32x4* c = reinterpret_cast<f32x4*>(w.carry + (at_part(i) * col_tiles + col0 / 16) * (KT * 256)) + lane;
    const bool last = i + 1 == parts;
#pragma unroll
    for (int t = 0; t < KT; ++t) E[t] = tiles && !last ? c[64 * t] : f32x4{0.f, 0.f, 0.f, 0.f};
    if (tiles)
#pragma unroll
      for (int t = 0; t < KT; ++t) c[64 * t] = S[t];
    if (last) break;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kItems; ++j) {
      const int x = (tid + 256 * j) / 64;  // column tile x / KT, row tile x % KT
      sM.put4(16 * (x / KT) + m, 16 * (x % KT) + 4 * grp, rM[j]);
    }
    if (i + 2 < parts) load(i + 1);
    __syncthreads();
    constexpr int KG = KT < 4 ? KT : 4;
    Frag<3> sf[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) sf[ks] = split_tiles<3>(S[2 * ks], S[2 * ks + 1]);
#pragma unroll
    for (int t = 0; t < KT; t += KG)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        Frag<3> f[KG];
#pragma unroll
        for (int j = 0; j < KG; ++j) f[j] = sM.cols(16 * (t + j), 32 * ks + 4 * grp, m);
        mma_n<3>(f, sf[ks], E + t);
      }
#pragma unroll
    for (int t = 0; t < KT; ++t) S[t] = E[t];
  }
}

}  // namespace

template <bool REV>
hipError_t launch_delta_carry(const DeltaGeom& g, const DeltaWork& w, const float* enter, hipStream_t s) {
  if (g.q.S == 0) return hipSuccess;
  const uint32_t ncb = delta_col_blocks(g.DV, 4);
  const dim3 grid(static_cast<unsigned>(static_cast<int64_t>(g.q.S) * g.HV * ncb));
  switch (delta_dkp(g.DK)) {
    case 32: hipLaunchKernelGGL((delta_carry_kernel<32, REV>), grid, dim3(256), 0, s, g, w, enter, ncb, delta_col_tiles(g)); break;
    case 64: hipLaunchKernelGGL((delta_carry_kernel<64, REV>), grid, dim3(256), 0, s, g, w, enter, ncb, delta_col_tiles(g)); break;
    default: hipLaunchKernelGGL((delta_carry_kernel<128, REV>), grid, dim3(256), 0, s, g, w, enter, ncb, delta_col_tiles(g)); break;
  }
  return hipGetLastError();
}
template hipError_t launch_delta_carry<false>(const DeltaGeom&, const DeltaWork&, const float*, hipStream_t);
template hipError_t launch_delta_carry<true>(const DeltaGeom&, const DeltaWork&, const float*, hipStream_t);

hipError_t launch_delta_fwd(const DeltaGeom& g, const DeltaIn& in, const DeltaWork& w, const float* h0, float* h1,
                            void* o, float* s0, float* vt, int dtype, hipStream_t s) {
  // (rows that are read value by value: more registers, so four waves)
  const int nw = g.vec ? g.waves : 4;
  const uint32_t vcb = delta_col_blocks(g.DV, nw);
  FwdArgs a{g, in, w, h0, h1, o, s0, vt, delta_col_tiles(g), vcb, vcb, static_cast<uint32_t>(chunk_slots(g.q, g.part))};
  hipError_t e = launch_delta_prep(g, in, w, dtype, s);
  if (e != hipSuccess) return e;
  const auto run = [&](auto t, auto dkp, auto waves, auto vec) {
    using T = decltype(t);
    constexpr int DKP = decltype(dkp)::value, NW = decltype(waves)::value;
    constexpr bool VEC = decltype(vec)::value;
    if (g.parts > 1) {
      a.ncb = vcb + delta_col_blocks(DKP, NW);
      hipLaunchKernelGGL((delta_fwd_kernel<T, DKP, NW, VEC, false, true>),
                         dim3(static_cast<unsigned>(delta_blocks(a.ncb, a.nslots, g.HV))), dim3(64 * NW), 0, s, a);
      hipError_t e = hipGetLastError();
      if (e != hipSuccess || (e = launch_delta_carry<false>(g, w, h0, s)) != hipSuccess) return e;
      a.ncb = vcb;
    }
    const dim3 grid(static_cast<unsigned>(delta_blocks(a.ncb, a.nslots, g.HV)));
    if (s0 != nullptr)
      hipLaunchKernelGGL((delta_fwd_kernel<T, DKP, NW, VEC, true, false>), grid, dim3(64 * NW), 0, s, a);
    else
      hipLaunchKernelGGL((delta_fwd_kernel<T, DKP, NW, VEC, false, false>), grid, dim3(64 * NW), 0, s, a);
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
