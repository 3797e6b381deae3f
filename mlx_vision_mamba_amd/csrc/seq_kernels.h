// Packed sequences with states: parameter blocks and launch entry points of
// the scan (seq_scan.hip) and the conv (seq_conv.hip), used by the C ABI
// (seq_capi.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mvm {

// Lengths of chunks that positions are cut by.  n / len for 0 <= n < 2^31 is
// (n * magic) >> (32 + shift): magic = ceil(2^(32 + shift) / len), shift =
// ceil(log2(len)) - 1, exact there because the error of magic, below len <=
// 2^(shift + 1), times n stays below 2^(32 + shift).
struct SeqCut {
  uint32_t len, magic, shift;  // len in [8, 2^31]
};
inline SeqCut seq_cut(int64_t len) {
  uint32_t l = 3;
  while ((uint64_t{1} << l) < static_cast<uint64_t>(len)) ++l;
  const uint64_t two = uint64_t{1} << (31 + l);
  return {static_cast<uint32_t>(len), static_cast<uint32_t>((two + len - 1) / len), l - 1};
}

// The cut of the token rows into sequences, and their state rows.  Work is
// handed out in chunks of positions of one sequence.  The chunk slots of
// sequence i start at offset(i) / len + i: floor(a) + 1 >= ceil(a)
// keeps the ranges apart, so a chunk finds its sequence by a search over the
// offsets, without a table made before the launch, and every sequence, an
// empty one too, has at least one slot.  Sequence S stands for the rows past
// the last offset, whose outputs are zero.
struct SeqGeom {
  int32_t T, S, M, L;    // token rows, sequences, state rows, length (off == nullptr)
  int64_t D;
  const int32_t* off;    // (S + 1) or nullptr
  const int32_t* slots;  // (S) or nullptr
  const uint8_t* fresh;  // (S) or nullptr
};
inline int64_t chunk_slots(const SeqGeom& g, const SeqCut& cut) {
  return static_cast<int64_t>(g.T) / cut.len + g.S + 1;
}

constexpr int kSeqTile = 8;       // positions per tile, and between checkpoints
constexpr int kSeqTileShift = 3;

struct SeqScanGeom {
  SeqGeom q;
  int64_t us, ds, bs, ys, zs;  // row strides
  int32_t N;
  SeqCut cut;
  int32_t multi;       // 0: every sequence is one chunk, no carries
  int32_t fold;        // 1: the main pass joins the chunks before its own itself, 0: a carry pass does
  int32_t max_chunks;  // of a sequence, as far as the caller's max_len holds
  int32_t a_log, softplus;
  int32_t a_vec, h_vec;  // rows of A, of the states, are read 16 bytes at a time
};

// Chunks whose aggregates a wave of the carry pass holds, and its waves.
constexpr int kCarryRun = 8;
inline int carry_waves(const SeqScanGeom& g) {
  const int w = (g.max_chunks + kCarryRun - 1) / kCarryRun;
  return w < 1 ? 1 : (w > 16 ? 16 : w);
}

struct SeqScanIn {
  const void* u;
  const void* delta;
  const float* dbias;  // or null
  const float* A;
  const void* Bm;
  const void* Cm;
  const float* Dv;
  const void* z;       // or null
};
struct SeqScanFwd {
  const float* h0;  // or null; may be h1
  float* h1;        // or null
  void* y;
  float* ckpt;      // or null
  float* agg_h;     // (slots, 4, D, 4; the groups that there are): end states from zero, then carry-ins; with
                    // fold the initial state at each sequence's last chunk
  float* agg_s;     // (slots, D): sum of delta
  float* bc;        // (T, 32) float32 copies of B | C, or null: read in place
};
struct SeqScanBwd {
  const float* ckpt;
  const void* dy;
  const float* dh1;  // or null
  void* du;
  void* ddelta;
  float* ddbias;     // or null
  float* dA;
  void* dB;
  void* dC;
  float* dD;
  void* dz;          // or null
  float* dh0;        // or null
  float* agg_h;      // adjoint aggregates, then carry-ins
  float* agg_s;
  float* part;       // (slots, 18, D): dA | dD | ddelta_bias of each chunk
  float* part_bc;    // (channel blocks, T, 32)
  float* bc;
};

// true when B and C rows are read where they lie by scalar loads: 16 states,
// rows that start on 4 bytes.  Others are first copied to float32 rows of 32.
bool seq_bc_in_place(const SeqScanGeom& g, const SeqScanIn& in, int dtype);
hipError_t launch_seq_scan_fwd(const SeqScanGeom& g, const SeqScanIn& in, const SeqScanFwd& b, int dtype,
                               int delta_dtype, hipStream_t s);
hipError_t launch_seq_scan_bwd(const SeqScanGeom& g, const SeqScanIn& in, const SeqScanBwd& b, int dtype,
                               int delta_dtype, hipStream_t s);
hipError_t launch_seq_scan_step(const SeqScanGeom& g, const SeqScanIn& in, float* states, void* y, int dtype,
                                int delta_dtype, hipStream_t s);

struct SeqConvGeom {
  SeqGeom q;
  int64_t xs, ys;
  int32_t kc;
  int32_t fwd_pos, bwd_pos;  // 4 or 8, 8 or 16: positions of a wave
  int32_t w_vec;  // taps and biases are read 16 bytes at a time
};
// A wave takes `pos` positions, a workgroup's chunk is four such runs: short
// ones while the card is not full, longer ones read fewer rows twice.
constexpr SeqCut conv_cut(int pos) {
  return {4u * pos, 1u << 31, pos == 4 ? 3u : (pos == 8 ? 4u : 5u)};
}
inline int64_t seq_conv_partial_floats(const SeqConvGeom& g) {
  return chunk_slots(g.q, conv_cut(g.bwd_pos)) * g.q.D * (g.kc + 1);
}
hipError_t launch_seq_conv_fwd(const SeqConvGeom& g, const void* x, const float* w, const float* b, const void* c0,
                               void* c1, void* y, int dtype, hipStream_t s);
hipError_t launch_seq_conv_bwd(const SeqConvGeom& g, const void* x, const float* w, const float* b, const void* c0,
                               const void* dy, const void* dc1, void* dx, float* dw, float* db, void* dc0,
                               float* part, int dtype, hipStream_t s);
hipError_t launch_seq_conv_step(const SeqConvGeom& g, const void* x, const float* w, const float* b, void* states,
                                void* y, int dtype, hipStream_t s);

}  // namespace mvm
