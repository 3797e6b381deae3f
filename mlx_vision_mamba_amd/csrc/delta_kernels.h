// The gated delta rule: parameter blocks and launch entry points
// (delta_prep.hip, delta_fwd.hip, delta_bwd.hip, delta_step.hip), used by the
// C ABI (delta_capi.hip).
#pragma once

#include "seq_kernels.h"

namespace mvm {

constexpr int kDeltaChunk = 64;   // tokens of a chunk
constexpr int64_t kDeltaMaxStride = 1 << 25;  // of v's and o's rows: 12 of them and a row are within 2^31 bytes
inline uint32_t delta_col_blocks(int cols, int waves) {
  return static_cast<uint32_t>((cols + 16 * waves - 1) / (16 * waves));
}

struct DeltaGeom {
  SeqGeom q;
  int32_t HK, HV, group;          // group = HV / HK
  int32_t DK, DV;
  int64_t qs, qh, ks, kh, vs, vh, gs, bs;
  float scale;
  int32_t l2;
  int32_t beta_f32;               // beta is float32, else of the activations' type
  int32_t vec;                    // rows of q, k, v, o (and of the gradients) are accessed 16 bytes at a time
  SeqCut cut;                     // chunks
  SeqCut part;                    // parts of the time axis, whole chunks
  int32_t parts;                  // 1: a sequence is one part
  int32_t waves;                  // of a workgroup of the passes along time, 16 columns of the state each
};

struct DeltaIn {
  const void* q;
  const void* k;
  const void* v;
  const float* g;
  const void* beta;
};

// States and rows that one pass leaves for another lie as the matrix units' result tiles, 16 x 16 values (256
// floats, 16 bytes a lane) each, the 16 columns' tiles one after the other.
inline int64_t delta_col_tiles(const DeltaGeom& g) { return (g.DV + 15) / 16; }

// What the chunks' own products leave for the passes along time, for every
// chunk slot and value head: the fragments of two 64 x 64 triangles as the
// matrix units take them, and four scalars for each token.  A training forward
// leaves all of it to the backward.
struct DeltaWork {
  void* tri;       // (slots, HV, 2, parts, 6, 64) 16-byte fragments
  float* dec;      // (slots, HV, 4, 64)
  float* gam;      // (slots, HV): the decay over the chunk
  float* trans;    // (part slots, HV, DKP / 16, DKP / 16 tiles) transitions of the parts, or null
  float* carry;    // (part slots, HV, column tiles, DKP / 16 tiles): end states of the parts from zero, then their
                   // initial states
};

struct DeltaBwd {
  const float* s0;   // (slots, HV, column tiles, DKP / 16 tiles): initial states of the chunks
  const float* vt;   // (slots, HV, column tiles, 4 tiles): d_t
  const void* d_o;
  const float* dh1;  // or null
  float* dh0;        // or null
  float* x;          // as vt: dv / beta
  float* dend;       // as s0: gradients of the chunks' final states
  void* dq;
  void* dk;
  void* dv;
  float* dg;
  void* dbeta;
};

// 16-byte fragments of one triangle of a chunk slot and value head
constexpr int kTriFrags = 6;                   // of 16 rows and 32 columns that are not all zero
constexpr int kTriParts = 3;
constexpr int kTriFragments = 2 * kTriFrags * kTriParts * 64;
constexpr int64_t kTriBytes = int64_t{kTriFragments} * 16;
// where lane 0's fragment f of part p of the which-th triangle lies: the second triangle last, so that a pass that
// does without it reads one run
constexpr int tri_index(int which, int p, int f) { return ((which * kTriParts + p) * kTriFrags + f) * 64; }

inline int delta_dkp(int dk) { return dk <= 32 ? 32 : (dk <= 64 ? 64 : 128); }

// joins the parts, from the initial states (REV: from the gradients of the final ones)
template <bool REV>
hipError_t launch_delta_carry(const DeltaGeom& g, const DeltaWork& w, const float* enter, hipStream_t s);
hipError_t launch_delta_prep(const DeltaGeom& g, const DeltaIn& in, const DeltaWork& w, int dtype, hipStream_t s);
hipError_t launch_delta_fwd(const DeltaGeom& g, const DeltaIn& in, const DeltaWork& w, const float* h0, float* h1,
                            void* o, float* s0, float* vt, int dtype, hipStream_t s);
hipError_t launch_delta_bwd(const DeltaGeom& g, const DeltaIn& in, const DeltaWork& w, const DeltaBwd& b, int dtype,
                            hipStream_t s);
hipError_t launch_delta_step(const DeltaGeom& g, const DeltaIn& in, float* states, void* o, int dtype, hipStream_t s);

}  // namespace mvm
