// Device helpers of the packed-sequence kernels.
#pragma once

#include "scan_common.h"
#include "seq_kernels.h"

namespace mvm {

typedef __attribute__((address_space(4))) const float const_f32;
typedef __attribute__((address_space(4))) const uint32_t const_u32;
typedef __attribute__((address_space(4))) const uint8_t const_u8;

// First token row of sequence i (i = S: the end of the last one), in [0, T].
// i may differ between lanes.
__device__ __forceinline__ int32_t seq_off(const SeqGeom& g, int32_t i) {
  if (g.off == nullptr) return i * g.L;
  const int32_t v = i == 0 ? 0 : g.off[i];
  return v < 0 ? 0 : (v > g.T ? g.T : v);
}
// the same for a wave-uniform i, by a scalar load
__device__ __forceinline__ int32_t seq_off_u(const SeqGeom& g, int32_t i) {
  if (g.off == nullptr) return i * g.L;
  if (i == 0) return 0;
  const int32_t v = ((const const_i32*)g.off)[i];
  return v < 0 ? 0 : (v > g.T ? g.T : v);
}

// State row of sequence i, or -1.
__device__ __forceinline__ int32_t seq_slot(const SeqGeom& g, int32_t i) {
  const int32_t v = g.slots == nullptr ? i : ((const const_i32*)g.slots)[i];
  return v < 0 || v >= g.M ? -1 : v;
}
__device__ __forceinline__ bool seq_fresh(const SeqGeom& g, int32_t i) {
  return g.fresh != nullptr && g.fresh[i] != 0;
}

// The state rows of sequences i0 .. i0 + R - 1 (past the last one: the last
// one's) and whether they start from zero, all asked for at once.  fresh is read
// from any valid address where there is none: a load in a branch would be
// waited for there.
template <int R>
struct StateRows {
  int32_t row[R];
  uint32_t fresh[R];
  __device__ __forceinline__ void load(const SeqGeom& g, int32_t i0, const void* any) {
    const uint8_t* f = g.fresh != nullptr ? g.fresh : static_cast<const uint8_t*>(any);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      row[r] = i0 + r < g.S ? i0 + r : g.S - 1;
      fresh[r] = f[g.fresh != nullptr ? row[r] : 0];
    }
    if (g.slots != nullptr) {
#pragma unroll
      for (int r = 0; r < R; ++r) row[r] = ((const const_i32*)g.slots)[row[r]];
    }
#pragma unroll
    for (int r = 0; r < R; ++r) row[r] = row[r] < 0 || row[r] >= g.M ? -1 : row[r];
  }
  // (once the loads that are to be in flight beside it have been issued)
  __device__ __forceinline__ void settle(const SeqGeom& g) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      asm volatile("" : "+v"(fresh[r]));
      fresh[r] = g.fresh != nullptr ? fresh[r] : 0u;
    }
  }
};

__device__ __forceinline__ int32_t cut_div(const SeqCut& cut, int32_t n) {
  return static_cast<int32_t>(__umulhi(static_cast<uint32_t>(n), cut.magic) >> cut.shift);
}

// The chunk that a slot stands for: rows [t0, t1) of sequence seq, which
// holds rows [start, end).  t0 < 0: none.  An empty sequence has one chunk,
// with t0 == t1 == start == end.
struct SeqChunk {
  int32_t seq, start, end, t0, t1, slot;
};
__device__ __forceinline__ SeqChunk seq_chunk(const SeqGeom& g, int32_t slot, const SeqCut& cut, int lane) {
  // the last i in [0, S] with offset(i) / len + i <= slot: each round 64 lanes
  // probe the range at even steps
  SeqChunk c;
  c.slot = slot;
  int32_t next;
  if (g.S <= 64) {  // one round, whose lanes hold the bounds too
    const int32_t i = lane + 1, off = seq_off(g, i <= g.S ? i : 0);
    c.seq = __popcll(__ballot(i <= g.S && cut_div(cut, off) + i <= slot));
    c.start = c.seq > 0 ? __builtin_amdgcn_readlane(off, c.seq - 1) : 0;
    next = c.seq < g.S ? __builtin_amdgcn_readlane(off, c.seq) : g.T;
  } else {
    int32_t lo = 0, hi = g.S;
    while (hi > lo) {
      const int32_t step = (hi - lo + 63) / 64;
      const int32_t i = lo + (lane + 1) * step;
      const bool in = i <= hi;
      const bool le = in && cut_div(cut, seq_off(g, in ? i : lo)) + i <= slot;
      const int32_t cnt = __popcll(__ballot(le));
      lo += cnt * step;
      const int32_t last = lo + step - 1;
      hi = hi < last ? hi : last;
    }
    c.seq = __builtin_amdgcn_readfirstlane(lo);
    c.start = seq_off_u(g, c.seq);
    next = c.seq == g.S ? g.T : seq_off_u(g, c.seq + 1);
  }
  c.end = next < c.start ? c.start : next;
  const int32_t nth = slot - cut_div(cut, c.start) - c.seq;
  const int64_t t0 = c.start + static_cast<int64_t>(nth) * cut.len;
  c.t0 = static_cast<int32_t>(t0 < c.end ? t0 : c.end);
  const int64_t t1 = t0 + cut.len;
  c.t1 = static_cast<int32_t>(t1 < c.end ? t1 : c.end);
  // a slot past the sequence's last chunk (or before its first, which only
  // offsets that decrease give)
  if (nth < 0 || (nth > 0 && t0 >= c.end)) c.t0 = c.t1 = -1;
  return c;
}

// the slot of the last chunk of c's sequence
__device__ __forceinline__ int32_t last_slot(const SeqCut& cut, const SeqChunk& c) {
  return cut_div(cut, c.start) + c.seq + (c.end > c.start ? cut_div(cut, c.end - c.start - 1) : 0);
}

// a pointer to global memory that the compiler knows nothing about
template <typename T>
__device__ __forceinline__ T* opaque(T* p) {
  uint64_t v = reinterpret_cast<uint64_t>(p);
  asm volatile("" : "+v"(v));
  return (T*)(__attribute__((address_space(1))) T*)v;
}

// V consecutive values, one access
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
  T v[V];
};
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
  return *reinterpret_cast<const Pack<T, V>*>(p);
}
template <typename T, int V>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, V>& x) {
  *reinterpret_cast<Pack<T, V>*>(p) = x;
}

// Workgroups are numbered with the channel blocks (ncb) innermost, so that
// neighbours read neighbouring columns of the same rows.
struct BlockPos {
  int32_t cb, slot;
};
__device__ __forceinline__ BlockPos block_pos(uint32_t ncb) {
  const uint32_t s = blockIdx.x / ncb;
  return {static_cast<int32_t>(blockIdx.x - s * ncb), static_cast<int32_t>(s)};
}

// Fixed-order float64 sums over the rows of part (nparts, ncols): lane =
// column, the block's 16 waves each add a run of the rows, and wave 0 the 16
// sums in order.  Each batch of loads is in flight together.
template <typename Store>
__device__ __forceinline__ void sum_columns(const float* part, int64_t nparts, int64_t ncols, Store store) {
  __shared__ double sums[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t col = static_cast<int64_t>(blockIdx.x) * 64 + lane;
  const int64_t at = col < ncols ? col : ncols - 1;
  const int64_t per = (nparts + 15) / 16;
  const int64_t q0 = wave * per, q1 = q0 + per < nparts ? q0 + per : nparts;
  constexpr int kBatch = 8;
  double s = 0.0;
  for (int64_t q = q0; q < q1; q += kBatch) {
    float v[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) v[i] = part[(q + i < q1 ? q + i : q0) * ncols + at];
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
      if (q + i < q1) s += v[i];
  }
  sums[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && col < ncols) {
    double t = 0.0;
#pragma unroll
    for (int w = 0; w < 16; ++w) t += sums[w][lane];
    store(col, static_cast<float>(t));
  }
}

}  // namespace mvm
