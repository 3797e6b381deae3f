// Device helpers of the packed selective scan's passes (seq_scan.hip forward,
// seq_scan_bwd.hip backward).
#pragma once

#include <algorithm>

#include "mvm_scan.h"
#include "seq_common.h"

namespace mvm {

constexpr int kWave = 64;
constexpr float kMaxA2 = 3.4028234e38f;
constexpr float kLog2eLow = 1.925963e-8f;  // log2(e) - kLog2e

// COUNT (a multiple of 4) values of row `row` of an array of N columns from
// column n0 on, zero past N.  vec: rows start on 16 bytes; a lane's own row
// then takes a quarter of the accesses, each of which touches 64 lines.
template <int COUNT>
__device__ __forceinline__ void load_states(float (&h)[COUNT], const float* p, int64_t row, int n0, int N, int vec) {
  const float* at = p + row * N;
  if (vec) {
    at = opaque(at);  // (else the compiler joins the branches, into single loads)
#pragma unroll
    for (int q = 0; q < COUNT / 4; ++q) {
      const Pack<float, 4> v = load_pack<float, 4>(at + state_col(n0 + 4 * q, N));
#pragma unroll
      for (int j = 0; j < 4; ++j) h[4 * q + j] = v.v[j];
    }
  } else {
#pragma unroll
    for (int n = 0; n < COUNT; ++n) h[n] = at[state_col(n0 + n, N)];
  }
#pragma unroll
  for (int n = 0; n < COUNT; ++n) h[n] = n0 + n < N ? h[n] : 0.f;
}
template <int COUNT>
__device__ __forceinline__ void store_states(const float (&h)[COUNT], float* p, int64_t row, int n0, int N, int vec) {
  float* at = p + row * N + n0;
  if (vec) {
#pragma unroll
    for (int q = 0; q < COUNT / 4; ++q)
      if (n0 + 4 * q < N)
        store_pack(at + 4 * q, Pack<float, 4>{h[4 * q], h[4 * q + 1], h[4 * q + 2], h[4 * q + 3]});
  } else {
#pragma unroll
    for (int n = 0; n < COUNT; ++n)
      if (n0 + n < N) at[n] = h[n];
  }
}

// A log2(e) of one channel's states from n0 on, 0 past N.  Kept finite, so
// that a delta of zero always means no decay.  A = -exp(A_log) by the
// exponential unit: the rounding error of A_log log2(e) is put back by its
// first-order term (2 ulp of A; the routine of the maths library costs 20
// instructions a state, as much as 4 tokens of the scan).
template <int COUNT>
__device__ __forceinline__ void load_a2(float (&a)[COUNT], const float* A, int64_t row, int n0, const SeqScanGeom& g) {
  load_states(a, A, row, n0, g.N, g.a_vec);
  if (g.a_log) {
#pragma unroll
    for (int j = 0; j < COUNT; ++j) {
      const float hi = a[j] * kLog2e, lo = fmaf(a[j], kLog2eLow, fmaf(a[j], kLog2e, -hi));
      const float e = fast_exp2(hi);
      a[j] = fabsf(hi) < 126.f ? -fmaf(e * kLn2, lo, e) : -e;  // (infinities and NaN as they come)
    }
  }
#pragma unroll
  for (int j = 0; j < COUNT; ++j) {
    float x = a[j] * kLog2e;
    x = x < -kMaxA2 ? -kMaxA2 : x;
    x = x > kMaxA2 ? kMaxA2 : x;
    a[j] = n0 + j < g.N ? x : 0.f;
  }
}

// What enters chunk nth (in order) of a sequence whose earlier chunks left their
// aggregates in `agg_h`, `agg_s` (DIR 1: slots base, base + 1, ..; -1: base,
// base - 1, ..), folded into h.
template <int DIR, int COUNT>
__device__ __forceinline__ void fold_chunks(float (&h)[COUNT], const float (&a2)[COUNT], const float* agg_h,
                                            const float* agg_s, int64_t base, int32_t nth, int64_t D, int64_t d) {
  constexpr int kBatch = 3;  // chunks whose loads are in flight together
  for (int32_t j0 = 0; j0 < nth; j0 += kBatch) {
    Pack<float, 4> v[kBatch][COUNT / 4];
    float s[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int64_t slot = base + DIR * (j0 + i < nth ? j0 + i : j0);
#pragma unroll
      for (int q = 0; q < COUNT / 4; ++q) v[i][q] = load_pack<float, 4>(agg_h + ((slot * 4 + q) * D + d) * 4);
      s[i] = agg_s[slot * D + d];
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
      if (j0 + i < nth) {
#pragma unroll
        for (int n = 0; n < COUNT; ++n) h[n] = fmaf(fast_exp2(a2[n] * s[i]), h[n], v[i][n >> 2].v[n & 3]);
      }
  }
}
template <int COUNT>
__device__ __forceinline__ void load_agg(float (&h)[COUNT], const float* agg_h, int64_t slot, int64_t D, int64_t d) {
#pragma unroll
  for (int q = 0; q < COUNT / 4; ++q) {
    const Pack<float, 4> v = load_pack<float, 4>(agg_h + ((slot * 4 + q) * D + d) * 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) h[4 * q + j] = v.v[j];
  }
}
// (a channel's values of a (row, 4, D, 4) array)
template <int COUNT>
__device__ __forceinline__ void store_agg(const float (&h)[COUNT], float* agg_h, int64_t slot, int64_t D, int64_t d) {
#pragma unroll
  for (int q = 0; q < COUNT / 4; ++q)
    store_pack(agg_h + ((slot * 4 + q) * D + d) * 4, Pack<float, 4>{h[4 * q], h[4 * q + 1], h[4 * q + 2], h[4 * q + 3]});
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

// x is computed here: the compiler would move a sum that only a branch uses
// into the branch, and keep all its terms in registers until then
__device__ __forceinline__ void pin(float& x) { asm volatile("" : "+v"(x)); }
// B and C of a tile on their way: lane l asks for states 4 (l & 3) .. + 3 of
// row l >> 3, of B or (l & 4) of C; rows past the chunk are zero.
template <typename T>
struct BcTile {
  T raw[4];
  __device__ __forceinline__ void fetch(const T* B, const T* C, int64_t st, int32_t t, int32_t t1, int N,
                                        uint32_t lane) {
    const int32_t i = t + static_cast<int32_t>(lane >> 3);
    const T* row = ((lane & 4) ? C : B) + (i < t1 ? i : t1 - 1) * st;
    const int n0 = 4 * (lane & 3);
#pragma unroll
    for (int j = 0; j < 4; ++j) raw[j] = row[state_col(n0 + j, N)];
  }
  __device__ __forceinline__ float value(int j, int N, uint32_t lane, int32_t t, int32_t t1) const {
    return static_cast<int>(4 * (lane & 3)) + j < N && t + static_cast<int32_t>(lane >> 3) < t1 ? to_f32(raw[j]) : 0.f;
  }
};
// orders a wave's own LDS accesses for the compiler (the unit keeps them in order)
__device__ __forceinline__ void lds_order() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

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
  // (or another address)
  __device__ __forceinline__ void next_or(bool go, uint64_t past) {
    at = go ? at + st : past;
    asm volatile("" : "+s"(at));
  }
  __device__ __forceinline__ void prev(bool go = true) {
    at -= go ? st : 0u;
    asm volatile("" : "+s"(at));
  }
  // (a 32-bit offset from the scalar address: one instruction, no address arithmetic)
  template <typename T>
  __device__ __forceinline__ T* elem(uint32_t lane) const {
    const uint32_t off = lane * static_cast<uint32_t>(sizeof(T));
    return (T*)((__attribute__((address_space(1))) char*)at + off);
  }
  template <typename T>
  __device__ __forceinline__ T load(uint32_t lane) const {
    return *elem<const T>(lane);
  }
  template <typename T>
  __device__ __forceinline__ void store(uint32_t lane, float v) const {
    *elem<T>(lane) = from_f32<T>(v);
  }
};

// The next kSeqTile rows, from row t on; rows past the chunk read its last one.
template <typename T>
__device__ __forceinline__ void load_next(T (&v)[kSeqTile], RowPtr& p, int32_t t, int32_t t1, uint32_t lane) {
  if (t + kSeqTile <= t1) {
#pragma unroll
    for (int i = 0; i < kSeqTile; ++i) {
      v[i] = p.load<T>(lane);
      p.next();
    }
  } else {
#pragma unroll
    for (int i = 0; i < kSeqTile; ++i) {
      v[i] = p.load<T>(lane);
      p.next(t + i + 1 < t1);
    }
  }
}
// The kSeqTile rows from row t on, last one first: p is at row t + 7, or at
// the chunk's last, and comes to rest at row t - 1.
template <typename T>
__device__ __forceinline__ void load_prev(T (&v)[kSeqTile], RowPtr& p, int32_t t, int32_t t1, uint32_t lane) {
  if (t + kSeqTile <= t1) {
#pragma unroll
    for (int i = kSeqTile - 1; i >= 0; --i) {
      v[i] = p.load<T>(lane);
      p.prev();
    }
  } else {
#pragma unroll
    for (int i = kSeqTile - 1; i >= 0; --i) {
      v[i] = p.load<T>(lane);
      p.prev(t + i < t1);
    }
  }
}
// The first `rows` of the next kSeqTile rows.
template <typename T>
__device__ __forceinline__ void store_next(RowPtr p, int32_t rows, uint32_t lane, const float (&v)[kSeqTile]) {
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

// B and C of positions past a chunk's end: a row of zeros at the front of the
// kernel's argument.  (What enters there is multiplied by a delta of zero, and
// infinities of the chunk's last row would make NaN of it.)
constexpr int kZeroRow = 16;
__device__ __forceinline__ uint64_t zero_row() { return (uint64_t)__builtin_amdgcn_kernarg_segment_ptr(); }

// f<T, DT>(): T the activations' type, DT delta's
template <typename F>
hipError_t by_types(int dtype, int delta_dtype, F&& f) {
  if (dtype == MVM_F32) return f(float{}, float{});
  return delta_dtype == MVM_F32 ? f(bf16_t{}, float{}) : f(bf16_t{}, bf16_t{});
}

inline uint32_t blocks_of(int64_t D) { return static_cast<uint32_t>((D + kWave - 1) / kWave); }
inline dim3 wave_grid(int64_t slots, uint32_t ncb) { return dim3(static_cast<unsigned>((slots * ncb + 3) / 4)); }

// workgroups of 256 over n elements that a kernel walks in steps of the grid
inline dim3 strided_grid(int64_t n) { return dim3(static_cast<unsigned>(std::min<int64_t>((n + 255) / 256, 1 << 20))); }

// Which rows of A and of the states are read 16 bytes at a time.
inline void set_vec(SeqScanGeom& g, const float* A, const float* h0, const float* h1) {
  const auto off = [](const float* p) { return reinterpret_cast<uintptr_t>(p) & 15; };
  g.a_vec = g.N % 4 == 0 && off(A) == 0;
  g.h_vec = g.N % 4 == 0 && (off(h0) | off(h1)) == 0;
}

// B and C as the kernels read them: in place, or (bc not null) from a float32
// copy that is made here.  f(BcRows)
template <typename T>
hipError_t launch_bc(const SeqScanGeom& g, const SeqScanIn& in, float* out, hipStream_t s);
template <typename T, typename F>
hipError_t with_bc(const SeqScanGeom& g, const SeqScanIn& in, float* bc, F&& f, hipStream_t s) {
  if (bc == nullptr) return f(BcRows<T>{static_cast<const T*>(in.Bm), static_cast<const T*>(in.Cm), g.bs});
  const hipError_t e = launch_bc<T>(g, in, bc, s);
  return e != hipSuccess ? e : f(BcRows<float>{bc, bc + 16, 32});
}

// The carry pass over the chunks' aggregates (seq_scan.hip); REV: from the end.
template <bool REV>
hipError_t launch_carry(const SeqScanGeom& g, const float* A, const float* enter, float* agg_h, const float* agg_s,
                        hipStream_t s);

}  // namespace mvm
