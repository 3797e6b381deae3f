// Device helpers of the gated delta rule's chunk kernels.
//
// Products run on the bf16 matrix units (16x16x32).  A float32 operand is the
// sum of three bf16 values, exactly (hi = bf16(x), mid = bf16(x - hi), lo = x -
// hi - mid: the method of gemm.hip), a bfloat16 one is its own only part.  The
// products of parts whose orders add up to less than 3 are kept: what is left
// out is below 2^-24 of a product.  So an operand of bfloat16 activations
// costs three instructions against a float32 state, one of float32 activations
// six.
//
// Lane layout (l = lane, m = l % 16, g = l / 16):
//   result   lane holds column m, rows 4g .. 4g + 3 of a 16 x 16 tile;
//   operands lane holds row (A) or column (B) m, 8 values of the summed index.
// The order of the summed index is free as long as both operands agree.  Here
// slot e of lane group g stands for 4g + e (e < 4) and 16 + 4g + e - 4 of the
// 32: then two result tiles one above the other are, converted, the next
// product's B operand, and the recurrence's chain of products never leaves the
// registers.  A operands come from LDS: rows as they lie, or columns by the
// transposing reads.
#pragma once

#include "delta_kernels.h"
#include "mvm_delta.h"
#include "mvm_scan.h"
#include "seq_common.h"

namespace mvm {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr int kC = kDeltaChunk;
constexpr float kL2Eps = 1e-6f;
constexpr float kMinLogDecay = -1e4f;

// bf16 parts of an operand of the activations' type
template <typename T>
constexpr int kRawParts = std::is_same_v<T, float> ? 3 : 1;

template <int P>
struct Frag {
  uint4 p[P];
};

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const f32x2 v = {a, b};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
}

// the P leading bf16 parts of 8 values
template <int P>
__device__ __forceinline__ Frag<P> split8(float v0, float v1, float v2, float v3, float v4, float v5, float v6,
                                          float v7) {
  float v[8] = {v0, v1, v2, v3, v4, v5, v6, v7};
  Frag<P> f;
#pragma unroll
  for (int q = 0; q < P; ++q) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
      if (q + 1 < P) {
        v[2 * i] -= __uint_as_float(w[i] << 16);
        v[2 * i + 1] -= __uint_as_float(w[i] & 0xffff0000u);
      }
    }
    f.p[q] = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return f;
}
template <int P>
__device__ __forceinline__ Frag<P> split_tiles(const f32x4& a, const f32x4& b) {
  return split8<P>(a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]);
}

// c + a b: the products of parts whose orders add up to less than ORD, small ones first
template <int ORD, int PA, int PB>
__device__ __forceinline__ f32x4 mma(const Frag<PA>& a, const Frag<PB>& b, f32x4 c) {
#pragma unroll
  for (int o = ORD - 1; o >= 0; --o)
#pragma unroll
    for (int i = 0; i < PA; ++i)
      if (o - i >= 0 && o - i < PB)
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a.p[i]),
                                                    __builtin_bit_cast(bf16x8, b.p[o - i]), c, 0, 0, 0);
  return c;
}

// The same for N tiles with operands of their own and one B: the products of one part after the other, so that
// neighbours in the instruction stream do not wait for each other's sums
template <int ORD, int PA, int PB, int N>
__device__ __forceinline__ void mma_n(const Frag<PA> (&a)[N], const Frag<PB>& b, f32x4* c) {
#pragma unroll
  for (int o = ORD - 1; o >= 0; --o)
#pragma unroll
    for (int i = 0; i < PA; ++i)
      if (o - i >= 0 && o - i < PB)
#pragma unroll
        for (int n = 0; n < N; ++n)
          c[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a[n].p[i]),
                                                         __builtin_bit_cast(bf16x8, b.p[o - i]), c[n], 0, 0, 0);
}

// The same for one A and B operands of their own: a result tile's operand of the chain is, as it is, the A operand
// of its transpose
template <int ORD, int PA, int PB, int N>
__device__ __forceinline__ void mma_t(const Frag<PA>& a, const Frag<PB> (&b)[N], f32x4* c) {
#pragma unroll
  for (int o = ORD - 1; o >= 0; --o)
#pragma unroll
    for (int i = 0; i < PA; ++i)
      if (o - i >= 0 && o - i < PB)
#pragma unroll
        for (int n = 0; n < N; ++n)
          c[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a.p[i]),
                                                         __builtin_bit_cast(bf16x8, b[n].p[o - i]), c[n], 0, 0, 0);
}

// A tile of ROWS rows of COLS values in LDS, one plane for each part.  Rows lie 16 values past a multiple of 64
// banks apart or an odd multiple of 16 values, and in every other eight of them the 16-byte words of a pair trade
// places: then neither 16 lanes' rows, nor the 8 rows by 16 columns of a transposing read, share a bank.
template <int ROWS, int COLS, int P>
struct Tile {
  static constexpr int LD = COLS + 16;
  static constexpr int kPlane = ROWS * LD;
  uint16_t v[P * kPlane];

  __device__ __forceinline__ static int at(int row, int col) { return row * LD + (col ^ (row & 8)); }

  // (columns c0, a multiple of 16, and offsets below it apart: an address register and constants)
  // row `row`, summed index 32 ks .. 32 ks + 31 in the chained order
  __device__ __forceinline__ Frag<P> rows(int row, int ks, int grp) const {
    Frag<P> f;
    const uint16_t* at0 = v + row * LD + ((4 * grp) ^ (row & 8)) + 32 * ks;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const uint2 a = *reinterpret_cast<const uint2*>(at0 + p * kPlane);
      const uint2 b = *reinterpret_cast<const uint2*>(at0 + p * kPlane + 16);
      f.p[p] = make_uint4(a.x, a.y, b.x, b.y);
    }
    return f;
  }
  // column c0 + m of the tile, summed index rows r0 .. r0 + 31 in the chained order (r0 includes 4g).  The
  // transposing read hands lane i of 16 the i % 4-th values of the 8-byte words at the addresses of lanes
  // i / 4, i / 4 + 4, + 8, + 12.
  __device__ __forceinline__ Frag<P> cols(int c0, int r0, int m) const {
    Frag<P> f;
    const int row = r0 + (m >> 2);
    const uint16_t* at0 = v + row * LD + ((4 * (m & 3)) ^ (row & 8)) + c0;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const uint16_t* x = at0 + p * kPlane;
      const uint2 a = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)x));
      const uint2 b = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(x + 16 * LD)));
      f.p[p] = make_uint4(a.x, a.y, b.x, b.y);
    }
    return f;
  }
  // rows r0 .. r0 + 3 of column c0 + m (r0 includes 4g), as a result tile holds them
  __device__ __forceinline__ f32x4 col4(int c0, int r0, int m) const {
    static_assert(P == 1, "one part");
    const int row = r0 + (m >> 2);
    const uint16_t* at0 = v + row * LD + ((4 * (m & 3)) ^ (row & 8)) + c0;
    const uint2 a = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at0));
    return {__uint_as_float(a.x << 16), __uint_as_float(a.x & 0xffff0000u), __uint_as_float(a.y << 16),
            __uint_as_float(a.y & 0xffff0000u)};
  }
  // four values of a row
  __device__ __forceinline__ void put4(int row, int col, const f32x4& x) {
    float a = x[0], b = x[1], c = x[2], d = x[3];
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const uint2 w = make_uint2(pack_bf16(a, b), pack_bf16(c, d));
      *reinterpret_cast<uint2*>(v + p * kPlane + at(row, col)) = w;
      a -= __uint_as_float(w.x << 16);
      b -= __uint_as_float(w.x & 0xffff0000u);
      c -= __uint_as_float(w.y << 16);
      d -= __uint_as_float(w.y & 0xffff0000u);
    }
  }
  __device__ __forceinline__ void put(int row, int col, const Frag<P>& f) {
#pragma unroll
    for (int p = 0; p < P; ++p) *reinterpret_cast<uint4*>(v + p * kPlane + at(row, col)) = f.p[p];
  }
  // values col .. col + 3 of a row (col a multiple of 4)
  __device__ __forceinline__ f32x4 get4(int row, int col) const {
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int p = P - 1; p >= 0; --p) {
      const uint2 a = *reinterpret_cast<const uint2*>(v + p * kPlane + at(row, col));
      s[0] += __uint_as_float(a.x << 16);
      s[1] += __uint_as_float(a.x & 0xffff0000u);
      s[2] += __uint_as_float(a.y << 16);
      s[3] += __uint_as_float(a.y & 0xffff0000u);
    }
    return s;
  }
};

// 8 values of a row of n from column c, zero past it
template <typename T>
__device__ __forceinline__ void load8f(float (&v)[8], const T* p, int c, int n, bool vec) {
  if (vec && c + 8 <= n) {
    if constexpr (std::is_same_v<T, float>) {
      const float4 a = *reinterpret_cast<const float4*>(p + c), b = *reinterpret_cast<const float4*>(p + c + 4);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      const uint4 w = *reinterpret_cast<const uint4*>(p + c);
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(u[i] << 16);
        v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < n ? to_f32(p[c + i]) : 0.f;
  }
}
template <int P>
__device__ __forceinline__ Frag<P> split8(const float (&v)[8]) {
  return split8<P>(v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]);
}
// the same as the parts of an operand: bfloat16 as it is
template <typename T>
__device__ __forceinline__ Frag<kRawParts<T>> load8(const T* p, int c, int n, bool vec) {
  if constexpr (std::is_same_v<T, float>) {
    float v[8];
    load8f(v, p, c, n, vec);
    return split8<3>(v);
  } else {
    Frag<1> f;
    if (vec && c + 8 <= n) {
      f.p[0] = *reinterpret_cast<const uint4*>(p + c);
    } else {
      uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c + i < n) w[i >> 1] |= static_cast<uint32_t>(p[c + i].bits) << (16 * (i & 1));
      f.p[0] = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return f;
  }
}

// 8 values of a row as they lie in memory
template <typename T>
struct Raw8 {
  uint4 v[std::is_same_v<T, float> ? 2 : 1];
};
// The 64 rows of a chunk's q or k, dk values each, on their way from global memory (load) into LDS (put), all
// loads in flight together; rows from n on and columns from dk on are zero.
template <typename T, int DKP, int NT>
struct StageRows {
  static constexpr int kPer = DKP / 8, kItems = (kC * kPer + NT - 1) / NT;
  Raw8<T> r[kItems];

  // (threads past the last item take part in the loads)
  __device__ __forceinline__ static int row(int i, int tid) { return (tid + NT * i) / kPer % kC; }
  __device__ __forceinline__ static int col(int i, int tid) { return (tid + NT * i) % kPer * 8; }

  template <bool VEC>
  __device__ __forceinline__ void load(const T* p, int64_t stride, int n, int dk, int tid) {
    if constexpr (VEC) {  // (dk is a multiple of a 16-byte access)
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        const int c = col(i, tid), rw = row(i, tid);
        const T* at = p + (rw < n ? rw : 0) * stride;
        constexpr int V = 16 / sizeof(T);
#pragma unroll
        for (int j = 0; j < 8 / V; ++j) {
          const uint4 x = *reinterpret_cast<const uint4*>(at + (c + V * j < dk ? c + V * j : 0));
          r[i].v[j] = x;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        const int c = col(i, tid), rw = row(i, tid);
        const T* at = p + (rw < n ? rw : 0) * stride;
        uint32_t w[8 * sizeof(T) / 4];
#pragma unroll
        for (int j = 0; j < static_cast<int>(8 * sizeof(T) / 4); ++j) {
          if constexpr (std::is_same_v<T, float>) {
            w[j] = __float_as_uint(at[c + j < dk ? c + j : 0]);
          } else {
            const uint32_t lo = at[c + 2 * j < dk ? c + 2 * j : 0].bits, hi = at[c + 2 * j + 1 < dk ? c + 2 * j + 1 : 0].bits;
            w[j] = (c + 2 * j < dk ? lo : 0u) | (c + 2 * j + 1 < dk ? hi << 16 : 0u);
          }
        }
#pragma unroll
        for (int j = 0; j < static_cast<int>(sizeof(T) / 2); ++j)
          r[i].v[j] = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
      }
    }
  }
  // the parts of item i
  __device__ __forceinline__ Frag<kRawParts<T>> parts(int i, int n, int dk, int tid) const {
    const bool ok = row(i, tid) < n;
    const int c = col(i, tid);
    if constexpr (std::is_same_v<T, float>) {
      float v[8];
      const uint32_t* u = reinterpret_cast<const uint32_t*>(r[i].v);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = ok && c + j < dk ? __uint_as_float(u[j]) : 0.f;
      return split8<3>(v);
    } else {
      // (columns past dk: whole accesses, or zero already)
      Frag<1> f;
      f.p[0] = ok && c < dk ? r[i].v[0] : make_uint4(0u, 0u, 0u, 0u);
      return f;
    }
  }
  __device__ __forceinline__ void put(Tile<kC, DKP, kRawParts<T>>& tile, int n, int dk, int tid) const {
#pragma unroll
    for (int i = 0; i < kItems; ++i)
      if (NT * (i + 1) <= kC * kPer || tid + NT * i < kC * kPer) tile.put(row(i, tid), col(i, tid), parts(i, n, dk, tid));
  }
};

// One column a lane of a chunk's n rows, as result tiles hold them (element 4 rt + r: row 16 rt + 4g + r).  `at` is
// the wave's first column in the chunk's first row, `stride` the rows' (at most kDeltaMaxStride: a scalar base for
// each row, and one 32-bit offset a lane).  Lanes past the last row read an earlier one.
template <typename T>
__device__ __forceinline__ uint32_t lane_offset(int64_t stride, int m, int grp) {
  return (4u * grp * static_cast<uint32_t>(stride) + m) * static_cast<uint32_t>(sizeof(T));
}
template <typename T>
struct Cols {
  T r[16];
  __device__ __forceinline__ void load(const T* at, int64_t stride, int m, int grp, int n, bool live) {
    const uint32_t off = live ? lane_offset<T>(stride, m, grp) : 0u;
    if (n == kC) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        r[i] = *reinterpret_cast<const T*>(reinterpret_cast<const char*>(at) + off);
        at += (i & 3) == 3 ? 13 * stride : stride;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int u = 16 * (i >> 2) + (i & 3);
        r[i] = *reinterpret_cast<const T*>(reinterpret_cast<const char*>(at + (u < n ? u : 0) * stride) +
                                           (u + 4 * grp < n ? off : 0u));
      }
    }
  }
  __device__ __forceinline__ f32x4 tile(int rt, int grp, int n, bool live) const {
    f32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = live && 16 * rt + 4 * grp + i < n ? to_f32(r[4 * rt + i]) : 0.f;
    return v;
  }
};
// Four values of a row in their type
template <typename T>
struct Quad {
  uint32_t w[sizeof(T)];
  __device__ __forceinline__ void set(const f32x4& v) {
    if constexpr (std::is_same_v<T, float>) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(v[i]);
    } else {
      w[0] = pack_bf16(v[0], v[1]);
      w[1] = pack_bf16(v[2], v[3]);
    }
  }
  // values c .. c + 3 of a row of n
  __device__ __forceinline__ void store(T* p, int c, int n, bool vec) const {
    if (vec) {  // (n is a multiple of 4)
      if (c < n) {
        if constexpr (std::is_same_v<T, float>)
          *reinterpret_cast<u32x4*>(p + c) = u32x4{w[0], w[1], w[2], w[3]};
        else
          *reinterpret_cast<u32x2*>(p + c) = u32x2{w[0], w[1]};
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (c + i < n) {
          if constexpr (std::is_same_v<T, float>)
            p[c + i] = __uint_as_float(w[i]);
          else
            p[c + i] = T{static_cast<uint16_t>(i & 1 ? w[i / 2] >> 16 : w[i / 2])};
        }
    }
  }
};
template <typename T>
__device__ __forceinline__ f32x4 load4(const T* p, int c, int n, bool vec) {
  f32x4 v;
  if (vec) {
    const T* at = p + (c < n ? c : 0);
    if constexpr (std::is_same_v<T, float>) {
      v = *reinterpret_cast<const f32x4*>(at);
    } else {
      const u32x2 a = *reinterpret_cast<const u32x2*>(at);
      v = {__uint_as_float(a[0] << 16), __uint_as_float(a[0] & 0xffff0000u), __uint_as_float(a[1] << 16),
           __uint_as_float(a[1] & 0xffff0000u)};
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = c < n ? v[i] : 0.f;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = c + i < n ? to_f32(p[c + i]) : 0.f;
  }
  return v;
}

// 1 where sequence i starts from the state in row `row` of `states`, else 0, for its users to multiply by.  (As `states
// && row >= 0 && (!fresh || !fresh[i]) ? rows : 0` this toolchain leaves the copy of `rows` out of the edge behind the
// load: a zero from before the conditions stays, and with flags no state is read.  A value that is set on both of that
// condition's edges, as the mask in delta_step.hip, is not touched by it.)
__device__ __forceinline__ int32_t seq_starts(const SeqGeom& g, int32_t i, int32_t row, const float* states) {
  const int32_t fresh = g.fresh != nullptr ? g.fresh[i] : 0;
  return (states != nullptr) & (row >= 0) & (__builtin_amdgcn_readfirstlane(fresh) == 0);
}

// The rows dk of a state's 16 columns: `at` is the wave's first column of row 0.  Rows are `ld` values apart.
template <int KT>
__device__ __forceinline__ void load_state(f32x4 (&S)[KT], const float* at, int ld, int rows, int m, int grp, bool live) {
  const uint32_t off = live ? (4u * grp * static_cast<uint32_t>(ld) + m) * 4u : 0u;
#pragma unroll
  for (int t = 0; t < KT; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const bool ok = live && 16 * t + 4 * grp + r < rows;
      S[t][r] = ok ? *reinterpret_cast<const float*>(reinterpret_cast<const char*>(at + (16 * t + r) * ld) + off) : 0.f;
    }
}
template <int KT>
__device__ __forceinline__ void store_state(float* at, int ld, int rows, const f32x4 (&S)[KT], int m, int grp, bool live) {
  if (!live) return;
  const uint32_t off = (4u * grp * static_cast<uint32_t>(ld) + m) * 4u;
#pragma unroll
  for (int t = 0; t < KT; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (rows == 16 * KT || 16 * t + 4 * grp + r < rows)
        *reinterpret_cast<float*>(reinterpret_cast<char*>(at + (16 * t + r) * ld) + off) = S[t][r];
}

// One row's operand: 8 values from column c on, zero past dk (or where !ok), as parts
template <typename T>
__device__ __forceinline__ Frag<kRawParts<T>> row_frag(const T* p, int c, int dk, bool vec, bool ok) {
  return load8<T>(p, c, ok ? dk : 0, vec);
}

// Number of the fragment of 16 rows (tile rt) and 32 columns (ks) of a lower triangle of 64 x 64, or -1 where all of
// it is zero.  Within a fragment the four lanes of a row lie together: so neither a row's readers nor those of a
// column share a bank.
constexpr int tri_frag(int rt, int ks) { return rt < 2 ? (ks == 0 ? rt : -1) : 2 * rt - 2 + ks; }
__device__ __forceinline__ int tri_lane(int m, int grp) { return 4 * m + grp; }

// Result tiles in memory as the lanes hold them, 16 bytes a lane: N tiles of one column block
template <int N>
__device__ __forceinline__ void store_tiles(float* at, const f32x4 (&v)[N], int lane) {
#pragma unroll
  for (int i = 0; i < N; ++i) reinterpret_cast<f32x4*>(at)[64 * i + lane] = v[i];
}

// A chunk's two triangles on their way into LDS: three parts of the first, PP of the second
template <int PP, int NT>
struct StageTri {
  static constexpr int kCount = tri_index(1, PP, 0), kItems = (kCount + NT - 1) / NT;
  u32x4 r[kItems];
  // (the items from a to b of 4)
  __device__ __forceinline__ void load(const uint4* tri, int tid, int a = 0, int b = 4) {
    const u32x4* at = reinterpret_cast<const u32x4*>(tri);
#pragma unroll
    for (int i = 0; i < kItems; ++i)
      if (i >= kItems * a / 4 && i < kItems * b / 4) r[i] = at[NT * (i + 1) <= kCount || tid + NT * i < kCount ? tid + NT * i : 0];
  }
  __device__ __forceinline__ void put(uint4* lds, int tid) const {
#pragma unroll
    for (int i = 0; i < kItems; ++i)
      if (NT * (i + 1) <= kCount || tid + NT * i < kCount) reinterpret_cast<u32x4*>(lds)[tid + NT * i] = r[i];
  }
};
// A triangle's operands for row tiles RT0 .. RT0 + N - 1, summed index 32 ks .. 32 ks + 31
template <int RT0, int N, int P>
__device__ __forceinline__ void tri_tiles(Frag<P> (&f)[N], const uint4* lds, int which, int ks, int m, int grp) {
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int q = 0; q < P; ++q) f[i].p[q] = lds[tri_index(which, q, tri_frag(RT0 + i, ks)) + tri_lane(m, grp)];
}
// the same of its transpose, whose summed index are the triangle's rows
template <int RT0, int N, int P>
__device__ __forceinline__ void tri_tiles_t(Frag<P> (&f)[N], const uint4* lds, int which, int ks, int m, int grp) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int jt = RT0 + i;
#pragma unroll
    for (int q = 0; q < P; ++q) {
      // 4 columns of row 32 ks (+ 16) + 4g + m / 4
      const uint2* at = reinterpret_cast<const uint2*>(lds + tri_lane(4 * grp + (m >> 2), m & 3)) + (jt & 1);
      const uint2 a = __builtin_bit_cast(
          uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + 2 * tri_index(which, q, tri_frag(2 * ks, jt / 2)))));
      const uint2 b = __builtin_bit_cast(
          uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + 2 * tri_index(which, q, tri_frag(2 * ks + 1, jt / 2)))));
      f[i].p[q] = make_uint4(a.x, a.y, b.x, b.y);
    }
  }
}

// Sum over the 4 lane groups of the lanes with the same m
__device__ __forceinline__ float sum_g(float x) {
  x += __shfl_xor(x, 16);
  x += __shfl_xor(x, 32);
  return x;
}

// Inclusive sums over a wave's lanes: within rows of 16 by shifts, then the rows' last lanes into the rows behind
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_part(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(u), CTRL, ROWS, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(u >> 32), CTRL, ROWS, 0xf, false);
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
__device__ __forceinline__ double wave_scan(double x) {
  x += dpp_part<0x111, 0xf>(x);
  x += dpp_part<0x112, 0xf>(x);
  x += dpp_part<0x114, 0xf>(x);
  x += dpp_part<0x118, 0xf>(x);
  x += dpp_part<0x142, 0xa>(x);
  x += dpp_part<0x143, 0xc>(x);
  return x;
}

// Lane = token of a chunk of n: the log decay summed from the chunk's start up to it, in 64 bits: the decay between
// two tokens is the exponential of a difference, which 32 bits would leave with the rounding of the sums.
__device__ __forceinline__ double log_decay(const DeltaGeom& g, const float* gp, int t0, int n, int h, int lane) {
  double s = 0.0;
  if (lane < n) {
    const float x = gp[(t0 + static_cast<int64_t>(lane)) * g.gs + h];
    s = x < kMinLogDecay ? kMinLogDecay : x;  // (NaN stays)
  }
  return wave_scan(s);
}
// exp of it: the whole part of the binary exponent is set apart in 64 bits, so that what the transcendental unit gets
// has the digits of a number below 1 (rounded whole, exp(-16) would be off by 7e-7 of itself)
__device__ __forceinline__ float exp_diff(double x) {
  const double t = x * 1.4426950408889634;
  const float n = rintf(__builtin_amdgcn_fmed3f(static_cast<float>(t), -1000.f, 1000.f));
  return ldexpf(fast_exp2(static_cast<float>(t - n)), static_cast<int>(n));
}

template <typename T>
__device__ __forceinline__ float load_beta(const DeltaGeom& g, const void* beta, int64_t t, int h) {
  return g.beta_f32 ? static_cast<const float*>(beta)[t * g.bs + h] : to_f32(static_cast<const T*>(beta)[t * g.bs + h]);
}

// The workgroup's item (a slot and value head) and column block.  Blocks are dealt to the 8 XCDs in turn: the column
// blocks of an item come 8 apart, so that its rows are read into one L2.
struct DeltaPos {
  int32_t slot, h, cb;
  bool ok;
};
__device__ __forceinline__ DeltaPos delta_pos(uint32_t ncb, uint32_t nslots, uint32_t heads) {
  const uint32_t b = blockIdx.x, r = b / (8 * ncb), in = b - r * 8 * ncb;
  const uint32_t item = r * 8 + in % 8;
  const uint32_t slot = item / heads;
  return {static_cast<int32_t>(slot), static_cast<int32_t>(item - slot * heads), static_cast<int32_t>(in / 8), slot < nslots};
}
inline int64_t delta_blocks(int64_t ncb, int64_t nslots, int64_t heads) { return (nslots * heads + 7) / 8 * 8 * ncb; }

// The tokens' scalars of a chunk, as delta_prep.hip leaves them: four rows of 64
enum DecRow { kDecKey, kDecUp, kDecOut, kDecBeta };
__device__ __forceinline__ f32x4 dec_at(const float (*dec)[kC], DecRow which, int rt, int grp) {
  return *reinterpret_cast<const f32x4*>(&dec[which][16 * rt + 4 * grp]);
}

// Instructions stay on their side: without it the reads of all operands are moved to the front, and their
// registers spill.  Each phase reads the next one's operands.
__device__ __forceinline__ void phase() { __builtin_amdgcn_sched_barrier(0); }
__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6)); }

// f(type of the activations, std::integral_constant<int, padded dk>)
template <typename F>
hipError_t delta_dispatch(int dtype, int dk, F&& f) {
  const auto by_dk = [&](auto t) {
    switch (delta_dkp(dk)) {
      case 32: return f(t, std::integral_constant<int, 32>{});
      case 64: return f(t, std::integral_constant<int, 64>{});
      default: return f(t, std::integral_constant<int, 128>{});
    }
  };
  return dtype == MVM_F32 ? by_dk(float{}) : by_dk(bf16_t{});
}

}  // namespace mvm
