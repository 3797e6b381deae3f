// Group norm with an activation, channels last (include/mvm_group_norm.h): C
// ABI and kernels.  Memory-bound: x (and z) are read and y is written once, as
// far as a group fits in registers.
//
// Rows (one position a sample: the heads of a mixer): a power of two of lanes
// takes a group, all its values in registers, so that x is read once: mean,
// then variance and what the mean was off by from the registers.  A wave keeps its groups and their weights
// and walks rows; the backward sums the channels' gradients in registers on the
// way and leaves one partial row a workgroup.  16384 rows of 12 gated groups of
// 128 in bfloat16: 33 us forward (151 MB, 4.6 TB/s), 49 backward (252 MB, 5.2).
//
// Tiles (a sample's group of up to 8 16-byte accesses a thread): a workgroup
// holds it, one launch a direction; 32 samples of 196 x 384 in 32 groups, float32:
// 7 us forward, 11 backward, of which 5 are launch and first loads.
//
// Maps: the values of a group do not fit, so x is read twice, the second time
// from the last-level cache where it fits there.  One pass leaves every
// channel's mean and sum of squared differences over a run of positions, a
// small one joins them to the groups' statistics, one forms y.  Sums are taken
// around a mean of the run itself, and joined as mean and squares (Chan, Golub
// and LeVeque, "Algorithms for computing the sample variance", 1983): a mean
// far from zero costs no digits.  The backward has the same three passes, of the
// sums of dn and dn xh.  4 maps of 50176 x 128 in bfloat16: 14 + 6 + 26 us, the
// last at 4.0 TB/s of reads from the cache and writes to memory.
//
// Statistics and sums are float32, those over runs float64; each output is
// rounded once.  No atomics: every sum has its order.
#include <algorithm>

#include "mvm_group_norm.h"
#include "mvm_scan.h"
#include "seq_common.h"
#include "status.h"

namespace mvm {
namespace {

struct GnGeom {
  int64_t N, P;
  int32_t C, G, Cg;
  int64_t xs, zs;
  float eps;
};
struct GnPtr {
  const void* x;
  const float* w;
  const float* b;
  const void* z;
};

__device__ __forceinline__ float silu_grad(float v, float s) { return s * fmaf(v, 1.f - s, 1.f); }

// One value: y and, backward, dn and dz, from n = xh w + b
template <bool SILU, bool GATE>
__device__ __forceinline__ float gn_out(float n, float z) {
  float y = SILU ? n * sigmoid_f(n) : n;
  if (GATE) y *= z * sigmoid_f(z);
  return y;
}
template <bool SILU, bool GATE>
__device__ __forceinline__ float gn_grad(float n, float z, float dy, float& dz) {
  const float sn = SILU ? sigmoid_f(n) : 0.f;
  if (GATE) {
    const float sz = sigmoid_f(z);
    dz = dy * (SILU ? n * sn : n) * silu_grad(z, sz);
    dy *= z * sz;
  }
  return SILU ? dy * silu_grad(n, sn) : dy;
}

// ------------------------------------------------------------------- rows

// Lanes of a group, groups of a wave, column of value i of lane l
struct GnLanes {
  int32_t log2;        // of the lanes of a group
  int32_t per_wave;
  uint32_t blocks;     // waves abreast over a row's groups
};

// A mean, near + off, and 1 / sqrt(var + eps)
struct GnMoments {
  float near, off, rstd;
};
// Of values whose differences from `near`, a number as close to their mean as its sum's rounding allows, have the mean
// `off` and the mean square `sq`: that rounding is taken out of both moments
__device__ __forceinline__ GnMoments moments_of(float near, float off, float sq, float eps) {
  const float var = fmaf(-off, off, sq);
  return {near, off, 1.f / sqrtf((var < 0.f ? 0.f : var) + eps)};  // (NaN stays)
}

template <int V>
__device__ __forceinline__ float group_sum(float v, int log2) {
  for (int o = 0; o < log2; ++o) v += __shfl_xor(v, 1 << o);
  return v;
}
// of two values, whose exchanges do not wait for each other
__device__ __forceinline__ float2 group_sums(float a, float b, int log2) {
  for (int o = 0; o < log2; ++o) {
    const float x = __shfl_xor(a, 1 << o), y = __shfl_xor(b, 1 << o);
    a += x;
    b += y;
  }
  return make_float2(a, b);
}

// The weights and biases of columns c .. c + V - 1.  (float32 of any alignment: the card's wide loads ask for 4 bytes)
template <int V>
__device__ __forceinline__ void load_weights(const GnPtr& p, int c, float (&w)[V], float (&b)[V]) {
  struct __attribute__((packed, aligned(4))) Run {
    float v[V];
  };
  Run x, y;
#pragma unroll
  for (int j = 0; j < V; ++j) x.v[j] = 1.f, y.v[j] = 0.f;
  if (p.w != nullptr) x = *reinterpret_cast<const Run*>(p.w + c);
  if (p.b != nullptr) y = *reinterpret_cast<const Run*>(p.b + c);
#pragma unroll
  for (int j = 0; j < V; ++j) w[j] = x.v[j], b[j] = y.v[j];
}

// A lane's weights: kept over the rows, unless 32 values would not fit in the registers beside the rest
template <int V, int PER>
struct RowWeights {
  static constexpr bool kKeep = PER * V < 32;
  float w[PER][V], b[PER][V];
  __device__ __forceinline__ void load(const GnGeom& g, const GnPtr& p, const GnLanes& ln, int i, int l, int c0, bool on) {
    const int c = (l + (i << ln.log2)) * V;
    load_weights<V>(p, c0 + (on && c < g.Cg ? c : 0), w[i], b[i]);
  }
};

template <typename T, int V, int PER, bool SILU, bool GATE>
__global__ void __launch_bounds__(256)
gn_rows_fwd_kernel(GnGeom g, GnPtr p, GnLanes ln, T* __restrict__ y, float2* __restrict__ stats) {
  const int lane = threadIdx.x & 63, l = lane & ((1 << ln.log2) - 1);
  const uint32_t wave = blockIdx.x * 4 + (threadIdx.x >> 6), rows = gridDim.x * 4 / ln.blocks;
  const uint32_t gb = wave % ln.blocks;
  const int grp = static_cast<int>(gb) * ln.per_wave + (lane >> ln.log2);
  const bool on = grp < g.G && (lane >> ln.log2) < ln.per_wave;
  const int c0 = (on ? grp : 0) * g.Cg;
  const float inv = 1.f / static_cast<float>(g.Cg);
  RowWeights<V, PER> wt;
  if constexpr (wt.kKeep)
#pragma unroll
    for (int i = 0; i < PER; ++i) wt.load(g, p, ln, i, l, c0, on);
  for (int64_t n = wave / ln.blocks; n < g.N; n += rows) {
    float v[PER][V];
    Pack<T, V> x[PER], z[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int c = (l + (i << ln.log2)) * V, at = c0 + (on && c < g.Cg ? c : 0);
      x[i] = load_pack<T, V>(static_cast<const T*>(p.x) + n * g.xs + at);
      if (GATE) z[i] = load_pack<T, V>(static_cast<const T*>(p.z) + n * g.zs + at);
    }
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const bool ok = on && (l + (i << ln.log2)) * V < g.Cg;
#pragma unroll
      for (int j = 0; j < V; ++j) s += v[i][j] = ok ? to_f32(x[i].v[j]) : 0.f;
    }
    const float near = group_sum<V>(s, ln.log2) * inv;
    float q = s = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        v[i][j] -= near;
        const bool in = (l + (i << ln.log2)) * V < g.Cg;
        s += in ? v[i][j] : 0.f;
        q = in ? fmaf(v[i][j], v[i][j], q) : q;
      }
    const float2 dev = group_sums(s, q, ln.log2);
    const GnMoments mo = moments_of(near, dev.x * inv, dev.y * inv, g.eps);
    if (on && l == 0 && stats != nullptr) stats[n * g.G + grp] = make_float2(near + mo.off, mo.rstd);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int c = (l + (i << ln.log2)) * V;
      if constexpr (!wt.kKeep) wt.load(g, p, ln, i, l, c0, on);
      if (on && c < g.Cg) {
        Pack<T, V> out;
#pragma unroll
        for (int j = 0; j < V; ++j)
          out.v[j] = from_f32<T>(gn_out<SILU, GATE>(fmaf((v[i][j] - mo.off) * mo.rstd, wt.w[i][j], wt.b[i][j]), GATE ? to_f32(z[i].v[j]) : 0.f));
        store_pack(y + n * g.C + c0 + c, out);
      }
    }
  }
}

template <typename T, int V, int PER, bool SILU, bool GATE>
__global__ void __launch_bounds__(256)
gn_rows_bwd_kernel(GnGeom g, GnPtr p, GnLanes ln, const float2* __restrict__ stats, const T* __restrict__ dy,
                   T* __restrict__ dx, T* __restrict__ dz, float* __restrict__ part) {
  const int lane = threadIdx.x & 63, l = lane & ((1 << ln.log2) - 1);
  const uint32_t gb = blockIdx.x % ln.blocks, rb = blockIdx.x / ln.blocks, rows = gridDim.x / ln.blocks * 4;
  const int grp = static_cast<int>(gb) * ln.per_wave + (lane >> ln.log2);
  const bool on = grp < g.G && (lane >> ln.log2) < ln.per_wave;
  const int c0 = (on ? grp : 0) * g.Cg;
  const float inv = 1.f / static_cast<float>(g.Cg);
  RowWeights<V, PER> wt;
  float dw[PER][V], db[PER][V];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if constexpr (wt.kKeep) wt.load(g, p, ln, i, l, c0, on);
#pragma unroll
    for (int j = 0; j < V; ++j) dw[i][j] = db[i][j] = 0.f;
  }
  for (int64_t n = rb * 4 + (threadIdx.x >> 6); n < g.N; n += rows) {
    const float2 st = stats[n * g.G + (on ? grp : 0)];
    float h[PER][V], xh[PER][V];
    Pack<T, V> gz[PER];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int c = (l + (i << ln.log2)) * V;
      const bool ok = on && c < g.Cg;
      const int64_t at = c0 + (ok ? c : 0);
      if constexpr (!wt.kKeep) wt.load(g, p, ln, i, l, c0, on);
      const Pack<T, V> x = load_pack<T, V>(static_cast<const T*>(p.x) + n * g.xs + at);
      const Pack<T, V> d = load_pack<T, V>(dy + n * g.C + at);
      Pack<T, V> z{};
      if (GATE) z = load_pack<T, V>(static_cast<const T*>(p.z) + n * g.zs + at);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        xh[i][j] = (to_f32(x.v[j]) - st.x) * st.y;
        float dzv = 0.f;
        const float dn = gn_grad<SILU, GATE>(fmaf(xh[i][j], wt.w[i][j], wt.b[i][j]), GATE ? to_f32(z.v[j]) : 0.f,
                                             to_f32(d.v[j]), dzv);
        if (GATE) gz[i].v[j] = from_f32<T>(dzv);
        h[i][j] = ok ? dn * wt.w[i][j] : 0.f;
        xh[i][j] = ok ? xh[i][j] : 0.f;
        if (ok) {
          dw[i][j] = fmaf(dn, xh[i][j], dw[i][j]);
          db[i][j] += dn;
        }
        s1 += h[i][j];
        s2 = fmaf(h[i][j], xh[i][j], s2);
      }
    }
    s1 = group_sum<V>(s1, ln.log2) * inv;
    s2 = group_sum<V>(s2, ln.log2) * inv;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int c = (l + (i << ln.log2)) * V;
      if (on && c < g.Cg) {
        Pack<T, V> out;
#pragma unroll
        for (int j = 0; j < V; ++j) out.v[j] = from_f32<T>(st.y * (h[i][j] - s1 - xh[i][j] * s2));
        store_pack(dx + n * g.C + c0 + c, out);
        if (GATE) store_pack(dz + n * g.C + c0 + c, gz[i]);
      }
    }
  }
  if (part == nullptr) return;
  // the workgroup's four waves in order
  __shared__ float sum[2][PER][V][64];
  for (int q = 0; q < 4; ++q) {
    if (static_cast<int>(threadIdx.x >> 6) == q)
#pragma unroll
      for (int i = 0; i < PER; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          sum[0][i][j][lane] = (q ? sum[0][i][j][lane] : 0.f) + dw[i][j];
          sum[1][i][j][lane] = (q ? sum[1][i][j][lane] : 0.f) + db[i][j];
        }
    __syncthreads();
  }
  float* out = part + static_cast<int64_t>(rb) * 2 * g.C;
  if (threadIdx.x < 64 && on)
#pragma unroll
    for (int i = 0; i < PER; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int c = (l + (i << ln.log2)) * V + j;
        if (c < g.Cg) {
          out[c0 + c] = sum[0][i][j][lane];
          out[g.C + c0 + c] = sum[1][i][j][lane];
        }
      }
}

// dweight | dbias: sums over the partial rows
__global__ void __launch_bounds__(1024)
gn_reduce_kernel(const float* part, int64_t nparts, int32_t C, float* dw, float* db) {
  sum_columns(part, nparts, 2 * static_cast<int64_t>(C), [&](int64_t c, float v) {
    if (c < C) {
      if (dw != nullptr) dw[c] = v;
    } else if (db != nullptr) {
      db[c - C] = v;
    }
  });
}

// ------------------------------------------------------------------- reductions of a workgroup

// The sums over a workgroup's rows of each of its columns, (1 << log2) lanes of V columns a row: every
// thread gets its own columns' sums.  A wave's rows by lane exchanges, the waves' through LDS.
template <int V>
__device__ __forceinline__ void column_sums(float (&s)[V], int log2, float (*lds)[64][V]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int o = 32; o >= (1 << log2); o >>= 1)
#pragma unroll
    for (int j = 0; j < V; ++j) s[j] += __shfl_xor(s[j], o);
  const int abreast = log2 > 6 ? 1 << (log2 - 6) : 1;  // waves along a row
  if (abreast == 4) return;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < V; ++j) lds[wave][lane][j] = s[j];
  __syncthreads();
#pragma unroll
  for (int j = 0; j < V; ++j) s[j] = 0.f;
  for (int w = wave & (abreast - 1); w < 4; w += abreast)
#pragma unroll
    for (int j = 0; j < V; ++j) s[j] += lds[w][lane][j];
}

__device__ __forceinline__ float2 workgroup_sum(float a, float b, float2* lds) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    a += __shfl_xor(a, o);
    b += __shfl_xor(b, o);
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = make_float2(a, b);
  __syncthreads();
  return make_float2((lds[0].x + lds[1].x) + (lds[2].x + lds[3].x), (lds[0].y + lds[1].y) + (lds[2].y + lds[3].y));
}

// ------------------------------------------------------------------- tiles

// A workgroup holds a sample's whole group in registers: PER rows a thread, V columns each, (1 << log2) lanes a row
struct TileAt {
  int64_t n;
  int grp, c, RI, ri;
  bool ok;
};
template <int V>
__device__ __forceinline__ TileAt tile_at(const GnGeom& g, int log2) {
  TileAt a;
  // neighbouring groups, which share cache lines, go to one of the 8 L2s
  const uint32_t per = gridDim.x / 8, b = blockIdx.x < per * 8 ? blockIdx.x % 8 * per + blockIdx.x / 8 : blockIdx.x;
  a.n = b / g.G;
  a.grp = static_cast<int>(b - static_cast<uint32_t>(a.n) * g.G);
  const int l = (threadIdx.x & ((1 << log2) - 1)) * V;
  a.ok = l < g.Cg;
  a.c = a.grp * g.Cg + (a.ok ? l : 0);
  a.ri = threadIdx.x >> log2;
  a.RI = 256 >> log2;
  return a;
}

template <typename T, int V, int PER, bool SILU, bool GATE>
__global__ void __launch_bounds__(256)
gn_tile_fwd_kernel(GnGeom g, GnPtr p, int log2, T* __restrict__ y, float2* __restrict__ stats) {
  __shared__ float2 lds[4];
  const TileAt a = tile_at<V>(g, log2);
  const int P = static_cast<int>(g.P);
  const T* xp = static_cast<const T*>(p.x) + a.n * g.P * g.xs + a.c;
  const T* zp = static_cast<const T*>(p.z) + a.n * g.P * g.zs + a.c;
  Pack<T, V> x[PER], z[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int t = a.ri + i * a.RI, at = t < P ? t : 0;
    x[i] = load_pack<T, V>(xp + at * g.xs);
    if (GATE) z[i] = load_pack<T, V>(zp + at * g.zs);
  }
  float w[V], b[V];
  load_weights<V>(p, a.c, w, b);
  const float inv = 1.f / (static_cast<float>(P) * g.Cg);
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) s += a.ok && a.ri + i * a.RI < P ? to_f32(x[i].v[j]) : 0.f;
  const float near = workgroup_sum(s, 0.f, lds).x * inv;
  float q = s = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float d = a.ok && a.ri + i * a.RI < P ? to_f32(x[i].v[j]) - near : 0.f;
      s += d;
      q = fmaf(d, d, q);
    }
  const float2 dev = workgroup_sum(s, q, lds);
  const GnMoments mo = moments_of(near, dev.x * inv, dev.y * inv, g.eps);
  if (threadIdx.x == 0 && stats != nullptr) stats[a.n * g.G + a.grp] = make_float2(near + mo.off, mo.rstd);
  T* yp = y + a.n * g.P * g.C + a.c;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int t = a.ri + i * a.RI;
    if (a.ok && t < P) {
      Pack<T, V> out;
#pragma unroll
      for (int j = 0; j < V; ++j)
        out.v[j] = from_f32<T>(gn_out<SILU, GATE>(fmaf((to_f32(x[i].v[j]) - near - mo.off) * mo.rstd, w[j], b[j]), GATE ? to_f32(z[i].v[j]) : 0.f));
      store_pack(yp + static_cast<int64_t>(t) * g.C, out);
    }
  }
}

// The two means that dx needs and the channels' sums (part (sample)[2][C]) from the same registers; dn is formed
// twice, which costs less than the registers that would keep it
template <typename T, int V, int PER, bool SILU, bool GATE>
__global__ void __launch_bounds__(256)
gn_tile_bwd_kernel(GnGeom g, GnPtr p, int log2, const float2* __restrict__ stats, const T* __restrict__ dy,
                   T* __restrict__ dx, T* __restrict__ dz, float* __restrict__ part) {
  __shared__ float2 lds[4];
  __shared__ float sCol[4][64][V];
  const TileAt a = tile_at<V>(g, log2);
  const int P = static_cast<int>(g.P);
  const T* xp = static_cast<const T*>(p.x) + a.n * g.P * g.xs + a.c;
  const T* zp = static_cast<const T*>(p.z) + a.n * g.P * g.zs + a.c;
  const int64_t out = a.n * g.P * g.C + a.c;
  Pack<T, V> x[PER], z[PER], d[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int t = a.ri + i * a.RI, at = t < P ? t : 0;
    x[i] = load_pack<T, V>(xp + at * g.xs);
    d[i] = load_pack<T, V>(dy + out + static_cast<int64_t>(at) * g.C);
    if (GATE) z[i] = load_pack<T, V>(zp + at * g.zs);
  }
  const float2 st = stats[a.n * g.G + a.grp];
  float w[V], b[V], s1[V], s2[V];
  load_weights<V>(p, a.c, w, b);
#pragma unroll
  for (int j = 0; j < V; ++j) s1[j] = s2[j] = 0.f;
  const auto grad = [&](int i, int j, float& xh, float& dzv) {
    xh = (to_f32(x[i].v[j]) - st.x) * st.y;
    return gn_grad<SILU, GATE>(fmaf(xh, w[j], b[j]), GATE ? to_f32(z[i].v[j]) : 0.f, to_f32(d[i].v[j]), dzv);
  };
#pragma unroll
  for (int i = 0; i < PER; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float xh, dzv = 0.f;
      const float dn = grad(i, j, xh, dzv);
      if (a.ok && a.ri + i * a.RI < P) {
        s1[j] = fmaf(dn, xh, s1[j]);
        s2[j] += dn;
      }
    }
  float u = 0.f, v = 0.f;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    u = fmaf(w[j], s1[j], u);
    v = fmaf(w[j], s2[j], v);
  }
  const float inv = 1.f / (static_cast<float>(P) * g.Cg);
  const float2 m = workgroup_sum(u, v, lds);
  const float m1 = m.x * inv, m2 = m.y * inv;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int t = a.ri + i * a.RI;
    Pack<T, V> ox, oz;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float xh, dzv = 0.f;
      const float dn = grad(i, j, xh, dzv);
      ox.v[j] = from_f32<T>(st.y * (dn * w[j] - m2 - xh * m1));
      if (GATE) oz.v[j] = from_f32<T>(dzv);
    }
    if (a.ok && t < P) {
      store_pack(dx + out + static_cast<int64_t>(t) * g.C, ox);
      if (GATE) store_pack(dz + out + static_cast<int64_t>(t) * g.C, oz);
    }
  }
  if (part == nullptr) return;
  column_sums<V>(s1, log2, sCol);
  column_sums<V>(s2, log2, sCol);
  if (a.ri == 0 && a.ok)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      part[a.n * 2 * g.C + a.c + j] = s1[j];
      part[(a.n * 2 + 1) * g.C + a.c + j] = s2[j];
    }
}

// ------------------------------------------------------------------- maps

constexpr int kAhead = 4;  // rows of a thread whose loads are in flight together

// A workgroup takes a run of positions of one sample and 256 V / RI columns, RI positions side by side
struct GnRun {
  int32_t log2;      // of the threads that lie along a row
  uint32_t cblocks;
  uint32_t runs;     // of a sample
  int32_t len;       // positions of a run
};
struct GnAt {
  int64_t n;
  int32_t run, c, ri, RI;
  int64_t p0, p1;
};
template <int V>
__device__ __forceinline__ GnAt gn_at(const GnGeom& g, const GnRun& r) {
  GnAt a;
  const uint32_t b = blockIdx.x, q = b / r.cblocks;
  a.n = q / r.runs;
  a.run = static_cast<int32_t>(q - static_cast<uint32_t>(a.n) * r.runs);
  a.c = static_cast<int32_t>(((b - q * r.cblocks) << r.log2) + (threadIdx.x & ((1 << r.log2) - 1))) * V;
  a.ri = threadIdx.x >> r.log2;
  a.RI = 256 >> r.log2;
  a.p0 = static_cast<int64_t>(a.run) * r.len;
  a.p1 = a.p0 + r.len < g.P ? a.p0 + r.len : g.P;
  return a;
}

// A channel's values over a run: a number near their mean, what it is off by, and their squared differences' sum.  (The
// mean as one float would have its rounding in it, of which a far mean's differences have few units.)
struct GnPart {
  float near, off, sq;
};
// Sums are taken around the mean of the run's first rows, one for all threads, so that they add up without a division
template <typename T, int V>
__global__ void __launch_bounds__(256)
gn_stats_kernel(GnGeom g, GnPtr p, GnRun r, GnPart* __restrict__ part) {
  __shared__ float lds[4][64][V];
  const GnAt a = gn_at<V>(g, r);
  const bool ok = a.c < g.C;
  float piv[V], s[V], q[V];
#pragma unroll
  for (int j = 0; j < V; ++j) piv[j] = s[j] = q[j] = 0.f;
  const T* x = static_cast<const T*>(p.x) + a.n * g.P * g.xs + (ok ? a.c : 0);
  const int rows = static_cast<int>(a.p1 - a.p0);  // (at least one)
  for (int t0 = 0; t0 < rows; t0 += kAhead * a.RI) {
    Pack<T, V> v[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int t = t0 + a.ri + i * a.RI;
      v[i] = load_pack<T, V>(x + (a.p0 + (t < rows ? t : 0)) * g.xs);
    }
    if (t0 == 0) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) piv[j] += a.ri + i * a.RI < rows ? to_f32(v[i].v[j]) : 0.f;
      column_sums<V>(piv, r.log2, lds);
      const float inv = 1.f / static_cast<float>(rows < kAhead * a.RI ? rows : kAhead * a.RI);
#pragma unroll
      for (int j = 0; j < V; ++j) piv[j] *= inv;
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = t0 + a.ri + i * a.RI < rows ? to_f32(v[i].v[j]) - piv[j] : 0.f;
        s[j] += d;
        q[j] = fmaf(d, d, q[j]);
      }
  }
  column_sums<V>(s, r.log2, lds);
  column_sums<V>(q, r.log2, lds);
  const float inv = 1.f / static_cast<float>(rows);
  if (a.ri == 0 && ok)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float m = s[j] * inv;
      part[(a.n * r.runs + a.run) * g.C + a.c + j] = {piv[j], m, fmaxf(q[j] - s[j] * m, 0.f)};
    }
}

// The sum over a team of W waves of a workgroup of four
template <int W>
__device__ __forceinline__ double team_sum(double x, double* lds) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
  if constexpr (W > 1) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    x = (lds[0] + lds[1]) + (lds[2] + lds[3]);
  }
  return x;
}

// W waves a group and sample (one, or the workgroup's four): its channels' partial statistics as one, for the backward
// (unless NULL) and for the forward's last pass
template <int W>
__global__ void __launch_bounds__(256)
gn_join_kernel(GnGeom g, GnRun r, const GnPart* __restrict__ part, float2* __restrict__ stats, GnMoments* __restrict__ out) {
  __shared__ double lds[4];
  const int64_t item = static_cast<int64_t>(blockIdx.x) * (4 / W) + (W == 1 ? threadIdx.x >> 6 : 0);
  if (item >= g.N * g.G) return;  // (of four waves: all or none)
  const int64_t n = item / g.G;
  const int c0 = static_cast<int>(item - n * g.G) * g.Cg, total = static_cast<int>(r.runs) * g.Cg;
  // the mean of the means, then the squares around it
  const auto each = [&](auto f) {
    for (int i = threadIdx.x & (64 * W - 1); i < total; i += 256 * W) {
      GnPart v[4];
      float cnt[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int at = i + 64 * W * j, k = at < total ? at : i, run = k / g.Cg;
        v[j] = part[(n * r.runs + run) * g.C + c0 + (k - run * g.Cg)];
        const int64_t left = g.P - static_cast<int64_t>(run) * r.len;
        cnt[j] = at < total ? static_cast<float>(left < r.len ? left : r.len) : 0.f;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) f(v[j], cnt[j]);
    }
  };
  const double count = static_cast<double>(g.P) * g.Cg;
  double m = 0.0, q = 0.0;
  each([&](const GnPart& v, float cnt) { m += (static_cast<double>(v.near) + v.off) * cnt; });
  m = team_sum<W>(m, lds) / count;
  each([&](const GnPart& v, float cnt) {
    const double d = v.near - m + v.off;
    q += cnt > 0.f ? v.sq + d * d * cnt : 0.0;
  });
  q = team_sum<W>(q, lds) / count;
  if ((threadIdx.x & (64 * W - 1)) == 0) {
    const float mean = static_cast<float>(m), rstd = static_cast<float>(1.0 / sqrt(q + g.eps));
    out[item] = {mean, static_cast<float>(m - mean), rstd};
    if (stats != nullptr) stats[item] = make_float2(mean, rstd);
  }
}

template <typename T, int V, bool SILU, bool GATE>
__global__ void __launch_bounds__(256)
gn_apply_kernel(GnGeom g, GnPtr p, GnRun r, const GnMoments* __restrict__ moments, T* __restrict__ y) {
  const GnAt a = gn_at<V>(g, r);
  if (a.c >= g.C) return;
  float mean[V], sc[V], b[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const GnMoments mo = moments[a.n * g.G + (a.c + j) / g.Cg];
    mean[j] = mo.near;
    sc[j] = mo.rstd * (p.w != nullptr ? p.w[a.c + j] : 1.f);
    b[j] = fmaf(-mo.off, sc[j], p.b != nullptr ? p.b[a.c + j] : 0.f);
  }
  for (int64_t t0 = a.p0 + a.ri; t0 < a.p1; t0 += kAhead * a.RI) {
    Pack<T, V> x[kAhead], z[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int64_t row = a.n * g.P + (t0 + i * a.RI < a.p1 ? t0 + i * a.RI : t0);
      x[i] = load_pack<T, V>(static_cast<const T*>(p.x) + row * g.xs + a.c);
      if (GATE) z[i] = load_pack<T, V>(static_cast<const T*>(p.z) + row * g.zs + a.c);
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (t0 + i * a.RI < a.p1) {
        Pack<T, V> out;
#pragma unroll
        for (int j = 0; j < V; ++j)
          out.v[j] = from_f32<T>(gn_out<SILU, GATE>(fmaf(to_f32(x[i].v[j]) - mean[j], sc[j], b[j]), GATE ? to_f32(z[i].v[j]) : 0.f));
        store_pack(y + (a.n * g.P + t0 + i * a.RI) * g.C + a.c, out);
      }
  }
}

// Every channel's sums of dn xh and dn over a run: part (sample, run)[2][C]
template <typename T, int V, bool SILU, bool GATE>
__global__ void __launch_bounds__(256)
gn_bwd_sums_kernel(GnGeom g, GnPtr p, GnRun r, const float2* __restrict__ stats, const T* __restrict__ dy,
                   float* __restrict__ part) {
  __shared__ float lds[4][64][V];
  const GnAt a = gn_at<V>(g, r);
  const bool ok = a.c < g.C;
  float mean[V], rs[V], w[V], b[V], s1[V], s2[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int c = ok ? a.c + j : 0;
    const float2 st = stats[a.n * g.G + c / g.Cg];
    mean[j] = st.x;
    rs[j] = st.y;
    w[j] = p.w != nullptr ? p.w[c] : 1.f;
    b[j] = p.b != nullptr ? p.b[c] : 0.f;
    s1[j] = s2[j] = 0.f;
  }
  for (int64_t t0 = a.p0 + a.ri; ok && t0 < a.p1; t0 += 2 * a.RI) {
    Pack<T, V> x[2], d[2], z[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t row = a.n * g.P + (t0 + i * a.RI < a.p1 ? t0 + i * a.RI : t0);
      x[i] = load_pack<T, V>(static_cast<const T*>(p.x) + row * g.xs + a.c);
      d[i] = load_pack<T, V>(dy + row * g.C + a.c);
      if (GATE) z[i] = load_pack<T, V>(static_cast<const T*>(p.z) + row * g.zs + a.c);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (t0 + i * a.RI < a.p1)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float xh = (to_f32(x[i].v[j]) - mean[j]) * rs[j];
          float dzv = 0.f;
          const float dn = gn_grad<SILU, GATE>(fmaf(xh, w[j], b[j]), GATE ? to_f32(z[i].v[j]) : 0.f, to_f32(d[i].v[j]), dzv);
          s1[j] = fmaf(dn, xh, s1[j]);
          s2[j] += dn;
        }
  }
  column_sums<V>(s1, r.log2, lds);
  column_sums<V>(s2, r.log2, lds);
  if (a.ri == 0 && ok) {
    float* out = part + (a.n * r.runs + a.run) * 2 * g.C + a.c;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      out[j] = s1[j];
      out[g.C + j] = s2[j];
    }
  }
}

// W waves a group and sample: the means of dn w xh and dn w
template <int W>
__global__ void __launch_bounds__(256)
gn_bwd_join_kernel(GnGeom g, GnPtr p, GnRun r, const float* __restrict__ part, float2* __restrict__ sums) {
  __shared__ double lds[4];
  const int64_t item = static_cast<int64_t>(blockIdx.x) * (4 / W) + (W == 1 ? threadIdx.x >> 6 : 0);
  if (item >= g.N * g.G) return;  // (of four waves: all or none)
  const int64_t n = item / g.G;
  const int c0 = static_cast<int>(item - n * g.G) * g.Cg, total = static_cast<int>(r.runs) * g.Cg;
  double u = 0.0, v = 0.0;
#pragma unroll 4
  for (int i = threadIdx.x & (64 * W - 1); i < total; i += 64 * W) {
    const int run = i / g.Cg, c = c0 + (i - run * g.Cg);
    const float* at = part + (n * r.runs + run) * 2 * g.C + c;
    const float w = p.w != nullptr ? p.w[c] : 1.f;
    u += static_cast<double>(at[0]) * w;
    v += static_cast<double>(at[g.C]) * w;
  }
  u = team_sum<W>(u, lds);
  v = team_sum<W>(v, lds);
  const double m = static_cast<double>(g.P) * g.Cg;
  if ((threadIdx.x & (64 * W - 1)) == 0) sums[item] = make_float2(static_cast<float>(u / m), static_cast<float>(v / m));
}

template <typename T, int V, bool SILU, bool GATE>
__global__ void __launch_bounds__(256)
gn_bwd_apply_kernel(GnGeom g, GnPtr p, GnRun r, const float2* __restrict__ stats, const float2* __restrict__ sums,
                    const T* __restrict__ dy, T* __restrict__ dx, T* __restrict__ dz) {
  const GnAt a = gn_at<V>(g, r);
  if (a.c >= g.C) return;
  float mean[V], rs[V], w[V], b[V], m1[V], m2[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int64_t at = a.n * g.G + (a.c + j) / g.Cg;
    const float2 st = stats[at], sm = sums[at];
    mean[j] = st.x;
    rs[j] = st.y;
    m1[j] = sm.x;
    m2[j] = sm.y;
    w[j] = p.w != nullptr ? p.w[a.c + j] : 1.f;
    b[j] = p.b != nullptr ? p.b[a.c + j] : 0.f;
  }
  for (int64_t t = a.p0 + a.ri; t < a.p1; t += a.RI) {
    const int64_t row = a.n * g.P + t;
    const Pack<T, V> x = load_pack<T, V>(static_cast<const T*>(p.x) + row * g.xs + a.c);
    const Pack<T, V> d = load_pack<T, V>(dy + row * g.C + a.c);
    Pack<T, V> z{}, ox, oz;
    if (GATE) z = load_pack<T, V>(static_cast<const T*>(p.z) + row * g.zs + a.c);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float xh = (to_f32(x.v[j]) - mean[j]) * rs[j];
      float dzv = 0.f;
      const float dn = gn_grad<SILU, GATE>(fmaf(xh, w[j], b[j]), GATE ? to_f32(z.v[j]) : 0.f, to_f32(d.v[j]), dzv);
      ox.v[j] = from_f32<T>(rs[j] * (dn * w[j] - m2[j] - xh * m1[j]));
      if (GATE) oz.v[j] = from_f32<T>(dzv);
    }
    store_pack(dx + row * g.C + a.c, ox);
    if (GATE) store_pack(dz + row * g.C + a.c, oz);
  }
}

// ------------------------------------------------------------- host side

constexpr int64_t kMaxRows = int64_t{1} << 31;
constexpr int64_t kMaxBlocks = (int64_t{1} << 24) - 8;  // of 256 threads, 2^32 a launch
constexpr int kRowValues = 2048;        // of a group, held in registers by 64 lanes
// waves that walk the rows forward: more of them load the weights more often, fewer leave loads unhidden (16384 rows of
// 12 heads of 128: 1024 86 us, 2048 52, 4096 40, 16384 50, all with weights in 4-byte loads; 33 now); four times as
// many where values come one by one (16384 rows of 1530 in 10 groups: 54 us against 67; in one, 117 against 103)
constexpr int64_t kRowWaves = 4096;
constexpr int64_t kTileRows = 8;        // of a thread, held in registers
constexpr int64_t kPartRows = 512;      // partial rows of the channels' gradients
constexpr size_t kAlign = 256;

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
size_t align_up(size_t x) { return (x + kAlign - 1) / kAlign * kAlign; }
int log2_ceil(int64_t n) {
  int l = 0;
  while ((int64_t{1} << l) < n) ++l;
  return l;
}

int check_fields(const mvm_group_norm_desc* d) {
  if (d == nullptr) return fail(MVM_ERR_INVALID_ARG, "desc is NULL");
  if (d->batch < 0 || d->positions < 0)
    return fail(MVM_ERR_INVALID_ARG, "negative size (batch=%lld positions=%lld)", (long long)d->batch,
                (long long)d->positions);
  if (d->channels < 1 || d->channels > MVM_GROUP_NORM_MAX_CHANNELS)
    return fail(MVM_ERR_UNSUPPORTED, "channels=%lld unsupported (1..%d)", (long long)d->channels,
                MVM_GROUP_NORM_MAX_CHANNELS);
  if (d->groups < 1 || d->groups > d->channels || d->channels % d->groups != 0)
    return fail(MVM_ERR_INVALID_ARG, "groups=%lld must divide channels=%lld", (long long)d->groups,
                (long long)d->channels);
  if (d->dtype != MVM_F32 && d->dtype != MVM_BF16) return fail(MVM_ERR_UNSUPPORTED, "dtype=%d unsupported", d->dtype);
  if (d->reserved != 0) return fail(MVM_ERR_INVALID_ARG, "reserved must be 0");
  if (d->silu != 0 && d->silu != 1) return fail(MVM_ERR_INVALID_ARG, "silu=%d must be 0 or 1", d->silu);
  if (!(d->eps >= 0.f)) return fail(MVM_ERR_INVALID_ARG, "eps must be >= 0");
  if (d->positions > 0 && d->batch > kMaxRows / d->positions)
    return fail(MVM_ERR_UNSUPPORTED, "batch=%lld * positions=%lld: at most %lld rows", (long long)d->batch,
                (long long)d->positions, (long long)kMaxRows);
  for (const int64_t s : {d->x_stride, d->z_stride})
    if (s < 0 || s > (int64_t{1} << 40))
      return fail(MVM_ERR_INVALID_ARG, "stride %lld must be in [0, 2^40]", (long long)s);
  return MVM_OK;
}

GnGeom geom_of(const mvm_group_norm_desc* d) {
  return {d->batch, d->positions, static_cast<int32_t>(d->channels), static_cast<int32_t>(d->groups),
          static_cast<int32_t>(d->channels / d->groups), d->x_stride, d->z_stride, d->eps};
}

bool by_rows(const GnGeom& g) { return g.P == 1 && g.Cg <= kRowValues; }

// The rows kernels' lanes for accesses of V values
GnLanes lanes_of(const GnGeom& g, int V) {
  GnLanes l;
  l.log2 = std::min(6, log2_ceil(ceil_div(g.Cg, V)));
  l.per_wave = std::min(64 >> l.log2, g.G);
  l.blocks = static_cast<uint32_t>(ceil_div(g.G, l.per_wave));
  return l;
}
// workgroups along the rows of the backward
int64_t row_blocks(const GnGeom& g, const GnLanes& l) {
  return std::max<int64_t>(1, std::min(ceil_div(g.N, 4), std::max<int64_t>(1, kPartRows * 4 / l.blocks)));
}

// A group in a workgroup's registers, for accesses of V values that groups start on: log2 of the lanes of a row and
// the rows of a thread, 0 where it does not fit.  (32 samples of 196 x 384 in 32 groups, gated: 9.4 us forward and 14
// backward, against 17 and 23 in passes; 256 of them 60 and 104, against 66 and 116)
struct GnTile {
  int32_t log2 = 0, per = 0;
};
GnTile tile_of(const GnGeom& g, int V) {
  GnTile t;
  if (V == 1 || g.Cg % V != 0 || g.Cg > 256 * V || g.N > kMaxBlocks / g.G) return t;
  t.log2 = log2_ceil(g.Cg / V);
  const int64_t per = ceil_div(g.P, 256 >> t.log2);
  if (per <= kTileRows) t.per = per <= 2 ? 2 : per <= 4 ? 4 : 8;
  return t;
}
template <typename F>
hipError_t with_tile(const GnTile& t, F&& f) {
  if (t.per == 2) return f(std::integral_constant<int, 2>{});
  if (t.per == 4) return f(std::integral_constant<int, 4>{});
  return f(std::integral_constant<int, 8>{});
}

// Four waves join a group's partial sums where one would take more than four turns of four loads
bool wide_join(const GnGeom& g, const GnRun& r) {
  return static_cast<int64_t>(r.runs) * g.Cg > 1024 && g.N <= kMaxBlocks / g.G;
}
unsigned join_blocks(const GnGeom& g, const GnRun& r) {
  return static_cast<unsigned>(wide_join(g, r) ? g.N * g.G : ceil_div(g.N * g.G, 4));
}

// The maps' runs: enough workgroups to fill the card, of 32 positions at least a thread
GnRun run_of(const GnGeom& g, int V) {
  GnRun r;
  r.log2 = std::min(8, log2_ceil(ceil_div(g.C, V)));
  r.cblocks = static_cast<uint32_t>(ceil_div(g.C, static_cast<int64_t>(V) << r.log2));
  const int64_t side = 256 >> r.log2;
  const int64_t want = std::max<int64_t>(1, ceil_div(2048, std::max<int64_t>(1, g.N * r.cblocks)));
  int64_t len = std::max(ceil_div(g.P, want), std::min<int64_t>(g.P, 8 * side));
  len = std::max<int64_t>(1, ceil_div(len, side) * side);
  // (no more workgroups than a launch takes, however many samples)
  r.len = static_cast<int32_t>(std::min<int64_t>(len, int64_t{1} << 30));
  r.runs = static_cast<uint32_t>(std::max<int64_t>(1, ceil_div(g.P, r.len)));
  return r;
}

// Everything that a call of either direction would be refused for.
int check_desc(const mvm_group_norm_desc* d) {
  const int rc = check_fields(d);
  if (rc != MVM_OK) return rc;
  const GnGeom g = geom_of(d);
  if (by_rows(g) || g.N == 0) return MVM_OK;
  const GnRun r = run_of(g, 1);
  if (g.N > kMaxBlocks / (static_cast<int64_t>(r.runs) * r.cblocks) || g.N > kMaxBlocks * 4 / g.G)
    return fail(MVM_ERR_UNSUPPORTED, "batch=%lld, positions=%lld, channels=%lld are too many for one launch",
                (long long)d->batch, (long long)d->positions, (long long)d->channels);
  return MVM_OK;
}

struct GnWs {
  size_t part = 0, stats = 0, total = 0;
};
GnWs ws_of(const GnGeom& g, bool backward) {
  GnWs w;
  // (the lanes and runs for the accesses that the pointers will allow: the larger of the two)
  const size_t row = static_cast<size_t>(g.C) * 8;
  for (const int V : {1, 4, 8}) {
    size_t part = 0;
    if (by_rows(g))
      part = backward ? static_cast<size_t>(row_blocks(g, lanes_of(g, V))) * row : 0;
    else
      part = static_cast<size_t>(g.N) * run_of(g, V).runs * (backward ? row : static_cast<size_t>(g.C) * sizeof(GnPart));
    w.part = std::max(w.part, align_up(part));
  }
  w.stats = by_rows(g) ? 0 : align_up(static_cast<size_t>(g.N) * g.G * (backward ? 8 : sizeof(GnMoments)));
  w.total = w.part + w.stats;
  return w;
}

int check_ws(const char* what, const void* ws, size_t have, size_t need) {
  if (need > 0 && (ws == nullptr || have < need))
    return fail(MVM_ERR_WORKSPACE, "%s: workspace %zu bytes < %zu needed", what, have, need);
  if (need > 0 && (reinterpret_cast<uintptr_t>(ws) & (kAlign - 1)) != 0)
    return fail(MVM_ERR_WORKSPACE, "%s: workspace must be %zu-byte aligned", what, kAlign);
  return MVM_OK;
}

// 16-byte accesses: every row and, for rows, every group starts on one
template <typename T>
bool wide(const GnGeom& g, std::initializer_list<const void*> ptrs, bool gate) {
  constexpr int V = 16 / sizeof(T);
  uintptr_t u = 0;
  for (const void* p : ptrs) u |= reinterpret_cast<uintptr_t>(p);
  const int64_t unit = by_rows(g) ? g.Cg : g.C;
  return (u & 15) == 0 && unit % V == 0 && g.xs % V == 0 && (!gate || g.zs % V == 0);
}

// f(type, values an access, silu, gate)
template <typename F>
hipError_t dispatch(const mvm_group_norm_desc* d, bool w32, bool w16, bool gate, F&& f) {
  const auto flags = [&](auto t, auto v) {
    using std::false_type;
    using std::true_type;
    if (d->silu) return gate ? f(t, v, true_type{}, true_type{}) : f(t, v, true_type{}, false_type{});
    return gate ? f(t, v, false_type{}, true_type{}) : f(t, v, false_type{}, false_type{});
  };
  using One = std::integral_constant<int, 1>;
  if (d->dtype == MVM_F32) return w32 ? flags(float{}, std::integral_constant<int, 4>{}) : flags(float{}, One{});
  return w16 ? flags(bf16_t{}, std::integral_constant<int, 8>{}) : flags(bf16_t{}, One{});
}

// f(std::integral_constant<int, accesses of a lane>)
template <int V, typename F>
hipError_t with_per(const GnGeom& g, const GnLanes& l, F&& f) {
  const int64_t per = ceil_div(g.Cg, static_cast<int64_t>(V) << l.log2);
  if (per <= 1) return f(std::integral_constant<int, 1>{});
  if (per <= 2) return f(std::integral_constant<int, 2>{});
  if (per <= 4) return f(std::integral_constant<int, 4>{});
  if constexpr (V <= 4) {
    if (per <= 8) return f(std::integral_constant<int, 8>{});
  }
  if constexpr (V == 1) {
    if (per <= 32) return f(std::integral_constant<int, 32>{});
  }
  return hipErrorInvalidValue;  // (kRowValues)
}

}  // namespace
}  // namespace mvm

extern "C" {

int mvm_group_norm_validate(const mvm_group_norm_desc* desc) {
  const int rc = mvm::check_desc(desc);
  return rc == MVM_OK ? mvm::ok() : rc;
}

int64_t mvm_group_norm_workspace_bytes(const mvm_group_norm_desc* desc, int which) {
  const int rc = mvm::check_desc(desc);
  if (rc != MVM_OK) return rc;
  if (which != 0 && which != 1) return mvm::fail(MVM_ERR_INVALID_ARG, "which=%d must be 0 or 1", which);
  return static_cast<int64_t>(mvm::ws_of(mvm::geom_of(desc), which == 1).total);
}

int mvm_group_norm_fwd(const mvm_group_norm_desc* desc, const void* x, const float* weight, const float* bias,
                       const void* z, void* y, float* stats, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace mvm;
  int rc = check_desc(desc);
  if (rc != MVM_OK) return rc;
  const GnGeom g = geom_of(desc);
  if (g.N == 0 || g.P == 0) return ok();
  if (!x || !y) return fail(MVM_ERR_INVALID_ARG, "mvm_group_norm_fwd: NULL pointer");
  const GnWs w = ws_of(g, false);
  if ((rc = check_ws("mvm_group_norm_fwd", workspace, workspace_bytes, w.total)) != MVM_OK) return rc;
  const GnPtr p{x, weight, bias, z};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const bool gate = z != nullptr;
  const hipError_t e = dispatch(desc, wide<float>(g, {x, z, y}, gate), wide<bf16_t>(g, {x, z, y}, gate), gate,
                                [&](auto t, auto v, auto silu, auto gt) {
    using T = decltype(t);
    constexpr int V = decltype(v)::value;
    constexpr bool SILU = decltype(silu)::value, GATE = decltype(gt)::value;
    if (by_rows(g)) {
      const GnLanes l = lanes_of(g, V);
      // (whole workgroups of waves that have one block of groups each)
      const int64_t waves = std::min<int64_t>(g.N, std::max<int64_t>(1, (V == 1 ? 4 : 1) * kRowWaves / l.blocks)) * l.blocks;
      const int64_t unit = static_cast<int64_t>(l.blocks) * 4;
      const dim3 grid(static_cast<unsigned>(ceil_div(ceil_div(waves, unit) * unit, 4)));
      return with_per<V>(g, l, [&](auto per) {
        hipLaunchKernelGGL((gn_rows_fwd_kernel<T, V, decltype(per)::value, SILU, GATE>), grid, dim3(256), 0, s, g, p, l,
                           static_cast<T*>(y), reinterpret_cast<float2*>(stats));
        return hipGetLastError();
      });
    }
    if constexpr (V > 1)
      if (const GnTile t = tile_of(g, V); t.per > 0)
        return with_tile(t, [&](auto per) {
          hipLaunchKernelGGL((gn_tile_fwd_kernel<T, V, decltype(per)::value, SILU, GATE>), dim3(static_cast<unsigned>(g.N * g.G)),
                             dim3(256), 0, s, g, p, t.log2, static_cast<T*>(y), reinterpret_cast<float2*>(stats));
          return hipGetLastError();
        });
    const GnRun r = run_of(g, V);
    const dim3 grid(static_cast<unsigned>(g.N * r.runs * r.cblocks));
    GnPart* part = static_cast<GnPart*>(workspace);
    GnMoments* mo = reinterpret_cast<GnMoments*>(static_cast<char*>(workspace) + w.part);
    hipLaunchKernelGGL((gn_stats_kernel<T, V>), grid, dim3(256), 0, s, g, p, r, part);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(wide_join(g, r) ? gn_join_kernel<4> : gn_join_kernel<1>, dim3(join_blocks(g, r)), dim3(256), 0, s, g, r,
                       part, reinterpret_cast<float2*>(stats), mo);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    hipLaunchKernelGGL((gn_apply_kernel<T, V, SILU, GATE>), grid, dim3(256), 0, s, g, p, r, mo, static_cast<T*>(y));
    return hipGetLastError();
  });
  return hip_status(e, "mvm_group_norm_fwd launch");
}

int mvm_group_norm_bwd(const mvm_group_norm_desc* desc, const void* x, const float* weight, const float* bias,
                       const void* z, const float* stats, const void* dy, void* dx, float* dweight, float* dbias,
                       void* dz, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace mvm;
  int rc = check_desc(desc);
  if (rc != MVM_OK) return rc;
  const GnGeom g = geom_of(desc);
  const bool some = g.N > 0 && g.P > 0, gate = z != nullptr;
  if (some && (!x || !stats || !dy || !dx || gate != (dz != nullptr)))
    return fail(MVM_ERR_INVALID_ARG, "mvm_group_norm_bwd: NULL pointer");
  const GnWs w = ws_of(g, true);
  if ((rc = check_ws("mvm_group_norm_bwd", workspace, workspace_bytes, w.total)) != MVM_OK) return rc;
  const GnPtr p{x, weight, bias, z};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  float* part = static_cast<float*>(workspace);
  const float2* st = reinterpret_cast<const float2*>(stats);
  int64_t nparts = 0;
  const bool params = dweight != nullptr || dbias != nullptr;
  hipError_t e = hipSuccess;
  if (some)
    e = dispatch(desc, wide<float>(g, {x, z, dy, dx, dz}, gate), wide<bf16_t>(g, {x, z, dy, dx, dz}, gate), gate,
                 [&](auto t, auto v, auto silu, auto gt) {
      using T = decltype(t);
      constexpr int V = decltype(v)::value;
      constexpr bool SILU = decltype(silu)::value, GATE = decltype(gt)::value;
      if (by_rows(g)) {
        const GnLanes l = lanes_of(g, V);
        nparts = row_blocks(g, l);
        const dim3 grid(static_cast<unsigned>(nparts * l.blocks));
        return with_per<V>(g, l, [&](auto per) {
          hipLaunchKernelGGL((gn_rows_bwd_kernel<T, V, decltype(per)::value, SILU, GATE>), grid, dim3(256), 0, s, g, p,
                             l, st, static_cast<const T*>(dy), static_cast<T*>(dx), static_cast<T*>(dz),
                             params ? part : nullptr);
          return hipGetLastError();
        });
      }
      if constexpr (V > 1)
        if (const GnTile t = tile_of(g, V); t.per > 0 && !(g.Cg == V && g.N * g.G > 8192)) {
          // (many groups of 16 bytes a row would take their lines several times: 1024 samples of 64 x 64 in 16 groups
          // 59 us against 28 in passes; 8 of 1024 x 256 in 32 groups 11 against 17)
          nparts = g.N;
          return with_tile(t, [&](auto per) {
            hipLaunchKernelGGL((gn_tile_bwd_kernel<T, V, decltype(per)::value, SILU, GATE>),
                               dim3(static_cast<unsigned>(g.N * g.G)), dim3(256), 0, s, g, p, t.log2, st,
                               static_cast<const T*>(dy), static_cast<T*>(dx), static_cast<T*>(dz), params ? part : nullptr);
            return hipGetLastError();
          });
        }
      const GnRun r = run_of(g, V);
      const dim3 grid(static_cast<unsigned>(g.N * r.runs * r.cblocks));
      nparts = g.N * r.runs;
      float2* sums = reinterpret_cast<float2*>(static_cast<char*>(workspace) + w.part);
      hipLaunchKernelGGL((gn_bwd_sums_kernel<T, V, SILU, GATE>), grid, dim3(256), 0, s, g, p, r, st,
                         static_cast<const T*>(dy), part);
      hipError_t e = hipGetLastError();
      if (e != hipSuccess) return e;
      hipLaunchKernelGGL(wide_join(g, r) ? gn_bwd_join_kernel<4> : gn_bwd_join_kernel<1>, dim3(join_blocks(g, r)), dim3(256), 0,
                         s, g, p, r, part, sums);
      if ((e = hipGetLastError()) != hipSuccess) return e;
      hipLaunchKernelGGL((gn_bwd_apply_kernel<T, V, SILU, GATE>), grid, dim3(256), 0, s, g, p, r, st, sums,
                         static_cast<const T*>(dy), static_cast<T*>(dx), static_cast<T*>(dz));
      return hipGetLastError();
    });
  if (e == hipSuccess && params) {
    hipLaunchKernelGGL(gn_reduce_kernel, dim3(static_cast<unsigned>(ceil_div(2 * static_cast<int64_t>(g.C), 64))),
                       dim3(1024), 0, s, part, nparts, g.C, dweight, dbias);
    e = hipGetLastError();
  }
  return hip_status(e, "mvm_group_norm_bwd launch");
}

}  // extern "C"
