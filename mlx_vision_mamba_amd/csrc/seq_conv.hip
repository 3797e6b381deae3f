// Causal depthwise conv + SiLU of packed sequences with states, forward,
// backward and one token, for gfx950.
//
// x~ is a sequence's rows with its state's kc - 1 rows before them:
//   pre_t = bias + sum_{j<kc} w[j] x~[t - (kc-1) + j],  y_t = pre_t sigmoid(pre_t)
// and the final state is the last kc - 1 rows of x~.
//
// Bound by the rows' traffic.  A lane holds V consecutive channels (16 bytes
// where the layout allows it), a wave P positions of one sequence with their
// whole window in registers, so that all its loads are in flight together; a
// block is four such waves.  The first wave of a sequence is the only one that
// reads its initial state (kc - 1 <= P), and it also writes the final one: both
// may be one buffer.
//
// MI355X: 8191 bf16 tokens of 1536 channels in 23 sequences 14.1 us, 3.6 TB/s (a
// large copy reaches 4.9), of 1535 channels, one a lane, 17.3; forward + backward
// of 6272 tokens of 768 channels 10 + 16 + 4 us of kernels, float32 or bf16 (the
// backward has two channels a lane).
#include <initializer_list>
#include <type_traits>

#include "mvm_conv.h"
#include "mvm_scan.h"
#include "seq_common.h"

namespace mvm {

namespace {

// Row p of x~ of a sequence, p counted from its first token (p < 0: the
// state's row kc - 1 + p); zero where there is none.
template <typename T, int V, int KC>
__device__ __forceinline__ Pack<T, V> row_of_seq(const T* x, int64_t xs, const SeqChunk& c, const T* state, int64_t D,
                                                 int64_t d, int64_t p) {
  Pack<T, V> r;
  if (p >= 0 && c.start + p < c.end) return load_pack<T, V>(x + (c.start + p) * xs + d);
  if (p < 0 && state != nullptr) return load_pack<T, V>(state + (KC - 1 + p) * D + d);
#pragma unroll
  for (int v = 0; v < V; ++v) r.v[v] = from_f32<T>(0.f);
  return r;
}

// The taps and biases of a lane's V channels.  Sixteen bytes a load where the
// channels' taps are whole multiples of that (vec: and the buffers aligned):
// one value a load would be more loads than the rows themselves.
template <int V, int KC>
struct Taps {
  float w[KC][V], b[V];
  __device__ __forceinline__ void load(const float* wp, const float* bp, int64_t d, int vec) {
    float t[V * KC];
    if ((V * KC) % 4 == 0 && V % 4 == 0 && vec) {
      wp = opaque(wp + d * KC);
#pragma unroll
      for (int i = 0; i < V * KC / 4; ++i) {
        const Pack<float, 4> p = load_pack<float, 4>(wp + 4 * i);
#pragma unroll
        for (int j = 0; j < 4; ++j) t[4 * i + j] = p.v[j];
      }
      if (bp) bp = opaque(bp + d);
#pragma unroll
      for (int i = 0; i < V / 4; ++i) {
        const Pack<float, 4> p = bp ? load_pack<float, 4>(bp + 4 * i) : Pack<float, 4>{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 4; ++j) b[4 * i + j] = p.v[j];
      }
    } else {
#pragma unroll
      for (int i = 0; i < V * KC; ++i) t[i] = wp[d * KC + i];
#pragma unroll
      for (int v = 0; v < V; ++v) b[v] = bp ? bp[d + v] : 0.f;
    }
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int j = 0; j < KC; ++j) w[j][v] = t[v * KC + j];
  }
};

template <typename T, int V, int KC, int P>
__global__ void __launch_bounds__(256)
seq_conv_fwd_kernel(SeqConvGeom g, uint32_t ncb, const T* __restrict__ x, const float* __restrict__ w,
                    const float* __restrict__ bias, const T* c0, T* c1, T* __restrict__ y) {
  static_assert(KC - 1 <= P, "a second wave would read the state that the first one writes");
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const BlockPos pos = block_pos(ncb);
  const SeqChunk c = seq_chunk(g.q, pos.slot, conv_cut(P), lane);
  const int64_t D = g.q.D, d = (static_cast<int64_t>(pos.cb) * 64 + lane) * V;
  if (c.t0 < 0 || d >= D) return;
  const int32_t s0 = c.t0 + wave * P;
  if (c.seq == g.q.S) {  // rows of no sequence
    Pack<T, V> zero;
#pragma unroll
    for (int v = 0; v < V; ++v) zero.v[v] = from_f32<T>(0.f);
    for (int32_t t = s0; t < c.t1 && t < s0 + P; ++t) store_pack(y + t * g.ys + d, zero);
    return;
  }
  const int32_t row = seq_slot(g.q, c.seq);
  Taps<V, KC> k;
  if (s0 < c.t1) k.load(w, bias, d, g.w_vec);
  const T* state = nullptr;
  if (c.t0 == c.start && c0 != nullptr && row >= 0 && !seq_fresh(g.q, c.seq))
    state = c0 + static_cast<int64_t>(row) * (KC - 1) * D;
  if (s0 < c.t1) {
    const int64_t p0 = s0 - c.start;
    Pack<T, V> win[P + KC - 1];
    if (p0 >= KC - 1 && s0 + P <= c.end) {
#pragma unroll
      for (int i = 0; i < P + KC - 1; ++i) win[i] = load_pack<T, V>(x + (s0 - (KC - 1) + i) * g.xs + d);
    } else {
#pragma unroll
      for (int i = 0; i < P + KC - 1; ++i)
        win[i] = row_of_seq<T, V, KC>(x, g.xs, c, state, D, d, p0 - (KC - 1) + i);
    }
#pragma unroll
    for (int i = 0; i < P; ++i) {
      if (s0 + i < c.t1) {
        Pack<T, V> o;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float pre = k.b[v];
#pragma unroll
          for (int j = 0; j < KC; ++j) pre = fmaf(k.w[j][v], to_f32(win[i + j].v[v]), pre);
          o.v[v] = from_f32<T>(pre * sigmoid_f(pre));
        }
        store_pack(y + (s0 + i) * g.ys + d, o);
      }
    }
  }
  if constexpr (KC > 1) {
    // The final state, by the wave that read the initial one (its loads are
    // done before these stores: the values have been used or are below).
    if (c.t0 == c.start && wave == 0 && c1 != nullptr && row >= 0) {
      Pack<T, V> f[KC - 1];
      const int64_t p0 = static_cast<int64_t>(c.end) - c.start - (KC - 1);
#pragma unroll
      for (int r = 0; r < KC - 1; ++r) f[r] = row_of_seq<T, V, KC>(x, g.xs, c, state, D, d, p0 + r);
#pragma unroll
      for (int r = 0; r < KC - 1; ++r) store_pack(c1 + (static_cast<int64_t>(row) * (KC - 1) + r) * D + d, f[r]);
    }
  }
}

template <typename T, int V, int KC, int P>
__global__ void __launch_bounds__(256)
seq_conv_bwd_kernel(SeqConvGeom g, uint32_t ncb, const T* __restrict__ x, const float* __restrict__ w,
                    const float* __restrict__ bias, const T* __restrict__ c0, const T* __restrict__ dy,
                    const T* __restrict__ dc1, T* __restrict__ dx, T* __restrict__ dc0, float* __restrict__ part) {
  __shared__ float sums[4][(KC + 1) * V][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const BlockPos pos = block_pos(ncb);
  const SeqChunk c = seq_chunk(g.q, pos.slot, conv_cut(P), lane);
  const int64_t D = g.q.D, d = (static_cast<int64_t>(pos.cb) * 64 + lane) * V;
  const bool valid = d < D;
  const int64_t dd = valid ? d : 0;
  const int32_t s0 = c.t0 + wave * P;
  float dw[KC][V], db[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    db[v] = 0.f;
#pragma unroll
    for (int j = 0; j < KC; ++j) dw[j][v] = 0.f;
  }
  if (c.seq == g.q.S && c.t0 >= 0) {
    Pack<T, V> zero;
#pragma unroll
    for (int v = 0; v < V; ++v) zero.v[v] = from_f32<T>(0.f);
    for (int32_t t = s0; t < c.t1 && t < s0 + P; ++t)
      if (valid) store_pack(dx + static_cast<int64_t>(t) * D + d, zero);
  } else if (c.t0 >= 0) {
    const T* state = c0 != nullptr ? c0 + static_cast<int64_t>(c.seq) * (KC - 1) * D : nullptr;
    const int64_t len = static_cast<int64_t>(c.end) - c.start, p0 = s0 - c.start;
    // the final state's gradient reaches rows len - (kc-1) .. len - 1 of x~
    auto add_final = [&](float (&a)[V], int64_t p) {
      const int64_t r = p - (len - (KC - 1));
      if (dc1 != nullptr && r >= 0 && r < KC - 1) {
        const Pack<T, V> f = load_pack<T, V>(dc1 + (static_cast<int64_t>(c.seq) * (KC - 1) + r) * D + dd);
#pragma unroll
        for (int v = 0; v < V; ++v) a[v] += to_f32(f.v[v]);
      }
    };
    const bool head = c.t0 == c.start && wave == 0;
    if (s0 < c.t1 || head) {
      Taps<V, KC> k;
      k.load(w, bias, dd, g.w_vec);
      constexpr int kG = P + KC - 1;  // positions whose dpre is needed
      Pack<T, V> xw[kG + KC - 1], gy[kG];
#pragma unroll
      for (int i = 0; i < kG + KC - 1; ++i)
        xw[i] = row_of_seq<T, V, KC>(x, g.xs, c, state, D, dd, p0 - (KC - 1) + i);
#pragma unroll
      for (int i = 0; i < kG; ++i) {
        if (p0 + i < len) {
          gy[i] = load_pack<T, V>(dy + (s0 + i) * g.ys + dd);
        } else {
#pragma unroll
          for (int v = 0; v < V; ++v) gy[i].v[v] = from_f32<T>(0.f);
        }
      }
      float gp[kG][V];
#pragma unroll
      for (int i = 0; i < kG; ++i)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float pre = k.b[v];
#pragma unroll
          for (int j = 0; j < KC; ++j) pre = fmaf(k.w[j][v], to_f32(xw[i + j].v[v]), pre);
          const float sg = sigmoid_f(pre);
          gp[i][v] = p0 + i < len ? to_f32(gy[i].v[v]) * sg * fmaf(pre, 1.f - sg, 1.f) : 0.f;
        }
#pragma unroll
      for (int i = 0; i < P; ++i) {
        if (s0 + i < c.t1) {
          float a[V];
#pragma unroll
          for (int v = 0; v < V; ++v) {
            a[v] = 0.f;
            db[v] += gp[i][v];
#pragma unroll
            for (int j = 0; j < KC; ++j) {
              a[v] = fmaf(k.w[j][v], gp[i + KC - 1 - j][v], a[v]);
              dw[j][v] = fmaf(gp[i][v], to_f32(xw[i + j].v[v]), dw[j][v]);
            }
          }
          add_final(a, p0 + i);
          Pack<T, V> o;
#pragma unroll
          for (int v = 0; v < V; ++v) o.v[v] = from_f32<T>(a[v]);
          if (valid) store_pack(dx + static_cast<int64_t>(s0 + i) * D + d, o);
        }
      }
      if constexpr (KC > 1) {
        if (head && dc0 != nullptr) {
          // x~ row p = r - (kc-1) < 0 enters pre of the tokens 0 .. r
#pragma unroll
          for (int r = 0; r < KC - 1; ++r) {
            float a[V];
#pragma unroll
            for (int v = 0; v < V; ++v) {
              a[v] = 0.f;
#pragma unroll
              for (int j = 0; j <= r; ++j) a[v] = fmaf(k.w[j][v], gp[r - j][v], a[v]);
            }
            add_final(a, r - (KC - 1));
            Pack<T, V> o;
#pragma unroll
            for (int v = 0; v < V; ++v) o.v[v] = from_f32<T>(a[v]);
            if (valid) store_pack(dc0 + (static_cast<int64_t>(c.seq) * (KC - 1) + r) * D + d, o);
          }
        }
      }
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
#pragma unroll
    for (int j = 0; j < KC; ++j) sums[wave][v * (KC + 1) + j][lane] = dw[j][v];
    sums[wave][v * (KC + 1) + KC][lane] = db[v];
  }
  __syncthreads();
  // the block's sums: columns (channel, tap | bias)
  constexpr int kCols = (KC + 1) * V;
  const int64_t first = static_cast<int64_t>(pos.cb) * 64 * kCols, ncols = D * (KC + 1);
  for (int i = threadIdx.x; i < 64 * kCols; i += 256) {
    const int l = i / kCols, k = i - l * kCols;
    if (first + i < ncols)
      part[static_cast<int64_t>(pos.slot) * ncols + first + i] =
          (sums[0][k][l] + sums[1][k][l]) + (sums[2][k][l] + sums[3][k][l]);
  }
}

__global__ void __launch_bounds__(1024)
seq_conv_reduce_kernel(int64_t ncols, int32_t kc, int64_t nparts, const float* __restrict__ part,
                       float* __restrict__ dw, float* __restrict__ db) {
  sum_columns(part, nparts, ncols, [&](int64_t col, float s) {
    const int64_t d = col / (kc + 1);
    const int j = static_cast<int>(col - d * (kc + 1));
    if (j < kc)
      dw[d * kc + j] = s;
    else if (db != nullptr)
      db[d] = s;
  });
}

// One token: the state's rows move up by one in place.  A wave keeps its
// channels' taps for R sequences, and has all their loads in flight together.
// MI355X, 1024 sequences of 1536 bf16 channels: 6.9 us, 3.6 TB/s; 0.8 more at one
// sequence a wave; 11.7 with 1535 channels, one a lane.
template <typename T, int V, int KC, int R>
__global__ void __launch_bounds__(64)
seq_conv_step_kernel(SeqConvGeom g, uint32_t ncb, const T* __restrict__ x, const float* __restrict__ w,
                     const float* __restrict__ bias, T* __restrict__ states, T* __restrict__ y) {
  const BlockPos pos = block_pos(ncb);
  const int64_t D = g.q.D, d = (static_cast<int64_t>(pos.cb) * 64 + threadIdx.x) * V;
  if (d >= D) return;
  const int32_t i0 = pos.slot * R;
  StateRows<R> rows;
  rows.load(g.q, i0, x);
  const int32_t(&row)[R] = rows.row;
  Pack<T, V> win[R][KC];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int32_t i = i0 + r < g.q.S ? i0 + r : g.q.S - 1;
    const T* at = states + static_cast<int64_t>(row[r] < 0 ? 0 : row[r]) * (KC - 1) * D + d;
    if (row[r] >= 0) {
#pragma unroll
      for (int k = 0; k < KC - 1; ++k) win[r][k] = load_pack<T, V>(at + k * D);
    }
    win[r][KC - 1] = load_pack<T, V>(x + i * g.xs + d);
  }
  Taps<V, KC> k;
  k.load(w, bias, d, g.w_vec);
  rows.settle(g.q);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (i0 + r >= g.q.S) break;
    Pack<T, V> o;
    if (row[r] < 0) {
#pragma unroll
      for (int v = 0; v < V; ++v) o.v[v] = from_f32<T>(0.f);
      store_pack(y + (i0 + r) * g.ys + d, o);
      continue;
    }
    if (__builtin_amdgcn_readfirstlane(rows.fresh[r]) != 0) {
#pragma unroll
      for (int j = 0; j < KC - 1; ++j)
#pragma unroll
        for (int v = 0; v < V; ++v) win[r][j].v[v] = from_f32<T>(0.f);
    }
    T* at = states + static_cast<int64_t>(row[r]) * (KC - 1) * D + d;
#pragma unroll
    for (int j = 0; j < KC - 1; ++j) store_pack(at + j * D, win[r][j + 1]);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float pre = k.b[v];
#pragma unroll
      for (int j = 0; j < KC; ++j) pre = fmaf(k.w[j][v], to_f32(win[r][j].v[v]), pre);
      o.v[v] = from_f32<T>(pre * sigmoid_f(pre));
    }
    store_pack(y + (i0 + r) * g.ys + d, o);
  }
}

// ----------------------------------------------------------------- launches

// Whether rows can be accessed V values at a time: whole packs in a row, and
// every row of every buffer aligned to them.
SeqConvGeom with_vec(SeqConvGeom g, const float* w, const float* b) {
  g.w_vec = ((reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(b)) & 15) == 0;
  return g;
}
template <typename T, int V>
bool packs(const SeqConvGeom& g, std::initializer_list<const void*> ptrs) {
  bool ok = g.q.D % V == 0 && g.xs % V == 0 && g.ys % V == 0;
  for (const void* p : ptrs) ok = ok && reinterpret_cast<uintptr_t>(p) % (sizeof(T) * V) == 0;
  return ok;
}

template <int V>
uint32_t conv_blocks(const SeqConvGeom& g) { return static_cast<uint32_t>((g.q.D + 64 * V - 1) / (64 * V)); }

// f<T, KC>()
template <typename F>
hipError_t by_width(int dtype, int kc, F&& f) {
  auto typed = [&](auto t) -> hipError_t {
    using T = decltype(t);
    switch (kc) {
      case 1: return f(T{}, std::integral_constant<int, 1>{});
      case 2: return f(T{}, std::integral_constant<int, 2>{});
      case 3: return f(T{}, std::integral_constant<int, 3>{});
      case 4: return f(T{}, std::integral_constant<int, 4>{});
      case 5: return f(T{}, std::integral_constant<int, 5>{});
      case 6: return f(T{}, std::integral_constant<int, 6>{});
      case 7: return f(T{}, std::integral_constant<int, 7>{});
      case 8: return f(T{}, std::integral_constant<int, 8>{});
      default: return hipErrorInvalidValue;
    }
  };
  return dtype == MVM_F32 ? typed(float{}) : typed(bf16_t{});
}

template <typename T, int V, int KC>
hipError_t fwd_v(const SeqConvGeom& g, const void* x, const float* w, const float* b, const void* c0, void* c1, void* y,
                 hipStream_t s) {
  const uint32_t ncb = conv_blocks<V>(g);
  auto run = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(chunk_slots(g.q, conv_cut(g.fwd_pos)) * ncb)), dim3(256), 0,
                       s, g, ncb, static_cast<const T*>(x), w, b, static_cast<const T*>(c0), static_cast<T*>(c1),
                       static_cast<T*>(y));
    return hipGetLastError();
  };
  if constexpr (KC - 1 <= 4) {
    if (g.fwd_pos == 4) return run(seq_conv_fwd_kernel<T, V, KC, 4>);
  }
  return run(seq_conv_fwd_kernel<T, V, KC, 8>);
}

template <typename T, int V, int KC>
hipError_t bwd_v(const SeqConvGeom& g, const void* x, const float* w, const float* b, const void* c0, const void* dy,
                 const void* dc1, void* dx, float* dw, float* db, void* dc0, float* part, hipStream_t s) {
  const uint32_t ncb = conv_blocks<V>(g);
  const int64_t slots = chunk_slots(g.q, conv_cut(g.bwd_pos)), ncols = g.q.D * (KC + 1);
  auto run = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(slots * ncb)), dim3(256), 0, s, g, ncb,
                       static_cast<const T*>(x), w, b, static_cast<const T*>(c0), static_cast<const T*>(dy),
                       static_cast<const T*>(dc1), static_cast<T*>(dx), static_cast<T*>(dc0), part);
    return hipGetLastError();
  };
  const hipError_t e =
      g.bwd_pos == 16 ? run(seq_conv_bwd_kernel<T, V, KC, 16>) : run(seq_conv_bwd_kernel<T, V, KC, 8>);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(seq_conv_reduce_kernel, dim3(static_cast<unsigned>((ncols + 63) / 64)), dim3(1024), 0, s, ncols,
                     static_cast<int32_t>(KC), slots, part, dw, db);
  return hipGetLastError();
}

template <typename T, int V, int KC>
hipError_t step_v(const SeqConvGeom& g, const void* x, const float* w, const float* b, void* states, void* y,
                  hipStream_t s) {
  const uint32_t ncb = conv_blocks<V>(g);
  auto run = [&](auto kernel, int R) {
    hipLaunchKernelGGL(kernel, dim3(ncb * static_cast<unsigned>((g.q.S + R - 1) / R)), dim3(64), 0, s, g, ncb,
                       static_cast<const T*>(x), w, b, static_cast<T*>(states), static_cast<T*>(y));
    return hipGetLastError();
  };
  // bf16: the taps of a lane's eight channels are more than a sequence's rows, so
  // two sequences share them once there is a wave for each SIMD.  MI355X, 1536
  // channels: 64 sequences 3.0 us by two, 2.6 by one; 384 4.6 and 4.6; 2048 10.9
  // and 12.5.  float32 (four channels): 2048 20.4 and 20.1
  if constexpr (V == 8) {
    if (static_cast<int64_t>(g.q.S) * ncb >= 1024) return run(seq_conv_step_kernel<T, V, KC, 2>, 2);
  }
  return run(seq_conv_step_kernel<T, V, KC, 1>, 1);
}

}  // namespace

hipError_t launch_seq_conv_fwd(const SeqConvGeom& geom, const void* x, const float* w, const float* b, const void* c0,
                               void* c1, void* y, int dtype, hipStream_t s) {
  const SeqConvGeom g = with_vec(geom, w, b);
  return by_width(dtype, g.kc, [&](auto t, auto kc) {
    using T = decltype(t);
    constexpr int KC = decltype(kc)::value, V = 16 / sizeof(T);
    return packs<T, V>(g, {x, c0, c1, y}) ? fwd_v<T, V, KC>(g, x, w, b, c0, c1, y, s)
                                          : fwd_v<T, 1, KC>(g, x, w, b, c0, c1, y, s);
  });
}

hipError_t launch_seq_conv_bwd(const SeqConvGeom& geom, const void* x, const float* w, const float* b, const void* c0,
                               const void* dy, const void* dc1, void* dx, float* dw, float* db, void* dc0,
                               float* part, int dtype, hipStream_t s) {
  const SeqConvGeom g = with_vec(geom, w, b);
  return by_width(dtype, g.kc, [&](auto t, auto kc) {
    using T = decltype(t);
    constexpr int KC = decltype(kc)::value;
    // two channels a lane: the whole window and its dpre stay in registers
    return packs<T, 2>(g, {x, c0, dy, dc1, dx, dc0})
               ? bwd_v<T, 2, KC>(g, x, w, b, c0, dy, dc1, dx, dw, db, dc0, part, s)
               : bwd_v<T, 1, KC>(g, x, w, b, c0, dy, dc1, dx, dw, db, dc0, part, s);
  });
}

hipError_t launch_seq_conv_step(const SeqConvGeom& geom, const void* x, const float* w, const float* b, void* states,
                                void* y, int dtype, hipStream_t s) {
  const SeqConvGeom g = with_vec(geom, w, b);
  return by_width(dtype, g.kc, [&](auto t, auto kc) {
    using T = decltype(t);
    constexpr int KC = decltype(kc)::value, V = 16 / sizeof(T);
    return packs<T, V>(g, {x, states, y}) ? step_v<T, V, KC>(g, x, w, b, states, y, s)
                                          : step_v<T, 1, KC>(g, x, w, b, states, y, s);
  });
}

}  // namespace mvm
