// The residual step on rows of any length: a block per row that passes over it
// once per row sum and once more to write, columns in steps of the block.  Rows
// that fit a block's registers never come here (resnorm_rows.cuh); this is for
// the rest: longer rows, rows of less than a vector, and the few forms that
// bwd_row_fits and fwd_row_fits name.
//
// Bound by HBM and, on the way there, by reading twice: the forward's later
// passes find the row in the caches ([512, 50000] float step of two
// LayerNormalizations 162 us, 2.1 times its bytes' time), the backward's two
// kernels each read every tensor ([2048, 16384] bf16, the same step, 196 - 204 us, 2.6
// times: 74 for the row sums, 109 - 114 for the rest, 11 for the fold).  Rows of less
// than a vector keep one thread of a block busy: [200000, 7] half RMS 980 us forward,
// 1460 backward, where rows of 8 take 13 and 20 (resnorm_rows.cuh).
#pragma once

#include <type_traits>

#include "resnorm.hpp"
#include "tokens.cuh"

namespace nblahip {

constexpr int kLongThreads = 512;

// A thread's share of a row sum: a vector's part in float, the vectors' in double.
// In float the share would be one chain of additions, each of equal values rounded the
// same way: off by 6e-5 for 8192 times 0.1 (a row of 2^22 columns), 2.5e-3 for 2^18.
// One conversion and one addition per vector do not show beside its memory accesses.
template <int N> struct RowShare {
  double s[N] = {};
  __device__ __forceinline__ void add(int i, float v) { s[i] += static_cast<double>(v); }
  __device__ __forceinline__ void get(float (&o)[N]) const {
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = static_cast<float>(s[i]);
  }
};

// Sum of N values over the block; every thread returns the same sums.
template <int N> __device__ __forceinline__ void long_sum(float (&v)[N]) {
  __shared__ float lds[N * (kLongThreads / kWave)];
  lds_barrier();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float w = wave_sum(v[i]);
    if ((threadIdx.x & (kWave - 1)) == 0) lds[i * (kLongThreads / kWave) + threadIdx.x / kWave] = w;
  }
  lds_barrier();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float s = 0.f;
    for (int k = 0; k < kLongThreads / kWave; ++k) s += lds[i * (kLongThreads / kWave) + k];
    v[i] = s;
  }
}

// A row's columns at c of the thread: gate values (ones without a gate).
template <typename T>
__device__ __forceinline__ void load_gate(const StepArgs &a, int64_t row, int64_t c, int n,
                                          float (&g)[Tok<T>::VEC]) {
  if (a.gate_kind == 2)
    Tok<T>::unpack(Tok<T>::load(static_cast<const T *>(a.gate) + row * a.cols + c, n), g);
  else
    load_param<Tok<T>::VEC>(a.gate_kind ? static_cast<const float *>(a.gate) : nullptr,
                            row / a.rows_per_gate * a.cols + c, n, g);
}

// One thread's vector of the step before the second norm.
template <typename T, bool POST>
__device__ __forceinline__ void long_h(const StepArgs &a, int64_t row, int64_t c, int n, float mean,
                                       float rho, float (&h)[Tok<T>::VEC]) {
  constexpr int V = Tok<T>::VEC;
  float g[V], r[V];
  Tok<T>::unpack(Tok<T>::load(static_cast<const T *>(a.x) + row * a.cols + c, n), h);
  if constexpr (POST) {
    float ga[V], be[V];
    load_param<V>(a.gamma_post, c, n, ga);
    load_bias<V>(a.beta_post, c, n, be);
#pragma unroll
    for (int j = 0; j < V; ++j) h[j] = fmaf((h[j] - mean) * rho, ga[j], be[j]);
  }
  load_gate<T>(a, row, c, n, g);
#pragma unroll
  for (int j = 0; j < V; ++j) h[j] = a.branch_scale * g[j] * h[j];
  if (a.res) {
    Tok<T>::unpack(Tok<T>::load(static_cast<const T *>(a.res) + row * a.cols + c, n), r);
#pragma unroll
    for (int j = 0; j < V; ++j) h[j] = fmaf(a.res_scale, r[j], h[j]);
  }
}

// Row moments of f(c, n, v): mean (LN) and variance, or the mean square.
template <int V, bool LN, typename F>
__device__ __forceinline__ void long_moments(int64_t cols, F f, float &mean, float &var) {
  const float inv = 1.f / static_cast<float>(cols);
  mean = 0.f;
  if constexpr (LN) {
    RowShare<1> share;
    for (int64_t c = threadIdx.x * V; c < cols; c += kLongThreads * V) {
      float v[V], t = 0.f;
      f(c, columns_left(cols - c, V), v);
#pragma unroll
      for (int j = 0; j < V; ++j) t += v[j];
      share.add(0, t);
    }
    float s[1];
    share.get(s);
    long_sum<1>(s);
    mean = s[0] * inv;
  }
  RowShare<1> share;
  for (int64_t c = threadIdx.x * V; c < cols; c += kLongThreads * V) {
    float v[V], t = 0.f;
    const int n = columns_left(cols - c, V);
    f(c, n, v);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float d = j < n ? v[j] - mean : 0.f;
      t = fmaf(d, d, t);
    }
    share.add(0, t);
  }
  float s[1];
  share.get(s);
  long_sum<1>(s);
  var = s[0] * inv;
}

template <typename T, bool LN, bool POST, bool PRE>
__global__ __launch_bounds__(kLongThreads) void step_fwd_long_kernel(const StepArgs a) {
  constexpr int V = Tok<T>::VEC;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    float m1 = 0.f, v1 = 0.f, r1 = 1.f, m2 = 0.f, v2 = 0.f, r2 = 1.f;
    if constexpr (POST) {
      long_moments<V, LN>(a.cols, [&](int64_t c, int n, float (&v)[V]) {
        Tok<T>::unpack(Tok<T>::load(static_cast<const T *>(a.x) + row * a.cols + c, n), v);
      }, m1, v1);
      r1 = inv_std(v1, a.eps);
    }
    if constexpr (PRE) {
      long_moments<V, LN>(a.cols, [&](int64_t c, int n, float (&v)[V]) {
        long_h<T, POST>(a, row, c, n, m1, r1, v);
      }, m2, v2);
      r2 = inv_std(v2, a.eps);
    }
    // h, which may be res or x in place, is written after its last read as an input
    const int64_t padded = (a.cols + kLongThreads * V - 1) / (kLongThreads * V) * (kLongThreads * V);
    for (int64_t c = threadIdx.x * V; c < padded; c += kLongThreads * V) {
      const int n = columns_left(a.cols - c, V);
      float h[V];
      if (a.x8) {
        float xv[V];
        Tok<T>::unpack(Tok<T>::load(static_cast<const T *>(a.x) + row * a.cols + c, n), xv);
        act8_put<V>(a.x8, a.x8_scale, row, a.cols, a.groups8, c, n, xv, a.format8);
      }
      long_h<T, POST>(a, row, c, n, m1, r1, h);
      const Packed hp = Tok<T>::pack(h);
      if (a.h8) {
        float hv[V];
        Tok<T>::unpack(hp, hv);
#pragma unroll
        for (int j = 0; j < V; ++j) hv[j] = j < n ? hv[j] : 0.f;
        act8_put<V>(a.h8, a.h8_scale, row, a.cols, a.groups8, c, n, hv, a.format8);
      }
      Tok<T>::store(static_cast<T *>(a.h) + row * a.cols + c, n, hp);
      if constexpr (PRE) {
        float ga[V], be[V];
        load_param<V>(a.gamma_pre, c, n, ga);
        load_bias<V>(a.beta_pre, c, n, be);
#pragma unroll
        for (int j = 0; j < V; ++j) h[j] = fmaf((h[j] - m2) * r2, ga[j], be[j]);
        Tok<T>::store(static_cast<T *>(a.y) + row * a.cols + c, n, Tok<T>::pack(h));
      }
    }
    if (threadIdx.x == 0) {
      if constexpr (POST) {
        if constexpr (LN) a.mean_post[row] = m1;
        a.var_post[row] = v1;
      }
      if constexpr (PRE) {
        if constexpr (LN) a.mean_pre[row] = m2;
        a.var_pre[row] = v2;
      }
    }
  }
}

// A kept tensor's vector: storage type, or an 8-bit copy.
template <typename T, bool Q8>
__device__ __forceinline__ void load_kept(const void *p, const uint8_t *scales, const StepArgs &a,
                                          int64_t row, int64_t c, int n, float (&o)[Tok<T>::VEC]) {
  if constexpr (Q8) {
    const uint32_t code = n > 0 ? scales[row * a.groups8 + c / kAct8Group] : 127u;
    act8_decode<Tok<T>::VEC>(
        act8_load<Tok<T>::VEC>(static_cast<const uint8_t *>(p) + row * a.cols + c, n), code,
        a.format8, o);
#pragma unroll
    for (int j = 0; j < Tok<T>::VEC; ++j) o[j] = j < n ? o[j] : 0.f;
  } else {
    Tok<T>::unpack(Tok<T>::load(static_cast<const T *>(p) + row * a.cols + c, n), o);
  }
}

struct RowMoments {
  float m1 = 0.f, r1 = 1.f, m2 = 0.f, r2 = 1.f;
};
template <bool LN, bool POST, bool PRE>
__device__ __forceinline__ RowMoments load_moments(const StepArgs &a, int64_t row) {
  RowMoments q;
  if constexpr (POST) {
    if constexpr (LN) q.m1 = a.mean_post[row];
    q.r1 = inv_std(a.var_post[row], a.eps);
  }
  if constexpr (PRE) {
    if constexpr (LN) q.m2 = a.mean_pre[row];
    q.r2 = inv_std(a.var_pre[row], a.eps);
  }
  return q;
}

// t = the whole gradient of h at a thread's vector, given the two row means
// s1 = mean(dy gamma), s2 = mean(dy gamma hh); hh the normalized h, dy the
// incoming gradient.
template <typename T, bool LN, bool PRE, bool Q8>
__device__ __forceinline__ void long_dh(const StepArgs &a, int64_t row, int64_t c, int n,
                                        const RowMoments &q, float s1, float s2,
                                        float (&t)[Tok<T>::VEC], float (&hh)[Tok<T>::VEC],
                                        float (&dy)[Tok<T>::VEC]) {
  constexpr int V = Tok<T>::VEC;
#pragma unroll
  for (int j = 0; j < V; ++j) t[j] = hh[j] = dy[j] = 0.f;
  if (a.dh) Tok<T>::unpack(Tok<T>::load(static_cast<const T *>(a.dh) + row * a.cols + c, n), t);
  if constexpr (PRE) {
    float ga[V];
    load_kept<T, Q8>(a.kept_h, a.kept_h_scale, a, row, c, n, hh);
    Tok<T>::unpack(Tok<T>::load(static_cast<const T *>(a.dy) + row * a.cols + c, n), dy);
    load_param<V>(a.gamma_pre, c, n, ga);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      hh[j] = j < n ? (hh[j] - q.m2) * q.r2 : 0.f;
      const float d = dy[j] * ga[j] - s1 - hh[j] * s2;
      t[j] = j < n ? fmaf(q.r2, d, t[j]) : 0.f;
    }
  }
}

// Row sums of the backward: row_sums[row] = {s1, s2, m1, m2}, the two means of
// each norm's backward.  The half RMS step from its tensors is held to the 80
// registers of six waves per SIMD, which it fits; left alone it takes 81 and runs
// five ([700, 40001] 86 -> 90 us).  The other forms of 80 and more would spill.
template <typename T, bool LN, bool Q8>
constexpr int kLongSumsWaves = std::is_same<T, __half>::value && !LN && !Q8 ? 6 : 1;
template <typename T, bool LN, bool POST, bool PRE, bool Q8>
__global__ __launch_bounds__(kLongThreads, (kLongSumsWaves<T, LN, Q8>))
void step_bwd_long_sums_kernel(const StepArgs a) {
  constexpr int V = Tok<T>::VEC;
  const float inv = 1.f / static_cast<float>(a.cols);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const RowMoments q = load_moments<LN, POST, PRE>(a, row);
    float s[2] = {0.f, 0.f}, m[2] = {0.f, 0.f};
    if constexpr (PRE) {
      RowShare<2> share;
      for (int64_t c = threadIdx.x * V; c < a.cols; c += kLongThreads * V) {
        const int n = columns_left(a.cols - c, V);
        float hh[V], dy[V], ga[V], g0 = 0.f, g1 = 0.f;
        load_kept<T, Q8>(a.kept_h, a.kept_h_scale, a, row, c, n, hh);
        Tok<T>::unpack(Tok<T>::load(static_cast<const T *>(a.dy) + row * a.cols + c, n), dy);
        load_param<V>(a.gamma_pre, c, n, ga);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float g = dy[j] * ga[j];
          if constexpr (LN) g0 += g;
          g1 = fmaf(g, j < n ? (hh[j] - q.m2) * q.r2 : 0.f, g1);
        }
        if constexpr (LN) share.add(0, g0);
        share.add(1, g1);
      }
      share.get(s);
      long_sum<2>(s);
      s[0] *= inv;
      s[1] *= inv;
    }
    if constexpr (POST) {
      RowShare<2> share;
      for (int64_t c = threadIdx.x * V; c < a.cols; c += kLongThreads * V) {
        const int n = columns_left(a.cols - c, V);
        float t[V], hh[V], dy[V], xh[V], g[V], ga[V], w0 = 0.f, w1 = 0.f;
        long_dh<T, LN, PRE, Q8>(a, row, c, n, q, s[0], s[1], t, hh, dy);
        load_kept<T, Q8>(a.x, a.kept_x_scale, a, row, c, n, xh);
        load_gate<T>(a, row, c, n, g);
        load_param<V>(a.gamma_post, c, n, ga);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float w = a.branch_scale * t[j] * g[j] * ga[j];
          if constexpr (LN) w0 += w;
          w1 = fmaf(w, j < n ? (xh[j] - q.m1) * q.r1 : 0.f, w1);
        }
        if constexpr (LN) share.add(0, w0);
        share.add(1, w1);
      }
      share.get(m);
      long_sum<2>(m);
      m[0] *= inv;
      m[1] *= inv;
    }
    if (threadIdx.x == 0)
      *reinterpret_cast<float4 *>(a.row_sums + 4 * row) = make_float4(s[0], s[1], m[0], m[1]);
  }
}

// Everything else: a block takes one run of rows with one gate row at
// kLongThreads vectors' worth of columns, writes dx, dres and a full gate's
// gradient, and leaves the run's column sums (of at most kLongRun rows, one after
// another).
template <typename T, bool LN, bool POST, bool PRE, bool Q8>
__global__ __launch_bounds__(kLongThreads) void step_bwd_long_cols_kernel(const StepArgs a) {
  constexpr int V = Tok<T>::VEC;
  const int64_t c = (static_cast<int64_t>(blockIdx.x) * kLongThreads + threadIdx.x) * V;
  if (c >= a.pitch) return;
  const int n = columns_left(a.cols - c, V);
  float ga[V], be[V];
  load_param<V>(POST ? a.gamma_post : nullptr, c, n, ga);
  load_bias<V>(POST ? a.beta_post : nullptr, c, n, be);
  for (int64_t chunk = blockIdx.y; chunk < a.chunks; chunk += gridDim.y) {
    const int64_t group = chunk / a.chunks_per_gate;
    const int64_t first = group * a.rows_per_gate + chunk % a.chunks_per_gate * a.chunk_rows;
    const int64_t last = least(first + a.chunk_rows, (group + 1) * a.rows_per_gate);
    float C[V] = {}, E[V] = {}, A[V] = {}, B[V] = {};
    for (int64_t row = first; row < last; ++row) {
      const RowMoments q = load_moments<LN, POST, PRE>(a, row);
      const float4 s = *reinterpret_cast<const float4 *>(a.row_sums + 4 * row);
      float t[V], hh[V], dy[V], xh[V], g[V], o[V];
      long_dh<T, LN, PRE, Q8>(a, row, c, n, q, s.x, s.y, t, hh, dy);
      load_gate<T>(a, row, c, n, g);
#pragma unroll
      for (int j = 0; j < V; ++j) xh[j] = 0.f;
      if (POST || a.gate_kind) load_kept<T, Q8>(a.x, a.kept_x_scale, a, row, c, n, xh);
      if constexpr (POST) {
#pragma unroll
        for (int j = 0; j < V; ++j) xh[j] = j < n ? (xh[j] - q.m1) * q.r1 : 0.f;
      }
      const int64_t at = row * a.cols + c;
      if (a.dres) {
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = a.res_scale * t[j];
        Tok<T>::put(static_cast<T *>(a.dres) + at, n, o, a.accum & NBLAHIP_ACCUM_DRES);
      }
      if (a.gate_kind == 2 && a.dgate) {
#pragma unroll
        for (int j = 0; j < V; ++j)
          o[j] = a.branch_scale * t[j] * (POST ? fmaf(xh[j], ga[j], be[j]) : xh[j]);
        Tok<T>::put(static_cast<T *>(a.dgate) + at, n, o, a.accum & NBLAHIP_ACCUM_DGATE);
      }
#pragma unroll
      for (int j = 0; j < V; ++j) {
        C[j] = fmaf(dy[j], hh[j], C[j]);
        E[j] += dy[j];
        const float w0 = a.branch_scale * t[j];
        const float w = w0 * g[j];
        const float p = a.gate_kind == 1 ? w0 : w; // a shared gate is multiplied in after the sum
        A[j] = fmaf(p, xh[j], A[j]);
        B[j] += p;
        o[j] = POST ? q.r1 * (w * ga[j] - s.z - xh[j] * s.w) : w;
      }
      if (a.dx) Tok<T>::put(static_cast<T *>(a.dx) + at, n, o, a.accum & NBLAHIP_ACCUM_DX);
    }
    constexpr int S = LN ? 2 : 1;
    if (a.part_pre) {
      float *p = a.part_pre + chunk * S * a.pitch + c;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        p[j] = C[j];
        if constexpr (LN) p[a.pitch + j] = E[j];
      }
    }
    if (a.part_post) {
      float *p = a.part_post + chunk * S * a.pitch + c;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        p[j] = A[j];
        if constexpr (LN) p[a.pitch + j] = B[j];
      }
    }
  }
}

} // namespace nblahip
