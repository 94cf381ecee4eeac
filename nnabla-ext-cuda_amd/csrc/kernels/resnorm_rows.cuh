// The residual step on rows that fit a block at one, two or four 16-byte vectors
// per thread: every tensor crosses HBM once per direction.
//
// TPR threads hold a row; a block takes several rows at a time where they are
// short.  A thread's columns are the same in every row, so the parameters (and,
// backward, the column sums of the parameter gradients) stay in its registers
// while the block walks its rows.  Row sums are float: a thread's columns, its
// wave by DPP, waves through LDS.
//
// What bounds it: HBM (6 tensors of 2 bytes an element backward, 4 forward).
// Forward [16384, 4096] bf16 RMS step 109 us, 4.9 TB/s of the 537 MB (a copy of
// that size: 5.3); [16384, 1024] half LayerNormalization step 25 us, 5.4 TB/s.
// Backward [8192, 8192] bf16 157 us + 5 of the fold, 5.1 TB/s; [16384, 1024] half
// LayerNormalization 44 + 6 us, 4.6 TB/s; from 8 bits [8192, 4096] bf16 72 + 6 us,
// 4.7 TB/s.  [2048, 16384] bf16 (four vectors) forward 56, backward 91 + 9 us.
// Rows that end inside a vector take more instructions and requests: [8191, 4097]
// bf16 backward 103 us, 3.9 TB/s; whole rows of [16384, 4096] reach 5.0 (160 us).
// A row's loads are asked for one row ahead and must stay in flight while the
// row before is worked on and stored.  This GPU counts loads and stores in one
// in-order counter per wave, and the compiler can wait for "all but the last
// n" only where it knows n on every path; after a branch around a load or a
// store it has to wait for everything, the row's own stores included (and keeps
// twice the registers: 170 against 80 in the backward).  So the loop has no such
// branch: every access is a buffer access whose bounds the hardware checks.  An
// absent tensor, a row past the end and a thread past the columns have no
// records in range: loads give 0, stores are dropped.
//
// Three forms (StepMode):
//   kWhole : rows of whole vectors, 16-byte aligned, no gate per element, no
//            accumulation onto dx / dres: the calls models make;
//   kRagged: rows or tensors at any element.  A row that ends inside a vector is
//            read as the vector that ends where the row ends, shifted down, and
//            written in pieces of 8, 4 and 2 bytes; nothing outside the row is
//            written, and nothing read outside the dwords it lies in;
//   kAny   : that, a gate per element and accumulation, whole rows too (absent ones
//            cost loads and stores that the bounds check drops).
#pragma once

#include "resnorm_long.cuh"

namespace nblahip {

// Sums of N values over the TPR threads of a row; every one of them gets the
// sums.  Rows of several waves go through LDS: two buffers taken in turn, so
// that one barrier per sum is enough (a wave writes a buffer again only after
// the barrier of the sum in between, which every wave reaches after its reads).
template <int TPR, int BLOCK, int N> struct RowTotal {
  static constexpr int kFloats = TPR > kWave ? 2 * (BLOCK / kWave) * N : 2;
};

template <int TPR, int N, int CAP>
__device__ __forceinline__ void row_total(float (&v)[N], float (&lds)[CAP], int &turn) {
  if constexpr (TPR < kWave) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = group_sum<TPR>(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = wave_sum(v[i]);
    if constexpr (TPR > kWave) {
      constexpr int W = TPR / kWave;
      const int wave = threadIdx.x / kWave;
      float *buf = lds + turn * (CAP / 2);
      if ((threadIdx.x & (kWave - 1)) == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) buf[wave * N + i] = v[i];
      }
      lds_barrier();
      const float *mine = buf + wave / W * (W * N);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) s += mine[w * N + i];
        v[i] = s;
      }
      turn ^= 1;
    }
  }
}


typedef __amdgpu_buffer_rsrc_t Buffer;
constexpr uint32_t kOutside = 0x7fffffffu; // an offset past every buffer here
constexpr int kStream = 2;                 // non-temporal

// `bytes` bytes at p + off (none where p is null).
__device__ __forceinline__ Buffer buffer(const void *p, int64_t off, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(static_cast<const char *>(p)) + off, 0,
                                           p ? static_cast<int>(bytes) : 0, 0x00020000);
}
// Tensors are stored non-temporally: 134 - 202 MB calls gain 3 - 20 % over ordinary
// stores ([8192, 2560] bf16 pre-norm forward 35.7 -> 28.5 us, [4096, 8192] RMS
// backward 43.4 -> 41.5), the largest up to 4 %; one loses 2 % ([16384, 4096]
// forward).  (Measured with outputs that are not written twice: a loop that
// writes the same buffers again finds them in the cache and shows the opposite.)
__device__ __forceinline__ Packed buffer_load(Buffer b, uint32_t at) {
  const native_u4 t = __builtin_amdgcn_raw_buffer_load_b128(b, at, 0, 0);
  Packed r;
  r.v = make_uint4(t.x, t.y, t.z, t.w);
  return r;
}
__device__ __forceinline__ float buffer_load_float(Buffer b, uint32_t at) {
  return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(b, at, 0, 0));
}
__device__ __forceinline__ void buffer_store(Buffer b, uint32_t at, const Packed &r) {
  const native_u4 t = {r.v.x, r.v.y, r.v.z, r.v.w};
  __builtin_amdgcn_raw_buffer_store_b128(t, b, at, 0, kStream);
}
__device__ __forceinline__ void buffer_store_float(Buffer b, uint32_t at, float v) {
  __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, v), b, at, 0, 0);
}

__device__ __forceinline__ uint4 shift_down_bits(uint4 v, uint32_t bits) {
  uint64_t lo = (static_cast<uint64_t>(v.y) << 32) | v.x;
  uint64_t hi = (static_cast<uint64_t>(v.w) << 32) | v.z;
  const bool far = bits >= 64;
  const uint32_t b = bits & 63u;
  lo = far ? hi : lo;
  hi = far ? 0 : hi;
  lo = (lo >> b) | ((hi << 1) << (63u - b));
  hi >>= b;
  return make_uint4(static_cast<uint32_t>(lo), static_cast<uint32_t>(lo >> 32),
                    static_cast<uint32_t>(hi), static_cast<uint32_t>(hi >> 32));
}

// Makes the compiler finish computing v here: it would otherwise carry both
// factors of a column sum's update to the end of the row.
template <int N> __device__ __forceinline__ void settle(float (&v)[N]) {
#pragma unroll
  for (int j = 0; j < N; ++j) asm volatile("" : "+v"(v[j]));
}

// Threads with four vectors work on them one after another: scheduled together
// they take more registers than there are.
template <int NV> __device__ __forceinline__ void one_vector_at_a_time() {
  if constexpr (NV == 4) __builtin_amdgcn_sched_barrier(0);
}

// Where a thread's NV vectors lie in the rows a block has in hand, in bytes from
// the first of them: of a tensor of the storage type, of 8-bit codes, of their
// scales, of a row statistic.  Of ragged rows the thread a row ends in reads the
// vector `drop` elements further ahead, and writes the first `n` of its own.
template <typename T, int TPR, int BLOCK, int MODE, int NV, bool DWORDS = false> struct Place {
  static constexpr int V = Tok<T>::VEC, W = NV * V;
  static constexpr uint32_t SZ = sizeof(T);
  static constexpr bool RAGGED = MODE != kWhole;
  // DWORDS: 16-bit rows may start in the middle of a dword, where a vector load takes
  // longer; the dwords that hold the vector are loaded, a fifth one where it straddles
  // them, and shifted when the vector is used.
  static constexpr bool HALVES = DWORDS && RAGGED && SZ == 2;
  struct Vec {
    Packed p[NV];
    uint32_t next[HALVES ? NV : 1], odd; // HALVES: the dword behind; bytes of the row's first dword before it
    // Hides the value from the optimiser, so that its widened form is made anew
    // where it is needed instead of being kept in twice the registers.
    __device__ __forceinline__ void pin() {
      if constexpr (SZ == 2) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
          asm volatile("" : "+v"(p[k].v.x), "+v"(p[k].v.y), "+v"(p[k].v.z), "+v"(p[k].v.w));
      }
    }
  };
  uint32_t wide[NV], codes[NV], scale[NV], stat;
  uint32_t drop[NV]; // ragged rows only
  int n[NV];         // columns of the thread's
  __device__ __forceinline__ static int first(int k) { // ... the first of them
    return (k * TPR + static_cast<int>(threadIdx.x % TPR)) * V;
  }
  __device__ __forceinline__ Place(const StepArgs &a) {
    const uint32_t cols = static_cast<uint32_t>(a.cols);
    const uint32_t sub = BLOCK == TPR ? 0 : threadIdx.x / TPR;
    stat = sub * 4;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = first(k);
      n[k] = columns_left(a.cols - c, V);
      drop[k] = RAGGED && n[k] > 0 ? V - n[k] : 0;
      wide[k] = n[k] > 0 ? (sub * cols + c - drop[k]) * SZ : kOutside;
      codes[k] = n[k] > 0 ? sub * cols + c - drop[k] : kOutside;
      scale[k] = n[k] > 0 ? sub * static_cast<uint32_t>(a.groups8) + c / kAct8Group : kOutside;
    }
  }
  // whether element j of the thread's W is a column of the row
  __device__ __forceinline__ bool has(int j) const { return j % V < n[j / V]; }
  __device__ __forceinline__ void param(const float *p, float (&o)[W]) const {
#pragma unroll
    for (int k = 0; k < NV; ++k) load_param<V>(p, first(k), n[k], reinterpret_cast<float(&)[V]>(o[k * V]));
  }
  __device__ __forceinline__ void bias(const float *p, float (&o)[W]) const {
#pragma unroll
    for (int k = 0; k < NV; ++k) load_bias<V>(p, first(k), n[k], reinterpret_cast<float(&)[V]>(o[k * V]));
  }
  __device__ __forceinline__ static void unpack(const Vec &r, float (&o)[W]) {
#pragma unroll
    for (int k = 0; k < NV; ++k) Tok<T>::unpack(r.p[k], reinterpret_cast<float(&)[V]>(o[k * V]));
  }
  __device__ __forceinline__ static Vec pack(const float (&o)[W]) {
    Vec r;
#pragma unroll
    for (int k = 0; k < NV; ++k) r.p[k] = Tok<T>::pack(reinterpret_cast<const float(&)[V]>(o[k * V]));
    return r;
  }
  // The thread's vectors of the `bytes` bytes of rows at p + off, to be settled by
  // fix(): when they are used, so that no load is waited for where it is asked for,
  // unless a form measures otherwise.
  __device__ __forceinline__ Vec load(const void *p, int64_t off, uint32_t bytes) const {
    Vec r;
    if constexpr (HALVES) {
      r.odd = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p) + off) & 2u;
      const Buffer b = buffer(p, off - r.odd, bytes ? (bytes + r.odd + 3u) & ~3u : 0u);
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const uint32_t at = wide[k] < bytes ? wide[k] + r.odd : kOutside;
        r.p[k] = buffer_load(b, at & ~3u);
        r.next[k] = __builtin_amdgcn_raw_buffer_load_b32(b, at & 2u ? at + 14u : kOutside, 0, 0);
      }
    } else {
      const Buffer b = buffer(p, off, bytes);
#pragma unroll
      for (int k = 0; k < NV; ++k) r.p[k] = buffer_load(b, wide[k]);
    }
    return r;
  }
  __device__ __forceinline__ void fix(Vec &r) const {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if constexpr (HALVES) {
        const uint32_t by = ((wide[k] + r.odd) & 2u) * 8u;
        uint4 &v = r.p[k].v;
        v = make_uint4(__builtin_amdgcn_alignbit(v.y, v.x, by), __builtin_amdgcn_alignbit(v.z, v.y, by),
                       __builtin_amdgcn_alignbit(v.w, v.z, by), __builtin_amdgcn_alignbit(r.next[k], v.w, by));
      }
      if constexpr (RAGGED) r.p[k].v = shift_down_bits(r.p[k].v, drop[k] * 8u * SZ);
    }
  }
  // Offset of the first of the thread's own elements, where it starts to write
  // the pieces of a vector that is cut short.
  __device__ __forceinline__ uint32_t own(uint32_t at, int k, uint32_t size) const {
    return n[k] > 0 ? at + drop[k] * size : kOutside;
  }
  __device__ __forceinline__ void store(Buffer b, const Vec &r) const {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if constexpr (!RAGGED) {
        buffer_store(b, wide[k], r.p[k]);
      } else {
        const uint4 v = r.p[k].v;
        buffer_store(b, n[k] == V ? wide[k] : kOutside, r.p[k]);
        const uint32_t left = static_cast<uint32_t>(n[k] < V ? n[k] : 0); // elements still to write
        const uint32_t at = own(wide[k], k, SZ);
        const uint32_t four = left & (8 / SZ), two = left & (4 / SZ);
        const native_u2 t = {v.x, v.y};
        __builtin_amdgcn_raw_buffer_store_b64(t, b, four ? at : kOutside, 0, 0);
        const uint4 q = shift_down_bits(v, four ? 64u : 0u);
        __builtin_amdgcn_raw_buffer_store_b32(q.x, b, two ? at + four * SZ : kOutside, 0, 0);
        if constexpr (SZ == 2) {
          const uint32_t w = two ? q.y : q.x;
          __builtin_amdgcn_raw_buffer_store_b16(static_cast<uint16_t>(w), b,
                                                left & 1u ? at + (four + two) * SZ : kOutside, 0, 0);
        }
      }
    }
  }
  // Rounds o and stores it in the rows at p + off, or adds it to what is there.
  __device__ __forceinline__ void put(void *p, bool add, int64_t off, uint32_t bytes, const float (&o)[W]) const {
    if constexpr (MODE == kAny) {
      float sum[W];
      Vec old = load(add ? p : nullptr, off, bytes);
      fix(old);
      unpack(old, sum);
#pragma unroll
      for (int j = 0; j < W; ++j) sum[j] += o[j];
      store(buffer(p, off, bytes), pack(sum));
    } else {
      store(buffer(p, off, bytes), pack(o));
    }
  }
  __device__ __forceinline__ uint2 load_codes(Buffer b, int k) const {
    uint2 q = make_uint2(0u, 0u);
    if constexpr (V == 8) {
      const native_u2 t = __builtin_amdgcn_raw_buffer_load_b64(b, codes[k], 0, 0);
      q = make_uint2(t.x, t.y);
    } else {
      q.x = __builtin_amdgcn_raw_buffer_load_b32(b, codes[k], 0, 0);
    }
    return q;
  }
  __device__ __forceinline__ void fix_codes(uint2 &q, int k) const {
    if constexpr (RAGGED) {
      const uint64_t v = ((static_cast<uint64_t>(q.y) << 32) | q.x) >> (8u * drop[k]);
      q = make_uint2(static_cast<uint32_t>(v), static_cast<uint32_t>(v >> 32));
    }
  }
  __device__ __forceinline__ void store_codes(Buffer b, uint2 q, int k) const {
    const uint32_t all = !RAGGED || n[k] == V ? codes[k] : kOutside;
    if constexpr (V == 8) {
      const native_u2 t = {q.x, q.y};
      __builtin_amdgcn_raw_buffer_store_b64(t, b, all, 0, 0);
    } else {
      __builtin_amdgcn_raw_buffer_store_b32(q.x, b, all, 0, 0);
    }
    if constexpr (RAGGED) {
      const uint32_t left = static_cast<uint32_t>(n[k] < V ? n[k] : 0), at = own(codes[k], k, 1);
      const uint32_t four = left & 4u, two = left & 2u;
      if constexpr (V == 8) __builtin_amdgcn_raw_buffer_store_b32(q.x, b, four ? at : kOutside, 0, 0);
      const uint32_t w = four ? q.y : q.x;
      __builtin_amdgcn_raw_buffer_store_b16(static_cast<uint16_t>(w), b, two ? at + four : kOutside, 0, 0);
      __builtin_amdgcn_raw_buffer_store_b8(static_cast<uint8_t>(two ? w >> 16 : w), b,
                                           left & 1u ? at + four + two : kOutside, 0, 0);
    }
  }
};

// The factor between the normalized x and its part of h, branch_scale * gate *
// gamma_post (without a norm: branch_scale * gate), at a thread's columns, and
// the same of beta_post.  A gate per element comes in later.
template <bool POST, typename P>
__device__ __forceinline__ void load_branch(const StepArgs &a, int64_t gate_row, const P &pl, float (&k)[P::W]) {
  float g[P::W];
  pl.param(POST ? a.gamma_post : nullptr, k);
  pl.param(a.gate_kind == 1 ? static_cast<const float *>(a.gate) + gate_row * a.cols : nullptr, g);
#pragma unroll
  for (int j = 0; j < P::W; ++j) k[j] *= a.branch_scale * g[j];
}
template <typename P>
__device__ __forceinline__ void load_branch_bias(const StepArgs &a, int64_t gate_row, const P &pl,
                                                 float (&k)[P::W]) {
  float g[P::W];
  pl.bias(a.beta_post, k);
  pl.param(a.gate_kind == 1 ? static_cast<const float *>(a.gate) + gate_row * a.cols : nullptr, g);
#pragma unroll
  for (int j = 0; j < P::W; ++j) k[j] *= a.branch_scale * g[j];
}

// Rows of [base, base + RPB) that lie before `last`.
template <int RPB> __device__ __forceinline__ uint32_t rows_in(int64_t base, int64_t last) {
  const int64_t n = last - base;
  return n >= RPB ? RPB : n > 0 ? static_cast<uint32_t>(n) : 0u;
}

// The second launch bound: waves per SIMD of the blocks a CU has at once.
constexpr int bwd_bound(int vec, bool layer, bool post, bool pre, bool q8, int mode, int tpr, int nv) {
  return (bwd_blocks_per_cu(vec, layer, post, pre, q8, mode, tpr, nv) * bwd_block(tpr) + 255) / 256;
}

// Forward.  A block takes runs of rows (chunks) that share a gate row.
template <typename T, bool LN, bool POST, bool PRE, bool COPY, int MODE, int TPR, int NV>
__global__ __launch_bounds__(fwd_block(TPR)) void step_fwd_rows_kernel(const StepArgs a) {
  using P = Place<T, TPR, fwd_block(TPR), MODE, NV>;
  using Vec = typename P::Vec;
  constexpr int V = P::V, W = P::W;
  constexpr bool OPTIONS = MODE == kAny;
  constexpr int BLOCK = fwd_block(TPR), RPB = BLOCK / TPR, D = fwd_depth(TPR, NV, MODE);
  __shared__ float lds[RowTotal<TPR, BLOCK, 1>::kFloats];
  int turn = 0;
  const P pl(a);
  const uint32_t row_bytes = static_cast<uint32_t>(a.cols) * static_cast<uint32_t>(sizeof(T));
  const float inv = 1.f / static_cast<float>(a.cols);
  const uint32_t stat_out = threadIdx.x % TPR == 0 ? pl.stat : kOutside;
  float gn[W], bn[W], kp[W], kb[W];
  // Two LayerNormalizations at four vectors: the second one's parameters wait in LDS.
  constexpr bool PARK = LN && POST && PRE && W == 32;
  __shared__ float4 park[PARK ? 2 * BLOCK * W / 4 : 1];
  if constexpr (PRE) pl.param(a.gamma_pre, gn);
  if constexpr (PRE && LN) pl.bias(a.beta_pre, bn);
  if constexpr (PARK) {
#pragma unroll
    for (int j = 0; j < W / 4; ++j) {
      park[(2 * j) * BLOCK + threadIdx.x] = make_float4(gn[4 * j], gn[4 * j + 1], gn[4 * j + 2], gn[4 * j + 3]);
      park[(2 * j + 1) * BLOCK + threadIdx.x] = make_float4(bn[4 * j], bn[4 * j + 1], bn[4 * j + 2], bn[4 * j + 3]);
    }
  }
  for (int64_t chunk = blockIdx.x; chunk < a.chunks; chunk += gridDim.x) {
    const int64_t group = chunk / a.chunks_per_gate;
    const int64_t first = group * a.rows_per_gate + chunk % a.chunks_per_gate * a.chunk_rows;
    const int64_t last = least(first + a.chunk_rows, (group + 1) * a.rows_per_gate);
    load_branch<POST>(a, group, pl, kp);
    if constexpr (POST && LN) load_branch_bias(a, group, pl, kb);
    // The form with a third tensor shifts where it asks ([8191, 4097] bf16 with a gate
    // per element 87 us, at the vectors' use 92; LayerNormalization 115 and 123), the
    // others where they use them (float [8191, 2049] 57 us, where they ask 59).
    Vec x[D], r[D], gf[D];
    auto ask = [&](int u, int64_t base) {
      const int64_t off = base * a.cols * static_cast<int64_t>(sizeof(T));
      const uint32_t bytes = rows_in<RPB>(base, last) * row_bytes;
      x[u] = pl.load(a.x, off, bytes);
      r[u] = pl.load(a.res, off, bytes);
      if constexpr (OPTIONS) {
        gf[u] = pl.load(a.gate_kind == 2 ? a.gate : nullptr, off, bytes);
        pl.fix(x[u]);
        pl.fix(r[u]);
        pl.fix(gf[u]);
      }
    };
#pragma unroll
    for (int u = 0; u < D; ++u) ask(u, first + u * RPB);
#pragma unroll 1
    for (int64_t base0 = first; base0 < last; base0 += D * RPB) {
#pragma unroll
     for (int u = 0; u < D; ++u) {
      const int64_t base = base0 + u * RPB;
      if (u > 0 && base >= last) break;
      const uint32_t rows = rows_in<RPB>(base, last), bytes = rows * row_bytes;
      const int64_t off = base * a.cols * static_cast<int64_t>(sizeof(T));
      float h[W], q[W];
      float m1 = 0.f, v1 = 0.f, m2 = 0.f, v2 = 0.f;
      if constexpr (!OPTIONS) {
        pl.fix(x[u]);
        pl.fix(r[u]);
      }
      P::unpack(x[u], h);
      P::unpack(r[u], q);
#pragma unroll
      for (int j = 0; j < W; ++j) q[j] *= a.res_scale;
      auto copy = [&](const float (&v)[W], void *codes, void *scales) {
        const Buffer to = buffer(codes, base * a.cols, rows * static_cast<uint32_t>(a.cols));
        const Buffer of = buffer(scales, base * a.groups8, rows * static_cast<uint32_t>(a.groups8));
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          uint32_t code;
          pl.store_codes(to, act8_encode<V>(reinterpret_cast<const float(&)[V]>(v[k * V]), a.format8, code), k);
          __builtin_amdgcn_raw_buffer_store_b8(static_cast<uint8_t>(code), of,
                                               P::first(k) % kAct8Group == 0 ? pl.scale[k] : kOutside, 0, 0);
        }
      };
      if constexpr (COPY) copy(h, a.x8, a.x8_scale);
      float g[W];
      if constexpr (OPTIONS) {
        P::unpack(gf[u], g);
#pragma unroll
        for (int j = 0; j < W; ++j) g[j] = a.gate_kind == 2 ? g[j] : 1.f;
        settle(g);
      }
      settle(h);
      settle(q);
      ask(u, base + D * RPB);
      auto moments = [&](float &mean, float &var) {
        float s[1] = {0.f};
        if constexpr (LN) {
#pragma unroll
          for (int j = 0; j < W; ++j) s[0] += h[j];
          row_total<TPR, 1>(s, lds, turn);
          mean = s[0] * inv;
        }
        s[0] = 0.f;
#pragma unroll
        for (int j = 0; j < W; ++j) {
          float d = LN ? h[j] - mean : h[j];
          if constexpr (LN && (MODE != kWhole || NV > 1)) d = pl.has(j) ? d : 0.f;
          s[0] = fmaf(d, d, s[0]);
        }
        if constexpr (LN && MODE == kWhole && NV == 1) s[0] = pl.n[0] > 0 ? s[0] : 0.f;
        row_total<TPR, 1>(s, lds, turn);
        var = s[0] * inv;
      };
      float rho = 1.f;
      if constexpr (POST) {
        moments(m1, v1);
        rho = inv_std(v1, a.eps);
      }
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const float xh = (POST && LN ? h[j] - m1 : h[j]) * rho;
        if constexpr (OPTIONS) {
          h[j] = fmaf(POST && LN ? fmaf(xh, kp[j], kb[j]) : xh * kp[j], g[j], q[j]);
        } else {
          if constexpr (POST && LN) q[j] += kb[j];
          h[j] = fmaf(xh, kp[j], q[j]);
        }
      }
      const Vec hp = P::pack(h);
      pl.store(buffer(a.h, off, bytes), hp);
      if constexpr (COPY && PRE) {
        float hv[W];
        P::unpack(hp, hv);
        copy(hv, a.h8, a.h8_scale);
      }
      if constexpr (PRE) {
        moments(m2, v2);
        const float rho2 = inv_std(v2, a.eps);
        float y[W];
#pragma unroll
        for (int j = 0; j < W; ++j) {
          if constexpr (PARK) {
            if (j % 4 == 0) {
              const float4 g = park[(j / 2) * BLOCK + threadIdx.x], b = park[(j / 2 + 1) * BLOCK + threadIdx.x];
              gn[j] = g.x; gn[j + 1] = g.y; gn[j + 2] = g.z; gn[j + 3] = g.w;
              bn[j] = b.x; bn[j + 1] = b.y; bn[j + 2] = b.z; bn[j + 3] = b.w;
            }
          }
          y[j] = LN ? fmaf((h[j] - m2) * rho2, gn[j], bn[j]) : h[j] * rho2 * gn[j];
        }
        pl.store(buffer(a.y, off, bytes), P::pack(y));
      }
      if constexpr (POST) {
        if constexpr (LN) buffer_store_float(buffer(a.mean_post, 4 * base, 4 * rows), stat_out, m1);
        buffer_store_float(buffer(a.var_post, 4 * base, 4 * rows), stat_out, v1);
      }
      if constexpr (PRE) {
        if constexpr (LN) buffer_store_float(buffer(a.mean_pre, 4 * base, 4 * rows), stat_out, m2);
        buffer_store_float(buffer(a.var_pre, 4 * base, 4 * rows), stat_out, v2);
      }
     }
    }
  }
}

// A kept tensor's vectors as they were loaded: storage type, or an 8-bit copy.
template <typename T, bool Q8, typename P> struct Kept {
  static constexpr int V = P::V;
  typename P::Vec p;
  __device__ __forceinline__ void ask(const StepArgs &a, const void *data, const uint8_t *, int64_t base,
                                      uint32_t rows, const P &pl) {
    p = pl.load(data, base * a.cols * static_cast<int64_t>(sizeof(T)),
                rows * static_cast<uint32_t>(a.cols) * static_cast<uint32_t>(sizeof(T)));
  }
  __device__ __forceinline__ void fix(const P &pl) { pl.fix(p); }
  __device__ __forceinline__ void get(const StepArgs &, int k, float (&o)[V]) const {
    Tok<T>::unpack(p.p[k], o);
  }
  // (value - mu) * rho, centred first: value * rho - mu * rho would carry the rounding
  // of mu * rho, 2^-24 of a value far from zero, into the float column sums.
  template <bool CENTRED>
  __device__ __forceinline__ void unit(const StepArgs &a, float mu, float rho, int k, float (&o)[V]) const {
    get(a, k, o);
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = (CENTRED ? o[j] - mu : o[j]) * rho;
  }
  __device__ __forceinline__ void pin() { p.pin(); }
};
template <typename T, typename P> struct Kept<T, true, P> {
  static constexpr int V = P::V, NV = P::W / V;
  uint2 q[NV];
  uint32_t code[NV];
  __device__ __forceinline__ void ask(const StepArgs &a, const void *data, const uint8_t *scales,
                                      int64_t base, uint32_t rows, const P &pl) {
    const Buffer codes = buffer(data, base * a.cols, rows * static_cast<uint32_t>(a.cols));
    const Buffer of = buffer(scales, base * a.groups8, rows * static_cast<uint32_t>(a.groups8));
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      q[k] = pl.load_codes(codes, k);
      code[k] = __builtin_amdgcn_raw_buffer_load_b8(of, pl.scale[k], 0, 0);
    }
  }
  __device__ __forceinline__ void fix(const P &pl) {
#pragma unroll
    for (int k = 0; k < NV; ++k) pl.fix_codes(q[k], k);
  }
  __device__ __forceinline__ void get(const StepArgs &a, int k, float (&o)[V]) const {
    act8_decode<V>(q[k], code[k], a.format8, o);
  }
  // Centred by one fma with the scale (a power of two: the product is exact); without
  // a mean one multiplication takes scale and rho.
  template <bool CENTRED>
  __device__ __forceinline__ void unit(const StepArgs &a, float mu, float rho, int k, float (&o)[V]) const {
    const float scale = CENTRED ? act8_scale(code[k]) : act8_scale(code[k]) * rho;
    act8_numbers<V>(q[k], a.format8, o);
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = CENTRED ? fmaf(o[j], scale, -mu) * rho : o[j] * scale;
  }
  __device__ __forceinline__ void pin() {
#pragma unroll
    for (int k = 0; k < NV; ++k) asm volatile("" : "+v"(q[k].x), "+v"(q[k].y), "+v"(code[k]));
  }
};

// Column sums of one kind for the thread's columns: in registers, or in LDS where
// a block of 1024 threads has none left for them (16 bytes of LDS traffic per
// column and row beside 12 of HBM's, at ten times its rate: it does not show).
template <int W, int TPR, bool IN_LDS> struct ColumnSum {
  float v[W];
  __device__ __forceinline__ void clear(float4 *) {
#pragma unroll
    for (int j = 0; j < W; ++j) v[j] = 0.f;
  }
  __device__ __forceinline__ void add(float4 *, int j, float a, float b) { v[j] = fmaf(a, b, v[j]); }
  template <int V> __device__ __forceinline__ void load(float4 *, int) {}
  template <int V> __device__ __forceinline__ void save(float4 *, int k) {
    settle(reinterpret_cast<float(&)[V]>(v[k * V]));
  }
  __device__ __forceinline__ void get(const float4 *, float (&o)[W]) const {
#pragma unroll
    for (int j = 0; j < W; ++j) o[j] = v[j];
  }
};
template <int W, int TPR> struct ColumnSum<W, TPR, true> {
  float v[W]; // of vector k only between its load and save
  __device__ __forceinline__ void clear(float4 *lds) {
#pragma unroll
    for (int j = 0; j < W / 4; ++j) lds[j * TPR + threadIdx.x] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  template <int V> __device__ __forceinline__ void load(float4 *lds, int k) {
#pragma unroll
    for (int j = k * V / 4; j < (k + 1) * V / 4; ++j) {
      const float4 t = lds[j * TPR + threadIdx.x];
      v[4 * j] = t.x; v[4 * j + 1] = t.y; v[4 * j + 2] = t.z; v[4 * j + 3] = t.w;
    }
  }
  __device__ __forceinline__ void add(float4 *, int j, float a, float b) { v[j] = fmaf(a, b, v[j]); }
  template <int V> __device__ __forceinline__ void save(float4 *lds, int k) {
#pragma unroll
    for (int j = k * V / 4; j < (k + 1) * V / 4; ++j)
      lds[j * TPR + threadIdx.x] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
  }
  __device__ __forceinline__ void get(const float4 *lds, float (&o)[W]) const {
#pragma unroll
    for (int j = 0; j < W / 4; ++j) {
      const float4 t = lds[j * TPR + threadIdx.x];
      o[4 * j] = t.x; o[4 * j + 1] = t.y; o[4 * j + 2] = t.z; o[4 * j + 3] = t.w;
    }
  }
};

// Vector loads in the middle of a dword: worth the dwords and the shifts in the
// backward of wide rows ([8191, 4097] bf16 RMS step 128 -> 109 us, [8191, 2049] 81 ->
// 67), not for two sums per norm (no gain), short rows ([8191, 1023] half 27.7 ->
// 29.5) and in the forward (68 -> 80), whose time the extra instructions are.
constexpr bool bwd_dwords(bool layer, int mode, int tpr) { return !layer && mode == kRagged && tpr >= 192; }

// Backward.  Each input vector is asked for again, for the next row, right
// after its last use.
template <typename T, bool LN, bool POST, bool PRE, bool Q8, int MODE, int TPR, int NV>
__global__ __launch_bounds__(bwd_block(TPR), bwd_bound(Tok<T>::VEC, LN, POST, PRE, Q8, MODE, TPR, NV))
void step_bwd_rows_kernel(const StepArgs a) {
  using P = Place<T, TPR, bwd_block(TPR), MODE, NV, bwd_dwords(LN, MODE, TPR)>;
  using Vec = typename P::Vec;
  constexpr int V = P::V, W = P::W;
  constexpr bool OPTIONS = MODE == kAny;
  constexpr int BLOCK = bwd_block(TPR), RPB = BLOCK / TPR, D = bwd_depth(V, LN, POST, PRE, Q8, MODE, TPR, NV);
  constexpr int S = LN ? 2 : 1; // row sums per norm, column sums per norm
  __shared__ float lds[RowTotal<TPR, BLOCK, S>::kFloats];
  __shared__ float fold[RPB > 1 ? BLOCK * V : 1];
  int turn = 0;
  const P pl(a);
  const uint32_t row_bytes = static_cast<uint32_t>(a.cols) * static_cast<uint32_t>(sizeof(T));
  const float inv = 1.f / static_cast<float>(a.cols);
  float kp[W], gn[W];
  // C, A: sums of gradient times normalized value; E, B: of the gradient (LN)
  // (which of them are in LDS: bwd_sums_in_lds)
  constexpr unsigned IN = bwd_sums_in_lds(W, LN, POST, PRE, Q8, MODE, TPR);
  constexpr int F4 = TPR * W / 4;
  __shared__ float4 c_lds[IN & kSumC ? F4 : 1], e_lds[IN & kSumE ? F4 : 1], a_lds[IN & kSumA ? F4 : 1],
      b_lds[IN & kSumB ? F4 : 1];
  ColumnSum<W, TPR, (IN & kSumC) != 0> C;
  ColumnSum<W, TPR, (IN & kSumE) != 0> E;
  ColumnSum<W, TPR, (IN & kSumA) != 0> A;
  ColumnSum<W, TPR, (IN & kSumB) != 0> B;
  if constexpr (PRE) pl.param(a.gamma_pre, gn);
  C.clear(c_lds);
  E.clear(e_lds);

  struct Row {
    Kept<T, Q8, P> x, h;
    Vec dh, dy, gf;
    float m1, v1, m2, v2;
  } slot[D];
  // Column sums (times `scale`) of the block's rows-at-a-time to `out`; every
  // thread of the block is here.
  auto flush = [&](float *out, const float (&s)[W], float scale) {
    if constexpr (RPB == 1) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        if (P::first(k) < a.pitch) {
#pragma unroll
          for (int j = k * V; j < (k + 1) * V; j += 4)
            *reinterpret_cast<float4 *>(out + P::first(k) + j - k * V) =
                make_float4(s[j] * scale, s[j + 1] * scale, s[j + 2] * scale, s[j + 3] * scale);
        }
      }
    } else {
      lds_barrier();
#pragma unroll
      for (int j = 0; j < V; ++j) fold[j * BLOCK + threadIdx.x] = s[j];
      lds_barrier();
      // the block over the TPR * V columns of the tile, RPB values each
      for (int i = threadIdx.x; i < TPR * V; i += BLOCK) {
        const int j = i / TPR, l = i % TPR;
        float t = 0.f;
#pragma unroll
        for (int q = 0; q < RPB; ++q) t += fold[j * BLOCK + q * TPR + l];
        if (l * V + j < a.pitch) out[l * V + j] = t * scale;
      }
    }
  };

  for (int64_t chunk = blockIdx.x; chunk < a.chunks; chunk += gridDim.x) {
    const int64_t group = chunk / a.chunks_per_gate;
    const int64_t first = group * a.rows_per_gate + chunk % a.chunks_per_gate * a.chunk_rows;
    const int64_t last = least(first + a.chunk_rows, (group + 1) * a.rows_per_gate);
    A.clear(a_lds);
    B.clear(b_lds);
    load_branch<POST>(a, group, pl, kp);
    auto ask_pre = [&](Row &r, int64_t base) {
      const uint32_t rows = rows_in<RPB>(base, last);
      const int64_t off = base * a.cols * static_cast<int64_t>(sizeof(T));
      if constexpr (PRE) {
        r.h.ask(a, a.kept_h, a.kept_h_scale, base, rows, pl);
        r.dy = pl.load(a.dy, off, rows * row_bytes);
        if constexpr (LN) r.m2 = buffer_load_float(buffer(a.mean_pre, 4 * base, 4 * rows), pl.stat);
        r.v2 = buffer_load_float(buffer(a.var_pre, 4 * base, 4 * rows), pl.stat);
      }
      r.dh = pl.load(a.dh, off, rows * row_bytes);
    };
    auto ask_post = [&](Row &r, int64_t base) {
      const uint32_t rows = rows_in<RPB>(base, last);
      r.x.ask(a, a.x, a.kept_x_scale, base, rows, pl);
      if constexpr (OPTIONS)
        r.gf = pl.load(a.gate_kind == 2 ? a.gate : nullptr, base * a.cols * static_cast<int64_t>(sizeof(T)),
                       rows * row_bytes);
      if constexpr (POST) {
        if constexpr (LN) r.m1 = buffer_load_float(buffer(a.mean_post, 4 * base, 4 * rows), pl.stat);
        r.v1 = buffer_load_float(buffer(a.var_post, 4 * base, 4 * rows), pl.stat);
      }
    };
#pragma unroll
    for (int u = 0; u < D; ++u) {
      ask_pre(slot[u], first + u * RPB);
      ask_post(slot[u], first + u * RPB);
    }
#pragma unroll 1
    for (int64_t base0 = first; base0 < last; base0 += D * RPB) {
#pragma unroll
     for (int u = 0; u < D; ++u) {
      const int64_t base = base0 + u * RPB;
      if (u > 0 && base >= last) break;
      Row &r = slot[u];
      const uint32_t rows = rows_in<RPB>(base, last);
      const int64_t off = base * a.cols * static_cast<int64_t>(sizeof(T));
      const bool in = RPB == 1 || pl.stat < 4 * rows;
      float t[W];
      if constexpr (PRE) {
        const float rho = in ? inv_std(r.v2, a.eps) : 0.f, mu = r.m2;
        float s[S];
        r.h.fix(pl);
        pl.fix(r.dy);
#pragma unroll
        for (int i = 0; i < S; ++i) s[i] = 0.f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          float hh[V], d[V];
          r.h.template unit<LN>(a, mu, rho, k, hh);
          Tok<T>::unpack(r.dy.p[k], d);
          C.template load<V>(c_lds, k);
          if constexpr (LN) E.template load<V>(e_lds, k);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            C.add(c_lds, k * V + j, d[j], hh[j]);
            if constexpr (LN) E.add(e_lds, k * V + j, d[j], 1.f);
            d[j] *= gn[k * V + j];
            if constexpr (LN) s[S - 1] += d[j];
            s[0] = fmaf(d[j], hh[j], s[0]);
          }
          C.template save<V>(c_lds, k);
          if constexpr (LN) E.template save<V>(e_lds, k);
          one_vector_at_a_time<NV>();
        }
        r.h.pin();
        r.dy.pin();
        row_total<TPR, S>(s, lds, turn);
        const float s2 = s[0] * inv, s1 = LN ? s[S - 1] * inv : 0.f;
        pl.fix(r.dh);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          float hh[V], d[V], g[V];
          r.h.template unit<LN>(a, mu, rho, k, hh);
          Tok<T>::unpack(r.dy.p[k], d);
          Tok<T>::unpack(r.dh.p[k], g);
#pragma unroll
          for (int j = 0; j < V; ++j)
            t[k * V + j] = fmaf(rho, fmaf(d[j], gn[k * V + j], -(LN ? fmaf(hh[j], s2, s1) : hh[j] * s2)), g[j]);
          one_vector_at_a_time<NV>();
        }
      } else {
        pl.fix(r.dh);
        P::unpack(r.dh, t);
      }
      settle(t);
      ask_pre(r, base + D * RPB);
      {
        float o[W];
#pragma unroll
        for (int j = 0; j < W; ++j) o[j] = a.res_scale * t[j];
        pl.put(a.dres, a.accum & NBLAHIP_ACCUM_DRES, off, rows * row_bytes, o);
      }
      const float rho = POST ? in ? inv_std(r.v1, a.eps) : 0.f : 1.f, mu = POST ? r.m1 : 0.f;
      float m[S], xh[W];
      r.x.fix(pl);
#pragma unroll
      for (int i = 0; i < S; ++i) m[i] = 0.f;
      auto get_x = [&](int k) {
        float(&o)[V] = reinterpret_cast<float(&)[V]>(xh[k * V]);
        if constexpr (POST)
          r.x.template unit<LN>(a, mu, rho, k, o);
        else
          r.x.get(a, k, o);
      };
      if constexpr (OPTIONS) {
#pragma unroll
        for (int k = 0; k < NV; ++k) get_x(k);
        const bool full = a.gate_kind == 2;
        float g[W];
        if constexpr (POST && LN) pl.bias(full ? a.beta_post : nullptr, g);
#pragma unroll
        for (int j = 0; j < W; ++j)
          g[j] = t[j] * (POST && LN ? fmaf(xh[j], kp[j], a.branch_scale * g[j]) : xh[j] * kp[j]);
        pl.put(full ? a.dgate : nullptr, a.accum & NBLAHIP_ACCUM_DGATE, off, rows * row_bytes, g);
        pl.fix(r.gf);
        P::unpack(r.gf, g);
#pragma unroll
        for (int j = 0; j < W; ++j) t[j] *= full ? g[j] : 1.f;
      }
      // branch_scale and a shared gate are multiplied in after the column sums
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        if constexpr (!OPTIONS) get_x(k);
        A.template load<V>(a_lds, k);
        if constexpr (LN && POST) B.template load<V>(b_lds, k);
#pragma unroll
        for (int j = k * V; j < (k + 1) * V; ++j) {
          A.add(a_lds, j, t[j], xh[j]);
          if constexpr (LN && POST) B.add(b_lds, j, t[j], 1.f);
          t[j] *= kp[j];
          if constexpr (POST) {
            if constexpr (LN) m[S - 1] += t[j];
            m[0] = fmaf(t[j], xh[j], m[0]);
          }
        }
        A.template save<V>(a_lds, k);
        if constexpr (LN && POST) B.template save<V>(b_lds, k);
        one_vector_at_a_time<NV>();
      }
      // (Columns beyond the row's end carry finite leftovers here; their gamma is
      // zero, so no row sum has them, and no sum or element of theirs is stored.)
      if constexpr (POST) {
        if constexpr (PRE) r.x.pin(); // (the first norm alone has registers to keep xh)
        row_total<TPR, S>(m, lds, turn);
        const float s2 = m[0] * inv, s1 = LN ? m[S - 1] * inv : 0.f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          if constexpr (PRE) get_x(k);
#pragma unroll
          for (int j = k * V; j < (k + 1) * V; ++j)
            t[j] = rho * (t[j] - (LN ? fmaf(xh[j], s2, s1) : xh[j] * s2));
          one_vector_at_a_time<NV>();
        }
      }
      settle(t);
      ask_post(r, base + D * RPB);
      pl.put(a.dx, a.accum & NBLAHIP_ACCUM_DX, off, rows * row_bytes, t);
     }
    }
    if (a.part_post) {
      float *out = a.part_post + chunk * S * a.pitch;
      float s[W];
      A.get(a_lds, s);
      flush(out, s, a.branch_scale);
      if constexpr (LN) {
        B.get(b_lds, s);
        flush(out + a.pitch, s, a.branch_scale);
      }
    }
  }
  if (PRE && a.part_pre) {
    float *out = a.part_pre + static_cast<int64_t>(blockIdx.x) * S * a.pitch;
    float s[W];
    C.get(c_lds, s);
    flush(out, s, 1.f);
    if constexpr (LN) {
      E.get(e_lds, s);
      flush(out + a.pitch, s, 1.f);
    }
  }
}

} // namespace nblahip
