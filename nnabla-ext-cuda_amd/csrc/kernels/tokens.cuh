// Building blocks of the transformer-block kernels (RMSNormalization, the
// residual step, 8-bit activation checkpoints): rows of any width read and
// written in 16-byte vectors at element alignment, three storage types, and
// the 8-bit group format.
//
// A thread's columns are the same in every row: vector k * TPR + lane of the
// row, so parameters and column sums stay in its registers from row to row.
// The vector a row ends inside is read and written element by element by its
// one thread; nothing outside the row is touched.
#pragma once

#include "common.cuh"

namespace nblahip {

typedef __bf16 bf16;
typedef __bf16 bf16_native2 __attribute__((ext_vector_type(2)));
typedef float native_f2 __attribute__((ext_vector_type(2)));
template <> struct FullVec<bf16> { static constexpr int value = 8; };

typedef uint32_t any_u4 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t any_u2 __attribute__((ext_vector_type(2), aligned(1)));
typedef uint32_t any_u1 __attribute__((aligned(1)));
typedef float any_f4 __attribute__((ext_vector_type(4), aligned(4)));

// How many of a vector's `vec` columns lie in the `remaining` ones of the row.
__device__ __forceinline__ int columns_left(int64_t remaining, int vec) {
  return remaining >= vec ? vec : remaining > 0 ? static_cast<int>(remaining) : 0;
}
__device__ __forceinline__ int64_t least(int64_t a, int64_t b) { return a < b ? a : b; }

// The element-by-element paths at a row's end are rare.  Hiding their count keeps
// the compiler from working out their masks and addresses ahead of the row loop,
// which costs more registers than the loop itself.
__device__ __forceinline__ int opaque(int n) {
  asm volatile("" : "+v"(n));
  return n;
}

// VEC elements as they are stored: 16 bytes.
struct Packed {
  uint4 v;
};

template <typename T> __device__ __forceinline__ float widen16(uint32_t w, bool high);
template <> __device__ __forceinline__ float widen16<__half>(uint32_t w, bool high) {
  const half2_native h = __builtin_bit_cast(half2_native, w);
  return static_cast<float>(high ? h.y : h.x);
}
template <> __device__ __forceinline__ float widen16<bf16>(uint32_t w, bool high) {
  return __builtin_bit_cast(float, high ? (w & 0xffff0000u) : (w << 16));
}
// Two floats rounded to nearest even and packed (one instruction each on gfx950).
template <typename T> __device__ __forceinline__ uint32_t narrow16(float lo, float hi);
template <> __device__ __forceinline__ uint32_t narrow16<__half>(float lo, float hi) {
  // (The compiler would round a product and sum to float16 at once, by a mixed-
  // precision instruction: another value than that of the float32 result, which it
  // computes beside it where that is needed too.)
  asm("" : "+v"(lo), "+v"(hi));
  const half2_native h = {static_cast<_Float16>(lo), static_cast<_Float16>(hi)};
  return __builtin_bit_cast(uint32_t, h);
}
template <> __device__ __forceinline__ uint32_t narrow16<bf16>(float lo, float hi) {
  const native_f2 f = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, bf16_native2));
}

template <typename T> struct Tok {
  static constexpr int VEC = FullVec<T>::value;

  // The n (clamped to 0 .. VEC) elements at p, zeros behind them.
  static __device__ __forceinline__ Packed load(const T *p, int n) {
    Packed r;
    r.v = make_uint4(0u, 0u, 0u, 0u);
    if (n >= VEC) {
      const any_u4 t = *reinterpret_cast<const any_u4 *>(p);
      r.v = make_uint4(t.x, t.y, t.z, t.w);
    } else if (n > 0) {
      uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int j = 0; j < VEC - 1; ++j) {
        if (j < n) {
          if constexpr (sizeof(T) == 4)
            w[j] = reinterpret_cast<const uint32_t *>(p)[j];
          else
            w[j / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t *>(p)[j]) << (16 * (j & 1));
        }
      }
      r.v = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return r;
  }
  static __device__ __forceinline__ void unpack(const Packed &r, float (&o)[VEC]) {
    const uint32_t w[4] = {r.v.x, r.v.y, r.v.z, r.v.w};
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      if constexpr (sizeof(T) == 4)
        o[j] = __builtin_bit_cast(float, w[j]);
      else
        o[j] = widen16<T>(w[j / 2], j & 1);
    }
  }
  static __device__ __forceinline__ Packed pack(const float (&o)[VEC]) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (sizeof(T) == 4)
        w[j] = __builtin_bit_cast(uint32_t, o[j]);
      else
        w[j] = narrow16<T>(o[2 * j], o[2 * j + 1]);
    }
    Packed r;
    r.v = make_uint4(w[0], w[1], w[2], w[3]);
    return r;
  }
  static __device__ __forceinline__ void store(T *p, int n, const Packed &r) {
    if (n >= VEC) {
      const any_u4 t = {r.v.x, r.v.y, r.v.z, r.v.w};
      __builtin_nontemporal_store(t, reinterpret_cast<any_u4 *>(p));
    } else if (n > 0) {
      n = opaque(n);
      const uint32_t w[4] = {r.v.x, r.v.y, r.v.z, r.v.w};
#pragma unroll
      for (int j = 0; j < VEC - 1; ++j) {
        if (j < n) {
          if constexpr (sizeof(T) == 4)
            reinterpret_cast<uint32_t *>(p)[j] = w[j];
          else
            reinterpret_cast<uint16_t *>(p)[j] = static_cast<uint16_t>(w[j / 2] >> (16 * (j & 1)));
        }
      }
    }
  }
  // Rounds o to the storage type, stores it (onto what is there when add), and
  // leaves the stored values' packed form.
  static __device__ __forceinline__ void put(T *p, int n, const float (&o)[VEC], bool add) {
    if (add) {
      float old[VEC], sum[VEC];
      unpack(load(p, n), old);
#pragma unroll
      for (int j = 0; j < VEC; ++j) sum[j] = old[j] + o[j];
      store(p, n, pack(sum));
    } else {
      store(p, n, pack(o));
    }
  }
};

// VEC float parameters at p (n valid, 0 behind them); a null p stands for ones.
template <int VEC>
__device__ __forceinline__ void load_param(const float *p, int64_t at, int n, float (&o)[VEC]) {
#pragma unroll
  for (int j = 0; j < VEC; ++j) o[j] = 0.f;
  if (!p) {
    n = opaque(n);
#pragma unroll
    for (int j = 0; j < VEC; ++j) o[j] = j < n ? 1.f : 0.f;
  } else {
    p += at;
    if (n >= VEC) {
#pragma unroll
      for (int i = 0; i < VEC / 4; ++i) {
        const any_f4 t = reinterpret_cast<const any_f4 *>(p)[i];
        o[4 * i] = t.x; o[4 * i + 1] = t.y; o[4 * i + 2] = t.z; o[4 * i + 3] = t.w;
      }
    } else if (n > 0) {
      n = opaque(n);
#pragma unroll
      for (int j = 0; j < VEC - 1; ++j)
        if (j < n) o[j] = p[j];
    }
  }
}
// The same for an additive parameter: a null p stands for zeros.
template <int VEC>
__device__ __forceinline__ void load_bias(const float *p, int64_t at, int n, float (&o)[VEC]) {
  if (p) {
    load_param<VEC>(p, at, n, o);
  } else {
#pragma unroll
    for (int j = 0; j < VEC; ++j) o[j] = 0.f;
  }
}

// ---------------------------------------------------------------------------
// 8-bit groups: 32 columns share one scale 2^(code - 127), the least (not
// below 2^-120) at which the group's largest magnitude fits the 8-bit type.  A
// power of two, so that x / scale and q * scale are exact and the one rounding
// is that to 8 bits: off by at most half a step of int8 (2^-7 of the largest
// magnitude at worst, 2^-8 at best) or, for e4m3, 2^-4 of the element (elements
// below 2^-6 of the scale: half the least step).  32 columns keep an outlier
// channel's reach short and cost one byte in 33; they are four lanes of 8
// elements or eight of 4, so the maximum stays inside a lane quad or pair of
// quads.  A group that holds an infinity or NaN has the code 255 and reads back
// as NaN throughout: a wrong number must not look like a right one.
// ---------------------------------------------------------------------------
constexpr int kAct8Group = 32;
enum Act8Format { kAct8None = 0, kAct8Int8 = 1, kAct8E4m3 = 2 };

template <int CTRL> __device__ __forceinline__ uint32_t dpp_u(uint32_t v) {
  return static_cast<uint32_t>(
      __builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xf, 0xf, true));
}

// Largest |v| of the thread's group as float bits (order of the bits = order of
// the magnitudes, infinities and NaN above every number).
template <int VEC> __device__ __forceinline__ uint32_t group_amax(const float (&v)[VEC]) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < VEC; ++j) m = max(m, __builtin_bit_cast(uint32_t, v[j]) & 0x7fffffffu);
  m = max(m, dpp_u<0xB1>(m));
  m = max(m, dpp_u<0x4E>(m));
  if constexpr (VEC == 4) m = max(m, dpp_u<0x141>(m));
  return m;
}

// Packs the thread's VEC values; code: the group's scale code.
template <int VEC>
__device__ __forceinline__ uint2 act8_encode(const float (&v)[VEC], int format, uint32_t &code) {
  const uint32_t amax = group_amax<VEC>(v);
  const bool finite = amax < 0x7f800000u;
  const uint32_t mant = amax & 0x7fffffu;
  int k = static_cast<int>(amax >> 23);
  // int8: 127.5 / 64 = 1.9921875 and above would round to 128; e4m3: above 448 / 256 = 1.75.
  k = format == kAct8Int8 ? k - 133 + (mant >= 0x7f0000u) : k - 135 + (mant > 0x600000u);
  k = max(k, -120);
  code = finite ? static_cast<uint32_t>(k + 127) : 255u;
  const float inv = finite ? __builtin_bit_cast(float, static_cast<uint32_t>(127 - k) << 23) : 0.f;
  uint32_t w[2] = {0u, 0u};
  if (format == kAct8Int8) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      // v * inv is exact; adding 1.5 * 2^23 rounds it to the nearest integer
      // (ties to even) and leaves it, two's complement, in the low byte.
      const uint32_t b = __builtin_bit_cast(uint32_t, fmaf(finite ? v[j] : 0.f, inv, 12582912.f));
      w[j / 4] |= (b & 0xffu) << (8 * (j & 3));
    }
  } else {
#pragma unroll
    for (int j = 0; j < VEC; j += 4) {
      int p = 0;
      p = __builtin_amdgcn_cvt_pk_fp8_f32(finite ? v[j] * inv : 0.f, finite ? v[j + 1] * inv : 0.f,
                                          p, false);
      p = __builtin_amdgcn_cvt_pk_fp8_f32(finite ? v[j + 2] * inv : 0.f,
                                          finite ? v[j + 3] * inv : 0.f, p, true);
      w[j / 4] = static_cast<uint32_t>(p);
    }
  }
  return make_uint2(w[0], w[1]);
}

__device__ __forceinline__ float act8_scale(uint32_t code) {
  return code == 255u ? __builtin_nanf("") : __builtin_bit_cast(float, code << 23);
}

// The numbers that the codes are, without their scale.
template <int VEC>
__device__ __forceinline__ void act8_numbers(uint2 q, int format, float (&o)[VEC]) {
  const uint32_t w[2] = {q.x, q.y};
  if (format == kAct8Int8) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) // (one instruction: conversion of a sign-extended byte)
      o[j] = static_cast<float>(static_cast<int>(static_cast<int8_t>(w[j / 4] >> (8 * (j & 3)))));
  } else {
#pragma unroll
    for (int j = 0; j < VEC; j += 4) {
      const native_f2 a = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w[j / 4]), false);
      const native_f2 b = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w[j / 4]), true);
      o[j] = a.x; o[j + 1] = a.y; o[j + 2] = b.x; o[j + 3] = b.y;
    }
  }
}
template <int VEC>
__device__ __forceinline__ void act8_decode(uint2 q, uint32_t code, int format, float (&o)[VEC]) {
  const float s = act8_scale(code);
  act8_numbers<VEC>(q, format, o);
#pragma unroll
  for (int j = 0; j < VEC; ++j) o[j] *= s;
}

// n of VEC codes at p, zeros behind them.
template <int VEC> __device__ __forceinline__ uint2 act8_load(const uint8_t *p, int n) {
  uint2 r = make_uint2(0u, 0u);
  if (n >= VEC) {
    if constexpr (VEC == 8) {
      const any_u2 t = *reinterpret_cast<const any_u2 *>(p);
      r = make_uint2(t.x, t.y);
    } else {
      r.x = *reinterpret_cast<const any_u1 *>(p);
    }
  } else if (n > 0) {
    uint32_t w[2] = {0u, 0u};
#pragma unroll
    for (int j = 0; j < VEC - 1; ++j)
      if (j < n) w[j / 4] |= static_cast<uint32_t>(p[j]) << (8 * (j & 3));
    r = make_uint2(w[0], w[1]);
  }
  return r;
}
template <int VEC> __device__ __forceinline__ void act8_store(uint8_t *p, int n, uint2 q) {
  if (n >= VEC) {
    if constexpr (VEC == 8) {
      const any_u2 t = {q.x, q.y};
      *reinterpret_cast<any_u2 *>(p) = t;
    } else {
      *reinterpret_cast<any_u1 *>(p) = q.x;
    }
  } else if (n > 0) {
    n = opaque(n);
    const uint32_t w[2] = {q.x, q.y};
#pragma unroll
    for (int j = 0; j < VEC - 1; ++j)
      if (j < n) p[j] = static_cast<uint8_t>(w[j / 4] >> (8 * (j & 3)));
  }
}

// Packs a thread's VEC values of a row into its 8-bit copy: codes at column c,
// the group's scale by the group's first thread.  Every thread of a group must
// be here (threads beyond the row's end with zeros and n <= 0).
template <int VEC>
__device__ __forceinline__ void act8_put(uint8_t *codes, uint8_t *scales, int64_t row, int64_t cols,
                                         int64_t groups, int64_t c, int n, const float (&v)[VEC],
                                         int format) {
  uint32_t code;
  const uint2 q = act8_encode<VEC>(v, format, code);
  act8_store<VEC>(codes + row * cols + c, n, q);
  if (n > 0 && (c & (kAct8Group - 1)) == 0)
    scales[row * groups + c / kAct8Group] = static_cast<uint8_t>(code);
}

} // namespace nblahip
