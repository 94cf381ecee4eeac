// 8-bit copies of activations: packing and reading back.
//
// Both directions are copies with a conversion, bound by HBM (2 + 33/32 bytes
// an element for half data): [16384, 4096] bf16 packs in 31.6 us and is read back
// in 29.0, 6.4 and 7.0 TB/s of the 203 MB (a copy of that size: 8).  A thread
// moves vectors of 16 bytes on the wide side, four of them in flight; the four or
// eight threads of a 32-column group share its scale.  Rows of a whole number of
// groups are one long row; others are padded to groups, so that no group crosses
// a row's end.
#include <algorithm>

#include "launch.hpp"
#include "tokens.cuh"

namespace nblahip {
namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;

struct Act8Args {
  const void *in;
  void *out;
  const uint8_t *scales_in;
  uint8_t *scales_out;
  int64_t rows, cols, groups; // after rows of whole groups have been joined
  int64_t vectors;            // of all rows, each padded to whole groups
  uint32_t row_vectors;       // per padded row (rows == 1: unused)
  FastDiv div;
  int format;
};

struct At {
  int64_t row, c;
  int n;
};
// The vector `v` of the padded rows; `row0`, `off0`: those of the block's first.
template <int VEC>
__device__ __forceinline__ At locate(const Act8Args &a, int64_t v, int64_t v0, int64_t row0,
                                     uint32_t off0) {
  At t;
  if (a.rows == 1) {
    t.row = 0;
    t.c = v * VEC;
  } else {
    const uint32_t w = off0 + static_cast<uint32_t>(v - v0);
    const uint32_t r = a.div.div(w);
    t.row = row0 + r;
    t.c = static_cast<int64_t>(w - r * a.row_vectors) * VEC;
  }
  t.n = v < a.vectors ? columns_left(a.cols - t.c, VEC) : 0;
  return t;
}

template <typename T> __global__ __launch_bounds__(kThreads) void act8_pack_kernel(const Act8Args a) {
  constexpr int V = Tok<T>::VEC;
  const int64_t v0 = static_cast<int64_t>(blockIdx.x) * (kThreads * kUnroll);
  int64_t row0 = 0;
  uint32_t off0 = 0;
  if (a.rows != 1) {
    row0 = v0 / a.row_vectors;
    off0 = static_cast<uint32_t>(v0 - row0 * a.row_vectors);
  }
  At at[kUnroll];
  Packed p[kUnroll];
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
    at[i] = locate<V>(a, v0 + i * kThreads + threadIdx.x, v0, row0, off0);
    p[i] = Tok<T>::load(static_cast<const T *>(a.in) + at[i].row * a.cols + at[i].c, at[i].n);
  }
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
    float x[V];
    Tok<T>::unpack(p[i], x);
    act8_put<V>(static_cast<uint8_t *>(a.out), a.scales_out, at[i].row, a.cols, a.groups, at[i].c,
                at[i].n, x, a.format);
  }
}

template <typename T> __global__ __launch_bounds__(kThreads) void act8_unpack_kernel(const Act8Args a) {
  constexpr int V = Tok<T>::VEC;
  const int64_t v0 = static_cast<int64_t>(blockIdx.x) * (kThreads * kUnroll);
  int64_t row0 = 0;
  uint32_t off0 = 0;
  if (a.rows != 1) {
    row0 = v0 / a.row_vectors;
    off0 = static_cast<uint32_t>(v0 - row0 * a.row_vectors);
  }
  At at[kUnroll];
  uint2 q[kUnroll];
  uint32_t code[kUnroll];
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
    at[i] = locate<V>(a, v0 + i * kThreads + threadIdx.x, v0, row0, off0);
    q[i] = act8_load<V>(static_cast<const uint8_t *>(a.in) + at[i].row * a.cols + at[i].c, at[i].n);
    code[i] = at[i].n > 0 ? a.scales_in[at[i].row * a.groups + at[i].c / kAct8Group] : 127u;
  }
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
    float x[V];
    act8_decode<V>(q[i], code[i], a.format, x);
    Tok<T>::store(static_cast<T *>(a.out) + at[i].row * a.cols + at[i].c, at[i].n, Tok<T>::pack(x));
  }
}

template <typename T> int launch(Act8Args a, bool pack, hipStream_t st) {
  constexpr int V = Tok<T>::VEC;
  if (a.cols % kAct8Group == 0) {
    a.cols *= a.rows;
    a.groups = a.cols / kAct8Group;
    a.rows = 1;
  }
  const int64_t per_row = a.groups * (kAct8Group / V);
  a.row_vectors = static_cast<uint32_t>(per_row);
  a.vectors = a.rows * per_row;
  a.div = a.rows == 1 ? FastDiv(1) : FastDiv(a.row_vectors);
  const int64_t blocks = (a.vectors + kThreads * kUnroll - 1) / (kThreads * kUnroll);
  if (blocks >= (int64_t(1) << 24)) return NBLAHIP_ERANGE; // fewer than 2^32 threads
  const dim3 grid(static_cast<unsigned>(blocks));
  if (pack) {
    NBLAHIP_LAUNCH("act8_pack_kernel", act8_pack_kernel<T>, grid, dim3(kThreads), 0, st, a);
  } else {
    NBLAHIP_LAUNCH("act8_unpack_kernel", act8_unpack_kernel<T>, grid, dim3(kThreads), 0, st, a);
  }
  return last_launch_status();
}

bool overlap(const void *a, size_t an, const void *b, size_t bn) {
  const uintptr_t p = reinterpret_cast<uintptr_t>(a), q = reinterpret_cast<uintptr_t>(b);
  return p < q + bn && q < p + an;
}

int run(const void *wide, const void *codes, const void *scales, int64_t rows, int64_t cols, int format,
        int dtype, bool pack, void *stream) {
  if (dtype != NBLAHIP_F32 && dtype != NBLAHIP_F16 && dtype != NBLAHIP_BF16) return NBLAHIP_EINVAL;
  if (format != NBLAHIP_ACT8_INT8 && format != NBLAHIP_ACT8_E4M3) return NBLAHIP_EINVAL;
  if (rows < 0 || cols < 0) return NBLAHIP_EINVAL;
  if (rows == 0 || cols == 0) return 0;
  if (cols >= (int64_t(1) << 27) || rows > (int64_t(1) << 46) / cols) return NBLAHIP_ERANGE;
  if (!wide || !codes || !scales) return NBLAHIP_EINVAL;
  Act8Args a;
  a.rows = rows;
  a.cols = cols;
  a.groups = (cols + kAct8Group - 1) / kAct8Group;
  a.format = format;
  const size_t n = static_cast<size_t>(rows) * cols, s = static_cast<size_t>(rows) * a.groups;
  const size_t w = n * (dtype == NBLAHIP_F32 ? 4 : 2);
  if (overlap(wide, w, codes, n) || overlap(wide, w, scales, s) || overlap(codes, n, scales, s))
    return NBLAHIP_EALIAS;
  a.in = pack ? wide : codes;
  a.out = const_cast<void *>(pack ? codes : wide);
  a.scales_in = static_cast<const uint8_t *>(scales);
  a.scales_out = static_cast<uint8_t *>(const_cast<void *>(scales));
  const hipStream_t st = static_cast<hipStream_t>(stream);
  switch (dtype) {
  case NBLAHIP_F32: return launch<float>(a, pack, st);
  case NBLAHIP_F16: return launch<__half>(a, pack, st);
  default: return launch<bf16>(a, pack, st);
  }
}

} // namespace
} // namespace nblahip

extern "C" {

int64_t nblahip_act8_scales_per_row(int64_t cols) {
  return cols <= 0 ? 0 : (cols + nblahip::kAct8Group - 1) / nblahip::kAct8Group;
}

int nblahip_act8_pack(const void *x, void *codes, uint8_t *scales, int64_t rows, int64_t cols,
                      int format, int dtype, void *stream) {
  return nblahip::run(x, codes, scales, rows, cols, format, dtype, true, stream);
}

int nblahip_act8_unpack(const void *codes, const uint8_t *scales, void *x, int64_t rows,
                        int64_t cols, int format, int dtype, void *stream) {
  return nblahip::run(x, codes, scales, rows, cols, format, dtype, false, stream);
}

} // extern "C"
