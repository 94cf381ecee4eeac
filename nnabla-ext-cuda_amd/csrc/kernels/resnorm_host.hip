// Plans, workspaces and C-ABI entry points of RMSNormalization, the residual
// step and the backward passes from 8-bit copies.  Nothing here allocates,
// throws or waits for the device.
#include <algorithm>
#include <initializer_list>

#include "resnorm.hpp"
#include "tokens.cuh"

using namespace nblahip;

namespace {

constexpr int64_t kMaxCols = (1ll << 27) - 1; // the fold's grid: 16 threads per column, fewer than 2^32
constexpr int64_t kGridY = 65535;

hipStream_t as_stream(void *s) { return static_cast<hipStream_t>(s); }
bool dtype_ok(int d) { return d == NBLAHIP_F32 || d == NBLAHIP_F16 || d == NBLAHIP_BF16; }
size_t elem_bytes(int dtype) { return dtype == NBLAHIP_F32 ? 4 : 2; }
bool format_ok(int f) { return f == NBLAHIP_ACT8_INT8 || f == NBLAHIP_ACT8_E4M3; }
int64_t groups_of(int64_t cols) { return (cols + kAct8Group - 1) / kAct8Group; }

// 0: proceed, 1: no rows or no columns, < 0: error.
int check_dims(int64_t rows, int64_t cols) {
  if (rows < 0 || cols < 0) return NBLAHIP_EINVAL;
  if (rows == 0 || cols == 0) return 1;
  if (cols > kMaxCols || rows > (int64_t(1) << 46) / cols) return NBLAHIP_ERANGE;
  return 0;
}

// Pointers of a call.  An output may be an input tensor of the same shape and
// type itself (every kernel reads a row's elements, by the thread that later
// writes them, before it writes the row); any other overlap of an output with
// an input or another output is refused.
struct Range {
  uintptr_t p;
  size_t n;
  bool whole; // may be the same tensor as an output marked whole
};
struct Aliases {
  Range in[16], out[16];
  int n_in = 0, n_out = 0;
  void read(const void *p, size_t n, bool whole = false) {
    if (p && n) in[n_in++] = Range{reinterpret_cast<uintptr_t>(p), n, whole};
  }
  void write(const void *p, size_t n, bool whole = false) {
    if (p && n) out[n_out++] = Range{reinterpret_cast<uintptr_t>(p), n, whole};
  }
  static bool overlap(const Range &a, const Range &b) { return a.p < b.p + b.n && b.p < a.p + a.n; }
  bool bad() const {
    for (int i = 0; i < n_out; ++i) {
      for (int k = 0; k < i; ++k)
        if (overlap(out[i], out[k])) return true;
      for (int k = 0; k < n_in; ++k) {
        if (!overlap(out[i], in[k])) continue;
        if (!(out[i].whole && in[k].whole && out[i].p == in[k].p && out[i].n == in[k].n)) return true;
      }
    }
    return false;
  }
};

constexpr int kCus = 256;

int vec_of(int dtype) { return dtype == NBLAHIP_F32 ? 4 : 8; }

// The layout with just enough threads for the row's vectors, of those that have the
// form (fits); rows longer than any of them, and those of less than a vector, go to
// the kernels for long rows.
template <typename F> void pick_layout(StepPlan &pl, int64_t cols, F fits) {
  const int64_t vec = vec_of(pl.dtype), vectors = (cols + vec - 1) / vec;
  pl.tpr = pl.nv = 0;
  if (cols < vec) return;
  int mode = pl.mode;
#define NBLAHIP_CASE(TPR, NV)                                                \
  if (NV > 1 && mode == kRagged) mode = kAny; /* (one form for both) */      \
  if (pl.tpr == 0 && vectors <= TPR * NV && fits(mode, TPR, NV)) {           \
    pl.mode = mode;                                                          \
    pl.tpr = TPR;                                                            \
    pl.nv = NV;                                                              \
  }
  NBLAHIP_STEP_LAYOUTS(NBLAHIP_CASE)
#undef NBLAHIP_CASE
}

// Whether every address that a 16-byte vector of the tensors (or its 8-bit
// codes) is at is a multiple of the vector's size.
bool whole_vectors(int dtype, int64_t cols, std::initializer_list<const void *> tensors,
                   std::initializer_list<const void *> codes) {
  const int vec = vec_of(dtype);
  if (cols % vec != 0) return false;
  for (const void *p : tensors)
    if (!aligned16(p)) return false;
  for (const void *p : codes)
    if ((reinterpret_cast<uintptr_t>(p) & (vec - 1)) != 0) return false;
  return true;
}

// Runs of rows for the backward: rows that share a gate row are cut into
// chunks_per_gate runs of chunk_rows, so that a run has one gate row and its
// column sums are one partial sum.  (Rounded up: with several gate rows the runs may
// pass the blocks, and some blocks walk two.)
void plan_chunks(StepArgs &a, int64_t gate_rows, int64_t want_chunks, int64_t min_rows) {
  a.rows_per_gate = std::max<int64_t>(1, a.rows / gate_rows);
  int64_t per = std::max<int64_t>(1, (want_chunks + gate_rows - 1) / gate_rows);
  int64_t rows = std::max((a.rows_per_gate + per - 1) / per, std::min(min_rows, a.rows_per_gate));
  a.chunk_rows = std::max<int64_t>(1, rows);
  a.chunks_per_gate = (a.rows_per_gate + a.chunk_rows - 1) / a.chunk_rows;
  a.chunks = a.rows > 0 ? a.chunks_per_gate * gate_rows : 0;
}

int64_t shared_gate_rows(const StepArgs &a, int64_t gate_rows) {
  return a.gate_kind == NBLAHIP_GATE_ROWS ? gate_rows : 1;
}

// The backward's split, and its workspace laid out from `ws` (null: sizes only).
size_t plan_bwd(StepArgs &a, StepPlan &pl, int64_t gate_rows, char *ws) {
  pick_layout(pl, a.cols, [&](int mode, int tpr, int nv) {
    return bwd_row_fits(vec_of(pl.dtype), pl.layer, pl.post, pl.pre, pl.kept8, mode, tpr, nv);
  });
  a.pitch = (a.cols + 7) / 8 * 8;
  if (pl.tpr == 0) {
    plan_chunks(a, gate_rows, std::max<int64_t>(kCus, (a.rows + kLongRun - 1) / kLongRun), 16);
    a.grid = a.chunks;
  } else {
    const int block = bwd_block(pl.tpr);
    const int64_t blocks = kCus * bwd_blocks_per_cu(vec_of(pl.dtype), pl.layer, pl.post, pl.pre, pl.kept8, pl.mode, pl.tpr, pl.nv);
    plan_chunks(a, gate_rows, blocks, block / pl.tpr);
    a.grid = std::min<int64_t>(a.chunks, blocks);
  }
  size_t at = 0;
  auto take = [&](int64_t floats) {
    float *p = ws ? reinterpret_cast<float *>(ws + at) : nullptr;
    at += align_up(static_cast<size_t>(floats) * sizeof(float), 256);
    return p;
  };
  const int sums = pl.layer ? 2 : 1;
  if (pl.tpr == 0) a.row_sums = take(4 * a.rows);
  if (pl.pre) a.part_pre = take(static_cast<int64_t>(a.grid) * sums * a.pitch);
  if (pl.post || a.gate_kind == NBLAHIP_GATE_ROWS) a.part_post = take(a.chunks * sums * a.pitch);
  return at;
}

// ---------------------------------------------------------------------------
// Column sums of the partial sums.  A block takes 32 columns (128 bytes of each
// partial row): 8 threads of 4 columns by 64 rows.  blockIdx.y: 0 / 1 the second
// norm's gamma / beta, 2 / 3 the first norm's (a shared gate's rows multiplied
// in), 4 + g gate row g.  The order of the additions is fixed by the sizes.
// Bound by its launch and the latency of a thread's reads, four at a time: 4 - 6.5
// us for the 2 - 8 MB that most calls leave ([16384, 1024] half with 32 gate rows:
// 6.2), 11 us for two LayerNormalizations of 16384 columns.
// ---------------------------------------------------------------------------
constexpr int kFoldLanes = 8, kFoldRows = 64;

struct FoldArgs {
  const float *part_pre, *part_post, *gate, *gamma_post, *beta_post;
  float *dgamma_pre, *dbeta_pre, *dgamma_post, *dbeta_post, *dgate;
  int64_t n_pre, chunks, chunks_per_gate, gate_rows, cols, pitch;
  unsigned accum;
  int sums;      // 1 or 2 sums per partial row
  int post;      // whether dgate goes through the first norm's parameters
};

__device__ __forceinline__ float4 add4(float4 a, float4 b) {
  return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w);
}

// Sum of n rows at p, `stride` floats apart, at the block's columns; the first
// 8 threads have it.  weight: row r counts times row r / per of it.
__device__ __forceinline__ float4 fold_rows(const float *p, int64_t n, int64_t stride,
                                            const float *weight, int64_t per, int64_t cols, int64_t c,
                                            int nc, float4 *lds) {
  const int row = threadIdx.x / kFoldLanes, lane = threadIdx.x % kFoldLanes;
  // Four rows in float, those in double: a gate row per token leaves a row per token,
  // and equal values added up one by one are rounded the same way each time.
  double sum[4] = {0., 0., 0., 0.};
  const int64_t step = kFoldRows * stride;
  const float *at = p + row * stride + c;
  auto load = [&](int64_t r, const float *from) {
    float4 v = *reinterpret_cast<const float4 *>(from);
    if (weight) {
      float w[4];
      load_param<4>(weight, r / per * cols + c, nc, w);
      v.x *= w[0]; v.y *= w[1]; v.z *= w[2]; v.w *= w[3];
    }
    return v;
  };
  int64_t r = row;
  for (; r + 3 * kFoldRows < n; r += 4 * kFoldRows, at += 4 * step) {
    float4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = load(r + i * kFoldRows, at + i * step);
    const float4 t = add4(add4(v[0], v[1]), add4(v[2], v[3]));
    sum[0] += t.x; sum[1] += t.y; sum[2] += t.z; sum[3] += t.w;
  }
  for (; r < n; r += kFoldRows, at += step) {
    const float4 t = load(r, at);
    sum[0] += t.x; sum[1] += t.y; sum[2] += t.z; sum[3] += t.w;
  }
  float4 s = make_float4(static_cast<float>(sum[0]), static_cast<float>(sum[1]),
                         static_cast<float>(sum[2]), static_cast<float>(sum[3]));
  __syncthreads();
  lds[threadIdx.x] = s;
  __syncthreads();
  if (row < 8) {
    for (int i = 1; i < 8; ++i) s = add4(s, lds[(row + 8 * i) * kFoldLanes + lane]);
  }
  __syncthreads();
  if (row < 8) lds[threadIdx.x] = s;
  __syncthreads();
  if (row == 0) {
    for (int i = 1; i < 8; ++i) s = add4(s, lds[i * kFoldLanes + lane]);
  }
  return s;
}

__device__ __forceinline__ void fold_put(float *out, int64_t c, int nc, float4 v, bool add) {
  if (threadIdx.x >= kFoldLanes) return;
  const float o[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (j < nc) out[c + j] = add ? out[c + j] + o[j] : o[j];
}

__global__ __launch_bounds__(kFoldLanes *kFoldRows) void step_fold_kernel(const FoldArgs a) {
  __shared__ float4 lds[kFoldLanes * kFoldRows];
  const int64_t c = (static_cast<int64_t>(blockIdx.x) * kFoldLanes + threadIdx.x % kFoldLanes) * 4;
  const int64_t cs = least(c, a.pitch - 4); // threads beyond the columns read the last ones
  const int nc = columns_left(a.cols - c, 4);
  const int64_t stride = a.sums * a.pitch;
  if (blockIdx.y < 4) {
    const bool beta = blockIdx.y & 1, first = blockIdx.y >= 2;
    float *out = first ? (beta ? a.dbeta_post : a.dgamma_post) : (beta ? a.dbeta_pre : a.dgamma_pre);
    if (!out) return;
    const float *p = (first ? a.part_post : a.part_pre) + (beta ? a.pitch : 0);
    const float4 s = fold_rows(p, first ? a.chunks : a.n_pre, stride, first ? a.gate : nullptr,
                               a.chunks_per_gate, a.cols, cs, nc, lds);
    fold_put(out, c, nc, s,
             a.accum & (first ? (beta ? NBLAHIP_ACCUM_DBETA_POST : NBLAHIP_ACCUM_DGAMMA_POST)
                              : (beta ? NBLAHIP_ACCUM_DBETA_PRE : NBLAHIP_ACCUM_DGAMMA_PRE)));
    return;
  }
  for (int64_t g = blockIdx.y - 4; g < a.gate_rows; g += gridDim.y - 4) {
    const float *p = a.part_post + g * a.chunks_per_gate * stride;
    const int64_t n = a.chunks > 0 ? a.chunks_per_gate : 0;
    float4 s = fold_rows(p, n, stride, nullptr, 1, a.cols, cs, nc, lds);
    if (a.post) {
      float ga[4], be[4];
      load_param<4>(a.gamma_post, c, nc, ga);
      s.x *= ga[0]; s.y *= ga[1]; s.z *= ga[2]; s.w *= ga[3];
      if (a.sums == 2 && a.beta_post) {
        load_bias<4>(a.beta_post, c, nc, be);
        const float4 t = fold_rows(p + a.pitch, n, stride, nullptr, 1, a.cols, cs, nc, lds);
        s.x = fmaf(t.x, be[0], s.x); s.y = fmaf(t.y, be[1], s.y);
        s.z = fmaf(t.z, be[2], s.z); s.w = fmaf(t.w, be[3], s.w);
      }
    }
    fold_put(a.dgate + g * a.cols, c, nc, s, a.accum & NBLAHIP_ACCUM_DGATE);
  }
}

int launch_fold(const StepArgs &a, const StepPlan &pl, int64_t gate_rows, hipStream_t st) {
  FoldArgs f = {};
  const bool shared = a.gate_kind == NBLAHIP_GATE_ROWS;
  f.part_pre = a.part_pre;
  f.part_post = a.part_post;
  f.gate = shared ? static_cast<const float *>(a.gate) : nullptr;
  f.gamma_post = a.gamma_post;
  f.beta_post = a.beta_post;
  f.dgamma_pre = pl.pre ? a.dgamma_pre : nullptr;
  f.dbeta_pre = pl.pre && pl.layer ? a.dbeta_pre : nullptr;
  f.dgamma_post = pl.post ? a.dgamma_post : nullptr;
  f.dbeta_post = pl.post && pl.layer ? a.dbeta_post : nullptr;
  f.dgate = shared ? static_cast<float *>(a.dgate) : nullptr;
  f.n_pre = a.chunks > 0 ? a.grid : 0;
  f.chunks = a.chunks;
  f.chunks_per_gate = std::max<int64_t>(1, a.chunks_per_gate);
  f.gate_rows = f.dgate ? gate_rows : 0;
  f.cols = a.cols;
  f.pitch = a.pitch;
  f.accum = a.accum;
  f.sums = pl.layer ? 2 : 1;
  f.post = pl.post;
  if (!f.dgamma_pre && !f.dbeta_pre && !f.dgamma_post && !f.dbeta_post && !f.dgate) return 0;
  const int64_t ny = 4 + std::min<int64_t>(f.gate_rows, kGridY - 4);
  const int span = 4 * kFoldLanes;
  const dim3 grid(static_cast<unsigned>((a.cols + span - 1) / span), static_cast<unsigned>(ny));
  NBLAHIP_LAUNCH("step_fold_kernel", step_fold_kernel, grid, dim3(kFoldLanes * kFoldRows), 0, st, f);
  return last_launch_status();
}

int run_fwd(const StepPlan &pl, const StepArgs &a, hipStream_t st) {
  switch (pl.dtype) {
  case NBLAHIP_F32: return launch_step_fwd_f32(pl, a, st);
  case NBLAHIP_F16: return launch_step_fwd_f16(pl, a, st);
  default: return launch_step_fwd_bf16(pl, a, st);
  }
}
int run_bwd(const StepPlan &pl, const StepArgs &a, hipStream_t st) {
  switch (pl.dtype) {
  case NBLAHIP_F32: return pl.kept8 ? launch_step_bwd8_f32(pl, a, st) : launch_step_bwd_f32(pl, a, st);
  case NBLAHIP_F16: return pl.kept8 ? launch_step_bwd8_f16(pl, a, st) : launch_step_bwd_f16(pl, a, st);
  default: return pl.kept8 ? launch_step_bwd8_bf16(pl, a, st) : launch_step_bwd_bf16(pl, a, st);
  }
}

int step_fwd(StepArgs a, StepPlan pl, int64_t gate_rows, hipStream_t st) {
  const int d = check_dims(a.rows, a.cols);
  if (d) return d < 0 ? d : 0;
  if (!a.x || !a.h || (pl.pre && !a.y)) return NBLAHIP_EINVAL;
  if (pl.post && (!a.var_post || (pl.layer && !a.mean_post))) return NBLAHIP_EINVAL;
  if (pl.pre && (!a.var_pre || (pl.layer && !a.mean_pre))) return NBLAHIP_EINVAL;
  if ((a.x8 == nullptr) != (a.x8_scale == nullptr) || (a.h8 == nullptr) != (a.h8_scale == nullptr))
    return NBLAHIP_EINVAL;
  if ((a.x8 || a.h8) && !format_ok(a.format8)) return NBLAHIP_EINVAL;
  if (a.h8 && !pl.pre) return NBLAHIP_EINVAL; // (the backward reads h for the second norm alone)
  if (!a.res) a.res_scale = 0.f;              // (an infinite one must not meet the zeros read for res)
  const size_t n = static_cast<size_t>(a.rows) * a.cols, tb = n * elem_bytes(pl.dtype);
  const size_t pb = 4 * static_cast<size_t>(a.cols), sb = 4 * static_cast<size_t>(a.rows);
  a.groups8 = groups_of(a.cols);
  const size_t qs = static_cast<size_t>(a.rows) * a.groups8;
  Aliases al;
  al.read(a.x, tb, true);
  al.read(a.res, tb, true);
  al.read(a.gate, a.gate_kind == NBLAHIP_GATE_FULL ? tb : gate_rows * pb, a.gate_kind == NBLAHIP_GATE_FULL);
  for (const float *p : {a.gamma_post, a.beta_post, a.gamma_pre, a.beta_pre}) al.read(p, pb);
  al.write(a.h, tb, true);
  if (pl.pre) al.write(a.y, tb, true);
  for (const float *p : {a.mean_post, a.var_post, a.mean_pre, a.var_pre}) al.write(p, sb);
  al.write(a.x8, n);
  al.write(a.h8, n);
  al.write(a.x8_scale, qs);
  al.write(a.h8_scale, qs);
  if (al.bad()) return NBLAHIP_EALIAS;
  pl.mode = a.gate_kind == NBLAHIP_GATE_FULL                                               ? kAny
            : whole_vectors(pl.dtype, a.cols, {a.x, a.res, a.h, a.y}, {a.x8, a.h8}) ? kWhole
                                                                                    : kRagged;
  pick_layout(pl, a.cols, [&](int mode, int, int nv) {
    return fwd_row_fits(vec_of(pl.dtype), pl.layer, pl.post, pl.pre, a.x8 || a.h8, mode, nv);
  });
  gate_rows = shared_gate_rows(a, gate_rows);
  const int block = pl.tpr ? fwd_block(pl.tpr) : 1024;
  const int64_t blocks = kCus * (pl.nv == 4 ? 1 : 2048 / block); // (four vectors: 256 registers a thread)
  plan_chunks(a, gate_rows, blocks, pl.tpr ? block / pl.tpr : 1);
  a.grid = std::min<int64_t>(a.chunks, blocks);
  return run_fwd(pl, a, st);
}

int step_bwd(StepArgs a, StepPlan pl, int64_t gate_rows, void *ws, size_t ws_bytes, hipStream_t st) {
  const int d = check_dims(a.rows, a.cols);
  if (d < 0) return d;
  if (a.cols == 0) return 0;
  const bool reads_x = pl.post || a.gate_kind;
  if (a.rows > 0) {
    if ((reads_x && !a.x) || (pl.pre && (!a.kept_h || !a.dy)) || (!pl.pre && !a.dh)) return NBLAHIP_EINVAL;
    if (pl.post && (!a.var_post || (pl.layer && !a.mean_post))) return NBLAHIP_EINVAL;
    if (pl.pre && (!a.var_pre || (pl.layer && !a.mean_pre))) return NBLAHIP_EINVAL;
    if (pl.kept8 && ((reads_x && !a.kept_x_scale) || (pl.pre && !a.kept_h_scale))) return NBLAHIP_EINVAL;
  }
  if (pl.kept8 && !format_ok(a.format8)) return NBLAHIP_EINVAL;
  gate_rows = shared_gate_rows(a, gate_rows);
  const bool full = a.gate_kind == NBLAHIP_GATE_FULL;
  const bool adds = (a.dx && (a.accum & NBLAHIP_ACCUM_DX)) || (a.dres && (a.accum & NBLAHIP_ACCUM_DRES));
  const bool whole = whole_vectors(pl.dtype, a.cols, {a.dh, a.dy, a.dx, a.dres}, {}) &&
                     (pl.kept8 ? whole_vectors(pl.dtype, a.cols, {}, {a.x, a.kept_h})
                               : whole_vectors(pl.dtype, a.cols, {a.x, a.kept_h}, {}));
  pl.mode = full || adds ? kAny : whole ? kWhole : kRagged;
  const size_t need = plan_bwd(a, pl, gate_rows, static_cast<char *>(ws));
  if (need && (!ws || (reinterpret_cast<uintptr_t>(ws) & 255u) != 0 || ws_bytes < need))
    return NBLAHIP_EWORKSPACE;
  const size_t n = static_cast<size_t>(a.rows) * a.cols, tb = n * elem_bytes(pl.dtype);
  const size_t pb = 4 * static_cast<size_t>(a.cols), sb = 4 * static_cast<size_t>(a.rows);
  const size_t kb = pl.kept8 ? n : tb;
  a.groups8 = groups_of(a.cols);
  const size_t qs = static_cast<size_t>(a.rows) * a.groups8;
  Aliases al;
  if (reads_x) al.read(a.x, kb, !pl.kept8);
  if (pl.pre) al.read(a.kept_h, kb, !pl.kept8);
  if (pl.kept8) {
    if (reads_x) al.read(a.kept_x_scale, qs);
    if (pl.pre) al.read(a.kept_h_scale, qs);
  }
  al.read(a.dh, tb, true);
  if (pl.pre) al.read(a.dy, tb, true);
  al.read(a.gate, full ? tb : gate_rows * pb, full);
  for (const float *p : {a.gamma_post, a.beta_post, a.gamma_pre}) al.read(p, pb);
  for (const float *p : {a.mean_post, a.var_post, a.mean_pre, a.var_pre}) al.read(p, sb);
  al.write(a.dx, tb, true);
  al.write(a.dres, tb, true);
  al.write(a.dgate, full ? tb : gate_rows * pb, full);
  for (const float *p : {a.dgamma_post, a.dbeta_post, a.dgamma_pre, a.dbeta_pre}) al.write(p, pb);
  al.write(ws, need);
  if (al.bad()) return NBLAHIP_EALIAS;
  if (!reads_x) a.x = nullptr;
  if (!pl.pre || !(a.dgamma_pre || a.dbeta_pre)) a.part_pre = nullptr;
  const bool post_sums = (pl.post && (a.dgamma_post || a.dbeta_post)) ||
                         (a.gate_kind == NBLAHIP_GATE_ROWS && a.dgate);
  if (!post_sums) a.part_post = nullptr;
  if (a.rows > 0) {
    if (!a.dx && !a.dres && !(full && a.dgate) && !a.part_pre && !a.part_post) return 0;
    if (const int e = run_bwd(pl, a, st)) return e;
  }
  return launch_fold(a, pl, gate_rows, st);
}

int check_gate(const void *gate, int kind, int64_t gate_rows, int64_t rows) {
  if (kind != NBLAHIP_GATE_NONE && kind != NBLAHIP_GATE_ROWS && kind != NBLAHIP_GATE_FULL) return NBLAHIP_EINVAL;
  if ((gate != nullptr) != (kind != NBLAHIP_GATE_NONE)) return NBLAHIP_EINVAL;
  if (kind == NBLAHIP_GATE_ROWS && (gate_rows <= 0 || rows < 0 || rows % gate_rows != 0)) return NBLAHIP_EINVAL;
  return 0;
}

} // namespace

extern "C" {

int nblahip_rms_fwd(const void *x, const float *gamma, void *y, float *ms, int64_t rows,
                    int64_t cols, float eps, int dtype, void *stream) {
  if (!dtype_ok(dtype)) return NBLAHIP_EINVAL;
  StepPlan pl;
  pl.dtype = dtype;
  pl.post = true;
  StepArgs a;
  a.x = x;
  a.gamma_post = gamma;
  a.h = y;
  a.var_post = ms;
  a.rows = rows;
  a.cols = cols;
  a.eps = eps;
  return step_fwd(a, pl, 1, as_stream(stream));
}

size_t nblahip_rms_bwd_workspace_bytes(int64_t rows, int64_t cols, int dtype) {
  return nblahip_resnorm_bwd_workspace_bytes(rows, cols, NBLAHIP_GATE_NONE, 0, NBLAHIP_NORM_RMS, 1,
                                             0, dtype);
}

// RMSNormalization / LayerNormalization backward: the step with its first norm alone.
static int norm_bwd(const void *x, const uint8_t *scale, int format, const void *dy,
                    const float *gamma, const float *mean, const float *var, void *dx,
                    float *dgamma, float *dbeta, int accum_dx, int accum_dgamma, int accum_dbeta,
                    int64_t rows, int64_t cols, float eps, bool layer, int dtype, void *ws,
                    size_t ws_bytes, void *stream) {
  if (!dtype_ok(dtype)) return NBLAHIP_EINVAL;
  if (rows > 0 && cols > 0 && !dy) return NBLAHIP_EINVAL;
  StepPlan pl;
  pl.dtype = dtype;
  pl.post = true;
  pl.layer = layer;
  pl.kept8 = format != NBLAHIP_ACT8_NONE;
  StepArgs a;
  a.x = x;
  a.kept_x_scale = scale;
  a.format8 = format;
  a.dh = dy;
  a.gamma_post = gamma;
  a.mean_post = const_cast<float *>(mean);
  a.var_post = const_cast<float *>(var);
  a.dx = dx;
  a.dgamma_post = dgamma;
  a.dbeta_post = dbeta;
  a.accum = (accum_dx ? NBLAHIP_ACCUM_DX : 0u) | (accum_dgamma ? NBLAHIP_ACCUM_DGAMMA_POST : 0u) |
            (accum_dbeta ? NBLAHIP_ACCUM_DBETA_POST : 0u);
  a.rows = rows;
  a.cols = cols;
  a.eps = eps;
  return step_bwd(a, pl, 1, ws, ws_bytes, as_stream(stream));
}

int nblahip_rms_bwd(const void *x, const uint8_t *x_scale, int x_format, const void *dy,
                    const float *gamma, const float *ms, void *dx, float *dgamma, int accum_dx,
                    int accum_dgamma, int64_t rows, int64_t cols, float eps, int dtype,
                    void *workspace, size_t workspace_bytes, void *stream) {
  return norm_bwd(x, x_scale, x_format, dy, gamma, nullptr, ms, dx, dgamma, nullptr, accum_dx,
                  accum_dgamma, 0, rows, cols, eps, false, dtype, workspace, workspace_bytes, stream);
}

size_t nblahip_ln_bwd_act8_workspace_bytes(int64_t outer, int64_t reduce, int dtype) {
  return nblahip_resnorm_bwd_workspace_bytes(outer, reduce, NBLAHIP_GATE_NONE, 0, NBLAHIP_NORM_LAYER,
                                             1, 0, dtype);
}

int nblahip_ln_bwd_act8(const void *x8, const uint8_t *x_scale, int x_format, const void *dy,
                        const float *gamma, const float *mean, const float *var, void *dx,
                        float *dgamma, float *dbeta, int accum_dx, int accum_dgamma,
                        int accum_dbeta, int64_t outer, int64_t reduce, float eps, int dtype,
                        void *workspace, size_t workspace_bytes, void *stream) {
  if (!format_ok(x_format)) return NBLAHIP_EINVAL;
  return norm_bwd(x8, x_scale, x_format, dy, gamma, mean, var, dx, dgamma, dbeta, accum_dx,
                  accum_dgamma, accum_dbeta, outer, reduce, eps, true, dtype, workspace,
                  workspace_bytes, stream);
}

int nblahip_resnorm_fwd(const void *x, const void *res, const void *gate, int gate_kind,
                        int64_t gate_rows, const float *gamma_post, const float *beta_post,
                        const float *gamma_pre, const float *beta_pre, void *h, void *y,
                        float *mean_post, float *var_post, float *mean_pre, float *var_pre,
                        void *x8, uint8_t *x8_scale, void *h8, uint8_t *h8_scale, int format8,
                        int64_t rows, int64_t cols, float res_scale, float branch_scale, float eps,
                        int norm, int post, int pre, int dtype, void *stream) {
  if (!dtype_ok(dtype) || (norm != NBLAHIP_NORM_RMS && norm != NBLAHIP_NORM_LAYER) || (!post && !pre))
    return NBLAHIP_EINVAL;
  if (const int e = check_gate(gate, gate_kind, gate_rows, rows)) return e;
  if (norm == NBLAHIP_NORM_RMS && (beta_post || beta_pre)) return NBLAHIP_EINVAL;
  if ((!post && (gamma_post || beta_post)) || (!pre && (gamma_pre || beta_pre))) return NBLAHIP_EINVAL;
  StepPlan pl;
  pl.dtype = dtype;
  pl.layer = norm == NBLAHIP_NORM_LAYER;
  pl.post = post;
  pl.pre = pre;
  StepArgs a;
  a.x = x;
  a.res = res;
  a.gate = gate;
  a.gate_kind = gate_kind;
  a.gamma_post = gamma_post;
  a.beta_post = beta_post;
  a.gamma_pre = gamma_pre;
  a.beta_pre = beta_pre;
  a.h = h;
  a.y = y;
  a.mean_post = post && pl.layer ? mean_post : nullptr;
  a.var_post = post ? var_post : nullptr;
  a.mean_pre = pre && pl.layer ? mean_pre : nullptr;
  a.var_pre = pre ? var_pre : nullptr;
  a.x8 = static_cast<uint8_t *>(x8);
  a.x8_scale = x8_scale;
  a.h8 = static_cast<uint8_t *>(h8);
  a.h8_scale = h8_scale;
  a.format8 = format8;
  a.rows = rows;
  a.cols = cols;
  a.res_scale = res_scale;
  a.branch_scale = branch_scale;
  a.eps = eps;
  return step_fwd(a, pl, gate_rows, as_stream(stream));
}

size_t nblahip_resnorm_bwd_workspace_bytes(int64_t rows, int64_t cols, int gate_kind,
                                           int64_t gate_rows, int norm, int post, int pre,
                                           int dtype) {
  if (!dtype_ok(dtype) || check_dims(rows, cols) != 0) return 0;
  if (gate_kind == NBLAHIP_GATE_ROWS && (gate_rows <= 0 || rows % gate_rows != 0)) return 0;
  StepPlan pl;
  pl.dtype = dtype;
  pl.layer = norm == NBLAHIP_NORM_LAYER;
  pl.post = post;
  pl.pre = pre;
  StepArgs a;
  a.rows = rows;
  a.cols = cols;
  a.gate_kind = gate_kind;
  const int64_t g = shared_gate_rows(a, gate_rows);
  size_t most = 0; // over the forms a call of these sizes may take
  for (const int mode : {kWhole, kRagged, kAny}) {
    for (const bool kept8 : {false, true}) {
      StepArgs b = a;
      StepPlan q = pl;
      q.mode = mode;
      q.kept8 = kept8;
      most = std::max(most, plan_bwd(b, q, g, nullptr));
    }
  }
  return most;
}

int nblahip_resnorm_bwd(const void *x, const uint8_t *x_scale, const void *h, const uint8_t *h_scale,
                        int kept_format, const void *dh, const void *dy, const void *gate,
                        int gate_kind, int64_t gate_rows, const float *gamma_post,
                        const float *beta_post, const float *gamma_pre, const float *mean_post,
                        const float *var_post, const float *mean_pre, const float *var_pre, void *dx,
                        void *dres, void *dgate, float *dgamma_post, float *dbeta_post,
                        float *dgamma_pre, float *dbeta_pre, unsigned accum, int64_t rows,
                        int64_t cols, float res_scale, float branch_scale, float eps, int norm,
                        int post, int pre, int dtype, void *workspace, size_t workspace_bytes,
                        void *stream) {
  if (!dtype_ok(dtype) || (norm != NBLAHIP_NORM_RMS && norm != NBLAHIP_NORM_LAYER) || (!post && !pre))
    return NBLAHIP_EINVAL;
  if (const int e = check_gate(gate, gate_kind, gate_rows, rows)) return e;
  const bool layer = norm == NBLAHIP_NORM_LAYER;
  if (!layer && (beta_post || dbeta_post || dbeta_pre)) return NBLAHIP_EINVAL;
  if (!post && (gamma_post || beta_post || dgamma_post || dbeta_post)) return NBLAHIP_EINVAL;
  if (!pre && (gamma_pre || dgamma_pre || dbeta_pre)) return NBLAHIP_EINVAL;
  if (dgate && !gate) return NBLAHIP_EINVAL;
  StepPlan pl;
  pl.dtype = dtype;
  pl.layer = layer;
  pl.post = post;
  pl.pre = pre;
  pl.kept8 = kept_format != NBLAHIP_ACT8_NONE;
  StepArgs a;
  a.x = x;
  a.kept_x_scale = x_scale;
  a.kept_h = h;
  a.kept_h_scale = h_scale;
  a.format8 = kept_format;
  a.dh = dh;
  a.dy = dy;
  a.gate = gate;
  a.gate_kind = gate_kind;
  a.gamma_post = gamma_post;
  a.beta_post = beta_post;
  a.gamma_pre = gamma_pre;
  a.mean_post = post && layer ? const_cast<float *>(mean_post) : nullptr;
  a.var_post = post ? const_cast<float *>(var_post) : nullptr;
  a.mean_pre = pre && layer ? const_cast<float *>(mean_pre) : nullptr;
  a.var_pre = pre ? const_cast<float *>(var_pre) : nullptr;
  a.dx = dx;
  a.dres = dres;
  a.dgate = dgate;
  a.dgamma_post = dgamma_post;
  a.dbeta_post = dbeta_post;
  a.dgamma_pre = dgamma_pre;
  a.dbeta_pre = dbeta_pre;
  a.accum = accum;
  a.rows = rows;
  a.cols = cols;
  a.res_scale = res_scale;
  a.branch_scale = branch_scale;
  a.eps = eps;
  return step_bwd(a, pl, gate_rows, workspace, workspace_bytes, as_stream(stream));
}

} // extern "C"
