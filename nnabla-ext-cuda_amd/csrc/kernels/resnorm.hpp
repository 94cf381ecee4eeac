// The residual step and the row norms of transformer blocks: problem
// description and launch functions (resnorm_host.hip plans, the units
// resnorm_fwd_*.hip and resnorm_bwd_*.hip hold the kernels).
#pragma once

#include "launch.hpp"

namespace nblahip {

// One step of `rows` rows of `cols` columns:
//   u = post ? norm(x; gamma_post, beta_post) : x
//   h = res_scale * res + branch_scale * gate * u
//   y = pre ? norm(h; gamma_pre, beta_pre) : none
// RMSNormalization is the step with post alone, no residual and no gate.
struct StepArgs {
  const void *x = nullptr;       // block output; backward: as kept (storage type or 8 bits)
  const void *res = nullptr;
  const void *gate = nullptr;    // gate_kind 1: float [gate_rows, cols]; 2: storage type [rows, cols]
  const float *gamma_post = nullptr, *beta_post = nullptr;
  const float *gamma_pre = nullptr, *beta_pre = nullptr;
  void *h = nullptr, *y = nullptr;                     // forward: out
  float *mean_post = nullptr, *var_post = nullptr;     // forward: out; backward: in
  float *mean_pre = nullptr, *var_pre = nullptr;
  uint8_t *x8 = nullptr, *x8_scale = nullptr;          // forward: 8-bit copies out
  uint8_t *h8 = nullptr, *h8_scale = nullptr;
  // backward
  const void *kept_h = nullptr;
  const uint8_t *kept_x_scale = nullptr, *kept_h_scale = nullptr; // 8-bit copies' scales
  const void *dh = nullptr, *dy = nullptr;
  void *dx = nullptr, *dres = nullptr, *dgate = nullptr; // dgate: float for gate_kind 1
  float *dgamma_post = nullptr, *dbeta_post = nullptr;
  float *dgamma_pre = nullptr, *dbeta_pre = nullptr;
  unsigned accum = 0;            // NBLAHIP_ACCUM_*
  float *row_sums = nullptr;     // workspace, long rows: [rows][4]
  float *part_pre = nullptr;     // workspace: [blocks][1 or 2][pitch]
  float *part_post = nullptr;    // workspace: [chunks][1 or 2][pitch]
  int64_t rows = 0, cols = 0;
  int64_t pitch = 0;             // floats between rows of the partial sums
  int64_t rows_per_gate = 1;
  int64_t chunk_rows = 1, chunks_per_gate = 1, chunks = 1; // backward: runs of rows with one gate row
  int64_t groups8 = 0;           // 8-bit groups per row
  int gate_kind = 0;
  int format8 = 0;
  int64_t grid = 1;              // row kernels: blocks launched; backward: rows of part_pre
  float res_scale = 1.f, branch_scale = 1.f, eps = 0.f;
};

// Most rows whose column sums one thread of the kernels for long rows adds up, one
// after another in float: rows of less than a vector come by the million, and equal
// values are rounded the same way each time (8192 times 0.1: 6e-5 off; 256: 2e-6).
constexpr int64_t kLongRun = 256;

// Forms of the row kernels (resnorm_rows.cuh).
enum StepMode { kWhole = 0, kRagged = 1, kAny = 2 };

// What selects a kernel.
struct StepPlan {
  int dtype = 0;
  bool layer = false, post = false, pre = false;
  bool kept8 = false;            // backward: x and h are 8-bit copies
  int mode = 0;                  // StepMode
  int tpr = 0, nv = 0;           // layout; 0: the kernels for long rows
};

// Layouts of the kernels that keep a row in registers: threads per row, 16-byte
// vectors per thread.
#define NBLAHIP_STEP_LAYOUTS(CASE)                                                            \
  CASE(16, 1) CASE(32, 1) CASE(64, 1) CASE(128, 1) CASE(192, 1) CASE(256, 1) CASE(384, 1)     \
  CASE(512, 1) CASE(640, 1) CASE(768, 1) CASE(1024, 1) CASE(1024, 2) CASE(512, 4)

// Threads of a block.  Backward: 512 where a row takes 256 or fewer, so that the
// rows of a block share one partial sum per column (half the partial sums of
// blocks of 256 at the same number of threads on the chip).
constexpr int fwd_block(int tpr) { return tpr == 192 ? 192 : tpr < 256 ? 256 : tpr; }
constexpr int bwd_block(int tpr) { return tpr == 192 ? 384 : tpr < 512 && tpr != 384 ? 512 : tpr; }

// Backward: waves per SIMD that the registers of the row kernels allow (what the
// compiler needs without a limit: 56 - 119 registers a thread, in the other forms
// 76 - 148), and from them how many blocks a CU has at once: as many as are
// launched, each walking its share of the rows.
constexpr int bwd_waves(int vec, bool layer, bool post, bool pre, bool q8, int mode, int tpr) {
  const bool both = post && pre;
  if (tpr == 1024) return 4;
  if (vec == 4) return mode == kAny && layer && both ? 4 : mode != kWhole || (layer && both) ? 5 : 6;
  if (layer) return (pre ? 4 : 5) - (mode != kWhole ? 1 : 0);
  if (mode == kRagged && pre && !q8 && (tpr % 192 == 0 || tpr == 640)) return 4; // (bwd_dwords)
  return mode == kWhole ? (pre ? 5 : 6) : mode == kRagged && !(both && q8) ? 5 : 4;
}
constexpr int bwd_blocks_per_cu(int vec, bool layer, bool post, bool pre, bool q8, int mode, int tpr, int nv) {
  if (nv == 4) return 1;
  const int n = 256 * bwd_waves(vec, layer, post, pre, q8, mode, tpr) / bwd_block(tpr);
  return n > 0 ? n : 1;
}
// Rows whose loads are in flight ahead of the one in hand: two where a CU has one
// block, which otherwise stands still while its next row arrives ([8192, 8192]
// bf16 175 -> 158 us), unless the registers of a block of 1024 are full; and in
// the RMS step at two blocks ([8192, 4096] bf16 162 -> 159).
constexpr int bwd_depth(int vec, bool layer, bool post, bool pre, bool q8, int mode, int tpr, int nv) {
  if (nv > 1) return 1;
  const bool full = tpr == 1024 && (vec == 8 ? mode != kWhole || (layer && post && pre) : mode != kWhole && layer);
  const int blocks = bwd_blocks_per_cu(vec, layer, post, pre, q8, mode, tpr, nv);
  return (blocks == 1 && !full) || (blocks == 2 && vec == 8 && !layer && mode == kWhole && tpr == 512) ? 2 : 1;
}
// Forward the same for blocks of 256 threads and more.
constexpr int fwd_depth(int tpr, int nv, int mode) {
  return tpr >= 256 && nv == 1 && !(mode != kWhole && tpr == 1024) ? 2 : 1;
}
// Column sums (C, A: of gradient times normalized value; E, B: of the gradient; C
// and E of the second norm) that a block keeps in LDS, at most 128 KB, because its
// registers are taken: 128 a thread of a block of 1024, 256 where threads have four
// vectors.  w: columns of a thread.
enum { kSumC = 1, kSumE = 2, kSumA = 4, kSumB = 8 };
constexpr unsigned bwd_sums_in_lds(int w, bool layer, bool post, bool pre, bool q8, int mode, int tpr) {
  if (w == 32) return layer ? (pre ? kSumC | kSumE : kSumA | kSumB) : (pre ? kSumC : 0) | kSumA;
  if (tpr != 1024 || w < 8) return 0;
  if (w == 8)
    return (layer ? kSumE | kSumB : 0) | (mode != kWhole || (layer && q8) ? kSumA : 0) |
           (layer && (mode != kWhole || q8) ? kSumC : 0);
  return kSumA; // (of 16 columns: the RMS norm alone, see bwd_row_fits)
}
// Which forms the layouts of the longest rows have: what fits their registers and
// LDS.  1024 threads of two vectors come first, 512 of four are for forms that do
// not fit those (as fast where both fit, slower for ragged rows: [2048, 8191] float
// pre-norm backward 111 us in twos, 143 in fours); what fits neither runs as long
// rows.  [2048, 16384] bf16 RMS step backward: long 183 us, fours 101.
constexpr bool bwd_row_fits(int vec, bool layer, bool post, bool pre, bool q8, int mode, int tpr, int nv) {
  const bool both = post && pre;
  if (tpr < 1024 && nv == 1) return true;
  if (nv == 1) return !(vec == 8 && layer && both && mode != kWhole);
  const bool twos = vec == 8         ? mode == kWhole && post && !pre && !layer
                    : mode == kWhole ? !(layer && both)
                                     : !both && !(layer && pre && q8);
  if (nv == 2) return twos;
  return !twos && (vec == 8 ? mode == kWhole && !(layer && both) : mode == kWhole || (!layer && !q8));
}
constexpr bool fwd_row_fits(int vec, bool layer, bool post, bool pre, bool copy, int mode, int nv) {
  if (nv == 1) return true;
  const bool twos = vec == 8 ? mode == kWhole && !(layer && post) && !(copy && pre)
                             : !(layer && post && mode != kWhole);
  if (nv == 2) return twos;
  return !twos && (vec == 8 ? mode == kWhole && !(layer && post && pre && copy) : !(pre && copy));
}

int launch_step_fwd_f32(const StepPlan &pl, const StepArgs &a, hipStream_t st);
int launch_step_fwd_f16(const StepPlan &pl, const StepArgs &a, hipStream_t st);
int launch_step_fwd_bf16(const StepPlan &pl, const StepArgs &a, hipStream_t st);
int launch_step_bwd_f32(const StepPlan &pl, const StepArgs &a, hipStream_t st);
int launch_step_bwd_f16(const StepPlan &pl, const StepArgs &a, hipStream_t st);
int launch_step_bwd_bf16(const StepPlan &pl, const StepArgs &a, hipStream_t st);
int launch_step_bwd8_f32(const StepPlan &pl, const StepArgs &a, hipStream_t st);
int launch_step_bwd8_f16(const StepPlan &pl, const StepArgs &a, hipStream_t st);
int launch_step_bwd8_bf16(const StepPlan &pl, const StepArgs &a, hipStream_t st);

} // namespace nblahip
