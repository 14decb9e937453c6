// Parameters of the FP8 row operators (fp8.cu).
#pragma once
#include "internal.cuh"

namespace colib {

struct QuantRowsParams {
  const void *x;             // [T, K] of `type`, rows `x_stride` elements apart
  int type;                  // COLI_TYPE_*
  long x_stride;
  bool x_vec;                // every row starts on 16 bytes
  const int32_t *row_token;  // [rows] source row of each row (outside [0, T): none, the row is left as it was), or null: the row itself
  int T, rows, K;
  const int32_t *rows_used = nullptr;  // device word: rows from it on are none
  uint8_t *codes;            // [rows, K], rows `ld` bytes apart (a multiple of 16); bytes K .. round_up(K, 16) become zero
  long ld;
  float *scales;             // scale of (row, block) at row * s_row + block * s_blk
  long s_row, s_blk;
};
constexpr int QR_COLS = 1024;  // columns of a row that a warp takes; the rest of the row lies along the grid's second axis
constexpr int QR_MOST_COLS = 65535 * QR_COLS;
int launch_quant_rows(const QuantRowsParams &p, cudaStream_t st);

struct Fp8MmParams {
  const void *codes;  // e4m3 rows [rows, K], `ld` bytes apart (a multiple of 16), 16-byte aligned
  long ld;
  const float *sx;    // their scales
  long s_row, s_blk;
  int rows, K, O;
  // segments of rows that share a weight: their lengths on the device, or null: one segment of all rows
  int nseg, rows_expected;
  const int32_t *seg_count, *seg_expert;
  WeightRef one;             // the weight of a single segment, or
  const WeightRef *w0, *w1;  // tables indexed by seg_expert (w1: up, where w0 is gate)
  void *y;                   // [rows, O] of y_type, rows y_stride elements apart, or
  int y_type;
  long y_stride;
  bool y_vec;                // every row of y starts on 16 bytes
  uint8_t *h_codes;          // when not null: h = act(w0 x, w1 x) quantised again: codes [rows, O], h_ld bytes apart,
  float *h_scales;           // and scales [ceil(O / 128)][rows]
  long h_ld;
  float *h32;                // segments of a few rows (fp8_stream_ok) instead: h as it is, f32 [rows, O]
  int32_t *rows_used;        // with h32: device word that receives the rows of all segments
  bool behind_gated;         // segments of a few rows: the launches before this one are the gated call's and the row quantiser's
  ActParams act;
  int *status;               // device word for a bounded wait that gave up, or null: the library's own
  // filled in by the launcher
  int KT, Op, n_tiles, split;
};
// Whether segments are short enough for the streaming kernel (fp8_stream.cu), a task of which takes up to 8 rows.  One segment up to
// 8 rows (streaming / tcgen05, us a call: 8 rows x 2048 x 2048 4.5 / 5.9, x 7168 x 4096 8.9 / 9.9); experts while
// segments have two rows on average (H 4096, I 1024, 32 experts: 32 rows 53 / 67, 128 rows 100 / 78; H 2048, I 768, 128 experts: 300
// rows 109 / 104, 512 rows 153 / 114).  A function of shapes alone.
static inline bool fp8_stream_ok(const Fp8MmParams &p) {
  if (!p.seg_count) return p.rows <= 8;
  const int segs = p.rows_expected < p.nseg ? p.rows_expected : p.nseg;
  return p.rows_expected <= 2L * segs;
}

// How the tensor-memory kernel cuts a product, all functions of the call's shapes alone: the cheapest of what was measured.
constexpr int F8_MAX_SPLIT = 4;  // CTAs that share a tile's k-tiles (clusters of 8 start late: 24 rows x 2048 x 2048 11.4 us, with 4 6.5)
// Us a k-tile, for the ends of a tile, and for joining the sums of CTAs that share one: fitted to K 512 to 7168 on 64 to 148 CTAs.
struct F8Shape {
  int ar, bn;
  double kt_us, end_us, join_us;
};
static const F8Shape F8_SHAPES[] = {{128, 256, 0.60, 3.3, 3.2}, {128, 128, 0.42, 1.7, 2.4}, {64, 256, 0.46, 1.9, 2.4}, {64, 128, 0.40, 0.9, 2.1}, {32, 256, 0.44, 1.7, 2.2}};

struct Fp8Plan {
  int ar, bn;   // rows and columns of a tile (gated: the columns are 128 features of gate and of up)
  int split;    // CTAs that share a tile
  int n_tiles;  // tiles over the features
  int most;     // tiles over the rows, at most
};
// Experts' rows of a tile follow from their average segment (a tile passes the weights once more): 32 up to 20 rows, 64 up to 56, 128
// from there where their tiles fill the SMs.  Us a call, 128 / 64 rows: H 7168, I 2048, 32 experts, 53 rows each 274 / 249,
// 64 rows 279 / 312; H 2048, I 768, 64 experts, 64 rows 100 / 82, 94 rows 103 / 103; 64 / 32 rows: 32 experts, 19 rows 49.6 / 46.0.
// (128-row tiles of gate and up are never shared: that they are taken says that there are more of them than SMs.)
static inline Fp8Plan fp8_plan(const Fp8MmParams &p) {
  const bool gated = p.h_codes != nullptr;
  const int segs = p.seg_count ? (p.rows_expected < p.nseg ? p.rows_expected : p.nseg) : 1;
  const long mean = p.seg_count ? ((long)p.rows_expected + segs - 1) / (segs > 0 ? segs : 1) : p.rows;
  const long full = ((mean + 127) / 128) * (segs > 0 ? segs : 1) * ((p.O + 127) / 128);
  const int wanted = !p.seg_count ? 0 : mean <= 20 ? 32 : mean <= (p.KT > 32 ? 56 : 64) || full <= COLI_SMS ? 64 : 128;
  Fp8Plan plan = {};
  double best = 0.0;
  for (const F8Shape &f : F8_SHAPES) {
    if ((wanted && f.ar != wanted) || (gated && f.bn != 256)) continue;
    const int fw = gated ? 128 : f.bn;
    const int row_tiles = p.seg_count ? p.rows_expected / f.ar + segs : (p.rows + f.ar - 1) / f.ar;
    const long tiles = (long)(row_tiles > 0 ? row_tiles : 1) * ((p.O + fw - 1) / fw);
    for (int split = 1; split <= F8_MAX_SPLIT && split <= p.KT && (split == 1 || tiles * split <= COLI_SMS); split *= 2) {
      const long rounds = (tiles * split + COLI_SMS - 1) / COLI_SMS;
      const double us = rounds * ((p.KT + split - 1) / split * f.kt_us + f.end_us) + (split > 1 ? f.join_us : 0.0);
      if (plan.ar && us >= best) continue;
      best = us;
      plan = {f.ar, f.bn, split, (p.O + fw - 1) / fw, p.seg_count ? p.rows / f.ar + (p.rows < p.nseg ? p.rows : p.nseg) : row_tiles};
    }
  }
  return plan;
}
int launch_fp8_mm(Fp8MmParams p, cudaStream_t st);
int launch_fp8_stream(Fp8MmParams p, cudaStream_t st);  // called by launch_fp8_mm
int *fp8_status_word();          // the library's own status word on the current device
int fp8_take_status(int *code);  // its value, and cleared when set

}  // namespace colib
