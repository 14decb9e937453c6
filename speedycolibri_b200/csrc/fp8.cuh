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
int launch_fp8_mm(Fp8MmParams p, cudaStream_t st);
int launch_fp8_stream(Fp8MmParams p, cudaStream_t st);  // called by launch_fp8_mm
int *fp8_status_word();          // the library's own status word on the current device
int fp8_take_status(int *code);  // its value, and cleared when set

}  // namespace colib
