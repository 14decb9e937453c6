// Device pieces that the FP8 row kernels share: the quantiser's arithmetic, the tables of segments and tiles, bulk copies.
#pragma once
#include "fp8.cuh"

namespace colib {

constexpr int F8_MAX_SEGS = 520;

// Both quotients are the correctly rounded ones: bf16 rows have many values exactly half-way between two codes, where
// a product with a rounded reciprocal falls to either side.  With y = 1 / b rounded to nearest and q within a unit of a / b,
// q + (a - q b) y rounds to the quotient (Markstein, IBM J. Res. Dev. 34, 1990): two FMAs, where a division
// is ten instructions and a branch (32768 rows of 7168 bf16: 287 us with divisions next to a border only).
__device__ __forceinline__ float quotient(float a, float b, float y) {
  const float q = a * y;
  return fmaf(fmaf(-q, b, a), y, q);
}
__device__ __forceinline__ float row_scale(float a) {
  constexpr float TINY = 1.17549435e-38f;              // 2^-126
  const float s = fmaxf(quotient(a, 448.0f, 1.0f / 448.0f), TINY);
  if (!(a >= 7.8886090522e-31f && a <= 3.4028235e38f))  // (the remainder is exact from 2^-100 up; none of an infinity)
    return a > 0.0f ? fmaxf(__fdiv_rn(a, 448.0f), TINY) : 1.0f;
  return s;
}
// Quotients by a block's scale.  The remainder of one of 2^-10 (below it the code is 0) or more is exact while the scale is 2^-93 or more:
// smaller blocks are divided 2^64 times as large, `up`, by which the caller multiplies.  Values by an infinite scale are their products
// with 0.
struct RowDivisor {
  static constexpr float UP = 18446744073709551616.0f;  // 2^64
  float scale, up, b, y;
  __device__ __forceinline__ explicit RowDivisor(float s) : scale(s) {
    const bool tiny = s < 8.0779356694631609e-28f;  // 2^-90
    up = tiny ? UP : 1.0f;
    const float d = s * up;
    y = __frcp_rn(d);
    b = d <= 3.4028235e38f ? d : 0.0f;
  }
  __device__ __forceinline__ float operator()(float v) const { return quotient(v, b, y); }
};
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t d;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(hi), "f"(lo));
  return d;
}
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) { return e4m3x2(a, b) | (e4m3x2(c, d) << 16); }

// The two scales of a k-tile are any f32.  They are multiplied with each other first, which is right while the product is a normal number
// (or one of them is 0): outside, scale x scale x sum may be one all the same (1e-38 and 1e-6 leave three bits of the product, 1e36
// and 1e5 none, and a sum of 0 becomes NaN).  A row with such a pair is summed again, by f8_sum_again: a branch among the additions, or
// one shared-memory read more a k-tile, costs every call 5 to 15 % (4096 x 7168 x 4096: 149.5 -> 157.7 and 170.7 us).
__device__ __forceinline__ bool f8_normal(float product) { return fabsf(product) >= 1.17549435e-38f && fabsf(product) <= 3.4028235e38f; }
// (an infinite scale or none gives the same either way)
__device__ __forceinline__ bool f8_ordinary(float x, float w) {
  return f8_normal(x * w) || x == 0.0f || w == 0.0f || !(fabsf(x) <= 3.4028235e38f && fabsf(w) <= 3.4028235e38f);
}
// sum * x * w, however far apart: factors of 2^64 keep what is on the way in range
__device__ __forceinline__ float f8_scaled(float sum, float x, float w) {
  if (f8_ordinary(x, w)) return sum * (x * w);
  constexpr float UP = 18446744073709551616.0f, DOWN = 1.0f / UP;
  return fabsf(x * w) < 1.0f ? sum * ((x * UP) * (w * UP)) * DOWN * DOWN : sum * ((x * DOWN) * (w * DOWN)) * UP * UP;
}
// Whether a row has such a pair in k-tiles kb0, kb0 + step .. kb1 - 1, with either of two blocks of features
__device__ __forceinline__ bool f8_again(const float *sx, long s_blk, const float *sw0, const float *sw1, int kb0, int kb1, int step = 1) {
  bool again = false;
#pragma unroll 1
  for (int kb = kb0; kb < kb1; kb += step) again = again || !f8_ordinary(sx[kb * s_blk], sw0[kb]) || !f8_ordinary(sx[kb * s_blk], sw1[kb]);
  return again;
}
// One result over k-tiles kb0 .. kb1 - 1, code by code: the row's codes, and the feature's, whose k-tiles lie w_step bytes apart
// (feature f, f & 7 = f7, with its chunks permuted).  Slow, and reached only by rows with scales as above; AHEAD chunks of 16 codes are
// requested at once, as many as the caller's registers allow.  (All rows of 4096 x 7168 x 4096: 37.6 ms, 9 ms a tile of 128 x 256, in
// which the tile's other warps wait; they would give up after 0.3 s, at a K of some 200000.)
template <int AHEAD>
static __device__ __noinline__ float f8_sum_again(const uint8_t *codes, const float *sx, long s_blk, int K, const uint8_t *w, size_t w_step, int f7,
                                                  const float *sw, int kb0, int kb1) {
  auto pair = [](uint32_t two) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)two));
    return __half22float2(*reinterpret_cast<const __half2 *>(&h));
  };
  float y = 0.0f;
  for (int kb = kb0; kb < kb1; ++kb) {
    float sum = 0.0f;
#pragma unroll 1
    for (int c0 = 0; c0 < 8; c0 += AHEAD) {
      uint4 a[AHEAD], b[AHEAD];
#pragma unroll
      for (int c = 0; c < AHEAD; ++c) {
        const int k = kb * 128 + (c0 + c) * 16;
        a[c] = k + 16 <= K ? *reinterpret_cast<const uint4 *>(codes + k) : make_uint4(0u, 0u, 0u, 0u);
        b[c] = *reinterpret_cast<const uint4 *>(w + kb * w_step + (size_t)(((c0 + c) ^ f7) << 4));
      }
#pragma unroll
      for (int c = 0; c < AHEAD; ++c) {
        const int k = kb * 128 + (c0 + c) * 16;
        uint32_t row[4] = {a[c].x, a[c].y, a[c].z, a[c].w};
        const uint32_t col[4] = {b[c].x, b[c].y, b[c].z, b[c].w};
        if (k < K && k + 16 > K)  // (nothing behind a row's last code is read)
          for (int i = 0; k + i < K; ++i) {
            const uint32_t code = (uint32_t)codes[k + i] << (8 * (i & 3));
            row[0] |= i < 4 ? code : 0u;
            row[1] |= i >= 4 && i < 8 ? code : 0u;
            row[2] |= i >= 8 && i < 12 ? code : 0u;
            row[3] |= i >= 12 ? code : 0u;
          }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float2 u = pair(row[i >> 1] >> (16 * (i & 1))), v = pair(col[i >> 1] >> (16 * (i & 1)));
          sum = fmaf(u.y, v.y, fmaf(u.x, v.x, sum));
        }
      }
    }
    y += f8_scaled(sum, sx[kb * s_blk], sw[kb]);
  }
  return y;
}

// `bytes` (a multiple of 16) in a row, global -> shared memory, counted by the barrier
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

template <typename OutT>
__device__ __forceinline__ OutT f8_out(float v);
template <>
__device__ __forceinline__ float f8_out<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half f8_out<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 f8_out<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

struct F8Tile {
  int seg, nt, row0, nrows;
};
// Rows and tiles before every segment, by one warp; counts that run past the buffer are cut.
template <int BM>
__device__ __forceinline__ void f8_tables(const Fp8MmParams &p, int *row_off, int *tile_off, int lane) {
  int rows = 0, tiles = 0;
  for (int s0 = 0; s0 < p.nseg; s0 += 32) {
    const int s = s0 + lane;
    int incl = s < p.nseg ? max(0, p.seg_count ? p.seg_count[s] : p.rows) : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl = (int)min((long)incl + u, (long)p.rows);
    }
    const int end = (int)min((long)rows + incl, (long)p.rows);
    int prev = __shfl_up_sync(0xffffffffu, end, 1);
    if (lane == 0) prev = rows;
    int t = (end - prev + BM - 1) / BM * p.n_tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, t, o);
      if (lane >= o) t += u;
    }
    if (s < p.nseg) {
      row_off[s + 1] = end;
      tile_off[s + 1] = tiles + t;
    }
    rows = __shfl_sync(0xffffffffu, end, 31);
    tiles += __shfl_sync(0xffffffffu, t, 31);
  }
  if (lane == 0) row_off[0] = tile_off[0] = 0;
}
// Tile t of the call, BM rows by one feature tile: segments in order, a segment's feature tiles in order, its row tiles
// inside one (they share the weights in L2).
template <int BM>
__device__ __forceinline__ F8Tile f8_tile(const int *tile_off, const int *row_off, int nseg, int t) {
  int lo = 0, hi = nseg;  // tile_off[lo] <= t < tile_off[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (tile_off[mid] <= t)
      lo = mid;
    else
      hi = mid;
  }
  const int n = row_off[lo + 1] - row_off[lo], mt = (n + BM - 1) / BM, l = t - tile_off[lo];
  F8Tile r;
  r.seg = lo;
  r.nt = l / mt;
  const int m = l - r.nt * mt;
  r.row0 = row_off[lo] + m * BM;
  r.nrows = min(BM, n - m * BM);
  return r;
}

}  // namespace colib
