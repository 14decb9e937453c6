// Products of 8-bit floating-point rows and weights with a scale for each block of 128, the quantiser that makes such
// rows, and the expert FFN over them.
//
//   rows     q[r,k] e4m3, sx[r,b] f32: row r, columns 128b .. 128b+127 stand for sx[r,b] * q
//   weights  FMT_FP8_B128 handles: codes qw[o,k], sw[o / 128, b] f32
//   product  y[r,o] = sum_b sx[r,b] * sw[o/128,b] * ( sum_{k in b} q[r,k] * qw[o,k] )
//
// (crates/colibri-engine/src/convert.rs:731-741 has the weights' half of it; the reference multiplies f32 activations.)
#include <type_traits>

#include "fp8.cuh"
#include "fp8_common.cuh"
#include "tc_common.cuh"

namespace colib {

// ---- row quantiser ---------------------------------------------------------------------------------------------
//   a = largest |x| of a block's non-NaN values, s = 1 if a == 0 else max(a / 448, 2^-126), code = e4m3(x / s)
// to nearest even, saturating; a NaN keeps a NaN code, and an infinity makes s infinite and its own code NaN, so
// that either shows in every product with the row.
// LANES lanes share a block, in pieces of 16 bytes; a warp takes QR_COLS columns of a row and goes through the rows with the next
// one's pieces already requested; the warps of a CTA take neighbouring rows, whose scales of a block lie side by side.  Four lanes
// halve what a block's scale costs (32768 gathered rows of 7168 bf16 99.7 -> 90.4 us before WHOLE, with eight lanes and two quotients an
// instruction; rows as they are 112 -> 108.5, 6.5 TB/s); values read one by one, off the 16-byte grid, and f32, whose codes would be
// stored half a sector at a time, keep eight (5000 rows of 1111 f16 11.0 us, with four 16.4).  WHOLE: gathered rows of whole pieces,
// which the L2 has as a rule and the instructions bound, are read without a branch per piece (the gathered rows 92.0 -> 83.8 us,
// and 85.3 since tiny blocks are told apart);
// rows as they are come faster from HBM with the branches, 108.7 against 131.
template <typename T, int LANES>
struct QrPieces {
  static constexpr int VEC = 16 / (int)sizeof(T), LOADS = 128 / LANES / VEC, COLS = 32 / LANES * 128, STEPS = QR_COLS / COLS;
  uint4 q[STEPS][LOADS];
};
// Rows and tokens (and in the products the rows' scales) are an earlier launch's results, which may be written while this one is already
// resident: no constants.  The quantiser's loads may pass its own stores all the same, which the language's would not (4096 rows
// gathered eight times 85.2 -> 91.4 us), but not the wait: their pointers are taken behind it.
template <typename P>
__device__ __forceinline__ const P *behind_wait(const P *p) {
  asm volatile("" : "+l"(p)::"memory");
  return p;
}
__device__ __forceinline__ uint4 qr_load16(const void *p) {
  uint4 v;
  asm("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ int qr_load4(const int32_t *p) {
  int v;
  asm("ld.global.s32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}
template <typename T, int LANES, bool WHOLE>
__device__ __forceinline__ void qr_request(QrPieces<T, LANES> &d, const QuantRowsParams &p, const T *rows, int src, int c0) {
  using P = QrPieces<T, LANES>;
  constexpr int VEC = P::VEC, STEPS = P::STEPS, COLS = P::COLS;
  const T *x = rows + (long)src * p.x_stride;
#pragma unroll
  for (int j = 0; j < STEPS; ++j)
#pragma unroll
    for (int l = 0; l < P::LOADS; ++l) {
      const int c = c0 + COLS * j + LANES * VEC * l;
      if constexpr (WHOLE) {
        d.q[j][l] = c < p.K ? qr_load16(x + c) : make_uint4(0u, 0u, 0u, 0u);
      } else if (p.x_vec && c + VEC <= p.K) {
        d.q[j][l] = qr_load16(x + c);
      } else {
        alignas(16) T raw[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) raw[i] = c + i < p.K ? x[c + i] : T(0.0f);
        d.q[j][l] = *reinterpret_cast<const uint4 *>(raw);
      }
    }
}
// largest magnitude of a word's one or two values (maxima drop NaN)
__device__ __forceinline__ float qr_amax(float a, uint32_t w, float) { return fmaxf(a, fabsf(__uint_as_float(w))); }
__device__ __forceinline__ __half2 qr_amax(__half2 a, uint32_t w, __half) { return __hmax2(a, __habs2(*reinterpret_cast<const __half2 *>(&w))); }
__device__ __forceinline__ __nv_bfloat162 qr_amax(__nv_bfloat162 a, uint32_t w, __nv_bfloat16) {
  return __hmax2(a, __habs2(*reinterpret_cast<const __nv_bfloat162 *>(&w)));
}
__device__ __forceinline__ float qr_amax_out(float a) { return a; }
__device__ __forceinline__ float qr_amax_out(__half2 a) { return fmaxf(__low2float(a), __high2float(a)); }
__device__ __forceinline__ float qr_amax_out(__nv_bfloat162 a) { return fmaxf(__low2float(a), __high2float(a)); }
__device__ __forceinline__ void qr_zero(float &a) { a = 0.0f; }
__device__ __forceinline__ void qr_zero(__half2 &a) { a = __half2(__half(0.0f), __half(0.0f)); }
__device__ __forceinline__ void qr_zero(__nv_bfloat162 &a) { a = __nv_bfloat162(__nv_bfloat16(0.0f), __nv_bfloat16(0.0f)); }
__device__ __forceinline__ float2 qr_pair(uint32_t w, __half) { return __half22float2(*reinterpret_cast<const __half2 *>(&w)); }
__device__ __forceinline__ float2 qr_pair(uint32_t w, __nv_bfloat16) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }

// a piece's values times 2^64, exactly
__device__ __forceinline__ float qr_lift(float v) { return v * RowDivisor::UP; }
__device__ __forceinline__ uint32_t qr_lift(uint32_t w, float) { return __float_as_uint(qr_lift(__uint_as_float(w))); }
__device__ __forceinline__ uint32_t qr_lift(uint32_t w, __nv_bfloat16 t) {
  const float2 v = qr_pair(w, t);
  return __float_as_uint(qr_lift(v.x)) >> 16 | (__float_as_uint(qr_lift(v.y)) & 0xffff0000u);
}

template <typename T>
struct QrMax {
  using type = float;
};
template <>
struct QrMax<__half> {
  using type = __half2;
};
template <>
struct QrMax<__nv_bfloat16> {
  using type = __nv_bfloat162;
};

template <typename T, int LANES, bool WHOLE>
__global__ void __launch_bounds__(256, sizeof(T) == 4 ? 2 : 4) k_quant_rows(QuantRowsParams p) {
  using P = QrPieces<T, LANES>;
  constexpr int STEPS = P::STEPS, COLS = P::COLS;
  coli_grid_dependency_sync();
  const T *x = behind_wait((const T *)p.x);
  const int32_t *tokens = behind_wait(p.row_token);
  const int kp = (p.K + 15) & ~15;
  const int lane = threadIdx.x & 31, sub = lane % LANES;
  const int c0 = blockIdx.y * QR_COLS + lane / LANES * 128 + sub * P::VEC;
  const int step = gridDim.x * 8;
  const int rows = p.rows_used ? min(p.rows, *p.rows_used) : p.rows;
  // source of a row; outside [0, T): none
  auto source = [&](long r) { return r < rows ? (tokens ? qr_load4(tokens + r) : (int)r) : -1; };
  auto valid = [&](int src) { return (unsigned)src < (unsigned)p.T; };
  long r = blockIdx.x * 8 + (threadIdx.x >> 5);
  P now, next;
  int src = source(r), src_next = source(r + step);
  if (valid(src)) qr_request<T, LANES, WHOLE>(now, p, x, src, c0);
  for (; r < rows; r += step) {
    const int src_after = source(r + 2 * (long)step);
    if (valid(src_next)) qr_request<T, LANES, WHOLE>(next, p, x, src_next, c0);
    if (valid(src)) {  // (no token: the row is left as it was)
#pragma unroll
      for (int j = 0; j < STEPS; ++j) {
        typename QrMax<T>::type m;
        qr_zero(m);
#pragma unroll
        for (int l = 0; l < P::LOADS; ++l) m = qr_amax(qr_amax(qr_amax(qr_amax(m, now.q[j][l].x, T()), now.q[j][l].y, T()), now.q[j][l].z, T()), now.q[j][l].w, T());
        float a = qr_amax_out(m);
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
        const RowDivisor by(row_scale(a));
        if constexpr (!std::is_same<T, __half>::value) {  // (16-bit floats have no such blocks: 2^-24 / 448)
          if (by.up != 1.0f) {
#pragma unroll
            for (int l = 0; l < P::LOADS; ++l) {
              uint4 &q = now.q[j][l];
              q = make_uint4(qr_lift(q.x, T()), qr_lift(q.y, T()), qr_lift(q.z, T()), qr_lift(q.w, T()));
            }
          }
        }
#pragma unroll
        for (int l = 0; l < P::LOADS; ++l) {
          const int c = c0 + COLS * j + LANES * P::VEC * l;
          const uint4 q = now.q[j][l];
          uint8_t *dst = p.codes + (size_t)r * p.ld + c;
          if constexpr (sizeof(T) == 4) {
            const uint32_t w = e4m3x4(by(__uint_as_float(q.x)), by(__uint_as_float(q.y)),
                                      by(__uint_as_float(q.z)), by(__uint_as_float(q.w)));
            if (c < kp) *reinterpret_cast<uint32_t *>(dst) = w;
          } else {
            const float2 v0 = qr_pair(q.x, T()), v1 = qr_pair(q.y, T()), v2 = qr_pair(q.z, T()), v3 = qr_pair(q.w, T());
            const uint2 w = make_uint2(e4m3x4(by(v0.x), by(v0.y), by(v1.x), by(v1.y)),
                                       e4m3x4(by(v2.x), by(v2.y), by(v3.x), by(v3.y)));
            if (c < kp) *reinterpret_cast<uint2 *>(dst) = w;
          }
        }
        const int block = (c0 + COLS * j) >> 7;
        if (sub == 0 && block * 128 < p.K) p.scales[r * p.s_row + (long)block * p.s_blk] = by.scale;
      }
    }
    now = next;
    src = src_next;
    src_next = src_after;
  }
}

int launch_quant_rows(const QuantRowsParams &p, cudaStream_t st) {
  if (p.rows == 0) return 1;
  const int chunks = (p.K + QR_COLS - 1) / QR_COLS;
  // CTAs that fit the SMs at once go through the rows
  const int fit = COLI_SMS * (p.type == COLI_TYPE_F32 ? 2 : 4), groups = (p.rows + 7) / 8;
  const int each = fit / chunks > 0 ? fit / chunks : 1;
  const dim3 grid((unsigned)(groups < each ? groups : each), (unsigned)chunks);
  coli_count_launch(1);
  const bool whole = p.x_vec && p.row_token && p.K % 8 == 0;
  auto of16 = [&](auto t) {
    using T = decltype(t);
    return whole ? k_quant_rows<T, 4, true> : p.x_vec ? k_quant_rows<T, 4, false> : k_quant_rows<T, 8, false>;
  };
  auto *kernel = p.type == COLI_TYPE_F32 ? k_quant_rows<float, 8, false> : p.type == COLI_TYPE_F16 ? of16(__half()) : of16(__nv_bfloat16());
  const cudaError_t e = launch_dependent(kernel, grid, dim3(256), 0, st, p);
  return coli_cuda_check(e, "row quantiser launch") ? 1 : 0;
}

// ---- product -----------------------------------------------------------------------------------------------------
// A persistent CTA per SM makes tiles of AR (128, 64 or 32) rows x BN features.  Per 128 columns (one k-tile, one scale block) a
// stage of the shared-memory ring holds the rows' codes (one TMA box, 128-byte swizzle) and the weights' codes, which lie in
// HBM in exactly that order (coli_fp8_chunk is the swizzle's permutation) and come as plain bulk copies; four tcgen05.mma
// kind::f8f6f4 form the k-tile's product in one of two TMEM buffers, and eight warps add it to f32 registers, scaled:
// a thread owns one row (its TMEM lane) and a share of the features, so sx is one register and sw is uniform.
// The scales are arbitrary f32, which the block-scaled MMA kinds do not take.  Four more warps copy, issue the products, look
// up the next tiles and bring the scales: whatever waits for memory in the summing warps is added to every k-tile.
// What bounds it: with short segments the weights' bytes; with long ones the hand-overs between products and sums, 1170 cycles
// a k-tile of 128 x 256 whose products take 512 (4096 rows x 7168 x 4096: 154 us, 1560 TFLOP/s, tensor pipe 39 % active;
// loads of the next k-tile always on their way across its end: 187 us), and in calls of many such tiles power (1.5 GHz at
// 1000 W; 8192 rows on 64 experts, H 7168, I 2048: 806 us, 895 TFLOP/s of products without their padding).
constexpr int F8_BM = 128;
constexpr int F8_EPI_WARPS = 8;
constexpr int F8_THREADS = (F8_EPI_WARPS + 4) * 32;  // (registers are moved between whole warpgroups: four other warps, a role each)
// 168 registers a thread at launch are 64512; the summing warps take 208 of them each, the others keep 88: all of them.
constexpr int F8_REGS_SUM = 208, F8_REGS_OTHER = 88;
constexpr int F8_MAPS = 5;  // boxes of 8, 16, 32, 64 and 128 rows
struct F8Maps {
  CUtensorMap m[F8_MAPS];
};
static __device__ int g_fp8_status;  // of products without a handle of their own

// What the roles need to know of a tile, looked up ahead of them by a warp of its own.
struct F8Info {
  const uint8_t *q0, *q1;  // codes of the tile's first feature, k-tile 0
  const float *s0, *s1;    // scales of its first block of features
  int nt, row0, nrows, pad;
};
constexpr int F8_INFOS = 4;
constexpr int F8_OUT_LD = 64 + 16;  // bytes a row of a warp's staged results: eight rows start in different banks
constexpr int F8_CHUNK = 4;   // k-tiles whose scales are handed over at once
// AR: rows of a tile.  The products always take 128: where segments are short, 64 or 32 rows stand two or four times in a stage, so
// that all four quarters of tensor memory hold them and every summing warp takes a half or a quarter of the features it would.
template <int BN, int AR>
struct F8Smem {
  static constexpr int DUP = F8_BM / AR, PARTS = 2 * DUP;  // copies of the rows; shares of the features
  static constexpr int A_BYTES = F8_BM * 128;
  static constexpr int B_BYTES = BN * 128;
  static constexpr int STAGE = A_BYTES + B_BYTES;
  static constexpr int STAGES = BN == 256 ? 4 : 6;
  static constexpr int RED_LD = BN + 4;  // f32 a row of partial sums: rows start 4 banks apart
  static constexpr int RING = STAGES * STAGE;
  static_assert(AR * RED_LD * 4 <= RING, "partial sums take the ring's place");
  static constexpr int OUT = F8_EPI_WARPS * 32 * F8_OUT_LD;
  static constexpr int INFOS = F8_INFOS * (int)sizeof(F8Info);
  static constexpr int SCALES = 2 * F8_CHUNK * (F8_BM + 2) * 4;  // two chunks: [k-tile][row] of sx, then [k-tile][block of features] of sw
  static constexpr int BARS = 2 * STAGES + 4 + 2 * F8_INFOS + 4;
  static constexpr int TABLES = 2 * (F8_MAX_SEGS + 1) * 4;
  static constexpr int BYTES = 1024 + RING + OUT + INFOS + SCALES + 8 * BARS + 16 + TABLES + 2 * 2 * F8_BM * 4;
  static_assert(BYTES <= 227 * 1024, "shared memory");
};

__device__ __forceinline__ void umma_f8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}" ::"r"(d_tmem), "l"(adesc), "l"(bdesc),
      "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr, uint32_t rank) {
  float4 v;
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
  return v;
}

// Four consecutive values of one row; `valid` of them exist.
template <typename OutT>
__device__ __forceinline__ void f8_store4(OutT *dst, const float (&v)[4], int valid, bool vec) {
  alignas(16) OutT o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = f8_out<OutT>(v[i]);
  if (vec && valid >= 4) {
    if constexpr (sizeof(OutT) == 4)
      *reinterpret_cast<uint4 *>(dst) = *reinterpret_cast<const uint4 *>(o);
    else
      *reinterpret_cast<uint2 *>(dst) = *reinterpret_cast<const uint2 *>(o);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < valid) dst[j] = o[j];
  }
}
// A warp's 32 rows x N columns, a row in each lane, to y: 64 bytes of every row at a time through shared memory, so that a
// store instruction writes eight rows' whole sectors (lane by lane it is 32 rows' halves: 5600 cycles a tile of 128 x 256,
// of 16 k-tiles at 1180).
template <typename OutT, int N>
__device__ __forceinline__ void f8_store_rows(unsigned char *stage, OutT *y, long stride, const float *acc, int rows, int cols, bool vec, int lane) {
  constexpr int LD = F8_OUT_LD, PER = 16 / (int)sizeof(OutT), CH = 64 / (int)sizeof(OutT);
  const uint32_t at = smem_u32(stage);
#pragma unroll
  for (int c = 0; c < N / CH; ++c) {
    if (c * CH >= cols) break;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      alignas(16) OutT o[PER];
#pragma unroll
      for (int j = 0; j < PER; ++j) o[j] = f8_out<OutT>(acc[c * CH + i * PER + j]);
      *reinterpret_cast<uint4 *>(stage + lane * LD + 16 * i) = *reinterpret_cast<const uint4 *>(o);
    }
    __syncwarp();
    if (vec && (c + 1) * CH <= cols) {
      const int col = c * CH + (lane & 3) * PER;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 8 * i + (lane >> 2);
        const uint4 v = lds128(at + (uint32_t)(r * LD + 16 * (lane & 3)));
        if (r < rows) *reinterpret_cast<uint4 *>(y + (long)r * stride + col) = v;
      }
    } else {  // off the 16-byte grid, or the last features: value by value, a row's next to each other
      const int e = lane % CH, col = c * CH + e;
#pragma unroll 8
      for (int r = lane / CH; r < 32; r += 32 / CH)
        if (r < rows && col < cols) y[(long)r * stride + col] = *reinterpret_cast<const OutT *>(stage + r * LD + e * (int)sizeof(OutT));
    }
    __syncwarp();
  }
}

// c += (x, y) * s
__device__ __forceinline__ void f8_add_scaled(float2 &c, float x, float y, float s) {
  uint64_t cc, v, ss;
  asm("mov.b64 %0, {%1, %2};" : "=l"(cc) : "f"(c.x), "f"(c.y));
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y));
  asm("mov.b64 %0, {%1, %1};" : "=l"(ss) : "f"(s));
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(cc) : "l"(v), "l"(ss));
  asm("mov.b64 {%0, %1}, %2;" : "=f"(c.x), "=f"(c.y) : "l"(cc));
}

// Row `row` of tile t from its codes, for scales that the tile's sums do not hold (f8_ordinary).
template <bool GATED, int BN, int AR>
struct F8Row {
  const uint8_t *codes, *q[2];
  const float *sx, *sw[2];  // sw: of all blocks of the feature's weight
  int f0;                   // the tile's first feature
  __device__ __forceinline__ F8Row(const Fp8MmParams &p, const int *row_off, const int *tile_off, int t, int row) {
    const F8Tile tile = f8_tile<AR>(tile_off, row_off, p.nseg, t);
    const int ex = p.seg_expert ? p.seg_expert[tile.seg] : tile.seg;
    const WeightRef w0 = p.w0 ? p.w0[ex] : p.one, w1 = GATED ? p.w1[ex] : w0;
    codes = (const uint8_t *)p.codes + (long)(tile.row0 + row) * p.ld;
    sx = p.sx + (long)(tile.row0 + row) * p.s_row;
    q[0] = w0.q;
    q[1] = w1.q;
    sw[0] = reinterpret_cast<const float *>(w0.s);
    sw[1] = reinterpret_cast<const float *>(w1.s);
    f0 = tile.nt * (GATED ? 128 : BN);
  }
  __device__ __forceinline__ bool asks(const Fp8MmParams &p, int first = 0, int step = 1) const {
    const float *s0 = sw[0] + (size_t)(f0 >> 7) * p.KT;
    return f8_again(sx, p.s_blk, s0, GATED ? sw[1] + (size_t)(f0 >> 7) * p.KT : BN == 256 && f0 + 128 < p.O ? s0 + p.KT : s0, first, p.KT, step);
  }
  __device__ __forceinline__ bool warp_asks(const Fp8MmParams &p, int lane) const { return __any_sync(0xffffffffu, asks(p, lane, 32)); }
  __device__ __forceinline__ float sum(const Fp8MmParams &p, int f, int up) const {
    return f < p.O ? f8_sum_again<8>(codes, sx, p.s_blk, p.K, q[up] + (size_t)f * 128, (size_t)p.Op * 128, f & 7, sw[up] + (size_t)(f >> 7) * p.KT, 0, p.KT) : 0.0f;
  }
};
// Four neighbouring features of one row of h by each lane of a warp: its scale and codes.
__device__ __forceinline__ void f8_store_h(const Fp8MmParams &p, const float (&g)[4], const float (&u)[4], long r, int nt, int lane) {
  const int f = nt * 128 + 4 * lane;
  float h[4], a = 0.0f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    h[j] = f + j < p.O ? coli_act_fast(g[j], u[j], p.act) : 0.0f;
    a = fmaxf(a, fabsf(h[j]));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
  const RowDivisor by(row_scale(a));
  if (f < p.h_ld) *reinterpret_cast<uint32_t *>(p.h_codes + (size_t)r * p.h_ld + f) = e4m3x4(by(h[0] * by.up), by(h[1] * by.up), by(h[2] * by.up), by(h[3] * by.up));
  if (lane == 0) p.h_scales[(size_t)nt * p.rows + r] = by.scale;
}

// One warp sums row i of the tile over the CTAs of the cluster and writes what becomes of it.
template <bool GATED, int BN, int AR, typename OutT>
__device__ __forceinline__ void f8_join_row(const Fp8MmParams &p, const F8Info &tile, const int *row_off, const int *tile_off, int t, uint32_t red, int world, int i,
                                            int lane) {
  // (all CTAs' sums are requested before the first is added)
  float4 v[BN / 128], u[F8_MAX_SPLIT][BN / 128];
#pragma unroll
  for (int r = 0; r < F8_MAX_SPLIT; ++r)
#pragma unroll
    for (int j = 0; j < BN / 128; ++j)
      if (r < world) u[r][j] = ld_cluster4(red + (uint32_t)(i * (BN + 4) + 128 * j + 4 * lane) * 4u, (uint32_t)r);
#pragma unroll
  for (int j = 0; j < BN / 128; ++j) v[j] = u[0][j];
#pragma unroll
  for (int r = 1; r < F8_MAX_SPLIT; ++r)
#pragma unroll
    for (int j = 0; j < BN / 128; ++j)
      if (r < world) {
        v[j].x += u[r][j].x;
        v[j].y += u[r][j].y;
        v[j].z += u[r][j].z;
        v[j].w += u[r][j].w;
      }
  const float first = __shfl_sync(0xffffffffu, v[0].x, 0);  // (columns behind the last feature hold anything)
  if (first != first) {
    const F8Row<GATED, BN, AR> row(p, row_off, tile_off, t, i);
    if (row.warp_asks(p, lane)) {
#pragma unroll
      for (int j = 0; j < BN / 128; ++j) {
        const int f = row.f0 + (GATED ? 0 : 128 * j) + 4 * lane;
        v[j] = make_float4(row.sum(p, f, GATED ? j : 0), row.sum(p, f + 1, GATED ? j : 0), row.sum(p, f + 2, GATED ? j : 0), row.sum(p, f + 3, GATED ? j : 0));
      }
    }
    __syncwarp();
  }
  if constexpr (GATED) {
    const float g[4] = {v[0].x, v[0].y, v[0].z, v[0].w}, u[4] = {v[1].x, v[1].y, v[1].z, v[1].w};
    f8_store_h(p, g, u, tile.row0 + i, tile.nt, lane);
  } else {
#pragma unroll
    for (int j = 0; j < BN / 128; ++j) {
      const int f = tile.nt * BN + 128 * j + 4 * lane;
      const float o[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
      if (f < p.O) f8_store4<OutT>((OutT *)p.y + (long)(tile.row0 + i) * p.y_stride + f, o, p.O - f, p.y_vec);
    }
  }
}

// GATED: features of two weights, h = act(gate, up), quantised again as rows (one scale per row and 128 features).
// SPLIT: the CTAs of a cluster share the k-tiles of one tile and join their sums, in rank order, through distributed
// shared memory: for calls with too few tiles for the SMs.
template <bool GATED, int BN, int AR, bool SPLIT, typename OutT>
__global__ void __launch_bounds__(F8_THREADS, 1) k_fp8_mm(const __grid_constant__ F8Maps maps, const Fp8MmParams p) {
  using S = F8Smem<BN, AR>;
  constexpr int DUP = S::DUP, PARTS = S::PARTS, NACC = BN / PARTS, HF = NACC / 2;  // a thread's sums; of those, GATED, of gate
  extern __shared__ unsigned char smem_raw[];
  unsigned char *smem = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const uint32_t ring = smem_u32(smem);
  F8Info *infos = reinterpret_cast<F8Info *>(smem + S::RING + S::OUT);
  float *scales = reinterpret_cast<float *>(infos + F8_INFOS);
  unsigned char *after = smem + S::RING + S::OUT + S::INFOS + S::SCALES;
  const uint32_t full = smem_u32(after), empty = full + 8 * S::STAGES, dfull = empty + 8 * S::STAGES, dempty = dfull + 16;
  const uint32_t known = dempty + 16, forgotten = known + 8 * F8_INFOS;
  const uint32_t scaled = forgotten + 8 * F8_INFOS, unscaled = scaled + 16;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(after + 8 * S::BARS);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
  int *row_off = reinterpret_cast<int *>(after + 8 * S::BARS + 16);
  int *tile_off = row_off + F8_MAX_SEGS + 1;
  float *amax_s = reinterpret_cast<float *>(tile_off + F8_MAX_SEGS + 1);  // [tile parity][share][row]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int *status = p.status;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::STAGES; ++s) {
      mbar_init(full + 8 * s, 1);
      mbar_init(empty + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(dfull + 8 * b, 1);
      mbar_init(dempty + 8 * b, F8_EPI_WARPS);
    }
    for (int i = 0; i < F8_INFOS; ++i) {
      mbar_init(known + 8 * i, 1);
      mbar_init(forgotten + 8 * i, F8_EPI_WARPS + 2);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(scaled + 8 * i, 1);
      mbar_init(unscaled + 8 * i, F8_EPI_WARPS);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == F8_EPI_WARPS + 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(2u * BN) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    tc_fence_before();
  }
  coli_grid_dependency_sync();  // (the set-up above overlaps the predecessor's end)
  if (warp == 0) f8_tables<AR>(p, row_off, tile_off, lane);
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int n_tiles = tile_off[p.nseg];
  const uint32_t rank = SPLIT ? cluster_rank() : 0u;
  const int world = SPLIT ? p.split : 1;
  const int cluster0 = (int)blockIdx.x / world, clusters = (int)gridDim.x / world;
  const int kb0 = SPLIT ? (int)((long)p.KT * rank / world) : 0, kb1 = SPLIT ? (int)((long)p.KT * (rank + 1) / world) : p.KT;
  // the CTAs of a cluster meet twice a tile: sums written, sums read
  auto meet = [&] {
    if constexpr (SPLIT) cluster_sync();
  };
  uint32_t it = 0;   // k-tiles so far: the ring's and the TMEM buffers' place and phase follow from it
  uint32_t nth = 0;  // tiles so far
  bool alive = true;
  // the nth tile of this CTA, as a reader; every lane must have it before the warp forgets it
  auto recall = [&](F8Info &i) {
    const uint32_t s = nth % F8_INFOS, ph = (nth / F8_INFOS) & 1u;
    alive = alive && __all_sync(0xffffffffu, mbar_wait(known + 8 * s, ph, abort_flag, status, TC_ERR_TMA_WAIT));
    i = infos[s];
    if (!alive) i.nrows = 0;
    __syncwarp();
    if (lane == 0) mbar_arrive(forgotten + 8 * s);
    ++nth;
  };

  if (warp >= F8_EPI_WARPS) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(F8_REGS_OTHER));
    if (warp == F8_EPI_WARPS) {
      // ---------------- copies ----------------
      asm volatile("fence.proxy.async.global;" ::: "memory");  // (the codes may be an earlier launch's ordinary stores)
      for (int t = cluster0; t < n_tiles; t += clusters) {
        F8Info tile;
        recall(tile);
        const int f0 = tile.nt * (GATED ? 128 : BN);
        const uint32_t nb = (uint32_t)min(GATED ? 128 : BN, p.Op - f0) * 128u;
        int box = 0;
        while ((8 << box) < tile.nrows) ++box;
        const uint32_t bytes = (uint32_t)(8 << box) * 128u * DUP + (GATED ? 2 * nb : nb);
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const uint32_t s = it % S::STAGES, ph = (it / S::STAGES) & 1u;
          alive = alive && __all_sync(0xffffffffu, mbar_wait(empty + 8 * s, ph ^ 1u, abort_flag, status, TC_ERR_TMA_WAIT));
          if (alive && elect_one()) {
            const uint32_t a = ring + s * S::STAGE, b = a + S::A_BYTES, bar = full + 8 * s;
            mbar_expect_tx(bar, bytes);
#pragma unroll
            for (int j = 0; j < DUP; ++j) tma_load_2d(a + j * AR * 128, &maps.m[box], kb * 128, tile.row0, bar);
            const size_t at = (size_t)kb * p.Op * 128;
            bulk_load(b, tile.q0 + at, nb, bar);
            if (GATED) bulk_load(b + 128 * 128, tile.q1 + at, nb, bar);
          }
          __syncwarp();
        }
        meet();
        meet();
      }
      if (*abort_flag) {
        // copies already issued still land in this CTA's shared memory: give them time before exit
        for (int i = 0; i < 2000; ++i) __nanosleep(1000);
      }
    } else if (warp == F8_EPI_WARPS + 1) {
      // ---------------- products ----------------
      // kind::f8f6f4: D = f32, A = B = e4m3 (format code 0), both K-major
      constexpr uint32_t idesc = (1u << 4) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(F8_BM >> 4) << 24);
      for (int t = cluster0; t < n_tiles; t += clusters) {
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const uint32_t s = it % S::STAGES, ph = (it / S::STAGES) & 1u, d = it & 1u, dph = (it >> 1) & 1u;
          // (the buffer last: the sums give it back late, and a look at a barrier takes over a hundred cycles here)
          alive = alive && __all_sync(0xffffffffu, mbar_wait(full + 8 * s, ph, abort_flag, status, TC_ERR_MMA_WAIT));
          alive = alive && __all_sync(0xffffffffu, mbar_wait(dempty + 8 * d, dph ^ 1u, abort_flag, status, TC_ERR_MMA_WAIT));
          tc_fence_after();
          if (alive && elect_one()) {
            const uint32_t a = ring + s * S::STAGE;
            const uint64_t ad = umma_smem_desc(a), bd = umma_smem_desc(a + S::A_BYTES);
#pragma unroll
            for (int k = 0; k < 4; ++k) umma_f8(tmem + d * BN, ad + 2 * k, bd + 2 * k, idesc, k != 0);
            umma_commit(dfull + 8 * d);
            umma_commit(empty + 8 * s);
          }
          __syncwarp();
        }
        meet();
        meet();
      }
    } else if (warp == F8_EPI_WARPS + 2) {
      // ---------------- tiles ahead ----------------
      for (int t = cluster0; t < n_tiles; t += clusters, ++nth) {
        const uint32_t s = nth % F8_INFOS, ph = (nth / F8_INFOS) & 1u;
        const F8Tile tile = f8_tile<AR>(tile_off, row_off, p.nseg, t);
        const int ex = p.seg_expert ? p.seg_expert[tile.seg] : tile.seg;
        const WeightRef w0 = p.w0 ? p.w0[ex] : p.one, w1 = GATED ? p.w1[ex] : w0;
        const int f0 = tile.nt * (GATED ? 128 : BN);
        F8Info i;
        i.q0 = w0.q + (size_t)f0 * 128;
        i.q1 = w1.q + (size_t)f0 * 128;
        i.s0 = reinterpret_cast<const float *>(w0.s) + (size_t)(f0 >> 7) * p.KT;
        i.s1 = reinterpret_cast<const float *>(w1.s) + (size_t)(f0 >> 7) * p.KT;
        i.nt = tile.nt;
        i.row0 = tile.row0;
        i.nrows = tile.nrows;
        alive = alive && __all_sync(0xffffffffu, mbar_wait(forgotten + 8 * s, ph ^ 1u, abort_flag, status, TC_ERR_TMA_WAIT));
        if (alive && lane == 0) {
          infos[s] = i;
          mbar_arrive(known + 8 * s);
        }
        __syncwarp();
        meet();
        meet();
      }
    } else {
      // ---------------- scales: sx of the tile's rows, sw of its one or two blocks of features ----------------
      for (int t = cluster0; t < n_tiles; t += clusters) {
        F8Info tile;
        recall(tile);
        // (a second block past the end has no scales, and is not stored; a tile that was not waited for is not known: no address of it
        // is used once a wait has given up)
        const float *sw = (lane & 1) == 0 ? tile.s0 : GATED ? tile.s1 : BN == 256 && tile.nt * BN + 128 < p.O ? tile.s0 + p.KT : tile.s0;
        const float *sx[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) sx[j] = p.sx + (long)(tile.row0 + min(lane + 32 * j, max(tile.nrows, 1) - 1)) * p.s_row;
        for (int kb = kb0; kb < kb1; kb += F8_CHUNK, ++it) {
          float x[F8_CHUNK][4];
          const float w = alive && lane < 2 * F8_CHUNK ? __ldg(sw + min(kb + (lane >> 1), kb1 - 1)) : 0.0f;
#pragma unroll
          for (int u = 0; u < F8_CHUNK; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j) x[u][j] = alive && kb + u < kb1 ? __ldcg(sx[j] + (long)(kb + u) * p.s_blk) : 0.0f;
          // A row with a pair that is not f8_ordinary becomes NaN, and the summing warps look closer at those.  (The chunk's extremes first:
          // the pairs one by one would make this warp the slowest.)
          float most = fabsf(x[0][0]), least = most;
#pragma unroll
          for (int u = 0; u < F8_CHUNK; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              most = fmaxf(most, fabsf(x[u][j]));
              least = fminf(least, kb + u < kb1 ? fabsf(x[u][j]) : least);
            }
          const uint32_t wbits = __float_as_uint(fabsf(w));
          const float wmost = __uint_as_float(__reduce_max_sync(0xffffffffu, wbits)), wleast = __uint_as_float(__reduce_min_sync(0xffffffffu, lane < 2 * F8_CHUNK ? wbits : 0x7fffffffu));
          if (!__all_sync(0xffffffffu, f8_normal(most * wmost) && f8_normal(least * wleast))) {
            bool again[4] = {};
#pragma unroll
            for (int u = 0; u < F8_CHUNK; ++u) {
              const float w0 = __shfl_sync(0xffffffffu, w, 2 * u), w1 = __shfl_sync(0xffffffffu, w, 2 * u + 1);
#pragma unroll
              for (int j = 0; j < 4; ++j) again[j] = again[j] || (kb + u < kb1 && (!f8_ordinary(x[u][j], w0) || !f8_ordinary(x[u][j], w1)));
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (again[j]) x[0][j] = __uint_as_float(0x7fffffffu);
          }
          const uint32_t s = it & 1u, ph = (it >> 1) & 1u;
          alive = alive && __all_sync(0xffffffffu, mbar_wait(unscaled + 8 * s, ph ^ 1u, abort_flag, status, TC_ERR_TMA_WAIT));
          if (alive) {
            float *at = scales + s * F8_CHUNK * (F8_BM + 2);
#pragma unroll
            for (int u = 0; u < F8_CHUNK; ++u)
#pragma unroll
              for (int j = 0; j < 4; ++j) at[u * F8_BM + lane + 32 * j] = x[u][j];
            if (lane < 2 * F8_CHUNK) at[F8_CHUNK * F8_BM + lane] = w;
          }
          __syncwarp();
          if (alive && lane == 0) mbar_arrive(scaled + 8 * s);
        }
        meet();
        meet();
      }
    }
  } else {
    // ---------------- scaled sums ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(F8_REGS_SUM));
    const int r0 = (warp & 3) % (AR / 32) * 32, row = r0 + lane, part = (warp >> 2) * DUP + (warp & 3) / (AR / 32);
    const uint32_t tbase = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    F8Info tile;
    tile.nrows = 0;
    uint32_t chunk = 0;  // of scales, so far
    // This thread's scales of the next k-tiles, read a chunk at a time: beside the products' operands a read of shared memory
    // takes some two hundred cycles.
    float sc0[F8_CHUNK] = {}, sc1[F8_CHUNK] = {};
    auto scales_of = [&](int kb) {
      if ((uint32_t)(kb - kb0) % F8_CHUNK == 0) {
        alive = alive && __all_sync(0xffffffffu, mbar_wait(scaled + 8 * (chunk & 1u), (chunk >> 1) & 1u, abort_flag, status, TC_ERR_EPI_WAIT));
        const float *at = scales + (chunk & 1u) * (F8_CHUNK * (F8_BM + 2)), *w = at + F8_CHUNK * F8_BM + (GATED ? 0 : (part * NACC) >> 7);
#pragma unroll
        for (int u = 0; u < F8_CHUNK; ++u) {
          const float x = at[u * F8_BM + row];
          sc0[u] = x * w[2 * u];
          if (GATED) sc1[u] = x * w[2 * u + 1];
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(unscaled + 8 * (chunk & 1u));
        ++chunk;
      } else {
#pragma unroll
        for (int u = 0; u + 1 < F8_CHUNK; ++u) {
          sc0[u] = sc0[u + 1];
          if (GATED) sc1[u] = sc1[u + 1];
        }
      }
    };
    if (cluster0 < n_tiles) recall(tile);
    for (int t = cluster0; t < n_tiles; t += clusters) {
      const bool any = r0 < tile.nrows;
      float2 acc[NACC / 2];
#pragma unroll
      for (int i = 0; i < NACC / 2; ++i) acc[i] = make_float2(0.0f, 0.0f);
      for (int kb = kb0; kb < kb1; ++kb, ++it) {
        const uint32_t d = it & 1u, dph = (it >> 1) & 1u;
        scales_of(kb);
        const float s0 = sc0[0], s1 = GATED ? sc1[0] : s0;
        alive = alive && __all_sync(0xffffffffu, mbar_wait(dfull + 8 * d, dph, abort_flag, status, TC_ERR_EPI_WAIT));
        tc_fence_after();
        if (any && alive) {
          // FLY loads of 16 columns at a time, the next ones requested as each is added, so that the buffer goes back to the
          // products after few round trips (48 columns on their way beside 128 sums leave 8 bytes of addresses a thread in memory, 64 would
          // leave sums); two sums an instruction.
          constexpr int CH = NACC / 16, FLY = CH == 8 ? 3 : CH;
          uint32_t v[FLY][16];
          auto column = [&](int c) { return tbase + d * BN + (uint32_t)(GATED ? (c < CH / 2 ? HF * part + 16 * c : 128 + HF * part + 16 * (c - CH / 2)) : part * NACC + 16 * c); };
#pragma unroll
          for (int c = 0; c < FLY; ++c) tmem_ld16(column(c), v[c]);
#pragma unroll
          for (int c0 = 0; c0 < CH; c0 += FLY) {
            tmem_ld_wait();
            if (c0 + FLY >= CH) {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(dempty + 8 * d);
            }
#pragma unroll
            for (int c = c0; c < c0 + FLY && c < CH; ++c) {
              const float s = GATED && c >= CH / 2 ? s1 : s0;
#pragma unroll
              for (int i = 0; i < 8; ++i) f8_add_scaled(acc[8 * c + i], __uint_as_float(v[c - c0][2 * i]), __uint_as_float(v[c - c0][2 * i + 1]), s);
              if (c + FLY < CH) tmem_ld16(column(c + FLY), v[c - c0]);
            }
          }
        } else {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(dempty + 8 * d);
        }
      }
      float *flat = reinterpret_cast<float *>(acc);
      const bool mine = row < tile.nrows;
      // a NaN: the row's own, or the scales' warp's (looked at once the sums are stored; columns behind the last feature hold anything)
      const bool none = mine && alive && flat[0] != flat[0] && tile.nt * (GATED ? 128 : BN) + (GATED ? HF : NACC) * part < p.O;
      if constexpr (SPLIT) {
        // partial sums into the ring's place: its last copies have been multiplied
        float *red = reinterpret_cast<float *>(smem);
        if (mine && alive) {
#pragma unroll
          for (int c = 0; c < NACC / 4; ++c) {
            const int col = GATED ? (4 * c < HF ? HF * part + 4 * c : 128 + HF * part + 4 * c - HF) : part * NACC + 4 * c;
            *reinterpret_cast<float4 *>(red + row * S::RED_LD + col) = make_float4(flat[4 * c], flat[4 * c + 1], flat[4 * c + 2], flat[4 * c + 3]);
          }
        }
        meet();
        alive = alive && !*abort_flag;
        for (int i = (int)rank + world * warp; alive && i < tile.nrows; i += world * F8_EPI_WARPS) f8_join_row<GATED, BN, AR, OutT>(p, tile, row_off, tile_off, t, ring, world, i, lane);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the ring is copied into again
        meet();
      } else if constexpr (GATED) {
        // h of this share's features, the row's largest together with the other shares', codes
        float a = 0.0f;
        const int f0 = tile.nt * 128 + HF * part, left = p.O - f0;  // features that exist
        if (any) {
#pragma unroll
          for (int i = 0; i < HF; ++i) {
            const float h = coli_act_fast(flat[i], flat[HF + i], p.act);  // (selected, not branched around: the chains overlap)
            flat[i] = i < left ? h : 0.0f;
            a = fmaxf(a, fabsf(flat[i]));
          }
        }
        float *am = amax_s + ((t / clusters) & 1) * PARTS * AR + row;
        am[part * AR] = a;
        asm volatile("bar.sync 1, %0;" ::"n"(F8_EPI_WARPS * 32) : "memory");
#pragma unroll
        for (int i = 0; i < PARTS; ++i) a = fmaxf(a, am[i * AR]);
        const RowDivisor by(row_scale(a));
        if (__any_sync(0xffffffffu, by.up != 1.0f)) {
#pragma unroll
          for (int i = 0; i < HF; ++i) flat[i] *= by.up;
        }
        const bool again = none && F8Row<GATED, BN, AR>(p, row_off, tile_off, t, row).asks(p);  // (every share of the row sees it)
        if (mine && alive && !again) {
          uint8_t *dst = p.h_codes + (size_t)(tile.row0 + row) * p.h_ld + f0;
#pragma unroll
          for (int c = 0; c < HF / 16; ++c) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              w[i] = e4m3x4(by(flat[16 * c + 4 * i]), by(flat[16 * c + 4 * i + 1]), by(flat[16 * c + 4 * i + 2]), by(flat[16 * c + 4 * i + 3]));
            if (f0 + 16 * c < p.h_ld) reinterpret_cast<uint4 *>(dst)[c] = make_uint4(w[0], w[1], w[2], w[3]);
          }
          if (part == 0) p.h_scales[(size_t)tile.nt * p.rows + tile.row0 + row] = by.scale;
        }
        for (uint32_t left = part == 0 ? __ballot_sync(0xffffffffu, again) : 0u; left; left &= left - 1u) {
          const int r = r0 + __ffs(left) - 1;
          const F8Row<GATED, BN, AR> one(p, row_off, tile_off, t, r);
          float g[4], u[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            g[j] = one.sum(p, one.f0 + 4 * lane + j, 0);
            u[j] = one.sum(p, one.f0 + 4 * lane + j, 1);
          }
          __syncwarp();
          f8_store_h(p, g, u, tile.row0 + r, tile.nt, lane);
        }
      } else {
        const int f = tile.nt * BN + part * NACC;
        if (any && alive && f < p.O)
          f8_store_rows<OutT, NACC>(smem + S::RING + warp * 32 * F8_OUT_LD, (OutT *)p.y + (long)(tile.row0 + r0) * p.y_stride + f, p.y_stride, flat,
                                    tile.nrows - r0, p.O - f, p.y_vec, lane);
        for (uint32_t left = __ballot_sync(0xffffffffu, none); left; left &= left - 1u) {
          const int r = r0 + __ffs(left) - 1;
          const F8Row<GATED, BN, AR> one(p, row_off, tile_off, t, r);
          if (!one.warp_asks(p, lane)) continue;
          for (int i = lane; i < NACC && f + i < p.O; i += 32) ((OutT *)p.y)[(long)(tile.row0 + r) * p.y_stride + f + i] = f8_out<OutT>(one.sum(p, f + i, 0));
        }
        __syncwarp();
      }
      if (t + clusters < n_tiles) recall(tile);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == F8_EPI_WARPS + 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2u * BN) : "memory");
  }
}

// e4m3 rows [rows, K] that start `ld` bytes apart; box = 128 columns x box_rows rows; reads past either end give zeros
static bool make_codes_map(CUtensorMap *map, const void *base, int rows, int K, long ld, int box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld};
  const cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    coli_set_error("cuTensorMapEncodeTiled failed with code %d (rows=%d K=%d ld=%ld)", (int)r, rows, K, ld);
    return false;
  }
  return true;
}

template <bool GATED, int BN, int AR, bool SPLIT, typename OutT>
static int launch_f8(const F8Maps &maps, const Fp8MmParams &p, int grid, cudaStream_t st) {
  static ColiPerDeviceOnce attr_once;
  auto *kernel = k_fp8_mm<GATED, BN, AR, SPLIT, OutT>;
  constexpr int bytes = F8Smem<BN, AR>::BYTES;
  if (!coli_set_smem_limit(attr_once, kernel, bytes, "fp8 product shared-memory attribute")) return 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(F8_THREADS);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)p.split;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = SPLIT ? 2 : 1;
  coli_count_launch(1);
  return coli_cuda_check(cudaLaunchKernelEx(&cfg, kernel, maps, p), "fp8 product launch") ? 1 : 0;
}
template <bool GATED, int BN, typename OutT>
static int launch_f8_rows(const F8Maps &maps, const Fp8MmParams &p, int ar, int grid, cudaStream_t st) {
  if constexpr (BN == 256)
    if (ar == 32) return p.split > 1 ? launch_f8<GATED, BN, 32, true, OutT>(maps, p, grid, st) : launch_f8<GATED, BN, 32, false, OutT>(maps, p, grid, st);
  if (ar <= 64) return p.split > 1 ? launch_f8<GATED, BN, 64, true, OutT>(maps, p, grid, st) : launch_f8<GATED, BN, 64, false, OutT>(maps, p, grid, st);
  if constexpr (!GATED)
    if (p.split > 1) return launch_f8<false, BN, 128, true, OutT>(maps, p, grid, st);
  return launch_f8<GATED, BN, 128, false, OutT>(maps, p, grid, st);
}
template <bool GATED, typename OutT>
static int launch_f8_shape(const F8Maps &maps, const Fp8MmParams &p, int bn, int ar, int grid, cudaStream_t st) {
  if constexpr (!GATED)
    if (bn == 128) return launch_f8_rows<false, 128, OutT>(maps, p, ar, grid, st);
  return launch_f8_rows<GATED, 256, OutT>(maps, p, ar, grid, st);
}

int launch_fp8_mm(Fp8MmParams p, cudaStream_t st) {
  if (p.rows == 0 || p.nseg == 0) return 1;
  if (!p.status && !(p.status = fp8_status_word())) return 0;
  if (p.nseg > F8_MAX_SEGS) {
    coli_set_error("fp8 product: %d segments (at most %d)", p.nseg, F8_MAX_SEGS);
    return 0;
  }
  p.KT = (p.K + 127) / 128;
  p.Op = round_up(p.O, 16);
  if (fp8_stream_ok(p)) return launch_fp8_stream(p, st);
  const bool gated = p.h_codes != nullptr;
  const Fp8Plan plan = fp8_plan(p);
  const int ar = plan.ar, bn = plan.bn, most = plan.most;
  p.split = plan.split;
  p.n_tiles = plan.n_tiles;
  F8Maps maps;
  // One segment has full boxes and a last one; behind counts on the device any may come (an encoding takes 0.3 us).
  auto box_of = [](int n) {
    int b = 0;
    while ((8 << b) < n) ++b;
    return b;
  };
  const int last = p.rows % ar ? p.rows % ar : ar;
  for (int b = 0; b < F8_MAPS; ++b)
    if (p.seg_count || b == box_of(last) || (b == box_of(ar) && p.rows >= ar))
      if (!make_codes_map(&maps.m[b], p.codes, p.rows, p.K, p.ld, 8 << b)) return 0;
  const long bound = (long)most * p.n_tiles;
  const int clusters = (int)(bound < COLI_SMS / p.split ? bound : COLI_SMS / p.split);
  if (gated) return launch_f8_shape<true, __nv_bfloat16>(maps, p, bn, ar, clusters * p.split, st);
  if (p.y_type == COLI_TYPE_F32) return launch_f8_shape<false, float>(maps, p, bn, ar, clusters * p.split, st);
  if (p.y_type == COLI_TYPE_F16) return launch_f8_shape<false, __half>(maps, p, bn, ar, clusters * p.split, st);
  return launch_f8_shape<false, __nv_bfloat16>(maps, p, bn, ar, clusters * p.split, st);
}

// Device address of the current device's status word, looked up once per device (as the routing scratch is).
static int *g_fp8_status_addr[COLI_CUDA_MAX_DEVICES];
int *fp8_status_word() {
  int dev = -1;
  if (!coli_cuda_check(cudaGetDevice(&dev), "fp8 status: cudaGetDevice") || dev < 0 || dev >= COLI_CUDA_MAX_DEVICES) return nullptr;
  int *at = __atomic_load_n(&g_fp8_status_addr[dev], __ATOMIC_ACQUIRE);
  if (!at) {
    if (!coli_cuda_check(cudaGetSymbolAddress((void **)&at, g_fp8_status), "fp8 status: cudaGetSymbolAddress")) return nullptr;
    __atomic_store_n(&g_fp8_status_addr[dev], at, __ATOMIC_RELEASE);
  }
  return at;
}
int fp8_take_status(int *code) {
  int *at = fp8_status_word();
  if (!at) return 0;
  CK(cudaMemcpy(code, at, sizeof(int), cudaMemcpyDeviceToHost), "fp8 status read");
  if (*code) CK(cudaMemset(at, 0, sizeof(int)), "fp8 status clear");
  return 1;
}

}  // namespace colib
