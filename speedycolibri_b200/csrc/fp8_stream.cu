// The product of a few 8-bit rows with resident weights, and the expert FFN over segments of a few rows: what a decode
// step asks for.  Every byte of the weights is read once and little is computed with it, so all there is to the
// kernel is to keep enough of them in flight on every SM.
//
// A warp owns slabs of 16 output features over all k-tiles (or `split` warps share a task's k-tiles and join their sums in
// a fixed order).  A slab's k-tile lies in HBM as 2 KB in a row; with the k-tile's columns of the task's rows and the scales of
// both it is copied into a ring of the warp's own, across the ends of tasks, 16 bytes a lane.  (A bulk copy costs the SM's copy
// engine 93 cycles however short it is: 2 KB at a time reach 22 bytes a clock, less than HBM gives an SM.  And whatever a
// warp loads into registers returns behind all copies the SM has asked for before, some 180 KB: with rows and scales
// loaded that way 64 rows on 128 experts, H 2048, I 768, took 81 us.)  Four mma.sync of 16 features x 8 rows x 32
// columns per 8 rows form the k-tile's product, which is added, scaled, to f32 registers.  The order of columns inside a
// k-tile is the same for both operands and otherwise free: a lane takes 16-byte chunks t and t + 4 of its feature and row.
#include "fp8.cuh"
#include "fp8_common.cuh"
#include "tc_common.cuh"

namespace colib {

constexpr int FS_WARPS = 16;
constexpr int FS_THREADS = FS_WARPS * 32;

constexpr int FS_ROWS = 8;  // of a task

template <int M>
struct FsSmem {
  static constexpr int ROWS = M * 2048, SCALES = ROWS + FS_ROWS * 128;  // a slot: slabs, rows' codes, scales (sx, then sw)
  static constexpr int UNIT = SCALES + 128;
  static constexpr int RED = FS_WARPS * M * 512;  // partial sums of warps that share a task
  static constexpr int RING = (218 * 1024 - RED) / UNIT * UNIT;
  static constexpr int SLOTS = RING / UNIT;
  static constexpr int TABLES = 2 * (F8_MAX_SEGS + 1) * 4;
  static constexpr int BYTES = 128 + RING + RED + 8 * SLOTS + 16 + TABLES;
  static_assert(BYTES <= 227 * 1024, "shared memory");
};

// `n` bytes (0 .. 16) from global memory and zeros behind them; 4 bytes, or a zero
__device__ __forceinline__ void cp_async_part(uint32_t dst, const void *src, int n) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_word(uint32_t dst, const void *src, int n) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ float lds32(uint32_t addr) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ void mma_e4m3(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// GATED: units hold a slab of gate and one of up.  M: slabs of a unit.
template <bool GATED, int M, typename OutT>
__global__ void __launch_bounds__(FS_THREADS, 1) k_fp8_stream(const __grid_constant__ Fp8MmParams p) {
  using S = FsSmem<M>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char *smem = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~(uintptr_t)127);
  float *red = reinterpret_cast<float *>(smem + S::RING);
  unsigned char *after = smem + S::RING + S::RED;
  const uint32_t ring0 = smem_u32(smem), bars = smem_u32(after);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(after + 8 * S::SLOTS);
  int *row_off = reinterpret_cast<int *>(after + 8 * S::SLOTS + 16), *tile_off = row_off + F8_MAX_SEGS + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  int *status = p.status;

  for (int i = threadIdx.x; i < S::SLOTS; i += FS_THREADS) mbar_init(bars + 8 * i, 32);
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // Counts, codes and scales of rows are written by earlier launches; weights are not.  One segment's table needs no counts.
  // Behind the gated call and the quantiser the counts are complete: the gated call lets its successor start after its own wait.
  const bool early = !p.seg_count || p.behind_gated;
  if (!early) coli_grid_wait();
  if (warp == 0) f8_tables<FS_ROWS>(p, row_off, tile_off, lane);
  __syncthreads();
  const int tasks = tile_off[p.nseg], ks = p.split;
  if (GATED && blockIdx.x == 0 && threadIdx.x == 0) *p.rows_used = row_off[p.nseg];
  // as many of the warps at work as make the rounds come out even, and the ring shared among those
  const int most = FS_WARPS / ks, rounds = (tasks + (int)gridDim.x * most - 1) / ((int)gridDim.x * most);
  const int groups = rounds > 0 ? min(most, (tasks + (int)gridDim.x * rounds - 1) / ((int)gridDim.x * rounds)) : 0;
  const int depth = groups > 0 ? S::SLOTS / (groups * ks) : 1;
  const int group = warp / ks, sub = warp % ks;
  const int stride = (int)gridDim.x * groups;
  const int kt0 = (int)((long)p.KT * sub / ks), kt1 = (int)((long)p.KT * (sub + 1) / ks), per_task = kt1 - kt0;
  const int first = (int)blockIdx.x * groups + group;
  const bool works = group < groups && first < tasks;
  const uint32_t ring = ring0 + (uint32_t)(warp * depth) * S::UNIT, bar = bars + 8u * (uint32_t)(warp * depth);
  const int n_units = works ? ((tasks - first + stride - 1) / stride) * per_task : 0;

  // the copies: unit u is k-tile kt0 + u % per_task of the warp's task u / per_task
  int issued = 0, i_task = first, i_kt = kt0, i_slot = 0, i_rows = 0;
  const uint8_t *q0 = nullptr, *q1 = nullptr, *codes = nullptr;
  const float *scale = nullptr;  // lanes 0 .. 7: their row's; the next two: the weights'
  bool both = true, alive = true;
  // where a task's operands are, looked up a task ahead (the expert's index and its table entry are two reads in a row)
  struct Task {
    const uint8_t *q0, *q1;
    const float *scale;
    int row0, nrows;
    bool both;
  } ahead_task = {};
  auto look_up = [&](int task) {
    if (task >= tasks) return;
    const F8Tile tile = f8_tile<FS_ROWS>(tile_off, row_off, p.nseg, task);
    const int ex = p.seg_expert ? p.seg_expert[tile.seg] : tile.seg;
    const WeightRef w0 = p.w0 ? p.w0[ex] : p.one, w1 = GATED ? p.w1[ex] : w0;
    const int f0 = tile.nt * (GATED ? 16 : 16 * M);
    ahead_task.q0 = w0.q + (size_t)f0 * 128;
    ahead_task.q1 = w1.q + (size_t)f0 * 128;
    ahead_task.scale = lane < FS_ROWS ? p.sx + (long)(tile.row0 + min(lane, tile.nrows - 1)) * p.s_row
                                   : reinterpret_cast<const float *>(lane == FS_ROWS ? w0.s : w1.s) + (size_t)(f0 >> 7) * p.KT;
    ahead_task.row0 = tile.row0;
    ahead_task.nrows = tile.nrows;
    ahead_task.both = f0 + 16 * M <= p.Op;
  };
  if (works) look_up(first);
  const long scale_step = lane < FS_ROWS ? p.s_blk : 1;
  auto issue_weights = [&]() {
    if (i_kt == kt0) {
      q0 = ahead_task.q0 + lane * 16;
      q1 = ahead_task.q1 + lane * 16;
      both = ahead_task.both;
      i_rows = ahead_task.nrows;
      codes = (const uint8_t *)p.codes + (long)(ahead_task.row0 + (lane >> 3)) * p.ld + (lane & 7) * 16;
      scale = ahead_task.scale;
      look_up(i_task + stride);
    }
    const uint32_t dst = ring + (uint32_t)i_slot * S::UNIT + (uint32_t)lane * 16;
    const size_t off = (size_t)i_kt * p.Op * 128;
#pragma unroll
    for (int c = 0; c < M * 4; ++c) {
      if (GATED && c >= 4)
        cp_async16(dst + c * 512, q1 + off + (c - 4) * 512);
      else if (GATED || M == 1 || c < 4 || both)  // (the last unit of an odd number of slabs is half a one)
        cp_async16(dst + c * 512, q0 + off + c * 512);
    }
  };
  auto issue_rows = [&]() {
    const uint32_t dst = ring + (uint32_t)i_slot * S::UNIT, c0 = (uint32_t)(lane & 7);
    const int left = p.K - i_kt * 128 - (lane & 7) * 16;
#pragma unroll
    for (int i = 0; i < FS_ROWS / 4; ++i) {  // rows 4 i + lane / 8; a missing row and columns past K are zeros
      const int r = 4 * i + (lane >> 3), n = r < i_rows ? max(0, min(16, left)) : 0;
      cp_async_part(dst + S::ROWS + (uint32_t)r * 128 + ((c0 ^ (uint32_t)(r & 7)) << 4), n ? codes + 4 * i * p.ld + (long)i_kt * 128 : codes, n);
    }
    if (lane < FS_ROWS + 2) cp_async_word(dst + S::SCALES + (uint32_t)lane * 4, scale + (long)i_kt * scale_step, 4);
    // the lane's copies count once they have landed
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar + 8u * (uint32_t)i_slot) : "memory");
    if (++i_slot == depth) i_slot = 0;
    ++issued;
    if (++i_kt == kt1) {
      i_kt = kt0;
      i_task += stride;
    }
  };
  // One segment: the weights of the ring's first fill (part of one task as a rule) before the wait, its rows behind it.
  const int ahead = early ? min(min(depth, n_units), per_task) : 0;
  for (int u = 0; u < ahead; ++u) {
    issue_weights();
    ++i_kt;
    ++i_slot;
  }
  if (early) coli_grid_wait();
  coli_grid_trigger();
  i_kt = kt0;
  i_slot = 0;
  for (int u = 0; u < ahead; ++u) issue_rows();
  auto issue = [&]() {
    issue_weights();
    issue_rows();
  };
  while (issued < depth && issued < n_units) issue();

  int used = 0, slot = 0;
  uint32_t phase = 0;
  for (int task = first; works && task < tasks; task += stride) {
    const F8Tile tile = f8_tile<FS_ROWS>(tile_off, row_off, p.nseg, task);
    const int f0 = tile.nt * (GATED ? 16 : 16 * M);
    float acc[M][4] = {};
    float least = 1.0f;  // product of scales so far (one that is too large shows in the sums)
    for (int kt = kt0; kt < kt1; ++kt, ++used) {
      alive = alive && __all_sync(0xffffffffu, mbar_wait(bar + 8u * (uint32_t)slot, phase, abort_flag, status, TC_ERR_TMA_WAIT));
      const uint32_t unit = ring + (uint32_t)slot * S::UNIT, c0 = (uint32_t)(t ^ g) * 16, c1 = (uint32_t)((t + 4) ^ g) * 16;
      const uint32_t r = unit + S::ROWS + (uint32_t)g * 128;
      const uint4 lo = lds128(r + c0), hi = lds128(r + c1);
      const float sx[2] = {lds32(unit + S::SCALES + (uint32_t)t * 8), lds32(unit + S::SCALES + (uint32_t)t * 8 + 4)};
      const float s0 = lds32(unit + S::SCALES + FS_ROWS * 4), s1 = GATED ? lds32(unit + S::SCALES + FS_ROWS * 4 + 4) : s0;
#pragma unroll
      for (int m = 0; m < M; ++m) {
        const uint32_t at = unit + (uint32_t)g * 128 + m * 2048;
        const uint4 a0 = lds128(at + c0), a1 = lds128(at + 1024 + c0), a2 = lds128(at + c1), a3 = lds128(at + 1024 + c1);
        const float sw = m == 0 || !GATED ? s0 : s1;
        float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        mma_e4m3(d, a0.x, a1.x, a2.x, a3.x, lo.x, hi.x);
        mma_e4m3(d, a0.y, a1.y, a2.y, a3.y, lo.y, hi.y);
        mma_e4m3(d, a0.z, a1.z, a2.z, a3.z, lo.z, hi.z);
        mma_e4m3(d, a0.w, a1.w, a2.w, a3.w, lo.w, hi.w);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[m][i] = fmaf(d[i], sx[i & 1] * sw, acc[m][i]);
        if (m == 0 || GATED) least = fminf(least, fminf(fabsf(sx[0] * sw), fabsf(sx[1] * sw)));
      }
      if (++slot == depth) {
        slot = 0;
        phase ^= 1u;
      }
      __syncwarp();  // the slot has been read
      if (alive && issued < n_units) issue();
    }
    if (alive && !(least >= 1.17549435e-38f)) {
      // too small a product, or a scale of 0: NaN where it asks for a closer look at the end
      const int ex = p.seg_expert ? p.seg_expert[tile.seg] : tile.seg;
      const WeightRef w0 = p.w0 ? p.w0[ex] : p.one, w1 = GATED ? p.w1[ex] : w0;
      const size_t sw = (size_t)(f0 >> 7) * p.KT;
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (f8_again(p.sx + (long)(tile.row0 + min(2 * t + j, tile.nrows - 1)) * p.s_row, p.s_blk, reinterpret_cast<const float *>(w0.s) + sw,
                     reinterpret_cast<const float *>(w1.s) + sw, kt0, kt1)) {
#pragma unroll
          for (int m = 0; m < M; ++m) acc[m][j] = acc[m][j + 2] = __uint_as_float(0x7fffffffu);
        }
    }
    __syncwarp();
    if (ks > 1) {
      // join the sums of the warps that share the task, in their order
      constexpr int N = M * 4;
      float *mine = red + (size_t)warp * N * 32;
#pragma unroll
      for (int i = 0; i < N; ++i) mine[i * 32 + lane] = acc[i / 4][i % 4];
      asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(ks * 32) : "memory");
      if (sub == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          float s = mine[i * 32 + lane];
          for (int w = 1; w < ks; ++w) s += mine[(size_t)w * N * 32 + i * 32 + lane];
          acc[i / 4][i % 4] = s;
        }
      }
      asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(ks * 32) : "memory");
    }
    if (sub == 0 && alive) {
      auto store = [&](int r, int m, int f, float v) {
        if constexpr (GATED)
          p.h32[(long)(tile.row0 + r) * p.O + f] = v;
        else
          ((OutT *)p.y)[(long)(tile.row0 + r) * p.y_stride + f + 16 * m] = f8_out<OutT>(v);
      };
      bool look = false;
#pragma unroll
      for (int i = 0; i < 4 * M; ++i) look = look || !(fabsf(acc[i / 4][i % 4]) <= 3.4028235e38f);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 2 * t + (i & 1), f = f0 + g + 8 * (i >> 1);
        if (r >= tile.nrows) continue;
        if constexpr (GATED) {
          if (f < p.O) store(r, 0, f, coli_act_fast(acc[0][i], acc[1][i], p.act));
        } else {
#pragma unroll
          for (int m = 0; m < M; ++m)
            if (f + 16 * m < p.O) store(r, m, f, acc[m][i]);
        }
      }
      if (look) {
        // a sum is infinite or none: where scales whose product is no normal number are the reason, the lane's results from their codes
        const int ex = p.seg_expert ? p.seg_expert[tile.seg] : tile.seg;
        const WeightRef w0 = p.w0 ? p.w0[ex] : p.one, w1 = GATED ? p.w1[ex] : w0;
        const size_t sw = (size_t)(f0 >> 7) * p.KT;
        const float *s0 = reinterpret_cast<const float *>(w0.s) + sw, *s1 = reinterpret_cast<const float *>(w1.s) + sw;
#pragma unroll 1
        for (int r = 2 * t; r < min(2 * t + 2, tile.nrows); ++r) {
          const uint8_t *q = (const uint8_t *)p.codes + (long)(tile.row0 + r) * p.ld;
          const float *sr = p.sx + (long)(tile.row0 + r) * p.s_row;
          if (!f8_again(sr, p.s_blk, s0, s1, 0, p.KT)) continue;
          auto sum = [&](const uint8_t *w, const float *s, int f) {
            return f8_sum_again<1>(q, sr, p.s_blk, p.K, w + (size_t)f * 128, (size_t)p.Op * 128, f & 7, s, 0, p.KT);
          };
#pragma unroll 1
          for (int f = f0 + g; f < min(f0 + (GATED ? 16 : 16 * M), p.O); f += 8) {
            const float v = sum(w0.q, s0, f);
            store(r, 0, f, GATED ? coli_act_fast(v, sum(w1.q, s1, f), p.act) : v);
          }
        }
      }
      __syncwarp();
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");  // (none are left unless a wait gave up)
}

template <bool GATED, int M, typename OutT>
static int launch_fs(const Fp8MmParams &p, int grid, cudaStream_t st) {
  static ColiPerDeviceOnce attr_once;
  auto *kernel = k_fp8_stream<GATED, M, OutT>;
  constexpr int bytes = FsSmem<M>::BYTES;
  if (!coli_set_smem_limit(attr_once, kernel, bytes, "fp8 stream shared-memory attribute")) return 0;
  coli_count_launch(1);
  return coli_cuda_check(launch_dependent(kernel, dim3((unsigned)grid), dim3(FS_THREADS), bytes, st, p), "fp8 stream launch") ? 1 : 0;
}
template <typename OutT>
static int launch_fs_slabs(const Fp8MmParams &p, int m, int grid, cudaStream_t st) {
  return m == 2 ? launch_fs<false, 2, OutT>(p, grid, st) : launch_fs<false, 1, OutT>(p, grid, st);
}

int launch_fp8_stream(Fp8MmParams p, cudaStream_t st) {
  const bool gated = p.w1 != nullptr;
  const int segs = p.seg_count ? (p.rows_expected < p.nseg ? p.rows_expected : p.nseg) : 1;
  const long chunks = p.seg_count ? segs + p.rows_expected / FS_ROWS : 1;
  // two slabs a unit where that still leaves every warp a task
  const int m = gated || chunks * ((p.O + 31) / 32) >= (long)COLI_SMS * FS_WARPS ? 2 : 1;
  p.n_tiles = (p.O + (gated ? 16 : 16 * m) - 1) / (gated ? 16 : 16 * m);
  const long tasks = (chunks > 0 ? chunks : 1) * p.n_tiles;
  p.split = 1;
  while (p.split < FS_WARPS && tasks * p.split * 2 <= (long)COLI_SMS * FS_WARPS && p.split * 2 <= p.KT) p.split *= 2;
  const long most = p.seg_count ? (p.rows / FS_ROWS + (p.rows < p.nseg ? p.rows : p.nseg)) * (long)p.n_tiles : tasks;
  const int grid = (int)(most < COLI_SMS ? most : COLI_SMS);
  if (gated) return launch_fs<true, 2, float>(p, grid, st);
  if (p.y_type == COLI_TYPE_F32) return launch_fs_slabs<float>(p, m, grid, st);
  if (p.y_type == COLI_TYPE_F16) return launch_fs_slabs<__half>(p, m, grid, st);
  return launch_fs_slabs<__nv_bfloat16>(p, m, grid, st);
}

}  // namespace colib
