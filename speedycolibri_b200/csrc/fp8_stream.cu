// The product of a few 8-bit rows with resident weights, and the expert FFN over segments of a few rows: what a decode
// step asks for.  Every byte of the weights is read once and little is computed with it, so all there is to the
// kernel is to keep enough of them in flight on every SM.
//
// A warp owns slabs of 16 output features over all k-tiles (or `ksplit` warps share a task's k-tiles and join their sums in
// a fixed order).  A slab's k-tile lies in HBM as 2 KB in a row and is copied into a ring of the warp's own, across
// the ends of tasks (16 bytes a lane: a bulk copy costs the SM's copy engine 93 cycles however short it is, and 2 KB
// at a time reach 22 bytes a clock, less than HBM gives an SM); four mma.sync of 16 features x 8 rows x 32 columns per 8 rows form the k-tile's product, which is added,
// scaled, to f32 registers.  The order of columns inside a k-tile is the same for both operands and otherwise free: a lane
// takes 16-byte chunks t and t + 4 of its feature and of its row.  Rows come straight from global memory (every warp of
// the SM reads the same few kilobytes, out of L1).
#include "fp8.cuh"
#include "fp8_common.cuh"
#include "tc_common.cuh"

namespace colib {

constexpr int FS_WARPS = 16;
constexpr int FS_THREADS = FS_WARPS * 32;

template <int M, int NT>
struct FsSmem {
  static constexpr int UNIT = M * 2048;
  static constexpr int RED = FS_WARPS * M * NT * 512;  // partial sums of warps that share a task
  static constexpr int RING = (220 * 1024 - RED) / UNIT * UNIT;
  static constexpr int SLOTS = RING / UNIT;
  static constexpr int TABLES = 2 * (F8_MAX_SEGS + 1) * 4;
  static constexpr int BYTES = 128 + RING + RED + 8 * SLOTS + 16 + TABLES;
  static_assert(BYTES <= 227 * 1024, "shared memory");
};

__device__ __forceinline__ void mma_e4m3(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int NT>
struct FsRows {
  uint4 lo[NT], hi[NT];  // chunks t and t + 4 of row 8 nt + g
  float sx[NT][2];       // scales of rows 8 nt + 2 t and the next
};
// 16 bytes of codes from column k0 on; columns past K give zeros, whatever lies there
__device__ __forceinline__ uint4 fs_chunk(const uint8_t *p, int left) {
  if (left <= 0) return make_uint4(0u, 0u, 0u, 0u);
  uint4 v = __ldg(reinterpret_cast<const uint4 *>(p));
  if (left < 16) {
    uint32_t *w = reinterpret_cast<uint32_t *>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = left - 4 * i;
      w[i] = n >= 4 ? w[i] : n <= 0 ? 0u : w[i] & (0xffffffffu >> (32 - 8 * n));
    }
  }
  return v;
}
// the same of an f32 row that is still to be quantised: four lanes share a row's 128 columns
__device__ __forceinline__ void fs_quantise(const float *x, int left, uint4 &lo, uint4 &hi, float &scale) {
  float4 v[8];
  float a = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int c = (i >> 2) * 64 + (i & 3) * 4;
    v[i] = c < left ? __ldcg(reinterpret_cast<const float4 *>(x + c)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    a = fmaxf(a, fmaxf(fmaxf(fabsf(v[i].x), fabsf(v[i].y)), fmaxf(fabsf(v[i].z), fabsf(v[i].w))));
  }
  a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 1));
  a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 2));
  scale = row_scale(a);
  const float inv = __frcp_rn(scale);
  auto word = [&](float4 f) { return e4m3x4(f.x * inv, f.y * inv, f.z * inv, f.w * inv); };
  lo = make_uint4(word(v[0]), word(v[1]), word(v[2]), word(v[3]));
  hi = make_uint4(word(v[4]), word(v[5]), word(v[6]), word(v[7]));
}

// GATED: units hold a slab of gate and one of up.  HIN: the rows are the f32 h of the gated call, quantised here.  M: slabs
// of a unit.  NT: groups of 8 rows.
template <bool GATED, bool HIN, int M, int NT, typename OutT>
__global__ void __launch_bounds__(FS_THREADS, 1) k_fp8_stream(const Fp8MmParams p) {
  using S = FsSmem<M, NT>;
  constexpr int ROWS = 8 * NT;
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
  // Counts and codes are written by earlier launches; weights are not.  One segment's table needs no counts; behind the
  // gated call the counts are complete already (it gives way to this one after its own wait).
  const bool early = !p.seg_count || HIN;
  if (!early) coli_grid_wait();
  if (warp == 0) f8_tables<ROWS>(p, row_off, tile_off, lane);
  __syncthreads();
  const int tasks = tile_off[p.nseg], ks = p.split;
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
  int issued = 0, i_task = first, i_kt = kt0;
  const uint8_t *q0 = nullptr, *q1 = nullptr;
  bool both = true;
  int i_slot = 0;
  bool alive = true;
  auto issue = [&]() {  // the next unit into its slot (whole warp)
    if (i_kt == kt0) {
      const F8Tile tile = f8_tile<ROWS>(tile_off, row_off, p.nseg, i_task);
      const int ex = p.seg_expert ? p.seg_expert[tile.seg] : tile.seg;
      const size_t at = (size_t)tile.nt * (GATED ? 16 : 16 * M) * 128;
      q0 = (p.w0 ? p.w0[ex].q : p.one.q) + at;
      q1 = GATED ? p.w1[ex].q + at : nullptr;
      both = (tile.nt + 1) * 16 * M <= p.Op;
    }
    const uint32_t dst = ring + (uint32_t)i_slot * S::UNIT + (uint32_t)lane * 16;
    const size_t off = (size_t)i_kt * p.Op * 128 + lane * 16;
#pragma unroll
    for (int c = 0; c < M * 4; ++c) {
      if (GATED && c >= 4)
        cp_async16(dst + c * 512, q1 + off + (c - 4) * 512);
      else if (GATED || M == 1 || c < 4 || both)  // (the last unit of an odd number of slabs is half a one)
        cp_async16(dst + c * 512, q0 + off + c * 512);
    }
    // the lane's copies count once they have landed
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar + 8u * (uint32_t)i_slot) : "memory");
    if (++i_slot == depth) i_slot = 0;
    ++issued;
    if (++i_kt == kt1) {
      i_kt = kt0;
      i_task += stride;
    }
  };
  while (issued < depth && issued < n_units) issue();
  if (early) coli_grid_wait();
  coli_grid_trigger();  // (behind the wait: what a successor reads early is complete then)

  int used = 0, slot = 0;
  uint32_t phase = 0;
  for (int task = first; works && task < tasks; task += stride) {
    const F8Tile tile = f8_tile<ROWS>(tile_off, row_off, p.nseg, task);
    const int ex = p.seg_expert ? p.seg_expert[tile.seg] : tile.seg;
    const int f0 = tile.nt * (GATED ? 16 : 16 * M);
    const float *w0s = reinterpret_cast<const float *>(p.w0 ? p.w0[ex].s : p.one.s) + (size_t)(f0 >> 7) * p.KT;
    const float *w1s = GATED ? reinterpret_cast<const float *>(p.w1[ex].s) + (size_t)(f0 >> 7) * p.KT : w0s;
    auto row_of = [&](int n) { return tile.row0 + min(n, tile.nrows - 1); };
    auto request = [&](FsRows<NT> &r, int kt) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int k0 = kt * 128 + 16 * t;
        if constexpr (HIN) {
          float s;
          fs_quantise(p.h32 + (long)row_of(8 * n + g) * p.K + k0, p.K - k0, r.lo[n], r.hi[n], s);
          r.sx[n][0] = __shfl_sync(0xffffffffu, s, 8 * t);
          r.sx[n][1] = __shfl_sync(0xffffffffu, s, 8 * t + 4);
        } else {
          const uint8_t *c = (const uint8_t *)p.codes + (long)row_of(8 * n + g) * p.ld + k0;
          r.lo[n] = fs_chunk(c, p.K - k0);
          r.hi[n] = fs_chunk(c + 64, p.K - k0 - 64);
#pragma unroll
          for (int i = 0; i < 2; ++i) r.sx[n][i] = __ldg(p.sx + (long)row_of(8 * n + 2 * t + i) * p.s_row + (long)kt * p.s_blk);
        }
      }
    };
    float acc[M][NT][4] = {};
    FsRows<NT> next;
    float sw0 = 0.0f, sw1 = 0.0f;
    request(next, kt0);
    sw0 = __ldg(w0s + kt0);
    if (GATED) sw1 = __ldg(w1s + kt0);
    for (int kt = kt0; kt < kt1; ++kt, ++used) {
      const FsRows<NT> rows = next;
      const float s0 = sw0, s1 = GATED ? sw1 : sw0;
      if (kt + 1 < kt1) {
        request(next, kt + 1);
        sw0 = __ldg(w0s + kt + 1);
        if (GATED) sw1 = __ldg(w1s + kt + 1);
      }
      alive = alive && __all_sync(0xffffffffu, mbar_wait(bar + 8u * (uint32_t)slot, phase, abort_flag, status, TC_ERR_TMA_WAIT));
      const uint32_t src = ring + (uint32_t)slot * S::UNIT + (uint32_t)g * 128;
#pragma unroll
      for (int m = 0; m < M; ++m) {
        const uint32_t at = src + m * 2048, c0 = (uint32_t)(t ^ g) * 16, c1 = (uint32_t)((t + 4) ^ g) * 16;
        const uint4 a0 = lds128(at + c0), a1 = lds128(at + 1024 + c0), a2 = lds128(at + c1), a3 = lds128(at + 1024 + c1);
        const float sw = m == 0 || !GATED ? s0 : s1;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          mma_e4m3(d, a0.x, a1.x, a2.x, a3.x, rows.lo[n].x, rows.hi[n].x);
          mma_e4m3(d, a0.y, a1.y, a2.y, a3.y, rows.lo[n].y, rows.hi[n].y);
          mma_e4m3(d, a0.z, a1.z, a2.z, a3.z, rows.lo[n].z, rows.hi[n].z);
          mma_e4m3(d, a0.w, a1.w, a2.w, a3.w, rows.lo[n].w, rows.hi[n].w);
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[m][n][i] = fmaf(d[i], rows.sx[n][i & 1] * sw, acc[m][n][i]);
        }
      }
      if (++slot == depth) {
        slot = 0;
        phase ^= 1u;
      }
      __syncwarp();  // the slot has been read
      if (alive && issued < n_units) issue();
    }
    if (ks > 1) {
      // join the sums of the warps that share the task, in their order
      constexpr int N = M * NT * 4;
      float *mine = red + (size_t)warp * N * 32;
#pragma unroll
      for (int i = 0; i < N; ++i) mine[i * 32 + lane] = acc[i / (4 * NT)][i / 4 % NT][i % 4];
      asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(ks * 32) : "memory");
      if (sub == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          float s = mine[i * 32 + lane];
          for (int w = 1; w < ks; ++w) s += mine[(size_t)w * N * 32 + i * 32 + lane];
          acc[i / (4 * NT)][i / 4 % NT][i % 4] = s;
        }
      }
      asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(ks * 32) : "memory");
    }
    if (sub == 0 && alive) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 8 * n + 2 * t + (i & 1);
          if (r >= tile.nrows) continue;
          if constexpr (GATED) {
            const int f = f0 + g + 8 * (i >> 1);
            if (f < p.O) p.h32[(long)(tile.row0 + r) * p.O + f] = coli_act_fast(acc[0][n][i], acc[1][n][i], p.act);
          } else {
#pragma unroll
            for (int m = 0; m < M; ++m) {
              const int f = f0 + 16 * m + g + 8 * (i >> 1);
              if (f < p.O) ((OutT *)p.y)[(long)(tile.row0 + r) * p.y_stride + f] = f8_out<OutT>(acc[m][n][i]);
            }
          }
        }
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");  // (none are left unless a wait gave up)
}

template <bool GATED, bool HIN, int M, int NT, typename OutT>
static int launch_fs(const Fp8MmParams &p, int grid, cudaStream_t st) {
  static ColiPerDeviceOnce attr_once;
  auto *kernel = k_fp8_stream<GATED, HIN, M, NT, OutT>;
  constexpr int bytes = FsSmem<M, NT>::BYTES;
  if (!coli_set_smem_limit(attr_once, kernel, bytes, "fp8 stream shared-memory attribute")) return 0;
  coli_count_launch(1);
  return coli_cuda_check(launch_dependent(kernel, dim3((unsigned)grid), dim3(FS_THREADS), bytes, st, p), "fp8 stream launch") ? 1 : 0;
}
template <bool HIN, typename OutT>
static int launch_fs_shape(const Fp8MmParams &p, int m, int nt, int grid, cudaStream_t st) {
  if (m == 2) return nt == 1 ? launch_fs<false, HIN, 2, 1, OutT>(p, grid, st) : launch_fs<false, HIN, 2, 2, OutT>(p, grid, st);
  return nt == 1 ? launch_fs<false, HIN, 1, 1, OutT>(p, grid, st) : launch_fs<false, HIN, 1, 2, OutT>(p, grid, st);
}

int launch_fp8_stream(Fp8MmParams p, cudaStream_t st) {
  const bool gated = p.w1 != nullptr;
  const int segs = p.seg_count ? (p.rows_expected < p.nseg ? p.rows_expected : p.nseg) : 1;
  // rows of a task: 8, or 16 where many segments have more than 8
  const int nt = p.rows_expected <= (p.seg_count ? 3L : 8L) * segs ? 1 : 2, rows = 8 * nt;
  const long chunks = p.seg_count ? segs + p.rows_expected / rows : (p.rows + rows - 1) / rows;
  // two slabs a unit where that still leaves every warp a task
  const int m = gated || chunks * ((p.O + 31) / 32) >= (long)COLI_SMS * FS_WARPS ? 2 : 1;
  p.n_tiles = (p.O + (gated ? 16 : 16 * m) - 1) / (gated ? 16 : 16 * m);
  const long tasks = (chunks > 0 ? chunks : 1) * p.n_tiles;
  p.split = 1;
  while (p.split < FS_WARPS && tasks * p.split * 2 <= (long)COLI_SMS * FS_WARPS && p.split * 2 <= p.KT) p.split *= 2;
  const long most = p.seg_count ? (p.rows / rows + (p.rows < p.nseg ? p.rows : p.nseg)) * (long)p.n_tiles : tasks;
  const int grid = (int)(most < COLI_SMS ? most : COLI_SMS);
  if (gated) return nt == 1 ? launch_fs<true, false, 2, 1, float>(p, grid, st) : launch_fs<true, false, 2, 2, float>(p, grid, st);
  if (p.h32) return launch_fs_shape<true, __nv_bfloat16>(p, m, nt, grid, st);
  if (p.y_type == COLI_TYPE_F32) return launch_fs_shape<false, float>(p, m, nt, grid, st);
  if (p.y_type == COLI_TYPE_F16) return launch_fs_shape<false, __half>(p, m, nt, grid, st);
  return launch_fs_shape<false, __nv_bfloat16>(p, m, nt, grid, st);
}

}  // namespace colib
