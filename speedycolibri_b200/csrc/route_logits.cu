// Routing from given logits: scores, choice of experts, weights, and the rows the chosen pairs take in expert order.
// The rules are those of the block's own router (crates/colibri-engine/src/moe.rs:1047-1132; groups and the logit bias
// as in routing.cu), with two differences that a caller's own logits make necessary: the choice is made on scores in 64
// bits, so that experts whose scores 32 bits do not tell apart still come in the order of their logits, and an expert whose
// logit is -inf or NaN is not chosen at all (a closed expert, a padded token), where the block's router falls back to expert 0.
#include "route_logits.cuh"

namespace colib {

constexpr int RL_WARPS = 8;
// per warp: candidate keys and scores, their ids
constexpr int RL_CAND_BYTES = 32 * (8 + 8 + 4);

template <typename T>
__device__ __forceinline__ double rl_load(const T *p);
template <>
__device__ __forceinline__ double rl_load<float>(const float *p) { return (double)__ldg(p); }
template <>
__device__ __forceinline__ double rl_load<__half>(const __half *p) { return (double)__half2float(__ldg(p)); }
template <>
__device__ __forceinline__ double rl_load<__nv_bfloat16>(const __nv_bfloat16 *p) { return (double)__bfloat162float(__ldg(p)); }

// order-preserving key of a value above -inf (never 0); 0 for what cannot be chosen
__device__ __forceinline__ uint64_t rl_key(double v) {
  const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);  // (-0 and 0 tie)
  return (b >> 63) ? ~b : (b | 0x8000000000000000ull);
}
__device__ __forceinline__ double rl_warp_max(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ double rl_warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct RlCand {
  uint64_t *key;
  double *score;
  int *id;
};

// The k best keys of a warp (lane + 32 s holds expert lane + 32 s; largest key, then lowest expert; 0 is none) into places
// 0 .. of `c`, in order.  Returns how many there are, at most k.  The k-th largest of the lanes' best keys bounds the k-th largest of
// all from below (taken by its upper word alone): a little over k candidates as a rule, and each finds its place by
// counting.  More than 32 of them (many equal logits) take k rounds.
template <int SLOTS>
__device__ __forceinline__ int rl_select(const uint64_t (&key)[SLOTS], const double (&score)[SLOTS], int k, const RlCand &c, int lane) {
  uint64_t best = 0;
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) best = key[s] > best ? key[s] : best;
  const uint32_t bhi = (uint32_t)(best >> 32);
  uint32_t *hi = reinterpret_cast<uint32_t *>(c.key);
  hi[lane] = bhi;
  __syncwarp();
  int above = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint4 q = reinterpret_cast<const uint4 *>(hi)[j];
    above += (q.x > bhi) + (q.y > bhi) + (q.z > bhi) + (q.w > bhi);
  }
  const uint32_t bound = max(1u, __reduce_min_sync(0xffffffffu, above < k ? bhi : 0xffffffffu));
  uint32_t holders[SLOTS];
  int n = 0;
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) {
    holders[s] = __ballot_sync(0xffffffffu, (uint32_t)(key[s] >> 32) >= bound);
    n += __popc(holders[s]);
  }
  if (n <= 32) {
    int at = 0;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
      if ((uint32_t)(key[s] >> 32) >= bound) {
        const int i = at + __popc(holders[s] & ((1u << lane) - 1u));
        c.key[i] = key[s];
        c.score[i] = score[s];
        c.id[i] = s * 32 + lane;
      }
      at += __popc(holders[s]);
    }
    __syncwarp();
    const uint64_t mk = lane < n ? c.key[lane] : 0;
    const double ms = lane < n ? c.score[lane] : 0.0;
    const int mi = lane < n ? c.id[lane] : 0;
    int rank = 0;
    for (int j = 0; j < n; ++j) {  // a slot's candidates precede the next slot's and lanes ascend: j < lane is the lower id
      const uint64_t other = c.key[j];
      rank += other > mk || (other == mk && j < lane);
    }
    __syncwarp();
    if (lane < n && rank < k) {
      c.score[rank] = ms;
      c.id[rank] = mi;
    }
    __syncwarp();
    return min(n, k);
  }
  uint64_t left[SLOTS];
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) left[s] = key[s];
  int found = 0;
  for (; found < k; ++found) {
    uint64_t bk = 0;
    double bs = 0.0;
    int bid = 0x7fffffff;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s)
      if (left[s] > bk) {
        bk = left[s];
        bs = score[s];
        bid = s * 32 + lane;
      }
    const uint32_t top_hi = __reduce_max_sync(0xffffffffu, (uint32_t)(bk >> 32));
    if (top_hi == 0u) break;
    const uint32_t top_lo = __reduce_max_sync(0xffffffffu, (uint32_t)(bk >> 32) == top_hi ? (uint32_t)bk : 0u);
    const bool holds = (uint32_t)(bk >> 32) == top_hi && (uint32_t)bk == top_lo;
    const int win = (int)__reduce_min_sync(0xffffffffu, holds ? (uint32_t)bid : 0x7fffffffu);
    if (holds && bid == win) {
      c.score[found] = bs;
      c.id[found] = win;
#pragma unroll
      for (int s = 0; s < SLOTS; ++s)
        if (s * 32 + lane == win) left[s] = 0;
    }
  }
  __syncwarp();
  return found;
}

// One warp routes one token; `row` is E doubles of shared memory of its own (groups only).
template <typename T, int SLOTS>
__device__ __forceinline__ void rl_token(const RouteLogitsParams &p, int t, const RlCand &c, double *row, int lane) {
  const T *z0 = (const T *)p.logits + (long)t * p.stride;
  const double NEG_INF = __longlong_as_double(0xfff0000000000000ll);
  double score[SLOTS];
  bool open[SLOTS];
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) {
    const int e = lane + 32 * s;
    double z = e < p.E ? rl_load<T>(z0 + e) : NEG_INF;
    if (p.logit_bias && e < p.E) z += (double)__ldg(p.logit_bias + e);
    open[s] = z > NEG_INF;
    score[s] = open[s] ? z : NEG_INF;
  }
  if (p.score == COLI_SCORE_SOFTMAX) {
    double m = NEG_INF;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) m = fmax(m, score[s]);
    m = rl_warp_max(m);
    double sum = 0.0;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
      // (an infinite largest logit shares the mass with its equals)
      score[s] = score[s] == m ? (open[s] ? 1.0 : 0.0) : exp(score[s] - m);
      sum += score[s];
    }
    sum = rl_warp_sum(sum);
    const double inv = sum > 0.0 ? 1.0 / sum : 0.0;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) score[s] *= inv;
  } else {
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) score[s] = 1.0 / (1.0 + exp(-score[s]));
  }
  uint64_t key[SLOTS];
  double choice[SLOTS];
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) {
    const int e = lane + 32 * s;
    choice[s] = p.select_bias && e < p.E ? score[s] + (double)__ldg(p.select_bias + e) : score[s];
    key[s] = open[s] ? rl_key(choice[s]) : 0;
  }
  if (p.n_group > 1) {
    // a group's mark is the sum of its two best (of one, where only one is open); `per` lanes share a group
    const int G = p.n_group, gs = p.E / G;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s)
      if (lane + 32 * s < p.E) row[lane + 32 * s] = key[s] ? choice[s] : NEG_INF;
    __syncwarp();
    int per = 1;
    while (2 * per * G <= 32) per *= 2;
    const int g = lane / per;
    double m1 = NEG_INF, m2 = NEG_INF;
    if (g < G)
      for (int i = lane % per; i < gs; i += per) {
        const double v = row[g * gs + i];
        m2 = v > m1 ? m1 : fmax(m2, v);
        m1 = fmax(m1, v);
      }
    for (int o = 1; o < per; o <<= 1) {
      const double o1 = __shfl_xor_sync(0xffffffffu, m1, o), o2 = __shfl_xor_sync(0xffffffffu, m2, o);
      m2 = fmax(fmin(m1, o1), fmax(m2, o2));
      m1 = fmax(m1, o1);
    }
    uint64_t *gk = c.key;
    const uint64_t mark = g < G && m1 > NEG_INF ? rl_key(m2 > NEG_INF ? m1 + m2 : m1) : 0;
    if (lane % per == 0 && g < G) gk[g] = mark;
    __syncwarp();
    int above = 0;
    for (int j = 0; j < G; ++j) above += gk[j] > mark || (gk[j] == mark && j < g);
    const uint32_t kept = __ballot_sync(0xffffffffu, g < G && mark != 0 && above < p.topk_group);
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
      const int e = lane + 32 * s;
      if (e < p.E && !((kept >> ((e / gs) * per)) & 1u)) key[s] = 0;
    }
    __syncwarp();
  }
  const int n = rl_select<SLOTS>(key, score, p.k, c, lane);
  double w = lane < n ? c.score[lane] : 0.0;
  if (p.norm_topk) w /= rl_warp_sum(w) + 1e-20;
  if (lane < p.k) {
    p.idx[(long)t * p.k + lane] = lane < n ? c.id[lane] : -1;
    p.w[(long)t * p.k + lane] = (float)(w * (double)p.routed_scale);
  }
}

template <typename T>
__device__ __forceinline__ void rl_route(const RouteLogitsParams &p, int t, const RlCand &c, double *row, int lane) {
  if (p.E <= 128)
    rl_token<T, 4>(p, t, c, row, lane);
  else if (p.E <= 256)
    rl_token<T, 8>(p, t, c, row, lane);
  else
    rl_token<T, 16>(p, t, c, row, lane);
}

// Which of a chunk's tokens chose each expert, one bit each: the number of bits below a token's own is the rank of its
// pair among the chunk's rows of that expert, whatever order the warps came in.
__device__ __forceinline__ void rl_mark(uint32_t *mask, int words, const int32_t *idx, int pairs, int k, int E) {
  for (int i = threadIdx.x; i < E * words; i += blockDim.x) mask[i] = 0u;
  __syncthreads();
  for (int i = threadIdx.x; i < pairs; i += blockDim.x) {
    const int e = idx[i], j = i / k;
    if (e >= 0) atomicOr(mask + e * words + (j >> 5), 1u << (j & 31));
  }
  __syncthreads();
}
__device__ __forceinline__ int rl_rank(const uint32_t *m, int words, int j) {
  int r = 0;
  for (int w = 0; w < words; ++w) r += w < (j >> 5) ? __popc(m[w]) : w == (j >> 5) ? __popc(m[w] & ((1u << (j & 31)) - 1u)) : 0;
  return r;
}

// A chunk's pairs take the rows base[e] + rank.
__device__ __forceinline__ void rl_place(const RouteLogitsParams &p, const uint32_t *mask, const int *base, int t0, int tokens) {
  const int words = p.chunk / 32;
  for (int i = threadIdx.x; i < tokens * p.k; i += blockDim.x) {
    const long at = (long)t0 * p.k + i;
    const int e = p.idx[at], j = i / p.k;
    int slot = -1;
    if (e >= 0) {
      slot = base[e] + rl_rank(mask + e * words, words, j);
      p.row_token[slot] = t0 + j;
    }
    p.slot[at] = slot;
  }
}
// exclusive sums of cnt[0 .. E) into off[0 .. E], by one warp
__device__ __forceinline__ void rl_scan(const int *cnt, int *off, int E, int lane) {
  int total = 0;
  for (int e0 = 0; e0 < E; e0 += 32) {
    const int n = e0 + lane < E ? cnt[e0 + lane] : 0;
    int s = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += u;
    }
    if (e0 + lane < E) off[e0 + lane] = total + s - n;
    total += __shfl_sync(0xffffffffu, s, 31);
  }
  if (lane == 0) off[E] = total;
}

// One CTA per chunk of tokens: routes them and counts their experts; where the call is one chunk, places them as well.
template <typename T>
__global__ void __launch_bounds__(RL_WARPS * 32) k_route_logits(RouteLogitsParams p) {
  extern __shared__ __align__(16) unsigned char rl_smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  unsigned char *mine = rl_smem + warp * RL_CAND_BYTES;
  const RlCand c = {reinterpret_cast<uint64_t *>(mine), reinterpret_cast<double *>(mine + 256), reinterpret_cast<int *>(mine + 512)};
  unsigned char *after = rl_smem + RL_WARPS * RL_CAND_BYTES;
  double *row = reinterpret_cast<double *>(after) + (size_t)warp * (p.n_group > 1 ? p.E : 0);
  coli_grid_dependency_sync();
  const int t0 = blockIdx.x * p.chunk, tokens = min(p.chunk, p.T - t0), words = p.chunk / 32;
  for (int j = warp; j < tokens; j += RL_WARPS) {
    rl_route<T>(p, t0 + j, c, row, lane);
    __syncwarp();
  }
  __syncthreads();
  // (from here the shared memory holds the masks, counts and offsets)
  uint32_t *mask = reinterpret_cast<uint32_t *>(rl_smem);
  int *cnt = reinterpret_cast<int *>(mask + p.E * words), *off = cnt + p.E;
  rl_mark(mask, words, p.idx + (long)t0 * p.k, tokens * p.k, p.k, p.E);
  const bool only = gridDim.x == 1;
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) {
    int n = 0;
    for (int w = 0; w < words; ++w) n += __popc(mask[e * words + w]);
    if (only) {
      cnt[e] = n;
      p.expert_rows[e] = n;
    } else {
      p.chunk_rows[(size_t)blockIdx.x * p.E + e] = (uint8_t)n;
    }
  }
  if (!only) return;
  __syncthreads();
  if (warp == 0) rl_scan(cnt, off, p.E, lane);
  __syncthreads();
  rl_place(p, mask, off, t0, tokens);
  for (int i = off[p.E] + (int)threadIdx.x; i < p.T * p.k; i += blockDim.x) p.row_token[i] = -1;
}

// One CTA per chunk: rows of every expert before the chunk from all chunks' counts, then the places of its pairs.
__global__ void __launch_bounds__(512) k_route_place(RouteLogitsParams p, int chunks) {
  extern __shared__ __align__(16) unsigned char rl_smem[];
  const int words = p.chunk / 32;
  uint32_t *mask = reinterpret_cast<uint32_t *>(rl_smem);
  int *cnt = reinterpret_cast<int *>(mask + p.E * words), *off = cnt + p.E, *before = off + p.E + 1;
  coli_grid_dependency_sync();
  const int t0 = blockIdx.x * p.chunk, tokens = min(p.chunk, p.T - t0);
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) {
    int all = 0, b = 0;
#pragma unroll 16
    for (int ch = 0; ch < chunks; ++ch) {
      const int n = p.chunk_rows[(size_t)ch * p.E + e];
      all += n;
      b += ch < (int)blockIdx.x ? n : 0;
    }
    cnt[e] = all;
    before[e] = b;
    if (blockIdx.x == 0) p.expert_rows[e] = all;
  }
  rl_mark(mask, words, p.idx + (long)t0 * p.k, tokens * p.k, p.k, p.E);
  if (threadIdx.x < 32) rl_scan(cnt, off, p.E, threadIdx.x);
  __syncthreads();
  const int total = off[p.E];
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) before[e] += off[e];
  __syncthreads();
  rl_place(p, mask, before, t0, tokens);
  for (long i = (long)total + blockIdx.x * blockDim.x + threadIdx.x; i < (long)p.T * p.k; i += (long)gridDim.x * blockDim.x) p.row_token[i] = -1;
}

int launch_route_logits(RouteLogitsParams p, cudaStream_t st) {
  p.chunk = route_logits_chunk(p.T);
  const int chunks = (p.T + p.chunk - 1) / p.chunk, words = p.chunk / 32;
  const size_t tables = (size_t)p.E * words * 4 + (3 * (size_t)p.E + 1) * 4;
  size_t smem = RL_WARPS * (RL_CAND_BYTES + (p.n_group > 1 ? (size_t)p.E * 8 : 0));
  if (smem < tables) smem = tables;
  coli_count_launch(1);
  cudaError_t e;
  if (p.type == COLI_TYPE_F32)
    e = launch_dependent(k_route_logits<float>, dim3(chunks), dim3(RL_WARPS * 32), smem, st, p);
  else if (p.type == COLI_TYPE_F16)
    e = launch_dependent(k_route_logits<__half>, dim3(chunks), dim3(RL_WARPS * 32), smem, st, p);
  else
    e = launch_dependent(k_route_logits<__nv_bfloat16>, dim3(chunks), dim3(RL_WARPS * 32), smem, st, p);
  if (!coli_cuda_check(e, "routing launch")) return 0;
  if (chunks == 1) return 1;
  coli_count_launch(1);
  return coli_cuda_check(launch_dependent(k_route_place, dim3(chunks), dim3(512), tables, st, p, chunks), "placement launch") ? 1 : 0;
}

}  // namespace colib
