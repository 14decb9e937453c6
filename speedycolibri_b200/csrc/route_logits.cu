// Routing from given logits: scores, choice of experts, weights, and the rows the chosen pairs take in expert order.
// The rules are those of the block's own router (crates/colibri-engine/src/moe.rs:1047-1132; groups and the logit bias
// as in routing.cu), with two differences that a caller's own logits make necessary: the choice is made on scores in 64
// bits (by the logits themselves, where neither a bias nor groups ask for scores), so that experts whose scores 32 bits
// do not tell apart still come in the order of their logits, and an expert whose
// logit is -inf or NaN is not chosen at all (a closed expert, a padded token), where the block's router falls back to expert 0.
#include "route_logits.cuh"

namespace colib {

constexpr int RL_MAX_WARPS = 32;
// per warp: keys of the candidates, their ids
constexpr int RL_CAND_BYTES = 32 * (8 + 4);

// Ordinary loads, of the biases too: an earlier launch may write them while this one is already resident, so that they are no constants.
template <typename T>
__device__ __forceinline__ double rl_load(const T *p);
template <>
__device__ __forceinline__ double rl_load<float>(const float *p) { return (double)*p; }
template <>
__device__ __forceinline__ double rl_load<__half>(const __half *p) { return (double)__half2float(*p); }
template <>
__device__ __forceinline__ double rl_load<__nv_bfloat16>(const __nv_bfloat16 *p) { return (double)__bfloat162float(*p); }

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

// exp of a non-positive (softmax) or any (sigmoid) argument, relative error below 1e-15: n = rint(x log2 e), Taylor's polynomial
// of degree 13 in r = x - n ln 2 (two steps), |r| <= 0.347: remainder 4e-18 / (1 - r) relative; times 2^n.  As coli_expf
// (coli_math.h), whose result is rounded to f32.  Arguments are cut to +-708: beyond, a weight is below f32's least either way.
__device__ __forceinline__ double rl_exp(double x) {
  x = fmin(fmax(x, -708.0), 708.0);
  const double n = rint(x * 1.4426950408889634074);
  double r = fma(n, -6.93147180369123816490e-01, x);
  r = fma(n, -1.90821492927058770002e-10, r);
  double p = 1.0 / 6227020800.0;
  p = fma(p, r, 1.0 / 479001600.0);
  p = fma(p, r, 1.0 / 39916800.0);
  p = fma(p, r, 1.0 / 3628800.0);
  p = fma(p, r, 1.0 / 362880.0);
  p = fma(p, r, 1.0 / 40320.0);
  p = fma(p, r, 1.0 / 5040.0);
  p = fma(p, r, 1.0 / 720.0);
  p = fma(p, r, 1.0 / 120.0);
  p = fma(p, r, 1.0 / 24.0);
  p = fma(p, r, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  return p * __hiloint2double((1023 + (int)n) << 20, 0);
}

// the same of an f32 value
__device__ __forceinline__ uint32_t rl_key32(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  return (b >> 31) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float rl_value32(uint32_t key) { return __uint_as_float((key >> 31) ? key & 0x7fffffffu : ~key); }

template <typename Key>
struct RlCand {
  Key *key;
  int *id;
};
__device__ __forceinline__ uint32_t rl_upper(uint32_t k) { return k; }
__device__ __forceinline__ uint32_t rl_upper(uint64_t k) { return (uint32_t)(k >> 32); }

// The k best keys of a warp (slot s of a lane holds expert lane + 32 s; largest key, then lowest expert; 0 is none) into places
// 0 .. of `c`, in order.  Returns how many there are, at most k.  The k-th largest of the lanes' best keys bounds the k-th largest of
// all from below (taken by its upper word alone): a little over k candidates as a rule, and each finds its place by
// counting.  More than 32 of them (many equal logits) take k rounds.
template <int SLOTS, typename Key>
__device__ __forceinline__ int rl_select(Key (&key)[SLOTS], int k, const RlCand<Key> &c, int lane) {
  Key best = 0;
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) best = key[s] > best ? key[s] : best;
  const uint32_t bhi = rl_upper(best);
  uint32_t *hi = reinterpret_cast<uint32_t *>(c.key);
  __syncwarp();
  hi[lane] = bhi;
  __syncwarp();
  int above = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint4 q = reinterpret_cast<const uint4 *>(hi)[j];
    above += (q.x > bhi) + (q.y > bhi) + (q.z > bhi) + (q.w > bhi);
  }
  const uint32_t bound = max(1u, __reduce_min_sync(0xffffffffu, above < k ? bhi : 0xffffffffu));
  uint32_t mine = 0u;  // this lane's slots at or above the bound
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) mine |= (uint32_t)(rl_upper(key[s]) >= bound) << s;
  const int n = (int)__reduce_add_sync(0xffffffffu, (unsigned)__popc(mine));
  if (n <= 32) {
    // places in any order, then everyone counts who comes before it
    int at = __popc(mine);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, at, o);
      if (lane >= o) at += u;
    }
    at -= __popc(mine);
#pragma unroll
    for (int s = 0; s < SLOTS; ++s)
      if ((mine >> s) & 1u) {
        c.key[at] = key[s];
        c.id[at] = s * 32 + lane;
        ++at;
      }
    __syncwarp();
    const Key mk = lane < n ? c.key[lane] : 0;
    const int mi = lane < n ? c.id[lane] : 0;
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) {
      const Key other = c.key[j];
      rank += other > mk || (other == mk && c.id[j] < mi);
    }
    __syncwarp();
    if (lane < n && rank < k) {
      c.key[rank] = mk;
      c.id[rank] = mi;
    }
    __syncwarp();
    return min(n, k);
  }
  int found = 0;
  for (; found < k; ++found) {
    Key bk = 0;
    int bid = 0x7fffffff;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s)
      if (key[s] > bk) {
        bk = key[s];
        bid = s * 32 + lane;
      }
    const uint32_t top = __reduce_max_sync(0xffffffffu, rl_upper(bk));
    if (top == 0u) break;
    const uint32_t low = __reduce_max_sync(0xffffffffu, rl_upper(bk) == top ? (uint32_t)bk : 0u);
    const bool holds = rl_upper(bk) == top && (uint32_t)bk == low;
    const int win = (int)__reduce_min_sync(0xffffffffu, holds ? (uint32_t)bid : 0x7fffffffu);
    if (holds && bid == win) {
      c.key[found] = bk;
      c.id[found] = win;
#pragma unroll
      for (int s = 0; s < SLOTS; ++s)
        if (s * 32 + lane == win) key[s] = 0;
    }
  }
  __syncwarp();
  return found;
}

// Experts outside the topk_group best groups lose their keys.  A group's mark is the sum of its two best choices (the one, where only
// one is open); `per` lanes share a group.  Returns how far the last mark kept lies above the first one left out.
template <int SLOTS, typename Key, typename Real>
__device__ __forceinline__ Real rl_groups(const RouteLogitsParams &p, Key (&key)[SLOTS], const Real (&choice)[SLOTS], Real none, Real *row, Real *marks,
                                          int lane) {
  const int G = p.n_group, gs = p.E / G;
#pragma unroll
  for (int s = 0; s < SLOTS; ++s)
    if (lane + 32 * s < p.E) row[lane + 32 * s] = key[s] ? choice[s] : none;
  __syncwarp();
  int per = 1;
  while (2 * per * G <= 32) per *= 2;
  const int g = lane / per;
  Real m1 = none, m2 = none;
  if (g < G)
#pragma unroll 4
    for (int i = lane % per; i < gs; i += per) {
      const Real v = row[g * gs + i];
      m2 = v > m1 ? m1 : (v > m2 ? v : m2);
      m1 = v > m1 ? v : m1;
    }
  for (int o = 1; o < per; o <<= 1) {
    const Real o1 = __shfl_xor_sync(0xffffffffu, m1, o), o2 = __shfl_xor_sync(0xffffffffu, m2, o);
    const Real lo = m1 < o1 ? m1 : o1, hi = m2 > o2 ? m2 : o2;
    m2 = lo > hi ? lo : hi;
    m1 = m1 > o1 ? m1 : o1;
  }
  const bool some = g < G && m1 > none;
  const Real mark = some ? (m2 > none ? m1 + m2 : m1) : none;
  if (lane % per == 0 && g < G) marks[g] = mark;
  __syncwarp();
  int above = 0;
  for (int j = 0; j < G; ++j) above += marks[j] > mark || (marks[j] == mark && j < g);
  const bool keep = some && above < p.topk_group;
  const uint32_t kept = __ballot_sync(0xffffffffu, keep);
  Real last = keep ? mark : -none, first = some && !keep ? mark : none;
  for (int o = 1; o < 32; o <<= 1) {
    const Real a = __shfl_xor_sync(0xffffffffu, last, o), b = __shfl_xor_sync(0xffffffffu, first, o);
    last = a < last ? a : last;
    first = b > first ? b : first;
  }
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) {
    const int e = lane + 32 * s;
    if (e < p.E && !((kept >> ((e / gs) * per)) & 1u)) key[s] = 0;
  }
  __syncwarp();
  return last - first;
}

// What the weights need besides a chosen expert's own logit.
struct RlNorm {
  double top, sum;  // softmax: the largest z, and the sum of exp(z - top); 0: not needed
  int n;            // experts chosen, -1: undecided
};
template <typename T>
__device__ __forceinline__ double rl_z(const RouteLogitsParams &p, const T *z0, int e) {
  const double z = rl_load<T>(z0 + e);
  return p.logit_bias ? z + (double)p.logit_bias[e] : z;
}
// (a largest logit of infinity shares the mass with its equals)
__device__ __forceinline__ double rl_over(double z, double top) { return z == top ? 1.0 : rl_exp(z - top); }

// The choice in 64 bits throughout: where 32 do not decide it.
template <typename T, int SLOTS>
__device__ __noinline__ RlNorm rl_choose64(const RouteLogitsParams &p, const T *z0, unsigned char *cand, double *row, int lane) {
  RlNorm norm;
  const double NEG_INF = __longlong_as_double(0xfff0000000000000ll);
  const RlCand<uint64_t> c = {reinterpret_cast<uint64_t *>(cand), reinterpret_cast<int *>(cand + 256)};
  double score[SLOTS];
  uint64_t key[SLOTS];
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) {
    const int e = lane + 32 * s;
    const double z = e < p.E ? rl_z<T>(p, z0, e) : NEG_INF;
    key[s] = z > NEG_INF;
    score[s] = key[s] ? z : NEG_INF;
  }
  norm.top = norm.sum = 0.0;
  if (p.score == COLI_SCORE_SOFTMAX) {
    double m = NEG_INF;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) m = fmax(m, score[s]);
    m = rl_warp_max(m);
    double sum = 0.0;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
      score[s] = key[s] ? rl_over(score[s], m) : 0.0;
      sum += score[s];
    }
    norm.top = m;
    norm.sum = sum = rl_warp_sum(sum);
    const double inv = sum > 0.0 ? 1.0 / sum : 0.0;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) score[s] *= inv;
  } else {
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) score[s] = 1.0 / (1.0 + rl_exp(-score[s]));
  }
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) {
    const int e = lane + 32 * s;
    if (p.select_bias && e < p.E) score[s] += (double)p.select_bias[e];
    key[s] = key[s] && score[s] > NEG_INF ? rl_key(score[s]) : 0;
  }
  if (p.n_group > 1) rl_groups<SLOTS, uint64_t, double>(p, key, score, NEG_INF, row, reinterpret_cast<double *>(cand), lane);
  norm.n = rl_select<SLOTS, uint64_t>(key, p.k, c, lane);
  return norm;
}

// The choice in 32 bits: by the logits themselves where neither a bias nor groups ask for scores, and else by f32 scores, as long as no
// two that it hangs on lie within their errors (-1: they do).  An f32 score is off by at most 2^-19 of itself (__expf: 2^-21 and
// 2^-23 of its argument, whose share of the score is below 2^-20) and by what the rounding of z takes from it, 2^-23 |z|
// with a logit bias; a choice by another 2^-23 of itself.
template <typename T, int SLOTS>
__device__ __forceinline__ int rl_choose32(const RouteLogitsParams &p, const T *z0, unsigned char *cand, float *row, int lane, RlNorm &norm) {
  const float NEG_INF = __uint_as_float(0xff800000u);
  const RlCand<uint32_t> c = {reinterpret_cast<uint32_t *>(cand), reinterpret_cast<int *>(cand + 256)};
  const bool softmax = p.score == COLI_SCORE_SOFTMAX;
  const bool scored = p.select_bias || p.logit_bias || p.n_group > 1;
  if (softmax && p.logit_bias) return -1;  // (top and sum are wanted to 64 bits)
  float z[SLOTS];
  uint32_t key[SLOTS];
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) z[s] = lane + 32 * s < p.E ? (float)rl_load<T>(z0 + lane + 32 * s) : NEG_INF;
  if (p.logit_bias) {
    // two finite values may leave f32: an expert that is open all the same
    bool leaves = false;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s)
      if (lane + 32 * s < p.E) {
        const float b = p.logit_bias[lane + 32 * s], sum = z[s] + b;
        leaves |= isinf(sum) && isfinite(z[s]) && isfinite(b);
        z[s] = sum;
      }
    if (__any_sync(0xffffffffu, leaves)) return -1;
  }
  uint32_t top = 0u;
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) {
    key[s] = z[s] > NEG_INF ? rl_key32(z[s]) : 0u;
    top = max(top, key[s]);
  }
  top = __reduce_max_sync(0xffffffffu, top);
  norm.top = norm.sum = 0.0;
  if (top == 0u) return 0;  // every expert is closed
  const float m = rl_value32(top);
  if (softmax) {
    norm.top = (double)m;
    // (where the weights are divided by their own sum, and that holds the largest, the sum over all experts drops out)
    if (!p.norm_topk || scored) {
      double sum = 0.0;
#pragma unroll
      for (int s = 0; s < SLOTS; ++s) sum += key[s] ? rl_over((double)z[s], norm.top) : 0.0;
      norm.sum = rl_warp_sum(sum);
    }
  }
  float apart = 0.0f;  // how far two choices must lie apart
  if (scored) {
    const float inv = softmax ? (float)(1.0 / norm.sum) : 0.0f;
    float choice[SLOTS], size = 0.0f, arg = 0.0f;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
      const int e = lane + 32 * s;
      choice[s] = softmax ? (z[s] == m ? 1.0f : __expf(z[s] - m)) * inv : __fdividef(1.0f, 1.0f + __expf(fminf(-z[s], 80.0f)));
      if (p.select_bias && e < p.E) choice[s] += p.select_bias[e];
      if (key[s]) key[s] = choice[s] > NEG_INF ? rl_key32(choice[s]) : 0u;
      if (key[s]) {
        size = fmaxf(size, fabsf(choice[s]));
        arg = fmaxf(arg, fminf(fabsf(z[s]), 128.0f));
      }
    }
    size = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(size)));
    arg = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(arg)));
    if (!(size <= 1.0e38f)) return -1;  // (the sum of two may leave f32)
    apart = 2.0f * (1.9e-6f + 2.4e-7f * size + (p.logit_bias ? 1.2e-7f * arg : 0.0f));
    if (p.n_group > 1) {
      const float gap = rl_groups<SLOTS, uint32_t, float>(p, key, choice, NEG_INF, row, reinterpret_cast<float *>(cand), lane);
      if (!(gap > 2.0f * apart)) return -1;
    }
  }
  const int n = rl_select<SLOTS, uint32_t>(key, min(scored ? p.k + 1 : p.k, 32), c, lane);
  if (scored) {
    if (n == 32 && p.k == 32) return -1;  // (the 33rd is not known)
    const bool near = lane + 1 < n && !(rl_value32(c.key[lane]) - rl_value32(c.key[lane + 1]) > apart);
    if (__any_sync(0xffffffffu, near)) return -1;
  }
  return min(n, p.k);
}

// One warp routes one token; `row` is E doubles of shared memory of its own (groups only).  The experts also go to ids_out.
template <typename T, int SLOTS>
__device__ __forceinline__ void rl_token(const RouteLogitsParams &p, int t, unsigned char *cand, double *row, int lane, int *ids_out) {
  const T *z0 = (const T *)p.logits + (long)t * p.stride;
  RlNorm norm;
  norm.n = rl_choose32<T, SLOTS>(p, z0, cand, reinterpret_cast<float *>(row), lane, norm);
  if (norm.n < 0) norm = rl_choose64<T, SLOTS>(p, z0, cand, row, lane);
  const int n = norm.n;
  const int *ids = reinterpret_cast<const int *>(cand + 256);
  double w = 0.0;
  if (lane < n) {
    const double z = rl_z<T>(p, z0, ids[lane]);
    if (p.score != COLI_SCORE_SOFTMAX)
      w = 1.0 / (1.0 + rl_exp(-z));
    else
      w = norm.sum > 0.0 ? rl_over(z, norm.top) / norm.sum : rl_over(z, norm.top);
  }
  if (p.norm_topk) w /= rl_warp_sum(w) + 1e-20;
  if (lane < p.k) {
    const int id = lane < n ? ids[lane] : -1;
    ids_out[lane] = id;
    p.idx[(long)t * p.k + lane] = id;
    p.w[(long)t * p.k + lane] = (float)(w * (double)p.routed_scale);
  }
}

template <typename T>
__device__ __forceinline__ void rl_route(const RouteLogitsParams &p, int t, unsigned char *cand, double *row, int lane, int *ids_out) {
  if (p.E <= 128)
    rl_token<T, 4>(p, t, cand, row, lane, ids_out);
  else if (p.E <= 256)
    rl_token<T, 8>(p, t, cand, row, lane, ids_out);
  else if (p.E <= 384)
    rl_token<T, 12>(p, t, cand, row, lane, ids_out);
  else
    rl_token<T, 16>(p, t, cand, row, lane, ids_out);
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
// exclusive sums of cnt[0 .. E) into off[0 .. E], by one warp: a run of experts each
__device__ __forceinline__ void rl_scan(const int *cnt, int *off, int E, int lane) {
  const int per = (E + 31) / 32, e0 = lane * per;
  int n = 0;
  for (int i = 0; i < per; ++i) n += e0 + i < E ? cnt[e0 + i] : 0;
  int s = n;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += u;
  }
  if (lane == 31) off[E] = s;
  s -= n;
  for (int i = 0; i < per && e0 + i < E; ++i) {
    off[e0 + i] = s;
    s += cnt[e0 + i];
  }
}

// The pairs of a chunk take their rows: off = rows of all experts below, before = rows of the expert in earlier chunks.
// cnt and before are summed, off has room for E + 1.
__device__ __forceinline__ void rl_place(const RouteLogitsParams &p, const uint32_t *mask, int words, const int32_t *ids, const int *cnt, int *before,
                                         int *off, int t0, int pairs) {
  if (threadIdx.x < 32) rl_scan(cnt, off, p.E, threadIdx.x);
  __syncthreads();
  const int total = off[p.E];
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) {
    before[e] += off[e];
    if (blockIdx.x == 0) p.expert_rows[e] = cnt[e];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < pairs; i += blockDim.x) {
    const int e = ids[i], j = i / p.k;
    int slot = -1;
    if (e >= 0) {
      slot = before[e] + rl_rank(mask + e * words, words, j);
      p.row_token[slot] = t0 + j;
    }
    p.slot[(long)t0 * p.k + i] = slot;
  }
  for (long i = (long)total + blockIdx.x * blockDim.x + threadIdx.x; i < (long)p.T * p.k; i += (long)gridDim.x * blockDim.x) p.row_token[i] = -1;
}
__device__ __forceinline__ void rl_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ int rl_cluster_load(const int *at, uint32_t rank) {
  uint32_t a;
  int v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(at)), "r"(rank));
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}

// One CTA per chunk of tokens: routes them and counts their experts.  Where the call is one chunk it places them as well, and where it
// is a few (CLUSTER: the chunks are one cluster, which reads one another's counts) they do together; else k_route_place does.
template <typename T, bool CLUSTER>
__global__ void __launch_bounds__(RL_MAX_WARPS * 32) k_route_logits(const __grid_constant__ RouteLogitsParams p) {
  extern __shared__ __align__(16) unsigned char rl_smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int t0 = blockIdx.x * p.chunk, tokens = max(0, min(p.chunk, p.T - t0)), pairs = tokens * p.k, words = (p.chunk + 31) / 32;
  int *ids = reinterpret_cast<int *>(rl_smem);  // the chunk's choices, then per-warp memory, later the tables
  unsigned char *after = rl_smem + (((size_t)p.chunk * p.k * 4 + 15) & ~(size_t)15);
  unsigned char *cand = after + warp * RL_CAND_BYTES;
  double *row = reinterpret_cast<double *>(after + warps * RL_CAND_BYTES) + (size_t)warp * (p.n_group > 1 ? p.E : 0);
  coli_grid_dependency_sync();
  for (int j = warp; j < tokens; j += warps) {
    rl_route<T>(p, t0 + j, cand, row, lane, ids + j * p.k);
    __syncwarp();
  }
  __syncthreads();
  if constexpr (CLUSTER) {
    const int pitch = (p.E + 3) & ~3;
    uint32_t *mask = reinterpret_cast<uint32_t *>(after);
    int *mine = reinterpret_cast<int *>(mask + p.E * words), *cnt = mine + pitch, *before = cnt + pitch, *off = before + pitch;
    rl_mark(mask, words, ids, pairs, p.k, p.E);
    for (int e = threadIdx.x; e < p.E; e += blockDim.x) {
      int n = 0;
      for (int w = 0; w < words; ++w) n += __popc(mask[e * words + w]);
      mine[e] = n;
    }
    rl_cluster_sync();
    for (int e = threadIdx.x; e < p.E; e += blockDim.x) {
      int all = 0, b = 0;
      for (uint32_t r = 0; r < gridDim.x; ++r) {
        const int n = rl_cluster_load(mine + e, r);
        all += n;
        b += r < blockIdx.x ? n : 0;
      }
      cnt[e] = all;
      before[e] = b;
    }
    __syncthreads();
    rl_place(p, mask, words, ids, cnt, before, off, t0, pairs);
    rl_cluster_sync();  // (the others have read this CTA's counts)
    return;
  }
  if (gridDim.x > 1) {
    uint32_t *mask = reinterpret_cast<uint32_t *>(after);
    rl_mark(mask, words, ids, pairs, p.k, p.E);
    const int pitch = (p.E + 3) & ~3;
    for (int e = threadIdx.x; e < pitch; e += blockDim.x) {
      int n = 0;
      for (int w = 0; w < words; ++w) n += e < p.E ? __popc(mask[e * words + w]) : 0;
      p.chunk_rows[(size_t)blockIdx.x * pitch + e] = (uint8_t)n;
    }
    return;
  }
  // The only chunk: every pair counts the pairs before it in expert order (a table of the experts would cost a scan over all).
  int *cnt = reinterpret_cast<int *>(after);
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) cnt[e] = 0;
  const int padded = (pairs + 3) & ~3;
  for (int i = pairs + threadIdx.x; i < padded; i += blockDim.x) ids[i] = -1;
  __syncthreads();
  int total = 0;
  for (int i0 = 0; i0 < pairs; i0 += blockDim.x) {
    const int i = i0 + (int)threadIdx.x, id = i < pairs ? ids[i] : -1;
    if (id >= 0) {
      int rank = 0;
      for (int j = 0; j < padded; j += 4) {
        const int4 o = *reinterpret_cast<const int4 *>(ids + j);
        rank += ((unsigned)o.x < (unsigned)id || (o.x == id && j < i)) + ((unsigned)o.y < (unsigned)id || (o.y == id && j + 1 < i)) +
                ((unsigned)o.z < (unsigned)id || (o.z == id && j + 2 < i)) + ((unsigned)o.w < (unsigned)id || (o.w == id && j + 3 < i));
      }
      atomicAdd(cnt + id, 1);
      p.slot[i] = rank;
      p.row_token[rank] = i / p.k;
    } else if (i < pairs) {
      p.slot[i] = -1;
    }
    total += __syncthreads_count(id >= 0);
  }
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) p.expert_rows[e] = cnt[e];
  for (int i = total + (int)threadIdx.x; i < pairs; i += blockDim.x) p.row_token[i] = -1;
}

// One CTA per chunk: rows of every expert before the chunk from all chunks' counts, then the places of its pairs.  Its CTAs wait for
// one another's memory most of the time: as large as they may be (16384 tokens, 384 experts, both kernels: 36.8 us with 512
// threads, 30.4 with 1024), and where they are no more than the SMs one on each, by the shared memory that they ask for: launched
// early, they would pack onto the SMs that their predecessor leaves first (27.5 us; 20000 tokens in 295 chunks 32.9, without 30.8).
constexpr int RL_PLACE_THREADS = 1024;
constexpr int RL_PLACE_ALONE = 116 * 1024;  // more than half of an SM's
__global__ void __launch_bounds__(RL_PLACE_THREADS) k_route_place(const __grid_constant__ RouteLogitsParams p, int chunks) {
  extern __shared__ __align__(16) unsigned char rl_smem[];
  const int words = (p.chunk + 31) / 32, pitch = (p.E + 3) & ~3;
  uint32_t *mask = reinterpret_cast<uint32_t *>(rl_smem);
  int *cnt = reinterpret_cast<int *>(mask + p.E * words), *before = cnt + pitch, *off = before + pitch;
  for (int e = threadIdx.x; e < 2 * pitch; e += blockDim.x) cnt[e] = 0;
  __syncthreads();
  coli_grid_dependency_sync();
  const int t0 = blockIdx.x * p.chunk, tokens = min(p.chunk, p.T - t0);
  {
    // four experts a thread, the chunks shared among as many groups of threads as there are
    const int quads = pitch / 4, groups = RL_PLACE_THREADS / quads, g = (int)threadIdx.x / quads, q = (int)threadIdx.x % quads;
    if (g < groups) {
      int all[4] = {}, b[4] = {};
#pragma unroll 8
      for (int ch = g; ch < chunks; ch += groups) {
        const uint32_t n = __ldcg(reinterpret_cast<const uint32_t *>(p.chunk_rows + (size_t)ch * pitch) + q);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int v = (int)((n >> (8 * i)) & 255u);
          all[i] += v;
          b[i] += ch < (int)blockIdx.x ? v : 0;
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        atomicAdd(cnt + 4 * q + i, all[i]);
        atomicAdd(before + 4 * q + i, b[i]);
      }
    }
  }
  const int32_t *idx = p.idx + (long)t0 * p.k;
  rl_mark(mask, words, idx, tokens * p.k, p.k, p.E);
  rl_place(p, mask, words, idx, cnt, before, off, t0, tokens * p.k);
}

template <typename T, bool CLUSTER>
static int launch_route_typed(const RouteLogitsParams &p, int ctas, int warps, size_t smem, cudaStream_t st) {
  static ColiPerDeviceOnce attr_once;
  if (!coli_set_smem_limit(attr_once, k_route_logits<T, CLUSTER>, 128 * 32 * 4 + RL_MAX_WARPS * (RL_CAND_BYTES + 512 * 8), "routing shared-memory attribute"))
    return 0;
  if (CLUSTER) {  // 16 CTAs are more than every GPU promises, and fit this one
    static ColiPerDeviceOnce cluster_once;
    bool done = false;
    const int dev = cluster_once.current(&done);
    if (!done) {
      if (!coli_cuda_check(cudaFuncSetAttribute(k_route_logits<T, CLUSTER>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1), "routing cluster attribute")) return 0;
      cluster_once.mark(dev);
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3((unsigned)warps * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)ctas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CLUSTER ? 2 : 1;
  coli_count_launch(1);
  return coli_cuda_check(cudaLaunchKernelEx(&cfg, k_route_logits<T, CLUSTER>, p), "routing launch") ? 1 : 0;
}
template <bool CLUSTER>
static int launch_route_kernel(const RouteLogitsParams &p, int ctas, int warps, size_t smem, cudaStream_t st) {
  if (p.type == COLI_TYPE_F32) return launch_route_typed<float, CLUSTER>(p, ctas, warps, smem, st);
  if (p.type == COLI_TYPE_F16) return launch_route_typed<__half, CLUSTER>(p, ctas, warps, smem, st);
  return launch_route_typed<__nv_bfloat16, CLUSTER>(p, ctas, warps, smem, st);
}

int launch_route_logits(RouteLogitsParams p, cudaStream_t st) {
  p.chunk = route_logits_chunk(p.T);
  const int chunks = (p.T + p.chunk - 1) / p.chunk, words = (p.chunk + 31) / 32;
  // a warp per token up to 32; a few more for the tables where there are few tokens
  const int tokens = p.T < p.chunk ? p.T : p.chunk, warps = tokens < 4 ? 4 : tokens < RL_MAX_WARPS ? tokens : RL_MAX_WARPS;
  const size_t pitch = (p.E + 3) & ~3, own = (size_t)warps * (RL_CAND_BYTES + (p.n_group > 1 ? (size_t)p.E * 8 : 0));
  const size_t marks = (size_t)p.E * words * 4, tables = marks + (3 * pitch + p.E + 1) * 4;
  const size_t smem = (((size_t)p.chunk * p.k * 4 + 15) & ~(size_t)15) + (own > tables ? own : tables);
  if (chunks == 1) return launch_route_kernel<false>(p, 1, warps, smem, st);
  if (chunks <= ROUTE_LOGITS_CLUSTER) return launch_route_kernel<true>(p, chunks <= 2 ? 2 : chunks <= 4 ? 4 : chunks <= 8 ? 8 : 16, warps, smem, st);
  if (!launch_route_kernel<false>(p, chunks, warps, smem, st)) return 0;
  static ColiPerDeviceOnce place_once;
  if (!coli_set_smem_limit(place_once, k_route_place, RL_PLACE_ALONE, "placement shared-memory attribute")) return 0;
  const size_t place = chunks <= COLI_SMS ? (size_t)RL_PLACE_ALONE : tables;  // (tables: 17 KB at most)
  coli_count_launch(1);
  return coli_cuda_check(launch_dependent(k_route_place, dim3(chunks), dim3(RL_PLACE_THREADS), place, st, p, chunks), "placement launch") ? 1 : 0;
}

}  // namespace colib
