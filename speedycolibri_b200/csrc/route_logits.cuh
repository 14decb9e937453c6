// Parameters of routing from given logits (route_logits.cu).
#pragma once
#include "internal.cuh"

namespace colib {

struct RouteLogitsParams {
  const void *logits;  // [T, E] of `type`, rows `stride` elements apart
  int type;            // COLI_TYPE_*
  long stride;
  int T, E, k;
  int score, norm_topk;
  float routed_scale;
  int n_group, topk_group;
  const float *select_bias, *logit_bias;  // [E] or null
  int32_t *idx;                           // [T, k]
  float *w;                               // [T, k]
  int32_t *expert_rows;                   // [E]
  int32_t *slot;                          // [T, k]
  int32_t *row_token;                     // [T * k]
  uint8_t *chunk_rows;                    // workspace: rows of each expert in each chunk of tokens (null for one chunk)
  int chunk;                              // filled in by the launcher
};
// Tokens that one CTA routes: 32 or 64 while that is no more CTAs than SMs, else an even share of whole rounds of at most 128 each
// (us a call, with 128 / a share: 16384 tokens, 384 experts 37.1 / 36.6; 20000 tokens, 128 experts 39.0 / 35.3; 5000 tokens in
// chunks of 64 / 34: 13.2 / 14.6).  Up to 512 tokens are one cluster, which places its pairs
// by itself; larger calls take a second launch.
constexpr int ROUTE_LOGITS_CLUSTER = 16;
static inline int route_logits_chunk(int T) {
  if (T <= 64 * COLI_SMS) return T <= 32 * COLI_SMS ? 32 : 64;
  const int ctas = (T + 128 * COLI_SMS - 1) / (128 * COLI_SMS) * COLI_SMS;
  return (T + ctas - 1) / ctas;
}
// bytes of counts that the chunks of a larger call leave for the placement
static inline size_t route_logits_workspace(int T, int E) {
  const int c = route_logits_chunk(T), chunks = (T + c - 1) / c;
  return chunks <= ROUTE_LOGITS_CLUSTER ? 0 : (size_t)chunks * ((E + 3) & ~3);
}
int launch_route_logits(RouteLogitsParams p, cudaStream_t st);

}  // namespace colib
