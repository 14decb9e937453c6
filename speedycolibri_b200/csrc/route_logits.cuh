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
// Tokens that one CTA routes: no more CTAs than SMs up to 128 tokens each.  Up to 512 tokens are one cluster, which places its pairs
// by itself; larger calls take a second launch.
constexpr int ROUTE_LOGITS_CLUSTER = 16;
static inline int route_logits_chunk(int T) { return T <= 32 * COLI_SMS ? 32 : T <= 64 * COLI_SMS ? 64 : 128; }
// bytes of counts that the chunks of a larger call leave for the placement
static inline size_t route_logits_workspace(int T, int E) {
  const int c = route_logits_chunk(T), chunks = (T + c - 1) / c;
  return chunks <= ROUTE_LOGITS_CLUSTER ? 0 : (size_t)chunks * ((E + 3) & ~3);
}
int launch_route_logits(RouteLogitsParams p, cudaStream_t st);

}  // namespace colib
