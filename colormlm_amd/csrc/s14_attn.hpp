// The attention operators between the FP8 projections and the expert layer:
// the residual norm before either, per-head norms with the position rotation,
// the paged key/value caches of 8 and of 4 bits, attention over them, and causal
// attention over packed prompts.  Shared
// between the kernel files (s14_attn_*.hip) and s14_attn_api.cpp.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "s14_attn_plan.h"
#include "s14_hip.h"

namespace s14 {

// Rows of one projection: value (token t, head h, d) at t * token + h * head
// + d, in elements.
struct AttnRows {
  const void *p;
  int bf16;
  uint32_t heads;
  uint64_t token;
  uint32_t head;
};
struct AttnOut {
  void *p;
  int bf16;
  uint64_t token;
  uint32_t head;
};

struct RopeArgs {
  const float *table;  // [positions][rot]: cos of rot / 2 angles, then their sines; NULL: no rotation
  uint32_t positions, rot, start;
  int interleaved;
};

struct NormRopeArgs {
  uint32_t tokens, dim;
  AttnRows in[2];   // queries, keys (heads 0: absent)
  AttnOut out[2];
  const float *weight[2];  // [dim] or NULL: no norm
  float eps;
  RopeArgs rope;
  const int32_t *positions;  // [tokens], read where rope.table is set
  uint32_t *status;
};

struct CacheArgs {     // of 8 bits, and of 4 (s14_hip.h has the layouts)
  uint8_t *k, *v;      // K codes [page][head][slot][dim], V codes [page][head][dim][slot]
  uint8_t *ks, *vs;    // E8M0 [page][head]
  uint32_t pages, heads, page, dim;  // page: tokens a page, a power of two
};

struct AppendArgs {
  CacheArgs cache;
  uint32_t tokens, seqs, max_new, table_width;
  AttnRows in[2];  // keys, values
  const float *k_weight;
  float eps;
  RopeArgs rope;
  const int32_t *page_table, *cu, *past;
  uint32_t *status;
};

struct PagedArgs {
  CacheArgs cache;
  uint32_t tokens, seqs, heads, max_new, max_len, table_width;
  const uint16_t *q;
  uint64_t q_token;
  uint32_t q_head;
  const int32_t *page_table, *cu, *len;
  AttnOut out;
  float *lse;  // [tokens][heads] or NULL
  float scale;
  uint32_t window;
  uint32_t *status, *count;  // count: kPagedCounters
};

struct PromptArgs {
  uint32_t tokens, seqs, heads, kv_heads, dim;
  const uint16_t *q, *k, *v;
  uint64_t q_token, k_token, v_token;
  uint32_t q_head, k_head, v_head;
  const int32_t *cu;
  AttnOut out;
  float *lse;
  float scale;
  uint32_t window;
};

// Rows of k values; x.heads is 1 throughout.  A NULL p: absent.
struct AddNormArgs {
  uint32_t rows, k;
  AttnRows x, residual;
  AttnOut residual_out, y;
  const float *weight;
  float eps;
  uint32_t group;  // of the codes' scales, 0: no codes
  uint8_t *q, *scales;
};

struct RopeTableArgs {
  uint32_t positions, rot;
  double theta, factor, original, fast, slow, amplitude;
  float *out;
};

hipError_t launch_add_norm(hipStream_t s, const AddNormArgs &a);
hipError_t launch_rope_table(hipStream_t s, const RopeTableArgs &a);
hipError_t launch_norm_rope(hipStream_t s, const NormRopeArgs &a);
hipError_t launch_kv_append(hipStream_t s, const AppendArgs &a);
hipError_t launch_kv4_append(hipStream_t s, const AppendArgs &a);
hipError_t launch_paged_attention(hipStream_t s, const PagedArgs &a, const PagedPlan &p, float *part);
hipError_t launch_paged4_attention(hipStream_t s, const PagedArgs &a, const PagedPlan &p, float *part);
hipError_t launch_prompt_attention(hipStream_t s, const PromptArgs &a);

}  // namespace s14
