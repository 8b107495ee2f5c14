/*
 * flagattention_amd_linear.h -- C ABI of rotary positions and of linear attention with a decay per
 * head (libflagattention_amd.so, with the conventions of flagattention_amd.h).  No counterpart in the
 * reference, whose operators take q and k as they are and whose linear attention
 * (chunk_gated_delta_rule) has another recurrence.
 */
#ifndef FLAGATTENTION_AMD_LINEAR_H
#define FLAGATTENTION_AMD_LINEAR_H

#include "flagattention_amd.h"

#ifdef __cplusplus
extern "C" {
#endif

#define FA_ROTARY_MAX_AXES 4

/*
 * Rotary positions.  Pair i of a head -- dims i and i + pairs, or 2i and 2i + 1 with adjacent -- turns
 * by the angle positions[axis(i)][t] * inv_freq[i]; dims from 2 * pairs on stay as they are.  axis(i):
 * with one axis 0; without mixed the axes have runs of sections[0], sections[1], ... pairs; with
 * mixed axis(i) = i % axes where i / axes < sections[i % axes], else 0.  The sections sum to pairs.
 *
 * q and k (and v) are [tokens][heads][d], element strides, last dimension contiguous; k may be NULL
 * with h_kv 0.  Outputs may be the inputs themselves (the same pointer and strides), but may not
 * overlap them otherwise.  With key_cache, k and v go to row slots[t] % block_size of block
 * slots[t] / block_size of caches [num_blocks][h_kv][block_size][d], and k to k_out only where
 * that is not NULL (nor k itself); tokens whose slot is negative or past the cache are skipped there.  fp16 or bf16; any alignment (rows
 * and strides of 16 bytes with pairs and d multiples of 8 are taken 16 bytes at a time).
 */
typedef struct fa_rotary_args {
  const void* q;
  int64_t q_stride_t, q_stride_h;
  const void* k;
  int64_t k_stride_t, k_stride_h;
  void* q_out;
  int64_t q_out_stride_t, q_out_stride_h;
  void* k_out; /* with caches NULL, or where k goes too */
  int64_t k_out_stride_t, k_out_stride_h;
  const void* v; /* with caches */
  int64_t v_stride_t, v_stride_h;
  void* key_cache; /* or NULL */
  void* value_cache;
  int64_t kc_stride_0, kc_stride_h, kc_stride_t, vc_stride_0, vc_stride_h, vc_stride_t;
  int64_t num_blocks;
  const void* slots; /* int32 or int64 [tokens] */
  const void* positions; /* int32 or int64 [axes][tokens] */
  int64_t pos_stride_a;
  const float* inv_freq; /* [pairs] */
  int32_t tokens, h_q, h_kv, d, pairs, axes;
  int32_t sections[FA_ROTARY_MAX_AXES];
  int32_t block_size, mixed, adjacent, pos64, slots64;
  int32_t dtype; /* 0 fp16, 1 bf16 */
} fa_rotary_args;

/* sizeof(fa_rotary_args) as compiled into the library. */
int64_t fa_rotary_args_size(void);

int fa_rotary(const fa_rotary_args* args, void* stream);

/*
 * Linear attention with a decay per head: for a KV head with log decay a, per sequence
 *   S_t = e^a S_{t-1} + k_t v_t^T  (fp32 [d][d], rows are k's dims),  o_t = scale * q_t S_t,
 * o_t for each query head of the KV head's group.  fp16 or bf16; head dims 64, 128, 256; element
 * strides; last dimensions contiguous, rows of q, k and v 16-byte aligned, strides of tokens below 2^23.
 *
 * state [num_slots][h_kv] of contiguous [d][d], strides multiples of 4: sequence s starts from slot
 * state_indices[s] (s itself if NULL) where has_state[s] is not 0 (or has_state is NULL), else from
 * zeros, and leaves its last state there.  An index outside the slots: it starts from zeros and keeps
 * nothing.
 */
typedef struct fa_linear_args {
  const void* q; /* [total][h_q][d] */
  int64_t q_stride_t, q_stride_h;
  const void* k; /* [total][h_kv][d] */
  const void* v;
  int64_t k_stride_t, k_stride_h, v_stride_t, v_stride_h;
  const float* log_decay; /* [h_kv] */
  const int32_t* cu_seqlens; /* [num_seqs + 1], fa_linear_prompt only */
  float* state; /* or NULL, fa_linear_prompt only: no sequence starts from a state or keeps one */
  int64_t state_stride_s, state_stride_h;
  const int32_t* state_indices; /* [num_seqs] or NULL */
  const uint8_t* has_state;     /* [num_seqs] or NULL, fa_linear_prompt only */
  void* out; /* contiguous [total][h_q][d] */
  float* part; /* workspace of fa_linear_plan's size, 16-byte aligned, where segment > 0 */
  int32_t num_slots, num_seqs, total, h_q, h_kv, d;
  /* fa_linear_prompt: tokens that a sequence is cut into, a multiple of 32, or 0; whether what the
   * pieces start from is added up in a launch of its own; whether the longest go first (up to 64
   * sequences) */
  int32_t segment, joined, sorted;
  float scale;
  int32_t dtype; /* 0 fp16, 1 bf16 */
} fa_linear_args;

/* sizeof(fa_linear_args) as compiled into the library. */
int64_t fa_linear_args_size(void);

/*
 * Fills in segment, joined and sorted, from the totals, heads and head dim of args, for sequences of up to max_seqlen
 * tokens on a device of cu_count compute units.  Returns the floats that part has to hold (0: none),
 * or a negative code.
 */
int64_t fa_linear_plan(fa_linear_args* args, int32_t max_seqlen, int32_t cu_count);

/*
 * Packed sequences: rows cu_seqlens[s] .. cu_seqlens[s + 1] - 1 of q, k and v are sequence s's
 * tokens.  Starts are taken as clipped to [0, total] and lengths as at least 0.  Rows of no sequence
 * (behind the last one, or before the first) get out = 0; a sequence without tokens leaves its slot
 * as it is.
 */
int fa_linear_prompt(const fa_linear_args* args, void* stream);

/* One token per sequence: total = num_seqs.  A sequence whose index is outside the slots gets
 * out = 0. */
int fa_linear_token(const fa_linear_args* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif
