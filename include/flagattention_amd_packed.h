/*
 * flagattention_amd_packed.h -- C ABI of prompt attention over packed sequences and of the paged
 * K/V cache in 4 bits (libflagattention_amd.so, with the conventions of flagattention_amd.h).
 */
#ifndef FLAGATTENTION_AMD_PACKED_H
#define FLAGATTENTION_AMD_PACKED_H

#include "flagattention_amd.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------------------------
 * Prompt attention over packed sequences, and grouped-query decode over a paged cache held in
 * 4 bits.  No counterpart in the reference (its operators take rectangular batches and 16-bit
 * caches).
 * ---------------------------------------------------------------------- */

/*
 * Packed sequences: rows cu_seqlens_q[s] .. cu_seqlens_q[s + 1] - 1 of q belong to sequence s, its
 * keys are rows cu_seqlens_k[s] .. cu_seqlens_k[s + 1] - 1 of k and v.  Starts are taken as clipped
 * to [0, total] and lengths as at least 0, so no list makes a call read or write past its tensors.
 * Rows of q that belong to no sequence (behind the last one, or before the first) get out = 0,
 * lse = -inf, as rows without a visible key do.  fp16 or bf16; element strides; last dimensions
 * contiguous, rows 16-byte aligned.  Head dims 64, 128, 256.
 */
typedef struct fa_varlen_args {
  const void* q; /* [total_q][h_q][d] */
  int64_t q_stride_t, q_stride_h;
  const void* k; /* [total_k][h_kv][d] */
  const void* v;
  int64_t k_stride_t, k_stride_h, v_stride_t, v_stride_h;
  const int32_t* cu_seqlens_q; /* [num_seqs + 1] */
  const int32_t* cu_seqlens_k; /* [num_seqs + 1] */
  void* out; /* [total_q][h_q][d] */
  int64_t o_stride_t, o_stride_h;
  float* lse;      /* optional fp32 [h_q][total_q] (natural log) */
  float* o_part;   /* split workspace fp32 [h_q][total_q][num_splits][d] */
  float* lse_part; /* fp32 [h_q][total_q][num_splits] */
  int32_t num_seqs; /* at most 65535 */
  int32_t total_q, total_k, h_q, h_kv, d;
  /* split s covers keys [s * split_tokens, (s + 1) * split_tokens) of every sequence, the last
   * one the keys behind it too */
  int32_t num_splits, split_tokens;
  float scale;
  int32_t causal; /* bottom-right aligned in each sequence */
  int32_t dtype;  /* 0 fp16, 1 bf16 */
} fa_varlen_args;

/* sizeof(fa_varlen_args) as compiled into the library. */
int64_t fa_varlen_args_size(void);

/*
 * Fills in num_splits and split_tokens, from the totals, heads, head dim and causal of args, for
 * sequences of up to max_q tokens and max_k keys on a device of cu_count compute units.
 */
int fa_varlen_plan(fa_varlen_args* args, int32_t max_q, int32_t max_k, int32_t cu_count);

/*
 * Attention of every packed row: with num_splits == 1 writes out (and lse if given), otherwise
 * the per-split partials for fa_varlen_combine.
 */
int fa_varlen_attention(const fa_varlen_args* args, void* stream);

/* LSE-weighted merge of the split partials into out (and lse if given). */
int fa_varlen_combine(const fa_varlen_args* args, void* stream);

#define FA_MXFP4_GROUP 32 /* dims that share a scale */

/*
 * A paged K/V cache in 4 bits.  Codes: uint8 [num_blocks][h_kv][block_size][d / 2], dim 2i in the
 * low half of byte i and dim 2i + 1 in the high half, each a sign bit over an e2m1 magnitude (0,
 * 0.5, 1, 1.5, 2, 3, 4, 6).  Scales: uint8 [num_blocks][h_kv][block_size][d / 32], byte e for
 * 2^(e - 127), 255 for a group that is NaN as a whole.  K and V have the same strides, in bytes;
 * last dimensions are contiguous, rows of codes aligned to min(16, d / 8) bytes, rows of scales to
 * d / 128 bytes (at least 1).  Head dims 64, 128, 256; block_size a power of
 * two of at least 16.
 */
typedef struct fa_mxfp4_cache {
  void* k_codes;
  void* k_scales;
  void* v_codes;
  void* v_scales;
  int64_t code_stride_0, code_stride_h, code_stride_t;
  int64_t scale_stride_0, scale_stride_h, scale_stride_t;
  int64_t num_blocks;
  int32_t block_size, h_kv, d;
} fa_mxfp4_cache;

/* sizeof(fa_mxfp4_cache) as compiled into the library. */
int64_t fa_mxfp4_cache_size(void);

/*
 * Cache write: token i's rows key[i] and value[i] ([h_kv][d], fp16 or bf16) go to slot
 * slots[i] = block * block_size + row; slots < 0 or past the cache are skipped, and the slots of
 * one call must differ.  Each group of 32 dims gets the smallest scale with amax <= 7 * scale
 * (at least 2^-127), at which no code is off by more than half of the widest step, and codes of
 * x / scale rounded to nearest, ties to the even code.  A group with a NaN or an infinity is NaN as a whole.
 * Strides in elements; slots int64 (slots64 != 0) or int32.
 */
int fa_mxfp4_cache_write(const fa_mxfp4_cache* cache, const void* key, int64_t key_stride_t,
                         int64_t key_stride_h, const void* value, int64_t value_stride_t,
                         int64_t value_stride_h, const void* slots, int32_t slots64,
                         int32_t num_tokens, int32_t dtype, void* stream);

/*
 * Read back: row cu_seqlens[s] + j of k_out and v_out ([total][h_kv][d] contiguous, fp16 or bf16)
 * is token j of sequence s, row j % block_size of block block_table[s][j / block_size].  Rows that
 * belong to no sequence and rows of blocks outside the cache are zeros.  At most 65535 sequences.
 */
int fa_mxfp4_gather(const fa_mxfp4_cache* cache, const int32_t* block_table, int64_t bt_stride_b,
                    int32_t max_blocks_per_seq, const int32_t* cu_seqlens, int32_t num_seqs,
                    int32_t total, void* k_out, void* v_out, int32_t dtype, void* stream);

/* One query token per sequence over the 4-bit cache. */
typedef struct fa_mxfp4_decode_args {
  fa_mxfp4_cache cache;
  const void* q; /* [batch][h_q][d] */
  int64_t q_stride_b, q_stride_h;
  const int32_t* block_table; /* [batch][max_blocks_per_seq]; a block outside the cache reads as
                                 masked keys */
  int64_t bt_stride_b;
  int32_t max_blocks_per_seq;
  const int32_t* seqlens; /* [batch] */
  void* out; /* [batch][h_q][d] */
  int64_t o_stride_b, o_stride_h;
  float* o_part;   /* split workspace fp32 [batch][h_q][num_splits][d] */
  float* lse_part; /* fp32 [batch][h_q][num_splits] */
  int32_t batch, h_q;
  int32_t num_splits, split_tokens; /* as in fa_gqa_decode_args; split_tokens a multiple of 32
                                       where there are several */
  float scale;
  int32_t dtype; /* 0 fp16, 1 bf16 */
} fa_mxfp4_decode_args;

/* sizeof(fa_mxfp4_decode_args) as compiled into the library. */
int64_t fa_mxfp4_decode_args_size(void);

/*
 * Fills in num_splits and split_tokens for sequences of up to max_len keys on a device of
 * cu_count compute units.
 */
int fa_mxfp4_decode_plan(int32_t batch, int32_t h_q, int32_t h_kv, int32_t d, int32_t max_len,
                         int32_t cu_count, fa_mxfp4_decode_args* args);

/* Decode: writes out with num_splits == 1, else the partials for fa_mxfp4_combine. */
int fa_mxfp4_decode(const fa_mxfp4_decode_args* args, void* stream);

/* LSE-weighted merge of the split partials into out. */
int fa_mxfp4_combine(const fa_mxfp4_decode_args* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* FLAGATTENTION_AMD_PACKED_H */
