/*
 * sp_hip_fp4.h -- the 4-bit block cache, and eviction by attention weight.
 *
 * Keys and values as OCP E2M1 numbers (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) with one
 * power of two as the scale of each 32 channels of a position and KV head (the OCP MXFP4 format):
 * 4.25 bits per element, half of the 8-bit cache's, in the same blocks of 64 positions. The
 * scale belongs to a position, so that a row is written or moved without another's being rounded
 * again; beside each position and KV head the cache keeps the attention weight that it has had,
 * by which sp_hip_fp4_evict shortens sequences. The reference has no counterpart.
 *
 * Batches, blocks and rows are those of the 8-bit cache (sp_hip_fp8_batch_t). Conventions
 * (return values, streams) are those of sp_hip.h.
 */
#ifndef SP_HIP_FP4_H
#define SP_HIP_FP4_H

#include "sp_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

#define SP_FP4_BLOCK 64

typedef sp_hip_fp8_batch_t sp_hip_fp4_batch_t;

typedef struct {
    sp_config_t config;    /* head_dim (64, 96, 128 or 256), n_layers, n_heads_kv are used */
    int         n_blocks;
    void       *d_k_codes; /* [n_layers][n_blocks][n_heads_kv][head_dim / 8][64][4] bytes: eight codes of a
                            * position, the lowest channel in the lowest four bits */
    void       *d_v_codes;
    void       *d_k_exp;   /* [n_layers][n_blocks][n_heads_kv][head_dim / 32][64] bytes b in [87, 167]: scale
                            * 2^(b - 127); position p's is the (p/4 % 4 * 16 + p/16 * 4 + p%4)-th */
    void       *d_v_exp;
    float      *d_weight;  /* [n_layers][n_blocks][n_heads_kv][64] attention weight of the positions */
    void       *stream;
    void       *priv;      /* device, attention workspace */
} sp_hip_fp4_cache_t;

/* As sp_hip_fp8_cache_init and _free: cleared, and with the same workspaces. */
int  sp_hip_fp4_cache_init(sp_hip_fp4_cache_t *c, const sp_config_t *cfg, int n_blocks, void *stream);
void sp_hip_fp4_cache_free(sp_hip_fp4_cache_t *c);

/* As sp_hip_fp8_write, at 4 bits: scale = 2^e with the least e in [-40, 40] that puts the largest
 * magnitude of the 32 channels at most at 6 * 2^e, code = E2M1 of x / scale rounded to nearest
 * even. NaN is stored as 0, magnitudes past 6 * 2^40 (infinity among them) as that. A position
 * whose K is written has attention weight 0. Only the rows' own positions are written, but
 * that a block whose first position is written starts anew: behind its rows it then counts as
 * empty. A call must not reach the same position twice, nor from two places a block that it starts anew. */
int  sp_hip_fp4_write(sp_hip_fp4_cache_t *c, int layer, const sp_hip_fp4_batch_t *batch, const void *d_k,
                      const void *d_v, long long row_stride, int dtype, void *stream);
/* The batch's rows read back: code * scale, rounded to dtype. */
int  sp_hip_fp4_read(const sp_hip_fp4_cache_t *c, int layer, const sp_hip_fp4_batch_t *batch, void *d_k, void *d_v,
                     long long row_stride, int dtype, void *stream);

/* As sp_hip_fp8_attn_decode and _prefill. Of a block's keys, and of its values, nothing finer
 * than 2^-25 of the largest scale that the block holds for the KV head is seen (a row that has been taken
 * back counts there until it is written over). Rows are written alone, but no call may write into a block
 * that an attention or weigh call under way reads. Which kernel serves a call goes by table_stride, which
 * stands for the length: tables much wider than their sequences make prompts of 100 to 300 rows slower. */
int  sp_hip_fp4_attn_decode(const sp_hip_fp4_cache_t *c, int layer, const sp_hip_fp4_batch_t *batch, const void *d_q,
                            long long q_stride, int n_q, int dtype, float kq_scale, int window, void *d_out,
                            long long out_stride, float *d_lse, void *stream);
int  sp_hip_fp4_attn_prefill(const sp_hip_fp4_cache_t *c, int layer, const sp_hip_fp4_batch_t *batch, const void *d_q,
                             long long q_stride, int n_q, int dtype, float kq_scale, int window, void *d_out,
                             long long out_stride, float *d_lse, void *stream);

/* Adds to d_weight, for each KV head and each position that the batch's rows see, the sum over the rows
 * and the KV head's query heads of exp(kq_scale * q . K - lse), K as attention sees it: with the arguments
 * of an attention call and the d_lse [n_rows][n_q] that it gave, its softmax weights. (A 16-bit query counts
 * whole, where attention sees nothing finer than 2^-39 of a row's largest entry; and d_lse is fp32, so that
 * scores near 2^n put a weight off by a factor of up to about e^(2^(n - 22)).) Any rows (d_row NULL or not),
 * so a prompt may be weighed by its last rows alone. A row and head whose lse or whose q is not finite
 * adds nothing. Needs no workspace: calls may overlap, but two that meet in a block, or a batch whose
 * sequences share one, add in no certain order (fp32 sums may differ in their last bits). */
int  sp_hip_fp4_weigh(sp_hip_fp4_cache_t *c, int layer, const sp_hip_fp4_batch_t *batch, const void *d_q,
                      long long q_stride, int n_q, int dtype, float kq_scale, int window, const float *d_lse,
                      void *stream);

/* Cuts each sequence of the batch that has more than `keep` positions to keep, for each KV head apart: its
 * `first` first ones, its `recent` last ones and, of those between, the keep - first - recent with the
 * largest attention weight (of equal ones the earlier; NaN is below all). They keep their order and are
 * moved, with their weights, into positions 0 .. keep - 1 of the sequence's table row; from there on
 * the sequence's length is keep, and blocks past that are the caller's again. Nothing is rounded.
 * d_kept [n_seq][n_heads_kv][keep] int32 gets the old position of each (a sequence of n <= keep is left as
 * it is, whatever its table holds, and gets 0 .. n - 1, then -1). A position of an attention call is then
 * its place, so a window counts kept positions, and keys should carry their rotation already. A longer
 * sequence with a table entry missing in its length is left as it is and gets -1. d_len is not changed,
 * d_row is not read (n_rows = n_seq without it). No other call may use the sequences' blocks meanwhile,
 * and no block is theirs twice or another sequence's too (a shared prefix would be moved under it;
 * nothing checks this). */
int  sp_hip_fp4_evict(sp_hip_fp4_cache_t *c, int layer, const sp_hip_fp4_batch_t *batch, int keep, int first, int recent,
                      int32_t *d_kept, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* SP_HIP_FP4_H */
