/*
 * llama3pure_paged.h -- the paged KV cache of libllama3pure_attn.so: many
 * sequences in one pool of pages, served in batches.
 *
 * The cache of llama3pure_attn.h holds one sequence of fixed capacity, as the
 * reference's engines do (llama3pure-c-engine.c:365-379).  A process that serves
 * several users needs what is here beside it: sequences that grow page by
 * page, share the pages of a common prompt, are copied, cut and freed, and one
 * attention call for a whole batch in which every sequence brings as many new
 * tokens as it has (one when it decodes, a chunk of its prompt before that).
 *
 * One step of a serving loop:
 *     l3p_paged_begin(ctx, n_seqs, seqs, n_new, stream);        once per step
 *     for each layer:
 *         l3p_paged_rope_append_dev(ctx, layer, q, k, v, ...);  rotate, write K/V
 *         l3p_paged_attn_dev(ctx, layer, q, out, ...);          attend
 *
 * Conventions (beside those of llama3pure_attn.h, whose codes are used)
 *   - Rows are of the pool's type: float with L3P_PAGED_F32, bfloat16 with
 *     L3P_PAGED_BF16.  Scores, softmax statistics and sums are fp32 in both;
 *     with BF16 rows a weight is rounded to bfloat16 ahead of its product with
 *     V, and so is the output; fp32 products are right to 2^-21 of themselves.
 *   - Token rows of a batch are stacked in the order of l3p_paged_begin's
 *     sequences: q, out [n_tok][n_heads][head_dim], k, v
 *     [n_tok][n_kv_heads][head_dim].  Strides are elements from one token to
 *     the next, 0 for dense rows; rows and strides are multiples of 16 bytes, so
 *     q, k and v may lie in one projection's output.
 *   - A stream of NULL is the legacy default stream.  Calls of one context are
 *     made from one host thread, and run on one stream or on streams that the
 *     caller orders: the batch description and the split workspace belong to
 *     the context.  Two captured graphs of one context must not run at once.
 *   - The calls that only keep books (new, fork, truncate, free, pages, tables)
 *     launch nothing.  A page that is freed may be given out by the next begin
 *     or copy; work on it that is already enqueued comes first when the stream
 *     is the same.
 *   - new, fork, begin, truncate, free, copy and compact check everything
 *     first: a call that they refuse changes nothing, also for want of host,
 *     pinned or device memory (L3P_E_NOMEM).  L3P_E_CUDA is a failure of the
 *     device, after which the pool's rows are not defined.
 *   - Freeing, truncating or compacting ends the current batch: append and
 *     attention are refused until the next begin.
 */
#ifndef LLAMA3PURE_PAGED_H
#define LLAMA3PURE_PAGED_H

#include "llama3pure_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

#define L3P_PAGED_F32 0  /* float pages, float q and out */
#define L3P_PAGED_BF16 1 /* bfloat16 pages, bfloat16 q and out */

/* Geometry of a pool.  Storage: one allocation
 * [n_pages][n_layers][2: K, V][n_kv_heads][page_size][head_dim], zeroed. */
typedef struct l3p_paged_config {
    int n_layers;
    int n_heads;      /* query heads; a multiple of n_kv_heads */
    int n_kv_heads;
    int head_dim;     /* 64, 128 or 256 */
    int page_size;    /* positions per page: 16, 32, 64 or 128 */
    int n_pages;      /* pages of the pool */
    int max_seqs;     /* sequences that may exist at once */
    int max_tokens;   /* new tokens of one batch at most */
    int max_seq_len;  /* positions of one sequence at most; 0 => n_pages * page_size.  The device block of a step's
                         description has room for max_seqs tables of that many positions (a word a page; F32 pools: and
                         four words per 128 positions): 64 sequences in a pool of 64K pages: 17 MB */
    int dtype;        /* L3P_PAGED_F32 or L3P_PAGED_BF16 */
    float scale;      /* multiplies q.k, not negative; 0 => 1/sqrt(head_dim) */
    int is_gemma3;    /* sliding-window layers as in l3p_attn_config: with is_gemma3, */
    int swa_window;   /*   swa_window > 0 and swa_pattern > 0, layer l with */
    int swa_pattern;  /*   l % swa_pattern < swa_pattern - 1 attends to the last swa_window positions */
    int device;
} l3p_paged_config;

typedef struct l3p_paged_ctx l3p_paged_ctx;

int l3p_paged_create(const l3p_paged_config* cfg, l3p_paged_ctx** out);
/* Why the last l3p_paged_create of the calling thread failed ("" after one that did not). */
const char* l3p_paged_create_error(void);
void l3p_paged_destroy(l3p_paged_ctx* ctx);
const char* l3p_paged_last_error(const l3p_paged_ctx* ctx);
/* Waits for `stream` and reports what its kernels recorded, clearing it:
 * L3P_E_TIMEOUT after a bounded wait gave up, L3P_E_INVAL when a captured
 * launch met a batch that it cannot serve (see l3p_paged_attn_dev).  Not during
 * stream capture. */
int l3p_paged_check(l3p_paged_ctx* ctx, void* stream);
/* Kernels launched since the context was created. */
long long l3p_paged_launch_count(const l3p_paged_ctx* ctx);
/* Device address and size of the storage. */
int l3p_paged_storage(l3p_paged_ctx* ctx, void** base, size_t* bytes);

/* ---- sequences and pages ------------------------------------------------- */
/* A sequence without tokens; ids are 0 .. max_seqs-1, the lowest free first. */
int l3p_paged_seq_new(l3p_paged_ctx* ctx, int* seq);
/* n sequences that share the first n_tokens positions of `seq` (n_tokens < 0:
 * all of them) with it, page by page, without moving data.  Whoever next grows
 * into a last page that others hold as well gets a copy of its rows first (in
 * l3p_paged_begin). */
int l3p_paged_seq_fork(l3p_paged_ctx* ctx, int seq, int n_tokens, int n, int* children);
/* New sequences children[i] with pages of their own that hold the rows of
 * seqs[i]; the rows move in one launch on `stream`. */
int l3p_paged_seq_copy(l3p_paged_ctx* ctx, int n, const int* seqs, int* children, void* stream);
/* Keeps the first n_tokens positions; pages behind them lose this holder. */
int l3p_paged_seq_truncate(l3p_paged_ctx* ctx, int seq, int n_tokens);
/* Ends the sequences.  Pages that nobody holds any more become free. */
int l3p_paged_seq_free(l3p_paged_ctx* ctx, int n, const int* seqs);
int l3p_paged_seq_length(l3p_paged_ctx* ctx, int seq, int* n_tokens);
/* Page tables of n sequences, row i at table + i*width, filled up with -1.
 * *need (may be NULL) is the widest row; with table NULL nothing else is
 * written; a width below *need is L3P_E_RANGE. */
int l3p_paged_tables(l3p_paged_ctx* ctx, int n, const int* seqs, int width, int* table, int* need);
int l3p_paged_free_pages(l3p_paged_ctx* ctx, int* n_free);
/* Moves the used pages with the highest indices to the free pages with the
 * lowest ones, in one launch on `stream`, until the pages in use are
 * 0 .. *n_used-1, and points the sequences' tables there. */
int l3p_paged_compact(l3p_paged_ctx* ctx, int* n_used, void* stream);

/* ---- a step ---------------------------------------------------------------- */
/* Begins a batch: sequence seqs[i] grows by n_new[i] >= 0 tokens.  Gives out
 * pages (always the free page of the lowest index), copies the rows of shared
 * last pages, and puts the batch's description on the device.  The rows of
 * the new tokens hold whatever the pages held until append writes them.
 * L3P_E_NOMEM when the free pages do not suffice.  Not during stream capture. */
int l3p_paged_begin(l3p_paged_ctx* ctx, int n_seqs, const int* seqs, const int* n_new, void* stream);

#define L3P_ROPE_INTERLEAVED 0 /* pairs (2i, 2i+1), c:3279-3296 */
#define L3P_ROPE_HALF 1        /* pairs (i, i + rotary_dim/2), c:3254-3278 */
#define L3P_ROPE_SCALE_NONE 0
#define L3P_ROPE_SCALE_LINEAR 1 /* every frequency / factor */
#define L3P_ROPE_SCALE_BANDS 2  /* by wavelength (Llama 3.1): above original_len/low_freq the frequency
                                   / factor, below original_len/high_freq as it is, blended between */
#define L3P_ROPE_SCALE_YARN 3   /* by pair: turns over original_len above beta_fast as it is, below
                                   beta_slow / factor, a linear ramp between; cosine and sine are
                                   multiplied by attn_factor */
typedef struct l3p_paged_rope_config {
    int max_pos;         /* positions the tables cover */
    int layout;          /* L3P_ROPE_INTERLEAVED or L3P_ROPE_HALF */
    int rotary_dim;      /* the first rotary_dim values of a head turn (even); 0 => head_dim */
    int scaling;         /* L3P_ROPE_SCALE_* */
    float theta;         /* 0 => 500000 */
    float theta_swa;     /* sliding-window layers; they are not scaled; 0 => 10000 */
    float factor;        /* >= 1 */
    float low_freq, high_freq;   /* BANDS; 0 => 1, 4 */
    float beta_fast, beta_slow;  /* YARN; 0 => 32, 1 */
    int original_len;    /* BANDS, YARN: positions the model was trained on */
    float attn_factor;   /* YARN; 0 => 0.1 ln(factor) + 1 */
    float rms_norm_eps;  /* 0 => 1e-5 */
    const float* q_norm; /* HOST [n_layers][head_dim] weights of an RMS norm of every q / k head ahead of the */
    const float* k_norm; /*   rotation (c:3150-3165), both or neither; NULL: none */
} l3p_paged_rope_config;
/* Builds the cosine and sine tables, angles in double precision.  Calling it
 * again replaces them; graphs captured before keep the ones they were captured
 * with.  Waits for the device. */
int l3p_paged_set_rope(l3p_paged_ctx* ctx, const l3p_paged_rope_config* rope);
/* Norm (when configured) and rotation of the batch's q and k rows; q goes to
 * q_out (which may be q), k and v into the pages.  One launch. */
int l3p_paged_rope_append_dev(l3p_paged_ctx* ctx, int layer, const void* q, long long q_stride, const void* k,
                              long long k_stride, const void* v, long long v_stride, void* q_out,
                              long long q_out_stride, void* stream);
/* The batch's k (already rotated) and v into the pages. */
int l3p_paged_append_dev(l3p_paged_ctx* ctx, int layer, const void* k, long long k_stride, const void* v,
                         long long v_stride, void* stream);
/* Attention of the batch's tokens over their sequences: the token at position
 * t attends to positions [max(0, t - window + 1), t] (windowed layers) or
 * [0, t].  The new tokens' K/V rows must have been appended.  Rows of out
 * behind the batch's last token are left as they were.  Positions that a token
 * does not attend to never reach its output, whatever they hold.  A value that
 * is not finite at a position that it does attend to leaves values that are not
 * finite (F32 pools: NaN also where the formula has an infinity or, for a key,
 * a weight of 0).
 *
 * Capture: a captured launch reads the batch's description when it is
 * replayed, so one graph of a decoding step serves every later step whose
 * batch takes the same path with at most as many tokens as the captured one:
 * with n_new * n_heads / n_kv_heads query rows per KV head, the largest count
 * of a batch of few tokens is at most 8, or 9 to 16 (F32 pools: 9 to 64, with
 * head_dim 256 9 and more).  A replay on a batch that does not fit writes
 * nothing for it and l3p_paged_check reports L3P_E_INVAL.  A graph of chunks
 * serves batches whose plan has no more parts, which goes by the lengths too. */
int l3p_paged_attn_dev(l3p_paged_ctx* ctx, int layer, const void* q, long long q_stride, void* out,
                       long long out_stride, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* LLAMA3PURE_PAGED_H */
