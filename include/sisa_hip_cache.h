/*
 * sisa_hip_cache.h -- entry points of libsisa_hip.so for generation caches in pages: writing new positions, the
 * attention of new tokens over the pages, the attention weights that a prompt's positions have received, and eviction
 * by them. Conventions (views, status codes, streams, caller-owned buffers) are those of sisa_hip.h.
 *
 * A pool holds `pages` pages of `page_size` positions for every head. Position j of sequence n lives in slot
 * j % page_size of page table[n * s_table + j / page_size]; each sequence has W entries, and what those behind its last
 * position hold does not matter. Lengths, tables and counts are device memory that the host does not see: where one of them
 * names a place outside the pool, no memory outside it is touched, and the call answers as its declaration says. The tables
 * of two sequences may name the same page for reading (a shared prefix), not for writing.
 *
 * No counterpart in the reference, whose cache is one tensor per layer that grows (src/sisa/generation.py:34-100).
 */
#ifndef SISA_HIP_CACHE_H
#define SISA_HIP_CACHE_H

#include "sisa_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

#define SISA_MIN_PAGE_SIZE 16
typedef struct {
    int32_t pages, heads;
    int32_t page_size;         /* positions of a page: a power of two, at least SISA_MIN_PAGE_SIZE */
    int32_t dtype;             /* of k, v, b: SISA_BF16, SISA_F16 or SISA_F32 */
    sisa_view k, v, b;         /* (pages, heads, page_size, 64|64|32): page, head and position strides */
    sisa_view g, f;            /* (pages, heads, page_size) fp32; f.ptr NULL = no forget term */
} sisa_page_pool;

/* New positions into the pages: row m < count[n] of k, v, b, g, f goes to position start[n] + m. Rows from count[n] on,
 * and rows whose position has no page of the pool, are left out. Sequences must not share a page that is written. */
typedef struct {
    int32_t B, M, W, reserved;
    sisa_page_pool pool;
    const int32_t* table; int64_t s_table;     /* (B, W) */
    const int32_t* start;      /* (B) */
    const int32_t* count;      /* (B), or NULL: M rows of each sequence */
    sisa_view k, v, b;         /* (B,H,M,64|64|32) in the pool's dtype */
    sisa_view g, f;            /* (B,H,M) fp32; f.ptr NULL exactly where the pool's is */
} sisa_paged_write_args;

int sisa_paged_write(const sisa_paged_write_args* a, void* stream);

/* Attention of the last M of each sequence's lengths[n] cached positions (written before) over the positions up to their
 * own, exact fp32 score and softmax as sisa_decode_attn, fp32 output:
 *   s_mj = q_m.k_j/8 + lam_h * exp(g_m - g_j) * (c_m.b_j) + (F_m - F_j)   for j <= lengths[n] - M + m,
 *   out_m = softmax_j(s_mj) v_j;  and, where w_out is given, w_out_j = w_in_j + sum over m of softmax_j(s_mj), for
 *   j < lengths[n] (the others are left as they are; w_in and w_out may be the same memory).
 * A row without a position (a sequence of no positions, or of fewer than M) is 0. The rows of a sequence whose length is
 * negative or above max_len or W pages, or one of whose pages is not in the pool, are NaN (its w_out is left as it is for
 * such a length, and NaN for such a page). max_len bounds the lengths for the launch: at most W * page_size. Workspace:
 * sisa_paged_decode_workspace_bytes(B, H, M, max_len, dtype, whether w_out is given), which may be none. */
typedef struct {
    int32_t B, M, W, max_len;
    sisa_page_pool pool;
    const int32_t* table; int64_t s_table;     /* (B, W) */
    const int32_t* lengths;    /* (B), the M new positions included */
    sisa_view q, c;            /* (B,H,M,64|32) in the pool's dtype */
    sisa_view gq, fq;          /* (B,H,M) fp32; fq.ptr NULL exactly where the pool's f is */
    const float* lam; int64_t s_lam;           /* (H) fp32 */
    sisa_view w_in, w_out;     /* (B,H,max_len) fp32, or both NULL */
    float* out;                /* (B,H,M,64) contiguous */
    void* workspace;           /* 16-byte aligned; NULL where none is needed */
} sisa_paged_decode_args;

int64_t sisa_paged_decode_workspace_bytes(int32_t B, int32_t H, int32_t M, int32_t max_len, int32_t dtype, int32_t tracked);
int sisa_paged_decode(const sisa_paged_decode_args* a, void* stream);

/* The softmax weights that each position j of a prompt receives from the last `window` queries of its sequence (0: from
 * all of them), summed:  out_j = sum over i >= j, n - window <= i < n, of softmax_j(s_ij), with the score of sisa_attn_fwd
 * and n = lengths[b] (NULL: L; values outside 0 .. L count as the nearer of the two); 0 for j >= n. g and f may rise, where a
 * rise of more than 16 costs time. Workspace:
 * sisa_attn_weights_workspace_bytes(B, H, L, window). */
#define SISA_ATTN_WEIGHTS_MAX_STRIDE (1 << 24)    /* of the positions of q, k, c and b, in elements */
typedef struct {
    int32_t B, H, L;
    int32_t window;            /* 0 .. L */
    int32_t dtype;             /* of q, k, c, b: SISA_BF16, SISA_F16 or SISA_F32 */
    int32_t reserved;
    sisa_view q, k;            /* (B,H,L,64) */
    sisa_view c, b;            /* (B,H,L,32) */
    sisa_view g, f;            /* (B,H,L) fp32, position stride 1; f.ptr NULL = no forget term */
    const float* lam; int64_t s_lam;           /* (H) fp32 */
    const int32_t* lengths;    /* (B) or NULL */
    float* out;                /* (B,H,L) contiguous */
    void* workspace;           /* 16-byte aligned */
} sisa_attn_weights_args;

int64_t sisa_attn_weights_workspace_bytes(int32_t B, int32_t H, int32_t L, int32_t window);
int sisa_attn_weights(const sisa_attn_weights_args* a, void* stream);

/* A cache cut down to at most `keep` positions per head, copied to pages of `to` in their order: the last `recent` of the
 * sequence and, of the others, those with the largest weights (of equal ones the lowest position; NaN is above all). The
 * positions that are kept, -1 behind them, and their weights, 0 behind them, are written beside. new_lengths[n] is
 * min(lengths[n], keep), or -1 where the length is negative or above max_len or W pages, where new_table has too few
 * pages, or where the old or the new page of a row that is kept is not in its pool (what the new pages then hold is of no
 * use). The pages of rows that are not kept are not looked at. -1 is an answer, not a length to count on from: a caller who
 * adds the next positions to it has an empty sequence, so negative lengths have to stay as they are (sisa_paged_decode then
 * gives NaN). No page may be both read and written. */
typedef struct {
    int32_t B, W, W_new, max_len;
    int32_t keep, recent;      /* 1 <= recent <= keep */
    sisa_page_pool from, to;   /* same heads and dtype, both with or both without f; page sizes may differ */
    const int32_t* table; int64_t s_table;     /* (B, W) */
    const int32_t* new_table; int64_t s_new;   /* (B, W_new) */
    const int32_t* lengths;    /* (B) */
    sisa_view weights;         /* (B,H,max_len) fp32 */
    int32_t* new_lengths;      /* (B) */
    float* new_weights;        /* (B,H,keep) contiguous */
    int32_t* positions;        /* (B,H,keep) contiguous */
} sisa_cache_evict_args;

int sisa_cache_evict(const sisa_cache_evict_args* a, void* stream);

/* sisa_step (sisa_hip_step.h) with its cache in pages: one new token of each of B rows through a decoder layer, sequence n's
 * at position start[n], lengths[n] = start[n] + 1. The recurrences continue from g_last, f_last and phi, which are advanced in
 * place. weights: accumulated weights as sisa_paged_decode's, in place, or NULL. A sequence whose position has no page of the
 * pool, or whose lengths[n] is not start[n] + 1, gives NaN, its weights are left as they are, and its g_last and f_last become
 * NaN: so do its later steps, until these are set anew. A length above max_len gives NaN. */
typedef struct {
    int32_t B, H, D, FF;       /* rows 1..SISA_STEP_MAX_ROWS, heads, width (64 H), hidden width of the FFN */
    int32_t dtype;             /* SISA_BF16 or SISA_F16, of the pool, too */
    int32_t W, max_len, reserved;
    float eps_attn, eps_ffn;
    const void* x; int64_t sx;         /* (B, D), row stride sx */
    const void* res;                   /* (B, D) contiguous, added to x first, or NULL */
    const void *attn_norm, *w_q, *w_k, *w_v, *w_b, *w_c, *w_theta, *w_alpha, *b_alpha, *w_forget, *b_forget, *w_o;
    const void *ffn_norm, *w_gate, *w_up, *w_down;     /* all contiguous, (outputs, inputs) */
    const float* lambda_raw;           /* (H) */
    sisa_page_pool pool;               /* with f */
    const int32_t* table; int64_t s_table;             /* (B, W) */
    const int32_t *start, *lengths;    /* (B) */
    float *g_last, *f_last, *phi;      /* (B,H), (B,H), (B,H,16) contiguous */
    sisa_view weights;                 /* (B,H,max_len) fp32 or NULL */
    void *h, *ffn;                     /* (B, D) contiguous outputs */
    void* workspace;                   /* sisa_step_paged_workspace_bytes(B,H,D,FF,max_len,dtype,tracked), 256-byte aligned */
} sisa_step_paged_args;

int64_t sisa_step_paged_workspace_bytes(int32_t B, int32_t H, int32_t D, int32_t FF, int32_t max_len, int32_t dtype,
                                        int32_t tracked);
int sisa_step_paged(const sisa_step_paged_args* a, void* stream);

#ifdef __cplusplus
}
#endif

#endif
