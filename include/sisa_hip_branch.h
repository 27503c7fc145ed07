/*
 * sisa_hip_branch.h -- entry points of libsisa_hip.so for branched and drafted generation: the attention of sequences that
 * have their first positions in common, and the verification of drafted tokens. Pages, tables, lengths and the conventions
 * (views, status codes, streams, caller-owned buffers) are those of sisa_hip_cache.h.
 *
 * No counterpart in the reference, which generates one continuation of a row, token by token
 * (src/sisa/generation.py:137-191).
 */
#ifndef SISA_HIP_BRANCH_H
#define SISA_HIP_BRANCH_H

#include "sisa_hip_cache.h"

#ifdef __cplusplus
extern "C" {
#endif

/* sisa_paged_decode for sequences in groups: those of group r are first[r] .. first[r+1] - 1, and their first shared[r]
 * positions are those of the group's first sequence (the places that its table row names), whatever the others' rows say of
 * them. Position j of a sequence from shared[r] on is where its own row says. Scores, softmax and the rows that are 0 or NaN
 * as sisa_paged_decode; so are the rows of a group whose shared[r] is negative or above max_shared: NaN. first rises from 0
 * to B and group[n] is the group of sequence n: where they do not agree no memory outside the arguments' is touched, and the
 * rows are of no use. An infinite v that a row sees may give NaN. The lengths of a group may be anything, below shared[r],
 * too. max_len bounds the lengths and max_shared the common positions, each at most W * page_size; the launch is sized by
 * them. The positions of a page of the pool are at least a row apart and those of a head within 2 GiB. Workspace:
 * sisa_prefix_decode_workspace_bytes(B, H, M, G, max_len, max_shared). */
typedef struct {
    int32_t B, M, W, G;
    int32_t max_len, max_shared;
    int32_t out_dtype;         /* SISA_F32, or the pool's */
    int32_t reserved;
    sisa_page_pool pool;
    const int32_t* table; int64_t s_table;     /* (B, W) */
    const int32_t* lengths;    /* (B), the M new positions included */
    const int32_t* first;      /* (G + 1) */
    const int32_t* group;      /* (B) */
    const int32_t* shared;     /* (G) */
    sisa_view q, c;            /* (B,H,M,64|32) in the pool's dtype */
    sisa_view gq, fq;          /* (B,H,M) fp32; fq.ptr NULL exactly where the pool's f is */
    const float* lam; int64_t s_lam;           /* (H) fp32 */
    sisa_view out;             /* (B,H,M,64) in out_dtype, unit last stride */
    void* workspace;           /* 16-byte aligned */
} sisa_prefix_decode_args;

int64_t sisa_prefix_decode_workspace_bytes(int32_t B, int32_t H, int32_t M, int32_t G, int32_t max_len, int32_t max_shared);
int sisa_prefix_decode(const sisa_prefix_decode_args* a, void* stream);

/* sisa_step_paged for M new positions of each of step.B sequences in groups: x, res, h and ffn are of step.B * M rows (at most
 * SISA_STEP_MAX_ROWS), row m of sequence n at n * M + m, at position step.start[n] + m; step.lengths[n] = start[n] + M. The
 * attention is sisa_prefix_decode's, first, group, shared and max_shared as there; step.weights is not used (NULL). A sequence
 * one of whose positions has no page of the pool ends with NaN from that row on, all of its attention with it. rows, or NULL:
 * what the recurrences continue from, (B,H,.) of 18 fp32 values (g, F, 16 phases) each s_rows values apart for a sequence
 * and head: before this call at row0, after position m at row0 + 1 + m. */
#define SISA_BRANCH_ROW 18
typedef struct {
    sisa_step_paged_args step;
    int32_t M, G, max_shared, row0;
    const int32_t *first, *group, *shared;     /* (G + 1), (B), (G) */
    float* rows; int64_t s_rows;
} sisa_step_branch_args;

int64_t sisa_step_branch_workspace_bytes(int32_t B, int32_t H, int32_t D, int32_t FF, int32_t M, int32_t G, int32_t max_len,
                                         int32_t max_shared);
int sisa_step_branch(const sisa_step_branch_args* a, void* stream);

/* Drafted tokens against the target's probabilities, by given random numbers. p[n,i] are the target's probabilities of what
 * follows i drafts of row n, q[n,i] those that draft i was drawn from. Draft i < counts[n] is accepted while all before it
 * are and u[n,i] q[n,i][x_i] < p[n,i][x_i] (as real numbers: the products are exact; a draft outside 0 .. V-1 is refused).
 * accepted[n] is how many are; tokens[n] are these, then one that is drawn, then -1. It is drawn with r = u[n,K] from the
 * weights max(p[n,i] - q[n,i], 0) of a refused draft i, or p[n,i] where these are all 0 or no draft is left: the lowest token
 * whose weight is not 0 with sum_{v <= token} w_v > r sum_v w_v, sums in fp64; where rounding leaves none (or r is 1 or more),
 * the last token whose weight is not 0; -1 where the weights are 0 or their sum is not finite. q.ptr NULL: the drafts were
 * not drawn (q is 1 at the draft and 0 elsewhere). counts[n] outside 0 .. K count as the nearer of the two. Workspace:
 * sisa_verify_workspace_bytes(B, V). */
typedef struct {
    int32_t B, K, V;           /* V at most SISA_VERIFY_MAX_V */
    int32_t p_dtype, q_dtype;  /* SISA_F32, SISA_BF16 or SISA_F16 */
    int32_t reserved;
    const void* p; int64_t p_b, p_k;           /* (B, K+1, V), strides of rows and positions, unit last stride */
    const void* q; int64_t q_b, q_k;           /* (B, K, V), or NULL */
    const int64_t* drafts; int64_t d_b, d_k;   /* (B, K) */
    const float* u; int64_t u_b, u_k;          /* (B, K+1) in [0, 1) */
    const int32_t* counts;     /* (B), or NULL: K of each row */
    int64_t* tokens;           /* (B, K+1) contiguous */
    int32_t* accepted;         /* (B) */
    void* workspace;           /* 16-byte aligned */
} sisa_verify_args;

#define SISA_VERIFY_MAX_V (1 << 24)
int64_t sisa_verify_workspace_bytes(int32_t B, int32_t V);
int sisa_verify(const sisa_verify_args* a, void* stream);

#ifdef __cplusplus
}
#endif

#endif
