/*
 * kvc-attn.h — attention over the caches that this library compacts: whole
 * prompts, and drafted or single tokens over a paged cache of stored rows.
 *
 * Query head h reads KV head h / (n_head / n_head_kv). Scores, the running
 * maximum and sum of each softmax and the output sums are held in 32 bits.
 * On the tensor cores the probabilities (for block types times the scale of
 * the row's block) meet V in fp16: with F16 queries rounded once, by up to
 * 2^-11 of each, while the sum that divides them is not rounded, so that F16
 * outputs carry this rounding beside their own; with F32 queries as two fp16
 * pieces, 22 bits together, as the queries themselves. Prompts of F32, and
 * shapes that the tensor-core kernels do not take, are 32-bit throughout.
 * A row that sees no key gets an output of 0 and a log-sum-exp of -inf.
 * The calls launch kernels on `stream` (a cudaStream_t; NULL = the legacy
 * default stream) and return; they read no device value on the host and
 * allocate nothing, so they can be captured into a graph. Pointers are device
 * memory of the current device. Return codes: 0; -1 a null argument; -2 bad
 * dimensions; -4 a row size that does not match; -10 no sm_100 device; -12
 * CUDA error; -13 a shape, alignment or workspace outside the limits. Waits
 * inside the kernels have a limit, which no call is known to reach; beyond it
 * kvc_attn_prompt gives rows of NaN, and kvc_attn_tree sets the cache's *status
 * to -12 and leaves outputs that mean nothing.
 */
#ifndef KVC_ATTN_H
#define KVC_ATTN_H

#include <stddef.h>
#include <stdint.h>

#include "kvc-pages.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Attention over whole prompts: n_seqs sequences packed one after another,
 * sequence s with queries cu_q[s] .. cu_q[s+1]-1 and keys cu_k[s] ..
 * cu_k[s+1]-1 (cumulative counts, ascending from 0; values past total_q /
 * total_k are cut). With causal != 0 query i of nq sees keys 0 .. i + nk - nq
 * (aligned to the end: the queries are the sequence's last tokens).
 * Element (token, head, i) of q lies at q + token*q_stride + head*q_head_stride
 * + i elements, and so on; i has stride 1. out and lse are dense [total_q x
 * n_head x d_v] and [total_q x n_head]. Rows of out and lse past the last
 * sequence are left as they were. q, k, v must be finite where a query of the
 * same sequence reads them or has them masked; other sequences never matter. */
typedef struct kvc_prompt_desc {
    const void * q;
    const void * k;
    const void * v;
    void *       out;
    float *      lse;            /* or NULL */
    const int *  cu_q;           /* [n_seqs + 1] */
    const int *  cu_k;           /* [n_seqs + 1] */
    int          type;           /* of q, k, v and out: KV_TYPE_F16 or KV_TYPE_F32 */
    int          n_seqs;
    int          total_q;
    int          total_k;
    int          n_head;
    int          n_head_kv;
    int          d_k;            /* <= 256 */
    int          d_v;            /* <= 256 */
    int          causal;
    float        scale;
    long long    q_stride, q_head_stride;
    long long    k_stride, k_head_stride;
    long long    v_stride, v_head_stride;
} kvc_prompt_desc;

int kvc_attn_prompt(const kvc_prompt_desc * desc, void * stream);

/* Attention of drafted tokens over a paged cache. Entry s of the batch has the
 * nodes cu[s] .. cu[s+1]-1 (rows of q) and reads sequence seqs[s] of the
 * cache, whose last nodes-many rows are the nodes' own rows (reserved and
 * written before the call). A node sees every earlier row, and the own row of
 * node j of its entry where bit j % 32 of mask[node*mask_words + j/32] is set
 * (mask NULL: all of them; nodes past 32*mask_words: none). One token per
 * sequence is a tree of one node. Row r of the cache adds beta (when the cache
 * has it) to its scaled score; beta = -inf hides the row from the head's
 * queries. An entry whose sequence id lies outside the cache sees no key. max_nodes
 * is the most nodes of any entry; of entries with more the first max_nodes are
 * computed, as they would be beside the others, whose own rows count as theirs
 * (the output rows of the nodes behind are left as they were). */
typedef struct kvc_tree_desc {
    const void *     q;          /* [total x n_head x d_k], rows q_stride elements apart */
    void *           out;        /* [total x n_head x d_v] dense, of q's type */
    float *          lse;        /* [total x n_head] or NULL */
    const int *      cu;         /* [n_seqs + 1] */
    const int *      seqs;       /* [n_seqs] */
    const uint32_t * mask;       /* [total x mask_words] or NULL */
    int              q_type;     /* KV_TYPE_F16 or KV_TYPE_F32 */
    int              mask_words;
    int              n_seqs;
    int              total;
    int              max_nodes;
    int              n_head;
    int              layer;      /* of the cache */
    float            scale;
    long long        q_stride;
} kvc_tree_desc;

/* Workspace bytes of a call with these sizes (not shared by concurrent calls);
 * 0 and a negative code in *rc (may be NULL) for bad arguments. */
size_t kvc_attn_tree_workspace(const kvc_page_cache * cache, const kvc_tree_desc * desc, int * rc);
int kvc_attn_tree(const kvc_page_cache * cache, const kvc_tree_desc * desc, void * workspace, size_t workspace_bytes,
                  void * stream);

#ifdef __cplusplus
}
#endif

#endif /* KVC_ATTN_H */
