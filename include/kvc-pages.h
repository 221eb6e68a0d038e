/*
 * kvc-pages.h — a paged KV cache of stored rows and the operations that move
 * its pages: reserving rows, writing and reading them, copying pages, forking
 * a sequence, compacting it to kept rows and freeing it.
 *
 * The cache keeps, for every layer, rows in the library's stored types (one
 * row holds all KV heads of a token, as kvc-batched.h's K and V do) in pages
 * of page_size rows. A sequence (slot) is a row of page_table and a length;
 * its row r lies in page page_table[slot][r / page_size] at r % page_size, in
 * every layer. ref_count[page] counts the table entries that hold the page;
 * 0 is a free page. All of it is device memory that the caller allocates; the
 * calls only launch kernels on the caller's stream, read no device value on
 * the host and allocate nothing, so they can be captured into a graph.
 * Consecutive calls on one cache must be ordered (same stream, or events).
 *
 * Pages are handed out lowest index first, among those that were free when
 * the call started (pages that the call itself gives back serve later calls).
 * A call whose pages do not suffice, or whose table rows are too short,
 * changes nothing but *status, which it sets to -11 or -13 (of both, -13);
 * calls that succeed leave *status as it is. A copy that does not arrive
 * within a kernel's limit sets *status to -12, and the call's rows mean
 * nothing. The workspace (kvc_pages_workspace bytes)
 * may be shared by ordered calls, not by concurrent ones.
 *
 * Sequence lists are HOST arrays, read before the call returns: ids in
 * [0, n_slots), at most KVC_PAGES_MAX_SEQS of them; each destination appears
 * once and is no other entry's source. A captured call keeps them, and host
 * counts and first rows, as they were. Everything else is device memory.
 * n_pages and max_pages times page_size are at most 2^31 - 1 - 65536.
 * Calls with n = 0 do nothing. Return codes: 0; -1 a null argument; -2 bad
 * counts, ids or a repeated destination; -4 a row size that does not match;
 * -10 no sm_100 device; -12 CUDA error; -13 a shape outside the limits, an
 * array that is not aligned to its elements (workspaces: to 16 bytes) or a
 * workspace that is too small. The current device must be the cache's.
 */
#ifndef KVC_PAGES_H
#define KVC_PAGES_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define KVC_PAGES_MAX_SEQS 256

typedef struct kvc_page_cache {
    int       n_layers;
    int       n_pages;      /* pages of the pool */
    int       page_size;    /* rows per page, any number >= 1 */
    int       n_slots;      /* rows of page_table */
    int       max_pages;    /* entries per row of page_table */
    int       n_head_kv;
    int       d_k;
    int       d_v;
    int       k_type;       /* KV_TYPE_* */
    int       v_type;
    size_t    k_row_bytes;  /* n_head_kv*d_k values */
    size_t    v_row_bytes;
    uint8_t * K;            /* [n_layers x n_pages x page_size x k_row_bytes] */
    uint8_t * V;            /* [n_layers x n_pages x page_size x v_row_bytes] */
    float *   beta;         /* [n_layers x n_pages x n_head_kv x page_size], or NULL (no bias) */
    int *     page_table;   /* [n_slots x max_pages]; unused entries are negative */
    int *     seq_len;      /* [n_slots] rows of each sequence */
    int *     ref_count;    /* [n_pages] */
    int *     status;       /* [1] */
} kvc_page_cache;

/* Workspace bytes that any of the calls below needs. */
size_t kvc_pages_workspace(const kvc_page_cache * cache);

/* Append add[i] >= 0 rows (host counts) to sequence seqs[i]; their content is
 * whatever the pages hold. */
int kvc_pages_reserve(const kvc_page_cache * cache, const int * seqs, const int * add, int n, void * workspace,
                      size_t workspace_bytes, void * stream);

/* Rows first[i] .. first[i]+count[i]-1 of sequence seqs[i] (host counts) from
 * / to packed rows k_rows [n_layers x sum(count) x k_row_bytes], v_rows and
 * beta_rows [n_layers x n_head_kv x sum(count)]; a null array is left out (a
 * write then sets no beta; beta_rows needs a cache with beta). Rows past the
 * sequence's length are skipped; a write also skips rows of pages that more
 * than one sequence holds, and then sets *status to -2. seqs may repeat in a
 * read.
 * One layer's rows (a decoder has layer l's K and V only after layer l - 1's
 * attention): these two calls, and kvc_attn_tree with layer 0, also take a
 * description of that layer alone, the same but for n_layers = 1 and K, V and
 * beta at the layer's own part (K + l * n_pages * page_size * k_row_bytes, and
 * so on). Calls that change tables want all layers. */
int kvc_pages_write(const kvc_page_cache * cache, const int * seqs, const int * first, const int * count, int n,
                    const uint8_t * k_rows, const uint8_t * v_rows, const float * beta_rows, void * stream);
int kvc_pages_read(const kvc_page_cache * cache, const int * seqs, const int * first, const int * count, int n,
                   uint8_t * k_rows, uint8_t * v_rows, float * beta_rows, void * stream);

/* Copy pages src[i] -> dst[i] (device arrays) in every layer: K, V and beta.
 * A pair with an index outside the pool is skipped. The destinations are
 * distinct and no sources. Tables and counts stay as they are. */
int kvc_pages_copy(const kvc_page_cache * cache, const int * src, const int * dst, int n, void * stream);

/* Sequence dst[i] becomes a copy of src[i]: it shares src's full pages; the
 * rows of a last, partly filled page are copied to a page of its own. dst's
 * former pages are given back. A source may serve several destinations. */
int kvc_pages_fork(const kvc_page_cache * cache, const int * src, const int * dst, int n, void * workspace,
                   size_t workspace_bytes, void * stream);

/* Sequence dst[i] becomes the first base[i] rows of src[i] followed by its
 * rows keep[..] in that order; src[i] == dst[i] compacts in place. base[n],
 * keep_n[n] and keep are device arrays: the list of layer l and entry i is
 * keep[l*keep_layer_stride + i*keep_ld + 0 .. keep_n[i]-1] (absolute rows;
 * keep_layer_stride 0: one list for all layers); base is cut to src's length
 * and keep_n to [0, keep_ld]. A kept row outside src leaves its place in the
 * new pages as it was. Full pages of the base are shared, the other rows go
 * to new pages. v_rows [n_layers x n x keep_ld x v_row_bytes] and beta_rows
 * [n_layers x n x n_head_kv x keep_ld], when not NULL, replace the kept rows'
 * V and beta (kvc_compact_layers_dev's V_out and beta have this layout for
 * n = 1 and keep_ld = t). */
int kvc_pages_compact(const kvc_page_cache * cache, const int * src, const int * dst, int n, const int * base,
                      const int * keep_n, const int * keep, int keep_ld, size_t keep_layer_stride,
                      const uint8_t * v_rows, const float * beta_rows, void * workspace, size_t workspace_bytes,
                      void * stream);

/* Give back the pages of seqs[i] and set their lengths to 0. */
int kvc_pages_free(const kvc_page_cache * cache, const int * seqs, int n, void * workspace, size_t workspace_bytes,
                   void * stream);

#ifdef __cplusplus
}
#endif

#endif /* KVC_PAGES_H */
