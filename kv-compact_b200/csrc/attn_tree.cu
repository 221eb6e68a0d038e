// attn_tree.cu — attention of drafted tokens over the paged cache
// (include/kvc-attn.h): argument checks and the choice of kernel.
#include "attn.h"
#include "attn_tree.h"

#include <limits.h>

namespace {

struct tree_plan {
    kvc_attn_args a;
    enum { SIMT, MMA, TC } kernel;
    size_t bytes, meta_at;
};

int head_bytes(int type, int d) {
    return type == KV_TYPE_F32 ? 4 * d : type == KV_TYPE_F16 ? 2 * d : d / 32 * kvc_block_bytes(type);
}

int make_plan(const kvc_page_cache * c, const kvc_tree_desc * t, int sms, tree_plan * p) {
    int rc = kvc_check_cache(c);
    if (rc) return rc;
    if (!t) return KVC_ERR_NULL;
    if (t->n_seqs < 0 || t->total < 0 || t->max_nodes < 0 || t->n_head <= 0 || t->mask_words < 0 || t->layer < 0 ||
        t->layer >= c->n_layers || t->n_head % c->n_head_kv != 0)
        return KVC_ERR_DIMS;
    if (t->q_type != KV_TYPE_F16 && t->q_type != KV_TYPE_F32) return KVC_ERR_DIMS;
    if (t->n_seqs > 0 && t->total > 0 && (!t->q || !t->out || !t->cu || !t->seqs)) return KVC_ERR_NULL;
    if (t->q_stride < (long long)t->n_head * c->d_k) return KVC_ERR_DIMS;
    if (c->d_k > KVC_MAX_D || c->d_v > KVC_MAX_D) return KVC_ERR_SHAPE;
    // a head's part of a row is whole blocks
    for (int i = 0; i < 2; i++) {
        const int type = i ? c->v_type : c->k_type, d = i ? c->d_v : c->d_k;
        if (type != KV_TYPE_F32 && type != KV_TYPE_F16 && d % 32 != 0) return KVC_ERR_SHAPE;
    }
    const uintptr_t qa = t->q_type == KV_TYPE_F32 ? 3 : 1;
    if (((uintptr_t)t->q & qa) || ((uintptr_t)t->out & qa)) return KVC_ERR_SHAPE;
    if (!kvc_words_aligned({t->lse, t->cu, t->seqs, t->mask})) return KVC_ERR_SHAPE;
    if ((long long)t->total * t->n_head > INT_MAX || (long long)t->max_nodes * t->n_head > INT_MAX) return KVC_ERR_SHAPE;
    if (sms < 0) return sms;                             // no device: after the argument checks
    kvc_attn_args & a = p->a;
    a = kvc_attn_args{};
    a.q = t->q;
    a.out = t->out;
    a.lse = t->lse;
    a.q_stride = t->q_stride;
    a.q_head = c->d_k;
    a.cu_q = t->cu;
    a.q_type = t->q_type;
    a.n_seqs = t->n_seqs;
    a.n_total = t->total;
    a.max_q = t->max_nodes;
    a.Hq = t->n_head;
    a.Hkv = c->n_head_kv;
    a.g = t->n_head / c->n_head_kv;
    a.dk = c->d_k;
    a.dv = c->d_v;
    a.scale = t->scale;
    const size_t rows = (size_t)c->n_pages * c->page_size;
    a.K = c->K + (size_t)t->layer * rows * c->k_row_bytes;
    a.V = c->V + (size_t)t->layer * rows * c->v_row_bytes;
    a.k_rb = (long long)c->k_row_bytes;
    a.v_rb = (long long)c->v_row_bytes;
    a.k_hb = head_bytes(c->k_type, c->d_k);
    a.v_hb = head_bytes(c->v_type, c->d_v);
    a.k_type = c->k_type;
    a.v_type = c->v_type;
    a.seqs = t->seqs;
    a.table = c->page_table;
    a.seq_len = c->seq_len;
    a.beta = c->beta ? c->beta + (size_t)t->layer * rows * c->n_head_kv : nullptr;
    a.mask = t->mask;
    a.mask_words = t->mask_words;
    a.status = c->status;
    a.n_slots = c->n_slots;
    a.n_pages = c->n_pages;
    a.max_pages = c->max_pages;
    a.page = c->page_size;
    a.by_page = kvc_make_divisor((uint32_t)c->page_size);
    a.by_group = kvc_make_divisor((uint32_t)a.g);
    if (t->n_seqs == 0 || t->total == 0 || t->max_nodes == 0) {
        p->bytes = 0;
        return KVC_OK;
    }
    long long blocks = 0;
    if (kvc_attn_tree_tc_plan(&a, sms, &blocks)) {
        p->kernel = tree_plan::TC;
    } else if (kvc_attn_tree_mma_plan(&a, sms, &blocks)) {
        p->kernel = tree_plan::MMA;
    } else {
        p->kernel = tree_plan::SIMT;
        kvc_attn_simt_split(&a, sms, false);
        blocks = a.n_parts;
    }
    p->bytes = kvc_attn_part_bytes(a, blocks, &p->meta_at);
    return KVC_OK;
}

}  // namespace

extern "C" {

KVC_EXPORT size_t kvc_attn_tree_workspace(const kvc_page_cache * cache, const kvc_tree_desc * desc, int * rc) {
    tree_plan p;
    const int r = make_plan(cache, desc, kvc_serve_device(), &p);
    if (rc) *rc = r;
    return r ? 0 : p.bytes;
}

KVC_EXPORT int kvc_attn_tree(const kvc_page_cache * cache, const kvc_tree_desc * desc, void * workspace,
                             size_t workspace_bytes, void * stream) {
    tree_plan p;
    const int sms = kvc_serve_device();
    const int rc = make_plan(cache, desc, sms, &p);
    if (rc) return rc;
    if (desc->n_seqs == 0 || desc->total == 0 || desc->max_nodes == 0) return KVC_OK;
    if (p.bytes && !workspace) return KVC_ERR_NULL;
    if (p.bytes > workspace_bytes || ((uintptr_t)workspace & 15)) return KVC_ERR_SHAPE;
    p.a.part = static_cast<float *>(workspace);
    p.a.meta = reinterpret_cast<int *>(static_cast<uint8_t *>(workspace) + p.meta_at);
    if (p.kernel == tree_plan::TC) return kvc_launch_attn_tree_tc(p.a, (cudaStream_t)stream);
    if (p.kernel == tree_plan::MMA) return kvc_launch_attn_tree_mma(p.a, (cudaStream_t)stream);
    return kvc_launch_attn_simt(p.a, (cudaStream_t)stream);
}

}  // extern "C"
