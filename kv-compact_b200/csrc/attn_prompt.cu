// attn_prompt.cu — attention over whole prompts (include/kvc-attn.h).
#include "attn.h"
#include "attn_prompt.h"

#include <limits.h>

extern "C" {

KVC_EXPORT int kvc_attn_prompt(const kvc_prompt_desc * t, void * stream) {
    if (!t) return KVC_ERR_NULL;
    if (t->n_seqs < 0 || t->total_q < 0 || t->total_k < 0 || t->n_head <= 0 || t->n_head_kv <= 0 ||
        t->n_head % t->n_head_kv != 0 || t->d_k <= 0 || t->d_v <= 0)
        return KVC_ERR_DIMS;
    if (t->type != KV_TYPE_F16 && t->type != KV_TYPE_F32) return KVC_ERR_DIMS;
    if (t->n_seqs > 0 && t->total_q > 0 && (!t->q || !t->out || !t->cu_q || !t->cu_k)) return KVC_ERR_NULL;
    if (t->n_seqs > 0 && t->total_q > 0 && t->total_k > 0 && (!t->k || !t->v)) return KVC_ERR_NULL;
    if (t->q_stride < 0 || t->k_stride < 0 || t->v_stride < 0 || t->q_head_stride < 0 || t->k_head_stride < 0 ||
        t->v_head_stride < 0)
        return KVC_ERR_DIMS;
    if (t->d_k > KVC_MAX_D || t->d_v > KVC_MAX_D || t->n_head > 65535) return KVC_ERR_SHAPE;
    const int size = t->type == KV_TYPE_F32 ? 4 : 2;
    for (const void * p : {t->q, t->k, t->v, (const void *)t->out})
        if ((uintptr_t)p % size) return KVC_ERR_SHAPE;
    if (!kvc_words_aligned({t->lse, t->cu_q, t->cu_k})) return KVC_ERR_SHAPE;
    if ((long long)t->total_q * t->n_head > INT_MAX) return KVC_ERR_SHAPE;
    const int sms = kvc_serve_device();
    if (sms < 0) return sms;
    if (t->n_seqs == 0 || t->total_q == 0) return KVC_OK;
    kvc_attn_args a{};
    a.q = t->q;
    a.out = t->out;
    a.lse = t->lse;
    a.q_stride = t->q_stride;
    a.q_head = t->q_head_stride;
    a.cu_q = t->cu_q;
    a.q_type = t->type;
    a.n_seqs = t->n_seqs;
    a.n_total = t->total_q;
    a.max_q = t->total_q;
    a.Hq = t->n_head;
    a.Hkv = t->n_head_kv;
    a.g = t->n_head / t->n_head_kv;
    a.dk = t->d_k;
    a.dv = t->d_v;
    a.scale = t->scale;
    a.K = static_cast<const uint8_t *>(t->k);
    a.V = static_cast<const uint8_t *>(t->v);
    a.k_rb = t->k_stride * size;
    a.v_rb = t->v_stride * size;
    a.k_hb = t->k_head_stride * size;
    a.v_hb = t->v_head_stride * size;
    a.k_type = a.v_type = t->type;
    a.cu_k = t->cu_k;
    a.n_keys = t->total_k;
    a.causal = t->causal != 0;
    a.page = 1;
    a.by_page = kvc_make_divisor(1);
    a.by_group = kvc_make_divisor((uint32_t)a.g);
    if (kvc_attn_prompt_tc_ok(a)) return kvc_launch_attn_prompt_tc(a, (cudaStream_t)stream);
    kvc_attn_simt_split(&a, sms, true);
    return kvc_launch_attn_simt(a, (cudaStream_t)stream);
}

}  // extern "C"
