// attn.h — what the attention kernels share: the launch arguments, the
// sequences of a batch as the device sees them, the split of their keys over
// the CTAs, and the stored elements.
#pragma once

#include <cuda_fp16.h>
#include <math.h>

#include "serve.h"

#include "kv-compact-api.h"

struct kvc_attn_args {
    // queries: element (token, head, i) at q + token*q_stride + head*q_head + i
    const void * q;
    void * out;             // [n_total x Hq x dv]
    float * lse;            // [n_total x Hq] or null
    long long q_stride, q_head;
    const int * cu_q;       // [n_seqs + 1]
    int q_type;
    int n_seqs, n_total, max_q;
    int Hq, Hkv, g, dk, dv;
    float scale;
    // keys: row r, head h at K + r*k_rb + h*k_hb bytes
    const uint8_t * K;
    const uint8_t * V;
    long long k_rb, k_hb, v_rb, v_hb;
    int k_type, v_type;
    // packed prompts (cu_k != null)
    const int * cu_k;       // [n_seqs + 1]
    int n_keys;
    int causal;
    // paged cache (seqs != null)
    const int * seqs;
    const int * table;
    const int * seq_len;
    const float * beta;     // [pages x Hkv x page] or null
    const uint32_t * mask;
    int mask_words;
    int n_slots, n_pages, max_pages, page;
    kvc_divisor by_page, by_group;
    // the split: blocks of rb query rows, tiles of `tile` keys, W workers per
    // KV head and stretch; n_parts stretches, each with partial results of its own:
    // one per row block, or 1 where the row blocks are laid end to end
    int rb, tile, W, n_parts;
    kvc_divisor by_tile;
    float * part;           // partial results
    int * meta;             // [row blocks][n_seqs][2]: first and last worker of a sequence (W > 1)
    int * status;           // set to KVC_ERR_CUDA by a device wait that ran out (or null)
};

// One sequence of a batch.
struct kvc_attn_seq {
    int q0, nq;             // rows of q
    int nodes;              // paged: nodes of the entry, of which nq are computed (fewer where max_q cuts them)
    int ln;                 // keys
    int k0;                 // packed: first key row
    int slot;               // paged: its slot, or -1
    const int * table;      // paged: its table row
};

__device__ __forceinline__ kvc_attn_seq attn_seq(const kvc_attn_args & a, int s) {
    kvc_attn_seq r;
    r.q0 = min(max(a.cu_q[s], 0), a.n_total);
    r.nodes = max(a.cu_q[s + 1], r.q0) - r.q0;
    r.nq = min(min(r.nodes, a.n_total - r.q0), a.max_q);
    r.k0 = 0;
    r.ln = 0;
    r.slot = -1;
    r.table = nullptr;
    if (a.cu_k) {
        r.k0 = min(max(a.cu_k[s], 0), a.n_keys);
        r.ln = min(max(a.cu_k[s + 1], r.k0), a.n_keys) - r.k0;
    } else {
        const int slot = a.seqs[s];
        if (slot >= 0 && slot < a.n_slots) {
            r.slot = slot;
            r.table = a.table + (size_t)slot * a.max_pages;
            r.ln = min(max(a.seq_len[slot], 0), a.max_pages * a.page);
        }
    }
    return r;
}

// Row number of key j in K and V (and its page and place), or -1.
__device__ __forceinline__ long long attn_row(const kvc_attn_args & a, const kvc_attn_seq & q, int j, int * page,
                                              int * off) {
    if (a.cu_k) return (long long)q.k0 + j;
    const int b = (int)a.by_page.div((uint32_t)j);
    const int p = q.table[b];
    if (p < 0 || p >= a.n_pages) return -1;
    *page = p;
    *off = j - b * a.page;
    return (long long)p * a.page + *off;
}

// Whether node / query i of a sequence sees key j (j < ln). The last rows of a paged sequence are its entry's nodes' own,
// those of nodes that are not computed among them.
__device__ __forceinline__ bool attn_sees(const kvc_attn_args & a, const kvc_attn_seq & q, int i, int j) {
    if (a.cu_k) return !a.causal || j <= i + (q.ln - q.nq);
    const int b = j - (q.ln - q.nodes);
    if (b < 0 || !a.mask) return true;
    return (b >> 5) < a.mask_words && ((a.mask[(size_t)(q.q0 + i) * a.mask_words + (b >> 5)] >> (b & 31)) & 1u);
}

// ---- the split of the keys ---------------------------------------------------
//
// For one (KV head, row block) the key tiles of all sequences that
// have rows in the block are laid end to end, and worker w of W (at most T)
// takes tiles [w*T/W, (w+1)*T/W). Sequences of any lengths then load the workers evenly.
// A worker's stretch meets at most two sequences that it does not cover whole:
// the one it starts inside of (slot 0) and the one it ends inside of (slot 1);
// their partial results go to those slots and are joined afterwards, in the
// workers' order.

// x / d of numbers >= 0, most of them below 2^31 (a 64-bit division takes several times as long).
__device__ __forceinline__ long long attn_quotient(long long x, long long d) {
    return ((x | d) >> 31) == 0 ? (long long)((uint32_t)x / (uint32_t)d) : x / d;
}
// Worker that holds tile x of T.
__device__ __forceinline__ int attn_worker(long long x, long long T, int W) {
    return (int)attn_quotient((x + 1) * W - 1, T);
}

// fn(qb, q, lo, hi, slot) for every piece of worker w's stretch: tiles lo..hi-1
// of a sequence in row block qb; slot -1 where that is all of them. Row blocks
// qb0 .. qb1-1 are laid end to end, each with its sequences. Every warp of a
// CTA takes the same steps. note: write which workers share a sequence, for the
// join.
template <typename F>
__device__ __forceinline__ void attn_walk(const kvc_attn_args & a, int qb0, int qb1, int w, bool note, F && fn) {
    const int lane = threadIdx.x & 31;
    auto tiles = [&](const kvc_attn_seq & q, int qb) {
        if ((long long)qb * a.rb >= (long long)q.nq * a.g || !q.ln) return 0;
        return (int)a.by_tile.div((uint32_t)q.ln - 1u) + 1;
    };
    kvc_attn_seq first{};                                // the first 32 sequences stay in registers
    if (lane < a.n_seqs) first = attn_seq(a, lane);
    long long T = 0;
    for (int s0 = 0; s0 < a.n_seqs; s0 += 32) {
        kvc_attn_seq q = first;
        if (s0) {
            q = kvc_attn_seq{};
            if (s0 + lane < a.n_seqs) q = attn_seq(a, s0 + lane);
        }
        const long long rows = (long long)q.nq * a.g;
        const long long blocks = rows <= 0 || !q.ln ? 0 : min((rows - 1) / a.rb + 1, (long long)qb1) - qb0;
        if (blocks > 0) T += blocks * ((int)a.by_tile.div((uint32_t)q.ln - 1u) + 1);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) T += __shfl_xor_sync(~0u, T, o);
    const int W = (int)min((long long)a.W, T);           // every worker has a tile
    if (w >= W) return;
    const long long from = attn_quotient(w * T, W), to = attn_quotient((w + 1) * T, W);
    long long at = 0;
    for (int qb = qb0; qb < qb1 && at < to; qb++)
        for (int s0 = 0; s0 < a.n_seqs && at < to; s0 += 32) {
            kvc_attn_seq mine = first;
            if (s0) {
                mine = kvc_attn_seq{};
                if (s0 + lane < a.n_seqs) mine = attn_seq(a, s0 + lane);
            }
            const int t = tiles(mine, qb);
            long long p = t;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long u = __shfl_up_sync(~0u, p, o);
                if (lane >= o) p += u;
            }
            const long long end = __shfl_sync(~0u, p, 31);
            p += at - t;
            const bool in = t > 0 && p < to && p + t > from;
            unsigned hit = __ballot_sync(~0u, in);
            if (note && in && p >= from && a.W > 1) {
                int * m = a.meta + ((size_t)qb * a.n_seqs + s0 + lane) * 2;
                m[0] = w;
                m[1] = attn_worker(p + t - 1, T, W);
            }
            while (hit) {
                const int l = __ffs(hit) - 1;
                hit &= hit - 1;
                const long long ps = __shfl_sync(~0u, p, l);
                const int ts = __shfl_sync(~0u, t, l);
                const int lo = (int)(max(from, ps) - ps), hi = (int)(min(to, ps + ts) - ps);
                kvc_attn_seq q;
                q.q0 = __shfl_sync(~0u, mine.q0, l);
                q.nq = __shfl_sync(~0u, mine.nq, l);
                q.nodes = __shfl_sync(~0u, mine.nodes, l);
                q.ln = __shfl_sync(~0u, mine.ln, l);
                q.k0 = __shfl_sync(~0u, mine.k0, l);
                q.slot = __shfl_sync(~0u, mine.slot, l);
                q.table = q.slot < 0 ? nullptr : a.table + (size_t)q.slot * a.max_pages;
                fn(qb, q, lo, hi, lo == 0 && hi == ts ? -1 : (from > ps ? 0 : 1));
            }
            at += end;
        }
}

// Partial results of worker w, slot s: rb sums of d_v, then rb maxima, rb sums.
__device__ __forceinline__ float * attn_part(const kvc_attn_args & a, int qb, int h, int w, int slot) {
    const size_t p = a.n_parts > 1 ? qb : 0;
    return a.part + (((p * a.Hkv + h) * a.W + w) * 2 + slot) * ((size_t)a.rb * (a.dv + 2));
}
// Workspace bytes for `blocks` row blocks: the partial results, then meta.
inline size_t kvc_attn_part_bytes(const kvc_attn_args & a, long long blocks, size_t * meta_at) {
    *meta_at = (size_t)a.n_parts * a.Hkv * a.W * 2 * a.rb * (a.dv + 2) * sizeof(float);
    return a.W > 1 ? *meta_at + (size_t)blocks * a.n_seqs * 2 * sizeof(int) : 0;
}

// Output row (token, head) from its sum and statistics.
__device__ __forceinline__ void attn_store(const kvc_attn_args & a, size_t row, int d, float o, float M, float L) {
    const float v = L > 0.0f ? o / L : (L == 0.0f ? 0.0f : L);       // no key seen: 0; NaN stays NaN
    if (a.q_type == KV_TYPE_F16) reinterpret_cast<__half *>(a.out)[row * a.dv + d] = __float2half_rn(v);
    else reinterpret_cast<float *>(a.out)[row * a.dv + d] = v;
    if (d == 0 && a.lse) a.lse[row] = L == 0.0f ? -INFINITY : M + logf(L);
}

// Joins the partial results and writes rows that no tile reached (attn_simt.cu).
// `overlap`: the kernel that ran lets its successor start early.
int kvc_launch_attn_join(const kvc_attn_args & a, bool overlap, cudaStream_t st);
// The general kernel: every type, d <= 256, any strides (attn_simt.cu).
// Sets the split for it; `whole`: one worker per row block (no partial results).
void kvc_attn_simt_split(kvc_attn_args * a, int sms, bool whole);
int kvc_launch_attn_simt(const kvc_attn_args & a, cudaStream_t st);

// Bytes of a 32-value block.
__host__ __device__ __forceinline__ constexpr int kvc_block_size(int type) {
    return type == KV_TYPE_Q8_0 ? 34 : type == KV_TYPE_Q4_0 ? 18 : type == KV_TYPE_Q4_1 ? 20 : type == KV_TYPE_F16 ? 64 : 128;
}

// ---- stored elements -----------------------------------------------------------
// Element e of a row's head segment at p (block types: segments start on a block).
__device__ __forceinline__ float attn_half(const uint8_t * p) {        // 2-byte aligned
    return __half2float(*reinterpret_cast<const __half *>(p));
}
__device__ __forceinline__ float attn_elem(const uint8_t * p, int type, int e) {
    switch (type) {
    case KV_TYPE_F32: return reinterpret_cast<const float *>(p)[e];
    case KV_TYPE_F16: return attn_half(p + 2 * e);
    case KV_TYPE_Q8_0: {
        const uint8_t * b = p + (e >> 5) * 34;
        return attn_half(b) * (float)(int8_t)b[2 + (e & 31)];
    }
    case KV_TYPE_Q4_0: {
        const uint8_t * b = p + (e >> 5) * 18;
        const int q = b[2 + ((e & 31) >> 1)];
        return attn_half(b) * ((float)((e & 1) ? q >> 4 : q & 15) - 8.0f);
    }
    default: {
        const uint8_t * b = p + (e >> 5) * 20;
        const int q = b[4 + ((e & 31) >> 1)];
        return fmaf(attn_half(b), (float)((e & 1) ? q >> 4 : q & 15), attn_half(b + 2));
    }
    }
}
