// pages.cu — the paged cache's operations (include/kvc-pages.h).
//
// A call that changes tables runs as three small launches: k_plan (one CTA:
// per entry how many pages are shared and how many are new, then the lowest
// free pages, found by scanning ref_count in order), k_move_rows (the row
// copies of all layers, from the old table to the new pages) and k_commit
// (tables, reference counts, lengths). The copies read the old table and only
// write pages that were free, and k_commit runs after them, so no step can
// see a half-made table; the counts change by integer additions, whose order
// does not matter.
#include "serve.h"
#include "tc_sm100.h"

#include "kv-compact-api.h"

#include <limits.h>
#include <stdlib.h>

#include <atomic>
#include <initializer_list>

std::atomic<uint64_t> g_serve_launches{0};

int kvc_serve_device() {
    static std::atomic<int> known[64];               // 0 unknown, else SM count + 1
    const char * e = getenv("KVC_FAULT_INJECT");
    if (e && strcmp(e, "nodev") == 0) return KVC_ERR_NODEV;
    int dev = -1;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) {
        cudaGetLastError();
        return KVC_ERR_NODEV;
    }
    int v = known[dev].load(std::memory_order_relaxed);
    if (v == 0) {
        int major = 0, sms = 0;
        if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess ||
            cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || major < 10 || sms <= 0) {
            cudaGetLastError();
            fprintf(stderr, "[kvc] device %d cannot run sm_100a kernels\n", dev);
            return KVC_ERR_NODEV;
        }
        v = sms + 1;
        known[dev].store(v, std::memory_order_relaxed);
    }
    return v - 1;
}

int kvc_check_cache(const kvc_page_cache * c) {
    if (!c || !c->K || !c->V || !c->page_table || !c->seq_len || !c->ref_count || !c->status) return KVC_ERR_NULL;
    if (c->n_layers <= 0 || c->n_pages <= 0 || c->page_size <= 0 || c->n_slots <= 0 || c->max_pages <= 0 ||
        c->n_head_kv <= 0 || c->d_k <= 0 || c->d_v <= 0)
        return KVC_ERR_DIMS;
    for (int t : {c->k_type, c->v_type})
        if (t != KV_TYPE_F32 && t != KV_TYPE_F16 && t != KV_TYPE_Q4_0 && t != KV_TYPE_Q4_1 && t != KV_TYPE_Q8_0)
            return KVC_ERR_DIMS;
    if (c->n_layers > 65535 || c->n_head_kv > 65535) return KVC_ERR_SHAPE;
    const long long ek = (long long)c->n_head_kv * c->d_k, ev = (long long)c->n_head_kv * c->d_v;
    if (ek > INT_MAX / 4 || ev > INT_MAX / 4 || c->k_row_bytes > INT_MAX || c->v_row_bytes > INT_MAX) return KVC_ERR_SHAPE;
    if (kvc_row_elements(c->k_type, c->k_row_bytes) != ek || kvc_row_bytes(c->k_type, (int)ek) != c->k_row_bytes ||
        kvc_row_elements(c->v_type, c->v_row_bytes) != ev || kvc_row_bytes(c->v_type, (int)ev) != c->v_row_bytes)
        return KVC_ERR_ROWSIZE;
    // row numbers of the pool and of a sequence are 32-bit, with room for the step past the end that scans and grids take
    constexpr int MOST_ROWS = INT_MAX - 65536;
    if ((long long)c->n_pages * c->page_size > MOST_ROWS || (long long)c->max_pages * c->page_size > MOST_ROWS)
        return KVC_ERR_SHAPE;
    // the widest element of the type decides how rows may be addressed
    const uintptr_t ka = c->k_type == KV_TYPE_F32 ? 4 : 2, va = c->v_type == KV_TYPE_F32 ? 4 : 2;
    if ((uintptr_t)c->K % ka || (uintptr_t)c->V % va) return KVC_ERR_SHAPE;
    if (!kvc_words_aligned({c->beta, c->page_table, c->seq_len, c->ref_count, c->status})) return KVC_ERR_SHAPE;
    return KVC_OK;
}

namespace {

enum { OP_RESERVE, OP_FORK, OP_COMPACT, OP_FREE };

// One entry of a planned call, as k_plan leaves it in the workspace.
struct plan_item {
    int whole;     // leading table entries of src that are shared
    int need;      // new pages
    int first;     // index of the first of them in the list of new pages
    int length;    // rows of dst afterwards
    int head;      // rows of src's page `whole` that go to the first new page
    int kept;      // rows that the keep list adds
};

struct plan_ids {
    int n;
    int src[KVC_PAGES_MAX_SEQS];
    int dst[KVC_PAGES_MAX_SEQS];
};

// Workspace: [0] 1 when the call may go on, then the items, then the new pages.
constexpr size_t WS_HEAD = 256;
constexpr size_t WS_ITEMS = WS_HEAD + KVC_PAGES_MAX_SEQS * sizeof(plan_item);

struct cache_dev {
    uint8_t * K;
    uint8_t * V;
    float * beta;
    int * table;
    int * seq_len;
    int * ref;
    int * status;
    int n_layers, n_pages, page, max_pages, H;
    kvc_divisor by_page;
};

cache_dev on_device(const kvc_page_cache * c) {
    return {c->K,        c->V,       c->beta,      c->page_table, c->seq_len,
            c->ref_count, c->status, c->n_layers,  c->n_pages,    c->page_size,
            c->max_pages, c->n_head_kv, kvc_make_divisor((uint32_t)c->page_size)};
}

// Pages of `rows` rows (rows + page may pass 2^31).
__device__ __forceinline__ int pages_of(int rows, kvc_divisor page) { return rows > 0 ? (int)page.div((uint32_t)rows - 1u) + 1 : 0; }

constexpr int PLAN_THREADS = 1024;
constexpr int PLAN_PER = 16;          // counts per thread and scan step

template <typename T>
__device__ __forceinline__ T warp_scan(T v, int lane) {              // inclusive
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T u = __shfl_up_sync(~0u, v, o);
        if (lane >= o) v += u;
    }
    return v;
}

// Exclusive scan over the CTA; every thread gets its prefix and the total.
template <typename T>
__device__ T block_scan(T v, T * sums, T * total) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const T inc = warp_scan(v, lane);
    __syncthreads();
    if (lane == 31) sums[w] = inc;
    __syncthreads();
    if (w == 0) sums[lane] = warp_scan(sums[lane], lane);
    __syncthreads();
    *total = sums[31];
    return inc - v + (w ? sums[w - 1] : 0);
}

// One CTA. Bound by latency: one pass over the entries, then the scan for free
// pages, 16 counts per thread and step (four 16-byte loads in flight), which
// stops as soon as enough were found.
__global__ void __launch_bounds__(PLAN_THREADS) k_plan(cache_dev c, const __grid_constant__ plan_ids ids, int op,
                                                       const int * __restrict__ base, const int * __restrict__ keep_n,
                                                       const __grid_constant__ plan_ids counts, int keep_ld,
                                                       int * __restrict__ ws) {
    __shared__ int sums[32];
    __shared__ long long needs[32];
    const int t = threadIdx.x;
    bool bad = false;
    plan_item it{};
    if (t < ids.n) {
        const int cap = c.max_pages * c.page;
        const int len = min(max(c.seq_len[ids.src[t]], 0), cap);
        long long length = len;
        if (op == OP_RESERVE) {
            it.whole = pages_of(len, c.by_page);
            length = (long long)len + counts.src[t];
        } else if (op == OP_FORK) {
            it.whole = (int)c.by_page.div((uint32_t)len);
            it.head = len - it.whole * c.page;
        } else {
            const int b = min(max(base[t], 0), len);
            it.kept = min(max(keep_n[t], 0), keep_ld);
            it.whole = (int)c.by_page.div((uint32_t)b);
            it.head = b - it.whole * c.page;
            length = (long long)b + it.kept;
        }
        if (length > cap) {
            bad = true;
        } else {
            it.length = (int)length;
            it.need = max(pages_of(it.length, c.by_page) - it.whole, 0);
        }
    }
    const bool too_long = __syncthreads_or(bad);
    long long total;                                     // of all entries: up to 256 times 2^31
    it.first = (int)block_scan<long long>(t < ids.n ? it.need : 0, needs, &total);
    plan_item * items = reinterpret_cast<plan_item *>(reinterpret_cast<char *>(ws) + WS_HEAD);
    if (t < ids.n) items[t] = it;
    int * fresh = reinterpret_cast<int *>(reinterpret_cast<char *>(ws) + WS_ITEMS);
    int found = 0;
    if (!too_long && total <= c.n_pages) {
        const bool wide = ((uintptr_t)c.ref & 15) == 0;
        for (int at = 0; found < total && at < c.n_pages; at += PLAN_THREADS * PLAN_PER) {
            const int p0 = at + t * PLAN_PER;
            unsigned free_bits = 0;
            if (wide && p0 + PLAN_PER <= c.n_pages) {
                int4 r[PLAN_PER / 4];
#pragma unroll
                for (int i = 0; i < PLAN_PER / 4; i++) r[i] = reinterpret_cast<const int4 *>(c.ref + p0)[i];
#pragma unroll
                for (int i = 0; i < PLAN_PER / 4; i++) {
                    free_bits |= (r[i].x == 0 ? 1u : 0u) << (4 * i);
                    free_bits |= (r[i].y == 0 ? 2u : 0u) << (4 * i);
                    free_bits |= (r[i].z == 0 ? 4u : 0u) << (4 * i);
                    free_bits |= (r[i].w == 0 ? 8u : 0u) << (4 * i);
                }
            } else {
                for (int i = 0; i < PLAN_PER; i++)
                    if (p0 + i < c.n_pages && c.ref[p0 + i] == 0) free_bits |= 1u << i;
            }
            int step;
            int k = found + block_scan(__popc(free_bits), sums, &step);
            while (free_bits && k < total) {
                const int i = __ffs(free_bits) - 1;
                free_bits &= free_bits - 1;
                fresh[k++] = p0 + i;
            }
            found += step;
        }
    }
    if (t == 0) {
        const bool ok = !too_long && found >= total;
        ws[0] = ok;
        if (!ok) *c.status = too_long ? KVC_ERR_SHAPE : KVC_ERR_OOM;
    }
}

// Table entries, counts and lengths of every entry; one thread per entry of a
// table row. Entry (dst, col) is read and written by its own thread alone, and
// a source row is nobody's destination but its own, so nothing races.
__global__ void __launch_bounds__(256) k_commit(cache_dev c, const __grid_constant__ plan_ids ids, int op,
                                                const int * __restrict__ ws) {
    const int i = blockIdx.y;
    if (op != OP_FREE && ws[0] == 0) return;
    const int col = blockIdx.x * 256 + threadIdx.x;
    plan_item it{};
    if (op != OP_FREE) it = reinterpret_cast<const plan_item *>(reinterpret_cast<const char *>(ws) + WS_HEAD)[i];
    if (col == 0) c.seq_len[ids.dst[i]] = it.length;
    if (col >= c.max_pages) return;
    const int * fresh = reinterpret_cast<const int *>(reinterpret_cast<const char *>(ws) + WS_ITEMS);
    int * at = c.table + (size_t)ids.dst[i] * c.max_pages + col;
    const int old = *at;
    int now = -1;
    if (col < it.whole) now = c.table[(size_t)ids.src[i] * c.max_pages + col];
    else if (col < it.whole + it.need) now = fresh[it.first + col - it.whole];
    if (old == now) return;
    if (old >= 0 && old < c.n_pages) atomicAdd(c.ref + old, -1);
    if (now >= 0 && now < c.n_pages) atomicAdd(c.ref + now, 1);
    *at = now;
}

// ---- row movement -----------------------------------------------------------
//
// Rows of whole 16-byte pieces go by bulk copies (k_move_bulk), others by
// k_move_rows: a CTA takes up to MOVE_ROWS rows of one layer (fewer where there
// are not enough to fill the machine), looks their places up once into shared
// memory, then all threads copy the K bytes and the V bytes in the widest
// pieces that the row sizes and base addresses allow, MOVE_DEPTH loads in
// flight per thread. 6,400 rows of 12 layers, 1,088 bytes of K and of V each:
// k_move_rows 66 us (74 with 8 loads in flight), k_move_bulk 54 us.
constexpr int MOVE_ROWS = 32;
constexpr int MOVE_THREADS = 256;
constexpr int MOVE_DEPTH = 4;
constexpr int BULK_BYTES = 9 * 1024, BULK_MOST = 200 * 1024;
constexpr uint32_t POLLS = 1u << 22;  // bound of every wait

__device__ __forceinline__ void bulk_load(void * dst, const uint8_t * src, uint32_t bytes, uint64_t * bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 :: "r"(kvc_tc::smem_u32(dst)), "l"(src), "r"(bytes), "r"(kvc_tc::smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void bulk_store(uint8_t * dst, const void * src, uint32_t bytes) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;"
                 :: "l"(dst), "r"(kvc_tc::smem_u32(src)), "r"(bytes) : "memory");
}

enum { MV_PAGES, MV_FORK, MV_COMPACT, MV_WRITE, MV_READ };

struct move_args {
    cache_dev c;
    int mode;
    long long krb, vrb;             // bytes per row
    int per;                        // rows of a CTA and step, <= MOVE_ROWS
    int rows;                       // rows per entry (MV_PAGES, MV_FORK, MV_COMPACT) or in all (MV_WRITE / MV_READ)
    kvc_divisor kdiv, vdiv;         // pieces per row
    const int * ws;
    const int * src_pages;          // MV_PAGES
    const int * dst_pages;
    const int * keep;               // MV_COMPACT
    int keep_ld;
    long long keep_layer;
    int n;
    uint8_t * k_rows;               // packed rows (MV_WRITE / MV_READ), or replacements (MV_COMPACT: V and beta)
    uint8_t * v_rows;
    float * b_rows;
};

template <typename T>
__device__ __forceinline__ void copy_pieces(const long long * src, const long long * dst, const uint8_t * from,
                                            uint8_t * to, kvc_divisor per, long long rb, int rows) {
    const uint32_t n = (uint32_t)rows * per.d;
    for (uint32_t p0 = threadIdx.x; p0 < n; p0 += MOVE_THREADS * MOVE_DEPTH) {
        T v[MOVE_DEPTH];
        long long out[MOVE_DEPTH];
#pragma unroll
        for (int i = 0; i < MOVE_DEPTH; i++) {
            const uint32_t p = p0 + i * MOVE_THREADS;
            out[i] = -1;
            if (p < n) {
                const uint32_t r = per.div(p), q = p - r * per.d;
                if (src[r] >= 0 && dst[r] >= 0) {
                    v[i] = *reinterpret_cast<const T *>(from + src[r] * rb + (long long)q * sizeof(T));
                    out[i] = dst[r] * rb + (long long)q * sizeof(T);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < MOVE_DEPTH; i++)
            if (out[i] >= 0) *reinterpret_cast<T *>(to + out[i]) = v[i];
    }
}

// Row numbers count rows of one layer's pool, or of a packed array; -1 = none, vsrc <= -2: row -2 - vsrc of the
// replacements.
struct row_place {
    long long src, dst, vsrc;
};

// What a CTA moves: the rows of one layer and entry.
struct move_part {
    plan_item it;
    int layer, item, count;
    const uint8_t * k_from;
    const uint8_t * v_from;
    uint8_t * k_to;
    uint8_t * v_to;
    const uint8_t * new_v;          // the entry's replacement rows, or null
};

__device__ __forceinline__ bool move_start(const move_args & a, int layer, int item, move_part * b) {
    const cache_dev & c = a.c;
    const bool planned = a.mode == MV_FORK || a.mode == MV_COMPACT;
    if (planned && a.ws[0] == 0) return false;
    const long long pool = (long long)c.n_pages * c.page;
    b->it = plan_item{};
    b->layer = layer;
    b->item = item;
    b->count = a.rows;
    if (planned) {
        b->it = reinterpret_cast<const plan_item *>(reinterpret_cast<const char *>(a.ws) + WS_HEAD)[item];
        b->count = b->it.head + b->it.kept;
    }
    b->k_from = b->k_to = c.K + (long long)layer * pool * a.krb;
    b->v_from = b->v_to = c.V + (long long)layer * pool * a.vrb;
    if (a.mode == MV_WRITE) {
        b->k_from = a.k_rows + (long long)layer * a.rows * a.krb;
        b->v_from = a.v_rows + (long long)layer * a.rows * a.vrb;
    } else if (a.mode == MV_READ) {
        b->k_to = a.k_rows + (long long)layer * a.rows * a.krb;
        b->v_to = a.v_rows + (long long)layer * a.rows * a.vrb;
    }
    b->new_v = a.mode == MV_COMPACT && a.v_rows ? a.v_rows + ((long long)layer * a.n + item) * a.keep_ld * a.vrb : nullptr;
    return true;
}

// Where row j of the part is read and written.
__device__ __forceinline__ row_place place_row(const move_args & a, const plan_ids & ids, const plan_ids & span,
                                               const move_part & b, int j) {
    const cache_dev & c = a.c;
    const plan_item & it = b.it;
    const int layer = b.layer, item = b.item;
    const int * fresh = reinterpret_cast<const int *>(reinterpret_cast<const char *>(a.ws) + WS_ITEMS);
    row_place w{-1, -1, -1};
    bool replaced = false;
    if (a.mode == MV_PAGES) {
        const int e = (int)c.by_page.div(j), off = j - e * c.page;
        const int ps = a.src_pages[e], pd = a.dst_pages[e];
        if (ps >= 0 && ps < c.n_pages && pd >= 0 && pd < c.n_pages && ps != pd) {
            w.src = (long long)ps * c.page + off;
            w.dst = (long long)pd * c.page + off;
        }
        w.vsrc = w.src;
    } else if (a.mode == MV_FORK || a.mode == MV_COMPACT) {
        const int * table = c.table + (size_t)ids.src[item] * c.max_pages;
        int row;
        if (j < it.head) {
            row = it.whole * c.page + j;
        } else {
            row = a.keep[(long long)layer * a.keep_layer + (long long)item * a.keep_ld + (j - it.head)];
            replaced = true;
        }
        const int len = min(max(c.seq_len[ids.src[item]], 0), c.max_pages * c.page);
        if (row >= 0 && row < len) {
            const int e = (int)c.by_page.div(row), p = table[e];
            if (p >= 0 && p < c.n_pages) w.src = (long long)p * c.page + (row - e * c.page);
        }
        const int e = (int)c.by_page.div(j);
        w.dst = (long long)fresh[it.first + e] * c.page + (j - e * c.page);
        w.vsrc = w.src;
        if (b.new_v && replaced && w.src >= 0) w.vsrc = -2 - (j - it.head);      // a replacement row
    } else {
        // packed rows: the entry that row j belongs to (few entries: a linear walk)
        int e = 0, at = 0;
        while (e < ids.n - 1 && j >= at + span.dst[e]) at += span.dst[e++];
        const int row = span.src[e] + (j - at);
        const int slot = ids.src[e];
        const int len = min(max(c.seq_len[slot], 0), c.max_pages * c.page);
        long long there = -1;
        if (row < len) {
            const int at_page = (int)c.by_page.div(row), p = c.table[(size_t)slot * c.max_pages + at_page];
            if (p >= 0 && p < c.n_pages) {
                there = (long long)p * c.page + (row - at_page * c.page);
                if (a.mode == MV_WRITE && c.ref[p] > 1) {
                    there = -1;
                    *c.status = KVC_ERR_DIMS;
                }
            }
        }
        w.src = a.mode == MV_WRITE ? j : there;
        w.dst = a.mode == MV_WRITE ? there : j;
        w.vsrc = w.src;
    }
    return w;
}

// beta of rows j0 .. j0+rows-1, whose places lie in shared memory.
__device__ __forceinline__ void move_beta(const move_args & a, const move_part & b, const long long * s_src,
                                          const long long * s_dst, int j0, int rows) {
    const cache_dev & c = a.c;
    const plan_item & it = b.it;
    const int layer = b.layer, item = b.item;
    // beta: [page][head][row in page]; neighbouring threads take
    // neighbouring rows, which lie side by side in a page
    if (c.beta && (a.mode < MV_WRITE || a.b_rows)) {
        float * pool_b = c.beta + (long long)layer * c.n_pages * c.page * c.H;
        for (int p = threadIdx.x; p < rows * c.H; p += blockDim.x) {
            const int h = p / rows, r = p - h * rows;
            const long long src = s_src[r], dst = s_dst[r];
            if (dst < 0) continue;
            auto place = [&](long long row) {
                const uint32_t pg = c.by_page.div((uint32_t)row);
                return ((long long)pg * c.H + h) * c.page + (row - (long long)pg * c.page);
            };
            if (a.mode == MV_WRITE) {
                pool_b[place(dst)] = a.b_rows[((long long)layer * c.H + h) * a.rows + src];
            } else if (a.mode == MV_READ) {
                if (src >= 0) a.b_rows[((long long)layer * c.H + h) * a.rows + dst] = pool_b[place(src)];
            } else {
                const int kept = j0 + r - it.head;
                if (src < 0) continue;
                if (a.mode == MV_COMPACT && a.b_rows && kept >= 0)
                    pool_b[place(dst)] = a.b_rows[(((long long)layer * a.n + item) * c.H + h) * a.keep_ld + kept];
                else
                    pool_b[place(dst)] = pool_b[place(src)];
            }
        }
    }
}

template <typename TK, typename TV>
__global__ void __launch_bounds__(MOVE_THREADS) k_move_rows(const __grid_constant__ move_args a,
                                                            const __grid_constant__ plan_ids ids,
                                                            const __grid_constant__ plan_ids span) {
    __shared__ long long s_src[MOVE_ROWS], s_dst[MOVE_ROWS], s_vsrc[MOVE_ROWS];
    move_part b;
    if (!move_start(a, blockIdx.y, blockIdx.z, &b)) return;
    for (long long j0 = (long long)blockIdx.x * a.per; j0 < b.count; j0 += (long long)gridDim.x * a.per) {
        const int rows = (int)min((long long)a.per, b.count - j0);
        __syncthreads();
        if (threadIdx.x < rows) {
            const row_place w = place_row(a, ids, span, b, (int)j0 + threadIdx.x);
            s_src[threadIdx.x] = w.src;
            s_dst[threadIdx.x] = w.dst;
            s_vsrc[threadIdx.x] = w.vsrc;
        }
        __syncthreads();
        if (a.mode < MV_WRITE || a.k_rows) copy_pieces<TK>(s_src, s_dst, b.k_from, b.k_to, a.kdiv, a.krb, rows);
        if (!b.new_v) {
            if (a.mode < MV_WRITE || a.v_rows) copy_pieces<TV>(s_src, s_dst, b.v_from, b.v_to, a.vdiv, a.vrb, rows);
        } else {
            const uint32_t n = (uint32_t)rows * a.vdiv.d;
            for (uint32_t p0 = threadIdx.x; p0 < n; p0 += MOVE_THREADS * MOVE_DEPTH) {
                TV v[MOVE_DEPTH];
                long long out[MOVE_DEPTH];
#pragma unroll
                for (int i = 0; i < MOVE_DEPTH; i++) {
                    const uint32_t p = p0 + i * MOVE_THREADS;
                    out[i] = -1;
                    if (p < n) {
                        const uint32_t r = a.vdiv.div(p), q = p - r * a.vdiv.d;
                        const long long vs = s_vsrc[r];
                        if (vs != -1) {
                            const uint8_t * f = vs >= 0 ? b.v_from + vs * a.vrb : b.new_v + (-2 - vs) * a.vrb;
                            v[i] = *reinterpret_cast<const TV *>(f + (long long)q * sizeof(TV));
                            out[i] = s_dst[r] * a.vrb + (long long)q * sizeof(TV);
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < MOVE_DEPTH; i++)
                    if (out[i] >= 0) *reinterpret_cast<TV *>(b.v_to + out[i]) = v[i];
            }
        }
        move_beta(a, b, s_src, s_dst, (int)j0, rows);
    }
}

// Rows of whole 16-byte pieces, each carried by two bulk copies: one warp per
// CTA, a row per lane, its K and V through shared memory of its own. A lane
// issues its loads, moves beta meanwhile with the others, and stores when all
// have landed; the CTAs of an SM (about 20) overlap one another's loads and
// stores. Bound by HBM: the copy above at 6.2 TB/s read and written, 0.95 of
// the measured copy rate; 6,540 kept rows of 12 layers 64 us (k_move_rows 80).
// 18 KB of rows per CTA 54.6 / 64.7 us, 36 KB 58 / 74, 72 KB 75 / 92. 64 MB of
// rows of 64, 128, 256 and 1,024 bytes: 79, 55, 43 and 43 us (172, 108, 68, 47).
__global__ void __launch_bounds__(32) k_move_bulk(const __grid_constant__ move_args a, const __grid_constant__ plan_ids ids,
                                                  const __grid_constant__ plan_ids span) {
    using namespace kvc_tc;
    extern __shared__ __align__(128) uint8_t slots[];
    __shared__ long long s_src[MOVE_ROWS], s_dst[MOVE_ROWS];
    __shared__ uint64_t bar;
    const int lane = threadIdx.x;
    move_part b;
    if (!move_start(a, blockIdx.y, blockIdx.z, &b)) return;
    if (lane == 0) {
        mbar_init(&bar, 32);
        mbar_init_fence();
    }
    __syncwarp();
    const uint32_t krb = (uint32_t)a.krb, vrb = (uint32_t)a.vrb;
    uint8_t * slot = slots + (size_t)min(lane, a.per - 1) * (krb + vrb);
    uint32_t phase = 0;
    for (long long j0 = (long long)blockIdx.x * a.per; j0 < b.count; j0 += (long long)gridDim.x * a.per) {
        const int rows = (int)min((long long)a.per, b.count - j0);
        row_place w{-1, -1, -1};
        if (lane < rows) w = place_row(a, ids, span, b, (int)j0 + lane);
        const bool k = w.src >= 0 && w.dst >= 0 && (a.mode < MV_WRITE || a.k_rows);
        const bool v = w.vsrc != -1 && w.dst >= 0 && (a.mode < MV_WRITE || a.v_rows);
        asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");     // the slot's stores have read it
        mbar_arrive_expect_tx(&bar, (k ? krb : 0u) + (v ? vrb : 0u));
        if (k) bulk_load(slot, b.k_from + w.src * a.krb, krb, &bar);
        if (v) bulk_load(slot + krb, w.vsrc >= 0 ? b.v_from + w.vsrc * a.vrb : b.new_v + (-2 - w.vsrc) * a.vrb, vrb, &bar);
        __syncwarp();
        if (lane < rows) {
            s_src[lane] = w.src;
            s_dst[lane] = w.dst;
        }
        __syncwarp();
        move_beta(a, b, s_src, s_dst, (int)j0, rows);
        if (!mbar_wait(&bar, phase, POLLS)) {
            *a.c.status = KVC_ERR_CUDA;
            mbar_wait(&bar, phase, POLLS);
            break;
        }
        phase ^= 1;
        if (k) bulk_store(b.k_to + w.dst * a.krb, slot, krb);
        if (v) bulk_store(b.v_to + w.dst * a.vrb, slot + krb, vrb);
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
    asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}

// The widest piece (16, 8, 4 or 2 bytes) that divides the row size and every base address.
int piece(size_t rb, std::initializer_list<const void *> bases) {
    uintptr_t m = rb;
    for (const void * b : bases) m |= (uintptr_t)b;
    return (m & 15) == 0 ? 16 : (m & 7) == 0 ? 8 : (m & 3) == 0 ? 4 : (m & 1) == 0 ? 2 : 1;
}

template <typename TK>
int launch_move_v(const move_args & a, int vp, const plan_ids & ids, const plan_ids & span, dim3 grid, cudaStream_t st) {
    switch (vp) {
    case 16: k_move_rows<TK, int4><<<grid, MOVE_THREADS, 0, st>>>(a, ids, span); break;
    case 8: k_move_rows<TK, int2><<<grid, MOVE_THREADS, 0, st>>>(a, ids, span); break;
    case 4: k_move_rows<TK, int><<<grid, MOVE_THREADS, 0, st>>>(a, ids, span); break;
    case 2: k_move_rows<TK, short><<<grid, MOVE_THREADS, 0, st>>>(a, ids, span); break;
    default: k_move_rows<TK, char><<<grid, MOVE_THREADS, 0, st>>>(a, ids, span); break;
    }
    g_serve_launches++;
    KVC_CUDA(cudaGetLastError());
    return KVC_OK;
}

// most: rows of the longest entry. Enough CTAs to fill the machine several
// times over, each looping when there are more rows.
int launch_move(move_args & a, const kvc_page_cache * c, const plan_ids & ids, const plan_ids & span, int items,
                long long most, int sms, cudaStream_t st) {
    if (most <= 0 || items <= 0) return KVC_OK;
    const bool packed = a.mode == MV_WRITE || a.mode == MV_READ;
    const int kp = piece(c->k_row_bytes, {c->K, packed ? a.k_rows : nullptr});
    const int vp = piece(c->v_row_bytes, {c->V, a.v_rows});
    a.krb = (long long)c->k_row_bytes;
    a.vrb = (long long)c->v_row_bytes;
    a.kdiv = kvc_make_divisor((uint32_t)(c->k_row_bytes / kp));
    a.vdiv = kvc_make_divisor((uint32_t)(c->v_row_bytes / vp));
    const long long both = a.krb + a.vrb;
    if (kp == 16 && vp == 16 && both <= BULK_MOST) {
        const int fit = (int)(BULK_BYTES / both);
        a.per = fit < 1 ? 1 : fit > MOVE_ROWS ? MOVE_ROWS : fit;
        while (a.per > 2 && (most + a.per - 1) / a.per * items * c->n_layers < 4LL * sms) a.per /= 2;
        const long long tiles = (most + a.per - 1) / a.per;
        const dim3 grid((unsigned)(tiles < 1 << 20 ? tiles : 1 << 20), (unsigned)c->n_layers, (unsigned)items);
        const int sm = (int)(a.per * both);
        static std::atomic<bool> set[64];
        int dev = 0;
        KVC_CUDA(cudaGetDevice(&dev));
        if (!set[dev & 63].load(std::memory_order_relaxed)) {
            KVC_CUDA(cudaFuncSetAttribute(k_move_bulk, cudaFuncAttributeMaxDynamicSharedMemorySize, BULK_MOST));
            set[dev & 63].store(true, std::memory_order_relaxed);
        }
        k_move_bulk<<<grid, 32, sm, st>>>(a, ids, span);
        g_serve_launches++;
        KVC_CUDA(cudaGetLastError());
        return KVC_OK;
    }
    // a quarter of the rows per CTA, and again, while there are fewer CTAs than two per SM
    a.per = MOVE_ROWS;
    while (a.per > 2 && (most + a.per - 1) / a.per * items * c->n_layers < 2LL * sms) a.per /= 4;
    const long long tiles = (most + a.per - 1) / a.per;
    const long long want = (16LL * sms * 8 + (long long)items * c->n_layers - 1) / ((long long)items * c->n_layers);
    const dim3 grid((unsigned)(tiles < want ? tiles : want), (unsigned)c->n_layers, (unsigned)items);
    switch (kp) {
    case 16: return launch_move_v<int4>(a, vp, ids, span, grid, st);
    case 8: return launch_move_v<int2>(a, vp, ids, span, grid, st);
    case 4: return launch_move_v<int>(a, vp, ids, span, grid, st);
    case 2: return launch_move_v<short>(a, vp, ids, span, grid, st);
    default: return launch_move_v<char>(a, vp, ids, span, grid, st);
    }
}

int check_ids(const kvc_page_cache * c, const int * src, const int * dst, int n, plan_ids * ids) {
    if (n < 0 || n > KVC_PAGES_MAX_SEQS) return KVC_ERR_DIMS;
    if (n > 0 && (!src || !dst)) return KVC_ERR_NULL;
    ids->n = n;
    for (int i = 0; i < n; i++) {
        if (src[i] < 0 || src[i] >= c->n_slots || dst[i] < 0 || dst[i] >= c->n_slots) return KVC_ERR_DIMS;
        ids->src[i] = src[i];
        ids->dst[i] = dst[i];
    }
    for (int i = 0; i < n; i++)
        for (int j = 0; j < n; j++)
            if (i != j && (dst[i] == dst[j] || dst[i] == src[j])) return KVC_ERR_DIMS;
    return KVC_OK;
}

int check_ws(const kvc_page_cache * c, const void * ws, size_t bytes) {
    if (!ws) return KVC_ERR_NULL;
    if (bytes < kvc_pages_workspace(c) || ((uintptr_t)ws & 15)) return KVC_ERR_SHAPE;
    return KVC_OK;
}

int launch_commit(const cache_dev & c, const plan_ids & ids, int op, const int * ws, cudaStream_t st) {
    k_commit<<<dim3((c.max_pages + 255) / 256, ids.n), 256, 0, st>>>(c, ids, op, ws);
    g_serve_launches++;
    KVC_CUDA(cudaGetLastError());
    return KVC_OK;
}

int launch_plan(const cache_dev & c, const plan_ids & ids, int op, const int * base, const int * keep_n,
                const plan_ids & counts, int keep_ld, int * ws, cudaStream_t st) {
    k_plan<<<1, PLAN_THREADS, 0, st>>>(c, ids, op, base, keep_n, counts, keep_ld, ws);
    g_serve_launches++;
    KVC_CUDA(cudaGetLastError());
    return KVC_OK;
}

// Rows of the packed forms: starts and counts of the entries, their sum.
int check_spans(const kvc_page_cache * c, const int * seqs, const int * first, const int * count, int n, plan_ids * ids,
                plan_ids * span, long long * total) {
    if (n < 0 || n > KVC_PAGES_MAX_SEQS) return KVC_ERR_DIMS;
    if (n > 0 && (!seqs || !first || !count)) return KVC_ERR_NULL;
    ids->n = span->n = n;
    *total = 0;
    for (int i = 0; i < n; i++) {
        if (seqs[i] < 0 || seqs[i] >= c->n_slots || first[i] < 0 || count[i] < 0 ||
            (long long)first[i] + count[i] > INT_MAX)
            return KVC_ERR_DIMS;
        ids->src[i] = seqs[i];
        span->src[i] = first[i];
        span->dst[i] = count[i];
        *total += count[i];
    }
    return *total > INT_MAX - 65536 ? KVC_ERR_SHAPE : KVC_OK;
}

int packed_move(int mode, const kvc_page_cache * cache, const int * seqs, const int * first, const int * count, int n,
                uint8_t * k_rows, uint8_t * v_rows, float * b_rows, cudaStream_t st) {
    int rc = kvc_check_cache(cache);
    if (rc) return rc;
    plan_ids ids, span;
    long long total;
    if ((rc = check_spans(cache, seqs, first, count, n, &ids, &span, &total))) return rc;
    if (b_rows && !cache->beta) return KVC_ERR_NULL;
    if (!kvc_words_aligned({b_rows})) return KVC_ERR_SHAPE;
    if (mode == MV_WRITE)               // two entries that write one row would race
        for (int i = 0; i < n; i++)
            for (int j = 0; j < i; j++)
                if (seqs[i] == seqs[j] && count[i] > 0 && count[j] > 0 && first[i] < first[j] + count[j] &&
                    first[j] < first[i] + count[i])
                    return KVC_ERR_DIMS;
    const int sms = kvc_serve_device();
    if (sms < 0) return sms;
    if (!k_rows && !v_rows && !b_rows) return KVC_OK;
    move_args a{};
    a.c = on_device(cache);
    a.mode = mode;
    a.rows = (int)total;
    a.k_rows = k_rows;
    a.v_rows = v_rows;
    a.b_rows = b_rows;
    a.n = n;
    return launch_move(a, cache, ids, span, 1, total, sms, st);
}

}  // namespace

extern "C" {

KVC_EXPORT size_t kvc_pages_workspace(const kvc_page_cache * cache) {
    if (kvc_check_cache(cache)) return 0;
    return (WS_ITEMS + (size_t)cache->n_pages * 4 + 255) & ~(size_t)255;
}

KVC_EXPORT int kvc_pages_reserve(const kvc_page_cache * cache, const int * seqs, const int * add, int n, void * ws,
                                 size_t ws_bytes, void * stream) {
    int rc = kvc_check_cache(cache);
    if (rc) return rc;
    plan_ids ids, counts{};
    if ((rc = check_ids(cache, seqs, seqs, n, &ids))) return rc;
    if (n > 0 && !add) return KVC_ERR_NULL;
    for (int i = 0; i < n; i++) {
        if (add[i] < 0) return KVC_ERR_DIMS;
        counts.src[i] = add[i];
    }
    if ((rc = check_ws(cache, ws, ws_bytes))) return rc;
    const int sms = kvc_serve_device();
    if (sms < 0) return sms;
    if (n == 0) return KVC_OK;
    const cache_dev c = on_device(cache);
    if ((rc = launch_plan(c, ids, OP_RESERVE, nullptr, nullptr, counts, 0, (int *)ws, (cudaStream_t)stream))) return rc;
    return launch_commit(c, ids, OP_RESERVE, (const int *)ws, (cudaStream_t)stream);
}

KVC_EXPORT int kvc_pages_write(const kvc_page_cache * cache, const int * seqs, const int * first, const int * count,
                               int n, const uint8_t * k_rows, const uint8_t * v_rows, const float * beta_rows,
                               void * stream) {
    return packed_move(MV_WRITE, cache, seqs, first, count, n, const_cast<uint8_t *>(k_rows),
                       const_cast<uint8_t *>(v_rows), const_cast<float *>(beta_rows), (cudaStream_t)stream);
}

KVC_EXPORT int kvc_pages_read(const kvc_page_cache * cache, const int * seqs, const int * first, const int * count,
                              int n, uint8_t * k_rows, uint8_t * v_rows, float * beta_rows, void * stream) {
    return packed_move(MV_READ, cache, seqs, first, count, n, k_rows, v_rows, beta_rows, (cudaStream_t)stream);
}

KVC_EXPORT int kvc_pages_copy(const kvc_page_cache * cache, const int * src, const int * dst, int n, void * stream) {
    int rc = kvc_check_cache(cache);
    if (rc) return rc;
    if (n < 0 || (long long)n * cache->page_size > INT_MAX - 65536) return KVC_ERR_DIMS;
    if (n > 0 && (!src || !dst)) return KVC_ERR_NULL;
    if (!kvc_words_aligned({src, dst})) return KVC_ERR_SHAPE;
    const int sms = kvc_serve_device();
    if (sms < 0) return sms;
    move_args a{};
    a.c = on_device(cache);
    a.mode = MV_PAGES;
    a.rows = n * cache->page_size;
    a.src_pages = src;
    a.dst_pages = dst;
    static const plan_ids none{};
    return launch_move(a, cache, none, none, 1, a.rows, sms, (cudaStream_t)stream);
}

KVC_EXPORT int kvc_pages_fork(const kvc_page_cache * cache, const int * src, const int * dst, int n, void * ws,
                              size_t ws_bytes, void * stream) {
    int rc = kvc_check_cache(cache);
    if (rc) return rc;
    plan_ids ids;
    if ((rc = check_ids(cache, src, dst, n, &ids))) return rc;
    for (int i = 0; i < n; i++)
        if (src[i] == dst[i]) return KVC_ERR_DIMS;
    if ((rc = check_ws(cache, ws, ws_bytes))) return rc;
    const int sms = kvc_serve_device();
    if (sms < 0) return sms;
    if (n == 0) return KVC_OK;
    const cache_dev c = on_device(cache);
    cudaStream_t st = (cudaStream_t)stream;
    static const plan_ids none{};
    if ((rc = launch_plan(c, ids, OP_FORK, nullptr, nullptr, none, 0, (int *)ws, st))) return rc;
    move_args a{};
    a.c = c;
    a.mode = MV_FORK;
    a.n = n;
    a.ws = (const int *)ws;
    if ((rc = launch_move(a, cache, ids, none, n, cache->page_size - 1, sms, st))) return rc;
    return launch_commit(c, ids, OP_FORK, (const int *)ws, st);
}

KVC_EXPORT int kvc_pages_compact(const kvc_page_cache * cache, const int * src, const int * dst, int n,
                                 const int * base, const int * keep_n, const int * keep, int keep_ld,
                                 size_t keep_layer_stride, const uint8_t * v_rows, const float * beta_rows, void * ws,
                                 size_t ws_bytes, void * stream) {
    int rc = kvc_check_cache(cache);
    if (rc) return rc;
    plan_ids ids;
    if ((rc = check_ids(cache, src, dst, n, &ids))) return rc;
    if (keep_ld < 0) return KVC_ERR_DIMS;
    if (n > 0 && (!base || !keep_n || (!keep && keep_ld > 0))) return KVC_ERR_NULL;
    if (beta_rows && !cache->beta) return KVC_ERR_NULL;
    if (!kvc_words_aligned({base, keep_n, keep, beta_rows})) return KVC_ERR_SHAPE;
    if ((rc = check_ws(cache, ws, ws_bytes))) return rc;
    const int sms = kvc_serve_device();
    if (sms < 0) return sms;
    if (n == 0) return KVC_OK;
    const cache_dev c = on_device(cache);
    cudaStream_t st = (cudaStream_t)stream;
    static const plan_ids none{};
    if ((rc = launch_plan(c, ids, OP_COMPACT, base, keep_n, none, keep_ld, (int *)ws, st))) return rc;
    move_args a{};
    a.c = c;
    a.mode = MV_COMPACT;
    a.n = n;
    a.ws = (const int *)ws;
    a.keep = keep;
    a.keep_ld = keep_ld;
    a.keep_layer = (long long)keep_layer_stride;
    a.v_rows = const_cast<uint8_t *>(v_rows);
    a.b_rows = const_cast<float *>(beta_rows);
    const long long most = (long long)cache->page_size - 1 + keep_ld;
    if ((rc = launch_move(a, cache, ids, none, n, most, sms, st))) return rc;
    return launch_commit(c, ids, OP_COMPACT, (const int *)ws, st);
}

KVC_EXPORT int kvc_pages_free(const kvc_page_cache * cache, const int * seqs, int n, void * ws, size_t ws_bytes,
                              void * stream) {
    int rc = kvc_check_cache(cache);
    if (rc) return rc;
    plan_ids ids;
    if ((rc = check_ids(cache, seqs, seqs, n, &ids))) return rc;
    if ((rc = check_ws(cache, ws, ws_bytes))) return rc;
    const int sms = kvc_serve_device();
    if (sms < 0) return sms;
    if (n == 0) return KVC_OK;
    return launch_commit(on_device(cache), ids, OP_FREE, (const int *)ws, (cudaStream_t)stream);
}

}  // extern "C"
