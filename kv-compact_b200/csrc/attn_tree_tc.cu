// attn_tree_tc.cu — attention of drafted trees over the paged cache on the
// 5th-generation tensor cores (tcgen05, accumulators in TMEM), for entries with
// many query rows per KV head (nodes x group), where k_tree_mma is bound by
// issuing its matrix instructions.
//
// A CTA takes up to 128 query rows of one KV head and a stretch of the keys, in
// tiles of 64 keys. F16 rows are copied as they are; a row of block codes
// becomes two fp16 pieces of value / 2^e, e the exponent of the row's largest
// block scale (22 bits of the row's range), once per CTA. F32 queries (times a
// power of two per row) and their probabilities enter as two pieces as well:
//
//   S[r][j] = sum of Qhi Khi, Qhi Klo, Qlo Khi        x = S 2^e_j scale + beta_j
//   O[r]   += 2^(R - 10) (Phi Vhi + Phi Vlo + Plo Vhi), P = exp(x - m) 2^(10 + e_j - R)
//
// with R the largest exponent of the tile's V rows. Every tile's product starts
// from zero and is added to O in fp32 registers, which rounds to nearest (the
// tensor cores' own sums truncate) and needs no correction of O in TMEM.
//
//   warps 0-3, 4-7   softmax of the even / odd tiles, each with its own S, m, l
//                    and O (two streams: one's products run under the other's
//                    softmax); a thread owns a row; joined at the end
//   warps 8-11       producers: rows of tile i + 1 are on their way while tile i
//                    is put into the swizzled tiles
//   warp 12          MMA issue (one thread); 13-15 idle (register shares go by
//                    warp group)
//
// Bound by latency inside a CTA: a stream's chain per tile (scores, maximum,
// exponentials, P, product, sums) takes about 6,000 cycles at 128 values with two
// softmax warps per scheduler, which the other stream half hides; and about 15 us
// per call go to the segments, the queries, the first tile and the join. Trees of
// 16 to 60 nodes on 26,122 F16 keys (8 heads of 4 query heads, 128 values) 108 us,
// 1.0 TB/s of rows; 25 nodes on 30,000 Q4_0 / Q4_1 keys (4 heads of 8, 64 values,
// F32 queries) 84 us. Queries read pair by pair before the first tile was asked
// for: 122 and 90 us.
#include "attn.h"
#include "attn_tc.h"
#include "attn_tree.h"

#include <limits.h>
#include <math.h>
#include <stddef.h>

namespace {

using namespace kvc_tc;
using namespace kvc_attn_tc;

constexpr int TM = 128, TN = 64;                // query rows, keys of a tile
constexpr int THREADS = 512;
constexpr int MAX_SEGS = 64;
constexpr uint32_t POLLS = 1u << 22;            // bound of every wait
constexpr float LOG2E = 1.4426950408889634f;
constexpr int P_SHIFT = 10;
// S is the product of the row's q / 2^u and the key's k / 2^e, e >= -15: with F32 queries 2^u S could pass fp32's range
// where q.k does not, so 2^u comes over this power of two and f times it.
template <int QP>
constexpr int HEADROOM = QP == 2 ? 16 : 0;
constexpr int HIDDEN = -200 * (1 << 23);        // exponent bits of a row that counts for nothing
// registers per thread of the warp groups; their sum x 128 is what the block is launched with
constexpr int REG_SOFTMAX = 192, REG_PRODUCE = 88, REG_MMA = 40, REG_LAUNCH = 128;
static_assert(2 * REG_SOFTMAX + REG_PRODUCE + REG_MMA <= 4 * REG_LAUNCH, "more registers than the block has");

template <int D, int QP, int KP>
struct cfg {
    static constexpr int HALVES = D / 64;
    static constexpr int KBLOCK = TN * 128, QBLOCK = TM * 128;      // 64 values x rows, 128 bytes a row
    static constexpr int PIECE = HALVES * KBLOCK;                   // one fp16 piece of a K or V tile
    static constexpr int SLOT = KP * PIECE;
    static constexpr int Q = QP * HALVES * QBLOCK;
    static constexpr int SLOTS = SLOT > 16384 ? 4 : 8;
    static constexpr int RING = SLOTS * SLOT;
    static constexpr int JOIN = TM * (D + 4) * 4;                   // one stream's O, over the ring
    static constexpr int REGION = RING > JOIN ? RING : JOIN;
    // TMEM: S of stream t at 64 t, O at 128 + D t, the pieces of P at 128 + 2 D + 64 t and 32 columns on
    static constexpr uint32_t S_COL = 0, O_COL = 128, P_COL = 128 + 2 * D;
    static constexpr uint32_t COLS = 512;
};

struct segment {
    int lo, hi, slot, qb, q0, nq, nodes, ln, table;
};

// Per key of a tile. Eight tiles deep: when tile i is filled, tile i - 5 and those before it have been read.
struct alignas(16) tile_info {      // read four at a time
    float f[TN];                // factor of S: scale 2^(e + HEADROOM)
    float b[TN];                // beta, or -inf
    int e[TN];                  // exponent of the V row << 23, or HIDDEN
};

struct shared {
    uint64_t full[8], empty[8], s_full[2], p_full[2], o_full[2], done;
    uint32_t tmem, lost;        // lost: a wait ran out
    int n_segs[2];
    unsigned long long bad[2][2];   // per stream, of even and odd steps (a slow warp may still read the step before's): rows
                                    // of the tile that are taken value by value
    segment segs[MAX_SEGS];
    int rows[2][TN];            // pool rows of a tile
    float mul[TM];              // power of two that a query row was divided by, over 2^HEADROOM
    float jm[TM], jl[TM];
    tile_info info[8];
};

static_assert(offsetof(shared, info) % 16 == 0, "tile_info on a 16-byte boundary");

template <int N>
__device__ __forceinline__ void reg_more() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(N)); }
template <int N>
__device__ __forceinline__ void reg_less() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(N)); }
__device__ __forceinline__ void group_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" :: "r"(id), "r"(threads) : "memory"); }
__device__ __forceinline__ void copy16(uint32_t dst, const void * src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(dst), "l"(src) : "memory");
}
// One column of this thread's TMEM lane.
__device__ __forceinline__ float ld1(uint32_t addr) {
    uint32_t r;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(addr));
    tmem_wait_ld();
    return __uint_as_float(r);
}
// 8 columns of this thread's TMEM lane.
__device__ __forceinline__ void st8(uint32_t addr, const uint32_t * r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 :: "r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
__device__ __forceinline__ float half_of(uint32_t h) { return __half2float(__ushort_as_half((unsigned short)h)); }
// 16 bytes of row r, chunk c of a 128-byte-swizzled block.
__device__ __forceinline__ uint32_t swizzled(int r, int c) { return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4)); }
__device__ __forceinline__ uint32_t h2mul(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t h2fma(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
__device__ __forceinline__ uint32_t h2add(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// One stored 32-value block as it was read: the aligned words that hold it.
struct raw_block {
    uint32_t w[9];
};
// A block at p (2-byte aligned). Q8_0 and Q4_0 blocks lie at either half of a word; the word before the block's
// first half-word belongs to the same pool, the half-word behind its last one is read alone.
__device__ __forceinline__ void read_block(raw_block & r, const uint8_t * p, int type) {
    const bool odd = ((uintptr_t)p & 2) != 0;
    const uint32_t * w = reinterpret_cast<const uint32_t *>(p - (odd ? 2 : 0));
    const int whole = type == KV_TYPE_Q8_0 ? (odd ? 9 : 8) : type == KV_TYPE_Q4_0 ? (odd ? 5 : 4) : 5;
#pragma unroll
    for (int i = 0; i < 9; i++) r.w[i] = i < whole ? w[i] : 0;
    if (!odd && type != KV_TYPE_Q4_1) r.w[type == KV_TYPE_Q8_0 ? 8 : 4] = *reinterpret_cast<const uint16_t *>(w + whole);
}
// Scale (and minimum) of a block as fp16 bits; the code words follow on a word boundary.
__device__ __forceinline__ void block_head(const raw_block & r, bool odd, int type, uint32_t & d, uint32_t & m) {
    d = odd ? r.w[0] >> 16 : r.w[0] & 0xFFFFu;
    m = type == KV_TYPE_Q4_1 ? r.w[0] >> 16 : 0;
}
__device__ __forceinline__ uint32_t code_word(const raw_block & r, bool odd, int type, int i) {
    return odd || type == KV_TYPE_Q4_1 ? r.w[i + 1] : __funnelshift_r(r.w[i], r.w[i + 1], 16);
}

// 32 values of a block over 2^e as two fp16 pieces, written as 16-byte chunks (8 values) through put(chunk, hi, lo).
template <int TYPE, typename F>
__device__ __forceinline__ void block_values(const raw_block & r, bool odd, float up, F && put) {
    uint32_t d, m;
    block_head(r, odd, TYPE, d, m);
    const float fd = half_of(d) * up, fm = half_of(m) * up;     // a power of two: exact but for tiny scales
    const uint32_t d2 = pack(fd, fd);
#pragma unroll
    for (int c = 0; c < 4; c++) {
        uint32_t hi[4], lo[4];
        if (TYPE == KV_TYPE_Q8_0) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const uint32_t w = code_word(r, odd, TYPE, 2 * c + i) ^ 0x80808080u;
                const uint32_t c0 = h2add(__byte_perm(w, 0x64646464u, 0x4140), 0xE480E480u);   // 1024 + 128 + code, less 1152
                const uint32_t c1 = h2add(__byte_perm(w, 0x64646464u, 0x4342), 0xE480E480u);
                hi[2 * i] = h2mul(c0, d2);
                hi[2 * i + 1] = h2mul(c1, d2);
                lo[2 * i] = h2fma(c0, d2, hi[2 * i] ^ 0x80008000u);                            // exact
                lo[2 * i + 1] = h2fma(c1, d2, hi[2 * i + 1] ^ 0x80008000u);
            }
        } else {
            // a byte holds values 2i (low) and 2i + 1 (high): 0x6400 | n is 1024 + n, 0x6400 | 16 n is 1024 + 16 n
            const uint32_t w = code_word(r, odd, TYPE, c);
#pragma unroll
            for (int b = 0; b < 4; b++) {
                const uint32_t n = __byte_perm(w, 0x64646464u, 0x4040 | b << 8 | b) & 0x64F0640Fu;
                if (TYPE == KV_TYPE_Q4_0) {              // (1024 + n0) - 1032, (1024 + 16 n1) / 16 - 72
                    const uint32_t q = h2fma(n, 0x2C003C00u, 0xD480E408u);
                    hi[b] = h2mul(q, d2);
                    lo[b] = h2fma(q, d2, hi[b] ^ 0x80008000u);                                 // exact
                } else {
                    const uint32_t q = h2fma(n, 0x2C003C00u, 0xD400E400u);
                    __half2 hq, hh;
                    memcpy(&hq, &q, 4);
                    const float2 x = __half22float2(hq);
                    const float v0 = fmaf(x.x, fd, fm), v1 = fmaf(x.y, fd, fm);
                    hi[b] = pack(v0, v1);
                    memcpy(&hh, &hi[b], 4);
                    const float2 f = __half22float2(hh);
                    lo[b] = pack(v0 - f.x, v1 - f.y);
                }
            }
        }
        put(c, make_uint4(hi[0], hi[1], hi[2], hi[3]), make_uint4(lo[0], lo[1], lo[2], lo[3]));
    }
}

template <int D, int QP, int KP>
__global__ void __launch_bounds__(THREADS, 1) k_tree_tc(const __grid_constant__ kvc_attn_args a, int n_blocks) {
    using C = cfg<D, QP, KP>;
    extern __shared__ uint8_t sm_raw[];
    uint8_t * sm = aligned_1024(sm_raw);
    uint8_t * sq = sm;                                   // [piece][half][128 rows][128 bytes]
    uint8_t * ring = sq + C::Q;                          // slots: [piece][half][64 rows][128 bytes]
    shared & X = *reinterpret_cast<shared *>(ring + C::REGION);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int h = blockIdx.y, w = blockIdx.x;
    if (warp == 12) tmem_alloc(&X.tmem, C::COLS);
    if (threadIdx.x == 0) {
        for (int i = 0; i < C::SLOTS; i++) {
            mbar_init(X.full + i, 128);
            mbar_init(X.empty + i, 1);
        }
        for (int t = 0; t < 2; t++) {
            mbar_init(X.s_full + t, 1);
            mbar_init(X.p_full + t, 4);
            mbar_init(X.o_full + t, 1);
        }
        mbar_init(&X.done, 1);
        X.lost = 0;
        mbar_init_fence();
    }
    cudaTriggerProgrammaticLaunchCompletion();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = X.tmem;
    // False: a wait ran out; the status says so. The thread goes on without waiting, whatever it then reads, and takes
    // every barrier of its group: these have no bound, and other warps may be behind them already.
    bool ok = true;
    auto await = [&](uint64_t * bar, uint32_t parity) {
        if (ok && !mbar_wait(bar, parity, POLLS)) {
            ok = false;
            X.lost = 1;
            if (a.status) *a.status = KVC_ERR_CUDA;
        }
    };
    // The same where the warp goes on to instructions of all its lanes: they agree.
    auto await_warp = [&](uint64_t * bar, uint32_t parity) {
        await(bar, parity);
        ok = __all_sync(~0u, ok);
    };
    int items = 0;                                       // K and V tiles through the ring before this segment
    int turns[2] = {0, 0};                               // tiles of each stream before it

    // every role walks the same segments
    auto each = [&](auto walks, auto && body) {
        for (int batch = 0;; batch += MAX_SEGS) {
            __syncthreads();
            if (decltype(walks)::value && warp == 0) {
                int n = 0;
                attn_walk(a, 0, n_blocks, w, h == 0, [&](int qb, const kvc_attn_seq & q, int lo, int hi, int slot) {
                    if (n >= batch && n < batch + MAX_SEGS && lane == 0)
                        X.segs[n - batch] = segment{lo, hi, slot, qb, q.q0, q.nq, q.nodes, q.ln, q.slot};
                    n++;
                });
                if (lane == 0) {
                    X.n_segs[0] = min(n - batch, MAX_SEGS);
                    X.n_segs[1] = n;
                }
            }
            __syncthreads();
            const int ns = X.n_segs[0], all = X.n_segs[1];
            for (int i = 0; i < ns; i++) {
                const segment S = X.segs[i];
                const int n = S.hi - S.lo;
                body(S, n);
                items += 2 * n;
                turns[0] += (n + 1) / 2;
                turns[1] += n / 2;
                __syncthreads();                         // the ring held the join, Q is read no more
            }
            if (all <= batch + MAX_SEGS) break;
        }
    };

    if (warp < 8) {
        // ---- softmax
        reg_more<REG_SOFTMAX>();
        const int t = warp >> 2, r = threadIdx.x & 127;
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const uint32_t s_addr = tmem + lanes + C::S_COL + t * TN, o_addr = tmem + lanes + C::O_COL + t * D;
        const uint32_t p_addr = tmem + lanes + C::P_COL + t * 64;
        each(kvc_int<1>{}, [&](const segment & S, int n) {
            const int qb = S.qb, r0 = qb * TM;
            const int rows_here = (int)min((long long)TM, (long long)S.nq * a.g - r0);
            {
                // Q: two threads per row, in 16-byte pieces where they are aligned, all of them on their way at once
                constexpr int SIZE = QP == 2 ? 4 : 2, PIECES = D / 2 * SIZE / 16;
                const bool whole = ((reinterpret_cast<uintptr_t>(a.q) | (uintptr_t)(a.q_stride * SIZE)) & 15) == 0;
                const int row = threadIdx.x >> 1, part = threadIdx.x & 1;
                const int i = (int)a.by_group.div(r0 + row);
                const long long at = (long long)(S.q0 + i) * a.q_stride + (long long)(h * a.g + (r0 + row - i * a.g)) * a.q_head;
                const uint8_t * src = reinterpret_cast<const uint8_t *>(a.q) + (at + part * (D / 2)) * SIZE;
                const int values = row < rows_here ? a.dk - part * (D / 2) : 0;      // of this thread's half
                uint4 raw[PIECES];
                if (whole) {
#pragma unroll
                    for (int k = 0; k < PIECES; k++)
                        raw[k] = 16 / SIZE * k < values ? *reinterpret_cast<const uint4 *>(src + 16 * k) : make_uint4(0, 0, 0, 0);
                } else {
#pragma unroll
                    for (int k = 0; k < PIECES; k++) {
                        uint32_t x[4] = {0, 0, 0, 0};
                        if (16 / SIZE * k < values) {
#pragma unroll
                            for (int u = 0; u < 4; u++) {
                                const uint8_t * p = src + 16 * k + 4 * u;
                                if (QP == 2) x[u] = *reinterpret_cast<const uint32_t *>(p);
                                else x[u] = *reinterpret_cast<const uint16_t *>(p) | (uint32_t)*reinterpret_cast<const uint16_t *>(p + 2) << 16;
                            }
                        }
                        raw[k] = make_uint4(x[0], x[1], x[2], x[3]);
                    }
                }
                float2 v[D / 4];
#pragma unroll
                for (int k = 0; k < PIECES; k++) {
                    const uint32_t x[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
#pragma unroll
                    for (int u = 0; u < 4; u++) {
                        if (QP == 2) {
                            float2 & y = v[2 * k + u / 2];
                            if (u & 1) y.y = __uint_as_float(x[u]);
                            else y.x = __uint_as_float(x[u]);
                        } else {
                            __half2 hh;
                            memcpy(&hh, &x[u], 4);
                            v[(4 * k + u) % (D / 4)] = __half22float2(hh);
                        }
                    }
                }
                float up = 1.0f;
                if (QP == 2) {
                    float top = 0.0f;
#pragma unroll
                    for (int k = 0; k < D / 4; k++) top = fmaxf(top, fmaxf(fabsf(v[k].x), fabsf(v[k].y)));
                    top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
                    float down = 1.0f;
                    // largest value of the row in [2^13, 2^14): both pieces normal numbers
                    if (top > 0.0f && top < INFINITY) {
                        const int e = min(13 - ilogbf(top), 100);
                        up = scalbnf(1.0f, e);
                        down = scalbnf(1.0f, -e);
                    }
                    down *= 1.0f / (1 << HEADROOM<QP>);
                    if (part == 0) X.mul[row] = down;
                }
#pragma unroll
                for (int c = 0; c < D / 16; c++) {       // chunks of 8 values
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const float x = v[4 * c + k].x * up, y = v[4 * c + k].y * up;
                        hi[k] = pack(x, y);
                        __half2 hh;
                        memcpy(&hh, &hi[k], 4);
                        const float2 f = __half22float2(hh);
                        lo[k] = pack(x - f.x, y - f.y);
                    }
                    const int chunk = part * (D / 16) + c;
                    uint8_t * dst = sq + (chunk >> 3) * C::QBLOCK + swizzled(row, chunk & 7);
                    *reinterpret_cast<uint4 *>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    if (QP == 2)
                        *reinterpret_cast<uint4 *>(dst + C::HALVES * C::QBLOCK) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                }
                fence_smem_to_async();
            }
            group_sync(4, 288);                          // Q is there: these warps and the one that issues the products
            const float mul = QP == 2 ? X.mul[r] : 1.0f;
            const bool real = r < rows_here;
            const int node = (int)a.by_group.div(r0 + r);
            const int first_own = a.mask ? S.ln - S.nodes : INT_MAX;
            const int steps = (n + 1 - t) / 2;
            float m = -INFINITY, l = 0.0f, back = 0.0f;  // back: 2^(R - 10) of the tile whose product is still in TMEM
            float2 O[D / 2];
#pragma unroll
            for (int k = 0; k < D / 2; k++) O[k] = make_float2(0.0f, 0.0f);
            // O = (O + product of the tile before) * f
            auto collect = [&](float f) {
                const float2 b2 = make_float2(back, back), f2 = make_float2(f, f);
                const bool moved = __any_sync(~0u, f != 1.0f);
#pragma unroll
                for (int c = 0; c < D; c += 32) {
                    uint32_t o[32];
                    tmem_ld16_nowait(o_addr + c, o);
                    tmem_ld16_nowait(o_addr + c + 16, o + 16);
                    tmem_wait_ld();
#pragma unroll
                    for (int k = 0; k < 16; k++) {
                        float2 & x = O[c / 2 + k];
                        x = fma2(make_float2(__uint_as_float(o[2 * k]), __uint_as_float(o[2 * k + 1])), b2, x);
                    }
                }
                if (moved) {
#pragma unroll
                    for (int k = 0; k < D / 2; k++) O[k] = mul2(O[k], f2);
                }
            };
            for (int j = 0; j < steps; j++) {
                const int i = 2 * j + t;                 // tile of the segment
                await_warp(X.s_full + t, (turns[t] + j) & 1);
                fence_after_sync();
                const tile_info & I = X.info[i & 7];
                const int j0 = (S.lo + i) * TN;
                const bool own = j0 + TN > first_own;
                unsigned long long vis = ~0ull;          // which of the tile's keys the mask shows to this row
                if (own) {
#pragma unroll 1
                    for (int k = max(0, first_own - j0); k < TN; k++) {
                        const int b = j0 + k - first_own;
                        const bool sees = j0 + k < S.ln && real && (b >> 5) < a.mask_words &&
                                          ((a.mask[(size_t)(S.q0 + node) * a.mask_words + (b >> 5)] >> (b & 31)) & 1u);
                        if (!sees) vis &= ~(1ull << k);
                    }
                }
                // x of columns c .. c+15 from v; `show`: the keys that count
                auto scores = [&](auto masked, int c, unsigned long long show, const uint32_t v[16], float2 x[8]) {
#pragma unroll
                    for (int k = 0; k < 16; k += 4) {
                        const float4 f = *reinterpret_cast<const float4 *>(&I.f[c + k]);
                        const float4 b = *reinterpret_cast<const float4 *>(&I.b[c + k]);
                        const float2 fk[2] = {make_float2(f.x, f.y), make_float2(f.z, f.w)};
                        const float2 bk[2] = {make_float2(b.x, b.y), make_float2(b.z, b.w)};
#pragma unroll
                        for (int u = 0; u < 2; u++) {
                            float2 s = make_float2(__uint_as_float(v[k + 2 * u]), __uint_as_float(v[k + 2 * u + 1]));
                            if (QP == 2) s = mul2(s, make_float2(mul, mul));
                            float2 & y = x[k / 2 + u];
                            y = fma2(s, fk[u], bk[u]);   // hidden rows: S = 0 and beta = -inf
                            if (decltype(masked)::value) {
                                if (!((show >> (c + k + 2 * u)) & 1)) y.x = -INFINITY;
                                if (!((show >> (c + k + 2 * u + 1)) & 1)) y.y = -INFINITY;
                            }
                        }
                    }
                };
                float top = -INFINITY;
                auto maximum = [&](auto masked) {
#pragma unroll 1
                    for (int c = 0; c < TN; c += 32) {
                        uint32_t v[2][16];
                        tmem_ld16_nowait(s_addr + c, v[0]);
                        tmem_ld16_nowait(s_addr + c + 16, v[1]);
                        tmem_wait_ld();
#pragma unroll
                        for (int u = 0; u < 2; u++) {
                            float2 x[8];
                            scores(masked, c + 16 * u, vis, v[u], x);
#pragma unroll
                            for (int k = 0; k < 8; k += 2)
                                top = fmaxf(fmaxf(top, fmaxf(x[k].x, x[k].y)), fmaxf(x[k + 1].x, x[k + 1].y));
                        }
                    }
                };
                if (own) maximum(kvc_int<1>{});
                else maximum(kvc_int<0>{});
                const float mn = fmaxf(m, top), base = mn == -INFINITY ? 0.0f : mn;
                const float f = ex2((m - base) * LOG2E);
                m = mn;
                l *= f;
                if (j > 0) {
                    await_warp(X.o_full + t, (turns[t] + j - 1) & 1);  // the product of the tile before
                    fence_after_sync();
                    collect(f);
                }
                // the tile's largest V exponent; rows that the mask hides from some of the queries and whose values are
                // no finite numbers, or far above the others', are added value by value
                int R = HIDDEN;
                float sum = 0.0f;
                float2 sums = make_float2(0.0f, 0.0f);
                if (KP == 2 || own) {
                    const int it = items + 2 * i + 1;    // the exponents are written with V
                    await_warp(X.full + it % C::SLOTS, (it / C::SLOTS) & 1);
                    const int2 e2 = *reinterpret_cast<const int2 *>(&I.e[2 * lane]);
                    R = __reduce_max_sync(~0u, max(e2.x, e2.y));
                    if (own) {
                        uint8_t * vt = ring + (it % C::SLOTS) * C::SLOT;
                        if (r == 0) X.bad[t][j & 1] = 0;
                        const int least = __reduce_min_sync(~0u, min(e2.x > HIDDEN ? e2.x : INT_MAX, e2.y > HIDDEN ? e2.y : INT_MAX));
                        group_sync(1 + t, 128);
                        if (r < TN && I.e[r] > HIDDEN) {
                            bool bad = (I.e[r] >> 23) - (least >> 23) > 8;
                            for (int c = 0; c < D / 8; c++) {
                                const uint4 v = *reinterpret_cast<const uint4 *>(vt + (c >> 3) * C::KBLOCK + swizzled(r, c & 7));
                                for (uint32_t y : {v.x, v.y, v.z, v.w})
                                    bad |= (y & 0x7C00u) == 0x7C00u || (y & 0x7C000000u) == 0x7C000000u;
                            }
                            if (bad) atomicOr(&X.bad[t][j & 1], 1ull << r);
                        }
                        group_sync(1 + t, 128);
                        const unsigned long long bad = X.bad[t][j & 1];
                        if (bad) {
                            R = max((bad >> (2 * lane)) & 1 ? HIDDEN : e2.x, (bad >> (2 * lane + 1)) & 1 ? HIDDEN : e2.y);
                            R = __reduce_max_sync(~0u, R);
                            for (unsigned long long left = bad; left;) {
                                const int k = __ffsll((long long)left) - 1;
                                left &= left - 1;
                                const float s = ld1(s_addr + k);
                                const float x = (vis >> k) & 1 ? fmaf(QP == 2 ? s * mul : s, I.f[k], I.b[k]) : -INFINITY;
                                const float p = ex2((x - base) * LOG2E), g = scalbnf(1.0f, I.e[k] >> 23);
                                sum += p;
#pragma unroll
                                for (int d = 0; d < D / 2; d++) {
                                    const uint32_t o = (d >> 5) * C::KBLOCK + swizzled(k, (d >> 2) & 7) + (d & 3) * 4;
                                    uint32_t hv = *reinterpret_cast<const uint32_t *>(vt + o), lv = 0;
                                    if (KP == 2) lv = *reinterpret_cast<const uint32_t *>(vt + C::PIECE + o);
                                    const bool fin0 = (hv & 0x7C00u) != 0x7C00u, fin1 = (hv & 0x7C000000u) != 0x7C000000u;
                                    const float v0 = half_of(hv) + (fin0 ? half_of(lv) : 0.0f);
                                    const float v1 = half_of(hv >> 16) + (fin1 ? half_of(lv >> 16) : 0.0f);
                                    if (p != 0.0f) {
                                        O[d].x = fmaf(p, v0 * g, O[d].x);
                                        O[d].y = fmaf(p, v1 * g, O[d].y);
                                    }
                                }
                            }
                            group_sync(1 + t, 128);
                            if (r < TN && ((bad >> r) & 1))      // 0 * V is to be 0
                                for (int pc = 0; pc < KP; pc++)
                                    for (int c = 0; c < D / 8; c++)
                                        *reinterpret_cast<uint4 *>(vt + pc * C::PIECE + (c >> 3) * C::KBLOCK + swizzled(r, c & 7)) =
                                            make_uint4(0, 0, 0, 0);
                            fence_smem_to_async();
                            vis &= ~bad;
                        }
                    }
                    if (R == HIDDEN) R = 0;
                } else {
                    R = 0;
                }
                back = scalbnf(1.0f, (R >> 23) - P_SHIFT);
                const int up_bits = (127 + P_SHIFT) * (1 << 23) - R;     // + exponent bits: 2^(10 + e - R)
                auto probabilities = [&](auto masked) {
                    uint32_t v[16];
                    tmem_ld16_nowait(s_addr, v);
#pragma unroll 1
                    for (int c = 0; c < TN; c += 16) {
                        float2 x[8];
                        tmem_wait_ld();
                        scores(masked, c, vis, v, x);
                        if (c + 16 < TN) tmem_ld16_nowait(s_addr + c + 16, v);     // under the exponentials
                        int4 e[4];
                        if (KP == 2) {
#pragma unroll
                            for (int k = 0; k < 4; k++) e[k] = *reinterpret_cast<const int4 *>(&I.e[c + 4 * k]);
                        }
                        uint32_t p0[8], p1[8];
#pragma unroll
                        for (int k = 0; k < 8; k++) {
                            const float2 y = mul2(add2(x[k], make_float2(-base, -base)), make_float2(LOG2E, LOG2E));
                            float2 p = make_float2(ex2(y.x), ex2(y.y));
                            sums = add2(sums, p);
                            float2 up = make_float2((float)(1 << P_SHIFT), (float)(1 << P_SHIFT));
                            if (KP == 2) {
                                const int4 & ek = e[k / 2];
                                up.x = __int_as_float(max((k & 1 ? ek.z : ek.x) + up_bits, 0));
                                up.y = __int_as_float(max((k & 1 ? ek.w : ek.y) + up_bits, 0));
                            }
                            p = mul2(p, up);
                            p0[k] = pack(p.x, p.y);
                            if (QP == 2) {
                                __half2 hh;
                                memcpy(&hh, &p0[k], 4);
                                const float2 z = __half22float2(hh);
                                p1[k] = pack(p.x - z.x, p.y - z.y);
                            }
                        }
                        st8(p_addr + c / 2, p0);
                        if (QP == 2) st8(p_addr + 32 + c / 2, p1);
                    }
                };
                if (own) probabilities(kvc_int<1>{});
                else probabilities(kvc_int<0>{});
                l += sum + (sums.x + sums.y);
                tmem_wait_st();
                fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(X.p_full + t);
            }
            if (steps > 0) {
                await_warp(X.o_full + t, (turns[t] + steps - 1) & 1);
                fence_after_sync();
                collect(1.0f);
            }
            // ---- join the streams (over the ring: every product has been taken)
            group_sync(3, 256);
            float * jo = reinterpret_cast<float *>(ring) + r * (D + 4);
            if (t == 1) {
#pragma unroll
                for (int k = 0; k < D / 4; k++)
                    *reinterpret_cast<float4 *>(jo + 4 * k) = make_float4(O[2 * k].x, O[2 * k].y, O[2 * k + 1].x, O[2 * k + 1].y);
                X.jm[r] = m;
                X.jl[r] = l;
            }
            group_sync(3, 256);
            if (t == 0) {
                const float om = X.jm[r], mn = fmaxf(m, om), base = mn == -INFINITY ? 0.0f : mn;
                const float f0 = ex2((m - base) * LOG2E), f1 = ex2((om - base) * LOG2E);
                l = l * f0 + X.jl[r] * f1;
                const float inv = S.slot >= 0 ? 1.0f : l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
                X.jm[r] = mn;
                X.jl[r] = l;
#pragma unroll
                for (int k = 0; k < D / 4; k++) {
                    float4 o = *reinterpret_cast<const float4 *>(jo + 4 * k);
                    o.x = (O[2 * k].x * f0 + o.x * f1) * inv;
                    o.y = (O[2 * k].y * f0 + o.y * f1) * inv;
                    o.z = (O[2 * k + 1].x * f0 + o.z * f1) * inv;
                    o.w = (O[2 * k + 1].y * f0 + o.w * f1) * inv;
                    *reinterpret_cast<float4 *>(jo + 4 * k) = o;
                }
            }
            group_sync(3, 256);
            // written side by side: a partial result is one stretch of rows
            float * part = S.slot >= 0 ? attn_part(a, qb, h, w, S.slot) : nullptr;
            if (t == 0 && real) {
                const size_t out = (size_t)(S.q0 + node) * a.Hq + h * a.g + (r0 + r - node * a.g);
                if (part) {
                    part[a.rb * a.dv + r] = X.jm[r];
                    part[a.rb * a.dv + a.rb + r] = X.jl[r];
                } else if (a.lse) {
                    a.lse[out] = X.jl[r] == 0.0f ? -INFINITY : X.jm[r] + logf(X.jl[r]);
                }
            }
            // 32 lanes = one row's D / 4 pieces of 16 bytes, twice for D = 64
            constexpr int PIECES = D / 4;
            const int piece = threadIdx.x % PIECES;
            if (4 * piece < a.dv)
#pragma unroll 4
                for (int rr = threadIdx.x / PIECES; rr < rows_here; rr += 256 / PIECES) {
                    const float4 o = *reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(ring) + rr * (D + 4) + 4 * piece);
                    if (part) {
                        *reinterpret_cast<float4 *>(part + rr * a.dv + 4 * piece) = o;
                    } else {
                        const int nd = (int)a.by_group.div(r0 + rr);
                        const size_t at = ((size_t)(S.q0 + nd) * a.Hq + h * a.g + (r0 + rr - nd * a.g)) * a.dv + 4 * piece;
                        const float v[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
                        for (int u = 0; u < 4; u++) {
                            if (QP == 2) reinterpret_cast<float *>(a.out)[at + u] = v[u];
                            else reinterpret_cast<__half *>(a.out)[at + u] = __float2half_rn(v[u]);
                        }
                    }
                }
        });
    } else if (warp < 12) {
        // ---- producers
        reg_less<REG_PRODUCE>();
        const int tid = threadIdx.x - 256;
        constexpr int PER = D / 64;                      // blocks of a thread: half a row (two threads per key)
        each(kvc_int<0>{}, [&](const segment & S, int n) {
            const int * table = a.table + (size_t)S.table * a.max_pages;
            // this thread's key of tile i: pool row, or -1; its bias
            const int key = KP == 2 ? tid >> 1 : tid & (TN - 1);
            auto place = [&](int i, int page) {
                const long long j = (long long)(S.lo + i) * TN + key;
                return i < n && j < S.ln && page >= 0 && page < a.n_pages
                           ? page * a.page + (int)(j - (long long)a.by_page.div((uint32_t)j) * a.page) : -1;
            };
            auto page_of = [&](int i) {
                const long long j = (long long)(S.lo + i) * TN + key;
                return i < n && j < S.ln ? table[a.by_page.div((uint32_t)j)] : -1;
            };
            auto bias_of = [&](int row) {
                if (row < 0) return -INFINITY;
                if (!a.beta) return 0.0f;
                const uint32_t p = a.by_page.div((uint32_t)row);
                return a.beta[((size_t)p * a.Hkv + h) * a.page + (row - (int)p * a.page)];
            };
            if constexpr (KP == 1) {
                const int chunk = tid & 7, first = tid >> 3;
                int page = page_of(0);
                int row = place(0, page);
                float bias = bias_of(row);
                page = page_of(1);
                auto arrive = [&](int i) {               // tile i has landed
                    fence_smem_to_async();
                    mbar_arrive(X.full + (items + 2 * i) % C::SLOTS);
                    mbar_arrive(X.full + (items + 2 * i + 1) % C::SLOTS);
                };
                for (int i = 0; i < n; i++) {
                    if (tid < TN) {
                        tile_info & I = X.info[i & 7];
                        const bool live = bias != -INFINITY;
                        X.rows[i & 1][key] = live ? row : -1;
                        I.f[key] = a.scale * (1 << HEADROOM<QP>);
                        I.b[key] = bias;
                        I.e[key] = live ? 0 : HIDDEN;
                    }
                    // the next tile's place and bias, the page of the one after
                    row = place(i + 1, page);
                    bias = bias_of(row);
                    page = page_of(i + 2);
                    group_sync(5, 128);
                    for (int side = 0; side < 2; side++) {
                        const int it = items + 2 * i + side;
                        await(X.empty + it % C::SLOTS, ((it / C::SLOTS) & 1) ^ 1);
                        const uint8_t * base = side ? a.V + (long long)h * a.v_hb : a.K + (long long)h * a.k_hb;
                        const long long rb = side ? a.v_rb : a.k_rb;
                        const int bytes = 2 * (side ? a.dv : a.dk);
                        uint8_t * dst = ring + (it % C::SLOTS) * C::SLOT;
#pragma unroll
                        for (int k = 0; k < TN / 16; k++) {
                            const int rr = first + 16 * k, at = X.rows[i & 1][rr];
#pragma unroll
                            for (int hf = 0; hf < C::HALVES; hf++) {
                                uint8_t * d = dst + hf * C::KBLOCK + swizzled(rr, chunk);
                                const int o = hf * 128 + chunk * 16;
                                if (at >= 0 && o < bytes && ok) copy16(smem_u32(d), base + at * rb + o);
                                else *reinterpret_cast<uint4 *>(d) = make_uint4(0, 0, 0, 0);
                            }
                        }
                    }
                    asm volatile("cp.async.commit_group;" ::: "memory");
                    if (i > 0) {
                        asm volatile("cp.async.wait_group 1;" ::: "memory");
                        arrive(i - 1);
                    }
                }
                asm volatile("cp.async.wait_group 0;" ::: "memory");
                if (n > 0) arrive(n - 1);
            } else {
                const int part = tid & 1;
                const int kbb = kvc_block_size(a.k_type), vbb = kvc_block_size(a.v_type);
                const int nbk = a.dk >> 5, nbv = a.dv >> 5;
                raw_block K[PER], V[PER], R[PER];
                uint32_t odd_k = 0, odd_v = 0;
                // an absent row reads the pool's first one: every address is one of the pool's
                auto read = [&](raw_block * R, uint32_t & odd, const uint8_t * base, long long rb, long long hb, int size, int nb,
                                int type, int row) {
                    odd = 0;
                    const uint8_t * at = base + (row < 0 ? 0 : row) * rb + (long long)h * hb;
#pragma unroll
                    for (int b = 0; b < PER; b++) {
                        const int bb = part * PER + b;
                        const uint8_t * p = at + (bb < nb ? bb : 0) * size;
                        odd |= (uint32_t)((uintptr_t)p >> 1 & 1) << b;
                        read_block(R[b], p, type);
                    }
                };
                // one side of tile i from its raw blocks: two pieces over 2^e, e the exponent of the row's largest finite
                // scale or minimum, which is returned
                auto convert = [&](uint32_t odd, int type, int nb, int it, bool live) {
                    uint32_t top = 0;
#pragma unroll
                    for (int b = 0; b < PER; b++)
                        if (part * PER + b < nb) {
                            uint32_t d, m;
                            block_head(R[b], (odd >> b) & 1, type, d, m);
                            d &= 0x7FFFu, m &= 0x7FFFu;
                            top = max(top, max(d < 0x7C00u ? d : 0u, m < 0x7C00u ? m : 0u));
                        }
                    top = max(top, __shfl_xor_sync(~0u, top, 1));
                    const int e = max((int)(top >> 10), 1) - 15;
                    const float up = __int_as_float((127 - e) << 23);
                    await(X.empty + it % C::SLOTS, ((it / C::SLOTS) & 1) ^ 1);
                    uint8_t * dst = ring + (it % C::SLOTS) * C::SLOT;
#pragma unroll
                    for (int b = 0; b < PER; b++) {
                        const int bb = part * PER + b;
                        uint8_t * at = dst + (bb >> 1) * C::KBLOCK;
                        auto put = [&](int c, uint4 hi, uint4 lo) {
                            uint8_t * p = at + swizzled(key, (bb & 1) * 4 + c);
                            *reinterpret_cast<uint4 *>(p) = hi;
                            *reinterpret_cast<uint4 *>(p + C::PIECE) = lo;
                        };
                        const bool o = (odd >> b) & 1;
                        if (!live || bb >= nb) {
#pragma unroll
                            for (int c = 0; c < 4; c++) put(c, make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0));
                        } else if (type == KV_TYPE_Q8_0) {
                            block_values<KV_TYPE_Q8_0>(R[b], o, up, put);
                        } else if (type == KV_TYPE_Q4_0) {
                            block_values<KV_TYPE_Q4_0>(R[b], o, up, put);
                        } else {
                            block_values<KV_TYPE_Q4_1>(R[b], o, up, put);
                        }
                    }
                    return e;
                };
                auto read_k = [&](int row) { read(K, odd_k, a.K, a.k_rb, a.k_hb, kbb, nbk, a.k_type, row); };
                auto read_v = [&](int row) { read(V, odd_v, a.V, a.v_rb, a.v_hb, vbb, nbv, a.v_type, row); };
                int page = page_of(0);
                int row = place(0, page);
                float bias = bias_of(row);
                read_k(row);
                read_v(row);
                page = page_of(1);
                for (int i = 0; i < n; i++) {
                    const bool live = row >= 0 && bias != -INFINITY;
                    const float bias_now = bias;
                    row = place(i + 1, page);
                    bias = bias_of(row);
                    page = page_of(i + 2);
#pragma unroll 1
                    for (int side = 0; side < 2; side++) {       // one body for both sides: the loop has to stay in the instruction cache
#pragma unroll
                        for (int b = 0; b < PER; b++)
#pragma unroll
                            for (int u = 0; u < 9; u++) R[b].w[u] = side ? V[b].w[u] : K[b].w[u];
                        const uint32_t odd = side ? odd_v : odd_k;
                        // the next tile's K comes in under this one's V, its V under the next K
                        if (side == 0) read_k(row);
                        else read_v(row);
                        const int it = items + 2 * i + side;
                        const int e = convert(odd, side ? a.v_type : a.k_type, side ? nbv : nbk, it, live);
                        if (part == 0) {
                            tile_info & I = X.info[i & 7];
                            if (side == 0) {
                                I.f[key] = a.scale * scalbnf(1.0f, e + HEADROOM<QP>);
                                I.b[key] = live ? bias_now : -INFINITY;
                            } else {
                                I.e[key] = live ? e * (1 << 23) : HIDDEN;
                            }
                        }
                        fence_smem_to_async();
                        mbar_arrive(X.full + it % C::SLOTS);
                    }
                }
            }
            // (the softmax warps' barriers of the join are theirs alone)
        });
    } else {
        reg_less<REG_MMA>();
        // ---- products
        each(kvc_int<0>{}, [&](const segment & S, int n) {
            if (warp == 12) {
                group_sync(4, 288);                      // Q is there
                fence_after_sync();
                constexpr uint32_t ID_S = (1u << 4) | ((uint32_t)(TN >> 3) << 17) | ((uint32_t)(TM >> 4) << 24);
                constexpr uint32_t ID_O = (1u << 4) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(TM >> 4) << 24);
                const uint32_t qa = smem_u32(sq), ra = smem_u32(ring);
                auto qk = [&](int i) {
                    const int it = items + 2 * i;
                    await_warp(X.full + it % C::SLOTS, (it / C::SLOTS) & 1);
                    if (!ok) return;
                    fence_after_sync();
                    const uint32_t ka = ra + (it % C::SLOTS) * C::SLOT;
                    uint32_t acc = 0;
#pragma unroll
                    for (int pr = 2; pr >= 0; pr--) {    // Qlo Khi, Qhi Klo, Qhi Khi: the small ones first
                        if ((pr == 2 && QP == 1) || (pr == 1 && KP == 1)) continue;
                        const uint32_t q = qa + (pr == 2 ? C::HALVES * C::QBLOCK : 0), k = ka + (pr == 1 ? C::PIECE : 0);
#pragma unroll
                        for (int s = 0; s < D / 16; s++) {
                            mma_f16_ss(tmem + C::S_COL + (i & 1) * TN, desc_k(q + (s >> 2) * C::QBLOCK + (s & 3) * 32),
                                    desc_k(k + (s >> 2) * C::KBLOCK + (s & 3) * 32), ID_S, acc);
                            acc = 1;
                        }
                    }
                    commit_mma(X.s_full + (i & 1));
                    commit_mma(X.empty + it % C::SLOTS);
                };
                auto pv = [&](int i) {
                    const int it = items + 2 * i + 1;
                    await_warp(X.full + it % C::SLOTS, (it / C::SLOTS) & 1);
                    if (!ok) return;
                    fence_after_sync();
                    const uint32_t va = ra + (it % C::SLOTS) * C::SLOT, p = tmem + C::P_COL + (i & 1) * 64;
                    uint32_t acc = 0;
#pragma unroll
                    for (int pr = 2; pr >= 0; pr--) {
                        if ((pr == 2 && QP == 1) || (pr == 1 && KP == 1)) continue;
#pragma unroll
                        for (int s = 0; s < TN / 16; s++) {
                            mma_f16_ts(tmem + C::O_COL + (i & 1) * D, p + (pr == 2 ? 32 : 0) + 8 * s,
                                       desc_n(va + (pr == 1 ? C::PIECE : 0) + s * 2048, C::KBLOCK), ID_O, acc);
                            acc = 1;
                        }
                    }
                    commit_mma(X.o_full + (i & 1));
                    commit_mma(X.empty + it % C::SLOTS);
                };
                if (n > 0) qk(0);
                if (n > 1) qk(1);
                for (int i = 0; i < n && ok; i++) {
                    await_warp(X.p_full + (i & 1), (turns[i & 1] + (i >> 1)) & 1);
                    if (!ok) break;
                    fence_after_sync();
                    if (i + 2 < n) qk(i + 2);            // first: the stream's next softmax can begin
                    pv(i);
                }
            }
            __syncwarp();
        });
    }
    fence_before_sync();
    __syncthreads();
    if (warp == 12) {
        fence_after_sync();
        if (X.lost) {                                    // products may be under way that nobody waited for
            commit_mma(&X.done);
            mbar_wait(&X.done, 0, POLLS);
            __syncwarp();
        }
        tmem_free(tmem, C::COLS);
    }
}

template <int D, int QP, int KP>
constexpr int smem_bytes() { return 1024 + cfg<D, QP, KP>::Q + cfg<D, QP, KP>::REGION + (int)sizeof(shared); }

template <int D, int QP, int KP>
int run(const kvc_attn_args & a, int ngr, cudaStream_t st) {
    static std::atomic<int> state[64];                   // 0 unknown, 1 ready, 2 does not fit
    int dev = 0;
    KVC_CUDA(cudaGetDevice(&dev));
    auto * k = k_tree_tc<D, QP, KP>;
    int s = state[dev & 63].load(std::memory_order_relaxed);
    if (s == 0) {
        // the register shares draw on what the block is launched with
        cudaFuncAttributes at;
        KVC_CUDA(cudaFuncGetAttributes(&at, k));
        s = at.numRegs * 4 >= 2 * REG_SOFTMAX + REG_PRODUCE + REG_MMA ? 1 : 2;
        KVC_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<D, QP, KP>()));
        state[dev & 63].store(s, std::memory_order_relaxed);
    }
    if (s == 2) {
        fprintf(stderr, "[kvc] k_tree_tc was built with too few registers per thread\n");
        return KVC_ERR_CUDA;
    }
    k<<<dim3((unsigned)a.W, (unsigned)a.Hkv), THREADS, smem_bytes<D, QP, KP>(), st>>>(a, ngr);
    g_serve_launches++;
    KVC_CUDA(cudaGetLastError());
    return kvc_launch_attn_join(a, true, st);
}

bool block_type(int t) { return t == KV_TYPE_Q8_0 || t == KV_TYPE_Q4_0 || t == KV_TYPE_Q4_1; }

}  // namespace

bool kvc_attn_tree_tc_plan(kvc_attn_args * a, int sms, long long * blocks) {
    const int top = a->dk > a->dv ? a->dk : a->dv;
    const long long rows = (long long)a->max_q * a->g;
    // k_tree_mma takes 32 rows at a time and its time grows with them; this
    // kernel's hardly does up to 128 rows, but putting two fp16 pieces of 128
    // values into the tiles costs it most. 43,000 keys x 8 heads, us here / there:
    //   rows                 32         36         64         80
    //   F16, d 64         65 / 71    65 / 99   68 / 105   69 / 172
    //   Q8_0, d 64       103 / 71  103 / 109  107 / 113  105 / 207
    //   F16, d 128       94 / 104   93 / 143   98 / 156  100 / 229
    //   Q8_0, d 128     208 / 117  208 / 165  211 / 175  211 / 296
    //   Q4_0, d 128     167 / 97   167 / 148  171 / 157  170 / 286
    // (F16 with 32 rows stays there: on short caches this kernel takes 25 us at
    // least, that one 19.)
    const long long few = a->k_type != KV_TYPE_F16 && top > 64 ? 64 : 32;
    if (rows <= few || top > 128 || a->dk % 32 || a->dv % 32) return false;
    if (a->k_type == KV_TYPE_F16 && a->v_type == KV_TYPE_F16) {
        // 16-byte pieces of a head's part of a row
        if (((uintptr_t)a->K | (uintptr_t)a->V | (uintptr_t)a->k_rb | (uintptr_t)a->v_rb) & 15) return false;
    } else if (block_type(a->k_type) && block_type(a->v_type)) {
        // words and half-words; Q4_1 blocks are read as words
        if (((uintptr_t)a->K | (uintptr_t)a->V) & 3) return false;
    } else {
        return false;
    }
    const long long n = (rows + TM - 1) / TM;
    if (n > 65535 || a->Hkv > 65535) return false;
    a->rb = TM;
    a->tile = TN;
    a->by_tile = kvc_make_divisor(TN);
    const long long w = sms / a->Hkv;                    // one CTA per SM; the row blocks are laid end to end
    a->W = (int)(w < 1 ? 1 : w);
    a->n_parts = 1;
    *blocks = n;
    return true;
}

int kvc_launch_attn_tree_tc(const kvc_attn_args & a, cudaStream_t st) {
    const int ngr = (int)(((long long)a.max_q * a.g + TM - 1) / TM);
    const bool wide = a.dk > 64 || a.dv > 64, f32 = a.q_type == KV_TYPE_F32, blocks = a.k_type != KV_TYPE_F16;
    if (wide) {
        if (f32) return blocks ? run<128, 2, 2>(a, ngr, st) : run<128, 2, 1>(a, ngr, st);
        return blocks ? run<128, 1, 2>(a, ngr, st) : run<128, 1, 1>(a, ngr, st);
    }
    if (f32) return blocks ? run<64, 2, 2>(a, ngr, st) : run<64, 2, 1>(a, ngr, st);
    return blocks ? run<64, 1, 2>(a, ngr, st) : run<64, 1, 1>(a, ngr, st);
}
