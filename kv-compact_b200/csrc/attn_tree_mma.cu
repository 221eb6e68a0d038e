// attn_tree_mma.cu — attention of drafted tokens over the paged cache on the
// warp-level tensor-core instructions (mma.sync m16n8k16, fp16 operands, fp32
// sums), for caches of F16, Q8_0, Q4_0 and Q4_1 rows.
//
// A decode step reads every stored byte once and does little with it: at one
// token per sequence and a group of four heads, 8 operations per value. The
// rows are therefore decoded straight into MMA fragments, in registers, and
// keys are the long side of the tile (M = 16 keys, N = 8 query rows), so that
// 8 query rows of a group fill it.
//
//   S[key][row] = sum_b dK[key][b] (sum_{i in b} code[key][i] Q[row][i])
//   O[i][row]   = sum_key code[key][i] (P[key][row] dV[key][b(i)])
//
// The codes of the block formats are small integers, exact in fp16; a block's
// scale is applied to its 32-value partial score on one side and to the
// probabilities on the other. With F32 queries both Q (times a power of two
// per row) and P dV (times a power of two, kept per warp) enter as two fp16
// pieces, 22 bits together; with F16 queries Q enters as it is and P dV is
// rounded once to fp16, as the output is. Q4_1's minima add m[key][b] (sum of
// Q over b) to the scores and a product of P m with ones to the output.
//
// One CTA per SM (16 or 8 warps) runs through its stretch of the keys with a
// ring of stages, each `tile` whole rows: the part of every row that belongs to
// the CTA's heads, loaded by TMA in boxes of as many rows as lie side by side
// in a page. The box is up to 31 bytes wider than that part, so that rows lie an
// odd number of 16 bytes apart and fragment reads meet no bank conflict. The
// warps take turns at refilling the ring, a tile or two behind the readers.
// A warp owns one KV head and one block of query rows for a sequence, takes
// every nsub-th group of 16 keys, and keeps its own maximum, sum and output;
// the warps of a head are joined at the end of the CTA's stretch of a
// sequence, the CTAs afterwards (k_attn_join). Rows or pages that TMA cannot
// read (row sizes that are no multiple of 16 bytes, pages without 8 rows side
// by side) are copied by all warps with cp.async instead.
//
// Bound by the work per key, not by memory: 160,000 Q8_0 keys of 8 heads, 4
// query rows each, 128 values take 141 us with F32 queries (2.5 TB/s of rows,
// 38 % of HBM's rate). 16 keys of a head cost about 1,000 instructions, 400 of
// them on the half-rate ALU pipe (codes to fp16, comparisons), and four warps per
// scheduler, all that 128 registers a thread allow, issue in 59 % of the cycles.
// 8 warps with twice the registers: 158 us.
#include "attn.h"
#include "attn_tree.h"
#include "attn_tc.h"

namespace {

constexpr int KEYS = 16;                  // keys of one MMA step
constexpr float LOG2E = 1.4426950408889634f;
constexpr int P_SHIFT = 10;               // P dV enters as P dV 2^(10 - R), R >= exponent of the largest dV so far
constexpr int MAX_STAGES = 8, MAX_TILE = 256, MAX_SEGS = 64;
constexpr uint32_t POLLS = 1u << 22;      // bound of every wait

struct mma_geom {
    int nw;                     // warps
    int hc, ngh;                // KV heads per CTA, groups of them
    int rc;                     // blocks of 8*NB query rows per CTA
    int kp, vp;                 // ring bytes per K / V row (16 * odd: no bank conflicts)
    int kg, vg;                 // cp.async piece: 16, 8 or 4 bytes
    int run;                    // rows per TMA box; 0: cp.async
    int bbox;                   // floats between the beta of two boxes
    int stages, stage_bytes;
    int lag;                    // tiles that a refill stays behind the reader
    int nbk, nbv;               // 32-value blocks per head
    int qvec;                   // rows of q may be read two elements at a time
    int ovec;                   // rows of out may be written four at a time
    kvc_divisor by_run;
};

// A piece of the CTA's stretch: key tiles lo .. hi-1 of one sequence.
struct segment {
    int lo, hi, slot;
    int q0, nq, nodes, ln;
    int table;                  // table row
};

__device__ __forceinline__ uint32_t smem_addr(const void * p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mma(float * d, const uint32_t * a, uint32_t b0, uint32_t b1, const float * c) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %11, %12, %13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
__device__ __forceinline__ void ldmatrix4(uint32_t * r, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t * r, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float2 unpack(uint32_t v) {
    __half2 h;
    memcpy(&h, &v, 4);
    return __half22float2(h);
}
__device__ __forceinline__ uint32_t hadd2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
__device__ __forceinline__ uint32_t lds16(const uint8_t * p) { return *reinterpret_cast<const uint16_t *>(p); }
// Four bytes at a 2-byte boundary; ALIGNED: at a 4-byte boundary.
template <bool ALIGNED>
__device__ __forceinline__ uint32_t lds32(const uint8_t * p) {
    if (ALIGNED) return *reinterpret_cast<const uint32_t *>(p);
    return lds16(p) | (lds16(p + 2) << 16);
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t pair16(uint32_t lo, uint32_t hi) { return __byte_perm(lo, hi, 0x5410); }
__device__ __forceinline__ float half_bits(uint32_t h) { return __half2float(__ushort_as_half((unsigned short)h)); }

// Two signed bytes (b0, b1 of v after v ^= 0x80808080) as fp16: 0x6400 | u is
// 1024 + u, and u = code + 128.
__device__ __forceinline__ uint32_t bytes_lo(uint32_t v) { return hadd2(__byte_perm(v, 0x64646464u, 0x4140), 0xE480E480u); }
__device__ __forceinline__ uint32_t bytes_hi(uint32_t v) { return hadd2(__byte_perm(v, 0x64646464u, 0x4342), 0xE480E480u); }
// Nibbles 0 and 4 (low) or 1 and 5 (high) of v as fp16 minus BIAS: 1024 + n,
// or (1024 + 16 n) / 16 = 64 + n.
template <int BIAS>
__device__ __forceinline__ uint32_t nibbles_lo(uint32_t v) {
    const uint32_t m = BIAS == 8 ? 0xE408E408u : 0xE400E400u;                 // -(1024 + BIAS)
    return hadd2((v & 0x000F000Fu) | 0x64006400u, m);
}
template <int BIAS>
__device__ __forceinline__ uint32_t nibbles_hi(uint32_t v) {
    const uint32_t m = BIAS == 8 ? 0xD480D480u : 0xD400D400u;                 // -(64 + BIAS)
    return hfma2((v & 0x00F000F0u) | 0x64006400u, 0x2C002C00u, m);
}

__device__ __forceinline__ constexpr int block_bytes(int type) {
    return type == KV_TYPE_Q8_0 ? 34 : type == KV_TYPE_Q4_0 ? 18 : type == KV_TYPE_Q4_1 ? 20 : 64;
}

// The dimension that accumulator row (r8: the upper eight) of lane group g
// stands for in m-tile mt of the output product.
__device__ __forceinline__ int v_dim(int type, int mt, int g, int r8) {
    return type == KV_TYPE_F16 ? 16 * mt + g + 8 * r8 : 4 * g + 2 * mt + r8;
}

// A fragments of the score product for block B: keys g and g + 8, both k-steps.
template <int KT, bool ODD>
__device__ __forceinline__ void k_frag(uint32_t a[2][4], const uint8_t * r0, const uint8_t * r1, uint32_t ld_addr, int t) {
    if (KT == KV_TYPE_F16) {
        ldmatrix4(a[0], ld_addr);
        ldmatrix4(a[1], ld_addr + 32);
    } else if (KT == KV_TYPE_Q8_0) {
#pragma unroll
        for (int s = 0; s < 2; s++) {
            const uint32_t x = lds32<ODD>(r0 + 2 + 4 * (t + 4 * s)) ^ 0x80808080u;
            const uint32_t y = lds32<ODD>(r1 + 2 + 4 * (t + 4 * s)) ^ 0x80808080u;
            a[s][0] = bytes_lo(x);
            a[s][1] = bytes_lo(y);
            a[s][2] = bytes_hi(x);
            a[s][3] = bytes_hi(y);
        }
    } else {
        constexpr int HEAD = KT == KV_TYPE_Q4_0 ? 2 : 4;
        constexpr bool AL = KT == KV_TYPE_Q4_1 || ODD;
        constexpr int BIAS = KT == KV_TYPE_Q4_0 ? 8 : 0;
        const uint32_t x = lds32<AL>(r0 + HEAD + 4 * t), y = lds32<AL>(r1 + HEAD + 4 * t);
        a[0][0] = nibbles_lo<BIAS>(x);
        a[0][1] = nibbles_lo<BIAS>(y);
        a[0][2] = nibbles_hi<BIAS>(x);
        a[0][3] = nibbles_hi<BIAS>(y);
        a[1][0] = nibbles_lo<BIAS>(x >> 8);
        a[1][1] = nibbles_lo<BIAS>(y >> 8);
        a[1][2] = nibbles_hi<BIAS>(x >> 8);
        a[1][3] = nibbles_hi<BIAS>(y >> 8);
    }
}

// A fragments of the output product for a block: dimensions 4g .. 4g+3 (two
// m-tiles) of keys 2t, 2t+1, 2t+8, 2t+9, whose rows start at `r` + key * vp.
// CENTRE: Q4_1 codes minus 8.
template <int VT, bool ODD, bool CENTRE>
__device__ __forceinline__ void v_frag(uint32_t a[2][4], const uint8_t * r, int vp, uint32_t ld_addr, int g) {
    if (VT == KV_TYPE_F16) {
        ldmatrix4_trans(a[0], ld_addr);
        ldmatrix4_trans(a[1], ld_addr + 32);
    } else if (VT == KV_TYPE_Q8_0) {
#pragma unroll
        for (int s = 0; s < 2; s++) {
            const uint32_t w0 = lds32<ODD>(r + (8 * s) * vp + 2 + 4 * g) ^ 0x80808080u;
            const uint32_t w1 = lds32<ODD>(r + (8 * s + 1) * vp + 2 + 4 * g) ^ 0x80808080u;
            const uint32_t x = __byte_perm(w0, w1, 0x5140), y = __byte_perm(w0, w1, 0x7362);
            a[0][2 * s] = bytes_lo(x);
            a[0][2 * s + 1] = bytes_hi(x);
            a[1][2 * s] = bytes_lo(y);
            a[1][2 * s + 1] = bytes_hi(y);
        }
    } else {
        constexpr int HEAD = VT == KV_TYPE_Q4_0 ? 2 : 4;
        constexpr int BIAS = VT == KV_TYPE_Q4_0 || CENTRE ? 8 : 0;
#pragma unroll
        for (int s = 0; s < 2; s++) {
            const uint32_t w = lds16(r + (8 * s) * vp + HEAD + 2 * g) | (lds16(r + (8 * s + 1) * vp + HEAD + 2 * g) << 16);
            a[0][2 * s] = nibbles_lo<BIAS>(w);
            a[0][2 * s + 1] = nibbles_hi<BIAS>(w);
            a[1][2 * s] = nibbles_lo<BIAS>(w >> 8);
            a[1][2 * s + 1] = nibbles_hi<BIAS>(w >> 8);
        }
    }
}

template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const uint8_t * src) {
    if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(dst), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" :: "r"(dst), "l"(src), "n"(BYTES) : "memory");
}
// One row's part, by a warp.
__device__ __forceinline__ void copy_row(uint32_t dst, const uint8_t * src, int g, int bytes, int lane) {
    if (g == 16) for (int o = 16 * lane; o < bytes; o += 512) copy_async<16>(dst + o, src + o);
    else if (g == 8) for (int o = 8 * lane; o < bytes; o += 256) copy_async<8>(dst + o, src + o);
    else for (int o = 4 * lane; o < bytes; o += 128) copy_async<4>(dst + o, src + o);
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const void * map, int x, int y, int z, uint64_t * bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 :: "r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_addr(bar)) : "memory");
}

// One slot of the shared region: a unit's query fragments in two pieces (in the
// loop), or a warp's output, maxima and sums (when the warps of a unit are joined).
constexpr int slot_bytes(int db, int nb) { return db * nb * 1024 + nb * 512; }

template <int DB, int NB, int NP, int MAXW, bool FULL>
__global__ void __launch_bounds__(32 * MAXW, 1) k_tree_mma(const __grid_constant__ kvc_attn_args a,
                                                           const __grid_constant__ mma_geom G,
                                                           const __grid_constant__ CUtensorMap k_map,
                                                           const __grid_constant__ CUtensorMap v_map,
                                                           const __grid_constant__ CUtensorMap b_map) {
    using namespace kvc_tc;
    constexpr int RW = 8 * NB;                           // query rows of a warp
    const int NBK = FULL ? DB : G.nbk, NBV = FULL ? DB : G.nbv;      // FULL: all blocks are there, no checks in the loops
    constexpr bool QS = NP == 2;                         // query fragments in shared memory
    constexpr int SLOT = slot_bytes(DB, NB);
    extern __shared__ __align__(128) uint8_t sm[];
    const int NW = G.nw, KT = a.tile;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const bool tma = G.run != 0;
    uint8_t * ring = sm;
    uint8_t * fixed = sm + (size_t)G.stages * G.stage_bytes;
    uint64_t * full = reinterpret_cast<uint64_t *>(fixed);
    uint64_t * empty = full + MAX_STAGES;
    uint32_t * bad = reinterpret_cast<uint32_t *>(empty + MAX_STAGES);       // [stages] boxes without a page
    int * n_segs = reinterpret_cast<int *>(bad + MAX_STAGES);                // [2]: of this batch, of all
    int * pages = n_segs + 8;                                                // [NW][32]
    segment * segs = reinterpret_cast<segment *>(pages + 32 * NW);
    float * qsum_all = reinterpret_cast<float *>(segs + MAX_SEGS);           // [NW][DB][RW]
    uint8_t * region = reinterpret_cast<uint8_t *>(qsum_all + NW * DB * RW);
    if (threadIdx.x == 0) {
        for (int i = 0; i < G.stages; i++) {
            mbar_init(full + i, tma ? 1 : 64 * NW);
            mbar_init(empty + i, NW);
        }
        mbar_init_fence();
    }
    cudaTriggerProgrammaticLaunchCompletion();           // the join may set up meanwhile; it waits for this grid

    const int hg = blockIdx.y % G.ngh, qb = blockIdx.y / G.ngh, w = blockIdx.x;
    const int h0 = hg * G.hc, nh = min(G.hc, a.Hkv - h0);
    // the heads' part of a row: where it starts, and from where it is copied
    const int k_at = h0 * (int)a.k_hb, v_at = h0 * (int)a.v_hb;
    const int k_off = tma || G.kg == 16 ? k_at & 15 : 0, v_off = tma || G.vg == 16 ? v_at & 15 : 0;
    const int kt = a.k_type, vt = a.v_type;
    const bool has_bias = !tma || a.beta != nullptr;
    float * qsum = qsum_all + warp * DB * RW;
    bool dead = false;                                   // a wait ran out: no more waits, the status says so
    auto await = [&](uint64_t * bar, uint32_t parity) {
        if (!dead && !mbar_wait_suspend(bar, parity, POLLS, 2000)) {
            dead = true;
            if (a.status) *a.status = KVC_ERR_CUDA;
        }
    };
    int c_stage = 0;                                     // next stage to read
    uint32_t c_phase = 0;
    int filled = 0;                                      // tiles of the batches before
    auto step = [&](int & st, uint32_t & ph) {
        if (++st == G.stages) {
            st = 0;
            ph ^= 1;
        }
    };

    for (int batch = 0;; batch += MAX_SEGS) {
        // ---- the pieces of this CTA's stretch, MAX_SEGS at a time
        __syncthreads();
        if (warp == 0) {
            int n = 0;
            attn_walk(a, qb, qb + 1, w, hg == 0, [&](int, const kvc_attn_seq & q, int lo, int hi, int slot) {
                if (n >= batch && n < batch + MAX_SEGS && lane == 0) {
                    segs[n - batch] = segment{lo, hi, slot, q.q0, q.nq, q.nodes, q.ln, q.slot};
                }
                n++;
            });
            if (lane == 0) {
                n_segs[0] = min(n - batch, MAX_SEGS);
                n_segs[1] = n;
            }
        }
        __syncthreads();
        const int ns = n_segs[0];

        // ---- filling: with TMA tile f of the batch is the business of warp f % NW alone (so that no warp has more to
        // do than another), with cp.async every warp's
        const int stride = tma ? NW : 1;
        int f_tile = tma ? warp : 0;                     // this warp's next tile to fill: its number in the batch,
        int f_seg = 0, f_at = ns > 0 ? segs[0].lo : 0;   // its piece and its tile there
        auto ahead = [&](int n) {
            f_at += n;
            while (f_seg < ns && f_at >= segs[f_seg].hi) {
                f_at -= segs[f_seg].hi;
                if (++f_seg < ns) f_at += segs[f_seg].lo;
            }
        };
        if (tma) ahead(warp);
        // TMA: the page of box `lane` of that tile, read ahead by an asynchronous copy
        int * p_page = pages + 32 * warp + lane;
        auto look = [&]() {
            if (f_seg < ns) {
                const segment & S = segs[f_seg];
                const long long j = (long long)f_at * KT + lane * G.run;
                if (lane * G.run < KT && j < S.ln)
                    copy_async<4>(smem_u32(p_page), reinterpret_cast<const uint8_t *>(
                                                       a.table + (size_t)S.table * a.max_pages + a.by_page.div((uint32_t)j)));
            }
        };
        auto fill = [&]() {
            if (f_seg >= ns) return;
            const segment & S = segs[f_seg];
            const int num = filled + f_tile, stage = num % G.stages;
            await(empty + stage, (num / G.stages & 1) ^ 1);
            uint8_t * st = ring + (size_t)stage * G.stage_bytes;
            uint8_t * sv = st + KT * G.kp;
            float * sb = reinterpret_cast<float *>(sv + KT * G.vp);
            uint64_t * bar = full + stage;
            if (tma) {
                const int k = lane * G.run;
                const long long j = (long long)f_at * KT + k;
                const bool want = k < KT && j < S.ln;
                asm volatile("cp.async.wait_all;" ::: "memory");
                const int page = want ? *p_page : -1;
                const bool have = page >= 0 && page < a.n_pages && !dead;
                const uint32_t boxes = __ballot_sync(~0u, have), missing = __ballot_sync(~0u, want && !have);
                if (lane == 0) {
                    bad[stage] = missing;
                    const uint32_t bytes = (uint32_t)G.run * (uint32_t)(G.kp + G.vp + (a.beta ? 4 * G.hc : 0));
                    mbar_arrive_expect_tx(bar, bytes * (uint32_t)__popc(boxes));
                }
                __syncwarp();
                if (have) {
                    const int off = (int)(j - (long long)a.by_page.div((uint32_t)j) * a.page);
                    const int row = page * a.page + off;
                    tma_load_2d(st + k * G.kp, &k_map, (k_at - k_off) >> 3, row, bar);
                    tma_load_2d(sv + k * G.vp, &v_map, (v_at - v_off) >> 3, row, bar);
                    if (a.beta) tma_load_3d(smem_addr(sb + lane * G.bbox), &b_map, off, h0, page, bar);
                }
            } else {
                // rows warp, warp + NW, ...; lane r knows the place of the r-th of them
                const int k0 = warp + NW * lane;
                const long long j = (long long)f_at * KT + k0;
                int row = -1;
                if (k0 < KT && j < S.ln) {
                    const int b = (int)a.by_page.div((uint32_t)j);
                    const int p = a.table[(size_t)S.table * a.max_pages + b];
                    if (p >= 0 && p < a.n_pages) row = p * a.page + (int)(j - (long long)b * a.page);
                }
                for (int r = 0; warp + NW * r < KT; r++) {
                    const int k = warp + NW * r;
                    const long long at = __shfl_sync(~0u, row, r);
                    for (int hh = lane; hh < nh; hh += 32) {
                        float b = at < 0 ? -INFINITY : 0.0f;
                        if (at >= 0 && a.beta) {
                            const uint32_t p = a.by_page.div((uint32_t)at);
                            b = a.beta[((size_t)p * a.Hkv + h0 + hh) * a.page + (at - (long long)p * a.page)];
                        }
                        sb[hh * KT + k] = b;
                    }
                    if (at < 0 || dead) continue;
                    copy_row(smem_addr(st + k * G.kp), a.K + at * a.k_rb + (k_at - k_off), G.kg,
                             (k_off + nh * (int)a.k_hb + G.kg - 1) & ~(G.kg - 1), lane);
                    copy_row(smem_addr(sv + k * G.vp), a.V + at * a.v_rb + (v_at - v_off), G.vg,
                             (v_off + nh * (int)a.v_hb + G.vg - 1) & ~(G.vg - 1), lane);
                }
                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" :: "r"(smem_addr(bar)) : "memory");
                mbar_arrive(bar);
            }
            f_tile += stride;
            ahead(stride);
            if (tma) look();
        };
        if (tma) look();
        while (f_seg < ns && f_tile < G.stages - G.lag) fill();
        int tile = 0;                                    // of the batch, being read

    int units_before = 0;
    for (int seg = 0; seg < ns; seg++) {
        const int lo = segs[seg].lo, hi = segs[seg].hi, slot = segs[seg].slot;
        kvc_attn_seq q;
        q.q0 = segs[seg].q0;
        q.nq = segs[seg].nq;
        q.nodes = segs[seg].nodes;
        q.ln = segs[seg].ln;
        // this warp's KV head, block of query rows and share of the keys
        const int rows_here = (int)min((long long)a.rb, (long long)q.nq * a.g - (long long)qb * a.rb);
        const int units = nh * ((rows_here + RW - 1) / RW);
        const int nsub = NW / units;
        if (units != units_before) __syncthreads();      // the units' barriers change hands
        units_before = units;
        const int sub = warp / units, unit = warp - sub * units;
        const bool active = sub < nsub;
        const int hc = unit % nh, h = h0 + hc;
        const int r0 = qb * a.rb + unit / nh * RW;
        const int nr = min(RW, rows_here - unit / nh * RW);
        // rows from here on are the nodes' own, and the mask decides on them (one node that sees itself needs none)
        const bool masked = a.mask && a.mask_words > 0 && !(q.nodes == 1 && (a.mask[(size_t)q.q0 * a.mask_words] & 1u));
        const int first_own = masked || (a.mask && !a.mask_words) ? q.ln - q.nodes : INT_MAX;

        // query fragments: lane (g, t) holds, of row g of each block of 8, the
        // elements that the k-steps of its K type ask of it; two pieces lie in
        // shared memory (32 registers less in the loop), written by a unit's
        // first warp
        uint32_t qf[QS ? 1 : DB][2][NB][2];
        uint4 * qs = reinterpret_cast<uint4 *>(region + (size_t)(active ? unit : 0) * SLOT) + lane;
        auto unit_sync = [&]() {                         // the warps of a unit
            if (nsub > 1) asm volatile("bar.sync %0, %1;" :: "r"(1 + unit), "r"(32 * nsub) : "memory");
            else __syncwarp();
        };
        float mul[NB][2];
#pragma unroll
        for (int nb = 0; nb < NB; nb++) {
            const int r = 8 * nb + g;
            const int i = (int)a.by_group.div(r0 + r);
            const long long at = (long long)(q.q0 + i) * a.q_stride + (long long)(h * a.g + (r0 + r - i * a.g)) * a.q_head;
            const bool there = active && r < nr;
            float x[DB][8];                              // in the order [k-step][element] of the fragments
#pragma unroll
            for (int b = 0; b < DB; b++) {
#pragma unroll
                for (int u = 0; u < 4; u++) {            // pairs of neighbouring elements
                    const int d = 32 * b + (kt == KV_TYPE_F16 ? 2 * t + 8 * u
                                            : kt == KV_TYPE_Q8_0 ? 4 * t + 2 * (u & 1) + 16 * (u >> 1) : 8 * t + 2 * u);
                    float2 v = make_float2(0.0f, 0.0f);
                    if (there && b < NBK) {
                        if (a.q_type == KV_TYPE_F16) {
                            const __half * p = reinterpret_cast<const __half *>(a.q) + at + d;
                            v = G.qvec ? __half22float2(*reinterpret_cast<const __half2 *>(p))
                                       : make_float2(__half2float(p[0]), __half2float(p[1]));
                        } else {
                            const float * p = reinterpret_cast<const float *>(a.q) + at + d;
                            v = G.qvec ? *reinterpret_cast<const float2 *>(p) : make_float2(p[0], p[1]);
                        }
                    }
                    x[b][2 * u] = v.x;
                    x[b][2 * u + 1] = v.y;
                }
                if (kt == KV_TYPE_Q4_0 || kt == KV_TYPE_Q4_1) {
                    // dimension i of the lane's eight is element e of step ks: i = 2 ks + (e >> 1) + 4 (e & 1)
                    const float y1 = x[b][1], y2 = x[b][2], y3 = x[b][3], y4 = x[b][4], y5 = x[b][5], y6 = x[b][6];
                    x[b][1] = y4;
                    x[b][2] = y1;
                    x[b][3] = y5;
                    x[b][4] = y2;
                    x[b][5] = y6;
                    x[b][6] = y3;
                }
            }
            float up = 1.0f, m = a.scale;
            if (NP == 2) {
                float top = 0.0f;
#pragma unroll
                for (int b = 0; b < DB; b++)
#pragma unroll
                    for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(x[b][e]));
                top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
                top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
                // largest value of the row in [2^13, 2^14): both pieces normal numbers
                if (top > 0.0f && top < INFINITY) {
                    const int e = min(13 - ilogbf(top), 100);
                    up = scalbnf(1.0f, e);
                    m = a.scale * scalbnf(1.0f, -e);
                }
            }
            mul[nb][0] = __shfl_sync(~0u, m, 8 * t);     // of rows 2t and 2t + 1
            mul[nb][1] = __shfl_sync(~0u, m, 8 * t + 4);
#pragma unroll
            for (int b = 0; b < DB; b++) {
                float sum = 0.0f;
#pragma unroll
                for (int ks = 0; ks < 2; ks++) {
                    uint32_t f[2], rest[2];
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        const float y0 = x[b][4 * ks + 2 * u] * up, y1 = x[b][4 * ks + 2 * u + 1] * up;
                        sum += y0 + y1;
                        f[u] = pack(y0, y1);
                        const float2 z = unpack(f[u]);
                        rest[u] = pack(y0 - z.x, y1 - z.y);
                    }
                    if (QS) {
                        if (sub == 0) qs[((b * 2 + ks) * NB + nb) * 32] = make_uint4(f[0], f[1], rest[0], rest[1]);
                    } else {
                        qf[QS ? 0 : b][ks][nb][0] = f[0];
                        qf[QS ? 0 : b][ks][nb][1] = f[1];
                    }
                }
                if (kt == KV_TYPE_Q4_1) {
                    sum += __shfl_xor_sync(~0u, sum, 1);
                    sum += __shfl_xor_sync(~0u, sum, 2);
                    if (t == 0) qsum[b * RW + r] = sum;
                }
            }
        }
        if (QS && active) unit_sync();
        else __syncwarp();
        float m[NB][2], l[NB][2], O[DB][2][NB][4];
#pragma unroll
        for (int nb = 0; nb < NB; nb++) {
            m[nb][0] = m[nb][1] = -INFINITY;
            l[nb][0] = l[nb][1] = 0.0f;
#pragma unroll
            for (int b = 0; b < DB; b++)
#pragma unroll
                for (int mt = 0; mt < 2; mt++)
#pragma unroll
                    for (int e = 0; e < 4; e++) O[b][mt][nb][e] = 0.0f;
        }
        int R = vt == KV_TYPE_F16 ? 0 : -1000;           // exponent that P dV is scaled by; -1000: none yet

        // 16 keys from j0 on, the k0-th of their tile; rows at ks / vs, the head's beta at sb
        auto group = [&](int j0, int k0, const uint8_t * ks, const uint8_t * vs, const float * sb, uint32_t missing) {
            const uint8_t * kr0 = ks + g * G.kp;
            const uint8_t * kr1 = kr0 + 8 * G.kp;
            // bias of key k of the group; -inf: not there, or hidden from the head
            auto key_bias = [&](int k) {
                if (j0 + k >= q.ln) return -INFINITY;
                if (!tma) return sb[hc * KT + k0 + k];
                float b = 0.0f;
                if (has_bias || missing) {
                    const int box = (int)G.by_run.div((uint32_t)(k0 + k));
                    if (has_bias) b = sb[box * G.bbox + hc * G.run + (k0 + k - box * G.run)];
                    if ((missing >> box) & 1u) b = -INFINITY;
                }
                return b;
            };
            const float b0 = key_bias(g), b1 = key_bias(g + 8);

            // ---- scores of 16 keys x RW rows: S[nb] = {(g, 2t), (g, 2t+1), (g+8, 2t), (g+8, 2t+1)}
            float S[NB][4];
#pragma unroll
            for (int nb = 0; nb < NB; nb++) S[nb][0] = S[nb][1] = S[nb][2] = S[nb][3] = 0.0f;
            const uint32_t k_ld = smem_addr(ks + ((lane & 7) + 8 * ((lane >> 3) & 1)) * G.kp + 16 * (lane >> 4));
            auto scores = [&](auto type) {
                constexpr int KT_ = decltype(type)::value;
#pragma unroll
                for (int b = 0; b < DB; b++) {
                    if (b < NBK) {
                        uint32_t fa[2][4];
                        const uint8_t * p0 = kr0 + b * block_bytes(KT_);
                        const uint8_t * p1 = kr1 + b * block_bytes(KT_);
                        if (b & 1) k_frag<KT_, true>(fa, p0, p1, k_ld + 64 * b, t);
                        else k_frag<KT_, false>(fa, p0, p1, k_ld + 64 * b, t);
                        float d0 = 1.0f, d1 = 1.0f, m0 = 0.0f, m1 = 0.0f;
                        if (KT_ != KV_TYPE_F16) {
                            d0 = half_bits(lds16(p0));
                            d1 = half_bits(lds16(p1));
                        }
                        if (KT_ == KV_TYPE_Q4_1) {
                            m0 = half_bits(lds16(p0 + 2));
                            m1 = half_bits(lds16(p1 + 2));
                        }
#pragma unroll
                        for (int nb = 0; nb < NB; nb++) {
                            float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                            for (int u = 0; u < 2; u++) {
                                if (QS) {                              // the small piece first
                                    const uint4 f = qs[((b * 2 + u) * NB + nb) * 32];
                                    mma(c, fa[u], f.z, f.w, c);
                                    mma(c, fa[u], f.x, f.y, c);
                                } else {
                                    mma(c, fa[u], qf[QS ? 0 : b][u][nb][0], qf[QS ? 0 : b][u][nb][1], c);
                                }
                            }
                            if (KT_ == KV_TYPE_Q4_1) {
                                const float2 s2 = *reinterpret_cast<const float2 *>(qsum + b * RW + 8 * nb + 2 * t);
                                S[nb][0] = fmaf(m0, s2.x, S[nb][0]);
                                S[nb][1] = fmaf(m0, s2.y, S[nb][1]);
                                S[nb][2] = fmaf(m1, s2.x, S[nb][2]);
                                S[nb][3] = fmaf(m1, s2.y, S[nb][3]);
                            }
                            S[nb][0] = fmaf(d0, c[0], S[nb][0]);
                            S[nb][1] = fmaf(d0, c[1], S[nb][1]);
                            S[nb][2] = fmaf(d1, c[2], S[nb][2]);
                            S[nb][3] = fmaf(d1, c[3], S[nb][3]);
                        }
                    }
                }
            };
            switch (kt) {
            case KV_TYPE_F16: scores(kvc_int<KV_TYPE_F16>{}); break;
            case KV_TYPE_Q8_0: scores(kvc_int<KV_TYPE_Q8_0>{}); break;
            case KV_TYPE_Q4_0: scores(kvc_int<KV_TYPE_Q4_0>{}); break;
            default: scores(kvc_int<KV_TYPE_Q4_1>{}); break;
            }

            // ---- softmax: running maximum per row (the 8 lane groups hold the keys), probabilities
            const bool own = j0 + KEYS > first_own;          // the group holds rows that the mask decides on
            const bool hidden = __any_sync(~0u, b0 == -INFINITY || b1 == -INFINITY);
            bool moved = false;
            float f[NB][2];
#pragma unroll
            for (int nb = 0; nb < NB; nb++) {
#pragma unroll
                for (int e = 0; e < 4; e++) S[nb][e] = fmaf(S[nb][e], mul[nb][e & 1], e < 2 ? b0 : b1);
                if (own || hidden) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        bool sees = (e < 2 ? b0 : b1) != -INFINITY;
                        if (own && sees) {
                            const int rr = r0 + 8 * nb + 2 * t + (e & 1);
                            sees = rr < r0 + nr && attn_sees(a, q, (int)a.by_group.div(rr), j0 + g + (e < 2 ? 0 : 8));
                        }
                        if (!sees) S[nb][e] = -INFINITY;
                    }
                }
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    float mt = fmaxf(S[nb][c], S[nb][c + 2]);
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) mt = fmaxf(mt, __shfl_xor_sync(~0u, mt, o));
                    const float mn = fmaxf(m[nb][c], mt);
                    const float base = mn == -INFINITY ? 0.0f : mn;
                    f[nb][c] = ex2((m[nb][c] - base) * LOG2E);
                    moved |= mn != m[nb][c];
                    m[nb][c] = mn;
                    S[nb][c] = ex2((S[nb][c] - base) * LOG2E);
                    S[nb][c + 2] = ex2((S[nb][c + 2] - base) * LOG2E);
                    l[nb][c] = fmaf(l[nb][c], f[nb][c], S[nb][c] + S[nb][c + 2]);
                }
            }
            if (__any_sync(~0u, moved)) {
#pragma unroll
                for (int b = 0; b < DB; b++)
#pragma unroll
                    for (int mt = 0; mt < 2; mt++)
#pragma unroll
                        for (int nb = 0; nb < NB; nb++)
#pragma unroll
                            for (int e = 0; e < 4; e++) O[b][mt][nb][e] *= f[nb][e & 1];
            }

            // ---- output
            // A key that some queries see and others do not may hold infinities or NaN: then value by value.
            auto by_value = [&]() {
                if (R == -1000) R = 0;
                const float up = scalbnf(1.0f, P_SHIFT - R);
                for (int k = 0; k < KEYS; k++) {
#pragma unroll
                    for (int nb = 0; nb < NB; nb++) {
                        const int from = (k & 7) * 4 + t;
                        const float x0 = __shfl_sync(~0u, S[nb][0], from), x1 = __shfl_sync(~0u, S[nb][1], from);
                        const float x2 = __shfl_sync(~0u, S[nb][2], from), x3 = __shfl_sync(~0u, S[nb][3], from);
                        const float p0 = (k < 8 ? x0 : x2) * up, p1 = (k < 8 ? x1 : x3) * up;
#pragma unroll
                        for (int b = 0; b < DB; b++)
#pragma unroll
                            for (int mt = 0; mt < 2; mt++)
#pragma unroll
                                for (int r8 = 0; r8 < 2; r8++) {
                                    if (b < NBV) {
                                        const float v = attn_elem(vs + k * G.vp, vt, 32 * b + v_dim(vt, mt, g, r8));
                                        if (p0 != 0.0f) O[b][mt][nb][2 * r8] = fmaf(p0, v, O[b][mt][nb][2 * r8]);
                                        if (p1 != 0.0f) O[b][mt][nb][2 * r8 + 1] = fmaf(p1, v, O[b][mt][nb][2 * r8 + 1]);
                                    }
                                }
                    }
                }
            };
            const uint32_t v_ld = smem_addr(vs + ((lane & 7) + 8 * (lane >> 4)) * G.vp + 16 * ((lane >> 3) & 1));
            const uint8_t * vk = vs + 2 * t * G.vp;      // keys 2t, 2t+1, 2t+8, 2t+9 are this lane's in the product
            auto product = [&](auto type) {
                constexpr int VT = decltype(type)::value;
                constexpr bool BLOCK = VT != KV_TYPE_F16;
                constexpr bool TWO = NP == 2 || BLOCK;   // P in two pieces
                // Q4_1 with one piece: codes minus 8 and m + 8 d, which nearly cancel no more
                constexpr bool CENTRE = VT == KV_TYPE_Q4_1 && NP == 1;
                uint32_t dl[DB], dh[DB];
                uint32_t live_l = ~0u, live_h = ~0u;     // rows hidden from the whole head: scales of 0
                uint32_t rs = 0x3C003C00u;               // 2^-R
                if (BLOCK) {
                    if (hidden) {
                        live_l = (key_bias(2 * t) == -INFINITY ? 0u : 0xFFFFu) |
                                 (key_bias(2 * t + 1) == -INFINITY ? 0u : 0xFFFF0000u);
                        live_h = (key_bias(2 * t + 8) == -INFINITY ? 0u : 0xFFFFu) |
                                 (key_bias(2 * t + 9) == -INFINITY ? 0u : 0xFFFF0000u);
                    }
                    uint32_t top = 0;
#pragma unroll
                    for (int b = 0; b < DB; b++) {
                        dl[b] = dh[b] = 0;
                        if (b < NBV) {
                            const uint8_t * p = vk + b * block_bytes(VT);
                            dl[b] = pair16(lds16(p), lds16(p + G.vp)) & live_l;
                            dh[b] = pair16(lds16(p + 8 * G.vp), lds16(p + 9 * G.vp)) & live_h;
                            top = __vmaxu2(top, __vmaxu2(dl[b] & 0x7FFF7FFFu, dh[b] & 0x7FFF7FFFu));
                            if (VT == KV_TYPE_Q4_1) {
                                const uint32_t x = pair16(lds16(p + 2), lds16(p + G.vp + 2)) & live_l;
                                const uint32_t y = pair16(lds16(p + 8 * G.vp + 2), lds16(p + 9 * G.vp + 2)) & live_h;
                                top = __vmaxu2(top, __vmaxu2(x & 0x7FFF7FFFu, y & 0x7FFF7FFFu));
                            }
                        }
                    }
                    top = __reduce_max_sync(~0u, max(top & 0xFFFFu, top >> 16));
                    if (top >= 0x7C00u) {
                        by_value();
                        return;
                    }
                    const int e = top ? max((int)(top >> 10), 1) - 15 : -14;    // |scale| < 2^(e+1)
                    if (own) {
                        // a node's row with scales far above the others' is not to cost the queries that do not see it
                        // their precision
                        int least = e;
                        if (R == -1000) {
#pragma unroll
                            for (int b = 0; b < DB; b++)
                                if (b < NBV) {
                                    const uint32_t x[4] = {dl[b] & 0x7FFFu, dl[b] >> 16 & 0x7FFFu, dh[b] & 0x7FFFu, dh[b] >> 16 & 0x7FFFu};
#pragma unroll
                                    for (int u = 0; u < 4; u++)
                                        if (x[u]) least = min(least, max((int)(x[u] >> 10), 1) - 15);
                                }
                            least = __reduce_min_sync(~0u, least);
                        } else {
                            least = R;
                        }
                        if (e > least + 8) {
                            by_value();
                            return;
                        }
                    }
                    if (e > R) {
                        if (R > -1000) {
                            const float fr = scalbnf(1.0f, R - e);
#pragma unroll
                            for (int b = 0; b < DB; b++)
#pragma unroll
                                for (int mt = 0; mt < 2; mt++)
#pragma unroll
                                    for (int nb = 0; nb < NB; nb++)
#pragma unroll
                                        for (int k = 0; k < 4; k++) O[b][mt][nb][k] *= fr;
                        }
                        R = e;
                    }
                    rs = pack(__int_as_float((127 - R) << 23), __int_as_float((127 - R) << 23));
                }
                // P 2^10 as B fragments: [nb][piece][keys 2t.. | 2t+8..]
                uint32_t pf[NB][2][2];
#pragma unroll
                for (int nb = 0; nb < NB; nb++)
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        const float x = S[nb][2 * u] * 1024.0f, y = S[nb][2 * u + 1] * 1024.0f;
                        const uint32_t hi2 = pack(x, y);
                        pf[nb][0][u] = transpose8(hi2);
                        if (TWO) {
                            const float2 k = unpack(hi2);
                            pf[nb][1][u] = transpose8(pack(x - k.x, y - k.y));
                        }
                    }
                // pieces of P times a factor per key (f: keys 2t, 2t+1 and 2t+8, 2t+9): the product's rounding
                // error is exact in fp16 (22 bits in all)
                auto times = [&](int nb, uint32_t fl, uint32_t fh, uint32_t bf[NP][2]) {
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        const uint32_t d = u ? fh : fl;
                        if (NP == 2) {
                            const uint32_t r = hmul2(pf[nb][0][u], d);
                            bf[0][u] = r;
                            bf[NP - 1][u] = hfma2(pf[nb][1][u], d, hfma2(pf[nb][0][u], d, r ^ 0x80008000u));
                        } else {
                            bf[0][u] = hfma2(pf[nb][0][u], d, hmul2(pf[nb][1][u], d));
                        }
                    }
                };
                auto add = [&](int b, int mt, int nb, const uint32_t * fa, const uint32_t bf[NP][2]) {
                    if (NP == 1) {
                        mma(O[b][mt][nb], fa, bf[0][0], bf[0][1], O[b][mt][nb]);
                    } else {                             // the group's sum apart, so that the running sum rounds to nearest
                        float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        mma(c, fa, bf[NP - 1][0], bf[NP - 1][1], c);
                        mma(c, fa, bf[0][0], bf[0][1], c);
#pragma unroll
                        for (int e = 0; e < 4; e++) O[b][mt][nb][e] += c[e];
                    }
                };
#pragma unroll
                for (int b = 0; b < DB; b++) {
                    if (b < NBV) {
                        uint32_t fa[2][4];
                        const uint8_t * p = vk + b * block_bytes(VT);
                        if (b & 1) v_frag<VT, true, CENTRE>(fa, p, G.vp, v_ld + 64 * b, g);
                        else v_frag<VT, false, CENTRE>(fa, p, G.vp, v_ld + 64 * b, g);
                        const uint32_t fl = hmul2(dl[b], rs), fh = hmul2(dh[b], rs);
#pragma unroll
                        for (int nb = 0; nb < NB; nb++) {
                            uint32_t bf[NP][2];
                            if (BLOCK) {
                                times(nb, fl, fh, bf);
                            } else {
#pragma unroll
                                for (int pc = 0; pc < NP; pc++) {
                                    bf[pc][0] = pf[nb][pc][0];
                                    bf[pc][1] = pf[nb][pc][1];
                                }
                            }
                            add(b, 0, nb, fa[0], bf);
                            add(b, 1, nb, fa[1], bf);
                            if (VT == KV_TYPE_Q4_1) {
                                const uint32_t ones[4] = {0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u};
                                uint32_t el = hmul2(pair16(lds16(p + 2), lds16(p + G.vp + 2)) & live_l, rs);
                                uint32_t eh = hmul2(pair16(lds16(p + 8 * G.vp + 2), lds16(p + 9 * G.vp + 2)) & live_h, rs);
                                if (CENTRE) {
                                    el = hfma2(fl, 0x48004800u, el);
                                    eh = hfma2(fh, 0x48004800u, eh);
                                }
                                times(nb, el, eh, bf);
                                add(b, 0, nb, ones, bf);
                                add(b, 1, nb, ones, bf);
                            }
                        }
                    }
                }
            };
            if (vt == KV_TYPE_F16) {
                if (hidden) {                            // rows that no query of the head sees: zeros, whatever they hold
                    unsigned rows = __ballot_sync(~0u, lane < KEYS && key_bias(lane & (KEYS - 1)) == -INFINITY);
                    while (rows) {
                        const int k = __ffs(rows) - 1;
                        rows &= rows - 1;
                        for (int o = lane; o < 4 * NBV; o += 32)
                            *reinterpret_cast<int4 *>(const_cast<uint8_t *>(vs) + k * G.vp + 16 * o) = make_int4(0, 0, 0, 0);
                    }
                    fence_smem_to_async();               // the next box goes over them
                    __syncwarp();
                }
                bool bad = false;
                if (own)
                    for (int k = 0; k < KEYS; k++)
                        for (int o = lane; o < 4 * NBV; o += 32) {
                            const uint4 v = *reinterpret_cast<const uint4 *>(vs + k * G.vp + 16 * o);
                            for (uint32_t x : {v.x, v.y, v.z, v.w})
                                bad |= (x & 0x7C00u) == 0x7C00u || (x & 0x7C000000u) == 0x7C000000u;
                        }
                if (__any_sync(~0u, bad)) by_value();
                else product(kvc_int<KV_TYPE_F16>{});
            } else if (vt == KV_TYPE_Q8_0) {
                product(kvc_int<KV_TYPE_Q8_0>{});
            } else if (vt == KV_TYPE_Q4_0) {
                product(kvc_int<KV_TYPE_Q4_0>{});
            } else {
                product(kvc_int<KV_TYPE_Q4_1>{});
            }
        };

        int turn = sub;                                  // groups until this warp's next one
        for (int i = lo; i < hi; i++) {
            await(full + c_stage, c_phase);
            const uint8_t * st = ring + (size_t)c_stage * G.stage_bytes;
            const uint8_t * sv = st + KT * G.kp;
            const uint32_t missing = tma ? bad[c_stage] : 0;
            const int keys = min(KT, q.ln - i * KT);
            for (int k = 0; k < keys; k += KEYS) {
                if (active && turn == 0)
                    group(i * KT + k, k, st + k * G.kp + k_off + hc * (int)a.k_hb, sv + k * G.vp + v_off + hc * (int)a.v_hb,
                          reinterpret_cast<const float *>(sv + KT * G.vp), missing);
                turn = turn == 0 ? nsub - 1 : turn - 1;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(empty + c_stage);
            step(c_stage, c_phase);
            if (f_tile == tile + G.stages - G.lag) fill();
            tile++;
        }

        // ---- join the warps of a unit, half of them giving their results to the other half at a time
#pragma unroll
        for (int nb = 0; nb < NB; nb++)
#pragma unroll
            for (int c = 0; c < 2; c++)
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) l[nb][c] += __shfl_xor_sync(~0u, l[nb][c], o);
        if (!active) continue;
        float back = R > -1000 ? scalbnf(1.0f, R - P_SHIFT) : 0.0f;    // of this warp's O
        if (nsub > 1) unit_sync();                       // the fragments have been read
        for (int n = nsub; n > 1;) {
            const int half = (n + 1) / 2;
            if (sub >= half && sub < n) {
                float4 * o = reinterpret_cast<float4 *>(region + (size_t)(unit + units * (sub - half)) * SLOT) + lane;
#pragma unroll
                for (int nb = 0; nb < NB; nb++) {
#pragma unroll
                    for (int b = 0; b < DB; b++)
#pragma unroll
                        for (int mt = 0; mt < 2; mt++)
                            o[((b * 2 + mt) * NB + nb) * 32] = make_float4(O[b][mt][nb][0] * back, O[b][mt][nb][1] * back,
                                                                           O[b][mt][nb][2] * back, O[b][mt][nb][3] * back);
                    o[(DB * 2 * NB + nb) * 32] = make_float4(m[nb][0], m[nb][1], l[nb][0], l[nb][1]);
                }
            }
            unit_sync();
            if (sub < n - half) {
                const float4 * o = reinterpret_cast<const float4 *>(region + (size_t)(unit + units * sub) * SLOT) + lane;
#pragma unroll
                for (int nb = 0; nb < NB; nb++) {
                    const float4 ml = o[(DB * 2 * NB + nb) * 32];
                    float f0[2], f1[2];
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        const float om = c ? ml.y : ml.x, ol = c ? ml.w : ml.z;
                        const float mn = fmaxf(m[nb][c], om), base = mn == -INFINITY ? 0.0f : mn;
                        f0[c] = ex2((m[nb][c] - base) * LOG2E);
                        f1[c] = ex2((om - base) * LOG2E);
                        l[nb][c] = l[nb][c] * f0[c] + ol * f1[c];
                        m[nb][c] = mn;
                        f0[c] *= back;
                    }
#pragma unroll
                    for (int b = 0; b < DB; b++)
#pragma unroll
                        for (int mt = 0; mt < 2; mt++) {
                            const float4 v = o[((b * 2 + mt) * NB + nb) * 32];
                            O[b][mt][nb][0] = O[b][mt][nb][0] * f0[0] + v.x * f1[0];
                            O[b][mt][nb][1] = O[b][mt][nb][1] * f0[1] + v.y * f1[1];
                            O[b][mt][nb][2] = O[b][mt][nb][2] * f0[0] + v.z * f1[0];
                            O[b][mt][nb][3] = O[b][mt][nb][3] * f0[1] + v.w * f1[1];
                        }
                }
                back = 1.0f;
            }
            n = half;
            if (n > 1) unit_sync();
        }
        if (sub == 0) {
#pragma unroll
            for (int nb = 0; nb < NB; nb++)
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const int r = 8 * nb + 2 * t + c;
                    if (r >= nr) continue;
                    const int rr = r0 - qb * a.rb + r, i = (int)a.by_group.div(r0 + r);
                    const size_t out = (size_t)(q.q0 + i) * a.Hq + h * a.g + (r0 + r - i * a.g);
                    float * part = slot >= 0 ? attn_part(a, qb, h, w, slot) : nullptr;
                    const float M = m[nb][c], L = l[nb][c];
                    const float mul_o = part ? back : L > 0.0f ? back / L : (L == 0.0f ? 0.0f : L);
                    if (g == 0) {
                        if (part) {
                            part[a.rb * a.dv + rr] = M;
                            part[a.rb * a.dv + a.rb + rr] = L;
                        } else if (a.lse) {
                            a.lse[out] = L == 0.0f ? -INFINITY : M + logf(L);
                        }
                    }
#pragma unroll
                    for (int b = 0; b < DB; b++) {
                        if (b >= NBV) break;
                        const float v[4] = {O[b][0][nb][c] * mul_o, O[b][0][nb][2 + c] * mul_o, O[b][1][nb][c] * mul_o,
                                            O[b][1][nb][2 + c] * mul_o};
                        if (vt == KV_TYPE_F16) {
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                const int d = 32 * b + v_dim(KV_TYPE_F16, e >> 1, g, e & 1);
                                if (part) part[rr * a.dv + d] = v[e];
                                else if (a.q_type == KV_TYPE_F16) reinterpret_cast<__half *>(a.out)[out * a.dv + d] = __float2half_rn(v[e]);
                                else reinterpret_cast<float *>(a.out)[out * a.dv + d] = v[e];
                            }
                        } else {                         // four neighbouring dimensions
                            const int d = 32 * b + 4 * g;
                            float * f = part ? part + rr * a.dv + d : reinterpret_cast<float *>(a.out) + out * a.dv + d;
                            if (part || (a.q_type == KV_TYPE_F32 && G.ovec)) {
                                *reinterpret_cast<float4 *>(f) = make_float4(v[0], v[1], v[2], v[3]);
                            } else if (a.q_type == KV_TYPE_F32) {
#pragma unroll
                                for (int e = 0; e < 4; e++) f[e] = v[e];
                            } else {
                                __half * o = reinterpret_cast<__half *>(a.out) + out * a.dv + d;
                                if (G.ovec) {
                                    *reinterpret_cast<uint2 *>(o) = make_uint2(pack(v[0], v[1]), pack(v[2], v[3]));
                                } else {
#pragma unroll
                                    for (int e = 0; e < 4; e++) o[e] = __float2half_rn(v[e]);
                                }
                            }
                        }
                    }
                }
        }
        // the region is free again (the next piece's fragments go there)
        if (nsub > 1) unit_sync();
        else __syncwarp();
    }
        filled += tile;
        if (n_segs[1] <= batch + MAX_SEGS) break;
    }
    if (dead && threadIdx.x < G.stages) {                // copies in flight land before the CTA ends
        mbar_wait(full + threadIdx.x, 0, POLLS);
        mbar_wait(full + threadIdx.x, 1, POLLS);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

int round_pitch(int bytes) {
    int p = (bytes + 15) & ~15;
    return (p / 16) % 2 ? p : p + 16;
}

constexpr int SMEM_MOST = 227 * 1024;

// Shared memory besides the ring, for that many (KV head, row block) units.
template <int DB, int NB, int NP, int MAXW>
int fixed_bytes(int nw, int units) {
    const int slots = NP == 2 && units > nw / 2 ? units : nw / 2;
    return MAX_STAGES * (8 + 8 + 4) + 32 + nw * 128 + MAX_SEGS * (int)sizeof(segment) + nw * 8 * NB * DB * 4 + slots * slot_bytes(DB, NB);
}

// Ring geometry and split, or false where the rows are not ones that the kernel reads.
using fixed_fn = int (*)(int, int);
bool geometry(const kvc_attn_args & a, int rw, int nw, fixed_fn fixed, mma_geom * G, int * tile) {
    if (a.k_type == KV_TYPE_F32 || a.v_type == KV_TYPE_F32 || a.dk % 32 || a.dv % 32) return false;
    auto piece = [](const void * base, long long rb, long long hb) {
        const uintptr_t all = (uintptr_t)base | (uintptr_t)rb;
        if ((all | (uintptr_t)hb) & 3) return 0;
        return (all & 15) == 0 ? 16 : ((all | (uintptr_t)hb) & 7) == 0 ? 8 : 4;
    };
    G->nw = nw;
    G->kg = piece(a.K, a.k_rb, a.k_hb);
    G->vg = piece(a.V, a.v_rb, a.v_hb);
    if (!G->kg || !G->vg) return false;
    G->nbk = a.dk / 32;
    G->nbv = a.dv / 32;
    G->ovec = (uintptr_t)a.out % (a.q_type == KV_TYPE_F32 ? 16 : 8) == 0;
    G->qvec = ((uintptr_t)a.q % (a.q_type == KV_TYPE_F32 ? 8 : 4)) == 0 && a.q_stride % 2 == 0;
    const long long rows = (long long)a.max_q * a.g, qb = (rows + rw - 1) / rw;
    // all row blocks of a head in one CTA where they fit, so that its rows are read once
    const long long ngr = (qb + nw - 1) / nw;
    G->rc = (int)((qb + ngr - 1) / ngr);
    auto pitch = [&](int hc, long long hb) { return round_pitch(hc * (int)hb + ((hb & 15) ? 15 : 0)); };
    // as many heads per CTA as leave a stage of 16 keys under 40 KB and a row in a TMA box (256 x 8 bytes)
    int hc = nw / G->rc < a.Hkv ? nw / G->rc : a.Hkv;
    while (hc > 1 && (KEYS * (pitch(hc, a.k_hb) + pitch(hc, a.v_hb)) > 40 * 1024 || pitch(hc, a.k_hb) > 2048 ||
                      pitch(hc, a.v_hb) > 2048))
        hc--;
    G->ngh = (a.Hkv + hc - 1) / hc;
    G->hc = (a.Hkv + G->ngh - 1) / G->ngh;
    G->kp = pitch(G->hc, a.k_hb);
    G->vp = pitch(G->hc, a.v_hb);
    // a stage of about 32 KB (16 to 256 keys), 2 to 8 of them
    int kt = 32 * 1024 / (KEYS * (G->kp + G->vp)) * KEYS;
    kt = kt < KEYS ? KEYS : kt > MAX_TILE ? MAX_TILE : kt;
    // rows side by side in a page that divide the tile: TMA boxes, at most 32 per tile, from 128-byte boundaries
    int run = 1;
    while (run < kt && run < a.page && a.page % (2 * run) == 0 && kt % (2 * run) == 0) run *= 2;
    const bool tma = G->kg == 16 && G->vg == 16 && run >= 8 && G->kp <= 2048 && G->vp <= 2048 &&
                     (!a.beta || ((uintptr_t)a.beta & 15) == 0);
    if (tma && kt > 32 * run) kt = 32 * run;
    G->run = tma ? run : 0;
    G->by_run = kvc_make_divisor((uint32_t)run);
    G->bbox = (run * G->hc * 4 + 127) / 128 * 32;
    if (!tma && kt > 32 * nw) kt = 32 * nw;              // a lane per row of a warp's share
    *tile = kt;
    const int bias = tma ? (a.beta ? kt / run * G->bbox * 4 : 0) : kt * G->hc * 4;
    G->stage_bytes = (kt * (G->kp + G->vp) + bias + 127) & ~127;
    G->stages = (SMEM_MOST - fixed(nw, G->hc * G->rc)) / G->stage_bytes;
    if (G->stages > MAX_STAGES) G->stages = MAX_STAGES;
    G->lag = G->stages >= 4 ? 2 : 1;
    return G->stages >= 2;
}

// Rows of `rb` bytes as 8-byte elements; a box is `pitch` bytes of `run` rows (bytes past the row read as 0).
bool row_map(CUtensorMap * m, const void * base, long long rb, long long rows, int pitch, int run) {
    const cuuint64_t dims[2] = {(cuuint64_t)rb / 8, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)rb};
    const cuuint32_t box[2] = {(cuuint32_t)pitch / 8, (cuuint32_t)run}, one[2] = {1, 1};
    return kvc_tensor_map_encoder()(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT64, 2, const_cast<void *>(base), dims, strides, box, one,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
bool beta_map(CUtensorMap * m, const kvc_attn_args & a, int hc, int run) {
    const cuuint64_t dims[3] = {(cuuint64_t)a.page, (cuuint64_t)a.Hkv, (cuuint64_t)a.n_pages};
    const cuuint64_t strides[2] = {(cuuint64_t)a.page * 4, (cuuint64_t)a.page * a.Hkv * 4};
    const cuuint32_t box[3] = {(cuuint32_t)run, (cuuint32_t)hc, 1}, one[3] = {1, 1, 1};
    return kvc_tensor_map_encoder()(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, const_cast<float *>(a.beta), dims, strides, box, one,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DB, int NB, int NP, int MAXW, bool FULL>
int run(const kvc_attn_args & a, const mma_geom & G, int ngr, cudaStream_t st) {
    static std::atomic<bool> set[64];
    int dev = 0;
    KVC_CUDA(cudaGetDevice(&dev));
    auto * k = k_tree_mma<DB, NB, NP, MAXW, FULL>;
    if (!set[dev & 63].load(std::memory_order_relaxed)) {
        KVC_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_MOST));
        set[dev & 63].store(true, std::memory_order_relaxed);
    }
    CUtensorMap maps[3] = {};
    if (G.run) {
        const long long rows = (long long)a.n_pages * a.page;
        if (!row_map(&maps[0], a.K, a.k_rb, rows, G.kp, G.run) || !row_map(&maps[1], a.V, a.v_rb, rows, G.vp, G.run) ||
            (a.beta && !beta_map(&maps[2], a, G.hc, G.run))) {
            fprintf(stderr, "[kvc] cuTensorMapEncodeTiled failed for a cache of %d pages\n", a.n_pages);
            return KVC_ERR_CUDA;
        }
    }
    const int sm = fixed_bytes<DB, NB, NP, MAXW>(G.nw, G.hc * G.rc) + G.stages * G.stage_bytes;
    k<<<dim3((unsigned)a.W, (unsigned)(G.ngh * ngr)), 32 * G.nw, sm, st>>>(a, G, maps[0], maps[1], maps[2]);
    g_serve_launches++;
    KVC_CUDA(cudaGetLastError());
    return kvc_launch_attn_join(a, true, st);
}

using run_fn = int (*)(const kvc_attn_args &, const mma_geom &, int, cudaStream_t);
struct variant {
    int db, nb, np, full, warps;
    fixed_fn fixed;
    run_fn run;
};
#define TREE_VARIANT(DB, NB, NP, W) \
    {DB, NB, NP, 0, W, fixed_bytes<DB, NB, NP, W>, run<DB, NB, NP, W, false>}, {DB, NB, NP, 1, W, fixed_bytes<DB, NB, NP, W>, run<DB, NB, NP, W, true>}
// Up to 8 query rows per KV head (single tokens): 16 warps of 8 rows. More rows: 8 warps of 16 rows, whose
// registers hold twice the output. d > 128: twice that again, 8 warps of 8 rows. Each with and without checks of
// the head's blocks (d_k = d_v = 32 DB: without; the checks cost the call of the header's figure 15 %).
const variant variants[] = {
    TREE_VARIANT(2, 1, 1, 16), TREE_VARIANT(2, 1, 2, 16), TREE_VARIANT(4, 1, 1, 16), TREE_VARIANT(4, 1, 2, 16),
    TREE_VARIANT(2, 2, 1, 8),  TREE_VARIANT(2, 2, 2, 8),  TREE_VARIANT(4, 2, 1, 8),  TREE_VARIANT(4, 2, 2, 8),
    TREE_VARIANT(8, 1, 1, 8),  TREE_VARIANT(8, 1, 2, 8),
};

const variant & select(const kvc_attn_args & a) {
    const int top = a.dk > a.dv ? a.dk : a.dv;
    const int db = top <= 64 ? 2 : top <= 128 ? 4 : 8;
    const int nb = db == 8 || (long long)a.max_q * a.g <= 8 ? 1 : 2;
    const int np = a.q_type == KV_TYPE_F32 ? 2 : 1;
    const int full = a.dk == 32 * db && a.dv == 32 * db;
    for (const variant & v : variants)
        if (v.db == db && v.nb == nb && v.np == np && v.full == full) return v;
    return variants[0];
}

bool plan(const kvc_attn_args & a, mma_geom * G, int * tile, int * ngr) {
    const variant & v = select(a);
    if (!geometry(a, 8 * v.nb, v.warps, v.fixed, G, tile)) return false;
    const long long qb = ((long long)a.max_q * a.g + 8 * v.nb - 1) / (8 * v.nb);
    const long long n = (qb + G->rc - 1) / G->rc;
    if (n * G->ngh > 65535 || (G->run && !kvc_tensor_map_encoder())) return false;
    *ngr = (int)n;
    return true;
}

}  // namespace

bool kvc_attn_tree_mma_plan(kvc_attn_args * a, int sms, long long * blocks) {
    mma_geom G;
    int tile, ngr;
    if (!plan(*a, &G, &tile, &ngr)) return false;
    a->rb = 8 * select(*a).nb * G.rc;
    a->tile = tile;
    a->by_tile = kvc_make_divisor((uint32_t)tile);
    const int w = sms / (G.ngh * ngr);                   // one CTA per SM, equal stretches
    a->W = w < 1 ? 1 : w;
    a->n_parts = ngr;
    *blocks = ngr;
    return true;
}

int kvc_launch_attn_tree_mma(const kvc_attn_args & a, cudaStream_t st) {
    mma_geom G;
    int tile, ngr;
    if (!plan(a, &G, &tile, &ngr)) return KVC_ERR_SHAPE;
    return select(a).run(a, G, ngr, st);
}
