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
// probabilities on the other, in fp32. With F32 queries both Q (times a power
// of two per row) and P dV (times a power of two, kept per warp) enter as two
// fp16 pieces, 22 bits together; with F16 queries as one. Q4_1's minima add
// m[key][b] (sum of Q over b) and a product of P m with ones.
//
// A warp works alone: 16 keys per step through its own ring of asynchronous
// copies, its own running maximum, sum and output, no barrier in the loop; the
// four warps of a CTA and the CTAs of a sequence are joined at the end.
#include "attn.h"
#include "attn_tree.h"

#include <math.h>

namespace {

constexpr int WARPS = 4, THREADS = 128, KEYS = 16;
constexpr int TILE = WARPS * KEYS;
constexpr float LOG2E = 1.4426950408889634f;
constexpr int P_SHIFT = 13;               // P dV enters as P dV 2^(13 - R), R >= exponent of the largest dV so far

struct mma_geom {
    int kp, vp;                 // ring bytes per K / V row (16 * odd: no bank conflicts)
    int kseg, vseg;             // bytes of a head's part of a row
    int kg, vg;                 // copy piece: 16, 8 or 4 bytes
    int stages;
    int ring;                   // bytes of the rings (and of the join's buffer)
    int nbk, nbv;               // 32-value blocks per head
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
template <int VT, bool ODD>
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
        constexpr int BIAS = VT == KV_TYPE_Q4_0 ? 8 : 0;
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
__device__ __forceinline__ void copy_async(uint32_t dst, const uint8_t * src, bool real) {
    const int n = real ? BYTES : 0;
    if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(dst), "l"(src), "r"(n) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" :: "r"(dst), "l"(src), "n"(BYTES), "r"(n) : "memory");
}

// One row's part for one head: `pieces` pieces of g bytes, four lanes side by side.
__device__ __forceinline__ void copy_row(uint32_t dst, const uint8_t * src, bool real, int g, int bytes, int t) {
    if (g == 16) {
        for (int o = 16 * t; o < bytes; o += 64) copy_async<16>(dst + o, src + o, real);
    } else if (g == 8) {
        for (int o = 8 * t; o < bytes; o += 32) copy_async<8>(dst + o, src + o, real);
    } else {
        for (int o = 4 * t; o < bytes; o += 16) copy_async<4>(dst + o, src + o, real);
    }
}

template <int DB, int NB, int NP>
__global__ void __launch_bounds__(THREADS) k_tree_mma(const __grid_constant__ kvc_attn_args a,
                                                      const __grid_constant__ mma_geom G) {
    constexpr int RB = 8 * NB;
    constexpr bool QREG = NB == 1 && DB <= 4;            // query fragments stay in registers
    extern __shared__ __align__(16) uint8_t sm[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int h = blockIdx.y % a.Hkv, qb = blockIdx.y / a.Hkv, w = blockIdx.x;
    uint2 * qf = reinterpret_cast<uint2 *>(sm);          // [DB][2][NP][NB][32 lanes] query fragments
    float * qsum = reinterpret_cast<float *>(qf + DB * 2 * NP * NB * 32);   // [DB][RB] sums of Q over a block
    float * qmul = qsum + DB * RB;                       // [RB] scale / power of two of the row
    float * jm = qmul + RB;                              // [WARPS][RB] maxima, [WARPS][RB] sums (join)
    float * jl = jm + WARPS * RB;
    uint8_t * ring_all = reinterpret_cast<uint8_t *>(jl + WARPS * RB);
    const int stage_bytes = KEYS * (G.kp + G.vp) + KEYS * 4;
    uint8_t * ring = ring_all + (size_t)warp * G.stages * stage_bytes;
    // where the head's part of a row starts, and from where it is copied
    const long long k_at = (long long)h * a.k_hb, v_at = (long long)h * a.v_hb;
    const int k_off = G.kg == 16 ? (int)(k_at & 15) : 0, v_off = G.vg == 16 ? (int)(v_at & 15) : 0;
    const int k_copy = G.kg == 16 ? (k_off + G.kseg + 15) & ~15 : G.kseg;
    const int v_copy = G.vg == 16 ? (v_off + G.vseg + 15) & ~15 : G.vseg;
    const uint8_t * Kh = a.K + (k_at - k_off);
    const uint8_t * Vh = a.V + (v_at - v_off);
    const int kt = a.k_type, vt = a.v_type;

    attn_walk<RB, TILE>(a, qb, w, [&](int s, int lo, int hi, int slot) {
        const kvc_attn_seq q = attn_seq(a, s);
        const int r0 = qb * RB;
        const int nr = (int)min((long long)RB, (long long)q.nq * a.g - r0);
        const int first_own = q.ln - q.nq;               // rows from here on are the nodes' own
        __syncthreads();
        // query fragments: a warp takes rows warp, warp + 4, ...
        for (int r = warp; r < RB; r += WARPS) {
            float v[DB];
            float top = 0.0f;
            const int i = (int)a.by_group.div(r0 + r);
            const long long at = (long long)(q.q0 + i) * a.q_stride + (long long)(h * a.g + (r0 + r - i * a.g)) * a.q_head;
#pragma unroll
            for (int b = 0; b < DB; b++) {
                v[b] = 0.0f;
                if (r < nr && b < G.nbk) {
                    const long long e = at + 32 * b + lane;
                    v[b] = a.q_type == KV_TYPE_F16 ? __half2float(reinterpret_cast<const __half *>(a.q)[e])
                                                   : reinterpret_cast<const float *>(a.q)[e];
                }
                top = fmaxf(top, fabsf(v[b]));
            }
            float up = 1.0f, mul = a.scale;
            if (NP == 2) {
#pragma unroll
                for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
                // largest value of the row in [2^13, 2^14): both pieces normal numbers
                if (top > 0.0f && top < INFINITY) {
                    const int e = min(max(13 - ilogbf(top), -100), 100);
                    up = scalbnf(1.0f, e);
                    mul = a.scale * scalbnf(1.0f, -e);
                }
            }
            if (lane == 0) qmul[r] = mul;
#pragma unroll
            for (int b = 0; b < DB; b++) {
                const float x = v[b] * up;
                float sum = x;
#pragma unroll
                for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
                if (lane == 0) qsum[b * RB + r] = sum;
                // element `lane` of the block goes to the fragment that reads it
                int fs, ft, fe;
                if (kt == KV_TYPE_F16) {
                    fs = lane >> 4;
                    ft = (lane & 7) >> 1;
                    fe = (lane & 1) + 2 * ((lane >> 3) & 1);
                } else if (kt == KV_TYPE_Q8_0) {
                    fs = lane >> 4;
                    ft = (lane & 15) >> 2;
                    fe = lane & 3;
                } else {
                    ft = lane >> 3;
                    fs = (lane >> 1) & 1;
                    fe = 2 * (lane & 1) + ((lane >> 2) & 1);
                }
                __half * f = reinterpret_cast<__half *>(qf);
                const int nb = r >> 3, n = r & 7;
                const __half hi16 = __float2half_rn(x);
                f[((((b * 2 + fs) * NP + 0) * NB + nb) * 32 + n * 4 + ft) * 4 + fe] = hi16;
                if (NP == 2)
                    f[((((b * 2 + fs) * NP + 1) * NB + nb) * 32 + n * 4 + ft) * 4 + fe] =
                        __float2half_rn(x - __half2float(hi16));
            }
        }
        __syncthreads();
        uint2 qr[QREG ? DB : 1][2][NP];
        if (QREG) {
#pragma unroll
            for (int b = 0; b < DB; b++)
#pragma unroll
                for (int st = 0; st < 2; st++)
#pragma unroll
                    for (int p = 0; p < NP; p++) qr[QREG ? b : 0][st][p] = qf[((b * 2 + st) * NP + p) * NB * 32 + lane];
        }
        float mul[NB][2];
#pragma unroll
        for (int nb = 0; nb < NB; nb++) {
            mul[nb][0] = qmul[8 * nb + 2 * t];
            mul[nb][1] = qmul[8 * nb + 2 * t + 1];
        }
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
        int R = -1000;                                   // exponent that P dV is scaled by; none yet
        if (vt == KV_TYPE_F16) R = 0;

        // ---- the ring: steps of 16 keys, table entries two steps ahead, beta one
        const int end = min(hi * TILE, q.ln);
        const int j00 = (lo * WARPS + warp) * KEYS;
        const int steps = j00 < end ? (end - j00 + TILE - 1) / TILE : 0;
        int pg[2];
        long long row[2];
        float bias[2];
        auto fetch_table = [&](int i) {
#pragma unroll
            for (int r = 0; r < 2; r++) {
                const int j = j00 + i * TILE + g + 8 * r;
                pg[r] = i < steps && j < end ? q.table[a.by_page.div((uint32_t)j)] : -1;
            }
        };
        auto fetch_bias = [&](int i) {
#pragma unroll
            for (int r = 0; r < 2; r++) {
                const int j = j00 + i * TILE + g + 8 * r;
                row[r] = -1;
                bias[r] = -INFINITY;
                if (pg[r] >= 0 && pg[r] < a.n_pages) {
                    const int off = j - (int)a.by_page.div((uint32_t)j) * a.page;
                    row[r] = (long long)pg[r] * a.page + off;
                    bias[r] = a.beta ? a.beta[((size_t)pg[r] * a.Hkv + h) * a.page + off] : 0.0f;
                }
            }
        };
        auto issue = [&](int i) {
            if (i < steps) {
                uint8_t * st = ring + (i % G.stages) * stage_bytes;
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    const bool real = row[r] >= 0 && bias[r] != -INFINITY;   // rows that nobody sees are read as zeros
                    const long long at = real ? row[r] : 0;
                    copy_row(smem_addr(st + (g + 8 * r) * G.kp), Kh + at * a.k_rb, real, G.kg, k_copy, t);
                    copy_row(smem_addr(st + KEYS * G.kp + (g + 8 * r) * G.vp), Vh + at * a.v_rb, real, G.vg, v_copy, t);
                    if (t == 0) reinterpret_cast<float *>(st + KEYS * (G.kp + G.vp))[g + 8 * r] = bias[r];
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            fetch_bias(i + 1);
            fetch_table(i + 2);
        };
        fetch_table(0);
        fetch_bias(0);
        fetch_table(1);
        for (int i = 0; i < G.stages - 1; i++) issue(i);

        for (int i = 0; i < steps; i++) {
            if (G.stages == 4) asm volatile("cp.async.wait_group 2;" ::: "memory");
            else if (G.stages == 3) asm volatile("cp.async.wait_group 1;" ::: "memory");
            else asm volatile("cp.async.wait_group 0;" ::: "memory");
            __syncwarp();
            issue(i + G.stages - 1);
            const uint8_t * st = ring + (i % G.stages) * stage_bytes;
            const uint8_t * kr0 = st + g * G.kp + k_off;
            const uint8_t * kr1 = kr0 + 8 * G.kp;
            const float * sb = reinterpret_cast<const float *>(st + KEYS * (G.kp + G.vp));
            const float b0 = sb[g], b1 = sb[g + 8];

            // ---- scores of 16 keys x RB rows: S[nb] = {(g, 2t), (g, 2t+1), (g+8, 2t), (g+8, 2t+1)}
            float S[NB][4];
#pragma unroll
            for (int nb = 0; nb < NB; nb++) S[nb][0] = S[nb][1] = S[nb][2] = S[nb][3] = 0.0f;
            const uint32_t k_ld = smem_addr(st + ((lane & 7) + 8 * ((lane >> 3) & 1)) * G.kp + k_off + 16 * (lane >> 4));
            auto scores = [&](auto type) {
                constexpr int KT = decltype(type)::value;
#pragma unroll
                for (int b = 0; b < DB; b++) {
                    if (b < G.nbk) {
                        uint32_t fa[2][4];
                        const uint8_t * p0 = kr0 + b * block_bytes(KT);
                        const uint8_t * p1 = kr1 + b * block_bytes(KT);
                        if (b & 1) k_frag<KT, true>(fa, p0, p1, k_ld + 64 * b, t);
                        else k_frag<KT, false>(fa, p0, p1, k_ld + 64 * b, t);
                        float d0 = 1.0f, d1 = 1.0f, m0 = 0.0f, m1 = 0.0f;
                        if (KT != KV_TYPE_F16) {
                            d0 = half_bits(lds16(p0));
                            d1 = half_bits(lds16(p1));
                        }
                        if (KT == KV_TYPE_Q4_1) {
                            m0 = half_bits(lds16(p0 + 2));
                            m1 = half_bits(lds16(p1 + 2));
                        }
#pragma unroll
                        for (int nb = 0; nb < NB; nb++) {
                            float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                            for (int p = NP - 1; p >= 0; p--)          // the small pieces first
#pragma unroll
                                for (int ks = 0; ks < 2; ks++) {
                                    const uint2 f = QREG ? qr[QREG ? b : 0][ks][p]
                                                         : qf[(((b * 2 + ks) * NP + p) * NB + nb) * 32 + lane];
                                    mma(c, fa[ks], f.x, f.y, c);
                                }
                            if (KT == KV_TYPE_Q4_1) {
                                const float s0 = qsum[b * RB + 8 * nb + 2 * t], s1 = qsum[b * RB + 8 * nb + 2 * t + 1];
                                S[nb][0] = fmaf(m0, s0, S[nb][0]);
                                S[nb][1] = fmaf(m0, s1, S[nb][1]);
                                S[nb][2] = fmaf(m1, s0, S[nb][2]);
                                S[nb][3] = fmaf(m1, s1, S[nb][3]);
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
            const int j0 = j00 + i * TILE;
            const bool own = a.mask && j0 + KEYS > first_own;      // the step holds rows that the mask decides on
            bool moved = false;
            float f[NB][2];
#pragma unroll
            for (int nb = 0; nb < NB; nb++) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float b = e < 2 ? b0 : b1;
                    bool sees = b != -INFINITY;
                    if (own && sees) {
                        const int rr = r0 + 8 * nb + 2 * t + (e & 1);
                        sees = rr < r0 + nr && attn_sees(a, q, (int)a.by_group.div(rr), j0 + g + (e < 2 ? 0 : 8));
                    }
                    S[nb][e] = sees ? fmaf(S[nb][e], mul[nb][e & 1], b) : -INFINITY;
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
            const uint8_t * vst = st + KEYS * G.kp + v_off;
            const uint32_t v_ld = smem_addr(vst + ((lane & 7) + 8 * (lane >> 4)) * G.vp + 16 * ((lane >> 3) & 1));
            auto product = [&](auto type) {
                constexpr int VT = decltype(type)::value;
                bool odd_values = false;                 // a scale that is no finite number
                float c13 = 8192.0f;                     // 2^(13 - R)
                if (VT != KV_TYPE_F16) {
                    uint32_t top = 0;
#pragma unroll
                    for (int b = 0; b < DB; b++)
                        if (b < G.nbv) {
#pragma unroll
                            for (int u = 0; u < (VT == KV_TYPE_Q4_1 ? 2 : 1); u++) {
                                const uint32_t x = lds16(vst + g * G.vp + b * block_bytes(VT) + 2 * u) & 0x7FFFu;
                                const uint32_t y = lds16(vst + (g + 8) * G.vp + b * block_bytes(VT) + 2 * u) & 0x7FFFu;
                                odd_values |= x >= 0x7C00u || y >= 0x7C00u;
                                top = max(top, max(x < 0x7C00u ? x : 0u, y < 0x7C00u ? y : 0u));
                            }
                        }
                    odd_values = __any_sync(~0u, odd_values);
                    top = __reduce_max_sync(~0u, top);
                    const int e = top ? max((int)(top >> 10), 1) - 15 : -14;    // |scale| < 2^(e+1)
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
                    c13 = __int_as_float((127 + P_SHIFT - R) << 23);
                }
                // B fragments of P times a factor per key (f0: key g, f1: key g + 8)
                auto probs = [&](int nb, float f0, float f1, uint32_t bf[NP][2]) {
                    float x[4] = {S[nb][0] * f0, S[nb][1] * f0, S[nb][2] * f1, S[nb][3] * f1};
                    if (VT != KV_TYPE_F16 && odd_values) {
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (S[nb][e] == 0.0f) x[e] = 0.0f;
                    }
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        const uint32_t hi2 = pack(x[2 * u], x[2 * u + 1]);
                        bf[0][u] = transpose8(hi2);
                        if (NP == 2) {
                            const float2 b = unpack(hi2);
                            bf[NP - 1][u] = transpose8(pack(x[2 * u] - b.x, x[2 * u + 1] - b.y));
                        }
                    }
                };
                auto add = [&](int b, int mt, int nb, const uint32_t * fa, const uint32_t bf[NP][2]) {
                    if (NP == 1) {
                        mma(O[b][mt][nb], fa, bf[0][0], bf[0][1], O[b][mt][nb]);
                    } else {                             // a step's sum apart, so that the running sum rounds to nearest
                        float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        mma(c, fa, bf[NP - 1][0], bf[NP - 1][1], c);
                        mma(c, fa, bf[0][0], bf[0][1], c);
#pragma unroll
                        for (int e = 0; e < 4; e++) O[b][mt][nb][e] += c[e];
                    }
                };
                uint32_t bf[NB][NP][2];
                if (VT == KV_TYPE_F16) {
#pragma unroll
                    for (int nb = 0; nb < NB; nb++) probs(nb, 8192.0f, 8192.0f, bf[nb]);
                }
#pragma unroll
                for (int b = 0; b < DB; b++) {
                    if (b < G.nbv) {
                        uint32_t fa[2][4];
                        const uint8_t * p = vst + b * block_bytes(VT);
                        if (b & 1) v_frag<VT, true>(fa, p + 2 * t * G.vp, G.vp, v_ld + 64 * b, g);
                        else v_frag<VT, false>(fa, p + 2 * t * G.vp, G.vp, v_ld + 64 * b, g);
                        float d0 = 0.0f, d1 = 0.0f;
                        if (VT != KV_TYPE_F16) {
                            d0 = half_bits(lds16(p + g * G.vp)) * c13;
                            d1 = half_bits(lds16(p + (g + 8) * G.vp)) * c13;
                        }
#pragma unroll
                        for (int nb = 0; nb < NB; nb++) {
                            if (VT != KV_TYPE_F16) probs(nb, d0, d1, bf[nb]);
                            add(b, 0, nb, fa[0], bf[nb]);
                            add(b, 1, nb, fa[1], bf[nb]);
                        }
                        if (VT == KV_TYPE_Q4_1) {
                            const float e0 = half_bits(lds16(p + g * G.vp + 2)) * c13;
                            const float e1 = half_bits(lds16(p + (g + 8) * G.vp + 2)) * c13;
                            const uint32_t ones[4] = {0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u};
#pragma unroll
                            for (int nb = 0; nb < NB; nb++) {
                                probs(nb, e0, e1, bf[nb]);
                                add(b, 0, nb, ones, bf[nb]);
                                add(b, 1, nb, ones, bf[nb]);
                            }
                        }
                    }
                }
            };
            bool by_value = false;
            if (own && vt == KV_TYPE_F16) {
                // a row that the mask hides from some of the queries may hold infinities or NaN
                bool bad = false;
                for (int k = 0; k < KEYS; k++)
                    for (int d = lane; d < 32 * G.nbv; d += 32) bad |= (lds16(vst + k * G.vp + 2 * d) & 0x7C00u) == 0x7C00u;
                by_value = __any_sync(~0u, bad);
            }
            if (by_value) {                              // then this step's products are taken value by value
                for (int k = 0; k < KEYS; k++) {
#pragma unroll
                    for (int nb = 0; nb < NB; nb++) {
                        const int from = (k & 7) * 4 + t;
                        const float x0 = __shfl_sync(~0u, S[nb][0], from), x1 = __shfl_sync(~0u, S[nb][1], from);
                        const float x2 = __shfl_sync(~0u, S[nb][2], from), x3 = __shfl_sync(~0u, S[nb][3], from);
                        const float p0 = (k < 8 ? x0 : x2) * 8192.0f, p1 = (k < 8 ? x1 : x3) * 8192.0f;
#pragma unroll
                        for (int b = 0; b < DB; b++)
#pragma unroll
                            for (int mt = 0; mt < 2; mt++)
#pragma unroll
                                for (int r8 = 0; r8 < 2; r8++) {
                                    if (b < G.nbv) {
                                        const float v = half_bits(
                                            lds16(vst + k * G.vp + 2 * (32 * b + v_dim(KV_TYPE_F16, mt, g, r8))));
                                        if (p0 != 0.0f) O[b][mt][nb][2 * r8] = fmaf(p0, v, O[b][mt][nb][2 * r8]);
                                        if (p1 != 0.0f) O[b][mt][nb][2 * r8 + 1] = fmaf(p1, v, O[b][mt][nb][2 * r8 + 1]);
                                    }
                                }
                    }
                }
            } else {
                switch (vt) {
                case KV_TYPE_F16: product(kvc_int<KV_TYPE_F16>{}); break;
                case KV_TYPE_Q8_0: product(kvc_int<KV_TYPE_Q8_0>{}); break;
                case KV_TYPE_Q4_0: product(kvc_int<KV_TYPE_Q4_0>{}); break;
                default: product(kvc_int<KV_TYPE_Q4_1>{}); break;
                }
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");

        // ---- join the warps: every warp's sums go to shared memory (over the rings)
        __syncthreads();
        float * jo = reinterpret_cast<float *>(ring_all);                       // [WARPS][RB][dv]
        const float back = R > -1000 ? scalbnf(1.0f, R - P_SHIFT) : 0.0f;
#pragma unroll
        for (int nb = 0; nb < NB; nb++) {
#pragma unroll
            for (int c = 0; c < 2; c++) {
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) l[nb][c] += __shfl_xor_sync(~0u, l[nb][c], o);
                if (g == 0) {
                    jm[warp * RB + 8 * nb + 2 * t + c] = m[nb][c];
                    jl[warp * RB + 8 * nb + 2 * t + c] = l[nb][c];
                }
            }
#pragma unroll
            for (int b = 0; b < DB; b++)
                if (b < G.nbv) {
#pragma unroll
                    for (int mt = 0; mt < 2; mt++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            jo[((size_t)warp * RB + 8 * nb + 2 * t + (e & 1)) * a.dv + 32 * b + v_dim(vt, mt, g, e >> 1)] =
                                O[b][mt][nb][e] * back;
                }
        }
        __syncthreads();
        float * part = slot >= 0 ? attn_part<RB>(a, qb, h, w, slot) : nullptr;
        for (int e = threadIdx.x; e < nr * a.dv; e += THREADS) {
            const int r = e / a.dv, d = e - r * a.dv;
            float M = -INFINITY;
#pragma unroll
            for (int u = 0; u < WARPS; u++) M = fmaxf(M, jm[u * RB + r]);
            const float base = M == -INFINITY ? 0.0f : M;
            float L = 0.0f, o = 0.0f;
#pragma unroll
            for (int u = 0; u < WARPS; u++) {
                const float fu = expf(jm[u * RB + r] - base);
                L = fmaf(fu, jl[u * RB + r], L);
                o = fmaf(fu, jo[((size_t)u * RB + r) * a.dv + d], o);
            }
            if (part) {
                part[r * a.dv + d] = o;
                if (d == 0) {
                    part[RB * a.dv + r] = M;
                    part[RB * a.dv + RB + r] = L;
                }
            } else {
                const int i = (int)a.by_group.div(r0 + r);
                const size_t at = (size_t)(q.q0 + i) * a.Hq + h * a.g + (r0 + r - i * a.g);
                const float v = L > 0.0f ? o / L : (L == 0.0f ? 0.0f : L);
                if (a.q_type == KV_TYPE_F16) reinterpret_cast<__half *>(a.out)[at * a.dv + d] = __float2half_rn(v);
                else reinterpret_cast<float *>(a.out)[at * a.dv + d] = v;
                if (d == 0 && a.lse) a.lse[at] = L == 0.0f ? -INFINITY : M + logf(L);
            }
        }
    });
}

// Ring geometry, or false where the rows are not ones that the kernel reads.
bool geometry(const kvc_attn_args & a, int rb, mma_geom * G) {
    if (a.k_type == KV_TYPE_F32 || a.v_type == KV_TYPE_F32 || a.dk % 32 || a.dv % 32) return false;
    auto side = [](const void * base, long long rbytes, long long hb, int * g, int * p, int seg) {
        const uintptr_t all = (uintptr_t)base | (uintptr_t)rbytes;
        if ((hb & 3) || (all & 3)) return false;
        int most = seg;
        if ((all & 15) == 0) {                           // 16-byte pieces from the boundary below the head's part
            *g = 16;
            most = seg + (int)(((hb & 15) == 0) ? 0 : (hb & 7) == 0 ? 8 : 12);
        } else {
            *g = ((all | (uintptr_t)hb) & 7) == 0 ? 8 : 4;
        }
        *p = (most + 15) & ~15;
        if ((*p / 16) % 2 == 0) *p += 16;
        return true;
    };
    G->kseg = (int)a.k_hb;
    G->vseg = (int)a.v_hb;
    if (!side(a.K, a.k_rb, a.k_hb, &G->kg, &G->kp, G->kseg) || !side(a.V, a.v_rb, a.v_hb, &G->vg, &G->vp, G->vseg))
        return false;
    G->nbk = a.dk / 32;
    G->nbv = a.dv / 32;
    const int stage = KEYS * (G->kp + G->vp) + KEYS * 4;
    // as many stages (2 to 4) as leave room for two CTAs and more per SM
    G->stages = WARPS * 4 * stage <= 76 * 1024 ? 4 : WARPS * 3 * stage <= 108 * 1024 ? 3 : 2;
    const int join = WARPS * rb * a.dv * 4;
    G->ring = WARPS * G->stages * stage;
    if (join > G->ring) G->ring = join;
    return true;
}

template <int DB, int NB, int NP>
size_t smem_bytes(const mma_geom & G) {
    constexpr int RB = 8 * NB;
    return (size_t)DB * 2 * NP * NB * 32 * 8 + (DB * RB + RB + 2 * WARPS * RB) * 4 + G.ring;
}

// CTAs per SM, asked once per shared-memory size and device.
template <int DB, int NB, int NP>
int resident(int * ctas, const mma_geom & G) {
    static std::atomic<uint64_t> known[64];
    const size_t sm = smem_bytes<DB, NB, NP>(G);
    int dev = 0;
    KVC_CUDA(cudaGetDevice(&dev));
    const uint64_t v = known[dev & 63].load(std::memory_order_relaxed);
    if ((v >> 8) == sm) {
        *ctas = (int)(v & 255);
        return KVC_OK;
    }
    KVC_CUDA(cudaFuncSetAttribute(k_tree_mma<DB, NB, NP>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
    KVC_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(ctas, k_tree_mma<DB, NB, NP>, THREADS, sm));
    known[dev & 63].store((uint64_t)sm << 8 | (uint64_t)*ctas, std::memory_order_relaxed);
    return KVC_OK;
}

template <int DB, int NB, int NP>
int run(const kvc_attn_args & a, const mma_geom & G, dim3 grid, cudaStream_t st) {
    k_tree_mma<DB, NB, NP><<<grid, THREADS, smem_bytes<DB, NB, NP>(G), st>>>(a, G);
    g_serve_launches++;
    KVC_CUDA(cudaGetLastError());
    return kvc_launch_attn_join(a, 8 * NB, TILE, st);
}

#define TREE_CASE(DB, NB, CALL) \
    return np == 2 ? CALL<DB, NB, 2> : CALL<DB, NB, 1>
#define TREE_SELECT(CALL)                              \
    if (db <= 2) {                                     \
        if (nb == 1) TREE_CASE(2, 1, CALL);            \
        if (nb == 2) TREE_CASE(2, 2, CALL);            \
        TREE_CASE(2, 4, CALL);                         \
    }                                                  \
    if (db <= 4) {                                     \
        if (nb == 1) TREE_CASE(4, 1, CALL);            \
        if (nb == 2) TREE_CASE(4, 2, CALL);            \
        TREE_CASE(4, 4, CALL);                         \
    }                                                  \
    if (nb == 1) TREE_CASE(8, 1, CALL);                \
    TREE_CASE(8, 2, CALL)

using resident_fn = int (*)(int *, const mma_geom &);
using run_fn = int (*)(const kvc_attn_args &, const mma_geom &, dim3, cudaStream_t);
resident_fn select_resident(int db, int nb, int np) { TREE_SELECT(resident); }
run_fn select_run(int db, int nb, int np) { TREE_SELECT(run); }

}  // namespace

bool kvc_attn_tree_mma_plan(kvc_attn_args * a, int sms, kvc_tree_mma_plan * p) {
    const int top = a->dk > a->dv ? a->dk : a->dv;
    const long long rows = (long long)a->max_q * a->g;
    p->db = top <= 64 ? 2 : top <= 128 ? 4 : 8;
    p->nb = rows <= 8 ? 1 : rows <= 16 || p->db == 8 ? 2 : 4;
    p->np = a->q_type == KV_TYPE_F32 ? 2 : 1;
    p->rb = 8 * p->nb;
    p->blocks = (rows + p->rb - 1) / p->rb;
    mma_geom G;
    if (p->blocks * a->Hkv > 65535 || !geometry(*a, p->rb, &G)) return false;
    int ctas = 0;
    if (select_resident(p->db, p->nb, p->np)(&ctas, G) != KVC_OK || ctas < 1) return false;
    // one wave: every CTA gets an equal stretch of the keys
    const long long w = (long long)sms * ctas / (p->blocks * a->Hkv);
    a->W = (int)(w < 1 ? 1 : w);
    return true;
}

int kvc_launch_attn_tree_mma(const kvc_attn_args & a, const kvc_tree_mma_plan & p, cudaStream_t st) {
    mma_geom G;
    if (!geometry(a, p.rb, &G)) return KVC_ERR_SHAPE;
    return select_run(p.db, p.nb, p.np)(a, G, dim3((unsigned)a.W, (unsigned)(p.blocks * a.Hkv)), st);
}
