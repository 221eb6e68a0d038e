// attn_prompt_tc.cu — attention over whole prompts on the 5th-generation
// tensor cores (tcgen05, accumulators in TMEM), F16 rows of up to 128 values.
//
//   S = Q K^T,  P = exp2(c S - c m),  O = P V,  out = O / l,  c = scale log2 e
//
// A tile is 128 rows of one KV head: floor(128 / g) tokens times the g query
// heads that share it, so that keys and values are loaded once for the group
// and short prompts fill the tile. A tile walks the keys in steps of 128; while
// one tile's softmax warps work, the tensor cores run the other's products. The
// two are two CTAs of one SM (NT = 1: one's start and end lie under the other's
// steps, and work is dealt in smaller pieces), or, for long sequences that fill
// the machine several times, in one CTA, which then loads keys and values once
// for both (NT = 2). 32 query heads on 8 KV heads, 128 values, us with one tile
// in a CTA / two, in a loop: ten packed prompts of 1 to 2,047 tokens 95 / 96, 812
// tokens on 10,333 keys 115 / 123, one prompt of 8,192 tokens 589 / 576.
//
//   warps 0-3 (, 4-7)  softmax of tile 0 (, 1): a thread owns a row. S comes
//                      from TMEM, P goes back as fp16 over S's columns, from
//                      where it is the second product's A operand (no shared
//                      memory). The reference maximum m moves only when a
//                      row's maximum has grown by more than 2^8 in P, so O is
//                      rarely rescaled.
//   then one warp      TMA: Q once, then K and V through one ring of slots
//   and one            MMA issue
//
// Rows, statistics and O are 32-bit; P is rounded to fp16 once (2^-11 relative, as
// the output is; l is the sum of the unrounded values): a second piece of P would be
// half as many products again. Against 64 bits the outputs' error grows from 1.9e-4
// (their own rounding) to 2.2e-4 - 2.9e-4. Bound by the exponentials (16 per clock
// and SM against 4,096 multiply-adds) and the tensor cores about equally at d = 128:
// a tile's step is a chain of softmax (about 2,350 cycles) and products (78 cycles
// for each of 16 instructions), and two tiles fill an SM's issue slots and tensor
// cores by turns.
// The 8,192-token prompt takes 496 us in bursts, 1,100 TFLOP/s or 65 % of a dense
// product's rate, and 574 in a loop of seconds, 960 TFLOP/s, 68 % of the sustained rate.
// Steps of 64 keys (723 us), two threads per row (513) and exponentials that do
// not wait for the step's maximum (544) were slower.
#include "attn.h"
#include "attn_prompt.h"
#include "attn_tc.h"
#include <math.h>

namespace {

using namespace kvc_tc;
using namespace kvc_attn_tc;

constexpr int TM = 128, TN = 128;               // rows and keys of a tile
constexpr uint32_t POLLS = 1u << 22;            // bound of every wait
constexpr float LOG2E = 1.4426950408889634f;

// NT tiles in a CTA.
template <int D, int NT>
struct cfg {
    static constexpr int HALVES = D / 64;                   // 64-value column blocks of 128 bytes a row
    static constexpr int BLOCK = TN * 128;                  // bytes of such a block (128 rows)
    static constexpr int TILE = HALVES * BLOCK;
    static constexpr int THREADS = 128 * NT + 64;
    static constexpr int SLOTS = NT == 2 ? (D == 128 ? 5 : 8) : (D == 128 ? 2 : 4);  // ring of K and V tiles
    static constexpr int SMEM = 1024 + NT * TILE + SLOTS * TILE + 256;
    static constexpr uint32_t S_COL = 0, O_COL = NT * 128;  // TMEM: S of tile t at t*128, O behind them at t*D
    static constexpr uint32_t COLS = NT * 256;
};

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const void * map, int x, int y, int z, uint64_t * bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 :: "r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar)) : "memory");
}

struct prompt_geom {
    int tokens;                 // of a tile: floor(128 / g)
    int tiles;                  // upper bound of the CTAs per KV head
};

template <int D, int NT>
__global__ void __launch_bounds__(cfg<D, NT>::THREADS, 3 - NT) k_prompt_tc(const __grid_constant__ kvc_attn_args a,
                                                          const __grid_constant__ prompt_geom G,
                                                          const __grid_constant__ CUtensorMap q_map,
                                                          const __grid_constant__ CUtensorMap k_map,
                                                          const __grid_constant__ CUtensorMap v_map) {
    using C = cfg<D, NT>;
    extern __shared__ uint8_t sm_raw[];
    uint8_t * sm = aligned_1024(sm_raw);
    uint8_t * sq = sm;                                   // Q tiles
    uint8_t * ring = sq + NT * C::TILE;
    uint64_t * bars = reinterpret_cast<uint64_t *>(ring + C::SLOTS * C::TILE);
    uint64_t * full = bars;                              // [SLOTS] by TMA
    uint64_t * empty = full + C::SLOTS;                  // [SLOTS] by the MMAs that read it
    uint64_t * q_full = empty + C::SLOTS;
    uint64_t * s_full = q_full + 1;                      // [2] S of a tile is in TMEM
    uint64_t * p_full = s_full + 2;                      // [2] P is, and O may be added to
    uint64_t * o_full = p_full + 2;                      // [2] the product has been added
    uint64_t * v_fixed = o_full + 2;                     // the last V tile's rows past the end are zero
    uint32_t * slot = reinterpret_cast<uint32_t *>(v_fixed + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int h = blockIdx.x % a.Hkv;

    // the CTA's token tile: the last ones of a sequence, which see most keys, first
    int s = -1, q0 = 0, nq = 0, k0 = 0, nk = 0, tok0 = 0;
    {
        const int per = NT * G.tokens;
        int want = blockIdx.x / a.Hkv, at = 0;
        for (int s0 = 0; s0 < a.n_seqs && s < 0; s0 += 32) {
            kvc_attn_seq x{};
            if (s0 + lane < a.n_seqs) x = attn_seq(a, s0 + lane);
            const int t = (x.nq + per - 1) / per;
            int p = t;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(~0u, p, o);
                if (lane >= o) p += u;
            }
            const unsigned hit = __ballot_sync(~0u, at + p > want);
            if (hit) {
                const int l = __ffs(hit) - 1;
                s = s0 + l;
                const int first = at + __shfl_sync(~0u, p - t, l), n = __shfl_sync(~0u, t, l);
                q0 = __shfl_sync(~0u, x.q0, l);
                nq = __shfl_sync(~0u, x.nq, l);
                k0 = __shfl_sync(~0u, x.k0, l);
                nk = __shfl_sync(~0u, x.ln, l);
                tok0 = (n - 1 - (want - first)) * per;
            }
            at += __shfl_sync(~0u, p, 31);
        }
    }
    if (s < 0) return;                                   // past the last tile
    // keys that the tiles see, in steps of 128
    int n_keys[NT], steps[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
        const int first = tok0 + t * G.tokens, last = min(first + G.tokens, nq) - 1;
        n_keys[t] = last < first ? 0 : a.causal ? min(nk, max(0, last + nk - nq + 1)) : nk;
        steps[t] = (n_keys[t] + TN - 1) / TN;
    }
    const int n = max(steps[0], steps[NT - 1]);

    if (warp == 4 * NT + 1) tmem_alloc(slot, C::COLS);
    if (threadIdx.x == 0) {
        for (int i = 0; i < C::SLOTS; i++) {
            mbar_init(full + i, 1);
            mbar_init(empty + i, 1);
        }
        mbar_init(q_full, 1);
        for (int t = 0; t < 2; t++) {
            mbar_init(s_full + t, 1);
            mbar_init(p_full + t, 4);
            mbar_init(o_full + t, 1);
        }
        mbar_init(v_fixed, 1);
        mbar_init_fence();
    }
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = *slot;

    bool ok = true;                                      // false: a wait ran out; the rows become NaN
    if (warp == 4 * NT) {
        // ---- loads: slot 2j holds K of step j, slot 2j + 1 its V
        const int last_rows = nk - (n - 1) * TN;         // valid rows of the last V tile
        if (lane == 0 && n > 0) {
            mbar_arrive_expect_tx(q_full, NT * C::HALVES * (uint32_t)(G.tokens * a.g * 128));
            for (int t = 0; t < NT; t++)
                for (int x = 0; x < C::HALVES; x++)
                    tma_load_3d(smem_u32(sq + t * C::TILE + x * C::BLOCK), &q_map, 64 * x, h * a.g,
                                q0 + tok0 + t * G.tokens, q_full);
            int i = 0;
            for (; i < 2 * n; i++) {
                const int st = i % C::SLOTS;
                ok = mbar_wait(empty + st, ((i / C::SLOTS) & 1) ^ 1, POLLS);
                if (!ok) break;
                uint8_t * dst = ring + st * C::TILE;
                mbar_arrive_expect_tx(full + st, C::TILE);
                for (int x = 0; x < C::HALVES; x++)
                    tma_load_3d(smem_u32(dst + x * C::BLOCK), i & 1 ? &v_map : &k_map, 64 * x, h, k0 + (i >> 1) * TN,
                                full + st);
            }
            // the copies land before the CTA ends, whether anybody still waits for them or not
            for (int k = max(0, i - C::SLOTS); k < i; k++) mbar_wait(full + k % C::SLOTS, (k / C::SLOTS) & 1, POLLS);
            mbar_wait(q_full, 0, POLLS);
        }
        ok = __shfl_sync(~0u, ok, 0);
        if (n > 0 && last_rows < TN) {
            // the rows behind the sequence's end may hold another sequence's values, of any kind: 0 * V has to be 0
            const int i = 2 * n - 1, st = i % C::SLOTS;
            const bool there = mbar_wait(full + st, (i / C::SLOTS) & 1, POLLS);
            if (there)
                for (int e = lane; e < (TN - last_rows) * 8 * C::HALVES; e += 32) {
                    const int row = last_rows + (e >> 3) % (TN - last_rows), x = (e >> 3) / (TN - last_rows);
                    *reinterpret_cast<int4 *>(ring + st * C::TILE + x * C::BLOCK + row * 128 + (e & 7) * 16) = make_int4(0, 0, 0, 0);
                }
            fence_smem_to_async();
            __syncwarp();
            if (lane == 0 && there) mbar_arrive(v_fixed);
        }
    } else if (warp == 4 * NT + 1) {
        // ---- products
        if (n > 0) {
            const uint32_t id_s = idesc_f16(TM, TN), id_o = idesc_f16(TM, D) | 1u << 16;      // V is N-major
            const bool fixed = nk - (n - 1) * TN < TN;
            auto qk = [&](int t, int j) {
                const uint32_t qa = smem_u32(sq + t * C::TILE), ka = smem_u32(ring + (2 * j) % C::SLOTS * C::TILE);
#pragma unroll
                for (int k = 0; k < D / 16; k++) {
                    const uint32_t o = (k >> 2) * C::BLOCK + (k & 3) * 32;
                    mma_f16_ss(tmem + C::S_COL + t * TN, desc_k(qa + o), desc_k(ka + o), id_s, k > 0);
                }
                commit_mma(s_full + t, ok);
            };
            auto pv = [&](int t, int j) {
                const uint32_t va = smem_u32(ring + (2 * j + 1) % C::SLOTS * C::TILE);
#pragma unroll
                for (int k = 0; k < TN / 16; k++)
                    mma_f16_ts(tmem + C::O_COL + t * D, tmem + C::S_COL + t * TN + 8 * k, desc_n(va + k * 2048, C::BLOCK),
                               id_o, j > 0 || k > 0);
                commit_mma(o_full + t, ok);
            };
            // The products are issued by whole warps, so no branch goes by `ok`, which a wait at its limit could leave
            // different from lane to lane (agreeing on it by a vote: ten packed prompts 95.0 us instead of 94.3).
            auto wait = [&](uint64_t * bar, uint32_t parity) { ok = ok && mbar_wait(bar, parity, POLLS); };
            auto wait_full = [&](int i) { wait(full + i % C::SLOTS, (i / C::SLOTS) & 1); };
            wait(q_full, 0);
            wait_full(0);
            fence_after_sync();
#pragma unroll
            for (int t = 0; t < NT; t++)
                if (steps[t] > 0) qk(t, 0);
            commit_mma(empty + 0, ok);
            for (int j = 0; j < n; j++) {
                wait_full(2 * j + 1);
                if (j == n - 1 && fixed) wait(v_fixed, 0);
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    if (j < steps[t]) {
                        wait(p_full + t, j & 1);
                        fence_after_sync();
                        pv(t, j);
                    }
                    if (t == NT - 1) commit_mma(empty + (2 * j + 1) % C::SLOTS, ok);
                    if (t == 0 && j + 1 < n) wait_full(2 * j + 2);
                    if (j + 1 < steps[t]) qk(t, j + 1);
                    if (t == NT - 1 && j + 1 < n) commit_mma(empty + (2 * j + 2) % C::SLOTS, ok);
                }
            }
            // the products end before TMEM is given back
#pragma unroll
            for (int t = 0; t < NT; t++)
                if (steps[t] > 0) mbar_wait(o_full + t, (steps[t] - 1) & 1, POLLS);
        }
        __syncwarp();
    } else {
        // ---- softmax: thread = row
        const int t = NT == 1 ? 0 : warp >> 2;
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const uint32_t s_addr = tmem + lanes + C::S_COL + t * TN, o_addr = tmem + lanes + C::O_COL + t * D;
        const int r = threadIdx.x & 127;
        const int tok = tok0 + t * G.tokens + (int)a.by_group.div(r);
        const bool real = r < G.tokens * a.g && tok < nq;
        const int see = !real ? 0 : a.causal ? min(nk, max(0, tok + nk - nq + 1)) : nk;      // keys 0 .. see-1
        const int see_all = tok0 + t * G.tokens + nk - nq + 1;                               // of the tile's first row
        const float c = a.scale * LOG2E;
        float m = -INFINITY, l = 0.0f;
        for (int j = 0; j < steps[t]; j++) {
            ok = ok && mbar_wait(s_full + t, j & 1, POLLS);
            if (!__all_sync(~0u, ok)) break;
            fence_after_sync();
            float x[TN];
            uint32_t * xr = reinterpret_cast<uint32_t *>(x);
#pragma unroll
            for (int i = 0; i < 4; i++) ld32(s_addr + 32 * i, xr + 32 * i);
            tmem_wait_ld();
            const int k_end = see - j * TN;
            if ((j + 1) * TN > (a.causal ? min(see_all, nk) : nk)) {      // some row of the tile sees less than all 128
#pragma unroll
                for (int i = 0; i < TN; i++)
                    if (i >= k_end) x[i] = -INFINITY;
            }
            float mx[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
            for (int i = 4; i < TN; i += 4) {
                mx[0] = fmaxf(mx[0], x[i]);
                mx[1] = fmaxf(mx[1], x[i + 1]);
                mx[2] = fmaxf(mx[2], x[i + 2]);
                mx[3] = fmaxf(mx[3], x[i + 3]);
            }
            const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
            // the reference moves where P would pass 2^8
            const bool move = top > m && !((top - m) * c <= 8.0f);
            if (j == 0) {
                m = top;
            } else if (__any_sync(~0u, move)) {
                const float mn = move ? top : m;
                const float f = ex2((m - (mn == -INFINITY ? 0.0f : mn)) * c);
                const float fr = move ? f : 1.0f;
                m = mn;
                l *= fr;
                ok = ok && mbar_wait(o_full + t, (j - 1) & 1, POLLS);
                if (!__all_sync(~0u, ok)) break;
                fence_after_sync();
#pragma unroll 1
                for (int i = 0; i < D; i += 32) {
                    float o[32];
                    ld32(o_addr + i, reinterpret_cast<uint32_t *>(o));
                    tmem_wait_ld();
#pragma unroll
                    for (int k = 0; k < 32; k++) o[k] *= fr;
                    st32(o_addr + i, reinterpret_cast<uint32_t *>(o));
                }
            }
            const float mc = m == -INFINITY ? 0.0f : -m * c;
            float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
            uint32_t p[TN / 2];
#pragma unroll
            for (int i = 0; i < TN / 2; i++) {
                float2 y = fma2(make_float2(x[2 * i], x[2 * i + 1]), make_float2(c, c), make_float2(mc, mc));
                y.x = ex2(y.x);
                y.y = ex2(y.y);
                sum[i & 1] = add2(sum[i & 1], y);
                p[i] = pack(y.x, y.y);
            }
            st32(s_addr, p);
            st32(s_addr + 32, p + 32);
            l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
            tmem_wait_st();
            fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + t);
        }
        // ---- output
        if (steps[t] > 0) ok = ok && mbar_wait(o_full + t, (steps[t] - 1) & 1, POLLS);
        ok = __all_sync(~0u, ok);
        fence_after_sync();
        const size_t row = (size_t)(q0 + tok) * a.Hq + h * a.g + (r - (int)a.by_group.div(r) * a.g);
        const float inv = !ok ? NAN : l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
        __half * out = reinterpret_cast<__half *>(a.out) + row * a.dv;
#pragma unroll 1
        for (int i = 0; i < D; i += 32) {
            float o[32];
            if (steps[t] > 0) {
                ld32(o_addr + i, reinterpret_cast<uint32_t *>(o));
                tmem_wait_ld();
            } else {
#pragma unroll
                for (int k = 0; k < 32; k++) o[k] = 0.0f;
            }
            if (real) {
#pragma unroll
                for (int k = 0; k < 32; k += 8)
                    if (i + k < a.dv) {
                        uint4 v;
                        v.x = pack(o[k] * inv, o[k + 1] * inv);
                        v.y = pack(o[k + 2] * inv, o[k + 3] * inv);
                        v.z = pack(o[k + 4] * inv, o[k + 5] * inv);
                        v.w = pack(o[k + 6] * inv, o[k + 7] * inv);
                        *reinterpret_cast<uint4 *>(out + i + k) = v;
                    }
            }
        }
        if (real && a.lse) a.lse[row] = !ok ? NAN : l == 0.0f ? -INFINITY : m * a.scale + logf(l);
        fence_before_sync();
    }
    __syncthreads();
    if (warp == 4 * NT + 1) {
        fence_after_sync();
        tmem_free(tmem, C::COLS);
    }
}

// [tokens][heads][d] F16 with the given byte strides; boxes of 64 values x `heads` x `rows` (values past d read as 0).
bool rows_map(CUtensorMap * m, const void * base, int d, int heads, int tokens, long long head_bytes, long long token_bytes,
              int box_heads, int box_rows) {
    const cuuint64_t dims[3] = {(cuuint64_t)d, (cuuint64_t)heads, (cuuint64_t)(tokens > 0 ? tokens : 1)};
    const cuuint64_t strides[2] = {(cuuint64_t)head_bytes, (cuuint64_t)token_bytes};
    const cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_rows}, one[3] = {1, 1, 1};
    return kvc_tensor_map_encoder()(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void *>(base), dims, strides, box, one,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, int NT>
int launch(const kvc_attn_args & a, prompt_geom G, const CUtensorMap * maps, cudaStream_t st) {
    static std::atomic<bool> set[64];
    int dev = 0;
    KVC_CUDA(cudaGetDevice(&dev));
    if (!set[dev & 63].load(std::memory_order_relaxed)) {
        KVC_CUDA(cudaFuncSetAttribute(k_prompt_tc<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, cfg<D, NT>::SMEM));
        set[dev & 63].store(true, std::memory_order_relaxed);
    }
    G.tiles = a.n_total / (NT * G.tokens) + a.n_seqs;    // each sequence's tiles, its last one perhaps partial
    k_prompt_tc<D, NT><<<(unsigned)G.tiles * (unsigned)a.Hkv, cfg<D, NT>::THREADS, cfg<D, NT>::SMEM, st>>>(a, G, maps[0], maps[1], maps[2]);
    g_serve_launches++;
    KVC_CUDA(cudaGetLastError());
    return KVC_OK;
}

}  // namespace

bool kvc_attn_prompt_tc_ok(const kvc_attn_args & a) {
    if (a.q_type != KV_TYPE_F16 || a.k_type != KV_TYPE_F16 || a.v_type != KV_TYPE_F16) return false;
    const int top = a.dk > a.dv ? a.dk : a.dv;
    // the running maximum is taken of the unscaled scores
    if (top > 128 || a.dk % 8 || a.dv % 8 || a.g > TM || !(a.scale > 0.0f) || !(a.scale < INFINITY)) return false;
    // TMA: 16-byte bases and strides (strides of dimensions of size 1 included), extents below 2^32
    const uintptr_t bases = (uintptr_t)a.q | (uintptr_t)a.K | (uintptr_t)a.V | (uintptr_t)a.out;
    const long long strides = a.q_stride * 2 | a.q_head * 2 | a.k_rb | a.k_hb | a.v_rb | a.v_hb;
    if ((bases & 15) || (strides & 15)) return false;
    for (long long x : {a.q_stride * 2, a.q_head * 2, a.k_rb, a.k_hb, a.v_rb, a.v_hb})
        if (x <= 0 || x >= 1LL << 40) return false;
    const long long tiles = a.n_total / (TM / a.g) + a.n_seqs;
    return a.n_keys > 0 && tiles * a.Hkv <= INT32_MAX && kvc_tensor_map_encoder() != nullptr;
}

int kvc_launch_attn_prompt_tc(const kvc_attn_args & a, cudaStream_t st) {
    prompt_geom G;
    G.tokens = TM / a.g;
    CUtensorMap maps[3];
    if (!rows_map(&maps[0], a.q, a.dk, a.Hq, a.n_total, a.q_head * 2, a.q_stride * 2, a.g, G.tokens) ||
        !rows_map(&maps[1], a.K, a.dk, a.Hkv, a.n_keys, a.k_hb, a.k_rb, 1, TN) ||
        !rows_map(&maps[2], a.V, a.dv, a.Hkv, a.n_keys, a.v_hb, a.v_rb, 1, TN)) {
        fprintf(stderr, "[kvc] cuTensorMapEncodeTiled failed for a prompt of %d rows\n", a.n_total);
        return KVC_ERR_CUDA;
    }
    // Two tiles in a CTA for sequences of 6,000 queries and more on average that make 4 CTAs per SM (the host knows no
    // more of the lengths). us with one tile / two, 32 heads on 8, 128 values: 4 x 2,000 queries 177 / 188, 3 x 4,100
    // 429 / 446, 5,000 215 / 221, 2 x 6,000 565 / 571, 8,192 506 / 510 (589 / 576 in a loop of seconds), 16,000
    // 1,843 / 1,791; 6,000 beside 16 of 100 301 / 313, 12,000 beside 8 of 300 1,071 / 1,050; 64 values: 4 x 2,000
    // 147 / 150, 2 x 6,000 491 / 483, 16,000 1,554 / 1,497.
    const bool two = a.n_total / a.n_seqs >= 6000 && (long long)a.n_total / (2 * G.tokens) * a.Hkv >= 4LL * kvc_serve_device();
    if (a.dk > 64 || a.dv > 64) return two ? launch<128, 2>(a, G, maps, st) : launch<128, 1>(a, G, maps, st);
    return two ? launch<64, 2>(a, G, maps, st) : launch<64, 1>(a, G, maps, st);
}
