// attn_simt.cu — the general attention kernel and the join of partial results
// (include/kvc-attn.h). The tensor-core kernels (attn_tree.cu,
// attn_prompt.cu) take the common types and shapes; this one takes the rest:
// F32 rows, head sizes and strides that those do not read.
//
//   x_ij = scale q_i.k_j (+ beta_j),  m = max_j x_ij,  l = sum_j exp(x_ij - m),
//   out_i = (sum_j exp(x_ij - m) v_j) / l,  lse_i = m + log l
//
// in one pass over the keys with a running m, l and sum.
#include "attn.h"
#include "attn_tc.h"

#include <math.h>

namespace {

constexpr int RB = 8, TILE = 128;        // query rows and keys per CTA and step
constexpr int WARPS = 4, THREADS = 32 * WARPS, WK = 32;
static_assert(TILE == WARPS * WK, "a tile is one key per lane");

// A shared-memory row of `d` values: whole float4s, an odd number of them, so that 8 lanes reading 8 rows hit all banks.
__host__ __device__ constexpr int simt_pitch(int d) { return 4 * (((d + 3) / 4) | 1); }

// 32 stored rows (this lane's is `row`; only those in `live` are read, the others become zeros) as fp32 into a warp's
// shared memory, d values each and zeros up to whole float4s. `direct`: fp32 rows on 16-byte boundaries, whose copies are
// all in flight at once; else 8 rows' elements at a time.
__device__ __forceinline__ void simt_load(float * buf, int pitch, const uint8_t * base, long long rb, int type, int d,
                                          long long row, unsigned live, bool direct, int lane) {
    const int d4 = (d + 3) & ~3;
    if (direct) {
        for (int k = 0; k < WK; k++) {
            const long long rk = __shfl_sync(~0u, row, k);
            const float * p = reinterpret_cast<const float *>(base + ((live >> k) & 1u ? rk : 0) * rb);
            for (int e = 4 * lane; e < d; e += 128) {
                if ((live >> k) & 1u)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
                                 :: "r"((uint32_t)__cvta_generic_to_shared(buf + k * pitch + e)), "l"(p + e) : "memory");
                else
                    *reinterpret_cast<float4 *>(buf + k * pitch + e) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        return;
    }
    for (int k0 = 0; k0 < WK; k0 += 8) {
        if (!((live >> k0) & 0xFFu)) {
            for (int e = lane; e < 8 * d4; e += 32) buf[(k0 + e / d4) * pitch + e % d4] = 0.0f;
            continue;
        }
        long long at[8];
#pragma unroll
        for (int u = 0; u < 8; u++) at[u] = __shfl_sync(~0u, row, k0 + u) * rb;
        for (int e = lane; e < d4; e += 32) {
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; u++) v[u] = e < d && ((live >> (k0 + u)) & 1u) ? attn_elem(base + at[u], type, e) : 0.0f;
#pragma unroll
            for (int u = 0; u < 8; u++) buf[(k0 + u) * pitch + e] = v[u];
        }
    }
}

// One CTA: 8 query rows of one KV head against its stretch of the keys. A
// warp takes 32 keys of a tile, brings their K rows as fp32 into its own shared
// memory, scores one key per lane, then does the same with V with up to 4
// neighbouring output dimensions per lane (8 in two runs): no barrier inside
// the loop. All shared-memory reads are of four values, 12 wavefronts for the
// 32 multiply-adds that a lane makes with them. Bound by a warp's wait for its
// rows (12 warps per SM at 128 values): 43,000 F32 keys of 8 heads, 4 query rows
// each, 128 values, 162 us (2.2 TB/s of rows); rows brought one by one and single
// values read from shared memory: 432 us.
template <int DV_LANES>
__global__ void __launch_bounds__(THREADS) k_attn_simt(const __grid_constant__ kvc_attn_args a) {
    extern __shared__ __align__(16) float sm[];
    constexpr int VEC = DV_LANES < 4 ? DV_LANES : 4;     // neighbouring output dimensions of a lane
    const int pitch = simt_pitch(max(a.dk, a.dv)), dk4 = (a.dk + 3) & ~3;
    // fp32 rows that can be copied 16 bytes at a time
    auto aligned = [](const uint8_t * p, long long rb, long long hb, int type, int d) {
        return type == KV_TYPE_F32 && (((uintptr_t)p | (uintptr_t)rb | (uintptr_t)hb) & 15) == 0 && d % 4 == 0;
    };
    const bool k_direct = aligned(a.K, a.k_rb, a.k_hb, a.k_type, a.dk), v_direct = aligned(a.V, a.v_rb, a.v_hb, a.v_type, a.dv);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float * qs = sm;                                     // [RB][dk]
    float * ps = qs + RB * dk4 + warp * (RB * WK);       // [32][RB] of this warp
    float * buf = qs + RB * dk4 + WARPS * RB * WK + (size_t)warp * WK * pitch;
    float * joinO = qs + RB * dk4 + WARPS * RB * WK;    // reused after the loop: [WARPS][RB][dv] (dv <= pitch, RB <= 32)
    __shared__ float s_m[WARPS][RB], s_l[WARPS][RB];
    const int h = blockIdx.y % a.Hkv, w = blockIdx.x;
    const int n_blocks = (int)(((long long)a.max_q * a.g + RB - 1) / RB);

    for (int qb = blockIdx.y / a.Hkv; qb < n_blocks; qb += gridDim.y / a.Hkv) {
    attn_walk(a, qb, qb + 1, w, h == 0 && threadIdx.x < 32, [&](int, const kvc_attn_seq & q, int lo, int hi, int slot) {
        const int r0 = qb * RB;
        const int nr = (int)min((long long)RB, (long long)q.nq * a.g - r0);
        __syncthreads();
        for (int e = threadIdx.x; e < RB * dk4; e += THREADS) {
            const int r = e / dk4, d = e - r * dk4;
            float v = 0.0f;
            if (r < nr && d < a.dk) {
                const int i = (int)a.by_group.div(r0 + r);
                const long long at = (long long)(q.q0 + i) * a.q_stride + (long long)(h * a.g + (r0 + r - i * a.g)) * a.q_head + d;
                v = a.q_type == KV_TYPE_F16 ? __half2float(reinterpret_cast<const __half *>(a.q)[at])
                                            : reinterpret_cast<const float *>(a.q)[at];
            }
            qs[e] = v;
        }
        __syncthreads();
        float m[RB], l[RB], o[RB][DV_LANES];
#pragma unroll
        for (int r = 0; r < RB; r++) {
            m[r] = -INFINITY;
            l[r] = 0.0f;
#pragma unroll
            for (int c = 0; c < DV_LANES; c++) o[r][c] = 0.0f;
        }
        int last = q.ln;                                 // keys behind every row of the block are not read
        if (a.cu_k && a.causal) {
            const long long see = (long long)a.by_group.div(r0 + nr - 1) + (q.ln - q.nq) + 1;
            last = (int)max(0LL, min((long long)q.ln, see));
        }
        for (int t = lo; t < hi; t++) {
            const int j0 = t * TILE + warp * WK;
            if (j0 >= last) continue;
            const int j = j0 + lane;
            int page = 0, off = 0;
            const long long row = j < last ? attn_row(a, q, j, &page, &off) : -1;
            float bias = 0.0f;
            if (row >= 0 && a.beta) bias = a.beta[((size_t)page * a.Hkv + h) * a.page + off];
            const bool there = row >= 0 && bias != -INFINITY;
            const unsigned live = __ballot_sync(~0u, there);
            if (!live) continue;
            simt_load(buf, pitch, a.K + (long long)h * a.k_hb, a.k_rb, a.k_type, a.dk, row, live, k_direct, lane);
            __syncwarp();
            float x[RB];
#pragma unroll
            for (int r = 0; r < RB; r++) x[r] = 0.0f;
#pragma unroll 4
            for (int d = 0; d < dk4; d += 4) {
                const float4 kv = *reinterpret_cast<const float4 *>(buf + lane * pitch + d);
#pragma unroll
                for (int r = 0; r < RB; r++) {
                    const float4 qv = *reinterpret_cast<const float4 *>(qs + r * dk4 + d);
                    x[r] = fmaf(qv.w, kv.w, fmaf(qv.z, kv.z, fmaf(qv.y, kv.y, fmaf(qv.x, kv.x, x[r]))));
                }
            }
            __syncwarp();
            simt_load(buf, pitch, a.V + (long long)h * a.v_hb, a.v_rb, a.v_type, a.dv, row, live, v_direct, lane);
            bool some = false;                           // a key that some rows see and others do not
#pragma unroll
            for (int r = 0; r < RB; r++) {
                const bool sees = there && r < nr && attn_sees(a, q, (int)a.by_group.div(r0 + r), j);
                some |= there && r < nr && !sees;
                const float xr = sees ? fmaf(x[r], a.scale, bias) : -INFINITY;
                float mt = xr;
#pragma unroll
                for (int o2 = 16; o2; o2 >>= 1) mt = fmaxf(mt, __shfl_xor_sync(~0u, mt, o2));
                const float mn = fmaxf(m[r], mt);
                const float base = mn == -INFINITY ? 0.0f : mn;
                const float p = sees ? expf(xr - base) : 0.0f;
                const float f = expf(m[r] - base);       // m = -inf: 0
                m[r] = mn;
                l[r] = l[r] * f + p;                     // per lane; summed over the lanes at the end
#pragma unroll
                for (int c = 0; c < DV_LANES; c++) o[r][c] *= f;
                ps[lane * RB + r] = p;
            }
            some = __any_sync(~0u, some);
            __syncwarp();
#pragma unroll 2
            for (int k = 0; k < WK; k++) {
                float v[DV_LANES], p[RB];
#pragma unroll
                for (int c = 0; c < DV_LANES; c += VEC) {
                    const int d = VEC * lane + 32 * c;
                    const float * at = buf + k * pitch + d;
                    const bool in = d < a.dv;
                    if (VEC == 4) {
                        const float4 w4 = in ? *reinterpret_cast<const float4 *>(at) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        v[c] = w4.x;
                        v[c + 1] = w4.y;
                        v[c + VEC - 2] = w4.z;
                        v[c + VEC - 1] = w4.w;
                    } else {
                        const float2 w2 = in ? *reinterpret_cast<const float2 *>(at) : make_float2(0.0f, 0.0f);
                        v[c] = w2.x;
                        v[c + 1] = w2.y;
                    }
                }
#pragma unroll
                for (int r = 0; r < RB; r += 4) {
                    const float4 p4 = *reinterpret_cast<const float4 *>(ps + k * RB + r);
                    p[r] = p4.x;
                    p[r + 1] = p4.y;
                    p[r + 2] = p4.z;
                    p[r + 3] = p4.w;
                }
                if (some) {                              // what a row does not see may be anything
#pragma unroll
                    for (int r = 0; r < RB; r++)
                        if (p[r] != 0.0f) {
#pragma unroll
                            for (int c = 0; c < DV_LANES; c++) o[r][c] = fmaf(p[r], v[c], o[r][c]);
                        }
                } else {
#pragma unroll
                    for (int r = 0; r < RB; r++)
#pragma unroll
                        for (int c = 0; c < DV_LANES; c++) o[r][c] = fmaf(p[r], v[c], o[r][c]);
                }
            }
            __syncwarp();
        }
        // join the warps
#pragma unroll
        for (int r = 0; r < RB; r++)
#pragma unroll
            for (int o2 = 16; o2; o2 >>= 1) l[r] += __shfl_xor_sync(~0u, l[r], o2);
        __syncthreads();
#pragma unroll
        for (int r = 0; r < RB; r++) {
            if (lane == 0) {
                s_m[warp][r] = m[r];
                s_l[warp][r] = l[r];
            }
#pragma unroll
            for (int c = 0; c < DV_LANES; c++) {
                const int d = VEC * lane + 32 * (c & ~(VEC - 1)) + (c & (VEC - 1));
                if (d < a.dv) joinO[((size_t)warp * RB + r) * a.dv + d] = o[r][c];
            }
        }
        __syncthreads();
        float * part = slot >= 0 ? attn_part(a, qb, h, w, slot) : nullptr;
        for (int e = threadIdx.x; e < nr * a.dv; e += THREADS) {
            const int r = e / a.dv, d = e - r * a.dv;
            float M = -INFINITY;
            for (int u = 0; u < WARPS; u++) M = fmaxf(M, s_m[u][r]);
            const float base = M == -INFINITY ? 0.0f : M;
            float L = 0.0f, O = 0.0f;
            for (int u = 0; u < WARPS; u++) {
                const float f = expf(s_m[u][r] - base);
                L = fmaf(f, s_l[u][r], L);
                O = fmaf(f, joinO[((size_t)u * RB + r) * a.dv + d], O);
            }
            if (part) {
                part[r * a.dv + d] = O;
                if (d == 0) {
                    part[RB * a.dv + r] = M;
                    part[RB * a.dv + RB + r] = L;
                }
            } else {
                const int i = (int)a.by_group.div(r0 + r);
                attn_store(a, (size_t)(q.q0 + i) * a.Hq + h * a.g + (r0 + r - i * a.g), d, O, M, L);
            }
        }
    });
    __syncthreads();
    }
}

// One CTA per (token, query head): the rows whose keys were split over several
// workers, joined in the workers' order, and rows of sequences without keys.
// Sequences that one worker covered are written already. Bound by the latency of
// its reads, so they are few and side by side: which workers share the sequence
// (meta), then all maxima and sums, then the outputs, four values a lane and
// eight partial results in flight per warp. What does not depend on the kernel
// before is done first, while that one still runs. 32 rows of 128 values, 148
// partial results: about 6 us of a single-token call's 19.
constexpr int JOIN_MOST = 512;                           // partial results whose factors fit shared memory at a time
__global__ void __launch_bounds__(128) k_attn_join(const __grid_constant__ kvc_attn_args a) {
    __shared__ float s_f[JOIN_MOST], s_o[4][KVC_MAX_D], s_red[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int token = (int)(blockIdx.x / (unsigned)a.Hq), hq = (int)(blockIdx.x - (unsigned)token * (unsigned)a.Hq);
    // the sequence of the token
    int s = -1;
    for (int s0 = 0; s0 < a.n_seqs && s < 0; s0 += 32) {
        bool in = false;
        if (s0 + lane < a.n_seqs) {
            const int q0 = min(max(a.cu_q[s0 + lane], 0), a.n_total), q1 = min(max(a.cu_q[s0 + lane + 1], q0), a.n_total);
            in = token >= q0 && token < q1;
        }
        const unsigned b = __ballot_sync(~0u, in);
        if (b) s = s0 + __ffs(b) - 1;
    }
    if (s < 0 || token - min(max(a.cu_q[s], 0), a.n_total) >= a.max_q) {
        cudaGridDependencySynchronize();     // on every path: what follows in the stream relies on it
        return;
    }
    const kvc_attn_seq q = attn_seq(a, s);
    const int i = token - q.q0;
    const int h = hq / a.g;
    const int rho = i * a.g + (hq - h * a.g);
    const int qb = rho / a.rb, r = rho - qb * a.rb;
    const size_t row = (size_t)token * a.Hq + hq;
    cudaGridDependencySynchronize();
    if (q.ln == 0) {
        for (int d = threadIdx.x; d < a.dv; d += 128) attn_store(a, row, d, 0.0f, 0.0f, 0.0f);
        return;
    }
    if (a.W == 1) return;
    const int w0 = a.meta[((size_t)qb * a.n_seqs + s) * 2], w1 = a.meta[((size_t)qb * a.n_seqs + s) * 2 + 1];
    if (w0 >= w1) return;
    // the first worker's piece lies in its slot 1 (its stretch began before the sequence or with it), the others' in slot 0
    const size_t step = 2 * (size_t)a.rb * (a.dv + 2);
    const float * first_p = attn_part(a, qb, h, w0, 1);
    auto at = [&](int w) { return w == w0 ? first_p : first_p + (size_t)(w - w0) * step - step / 2; };
    auto over = [&](float v, bool largest) {             // of all threads
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            const float u = __shfl_xor_sync(~0u, v, o);
            v = largest ? fmaxf(v, u) : v + u;
        }
        float * red = s_red + (largest ? 0 : 4);
        if (lane == 0) red[warp] = v;
        __syncthreads();
        return largest ? fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])) : (red[0] + red[1]) + (red[2] + red[3]);
    };
    const int n = w1 - w0 + 1;
    float M = -INFINITY;
    for (int k = threadIdx.x; k < n; k += 128) M = fmaxf(M, at(w0 + k)[a.rb * a.dv + r]);
    M = over(M, true);
    const float base = M == -INFINITY ? 0.0f : M;
    const bool wide = (a.dv & 3) == 0;                   // the partial results' rows lie on 16-byte boundaries
    float L = 0.0f;
    float4 O[2] = {make_float4(0, 0, 0, 0), make_float4(0, 0, 0, 0)};
    float O1[KVC_MAX_D / 32];
#pragma unroll
    for (int c = 0; c < KVC_MAX_D / 32; c++) O1[c] = 0.0f;
    for (int k0 = 0; k0 < n; k0 += JOIN_MOST) {
        const int m = min(n - k0, JOIN_MOST);
        __syncthreads();
        for (int k = threadIdx.x; k < m; k += 128) {
            const float * p = at(w0 + k0 + k) + a.rb * a.dv + r;
            const float f = expf(p[0] - base);
            s_f[k] = f;
            L = fmaf(f, p[a.rb], L);
        }
        __syncthreads();
        if (wide) {
#pragma unroll
            for (int c = 0; c < 2; c++) {
                const int d = 4 * lane + 128 * c;
                if (d >= a.dv) break;
                for (int k = warp; k < m; k += 32) {
                    float4 v[8];
#pragma unroll
                    for (int u = 0; u < 8; u++)
                        if (k + 4 * u < m) v[u] = *reinterpret_cast<const float4 *>(at(w0 + k0 + k + 4 * u) + r * a.dv + d);
#pragma unroll
                    for (int u = 0; u < 8; u++)
                        if (k + 4 * u < m) {
                            const float f = s_f[k + 4 * u];
                            O[c].x = fmaf(f, v[u].x, O[c].x);
                            O[c].y = fmaf(f, v[u].y, O[c].y);
                            O[c].z = fmaf(f, v[u].z, O[c].z);
                            O[c].w = fmaf(f, v[u].w, O[c].w);
                        }
                }
            }
        } else {
            for (int k = warp; k < m; k += 4) {
                const float * p = at(w0 + k0 + k) + r * a.dv;
                const float f = s_f[k];
#pragma unroll
                for (int c = 0; c < KVC_MAX_D / 32; c++)
                    if (lane + 32 * c < a.dv) O1[c] = fmaf(f, p[lane + 32 * c], O1[c]);
            }
        }
    }
    if (wide) {
#pragma unroll
        for (int c = 0; c < 2; c++)
            if (4 * lane + 128 * c < a.dv) *reinterpret_cast<float4 *>(&s_o[warp][4 * lane + 128 * c]) = O[c];
    } else {
#pragma unroll
        for (int c = 0; c < KVC_MAX_D / 32; c++)
            if (lane + 32 * c < a.dv) s_o[warp][lane + 32 * c] = O1[c];
    }
    L = over(L, false);
    for (int d = threadIdx.x; d < a.dv; d += 128)
        attn_store(a, row, d, (s_o[0][d] + s_o[1][d]) + (s_o[2][d] + s_o[3][d]), M, L);
}

size_t simt_smem(int dk, int dv) {
    const int pitch = simt_pitch(dk > dv ? dk : dv);
    return (size_t)(RB * ((dk + 3) & ~3) + WARPS * RB * WK + WARPS * WK * pitch) * sizeof(float);
}

template <int C>
int launch_simt(const kvc_attn_args & a, dim3 grid, cudaStream_t st) {
    // the limit is the function's, whoever calls it: one value for all sizes
    static std::atomic<bool> set[64];
    int dev = 0;
    KVC_CUDA(cudaGetDevice(&dev));
    if (!set[dev & 63].load(std::memory_order_relaxed)) {
        KVC_CUDA(cudaFuncSetAttribute(k_attn_simt<C>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)simt_smem(KVC_MAX_D, KVC_MAX_D)));
        set[dev & 63].store(true, std::memory_order_relaxed);
    }
    const size_t sm = simt_smem(a.dk, a.dv);
    k_attn_simt<C><<<grid, THREADS, sm, st>>>(a);
    g_serve_launches++;
    KVC_CUDA(cudaGetLastError());
    return KVC_OK;
}

}  // namespace

void kvc_attn_simt_split(kvc_attn_args * a, int sms, bool whole) {
    a->rb = RB;
    a->tile = TILE;
    a->by_tile = kvc_make_divisor(TILE);
    // enough CTAs for four waves' worth of two per SM
    const long long blocks = ((long long)a->max_q * a->g + RB - 1) / RB * a->Hkv;
    const long long w = whole || blocks <= 0 ? 1 : (8LL * sms + blocks - 1) / blocks;
    a->W = (int)(w < 1 ? 1 : w);
    a->n_parts = (int)(blocks / a->Hkv);
}

int kvc_launch_attn_simt(const kvc_attn_args & a, cudaStream_t st) {
    const long long blocks = ((long long)a.max_q * a.g + RB - 1) / RB;
    if (blocks <= 0 || a.n_seqs == 0 || a.n_total == 0) return KVC_OK;
    const long long cap = 65535 / a.Hkv;
    const dim3 grid((unsigned)a.W, (unsigned)((blocks < cap ? blocks : cap) * a.Hkv));
    int rc;
    if (a.dv <= 64) rc = launch_simt<2>(a, grid, st);
    else if (a.dv <= 128) rc = launch_simt<4>(a, grid, st);
    else rc = launch_simt<8>(a, grid, st);
    return rc ? rc : kvc_launch_attn_join(a, false, st);
}

int kvc_launch_attn_join(const kvc_attn_args & a, bool overlap, cudaStream_t st) {
    const long long units = (long long)a.n_total * a.Hq;
    if (units == 0) return KVC_OK;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)units);
    cfg.blockDim = dim3(128);
    cfg.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = overlap ? 1 : 0;
    KVC_CUDA(cudaLaunchKernelEx(&cfg, k_attn_join, a));
    g_serve_launches++;
    return KVC_OK;
}

kvc_encode_fn kvc_tensor_map_encoder() {
    static const kvc_encode_fn fn = [] {
        void * p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            p = nullptr;
        }
        return (kvc_encode_fn)p;
    }();
    return fn;
}
