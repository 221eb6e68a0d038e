// attn_simt.cu — the general attention kernel and the join of partial results
// (include/kvc-attn.h). The tensor-core kernels (attn_tree.cu,
// attn_prompt.cu) take the common types and shapes; this one takes the rest:
// F32 rows, head sizes and strides that those do not read.
//
//   x_ij = scale q_i.k_j (+ beta_j),  m = max_j x_ij,  l = sum_j exp(x_ij - m),
//   out_i = (sum_j exp(x_ij - m) v_j) / l,  lse_i = m + log l
//
// in one pass over the keys with a running m, l and sum. 160,000 Q8_0 keys of 8
// heads, 4 query rows each, 128 values: 1.41 ms here, 0.14 ms in k_tree_mma.
#include "attn.h"
#include "attn_tc.h"

#include <math.h>

namespace {

constexpr int RB = 8, TILE = 128;        // query rows and keys per CTA and step
constexpr int WARPS = 4, THREADS = 32 * WARPS, WK = 32;
static_assert(TILE == WARPS * WK, "a tile is one key per lane");

// One CTA: 8 query rows of one KV head against its stretch of the keys. A
// warp takes 32 keys of a tile, decodes their K rows into its own shared
// memory, scores one key per lane, then does the same with V with one output
// dimension per lane: no barrier inside the loop. Bound by the shared-memory
// reads of the two products (9 words per 8 multiply-adds).
template <int DV_LANES>
__global__ void __launch_bounds__(THREADS) k_attn_simt(const __grid_constant__ kvc_attn_args a) {
    extern __shared__ float sm[];
    const int pitch = max(a.dk, a.dv) | 1;               // odd: a column read hits 32 banks
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float * qs = sm;                                     // [RB][dk]
    float * ps = qs + RB * a.dk + warp * (RB * WK);      // [RB][32] of this warp
    float * buf = qs + RB * a.dk + WARPS * RB * WK + (size_t)warp * WK * pitch;
    float * joinO = qs + RB * a.dk + WARPS * RB * WK;    // reused after the loop: [WARPS][RB][dv] (dv <= pitch, RB <= 32)
    __shared__ float s_m[WARPS][RB], s_l[WARPS][RB];
    const int h = blockIdx.y % a.Hkv, w = blockIdx.x;
    const int n_blocks = (int)(((long long)a.max_q * a.g + RB - 1) / RB);

    for (int qb = blockIdx.y / a.Hkv; qb < n_blocks; qb += gridDim.y / a.Hkv) {
    attn_walk(a, qb, qb + 1, w, h == 0 && threadIdx.x < 32, [&](int, const kvc_attn_seq & q, int lo, int hi, int slot) {
        const int r0 = qb * RB;
        const int nr = (int)min((long long)RB, (long long)q.nq * a.g - r0);
        __syncthreads();
        for (int e = threadIdx.x; e < RB * a.dk; e += THREADS) {
            const int r = e / a.dk, d = e - r * a.dk;
            float v = 0.0f;
            if (r < nr) {
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
            for (int k = 0; k < WK; k++) {
                const long long rk = __shfl_sync(~0u, row, k);
                const bool ok = (live >> k) & 1u;
                const uint8_t * p = a.K + (ok ? rk : 0) * a.k_rb + (long long)h * a.k_hb;
                for (int d = lane; d < a.dk; d += 32) buf[k * pitch + d] = ok ? attn_elem(p, a.k_type, d) : 0.0f;
            }
            __syncwarp();
            float x[RB];
#pragma unroll
            for (int r = 0; r < RB; r++) x[r] = 0.0f;
            for (int d = 0; d < a.dk; d++) {
                const float kv = buf[lane * pitch + d];
#pragma unroll
                for (int r = 0; r < RB; r++) x[r] = fmaf(qs[r * a.dk + d], kv, x[r]);
            }
            __syncwarp();
            for (int k = 0; k < WK; k++) {
                const long long rk = __shfl_sync(~0u, row, k);
                const bool ok = (live >> k) & 1u;
                const uint8_t * p = a.V + (ok ? rk : 0) * a.v_rb + (long long)h * a.v_hb;
                for (int d = lane; d < a.dv; d += 32) buf[k * pitch + d] = ok ? attn_elem(p, a.v_type, d) : 0.0f;
            }
#pragma unroll
            for (int r = 0; r < RB; r++) {
                const bool sees = there && r < nr && attn_sees(a, q, (int)a.by_group.div(r0 + r), j);
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
                ps[r * WK + lane] = p;
            }
            __syncwarp();
            for (int k = 0; k < WK; k++) {
                float v[DV_LANES];
#pragma unroll
                for (int c = 0; c < DV_LANES; c++) v[c] = lane + 32 * c < a.dv ? buf[k * pitch + lane + 32 * c] : 0.0f;
#pragma unroll
                for (int r = 0; r < RB; r++) {
                    const float p = ps[r * WK + k];
                    if (p != 0.0f) {                     // a hidden row's V may be anything
#pragma unroll
                        for (int c = 0; c < DV_LANES; c++) o[r][c] = fmaf(p, v[c], o[r][c]);
                    }
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
            for (int c = 0; c < DV_LANES; c++)
                if (lane + 32 * c < a.dv) joinO[((size_t)warp * RB + r) * a.dv + lane + 32 * c] = o[r][c];
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
    const int pitch = (dk > dv ? dk : dv) | 1;
    return (size_t)(RB * dk + WARPS * RB * WK + WARPS * WK * pitch) * sizeof(float);
}

template <int C>
int launch_simt(const kvc_attn_args & a, dim3 grid, cudaStream_t st) {
    const size_t sm = simt_smem(a.dk, a.dv);
    KVC_CUDA(cudaFuncSetAttribute(k_attn_simt<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sm));
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
