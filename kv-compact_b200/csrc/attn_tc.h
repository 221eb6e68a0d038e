// attn_tc.h — what the tcgen05 attention kernels share: descriptors of
// 128-byte-swizzled tiles, TMEM access and packed fp32 arithmetic.
#pragma once

#include <cuda.h>

#include "tc_sm100.h"

namespace kvc_attn_tc {

using kvc_tc::smem_u32;

// Shared-memory descriptors of tiles whose rows are 128 bytes, 128-byte swizzled
// as TMA writes them (start addresses below are multiples of 16 bytes).
// K-major operand (rows = M or N, 64 values of K a row): groups of 8 rows 1,024 bytes apart.
__device__ __forceinline__ uint64_t desc_k(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
           (uint64_t)2 << 61;
}
// N-major operand (rows = K, 64 values of N a row): blocks of 64 N `next` bytes apart, groups of 8 K 1,024 bytes.
__device__ __forceinline__ uint64_t desc_n(uint32_t addr, uint32_t next) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | (uint64_t)(next >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
           (uint64_t)2 << 61;
}

// The MMA warp runs these with all its lanes, and one of them (always the same)
// issues: in warp-uniform code the operands stay in uniform registers (a branch
// on the lane made the prompt kernel's issue 78 cycles per instruction, more
// than the instruction itself takes).
// D[tmem] (+)= A[tmem] B[smem], fp16 operands.
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n"
        :: "r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc));
}
// D[tmem] (+)= A[smem] B[smem].
__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n"
        :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc));
}
// `go` false in that lane: nothing is committed (a warp whose lanes may differ in it takes no branch on it).
__device__ __forceinline__ void commit_mma(uint64_t * mbar, bool go = true) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "setp.ne.and.b32 q, %1, 0, q;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n"
        :: "r"(smem_u32(mbar)), "r"((uint32_t)go) : "memory");
}

#define KVC_R8(r, o) "=r"(r[o]), "=r"(r[o + 1]), "=r"(r[o + 2]), "=r"(r[o + 3]), "=r"(r[o + 4]), "=r"(r[o + 5]), "=r"(r[o + 6]), "=r"(r[o + 7])
#define KVC_I8(r, o) "r"(r[o]), "r"(r[o + 1]), "r"(r[o + 2]), "r"(r[o + 3]), "r"(r[o + 4]), "r"(r[o + 5]), "r"(r[o + 6]), "r"(r[o + 7])
// 32 consecutive columns of this thread's lane, without waiting.
__device__ __forceinline__ void ld32(uint32_t addr, uint32_t * r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : KVC_R8(r, 0), KVC_R8(r, 8), KVC_R8(r, 16), KVC_R8(r, 24) : "r"(addr));
}
__device__ __forceinline__ void st32(uint32_t addr, const uint32_t * r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
        :: "r"(addr), KVC_I8(r, 0), KVC_I8(r, 8), KVC_I8(r, 16), KVC_I8(r, 24) : "memory");
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
// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    unsigned long long x, y, z, d;
    memcpy(&x, &a, 8), memcpy(&y, &b, 8), memcpy(&z, &c, 8);
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(x), "l"(y), "l"(z));
    float2 r;
    memcpy(&r, &d, 8);
    return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    unsigned long long x, y, d;
    memcpy(&x, &a, 8), memcpy(&y, &b, 8);
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(x), "l"(y));
    float2 r;
    memcpy(&r, &d, 8);
    return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    unsigned long long x, y, d;
    memcpy(&x, &a, 8), memcpy(&y, &b, 8);
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(x), "l"(y));
    float2 r;
    memcpy(&r, &d, 8);
    return r;
}

// Dynamic shared memory from its next 1,024-byte boundary (the swizzle's period); stays a shared-memory pointer.
__device__ __forceinline__ uint8_t * aligned_1024(uint8_t * p) { return p + ((1024u - (smem_u32(p) & 1023u)) & 1023u); }

#undef KVC_R8
#undef KVC_I8

}  // namespace kvc_attn_tc

using kvc_encode_fn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                               const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                               CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
// cuTensorMapEncodeTiled of the driver, or null (attn_simt.cu).
kvc_encode_fn kvc_tensor_map_encoder();
