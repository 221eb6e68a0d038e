// serve.h — shared pieces of the serving operators (pages.cu, attn_*.cu).
#pragma once

#include "kvc-attn.h"
#include "kvc-pages.h"
#include "kvc_internal.h"

#include <atomic>
#include <initializer_list>

// The current device, checked once per device: >= 0 SM count, or a negative
// error code when it cannot run the library's kernels.
int kvc_serve_device();
// Kernels launched by the serving operators (part of kvc_launch_count).
extern std::atomic<uint64_t> g_serve_launches;

// Whether arrays of 32-bit numbers lie on 4-byte boundaries (a kernel that reads others faults).
inline bool kvc_words_aligned(std::initializer_list<const void *> arrays) {
    for (const void * p : arrays)
        if ((uintptr_t)p & 3) return false;
    return true;
}

// Argument checks of a page cache (null pointers, counts, row sizes).
int kvc_check_cache(const kvc_page_cache * c);

// Quotient and remainder by a run-time divisor that stays the same for a
// launch: n / d for 0 <= n < 2^31 as the high word of n * m, m =
// ceil(2^(32+s) / d) with s = ceil(log2 d) - 1 so that m < 2^32 (d >= 2; the
// error m*d - 2^(32+s) < d <= 2^(s+1) keeps the quotient exact for n < 2^31).
struct kvc_divisor {
    uint32_t d, m, s;
    KVC_HD uint32_t div(uint32_t n) const {
#ifdef __CUDA_ARCH__
        return d == 1 ? n : __umulhi(n, m) >> s;
#else
        return d == 1 ? n : (uint32_t)(((uint64_t)n * m) >> 32) >> s;
#endif
    }
};
inline kvc_divisor kvc_make_divisor(uint32_t d) {
    kvc_divisor v{d, 0, 0};
    if (d > 1) {
        uint32_t s = 0;
        while ((2u << s) < d) s++;
        v.s = s;
        v.m = (uint32_t)(((1ull << (32 + s)) + d - 1) / d);
    }
    return v;
}
