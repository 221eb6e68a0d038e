// attn_tree.h — the tensor-core tree attention's entry points within the library.
#pragma once

#include "attn.h"

template <int V>
struct kvc_int {
    static constexpr int value = V;
};

struct kvc_tree_mma_plan {
    int db, nb, np;        // 32-value blocks, 8-row blocks and fp16 pieces that the kernel is built for
    int rb;                // query rows per CTA
    long long blocks;      // row blocks
};

// Whether the kernel takes these rows and shapes; sets a->W and the plan.
bool kvc_attn_tree_mma_plan(kvc_attn_args * a, int sms, kvc_tree_mma_plan * p);
int kvc_launch_attn_tree_mma(const kvc_attn_args & a, const kvc_tree_mma_plan & p, cudaStream_t st);
