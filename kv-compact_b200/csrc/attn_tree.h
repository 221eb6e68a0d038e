// attn_tree.h — the tensor-core tree attention's entry points within the library.
#pragma once

#include "attn.h"

template <int V>
struct kvc_int {
    static constexpr int value = V;
};

// Whether the kernel takes these rows and shapes; sets a's split and the number
// of row blocks.
bool kvc_attn_tree_mma_plan(kvc_attn_args * a, int sms, long long * blocks);
int kvc_launch_attn_tree_mma(const kvc_attn_args & a, cudaStream_t st);

// The same for entries with many query rows (attn_tree_tc.cu).
bool kvc_attn_tree_tc_plan(kvc_attn_args * a, int sms, long long * blocks);
int kvc_launch_attn_tree_tc(const kvc_attn_args & a, cudaStream_t st);
