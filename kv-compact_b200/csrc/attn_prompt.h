// attn_prompt.h — the tensor-core prompt attention's entry points within the library.
#pragma once

#include "attn.h"

// Whether the kernel takes these types, sizes, strides and addresses.
bool kvc_attn_prompt_tc_ok(const kvc_attn_args & a);
int kvc_launch_attn_prompt_tc(const kvc_attn_args & a, cudaStream_t st);
