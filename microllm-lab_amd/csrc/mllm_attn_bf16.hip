// mllm_attn_bf16.hip -- mllm_attn_paged's kernels for a cache of bf16.
#include "mllm_paged_attn.h"

int mllm::paged::attn_bf16(const AttnArgs &A, dim3 grid, hipStream_t st) { return attn_dispatch<KvBf16>(A, grid, st); }
