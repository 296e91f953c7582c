// mllm_attn_f16.hip -- mllm_attn_paged's kernels for a cache of f16.
#include "mllm_paged_attn.h"

int mllm::paged::attn_f16(const AttnArgs &A, dim3 grid, hipStream_t st) { return attn_dispatch<KvF16>(A, grid, st); }
