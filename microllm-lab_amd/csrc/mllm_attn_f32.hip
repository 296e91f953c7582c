// mllm_attn_f32.hip -- mllm_attn_paged's kernels for a cache of f32.
#include "mllm_paged_attn.h"

int mllm::paged::attn_f32(const AttnArgs &A, dim3 grid, hipStream_t st) { return attn_dispatch<KvF32>(A, grid, st); }
