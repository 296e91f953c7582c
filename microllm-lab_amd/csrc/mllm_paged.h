// mllm_paged.h -- what the translation units of the paged operators share: the
// cache's storages, a pool of pages as the kernels take it, and the attention's
// arguments and layouts.
#pragma once

#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mllm {
namespace paged {

typedef float v4f __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------- storages
// An element of the cache: f32, f16 or bf16, rounded to nearest even.
struct KvF32 {
  using T = float;
  static __device__ __forceinline__ T put(float v) { return v; }
};
struct KvF16 {
  using T = uint16_t;
  static __device__ __forceinline__ T put(float v) { return __half_as_ushort(__float2half_rn(v)); }
};
struct KvBf16 {
  using T = uint16_t;
  static __device__ __forceinline__ T put(float v) {
    const uint32_t u = __float_as_uint(v);
    if (v != v) return (uint16_t)((u >> 16) | 0x40u);  // NaN stays NaN
    return (uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
  }
};

// A pool of pages as the kernels take it.
struct Pages {
  void *k, *v;
  const int32_t *table;
  int64_t page_stride, head_stride, row_stride;
  int pages, page_size, sequences, table_cols, n_kv, hd;
  uint32_t page_magic;  // floor(2^32 / page_size) + 1
};

// pos / page_size: with magic = 2^32 / d + e, 0 < e <= 1, the product's high
// word is the quotient or one more (pos e / 2^32 < 1).
__device__ __forceinline__ int page_of(const Pages &P, int pos) {
  if (P.page_size == 1) return pos;
  const uint32_t q = __umulhi((uint32_t)pos, P.page_magic);
  return (int)(q - (q * (uint32_t)P.page_size > (uint32_t)pos ? 1u : 0u));
}

// ---------------------------------------------------------------- attention over pages
constexpr int APLACES = 512;           // positions whose places in the pool are in LDS at a time, for each wave
constexpr int kCounters = 4096;        // rows' heads that may be split, each with its counter
constexpr int kParts = 256;            // parts of a row at most
constexpr float LOG2E = 1.44269504088896340736f;

struct AttnArgs {
  Pages P;
  const float *q;
  const int32_t *seq, *len;
  float *out, *part;  // part: [units][splits], each the heads' sums [heads][hd], then their (maximum, sum)
  unsigned *count;    // [kCounters] parts that are there, zero between calls
  int n_heads, rep, tiles, heads, max_len, chunk, splits;  // heads: query heads of a workgroup at most
  float scale;
  int waves;          // of a workgroup: four, or one for many short rows (splits = 1)
  int stream;         // loads past the caches
};

// How a head's row of HD elements is laid on lanes: keys in runs of 16 bytes
// (RUN elements, NR of them to a lane), values EL elements to each of LPR lanes,
// 16 bytes where the row's size allows it.
template <class KV, int DC>
struct Lay {
  static constexpr int HD = 32 * DC, ES = (int)sizeof(typename KV::T), RUN = 16 / ES, NR = HD / (4 * RUN);
  static constexpr bool fits(int l) { return l <= 64 && HD % l == 0 && HD / l * ES % 4 == 0; }
  static constexpr int lanes() {
    int l = 4;
    while (l * 16 < HD * ES) l *= 2;
    while (!fits(l)) l /= 2;
    return l;
  }
  static constexpr int LPR = lanes(), EL = HD / LPR, G = 64 / LPR;  // G: positions of one load
  static constexpr int ROW = HD * ES, PT = ROW <= 128 ? 4 : ROW < 256 ? 2 : 1, TP = 16 * PT, NU = TP / G;
  static constexpr int AQ = EL <= 8 ? 16 : 8;                       // query heads of a workgroup at most
  static constexpr int PS = TP + (G < 4 ? 4 : G);                   // floats of a row of weights, off the banks' period
};

// The kernel for A.heads query heads and A.P.hd elements, on the storage's own
// translation unit (mllm_attn_f32.hip, mllm_attn_f16.hip, mllm_attn_bf16.hip).
int attn_f32(const AttnArgs &A, dim3 grid, hipStream_t st);
int attn_f16(const AttnArgs &A, dim3 grid, hipStream_t st);
int attn_bf16(const AttnArgs &A, dim3 grid, hipStream_t st);

}  // namespace paged
}  // namespace mllm
