// mllm_sample.hip -- drawing tokens from logits (include/mllm.h mllm_sample).
// All pointers are device pointers.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mllm_device.h"
#include "mllm_host.h"

using namespace mllm;

namespace {

// One workgroup per row.  With d = max - z, a token's weight is
//   W = round(2^44 2^(-d log2(e) / T)),  0 below 2^0 (d > dlim),
// an integer, so that every sum is exact and the same in any order: the
// weights of up to 2^19 tokens fit 64 bits, and 2^-45 of the largest is a
// thousandth of what float64 sums of float64 weights would need to name
// another token once in a million rows.
//
// The order of the tokens is: larger logit first, equal ones by index.  top-k
// and top-p both keep a prefix of it -- the shortest whose count reaches k, or
// whose weight reaches top_p of the total -- and so does min-p.  No sort: the
// last token of a prefix is found by histograms (count or weight per bin, in
// LDS), each level taking the bin in which the sum passes its target: first
// 2048 bins of equal width in d, then of equal width in the bits of the logit,
// at most three times, and tokens that still tie by index.
//
// The draw itself sums the kept weights by 256-token chunks in index order and
// takes the first token whose running sum is more than u of the total.
constexpr int ST = 1024;        // threads
constexpr int SW = ST / 64;     // waves
constexpr int SB = 2048;        // bins of a histogram, and chunks of a row at most
constexpr int kMaxVocab = SB * 256;
constexpr int WBITS = 44;

typedef unsigned long long u64;

struct SampleArgs {
  const float *logits, *temperature, *top_p, *min_p, *u;
  const int32_t *top_k;
  int32_t *ids;
  float *probs;
  int vocab;
};

// Order-preserving bits of a float (-0 and +0 tie, as the numbers do).
__device__ __forceinline__ uint32_t key_of(float z) {
  const uint32_t b = __float_as_uint(z + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// A row's state, the same in every thread.
struct Row {
  float zmax, dlim;
  double c;           // log2(e) / T
  uint32_t key_cut;   // kept: key > key_cut, or key == key_cut and index <= idx_cut
  int idx_cut;
  u64 wmin;           // kept: weight at least this
  int first;          // the first token of the order, always kept
};

__device__ __forceinline__ float dist(const Row &R, float z) { return z == R.zmax ? 0.f : R.zmax - z; }
__device__ __forceinline__ bool live(const Row &R, float z) { return dist(R, z) <= R.dlim; }  // not NaN, not -inf

// W of a live token: 2^t by its Taylor series about the nearest integer, whose
// next term is below 2^-47, and the scaling in the exponent.
__device__ __forceinline__ u64 weight(const Row &R, float z) {
  const double d = z == R.zmax ? 0.0 : (double)R.zmax - (double)z, t = -d * R.c, n = rint(t), f = t - n;
  double p = 4.4455382718708116e-10;                       // ln2^k / k!, k = 11
  p = __builtin_fma(p, f, 7.0549116208011233e-09);
  p = __builtin_fma(p, f, 1.0178086009239700e-07);
  p = __builtin_fma(p, f, 1.3215486790144309e-06);
  p = __builtin_fma(p, f, 1.5252733804059840e-05);
  p = __builtin_fma(p, f, 1.5403530393381609e-04);
  p = __builtin_fma(p, f, 1.3333558146428443e-03);
  p = __builtin_fma(p, f, 9.6181291076284772e-03);
  p = __builtin_fma(p, f, 5.5504108664821580e-02);
  p = __builtin_fma(p, f, 2.4022650695910072e-01);
  p = __builtin_fma(p, f, 6.9314718055994531e-01);
  p = __builtin_fma(p, f, 1.0);
  const long long e = (long long)__double_as_longlong(p) + ((long long)((int)n + WBITS) << 52);
  return (u64)__double_as_longlong(__longlong_as_double(e) + 4503599627370496.0) & 0xfffffffffffffull;
}

__device__ __forceinline__ bool in_cut(const Row &R, float z, int i) {
  const uint32_t k = key_of(z);
  return live(R, z) && (k > R.key_cut || (k == R.key_cut && i <= R.idx_cut));
}

__device__ __forceinline__ u64 wave_incl(u64 v) {  // inclusive scan over the lanes
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const u64 o = __shfl_up(v, s);
    if (lane >= s) v += o;
  }
  return v;
}

struct Lds {
  u64 bin[SB];
  u64 wave[SW];
  uint32_t wk[2 * SW];
  // the bin that scan_find has found: its number, the sum before it, its own sum
  int at;
  u64 before, own;
  float wv[SW];
  int wi[SW];
  int id;
};

// The first bin at which the running sum reaches target (>= 1), in L.at /
// before / own; the total (all bins) is returned.  L.at = -1 where the total
// does not reach it.  Ends in a barrier.
__device__ u64 scan_find(Lds &L, u64 target) {
  const int t = threadIdx.x, wv = t >> 6;
  __syncthreads();
  const u64 a = L.bin[2 * t], b = L.bin[2 * t + 1], incl = wave_incl(a + b);
  if ((t & 63) == 63) L.wave[wv] = incl;
  if (t == 0) L.at = -1;
  __syncthreads();
  u64 off = 0, total = 0;
#pragma unroll
  for (int w = 0; w < SW; ++w) {
    const u64 v = L.wave[w];
    if (w < wv) off += v;
    total += v;
  }
  const u64 e0 = off + incl - a - b, e1 = e0 + a, e2 = e1 + b;
  if (e0 < target && target <= e2) {
    const bool lo = target <= e1;
    L.at = 2 * t + (lo ? 0 : 1);
    L.before = lo ? e0 : e1;
    L.own = lo ? a : b;
  }
  __syncthreads();
  return total;
}

__device__ __forceinline__ void clear_bins(Lds &L) {
  __syncthreads();
  L.bin[2 * threadIdx.x] = 0;
  L.bin[2 * threadIdx.x + 1] = 0;
  __syncthreads();
}

// The tokens of a row, chunk by chunk: lane l of chunk c holds the tokens
// 256 c + 4 l .. + 3.  A wave takes a run of neighbouring chunks.
struct Span {
  const float *x;
  int vocab, c0, c1;
  __device__ __forceinline__ float4 load(int c) const {
    const int i = 256 * c + 4 * (int)(threadIdx.x & 63);
    if (i + 4 <= vocab) return ld4u(x + i);
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = i + e < vocab ? x[i + e] : -INFINITY;
    return make_float4(v[0], v[1], v[2], v[3]);
  }
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    for (int c = c0; c < c1; ++c) {
      const float4 v = load(c);
      const int i = 256 * c + 4 * (int)(threadIdx.x & 63);
      f(v.x, i), f(v.y, i + 1), f(v.z, i + 2), f(v.w, i + 3);
    }
  }
};

// Shortens the cut to the shortest prefix of the order whose sum -- the count
// of its tokens, or their weight -- reaches target; nothing where the tokens
// inside the present cut do not reach it.
template <bool MASS>
__device__ void cut(Lds &L, const Span &S, Row &R, u64 target) {
  const float s0 = R.dlim > 0.f ? (float)SB / R.dlim : 0.f;
  auto bin0 = [&](float z) { return min(SB - 1, (int)(dist(R, z) * s0)); };
  clear_bins(L);
  S.each([&](float z, int i) {
    if (in_cut(R, z, i)) atomicAdd(&L.bin[bin0(z)], MASS ? weight(R, z) : 1ull);
  });
  scan_find(L, target);
  const int b0 = L.at;
  if (b0 < 0) return;
  u64 rest = target - L.before;
  // the range of the bin's keys
  uint32_t hi = 0u, lo = 0xffffffffu;
  S.each([&](float z, int i) {
    if (in_cut(R, z, i) && bin0(z) == b0) {
      const uint32_t k = key_of(z);
      hi = max(hi, k);
      lo = min(lo, k);
    }
  });
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    hi = max(hi, (uint32_t)__shfl_xor((int)hi, s));
    lo = min(lo, (uint32_t)__shfl_xor((int)lo, s));
  }
  if ((threadIdx.x & 63) == 0) L.wk[threadIdx.x >> 6] = hi, L.wk[SW + (threadIdx.x >> 6)] = lo;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < SW; ++w) hi = max(hi, L.wk[w]), lo = min(lo, L.wk[SW + w]);
  u64 own = L.own;
  while (hi != lo) {
    const uint32_t range = hi - lo;
    const int sh = max(0, 32 - __clz(range) - 11);
    clear_bins(L);
    S.each([&](float z, int i) {
      const uint32_t k = key_of(z);
      if (k <= hi && k >= lo && in_cut(R, z, i) && bin0(z) == b0)
        atomicAdd(&L.bin[(hi - k) >> sh], MASS ? weight(R, z) : 1ull);
    });
    scan_find(L, rest);
    rest -= L.before;
    own = L.own;
    const uint32_t h = hi - ((uint32_t)L.at << sh);
    lo = h - lo < (1u << sh) ? lo : h - ((1u << sh) - 1u);
    hi = h;
  }
  // the first `need` of the tokens that tie at this key, by index
  const u64 unit = MASS ? weight(R, hi & 0x80000000u ? __uint_as_float(hi ^ 0x80000000u) : __uint_as_float(~hi)) : 1ull;
  const u64 need = (rest + unit - 1) / unit;
  int idx = R.key_cut == hi ? R.idx_cut : 0x7fffffff;
  if (need * unit < own) {
    // tokens at the key by chunk, in index order
    clear_bins(L);
    for (int c = S.c0; c < S.c1; ++c) {
      const float4 v = S.load(c);
      const int i = 256 * c + 4 * (int)(threadIdx.x & 63);
      auto hit = [&](float z, int e) { return key_of(z) == hi && in_cut(R, z, i + e); };
      const int n = __popcll(__ballot(hit(v.x, 0))) + __popcll(__ballot(hit(v.y, 1))) + __popcll(__ballot(hit(v.z, 2))) +
                    __popcll(__ballot(hit(v.w, 3)));
      if ((threadIdx.x & 63) == 0) L.bin[c] = (u64)n;
    }
    scan_find(L, need);
    const int c = L.at;
    if (c >= S.c0 && c < S.c1) {
      const float4 v = S.load(c);
      const float z[4] = {v.x, v.y, v.z, v.w};
      const int i = 256 * c + 4 * (int)(threadIdx.x & 63);
      u64 n = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) n += key_of(z[e]) == hi && in_cut(R, z[e], i + e);
      u64 k = L.before + wave_incl(n) - n;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (key_of(z[e]) == hi && in_cut(R, z[e], i + e) && ++k == need) L.id = i + e;
    }
    __syncthreads();
    idx = L.id;
  }
  R.key_cut = hi;
  R.idx_cut = idx;
}

__global__ __launch_bounds__(ST) void k_sample(SampleArgs A) {
  __shared__ Lds L;
  const int row = blockIdx.x, t = threadIdx.x, wv = t >> 6;
  const int chunks = (A.vocab + 255) / 256, per = (chunks + SW - 1) / SW;
  const Span S{A.logits + (size_t)row * A.vocab, A.vocab, min(wv * per, chunks), min((wv + 1) * per, chunks)};
  // the first token of the order
  float zv = -INFINITY;
  int zi = 0x7fffffff;
  S.each([&](float z, int i) {
    if (z > zv) zv = z, zi = i;
  });
  wave_argmax(zv, zi);
  if ((t & 63) == 0) L.wv[wv] = zv, L.wi[wv] = zi;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < SW; ++w)
    if (amax_better(L.wv[w], L.wi[w], zv, zi)) zv = L.wv[w], zi = L.wi[w];
  const float temp = A.temperature ? A.temperature[row] : 1.f;
  if (zv == -INFINITY || !(temp > 0.f)) {  // nothing above -inf; greedy
    if (t == 0) {
      A.ids[row] = zv == -INFINITY ? 0 : zi;
      if (A.probs) A.probs[row] = zv == -INFINITY ? 0.f : 1.f;
    }
    return;
  }
  Row R;
  R.zmax = zv;
  R.first = zi;
  R.c = 1.4426950408889634074 / (double)temp;
  R.dlim = fminf((float)((double)WBITS / R.c), 3.402823466e38f);
  if (R.dlim < 1e-35f) R.dlim = 0.f;  // a temperature below 2e-37: the tokens that tie at the maximum
  R.key_cut = 0u;
  R.idx_cut = 0x7fffffff;
  const int k = A.top_k ? A.top_k[row] : 0;
  if (k > 0 && k < A.vocab) cut<false>(L, S, R, (u64)k);
  const float p = A.top_p ? A.top_p[row] : 1.f;
  if (p < 1.f) {
    u64 sum = 0;
    S.each([&](float z, int i) {
      if (in_cut(R, z, i)) sum += weight(R, z);
    });
    sum = wave_incl(sum);
    __syncthreads();
    if ((t & 63) == 63) L.wave[wv] = sum;
    __syncthreads();
    u64 total = 0;
#pragma unroll
    for (int w = 0; w < SW; ++w) total += L.wave[w];
    const double x = (double)fmaxf(p, 0.f) * (double)total;
    u64 target = (u64)ceil(x);
    if (target < 1) target = 1;
    cut<true>(L, S, R, target);
  }
  const float mp = A.min_p ? A.min_p[row] : 0.f;
  R.wmin = mp > 0.f ? (u64)ceil(fmin((double)mp, 2.0) * (double)(1ull << WBITS)) : 0;
  auto kept = [&](float z, int i) -> u64 {
    if (!in_cut(R, z, i)) return 0;
    const u64 w = weight(R, z);
    return w >= R.wmin || i == R.first ? w : 0;
  };
  clear_bins(L);
  for (int c = S.c0; c < S.c1; ++c) {
    const float4 v = S.load(c);
    const int i = 256 * c + 4 * (int)(t & 63);
    const u64 w = kept(v.x, i) + kept(v.y, i + 1) + kept(v.z, i + 2) + kept(v.w, i + 3);
    const u64 s = wave_incl(w);
    if ((t & 63) == 63) L.bin[c] = s;
  }
  // the total, then the chunk in which the running sum passes u of it
  u64 total = scan_find(L, 1);
  const float u = A.u[row];
  u64 target = u > 0.f ? (u64)((double)u * (double)total) : 0;
  if (target > total - 1) target = total - 1;
  scan_find(L, target + 1);
  const int c = L.at;
  if (c >= S.c0 && c < S.c1) {
    const float4 v = S.load(c);
    const int i = 256 * c + 4 * (int)(t & 63);
    const u64 w[4] = {kept(v.x, i), kept(v.y, i + 1), kept(v.z, i + 2), kept(v.w, i + 3)};
    const u64 sum = w[0] + w[1] + w[2] + w[3];
    u64 run = L.before + wave_incl(sum) - sum;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (run <= target && target < run + w[e]) {
        A.ids[row] = i + e;
        if (A.probs) A.probs[row] = (float)((double)w[e] / (double)total);
      }
      run += w[e];
    }
  }
}

}  // namespace

extern "C" int mllm_sample(int rows, int vocab, const float *logits, const float *temperature, const int32_t *top_k,
                           const float *top_p, const float *min_p, const float *u, int32_t *ids, float *probs,
                           void *stream) {
  MLLM_CHECK(rows > 0 && vocab > 0, "invalid shape rows=%d vocab=%d", rows, vocab);
  if (vocab > kMaxVocab) return set_error(MLLM_ERR_UNSUPPORTED, "vocab=%d exceeds %d", vocab, kMaxVocab);
  MLLM_CHECK(logits && u && ids, "null pointer");
  const SampleArgs A{logits, temperature, top_p, min_p, u, top_k, ids, probs, vocab};
  hipLaunchKernelGGL(k_sample, dim3((unsigned)rows), dim3(ST), 0, reinterpret_cast<hipStream_t>(stream), A);
  MLLM_HIP(hipGetLastError());
  return 0;
}
