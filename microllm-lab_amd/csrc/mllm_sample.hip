// mllm_sample.hip -- drawing tokens from logits (include/mllm.h mllm_sample).
// All pointers are device pointers.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mllm_device.h"
#include "mllm_host.h"

using namespace mllm;

namespace {

// One workgroup per row.  With d = max - z, a token's weight is
//   W = round(2^44 2^(-d log2(e) / T)),  0 past 2^-44 of the largest,
// an integer, so that every sum is exact and the same in any order: the
// weights of up to 2^19 tokens fit 64 bits, and 2^-45 of the largest is a
// thousandth of what float64 sums of float64 weights would need to name
// another token once in a million rows.
//
// The order of the tokens is: larger logit first, equal ones by index.  top-k
// and top-p both keep a prefix of it -- the shortest whose count reaches k, or
// whose weight reaches top_p of the total -- and so does min-p.  No sort:
//   1 the maximum, of the row, of each thread and of each 1024 tokens;
//   2 a bound on the logits that can be left: the k-th of the threads' maxima
//     for top-k, the least weight for min-p; for top-p alone the weights of all
//     tokens are summed into 2048 bins of equal width in d (LDS atomics on
//     64-bit integers), and the bin in which the sum passes its target bounds
//     them;
//   3 the tokens within the bound are listed in LDS, from the 1024s whose
//     maximum is;
//   4 128 tokens or fewer are ranked each against each, and drawn from; a longer
//     list goes through histograms as in 2, whose last bin is ranked so (a bin of
//     more than 128 tokens is split by the bits of its logits, at most three
//     times, and then by index);
//   5 the kept weights are summed by chunks in index order, and the first token
//     whose running sum is more than u of the total is drawn.
//
// What bounds it: a row's own chain, since a row has one CU.  Of 49152 logits,
// us: the maxima 4.5 (44 GB/s), the histogram of all weights 14.7 (each wave
// issues about 1000 instructions, 6.7 on the four SIMDs, the rest is the
// atomics), the list 5, a draw from a short list 5.  Measured, the mean of four
// sets of inputs: one row with top-k and top-p 16, without a filter 24; 100 rows of
// 131072 with min-p 26.5 (2.0 TB/s), 64 rows of 49152 without a filter 26, 200 rows
// of 49152 with top-p alone 56, 64 rows of 50257 with every setting 50 -- there the
// rows whose top-p leaves more tokens than the list holds set the time: they weigh
// all tokens twice.  Tried without gain: the row kept in registers between the
// passes (it spills), more waves (there are none).
constexpr int ST = 1024;        // threads
constexpr int SW = ST / 64;     // waves
constexpr int SB = 2048;        // bins of a histogram, and chunks of a row at most
constexpr int SG = 128;         // tokens of a bin that are ranked against each other
constexpr int SL = 16384;       // tokens that fit the list of those that can be left
constexpr int kMaxVocab = SB * 256;
constexpr int WBITS = 44;

typedef unsigned long long u64;

struct SampleArgs {
  const float *logits, *temperature, *top_p, *min_p, *u;
  const int32_t *top_k;
  int32_t *ids;
  float *probs;
  int vocab;
  // every row's, where the array is null
  float temperature1, top_p1, min_p1, u1;
  int32_t top_k1;
};

// Order-preserving bits of a float (-0 and +0 tie, as the numbers do).
__device__ __forceinline__ uint32_t key_of(float z) {
  const uint32_t b = __float_as_uint(z + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

// Values that are the same in every thread, for the scalar registers.
__device__ __forceinline__ float uni(float v) { return readlane_f(v, 0); }
__device__ __forceinline__ int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ u64 uni(u64 v) {
  return (u64)(uint32_t)uni((int)(uint32_t)(v >> 32)) << 32 | (uint32_t)uni((int)(uint32_t)v);
}
__device__ __forceinline__ double uni(double v) { return __longlong_as_double((long long)uni((u64)__double_as_longlong(v))); }

// A row's state, the same in every thread.
struct Row {
  float zmax, slack;  // slack: more than two roundings of max - d
  float s0;           // bins per unit of d
  double dmax, c;     // zmax (the largest float for infinity); log2(e) / T
  float zcut;         // kept: z > zcut, or z == zcut and index <= icut (never NaN or -inf)
  int icut;
  double poly[9];     // weight()'s polynomial, without its constant 1
};

__device__ __forceinline__ bool kept(const Row &R, float z, int i) {
  return z > R.zcut || (z == R.zcut && i <= R.icut);
}
__device__ __forceinline__ int bin_of(const Row &R, float z) { return (int)fminf((R.zmax - z) * R.s0, (float)(SB - 1)); }
// Logits below this cannot be in bins up to b, nor those above hi_of(b) in bin b.
__device__ __forceinline__ float lo_of(const Row &R, int b) {
  return b >= SB - 1 || R.zmax == INFINITY ? -INFINITY : R.zmax - (float)(b + 2) / R.s0 - R.slack;
}
__device__ __forceinline__ float hi_of(const Row &R, int b) {
  return b <= 1 || R.zmax == INFINITY ? R.zmax : R.zmax - (float)(b - 1) / R.s0 + R.slack;
}

// W of a kept token: 2^t by a polynomial in the distance to the nearest
// integer (interpolated at Chebyshev nodes, within 4e-14; 1 at 0), the integer
// into the exponent.  Adding 1.5 2^52 + 44 rounds t and leaves its integer + 44
// in the low word; adding 2^52 leaves the weight's.  (Conversions of doubles to
// integers, roundings and ldexp take four times an addition.)
// The coefficients come from scalar registers: from vector registers the
// compiler copies each before the multiply-add that overwrites the copy.
__device__ __forceinline__ void set_poly(Row &R) {
  constexpr double c[9] = {1.0203121063391729e-07, 1.3255224878668817e-06, 1.525268684626772e-05,
                           1.5403455852453838e-04, 1.3333558179043112e-03, 9.618129159402558e-03,
                           5.5504108664760424e-02, 2.402265069581299e-01,  6.931471805599453e-01};
#pragma unroll
  for (int k = 0; k < 9; ++k) {
    R.poly[k] = c[k];
    asm("" : "+s"(R.poly[k]));
  }
}
__device__ __forceinline__ u64 weight(const Row &R, float z) {
  constexpr double ROUND = 6755399441055744.0 + WBITS;
  const double t = ((double)fminf(z, 3.402823466e38f) - R.dmax) * R.c, m = t + ROUND, f = t - (m - ROUND);
  double p = R.poly[0];
#pragma unroll
  for (int k = 1; k < 9; ++k) p = __builtin_fma(p, f, R.poly[k]);
  p = __builtin_fma(p, f, 1.0);
  const double w = __hiloint2double(__double2hiint(p) + (__double2loint(m) << 20), __double2loint(p)) + 4503599627370496.0;
  return (u64)(uint32_t)(__double2hiint(w) & 0xfffff) << 32 | (uint32_t)__double2loint(w);
}

template <int CTRL>
__device__ __forceinline__ u64 dpp64(u64 v) {
  const uint32_t lo = (uint32_t)dpp_i<CTRL>((int)(uint32_t)v), hi = (uint32_t)dpp_i<CTRL>((int)(uint32_t)(v >> 32));
  return (u64)hi << 32 | lo;
}
__device__ __forceinline__ u64 lane64(u64 v, int lane) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane),
                 hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane);
  return (u64)hi << 32 | lo;
}
__device__ __forceinline__ u64 sum8_64(u64 v) {  // over the 8 lanes of each half-row
  v += dpp64<0xB1>(v);
  v += dpp64<0x4E>(v);
  return v + dpp64<0x141>(v);
}
__device__ __forceinline__ u64 sum16_64(u64 v) {  // over each row of 16
  v = sum8_64(v);
  return v + dpp64<0x140>(v);
}
__device__ __forceinline__ u64 wave_sum64(u64 v) {
  v = sum16_64(v);
  return (lane64(v, 0) + lane64(v, 16)) + (lane64(v, 32) + lane64(v, 48));
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
  float top[SB / 4];  // the maxima of the waves' groups of four chunks
  u64 wave[SW];
  // the bin that scan_find has found: its number, the sum before it, its own sum
  int at;
  u64 before, own;
  // the tokens that can be left: logits' bits and indices
  uint2 list[SL];
  int ln;
  // the tokens of a bin
  u64 gw[SG];
  float gz[SG];
  int gi[SG];
  int n;
  float zcut;
  int icut;
  float wv[SW];
  int id;
};

// The first bin at which the running sum reaches target(total) (>= 1), in L.at
// / before / own, and the target itself; L.at = -1 where the total does not
// reach it.  Ends in a barrier.
template <class F>
__device__ __forceinline__ u64 scan_find(Lds &L, F target_of, u64 &total) {
  const int t = threadIdx.x, wv = t >> 6;
  __syncthreads();
  constexpr int BT = SB / ST;  // bins of a thread
  u64 e[BT + 1];
  e[0] = 0;
#pragma unroll
  for (int k = 0; k < BT; ++k) e[k + 1] = e[k] + L.bin[BT * t + k];
  const u64 incl = wave_incl(e[BT]);
  if ((t & 63) == 63) L.wave[wv] = incl;
  if (t == 0) L.at = -1;
  __syncthreads();
  static_assert(SW == 16, "the waves' sums in a row of lanes");
  const u64 v = L.wave[t & 15];
  total = uni(sum16_64(v));
  const u64 target = uni(target_of(total)), off = uni(sum16_64((t & 15) < wv ? v : 0ull)) + incl - e[BT];
  if (off < target && target <= off + e[BT]) {
#pragma unroll
    for (int k = 0; k < BT; ++k)
      if (off + e[k] < target && target <= off + e[k + 1]) {
        L.at = BT * t + k;
        L.before = off + e[k];
        L.own = e[k + 1] - e[k];
      }
  }
  __syncthreads();
  return target;
}

__device__ __forceinline__ void clear_bins(Lds &L) {
  __syncthreads();
#pragma unroll
  for (int k = 0; k < SB / ST; ++k) L.bin[threadIdx.x + k * ST] = 0;
  if (threadIdx.x == 0) L.n = 0;
  __syncthreads();
}

// Where the passes take the tokens from.  A row in memory, chunk by chunk: lane
// l of chunk c holds the tokens 256 c + 4 l .. + 3, a wave takes a run of
// neighbouring chunks.
struct Tokens {
  const float *x;
  int vocab, c0, c1;
  int g0;  // its first group in Lds::top
  __device__ __forceinline__ float4 load(int c) const {
    const int i = 256 * c + 4 * (int)(threadIdx.x & 63);
    if (256 * (c + 1) <= vocab) return ld4u(x + i);
    float e[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) e[k] = i + k < vocab ? x[i + k] : -INFINITY;
    return make_float4(e[0], e[1], e[2], e[3]);
  }
  // f(c, index, values) for each chunk, the next N in flight
  template <int N = 4, class F>
  __device__ __forceinline__ void chunks(F f) const {
    if (c0 >= c1) return;
    float4 w[N], next[N];
#pragma unroll
    for (int j = 0; j < N; ++j) next[j] = load(min(c0 + j, c1 - 1));
    for (int c = c0; c < c1; c += N) {
#pragma unroll
      for (int j = 0; j < N; ++j) w[j] = next[j];
      if (c + N < c1)
#pragma unroll
        for (int j = 0; j < N; ++j) next[j] = load(min(c + N + j, c1 - 1));
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (c + j < c1) f(c + j, 256 * (c + j) + 4 * (int)(threadIdx.x & 63), w[j]);
    }
  }
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    chunks([&](int, int i, const float4 &w) { f(w.x, i), f(w.y, i + 1), f(w.z, i + 2), f(w.w, i + 3); });
  }
  // L.bin[c]: the sum of f over chunk c
  template <class F>
  __device__ __forceinline__ void by_chunk(Lds &L, F f) const {
    chunks([&](int c, int i, const float4 &w) {
      const u64 s = (f(w.x, i) + f(w.y, i + 1)) + (f(w.z, i + 2) + f(w.w, i + 3));
      if (!__any(s != 0)) return;
      const u64 sum = wave_sum64(s);
      if ((threadIdx.x & 63) == 0) L.bin[c] = sum;
    });
  }
};
// The list in LDS, in no order: a thread takes K neighbours (K odd, for the LDS
// banks), so that the lanes of a wave stand in different chunks of the row.
struct List {
  const Lds *L;
  int n;
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    const int K = ((n + ST - 1) / ST) | 1, m1 = min(n, ((int)threadIdx.x + 1) * K);
    for (int m = threadIdx.x * K; m < m1; ++m) {
      const uint2 e = L->list[m];
      f(__uint_as_float(e.x), (int)e.y);
    }
  }
  template <class F>
  __device__ __forceinline__ void by_chunk(Lds &L, F f) const {
    each([&](float z, int i) {
      const u64 w = f(z, i);
      if (w) atomicAdd(&L.bin[i >> 8], w);
    });
  }
};

// The bin in which a running sum reaches its target.
struct Found {
  int bin;        // -1: it does not reach it
  u64 rest, own;  // of the target, past what stands before the bin; the bin's sum
};

// The cut at the first token (in order) of bin b0 at which the running sum
// reaches target, the bin holding more tokens than can be ranked: by the bits
// of the logit, then by index.  before: the sum in front of the bin.
template <bool MASS, class S>
__device__ __forceinline__ void cut_wide(Lds &L, const S &src, const Tokens &row, Row &R, const Found &F) {
  const int b0 = F.bin;
  u64 rest = F.rest, own = F.own;
  uint32_t hi = 0xffffffffu, lo = 0u;
  auto member = [&](float z, int i, uint32_t k) { return kept(R, z, i) && k <= hi && k >= lo && bin_of(R, z) == b0; };
  for (;;) {
    // the range of the keys that are left; one where they tie
    uint32_t h = 0u, l = 0xffffffffu;
    src.each([&](float z, int i) {
      const uint32_t k = key_of(z);
      if (member(z, i, k)) h = max(h, k), l = min(l, k);
    });
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
      h = max(h, (uint32_t)__shfl_xor((int)h, s));
      l = min(l, (uint32_t)__shfl_xor((int)l, s));
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) L.wave[threadIdx.x >> 6] = (u64)h << 32 | l;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SW; ++w) h = max(h, (uint32_t)(L.wave[w] >> 32)), l = min(l, (uint32_t)L.wave[w]);
    hi = (uint32_t)uni((int)h), lo = (uint32_t)uni((int)l);
    if (hi == lo) break;
    const int sh = max(0, 32 - __clz((int)(hi - lo)) - 11);
    clear_bins(L);
    src.each([&](float z, int i) {
      const uint32_t k = key_of(z);
      if (member(z, i, k)) atomicAdd(&L.bin[(hi - k) >> sh], MASS ? weight(R, z) : 1ull);
    });
    u64 total;
    scan_find(L, [&](u64) { return rest; }, total);
    rest -= uni(L.before);
    own = uni(L.own);
    hi -= (uint32_t)uni(L.at) << sh;
    lo = hi - lo < (1u << sh) ? lo : hi - ((1u << sh) - 1u);
  }
  // the first `need` of the tokens that tie at this logit, by index
  const float zc = of_key(hi);
  const u64 unit = MASS ? weight(R, zc) : 1ull, need = (rest + unit - 1) / unit;
  int idx = R.zcut == zc ? R.icut : 0x7fffffff;
  if (need * unit < own) {
    // their number in each chunk
    clear_bins(L);
    src.by_chunk(L, [&](float z, int i) -> u64 { return z == zc && kept(R, z, i); });
    u64 total;
    scan_find(L, [&](u64) { return need; }, total);
    const int c = uni(L.at);
    if (c >= row.c0 && c < row.c1) {
      const float4 w = row.load(c);
      const float z[4] = {w.x, w.y, w.z, w.w};
      const int i = 256 * c + 4 * (int)(threadIdx.x & 63);
      u64 n = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) n += z[e] == zc && kept(R, z[e], i + e);
      u64 k = L.before + wave_incl(n) - n;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (z[e] == zc && kept(R, z[e], i + e) && ++k == need) L.id = i + e;
    }
    __syncthreads();
    idx = L.id;
  }
  R.zcut = uni(zc);
  R.icut = uni(idx);
}

// The bin in which the running sum of the order -- the count of the tokens in
// the present cut, or their weight -- reaches target_of(total).  Logits below
// zq need not be counted.
template <bool MASS, class S, class F>
__device__ __forceinline__ Found find_bin(Lds &L, const S &src, const Row &R, float zq, F target_of) {
  clear_bins(L);
  src.each([&](float z, int i) {
    if (!(z < zq) && kept(R, z, i)) atomicAdd(&L.bin[bin_of(R, z)], MASS ? weight(R, z) : 1ull);
  });
  u64 total;
  const u64 target = scan_find(L, target_of, total);
  return Found{uni(L.at), target - uni(L.before), uni(L.own)};
}

// Shortens the cut to the token of that bin at which the sum reaches its
// target.
template <bool MASS, class S>
__device__ __forceinline__ void settle(Lds &L, const S &src, const Tokens &row, Row &R, const Found &F) {
  if (F.bin < 0) return;
  const int b0 = F.bin;
  // the bin's tokens (L.n is 0)
  const float zl = uni(lo_of(R, b0)), zh = uni(hi_of(R, b0));
  src.each([&](float z, int i) {
    if (!(z < zl) && !(z > zh) && kept(R, z, i) && bin_of(R, z) == b0) {
      const int k = atomicAdd(&L.n, 1);
      if (k < SG) L.gz[k] = z, L.gi[k] = i, L.gw[k] = MASS ? weight(R, z) : 1ull;
    }
  });
  __syncthreads();
  const int n = uni(L.n);
  if (n > SG) return cut_wide<MASS>(L, src, row, R, F);
  // eight lanes to a token sum what stands before it
  static_assert(ST == 8 * SG, "eight lanes to a token");
  const int m = min((int)threadIdx.x >> 3, n - 1);
  const float zm = L.gz[m];
  const int im = L.gi[m];
  u64 sum = 0;
  for (int k = threadIdx.x & 7; k < n; k += 8) {
    const float zk = L.gz[k];
    if (zk > zm || (zk == zm && L.gi[k] < im)) sum += L.gw[k];
  }
  sum = sum8_64(sum);
  if (sum < F.rest && F.rest <= sum + L.gw[m]) L.zcut = zm, L.icut = im;  // the same values from each of its lanes
  __syncthreads();
  R.zcut = uni(L.zcut);
  R.icut = uni(L.icut);
}

// What a row's settings leave, and the draw, from the tokens of src (those of
// the row that can be left, at least).
struct Settings {
  int k;
  float p, zq, zp;  // zq: the top k are at least this; zp: min-p leaves nothing below this
  u64 wmin;         // min-p: the least weight left
  float u;
  int32_t *id;
  float *prob;
};
__device__ __forceinline__ u64 top_p_target(float p, u64 total) {
  const u64 target = (u64)ceil((double)fmaxf(p, 0.f) * (double)total);
  return target < 1 ? 1ull : target;
}
// The running sum to reach, of the weights that are left.
__device__ __forceinline__ u64 draw_target(float u, u64 total) {
  const u64 x = u > 0.f ? (u64)((double)fminf(u, 1.f) * (double)total) : 0;
  return (x > total - 1 ? total - 1 : x) + 1;
}
__device__ __forceinline__ void put(const Settings &A, int i, u64 w, u64 total) {
  *A.id = i;
  if (A.prob) *A.prob = (float)((double)w / (double)total);
}

// The sum over the workgroup of a value that the first of every eight lanes has.
__device__ __forceinline__ u64 sum_of_eighths(Lds &L, u64 v) {
  v = wave_sum64((threadIdx.x & 7) == 0 ? v : 0ull);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) L.wave[threadIdx.x >> 6] = v;
  __syncthreads();
  return uni(sum16_64(L.wave[threadIdx.x & 15]));
}

// n <= SG tokens in the list, eight lanes to each: what stands before a token in
// the order decides whether it is left, what stands before it by index whether
// it is drawn.
__device__ __forceinline__ void draw_few(Lds &L, int n, const Row &R, const Settings &A) {
  const int m = min((int)threadIdx.x >> 3, n - 1), part = threadIdx.x & 7;
  const bool own = (int)threadIdx.x >> 3 < n;
  const float z = __uint_as_float(L.list[m].x);
  const int i = (int)L.list[m].y;
  u64 w = weight(R, z);
  if (own && part == 0) L.gw[m] = w;
  __syncthreads();
  u64 before = 0, rank = 0;
  for (int j = part; j < n; j += 8) {
    const uint2 e = L.list[j];
    const float zj = __uint_as_float(e.x);
    if (zj > z || (zj == z && (int)e.y < i)) before += L.gw[j], ++rank;
  }
  before = sum8_64(before);
  rank = sum8_64(rank);
  bool in = own && (A.k == 0 || rank < (u64)A.k);
  if (A.p < 1.f) {
    const u64 target = top_p_target(A.p, sum_of_eighths(L, in ? w : 0ull));
    in = in && before < target;
  }
  w = in && w >= A.wmin ? w : 0;
  const u64 total = sum_of_eighths(L, w);
  if (own && part == 0) L.gw[m] = w;
  __syncthreads();
  u64 run = 0;
  for (int j = part; j < n; j += 8)
    if ((int)L.list[j].y < i) run += L.gw[j];
  run = sum8_64(run);
  const u64 target = draw_target(A.u, total);
  if (own && part == 0 && run < target && target <= run + w) put(A, i, w, total);
}

// The cuts of top-k and top-p, and their tokens' sums, from src.  F: top-p's
// bin, where there is no top-k; border: a source of that bin's tokens.
template <class S, class B>
__device__ __forceinline__ void draw(Lds &L, const S &src, const B &border, const Tokens &row, Row &R, const Settings &A,
                                     Found F) {
  if (A.k) {
    settle<false>(L, src, row, R, find_bin<false>(L, src, R, A.zq, [&](u64) { return (u64)A.k; }));
    if (A.p < 1.f)
      settle<true>(L, src, row, R, find_bin<true>(L, src, R, -INFINITY, [&](u64 total) { return top_p_target(A.p, total); }));
  } else if (A.p < 1.f) {
    settle<true>(L, border, row, R, F);
  }
  auto left = [&](float z, int i) -> u64 {
    if (z < A.zp || !kept(R, z, i)) return 0;
    const u64 w = weight(R, z);
    return w >= A.wmin ? w : 0;
  };
  clear_bins(L);
  src.by_chunk(L, left);
  // the chunk in which the running sum passes u of the total
  u64 total;
  const u64 target = scan_find(L, [&](u64 all) { return draw_target(A.u, all); }, total);
  const int c = uni(L.at);
  if (c < row.c0 || c >= row.c1) return;
  const float4 v = row.load(c);
  const int i = 256 * c + 4 * (int)(threadIdx.x & 63);
  const u64 w[4] = {left(v.x, i), left(v.y, i + 1), left(v.z, i + 2), left(v.w, i + 3)};
  const u64 sum = (w[0] + w[1]) + (w[2] + w[3]);
  u64 run = L.before + wave_incl(sum) - sum;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (run < target && target <= run + w[e]) put(A, i + e, w[e], total);
    run += w[e];
  }
}

// The row's tokens from zl on (BOUNDED: up to zh) into the list, in no order,
// from the groups of chunks whose maximum is at least zl.  L.ln: their number, or
// any above SL where the list has no room for them.
template <bool BOUNDED>
__device__ __forceinline__ void list_tokens(Lds &L, const Tokens &row, float zl, float zh) {
  const int lane = threadIdx.x & 63, groups = (row.c1 - row.c0 + 3) / 4;  // at most 32
  __syncthreads();
  if (threadIdx.x == 0) L.ln = 0;
  __syncthreads();
  u64 todo = __ballot(lane < groups && L.top[min(row.g0 + lane, SB / 4 - 1)] >= zl);
  float4 next[4];
  auto fetch = [&](u64 which) {
    const int c = row.c0 + 4 * (which ? __builtin_ctzll(which) : 0);
#pragma unroll
    for (int j = 0; j < 4; ++j) next[j] = row.load(min(c + j, row.c1 - 1));
  };
  if (todo) fetch(todo);
  while (todo) {
    const int c0 = row.c0 + 4 * __builtin_ctzll(todo);
    float4 w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = next[j];
    todo &= todo - 1;
    if (todo) fetch(todo);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (c0 + j >= row.c1) break;
      const float z[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
      auto listed = [&](int e) { return z[e] >= zl && (!BOUNDED || z[e] <= zh); };
      u64 hit[4];  // the lanes whose token is listed
#pragma unroll
      for (int e = 0; e < 4; ++e) hit[e] = __ballot(listed(e));
      if ((hit[0] | hit[1] | hit[2] | hit[3]) == 0) continue;
      const int n = __popcll(hit[0]) + __popcll(hit[1]) + __popcll(hit[2]) + __popcll(hit[3]);
      int m = 0;  // places in the list, taken at once
      if (lane == 0) m = atomicAdd(&L.ln, n);
      m = uni(m);
      if (m + n > SL) return;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (listed(e)) {
          const int at = __builtin_amdgcn_mbcnt_hi((uint32_t)(hit[e] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)hit[e], m));
          L.list[at] = make_uint2(__float_as_uint(z[e]), (uint32_t)(256 * (c0 + j) + 4 * lane + e));
        }
        m += __popcll(hit[e]);
      }
    }
  }
}

__global__ __launch_bounds__(ST) void k_sample(SampleArgs A) {
  __shared__ Lds L;
  const int r = blockIdx.x, t = threadIdx.x, wv = uni(t >> 6);
  const int chunks = (A.vocab + 255) / 256, per = (chunks + SW - 1) / SW;
  const Tokens row{A.logits + (size_t)r * A.vocab, A.vocab, min(wv * per, chunks), min((wv + 1) * per, chunks),
                   wv * ((per + 3) / 4)};
  float zt = -INFINITY, zg = -INFINITY;  // this thread's maximum, and its group's
  row.chunks<8>([&](int c, int, const float4 &w) {
    zg = fmaxf(fmaxf(fmaxf(w.x, w.y), fmaxf(w.z, w.w)), zg);
    if (((c - row.c0) & 3) == 3 || c == row.c1 - 1) {
      const float z = wave_max(zg);
      if ((t & 63) == 0) L.top[row.g0 + (c - row.c0) / 4] = z;
      zt = fmaxf(zg, zt);
      zg = -INFINITY;
    }
  });
  float zv = wave_max(zt);
  if ((t & 63) == 0) L.wv[wv] = zv;
  if (t == 0) L.id = 0x7fffffff;
  __syncthreads();
  zv = uni(row16_max(L.wv[t & 15]));
  const float temp = A.temperature ? A.temperature[r] : A.temperature1, mp = A.min_p ? A.min_p[r] : A.min_p1;
  if (zv == -INFINITY || !(temp > 0.f) || mp > 1.f) {  // nothing above -inf; greedy; the first token alone is left
    for (int c = row.c0; c < row.c1 && zv != -INFINITY; c += 4)
      if (L.top[row.g0 + (c - row.c0) / 4] == zv) {  // the wave's first group that has it
        for (int j = 0; j < 4; ++j) {
          const float4 w = row.load(min(c + j, row.c1 - 1));
          const int i = 256 * min(c + j, row.c1 - 1) + 4 * (t & 63);
          const int at = w.x == zv ? i : w.y == zv ? i + 1 : w.z == zv ? i + 2 : w.w == zv ? i + 3 : 0x7fffffff;
          if (at != 0x7fffffff) atomicMin(&L.id, at);
        }
        break;
      }
    __syncthreads();
    if (t == 0) {
      A.ids[r] = zv == -INFINITY ? 0 : L.id;
      if (A.probs) A.probs[r] = zv == -INFINITY ? 0.f : 1.f;
    }
    return;
  }
  Row R;
  set_poly(R);
  R.zmax = zv;
  R.dmax = (double)fminf(zv, 3.402823466e38f);
  R.c = uni(1.4426950408889634074 / (double)temp);
  R.slack = uni(fabsf(zv) * 2.4e-7f);
  const double far = (double)WBITS / R.c;
  float dlim = fminf((float)far, 3.402823466e38f);
  if (dlim < 1e-35f) dlim = 0.f;  // a temperature below 2e-37: the tokens that tie at the maximum
  R.s0 = uni(dlim > 0.f ? (float)SB / dlim : 0.f);
  // from a temperature of 1.1e37 on, logits further apart than the largest float have weight
  const float zfar = dlim < 3.402823466e38f || zv == INFINITY ? zv - dlim : (float)fmax((double)zv - far, -3.402823466e38);
  R.zcut = uni(fmaxf(zfar, -3.402823466e38f));
  R.icut = 0x7fffffff;
  Settings s;
  s.id = A.ids + r, s.prob = A.probs ? A.probs + r : nullptr;
  s.u = A.u ? A.u[r] : A.u1;
  s.k = A.top_k ? A.top_k[r] : A.top_k1;
  if (s.k < 0 || s.k >= A.vocab) s.k = 0;
  s.p = A.top_p ? A.top_p[r] : A.top_p1;
  s.wmin = mp > 0.f ? (u64)ceil((double)mp * (double)(1ull << WBITS)) : 0;
  s.zq = s.zp = -INFINITY;
  if (mp > 0.f && zv != INFINITY) s.zp = uni(zv + logf(mp) * temp * 1.00001f - 1e-5f * temp - R.slack);
  if (s.k && s.k <= ST) {
    // k of the threads' maxima lie in the bins up to the k-th one's: so do the
    // top k
    clear_bins(L);
    if (zt >= R.zcut) atomicAdd(&L.bin[bin_of(R, zt)], 1ull);
    u64 total;
    scan_find(L, [&](u64) { return (u64)s.k; }, total);
    if (L.at >= 0) s.zq = uni(lo_of(R, L.at));
  }
  // the tokens that can be left: top-p's total takes all of the top k
  Found F{-1, 0, 0};
  float zl = s.p < 1.f ? s.zq : fmaxf(s.zq, s.zp);
  const bool p_alone = !s.k && s.p < 1.f;
  if (p_alone) {
    F = find_bin<true>(L, row, R, -INFINITY, [&](u64 total) { return top_p_target(s.p, total); });
    zl = uni(lo_of(R, F.bin));
  }
  if (zl > -INFINITY) {
    zl = uni(fmaxf(zl, R.zcut));
    list_tokens<false>(L, row, zl, INFINITY);
    __syncthreads();
    int n = uni(L.ln);
    if (n <= SL) {
      if (!p_alone && n <= SG) return draw_few(L, n, R, s);
      const List list{&L, n};
      return draw(L, list, list, row, R, s, F);
    }
    if (p_alone) {  // too many: those of top-p's bin alone
      list_tokens<true>(L, row, zl, uni(hi_of(R, F.bin)));
      __syncthreads();
      n = uni(L.ln);
      if (n <= SL) return draw(L, row, List{&L, n}, row, R, s, F);
    }
  }
  draw(L, row, row, row, R, s, F);
}

int launch(int rows, const SampleArgs &A, hipStream_t st) {
  MLLM_CHECK(rows > 0 && A.vocab > 0, "invalid shape rows=%d vocab=%d", rows, A.vocab);
  if (A.vocab > kMaxVocab) return set_error(MLLM_ERR_UNSUPPORTED, "vocab=%d exceeds %d", A.vocab, kMaxVocab);
  MLLM_CHECK((int64_t)rows * ST < (1ll << 32), "%d rows exceed a launch", rows);
  hipLaunchKernelGGL(k_sample, dim3((unsigned)rows), dim3(ST), 0, st, A);
  MLLM_HIP(hipGetLastError());
  return 0;
}

}  // namespace

int mllm::sample_row(int vocab, const float *logits, float temperature, int32_t top_k, float top_p, float min_p, float u,
                     int32_t *id, float *prob, hipStream_t st) {
  const SampleArgs A{logits, nullptr, nullptr, nullptr, nullptr,     nullptr, id,
                     prob,   vocab,   temperature, top_p, min_p, u, top_k};
  return launch(1, A, st);
}

extern "C" int mllm_sample(int rows, int vocab, const float *logits, const float *temperature, const int32_t *top_k,
                           const float *top_p, const float *min_p, const float *u, int32_t *ids, float *probs,
                           void *stream) {
  MLLM_CHECK(logits && u && ids, "null pointer");
  const SampleArgs A{logits, temperature, top_p, min_p, u, top_k, ids, probs, vocab, 1.f, 1.f, 0.f, 0.f, 0};
  return launch(rows, A, reinterpret_cast<hipStream_t>(stream));
}
