// mllm_paged.hip -- the operators of a batched decode step that touch the
// pages of a key-value cache (include/mllm.h): mllm_rope_kv_paged writes new
// tokens' keys and values, mllm_attn_paged attends to them.  All pointers are
// device pointers.
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "mllm_device.h"
#include "mllm_host.h"

using namespace mllm;

namespace {

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

// ---------------------------------------------------------------- rotation into the pages
struct RopeArgs {
  Pages P;
  const float *qkv, *inv_freq, *q_gain, *k_gain;
  const int32_t *seq, *pos;
  float *q;
  int n_heads, rot, lph, lg_lph, per_wg, n_wg;  // lanes per head (a power of two), heads per workgroup, workgroups per token
  int interleaved;
  float eps;
};

// A token's heads, lph lanes to each: lane s holds the four pairs 4s .. 4s + 3.
// Pair p is rotated below rot / 2 -- elements (p, p + rot/2), or (2p, 2p + 1)
// interleaved -- and passes through above, as elements (2p, 2p + 1).  VEC: rot
// is a multiple of 8, so a lane's pairs are two runs of four floats.
//
// The angle is formed in double and in turns: a position of 2^20 keeps 2^-33
// of a turn, where a float product would keep 2^-4.
template <class KV, bool VEC>
__global__ __launch_bounds__(WG) void k_rope_kv(RopeArgs A) {
  const int token = blockIdx.x / A.n_wg, part = blockIdx.x - token * A.n_wg;
  const int s = threadIdx.x & (A.lph - 1), head = part * A.per_wg + (threadIdx.x >> A.lg_lph);
  const int nh = A.n_heads, nkv = A.P.n_kv, hd = A.P.hd, rows = nh + 2 * nkv;
  if ((int)(threadIdx.x >> A.lg_lph) >= A.per_wg || head >= rows) return;  // whole heads
  const int seq = A.seq ? A.seq[token] : token, pos = A.pos[token];
  if (seq < 0 || seq >= A.P.sequences || pos < 0) return;  // padding
  const bool in = 8 * s < hd, turned = head < nh + nkv && 8 * s < A.rot;
  const float *x = A.qkv + ((size_t)token * rows + head) * hd;
  // element e of the lane's pair j
  auto at = [&](int j, int e) {
    const int p = 4 * s + j;
    const bool r = head < nh + nkv && 2 * p < A.rot;
    return r && !A.interleaved ? p + e * (A.rot >> 1) : 2 * p + e;
  };
  const bool halves = turned && !A.interleaved;
  const int o0 = halves ? 4 * s : 8 * s, o1 = halves ? 4 * s + (A.rot >> 1) : 8 * s + 4;
  float a[4], b[4];  // the pairs' elements
  if (!in) {
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] = b[j] = 0.f;
  } else if (VEC) {
    const float4 u = *reinterpret_cast<const float4 *>(x + o0), w = *reinterpret_cast<const float4 *>(x + o1);
    if (halves) {
      a[0] = u.x, a[1] = u.y, a[2] = u.z, a[3] = u.w, b[0] = w.x, b[1] = w.y, b[2] = w.z, b[3] = w.w;
    } else {
      a[0] = u.x, b[0] = u.y, a[1] = u.z, b[1] = u.w, a[2] = w.x, b[2] = w.y, a[3] = w.z, b[3] = w.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] = x[at(j, 0)], b[j] = x[at(j, 1)];
  }
  const float *gain = head < nh ? A.q_gain : head < nh + nkv ? A.k_gain : nullptr;
  if (gain) {
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) ss = __builtin_fmaf(a[j], a[j], __builtin_fmaf(b[j], b[j], ss));
    for (int m = 1; m < A.lph; m <<= 1) ss += __shfl_xor(ss, m);
    const float inv = 1.0f / sqrtf(ss / (float)hd + A.eps);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (in) a[j] = a[j] * inv * gain[at(j, 0)], b[j] = b[j] * inv * gain[at(j, 1)];
  }
  if (!in) return;
  if (turned) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int p = 4 * s + j;
      if (2 * p < A.rot) {
        const double t = (double)pos * ((double)A.inv_freq[p] * 0.15915494309189533577);  // turns
        float sn, cs;
        sincospif((float)(2.0 * (t - rint(t))), &sn, &cs);
        const float u = a[j], w = b[j];
        a[j] = u * cs - w * sn;
        b[j] = w * cs + u * sn;
      }
    }
  }
  auto store = [&](auto *to, auto put) {
    using T = decltype(put(0.f));
    if (VEC) {
      typedef T v4 __attribute__((ext_vector_type(4)));
      v4 u, w;
      if (halves) {
        u = v4{put(a[0]), put(a[1]), put(a[2]), put(a[3])};
        w = v4{put(b[0]), put(b[1]), put(b[2]), put(b[3])};
      } else {
        u = v4{put(a[0]), put(b[0]), put(a[1]), put(b[1])};
        w = v4{put(a[2]), put(b[2]), put(a[3]), put(b[3])};
      }
      *reinterpret_cast<v4 *>(to + o0) = u;
      *reinterpret_cast<v4 *>(to + o1) = w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) to[at(j, 0)] = put(a[j]), to[at(j, 1)] = put(b[j]);
    }
  };
  if (head < nh) {
    store(A.q + ((size_t)token * nh + head) * hd, KvF32::put);
    return;
  }
  const int col = page_of(A.P, pos), slot = pos - col * A.P.page_size;
  if (col >= A.P.table_cols) return;
  const int page = A.P.table[(size_t)seq * A.P.table_cols + col];
  if (page < 0 || page >= A.P.pages) return;
  const int kvh = head < nh + nkv ? head - nh : head - nh - nkv;
  typename KV::T *pool = static_cast<typename KV::T *>(head < nh + nkv ? A.P.k : A.P.v);
  store(pool + page * A.P.page_stride + kvh * A.P.head_stride + slot * A.P.row_stride, KV::put);
}

// ---------------------------------------------------------------- attention over pages
constexpr int AW = 4;                  // waves of a workgroup
constexpr int ASUB = 2048;             // positions whose places in the pool are in LDS at a time
constexpr int kUnits = 1024;           // workgroups that fill the chip: four on each of the 256 CUs
constexpr float LOG2E = 1.44269504088896340736f;

struct AttnArgs {
  Pages P;
  const float *q;
  const int32_t *seq, *len;
  float *out, *part;  // part: [units][splits][heads of a unit][hd + 2], the sums, then maximum and sum
  unsigned *count;    // [kUnits] parts that are there, zero between calls
  int n_heads, rep, tiles, heads, max_len, chunk, splits;  // heads: query heads of a workgroup at most
  float scale;
};

// A row's length as the kernels use it: -1 padding (the row is left as it
// was), -2 not possible (NaN).
__device__ __forceinline__ int row_len(const AttnArgs &A, int row, int &seq) {
  seq = A.seq ? A.seq[row] : row;
  if (seq < 0 || seq >= A.P.sequences) return -1;
  const int n = A.len[row];
  return n < 0 || n > A.max_len ? -2 : n;
}

// E elements of the cache at p as floats, loaded in runs of at most 16 bytes.
template <class KV, int E>
struct Raw {
  static constexpr int N = E * (int)sizeof(typename KV::T) / 4;  // dwords
  uint32_t d[N];
  __device__ __forceinline__ void load(const void *p) {
    typedef uint32_t u4 __attribute__((ext_vector_type(4), aligned(4)));
    typedef uint32_t u2 __attribute__((ext_vector_type(2), aligned(4)));
    const uint32_t *s = static_cast<const uint32_t *>(p);
#pragma unroll
    for (int i = 0; i + 4 <= N; i += 4) {
      const u4 v = *reinterpret_cast<const u4 *>(s + i);
      d[i] = v.x, d[i + 1] = v.y, d[i + 2] = v.z, d[i + 3] = v.w;
    }
    if constexpr ((N & 2) != 0) {
      const u2 v = *reinterpret_cast<const u2 *>(s + (N & ~3));
      d[N & ~3] = v.x, d[(N & ~3) + 1] = v.y;
    }
    if constexpr ((N & 1) != 0) d[N - 1] = s[N - 1];
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < N; ++i) d[i] = 0u;
  }
  __device__ __forceinline__ float get(int e) const {
    if constexpr (sizeof(typename KV::T) == 4) return __uint_as_float(d[e]);
    else if constexpr (__is_same(KV, KvBf16)) return __uint_as_float(e & 1 ? d[e >> 1] & 0xffff0000u : d[e >> 1] << 16);
    else return __half2float(__ushort_as_half((uint16_t)(e & 1 ? d[e >> 1] >> 16 : d[e >> 1] & 0xffffu)));
  }
};

// The 16-bit pieces of a float: a sum of NP of them is the float to 24 bits (22
// in f16, where the caller scales it away from the type's ends).
template <class KV>
struct Piece;
template <>
struct Piece<KvF16> {
  static constexpr int NP = 2;
  static __device__ __forceinline__ float val(uint16_t h) { return __half2float(__ushort_as_half(h)); }
};
template <>
struct Piece<KvBf16> {
  static constexpr int NP = 3;
  static __device__ __forceinline__ float val(uint16_t h) { return __uint_as_float((uint32_t)h << 16); }
};
template <>
struct Piece<KvF32> {
  static constexpr int NP = 1;  // no pieces: the products are float32 as they are
  static __device__ __forceinline__ float val(float v) { return v; }
};

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));

template <class KV>
__device__ __forceinline__ v4f mma32(u32x4 a, u32x4 b, v4f c) {
  if constexpr (__is_same(KV, KvBf16))
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, a), __builtin_bit_cast(b16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h16x8, a), __builtin_bit_cast(h16x8, b), c, 0, 0, 0);
}

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
  static constexpr int ROW = HD * ES, PT = ROW <= 128 ? 4 : ROW <= 256 ? 2 : 1, TP = 16 * PT, NU = TP / G;
  static constexpr int AQ = EL <= 8 ? 16 : 8;                       // query heads of a workgroup at most
  static constexpr int PS = TP + (G < 4 ? 4 : G);                   // floats of a row of weights, off the banks' period
};

// One row's attention to `chunk` positions of one KV head, for up to 4 RT of the
// query heads that share it.  The positions go to the waves in turns of TP, and
// each wave keeps its own reference m (the maximum when it last moved: it moves
// where a score is 8 past it) and sum l.
//   S = K Q^T  A = 16 positions (lane j + 16 g: position j, the elements of its
//              16-byte runs g, g + 4, ...), B = the query heads.  Keys of 16
//              bits go into v_mfma_f32_16x16x32 as they are, against the 16-bit
//              pieces of the queries; f32 keys, and EXACT, take
//              v_mfma_f32_16x16x4_f32.  Lane j + 16 g then holds head j's scores
//              of positions 4 g .. 4 g + 3.
//   O += P V   v_mfma_f32_4x4x1_16b: each block of four lanes is a product of
//              its own, so a load of 16 bytes a lane -- G positions side by
//              side, LPR lanes to a row -- is the A operand as it stands: block
//              b takes its own position's 4 EL elements, one MFMA per element of
//              a lane, against the weights of four heads.  Positions G apart are
//              summed in the instruction, the G sums at the end.
// The products of the values are float32, the sums all are.  A score that is
// NaN (an infinite key times a piece that is 0, or a real one) sends the
// workgroup through the chunk again in float32, where it acts as in the plain
// formula.
//
// What bounds it: the cache's bytes.  Per 64 positions of an f16 head of 64
// elements, 16 KB, a wave spends 16 + 64 MFMAs (770 cycles) and about 1000 VALU
// cycles; a CU's share of 7 TB/s is 1440 cycles for them.
template <class KV, int DC, int RT>
__global__ __launch_bounds__(64 * AW) void k_attn_paged(AttnArgs A) {
  using Y = Lay<KV, DC>;
  constexpr int HD = Y::HD, EL = Y::EL, RUN = Y::RUN, NR = Y::NR, LPR = Y::LPR, G = Y::G, PT = Y::PT, TP = Y::TP,
                NU = Y::NU, PS = Y::PS, NP = Piece<KV>::NP;
  static_assert(ASUB % (AW * TP) == 0, "whole turns");
  using T = typename KV::T;
  // the places of the positions and the waves' weights; then the waves' sums
  constexpr int kPlaces = 2 * ASUB, kWeights = AW * 4 * RT * PS, kSums = AW * G * 4 * HD;
  constexpr int kLds = kPlaces + kWeights > kSums ? kPlaces + kWeights : kSums;
  __shared__ __attribute__((aligned(16))) float lds[kLds];
  __shared__ float ml[2][AW][16];
  __shared__ int last;
  int64_t *place = reinterpret_cast<int64_t *>(lds);
  int unit = blockIdx.x;
  const int tile = unit % A.tiles;
  unit /= A.tiles;
  const int kvh = unit % A.P.n_kv, row = unit / A.P.n_kv;
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), j = lane & 15, g = lane >> 4;
  float *pw = lds + kPlaces + wv * (4 * RT * PS);
  const int h0 = kvh * A.rep + tile * A.heads, nq = min(A.heads, A.rep - tile * A.heads);
  int seq;
  int n = row_len(A, row, seq);
  if (n == -1) return;
  bool bad = n < 0;
  if (bad) n = 0;
  const int p0 = blockIdx.y * A.chunk, p1 = min(n, p0 + A.chunk);
  if (blockIdx.y > 0 && p0 >= n) return;
  const T *kb = static_cast<const T *>(A.P.k) + kvh * A.P.head_stride + g * RUN;
  const T *vb = static_cast<const T *>(A.P.v) + kvh * A.P.head_stride + (lane & (LPR - 1)) * EL;
  const float *qr = A.q + ((size_t)row * A.n_heads + h0 + (j < nq ? j : 0)) * HD + g * RUN;

  float m, l;
  v4f o[RT][EL];
  auto pass = [&](auto exact_) {
    constexpr bool EXACT = decltype(exact_)::value;
    // the queries: floats, or pieces scaled by a power of two
    float qf[EXACT ? NR * RUN : 1];
    u32x4 qp[EXACT ? 1 : NP][EXACT ? 1 : NR];
    float fac = A.scale;  // of a score
    if constexpr (EXACT) {
#pragma unroll
      for (int i = 0; i < NR; ++i)
#pragma unroll
        for (int e = 0; e < RUN; ++e) qf[i * RUN + e] = j < nq ? qr[4 * i * RUN + e] : 0.f;
    } else {
      float x[NR * RUN], top = 0.f;
#pragma unroll
      for (int i = 0; i < NR; ++i)
#pragma unroll
        for (int e = 0; e < RUN; ++e) {
          x[i * RUN + e] = j < nq ? qr[4 * i * RUN + e] : 0.f;
          top = fmaxf(top, fabsf(x[i * RUN + e]));
        }
      if constexpr (__is_same(KV, KvF16)) {
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        // the head's largest element to [2^14, 2^15): its pieces end at 2^-24
        const int ex = min(max(141 - (int)(__float_as_uint(top) >> 23), -126), 100);
        const float up = __uint_as_float((uint32_t)(127 + ex) << 23);
#pragma unroll
        for (int i = 0; i < NR * RUN; ++i) x[i] *= up;
        fac *= __uint_as_float((uint32_t)(127 - ex) << 23);
      }
#pragma unroll
      for (int k = 0; k < NP; ++k)
#pragma unroll
        for (int i = 0; i < NR; ++i) {
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint16_t a = KV::put(x[i * RUN + 2 * e]), b = KV::put(x[i * RUN + 2 * e + 1]);
            x[i * RUN + 2 * e] -= Piece<KV>::val(a);
            x[i * RUN + 2 * e + 1] -= Piece<KV>::val(b);
            w[e] = (uint32_t)a | (uint32_t)b << 16;
          }
          qp[k][i] = u32x4{w[0], w[1], w[2], w[3]};
        }
    }
    m = -INFINITY, l = 0.f;
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int e = 0; e < EL; ++e) o[r][e] = v4f{0.f, 0.f, 0.f, 0.f};
    for (int s0 = p0; s0 < p1; s0 += ASUB) {
      const int s1 = min(p1, s0 + ASUB), fill = (s1 - s0 + TP - 1) / TP * TP;
      __syncthreads();
      for (int i = threadIdx.x; i < fill; i += 64 * AW) {
        const int pos = min(s0 + i, s1 - 1), c = page_of(A.P, pos);  // the last position's place behind the end
        int page = A.P.table[(size_t)seq * A.P.table_cols + c];
        if (page < 0 || page >= A.P.pages) bad = true, page = 0;
        place[i] = page * A.P.page_stride + (pos - c * A.P.page_size) * A.P.row_stride;
      }
      __syncthreads();
      Raw<KV, RUN> kr[PT][NR];
      Raw<KV, EL> vr[NU];
      auto load_k = [&](int t0) {
#pragma unroll
        for (int t = 0; t < PT; ++t) {
          const T *k = kb + place[t0 - s0 + 16 * t + j];
#pragma unroll
          for (int i = 0; i < NR; ++i) kr[t][i].load(k + 4 * i * RUN);
        }
      };
      auto load_v = [&](int t0) {
#pragma unroll
        for (int u = 0; u < NU; ++u) vr[u].load(vb + place[t0 - s0 + u * G + lane / LPR]);
      };
      int t0 = s0 + wv * TP;
      if (t0 < s1) load_k(t0), load_v(t0);
      for (; t0 < s1; t0 += AW * TP) {
        const bool more = t0 + AW * TP < s1;
        v4f s[PT];
#pragma unroll
        for (int t = 0; t < PT; ++t) {
          s[t] = v4f{0.f, 0.f, 0.f, 0.f};
          if constexpr (EXACT) {
#pragma unroll
            for (int i = 0; i < NR; ++i)
#pragma unroll
              for (int e = 0; e < RUN; ++e)
                s[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(kr[t][i].get(e), qf[i * RUN + e], s[t], 0, 0, 0);
          } else {
#pragma unroll
            for (int k = NP - 1; k >= 0; --k)
#pragma unroll
              for (int i = 0; i < NR; ++i)
                s[t] = mma32<KV>(u32x4{kr[t][i].d[0], kr[t][i].d[1], kr[t][i].d[2], kr[t][i].d[3]}, qp[k][i], s[t]);
          }
        }
        if (more) load_k(t0 + AW * TP);
        float mx = -INFINITY;
#pragma unroll
        for (int t = 0; t < PT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[t][i] *= fac;
        if (t0 + TP > s1) {  // the last turn: positions behind the end
#pragma unroll
          for (int t = 0; t < PT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[t][i] = t0 + 16 * t + 4 * g + i < s1 ? s[t][i] : -INFINITY;
#pragma unroll
          for (int u = 0; u < NU; ++u)
            if (t0 + u * G + lane / LPR >= s1) vr[u].clear();
        }
#pragma unroll
        for (int t = 0; t < PT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[t][i]);
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        if (__any(mx > m + 8.f)) {
          const float mn = fmaxf(m, mx), corr = __builtin_amdgcn_exp2f((m - score_ref(mn)) * LOG2E);
          l *= corr;
#pragma unroll
          for (int r = 0; r < RT; ++r) {
            const float c = __shfl(corr, 4 * r + (lane & 3));
#pragma unroll
            for (int e = 0; e < EL; ++e)
#pragma unroll
              for (int i = 0; i < 4; ++i) o[r][e][i] *= c;
          }
          m = mn;
        }
        const float ref = score_ref(m);
#pragma unroll
        for (int t = 0; t < PT; ++t) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s[t][i] = __builtin_amdgcn_exp2f((s[t][i] - ref) * LOG2E);
            l += s[t][i];
          }
          if (j < 4 * RT) *reinterpret_cast<v4f *>(pw + j * PS + 16 * t + 4 * g) = s[t];
        }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int u = 0; u < NU; ++u) {
          float w[RT];
#pragma unroll
          for (int r = 0; r < RT; ++r) w[r] = pw[(4 * r + (lane & 3)) * PS + u * G + lane / LPR];
#pragma unroll
          for (int e = 0; e < EL; ++e)
#pragma unroll
            for (int r = 0; r < RT; ++r) o[r][e] = __builtin_amdgcn_mfma_f32_4x4x1f32(vr[u].get(e), w[r], o[r][e], 0, 0, 0);
        }
        __builtin_amdgcn_wave_barrier();
        if (more) load_v(t0 + AW * TP);
      }
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
  };
  if constexpr (NP == 1) {
    pass(std::true_type{});
  } else {
    pass(std::false_type{});
    if (__syncthreads_or(l != l && j < nq)) pass(std::true_type{});
  }
  bad = __syncthreads_or(bad);
  // the waves' parts
  if (g == 0) ml[0][wv][j] = m, ml[1][wv][j] = l;
  float *part = A.part + ((size_t)blockIdx.x * A.splits + blockIdx.y) * A.heads * (HD + 2);
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    if (4 * r >= nq) break;
    __syncthreads();
    // lane: head 4 r + lane % 4, the elements of the lanes of its block
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float *to = lds + ((wv * G + lane / LPR) * 4 + (lane & 3)) * HD + (((lane & ~3) + i) & (LPR - 1)) * EL;
#pragma unroll
      for (int e = 0; e < EL; ++e) to[e] = o[r][e][i];
    }
    __syncthreads();
    for (int x = threadIdx.x; x < min(4, nq - 4 * r) * HD; x += 64 * AW) {
      const int h = x / HD, d = x - h * HD, hh = 4 * r + h;
      float mm = -INFINITY;
#pragma unroll
      for (int w = 0; w < AW; ++w) mm = fmaxf(mm, ml[0][w][hh]);
      const float ref = score_ref(mm);
      float ll = 0.f, oo = 0.f;
#pragma unroll
      for (int w = 0; w < AW; ++w) {
        const float c = __builtin_amdgcn_exp2f((ml[0][w][hh] - ref) * LOG2E);
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < G; ++k) sum += lds[((w * G + k) * 4 + h) * HD + d];
        ll += c * ml[1][w][hh];
        oo += c * sum;
      }
      if (bad) ll = oo = __builtin_nanf("");
      if (A.splits == 1) {
        A.out[((size_t)row * A.n_heads + h0 + hh) * HD + d] = n == 0 && !bad ? 0.f : oo / ll;
      } else {
        coh_stf(part, 4u * (hh * (HD + 2) + d), oo);
        if (d == 0) coh_stf(part, 4u * (hh * (HD + 2) + HD), mm), coh_stf(part, 4u * (hh * (HD + 2) + HD + 1), ll);
      }
    }
  }
  if (A.splits == 1) return;
  // the last part to be there joins them
  const int parts = n == 0 ? 1 : (n + A.chunk - 1) / A.chunk;
  wait_stores();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(A.count + blockIdx.x, 1u) == (unsigned)parts - 1;
  __syncthreads();
  if (!last) return;
  const float *all = A.part + (size_t)blockIdx.x * A.splits * A.heads * (HD + 2);
  const uint32_t step = 4u * A.heads * (HD + 2);
  for (int x = threadIdx.x; x < nq * HD; x += 64 * AW) {
    const int h = x / HD, d = x - h * HD;
    const uint32_t at = 4u * (h * (HD + 2));
    float mm = -INFINITY;
    for (int i = 0; i < parts; ++i) mm = fmaxf(mm, coh_ldf(all, i * step + at + 4u * HD));
    const float ref = score_ref(mm);
    float ll = 0.f, oo = 0.f;
#pragma unroll 4
    for (int i = 0; i < parts; ++i) {
      const float c = __builtin_amdgcn_exp2f((coh_ldf(all, i * step + at + 4u * HD) - ref) * LOG2E);
      ll += c * coh_ldf(all, i * step + at + 4u * HD + 4u);
      oo += c * coh_ldf(all, i * step + at + 4u * d);
    }
    A.out[((size_t)row * A.n_heads + h0 + h) * HD + d] = n == 0 && !bad ? 0.f : oo / ll;
  }
  if (threadIdx.x == 0) __hip_atomic_store(A.count + blockIdx.x, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// ---------------------------------------------------------------- host side
int check_pages(const mllm_kv_pages *kv, Pages *out) {
  MLLM_CHECK(kv, "null pointer");
  MLLM_CHECK(kv->k && kv->v && kv->table, "null pointer in the pages");
  MLLM_CHECK(kv->n_kv_heads > 0 && kv->pages > 0 && kv->page_size > 0 && kv->sequences > 0 && kv->table_cols > 0,
             "invalid pages: %d KV heads, %d pages of %d positions, %d sequences of %d pages", kv->n_kv_heads, kv->pages,
             kv->page_size, kv->sequences, kv->table_cols);
  if (kv->storage != MLLM_F32 && kv->storage != MLLM_F16 && kv->storage != MLLM_BF16)
    return set_error(MLLM_ERR_UNSUPPORTED, "storage %d unsupported (f32, f16 or bf16)", kv->storage);
  if (kv->head_dim <= 0 || kv->head_dim % 32 || kv->head_dim > 256)
    return set_error(MLLM_ERR_UNSUPPORTED, "head_dim %d unsupported (a multiple of 32, at most 256)", kv->head_dim);
  MLLM_CHECK((int64_t)kv->page_size * kv->table_cols < (1ll << 31), "%d pages of %d positions a sequence exceed 2^31",
             kv->table_cols, kv->page_size);
  int64_t ps = kv->page_stride, hs = kv->head_stride, rs = kv->row_stride;
  if (!ps && !hs && !rs) {
    rs = kv->head_dim;
    hs = rs * kv->page_size;
    ps = hs * kv->n_kv_heads;
  }
  const int es = kv->storage == MLLM_F32 ? 4 : 2;
  MLLM_CHECK(ps > 0 && hs > 0 && rs >= kv->head_dim, "invalid strides %lld, %lld, %lld", (long long)ps, (long long)hs,
             (long long)rs);
  MLLM_CHECK((((uintptr_t)kv->k | (uintptr_t)kv->v | (uint64_t)(ps | hs | rs) * es) & 15) == 0,
             "k, v and the strides must be 16-byte aligned");
  *out = Pages{kv->k,   kv->v,         kv->table,     ps,
               hs,      rs,            kv->pages,     kv->page_size,
               kv->sequences, kv->table_cols, kv->n_kv_heads, kv->head_dim,
               (uint32_t)((1ull << 32) / (uint64_t)kv->page_size + 1)};
  return 0;
}

hipStream_t as_stream(void *s) { return reinterpret_cast<hipStream_t>(s); }

// Positions per workgroup and the number of parts for rows of up to max_len
// positions: parts only where the rows and heads alone would not fill the chip,
// each of 256 positions (a turn of the four waves) at least.
void attn_plan(int64_t units, int max_len, int *chunk, int *splits) {
  const int64_t most = (max_len + 255) / 256;
  int64_t s = (kUnits + units - 1) / units;
  s = s > most ? most : s;
  s = s < 1 ? 1 : s;
  const int64_t c = ((max_len + s - 1) / s + 255) / 256 * 256;
  *chunk = c > 0x7fffff00 ? 0x7fffff00 : (int)(c < 256 ? 256 : c);
  *splits = units >= kUnits || max_len == 0 ? 1 : (int)(((int64_t)max_len + *chunk - 1) / *chunk);
}

template <class KV>
constexpr int heads_at_most(int dc) {
  return dc == 1   ? Lay<KV, 1>::AQ
         : dc == 2 ? Lay<KV, 2>::AQ
         : dc == 3 ? Lay<KV, 3>::AQ
         : dc == 4 ? Lay<KV, 4>::AQ
         : dc == 5 ? Lay<KV, 5>::AQ
         : dc == 6 ? Lay<KV, 6>::AQ
         : dc == 7 ? Lay<KV, 7>::AQ
                   : Lay<KV, 8>::AQ;
}

struct AttnPlan {
  int rep, tiles, heads, chunk, splits;
  int64_t units;
  uint64_t bytes;  // of the workspace: the counters, then the parts
};

int attn_shape(const mllm_kv_pages *kv, const Pages &P, int rows, int n_heads, int max_len, AttnPlan *pl) {
  MLLM_CHECK(rows > 0 && n_heads > 0 && n_heads % P.n_kv == 0, "invalid shape rows=%d n_heads=%d over %d KV heads", rows,
             n_heads, P.n_kv);
  MLLM_CHECK(max_len >= 0 && max_len <= (int64_t)P.page_size * P.table_cols,
             "max_len=%d beyond the %d pages of %d positions of a sequence", max_len, P.table_cols, P.page_size);
  pl->rep = n_heads / P.n_kv;
  const int dc = P.hd / 32, aq = kv->storage == MLLM_F32   ? heads_at_most<KvF32>(dc)
                                 : kv->storage == MLLM_F16 ? heads_at_most<KvF16>(dc)
                                                           : heads_at_most<KvBf16>(dc);
  pl->heads = pl->rep < aq ? pl->rep : aq;
  pl->tiles = (pl->rep + aq - 1) / aq;
  pl->units = (int64_t)rows * P.n_kv * pl->tiles;
  MLLM_CHECK(pl->units < (1ll << 31) && (int64_t)rows * n_heads < (1ll << 31), "%d rows of %d heads exceed a launch", rows,
             n_heads);
  attn_plan(pl->units, max_len, &pl->chunk, &pl->splits);
  pl->bytes = pl->splits > 1 ? kUnits * sizeof(unsigned) +
                                   (uint64_t)pl->units * pl->splits * pl->heads * (P.hd + 2) * sizeof(float)
                             : 0;
  return 0;
}

template <class KV, int DC>
int attn_launch(const AttnArgs &A, dim3 grid, hipStream_t st) {
  if (A.heads <= 4) hipLaunchKernelGGL((k_attn_paged<KV, DC, 1>), grid, dim3(64 * AW), 0, st, A);
  else if (A.heads <= 8) hipLaunchKernelGGL((k_attn_paged<KV, DC, 2>), grid, dim3(64 * AW), 0, st, A);
  else if constexpr (Lay<KV, DC>::AQ > 8) hipLaunchKernelGGL((k_attn_paged<KV, DC, 4>), grid, dim3(64 * AW), 0, st, A);
  MLLM_HIP(hipGetLastError());
  return 0;
}

template <class KV>
int attn_dispatch(const AttnArgs &A, dim3 grid, hipStream_t st) {
  switch (A.P.hd / 32) {
  case 1: return attn_launch<KV, 1>(A, grid, st);
  case 2: return attn_launch<KV, 2>(A, grid, st);
  case 3: return attn_launch<KV, 3>(A, grid, st);
  case 4: return attn_launch<KV, 4>(A, grid, st);
  case 5: return attn_launch<KV, 5>(A, grid, st);
  case 6: return attn_launch<KV, 6>(A, grid, st);
  case 7: return attn_launch<KV, 7>(A, grid, st);
  default: return attn_launch<KV, 8>(A, grid, st);
  }
}

}  // namespace

extern "C" int mllm_rope_kv_paged(const mllm_kv_pages *kv, int tokens, int n_heads, const float *qkv,
                                  const int32_t *seq, const int32_t *pos, const float *inv_freq, int rot,
                                  int interleaved, const float *q_gain, const float *k_gain, float eps, float *q,
                                  void *stream) {
  RopeArgs A{};
  if (int rc = check_pages(kv, &A.P)) return rc;
  MLLM_CHECK(tokens > 0 && n_heads > 0 && n_heads % A.P.n_kv == 0, "invalid shape tokens=%d n_heads=%d over %d KV heads",
             tokens, n_heads, A.P.n_kv);
  MLLM_CHECK(rot >= 0 && rot % 2 == 0 && rot <= A.P.hd, "rot=%d: an even part of the head's %d", rot, A.P.hd);
  MLLM_CHECK(qkv && pos && q && (rot == 0 || inv_freq), "null pointer");
  MLLM_CHECK(seq || tokens <= A.P.sequences, "%d tokens without seq, %d sequences", tokens, A.P.sequences);
  MLLM_CHECK((((uintptr_t)qkv | (uintptr_t)q) & 15) == 0, "qkv and q must be 16-byte aligned");
  A.qkv = qkv, A.inv_freq = inv_freq, A.q_gain = q_gain, A.k_gain = k_gain;
  A.seq = seq, A.pos = pos, A.q = q;
  A.n_heads = n_heads, A.rot = rot, A.interleaved = interleaved != 0, A.eps = eps;
  A.lph = 4, A.lg_lph = 2;
  while (8 * A.lph < A.P.hd) A.lph <<= 1, ++A.lg_lph;
  const int64_t heads = (int64_t)n_heads + 2 * (int64_t)A.P.n_kv;
  const int fit = WG >> A.lg_lph;
  A.n_wg = (int)((heads + fit - 1) / fit);
  A.per_wg = (int)((heads + A.n_wg - 1) / A.n_wg);
  MLLM_CHECK(heads < (1 << 20) && (int64_t)tokens * A.n_wg < (1ll << 31), "%d tokens of %lld heads exceed a launch",
             tokens, (long long)heads);
  const dim3 grid((unsigned)(tokens * A.n_wg)), block((unsigned)((A.per_wg * A.lph + 63) & ~63));
  const bool vec = rot % 8 == 0;
  const auto kern = kv->storage == MLLM_F32   ? (vec ? k_rope_kv<KvF32, true> : k_rope_kv<KvF32, false>)
                    : kv->storage == MLLM_F16 ? (vec ? k_rope_kv<KvF16, true> : k_rope_kv<KvF16, false>)
                                              : (vec ? k_rope_kv<KvBf16, true> : k_rope_kv<KvBf16, false>);
  hipLaunchKernelGGL(kern, grid, block, 0, as_stream(stream), A);
  MLLM_HIP(hipGetLastError());
  return 0;
}

extern "C" uint64_t mllm_attn_paged_workspace(const mllm_kv_pages *kv, int rows, int n_heads, int max_len) {
  Pages P;
  AttnPlan pl;
  if (check_pages(kv, &P) || attn_shape(kv, P, rows, n_heads, max_len, &pl)) return 0;
  return pl.bytes;
}

extern "C" int mllm_attn_paged(const mllm_kv_pages *kv, int rows, int n_heads, const float *q, const int32_t *seq,
                               const int32_t *len, int max_len, float scale, float *out, void *workspace,
                               uint64_t workspace_bytes, void *stream) {
  AttnArgs A{};
  AttnPlan pl;
  if (int rc = check_pages(kv, &A.P)) return rc;
  if (int rc = attn_shape(kv, A.P, rows, n_heads, max_len, &pl)) return rc;
  MLLM_CHECK(q && len && out, "null pointer");
  MLLM_CHECK(seq || rows <= A.P.sequences, "%d rows without seq, %d sequences", rows, A.P.sequences);
  MLLM_CHECK(pl.bytes == 0 || workspace, "null workspace, %llu bytes needed", (unsigned long long)pl.bytes);
  MLLM_CHECK(workspace_bytes >= pl.bytes, "workspace of %llu bytes, %llu needed", (unsigned long long)workspace_bytes,
             (unsigned long long)pl.bytes);
  MLLM_CHECK(pl.bytes == 0 || ((uintptr_t)workspace & 15) == 0, "the workspace must be 16-byte aligned");
  A.q = q, A.seq = seq, A.len = len, A.out = out;
  A.count = static_cast<unsigned *>(workspace);
  A.part = reinterpret_cast<float *>(A.count + kUnits);
  A.n_heads = n_heads, A.rep = pl.rep, A.tiles = pl.tiles, A.heads = pl.heads, A.max_len = max_len;
  A.chunk = pl.chunk, A.splits = pl.splits, A.scale = scale;
  const dim3 grid((unsigned)pl.units, (unsigned)pl.splits);
  hipStream_t st = as_stream(stream);
  return kv->storage == MLLM_F32   ? attn_dispatch<KvF32>(A, grid, st)
         : kv->storage == MLLM_F16 ? attn_dispatch<KvF16>(A, grid, st)
                                   : attn_dispatch<KvBf16>(A, grid, st);
}
