// mllm_paged_attn.h -- the attention kernel of mllm_attn_paged, for one storage
// of the cache to a translation unit.
#pragma once

#include <type_traits>

#include "mllm_device.h"
#include "mllm_host.h"
#include "mllm_paged.h"

namespace {

using namespace mllm;
using namespace mllm::paged;

// A row's length as the kernels use it: -1 padding (the row is left as it
// was), -2 not possible (NaN).
__device__ __forceinline__ int row_len(const AttnArgs &A, int row, int &seq) {
  const int n = A.len[row];  // both loads in flight
  seq = A.seq ? A.seq[row] : row;
  if (seq < 0 || seq >= A.P.sequences) return -1;
  return n < 0 || n > A.max_len ? -2 : n;
}

// E elements of the cache at p as floats, loaded in runs of at most 16 bytes.
template <class KV, int E>
struct Raw {
  static constexpr int N = E * (int)sizeof(typename KV::T) / 4;  // dwords
  uint32_t d[N];
  template <bool STREAM>
  __device__ __forceinline__ void load(const void *p) {
    typedef uint32_t u4 __attribute__((ext_vector_type(4), aligned(4)));
    typedef uint32_t u2 __attribute__((ext_vector_type(2), aligned(4)));
    const uint32_t *s = static_cast<const uint32_t *>(p);
#pragma unroll
    for (int i = 0; i + 4 <= N; i += 4) {
      const u4 *q = reinterpret_cast<const u4 *>(s + i);
      const u4 v = STREAM ? __builtin_nontemporal_load(q) : *q;
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

// The 16-bit pieces of a float: take() takes the leading one off x.  Two f16
// pieces, rounded to nearest, hold 22 bits (the caller scales them away from
// the type's ends); three bf16 pieces, cut off, all 24.
template <class KV>
struct Piece;
template <>
struct Piece<KvF16> {
  static constexpr int NP = 2;
  static __device__ __forceinline__ uint32_t take(float &x) {
    const __half h = __float2half_rn(x);
    x -= __half2float(h);
    return __half_as_ushort(h);
  }
};
template <>
struct Piece<KvBf16> {
  static constexpr int NP = 3;
  static __device__ __forceinline__ uint32_t take(float &x) {
    const uint32_t u = __float_as_uint(x);
    x -= __uint_as_float(u & 0xffff0000u);
    return u >> 16;
  }
};
template <>
struct Piece<KvF32> {
  static constexpr int NP = 1;  // no pieces: the products are float32 as they are
  static __device__ __forceinline__ uint32_t take(float &x) { return __float_as_uint(x); }
};

// Sums of registers over the lanes 32, 16, 8, 4 apart (down to LPR): the first
// two steps halve the registers -- v_permlane32_swap puts v[k] and v[k + N / 2]
// into one register, the lower lanes' and the upper lanes' -- the others leave
// the sum in every lane.  Returns the index of v[0] in this lane.
__device__ __forceinline__ float swap_sum32(float x, float y) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(y), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float swap_sum16(float x, float y) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(y), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
template <int LPR, int N>
__device__ __forceinline__ int lane_sums(float (&v)[N]) {
  const int lane = threadIdx.x & 63;
  int at = 0;
  if constexpr (LPR <= 32) {
#pragma unroll
    for (int k = 0; k < N / 2; ++k) v[k] = swap_sum32(v[k], v[k + N / 2]);
    at += lane & 32 ? N / 2 : 0;
  }
  if constexpr (LPR <= 16) {
#pragma unroll
    for (int k = 0; k < N / 4; ++k) v[k] = swap_sum16(v[k], v[k + N / 4]);
    at += lane & 16 ? N / 4 : 0;
  }
  constexpr int L = LPR <= 16 ? N / 4 : LPR <= 32 ? N / 2 : N;
  if constexpr (LPR <= 8) {
#pragma unroll
    for (int k = 0; k < L; ++k) v[k] += dpp_f<0x128>(v[k]);  // row_ror:8
  }
  if constexpr (LPR <= 4) {
#pragma unroll
    for (int k = 0; k < L; ++k) v[k] += dpp_f<0x124>(v[k]);  // row_ror:4
  }
  return at;
}

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
// What bounds it: the cache's bytes, at about 28 GB/s to a CU (what these loads
// come to, not what a CU can read) and 6.2 to 6.4 TB/s in all, and for short rows a
// workgroup's start and end.  Per 64 positions of an f16 head of 64 elements, 16
// KB, a wave spends 16 + 64 MFMAs (770 cycles) and about 1000 VALU cycles; a
// SIMD's share of the CU's 28 GB/s is 5600 cycles for them.  Measured, us: 2 rows
// of 100000 positions, 8 heads of 128 bf16 or f16 elements (819 MB), 143 (5.7
// TB/s), of f32 (1638 MB) 255; 64 rows of 512 to 2048, 5 heads of 64 f16 or bf16
// elements (102 MB), 30.5, of f32 (203 MB) 45.8;
// 2560 units of 128 positions, a wave to each (88 MB), 22; 64 rows, 8 query heads
// to a KV head of 256, one workgroup to a CU: bf16 (177 MB) 48, f32 (349 MB) 76.
// In the 102 MB of f16 a workgroup takes 1.0 to its row's length, 1.4 to its pages,
// 2.4 to its first scores, 0.8 for the sums of the lanes and waves, 0.8 to store
// them and 1.7 to join them.  Tried there without gain: three workgroups to a CU
// in place of two (fewer positions in flight), pages looked up a block ahead (its
// barriers in the loop cost more than the stops it saves), finer parts under the
// same two workgroups (33 to 40), parts of one wave each (29.5 to 37).
// STREAM: the cache is read past the caches.  AW: waves of a workgroup; with one
// there is no joining.
template <class KV, int DC, int RT, bool STREAM, int AW>
__global__ __launch_bounds__(64 * AW) void k_attn_paged(AttnArgs A) {
  constexpr int ASUB = APLACES * AW;  // positions whose places in the pool are in LDS at a time
  using Y = Lay<KV, DC>;
  constexpr int HD = Y::HD, EL = Y::EL, RUN = Y::RUN, NR = Y::NR, LPR = Y::LPR, G = Y::G, PT = Y::PT, TP = Y::TP,
                NU = Y::NU, PS = Y::PS, NP = Piece<KV>::NP;
  static_assert(ASUB % (AW * TP) == 0, "whole turns");
  using T = typename KV::T;
  // the places of the positions and the waves' weights; then the waves' sums
  constexpr int kPlaces = 2 * ASUB, kWeights = AW * 4 * RT * PS, kSums = AW * 4 * HD;
  constexpr int kJoin = AW == 1 ? 0 : 17 * kParts;  // a join's weights and the heads' sums
  constexpr int kMain = kPlaces + kWeights > kSums ? kPlaces + kWeights : kSums, kLds = kMain > kJoin ? kMain : kJoin;
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
  // the queries; in flight while the row is looked up
  float qf[NR * RUN];
  auto load_q = [&] {
    const float *qr = A.q + ((size_t)row * A.n_heads + h0 + min(j, nq - 1)) * HD + g * RUN;
#pragma unroll
    for (int i = 0; i < NR; ++i)
#pragma unroll
      for (int e = 0; e < RUN; e += 4) {
        const float4 v = *reinterpret_cast<const float4 *>(qr + 4 * i * RUN + e);
        float *to = qf + i * RUN + e;
        to[0] = v.x, to[1] = v.y, to[2] = v.z, to[3] = v.w;
      }
  };
  load_q();
  int seq;
  int n = row_len(A, row, seq);
  if (n == -1) return;
  bool bad = n < 0;
  if (bad) n = 0;
  const int p0 = blockIdx.y * A.chunk, p1 = min(n, p0 + A.chunk);
  if (blockIdx.y > 0 && p0 >= n) return;
  const T *kb = static_cast<const T *>(A.P.k) + kvh * A.P.head_stride + g * RUN;
  const T *vb = static_cast<const T *>(A.P.v) + kvh * A.P.head_stride + (lane & (LPR - 1)) * EL;
  float m, l;
  v4f o[RT][EL];
  auto pass = [&](auto exact_) {
    constexpr bool EXACT = decltype(exact_)::value;
    if constexpr (EXACT && NP > 1) load_q();
#pragma unroll
    for (int i = 0; i < NR * RUN; ++i) qf[i] = j < nq ? qf[i] : 0.f;  // zeros past the last head
    float fac = A.scale;  // of a score
    u32x4 qp[EXACT ? 1 : NP][EXACT ? 1 : NR];
    auto pieces = [&] {
      float x[NR * RUN], up = 1.f;
      if constexpr (__is_same(KV, KvF16)) {
        // the head's largest element to [2^14, 2^15): its pieces end at 2^-24
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < NR * RUN; ++i) top = fmaxf(top, fabsf(qf[i]));
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const int ex = min(max(141 - (int)(__float_as_uint(top) >> 23), -126), 100);
        up = __uint_as_float((uint32_t)(127 + ex) << 23);
        fac *= __uint_as_float((uint32_t)(127 - ex) << 23);
      }
#pragma unroll
      for (int i = 0; i < NR * RUN; ++i) x[i] = qf[i] * up;
#pragma unroll
      for (int k = 0; k < NP; ++k)
#pragma unroll
        for (int i = 0; i < NR; ++i) {
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            w[e] = Piece<KV>::take(x[i * RUN + 2 * e]);
            w[e] |= Piece<KV>::take(x[i * RUN + 2 * e + 1]) << 16;
          }
          qp[k][i] = u32x4{w[0], w[1], w[2], w[3]};
        }
    };
    if constexpr (!EXACT) pieces();
    m = -INFINITY, l = 0.f;
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int e = 0; e < EL; ++e) o[r][e] = v4f{0.f, 0.f, 0.f, 0.f};
    for (int s0 = p0; s0 < p1; s0 += ASUB) {
      const int s1 = min(p1, s0 + ASUB), fill = (s1 - s0 + TP - 1) / TP * TP;
      __syncthreads();
      // the last position's place behind the end; all of a thread's pages at once
      constexpr int NF = ASUB / (64 * AW);
      int page[NF], slot[NF];
#pragma unroll
      for (int k = 0; k < NF; ++k)
        if (64 * AW * k < fill) {
          const int pos = min(s0 + (int)threadIdx.x + 64 * AW * k, s1 - 1), c = page_of(A.P, pos);
          slot[k] = pos - c * A.P.page_size;
          page[k] = A.P.table[(size_t)seq * A.P.table_cols + c];
        }
#pragma unroll
      for (int k = 0; k < NF; ++k)
        if (64 * AW * k < fill) {
          if (page[k] < 0 || page[k] >= A.P.pages) bad = true, page[k] = 0;
          place[threadIdx.x + 64 * AW * k] = page[k] * A.P.page_stride + slot[k] * A.P.row_stride;
        }
      __syncthreads();
      Raw<KV, RUN> kr[PT][NR];
      Raw<KV, EL> vr[NU];
      auto load_k = [&](int t0) {
#pragma unroll
        for (int t = 0; t < PT; ++t) {
          const T *k = kb + place[t0 - s0 + 16 * t + j];
#pragma unroll
          for (int i = 0; i < NR; ++i) kr[t][i].template load<STREAM>(k + 4 * i * RUN);
        }
      };
      auto load_v = [&](int t0) {
#pragma unroll
        for (int u = 0; u < NU; ++u) vr[u].template load<STREAM>(vb + place[t0 - s0 + u * G + lane / LPR]);
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
  const uint32_t part_size = ((uint32_t)A.heads * (HD + 2) + 3) & ~3u;  // floats: the heads' sums, then maxima and sums
  float *part = A.part + ((size_t)blockIdx.x * A.splits + blockIdx.y) * part_size;
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    if (4 * r >= nq) break;
    // lane: head 4 r + lane % 4, the elements of the lanes of its block
    float v[4 * EL];
#pragma unroll
    for (int e = 0; e < EL; ++e)
#pragma unroll
      for (int i = 0; i < 4; ++i) v[4 * e + i] = o[r][e][i];
    const int at = lane_sums<LPR>(v);
    constexpr int NV = LPR <= 16 ? EL : LPR <= 32 ? 2 * EL : 4 * EL;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int e = (at + k) >> 2, i = (at + k) & 3;
      lds[(wv * 4 + (lane & 3)) * HD + (((lane & ~3) + i) & (LPR - 1)) * EL + e] = v[k];
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
        ll += c * ml[1][w][hh];
        oo += c * lds[(w * 4 + h) * HD + d];
      }
      if (bad) ll = oo = __builtin_nanf("");
      if (A.splits == 1) {
        A.out[((size_t)row * A.n_heads + h0 + hh) * HD + d] = n == 0 && !bad ? 0.f : oo / ll;
      } else {
        coh_stf(part, 4u * (hh * HD + d), oo);
        if (d == 0) coh_stf(part, 4u * (A.heads * HD + 2 * hh), mm), coh_stf(part, 4u * (A.heads * HD + 2 * hh + 1), ll);
      }
    }
  }
  if (AW == 1 || A.splits == 1) return;
  if constexpr (AW > 1) {
  // the last part to be there joins them
  const int parts = n == 0 ? 1 : (n + A.chunk - 1) / A.chunk;
  wait_stores();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(A.count + blockIdx.x, 1u) == (unsigned)parts - 1;
  __syncthreads();
  if (!last) return;
  const float *all = A.part + (size_t)blockIdx.x * A.splits * part_size;
  const uint32_t step = 4u * part_size, at_ml = 4u * A.heads * HD;
  // four elements of the sums to a thread, the first of them in flight over the
  // weights
  constexpr int JB = 16;
  const int items = nq * (HD / 4);
  float4 v[JB];
  auto load_sums = [&](int x, int i0) {
#pragma unroll
    for (int k = 0; k < JB; ++k)
      if (i0 + k < parts) v[k] = coh_ld4(all, (i0 + k) * step + 16u * x);
  };
  if ((int)threadIdx.x < items) load_sums(threadIdx.x, 0);
  // the parts' weights, and the sums of their sums: a wave to a head, the loads
  // of all its heads in flight
  constexpr int PL = kParts / 64, HW = RT;  // heads of a wave
  float mi[HW][PL], li[HW][PL];
#pragma unroll
  for (int k = 0; k < PL; ++k)
    if (64 * k < parts)
#pragma unroll
      for (int w = 0; w < HW; ++w) {
        const uint32_t at = min(lane + 64 * k, parts - 1) * step + at_ml + 8u * min(wv + AW * w, nq - 1);
        const uint2 u = coh_ld8(all, at);
        mi[w][k] = __uint_as_float(u.x), li[w][k] = __uint_as_float(u.y);
      }
  for (int w = 0; w < HW; ++w) {
    const int h = wv + AW * w;
    if (h >= nq) break;
    float mm = -INFINITY, ll = 0.f;
#pragma unroll
    for (int k = 0; k < PL; ++k)
      if (64 * k < parts) mm = fmaxf(mm, mi[w][k]);
    const float ref = score_ref(wave_max(mm));
#pragma unroll
    for (int k = 0; k < PL; ++k)
      if (64 * k < parts) {
        const float c = lane + 64 * k < parts ? __builtin_amdgcn_exp2f((mi[w][k] - ref) * LOG2E) : 0.f;
        ll += c * (lane + 64 * k < parts ? li[w][k] : 0.f);
        lds[h * kParts + lane + 64 * k] = c;
      }
    ll = wave_sum(ll);
    if (lane == 0) lds[16 * kParts + h] = ll;
  }
  __syncthreads();
  for (int x = threadIdx.x; x < items; x += 64 * AW) {
    const int h = x / (HD / 4);
    v4f oo = {0.f, 0.f, 0.f, 0.f};
    for (int i0 = 0; i0 < parts; i0 += JB) {
      if (i0 > 0 || x >= 64 * AW) load_sums(x, i0);
#pragma unroll
      for (int k = 0; k < JB; ++k)
        if (i0 + k < parts) {
          const float c = lds[h * kParts + i0 + k];
          oo[0] += c * v[k].x, oo[1] += c * v[k].y, oo[2] += c * v[k].z, oo[3] += c * v[k].w;
        }
    }
    const float ll = lds[16 * kParts + h];
    float *to = A.out + ((size_t)row * A.n_heads + h0) * HD + 4 * x;
#pragma unroll
    for (int k = 0; k < 4; ++k) to[k] = n == 0 && !bad ? 0.f : oo[k] / ll;
  }
  if (threadIdx.x == 0) __hip_atomic_store(A.count + blockIdx.x, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
}

// ---------------------------------------------------------------- launch
template <class KV, int DC>
int attn_launch(const AttnArgs &A, dim3 grid, hipStream_t st) {
  constexpr int RT4 = Lay<KV, DC>::AQ > 8 ? 4 : 2;
  const auto pick = [&](auto stream, auto waves) {
    constexpr bool S = decltype(stream)::value;
    constexpr int W = decltype(waves)::value;
    const auto kern = A.heads <= 4   ? k_attn_paged<KV, DC, 1, S, W>
                      : A.heads <= 8 ? k_attn_paged<KV, DC, 2, S, W>
                                     : k_attn_paged<KV, DC, RT4, S, W>;
    hipLaunchKernelGGL(kern, grid, dim3(64 * W), 0, st, A);
  };
  // a wave to a unit: short rows, through the caches
  if (A.waves == 1) pick(std::false_type{}, std::integral_constant<int, 1>{});
  else if (A.stream) pick(std::true_type{}, std::integral_constant<int, 4>{});
  else pick(std::false_type{}, std::integral_constant<int, 4>{});
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
