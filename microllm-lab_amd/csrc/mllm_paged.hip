// mllm_paged.hip -- the operators of a batched decode step that touch the
// pages of a key-value cache (include/mllm.h): mllm_rope_kv_paged writes new
// tokens' keys and values, mllm_attn_paged attends to them.  All pointers are
// device pointers.
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

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
constexpr int AQ = 16;                 // query heads of a workgroup
constexpr float LOG2E = 1.44269504088896340736f;

struct AttnArgs {
  Pages P;
  const float *q;
  const int32_t *seq, *len;
  float *out, *part;  // part: [rows][n_heads][splits][hd + 2], the sums, then maximum and sum
  int n_heads, rep, tiles, max_len, chunk, splits;
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
    if (N & 2) {
      const u2 v = *reinterpret_cast<const u2 *>(s + (N & ~3));
      d[N & ~3] = v.x, d[(N & ~3) + 1] = v.y;
    }
    if (N & 1) d[N - 1] = s[N - 1];
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < N; ++i) d[i] = 0u;
  }
  __device__ __forceinline__ float get(int e) const;
};
template <class KV, int E>
__device__ __forceinline__ float Raw<KV, E>::get(int e) const {
  if constexpr (sizeof(typename KV::T) == 4) return __uint_as_float(d[e]);
  else if constexpr (__is_same(KV, KvBf16)) return __uint_as_float(e & 1 ? d[e >> 1] & 0xffff0000u : d[e >> 1] << 16);
  else return __half2float(__ushort_as_half((uint16_t)(e & 1 ? d[e >> 1] >> 16 : d[e >> 1] & 0xffffu)));
}

__device__ __forceinline__ v4f mma(float a, float b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// One row's attention to `chunk` positions of one KV head, for up to 16 of the
// query heads that share it.  Waves take the positions in turns of 16 * PT, each
// with its own running maximum m and sum l:
//   S = K Q^T  on the float32 matrix cores: A = 16 positions (lane r + 16 g:
//              position r, the elements of its 16-byte runs g, g + 4, ...),
//              B = the query heads.  Lane j + 16 g then holds head j's scores of
//              the positions 4 g .. 4 g + 3,
//   O += P V   which is the layout of the A operand of the second product, one
//              position of each group of four a step; B = the values, lane c +
//              16 g the elements c hd / 16 ... of its position.
// Products and sums are float32, as the plain formula's, so an infinite key or
// value acts as it does there.
template <class KV, int DC, int PT>
__global__ __launch_bounds__(64 * AW) void k_attn_paged(AttnArgs A) {
  constexpr int HD = 32 * DC, EL = HD / 16, RUN = 16 / (int)sizeof(typename KV::T), NR = HD / (4 * RUN);
  using T = typename KV::T;
  extern __shared__ __attribute__((aligned(16))) float lds[];  // pages, then [AW][heads][HD] sums, [AW][2][16]
  int unit = blockIdx.x;
  const int tile = unit % A.tiles;
  unit /= A.tiles;
  const int kvh = unit % A.P.n_kv, row = unit / A.P.n_kv;
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, j = lane & 15, g = lane >> 4;
  const int h0 = kvh * A.rep + tile * AQ, nq = min(AQ, A.rep - tile * AQ);
  int seq;
  int n = row_len(A, row, seq);
  if (n == -1) return;
  const bool impossible = n < 0;
  if (impossible) n = 0;
  const int p0 = blockIdx.y * A.chunk, p1 = min(n, p0 + A.chunk);
  if (blockIdx.y > 0 && p0 >= n) return;
  // the chunk's pages
  int *pg = reinterpret_cast<int *>(lds);
  const int c0 = page_of(A.P, p0), nc = p1 > p0 ? page_of(A.P, p1 - 1) - c0 + 1 : 0;
  bool bad = impossible;
  for (int i = threadIdx.x; i < nc; i += 64 * AW) {
    const int page = A.P.table[(size_t)seq * A.P.table_cols + c0 + i];
    const bool ok = page >= 0 && page < A.P.pages;
    bad |= !ok;
    pg[i] = ok ? page : 0;
  }
  bad = __syncthreads_or(bad);
  // the queries
  float q[NR * RUN];
#pragma unroll
  for (int i = 0; i < NR; ++i)
#pragma unroll
    for (int e = 0; e < RUN; ++e)
      q[i * RUN + e] = j < nq ? A.q[((size_t)row * A.n_heads + h0 + j) * HD + (g + 4 * i) * RUN + e] : 0.f;
  const T *kb = static_cast<const T *>(A.P.k) + kvh * A.P.head_stride;
  const T *vb = static_cast<const T *>(A.P.v) + kvh * A.P.head_stride;
  auto at = [&](int pos) {
    const int c = page_of(A.P, pos);
    return pg[c - c0] * A.P.page_stride + (pos - c * A.P.page_size) * A.P.row_stride;
  };
  float m = -INFINITY, l = 0.f;
  v4f o[EL];
#pragma unroll
  for (int i = 0; i < EL; ++i) o[i] = v4f{0.f, 0.f, 0.f, 0.f};
  for (int t0 = p0 + wv * 16 * PT; t0 < p1; t0 += AW * 16 * PT) {
    Raw<KV, RUN> kr[PT][NR];
    Raw<KV, EL> vr[PT][4];
#pragma unroll
    for (int t = 0; t < PT; ++t) {
      const T *k = kb + at(min(t0 + 16 * t + j, p1 - 1)) + g * RUN;
#pragma unroll
      for (int i = 0; i < NR; ++i) kr[t][i].load(k + 4 * i * RUN);
    }
#pragma unroll
    for (int t = 0; t < PT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int pos = t0 + 16 * t + 4 * g + i;
        vr[t][i].load(vb + at(min(pos, p1 - 1)) + j * EL);
        if (pos >= p1) vr[t][i].clear();
      }
    v4f s[PT];
    float mx = -INFINITY;
#pragma unroll
    for (int t = 0; t < PT; ++t) {
      s[t] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < NR; ++i)
#pragma unroll
        for (int e = 0; e < RUN; ++e) s[t] = mma(kr[t][i].get(e), q[i * RUN + e], s[t]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[t][i] = j < nq && t0 + 16 * t + 4 * g + i < p1 ? s[t][i] * A.scale : -INFINITY;
        mx = fmaxf(mx, s[t][i]);
      }
    }
    mx = fmaxf(mx, __shfl_xor(mx, 16));
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    const float mn = fmaxf(m, mx), ref = score_ref(mn);
    if (__any(mn > m)) {
      const float corr = exp2f((m - ref) * LOG2E);
      l *= corr;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float c = __shfl(corr, 4 * g + i);
#pragma unroll
        for (int d = 0; d < EL; ++d) o[d][i] *= c;
      }
      m = mn;
    }
#pragma unroll
    for (int t = 0; t < PT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p = exp2f((s[t][i] - ref) * LOG2E);
        l += p;
#pragma unroll
        for (int d = 0; d < EL; ++d) o[d] = mma(p, vr[t][i].get(d), o[d]);
      }
  }
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  // the waves' parts
  __syncthreads();
  float *sums = lds, *ml = lds + AW * nq * HD;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (4 * g + i < nq)
#pragma unroll
      for (int d = 0; d < EL; ++d) sums[(wv * nq + 4 * g + i) * HD + j * EL + d] = o[d][i];
  if (g == 0) ml[wv * 32 + j] = m, ml[wv * 32 + 16 + j] = l;
  __syncthreads();
  for (int e = threadIdx.x; e < nq * HD; e += 64 * AW) {
    const int h = e / HD, d = e - h * HD;
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < AW; ++w) mm = fmaxf(mm, ml[w * 32 + h]);
    const float ref = score_ref(mm);
    float ll = 0.f, oo = 0.f;
#pragma unroll
    for (int w = 0; w < AW; ++w) {
      const float c = exp2f((ml[w * 32 + h] - ref) * LOG2E);
      ll += c * ml[w * 32 + 16 + h];
      oo += c * sums[(w * nq + h) * HD + d];
    }
    if (bad) ll = oo = __builtin_nanf("");
    const size_t at_row = (size_t)row * A.n_heads + h0 + h;
    if (A.splits == 1) {
      A.out[at_row * HD + d] = n == 0 && !bad ? 0.f : oo / ll;
    } else {
      float *p = A.part + (at_row * A.splits + blockIdx.y) * (HD + 2);
      p[d] = oo;
      if (d == 0) p[HD] = mm, p[HD + 1] = ll;
    }
  }
}

// The parts of a row's head, joined: a wave to each.
__global__ __launch_bounds__(64) void k_attn_join(AttnArgs A) {
  __shared__ float w[64];
  const int row = blockIdx.x / A.n_heads, lane = threadIdx.x, HD = A.P.hd;
  int seq;
  const int n = row_len(A, row, seq);
  if (n == -1) return;
  const int parts = n <= 0 ? 1 : (n + A.chunk - 1) / A.chunk;
  const float *p = A.part + (size_t)blockIdx.x * A.splits * (HD + 2);
  float mm = -INFINITY;
  for (int i = lane; i < parts; i += 64) mm = fmaxf(mm, p[(size_t)i * (HD + 2) + HD]);
  const float ref = score_ref(wave_max(mm));
  float ll = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int i0 = 0; i0 < parts; i0 += 64) {
    float c = 0.f;
    if (i0 + lane < parts) {
      const float *pi = p + (size_t)(i0 + lane) * (HD + 2) + HD;
      c = exp2f((pi[0] - ref) * LOG2E);
      ll += c * pi[1];
    }
    __syncthreads();
    w[lane] = c;
    __syncthreads();
    const int ni = min(64, parts - i0);
    for (int i = 0; i < ni; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (lane + 64 * k < HD) o[k] += w[i] * p[(size_t)(i0 + i) * (HD + 2) + lane + 64 * k];
  }
  ll = wave_sum(ll);
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (lane + 64 * k < HD) A.out[(size_t)blockIdx.x * HD + lane + 64 * k] = n == 0 ? 0.f : o[k] / ll;
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
// positions.
constexpr int kUnits = 1024;  // workgroups that fill the chip: four on each of the 256 CUs
void attn_plan(int units, int max_len, int *chunk, int *splits) {
  const int most = (max_len + 255) / 256;
  int s = (kUnits + units - 1) / units;
  s = s < 1 ? 1 : s > most ? most : s;
  int c = (max_len + s - 1) / s;
  c = (c + 63) / 64 * 64;
  if (c > 4096) c = 4096;
  if (c < 64) c = 64;
  *chunk = c;
  *splits = max_len > 0 ? (max_len + c - 1) / c : 1;
}

struct AttnPlan {
  int rep, tiles, chunk, splits;
  uint64_t bytes;  // of the workspace
};

int attn_shape(const Pages &P, int rows, int n_heads, int max_len, AttnPlan *pl) {
  MLLM_CHECK(rows > 0 && n_heads > 0 && n_heads % P.n_kv == 0, "invalid shape rows=%d n_heads=%d over %d KV heads", rows,
             n_heads, P.n_kv);
  MLLM_CHECK(max_len >= 0 && max_len <= (int64_t)P.page_size * P.table_cols,
             "max_len=%d beyond the %d pages of %d positions of a sequence", max_len, P.table_cols, P.page_size);
  pl->rep = n_heads / P.n_kv;
  pl->tiles = (pl->rep + AQ - 1) / AQ;
  const int64_t units = (int64_t)rows * P.n_kv * pl->tiles;
  MLLM_CHECK(units < (1ll << 31) && (int64_t)rows * n_heads < (1ll << 31), "%d rows of %d heads exceed a launch", rows,
             n_heads);
  attn_plan((int)units, max_len, &pl->chunk, &pl->splits);
  MLLM_CHECK(pl->splits <= 65535, "max_len=%d exceeds a launch", max_len);
  pl->bytes = pl->splits > 1 ? (uint64_t)rows * n_heads * pl->splits * (P.hd + 2) * sizeof(float) : 0;
  return 0;
}

template <class KV, int DC>
int attn_launch(const AttnArgs &A, dim3 grid, size_t lds, hipStream_t st) {
  // positions a wave has in flight: 64, fewer where their registers would not
  // leave two waves to a SIMD
  constexpr int row_bytes = 32 * DC * (int)sizeof(typename KV::T), PT = row_bytes <= 128 ? 4 : row_bytes <= 256 ? 2 : 1;
  const auto kern = k_attn_paged<KV, DC, PT>;
  if (lds > 64 * 1024)
    MLLM_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(kern), hipFuncAttributeMaxDynamicSharedMemorySize,
                                 (int)lds));
  hipLaunchKernelGGL(kern, grid, dim3(64 * AW), lds, st, A);
  MLLM_HIP(hipGetLastError());
  return 0;
}

template <class KV>
int attn_dispatch(const AttnArgs &A, dim3 grid, size_t lds, hipStream_t st) {
  switch (A.P.hd / 32) {
  case 1: return attn_launch<KV, 1>(A, grid, lds, st);
  case 2: return attn_launch<KV, 2>(A, grid, lds, st);
  case 3: return attn_launch<KV, 3>(A, grid, lds, st);
  case 4: return attn_launch<KV, 4>(A, grid, lds, st);
  case 5: return attn_launch<KV, 5>(A, grid, lds, st);
  case 6: return attn_launch<KV, 6>(A, grid, lds, st);
  case 7: return attn_launch<KV, 7>(A, grid, lds, st);
  default: return attn_launch<KV, 8>(A, grid, lds, st);
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
  if (check_pages(kv, &P) || attn_shape(P, rows, n_heads, max_len, &pl)) return 0;
  return pl.bytes;
}

extern "C" int mllm_attn_paged(const mllm_kv_pages *kv, int rows, int n_heads, const float *q, const int32_t *seq,
                               const int32_t *len, int max_len, float scale, float *out, void *workspace,
                               uint64_t workspace_bytes, void *stream) {
  AttnArgs A{};
  AttnPlan pl;
  if (int rc = check_pages(kv, &A.P)) return rc;
  if (int rc = attn_shape(A.P, rows, n_heads, max_len, &pl)) return rc;
  MLLM_CHECK(q && len && out, "null pointer");
  MLLM_CHECK(seq || rows <= A.P.sequences, "%d rows without seq, %d sequences", rows, A.P.sequences);
  MLLM_CHECK(pl.bytes == 0 || workspace, "null workspace, %llu bytes needed", (unsigned long long)pl.bytes);
  MLLM_CHECK(workspace_bytes >= pl.bytes, "workspace of %llu bytes, %llu needed", (unsigned long long)workspace_bytes,
             (unsigned long long)pl.bytes);
  MLLM_CHECK(pl.bytes == 0 || ((uintptr_t)workspace & 15) == 0, "the workspace must be 16-byte aligned");
  A.q = q, A.seq = seq, A.len = len, A.out = out, A.part = static_cast<float *>(workspace);
  A.n_heads = n_heads, A.rep = pl.rep, A.tiles = pl.tiles, A.max_len = max_len;
  A.chunk = pl.chunk, A.splits = pl.splits, A.scale = scale;
  const dim3 grid((unsigned)(rows * A.P.n_kv * pl.tiles), (unsigned)pl.splits);
  const int nq = pl.rep < AQ ? pl.rep : AQ;
  const size_t pages = ((size_t)pl.chunk / kv->page_size + 2) * sizeof(int);
  const size_t sums = ((size_t)AW * nq * A.P.hd + AW * 32) * sizeof(float);
  const size_t lds = pages > sums ? pages : sums;
  hipStream_t st = as_stream(stream);
  const int rc = kv->storage == MLLM_F32   ? attn_dispatch<KvF32>(A, grid, lds, st)
                 : kv->storage == MLLM_F16 ? attn_dispatch<KvF16>(A, grid, lds, st)
                                           : attn_dispatch<KvBf16>(A, grid, lds, st);
  if (rc || pl.splits == 1) return rc;
  hipLaunchKernelGGL(k_attn_join, dim3((unsigned)(rows * n_heads)), dim3(64), 0, st, A);
  MLLM_HIP(hipGetLastError());
  return 0;
}
