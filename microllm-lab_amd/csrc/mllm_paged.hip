// mllm_paged.hip -- the operators of a batched decode step that touch the
// pages of a key-value cache (include/mllm.h): mllm_rope_kv_paged writes new
// tokens' keys and values, mllm_attn_paged attends to them (its kernels:
// mllm_paged_attn.h).  All pointers are device pointers.
#include "mllm_device.h"
#include "mllm_host.h"
#include "mllm_paged.h"

using namespace mllm;
using namespace mllm::paged;

namespace {

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

// Positions per workgroup (turns of the four waves) and the number of parts for
// rows of up to max_len positions.  A CU reads at most about 28 GB/s, whatever
// the number of its workgroups, and the chip 6.2 TB/s: the time goes by the
// bytes of the CU that has most, a workgroup's start and end (about 64 KB of
// reading) and a join (96 KB).  Measured, us: 2 rows of 100000 positions, 16
// units, 8 / 12 / 16 / 20 / 24 / 32 parts 239 / 174 / 143 / 199 / 168 / 152; 320
// units of 6144 positions, 1 / 2 / 3 / 4 / 6 parts 111 / 98 / 89 / 88 / 99; 100
// units of 4000, 2 / 3 / 4 / 8 parts 23 / 27 / 24 / 28.
constexpr int64_t kMallBytes = 256 << 20;  // the Infinity Cache
constexpr int64_t kCus = 256, kStart = 64 << 10, kJoinCost = 96 << 10;
void attn_plan(int64_t units, int max_len, int64_t pos_bytes, int *chunk, int *splits) {
  int64_t best = 0;
  *chunk = 0;
  for (int64_t s = 1; s <= kParts; ++s) {
    int64_t c = ((max_len + s - 1) / s + 255) / 256 * 256;
    c = c < 256 ? 256 : c > 0x7fffff00 ? 0x7fffff00 : c;
    const int64_t parts = max_len > c ? (max_len + c - 1) / c : 1;
    const int64_t cost = (units * parts + kCus - 1) / kCus * (c * pos_bytes + kStart) + (parts > 1 ? kJoinCost : 0);
    if (*chunk == 0 || cost < best) best = cost, *chunk = (int)c, *splits = (int)parts;
    if (units > kCounters || c == 256) break;
  }
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
  int64_t units, pos_bytes;  // pos_bytes: a head's key and value
  uint64_t bytes;            // of the workspace: the counters, then the parts
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
  pl->pos_bytes = 2 * P.hd * (kv->storage == MLLM_F32 ? 4 : 2);
  MLLM_CHECK(pl->units < (1ll << 31) && (int64_t)rows * n_heads < (1ll << 31), "%d rows of %d heads exceed a launch", rows,
             n_heads);
  attn_plan(pl->units, max_len, pl->pos_bytes, &pl->chunk, &pl->splits);
  pl->bytes = pl->splits > 1 ? kCounters * sizeof(unsigned) +
                                   (uint64_t)pl->units * pl->splits * (((uint64_t)pl->heads * (P.hd + 2) + 3) & ~3ull) * sizeof(float)
                             : 0;
  return 0;
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
  MLLM_CHECK(((uintptr_t)q & 15) == 0, "q must be 16-byte aligned");
  MLLM_CHECK(seq || rows <= A.P.sequences, "%d rows without seq, %d sequences", rows, A.P.sequences);
  MLLM_CHECK(pl.bytes == 0 || workspace, "null workspace, %llu bytes needed", (unsigned long long)pl.bytes);
  MLLM_CHECK(workspace_bytes >= pl.bytes, "workspace of %llu bytes, %llu needed", (unsigned long long)workspace_bytes,
             (unsigned long long)pl.bytes);
  MLLM_CHECK(pl.bytes == 0 || ((uintptr_t)workspace & 15) == 0, "the workspace must be 16-byte aligned");
  A.q = q, A.seq = seq, A.len = len, A.out = out;
  A.count = static_cast<unsigned *>(workspace);
  A.part = reinterpret_cast<float *>(A.count + kCounters);
  A.n_heads = n_heads, A.rep = pl.rep, A.tiles = pl.tiles, A.heads = pl.heads, A.max_len = max_len;
  A.chunk = pl.chunk, A.splits = pl.splits, A.scale = scale;
  // what the Infinity Cache cannot hold until the next call is read past the
  // caches (64 rows of 6144 positions, 503 MB: 95 to 88 us; 126 MB that it does
  // hold: 29 to 32)
  const int64_t positions = (int64_t)rows * max_len, pool = (int64_t)kv->pages * kv->page_size;
  A.stream = (positions < pool ? positions : pool) * A.P.n_kv * pl.pos_bytes > kMallBytes;
  const dim3 grid((unsigned)pl.units, (unsigned)pl.splits);
  hipStream_t st = as_stream(stream);
  return kv->storage == MLLM_F32   ? attn_f32(A, grid, st)
         : kv->storage == MLLM_F16 ? attn_f16(A, grid, st)
                                   : attn_bf16(A, grid, st);
}
