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
  int n_heads, rot, lg_lph;  // 2^lg_lph lanes per head
  int interleaved;
  float eps;
};

// A token's heads, lph lanes to each: lane s takes the same four pairs of every
// head that its group of lanes reaches, so that their angles are formed once.
// Pair p is rotated below rot / 2 -- elements (p, p + rot/2), or (2p, 2p + 1)
// interleaved.  VEC (rot a multiple of 8): a lane's elements are two runs of
// four, each side by side with the next lane's -- p = 4s .. 4s + 3 in halves,
// and 4s .., hd/2 + 4s .. of what is interleaved or not rotated.  Otherwise a
// lane's pairs are 4s .. 4s + 3, element by element.
//
// What bounds it: the bytes, at the rate of a copy.  8000 tokens with 48 heads
// of 128 (360 MB), us: runs of eight elements a lane, which touch every cache
// line twice, 124; runs of four 75, three heads of a lane in flight 88, three
// times the threads 98; loads and stores past the caches, whose readers sit
// behind another L2, 70 (5.2 TB/s; a copy of the same bytes takes 72).  Element
// by element, 60 of the 128 rotated: 222.
//
// The angle is formed in double and in turns: a position of 2^20 keeps 2^-33
// of a turn, where a float product would keep 2^-4.  What is left of it within
// half a turn is taken as two floats, hi + lo: the functions of hi, and their
// slopes times lo (at most 2^-25 of half a turn; its square is below 2^-47).
template <class KV, bool VEC>
__global__ __launch_bounds__(WG) void k_rope_kv(RopeArgs A) {
  const int token = blockIdx.x, lph = 1 << A.lg_lph, s = threadIdx.x & (lph - 1);
  const int nh = A.n_heads, nkv = A.P.n_kv, hd = A.P.hd, rows = nh + 2 * nkv, step = (int)blockDim.x >> A.lg_lph;
  const float *row = A.qkv + (size_t)token * rows * hd;
  const bool in = 8 * s < hd;
  const int half = A.rot >> 1;
  // the lane's pair j, where it is rotated (2 pair < rot)
  auto pair = [&](int j) { return VEC && A.interleaved ? (j < 2 ? 2 * s + j : (hd >> 2) + 2 * s + j - 2) : 4 * s + j; };
  // r: a head of the queries or keys.  Element e of pair j, without runs
  auto at1 = [&](bool r, int j, int e) {
    const int p = 4 * s + j;
    return r && 2 * p < A.rot && !A.interleaved ? p + e * half : 2 * p + e;
  };
  // the runs: halves of the rotated part, or of what passes through behind it
  auto halves = [&](bool r) { return r && !A.interleaved && 8 * s < A.rot; };
  auto run0 = [&](bool r) { return r && !A.interleaved && 8 * s >= A.rot ? 4 * s + half : 4 * s; };
  auto run1 = [&](bool r) {
    return !r || A.interleaved ? (hd >> 1) + 4 * s : 8 * s < A.rot ? half + 4 * s : (hd >> 1) + 4 * s;
  };
  auto at = [&](bool r, int j, int e) {
    if (!VEC) return at1(r, j, e);
    if (halves(r)) return e ? run1(r) + j : run0(r) + j;
    return (j < 2 ? run0(r) : run1(r)) + 2 * (j & 1) + e;
  };
  float a[4], b[4];  // the pairs' elements
  auto load = [&](int head, float (&u)[4], float (&w)[4]) {
    const bool r = head < nh + nkv;
    const float *x = row + (size_t)head * hd;
#pragma unroll
    for (int j = 0; j < 4; ++j) u[j] = w[j] = 0.f;
    if (!in || head >= rows) return;
    if (VEC) {
      const v4f f = __builtin_nontemporal_load(reinterpret_cast<const v4f *>(x + run0(r)));
      const v4f g = __builtin_nontemporal_load(reinterpret_cast<const v4f *>(x + run1(r)));
      const bool h = halves(r);
      u[0] = f.x, u[1] = h ? f.y : f.z, u[2] = h ? f.z : g.x, u[3] = h ? f.w : g.z;
      w[0] = h ? g.x : f.y, w[1] = h ? g.y : f.w, w[2] = h ? g.z : g.y, w[3] = g.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) u[j] = x[at1(r, j, 0)], w[j] = x[at1(r, j, 1)];
    }
  };
  const int first = threadIdx.x >> A.lg_lph;
  load(first, a, b);
  const int seq = A.seq ? A.seq[token] : token, pos = A.pos[token];
  if (seq < 0 || seq >= A.P.sequences || pos < 0) return;  // padding
  // the slot, if there is one
  const int col = page_of(A.P, pos), slot = pos - col * A.P.page_size;
  int page = -1;
  if (col < A.P.table_cols) page = A.P.table[(size_t)seq * A.P.table_cols + col];
  const bool placed = page >= 0 && page < A.P.pages;
  const int64_t place = placed ? page * A.P.page_stride + slot * A.P.row_stride : 0;
  float sn[4], cs[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    sn[j] = 0.f, cs[j] = 1.f;
    if (in && 2 * pair(j) < A.rot) {
      const double t = (double)pos * ((double)A.inv_freq[pair(j)] * 0.15915494309189533577);  // turns
      const double x = 2.0 * (t - rint(t));
      const float hi = (float)x, lo = (float)(x - (double)hi) * 3.14159265f;
      float sh, ch;
      sincospif(hi, &sh, &ch);
      sn[j] = __builtin_fmaf(ch, lo, sh), cs[j] = __builtin_fmaf(-sh, lo, ch);
    }
  }
  auto store = [&](bool r, const float (&u)[4], const float (&w)[4], auto *to, auto put) {
    using T = decltype(put(0.f));
    if (VEC) {
      typedef T v4 __attribute__((ext_vector_type(4)));
      const bool h = halves(r);
      const float f[8] = {u[0], h ? u[1] : w[0], h ? u[2] : u[1], h ? u[3] : w[1],
                          h ? w[0] : u[2], h ? w[1] : w[2], h ? w[2] : u[3], w[3]};
      __builtin_nontemporal_store(v4{put(f[0]), put(f[1]), put(f[2]), put(f[3])}, reinterpret_cast<v4 *>(to + run0(r)));
      __builtin_nontemporal_store(v4{put(f[4]), put(f[5]), put(f[6]), put(f[7])}, reinterpret_cast<v4 *>(to + run1(r)));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) to[at1(r, j, 0)] = put(u[j]), to[at1(r, j, 1)] = put(w[j]);
    }
  };
  for (int head = first; head < rows; head += step) {
    if (head != first) load(head, a, b);
    const bool r = head < nh + nkv;
    const float *gain = head < nh ? A.q_gain : r ? A.k_gain : nullptr;
    if (gain) {
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) ss = __builtin_fmaf(a[j], a[j], __builtin_fmaf(b[j], b[j], ss));
      for (int m = 1; m < lph; m <<= 1) ss += __shfl_xor(ss, m);
      const float inv = 1.0f / sqrtf(ss / (float)hd + A.eps);
      if (in)
#pragma unroll
        for (int j = 0; j < 4; ++j) a[j] = a[j] * inv * gain[at(r, j, 0)], b[j] = b[j] * inv * gain[at(r, j, 1)];
    }
    if (!in) continue;
    if (r)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (2 * pair(j) < A.rot) {
          const float u = a[j], w = b[j];
          a[j] = u * cs[j] - w * sn[j];
          b[j] = w * cs[j] + u * sn[j];
        }
    if (head < nh) {
      store(r, a, b, A.q + ((size_t)token * nh + head) * hd, KvF32::put);
    } else if (placed) {
      typename KV::T *pool = static_cast<typename KV::T *>(r ? A.P.k : A.P.v);
      store(r, a, b, pool + place + (r ? head - nh : head - nh - nkv) * A.P.head_stride, KV::put);
    }
  }
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
  // the kernels step past a position in 32 bits
  MLLM_CHECK((int64_t)kv->page_size * kv->table_cols <= (1ll << 30), "%d pages of %d positions a sequence exceed 2^30",
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

constexpr int64_t kMallBytes = 256 << 20;  // the Infinity Cache

// Positions per workgroup (turns of the four waves) and the number of parts for
// rows of up to max_len positions.  With this kernel's loads a CU comes to about
// 28 GB/s, with one workgroup or more, and the chip to 6.2 TB/s: the time goes by
// the bytes of the CU that has most, a workgroup's start and end (about 64 KB of
// reading) and a join (96 KB).  Measured, us: 2 rows of 100000 positions, 16
// units, 8 / 12 / 16 / 20 / 24 / 32 parts 239 / 174 / 143 / 199 / 168 / 152; 320
// units of 6144 positions, 1 / 2 / 3 / 4 / 6 parts 111 / 98 / 89 / 88 / 99; 100
// units of 4000, 2 / 3 / 4 / 8 parts 23 / 27 / 24 / 28.
// A part is a multiple of kChunk positions: one row of 700 positions in float32
// (3 units), parts of 64 / 128 / 256 positions 8.0 / 8.1 / 9.1 us; five rows of
// 516 in f16 9.7 / 9.1 / 9.2.
// At most kCounters workgroups where rows are split: a workspace for many rows
// and long ones serves fewer and shorter.
// Many short rows (more than two units to a CU, of at most kShort bytes each)
// take a wave to a unit, so that eight of them are at their starts and ends at
// once.  Two is what a CU holds of the workgroups of four waves measured here;
// by its registers a form has one to four (f32 heads of 64 four, f32 and bf16
// heads of 256 with more than four query heads one), where it was not measured.
// Four waves / one, us: 640 units of 64 f16 elements, 16 / 128 / 512 / 1024
// positions 10.6 / 9.0, 12.0 / 9.1, 20.2 / 17.6, 36.1 / 35.3; 320 units 8.7 /
// 8.7, 8.8 / 8.7, 13.4 / 16.6, 20.3 / 28.3; 2560 units 28.6 / 11.7, 32.9 / 19.3,
// 65.8 / 66.5, 110 / 126; 2048 units of 128 bf16 elements, 25 / 128 / 256 / 512
// positions 24.7 / 11.7, 35.5 / 25.5, 61.4 / 52.2, 91.0 / 95.4.
constexpr int64_t kShort = 128 << 10;
constexpr int64_t kChunk = 128, kCus = 256, kStart = 64 << 10, kJoinCost = 96 << 10;
void attn_plan(int64_t units, int max_len, int64_t pos_bytes, int *waves, int *chunk, int *splits) {
  int64_t best = 0;
  *waves = units > 2 * kCus && max_len * pos_bytes <= kShort ? 1 : 4;
  *chunk = 0;
  for (int64_t s = 1; s <= kParts; ++s) {
    int64_t c = ((max_len + s - 1) / s + kChunk - 1) / kChunk * kChunk;
    c = c < kChunk ? kChunk : c;
    const int64_t parts = max_len > c ? (max_len + c - 1) / c : 1;
    const int64_t cost = (units * parts + kCus - 1) / kCus * ((c < max_len ? c : max_len) * pos_bytes + kStart) +
                         (parts > 1 ? kJoinCost : 0);
    if (*chunk == 0 || cost < best) best = cost, *chunk = (int)c, *splits = (int)parts;
    if (*waves == 1 || units * (s + 1) > kCounters || c == kChunk) break;
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
  int rep, tiles, heads, waves, chunk, splits;
  int64_t units, pos_bytes;  // pos_bytes: a head's key and value
  uint64_t part_bytes;
  // of a workspace: the counters, then the parts
  uint64_t bytes(int64_t parts) const { return kCounters * sizeof(unsigned) + (uint64_t)parts * part_bytes; }
  uint64_t need() const { return splits > 1 ? bytes(units * splits) : 0; }
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
  MLLM_CHECK(pl->units < (1ll << 32) / 256, "%d rows of %d heads exceed a launch", rows, n_heads);
  attn_plan(pl->units, max_len, pl->pos_bytes, &pl->waves, &pl->chunk, &pl->splits);
  pl->part_bytes = (((uint64_t)pl->heads * (P.hd + 2) + 3) & ~3ull) * sizeof(float);
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
  A.lg_lph = 2;
  while (8 << A.lg_lph < A.P.hd) ++A.lg_lph;
  const int64_t heads = (int64_t)n_heads + 2 * (int64_t)A.P.n_kv;
  MLLM_CHECK(heads < (1 << 20), "%lld heads", (long long)heads);
  const int threads = heads << A.lg_lph < WG ? (int)(heads << A.lg_lph) : WG;  // whole waves
  const dim3 grid((unsigned)tokens), block((unsigned)((threads + 63) & ~63));
  MLLM_CHECK((uint64_t)tokens * block.x < (1ull << 32), "%d tokens of %lld heads exceed a launch", tokens,
             (long long)heads);
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
  // parts of no plan for as many rows or fewer and as long or shorter exceed these
  const int64_t longest = ((int64_t)max_len + kChunk - 1) / kChunk, splits = longest < kParts ? longest : kParts;
  return splits > 1 ? pl.bytes(pl.units * splits < kCounters ? pl.units * splits : kCounters) : 0;
}

extern "C" int mllm_attn_paged(const mllm_kv_pages *kv, int rows, int n_heads, const float *q, const int32_t *seq,
                               const int32_t *len, int max_len, float scale, float *out, void *workspace,
                               uint64_t workspace_bytes, void *stream) {
  AttnArgs A{};
  AttnPlan pl;
  if (int rc = check_pages(kv, &A.P)) return rc;
  if (int rc = attn_shape(kv, A.P, rows, n_heads, max_len, &pl)) return rc;
  MLLM_CHECK(seq || rows <= A.P.sequences, "%d rows without seq, %d sequences", rows, A.P.sequences);
  const uint64_t need = pl.need();
  MLLM_CHECK(need == 0 || workspace, "null workspace, %llu bytes needed", (unsigned long long)need);
  MLLM_CHECK(workspace_bytes >= need, "workspace of %llu bytes, %llu needed", (unsigned long long)workspace_bytes,
             (unsigned long long)need);
  MLLM_CHECK(need == 0 || ((uintptr_t)workspace & 15) == 0, "the workspace must be 16-byte aligned");
  MLLM_CHECK(q && len && out, "null pointer");
  MLLM_CHECK(((uintptr_t)q & 15) == 0, "q must be 16-byte aligned");
  A.q = q, A.seq = seq, A.len = len, A.out = out;
  A.count = static_cast<unsigned *>(workspace);
  A.part = reinterpret_cast<float *>(A.count + kCounters);
  A.n_heads = n_heads, A.rep = pl.rep, A.tiles = pl.tiles, A.heads = pl.heads, A.max_len = max_len;
  A.chunk = pl.chunk, A.splits = pl.splits, A.scale = scale;
  A.waves = pl.waves;
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
