// Attention of drafted tokens over a paged cache: row b's n tokens lie at the end of its
// context, and token j sees the context before them and those of them that its mask names.
//
//   out_j = softmax(scale q_j K^T) V over the tokens t < c and the c + k with bit k of mask_j,
//   c = seq_len - n
#include "attn_tile.hpp"

#include <float.h>
#include <math.h>

namespace cir {
namespace {

constexpr int kMaxDrafts = 256;  // tokens of a row

struct Args {
  const int32_t *table, *lens, *offsets, *counts;
  const uint32_t* masks;  // [tokens][2 words]: bit k % 32 of word k / 32
  float *part_o, *part_ml;
  int tokens, batch, Hq, Hkv, D, P, max_pages, words, splits;
  float scale_log2;
};

__device__ __forceinline__ int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }

// A row's first token, their number, where they begin in its context, and what is stored of it; inside the step's
// tokens and the table whatever the device's numbers are.
struct Row {
  int first, n, context, limit;
};
__device__ __forceinline__ Row row_of(const Args& A, int b) {
  const int o = A.offsets[b], e = A.offsets[b + 1], c = A.counts[b], len = A.lens[b];
  Row r;
  r.first = min(max(o, 0), A.tokens);
  r.n = max(0, min(min(c, 64 * A.words), min(e, A.tokens) - r.first));
  r.context = max(0, len - r.n);
  r.limit = max(0, min(len, A.max_pages * A.P));
  return r;
}
// Drafted tokens 32 w .. 32 w + 31 that token j sees.
__device__ __forceinline__ uint32_t mask_word(const Args& A, int j, int w, int n) {
  if (w < 0 || 32 * w >= n) return 0;
  const uint32_t m = A.masks[(size_t)j * 2 * A.words + w];
  return 32 * w + 32 > n ? m & ((1u << (n - 32 * w)) - 1) : m;
}
// The same for the 32 tokens of the context's axis from `token` on (those before the drafted ones count as seen).
__device__ __forceinline__ uint32_t seen_from(const Args& A, int j, int token, int context, int n) {
  const int k = token - context;
  if (k + 32 <= 0) return 0xffffffffu;
  const int w = k >> 5, s = k & 31;  // (floor)
  const uint32_t lo = k < 0 ? 0xffffffffu : mask_word(A, j, w, n), hi = s ? mask_word(A, j, w + 1, n) : 0;
  return s ? (lo >> s) | (hi << (32 - s)) : lo;
}

// Whether token j sees any token at all.
__device__ __forceinline__ bool sees(const Args& A, const Row& r, int j) {
  if (min(r.context, r.limit) > 0) return true;
  const int n = min(r.n, r.limit - r.context);
  uint32_t any = 0;
  for (int w = 0; 32 * w < n; ++w) any |= mask_word(A, j, w, n);
  return any != 0;
}

// -------------------------------------------------------------- any sizes -----
// fp32 arithmetic for any head_dim up to 256, type and page size.  A workgroup takes up to kVec query vectors of one row
// and KV head (a tile) over a stretch of the row's tokens, 64 at a time: K and V through LDS as fp32, a wavefront's
// lanes are tokens for the scores and dims for the sum over V, each wavefront with its own four vectors.
constexpr int kGenThreads = 256;
constexpr int kGenWaves = kGenThreads / 64;
constexpr int kPerWave = 4;
constexpr int kVec = kGenWaves * kPerWave;
constexpr int kTok = 64;
constexpr int kMaxD = 256;

__device__ __forceinline__ int tiles_of(const Args& A, int n) { return (n * (A.Hq / A.Hkv) + kVec - 1) / kVec; }

template <typename T, int DM>  // DM: head_dim at most
__global__ __launch_bounds__(kGenThreads) void tree_generic(const T* __restrict__ q, const T* __restrict__ kp,
                                                            const T* __restrict__ vp, T* __restrict__ out, Args A) {
  constexpr int ldk = DM + 4;
  __shared__ __align__(16) float sm_q[kVec * DM], sm_k[kTok * ldk], sm_v[kTok * DM];
  __shared__ int sm_sum[kGenWaves], sm_find[2];
  const int D = A.D, Dp = (D + 3) / 4 * 4;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int G = A.Hq / A.Hkv, h = blockIdx.y;

  // The row and tile of this workgroup: tiles are numbered row after row.
  if (t == 0) sm_find[0] = -1;
  int before = 0;
  for (int b0 = 0; b0 < A.batch; b0 += kGenThreads) {  // uniform
    const int b = b0 + t;
    const int mine = b < A.batch ? tiles_of(A, row_of(A, b).n) : 0;
    int upto = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int o = __shfl_up(upto, off, 64);
      upto += lane >= off ? o : 0;
    }
    if (lane == 63) sm_sum[wave] = upto;
    __syncthreads();
    int total = before;
#pragma unroll
    for (int w = 0; w < kGenWaves; ++w) {
      upto += w < wave ? sm_sum[w] : 0;
      total += sm_sum[w];
    }
    upto += before;
    const int id = blockIdx.x;
    if (id >= upto - mine && id < upto) {
      sm_find[0] = b;
      sm_find[1] = id - (upto - mine);
    }
    before = total;
    __syncthreads();
    if (before > id) break;  // uniform
  }
  __syncthreads();
  const int b = uni(sm_find[0]);
  if (b < 0) return;  // uniform: more workgroups than tiles
  const Row r = row_of(A, b);
  const int v0 = uni(sm_find[1]) * kVec, nv = min(kVec, r.n * G - v0);
  // This workgroup's stretch of the row's tokens.
  const int stretch = ((r.limit + A.splits - 1) / A.splits + kTok - 1) / kTok * kTok;
  const int k0 = min((int64_t)r.limit, (int64_t)blockIdx.z * stretch), k1 = min(r.limit, k0 + stretch);

  for (int i = t; i < kVec * Dp; i += kGenThreads) {
    const int v = i / Dp, d = i - v * Dp, vv = v0 + v;
    float x = 0.f;
    if (v < nv && d < D)
      x = to_f32(q[((size_t)(r.first + vv / G) * A.Hq + (size_t)h * G + vv % G) * D + d]) * A.scale_log2;
    sm_q[i] = x;
  }
  float m[kPerWave], l[kPerWave], acc[kPerWave][DM / 64];
  int row[kPerWave];
#pragma unroll
  for (int i = 0; i < kPerWave; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
    row[i] = r.first + min(v0 + wave * kPerWave + i, r.n * G - 1) / G;
#pragma unroll
    for (int c = 0; c < DM / 64; ++c) acc[i][c] = 0.f;
  }
  for (int k = k0; k < k1; k += kTok) {  // uniform
    const int nt = min(kTok, k1 - k);
    __syncthreads();
    for (int i = t; i < kTok * Dp; i += kGenThreads) {
      const int tok = i / Dp, d = i - tok * Dp;
      float x = 0.f, y = 0.f;
      if (tok < nt && d < D) {
        const int pos = k + tok, page = pos / A.P;
        const size_t at = (((size_t)A.table[(size_t)b * A.max_pages + page] * A.Hkv + h) * A.P + (pos - page * A.P)) * D + d;
        x = to_f32(kp[at]);
        y = to_f32(vp[at]);
      }
      sm_k[tok * ldk + d] = x;
      sm_v[tok * Dp + d] = y;
    }
    __syncthreads();
    float s[kPerWave];
#pragma unroll
    for (int i = 0; i < kPerWave; ++i) s[i] = 0.f;
    for (int d = 0; d < Dp; d += 4) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(sm_k + lane * ldk + d);
#pragma unroll
      for (int i = 0; i < kPerWave; ++i) {
        const f32x4 y = *reinterpret_cast<const f32x4*>(sm_q + (wave * kPerWave + i) * Dp + d);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[i] = fmaf(x[e], y[e], s[i]);
      }
    }
    const bool drafted = k + nt > r.context;  // uniform: some tokens that not every vector sees
    uint64_t seen[kPerWave];
#pragma unroll
    for (int i = 0; i < kPerWave; ++i) {
      seen[i] = nt < 64 ? (1ull << nt) - 1 : ~0ull;
      if (drafted)
        seen[i] &= seen_from(A, row[i], k, r.context, r.n) | (uint64_t)seen_from(A, row[i], k + 32, r.context, r.n) << 32;
      const bool mine = seen[i] >> lane & 1;
      const float x = mine ? s[i] : -INFINITY;
      const float mn = fmaxf(m[i], wave_max(x)), ms = mn == -INFINITY ? 0.f : mn;
      const float alpha = __builtin_amdgcn_exp2f(m[i] - ms);
      s[i] = mine ? __builtin_amdgcn_exp2f(s[i] - ms) : 0.f;
      l[i] = fmaf(l[i], alpha, wave_sum(s[i]));
      m[i] = mn;
#pragma unroll
      for (int c = 0; c < DM / 64; ++c) acc[i][c] *= alpha;
    }
    for (int tok = 0; tok < nt; ++tok) {
      float p[kPerWave];
#pragma unroll
      for (int i = 0; i < kPerWave; ++i) p[i] = __shfl(s[i], tok, 64);
#pragma unroll
      for (int c = 0; c < DM / 64; ++c) {
        const int d = lane + 64 * c;
        if (64 * c >= D) break;  // uniform
        const float y = d < D ? sm_v[tok * Dp + d] : 0.f;
#pragma unroll
        for (int i = 0; i < kPerWave; ++i)
          if (!drafted || (seen[i] >> tok & 1)) acc[i][c] = fmaf(p[i], y, acc[i][c]);  // (what is not seen may be NaN)
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kPerWave; ++i) {
    const int v = wave * kPerWave + i;
    if (v >= nv) continue;
    const int j = r.first + (v0 + v) / G, head = h * G + (v0 + v) % G;
    const size_t id = (size_t)j * A.Hq + head;
    const size_t at = id * A.splits + blockIdx.z;
    const float inv = A.splits > 1 ? 1.f : l[i] != 0.f ? 1.f / l[i] : sees(A, r, j) ? NAN : 0.f;
#pragma unroll
    for (int c = 0; c < DM / 64; ++c) {
      if (lane + 64 * c >= D) continue;
      if (A.splits > 1) A.part_o[at * D + lane + 64 * c] = acc[i][c];
      else out[id * D + lane + 64 * c] = from_f32<T>(as_f32_value(l[i] != 0.f ? acc[i][c] * inv : inv));
    }
    if (A.splits > 1 && lane == 0) {
      A.part_ml[2 * at] = m[i];
      A.part_ml[2 * at + 1] = l[i];
    }
  }
}

// out = sum 2^(m_s - M) O_s / sum 2^(m_s - M) l_s over the stretches.  One workgroup per token.
template <typename T>
__global__ __launch_bounds__(kGenThreads) void tree_generic_join(T* __restrict__ out, Args A) {
  const int j = blockIdx.x, t = threadIdx.x;
  int b = -1;  // the row whose tokens hold j
  for (int b0 = 0; b0 < A.batch; b0 += kGenThreads) {  // uniform
    const int mine = b0 + t < A.batch ? b0 + t : -1;
    bool has = false;
    if (mine >= 0) {
      const Row r = row_of(A, mine);
      has = j >= r.first && j < r.first + r.n;
    }
    __shared__ int sm_row;
    if (t == 0) sm_row = -1;
    __syncthreads();
    if (has) sm_row = mine;
    __syncthreads();
    b = uni(sm_row);
    if (b >= 0) break;  // uniform
    __syncthreads();
  }
  if (b < 0) return;  // uniform: a token of no row is left as it was
  const bool any = sees(A, row_of(A, b), j);
  for (int i = t; i < A.Hq * A.D; i += kGenThreads) {
    const int head = i / A.D, d = i - head * A.D;
    const size_t at = ((size_t)j * A.Hq + head) * A.splits;
    float M = -INFINITY, den = 0.f, o = 0.f;
    for (int s = 0; s < A.splits; ++s) M = fmaxf(M, A.part_ml[2 * (at + s)]);
    const float ms = M == -INFINITY ? 0.f : M;
    for (int s = 0; s < A.splits; ++s) {
      const float f = __builtin_amdgcn_exp2f(A.part_ml[2 * (at + s)] - ms);
      den = fmaf(A.part_ml[2 * (at + s) + 1], f, den);
      o = fmaf(A.part_o[(at + s) * A.D + d], f, o);
    }
    out[((size_t)j * A.Hq + head) * A.D + d] = from_f32<T>(as_f32_value(den != 0.f ? o / den : any ? NAN : 0.f));
  }
}

struct GenericPlan {
  unsigned tiles;
  int splits;
};
// Splits that give some 1024 workgroups, of 256 tokens at least (were every row as long as the table).
GenericPlan generic_plan(int tokens, int batch, int Hq, int Hkv, int P, int max_pages) {
  const long vectors = (long)tokens * (Hq / Hkv);
  GenericPlan p;
  p.tiles = (unsigned)((vectors + kVec - 1) / kVec + min(batch, tokens));  // (a part of a tile a row besides)
  const long wgs = (long)p.tiles * Hkv, most = ((long)max_pages * P + 255) / 256;
  p.splits = (int)max(1L, min(min(32L, most), 1024 / wgs));
  return p;
}
size_t generic_floats(const GenericPlan& p, int tokens, int Hq, int D) {
  return p.splits > 1 ? (size_t)tokens * Hq * p.splits * (D + 2) : 0;
}

}  // namespace
}  // namespace cir

using namespace cir;

extern "C" size_t cir_tree_attention_workspace_bytes(int tokens, int batch, int num_heads, int num_kv_heads,
                                                     int head_dim, int page_size, int max_pages, int kv_dtype) {
  if (tokens <= 0 || batch <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads || head_dim <= 0 ||
      head_dim > kMaxD || page_size <= 0 || max_pages <= 0 || (long)page_size * max_pages > 0x7fffffffL ||
      (long)tokens * num_heads >= 1L << 26)
    return 0;
  const GenericPlan g = generic_plan(tokens, batch, num_heads, num_kv_heads, page_size, max_pages);
  return generic_floats(g, tokens, num_heads, head_dim) * sizeof(float);
}

extern "C" int cir_paged_tree_attention(const void* q, const void* k_pool, const void* v_pool,
                                        const int32_t* page_table, const int32_t* seq_lens, const int32_t* offsets,
                                        const int32_t* counts, const int64_t* masks, int words, void* out,
                                        void* workspace, size_t workspace_bytes, int tokens, int batch, int num_heads,
                                        int num_kv_heads, int head_dim, int page_size, int max_pages, float scale,
                                        int kv_dtype, void* stream) {
  CIR_CHECK_ARG(tokens >= 0 && batch >= 0, "tree_attention: tokens and batch must be >= 0");
  if (tokens == 0 || batch == 0) return 0;
  CIR_CHECK_ARG(q && k_pool && v_pool && page_table && seq_lens && offsets && counts && masks && out,
                "tree_attention: null pointer");
  CIR_CHECK_ARG(num_kv_heads > 0 && num_heads > 0 && num_heads % num_kv_heads == 0,
                "tree_attention: num_heads (%d) must be a multiple of num_kv_heads (%d)", num_heads, num_kv_heads);
  CIR_CHECK_ARG(head_dim > 0 && head_dim <= kMaxD, "tree_attention: head_dim %d out of range (1..%d)", head_dim, kMaxD);
  CIR_CHECK_ARG(page_size > 0 && max_pages > 0 && (long)page_size * max_pages <= 0x7fffffffL,
                "tree_attention: page_size and max_pages must be positive, and their product a 32-bit number");
  CIR_CHECK_ARG(kv_dtype == CIR_F16 || kv_dtype == CIR_F32, "tree_attention: kv_dtype must be CIR_F16 or CIR_F32");
  CIR_CHECK_ARG(words >= 1 && words * 64 <= kMaxDrafts, "tree_attention: words must be 1..%d (got %d)", kMaxDrafts / 64,
                words);
  CIR_CHECK_ARG((long)tokens * num_heads < 1L << 26 && num_kv_heads < 1 << 16 && batch < 1 << 20,
                "tree_attention: 2^26 query vectors, 2^16 KV heads or 2^20 rows and more");
  const GenericPlan g = generic_plan(tokens, batch, num_heads, num_kv_heads, page_size, max_pages);
  const size_t floats = generic_floats(g, tokens, num_heads, head_dim), need = floats * sizeof(float);
  CIR_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need && (uintptr_t)workspace % 16 == 0),
                "tree_attention: workspace too small or not on 16 bytes (%zu < %zu)", workspace_bytes, need);
  float* ws = static_cast<float*>(workspace);
  const float scale_log2 = scale * kLog2e;
  const Args A{page_table, seq_lens, offsets, counts, reinterpret_cast<const uint32_t*>(masks), ws,
               ws + (size_t)tokens * num_heads * g.splits * head_dim, tokens, batch, num_heads, num_kv_heads, head_dim,
               page_size, max_pages, words, g.splits, scale_log2};
  hipStream_t s = as_stream(stream);
  const auto go = [&]<typename T>() {
    const dim3 grid(g.tiles, num_kv_heads, g.splits);
    const T *qt = static_cast<const T*>(q), *kt = static_cast<const T*>(k_pool), *vt = static_cast<const T*>(v_pool);
    if (head_dim <= 64) tree_generic<T, 64><<<grid, kGenThreads, 0, s>>>(qt, kt, vt, static_cast<T*>(out), A);
    else if (head_dim <= 128) tree_generic<T, 128><<<grid, kGenThreads, 0, s>>>(qt, kt, vt, static_cast<T*>(out), A);
    else tree_generic<T, 256><<<grid, kGenThreads, 0, s>>>(qt, kt, vt, static_cast<T*>(out), A);
    const int st = launch_status();
    if (st || g.splits == 1) return st;
    tree_generic_join<T><<<tokens, kGenThreads, 0, s>>>(static_cast<T*>(out), A);
    return launch_status();
  };
  return kv_dtype == CIR_F16 ? go.template operator()<f16>() : go.template operator()<float>();
}
