// Attention of drafted tokens over a paged cache: row b's n tokens lie at the end of its
// context, and token j sees the context before them and those of them that its mask names.
//
//   out_j = softmax(scale q_j K^T) V over the tokens t < c and the c + k with bit k of mask_j,
//   c = seq_len - n
#include "attn_tile.hpp"

#include <float.h>
#include <math.h>

#include <algorithm>

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
// tokens and the table whatever the device's numbers are.  A row of more tokens than the masks have bits for is refused:
// what its tokens see is not known, so nothing is stored of it and all of them yield NaN.
struct Row {
  int first, n, context, limit;
};
__device__ __forceinline__ bool refused(const Args& A, int n) { return n > 64 * A.words; }
__device__ __forceinline__ Row row_of(const Args& A, int b) {
  const int o = A.offsets[b], e = A.offsets[b + 1], c = A.counts[b], len = A.lens[b];
  Row r;
  r.first = min(max(o, 0), A.tokens);
  r.n = max(0, min(c, min(e, A.tokens) - r.first));
  r.context = max(0, len - r.n);
  r.limit = refused(A, r.n) ? 0 : max(0, min(len, A.max_pages * A.P));
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

// Whether token j sees any token at all (and yields NaN if none of them counts).
__device__ __forceinline__ bool sees(const Args& A, const Row& r, int j) {
  if (min(r.context, r.limit) > 0 || refused(A, r.n)) return true;
  const int n = min(r.n, r.limit - r.context);
  uint32_t any = 0;
  for (int w = 0; 32 * w < n; ++w) any |= mask_word(A, j, w, n);
  return any != 0;
}

// -------------------------------------------------------------- any sizes -----
// Any head_dim up to 256, type and page size, in fp32.  A workgroup takes up to 16 query vectors of one row and KV head (a
// tile) over a stretch of the row's tokens; its wavefronts take turns at blocks of 16 tokens, each with a softmax of its
// own, and are joined through LDS at the end.  MFMA 16x16x4 in fp32, S^T = K Q^T and O^T = V^T P^T, from registers alone:
// the order of the summed dims and tokens is free, so lane l takes dims 16 c + 4 (l / 16) .. of K and Q by one load, its
// scores are those of tokens 4 (l / 16) .. of vector l % 16, which is how the second product wants the weights, and its
// rows of V^T are dims 64 g + 4 (l % 16) .., again one load.  K of the next block and V of this one are on their way
// during the products.  16 rows of 1 or 2 tokens over 7800, 16 heads on 8 of 96 dims in fp32 (767 MB): 128 us, 6.0 TB/s;
// 7 tokens over 97, 4 heads on 2 of 64 dims: 8.4, latency (plan, table, K, two blocks, the join through LDS).
constexpr int kGenThreads = 256;
constexpr int kGenWaves = kGenThreads / 64;
constexpr int kVec = 16;
constexpr int kTok = 16;
constexpr int kMaxD = 256;

__device__ __forceinline__ int tiles_of(const Args& A, int n) { return (n * (A.Hq / A.Hkv) + kVec - 1) / kVec; }

template <typename T, int DM, bool QUADS>  // DM: head_dim at most; QUADS: it is a multiple of 4
__global__ __launch_bounds__(kGenThreads) void tree_generic(const T* __restrict__ q, const T* __restrict__ kp,
                                                            const T* __restrict__ vp, T* __restrict__ out, Args A) {
  constexpr int C = DM / 16, NGr = DM / 64;
  typedef T mt __attribute__((ext_vector_type(4), aligned(sizeof(T))));  // (at any address)
  typedef T vt __attribute__((ext_vector_type(4)));
  __shared__ __align__(16) float sm_o[kGenWaves][kVec][DM + 4];
  __shared__ float sm_ml[kGenWaves][2][kVec];
  __shared__ int sm_sum[kGenWaves], sm_find[2];
  const int D = A.D;
  const int t = threadIdx.x, lane = t & 63, wave = uni(t >> 6), col = lane & 15, quarter = lane >> 4;
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
  constexpr int kTurn = kTok * kGenWaves;
  const int64_t stretch = (((int64_t)r.limit + A.splits - 1) / A.splits + kTurn - 1) / kTurn * kTurn;
  const int k0 = (int)min((int64_t)r.limit, blockIdx.z * stretch), k1 = (int)min((int64_t)r.limit, k0 + stretch);

  // Dims d .. d + 3 of a row; what stands for those past the last is some other dim's.  Without a branch, and so is what
  // follows: where lanes take different paths to a register, the compiler waits for the load there.
  const auto part_of = [&](const T* row, int d) __attribute__((always_inline)) {
    if constexpr (QUADS) return static_cast<vt>(*reinterpret_cast<const mt*>(row + min(d, D - 4)));
    asm volatile("" : "+v"(d));  // (else the places of all elements are kept through the loop: 20 registers too many at 256)
    vt x;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = row[min(d + e, D - 1)];
    return x;
  };
  const auto f32_of = [](vt x) { return f32x4{to_f32(x[0]), to_f32(x[1]), to_f32(x[2]), to_f32(x[3])}; };
  const auto dims_of = [&](f32x4 x, int d) __attribute__((always_inline)) {  // zeros past the last dim
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = d + e < D ? x[e] : 0.f;
    return x;
  };
  // Token k + l % 16 of block k, or the stretch's last: its page, and the place of its row in the pools.
  const auto token_at = [&](int64_t k) { return (int)min(k + col, (int64_t)k1 - 1); };
  const auto page_of = [&](int64_t k) { return A.table[(size_t)b * A.max_pages + token_at(k) / A.P]; };
  const auto row_at = [&](int64_t k, int page) { return (((int64_t)page * A.Hkv + h) * A.P + token_at(k) % A.P) * D; };
  vt nk[C];
  const auto load_k = [&](int64_t at) __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (16 * c < D) nk[c] = part_of(kp + at, 16 * c + 4 * quarter);  // uniform
  };
  int64_t k = (int64_t)k0 + kTok * wave;
  int64_t at = 0;
  if (k < k1) {  // uniform in a wavefront
    at = row_at(k, page_of(k));
    load_k(at);
  }
  const int live = min(v0 + col, r.n * G - 1), j = r.first + live / G;  // (vectors past the last: the last one again)
  f32x4 qf[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    qf[c] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (16 * c >= D) continue;  // uniform
    const T* row = q + ((size_t)j * A.Hq + (size_t)h * G + live % G) * D;
    qf[c] = dims_of(f32_of(part_of(row, 16 * c + 4 * quarter)) * A.scale_log2, 16 * c + 4 * quarter);
  }
  float m = -INFINITY, l = 0.f;
  f32x4 acc[NGr][4];  // [64 dims][dim % 4]: dims 64 g + 16 (l / 16) + 4 i + dim % 4
#pragma unroll
  for (int g = 0; g < NGr; ++g)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[g][e] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (; k < k1; k += kTurn) {  // uniform in a wavefront
    const int page = page_of(k + kTurn);
    vt nv_[4][NGr];
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // token 4 (l / 16) + i
      const T* row = vp + __shfl(at, 4 * quarter + i, 64);
#pragma unroll
      for (int g = 0; g < NGr; ++g)
        if (64 * g < D) nv_[i][g] = part_of(row, 64 * g + 4 * col);  // uniform
    }
    f32x4 s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (16 * c >= D) continue;  // uniform
      f32x4 x = f32_of(nk[c]);
      if (16 * c + 16 > D) x = dims_of(x, 16 * c + 4 * quarter);  // uniform
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], qf[c][e], s[e & 1], 0, 0, 0);
    }
    const int64_t here = at;
    at = row_at(k + kTurn, page);
    load_k(at);
    const int nt = (int)min((int64_t)kTok, k1 - k);
    const bool drafted = k + nt > r.context;  // uniform: some tokens that not every vector sees
    uint32_t seen = (1u << nt) - 1;
    if (drafted) seen &= seen_from(A, j, (int)k, r.context, r.n);
    float p[4], mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      p[i] = seen >> (4 * quarter + i) & 1 ? as_f32_value(s[0][i] + s[1][i]) : -INFINITY;
      mx = fmaxf(mx, p[i]);
    }
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    const float mn = fmaxf(m, mx), ms = mn == -INFINITY ? 0.f : mn, alpha = __builtin_amdgcn_exp2f(m - ms);
    l *= alpha;
    m = mn;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      p[i] = __builtin_amdgcn_exp2f(p[i] - ms);
      l += p[i];
    }
    if (__builtin_amdgcn_ballot_w64(alpha != 1.f) != 0) {  // uniform
#pragma unroll
      for (int g = 0; g < NGr; ++g)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[g][e] *= alpha;
    }
    bool dirty = false;
#pragma unroll
    for (int g = 0; g < NGr; ++g) {
      if (64 * g >= D) continue;  // uniform
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f32x4 x = f32_of(nv_[i][g]);
        if (nt < kTok) {  // uniform: the last token again
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = 4 * quarter + i < nt ? x[e] : 0.f;
        }
        if (drafted) {  // uniform: what is no finite number must not meet the zero weights of what is not seen
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const bool bad = !(fabsf(x[e]) < INFINITY);
            dirty |= bad;
            x[e] = bad ? 0.f : x[e];
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[g][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], p[i], acc[g][e], 0, 0, 0);
      }
    }
    if (__builtin_amdgcn_ballot_w64(dirty) != 0) {  // uniform: and is added to the sums of the vectors that see its token
#pragma unroll 1
      for (int tok = 0; tok < nt; ++tok) {
        const T* row = vp + __shfl(here, tok, 64);
#pragma unroll
        for (int g = 0; g < NGr; ++g)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int d = 64 * g + 16 * quarter + 4 * i + e;
              const float x = d < D ? to_f32(row[d]) : 0.f;
              if ((seen >> tok & 1) && !(fabsf(x) < INFINITY)) acc[g][e][i] += x;
            }
      }
    }
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
#pragma unroll
  for (int g = 0; g < NGr; ++g)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<f32x4*>(&sm_o[wave][col][64 * g + 16 * quarter + 4 * i]) =
          f32x4{acc[g][0][i], acc[g][1][i], acc[g][2][i], acc[g][3][i]};
  if (quarter == 0) {
    sm_ml[wave][0][col] = m;
    sm_ml[wave][1][col] = l;
  }
  __syncthreads();
  // 16 threads per vector from here on.
  const int v = t >> 4, part = t & 15;
  if (v >= nv) return;
  float M = -INFINITY, f[kGenWaves], den = 0.f;
#pragma unroll
  for (int w = 0; w < kGenWaves; ++w) M = fmaxf(M, sm_ml[w][0][v]);
#pragma unroll
  for (int w = 0; w < kGenWaves; ++w) {
    f[w] = __builtin_amdgcn_exp2f(sm_ml[w][0][v] - (M == -INFINITY ? 0.f : M));
    den = fmaf(sm_ml[w][1][v], f[w], den);
  }
  const int token = r.first + (v0 + v) / G;
  const size_t id = (size_t)token * A.Hq + h * G + (v0 + v) % G;
  const size_t place = id * A.splits + blockIdx.z;
  const float inv = den != 0.f ? 1.f / den : 0.f, none = den != 0.f || !sees(A, r, token) ? 0.f : NAN;
#pragma unroll
  for (int g = 0; g < NGr; ++g) {
    const int d = 64 * g + 4 * part;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kGenWaves; ++w)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(sm_o[w][v][d + e], f[w], o[e]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (d + e >= D) continue;
      if (A.splits > 1) A.part_o[place * D + d + e] = o[e];
      else out[id * D + d + e] = from_f32<T>(as_f32_value(den != 0.f ? o[e] * inv : none));
    }
  }
  if (A.splits > 1 && part == 0) {
    A.part_ml[2 * place] = M;
    A.part_ml[2 * place + 1] = den;
  }
}

// out = sum 2^(m_s - M) O_s / sum 2^(m_s - M) l_s over the stretches.  A wavefront per token and head: lanes are stretches
// for the statistics, dims for the sums, 16 O on their way.
constexpr int kMaxSplits = 64;
template <typename T>
__global__ __launch_bounds__(kGenThreads) void tree_generic_join(T* __restrict__ out, Args A) {
  const int lane = threadIdx.x & 63;
  const int64_t id = (int64_t)blockIdx.x * kGenWaves + uni(threadIdx.x >> 6);
  const int j = (int)(id / A.Hq);
  if (j >= A.tokens) return;  // uniform in a wavefront
  const float2 ml = lane < A.splits ? *reinterpret_cast<const float2*>(A.part_ml + 2 * (id * A.splits + lane))
                                    : make_float2(-INFINITY, 0.f);
  int b = -1;  // the row whose tokens hold j
  for (int b0 = 0; b0 < A.batch && b < 0; b0 += 64) {  // uniform
    bool has = false;
    if (b0 + lane < A.batch) {
      const Row r = row_of(A, b0 + lane);
      has = j >= r.first && j < r.first + r.n;
    }
    const uint64_t rows = __builtin_amdgcn_ballot_w64(has);
    if (rows) b = b0 + __builtin_ctzll(rows);
  }
  if (b < 0) return;  // uniform: a token of no row is left as it was
  const float M = wave_max(ml.x), f = __builtin_amdgcn_exp2f(ml.x - (M == -INFINITY ? 0.f : M)), den = wave_sum(ml.y * f);
  const float none = den != 0.f || !sees(A, row_of(A, b), j) ? 0.f : NAN;
  for (int d0 = 0; d0 < A.D; d0 += 64) {  // uniform
    const int d = min(d0 + lane, A.D - 1);
    float o = 0.f;
    constexpr int U = 16;
    for (int s0 = 0; s0 < A.splits; s0 += U) {  // uniform
      float x[U];
#pragma unroll
      for (int i = 0; i < U; ++i) x[i] = A.part_o[(id * A.splits + min(s0 + i, A.splits - 1)) * A.D + d];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const float fi = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), min(s0 + i, 63)));
        if (s0 + i < A.splits) o = fmaf(x[i], fi, o);
      }
    }
    if (d0 + lane < A.D) out[id * A.D + d] = from_f32<T>(as_f32_value(den != 0.f ? o / den : none));
  }
}

struct GenericPlan {
  unsigned tiles;
  int splits;
};
// Splits that give some 1024 workgroups, of 128 tokens at least (were every row as long as the table).
GenericPlan generic_plan(int tokens, int batch, int Hq, int Hkv, int P, int max_pages) {
  const long vectors = (long)tokens * (Hq / Hkv);
  GenericPlan p;
  p.tiles = (unsigned)((vectors + kVec - 1) / kVec + min(batch, tokens));  // (a part of a tile a row besides)
  const long wgs = (long)p.tiles * Hkv, most = ((long)max_pages * P + 127) / 128;
  p.splits = (int)max(1L, min(min((long)kMaxSplits, most), 1024 / wgs));
  return p;
}
size_t generic_floats(const GenericPlan& p, int tokens, int Hq, int D) {
  return p.splits > 1 ? (size_t)tokens * Hq * p.splits * (D + 2) : 0;
}

// Whether x is an infinity or NaN (not 0: it is), in a form that ors.
__device__ __forceinline__ uint32_t not_finite(f16 x) {
  const uint16_t u = __builtin_bit_cast(uint16_t, x);
  return (u & 0x7c00) == 0x7c00;
}

// ------------------------------------------------- fp16, head_dim 128: MFMA -----
// Work.  An item is a row's tile of up to 256 query vectors (drafted token and head of the KV head's group) over all that
// the row holds; it costs kItemCost + its 32-token blocks.  The items lie on one axis and each team of workgroups (one per
// KV head) takes an equal stretch of it: lengths and counts live on the device, and a grid cut by rows leaves CUs idle
// behind the longest.  Every workgroup scans the rows for itself.  A stretch's part of an item is a piece, which leaves
// (max, sum, O) of its vectors; the piece of team w and of the tile that begins at vector e of all (e = first token * G +
// 256 tile) lies at vector 256 w + e of the workspace: along the axis one of the two grows by at least the piece's
// vectors, so pieces do not overlap, and the join finds a tile's pieces from its start and the stretch alone.
//
// Body (4 wavefronts, one workgroup per CU, up to 512 registers a lane).  Each wavefront takes NG groups of 32 query
// vectors (Q in accumulator registers) and, of VW = 4 / CW wavefronts side by side, every CW-th block.  Stages of 64 tokens
// of K and V come by DMA into a ring of four in LDS: two are on their way while one is worked on.  S^T = K Q^T and
// O^T = V^T P^T on MFMA 32x32x16: a lane holds one vector's scores and sums, 64 vectors a wavefront halve the LDS reads of
// 32.  The scores of the next block run on the matrix cores while the VALU takes this block's exponentials.
//
// Bound, and measured (kernel, then join): 8 trees of 57 to 64 tokens over 11000 to 16000, 32 query heads on 8 (107 GFLOP):
// 155 + 10 us in a long run of calls, 690 TFLOP/s (up to 181 where the card's clocks fall), the matrix cores busy 40% of the
// cycles: a block of 32 tokens and 64 vectors a wavefront takes 2500 cycles for 1024 of products.  Its 330 instructions, one
// in 4 to 5 cycles from one wavefront per SIMD and 32 exponentials at a quarter of that rate, make some 2000 of them; what
// the rest waits for is not known.  32 trees of 5 to 16 tokens, 28 heads on 4 (238 MB of K and V): 63 + 6 us, 3.8 TB/s; 26 us of it
// are what comes before and behind the blocks of a workgroup's one or two pieces (plan 3.3 us, a piece's first loads 4, its
// sums 3).  4 trees of 26 tokens over 300 to 3000: 22 + 5, all of it such.  K and V straight into registers, without a ring,
// took 32 and 100 us where this took 31 and 75.
constexpr int D = 128;
constexpr int kBlock = 32;       // tokens of an MFMA tile
constexpr int kGroup = 32;       // query vectors of an MFMA tile
constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kTileVec = 256;    // query vectors of a tile
constexpr int kWorkgroups = 256;
constexpr int kItemCost = 10;    // a piece's start and join, in blocks (32 and 8 trees above: 63 and 168 us, with 6 70 and 176,
                                 // with 16 63 and 174)
constexpr int kMinStretch = 4;   // (2 trees of 5 and 26 tokens over 300: 15 us, with 8 17, with 16 23)
constexpr int kMaxRows = 1024;
constexpr int kMaxGroup = 2048;   // query heads per KV head (256 G G < 2^32: token_of is exact)
constexpr int kRowB = 2 * D;     // bytes of a K or V row
constexpr int kStageTok = 64;    // tokens of a stage
constexpr int kStage = 2 * kStageTok * kRowB;  // bytes: K, then V

// What the join wants to know of a token's row: place of the first tile's blocks on the axis, their number (kNoRow: no row
// counts the token, kRefused: its row is), the stretch, and 256 row + the token's number in it.
constexpr int kNoRow = -1, kRefused = -2;
struct TokRec {
  int start, blocks, stretch, row;
};
struct Fast {
  Args a;
  TokRec* rec;      // [tokens]
  float *o, *ml;    // [vector of the workspace][KV head][D] and [2]
  int P16;          // page size / 16
  uint32_t page_magic;  // ceil(2^32 / P16): n / P16 = n * page_magic >> 32 (P16 > 1)
  uint32_t head_magic;  // the same of G = Hq / Hkv, for a row's vectors (fewer than 256 G + 256, G <= kMaxGroup)
};

__device__ __forceinline__ int page_index(const Fast& F, int n) {
  return F.P16 == 1 ? n : (int)__umulhi((uint32_t)n, F.page_magic);
}
__device__ __forceinline__ int token_of(const Fast& F, int G, int v) {  // v / G
  return G == 1 ? v : (int)__umulhi((uint32_t)v, F.head_magic);
}
__device__ __forceinline__ size_t rows16_at(const Fast& F, int h, int page, int n, int index) {
  return (((size_t)page * F.a.Hkv + h) * F.P16 + (n - index * F.P16)) * (16 * D);
}

// A piece: vectors v0 .. v0 + nv - 1 of row r (its tile) and KV head h over blocks blk0 .. blk1 - 1.
struct Piece {
  const f16 *q, *kp, *vp;
  const int32_t* ptrow;
  Row r;
  int h, v0, nv, blk0, blk1;
  size_t at;  // first vector in the workspace
};

struct Smem {
  float ml[kWaves][2][2 * kGroup];
  uint32_t mask[kTileVec][2 * kMaxDrafts / 64 + 1];
  int4 row[kMaxRows + 1];  // first token, their number, length (kRefused), place on the axis
  int scan[kWaves], find;
};

// 16 bytes per lane from a buffer (raw, bytes past its end read as 0) into LDS: lane l's land at lds + 16 l.  In asm, and so
// unknown to the compiler's counts: for a DMA that it knows it puts a wait before every read of the same LDS array, the
// ring's other stages among them.  The waits are the ones written out below (those that the compiler puts for loads of its
// own can only come out stricter); no register is written.
typedef int i32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ i32x4 buffer_of(const void* p, int bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(p);
  return i32x4{uni((int)a), uni((int)(a >> 32) & 0xffff), uni(bytes), 0x00020000};
}
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // (m0 is reserved; nothing else here uses it)
template <int ROWS4>  // 4 ROWS4 rows further, in the buffer and in LDS
__device__ __forceinline__ void dma16(i32x4 buffer, uint32_t lds, uint32_t offset) {
  constexpr int kMore = 4 * ROWS4 * kRowB;
  if constexpr (kMore == 0)
    asm volatile(
        "s_mov_b32 m0, %0\n\t"
        "s_nop 0\n\t"
        "buffer_load_dwordx4 %1, %2, 0 offen lds"
        :: "s"(lds), "v"(offset), "s"(buffer) : "memory", "m0");
  else
    asm volatile(
        "s_add_u32 m0, %0, %3\n\t"
        "s_nop 0\n\t"
        "buffer_load_dwordx4 %1, %2, %4 offen lds"
        :: "s"(lds), "v"(offset), "s"(buffer), "n"(kMore), "s"(kMore) : "memory", "m0", "scc");
}
#pragma clang diagnostic pop

template <typename F>
__device__ __forceinline__ void for_each4(const F& f) {
  f.template operator()<0>();
  f.template operator()<1>();
  f.template operator()<2>();
  f.template operator()<3>();
}

// Running softmax of one query vector per lane (lane l and l + 32: the same vector).
struct Soft {
  float m, l;
  f32x16 acc[D / 32];
};

template <int VW, int NG>
__device__ __forceinline__ void tree_piece(const Fast& F, const Piece& p, Smem& sm, uint8_t* ring) {
  constexpr int CW = kWaves / VW;     // wavefronts that take turns at the blocks
  constexpr int PW = 2 / CW;          // blocks of a stage that a wavefront takes
  static_assert(CW == 1 || CW == 2, "");
  const Args& A = F.a;
  int t = threadIdx.x;
  asm volatile("" : "+v"(t));  // (else what all variants form from it is formed, and kept, before the first piece: 500 lines)
  const int wave = uni(t >> 6), lane = t & 63;
  const int l32 = lane & 31, h = lane >> 5;
  const int col = wave % VW, par = wave / VW;
  const float sc = fabsf(A.scale_log2);
  const int G = A.Hq / A.Hkv;
  const int limit = min(p.r.limit, p.blk1 * kBlock);  // tokens of the piece end here
  const int nst = (p.blk1 - p.blk0 + 1) / 2;

  // DMA of a stage: each wavefront brings in 16 rows of K and of V, 4 rows per instruction (lane / 16 = row, lane % 16 =
  // LDS slot); chunk c of K row r goes to slot c ^ (r % 16), of V row r to slot c ^ (4 (r % 4) + r / 4 % 4).  Rows past the
  // piece's last token lie past the buffer's end and are zero.
  const int lr = lane >> 4, ls = lane & 15;
  // Byte offset of the lane's chunk in the first four rows; rows 4 u on: ^ 64 u or 16 u, and 1024 u further.
  const uint32_t at_k = lr * kRowB + 16 * (ls ^ lr), at_v = lr * kRowB + 16 * (ls ^ (lr << 2));
  const int first16 = 2 * p.blk0 + wave, last16 = (limit - 1) >> 4;
  // Pages of 64 stages' rows, one a lane.  (Scalar loads count with those from LDS and return in any order, so that every
  // wait for LDS would wait for them: some 700 cycles a stage.)
  int pages;
  const auto fetch = [&](int st) __attribute__((always_inline)) {
    pages = p.ptrow[page_index(F, min(first16 + 4 * (st + lane), last16))];
    asm volatile("" : "+v"(pages));  // (waits here)
  };
  struct Rows {  // the rows of a stage
    i32x4 k, v;
    uint32_t to;  // in LDS
  };
  const uint32_t ring_at = uni((int)(uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)ring) + 16 * wave * kRowB;
  const auto rows_of = [&](int st) __attribute__((always_inline)) {
    const int n = first16 + 4 * st, m = min(n, last16);
    const size_t base = rows16_at(F, p.h, __builtin_amdgcn_readlane(pages, st & 63), m, page_index(F, m));
    const int bytes = max(0, min(16, limit - 16 * n)) * kRowB;
    return Rows{buffer_of(p.kp + base, bytes), buffer_of(p.vp + base, bytes), ring_at + (st & 3) * kStage};
  };
  const auto issue = [&](int st) __attribute__((always_inline)) {
    const Rows r = rows_of(st);
    for_each4([&]<int U>() __attribute__((always_inline)) { dma16<U>(r.k, r.to, at_k ^ (64 * U)); });
    for_each4([&]<int U>() __attribute__((always_inline)) { dma16<U>(r.v, r.to + kStage / 2, at_v ^ (16 * U)); });
  };
  fetch(0);

  // Q^T as the B operand: lane l32's vector of each group, dims 16 s + 8 h + e; a negative
  // scale goes into its sign, so that the maximum can be taken before scaling.
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  const uint32_t flip = A.scale_log2 < 0.f ? 0x80008000u : 0u;
  f16x8 qb[NG][8];
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const int v = (col * NG + g) * kGroup + l32;
    const int vv = p.v0 + min(v, p.nv - 1), tok = token_of(F, G, vv);  // (vectors past the last: the last one again)
    const f16* row = p.q + ((size_t)(p.r.first + tok) * A.Hq + (size_t)p.h * G + (vv - tok * G)) * D + 8 * h;
#pragma unroll
    for (int s = 0; s < 8; ++s) qb[g][s] = *reinterpret_cast<const f16x8*>(row + 16 * s);
  }
  issue(0);
  // The masks of the tile's vectors, where a block of the piece holds drafted tokens.
  const int drafts = min(p.r.n, p.r.limit - p.r.context);  // of the row, as far as the table holds them
  if (p.blk1 * kBlock > p.r.context) {                     // uniform
    static_assert(kTileVec <= kThreads, "");
    if (t < p.nv) {
      const int j = p.r.first + token_of(F, G, p.v0 + t);
#pragma unroll 1
      for (int w = 0; w < 2 * A.words; ++w) sm.mask[t][w] = mask_word(A, j, w, drafts);
    }
  }

  Soft a[NG];
  bool huge = false;  // uniform: some vector's |m| is 2^24 or more
  uint32_t dirty = 0;
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    a[g].m = -INFINITY;
    a[g].l = 0.f;
#pragma unroll
    for (int t = 0; t < D / 32; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) a[g].acc[t][r] = 0.f;
  }
  // LDS bytes of the lane's part of K rows (chunk 2 s + h: ^ 32 s) and of V rows (dims from 32 dt on: ^ 64 dt; token rows
  // 8 i + 4 h ..).
  const int ti = lane & 15, sub = (lane >> 4) & 1;
  const uint32_t k_at = l32 * kRowB + 16 * (h ^ (l32 & 15));
  uint32_t v_at[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    v_at[i] = kStage / 2 + (8 * i + 4 * h + (ti >> 2)) * kRowB + 64 * (ti >> 2) +
              16 * ((2 * sub + ((ti & 3) >> 1)) ^ (2 * i + h)) + 8 * (ti & 1);
  // Tokens of a block that the lane's vector of group g sees; score r is that of token bit_of(r).
  const auto seen_of = [&](int g, int blk) __attribute__((always_inline)) {
    const int k = blk * kBlock - p.r.context, rest = limit - blk * kBlock;  // drafted token of the block's first
    const uint32_t* m = sm.mask[min((col * NG + g) * kGroup + l32, p.nv - 1)];
    const int w = k >> 5, s = k & 31;
    const uint32_t lo = k < 0 ? 0xffffffffu : w < 2 * A.words ? m[w] : 0;
    const uint32_t hi = w + 1 >= 0 && w + 1 < 2 * A.words ? m[w + 1] : 0;
    const uint32_t seen = k <= -32 ? 0xffffffffu : s ? (lo >> s) | (hi << (32 - s)) : lo;
    return rest >= 32 ? seen : rest <= 0 ? 0u : seen & ((1u << rest) - 1);
  };
  const auto bit_of = [&](int r) { return 8 * (r >> 2) + 4 * h + (r & 3); };

  // Blocks from here on hold tokens that not every vector sees, or none.
  const int special = min(p.r.context, limit) / kBlock;
  f32x16 c[NG];  // scores of the block at hand
  f16x8 ka[8];   // K of the next one
  const auto read_k = [&](uint32_t at, int s) __attribute__((always_inline)) {
    ka[s] = *reinterpret_cast<const f16x8*>(ring + ((at + k_at) ^ (32 * s)));
  };
  // Rows of a stage on their way, in eight parts (K, then V): from a turn (below) on, a quarter of a stage's beside the
  // second products of a block and beside the first ones of the next, spread out: an LDS load takes a CU's four wavefronts
  // some 170 cycles together, and a wavefront that issues several at once stands still.
  Rows rows{};
  const auto load_part = [&]<int B, int U>(int i) __attribute__((always_inline)) {  // B: beside second products; U < 4 / PW
    if constexpr (PW == 1) {
      if constexpr (B) dma16<U>(rows.k, rows.to, at_k ^ (64 * U));
      else dma16<U>(rows.v, rows.to + kStage / 2, at_v ^ (16 * U));
    } else {
      const bool v = B ? (i & 1) : !(i & 1);
      constexpr int W = B ? U : U + 2;
      dma16<W>(v ? rows.v : rows.k, rows.to + (v ? kStage / 2 : 0), (v ? at_v : at_k) ^ ((v ? 16 : 64) * W));
    }
  };
  // One block, `blk` (its V at byte `vcur` of the ring), and the scores of the next one, `bnext`; K of the one after that
  // (at `kafter`) is read beside the second products.
  //
  // p = 2^(c sc - m) by one FMA, in fp16: the B operand of the second product, since fp32 products are an eighth as fast.
  // Each weight is rounded once (2^-11 of it, or 2^-25 below fp16's normal range) and the sum takes the rounded ones; the
  // results' error against 64 bits is 2.8e-4 where fp32 weights, and the same fp16 output, leave 2.1e-4.  The first block's scores set m, which
  // follows the maximum only once a lane's 16 weights of a block sum to more than 2^8: then no p is larger, and fp16 holds it
  // as exactly as p <= 1; after a piece's first blocks the accumulators are hardly ever scaled, and no maximum is taken.
  // m is a rounded product, off by up to half an ulp: a factor that all p of the vector share.  From |m| = 2^24 on (where it
  // could leave fp16) the rounded products are subtracted instead.
  //
  // One wavefront per SIMD issues one instruction in 4 to 5 cycles, whatever it is for: products, exponentials and loads
  // stand by turns in the order wanted (sched_barrier), and what the 32 cycles of a product leave is filled.
  auto block = [&]<bool SPECIAL>(int i, int blk, int bnext, uint32_t kafter, uint32_t vcur) __attribute__((always_inline)) {
    f16x8 va[D / 32][2], pa[NG][2];
    f32x16 cn[NG];
    float sum[NG], e0, e1;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      sum[g] = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) cn[g][r] = 0.f;
    }
    const auto put = [&](int g, int r, float x, float y) __attribute__((always_inline)) {  // weights r and r + 1
      const f16x2 two = {static_cast<f16>(x), static_cast<f16>(y)};
      pa[g][r >> 3][r & 7] = two.x;
      pa[g][r >> 3][(r & 7) + 1] = two.y;
      sum[g] = __builtin_amdgcn_fdot2(two, f16x2{(f16)1.f, (f16)1.f}, sum[g], false);  // exact products, fp32 sum
    };
    const auto exps = [&](int g, int r) __attribute__((always_inline)) {
      e0 = __builtin_amdgcn_exp2f(fmaf(c[g][r], sc, -a[g].m));
      e1 = __builtin_amdgcn_exp2f(fmaf(c[g][r + 1], sc, -a[g].m));
    };
    exps(0, 0);
    __builtin_amdgcn_sched_barrier(0);
    const auto first = [&]<int S>() __attribute__((always_inline)) {
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        cn[g] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka[S], qb[g][S], cn[g], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
        const int pair = S * NG + g, gp = pair >> 3, r = 2 * (pair & 7);  // the pair whose exponentials were taken before
        const float x = e0, y = e1;
        if (pair + 1 < 8 * NG) exps((pair + 1) >> 3, 2 * ((pair + 1) & 7));
        put(gp, r, x, y);
        if (g == 0) {
          constexpr int dt = S & 3, ks = S >> 2;
          const f16x4 lo = lds_read_tr(ring + (((vcur + v_at[0]) ^ (64 * dt)) + ks * 16 * kRowB));
          const f16x4 hi = lds_read_tr(ring + (((vcur + v_at[1]) ^ (64 * dt)) + ks * 16 * kRowB));
          va[dt][ks] = f16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        }
        if constexpr (S % (2 * PW) == PW) {
          if (g == NG - 1) load_part.template operator()<0, S / (2 * PW)>(i);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    for_each4([&]<int U>() __attribute__((always_inline)) { first.template operator()<U>(); });
    for_each4([&]<int U>() __attribute__((always_inline)) { first.template operator()<U + 4>(); });
    bool over = huge;
#pragma unroll
    for (int g = 0; g < NG; ++g) over |= !(sum[g] <= 256.f);
    if (__builtin_amdgcn_ballot_w64(over) != 0) {  // uniform
      bool far = false;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float mx = c[g][0];
#pragma unroll
        for (int r = 1; r < 16; ++r) mx = fmaxf(mx, c[g][r]);
        mx = as_f32_value(mx * sc);
        const float mn = fmaxf(a[g].m, fmaxf(mx, __shfl_xor(mx, 32, 64)));
        const float ms = mn == -INFINITY ? 0.f : mn, alpha = __builtin_amdgcn_exp2f(a[g].m - ms);
        a[g].l *= alpha;
        a[g].m = mn;
        far |= fabsf(ms) >= 0x1p24f;
#pragma unroll
        for (int t = 0; t < D / 32; ++t) a[g].acc[t] *= alpha;
        sum[g] = 0.f;
#pragma unroll
        for (int r = 0; r < 16; r += 2) {
          const float x = fabsf(ms) >= 0x1p24f ? as_f32_value(c[g][r] * sc) - ms : fmaf(c[g][r], sc, -ms);
          const float y = fabsf(ms) >= 0x1p24f ? as_f32_value(c[g][r + 1] * sc) - ms : fmaf(c[g][r + 1], sc, -ms);
          put(g, r, __builtin_amdgcn_exp2f(x), __builtin_amdgcn_exp2f(y));
        }
      }
      huge = __builtin_amdgcn_ballot_w64(far) != 0;
    }
    if constexpr (SPECIAL) {
      // Scores of tokens that a vector does not see become -inf.
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const uint32_t seen = seen_of(g, bnext);
#pragma unroll
        for (int r = 0; r < 16; ++r) cn[g][r] = seen >> bit_of(r) & 1 ? cn[g][r] : -INFINITY;
      }
      // V that is no finite number must not meet the zero weights of what is not seen: it is left out here and added after
      // the last block (below).
      if (blk >= special) {  // uniform
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
          for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const f16 x = va[dt][ks][e];
              dirty |= not_finite(x);
              va[dt][ks][e] = not_finite(x) ? (f16)0.f : x;
            }
      }
    }
    // A turn, before the block's second products and with V of it in registers: K of the block after the next one is to
    // have landed (all but the youngest eight loads), and every wavefront has left the stage that stage `far` takes.
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    if (PW == 1 || !(i & 1)) {  // uniform
      const int far = i / PW + (PW == 1 ? 4 : 3);
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_waitcnt(0x0F78);  // vmcnt(8)
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if ((far & 63) == 0) fetch(far);  // uniform
    }
    const auto second = [&]<int J>() __attribute__((always_inline)) {
      constexpr int g = J >> 3, dt = J & 3, ks = (J >> 2) & 1;  // (ks, then dt: four chains)
      a[g].acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va[dt][ks], pa[g][ks], a[g].acc[dt], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (J == 0) rows = rows_of(i / PW + (PW == 1 ? 4 : 3));
      if constexpr (NG == 1 || J >= 8) read_k(kafter, J & 7);
      if constexpr (J % (2 * PW * NG) == 2 * PW * NG - 1) load_part.template operator()<1, J / (2 * PW * NG)>(i);
      __builtin_amdgcn_sched_barrier(0);
    };
    for_each4([&]<int U>() __attribute__((always_inline)) { second.template operator()<U>(); });
    for_each4([&]<int U>() __attribute__((always_inline)) { second.template operator()<U + 4>(); });
    if constexpr (NG == 2) {
      for_each4([&]<int U>() __attribute__((always_inline)) { second.template operator()<U + 8>(); });
      for_each4([&]<int U>() __attribute__((always_inline)) { second.template operator()<U + 12>(); });
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      c[g] = cn[g];
      a[g].l += sum[g];
    }
  };
  // A wavefront's blocks in order: block i lies in stage i / PW.
  constexpr int kOther = kBlock * kRowB;  // the stage's second block
  const auto place = [&](int i) { return (uint32_t)((i / PW) & 3) * kStage + (PW == 1 ? par : i & 1) * kOther; };
#pragma unroll 1
  for (int st = 1; st < (PW == 1 ? 3 : 2); ++st) issue(st);
  rows = rows_of(PW == 1 ? 3 : 2);
  for_each4([&]<int U>() __attribute__((always_inline)) { dma16<U>(rows.k, rows.to, at_k ^ (64 * U)); });
  if constexpr (PW == 2) {
    dma16<0>(rows.v, rows.to + kStage / 2, at_v);
    dma16<1>(rows.v, rows.to + kStage / 2, at_v ^ 16);
  }
#pragma unroll
  for (int g = 0; g < NG; ++g)
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      qb[g][s] = __builtin_bit_cast(f16x8, __builtin_bit_cast(u32x4, qb[g][s]) ^ flip);
      // (Here, before the next stages are on their way: its wait would be for them too.  In accumulator registers, which an
      // MFMA reads as well as the others.)
      asm volatile("" : "+a"(qb[g][s]));
    }
  asm volatile("" ::: "memory");
  // Block 0 and K of block 1 have landed, the masks are written: lgkmcnt(0), vmcnt(12) (a stage and K of one) or 14.
  __builtin_amdgcn_s_waitcnt(PW == 1 ? 0x007C : 0x007E);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  {  // scores of the first block, and K of the second
    const int first = p.blk0 + (PW == 1 ? par : 0);
#pragma unroll
    for (int s = 0; s < 8; ++s) read_k(place(0), s);
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int r = 0; r < 16; ++r) c[g][r] = 0.f;
#pragma unroll
    for (int s = 0; s < 8; ++s)
#pragma unroll
      for (int g = 0; g < NG; ++g) c[g] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka[s], qb[g][s], c[g], 0, 0, 0);
#pragma unroll
    for (int s = 0; s < 8; ++s) read_k(place(1), s);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      if (first >= special) {  // uniform
        const uint32_t seen = seen_of(g, first);
#pragma unroll
        for (int r = 0; r < 16; ++r) c[g][r] = seen >> bit_of(r) & 1 ? c[g][r] : -INFINITY;
      }
      float mx = c[g][0];
#pragma unroll
      for (int r = 1; r < 16; ++r) mx = fmaxf(mx, c[g][r]);
      mx = as_f32_value(mx * sc);
      a[g].m = fmaxf(mx, __shfl_xor(mx, 32, 64));
      huge |= fabsf(a[g].m) >= 0x1p24f && a[g].m != -INFINITY;
    }
    huge = __builtin_amdgcn_ballot_w64(huge) != 0;
  }
  const auto turns = [&]<bool SPECIAL>(int from, int to) __attribute__((always_inline)) {
#pragma unroll 1
    for (int i = from; i < to; ++i) {
      const int blk = p.blk0 + (PW == 1 ? 2 * i + par : i);
      block.template operator()<SPECIAL>(i, blk, blk + CW, place(i + 2), place(i));
    }
  };
  const int plain = max(0, min(nst * PW, (special - p.blk0) / CW - 1));  // (a block scores the next one too)
  turns.template operator()<false>(0, plain);
  turns.template operator()<true>(plain, nst * PW);
  // Infinities and NaN of V among the drafted tokens: each is added to the sums of the vectors that see its token.
  if (__builtin_amdgcn_ballot_w64(dirty) != 0) {  // uniform
    for (int blk = p.blk0 + (PW == 1 ? par : 0); blk < p.blk1; blk += CW) {
      if (blk < special) continue;
#pragma unroll 1
      for (int dt = 0; dt < D / 32; ++dt) {
        f16x8 plus[2], minus[2];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int tok = min(blk * kBlock + bit_of(r), limit - 1), n = tok >> 4, index = page_index(F, n);
          const f16 x = p.vp[rows16_at(F, p.h, p.ptrow[index], n, index) + (tok & 15) * D + 32 * dt + l32];
          const uint16_t u = __builtin_bit_cast(uint16_t, x);
          const bool bad = not_finite(x), nan = bad && (u & 0x3ff);
          plus[r >> 3][r & 7] = nan || (bad && !(u & 0x8000)) ? (f16)1.f : (f16)0.f;
          minus[r >> 3][r & 7] = nan || (bad && (u & 0x8000)) ? (f16)1.f : (f16)0.f;
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const uint32_t seen = seen_of(g, blk);
          f16x8 on[2];  // the vector's tokens as 0 or 1, laid out as its weights
#pragma unroll
          for (int r = 0; r < 16; ++r) on[r >> 3][r & 7] = seen >> bit_of(r) & 1 ? (f16)1.f : (f16)0.f;
          f32x16 up, down;
#pragma unroll
          for (int r = 0; r < 16; ++r) up[r] = down[r] = 0.f;
#pragma unroll
          for (int ks = 0; ks < 2; ++ks) {
            up = __builtin_amdgcn_mfma_f32_32x32x16_f16(plus[ks], on[ks], up, 0, 0, 0);
            down = __builtin_amdgcn_mfma_f32_32x32x16_f16(minus[ks], on[ks], down, 0, 0, 0);
          }
#pragma unroll
          for (int t = 0; t < D / 32; ++t) {
            if (t != dt) continue;  // (uniform: dt is no constant, the accumulators are registers)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              a[g].acc[t][r] += up[r] > 0.f ? INFINITY : 0.f;
              a[g].acc[t][r] -= down[r] > 0.f ? INFINITY : 0.f;
            }
          }
        }
      }
    }
  }

  // The wavefronts' (m, l, O) go to LDS, 16-byte chunk c of vector v in slot c ^ (v % 32) of its 512 bytes; all threads join
  // those of wavefronts that took turns at the blocks, and write rows.
  static_assert(kWaves * 2 * kGroup * D * sizeof(float) <= 4 * kStage, "");
  dma_wait_barrier();  // (every wavefront is done with its blocks, and no DMA is on its way into them)
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    uint8_t* to = ring + (wave * NG + g) * kGroup * 512 + l32 * 512;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<f32x4*>(to + 16 * ((8 * dt + 2 * j + h) ^ l32)) =
            f32x4{a[g].acc[dt][4 * j], a[g].acc[dt][4 * j + 1], a[g].acc[dt][4 * j + 2], a[g].acc[dt][4 * j + 3]};
    a[g].l += __shfl_xor(a[g].l, 32, 64);
    if (h == 0) {
      sm.ml[wave][0][g * kGroup + l32] = a[g].m;
      sm.ml[wave][1][g * kGroup + l32] = a[g].l;
    }
  }
  __syncthreads();
  if (t < p.nv) {  // (max, sum) of vector t, and the factors of its parts' O
    constexpr int V = NG * kGroup;  // vectors of a wavefront
    float* m0 = &sm.ml[t / V][0][t % V];
    const size_t at = (p.at + t) * A.Hkv + p.h;
    float m = m0[0], l = m0[2 * kGroup];
    if constexpr (CW == 2) {
      float* m1 = &sm.ml[t / V + VW][0][t % V];
      const float M = fmaxf(m, m1[0]), ms = M == -INFINITY ? 0.f : M;
      const float f0 = __builtin_amdgcn_exp2f(m - ms), f1 = __builtin_amdgcn_exp2f(m1[0] - ms);
      l = fmaf(m1[2 * kGroup], f1, l * f0);
      m = M;
      m0[0] = f0;
      m1[0] = f1;
    }
    F.ml[2 * at] = m;
    F.ml[2 * at + 1] = l;
  }
  if constexpr (CW == 2) __syncthreads();
#pragma unroll 4
  for (int id = t; id < p.nv * (D / 4); id += kThreads) {
    const int v = id / (D / 4), c = id % (D / 4), slot = v * 512 + 16 * (c ^ (v & 31));
    f32x4 o = *reinterpret_cast<const f32x4*>(ring + slot);
    if constexpr (CW == 2) {
      constexpr int V = NG * kGroup;
      const float f0 = sm.ml[v / V][0][v % V], f1 = sm.ml[v / V + VW][0][v % V];
      const f32x4 x = *reinterpret_cast<const f32x4*>(ring + VW * V * 512 + slot);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(x[e], f1, o[e] * f0);
    }
    *reinterpret_cast<f32x4*>(F.o + ((p.at + v) * A.Hkv + p.h) * D + 4 * c) = o;
  }
  __syncthreads();  // the next piece writes the same LDS
}

__global__ __launch_bounds__(kThreads, 1) void tree_f16_d128(const f16* __restrict__ q, const f16* __restrict__ kp,
                                                             const f16* __restrict__ vp,
                                                             const int32_t* __restrict__ table, Fast F) {
  __shared__ __align__(16) uint8_t ring[4 * kStage];
  __shared__ Smem sm;
  const Args& A = F.a;
  const int G = A.Hq / A.Hkv, B = A.batch, Hkv = A.Hkv;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int w = blockIdx.x / Hkv, h = blockIdx.x - w * Hkv;  // team, KV head

  int all = 0;
  for (int b0 = 0; b0 < B; b0 += kThreads) {  // uniform
    const int b = b0 + t;
    int cost = 0;
    int4 row = make_int4(0, 0, 0, 0);
    if (b < B) {
      const Row r = row_of(A, b);
      const int blocks = (r.limit + kBlock - 1) / kBlock, tiles = (r.n * G + kTileVec - 1) / kTileVec;
      cost = blocks > 0 ? tiles * (blocks + kItemCost) : 0;
      row = make_int4(r.first, r.n, refused(A, r.n) ? kRefused : max(0, A.lens[b]), 0);
    }
    int upto = cost;
    for (int off = 1; off < min(B, 64); off <<= 1) {  // uniform
      const int o = __shfl_up(upto, off, 64);
      upto += lane >= off ? o : 0;
    }
    if (lane == min(B, 64) - 1) sm.scan[wave] = upto;
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      upto += i < wave ? sm.scan[i] : 0;
      total += sm.scan[i];
    }
    row.w = all + upto - cost;
    if (b < B) sm.row[b] = row;
    all += total;
    __syncthreads();
  }
  if (t == 0) sm.row[B].w = all;
  const int teams = gridDim.x / Hkv;
  const int stretch = max((all + teams - 1) / teams, kMinStretch);
  const int lo = w * stretch, hi = min(all, lo + stretch);
  __syncthreads();
  // What the join needs, shared out over the workgroups from the last one on (the ones without work of their own).
  const int id = (int)(gridDim.x - 1 - blockIdx.x) + t * (int)gridDim.x, step = kThreads * (int)gridDim.x;
  for (int j = id; j < A.tokens; j += step) {
    int a = 0, z = B - 1;  // the last row that begins at or before j (rows without tokens begin where the next does)
    while (a < z) {
      const int m = (a + z + 1) >> 1;
      if (sm.row[m].x <= j) a = m;
      else z = m - 1;
    }
    const int4 r = sm.row[a];
    const bool counted = j >= r.x && j < r.x + r.y;
    const int blocks = r.z == kRefused ? kRefused : (min(r.z, A.max_pages * A.P) + kBlock - 1) / kBlock;
    F.rec[j] = TokRec{r.w + kItemCost, counted ? blocks : kNoRow, stretch, kMaxDrafts * a + (j - r.x)};
  }
  if (lo >= hi) return;  // uniform
  for (int b = t; b < B; b += kThreads)
    if (sm.row[b].w <= lo && lo < sm.row[b + 1].w) sm.find = b;
  __syncthreads();

  for (int b = uni(sm.find); b < B; ++b) {  // uniform
    const int4 row = sm.row[b];
    const int start = uni(row.w);
    if (start >= hi) break;
    if (uni(sm.row[b + 1].w) == start) continue;
    Piece p;
    p.r.first = uni(row.x);
    p.r.n = uni(row.y);
    p.r.context = max(0, uni(row.z) - p.r.n);
    p.r.limit = min(uni(row.z), A.max_pages * A.P);
    const int blocks = (p.r.limit + kBlock - 1) / kBlock, cost = blocks + kItemCost;
    const int tiles = (p.r.n * G + kTileVec - 1) / kTileVec;
    for (int i = start >= lo || tiles == 1 ? 0 : (lo - start) / cost; i < tiles && start + i * cost < hi; ++i) {
      const int at = start + i * cost + kItemCost;
      const int k0 = max(0, min(lo - at, blocks)), k1 = max(0, min(hi - at, blocks));
      if (k0 >= k1) continue;
      p.q = q;
      p.kp = kp;
      p.vp = vp;
      p.h = h;
      p.ptrow = table + (size_t)b * A.max_pages;
      p.v0 = i * kTileVec;
      p.nv = min(kTileVec, p.r.n * G - p.v0);
      p.blk0 = k0;
      p.blk1 = k1;
      p.at = (size_t)w * kTileVec + (size_t)p.r.first * G + p.v0;
      // The fewest vectors a wavefront that hold the tile; 112 vectors of 32 trees: 63 us, as <4, 2> 92; up to 48 of 32 trees
      // over up to 4000 tokens: 62, as <2, 2> 71, as <4, 2> 101.
      if (p.nv <= 2 * kGroup) tree_piece<2, 1>(F, p, sm, ring);
      else if (p.nv <= 4 * kGroup) tree_piece<2, 2>(F, p, sm, ring);
      else tree_piece<4, 2>(F, p, sm, ring);
    }
  }
}

// out = sum 2^(m_i - M) O_i / sum 2^(m_i - M) l_i over the pieces of a vector's tile.  Half a wavefront per vector, four dims
// a lane; lane k takes (m, l) of every 32nd piece.  Bound by latency (record, then pieces): four O are on their way, the first
// ones along with the (m, l).  15.5k vectors of 4 to 5 pieces: 10.1 us, of 41k vectors with one or two 12.3; two halves per
// vector, with every second piece each: 12.8 and 22.5, eight O on their way 10.5 and 14.4.
constexpr int kJoinVec = 8;  // of a workgroup
__global__ __launch_bounds__(32 * kJoinVec) void tree_join(Fast F, f16* __restrict__ out) {
  constexpr int U = 4;
  const Args& A = F.a;
  const int lane = threadIdx.x & 31;
  const int id = blockIdx.x * kJoinVec + (threadIdx.x >> 5), G = A.Hq / A.Hkv;
  const int j = id / A.Hq, head = id - j * A.Hq, h = head / G;
  TokRec rec = F.rec[min(j, A.tokens - 1)];
  if (j >= A.tokens) rec.blocks = kNoRow;
  const bool live = rec.blocks != kNoRow;
  const int v = rec.row % kMaxDrafts * G + (head - h * G), tile = v / kTileVec;
  const int start = rec.start + tile * (rec.blocks + kItemCost), w0 = start / rec.stretch;
  const int n = live && rec.blocks > 0 ? (start + rec.blocks - 1) / rec.stretch - w0 + 1 : 0;
  const auto at = [&](int k) {
    return ((size_t)(w0 + k) * kTileVec + (size_t)j * G + (head - h * G)) * A.Hkv + h;
  };
  const auto ml_of = [&](int k) { return *reinterpret_cast<const float2*>(F.ml + 2 * at(k)); };
  const auto o_of = [&](int k) { return *reinterpret_cast<const f32x4*>(F.o + D * at(k) + 4 * lane); };
  float den = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  if (n > 0) {
    float2 ml = lane < n ? ml_of(lane) : make_float2(-INFINITY, 0.f);
    f32x4 x[U];
    const auto load = [&](int k0) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < U; ++i) x[i] = o_of(min(k0 + i, n - 1));
    };
    load(0);
    float M = ml.x;
    for (int k = lane + 32; k < n; k += 32) M = fmaxf(M, ml_of(k).x);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) M = fmaxf(M, __shfl_xor(M, d, 32));
    const float ms = M == -INFINITY ? 0.f : M;
    for (int k0 = 0; k0 < n; k0 += 32) {
      if (k0) ml = k0 + lane < n ? ml_of(k0 + lane) : make_float2(-INFINITY, 0.f);
      const float f = __builtin_amdgcn_exp2f(ml.x - ms);
      den = fmaf(ml.y, f, den);
      for (int j0 = k0; j0 < min(n, k0 + 32); j0 += U) {
#pragma unroll
        for (int i = 0; i < U; ++i) {
          const int k = j0 + i;
          const float fk = __shfl(f, k - k0, 32);
          if (k < n) {
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = fmaf(x[i][e], fk, o[e]);
          }
        }
        if (j0 + U < n) load(j0 + U);
      }
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) den += __shfl_xor(den, d, 32);
  }
  if (!live) return;
  float inv = 1.f / den;
  if (den == 0.f)
    inv = rec.blocks == kRefused || (n > 0 && sees(A, row_of(A, rec.row / kMaxDrafts), j)) ? NAN : 0.f;
  f16x4 y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = static_cast<f16>(as_f32_value(o[e] * inv));
  *reinterpret_cast<f16x4*>(out + (size_t)id * D + 4 * lane) = y;
}

int teams_of(int Hkv) { return max(1, kWorkgroups / Hkv); }

size_t round16(size_t n) { return (n + 15) / 16 * 16; }

struct Layout {
  size_t rec, o, ml, total;  // bytes
};
Layout layout(int tokens, int Hq, int Hkv) {
  Layout l{};
  size_t at = 0;
  const auto take = [&](size_t bytes) {
    const size_t p = at;
    at += round16(bytes);
    return p;
  };
  const size_t vectors = ((size_t)teams_of(Hkv) * kTileVec + (size_t)tokens * (Hq / Hkv)) * Hkv;
  l.rec = take(sizeof(TokRec) * tokens);
  l.o = take(vectors * D * sizeof(float));
  l.ml = take(vectors * 2 * sizeof(float));
  l.total = at;
  return l;
}

// Sizes that the MFMA kernel takes; others run the generic one (which takes 107, 544 and 2104 us for the three above, and 13
// where this takes 9: 7 tokens over 97).
bool fast_sizes(int tokens, int batch, int Hq, int Hkv, int head_dim, int P, int max_pages, int kv_dtype) {
  const long blocks = (long)max_pages * P / kBlock + 1 + kItemCost;
  const long tiles = (long)tokens * (Hq / Hkv) / kTileVec + batch;
  return kv_dtype == CIR_F16 && head_dim == D && P % 16 == 0 && Hq / Hkv <= kMaxGroup && batch <= kMaxRows &&
         (long)max_pages * P / 16 * (P / 16) < (1L << 32) && (long)max_pages * P < (1L << 31) - 4096 &&
         blocks * tiles < (1L << 31) - kWorkgroups;
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
  // (the larger of the two paths: the addresses, which are not known here, decide between them too)
  const GenericPlan g = generic_plan(tokens, batch, num_heads, num_kv_heads, page_size, max_pages);
  const size_t plain = generic_floats(g, tokens, num_heads, head_dim) * sizeof(float);
  if (!fast_sizes(tokens, batch, num_heads, num_kv_heads, head_dim, page_size, max_pages, kv_dtype)) return plain;
  return std::max(plain, layout(tokens, num_heads, num_kv_heads).total);
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
  const float scale_log2 = scale * kLog2e;
  hipStream_t s = as_stream(stream);
  Args A{page_table, seq_lens, offsets, counts, reinterpret_cast<const uint32_t*>(masks), nullptr, nullptr, tokens, batch,
         num_heads, num_kv_heads, head_dim, page_size, max_pages, words, 1,
         scale_log2 == 0.f ? FLT_MIN : scale_log2};  // (a masked score is -inf: -inf * 0 would be NaN)
  // DMA takes 16-byte groups of the pools; q is read by 16 bytes, out written by 8.
  if (fast_sizes(tokens, batch, num_heads, num_kv_heads, head_dim, page_size, max_pages, kv_dtype) &&
      ((uintptr_t)q | (uintptr_t)k_pool | (uintptr_t)v_pool) % 16 == 0 && (uintptr_t)out % 8 == 0) {
    const Layout l = layout(tokens, num_heads, num_kv_heads);
    CIR_CHECK_ARG(workspace && workspace_bytes >= l.total && (uintptr_t)workspace % 16 == 0,
                  "tree_attention: workspace too small or not on 16 bytes (%zu < %zu)", workspace_bytes, l.total);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    const uint32_t P16 = page_size / 16, G = num_heads / num_kv_heads;
    const Fast F{A, reinterpret_cast<TokRec*>(ws + l.rec), reinterpret_cast<float*>(ws + l.o),
                 reinterpret_cast<float*>(ws + l.ml), (int)P16, (uint32_t)(((1ull << 32) + P16 - 1) / P16),
                 (uint32_t)(((1ull << 32) + G - 1) / G)};
    tree_f16_d128<<<teams_of(num_kv_heads) * num_kv_heads, kThreads, 0, s>>>(
        static_cast<const f16*>(q), static_cast<const f16*>(k_pool), static_cast<const f16*>(v_pool), page_table, F);
    const int st = launch_status();
    if (st) return st;
    tree_join<<<((unsigned)tokens * num_heads + kJoinVec - 1) / kJoinVec, 32 * kJoinVec, 0, s>>>(F, static_cast<f16*>(out));
    return launch_status();
  }
  const GenericPlan g = generic_plan(tokens, batch, num_heads, num_kv_heads, page_size, max_pages);
  const size_t floats = generic_floats(g, tokens, num_heads, head_dim), need = floats * sizeof(float);
  CIR_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need && (uintptr_t)workspace % 16 == 0),
                "tree_attention: workspace too small or not on 16 bytes (%zu < %zu)", workspace_bytes, need);
  A.part_ml = static_cast<float*>(workspace);
  A.part_o = A.part_ml + 2 * (size_t)tokens * num_heads * g.splits;
  A.splits = g.splits;
  A.scale_log2 = scale_log2;
  const auto go = [&]<typename T>() {
    const dim3 grid(g.tiles, num_kv_heads, g.splits);
    const T *qt = static_cast<const T*>(q), *kt = static_cast<const T*>(k_pool), *vt = static_cast<const T*>(v_pool);
    const auto sized = [&]<int DM>() {
      if (head_dim % 4 == 0) tree_generic<T, DM, true><<<grid, kGenThreads, 0, s>>>(qt, kt, vt, static_cast<T*>(out), A);
      else tree_generic<T, DM, false><<<grid, kGenThreads, 0, s>>>(qt, kt, vt, static_cast<T*>(out), A);
    };
    if (head_dim <= 64) sized.template operator()<64>();
    else if (head_dim <= 128) sized.template operator()<128>();
    else sized.template operator()<256>();
    const int st = launch_status();
    if (st || g.splits == 1) return st;
    const unsigned wgs = (unsigned)(((long)tokens * num_heads + kGenWaves - 1) / kGenWaves);
    tree_generic_join<T><<<wgs, kGenThreads, 0, s>>>(static_cast<T*>(out), A);
    return launch_status();
  };
  return kv_dtype == CIR_F16 ? go.template operator()<f16>() : go.template operator()<float>();
}
