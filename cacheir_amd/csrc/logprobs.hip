// Log probabilities of given tokens, entropy and the most likely alternatives of rows of
// logits, in one pass over the logits.
//
// With m = max x, S = sum e^(x - m) and T = sum e^(x - m) (x - m):
//   log p(i) = x_i - m - log S,   H = -sum p log p = log S - T / S
// (both terms of H are positive: no cancellation).  Each thread keeps (m, S, T) in fp32 over
// its share and rescales when its maximum moves: with a = e^(m - m'), S' = a S and
// T' = a (T + (m - m') S).  The alternatives are the K largest by (value, then lowest
// index): a wavefront keeps the best 64 of its share sorted across its lanes, as 64-bit keys
// (order-preserving bits of the value | complement of the index), and inserts what beats
// the K-th.  Wavefronts, then workgroups of a row, are merged in order, so results do not
// depend on timing.
//
// Bound by the read of the logits.
#include "common.hpp"

#include <float.h>
#include <math.h>

namespace cir {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxTop = 64;       // a wavefront's lanes
constexpr int kMinChunk = 4096;   // logits of a workgroup that shares its row with others
constexpr float kLog2e = 1.4426950408889634f;
// e^-200 is zero in fp32: differences below it add nothing, and 0 * (x - m) stays 0 for x = -inf.
constexpr float kFloor = -200.f;

typedef unsigned long long u64;

// Larger key = larger value (NaN above all, -0 as 0), then lower index.
__device__ __forceinline__ u64 make_key(float v, int i) {
  uint32_t b = __builtin_bit_cast(uint32_t, v + 0.f);
  b = (v != v) ? 0xffffffffu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
  return ((u64)b << 32) | (uint32_t)~i;
}
__device__ __forceinline__ float key_value(u64 k) {
  const uint32_t b = (uint32_t)(k >> 32);
  if (b == 0xffffffffu) return NAN;
  return __builtin_bit_cast(float, (b & 0x80000000u) ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ int key_index(u64 k) { return (int)~(uint32_t)k; }

__device__ __forceinline__ u64 read_lane(u64 v, int l) {
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)v, l), hi = __builtin_amdgcn_readlane((int)(v >> 32), l);
  return ((u64)hi << 32) | lo;
}

struct Stats {
  float m, s, t;
};
__device__ __forceinline__ void raise(Stats& a, float m) {  // to a maximum m >= a.m
  const float d = fmaxf(a.m - m, kFloor), f = __builtin_amdgcn_exp2f(d * kLog2e);
  a.t = f * fmaf(d, a.s, a.t);
  a.s *= f;
  a.m = m;
}
__device__ __forceinline__ void add(Stats& a, float x) {  // x <= a.m, or NaN or +inf (S becomes NaN)
  const float d = x - a.m, e = __builtin_amdgcn_exp2f(d * kLog2e);
  a.s += e;
  a.t = fmaf(e, fmaxf(d, kFloor), a.t);
}
__device__ __forceinline__ Stats join(Stats a, Stats b) {
  const float m = fmaxf(a.m, b.m);
  raise(a, m);
  raise(b, m);
  return {m, a.s + b.s, a.t + b.t};
}

// The wavefront's sorted list: lane i holds the i-th best key (0: none).
struct Top {
  u64 key, least;  // least: the K-th best (uniform)
  __device__ __forceinline__ void init() { key = least = 0; }
  // Every lane offers one key (0: none).
  __device__ __forceinline__ void offer(u64 k, int K, int lane) {
    u64 want = __builtin_amdgcn_ballot_w64(k > least);
    while (want) {  // uniform
      const int l = __builtin_ctzll(want);
      const u64 b = read_lane(k, l);
      const int at = __builtin_popcountll(__builtin_amdgcn_ballot_w64(key > b));
      const u64 up = __shfl_up(key, 1);
      key = lane < at ? key : lane == at ? b : up;
      least = read_lane(key, K - 1);
      want = __builtin_amdgcn_ballot_w64(k > least) & ~((2ull << l) - 1);
    }
  }
};

template <typename T>
struct Words;
template <>
struct Words<float> {
  static constexpr int kN = 4;
  typedef float vec __attribute__((ext_vector_type(4)));
};
template <>
struct Words<f16> {
  static constexpr int kN = 8;
  typedef f16 vec __attribute__((ext_vector_type(8)));
};

struct Out {
  float* lp;
  float* entropy;
  int64_t* top_ids;
  float* top_lp;
};

// A row's results from its whole statistics (valid in every lane of the wavefront) and list.
__device__ __forceinline__ void finish(const Out& o, int64_t row, const Stats& a, const Top& top, int K, float x,
                                       bool known, int lane) {
  // no probability anywhere (logits of -inf alone): NaN, as the log of 0 / 0
  const float log_s = a.s > 0.f || a.s != a.s ? logf(a.s) : NAN;
  if (lane == 0) {
    if (o.lp) o.lp[row] = known ? (x - a.m) - log_s : NAN;
    o.entropy[row] = log_s - a.t / a.s;
  }
  if (lane < K) {
    const int64_t at = row * K + lane;
    o.top_ids[at] = key_index(top.key);
    o.top_lp[at] = (key_value(top.key) - a.m) - log_s;
  }
}

// One workgroup per (row, split): grid x = row * S + split.
template <typename T, bool TOP>
__global__ __launch_bounds__(kThreads) void logprobs_kernel(const T* __restrict__ logits, int64_t ld,
                                                            const int64_t* __restrict__ ids, int vocab, int K, int S,
                                                            Out out, float* __restrict__ part,
                                                            u64* __restrict__ part_top) {
  constexpr int N = Words<T>::kN, U = 4;
  typedef typename Words<T>::vec vec;
  __shared__ float sm[kWaves][3];
  __shared__ u64 sm_top[kWaves][kMaxTop];
  const int64_t row = blockIdx.x / (unsigned)S;
  const int split = blockIdx.x % (unsigned)S;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const T* x = logits + row * ld;
  // Vectors of 16 aligned bytes: `skip` values before the first, then nv vectors, then a tail.
  const int skip = min(vocab, (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(T));
  const int nv = (vocab - skip) / N, tail = skip + nv * N;
  const int per = (nv + S - 1) / S, v0 = min(nv, split * per), v1 = min(nv, v0 + per);
  const vec* xv = reinterpret_cast<const vec*>(x + skip);

  Stats a = {-FLT_MAX, 0.f, 0.f};
  Top top;
  top.init();
  const auto one = [&](bool have, int i) __attribute__((always_inline)) {  // a value of the head or tail
    const float v = have ? to_f32(x[i]) : -INFINITY;
    raise(a, fmaxf(a.m, v));
    if (have) add(a, v);
    if (TOP) top.offer(have ? make_key(v, i) : 0, K, lane);
  };
  if (split == 0 && wave == 0 && skip) one(lane < skip, lane);
  for (int base = v0 + wave * 64; base < v1; base += kThreads * U) {  // uniform
    vec w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = base + u * kThreads + lane;
      if (i < v1) w[u] = xv[i];
      else
#pragma unroll
        for (int e = 0; e < N; ++e) w[u][e] = (T)-INFINITY;
    }
    float v[U][N], mx = -FLT_MAX;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        v[u][e] = to_f32(w[u][e]);
        mx = fmaxf(mx, v[u][e]);
      }
    if (mx > a.m) raise(a, mx);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < N; ++e) add(a, v[u][e]);
    if (TOP) {
      // A value equal to the K-th best cannot enter: what the list holds came earlier, at lower indices.  A NaN (or an
      // infinity) has made the sum NaN, and is looked for value by value from then on.
      const float least = key_value(top.least);
      const bool look = top.least == 0 || mx > least || a.s != a.s;
      if (__builtin_amdgcn_ballot_w64(look)) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int i = base + u * kThreads + lane;
#pragma unroll
          for (int e = 0; e < N; ++e) top.offer(i < v1 ? make_key(v[u][e], skip + i * N + e) : 0, K, lane);
        }
      }
    }
  }
  if (split == S - 1 && wave == kWaves - 1 && tail < vocab) one(tail + lane < vocab, tail + lane);

#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const Stats b = {__shfl_xor(a.m, off), __shfl_xor(a.s, off), __shfl_xor(a.t, off)};
    a = (lane & off) ? join(b, a) : join(a, b);
  }
  if (lane == 0) {
    sm[wave][0] = a.m;
    sm[wave][1] = a.s;
    sm[wave][2] = a.t;
  }
  if (TOP) sm_top[wave][lane] = top.key;
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int w = 1; w < kWaves; ++w) {
    a = join(a, Stats{sm[w][0], sm[w][1], sm[w][2]});
    if (TOP) top.offer(lane < K ? sm_top[w][lane] : 0, K, lane);
  }
  if (S == 1) {
    const int64_t id = ids ? ids[row] : -1;
    const bool known = id >= 0 && id < vocab;
    finish(out, row, a, top, TOP ? K : 0, known ? to_f32(x[id]) : 0.f, known, lane);
    return;
  }
  if (lane == 0) {
    float* p = part + (size_t)blockIdx.x * 3;
    p[0] = a.m;
    p[1] = a.s;
    p[2] = a.t;
  }
  if (TOP && lane < K) part_top[(size_t)blockIdx.x * K + lane] = top.key;
}

// Joins the S splits of a row, one wavefront per row.
template <typename T, bool TOP>
__global__ __launch_bounds__(64) void logprobs_merge(const T* __restrict__ logits, int64_t ld,
                                                     const int64_t* __restrict__ ids, int vocab, int K, int S, Out out,
                                                     const float* __restrict__ part, const u64* __restrict__ part_top) {
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x;
  const int64_t id = ids ? ids[row] : -1;
  const bool known = id >= 0 && id < vocab;
  const float x = known ? to_f32(logits[row * ld + id]) : 0.f;
  Stats a = {-FLT_MAX, 0.f, 0.f};
  if (lane < S) {  // (S <= 64)
    const float* p = part + (row * S + lane) * 3;
    a = {p[0], p[1], p[2]};
  }
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const Stats b = {__shfl_xor(a.m, off), __shfl_xor(a.s, off), __shfl_xor(a.t, off)};
    a = (lane & off) ? join(b, a) : join(a, b);
  }
  Top top;
  top.init();
  if (TOP) {
    const u64* p = part_top + row * S * K;
    for (int i = 0; i < S * K; i += 64) top.offer(i + lane < S * K ? p[i + lane] : 0, K, lane);
  }
  finish(out, row, a, top, TOP ? K : 0, x, known, lane);
}

// Workgroups that share a row: enough for two per CU, each with kMinChunk logits at least.
int row_splits(int rows, int vocab) {
  const int fill = 512 / max(1, min(rows, 512)), most = max(1, vocab / kMinChunk);
  return max(1, min(min(fill, most), 64));
}

}  // namespace
}  // namespace cir

using namespace cir;

extern "C" size_t cir_token_logprobs_workspace_bytes(int rows, int vocab, int top_k) {
  if (rows <= 0 || vocab <= 0 || top_k < 0) return 0;
  const int S = row_splits(rows, vocab);
  return S == 1 ? 0 : (size_t)rows * S * ((size_t)top_k * sizeof(u64) + 3 * sizeof(float));
}

extern "C" int cir_token_logprobs(const void* logits, int dt, int64_t ld, const int64_t* ids, int rows, int vocab,
                                  int top_k, float* logprobs, float* entropy, int64_t* top_ids, float* top_logprobs,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  CIR_CHECK_ARG(dt == CIR_F32 || dt == CIR_F16, "token_logprobs: bad dtype");
  CIR_CHECK_ARG(rows >= 0 && vocab > 0 && ld >= vocab, "token_logprobs: bad sizes");
  CIR_CHECK_ARG(top_k >= 0 && top_k <= kMaxTop && top_k <= vocab, "token_logprobs: top_k %d out of range (0..%d, at most "
                "the vocabulary)", top_k, kMaxTop);
  if (rows == 0) return 0;
  CIR_CHECK_ARG(logits && entropy && (!ids || logprobs) && (top_k == 0 || (top_ids && top_logprobs)),
                "token_logprobs: null pointer");
  CIR_CHECK_ARG((uintptr_t)logits % (dt == CIR_F16 ? 2 : 4) == 0, "token_logprobs: logits off their type's alignment");
  const int S = row_splits(rows, vocab);
  const size_t need = cir_token_logprobs_workspace_bytes(rows, vocab, top_k);
  CIR_CHECK_ARG((workspace || need == 0) && workspace_bytes >= need && (uintptr_t)workspace % 8 == 0,
                "token_logprobs: workspace too small or not on 8 bytes (%zu < %zu)", workspace_bytes, need);
  CIR_CHECK_ARG((long)rows * S < (1L << 31), "token_logprobs: grid too large");
  hipStream_t s = as_stream(stream);
  const Out out{ids ? logprobs : nullptr, entropy, top_ids, top_logprobs};
  u64* part_top = static_cast<u64*>(workspace);
  float* part = reinterpret_cast<float*>(part_top + (size_t)rows * S * top_k);
  const auto go = [&]<typename T, bool TOP>() {
    const T* x = static_cast<const T*>(logits);
    logprobs_kernel<T, TOP><<<(unsigned)(rows * S), kThreads, 0, s>>>(x, ld, ids, vocab, top_k, S, out, part, part_top);
    const int st = launch_status();
    if (st || S == 1) return st;
    logprobs_merge<T, TOP><<<rows, 64, 0, s>>>(x, ld, ids, vocab, top_k, S, out, part, part_top);
    return launch_status();
  };
  if (dt == CIR_F16) return top_k ? go.template operator()<f16, true>() : go.template operator()<f16, false>();
  return top_k ? go.template operator()<float, true>() : go.template operator()<float, false>();
}
