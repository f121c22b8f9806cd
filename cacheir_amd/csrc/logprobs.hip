// Log probabilities of given tokens, entropy and the most likely alternatives of rows of
// logits, in one pass over the logits.
//
// In base 2, with a reference r near max x, y = (x - r) log2 e, S = sum 2^y, T = sum 2^y y:
//   log p(i) = ln 2 (y_i - log2 S),   H = -sum p log p = ln 2 (log2 S - T / S)
// (both terms of H are positive: no cancellation).  Each thread keeps (r, S, T) in fp32 over
// its share and rescales when its maximum moves: with d = (r - r') log2 e, S' = 2^d S and
// T' = 2^d (T + d S).
//
// The alternatives are the K largest by (value, then lowest index), as 64-bit keys
// (order-preserving bits of the value | complement of the index).  While it streams, a lane
// only keeps the largest value of each of up to kCells stretches of its share ("cells"), which
// the statistics need anyway.  The K-th largest of a wavefront's 64 lane maxima bounds the
// row's K-th largest value from below; so does the largest such bound of the row's
// wavefronts.  The values that reach the bound lie in the few cells whose maximum does:
// those are read again, what reaches the bound is gathered in LDS, sorted by a bitonic
// network and kept as the wavefront's list, 64 keys across its lanes.  Where too many cells
// qualify (equal logits, a mask that leaves less than K tokens) or a NaN is about, the share
// is walked in order instead, past every group that cannot change the list.  Sorted lists
// are joined in 7 exchange steps: wavefronts, then workgroups of a row, in order, so results
// do not depend on timing.  (Inserting what beat a running K-th best as it streamed by took
// 101 us where this took 67, 1021 x 152064 fp16 and K = 2.)
//
// Bound by the read of the logits: 1021 x 152064 fp16 62 us with two alternatives and 55
// without (5.0 and 5.6 TB/s; without the exponentials 58 and 53); 32 x 128256 fp32 with 20 by
// the latency of two launches (10.5 and 4.6 us).
#include "common.hpp"

#include <float.h>
#include <math.h>

namespace cir {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxTop = 64;       // a wavefront's lanes
constexpr int kCells = 16;        // maxima a lane keeps
constexpr int kPicks = 128;       // cells of a wavefront that are read again
constexpr int kKeys = 256;        // keys a wavefront gathers
constexpr int kAhead = 8;         // values per lane that are read again at once
constexpr int kMinChunk = 4096;   // logits of a workgroup that shares its row with others
// Logits that the last cache cannot hold are read past it (1021 x 152064 fp16 66.9 -> 62.5 us; 32 x 128256, which a
// product has just written, 14.6 -> 15.4).
constexpr size_t kCacheBytes = (size_t)256 << 20;
constexpr int kManyRows = 1024;   // rows of one wavefront each, where they are short
constexpr int kMaxRows = 1 << 24;  // (rows * kThreads < 2^32)
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// 2^-300 is zero in fp32: y below it adds nothing, and 0 * y stays 0 for x = -inf.
constexpr float kFloor = -300.f;

typedef unsigned long long u64;

// Order-preserving bits (NaN aside).
__device__ __forceinline__ uint32_t rank_bits(float v) {
  const uint32_t b = __builtin_bit_cast(uint32_t, v + 0.f);
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float rank_value(uint32_t b) {
  return __builtin_bit_cast(float, (b & 0x80000000u) ? b & 0x7fffffffu : ~b);
}
// Larger key = larger value (NaN above all, -0 as 0), then lower index.
__device__ __forceinline__ u64 make_key(float v, int i) {
  return ((u64)((v != v) ? 0xffffffffu : rank_bits(v)) << 32) | (uint32_t)~i;
}
__device__ __forceinline__ float key_value(u64 k) {
  const uint32_t b = (uint32_t)(k >> 32);
  return b == 0xffffffffu ? NAN : rank_value(b);
}
__device__ __forceinline__ int key_index(u64 k) { return (int)~(uint32_t)k; }

__device__ __forceinline__ u64 read_lane(u64 v, int l) {
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)v, l), hi = __builtin_amdgcn_readlane((int)(v >> 32), l);
  return ((u64)hi << 32) | lo;
}

// fp32 logits: the reference is the maximum itself.  fp16 logits: it is fl(max log2 e), so that y is one mixed-precision
// FMA on the logit as it was loaded (values up to 65504: no overflow); the rounding of the reference is shared by all.
template <typename T>
struct Words;
template <>
struct Words<float> {
  static constexpr int kN = 4, kUnroll = 4;
  typedef float vec __attribute__((ext_vector_type(4)));
  static __device__ __forceinline__ float ref_of(float m) { return m; }
  static __device__ __forceinline__ float y_of(float x, float ref) { return (x - ref) * kLog2e; }
  static __device__ __forceinline__ float gap(float ref, float to) { return (ref - to) * kLog2e; }
  static __device__ __forceinline__ float log_p(float x, float ref, float log2_s) { return (x - ref) - log2_s * kLn2; }
};
template <>
struct Words<f16> {
  static constexpr int kN = 8, kUnroll = 4;
  typedef f16 vec __attribute__((ext_vector_type(8)));
  // (as_f32_value: contracted into the subtraction in gap, the unrounded product would not cancel)
  static __device__ __forceinline__ float ref_of(float m) { return as_f32_value(m * kLog2e); }
  static __device__ __forceinline__ float y_of(f16 x, float ref) { return fmaf((float)x, kLog2e, -ref); }
  static __device__ __forceinline__ float gap(float ref, float to) { return ref - to; }
  static __device__ __forceinline__ float log_p(f16 x, float ref, float log2_s) { return (y_of(x, ref) - log2_s) * kLn2; }
};

__device__ __forceinline__ uint32_t read_lane32(uint32_t v, int l) {
  return (uint32_t)__builtin_amdgcn_readlane((int)v, l);
}
__device__ __forceinline__ int lanes_below(u64 m) {  // set bits of lanes before this one
  return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
}

struct Stats {
  float m, ref, s, t;
};
template <typename T>
__device__ __forceinline__ Stats none() {
  const float low = sizeof(T) == 2 ? -65504.f : -FLT_MAX;
  return {low, Words<T>::ref_of(low), 0.f, 0.f};
}
template <typename T>
__device__ __forceinline__ void raise(Stats& a, float m) {  // to a maximum m >= a.m
  const float ref = Words<T>::ref_of(m);
  const float d = fmaxf(Words<T>::gap(a.ref, ref), kFloor), f = __builtin_amdgcn_exp2f(d);
  a.t = f * fmaf(d, a.s, a.t);
  a.s *= f;
  a.ref = ref;
  a.m = m;
}
template <typename T>
__device__ __forceinline__ void add(Stats& a, T x) {  // x <= a.m, or NaN or +inf (S becomes NaN)
  const float y = Words<T>::y_of(x, a.ref), e = __builtin_amdgcn_exp2f(y);
  a.s += e;
  a.t = fmaf(e, fmaxf(y, kFloor), a.t);
}
template <typename T>
__device__ __forceinline__ Stats join(Stats a, Stats b) {
  const float m = fmaxf(a.m, b.m);
  raise<T>(a, m);
  raise<T>(b, m);
  return {m, a.ref, a.s + b.s, a.t + b.t};
}
template <typename T>
__device__ __forceinline__ Stats join_wave(Stats a) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const Stats b = {__shfl_xor(a.m, off), __shfl_xor(a.ref, off), __shfl_xor(a.s, off), __shfl_xor(a.t, off)};
    a = join<T>(a, b);
  }
  return a;
}

// The key of lane ^ MASK, by DPP inside a row of 16 lanes and gfx950's lane swaps past it.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false);
}
template <int MASK>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v) {
  if constexpr (MASK == 1) return dpp<0xB1>(v);              // quad_perm [1,0,3,2]
  else if constexpr (MASK == 2) return dpp<0x4E>(v);         // quad_perm [2,3,0,1]
  else if constexpr (MASK == 4) return dpp<0x1B>(dpp<0x141>(v));  // half-row mirror (^7), quad_perm [3,2,1,0] (^3)
  else if constexpr (MASK == 8) return dpp<0x128>(v);        // row_ror:8
  else if constexpr (MASK == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);  // (r0, r0, r2, r2), (r1, r1, r3, r3) by rows
    const uint32_t a = r[0], b = r[1];
    return (threadIdx.x & 16) ? a : b;
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);  // (low, low), (high, high) halves
    const uint32_t a = r[0], b = r[1];
    return (threadIdx.x & 32) ? a : b;
  }
}
// Compare-exchange with lane ^ MASK; `up`: this lane keeps the larger key.
template <int MASK>
__device__ __forceinline__ void exchange(u64& k, bool up) {
  const u64 o = ((u64)lane_xor<MASK>((uint32_t)(k >> 32)) << 32) | lane_xor<MASK>((uint32_t)k);
  k = (k > o) == up ? k : o;
}
template <int MASK>
__device__ __forceinline__ void exchange(uint32_t& k, bool up) {
  const uint32_t o = lane_xor<MASK>(k), hi = max(k, o), lo = min(k, o);
  k = up ? hi : lo;
}
template <int MASK, typename Key>
__device__ __forceinline__ void merge_steps(Key& k, int lane, bool desc) {  // a bitonic run of 2 MASK lanes, sorted
  exchange<MASK>(k, ((lane & MASK) == 0) == desc);
  if constexpr (MASK > 1) merge_steps<MASK / 2>(k, lane, desc);
}

template <typename Key>
__device__ __forceinline__ Key sorted(Key k, int lane) {  // one key per lane, the largest in lane 0
  merge_steps<1>(k, lane, (lane & 2) == 0);
  merge_steps<2>(k, lane, (lane & 4) == 0);
  merge_steps<4>(k, lane, (lane & 8) == 0);
  merge_steps<8>(k, lane, (lane & 16) == 0);
  merge_steps<16>(k, lane, (lane & 32) == 0);
  merge_steps<32>(k, lane, true);
  return k;
}

// The wavefront's list: lane i holds the i-th best key (0: none).
struct Top {
  u64 key, least;  // least: the K-th best (uniform)
  // Joins another sorted list: the larger of lane i and lane 63 - i of the other are the best 64, as a bitonic run.
  __device__ __forceinline__ void join(u64 k, int K, int lane) {
    const u64 o = __shfl(k, 63 - lane);
    key = key > o ? key : o;
    merge_steps<32>(key, lane, true);
    least = read_lane(key, K - 1);
  }
  // Every lane offers one key (0: none).
  __device__ __forceinline__ void absorb(u64 k, int K, int lane) {
    if (!__builtin_amdgcn_ballot_w64(k > least)) return;
    k = sorted(k, lane);
    if (read_lane(key, 0) != 0) {  // uniform
      join(k, K, lane);
    } else {
      key = k;
      least = read_lane(key, K - 1);
    }
  }
};

struct Out {
  float* lp;
  float* entropy;
  int64_t* top_ids;
  float* top_lp;
};

// A row's results from its whole statistics (valid in every lane of the wavefront) and list; x: the given token's logit.
template <typename T>
__device__ __forceinline__ void finish(const Out& o, int64_t row, const Stats& a, const Top& top, int K, T x, bool known,
                                       int lane) {
  // no probability anywhere (logits of -inf alone): NaN, as the log of 0 / 0
  const float log_s = a.s > 0.f || a.s != a.s ? log2f(a.s) : NAN;
  if (lane == 0) {
    if (o.lp) o.lp[row] = known ? Words<T>::log_p(x, a.ref, log_s) : NAN;
    o.entropy[row] = (log_s - a.t / a.s) * kLn2;
  }
  if (lane < K) {
    const int64_t at = row * K + lane;
    o.top_ids[at] = key_index(top.key);
    o.top_lp[at] = Words<T>::log_p(from_f32<T>(key_value(top.key)), a.ref, log_s);
  }
}

// WPR wavefronts per row: four, one workgroup per (row, split), grid x = row * S + split; or one, four rows per
// workgroup (S = 1).  U vectors per lane and group; ONE: every wavefront's share is one group (what may enter the list
// is then taken from registers); ONCE: non-temporal loads.
template <typename T, bool TOP, int WPR, int U, bool ONE, bool ONCE>
__global__ __launch_bounds__(kThreads) void logprobs_kernel(const T* __restrict__ logits, int64_t ld,
                                                            const int64_t* __restrict__ ids, int rows, int vocab, int K,
                                                            int S, Out out, float* __restrict__ part,
                                                            u64* __restrict__ part_top) {
  typedef Words<T> W;
  constexpr int N = W::kN;
  typedef typename W::vec vec;
  __shared__ float sm[kWaves][4];
  __shared__ float sm_cell[TOP && !ONE ? kWaves : 1][TOP && !ONE ? kCells : 1][64];
  __shared__ u64 sm_keys[TOP ? kWaves : 1][TOP ? kKeys : 1];
  __shared__ int sm_pick[TOP && !ONE ? kWaves : 1][TOP && !ONE ? kPicks : 1], sm_n[kWaves];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int64_t row = WPR == 1 ? (int64_t)blockIdx.x * kWaves + wave : blockIdx.x / (unsigned)S;
  const int split = WPR == 1 ? 0 : blockIdx.x % (unsigned)S, turn = WPR == 1 ? 0 : wave;
  if (WPR == 1 && row >= rows) return;
  const T* x = logits + row * ld;
  // Vectors of 16 aligned bytes: `skip` values before the first, then nv vectors, then a tail.
  const int skip = min(vocab, (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(T));
  const int nv = (vocab - skip) / N, tail = skip + nv * N;
  const int per = (nv + S - 1) / S, v0 = min(nv, split * per), v1 = min(nv, v0 + per);
  const vec* xv = reinterpret_cast<const vec*>(x + skip);
  // The given token's logit, on its way meanwhile.
  const int64_t id = S == 1 && ids ? ids[row] : -1;
  const bool known = id >= 0 && id < vocab;
  const T given = x[known ? id : 0];

  // This wavefront's groups: vectors base0 + g * kGroup + u * 64 WPR + lane, u < U; cells of `wide` groups.
  constexpr int kGroup = 64 * WPR * U;
  const int base0 = v0 + turn * 64;
  const int groups = base0 < v1 ? (ONE ? 1 : (v1 - base0 + kGroup - 1) / kGroup) : 0;
  const int wide = (groups + kCells - 1) / kCells;
  Stats a = none<T>();
  float most = -INFINITY;  // the lane's largest value (NaN aside)
  const auto load = [&](vec (&w)[U], int base) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = base + u * 64 * WPR + lane;
      if (i < v1) w[u] = ONCE ? __builtin_nontemporal_load(xv + i) : xv[i];
      else
#pragma unroll
        for (int e = 0; e < N; ++e) w[u][e] = (T)-INFINITY;
    }
  };
  const auto take = [&](const vec (&w)[U]) __attribute__((always_inline)) {  // into the statistics; the largest value
    vec top_of = w[0];
#pragma unroll
    for (int u = 1; u < U; ++u) top_of = __builtin_elementwise_max(top_of, w[u]);
    float mx = to_f32(top_of[0]);
#pragma unroll
    for (int e = 1; e < N; ++e) mx = fmaxf(mx, to_f32(top_of[e]));
    if (mx > a.m) raise<T>(a, mx);
    // (a sum of its own per group: next to a likely token's 1 hundreds of terms below 2^-25 would be lost one by one)
    Stats b = {a.m, a.ref, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < N; ++e) add<T>(b, w[u][e]);
    a.s += b.s;
    a.t += b.t;
    return mx;
  };
  vec one[ONE ? U : 1];
  if constexpr (ONE) {
    load(one, base0);
    most = take(one);
  } else {
    float cell = -INFINITY;
    for (int g = 0; g < groups; ++g) {  // uniform
      vec w[U];
      load(w, base0 + g * kGroup);
      const float mx = take(w);
      if constexpr (TOP) {
        cell = fmaxf(cell, mx);
        if ((g + 1) % wide == 0 || g + 1 == groups) {  // uniform
          sm_cell[wave][g / wide][lane] = cell;
          most = fmaxf(most, cell);
          cell = -INFINITY;
        }
      }
    }
  }
  // The values before the first vector and behind the last one (at most N - 1 each), one per lane.
  const bool has_head = split == 0 && turn == 0 && skip > 0, has_tail = split == S - 1 && turn == WPR - 1 && tail < vocab;
  const int end_at = has_head && lane < skip                            ? lane
                     : has_tail && lane >= 32 && tail + lane - 32 < vocab ? tail + lane - 32
                                                                        : -1;
  if (has_head || has_tail) {
    const T v = end_at >= 0 ? x[end_at] : (T)-INFINITY;
    raise<T>(a, fmaxf(a.m, to_f32(v)));
    if (end_at >= 0) add<T>(a, v);
  }

  Top top{0, 0};
  if constexpr (TOP) {
    // The bound: at least K values of the row reach it.
    float bound = rank_value(read_lane32(sorted(rank_bits(most), lane), K - 1));
    const bool odd = __builtin_amdgcn_ballot_w64(a.s != a.s) != 0;  // uniform: a NaN or an infinity
    if (WPR > 1) {
      if (lane == 0) sm[wave][3] = bound;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kWaves; ++w) bound = fmaxf(bound, sm[w][3]);
    }
    int n = 0;  // keys gathered, uniform
    const auto gather = [&](bool may, float v, int at) __attribute__((always_inline)) {
      const u64 m = __builtin_amdgcn_ballot_w64(may);
      if (m) {
        const int to = n + lanes_below(m);
        if (may && to < kKeys) sm_keys[wave][to] = make_key(v, at);
        n += __builtin_popcountll(m);
      }
    };
    if (has_head || has_tail) gather(end_at >= 0, end_at >= 0 ? to_f32(x[end_at]) : 0.f, end_at);
    const int ends = n;  // (at most 2 N - 2, those before the first vector first)
    int picks = 0;  // uniform
    if constexpr (ONE) {
      if (!odd) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int i = base0 + u * 64 * WPR + lane;
#pragma unroll
          for (int e = 0; e < N; ++e) {
            const float v = to_f32(one[u][e]);
            gather(i < v1 && v >= bound, v, skip + i * N + e);
          }
        }
      }
    } else if (!odd) {
      // The cells that reach the bound.
      const int cells = wide ? (groups + wide - 1) / wide : 0;
      for (int c = 0; c < cells; ++c) {
        const u64 hit = __builtin_amdgcn_ballot_w64(sm_cell[wave][c][lane] >= bound);
        const int at = picks + lanes_below(hit);
        if (((hit >> lane) & 1) && at < kPicks) sm_pick[wave][at] = c * 64 + lane;
        picks += __builtin_popcountll(hit);
      }
      if (picks <= kPicks) {
        for (int g = 0; g < wide; ++g)                                 // (group of the cell)
          for (int j0 = 0; j0 < picks * U * N; j0 += 64 * kAhead) {    // uniform
            float v[kAhead];
            int at[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
              const int j = j0 + 64 * k + lane, p = j / (U * N), r = j % (U * N);
              const int pick = sm_pick[wave][min(p, kPicks - 1)];
              const int i = base0 + ((pick >> 6) * wide + g) * kGroup + r / N * 64 * WPR + (pick & 63);
              const bool in = p < picks && i < v1;
              at[k] = in ? skip + i * N + r % N : -1;
              v[k] = to_f32(x[in ? at[k] : 0]);
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k) gather(at[k] >= 0 && v[k] >= bound, v[k], at[k]);
          }
      }
    }
    if (picks > kPicks || n > kKeys || odd) {  // uniform
      // What lies before the groups, then the groups, then what lies behind them: a group whose values are no larger than
      // the list's least can be passed over because the list holds lower indices only.
      const int head = has_head ? skip : 0;
      top.absorb(lane < head ? sm_keys[wave][lane] : 0, K, lane);
      for (int g = 0; g < groups; ++g) {           // uniform
        const float least = key_value(top.least);  // (none yet: NaN)
        if (!ONE && !odd) {
          const float m = sm_cell[wave][ONE ? 0 : g / wide][lane];
          if (!__builtin_amdgcn_ballot_w64(m >= bound && !(m <= least))) continue;
        }
        for (int j = 0; j < U * N; ++j) {
          const int i = base0 + g * kGroup + j / N * 64 * WPR + lane, at = skip + i * N + j % N;
          const bool in = i < v1;
          const float v = to_f32(x[in ? at : 0]);
          top.absorb(in && !(v < bound) ? make_key(v, at) : 0, K, lane);
        }
      }
      top.absorb(lane >= head && lane < ends ? sm_keys[wave][lane] : 0, K, lane);
      n = 64;
      sm_keys[wave][lane] = top.key;
      top = Top{0, 0};
    }
    if (lane == 0) sm_n[wave] = n;
  }

  a = join_wave<T>(a);
  if constexpr (WPR > 1) {
    if (lane == 0) {
      sm[wave][0] = a.m;
      sm[wave][1] = a.s;
      sm[wave][2] = a.t;
    }
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) a = join<T>(a, Stats{sm[w][0], W::ref_of(sm[w][0]), sm[w][1], sm[w][2]});
  }
  if constexpr (TOP) {  // every wavefront's keys, 64 at a time
    constexpr int kOf = WPR > 1 ? kWaves : 1;
    int from[kOf + 1];
    from[0] = 0;
#pragma unroll
    for (int w = 0; w < kOf; ++w) from[w + 1] = from[w] + __builtin_amdgcn_readfirstlane(sm_n[WPR > 1 ? w : wave]);
    for (int j = 0; j < from[kOf]; j += 64) {
      int w = 0;
#pragma unroll
      for (int k = 1; k < kOf; ++k) w += j + lane >= from[k] ? 1 : 0;
      int start = 0;
#pragma unroll
      for (int k = 1; k < kOf; ++k) start = w == k ? from[k] : start;
      top.absorb(j + lane < from[kOf] ? sm_keys[WPR > 1 ? w : wave][j + lane - start] : 0, K, lane);
    }
  }
  if (S == 1) {
    finish<T>(out, row, a, top, TOP ? K : 0, given, known, lane);
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

// Joins the S <= 64 splits of a row, one wavefront per row: the K-th largest of the lanes' best keys bounds what can
// enter, what reaches it is gathered and sorted (all of it, 64 at a time, where equal values make it too much).
template <typename T, bool TOP>
__global__ __launch_bounds__(64) void logprobs_merge(const T* __restrict__ logits, int64_t ld,
                                                     const int64_t* __restrict__ ids, int vocab, int K, int S, Out out,
                                                     const float* __restrict__ part, const u64* __restrict__ part_top) {
  __shared__ u64 sm_keys[kKeys];
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x;
  const int64_t id = ids ? ids[row] : -1;
  const bool known = id >= 0 && id < vocab;
  Stats a = none<T>();
  if (lane < S) {
    const float* p = part + (row * S + lane) * 3;
    a = {p[0], Words<T>::ref_of(p[0]), p[1], p[2]};
  }
  const T x = logits[row * ld + (known ? id : 0)];
  Top top{0, 0};
  if (TOP) {
    const u64* p = part_top + row * S * K;
    const int all = S * K;
    uint32_t best = 0;
    for (int i0 = 0; i0 < all; i0 += 64 * kAhead) {
      u64 k[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) k[j] = p[min(i0 + 64 * j + lane, all - 1)];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) best = max(best, i0 + 64 * j + lane < all ? (uint32_t)(k[j] >> 32) : 0);
    }
    const uint32_t bound = read_lane32(sorted(best, lane), K - 1);
    int n = 0;
    for (int i0 = 0; i0 < all; i0 += 64 * kAhead) {
      u64 k[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) k[j] = p[min(i0 + 64 * j + lane, all - 1)];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const bool may = i0 + 64 * j + lane < all && k[j] != 0 && (uint32_t)(k[j] >> 32) >= bound;
        const u64 m = __builtin_amdgcn_ballot_w64(may);
        const int to = n + lanes_below(m);
        if (may && to < kKeys) sm_keys[to] = k[j];
        n += __builtin_popcountll(m);
      }
    }
    const bool fits = n <= kKeys;
    if (!fits) n = all;
    for (int i = 0; i < n; i += 64) top.absorb(i + lane < n ? (fits ? sm_keys[i + lane] : p[i + lane]) : 0, K, lane);
  }
  a = join_wave<T>(a);
  finish<T>(out, row, a, top, TOP ? K : 0, x, known, lane);
}

template <typename T>
constexpr int kGroupOf = 64 * 4 * Words<T>::kN;  // logits of a wavefront's group

// Workgroups that share a row: enough for two per CU, each with kMinChunk logits at least (one from 257 rows on).
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
  // A grid has fewer than 2^32 threads: one bound for all forms, which asks for a workgroup per row at most.
  CIR_CHECK_ARG(rows < kMaxRows, "token_logprobs: %d rows are too many for a launch (fewer than 2^24)", rows);
  if (rows == 0) return 0;
  CIR_CHECK_ARG(logits && entropy && (!ids || logprobs) && (top_k == 0 || (top_ids && top_logprobs)),
                "token_logprobs: null pointer");
  CIR_CHECK_ARG((uintptr_t)logits % (dt == CIR_F16 ? 2 : 4) == 0, "token_logprobs: logits off their type's alignment");
  const int S = row_splits(rows, vocab);
  const size_t need = cir_token_logprobs_workspace_bytes(rows, vocab, top_k);
  CIR_CHECK_ARG((workspace || need == 0) && workspace_bytes >= need && (uintptr_t)workspace % 8 == 0,
                "token_logprobs: workspace too small or not on 8 bytes (%zu < %zu)", workspace_bytes, need);
  const bool many = rows >= kManyRows && vocab <= 4 * (dt == CIR_F16 ? kGroupOf<f16> : kGroupOf<float>);
  hipStream_t s = as_stream(stream);
  const Out out{ids ? logprobs : nullptr, entropy, top_ids, top_logprobs};
  u64* part_top = static_cast<u64*>(workspace);
  float* part = reinterpret_cast<float*>(part_top + (size_t)rows * S * top_k);
  const auto go = [&]<typename T, bool TOP>() {
    const T* x = static_cast<const T*>(logits);
    constexpr int kGroup = kGroupOf<T>;
    const auto run = [&]<int WPR, int U, bool ONE, bool ONCE>() {
      const unsigned wgs = WPR == 1 ? (unsigned)(((long)rows + kWaves - 1) / kWaves) : (unsigned)(rows * S);
      logprobs_kernel<T, TOP, WPR, U, ONE, ONCE><<<wgs, kThreads, 0, s>>>(x, ld, ids, rows, vocab, top_k, S, out, part,
                                                                          part_top);
    };
    if (many) {
      if (vocab <= kGroup / 4) run.template operator()<1, 1, true, false>();
      else if (vocab <= kGroup) run.template operator()<1, 4, true, false>();
      else run.template operator()<1, 4, false, false>();
      return launch_status();
    }
    if (((vocab / Words<T>::kN + S - 1) / S) <= 64 * 4 * kWaves) run.template operator()<kWaves, 4, true, false>();
    else if ((size_t)rows * vocab * sizeof(T) < kCacheBytes) run.template operator()<kWaves, 4, false, false>();
    else run.template operator()<kWaves, 4, false, true>();
    const int st = launch_status();
    if (st || S == 1) return st;
    logprobs_merge<T, TOP><<<rows, 64, 0, s>>>(x, ld, ids, vocab, top_k, S, out, part, part_top);
    return launch_status();
  };
  if (dt == CIR_F16) return top_k ? go.template operator()<f16, true>() : go.template operator()<f16, false>();
  return top_k ? go.template operator()<float, true>() : go.template operator()<float, false>();
}
