// What a step needs before its attention, without the host: page tables, positions and
// slot maps from request lengths (extend_tables_kernel), and the rotary positions of q and
// k with the append of k and v to the slots of that map (rope_append_kernel).
#include "common.hpp"

#include <limits.h>

#include <utility>

namespace cir {
namespace {

bool valid_dt(int dt) { return dt == CIR_F32 || dt == CIR_F16; }

// ------------------------------------------------------------- page tables ----
// Row b holds lens[b] tokens and gets new[b] more: it needs
//   need_b = ceil((lens[b] + new[b]) / P) - ceil(lens[b] / P)
// pages, handed out in row order from free_slots[head ..]; with upto_b = need_0 + .. + need_b
// the row gets them if head + upto_b <= free_total (rows that do not fit the table or the
// slot map count no need).  Token j of row b lies at position lens[b] + j, in page
// p = pos / P: an old entry of the table for p < ceil(lens[b] / P), else
// free_slots[head + upto_b - need_b + p - ceil(lens[b] / P)], so no workgroup reads an entry
// that another writes, and every workgroup runs the scan over the rows by itself and then
// takes its span of the tokens (the first token of a new page also writes the table entry).
// Bound by latency: three dependent loads (lengths; table entry or free slot) and a block
// scan of kRows rows.  Sums saturate at kCap, above any max_tokens or free_total, so 32 bits
// hold them (64-bit sums and divisions made 128 rows of a token each 8.3 us instead of 4.3).
constexpr int kRows = 256;     // rows per scan = threads
constexpr int kSpan = 1024;    // tokens per workgroup
constexpr int kFill = 1;       // write tables, positions, slots, offsets and granted
constexpr int kAdvance = 2;    // write seq_lens_out and free_head_out
constexpr uint32_t kCap = 1u << 30;

__device__ __forceinline__ uint32_t sat_add(uint32_t a, uint32_t b) { return min(a + b, kCap); }  // (each <= kCap)

// Inclusive saturating sum over the workgroup, from `before` on; the last thread's value is the total.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t before, uint32_t* scratch) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t o = __shfl_up(v, off, 64);
    v = sat_add(v, lane >= off ? o : 0);
  }
  if (lane == 63) scratch[wave] = v;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kRows / 64; ++w) before = sat_add(before, w < wave ? scratch[w] : 0);
  return sat_add(v, before);
}
__device__ __forceinline__ uint32_t pages_of(uint32_t tokens, uint32_t P) { return tokens / P + (tokens % P ? 1 : 0); }

__global__ __launch_bounds__(kRows) void extend_tables_kernel(
    int32_t* table, const int32_t* lens, const int32_t* news, const int32_t* __restrict__ free_slots, int free_total,
    const int32_t* head_in, int32_t* lens_out, int32_t* head_out, int32_t* __restrict__ offsets,
    int32_t* __restrict__ granted, int32_t* __restrict__ positions, int64_t* __restrict__ slot_map, int batch,
    int max_pages, int P, int max_tokens, int what) {
  __shared__ uint32_t sm_tok[kRows / 64], sm_pag[kRows / 64];
  __shared__ uint32_t sm_end[kRows];  // tokens up to and with the row
  __shared__ uint32_t sm_len[kRows], sm_old[kRows];  // sm_old: pages held
  __shared__ int sm_from[kRows];      // free_slots index of the row's page 0, were it new; kNone: not granted
  __shared__ uint32_t sm_total[2];
  constexpr int kNone = INT_MIN;
  const int t = threadIdx.x;
  const bool first = blockIdx.x == 0;
  const int head = head_in[0];
  const uint32_t room = head >= 0 && head < free_total ? free_total - head : 0;  // free slots left
  const uint32_t span0 = blockIdx.x * (uint32_t)kSpan, span1 = min(span0 + kSpan, (uint32_t)max_tokens);
  uint32_t tokens = 0, pages = 0, used = 0;  // of the rows before this chunk; `used`: pages handed out
  for (int r0 = 0; r0 < batch; r0 += kRows) {  // uniform
    const int r = r0 + t;
    const bool in = r < batch;
    const uint32_t len = in ? max(lens[r], 0) : 0, add = in ? max(news[r], 0) : 0;
    const uint32_t have = pages_of(len, P), want = pages_of(len + add, P);  // (len + add < 2^32)
    const uint32_t end = block_scan(min(add, kCap), tokens, sm_tok);
    const bool fits = want <= (uint32_t)max_pages && end <= (uint32_t)max_tokens && len + add <= (uint32_t)INT_MAX;
    const uint32_t need = fits ? want - have : 0;
    const uint32_t upto = block_scan(need, pages, sm_pag);
    const bool ok = fits && (need == 0 || upto <= room);
    sm_end[t] = end;
    sm_len[t] = len;
    sm_old[t] = have;
    sm_from[t] = ok ? head + (int)(upto - need) - (int)have : kNone;
    if (t == kRows - 1) {
      sm_total[0] = end;
      sm_total[1] = upto;
    }
    // Pages of the rows served so far: `upto` grows with the row, so the largest of an ok row that needed some.
    used = (ok && need > 0) ? upto : used;
    if (first && in) {
      if (what & kFill) {
        offsets[r + 1] = (int)end;
        granted[r] = ok ? add : 0;
      }
      if (what & kAdvance) lens_out[r] = (int)(len + (ok ? add : 0));
    }
    __syncthreads();
    if (what & kFill) {
      const uint32_t lo = max(span0, tokens), hi = min(span1, sm_total[0]);
      for (uint32_t j = lo + t; j < hi; j += kRows) {
        int a = 0;  // first row whose end lies past j
#pragma unroll
        for (int step = kRows / 2; step > 0; step >>= 1) a += sm_end[a + step - 1] <= j ? step : 0;
        const uint32_t pos = sm_len[a] + (j - (a ? sm_end[a - 1] : tokens));
        const uint32_t page = pos / (uint32_t)P, off = pos - page * P;
        const int from = sm_from[a];
        int64_t slot = -1;
        if (from != kNone) {
          int32_t* entry = table + (size_t)(r0 + a) * max_pages + page;
          const int s = page < sm_old[a] ? *entry : free_slots[from + (int)page];
          if (page >= sm_old[a] && off == 0) *entry = s;
          slot = (int64_t)s * P + off;
        }
        positions[j] = (int)min(pos, (uint32_t)INT_MAX);
        slot_map[j] = slot;
      }
    }
    tokens = sm_total[0];
    pages = sm_total[1];
    __syncthreads();  // the next chunk writes the same arrays
  }
  if (what & kFill) {  // tokens past the last row's
    for (uint32_t j = max(span0, tokens) + t; j < span1; j += kRows) {
      positions[j] = 0;
      slot_map[j] = -1;
    }
    if (first && t == 0) offsets[0] = 0;
  }
  if ((what & kAdvance) && first) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) used = max(used, (uint32_t)__shfl_xor(used, off, 64));
    if ((t & 63) == 0) sm_tok[t >> 6] = used;
    __syncthreads();
    if (t == 0) {
#pragma unroll
      for (int w = 1; w < kRows / 64; ++w) used = max(used, sm_tok[w]);
      head_out[0] = head + (int)used;
    }
  }
}

// ------------------------------------------------------------- rotary append --
// y = factor * R(pos * f_i) x on pair i of the first `rot` dims (i < rot / 2; pairs (2i, 2i + 1), or (i, i + rot / 2)
// with `halves`); dims past `rot` are copied.  The angle is formed and reduced in 64 bits: pos * f in 32 bits is off by
// 2^-24 pos, which at position 100k is 0.006 radian, and a float argument past a few thousand takes
// the long range reduction besides.  One workgroup takes kTokens tokens (or a share of one token's heads): its threads
// first evaluate the tokens' sines once for all heads into LDS, then stream items of NP pairs (two vectors of NP values).
// Bound by the copy: 75.5 MB of 4093 tokens in 15.0 us (5.0 TB/s, a large copy's rate), of 32 tokens by latency (4.1 us).
constexpr int kRopeThreads = 256;
constexpr int kMaxDim = 256;
constexpr int kTokens = 4;
constexpr int kMaxTokens = (1 << 26) - kTokens;  // (a grid, whole workgroups, has fewer than 2^32 threads)
constexpr int kMaxHeads = 1 << 20;

template <typename T, int N>
struct Vec {
  T v[N];
};
template <typename T, int N>
__device__ __forceinline__ Vec<T, N> load_vec(const T* p) {
  typedef T vt __attribute__((ext_vector_type(N)));
  const vt x = *reinterpret_cast<const vt*>(p);
  Vec<T, N> o;
#pragma unroll
  for (int i = 0; i < N; ++i) o.v[i] = x[i];
  return o;
}
template <typename T, int N>
__device__ __forceinline__ void store_vec(T* p, const float (&y)[N]) {
  typedef T vt __attribute__((ext_vector_type(N)));
  vt x;
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = from_f32<T>(y[i]);
  *reinterpret_cast<vt*>(p) = x;
}

// factor (cos, sin) of pos * f: the product reduced by 2 pi rint(a / 2 pi), 2 pi in two parts
__device__ __forceinline__ float2 turn_of(int pos, double f, float factor) {
  const double a = (double)pos * f;
  const double n = rint(a * 0.15915494309189535);
  const double r = fma(-n, 2.4492935982947064e-16, fma(-n, 6.283185307179586, a));
  float s, c;
  sincosf((float)r, &s, &c);
  return make_float2(c * factor, s * factor);
}

struct RopeIn {
  const void *q, *k, *v;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head, o_token, o_head;  // strides, elements
};

template <typename T, typename TK, int NP>
__global__ __launch_bounds__(kRopeThreads) void rope_append_kernel(
    RopeIn in, const int32_t* __restrict__ positions, const int64_t* __restrict__ slot_map,
    const double* __restrict__ freq, float factor, T* q_out, TK* __restrict__ kp, TK* __restrict__ vp, int tokens,
    int Hq, int Hkv, int D, int rot, int halves, int P, int64_t slots) {
  __shared__ float2 sm_cs[kTokens][kMaxDim / 2];
  __shared__ int64_t sm_at[kTokens];  // pool element of the token's row in KV head 0 (negative: padding)
  const int t0 = blockIdx.x * kTokens, nt = min(kTokens, tokens - t0);
  const int half = rot / 2;
  for (int i = threadIdx.x; i < nt * half; i += kRopeThreads) {
    const int u = i / half, p = i - u * half;
    sm_cs[u][p] = turn_of(positions[t0 + u], freq[p], factor);
  }
  if ((int)threadIdx.x < nt) {
    const int64_t s = slot_map[t0 + threadIdx.x];
    int64_t at = -1;
    if (s >= 0 && s < slots) {
      const int64_t page = s / P;
      at = (page * Hkv * P + (s - page * P)) * (int64_t)D;
    }
    sm_at[threadIdx.x] = at;
  }
  __syncthreads();
  const int per_head = D / 2 / NP;               // items of a head
  const int items = (Hq + 2 * Hkv) * per_head;   // of a token
  const int share = (items + gridDim.y - 1) / gridDim.y;
  const int i0 = blockIdx.y * share, n = max(0, min(items, i0 + share) - i0);
  for (int id = threadIdx.x; id < nt * n; id += kRopeThreads) {
    const int u = id / n, it = i0 + id - u * n;
    const int64_t at = sm_at[u];
    if (at < 0) continue;
    const int h = it / per_head, c = it - h * per_head;  // head (q, then k, then v), item of it
    const int p0 = c * NP;                               // first pair
    const bool turn = p0 < half && h < Hq + Hkv;
    const bool apart = halves && p0 < half;
    const int lo = apart ? p0 : 2 * p0, hi = apart ? p0 + half : 2 * p0 + NP;
    const int64_t tok = t0 + u;
    const T* src = h < Hq         ? (const T*)in.q + tok * in.q_token + h * in.q_head
                   : h < Hq + Hkv ? (const T*)in.k + tok * in.k_token + (h - Hq) * in.k_head
                                  : (const T*)in.v + tok * in.v_token + (h - Hq - Hkv) * in.v_head;
    const Vec<T, NP> a = load_vec<T, NP>(src + lo), b = load_vec<T, NP>(src + hi);
    float x[2 * NP], y[2 * NP];
#pragma unroll
    for (int e = 0; e < NP; ++e) {
      x[e] = to_f32(a.v[e]);
      x[NP + e] = to_f32(b.v[e]);
    }
#pragma unroll
    for (int e = 0; e < 2 * NP; ++e) y[e] = x[e];
    if (turn) {
#pragma unroll
      for (int e = 0; e < NP; ++e) {
        const float2 cs = sm_cs[u][p0 + e];
        // halves: elements e and NP + e; neighbours: 2e and 2e + 1
        const float re = halves ? x[e] : x[2 * e], im = halves ? x[NP + e] : x[2 * e + 1];
        const float yr = as_f32_value(fmaf(re, cs.x, -(im * cs.y))), yi = as_f32_value(fmaf(re, cs.y, im * cs.x));
        if (halves) {
          y[e] = yr;
          y[NP + e] = yi;
        } else {
          y[2 * e] = yr;
          y[2 * e + 1] = yi;
        }
      }
    }
    float ya[NP], yb[NP];
#pragma unroll
    for (int e = 0; e < NP; ++e) {
      ya[e] = y[e];
      yb[e] = y[NP + e];
    }
    if (h < Hq) {
      T* dst = q_out + tok * in.o_token + h * in.o_head;
      store_vec<T, NP>(dst + lo, ya);
      store_vec<T, NP>(dst + hi, yb);
    } else {
      TK* dst = (h < Hq + Hkv ? kp + (int64_t)(h - Hq) * P * D : vp + (int64_t)(h - Hq - Hkv) * P * D) + at;
      store_vec<TK, NP>(dst + lo, ya);
      store_vec<TK, NP>(dst + hi, yb);
    }
  }
}

// ---------------------------------------------------- norm and rotary append --
// y = factor * R(pos * f_i) (x / sqrt(mean x^2 + eps) * w), heads of q and k; v is copied: the rotary append with the
// norm of each head before the turn, x read once and y rounded once.  A head is taken by LPH lanes (a power of two, items
// of NP pairs as above, at most two a lane), which join their sums of squares by shuffles, so nothing passes through LDS
// but the sines.  A lane keeps its own part of both weights.  Bound by the copy: 100.6 MB of 4093 tokens of 48 heads in 20.7
// us (4.9 TB/s; without the next head's values on their way and with weights one by one 31.6), of one token by latency (3.4).
struct NormIn {
  const void *qw, *kw;
  int wf32;  // weights in fp32 (else fp16)
  float eps;
};
template <int NP>
__device__ __forceinline__ void load_weights(const void* w, int f32, int at, float* y) {  // (any address)
  typedef float wide __attribute__((ext_vector_type(NP), aligned(4)));
  typedef f16 half __attribute__((ext_vector_type(NP), aligned(2)));
  if (f32) {  // uniform
    const wide x = *reinterpret_cast<const wide*>((const float*)w + at);
#pragma unroll
    for (int e = 0; e < NP; ++e) y[e] = x[e];
  } else {
    const half x = *reinterpret_cast<const half*>((const f16*)w + at);
#pragma unroll
    for (int e = 0; e < NP; ++e) y[e] = to_f32(x[e]);
  }
}

template <typename T, typename TK, int NP>
__global__ __launch_bounds__(kRopeThreads) void norm_rope_append_kernel(
    RopeIn in, NormIn nm, const int32_t* __restrict__ positions, const int64_t* __restrict__ slot_map,
    const double* __restrict__ freq, float factor, T* q_out, TK* __restrict__ kp, TK* __restrict__ vp, int tokens,
    int Hq, int Hkv, int D, int rot, int halves, int P, int64_t slots, int lph) {
  constexpr int kItems = 64 * 2 * NP >= kMaxDim ? 1 : 2;  // of a lane: 64 lanes at most have a head
  __shared__ float2 sm_cs[kTokens][kMaxDim / 2];
  __shared__ int64_t sm_at[kTokens];  // pool element of the token's row in KV head 0 (negative: padding)
  const int t0 = blockIdx.x * kTokens, nt = min(kTokens, tokens - t0);
  const int half = rot / 2;
  const int per_head = D / 2 / NP;
  const int lane = threadIdx.x & (lph - 1), group = threadIdx.x / lph, groups = kRopeThreads / lph;
  const int heads = Hq + 2 * Hkv, share = (heads + gridDim.y - 1) / gridDim.y;
  const int h0 = blockIdx.y * share, n = max(0, min(heads, h0 + share) - h0);
  // The lane's items: pair p0 = c NP on, whose elements are lo .. lo + NP - 1 and hi .. hi + NP - 1.
  int lo[kItems], hi[kItems];
  bool live[kItems];
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const int c = lane + i * lph, p0 = c * NP;
    live[i] = c < per_head;
    const bool apart = halves && p0 < half;
    lo[i] = apart ? p0 : 2 * p0;
    hi[i] = apart ? p0 + half : 2 * p0 + NP;
  }
  // Head `h` of token t0 + u, and the group's next one; its x is on its way while the one before is worked on.
  int u = n > 0 ? group / n : nt, h = n > 0 ? group - u * n : 0;
  Vec<T, NP> na[kItems], nb[kItems];
  const auto load = [&]() __attribute__((always_inline)) {
    const int64_t tok = t0 + u;
    const int hh = h0 + h;
    const T* src = hh < Hq         ? (const T*)in.q + tok * in.q_token + hh * in.q_head
                   : hh < Hq + Hkv ? (const T*)in.k + tok * in.k_token + (hh - Hq) * in.k_head
                                   : (const T*)in.v + tok * in.v_token + (hh - Hq - Hkv) * in.v_head;
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      if (!live[i]) continue;
      na[i] = load_vec<T, NP>(src + lo[i]);
      nb[i] = load_vec<T, NP>(src + hi[i]);
    }
  };
  if (u < nt) load();
  float qw[kItems][2 * NP], kw[kItems][2 * NP];
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    if (!live[i]) continue;
    load_weights<NP>(nm.qw, nm.wf32, lo[i], qw[i]);
    load_weights<NP>(nm.qw, nm.wf32, hi[i], qw[i] + NP);
    load_weights<NP>(nm.kw, nm.wf32, lo[i], kw[i]);
    load_weights<NP>(nm.kw, nm.wf32, hi[i], kw[i] + NP);
  }
  for (int i = threadIdx.x; i < nt * half; i += kRopeThreads) {
    const int w = i / half, p = i - w * half;
    sm_cs[w][p] = turn_of(positions[t0 + w], freq[p], factor);
  }
  if ((int)threadIdx.x < nt) {
    const int64_t s = slot_map[t0 + threadIdx.x];
    int64_t at = -1;
    if (s >= 0 && s < slots) {
      const int64_t page = s / P;
      at = (page * Hkv * P + (s - page * P)) * (int64_t)D;
    }
    sm_at[threadIdx.x] = at;
  }
  __syncthreads();
  const float inv_d = 1.f / (float)D;
  while (u < nt) {  // (the lanes of a head stay together)
    const int64_t at = sm_at[u], tok = t0 + u;
    const int hh = h0 + h, was = u;
    float x[kItems][2 * NP], sum = 0.f;
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      if (!live[i]) continue;
#pragma unroll
      for (int e = 0; e < NP; ++e) {
        x[i][e] = to_f32(na[i].v[e]);
        x[i][NP + e] = to_f32(nb[i].v[e]);
      }
#pragma unroll
      for (int e = 0; e < 2 * NP; ++e) sum = fmaf(x[i][e], x[i][e], sum);
    }
    h += groups;
    while (h >= n) h -= n, ++u;
    if (u < nt) load();
    if (at < 0) continue;
    if (hh < Hq + Hkv) {
      for (int off = lph >> 1; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
      const float r = 1.f / sqrtf(fmaf(sum, inv_d, nm.eps));
      const bool is_q = hh < Hq;
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        if (!live[i]) continue;
        const int p0 = (lane + i * lph) * NP;
#pragma unroll
        for (int e = 0; e < 2 * NP; ++e) x[i][e] = x[i][e] * r * (is_q ? qw[i][e] : kw[i][e]);
        if (p0 >= half) continue;
#pragma unroll
        for (int e = 0; e < NP; ++e) {
          const float2 cs = sm_cs[was][p0 + e];
          const int re = halves ? e : 2 * e, im = halves ? NP + e : 2 * e + 1;
          const float a = x[i][re], b = x[i][im];
          x[i][re] = as_f32_value(fmaf(a, cs.x, -(b * cs.y)));
          x[i][im] = as_f32_value(fmaf(a, cs.y, b * cs.x));
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      if (!live[i]) continue;
      float ya[NP], yb[NP];
#pragma unroll
      for (int e = 0; e < NP; ++e) {
        ya[e] = as_f32_value(x[i][e]);
        yb[e] = as_f32_value(x[i][NP + e]);
      }
      if (hh < Hq) {
        T* dst = q_out + tok * in.o_token + hh * in.o_head;
        store_vec<T, NP>(dst + lo[i], ya);
        store_vec<T, NP>(dst + hi[i], yb);
      } else {
        TK* dst = (hh < Hq + Hkv ? kp + (int64_t)(hh - Hq) * P * D : vp + (int64_t)(hh - Hq - Hkv) * P * D) + at;
        store_vec<TK, NP>(dst + lo[i], ya);
        store_vec<TK, NP>(dst + hi[i], yb);
      }
    }
  }
}

// Whether any two of the heads at t * ts + h * hs (t < nt, h < nh; `len` elements each) overlap: some (i, j) != (0, 0),
// |i| < nt, |j| < nh, has |i ts + j hs| < len.
bool heads_overlap(int64_t ts, int nt, int64_t hs, int nh, int len) {
  typedef __int128 wide;  // (any strides)
  const auto mag = [](wide v) { return v < 0 ? -v : v; };
  wide a = ts, b = hs;
  int na = nt, nb = nh;
  if (na < nb) {
    std::swap(a, b);
    std::swap(na, nb);
  }
  if (na <= 1) return false;
  if (mag(a) < len || (nb > 1 && mag(b) < len)) return true;
  // One axis lies within a step of the other, as in every ordinary tensor.
  if (nb <= 1 || mag(a) >= (nb - 1) * mag(b) + len || mag(b) >= (na - 1) * mag(a) + len) return false;
  for (int j = 1; j < nb; ++j) {  // i = -j b / a, rounded to both sides, comes nearest
    const wide i = mag(j * b) / mag(a), rest = mag(j * b) - i * mag(a);
    if ((i < na && rest < len) || (i + 1 < na && mag(a) - rest < len)) return true;
  }
  return false;
}

// What rope_append and norm_rope_append take (a call without tokens passes with null pointers).
int check_rope(const char* who, const RopeIn& in, int dt, const int32_t* positions, const int64_t* slot_map,
               const double* inv_freq, int rotary_dim, int layout, void* q_out, void* k_pool, void* v_pool, int kv_dtype,
               int64_t slots, int tokens, int num_heads, int num_kv_heads, int head_dim, int page_size) {
  CIR_CHECK_ARG(valid_dt(dt) && valid_dt(kv_dtype), "%s: bad dtype", who);
  CIR_CHECK_ARG(layout == CIR_ROPE_INTERLEAVED || layout == CIR_ROPE_HALF, "%s: bad layout %d", who, layout);
  CIR_CHECK_ARG(head_dim > 0 && head_dim <= kMaxDim && head_dim % 2 == 0, "%s: head_dim %d must be even, 2..%d", who,
                head_dim, kMaxDim);
  CIR_CHECK_ARG(rotary_dim >= 0 && rotary_dim <= head_dim && rotary_dim % 2 == 0,
                "%s: rotary_dim %d must be even and at most head_dim", who, rotary_dim);
  CIR_CHECK_ARG(tokens >= 0 && num_heads >= 0 && num_kv_heads > 0 && page_size > 0 && slots >= 0,
                "%s: bad sizes", who);
  CIR_CHECK_ARG(tokens <= kMaxTokens && num_heads <= kMaxHeads && num_kv_heads <= kMaxHeads,
                "%s: more than 2^26 - 4 tokens or 2^20 heads", who);
  CIR_CHECK_ARG(slots % page_size == 0, "%s: slots must be whole pages", who);
  if (tokens == 0) return 0;
  CIR_CHECK_ARG((num_heads == 0 || (in.q && q_out)) && in.k && in.v && positions && slot_map && k_pool && v_pool &&
                    (inv_freq || rotary_dim == 0),
                "%s: null pointer", who);
  // Written heads that overlap, or q in place at other strides, would be read and written by different threads.
  CIR_CHECK_ARG(num_heads == 0 || !heads_overlap(in.o_token, tokens, in.o_head, num_heads, head_dim),
                "%s: heads of q_out overlap", who);
  CIR_CHECK_ARG(num_heads == 0 || q_out != in.q ||
                    ((tokens == 1 || in.o_token == in.q_token) &&
                     (num_heads == 1 || in.o_head == in.q_head)),
                "%s: q_out is q with other strides", who);
  const uintptr_t pool_bytes = (uintptr_t)slots * num_kv_heads * head_dim * (kv_dtype == CIR_F16 ? 2 : 4);
  const uintptr_t k_at = (uintptr_t)k_pool, v_at = (uintptr_t)v_pool;
  CIR_CHECK_ARG((k_at < v_at ? v_at - k_at : k_at - v_at) >= pool_bytes, "%s: k_pool and v_pool overlap", who);
  return 0;
}

// Values in a vector of an item (NP pairs take two): every row, head and half starts on a whole vector.
int rope_vector(const RopeIn& in, int dt, int rotary_dim, const void* q_out, const void* k_pool, const void* v_pool,
                int kv_dtype, int num_heads, int head_dim) {
  const auto aligned = [&](int np) {
    const int64_t strides = in.q_token | in.q_head | in.k_token | in.k_head | in.v_token | in.v_head | in.o_token | in.o_head;
    const uintptr_t io = (num_heads ? (uintptr_t)in.q | (uintptr_t)q_out : 0) | (uintptr_t)in.k | (uintptr_t)in.v;
    const uintptr_t pool = (uintptr_t)k_pool | (uintptr_t)v_pool;
    return head_dim % (2 * np) == 0 && rotary_dim % (2 * np) == 0 && strides % np == 0 &&
           io % (np * (dt == CIR_F16 ? 2 : 4)) == 0 && pool % (np * (kv_dtype == CIR_F16 ? 2 : 4)) == 0;
  };
  return dt == CIR_F16 && kv_dtype == CIR_F16 && aligned(8) ? 8 : aligned(4) ? 4 : 1;
}

// go<T, TK, NP>() for these types and vectors.
template <typename F>
void by_rope_types(int dt, int kv_dtype, int np, const F& go) {
  const auto by_pool = [&]<typename T, int NP>() {
    kv_dtype == CIR_F16 ? go.template operator()<T, f16, NP>() : go.template operator()<T, float, NP>();
  };
  if (dt == CIR_F16) {
    if (np == 8) go.template operator()<f16, f16, 8>();
    else if (np == 4) by_pool.template operator()<f16, 4>();
    else by_pool.template operator()<f16, 1>();
  } else {
    if (np == 4) by_pool.template operator()<float, 4>();
    else by_pool.template operator()<float, 1>();
  }
}

}  // namespace
}  // namespace cir

using namespace cir;

extern "C" int cir_extend_page_tables(int32_t* page_table, const int32_t* seq_lens, const int32_t* new_tokens,
                                      const int32_t* free_slots, int free_total, const int32_t* free_head,
                                      int32_t* seq_lens_out, int32_t* free_head_out, int32_t* offsets,
                                      int32_t* granted, int32_t* positions, int64_t* slot_map, int batch,
                                      int max_pages, int page_size, int max_tokens, void* stream) {
  CIR_CHECK_ARG(batch >= 0 && max_tokens >= 0 && free_total >= 0, "extend_page_tables: bad sizes");
  CIR_CHECK_ARG(page_size > 0 && max_pages > 0, "extend_page_tables: page_size and max_pages must be positive");
  CIR_CHECK_ARG(max_tokens < (int)kCap && free_total < (int)kCap, "extend_page_tables: 2^30 tokens or free slots");
  // (no rows: the slot map is still filled with -1)
  CIR_CHECK_ARG((page_table && seq_lens && new_tokens && seq_lens_out && granted) || batch == 0,
                "extend_page_tables: null pointer");
  CIR_CHECK_ARG(free_head && free_head_out && offsets, "extend_page_tables: null pointer");
  CIR_CHECK_ARG((free_slots || free_total == 0) && ((positions && slot_map) || max_tokens == 0),
                "extend_page_tables: null pointer");
  hipStream_t s = as_stream(stream);
  const unsigned wgs = (unsigned)(((long)max_tokens + kSpan - 1) / kSpan);
  // Lengths and head written in place: with several workgroups the ones that scan late would read what the first has
  // advanced, so a second launch advances them.
  const bool in_place = seq_lens_out == seq_lens || free_head_out == free_head;
  const auto go = [&](unsigned n, int what) {
    extend_tables_kernel<<<n, kRows, 0, s>>>(page_table, seq_lens, new_tokens, free_slots, free_total, free_head,
                                             seq_lens_out, free_head_out, offsets, granted, positions, slot_map, batch,
                                             max_pages, page_size, max_tokens, what);
    return launch_status();
  };
  if (wgs <= 1 || !in_place) return go(wgs ? wgs : 1, kFill | kAdvance);
  const int st = go(wgs, kFill);
  return st ? st : go(1, kAdvance);
}

extern "C" int cir_rope_append(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k,
                               int64_t k_token_stride, int64_t k_head_stride, const void* v, int64_t v_token_stride,
                               int64_t v_head_stride, int dt, const int32_t* positions, const int64_t* slot_map,
                               const double* inv_freq, float factor, int rotary_dim, int layout, void* q_out,
                               int64_t o_token_stride, int64_t o_head_stride, void* k_pool, void* v_pool, int kv_dtype,
                               int64_t slots, int tokens, int num_heads, int num_kv_heads, int head_dim, int page_size,
                               void* stream) {
  const RopeIn in{q, k, v, q_token_stride, q_head_stride, k_token_stride, k_head_stride, v_token_stride, v_head_stride,
                  o_token_stride, o_head_stride};
  if (const int bad = check_rope("rope_append", in, dt, positions, slot_map, inv_freq, rotary_dim, layout, q_out, k_pool,
                                 v_pool, kv_dtype, slots, tokens, num_heads, num_kv_heads, head_dim, page_size))
    return bad;
  if (tokens == 0) return 0;
  hipStream_t s = as_stream(stream);
  const int np = rope_vector(in, dt, rotary_dim, q_out, k_pool, v_pool, kv_dtype, num_heads, head_dim);
  const unsigned blocks = (unsigned)((tokens + kTokens - 1) / kTokens);
  const int items = (num_heads + 2 * num_kv_heads) * (head_dim / 2 / np);
  // Few tokens: a workgroup takes a share of the heads (one item per thread and token at least).
  const unsigned shares = (unsigned)max(1, min(min(16, (items * kTokens + kRopeThreads - 1) / kRopeThreads),
                                               (int)(512 / blocks)));
  by_rope_types(dt, kv_dtype, np, [&]<typename T, typename TK, int NP>() {
    rope_append_kernel<T, TK, NP><<<dim3(blocks, shares), kRopeThreads, 0, s>>>(
        in, positions, slot_map, inv_freq, factor, (T*)q_out, (TK*)k_pool, (TK*)v_pool, tokens, num_heads, num_kv_heads,
        head_dim, rotary_dim, layout == CIR_ROPE_HALF, page_size, slots);
  });
  return launch_status();
}

extern "C" int cir_norm_rope_append(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k,
                                    int64_t k_token_stride, int64_t k_head_stride, const void* v, int64_t v_token_stride,
                                    int64_t v_head_stride, int dt, const void* q_weight, const void* k_weight, int wdt,
                                    float eps, const int32_t* positions, const int64_t* slot_map, const double* inv_freq,
                                    float factor, int rotary_dim, int layout, void* q_out, int64_t o_token_stride,
                                    int64_t o_head_stride, void* k_pool, void* v_pool, int kv_dtype, int64_t slots,
                                    int tokens, int num_heads, int num_kv_heads, int head_dim, int page_size,
                                    void* stream) {
  const RopeIn in{q, k, v, q_token_stride, q_head_stride, k_token_stride, k_head_stride, v_token_stride, v_head_stride,
                  o_token_stride, o_head_stride};
  CIR_CHECK_ARG(valid_dt(wdt), "norm_rope_append: bad dtype");
  if (const int bad = check_rope("norm_rope_append", in, dt, positions, slot_map, inv_freq, rotary_dim, layout, q_out,
                                 k_pool, v_pool, kv_dtype, slots, tokens, num_heads, num_kv_heads, head_dim, page_size))
    return bad;
  if (tokens == 0) return 0;
  CIR_CHECK_ARG((q_weight || num_heads == 0) && k_weight, "norm_rope_append: null pointer");
  const int np = rope_vector(in, dt, rotary_dim, q_out, k_pool, v_pool, kv_dtype, num_heads, head_dim);
  const int per_head = head_dim / 2 / np;  // (at most 128: two items a lane)
  int lph = 1;
  while (lph < per_head && lph < 64) lph *= 2;
  const unsigned blocks = (unsigned)((tokens + kTokens - 1) / kTokens);
  // Few tokens: a workgroup takes a share of the heads (a head per group of lanes and token at least).
  const int heads = num_heads + 2 * num_kv_heads, groups = kRopeThreads / lph;
  const unsigned shares = (unsigned)max(1, min(min(64, (heads * kTokens + groups - 1) / groups), (int)(512 / blocks)));
  by_rope_types(dt, kv_dtype, np, [&]<typename T, typename TK, int NP>() {
    norm_rope_append_kernel<T, TK, NP><<<dim3(blocks, shares), kRopeThreads, 0, as_stream(stream)>>>(
        in, NormIn{num_heads ? q_weight : k_weight, k_weight, wdt == CIR_F32, eps}, positions, slot_map, inv_freq, factor,
        (T*)q_out, (TK*)k_pool, (TK*)v_pool, tokens, num_heads, num_kv_heads, head_dim, rotary_dim,
        layout == CIR_ROPE_HALF, page_size, slots, lph);
  });
  return launch_status();
}
