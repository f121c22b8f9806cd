// Logits before sampling: penalties for repeated tokens, biases of single tokens, and masks
// of the tokens that a grammar allows.
//
// For a row of sequence b and token v that occurs c times in what the sequence has said (its
// history behind the prompt, and the drafted tokens on the row's path), and at all in its
// prompt or there:
//   x = logit > 0 ? logit / rep_b : logit rep_b   (if v occurs at all)
//   y = x - freq_b c - (c > 0 ? pres_b : 0) + bias_b(v),   -inf where the row's mask has no bit
#include "common.hpp"

#include <math.h>

namespace cir {
namespace {

// One workgroup takes kChunk tokens of the vocabulary for some of a sequence's rows.  Counts
// of a whole vocabulary do not fit LDS, so each chunk's workgroup reads the sequence's history
// by itself (from L2: 64 KB for 8000 tokens) and counts what falls into its chunk, once for all
// of its rows; between two rows the drafted tokens on the one's path and not on the other's are
// added or taken off.  A word per token: how often it was said, its place in the bias list, and
// whether it was given in the prompt.  Bound by the read and write of the logits: a row's are on
// their way while the one before is worked on, the first row's while the history is counted.
// 485 rows of 152064 in fp16 (295 MB, histories of up to 4000): 68 us, a copy of them takes 57; before the loads and stores
// past the caches (below) 73, then with 512 threads 77, with chunks of 4096 or 16384 tokens, which read the history twice or
// half as often, 90 and 85.
constexpr int kChunk = 8192;
constexpr int kThreads = 1024;
constexpr int kCountBits = 20;                        // history and drafts hold fewer than 2^20 tokens
constexpr uint32_t kCount = (1u << kCountBits) - 1;
constexpr int kMaxBias = (1 << (31 - kCountBits)) - 1;  // 11 bits: index + 1
constexpr uint32_t kGiven = 1u << 31;
constexpr int kMaxDrafts = 256;
constexpr int kMaxHistory = (1 << kCountBits) - 1 - kMaxDrafts;

struct Args {
  const int32_t* offsets;  // NULL: one row per sequence
  const int64_t* history;
  const int32_t *history_lens, *prompt_lens;
  const int64_t *drafts, *masks;
  const float *rep, *pres, *freq;
  const int64_t* bias_ids;
  const float* bias;
  const int32_t* allowed;
  int64_t ld_in, ld_out;
  int rows, vocab, history_width, bias_width, words, allowed_words, in_place;
};

template <typename T>
__device__ __forceinline__ uint32_t raw_of(T x) {
  if constexpr (sizeof(T) == 2) return __builtin_bit_cast(uint16_t, x);
  else return __builtin_bit_cast(uint32_t, x);
}
template <typename T>
__device__ __forceinline__ T elem_of(uint32_t raw) {
  if constexpr (sizeof(T) == 2) return __builtin_bit_cast(T, (uint16_t)raw);
  else return __builtin_bit_cast(T, raw);
}

template <typename T, bool PAST>  // PAST: loads and stores past the caches
__global__ __launch_bounds__(kThreads) void adjust_logits_kernel(const T* in, T* out, Args A) {
  constexpr int VE = 16 / sizeof(T), J = kChunk / (kThreads * VE);  // tokens of a vector, vectors of a thread
  constexpr uint32_t kAll = (1u << VE) - 1;
  // (rows of any stride and address: the hardware takes vectors at any element)
  typedef T mt __attribute__((ext_vector_type(VE), aligned(sizeof(T))));
  typedef uint32_t vt __attribute__((ext_vector_type(4)));
  constexpr int kBits = 8 * sizeof(T), kPer = 32 / kBits;  // of an element; elements of a word
  constexpr uint32_t kElem = kPer == 1 ? ~0u : (1u << kBits % 32) - 1;
  __shared__ uint32_t sm_tab[kChunk], sm_drafted[kChunk / 32];
  const int t = threadIdx.x, b = blockIdx.y;
  const int v0 = blockIdx.x * kChunk, nv = min(kChunk, A.vocab - v0);
  // The sequence's rows, and this workgroup's share of them.
  int first = b, n = 1;
  if (A.offsets) {
    first = min(max(A.offsets[b], 0), A.rows);
    n = min(max(A.offsets[b + 1], first), A.rows) - first;
  }
  const int share = (n + gridDim.z - 1) / gridDim.z;
  const int i0 = blockIdx.z * share, i1 = min(n, i0 + share);
  if (i0 >= i1) return;  // uniform
  const int drafts = A.drafts ? min(n, 64 * A.words) : 0;

  // Tokens of vector k that the mask of the sequence's row i allows (none behind the vocabulary).
  const auto allowed = [&](int i, uint32_t (&ok)[J]) __attribute__((always_inline)) {
    const uint8_t* bits = reinterpret_cast<const uint8_t*>(A.allowed + (int64_t)(first + i) * A.allowed_words) + v0 / 8;
#pragma unroll
    for (int k = 0; k < J; ++k) {
      const int j = (t + k * kThreads) * VE;
      ok[k] = j >= nv || i >= i1 ? 0 : A.allowed ? bits[j >> 3] >> (j & 7) & kAll : kAll;
    }
  };
  const auto load = [&](int i, int k) __attribute__((always_inline)) {
    const T* src = in + (first + i) * A.ld_in + v0 + (t + k * kThreads) * VE;
    const int rest = nv - (t + k * kThreads) * VE;
    if (rest >= VE) {
      if constexpr (PAST) return __builtin_bit_cast(vt, __builtin_nontemporal_load(reinterpret_cast<const mt*>(src)));
      else return __builtin_bit_cast(vt, *reinterpret_cast<const mt*>(src));
    }
    vt x = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < VE; ++e)
      if (e < rest) x[e / kPer] |= raw_of(src[e]) << e % kPer * kBits;
    return x;
  };
  // The draft token of this thread: its place in the chunk.
  int place = -1;
  const auto in_chunk = [&](int64_t id) { return (uint64_t)(id - v0) < (uint64_t)nv; };
  const auto on_path = [&](int i) __attribute__((always_inline)) {
    return place >= 0 && i < i1 && (A.masks[(int64_t)(first + i) * A.words + (t >> 6)] >> (t & 63) & 1);
  };
  // The first tokens of the history, before the logits: loads come back in order.
  constexpr int U = 4;  // pairs on their way
  typedef int64_t i64x2 __attribute__((ext_vector_type(2), aligned(8)));
  const int len = A.history ? min(max(A.history_lens[b], 0), A.history_width) : 0;
  const int64_t* hist = A.history + (int64_t)b * A.history_width;
  i64x2 said[U];
  const auto said_from = [&](int k0) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + 2 * (t + u * kThreads);
      said[u] = i64x2{-1, -1};
      if (k + 1 < len) said[u] = *reinterpret_cast<const i64x2*>(hist + k);
      else if (k < len) said[u].x = hist[k];
    }
  };
  said_from(0);
  vt x[J], xn[J];
  uint32_t ok[J], okn[J];
  allowed(i0, ok);
  allowed(i0 + 1, okn);
  if (!A.in_place) {  // (in place most vectors need no load: below)
#pragma unroll
    for (int k = 0; k < J; ++k)
      if (ok[k]) x[k] = load(i0, k);
  }
  if (t < drafts) {
    const int64_t id = A.drafts[first + t];
    if (in_chunk(id)) place = (int)(id - v0);
  }
  bool on = on_path(i0), was = false;

  for (int i = t; i < kChunk / 4; i += kThreads) *reinterpret_cast<uint4*>(sm_tab + 4 * i) = make_uint4(0, 0, 0, 0);
  for (int i = t; i < kChunk / 32; i += kThreads) sm_drafted[i] = 0;
  const bool tree = __syncthreads_or(place >= 0);  // some token of the sequence's tree lies in the chunk
  if (place >= 0) atomicOr(&sm_drafted[place >> 5], 1u << (place & 31));
  if (A.bias_ids) {  // (of equal ids the last one counts)
    for (int k = t; k < A.bias_width; k += kThreads) {
      const int64_t id = A.bias_ids[(int64_t)b * A.bias_width + k];
      if (in_chunk(id)) atomicMax(&sm_tab[id - v0], (uint32_t)(k + 1) << kCountBits);
    }
    __syncthreads();
  }
  const int prompt = A.prompt_lens ? A.prompt_lens[b] : 0;
  const auto count = [&](int64_t id, int k) __attribute__((always_inline)) {
    if (!in_chunk(id)) return;
    if (k < prompt) atomicOr(&sm_tab[id - v0], kGiven);
    else atomicAdd(&sm_tab[id - v0], 1u);
  };
  for (int k0 = 0; k0 < len; k0 += 2 * U * kThreads) {
    if (k0) said_from(k0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + 2 * (t + u * kThreads);
      count(said[u].x, k);
      count(said[u].y, k + 1);
    }
  }
  __syncthreads();
  // Tokens of the thread's vectors that some row adjusts.  They are few, so a lane works on its own one after another: the
  // same for every element, needed or not, took as long as the memory (85 us instead of 77).
  uint32_t touched[J];
#pragma unroll
  for (int k = 0; k < J; ++k) {
    const int j = (t + k * kThreads) * VE;
    touched[k] = sm_drafted[j >> 5] >> (j & 31) & kAll;
#pragma unroll
    for (int e = 0; e < VE; ++e) touched[k] |= sm_tab[j + e] ? 1u << e : 0;
  }
  const float rep = A.rep ? A.rep[b] : 1.f, pres = A.pres ? A.pres[b] : 0.f, freq = A.freq ? A.freq[b] : 0.f;
  const auto adjust = [&](float x, uint32_t w) __attribute__((always_inline)) {
    const uint32_t c = w & kCount, k = (w & ~kGiven) >> kCountBits;
    if ((w & kGiven) || c) x = x > 0.f ? x / rep : x * rep;
    if (c) x = fmaf(-freq, (float)c, x) - pres;
    if (k) x += A.bias[(int64_t)b * A.bias_width + k - 1];
    return x;
  };
  for (int i = i0; i < i1; ++i) {
    if (tree) __syncthreads();  // uniform: the row before is done
    if (on != was) atomicAdd(&sm_tab[place], on ? 1u : ~0u);
    was = on;
    on = on_path(i + 1);
    if (!A.in_place) {
#pragma unroll
      for (int k = 0; k < J; ++k)
        if (okn[k]) xn[k] = load(i + 1, k);
    }
    uint32_t oka[J];
    allowed(i + 2, oka);
    if (tree) __syncthreads();  // uniform
    T* dst = out + (first + i) * A.ld_out + v0;
#pragma unroll
    for (int k = 0; k < J; ++k) {
      const int j = (t + k * kThreads) * VE;
      if (j >= nv) break;
      uint32_t left = touched[k] & ok[k];
      if (A.in_place) {
        if (ok[k] == kAll && !left) continue;
        if (ok[k]) x[k] = load(i, k);
      }
      while (left) {
        const int e = __builtin_ctz(left);
        left &= left - 1;
        const uint32_t w = sm_tab[j + e];
        const int d = e / kPer, shift = e % kPer * kBits;
        const uint32_t word = d == 0 ? x[k][0] : d == 1 ? x[k][1] : d == 2 ? x[k][2] : x[k][3];
        const T old = elem_of<T>(word >> shift);
        const uint32_t y = raw_of(w ? from_f32<T>(adjust(to_f32<T>(old), w)) : old) << shift;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[k][i] = d == i ? (x[k][i] & ~(kElem << shift)) | y : x[k][i];
      }
      const uint32_t lowest = raw_of(from_f32<T>(-INFINITY));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t off = 0;  // the elements that the mask takes out
#pragma unroll
        for (int e = 0; e < kPer; ++e) off |= ok[k] >> (i * kPer + e) & 1 ? 0 : kElem << e * kBits;
        x[k][i] = (x[k][i] & ~off) | ((kPer == 1 ? lowest : lowest * 0x10001u) & off);
      }
      if (nv - j >= VE) {
        if constexpr (PAST) __builtin_nontemporal_store(__builtin_bit_cast(mt, x[k]), reinterpret_cast<mt*>(dst + j));
        else *reinterpret_cast<mt*>(dst + j) = __builtin_bit_cast(mt, x[k]);
      } else {
#pragma unroll
        for (int e = 0; e < VE; ++e)
          if (e < nv - j) dst[j + e] = elem_of<T>(x[k][e / kPer] >> e % kPer * kBits);
      }
    }
#pragma unroll
    for (int k = 0; k < J; ++k) {
      x[k] = xn[k];
      ok[k] = okn[k];
      okn[k] = oka[k];
    }
  }
}

}  // namespace
}  // namespace cir

using namespace cir;

extern "C" int cir_adjust_logits(const void* logits, int64_t ld_in, void* out, int64_t ld_out, int dt,
                                 const int32_t* offsets, const int64_t* history, const int32_t* history_lens,
                                 const int32_t* prompt_lens, int history_width, const int64_t* drafts,
                                 const int64_t* masks, int words, const float* repetition, const float* presence,
                                 const float* frequency, const int64_t* bias_ids, const float* bias, int bias_width,
                                 const int32_t* allowed, int rows, int batch, int vocab, void* stream) {
  CIR_CHECK_ARG(dt == CIR_F32 || dt == CIR_F16, "adjust_logits: bad dtype");
  CIR_CHECK_ARG(rows >= 0 && batch >= 0 && vocab > 0, "adjust_logits: bad sizes");
  CIR_CHECK_ARG(rows < 1 << 24 && batch < 1 << 16, "adjust_logits: 2^24 rows or 2^16 sequences and more");
  CIR_CHECK_ARG(vocab <= 1 << 30, "adjust_logits: more than 2^30 tokens");
  CIR_CHECK_ARG(offsets || rows == batch, "adjust_logits: rows of sequences that offsets do not name");
  CIR_CHECK_ARG(ld_in >= vocab && ld_out >= vocab, "adjust_logits: rows overlap");
  CIR_CHECK_ARG(history_width >= 0 && history_width <= kMaxHistory, "adjust_logits: history of more than %d tokens",
                kMaxHistory);
  CIR_CHECK_ARG(bias_width >= 0 && bias_width <= kMaxBias, "adjust_logits: more than %d biases", kMaxBias);
  CIR_CHECK_ARG(!drafts || (words >= 1 && words * 64 <= kMaxDrafts), "adjust_logits: words must be 1..%d",
                kMaxDrafts / 64);
  if (rows == 0 || batch == 0) return 0;
  CIR_CHECK_ARG(logits && out && (!history || history_lens) && !drafts == !masks && !bias_ids == !bias,
                "adjust_logits: null pointer");
  CIR_CHECK_ARG(!drafts || offsets, "adjust_logits: drafts need offsets");
  const int size = dt == CIR_F16 ? 2 : 4;
  // In place at other strides, or onto other rows of the input, threads would read what others wrote.
  const uintptr_t a = (uintptr_t)logits, z = (uintptr_t)out;
  const uintptr_t a_bytes = ((uintptr_t)(rows - 1) * ld_in + vocab) * size;
  const uintptr_t z_bytes = ((uintptr_t)(rows - 1) * ld_out + vocab) * size;
  CIR_CHECK_ARG(a == z ? (rows == 1 || ld_in == ld_out) : a < z ? z - a >= a_bytes : a - z >= z_bytes,
                "adjust_logits: out overlaps the logits");
  const int chunks = (vocab + kChunk - 1) / kChunk;
  // Rows of a sequence are shared out until some 2048 workgroups fill the GPU, four times over (1024: 87 us instead of 76,
  // 4096: 80, each workgroup counts the history again).
  const int mean = (rows + batch - 1) / batch;
  const int shares = max(1, min(min(mean, 64), (int)(2048 / ((long)chunks * batch))));
  const Args A{offsets, history_width ? history : nullptr, history_lens, prompt_lens, drafts, masks, repetition, presence,
               frequency, bias_width ? bias_ids : nullptr, bias, allowed, ld_in, ld_out, rows, vocab, history_width, bias_width,
               words, (vocab + 31) / 32, a == z};
  const dim3 grid(chunks, batch, shares);
  // Logits that the L2s (32 MB in all) do not hold go past them: 147 MB 68.4 us instead of 73.2, and 119.6 instead of 122.2
  // with the call that reads them next; 16 MB 15.3 instead of 16.0, but 53.0 instead of 48.5 with the argmax that follows.
  const bool past = (long)rows * vocab * size > 32L << 20;
  const auto go = [&]<typename T>() {
    const auto kernel = past ? adjust_logits_kernel<T, true> : adjust_logits_kernel<T, false>;
    kernel<<<grid, kThreads, 0, as_stream(stream)>>>((const T*)logits, (T*)out, A);
  };
  dt == CIR_F16 ? go.template operator()<f16>() : go.template operator()<float>();
  return launch_status();
}
