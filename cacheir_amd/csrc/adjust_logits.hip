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
// of its rows; the drafted tokens on a row's path are added before the row and taken off after
// it.  A word per token: how often it was said, its place in the bias list, and whether it was
// given in the prompt.  Bound by the read and write of the logits.
constexpr int kChunk = 8192;
constexpr int kThreads = 512;
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

template <typename T, int VE>
__global__ __launch_bounds__(kThreads) void adjust_logits_kernel(const T* in, T* out, Args A) {
  typedef T vt __attribute__((ext_vector_type(VE)));
  __shared__ uint32_t sm_tab[kChunk];
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

  for (int i = t; i < kChunk; i += kThreads) sm_tab[i] = 0;
  __syncthreads();
  const auto in_chunk = [&](int64_t id) { return (uint64_t)(id - v0) < (uint64_t)nv; };
  if (A.bias_ids) {  // (of equal ids the last one counts)
    for (int k = t; k < A.bias_width; k += kThreads) {
      const int64_t id = A.bias_ids[(int64_t)b * A.bias_width + k];
      if (in_chunk(id)) atomicMax(&sm_tab[id - v0], (uint32_t)(k + 1) << kCountBits);
    }
    __syncthreads();
  }
  if (A.history) {
    const int len = min(max(A.history_lens[b], 0), A.history_width);
    const int prompt = A.prompt_lens ? A.prompt_lens[b] : 0;
    const int64_t* h = A.history + (int64_t)b * A.history_width;
    for (int k = t; k < len; k += kThreads) {
      const int64_t id = h[k];
      if (in_chunk(id)) {
        if (k < prompt) atomicOr(&sm_tab[id - v0], kGiven);
        else atomicAdd(&sm_tab[id - v0], 1u);
      }
    }
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
    const int row = first + i;
    // Whether token t of the row's tree is on its path, and falls into the chunk.
    int64_t said = -1;
    if (t < drafts && (A.masks[(int64_t)row * A.words + (t >> 6)] >> (t & 63) & 1)) {
      const int64_t id = A.drafts[first + t];
      if (in_chunk(id)) said = id - v0;
    }
    __syncthreads();  // (the history is counted, the row before is done)
    if (said >= 0) atomicAdd(&sm_tab[said], 1u);
    __syncthreads();
    const T* src = in + row * A.ld_in + v0;
    T* dst = out + row * A.ld_out + v0;
    const int32_t* bits = A.allowed ? A.allowed + (int64_t)row * A.allowed_words + v0 / 32 : nullptr;
    for (int j = t * VE; j < nv; j += kThreads * VE) {  // (nv is a multiple of VE)
      constexpr uint32_t kAll = (1u << VE) - 1;
      const uint32_t ok = bits ? ((uint32_t)bits[j >> 5] >> (j & 31)) & kAll : kAll;
      uint32_t w[VE], any = 0;
#pragma unroll
      for (int e = 0; e < VE; ++e) any |= w[e] = sm_tab[j + e];
      if (A.in_place && ok == kAll && !any) continue;
      vt x = {};
      if (ok) x = *reinterpret_cast<const vt*>(src + j);
      if (any | (ok ^ kAll)) {
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const float y = adjust(to_f32<T>(x[e]), w[e]);
          x[e] = ok >> e & 1 ? w[e] ? from_f32<T>(y) : x[e] : from_f32<T>(-INFINITY);
        }
      }
      *reinterpret_cast<vt*>(dst + j) = x;
    }
    if (i + 1 < i1) {
      __syncthreads();
      if (said >= 0) atomicSub(&sm_tab[said], 1u);
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
  const Args A{offsets, history_width ? history : nullptr, history_lens, prompt_lens, drafts, masks, repetition, presence, frequency,
               bias_width ? bias_ids : nullptr, bias, allowed, ld_in, ld_out, rows, vocab, history_width, bias_width,
               words, (vocab + 31) / 32, a == z};
  const int chunks = (vocab + kChunk - 1) / kChunk;
  // Rows of a sequence are shared out until some 2048 workgroups fill the GPU.
  const int mean = (rows + batch - 1) / batch;
  const int shares = max(1, min(min(mean, 64), (int)(2048 / ((long)chunks * batch))));
  const int ve = 16 / size;
  const bool wide = (a | z) % 16 == 0 && ld_in % ve == 0 && ld_out % ve == 0 && vocab % ve == 0;
  const dim3 grid(chunks, batch, shares);
  const auto go = [&]<typename T, int VE>() {
    adjust_logits_kernel<T, VE><<<grid, kThreads, 0, as_stream(stream)>>>((const T*)logits, (T*)out, A);
  };
  if (dt == CIR_F16) wide ? go.template operator()<f16, 8>() : go.template operator()<f16, 1>();
  else wide ? go.template operator()<float, 4>() : go.template operator()<float, 1>();
  return launch_status();
}
