// Trees of drafted tokens, before and after a step verifies them: which tokens each one
// sees and where it stands (draft_tree_kernel); the path that the model's own choices
// confirm, and its K and V moved behind the context (accept_kernel, settle_kernel).
//
// Row b's tokens are offsets[b] .. offsets[b] + n - 1 of the step's, n = counts[b], and lie
// in the cache as the last n of its seq_lens[b] tokens; parents name a token of the same
// row that comes before, or none (negative).
#include "common.hpp"

namespace cir {
namespace {

constexpr int kMaxDrafts = 256;  // of a row: one per thread
constexpr int kThreads = 256;

// A row's first token and their number, inside the step's tokens whatever the device's numbers are.  The cache holds all of
// them behind the context, however many a kernel takes.
struct Drafts {
  int first, all, n, end;  // n: of all, those that the kernel takes (`most` at most); end: where the next row's begin
};
__device__ __forceinline__ Drafts drafts_of(const int32_t* offsets, const int32_t* counts, int b, int tokens, int most) {
  const int o = offsets[b], e = offsets[b + 1], c = counts[b];
  Drafts d;
  d.first = min(max(o, 0), tokens);
  d.end = min(max(e, d.first), tokens);
  d.all = max(0, min(c, d.end - d.first));
  d.n = min(d.all, most);
  return d;
}

// ---------------------------------------------------------------- masks -------
// seen(j) = {j} + seen(parent(j)).  Pointer jumping: with mask(j) the ancestors up to 2^i - 1
// steps away and up(j) the one 2^i away, mask(j) |= mask(up(j)), up(j) = up(up(j)) doubles
// the reach, so a chain of 200 tokens takes 8 rounds and a tree of depth 5 three (a walk from
// parent to parent is one LDS latency a step: some 8 us for the chain).  One workgroup per
// row, one token per thread; a token's depth is the number of its ancestors.  Bound by
// latency: offsets, then parents, then the rounds (26 tokens 2.6 us, 128 rows of up to 200 6.0).
// A row of more tokens than masks of W words have bits for is refused: all of its masks are
// empty, and its positions, as if the first 64 W tokens were all it has, mean nothing.
template <int W>
__global__ __launch_bounds__(kThreads) void draft_tree_kernel(const int32_t* __restrict__ parents,
                                                              const int32_t* __restrict__ lens,
                                                              const int32_t* __restrict__ offsets,
                                                              const int32_t* __restrict__ counts,
                                                              int64_t* __restrict__ masks,
                                                              int32_t* __restrict__ positions, int tokens, int batch) {
  __shared__ uint64_t sm_mask[W][kMaxDrafts];
  __shared__ int sm_up[kMaxDrafts];
  const int b = blockIdx.x, t = threadIdx.x;
  const Drafts d = drafts_of(offsets, counts, b, tokens, 64 * W);
  const int len = lens[b];
  const bool in = t < d.n;
  int up = in ? parents[d.first + t] : -1;
  if (up >= t) up = -1;
  uint64_t m[W];
#pragma unroll
  for (int w = 0; w < W; ++w) {
    m[w] = in && (t >> 6) == w ? 1ull << (t & 63) : 0;
    sm_mask[w][t] = m[w];
  }
  sm_up[t] = up;
  while (__syncthreads_or(up >= 0)) {  // (up falls with every round: at most 8)
    int next = -1;
    if (up >= 0) {
#pragma unroll
      for (int w = 0; w < W; ++w) m[w] |= sm_mask[w][up];
      next = sm_up[up];
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) sm_mask[w][t] = m[w];
    sm_up[t] = up = next;
  }
  if (in) {
    int above = -1;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      above += __popcll(m[w]);
      masks[(size_t)(d.first + t) * W + w] = d.all > 64 * W ? 0 : (int64_t)m[w];
    }
    positions[d.first + t] = max(0, len - d.n) + above;
  }
  // Tokens that no row counts: those of rows that were not granted, and past the last row.
  const int lo = b == 0 ? 0 : d.first + d.n, hi = b == batch - 1 ? tokens : d.end;
  for (int j = lo + t; j < hi; j += kThreads) {
    if (j >= d.first && j < d.first + d.n) continue;
#pragma unroll
    for (int w = 0; w < W; ++w) masks[(size_t)j * W + w] = 0;
    positions[j] = 0;
  }
}

// --------------------------------------------------------------- accept -------
// The path starts at the row's token 0 (which the step before chose, so it stands) and goes
// from a token to the child that the model chose after it, the first one among equals, until
// there is none: next(p) = min {j : parent(j) = p, draft(j) = target(p)}, found for all
// tokens at once, then followed.  Token path[i] moves from position c + path[i] of the cache
// (c tokens of context) to c + i.  Parents come first, so path[i] >= i and path rises: no
// move reads what an earlier one wrote, each thread moves its 16 bytes of a head of all
// tokens, and the order among threads is free.  Every workgroup of a row finds the path for
// itself; the row's share of (layer, K or V, head, 16 bytes) is split over them.  Bound by
// the moved bytes; below some 10 MB by latency (lengths, tokens, path, page table, K and V).
struct AcceptArgs {
  const int32_t *parents, *lens, *offsets, *counts, *table;
  const int64_t *drafts, *targets;
  int32_t *accepted, *path, *lens_out;  // lens_out: NULL where settle_kernel writes them
  int64_t* tokens_out;
  uint8_t *k, *v;
  int64_t layer_bytes;  // of one pool
  int64_t slots;
  int tokens, max_pages, most, layers, Hkv, P, head_bytes;
};
constexpr int kAhead = 8;  // tokens whose loads are on their way together

template <typename V>
__global__ __launch_bounds__(kThreads) void accept_kernel(AcceptArgs A) {
  __shared__ int64_t sm_target[kMaxDrafts];
  __shared__ int sm_next[kMaxDrafts], sm_path[kMaxDrafts];
  __shared__ int sm_count, sm_moves;
  __shared__ int64_t sm_of[kMaxDrafts], sm_to[kMaxDrafts];  // byte of the token's row in head 0 of a layer's pool
  const int b = blockIdx.x, t = threadIdx.x;
  const Drafts d = drafts_of(A.offsets, A.counts, b, A.tokens, kMaxDrafts);
  const int len = A.lens[b], ctx = max(0, len - d.all);
  const bool in = t < d.n;
  const int p = in ? A.parents[d.first + t] : -1;
  const int64_t draft = in ? A.drafts[d.first + t] : 0;
  if (in) sm_target[t] = A.targets[d.first + t];
  sm_next[t] = kMaxDrafts;
  __syncthreads();
  if (in && p >= 0 && p < t && draft == sm_target[p]) atomicMin(&sm_next[p], t);
  __syncthreads();
  if (t == 0) {
    int n = 0;
    for (int at = 0; n < A.most && at < d.n; at = sm_next[at]) sm_path[n++] = at;  // (next > at)
    sm_count = n;
  }
  __syncthreads();
  const int n = sm_count;
  if (blockIdx.y == 0) {
    if (t < A.most) {
      A.path[(size_t)b * A.most + t] = t < n ? sm_path[t] : -1;
      A.tokens_out[(size_t)b * A.most + t] = t < n ? sm_target[sm_path[t]] : -1;
    }
    if (t == 0) {
      A.accepted[b] = n;
      if (A.lens_out) A.lens_out[b] = ctx + n;
    }
  }
  // Moves, those that stay where they are left out (the first tokens of the path: path[i] - i never falls).
  if (t < n) {
    const auto place = [&](int pos) -> int64_t {  // (entries outside the pool: nothing moves)
      const int page = pos / A.P;
      const int64_t slot = page < A.max_pages ? A.table[(size_t)b * A.max_pages + page] : -1;
      return slot < 0 || slot >= A.slots ? -1 : (slot * A.Hkv * A.P + pos % A.P) * (int64_t)A.head_bytes;
    };
    const bool moves = sm_path[t] != t;
    sm_of[t] = moves ? place(ctx + sm_path[t]) : -1;
    sm_to[t] = moves ? place(ctx + t) : -1;
    if (moves && (t == 0 || sm_path[t - 1] == t - 1)) sm_moves = t;
    if (t == n - 1 && !moves) sm_moves = n;
  }
  __syncthreads();
  if (n == 0) return;  // uniform
  const int first = sm_moves;
  if (first >= n) return;  // uniform
  const int per_head = A.head_bytes / (int)sizeof(V);
  const int units = A.layers * 2 * A.Hkv * per_head;
  for (int u = blockIdx.y * kThreads + t; u < units; u += gridDim.y * kThreads) {
    const int c = u % per_head, hl = u / per_head;
    const int h = hl % A.Hkv, kl = hl / A.Hkv;
    uint8_t* base = ((kl & 1) ? A.v : A.k) + (kl >> 1) * A.layer_bytes + (int64_t)h * A.P * A.head_bytes +
                    c * (int)sizeof(V);
    for (int i0 = first; i0 < n; i0 += kAhead) {
      V x[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (i0 + i < n && sm_of[i0 + i] >= 0) x[i] = *reinterpret_cast<const V*>(base + sm_of[i0 + i]);
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (i0 + i < n && sm_of[i0 + i] >= 0 && sm_to[i0 + i] >= 0) *reinterpret_cast<V*>(base + sm_to[i0 + i]) = x[i];
    }
  }
}

// Lengths written in place (every workgroup of accept_kernel reads them), and the pages behind the new lengths back to
// the free slots: row after row, so that they end where free_head was.
__global__ __launch_bounds__(kThreads) void settle_kernel(const int32_t* lens, const int32_t* __restrict__ offsets,
                                                          const int32_t* __restrict__ counts,
                                                          const int32_t* __restrict__ accepted,
                                                          const int32_t* __restrict__ table, int32_t* lens_out,
                                                          int32_t* __restrict__ free_slots, int free_total,
                                                          int32_t* free_head, int tokens, int batch, int max_pages,
                                                          int P) {
  __shared__ int sm_wave[kThreads / 64];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int per = (batch + kThreads - 1) / kThreads;
  const int b0 = min(batch, t * per), b1 = min(batch, b0 + per);
  const auto pages = [&](int n) { return min(n / P + (n % P ? 1 : 0), max_pages); };
  const auto row = [&](int b, int& keep, int& now, int& had) __attribute__((always_inline)) {
    const Drafts d = drafts_of(offsets, counts, b, tokens, kMaxDrafts);
    const int len = max(0, lens[b]);
    keep = max(0, len - d.all) + accepted[b];
    now = pages(keep);
    had = pages(len);
  };
  int mine = 0;
  if (free_slots)
    for (int b = b0; b < b1; ++b) {
      int keep, now, had;
      row(b, keep, now, had);
      mine += max(0, had - now);
    }
  int upto = mine;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int o = __shfl_up(upto, off, 64);
    upto += lane >= off ? o : 0;
  }
  if (lane == 63) sm_wave[wave] = upto;
  const int head = free_slots ? free_head[0] : 0;
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    upto += w < wave ? sm_wave[w] : 0;
    total += sm_wave[w];
  }
  const bool fits = free_slots && total <= head && head <= free_total;  // (else slots were counted elsewhere: none is written)
  int at = head - total + upto - mine;
  for (int b = b0; b < b1; ++b) {
    int keep, now, had;
    row(b, keep, now, had);
    if (fits)
      for (int p = now; p < had; ++p) free_slots[at++] = table[(size_t)b * max_pages + p];
    lens_out[b] = keep;
  }
  if (t == 0 && fits) free_head[0] = head - total;
}

}  // namespace
}  // namespace cir

using namespace cir;

extern "C" int cir_draft_tree(const int32_t* parents, const int32_t* seq_lens, const int32_t* offsets,
                              const int32_t* counts, int64_t* masks, int32_t* positions, int tokens, int batch,
                              int words, void* stream) {
  CIR_CHECK_ARG(tokens >= 0 && batch >= 0, "draft_tree: bad sizes");
  CIR_CHECK_ARG(words >= 1 && words * 64 <= kMaxDrafts, "draft_tree: words must be 1..%d (got %d)", kMaxDrafts / 64, words);
  CIR_CHECK_ARG(batch < (1 << 24), "draft_tree: 2^24 rows and more");
  if (tokens == 0) return 0;
  CIR_CHECK_ARG(batch > 0, "draft_tree: tokens of no row");
  CIR_CHECK_ARG(parents && seq_lens && offsets && counts && masks && positions, "draft_tree: null pointer");
  const auto go = [&]<int W>() {
    draft_tree_kernel<W><<<batch, kThreads, 0, as_stream(stream)>>>(parents, seq_lens, offsets, counts, masks, positions,
                                                                    tokens, batch);
  };
  switch (words) {
    case 1: go.template operator()<1>(); break;
    case 2: go.template operator()<2>(); break;
    case 3: go.template operator()<3>(); break;
    default: go.template operator()<4>(); break;
  }
  return launch_status();
}

extern "C" int cir_accept_drafts(const int32_t* parents, const int64_t* drafts, const int64_t* targets,
                                 const int32_t* seq_lens, const int32_t* offsets, const int32_t* counts,
                                 const int32_t* page_table, int32_t* accepted, int32_t* path, int64_t* tokens_out,
                                 int32_t* seq_lens_out, void* k_pools, void* v_pools, int kv_dtype, int64_t slots,
                                 int32_t* free_slots, int free_total, int32_t* free_head, int tokens, int batch, int most,
                                 int max_pages, int layers, int num_kv_heads, int head_dim, int page_size,
                                 void* stream) {
  CIR_CHECK_ARG(tokens >= 0 && batch >= 0 && layers >= 0 && slots >= 0 && free_total >= 0, "accept_drafts: bad sizes");
  CIR_CHECK_ARG(most >= 1 && most <= kMaxDrafts, "accept_drafts: most must be 1..%d (got %d)", kMaxDrafts, most);
  CIR_CHECK_ARG(kv_dtype == CIR_F16 || kv_dtype == CIR_F32, "accept_drafts: bad dtype");
  CIR_CHECK_ARG(num_kv_heads > 0 && num_kv_heads <= 1 << 12 && head_dim > 0 && head_dim <= 1 << 12 && layers <= 1 << 12 &&
                    page_size > 0 && max_pages > 0,
                "accept_drafts: heads, dims, layers (up to 4096) and pages must be positive");
  CIR_CHECK_ARG(slots < (1LL << 31) && batch < 1 << 20, "accept_drafts: 2^31 pages or 2^20 rows and more");
  if (batch == 0) return 0;
  CIR_CHECK_ARG(seq_lens && offsets && counts && page_table && accepted && path && tokens_out && seq_lens_out,
                "accept_drafts: null pointer");
  CIR_CHECK_ARG((parents && drafts && targets) || tokens == 0, "accept_drafts: null pointer");
  CIR_CHECK_ARG((k_pools && v_pools) || layers == 0 || slots == 0, "accept_drafts: null pools");
  CIR_CHECK_ARG(!free_slots == !free_head, "accept_drafts: free_slots and free_head go together");
  const int size = kv_dtype == CIR_F16 ? 2 : 4, head_bytes = head_dim * size;
  const int64_t layer_bytes = slots * num_kv_heads * page_size * (int64_t)head_bytes;
  const uintptr_t k_at = (uintptr_t)k_pools, v_at = (uintptr_t)v_pools;
  CIR_CHECK_ARG((k_at < v_at ? v_at - k_at : k_at - v_at) >= (uintptr_t)(layer_bytes * layers),
                "accept_drafts: k_pools and v_pools overlap");
  hipStream_t s = as_stream(stream);
  const bool settle = seq_lens_out == seq_lens || free_slots;
  const AcceptArgs A{parents, seq_lens, offsets, counts, page_table, drafts, targets, accepted, path,
                     settle ? nullptr : seq_lens_out, tokens_out, static_cast<uint8_t*>(k_pools),
                     static_cast<uint8_t*>(v_pools), layer_bytes, slots, tokens, max_pages, most,
                     slots ? layers : 0, num_kv_heads, page_size, head_bytes};
  const bool wide = head_bytes % 16 == 0 && (k_at | v_at) % 16 == 0;
  const int per_head = head_bytes / (wide ? 16 : size);
  const long units = (long)A.layers * 2 * num_kv_heads * per_head;
  CIR_CHECK_ARG(units < 1L << 30, "accept_drafts: 2^30 parts of a token's heads and more");
  // One unit a thread, up to some 16 workgroups per CU in all.
  const unsigned shares = (unsigned)max(1L, min((units + kThreads - 1) / kThreads, max(1L, 4096L / batch)));
  if (wide) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    accept_kernel<u32x4><<<dim3(batch, shares), kThreads, 0, s>>>(A);
  } else if (size == 4) {
    accept_kernel<uint32_t><<<dim3(batch, shares), kThreads, 0, s>>>(A);
  } else {
    accept_kernel<uint16_t><<<dim3(batch, shares), kThreads, 0, s>>>(A);
  }
  const int st = launch_status();
  if (st || !settle) return st;
  settle_kernel<<<1, kThreads, 0, s>>>(seq_lens, offsets, counts, accepted, page_table, seq_lens_out, free_slots,
                                       free_total, free_head, tokens, batch, max_pages, page_size);
  return launch_status();
}
