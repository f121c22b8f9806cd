// Decode attention for a batch whose rows share prefixes by groups: the K and V of a prefix
// are read once for the query vectors of all rows of its group, not once per row.
//
// out[b] = softmax(scale q[b] K[b]^T) V[b] over the row's paged context, as the decode
// attention computes it.  Softmax over a context in pieces: each piece gives (m, l, O) =
// (max, sum of e^(s - m), sum of e^(s - m) v), and the pieces of a row, its group's prefix
// among them, are joined by sum 2^(m_i - M) (l_i, O_i) in a second launch.
//
// Work.  Two kinds of item: (group, tile of 128 query vectors) over the prefix, and a row
// over what follows it; a group of up to 32 vectors makes one tile of 32.  An item costs
// kItemCost + its 32-token blocks; the items lie on one axis, prefixes first, and each team
// of workgroups (one per KV head) takes an equal stretch of that axis, whatever rows it
// crosses: lengths live on the device, and a grid cut by rows or by a fixed number of splits
// leaves CUs idle behind the longest row.  Every workgroup finds its stretch by a scan over
// the groups and rows (from L2, ~1 us).  A piece of item i computed by team w has the slot
// w + i: along the axis one of the two grows from piece to piece, so slots are unique, and
// the join finds an item's pieces from its start and the stretch alone.  The workgroups of a
// team walk the same pages in step, one head of each.
//
// Bodies (4 wavefronts, two workgroups per CU, so that one streams while the other starts or
// ends a piece; MFMA 32x32x16 f16, S^T = K Q^T and O^T = V^T P^T as in the prefill
// attention, whose LDS swizzles these are):
//   * piece_stream, up to 32 query vectors: bound by the read of K and V.  Each wavefront
//     walks blocks of its own (every 4th) and stages them by DMA in LDS of its own: no
//     barriers, K of the next block is on its way once this block's K is in registers, and
//     V likewise, so a CU has 64 to 128 KiB in flight.  The loads are non-temporal (128 rows
//     of 64 to 7168 tokens, 28/4 heads: 180 -> 158 us, 6.0 TB/s).
//   * piece_tile, up to 128 vectors: bound by the chain of a stage (LDS reads, products,
//     softmax), which the second workgroup hides in part.  Each wavefront takes 32 vectors;
//     stages of 64 tokens of K and V go through LDS for all.  64 rows after 32672 tokens,
//     32/8 heads: 59 us, 576 TFLOP/s.
// P is rounded to fp16 for the second product (relative 2^-11 of a weight) and l sums the
// rounded values, so a row's weights still add up to one; everything else is fp32.
// Measured, both launches: 128 rows of 64 to 7168 tokens after 1024 shared ones, 28/4 heads,
// 165 us (5.8 TB/s; each row alone 197); 64 rows after 16000, 32/8 heads, 45 us (each row
// alone 320); 4 rows after 500 11.5 us, where each row alone takes 11.0.
#include "attn_tile.hpp"

#include <float.h>
#include <math.h>

namespace cir {
namespace {

constexpr int D = 128;
constexpr int kBlock = 32;        // tokens of an MFMA tile
constexpr int kVec = 32;          // query vectors of an MFMA tile
constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kGroups = 512;      // workgroups, about: two per CU
constexpr int kTileVec = 128;     // query vectors of a prefix tile
// A piece's start and join in blocks (6 against 3, us: 64 rows after 16000 tokens 49.3 -> 47.9, 64 after 2048
// 22.3 -> 20.8, 32 after 8000 24.5 -> 22.6), and the blocks per workgroup at least (one per wavefront; 4 against 8: 4 rows after 500
// tokens 12.8 -> 11.8, 16 after 1000 16.8 -> 15.6, 8 after 3000 14.3 -> 15.6).
constexpr int kItemCost = 6;
constexpr int kMinStretch = 4;
constexpr int kMaxPrefixes = 256;  // groups: one per thread
constexpr int kMaxRows = 2048;
// Fewer query vectors than this in the batch (the join's rounded-up grid stays below 2^32 threads), and fewer KV heads (a
// workgroup each at least; the records' loop steps by kThreads grids in 32 bits).
constexpr long kMaxVectors = (1L << 26) - 3;
constexpr int kMaxKvHeads = 1 << 23;
constexpr int kRowB = 2 * D;      // bytes of a K or V row

// Workspace: one record per row, then the pieces.
struct Pieces {
  int slot, count;  // of an item: piece k lies in slot + k
};
struct RowRec {
  Pieces prefix[2];  // of the tile that holds the row's first query vector of a KV head, and of the next one
  Pieces own;
  int first, pad;  // that vector in its group
};
struct Layout {
  size_t rows, pre_o, pre_ml, suf_o, suf_ml, total;  // bytes
};

struct Args {
  RowRec* rows;
  float *pre_o, *pre_ml, *suf_o, *suf_ml;
  int B, NG, Hq, Hkv, P16, max_pages;  // P16: page size / 16
  uint32_t page_magic;                 // ceil(2^32 / P16): n / P16 = n * page_magic >> 32 (P16 > 1)
  float scale_log2;
};

// A piece: query vectors v0 .. v0 + nv - 1 of (rows from vrow, KV head h) over blocks blk0 .. blk1 - 1 of the
// table row `ptrow`; tokens from `limit` on do not count.
struct Piece {
  const f16 *q, *kp, *vp;
  const int32_t* ptrow;
  int h, vrow, v0, nv, blk0, blk1, limit;
  float *o, *ml;
};

__device__ __forceinline__ int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Inclusive sums of N values over the workgroup, and their totals.
template <int N>
__device__ __forceinline__ void block_scan(int (&v)[N], int (&total)[N], int (*scratch)[kWaves]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int i = 0; i < N; ++i) {
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int o = __shfl_up(v[i], off, 64);
      v[i] += lane >= off ? o : 0;
    }
    if (lane == 63) scratch[i][wave] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    total[i] = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      v[i] += w < wave ? scratch[i][w] : 0;
      total[i] += scratch[i][w];
    }
  }
  __syncthreads();
}

// Running softmax of one query vector per lane (lane l and l + 32: the same vector).
struct Soft {
  float m, l;
  bool huge;  // uniform: some vector's |m| is 2^24 or more
  f32x16 acc[D / 32];
};
__device__ __forceinline__ void soft_init(Soft& a) {
  a.m = -INFINITY;
  a.l = 0.f;
  a.huge = false;
#pragma unroll
  for (int t = 0; t < D / 32; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) a.acc[t][r] = 0.f;
}
// Scores c (unscaled) of NB blocks -> p in fp16, the B operand of the second product, with the running max and the
// accumulators moved; `ps` are the sums of p.  A vector that has seen no finite score keeps m = -inf and subtracts 0.
// m follows the maximum only once some score lies more than 8 above it: p stays at 2^8 or less, which fp16 holds as
// exactly as p <= 1, and after a piece's first blocks the 64 accumulators are hardly ever scaled (128 rows after 16384
// shared tokens, 28/4 heads: 61 -> 57 us).  The two lanes of a vector compare their own halves of the scores.
template <int NB>
__device__ __forceinline__ void soft_step(Soft& a, f32x16 (&c)[NB], float sc, f16x8 (&pa)[NB][2], float (&ps)[NB]) {
  float mx = c[0][0];
#pragma unroll
  for (int r = 1; r < 16 * NB; ++r) mx = fmaxf(mx, c[r >> 4][r & 15]);
  mx = as_f32_value(mx * sc);
  // The difference, not a.m + 8: from |m| = 2^27 on that can round up to the next score, 16 above, whose p is no fp16.
  if (__builtin_amdgcn_ballot_w64(mx - a.m > 8.f) != 0) {  // uniform
    const float mn = fmaxf(a.m, fmaxf(mx, __shfl_xor(mx, 32, 64)));
    const float alpha = __builtin_amdgcn_exp2f(a.m - (mn == -INFINITY ? 0.f : mn));
    a.l *= alpha;
    a.m = mn;
    a.huge = __builtin_amdgcn_ballot_w64(fabsf(a.m) >= 0x1p24f && a.m != -INFINITY) != 0;
#pragma unroll
    for (int t = 0; t < D / 32; ++t) a.acc[t] *= alpha;
  }
  // p = 2^(c sc - m) by one FMA.  m is a rounded product, off by up to half an ulp: a factor that all p of the vector
  // share.  From |m| = 2^24 on (where it could leave fp16) the rounded products are subtracted instead.
  float ms = a.m == -INFINITY ? 0.f : a.m, pc = sc;
  if (__builtin_expect(a.huge, 0)) {
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) c[j][r] = as_f32_value(c[j][r] * sc) - ms;
    ms = 0.f;
    pc = 1.f;
  }
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    ps[j] = 0.f;
#pragma unroll
    for (int r = 0; r < 16; r += 2) {
      const f16x2 two = {static_cast<f16>(__builtin_amdgcn_exp2f(fmaf(c[j][r], pc, -ms))),
                         static_cast<f16>(__builtin_amdgcn_exp2f(fmaf(c[j][r + 1], pc, -ms)))};
      pa[j][r >> 3][r & 7] = two.x;
      pa[j][r >> 3][(r & 7) + 1] = two.y;
      ps[j] = __builtin_amdgcn_fdot2(two, f16x2{(f16)1.f, (f16)1.f}, ps[j], false);  // exact products, fp32 sum
    }
  }
}

// Q^T as the B operand: lane l32's vector, dims 16 s + 8 h + e (zero past the last vector); a negative scale goes into
// its sign, so that the maximum can be taken before scaling.
__device__ __forceinline__ void load_q(const Args& A, const Piece& p, int v, f16x8 (&qb)[8]) {
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int G = A.Hq / A.Hkv;
  const bool live = v < p.nv;
  const int vv = p.v0 + (live ? v : 0);
  const int r = vv / G, g = vv - r * G;
  const f16* row = p.q + ((size_t)(p.vrow + r) * A.Hq + (size_t)p.h * G + g) * D + 8 * half;
  const uint32_t flip = A.scale_log2 < 0.f ? 0x80008000u : 0u;
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
#pragma unroll
  for (int s = 0; s < 8; ++s) {
    const u32x4 x = *reinterpret_cast<const u32x4*>(row + 16 * s) ^ flip;
    qb[s] = live ? __builtin_bit_cast(f16x8, x) : f16x8{0, 0, 0, 0, 0, 0, 0, 0};
  }
}

// V^T fragments of a block whose V rows start at `v`: see the prefill attention.
__device__ __forceinline__ void load_vt(const uint8_t* v, const int (&vo)[2], int ti, f16x8 (&va)[D / 32][2]) {
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const uint8_t* p = v + 64 * (dt ^ (ti >> 2)) + ks * 16 * kRowB;
      const f16x4 lo = lds_read_tr(p + vo[0]), hi = lds_read_tr(p + vo[1]);
      va[dt][ks] = f16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    }
}

constexpr int kStage = 32 * 1024;  // bytes of each of the two LDS arrays

// Pool rows of 16 tokens (one page holds them whole), token 16 n first: page table entry, then elements from the pool.
__device__ __forceinline__ int page_index(const Args& A, int n) {
  return A.P16 == 1 ? n : (int)__umulhi((uint32_t)n, A.page_magic);
}
__device__ __forceinline__ size_t rows16_at(const Args& A, int h, int page, int n, int index) {
  return (((size_t)page * A.Hkv + h) * A.P16 + (n - index * A.P16)) * (16 * D);
}

// ------------------------------------------------------- up to 32 vectors -----
__device__ __forceinline__ void piece_stream(const Args& A, const Piece& p, uint8_t* st0, uint8_t* st1,
                                             float (*sm_ml)[2][kVec]) {
  const int wave = uni(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int l32 = lane & 31, h = lane >> 5;
  uint8_t* kb = st0 + wave * (kBlock * kRowB);
  uint8_t* vb = st1 + wave * (kBlock * kRowB);
  const float sc = fabsf(A.scale_log2);
  const int last = p.limit - 1, last16 = last >> 4;

  // DMA of a block: 4 rows per instruction (lane / 16 = row, lane % 16 = LDS slot); chunk c of K row r goes to slot
  // c ^ (r % 16), of V row r to slot c ^ (4 (r % 4) + r / 4 % 4).  Rows past the limit re-read the last token
  // (masked; p = 0 meets finite values unless that token's own are not).
  const int lr = lane >> 4, ls = lane & 15;
  uint32_t at_k[4], at_v[4];  // byte offsets of the lane's chunk in 16 whole rows
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    at_k[u] = (4 * u + lr) * kRowB + 16 * (ls ^ (4 * u + lr));
    at_v[u] = (4 * u + lr) * kRowB + 16 * (ls ^ ((lr << 2) | u));
  }
  int page[2];
  auto fetch = [&](int blk) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 2; ++j) page[j] = p.ptrow[page_index(A, min(2 * blk + j, last16))];
  };
  auto issue = [&](const f16* pool, uint8_t* buf, int blk, const uint32_t (&at)[4]) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int n = min(2 * blk + j, last16), end = last - 16 * n;  // end: the last row that counts, if below 15
      const rsrc_t r = make_rsrc(pool + rows16_at(A, p.h, page[j], n, page_index(A, n)), 16 * kRowB);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        uint32_t off = at[u];
        if (end < 15) off = off - max(0, 4 * u + lr - end) * kRowB;  // uniform
        buf16_to_lds_once(r, buf + (16 * j + 4 * u) * kRowB, off, 0);
      }
    }
  };

  int blk = p.blk0 + wave;
  f16x8 qb[8];
  load_q(A, p, l32, qb);
  Soft a;
  soft_init(a);
  const int krow = l32 * kRowB, kx = 16 * (h ^ (l32 & 15));
  const int ti = lane & 15, sub = (lane >> 4) & 1;
  int vo[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    vo[i] = (8 * i + 4 * h + (ti >> 2)) * kRowB + 16 * ((2 * sub + ((ti & 3) >> 1)) ^ (2 * i + h)) + 8 * (ti & 1);

  // One block; MORE: the next one is issued.  (The last block is peeled off: loads under a condition would make the
  // compiler wait for all of them before each read of LDS.)
  auto step = [&]<bool MORE>() __attribute__((always_inline)) {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0F78);  // vmcnt(8): this block's K has landed (its V may be on its way)
    asm volatile("" ::: "memory");
    f16x8 ka[8];
#pragma unroll
    for (int s = 0; s < 8; ++s) ka[s] = *reinterpret_cast<const f16x8*>(kb + krow + (kx ^ (32 * s)));
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): K is in registers, its LDS free
    asm volatile("" ::: "memory");
    if constexpr (MORE) issue(p.kp, kb, blk + kWaves, at_k);
    f32x16 c[1];
#pragma unroll
    for (int r = 0; r < 16; ++r) c[0][r] = 0.f;
#pragma unroll
    for (int s = 0; s < 8; ++s) c[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka[s], qb[s], c[0], 0, 0, 0);
    if ((blk + 1) * kBlock > p.limit) {  // uniform
#pragma unroll
      for (int r = 0; r < 16; ++r)
        c[0][r] = (blk * kBlock + 8 * (r >> 2) + 4 * h + (r & 3) < p.limit) ? c[0][r] : -INFINITY;
    }
    f16x8 pa[1][2];
    float ps[1];
    soft_step<1>(a, c, sc, pa, ps);
    a.l += ps[0];
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(MORE ? 0x0F78 : 0x0F70);  // this block's V has landed (vmcnt(8): the next K may not)
    asm volatile("" ::: "memory");
    f16x8 va[D / 32][2];
    load_vt(vb, vo, ti, va);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);
    asm volatile("" ::: "memory");
    if constexpr (MORE) {
      issue(p.vp, vb, blk + kWaves, at_v);
      fetch(min(blk + 2 * kWaves, p.blk1 - 1));
    }
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt)
        a.acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va[dt][ks], pa[0][ks], a.acc[dt], 0, 0, 0);
  };
  if (blk < p.blk1) {  // uniform
    fetch(blk);
    issue(p.kp, kb, blk, at_k);
    issue(p.vp, vb, blk, at_v);
    fetch(min(blk + kWaves, p.blk1 - 1));
    for (; blk + kWaves < p.blk1; blk += kWaves) step.template operator()<true>();
    step.template operator()<false>();
  }
  a.l += __shfl_xor(a.l, 32, 64);
  // Each wavefront leaves its O in its own staging rows, [vector][dim], 64 dims in each array; chunk c of vector v in
  // slot c ^ (v % 16).
  if (l32 < p.nv) {
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = 8 * (dt & 1) + 2 * j + h;
        *reinterpret_cast<f32x4*>((dt < 2 ? kb : vb) + l32 * 256 + 16 * (c ^ (l32 & 15))) =
            f32x4{a.acc[dt][4 * j], a.acc[dt][4 * j + 1], a.acc[dt][4 * j + 2], a.acc[dt][4 * j + 3]};
      }
    if (h == 0) {
      sm_ml[wave][0][l32] = a.m;
      sm_ml[wave][1][l32] = a.l;
    }
  }
  __syncthreads();
  for (int it = threadIdx.x; it < p.nv * 32; it += kThreads) {
    const int v = it >> 5, c4 = it & 31;
    const uint8_t* base = (c4 < 16 ? st0 : st1) + v * 256 + 16 * ((c4 & 15) ^ (v & 15));
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) M = fmaxf(M, sm_ml[w][0][v]);
    const float ms = M == -INFINITY ? 0.f : M;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    float l = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = __builtin_amdgcn_exp2f(sm_ml[w][0][v] - ms);
      const f32x4 x = *reinterpret_cast<const f32x4*>(base + w * (kBlock * kRowB));
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(x[e], f, o[e]);
      l = fmaf(sm_ml[w][1][v], f, l);
    }
    *reinterpret_cast<f32x4*>(p.o + (size_t)v * D + 4 * c4) = o;
    if (c4 == 0) {
      p.ml[2 * v] = M;
      p.ml[2 * v + 1] = l;
    }
  }
  __syncthreads();  // the next piece writes the same LDS
}

// ------------------------------------------------------ up to 128 vectors -----
__device__ __forceinline__ void piece_tile(const Args& A, const Piece& p, uint8_t* st0, uint8_t* st1) {
  constexpr int NB = 2;
  constexpr int kTok = kBlock * NB;               // tokens per stage
  constexpr int kHalf = kTok * kRowB;             // bytes of K, then V
  constexpr int kRows = kTok / kWaves;            // rows of each a wavefront brings in
  static_assert(kRows == 16 && 2 * kHalf == kStage, "a wavefront's rows lie in one page");
  const int wave = uni(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int l32 = lane & 31, h = lane >> 5;
  const float sc = fabsf(A.scale_log2);
  const int nst = (p.blk1 - p.blk0 + NB - 1) / NB;  // (every token of the blocks counts)
  const int first16 = 2 * p.blk0 + wave, last16 = 2 * p.blk1 - 1;
  const bool busy = wave * kVec < p.nv;  // uniform

  // DMA of a stage: each wavefront brings in 16 rows of K and of V; past the last block it re-reads the last rows.
  const int lr = lane >> 4, ls = lane & 15;
  uint32_t at_k[4], at_v[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    at_k[u] = (4 * u + lr) * kRowB + 16 * (ls ^ (4 * u + lr));
    at_v[u] = (4 * u + lr) * kRowB + 16 * (ls ^ ((lr << 2) | u));
  }
  int page = 0;
  auto fetch = [&](int st) __attribute__((always_inline)) {
    page = p.ptrow[page_index(A, min(first16 + st * (kTok / 16), last16))];
  };
  auto issue = [&](uint8_t* buf, int st) __attribute__((always_inline)) {
    const int n = min(first16 + st * (kTok / 16), last16);
    const size_t base = rows16_at(A, p.h, page, n, page_index(A, n));
    const rsrc_t rk = make_rsrc(p.kp + base, 16 * kRowB), rv = make_rsrc(p.vp + base, 16 * kRowB);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      uint8_t* to = buf + (kRows * wave + 4 * u) * kRowB;
      buf16_to_lds(rk, to, at_k[u], 0);
      buf16_to_lds(rv, to + kHalf, at_v[u], 0);
    }
  };

  f16x8 qb[8];
  load_q(A, p, wave * kVec + l32, qb);
  Soft a;
  soft_init(a);
  const int krow = l32 * kRowB, kx = 16 * (h ^ (l32 & 15));
  const int ti = lane & 15, sub = (lane >> 4) & 1;
  int vo[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    vo[i] = kHalf + (8 * i + 4 * h + (ti >> 2)) * kRowB +
            16 * ((2 * sub + ((ti & 3) >> 1)) ^ (2 * i + h)) + 8 * (ti & 1);

  // The products run at a higher wave priority than the softmax: of the two wavefronts of a SIMD the one that feeds the
  // matrix cores goes first (64 rows after 32672 tokens 64.5 -> 62.6 us).
  auto blocks = [&](const uint8_t* buf, int blk) __attribute__((always_inline)) {
    __builtin_amdgcn_s_setprio(1);
    f32x16 c[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      f16x8 ka[8];
#pragma unroll
      for (int s = 0; s < 8; ++s)
        ka[s] = *reinterpret_cast<const f16x8*>(buf + krow + j * kBlock * kRowB + (kx ^ (32 * s)));
#pragma unroll
      for (int r = 0; r < 16; ++r) c[j][r] = 0.f;
#pragma unroll
      for (int s = 0; s < 8; ++s) c[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka[s], qb[s], c[j], 0, 0, 0);
    }
    f16x8 va[NB][D / 32][2];
    load_vt(buf, vo, ti, va[0]);  // before the softmax, which hides the LDS latency
    __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_sched_barrier(0);
    const bool both = blk + 1 < p.blk1;  // uniform
    if (!both) {
      asm volatile("" : "+v"(c[1]));  // (stays a branch: 16 selects a stage otherwise)
#pragma unroll
      for (int r = 0; r < 16; ++r) c[1][r] = -INFINITY;
    }
    f16x8 pa[NB][2];
    float ps[NB];
    soft_step<NB>(a, c, sc, pa, ps);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      if (j > 0 && !both) break;  // uniform
      a.l += ps[j];
      if (j > 0) load_vt(buf + j * kBlock * kRowB, vo, ti, va[j]);
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt)
          a.acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va[j][dt][ks], pa[j][ks], a.acc[dt], 0, 0, 0);
    }
  };
  auto step = [&](const uint8_t* cur, uint8_t* other, int st) __attribute__((always_inline)) {
    dma_wait_barrier();
    if (st + 1 < nst) {
      issue(other, st + 1);
      fetch(min(st + 2, nst - 1));
    }
    if (busy) blocks(cur, p.blk0 + st * NB);
    __builtin_amdgcn_s_setprio(0);
  };
  fetch(0);
  issue(st0, 0);
  fetch(min(1, nst - 1));
  for (int st = 0;;) {  // uniform
    step(st0, st1, st);
    if (++st >= nst) break;
    step(st1, st0, st);
    if (++st >= nst) break;
  }
  a.l += __shfl_xor(a.l, 32, 64);

  const int v = wave * kVec + l32;
  if (v < p.nv) {
    float* po = p.o + (size_t)v * D + 4 * h;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<f32x4*>(po + 32 * dt + 8 * j) =
            f32x4{a.acc[dt][4 * j], a.acc[dt][4 * j + 1], a.acc[dt][4 * j + 2], a.acc[dt][4 * j + 3]};
    if (h == 0) {
      p.ml[2 * v] = a.m;
      p.ml[2 * v + 1] = a.l;
    }
  }
  __syncthreads();  // every wavefront has read its last stage
}

// A row's place on the axis, whether it takes its group's prefix, and the tokens its last block lacks.
constexpr int kPadBits = 5, kTakes = 1 << kPadBits, kPlace = kPadBits + 1;

__global__ __launch_bounds__(kThreads, 2) void attn_shared_f16_d128(
    const f16* __restrict__ q, const f16* __restrict__ kp, const f16* __restrict__ vp, const int32_t* __restrict__ pt,
    const int32_t* __restrict__ lens, const int32_t* __restrict__ group_rows, const int32_t* __restrict__ prefix_lens,
    Args A) {
  __shared__ __align__(16) uint8_t st0[kStage];
  __shared__ __align__(16) uint8_t st1[kStage];
  __shared__ float sm_ml[kWaves][2][kVec];
  __shared__ int sm_scan[3][kWaves];
  // Group g: rows sm_row0[g] .. sm_row0[g + 1] - 1, shared blocks, place on the axis, first item.
  __shared__ int sm_row0[kMaxPrefixes + 1], sm_eff[kMaxPrefixes], sm_gstart[kMaxPrefixes], sm_item[kMaxPrefixes];
  __shared__ int sm_row[kMaxRows + 1];
  __shared__ int sm_find;
  const int G = A.Hq / A.Hkv, NG = A.NG, B = A.B, Hkv = A.Hkv;
  const int t = threadIdx.x, w = blockIdx.x / Hkv, h = blockIdx.x - w * Hkv;  // team, KV head
  const int max_ctx = A.max_pages * A.P16 * 16;

  // Everything the plan needs is loaded at once (it is bound by latency); lengths wait in the staging rows.
  int* sm_len = reinterpret_cast<int*>(st0);
  static_assert(kMaxRows * 4 <= kStage, "");
  int g0 = 0, g1 = 0, prefix = 0;
  if (t < NG) {
    g0 = group_rows[t];
    g1 = group_rows[t + 1];
    prefix = prefix_lens[t];
  }
  for (int r = t; r < B; r += kThreads) sm_len[r] = max(0, min(lens[r], max_ctx));
  if (t < NG) {
    sm_row0[t] = g0;
    if (t == NG - 1) sm_row0[NG] = g1;
  }
  // Rows out of order switch sharing off.
  const bool off = __syncthreads_or(t < NG && (g0 < 0 || g1 > B || g1 < g0)) || NG == 0;
  // Groups.  What is shared ends at the first row's own length (its pages are the ones read) and at whole blocks; a row
  // alone shares nothing.
  int v[3] = {0, 0, 0}, total[3], eff = 0;  // cost of the group's items, their number, cost of a row
  if (t < NG) {
    const int rows = off ? 0 : g1 - g0;
    if (rows > 1) eff = max(0, min(prefix, sm_len[g0])) / kBlock;
    v[1] = eff > 0 ? (rows * G + kTileVec - 1) / kTileVec : 0;
    v[0] = v[1] * (eff + kItemCost);
    sm_eff[t] = eff;
  }
  __syncthreads();
  const auto group_of = [&](int r) __attribute__((always_inline)) {  // -1: none
    if (off || r < sm_row0[0] || r >= sm_row0[NG]) return -1;
    int lo = 0, hi = NG - 1;  // the last group that starts at or before r (empty ones start where the next does)
    while (lo < hi) {
      const int m = (lo + hi + 1) >> 1;
      if (sm_row0[m] <= r) lo = m;
      else hi = m - 1;
    }
    return lo;
  };
  int rows_total = 0;
  const int gcost = v[0], gitems = v[1];
  int gstart = 0;
  for (int r0 = 0; r0 < B; r0 += kThreads) {  // uniform
    const int r = r0 + t;
    int cost = 0, word = 0;
    if (r < B) {
      const int L = sm_len[r], g = group_of(r), e = g >= 0 ? sm_eff[g] : 0;
      const bool takes = e > 0 && L >= e * kBlock;  // a row shorter than the prefix reads it alone
      const int blocks = (L + kBlock - 1) / kBlock - (takes ? e : 0);
      cost = blocks > 0 ? blocks + kItemCost : 0;
      word = (takes ? kTakes : 0) | (-L & (kBlock - 1));
    }
    if (r0 == 0) {
      v[2] = cost;
      block_scan<3>(v, total, sm_scan);
      gstart = v[0] - gcost;
      if (t < NG) {
        sm_gstart[t] = gstart;
        sm_item[t] = v[1] - gitems;
      }
    } else {
      int c[1] = {cost}, sum[1];
      block_scan<1>(c, sum, sm_scan);
      v[2] = c[0];
      total[2] = sum[0];
    }
    if (r < B) sm_row[r] = ((total[0] + rows_total + v[2] - cost) << kPlace) | word;
    rows_total += total[2];
  }
  const int prefix_total = total[0], all = prefix_total + rows_total;
  if (t == 0) sm_row[B] = all << kPlace;
  const int teams = gridDim.x / Hkv;
  const int stretch = max((all + teams - 1) / teams, kMinStretch);
  const int a = w * stretch, b = min(all, a + stretch);
  __syncthreads();

  // The join's records, shared out over the workgroups from the last one on (the ones without work of their own).
  for (int r = (int)(gridDim.x - 1 - blockIdx.x) + t * (int)gridDim.x; r < B; r += kThreads * (int)gridDim.x) {
    const int word = sm_row[r], place = word >> kPlace, span = (sm_row[r + 1] >> kPlace) - place;
    const auto pieces = [&](int start, int blocks, int item) {  // item's blocks from `start` on
      const int w0 = start / stretch;
      return Pieces{w0 + item, (start + blocks - 1) / stretch - w0 + 1};
    };
    RowRec rec{{{0, 0}, {0, 0}}, {0, 0}, 0, 0};
    if (word & kTakes) {
      const int g = group_of(r), tiles = ((sm_row0[g + 1] - sm_row0[g]) * G + kTileVec - 1) / kTileVec;
      const int shared = sm_eff[g];
      rec.first = (r - sm_row0[g]) * G;
      const int tile = rec.first / kTileVec;
      for (int k = 0; k < 2 && tile + k < tiles; ++k)
        rec.prefix[k] = pieces(sm_gstart[g] + (tile + k) * (shared + kItemCost) + kItemCost, shared,
                               sm_item[g] + tile + k);
    }
    if (span > 0) rec.own = pieces(place + kItemCost, span - kItemCost, r);
    A.rows[r] = rec;
  }
  if (a >= b) return;  // uniform
  // The unit (group, then NG + row) in which the stretch begins.
  if (a < prefix_total) {
    if (t < NG && gstart <= a && a < gstart + gcost) sm_find = t;
  } else {
    for (int r = t; r < B; r += kThreads)
      if ((sm_row[r] >> kPlace) <= a && a < (sm_row[r + 1] >> kPlace)) sm_find = NG + r;
  }
  __syncthreads();

  for (int u = uni(sm_find); u < NG + B; ++u) {  // uniform
    const bool pre = u < NG;
    const int r = u - NG;
    int rows = 0, count = 1, start, first = 0, blocks, limit;  // items, their place, blocks, tokens
    if (pre) {
      rows = uni(sm_row0[u + 1]) - uni(sm_row0[u]);
      blocks = uni(sm_eff[u]);
      count = (rows * G + kTileVec - 1) / kTileVec;
      start = uni(sm_gstart[u]);
      limit = blocks * kBlock;
    } else {
      const int word = uni(sm_row[r]);
      start = word >> kPlace;
      blocks = (uni(sm_row[r + 1]) >> kPlace) - start - kItemCost;
      if (word & kTakes) first = uni(sm_eff[uni(group_of(r))]);
      limit = (first + blocks) * kBlock - (word & (kBlock - 1));
    }
    if (start >= b) break;
    if (blocks <= 0) continue;
    const int c = blocks + kItemCost;
    for (int i = max(0, (a - start) / c); i < count && start + i * c < b; ++i) {
      const int st = start + i * c + kItemCost;
      const int k0 = max(0, min(a - st, blocks)), k1 = max(0, min(b - st, blocks));
      if (k0 >= k1) continue;
      Piece p;
      p.q = q;
      p.kp = kp;
      p.vp = vp;
      p.h = h;
      p.blk0 = first + k0;
      p.blk1 = first + k1;
      p.limit = limit;
      p.vrow = pre ? uni(sm_row0[u]) : r;
      p.v0 = pre ? i * kTileVec : 0;
      p.nv = pre ? min(kTileVec, rows * G - p.v0) : G;
      p.ptrow = pt + (size_t)p.vrow * A.max_pages;
      const int slot = w + (pre ? uni(sm_item[u]) + i : r);
      const size_t at = ((size_t)slot * Hkv + h) * (pre ? kTileVec : G);
      p.o = (pre ? A.pre_o : A.suf_o) + at * D;
      p.ml = (pre ? A.pre_ml : A.suf_ml) + at * 2;
      if (p.nv > kVec) piece_tile(A, p, st0, st1);
      else piece_stream(A, p, st0, st1, sm_ml);
    }
  }
}

// out = sum 2^(m_i - M) O_i / sum 2^(m_i - M) l_i over the pieces of a query vector: those of its group's prefix, then
// those of its own part.  Two half-wavefronts per vector, each with every second piece, four dims a lane; lane k takes
// (m, l) of every 32nd piece.  Bound by latency (record, then pieces), so a half-wavefront has four O on their way, the
// first ones along with the (m, l).  Half-wavefronts per vector, us of the whole call: 64 rows after 2048 tokens, 9
// pieces a vector, 24.8 with one, 21.0 with two, 24.6 with four; 20 groups of 4 rows 31.4, 30.9, 32.7.
// A row without tokens gives zeros; one whose scores are all -inf NaN, as a softmax over them does.
__global__ __launch_bounds__(256) void attn_shared_join(Args A, f16* __restrict__ out) {
  constexpr int W = 2, U = 4, kVecs = 8 / W;
  __shared__ f32x4 sm_o[kVecs][32];
  const int part = threadIdx.x >> 5, lane = threadIdx.x & 31, s = part % W, vec = part / W;
  const int id = blockIdx.x * kVecs + vec;
  const bool live = id < A.B * A.Hq;
  const int row = live ? id / A.Hq : 0;
  const int head = live ? id - row * A.Hq : 0, G = A.Hq / A.Hkv;
  const int h = head / G, g = head - h * G;
  const RowRec rec = A.rows[row];
  const int v = rec.first + g, later = v / kTileVec != rec.first / kTileVec;
  const Pieces pre = later ? rec.prefix[1] : rec.prefix[0];
  const int n = live ? pre.count + rec.own.count : 0;
  // Query vector `at` of piece k's slot: (m, l) and O.
  const size_t pre_at = ((size_t)pre.slot * A.Hkv + h) * kTileVec + v % kTileVec;
  const size_t own_at = ((size_t)rec.own.slot * A.Hkv + h) * G + g;
  const auto at = [&](int k) {
    return k < pre.count ? pre_at + (size_t)k * A.Hkv * kTileVec : own_at + (size_t)(k - pre.count) * A.Hkv * G;
  };
  const auto ml_of = [&](int k) {
    return *reinterpret_cast<const float2*>((k < pre.count ? A.pre_ml : A.suf_ml) + 2 * at(k));
  };
  const auto o_of = [&](int k) {
    return *reinterpret_cast<const f32x4*>((k < pre.count ? A.pre_o : A.suf_o) + D * at(k) + 4 * lane);
  };
  float den = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  if (n > 0) {
    float2 ml = lane < n ? ml_of(lane) : make_float2(-INFINITY, 0.f);
    f32x4 x[U];
    const auto load = [&](int k0) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int k = k0 + s + W * j;
        x[j] = o_of(min(k, n - 1));
      }
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
      for (int j0 = k0; j0 < min(n, k0 + 32); j0 += W * U) {
#pragma unroll
        for (int j = 0; j < U; ++j) {
          const int k = j0 + s + W * j;
          const float fk = __shfl(f, k - k0, 32);
          if (k < n) {
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = fmaf(x[j][e], fk, o[e]);
          }
        }
        if (j0 + W * U < n) load(j0 + W * U);
      }
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) den += __shfl_xor(den, d, 32);
  }
  if (s > 0) sm_o[vec][lane] = o;
  __syncthreads();
  if (s > 0 || !live) return;
  o += sm_o[vec][lane];
  const float inv = n == 0 ? 0.f : den == 0.f ? NAN : 1.f / den;
  f16x4 y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = static_cast<f16>(as_f32_value(o[e] * inv));
  *reinterpret_cast<f16x4*>(out + (size_t)id * D + 4 * lane) = y;
}

int teams_of(int Hkv) { return max(1, kGroups / Hkv); }

size_t round16(size_t n) { return (n + 15) / 16 * 16; }

Layout layout(int B, int NG, int Hq, int Hkv) {
  const int G = Hq / Hkv;
  Layout l{};
  size_t at = 0;
  const auto take = [&](size_t bytes) {
    const size_t p = at;
    at += round16(bytes);
    return p;
  };
  // tiles of n_g rows: ceil(n_g G / 128), so at most B G / 128 + NG in all
  const size_t pre = NG ? (size_t)(teams_of(Hkv) + (long)B * G / kTileVec + NG) * Hkv * kTileVec : 0;
  const size_t suf = (size_t)(teams_of(Hkv) + B) * Hkv * G;
  l.rows = take(sizeof(RowRec) * B);
  l.pre_o = take(pre * D * sizeof(float));
  l.pre_ml = take(pre * 2 * sizeof(float));
  l.suf_o = take(suf * D * sizeof(float));
  l.suf_ml = take(suf * 2 * sizeof(float));
  l.total = at;
  return l;
}

// Sizes that the shared kernel takes: fp16, head_dim 128, pages of a multiple of 16 tokens, up to 32 query heads per
// KV head, and an axis that sm_row holds.  Others run the decode attention over each row's whole context.
bool shares(int B, int NG, int Hq, int Hkv, int head_dim, int P, int max_pages, int kv_dtype) {
  const int G = Hq / Hkv;
  const long per_item = (long)max_pages * P / kBlock + 1 + kItemCost;
  const long items = (long)B * G / kTileVec + NG + B;
  // (page_index is exact while (tokens / 16) (P / 16) < 2^32)
  return kv_dtype == CIR_F16 && head_dim == D && P % 16 == 0 && (long)max_pages * P / 16 * (P / 16) < (1L << 32) &&
         G <= kVec && NG <= kMaxPrefixes && B <= kMaxRows && (long)B * Hq < kMaxVectors && Hkv < kMaxKvHeads &&
         per_item < (1L << 31) && per_item * items < (1L << (31 - kPlace));
}

}  // namespace
}  // namespace cir

using namespace cir;

extern "C" size_t cir_shared_attention_workspace_bytes(int batch, int groups, int num_heads, int num_kv_heads,
                                                       int head_dim, int page_size, int max_pages, int kv_dtype) {
  if (batch <= 0 || groups < 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads || head_dim <= 0 ||
      page_size <= 0 || max_pages <= 0 || (long)page_size * max_pages > 0x7fffffffL)
    return 0;
  // (the larger of the two paths: the pools' addresses, which are not known here, decide between them too)
  const size_t plain = cir_paged_attention_workspace_bytes(batch, num_heads, head_dim, max_pages * page_size);
  if (!shares(batch, groups, num_heads, num_kv_heads, head_dim, page_size, max_pages, kv_dtype)) return plain;
  const size_t own = layout(batch, groups, num_heads, num_kv_heads).total;
  return own > plain ? own : plain;
}

extern "C" int cir_paged_decode_attention_shared(const void* q, const void* k_pool, const void* v_pool,
                                                 const int32_t* page_table, const int32_t* seq_lens,
                                                 const int32_t* group_rows, const int32_t* prefix_lens, int groups,
                                                 void* out, void* workspace, size_t workspace_bytes, int batch,
                                                 int num_heads, int num_kv_heads, int head_dim, int page_size,
                                                 int max_pages, float scale, int kv_dtype, void* stream) {
  CIR_CHECK_ARG(batch >= 0 && groups >= 0, "attention_shared: batch and groups must be >= 0");
  if (batch == 0) return 0;
  CIR_CHECK_ARG(q && k_pool && v_pool && page_table && seq_lens && out, "attention_shared: null pointer");
  CIR_CHECK_ARG(groups == 0 || (group_rows && prefix_lens), "attention_shared: null group_rows or prefix_lens");
  CIR_CHECK_ARG(num_kv_heads > 0 && num_heads > 0 && num_heads % num_kv_heads == 0,
                "attention_shared: num_heads (%d) must be a multiple of num_kv_heads (%d)", num_heads, num_kv_heads);
  CIR_CHECK_ARG(head_dim > 0 && head_dim <= 256, "attention_shared: head_dim %d out of range (1..256)", head_dim);
  CIR_CHECK_ARG(page_size > 0 && max_pages > 0 && (long)page_size * max_pages <= 0x7fffffffL,
                "attention_shared: page_size and max_pages must be positive, and their product a 32-bit number");
  CIR_CHECK_ARG(kv_dtype == CIR_F16 || kv_dtype == CIR_F32, "attention_shared: kv_dtype must be CIR_F16 or CIR_F32");
  // DMA takes 16-byte groups of the pools; q is read by 16 bytes, out written by 8.
  if (!shares(batch, groups, num_heads, num_kv_heads, head_dim, page_size, max_pages, kv_dtype) ||
      ((uintptr_t)q | (uintptr_t)k_pool | (uintptr_t)v_pool) % 16 || (uintptr_t)out % 8)
    return cir_paged_decode_attention(q, k_pool, v_pool, page_table, seq_lens, out, workspace, workspace_bytes, batch,
                                      num_heads, num_kv_heads, head_dim, page_size, max_pages, scale, kv_dtype, stream);
  const Layout l = layout(batch, groups, num_heads, num_kv_heads);
  CIR_CHECK_ARG(workspace && workspace_bytes >= l.total && (uintptr_t)workspace % 16 == 0,
                "attention_shared: workspace too small or not on 16 bytes (%zu < %zu)", workspace_bytes, l.total);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const float scale_log2 = scale * kLog2e;
  const uint32_t P16 = page_size / 16;
  const Args A{reinterpret_cast<RowRec*>(ws + l.rows),
               reinterpret_cast<float*>(ws + l.pre_o), reinterpret_cast<float*>(ws + l.pre_ml),
               reinterpret_cast<float*>(ws + l.suf_o), reinterpret_cast<float*>(ws + l.suf_ml), batch, groups, num_heads,
               num_kv_heads, (int)P16, max_pages, (uint32_t)(((1ull << 32) + P16 - 1) / P16),
               scale_log2 == 0.f ? FLT_MIN : scale_log2};  // (a masked score is -inf: -inf * 0 would be NaN)
  hipStream_t s = as_stream(stream);
  attn_shared_f16_d128<<<teams_of(num_kv_heads) * num_kv_heads, kThreads, 0, s>>>(
      static_cast<const f16*>(q), static_cast<const f16*>(k_pool), static_cast<const f16*>(v_pool), page_table, seq_lens,
      group_rows, prefix_lens, A);
  const int st = launch_status();
  if (st) return st;
  const unsigned vectors = (unsigned)batch * num_heads;
  attn_shared_join<<<(vectors + 3) / 4, 256, 0, s>>>(A, static_cast<f16*>(out));
  return launch_status();
}
