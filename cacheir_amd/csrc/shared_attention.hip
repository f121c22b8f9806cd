// Decode attention for a batch whose rows share prefixes by groups: the K and V of a prefix
// are read once for the query vectors of all rows of its group, not once per row.
//
// out[b] = softmax(scale q[b] K[b]^T) V[b] over the row's paged context, as the decode
// attention computes it.  Softmax over a context in pieces: each piece gives (m, l, O) =
// (max, sum of e^(s - m), sum of e^(s - m) v), and the pieces of a row, its group's prefix
// among them, are joined by sum 2^(m_i - M) (l_i, O_i) in a second launch.
//
// Work.  Two kinds of item: (group, tile of 128 query vectors, KV head) over the prefix, and
// (row, KV head) over what follows it; a group of up to 32 vectors makes one tile of 32.
// An item costs kItemCost + its 32-token blocks; the items lie on one axis, prefixes first,
// and each of kGroups persistent workgroups takes an equal stretch of that axis, whatever
// rows it crosses: lengths live on the device, and a grid cut by rows or by a fixed number
// of splits leaves CUs idle behind the longest row.  Every workgroup finds its stretch by a
// scan over the groups and rows (from L2, ~1 us).  A piece of item i computed by workgroup w
// has the slot w + i: along the axis one of the two grows from piece to piece, so slots are
// unique, and the join finds an item's pieces from its start and the stretch alone.
//
// Bodies (8 wavefronts, one workgroup per CU, MFMA 32x32x16 f16, S^T = K Q^T and
// O^T = V^T P^T as in the prefill attention, whose LDS swizzles these are):
//   * piece_stream, up to 32 query vectors: bound by the read of K and V.  Each wavefront
//     walks blocks of its own (every 8th) and stages them by DMA in LDS of its own: no
//     barriers, K of the next block is on its way once this block's K is in registers, and
//     V likewise, so a CU has 64 to 128 KiB in flight.
//   * piece_tile, up to 128 vectors: bound by the matrix cores and the softmax.  Four
//     wavefronts of 32 vectors, twice: two sets take turns of 64-token pairs of blocks; K
//     and V go through LDS once for all.
// P is rounded to fp16 for the second product (relative 2^-11 of a weight) and l sums the
// rounded values, so a row's weights still add up to one; everything else is fp32.
#include "attn_tile.hpp"

#include <float.h>
#include <math.h>

namespace cir {
namespace {

constexpr int D = 128;
constexpr int kBlock = 32;        // tokens of an MFMA tile
constexpr int kVec = 32;          // query vectors of an MFMA tile
constexpr int kWaves = 8;
constexpr int kThreads = 64 * kWaves;
constexpr int kGroups = 256;      // workgroups: one per CU
constexpr int kTileVec = 128;     // query vectors of a prefix tile
constexpr int kItemCost = 3;      // start and join of a piece, in blocks
constexpr int kMinStretch = 8;    // blocks per workgroup at least (one per wavefront)
constexpr int kMaxPrefixes = 512;   // groups: one per thread
constexpr int kMaxRows = 4096;
constexpr int kRowB = 2 * D;      // bytes of a K or V row

// Workspace: header, then one record per group and row, then the pieces.
struct Plan {
  int stretch, pad[3];
};
struct GroupRec {
  int start, first_item, blocks, row0;  // blocks 0: nothing shared
};
struct RowRec {
  int start, blocks, group, length;  // group -1: the row takes no prefix piece
};
struct Layout {
  size_t groups, rows, pre_o, pre_ml, suf_o, suf_ml, total;  // bytes
  int pre_slots, suf_slots;
};

struct Args {
  Plan* plan;
  GroupRec* groups;
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

// Inclusive sum over the workgroup, and its total.
__device__ __forceinline__ int block_scan(int v, int* scratch, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int o = __shfl_up(v, off, 64);
    v += lane >= off ? o : 0;
  }
  if (lane == 63) scratch[wave] = v;
  __syncthreads();
  total = 0;
  int before = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    before += w < wave ? scratch[w] : 0;
    total += scratch[w];
  }
  __syncthreads();
  return v + before;
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
template <int NB>
__device__ __forceinline__ void soft_step(Soft& a, f32x16 (&c)[NB], float sc, f16x8 (&pa)[NB][2], float (&ps)[NB]) {
  float mx = c[0][0];
#pragma unroll
  for (int r = 1; r < 16 * NB; ++r) mx = fmaxf(mx, c[r >> 4][r & 15]);
  mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * sc;
  if (__builtin_amdgcn_ballot_w64(mx > a.m) != 0) {  // uniform
    const float mn = fmaxf(a.m, mx);
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
    for (int r = 0; r < 16; ++r) {
      pa[j][r >> 3][r & 7] = static_cast<f16>(__builtin_amdgcn_exp2f(fmaf(c[j][r], pc, -ms)));
      ps[j] += static_cast<float>(pa[j][r >> 3][r & 7]);
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

constexpr int kStage = 64 * 1024;  // bytes of each of the two LDS arrays

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
        buf16_to_lds(r, buf + (16 * j + 4 * u) * kRowB, off, 0);
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
// VW x CW wavefronts: VW tiles of 32 vectors, CW sets that take turns of NB blocks.
__device__ __forceinline__ void piece_tile(const Args& A, const Piece& p, uint8_t* st0, uint8_t* st1,
                                           float (*sm_ml)[2][kVec]) {
  constexpr int VW = 4, CW = 2, NB = 2;
  constexpr int kTok = kBlock * NB * CW;          // tokens per stage
  constexpr int kHalf = kTok * kRowB;             // bytes of K, then V
  constexpr int kRows = kTok / kWaves;            // rows of each a wavefront brings in
  static_assert(kRows == 16 && 2 * kHalf == kStage, "a wavefront's rows lie in one page");
  const int wave = uni(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int vw = wave % VW, cw = wave / VW;
  const int l32 = lane & 31, h = lane >> 5;
  const float sc = fabsf(A.scale_log2);
  const int nst = (p.blk1 - p.blk0 + NB * CW - 1) / (NB * CW);  // (every token of the blocks counts)
  const int first16 = 2 * p.blk0 + wave, last16 = 2 * p.blk1 - 1;
  const bool busy = vw * kVec < p.nv;  // uniform

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
  load_q(A, p, vw * kVec + l32, qb);
  Soft a;
  soft_init(a);
  const int krow = (kBlock * NB * cw + l32) * kRowB, kx = 16 * (h ^ (l32 & 15));
  const int ti = lane & 15, sub = (lane >> 4) & 1;
  int vo[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    vo[i] = kHalf + (kBlock * NB * cw + 8 * i + 4 * h + (ti >> 2)) * kRowB +
            16 * ((2 * sub + ((ti & 3) >> 1)) ^ (2 * i + h)) + 8 * (ti & 1);

  auto blocks = [&](const uint8_t* buf, int blk) __attribute__((always_inline)) {
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
    __builtin_amdgcn_sched_barrier(0);
    const bool both = blk + 1 < p.blk1;  // uniform
    if (!both) {
#pragma unroll
      for (int r = 0; r < 16; ++r) c[1][r] = -INFINITY;
    }
    f16x8 pa[NB][2];
    float ps[NB];
    soft_step<NB>(a, c, sc, pa, ps);
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
    const int blk = p.blk0 + (st * CW + cw) * NB;
    if (busy && blk < p.blk1) blocks(cur, blk);
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

  // Join the two sets: the second parks (m, l, O) in the first array.
  dma_wait_barrier();  // every wavefront has read its last stage
  float* park = reinterpret_cast<float*>(st0 + vw * (64 * 64 * 4)) + lane;
  if (cw > 0 && busy) {
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) park[(16 * dt + r) * 64] = a.acc[dt][r];
    if (h == 0) {
      sm_ml[vw][0][l32] = a.m;
      sm_ml[vw][1][l32] = a.l;
    }
  }
  __syncthreads();
  if (cw == 0 && busy) {
    const float mg = sm_ml[vw][0][l32], lg = sm_ml[vw][1][l32];
    const float mn = fmaxf(a.m, mg), ms = mn == -INFINITY ? 0.f : mn;
    const float fa = __builtin_amdgcn_exp2f(a.m - ms), fb = __builtin_amdgcn_exp2f(mg - ms);
    const int v = vw * kVec + l32;
    const float l = fmaf(a.l, fa, lg * fb);
    f32x4 o[D / 32][4];
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[dt][r >> 2][r & 3] = fmaf(a.acc[dt][r], fa, park[(16 * dt + r) * 64] * fb);
    if (v < p.nv) {
      float* po = p.o + (size_t)v * D + 4 * h;
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int j = 0; j < 4; ++j) *reinterpret_cast<f32x4*>(po + 32 * dt + 8 * j) = o[dt][j];
      if (h == 0) {
        p.ml[2 * v] = mn;
        p.ml[2 * v + 1] = l;
      }
    }
  }
  __syncthreads();
}

// Blocks of a row's own part, where it starts, the group whose prefix it takes (-1: none) and its length.
struct Own {
  int first, blocks, group, length;
};

__global__ __launch_bounds__(kThreads, 2) void attn_shared_f16_d128(
    const f16* __restrict__ q, const f16* __restrict__ kp, const f16* __restrict__ vp, const int32_t* __restrict__ pt,
    const int32_t* __restrict__ lens, const int32_t* __restrict__ group_rows, const int32_t* __restrict__ prefix_lens,
    Args A) {
  __shared__ __align__(16) uint8_t st0[kStage];
  __shared__ __align__(16) uint8_t st1[kStage];
  __shared__ float sm_ml[kWaves][2][kVec];
  __shared__ int sm_scan[kWaves];
  // Group g: rows sm_row0[g] .. sm_row0[g + 1] - 1, shared blocks, place on the axis, first item.
  __shared__ int sm_row0[kMaxPrefixes + 1], sm_eff[kMaxPrefixes], sm_gstart[kMaxPrefixes], sm_item[kMaxPrefixes];
  __shared__ int sm_rstart[kMaxRows + 1];  // place of row r's items on the axis
  __shared__ int sm_find;
  const int t = threadIdx.x, w = blockIdx.x;
  const int G = A.Hq / A.Hkv, NG = A.NG, B = A.B, Hkv = A.Hkv;
  const int max_ctx = A.max_pages * A.P16 * 16;

  // Groups.  What is shared ends at the first row's own length (its pages are the ones read) and at whole blocks;
  // a row alone shares nothing, and rows out of order switch sharing off.
  bool bad = false;
  for (int g = t; g <= NG; g += kThreads) {
    const int r = group_rows[g];
    bad |= r < 0 || r > B || (g < NG && group_rows[g + 1] < r);
    sm_row0[g] = r;
  }
  const bool off = __syncthreads_or(bad);
  int eff = 0, cost = 0, n = 0;
  if (t < NG) {
    const int r0 = sm_row0[t], rows = off ? 0 : sm_row0[t + 1] - r0;
    if (rows > 1) eff = max(0, min(min(prefix_lens[t], lens[r0]), max_ctx)) / kBlock;
    n = eff > 0 ? (rows * G + kTileVec - 1) / kTileVec * Hkv : 0;
    cost = n * (eff + kItemCost);
    sm_eff[t] = eff;
  }
  int total, items;
  const int gstart = block_scan(cost, sm_scan, total) - cost, item = block_scan(n, sm_scan, items) - n;
  if (t < NG) {
    sm_gstart[t] = gstart;
    sm_item[t] = item;
    if (w == 0) A.groups[t] = GroupRec{gstart, item, eff, sm_row0[t]};
  }
  __syncthreads();
  const int prefix_total = total;

  const auto own_of = [&](int r) __attribute__((always_inline)) {
    const int L = max(0, min(lens[r], max_ctx));
    int g = -1;
    if (!off && NG > 0 && r >= sm_row0[0] && r < sm_row0[NG]) {
      int lo = 0, hi = NG - 1;  // the last group that starts at or before r (empty ones start where the next does)
      while (lo < hi) {
        const int m = (lo + hi + 1) >> 1;
        if (sm_row0[m] <= r) lo = m;
        else hi = m - 1;
      }
      // a row shorter than the prefix reads it alone
      if (sm_eff[lo] > 0 && L >= sm_eff[lo] * kBlock) g = lo;
    }
    const int first = g >= 0 ? sm_eff[g] : 0;
    return Own{first, (L + kBlock - 1) / kBlock - first, g, L};
  };
  for (int r0 = 0; r0 < B; r0 += kThreads) {  // uniform
    const int r = r0 + t;
    Own o{0, 0, -1, 0};
    if (r < B) o = own_of(r);
    const int c = o.blocks > 0 ? Hkv * (o.blocks + kItemCost) : 0;
    int sum;
    const int start = total + block_scan(c, sm_scan, sum) - c;
    if (r < B) {
      sm_rstart[r] = start;
      if (w == 0) A.rows[r] = RowRec{start, o.blocks, o.group, o.length};
    }
    total += sum;
  }
  if (t == 0) sm_rstart[B] = total;
  const int stretch = max((total + kGroups - 1) / kGroups, kMinStretch);
  if (w == 0 && t == 0) A.plan->stretch = stretch;
  const int a = w * stretch, b = min(total, a + stretch);
  if (a >= b) return;  // uniform
  // The unit (group, then NG + row) in which the stretch begins.
  __syncthreads();
  if (a < prefix_total) {
    if (t < NG && gstart <= a && a < gstart + cost) sm_find = t;
  } else {
    for (int r = t; r < B; r += kThreads)
      if (sm_rstart[r] <= a && a < sm_rstart[r + 1]) sm_find = NG + r;
  }
  __syncthreads();

  for (int u = uni(sm_find); u < NG + B; ++u) {  // uniform
    const bool pre = u < NG;
    const int r = u - NG;
    Own o{0, 0, -1, 0};
    int rows = 0, count = Hkv, start;
    if (pre) {
      rows = uni(sm_row0[u + 1]) - uni(sm_row0[u]);
      o.blocks = uni(sm_eff[u]);
      o.length = o.blocks * kBlock;
      count = (rows * G + kTileVec - 1) / kTileVec * Hkv;
      start = uni(sm_gstart[u]);
    } else {
      o = own_of(r);
      o.first = uni(o.first);
      o.blocks = uni(o.blocks);
      o.length = uni(o.length);
      start = uni(sm_rstart[r]);
    }
    if (start >= b) break;
    if (o.blocks <= 0) continue;
    const int c = o.blocks + kItemCost;
    for (int i = max(0, (a - start) / c); i < count && start + i * c < b; ++i) {
      const int st = start + i * c + kItemCost;
      const int k0 = max(0, min(a - st, o.blocks)), k1 = max(0, min(b - st, o.blocks));
      if (k0 >= k1) continue;
      Piece p;
      p.q = q;
      p.kp = kp;
      p.vp = vp;
      p.blk0 = o.first + k0;
      p.blk1 = o.first + k1;
      p.limit = o.length;
      if (pre) {
        const int tile = i / Hkv;
        p.h = i - tile * Hkv;
        p.vrow = uni(sm_row0[u]);
        p.v0 = tile * kTileVec;
        p.nv = min(kTileVec, rows * G - p.v0);
        const size_t slot = (size_t)(w + uni(sm_item[u]) + i) * kTileVec;
        p.o = A.pre_o + slot * D;
        p.ml = A.pre_ml + slot * 2;
      } else {
        p.h = i;
        p.vrow = r;
        p.v0 = 0;
        p.nv = G;
        const size_t slot = (size_t)(w + r * Hkv + i) * G;
        p.o = A.suf_o + slot * D;
        p.ml = A.suf_ml + slot * 2;
      }
      p.ptrow = pt + (size_t)p.vrow * A.max_pages;
      if (p.nv > kVec) piece_tile(A, p, st0, st1, sm_ml);
      else piece_stream(A, p, st0, st1, sm_ml);
    }
  }
}

// out = sum 2^(m_i - M) O_i / sum 2^(m_i - M) l_i over the pieces of a query vector: those of its group's prefix, then
// those of its own part, in order.  32 lanes per vector, four dims each; lane k takes (m, l) of every 32nd piece.
// A row without tokens gives zeros; one whose scores are all -inf NaN, as a softmax over them does.
__global__ __launch_bounds__(256) void attn_shared_join(Args A, f16* __restrict__ out) {
  const int id = (int)((blockIdx.x * 256u + threadIdx.x) >> 5), lane = threadIdx.x & 31;
  const int row = id / A.Hq;
  if (row >= A.B) return;
  const int head = id - row * A.Hq, G = A.Hq / A.Hkv;
  const int h = head / G, g = head - h * G;
  const int stretch = A.plan->stretch;
  const RowRec rr = A.rows[row];
  const float *po[2], *pm[2];  // O and (m, l) of the first piece of each kind
  size_t step[2];              // vectors from one piece to the next
  int count[2] = {0, 0};
  if (rr.group >= 0) {
    const GroupRec gr = A.groups[rr.group];
    const int v = (row - gr.row0) * G + g, tile = v / kTileVec, i = tile * A.Hkv + h;
    const int st = gr.start + i * (gr.blocks + kItemCost) + kItemCost;
    const int w0 = st / stretch, w1 = (st + gr.blocks - 1) / stretch;
    const size_t at = (size_t)(w0 + gr.first_item + i) * kTileVec + (v - tile * kTileVec);
    po[0] = A.pre_o + at * D;
    pm[0] = A.pre_ml + at * 2;
    step[0] = kTileVec;
    count[0] = w1 - w0 + 1;
  }
  if (rr.blocks > 0) {
    const int st = rr.start + h * (rr.blocks + kItemCost) + kItemCost;
    const int w0 = st / stretch, w1 = (st + rr.blocks - 1) / stretch;
    const size_t at = (size_t)(w0 + row * A.Hkv + h) * G + g;
    po[1] = A.suf_o + at * D;
    pm[1] = A.suf_ml + at * 2;
    step[1] = G;
    count[1] = w1 - w0 + 1;
  }
  float M = -INFINITY;
#pragma unroll
  for (int s = 0; s < 2; ++s)
    for (int k = lane; k < count[s]; k += 32) M = fmaxf(M, pm[s][k * step[s] * 2]);
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) M = fmaxf(M, __shfl_xor(M, x, 32));
  const float ms = M == -INFINITY ? 0.f : M;
  float den = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < 2; ++s)
    for (int k0 = 0; k0 < count[s]; k0 += 32) {
      float f = 0.f;
      if (k0 + lane < count[s]) {
        const float* ml = pm[s] + (k0 + lane) * step[s] * 2;
        f = __builtin_amdgcn_exp2f(ml[0] - ms);
        den = fmaf(ml[1], f, den);
      }
      const int n = min(32, count[s] - k0);
      for (int j = 0; j < n; ++j) {
        const float fj = __shfl(f, j, 32);
        const f32x4 x = *reinterpret_cast<const f32x4*>(po[s] + (k0 + j) * step[s] * D + 4 * lane);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = fmaf(x[e], fj, o[e]);
      }
    }
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) den += __shfl_xor(den, x, 32);
  const float inv = den == 0.f ? (rr.length > 0 ? NAN : 0.f) : 1.f / den;
  f16x4 y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = static_cast<f16>(as_f32_value(o[e] * inv));
  *reinterpret_cast<f16x4*>(out + (size_t)id * D + 4 * lane) = y;
}

size_t round16(size_t n) { return (n + 15) / 16 * 16; }

Layout layout(int B, int NG, int Hq, int Hkv) {
  const int G = Hq / Hkv;
  Layout l{};
  // tiles of n_g rows: ceil(n_g G / 128), so at most B G / 128 + NG in all
  l.pre_slots = kGroups + (int)(((long)B * G / kTileVec + NG) * Hkv);
  l.suf_slots = kGroups + B * Hkv;
  size_t at = round16(sizeof(Plan));
  const auto take = [&](size_t bytes) {
    const size_t p = at;
    at += round16(bytes);
    return p;
  };
  l.groups = take(sizeof(GroupRec) * NG);
  l.rows = take(sizeof(RowRec) * B);
  l.pre_o = take((size_t)(NG ? l.pre_slots : 0) * kTileVec * D * sizeof(float));
  l.pre_ml = take((size_t)(NG ? l.pre_slots : 0) * kTileVec * 2 * sizeof(float));
  l.suf_o = take((size_t)l.suf_slots * G * D * sizeof(float));
  l.suf_ml = take((size_t)l.suf_slots * G * 2 * sizeof(float));
  l.total = at;
  return l;
}

// Sizes that the shared kernel takes: fp16, head_dim 128, pages of a multiple of 16 tokens, up to 32 query heads per KV
// head, and an axis that 32 bits number.  Others run the decode attention over each row's whole context.
bool shares(int B, int NG, int Hq, int Hkv, int head_dim, int P, int max_pages, int kv_dtype) {
  const int G = Hq / Hkv;
  const long per_item = (long)max_pages * P / kBlock + 1 + kItemCost;
  const long items = ((long)B * G / kTileVec + NG + B) * Hkv;
  // (page_index is exact while (tokens / 16) (P / 16) < 2^32)
  return kv_dtype == CIR_F16 && head_dim == D && P % 16 == 0 && (long)max_pages * P / 16 * (P / 16) < (1L << 32) &&
         G <= kVec && NG <= kMaxPrefixes && B <= kMaxRows && per_item < (1L << 30) && items < (1L << 30) && per_item * items < (1L << 30);
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
  // DMA takes 16-byte groups of the pools.
  if (!shares(batch, groups, num_heads, num_kv_heads, head_dim, page_size, max_pages, kv_dtype) ||
      ((uintptr_t)k_pool | (uintptr_t)v_pool) % 16)
    return cir_paged_decode_attention(q, k_pool, v_pool, page_table, seq_lens, out, workspace, workspace_bytes, batch,
                                      num_heads, num_kv_heads, head_dim, page_size, max_pages, scale, kv_dtype, stream);
  const Layout l = layout(batch, groups, num_heads, num_kv_heads);
  CIR_CHECK_ARG(workspace && workspace_bytes >= l.total && (uintptr_t)workspace % 16 == 0,
                "attention_shared: workspace too small or not on 16 bytes (%zu < %zu)", workspace_bytes, l.total);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const float scale_log2 = scale * kLog2e;
  const uint32_t P16 = page_size / 16;
  const Args A{reinterpret_cast<Plan*>(ws),
               reinterpret_cast<GroupRec*>(ws + l.groups), reinterpret_cast<RowRec*>(ws + l.rows),
               reinterpret_cast<float*>(ws + l.pre_o), reinterpret_cast<float*>(ws + l.pre_ml),
               reinterpret_cast<float*>(ws + l.suf_o), reinterpret_cast<float*>(ws + l.suf_ml), batch, groups, num_heads,
               num_kv_heads, (int)P16, max_pages, (uint32_t)(((1ull << 32) + P16 - 1) / P16),
               scale_log2 == 0.f ? FLT_MIN : scale_log2};  // (a masked score is -inf: -inf * 0 would be NaN)
  hipStream_t s = as_stream(stream);
  attn_shared_f16_d128<<<kGroups, kThreads, 0, s>>>(
      static_cast<const f16*>(q), static_cast<const f16*>(k_pool), static_cast<const f16*>(v_pool), page_table, seq_lens,
      group_rows, prefix_lens, A);
  const int st = launch_status();
  if (st) return st;
  const unsigned vectors = (unsigned)batch * num_heads;
  attn_shared_join<<<(vectors + 7) / 8, 256, 0, s>>>(A, static_cast<f16*>(out));
  return launch_status();
}
