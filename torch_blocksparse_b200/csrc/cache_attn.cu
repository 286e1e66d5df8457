// Attention of the newest tokens of every sequence over the 4-bit cache, along the rows of a sparse layout:
//
//   o = softmax(scale q K^T) V  over the keys j <= position in the nonzero blocks of the position's block-row,
//
// with K = s c and V = s c from codes c and a scale s for 32 channels (cache.cuh).  One launch, no workspace.
//
// Bound by memory (4.5 bits a value, each read once) if the codes reach the tensor cores in few enough
// instructions, which is what the format is for.  A warp takes 16 tokens (a granule) at a time:
//   S^T = K q^T   m16n8k16: 16 tokens x 16 channels by 16 channels x 8 queries.  The operand is a code word
//                 under a mask: c + 8 as a half, times 2^-21 (2^-17 in the odd quarters, for which
//                 q is divided by 16), exact.  The + 8 leaves through the accumulator's start, -8 * sum(q).
//                 One multiply-add per group of 32 channels, token and query brings the scale in.
//   O^T = V^T P   16 channels x 16 tokens by 16 tokens x 8 queries, P = p * s for each group, so that the codes
//                 are used as they are here too; the + 8 leaves through one product with a matrix of eights for each
//                 group.  P comes out of S^T's accumulators by two transposes of 8 x 8 (movmatrix).
// Eight queries (query heads that share a head of the cache, times new tokens) ride along for one.  Where there are at most four,
// or two of 128 channels, a column is a (query, group) of GC groups: q is zero outside its group, S^T comes out by groups, P of GC
// groups is one operand with one transpose and one product of eights, and a lane deals with one query.  tcgen05 has no
// place here: its operands come from shared or tensor memory, and storing unpacked codes there would
// cost more than the products, which use a fraction of mma.sync's rate at this width.
//
// Numbers.  q is scaled by a power of two to the top of fp16's range and so keeps every bit of either type down to
// 2^-24 of the row's largest.  Scores, sums, maxima and accumulators are floats.  P is rounded to half:
// 2^-11 relative, an eighth of bf16's half step; for fp16 results a second product adds what the rounding
// cut off (SPLIT).  A power of two for each query and group keeps P in half's range.  It follows the largest p * s, not
// the largest s (a large value that a query gives no weight would push the others' P into half's subnormal range), so what is lost
// there is at most 2^-32 of the largest product of a weight and a scale for each key.  A warp usually finds with one vote that
// it need not look closer: no score is 2^4 above the maximum, and no scale so large that its P could pass 2^15.  Where one is, or some
// queries do not see all tokens, every P is checked and the powers are lowered where one is above 2^8 (exact, since everything is
// relative to them); a new maximum, which makes all weights smaller, raises them.
//
// Work: a CTA's warps, times the CTAs of a cluster, take the granules of one (sequence, head, eight
// queries) in turn, each through a ring of its own (cp.async, no barriers), and join their sums
// once, in shared memory, then by sending them over the cluster, in a fixed order: results do not depend on timing.
//
// What bounds it now.  592 heads x 8192 keys, all of a layout, bf16: 128 channels, one query each 111 us, 96 % of the copy rate, four
// 122 us, 87 %, eight 146 us, 73 %; 64 channels, up to four queries 71 us, 75 %, eight 84, 64 % (fp16: 126, 144 and 182 us, 85, 74 and 59 %; 81 and
// 99 us, 66 and 54 %).  Short of the memory's rate it is instructions: masks, permutations, packing and maxima hold an SM's issue
// ports two cycles each (for 16 tokens of 128 channels and eight queries 64 + 16 + 8 + 8 of them), a product of 16 x 8 x 16 the tensor pipe
// 8.3 and the port two, everything else one: 510 cycles of an SM's quarter where loading takes 375.  More warps an SM (96 or 80 registers)
// change nothing.  Short rows are bound by the chain of loads (length, row, block, page, data), the launch and the join: 4.8 us for 5
// granules a warp.  More than eight queries take the granules again for every eight (16 x 8 heads of 32768 keys, bf16, 128 channels: 8, 16, 32 and
// 128 queries 150, 283, 542 and 1818 us).
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <algorithm>

#include "cache.cuh"
#include "common.h"
#include "launch.cuh"
#include "tile.cuh"

namespace bsp {
namespace {

namespace cg = cooperative_groups;

constexpr int kWarps = 4;
constexpr int kStages = 2;
constexpr int kCtas = 4;            // on an SM
constexpr int kSms = 148;
constexpr int kQueries = 8;
constexpr int kMaxCluster = 8;
constexpr float kNothing = -3e38f; // the maximum of no scores
constexpr float kSlack = 4.f;      // p <= 2^4
constexpr uint32_t kEights = 0x04000400u;        // halves 2^-14: 8 as a code in a high field
constexpr uint32_t kSixteenth = 0x3d803d80u;     // a pair of bf16
constexpr int kHighest = 234, kLowest = 12;   // biased exponents of the powers of two on P: 2^107, 2^-115
constexpr int kNone = 0x7ffffff0;  // the token of a granule that is not there: nobody sees it

struct AttnParams {
  const void* q;
  void* o;
  int64_t q_sz, q_sh, q_st, o_sz, o_sh, o_st;
  const uint8_t* data;
  CachePages pages;
  const int32_t* lengths;
  const int32_t *row_ptr, *blk_col;
  int layout_heads, layout_rows, rows, block_shift;   // rows: those that count; block_shift: log2(granules of a block)
  int T, G, tiles, cluster;                     // G: query heads of a cache head; tiles of 8 queries
  float scale_log2e;
};

__device__ __forceinline__ void mma_half(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same on top of c0, c1 in both halves of the rows.
__device__ __forceinline__ void mma_half_from(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1,
                                              float c0, float c1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%10,%11};\n"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(to), "l"(from));
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float exact_exp2(int e) { return __int_as_float((e + 127) << 23); }   // -126 <= e <= 127
__device__ __forceinline__ int exponent_of(float x, int most) { return max(-100, min(most, static_cast<int>(__float_as_uint(x) >> 23) - 127)); }
// One of a pair of bf16 as a float, and times another (exact: 16 significant bits).  Both on the FMA pipe in one instruction:
// a shift or mask takes the integer pipe two cycles, and that pipe is what the kernel runs out of.
__device__ __forceinline__ float bf16_at(uint32_t pair, int i) {
  float x;
  if (i) asm("{.reg .b16 l, h; mov.b32 {l, h}, %1; add.rn.f32.bf16 %0, h, 0f00000000;}" : "=f"(x) : "r"(pair));
  else asm("{.reg .b16 l, h; mov.b32 {l, h}, %1; add.rn.f32.bf16 %0, l, 0f00000000;}" : "=f"(x) : "r"(pair));
  return x;
}
__device__ __forceinline__ float bf16_product(uint32_t pair, int i, uint32_t other, int j) {
  float x;
  if (i && j) asm("{.reg .b16 l, h, m, n; mov.b32 {l, h}, %1; mov.b32 {m, n}, %2; fma.rn.f32.bf16 %0, h, n, 0f00000000;}" : "=f"(x) : "r"(pair), "r"(other));
  else if (i) asm("{.reg .b16 l, h, m, n; mov.b32 {l, h}, %1; mov.b32 {m, n}, %2; fma.rn.f32.bf16 %0, h, m, 0f00000000;}" : "=f"(x) : "r"(pair), "r"(other));
  else if (j) asm("{.reg .b16 l, h, m, n; mov.b32 {l, h}, %1; mov.b32 {m, n}, %2; fma.rn.f32.bf16 %0, l, n, 0f00000000;}" : "=f"(x) : "r"(pair), "r"(other));
  else asm("{.reg .b16 l, h, m, n; mov.b32 {l, h}, %1; mov.b32 {m, n}, %2; fma.rn.f32.bf16 %0, l, m, 0f00000000;}" : "=f"(x) : "r"(pair), "r"(other));
  return x;
}
// The biased exponents of a pair of powers of two in bf16.
__device__ __forceinline__ int exponent_at(uint32_t pair, int i) { return pair >> (16 * i + 7) & 255; }
__device__ __forceinline__ void set_exponent(uint32_t& pair, int i, int e) {
  pair = (pair & (i ? 0x0000ffffu : 0xffff0000u)) | static_cast<uint32_t>(e) << (16 * i + 7);
}
__device__ __forceinline__ __nv_bfloat162 as_bf162(uint32_t x) { return *reinterpret_cast<const __nv_bfloat162*>(&x); }

template <typename T, int D, bool SPLIT, int GC, int NP>
__global__ void __launch_bounds__(kWarps * 32, kCtas) cache_attn_kernel(const __grid_constant__ AttnParams p) {
  constexpr int REC = record_bytes(D), HALF = REC / 2, STAGE = NP * REC, NC = D / 64, NG = D / kGroup, NK = D / 16;
  // Columns of the products: 8 / GC queries by GC groups of channels.  q is zero in a column outside its group, so that a
  // column's sums over GC groups of channels (a set) belong to one of them.  A lane has columns 2 t4 and 2 t4 + 1: two queries and
  // all groups (GC = 1), or QL = 1 query and two groups of each set, whose scales are SW words for each of its tokens.
  constexpr int SETS = NG / GC, QL = GC == 1 ? 2 : 1, SW = GC == 4 ? 1 : NG / 2;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ uint4 q_operand[NG][32];              // of both quarters of a group, by lane
  __shared__ float2 q_start[NG][4];                // by pair of queries
  __shared__ int2 listed[kWarps][32];              // granules looked up: record, first token + row (0, 1)
  __shared__ float part_m[kWarps][kQueries], part_l[kWarps][kQueries];
  __shared__ float inbox[kQueries * D + kMaxCluster], inbox_m[kMaxCluster][kQueries], inbox_l[kMaxCluster][kQueries];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t4 = lane % 4;
  uint8_t* ring = smem + warp * (kStages * STAGE);
  const int my_query = 2 * t4 / GC, my_word = GC == 4 ? t4 % 2 : 0;
  const int q_column = g / GC;                     // the query of column g

  wait_for_earlier_kernels();
  if (p.cluster > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;\n");   // (this CTA runs: others may write here)

  // ---- which queries
  const int rank = blockIdx.x % p.cluster;
  int w = blockIdx.x / p.cluster;
  const int tile = w % p.tiles;
  w /= p.tiles;
  const int hk = w % p.pages.heads, z = w / p.pages.heads;
  const int32_t* row_ptr = p.row_ptr + static_cast<int64_t>(p.layout_heads > 1 ? hk : 0) * p.layout_rows;
  const int len = max(p.lengths[z], 0);
  const int r0 = tile * kQueries, nq = min(kQueries, p.T * p.G - r0);
  // (two channels a load: see the entry point)
  uint32_t qraw[NK][2];
  {
    const int r = r0 + min(q_column, nq - 1), t = p.T == 1 ? 0 : r / p.G;
    const T* q = static_cast<const T*>(p.q) + z * p.q_sz + (hk * p.G + r - t * p.G) * p.q_sh + t * p.q_st + t4 * 2;
#pragma unroll
    for (int n = 0; n < NK; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) qraw[n][i] = *reinterpret_cast<const uint32_t*>(q + n * 16 + i * 8);
  }

  // ---- which rows of the layout: the first query's and, if that is another, the last one's (8 queries span
  // at most 8 positions, a block at least 16); of each its entries in blk_col, the granules of all its blocks, and the
  // last token that any query sees.  limit: that token for this lane's queries (-1: none); all_see: what
  // every query sees (-1: nothing is sure).
  const int block_log2 = p.block_shift + 4;
  int begin[2] = {0, 0}, granules[2] = {0, 0}, last[2] = {-1, -1}, limit[2][QL], all_see;
  {
    const int first_pos = len - p.T + (p.T == 1 ? 0 : r0 / p.G), last_pos = len - p.T + (p.T == 1 ? 0 : (r0 + nq - 1) / p.G);
    const int row[2] = {max(first_pos, 0) >> block_log2, last_pos >> block_log2};
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int i = 0; i < QL; ++i) limit[s][i] = s ? -1 : last_pos;
      if (last_pos < 0 || row[s] >= p.rows || (s && row[1] == row[0])) continue;
      begin[s] = row_ptr[row[s]];
      granules[s] = (row_ptr[row[s] + 1] - begin[s]) << p.block_shift;
      last[s] = static_cast<int>(min(static_cast<int64_t>(last_pos), (static_cast<int64_t>(row[s] + 1) << block_log2) - 1));
    }
    all_see = first_pos >= 0 && row[0] == row[1] ? first_pos : -1;
    if (p.T > 1) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
#pragma unroll
        for (int i = 0; i < QL; ++i) {
          const int r = my_query + i, pos = r < nq ? len - p.T + (r0 + r) / p.G : -1;
          limit[s][i] = pos >= 0 && pos >> block_log2 == row[s] ? pos : -1;
        }
      }
    }
  }

  // ---- the warp's granules: number wid + n * nw of both rows, one after the other
  const int nw = kWarps * p.cluster, wid = rank * kWarps + warp, total = granules[0] + granules[1];
  const int mine = total > wid ? (total - wid + nw - 1) / nw : 0;
  int n0 = 0, at = 0, found = 0;   // looked up so far; of the last 32 those loaded, and those to be loaded
  const uint8_t* data = p.data + lane * 16;
  const uint32_t ring_at = smem_u32(ring) + lane * 16;
  // Loads the next NP granules that have a page and a visible token into a stage; their tokens + rows, kNone: no more.
  auto fetch = [&](int stage_offset, int (&tokens)[NP]) {
#pragma unroll
    for (int u = 0; u < NP; ++u) {
      tokens[u] = kNone;
      while (at == found && n0 < mine) {
        const int n = n0 + lane;
        int record = -1, first = 0;
        if (n < mine) {
          int i = wid + n * nw;
          const int s = i >= granules[0];
          if (s) i -= granules[0];
          const int gran = (p.blk_col[(s ? begin[1] : begin[0]) + (i >> p.block_shift)] << p.block_shift) + (i & ((1 << p.block_shift) - 1));
          first = gran * kGranule + s;
          if (gran * kGranule <= (s ? last[1] : last[0])) record = static_cast<int>(p.pages.granule(z, hk, gran));
        }
        __syncwarp();                              // (the last 32 have been read)
        const uint32_t has = __ballot_sync(~0u, record >= 0);
        if (record >= 0) listed[warp][__popc(has & ((1u << lane) - 1))] = make_int2(record, first);
        __syncwarp();
        at = 0;
        found = __popc(has);
        n0 += 32;
      }
      if (at < found) {
        const int2 next = listed[warp][at++];
        tokens[u] = next.y;
        const uint8_t* from = data + static_cast<uint64_t>(static_cast<uint32_t>(next.x)) * REC;
        const uint32_t to = ring_at + stage_offset + u * REC;
#pragma unroll
        for (int i = 0; i < REC / 512; ++i) copy16(to + i * 512, from + i * 512);
        if (lane < REC / 16 % 32) copy16(to + REC / 512 * 512, from + REC / 512 * 512);
      }
    }
    cp_async_commit();
  };
  int tokens[NP], ahead[NP];
  fetch(0, tokens);
  fetch(STAGE, ahead);

  // ---- q as operands: halves scaled by a power of two, and what the codes' offset adds up to; one group of 32
  // channels a warp, kept in shared memory (registers are what limits the warps of an SM)
  float unscale[QL];
  {
    auto pair_at = [&](int n, int i) {
      if constexpr (std::is_same_v<T, __half>) return __half22float2(*reinterpret_cast<const __half2*>(&qraw[n][i]));
      else return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&qraw[n][i]));
    };
    float amax = 0.f;
#pragma unroll
    for (int n = 0; n < NK; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) amax = fmaxf(amax, fmaxf(fabsf(pair_at(n, i).x), fabsf(pair_at(n, i).y)));
    amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 2));
    // |q| < 2^(e + 1); q * 2^(13 - e) < 2^14, and a sixteenth of it in the odd quarters.  (Where scale * 2^e is above 2^119 the
    // factor that takes this back, 2^8 times that, is infinite, and so the query's scores are no numbers.)
    const int e = exponent_of(amax, 127);
    const float sign = p.scale_log2e > 0.f ? 1.f : p.scale_log2e < 0.f ? -1.f : p.scale_log2e;   // (scores come out scaled by > 0)
    const float down = fmaxf(fabsf(p.scale_log2e) * 256.f * exact_exp2(e), 0x1p-100f);           // 2^21 * 2^(e - 13)
#pragma unroll
    for (int i = 0; i < QL; ++i) unscale[i] = __shfl_sync(~0u, down, (GC == 1 ? my_query + i : my_query * GC) * 4);
    const float up = exact_exp2(13 - e) * sign;
#pragma unroll
    for (int k = 0; k < NG; ++k) {
      if (k % kWarps != warp) continue;
      uint32_t h[4];
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 x = pair_at(2 * k + j / 2, j % 2);
        const float f = j / 2 ? up * 0.0625f : up;
        h[j] = pack_half(x.x * f, x.y * f);
        const float2 r = __half22float2(*reinterpret_cast<const __half2*>(&h[j]));
        sum += (r.x + r.y) * (j / 2 ? 16.f : 1.f);
      }
      sum += __shfl_xor_sync(~0u, sum, 1);
      sum += __shfl_xor_sync(~0u, sum, 2);
      const bool mine = g % GC == k % GC;          // (a column of another group: zeros)
      q_operand[k][lane] = mine ? make_uint4(h[0], h[1], h[2], h[3]) : make_uint4(0, 0, 0, 0);
      if (t4 == 0 && mine) reinterpret_cast<float*>(q_start[k / GC])[g] = sum * -0x1p-18f;
    }
  }
  __syncthreads();

  // O^T: 16 channels each by the columns (those of their own group count); sums of P times 2^-14
  float acc[NK][4] = {}, eights[SETS][4] = {};
  // largest score before `unscale`; that it is time for a new one; minus the largest, scaled; sums of weights
  float m[QL], limit_m[QL], neg_m[QL], l[QL];
#pragma unroll
  for (int i = 0; i < QL; ++i) {
    m[i] = limit_m[i] = -INFINITY;
    neg_m[i] = l[i] = 0.f;
  }
  // Powers of two on P, pairs of bf16: of a set's two groups, or (GC = 1) of a group's two queries.  Scales of V above which
  // P could pass 2^15 while p <= 2^4, by group; none for a query that has seen nothing, whose P are zeros.
  uint32_t boost[SETS];
  __nv_bfloat162 ceiling[SW];
#pragma unroll
  for (int k = 0; k < SETS; ++k) boost[k] = 0x3f803f80u;
#pragma unroll
  for (int k = 0; k < SW; ++k) ceiling[k] = as_bf162(0x7f807f80u);
  auto renew_ceilings = [&] {
    auto most = [&](int k, int j) { return m[GC == 1 ? j : 0] == -INFINITY ? 0x7f80u : static_cast<uint32_t>(265 - exponent_at(boost[k], j)) << 7; };
#pragma unroll
    for (int k = 0; k < SW; ++k) {
      if constexpr (GC == 1) ceiling[k] = as_bf162(min(most(2 * k, 0), most(2 * k, 1)) | min(most(2 * k + 1, 0), most(2 * k + 1, 1)) << 16);
      else ceiling[k] = as_bf162(most(k, 0) | most(k, 1) << 16);
    }
  };
  // Sums of the k-th set by columns, times f
  auto scale_sums = [&](int k, float f0, float f1) {
#pragma unroll
    for (int n = 2 * GC * k; n < 2 * GC * (k + 1); ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[n][i] *= i % 2 ? f1 : f0;
#pragma unroll
    for (int i = 0; i < 4; ++i) eights[k][i] *= i % 2 ? f1 : f0;
  };

  // NP granules at a time: what is done once for them (waiting, voting, branching) is a good part of the work,
  // and they hide each other's latencies
  for (int stage = 0;; stage ^= STAGE) {
    cp_async_wait<kStages - 1>();
    __syncwarp();
    if (tokens[0] == kNone) break;
    const uint8_t* rec = ring + stage;

    // scores of tokens g (the first QL) and g + 8 for the lane's queries, before `unscale`
    uint32_t ks[NP][2][SW], vs[NP][2][SW];
    float x[NP][2 * QL];
#pragma unroll
    for (int u = 0; u < NP; ++u)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int k = 0; k < SW; ++k) {
          ks[u][i][k] = reinterpret_cast<const uint32_t*>(rec + u * REC + 8 * D)[(g + 8 * i) * (NG / 2) + my_word + k];
          vs[u][i][k] = reinterpret_cast<const uint32_t*>(rec + u * REC + HALF + 8 * D)[(g + 8 * i) * (NG / 2) + my_word + k];
        }
    float a[NP][4], a_odd[NP][4];                  // a set's sums; GC = 4: of the odd quarters
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      uint4 w[NP];
#pragma unroll
      for (int u = 0; u < NP; ++u) w[u] = reinterpret_cast<const uint4*>(rec + u * REC + c * 512)[lane];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int k = 2 * c + half;
        const uint4 qf = q_operand[k][lane];
        const float2 start = q_start[k / GC][t4];
#pragma unroll
        for (int u = 0; u < NP; ++u) {
          const uint4 lo = make_uint4(w[u].x & kLowField, w[u].y & kLowField, w[u].z & kLowField, w[u].w & kLowField);
          const uint4 hi = make_uint4(w[u].x & kHighField, w[u].y & kHighField, w[u].z & kHighField, w[u].w & kHighField);
          if (k % GC) mma_half(a[u], lo.x, lo.y, lo.z, lo.w, qf.x, qf.y);
          else mma_half_from(a[u], lo.x, lo.y, lo.z, lo.w, qf.x, qf.y, start.x, start.y);
          if (GC < 4) mma_half(a[u], hi.x, hi.y, hi.z, hi.w, qf.z, qf.w);
          else if (k) mma_half(a_odd[u], hi.x, hi.y, hi.z, hi.w, qf.z, qf.w);
          else mma_half_from(a_odd[u], hi.x, hi.y, hi.z, hi.w, qf.z, qf.w, 0.f, 0.f);
          if constexpr (GC == 1) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float s = bf16_at(ks[u][i / 2][k / 2], k % 2);
              x[u][i] = k ? fmaf(a[u][i], s, x[u][i]) : a[u][i] * s;
            }
          } else if (k % GC == GC - 1) {
            const int word = GC == 4 ? 0 : c;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float s0 = bf16_at(ks[u][i][word], 0), s1 = bf16_at(ks[u][i][word], 1);
              const float a0 = GC == 4 ? a[u][2 * i] + a_odd[u][2 * i] : a[u][2 * i];
              const float a1 = GC == 4 ? a[u][2 * i + 1] + a_odd[u][2 * i + 1] : a[u][2 * i + 1];
              x[u][i] = fmaf(a1, s1, word ? fmaf(a0, s0, x[u][i]) : a0 * s0);
              if constexpr (GC == 4) x[u][i] += __shfl_xor_sync(~0u, x[u][i], 1);   // (the query's other two groups)
            }
          }
          if (half == 0) w[u] = make_uint4(swap_bytes(w[u].x), swap_bytes(w[u].y), swap_bytes(w[u].z), swap_bytes(w[u].w));
        }
      }
    }
    // take out what some queries do not see
    uint32_t keep[NP][2];                          // halves of P that their query sees
    const bool masked = tokens[NP - 1] + 15 > all_see;   // (a row's tokens ascend; where there are two rows, all_see is -1)
    if (masked) {
#pragma unroll
      for (int u = 0; u < NP; ++u) {
        const int token = (tokens[u] & ~15) + g;
        const bool s = tokens[u] & 15;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          bool any = false;
          keep[u][i] = 0;
#pragma unroll
          for (int j = 0; j < QL; ++j) {
            const bool sees = token + 8 * i <= (s ? limit[1][j] : limit[0][j]);
            any = any || sees;
            keep[u][i] |= sees ? (GC > 1 ? ~0u : j ? 0xffff0000u : 0x0000ffffu) : 0u;
            if (!sees) x[u][QL * i + j] = -INFINITY;
          }
          if (!any)
#pragma unroll
            for (int k = 0; k < SW; ++k) vs[u][i][k] = 0;
        }
      }
    }

    // new maxima where they are exceeded; whether every P is to be checked
    float top[QL];
    __nv_bfloat162 scale_top[SW];
#pragma unroll
    for (int u = 0; u < NP; ++u) {
#pragma unroll
      for (int i = 0; i < QL; ++i) top[i] = u ? fmaxf(top[i], fmaxf(x[u][i], x[u][i + QL])) : fmaxf(x[u][i], x[u][i + QL]);
#pragma unroll
      for (int k = 0; k < SW; ++k) {
        const __nv_bfloat162 s = __hmax2(as_bf162(vs[u][0][k]), as_bf162(vs[u][1][k]));
        scale_top[k] = u ? __hmax2(scale_top[k], s) : s;
      }
    }
    uint32_t over = 0;
#pragma unroll
    for (int k = 0; k < SW; ++k) over |= __hgt2_mask(scale_top[k], ceiling[k]);
    bool due = false;
#pragma unroll
    for (int i = 0; i < QL; ++i) due = due || top[i] > limit_m[i];
    bool careful = masked, fallen = false;
    float fall[QL];                                // of all weights so far, as a power of two
#pragma unroll
    for (int i = 0; i < QL; ++i) fall[i] = 0.f;
    if (__any_sync(~0u, due || over)) {
      careful = true;
      fallen = __any_sync(~0u, due);
      if (fallen) {
#pragma unroll
        for (int i = 0; i < QL; ++i) {
          float t = top[i];
#pragma unroll
          for (int d = 4; d < 32; d *= 2) t = fmaxf(t, __shfl_xor_sync(~0u, t, d));
          if (t > m[i]) {
            fall[i] = (t - m[i]) * unscale[i];
            m[i] = t;
            neg_m[i] = -t * unscale[i];
            limit_m[i] = t + kSlack / unscale[i];
            l[i] *= fast_exp2(-fall[i]);
          }
        }
      }
      if (!masked)
#pragma unroll
        for (int u = 0; u < NP; ++u) keep[u][0] = keep[u][1] = ~0u;
    }

#pragma unroll
    for (int u = 0; u < NP; ++u)
#pragma unroll
      for (int i = 0; i < 2 * QL; ++i) {
        x[u][i] = fast_exp2(fmaf(x[u][i], unscale[i % QL], neg_m[i % QL]));
        l[i % QL] += x[u][i];
      }
    auto add_values = [&](auto check) {
#pragma unroll
      for (int u = 0; u < NP; ++u) {
        // P as operands, of the k-th set, and with SPLIT what its rounding cut off
        uint32_t b[SPLIT ? 2 : 1][2];
        auto weights = [&](int k) {
          float w[2][2];                           // by token half and column
          if constexpr (check) {
            // (x * s first: s * boost may leave a float's range where x is small; a sixteenth, for x is up to 2^4)
            auto part = [&](int v, int i, int j) {
              return GC > 1 ? x[v][i] * bf16_product(vs[v][i][k], j, kSixteenth, 0) : x[v][2 * i + j] * bf16_product(vs[v][i][k / 2], k % 2, kSixteenth, 0);
            };
            auto multiply = [&] {
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                const float by = bf16_at(boost[k], j) * 16.f;
#pragma unroll
                for (int i = 0; i < 2; ++i) w[i][j] = part(u, i, j) * by;
              }
            };
            multiply();
            if ((u == 0 && fallen) || __any_sync(~0u, fmaxf(fmaxf(w[0][0], w[1][0]), fmaxf(w[0][1], w[1][1])) > 256.f)) {
              float f[2];
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                float t = 0.f;
#pragma unroll
                for (int v = 0; v < NP; ++v) t = fmaxf(t, fmaxf(part(v, 0, j), part(v, 1, j)));
#pragma unroll
                for (int d = 4; d < 32; d *= 2) t = fmaxf(t, __shfl_xor_sync(~0u, t, d));
                // as high as the fall of the weights allows, and the largest P of the step at 2^7 .. 2^8 at most
                const float by = u ? 0.f : fall[GC == 1 ? j : 0];
                const int old = exponent_at(boost[k], j), most = by < 126.f ? min(old + static_cast<int>(ceilf(by)), kHighest) : kHighest;
                const int e = max(kLowest, min(most, 134 - (static_cast<int>(__float_as_uint(t) >> 23) - 127 + 4)));
                set_exponent(boost[k], j, e);
                f[j] = by < 126.f && old - e < 127 ? exact_exp2(e - old) * fast_exp2(-by) : 0.f;
              }
              scale_sums(k, f[0], f[1]);
              multiply();
            }
          } else {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int j = 0; j < 2; ++j)
                w[i][j] = GC > 1 ? x[u][i] * bf16_product(vs[u][i][k], j, boost[k], j) : x[u][2 * i + j] * bf16_product(vs[u][i][k / 2], k % 2, boost[k], j);
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t h = pack_half(w[i][0], w[i][1]);
            if constexpr (check) h &= keep[u][i];  // (0 times a NaN scale of a token that this query does not see)
            b[0][i] = transpose8(h);
            if constexpr (SPLIT) {
              const float2 r = __half22float2(*reinterpret_cast<const __half2*>(&h));
              uint32_t rest = pack_half(w[i][0] - r.x, w[i][1] - r.y);
              if constexpr (check) rest &= keep[u][i];
              b[1][i] = transpose8(rest);
            }
          }
#pragma unroll
          for (int j = 0; j < (SPLIT ? 2 : 1); ++j) mma_half(eights[k], kEights, kEights, kEights, kEights, b[j][0], b[j][1]);
        };
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          uint4 w = reinterpret_cast<const uint4*>(rec + u * REC + HALF + c * 512)[lane];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int k = 2 * c + half, n = 4 * c + 2 * half;
            if (k % GC == 0) weights(k / GC);
            const uint4 lo = make_uint4(w.x & kLowField, w.y & kLowField, w.z & kLowField, w.w & kLowField);
            const uint4 hi = make_uint4(w.x & kHighField, w.y & kHighField, w.z & kHighField, w.w & kHighField);
#pragma unroll
            for (int j = 0; j < (SPLIT ? 2 : 1); ++j) {
              mma_half(acc[n], lo.x, lo.y, lo.z, lo.w, b[j][0], b[j][1]);
              mma_half(acc[n + 1], hi.x, hi.y, hi.z, hi.w, b[j][0], b[j][1]);
            }
            if (half == 0) w = make_uint4(swap_bytes(w.x), swap_bytes(w.y), swap_bytes(w.z), swap_bytes(w.w));
          }
        }
      }
    };
    if (careful) {
      add_values(std::true_type());
      renew_ceilings();
    } else {
      add_values(std::false_type());
    }
    __syncwarp();                                  // (all lanes are done with the stage)
#pragma unroll
    for (int u = 0; u < NP; ++u) tokens[u] = ahead[u];
    fetch(stage, ahead);
  }
  cp_async_wait<0>();
  __syncwarp();

  // ---- join: the warp's averages into its ring, then all warps', then all CTAs' of the cluster, each with its share of the weight
  // (sums of values near the end of bf16's range would leave a float's)
  float* own = reinterpret_cast<float*>(ring);     // [queries][D]
#pragma unroll
  for (int i = 0; i < QL; ++i) {
#pragma unroll
    for (int d = 4; d < 32; d *= 2) l[i] += __shfl_xor_sync(~0u, l[i], d);
    if (g == 0 && my_word == 0) {
      part_m[warp][my_query + i] = l[i] > 0.f || l[i] != l[i] ? -neg_m[i] : kNothing;
      part_l[warp][my_query + i] = l[i];
    }
  }
#pragma unroll
  for (int k = 0; k < NG; ++k) {
    if (GC == 4 && k / 2 != my_word) continue;
#pragma unroll
    for (int i = 0; i < QL; ++i)
      if (my_query + i < nq) {
        const float back = 1.f / bf16_at(boost[k / GC], GC > 1 ? k % 2 : i);
        const int column = GC > 1 ? k % 2 : i;
        const float each = l[i] == 0.f ? 0.f : 0x1p17f / l[i];
#pragma unroll
        for (int j = 0; j < 4; ++j)                // channel g + 8 j of the group
          own[(my_query + i) * D + k * 32 + g + 8 * j] =
              (acc[2 * k + j / 2][column + j % 2 * 2] * (j / 2 ? 1.f : 16.f) - eights[k / GC][column]) * each * back;
      }
  }
  __syncthreads();
  T* o = static_cast<T*>(p.o) + z * p.o_sz;
  auto store = [&](int r, int d, float value) {
    const int q = r0 + r, t = p.T == 1 ? 0 : q / p.G;
    o[(hk * p.G + q - t * p.G) * p.o_sh + t * p.o_st + d] = cvt_out<T>(value);
  };
  // Where there are more CTAs, each sends every one of them the part of its averages that it stores in the end: rank v
  // has v * share .. v * share + share - 1.
  const int share = (nq * D + p.cluster - 1) / p.cluster;
  cg::cluster_group cluster = cg::this_cluster();
  if (p.cluster > 1) asm volatile("barrier.cluster.wait.aligned;\n");
  for (int at = threadIdx.x; at < nq * D; at += kWarps * 32) {
    const int r = at / D;
    float top = kNothing, sum = 0.f, weight = 0.f, share_of[kWarps];
#pragma unroll
    for (int v = 0; v < kWarps; ++v) top = fmaxf(top, part_m[v][r]);
#pragma unroll
    for (int v = 0; v < kWarps; ++v) {
      share_of[v] = part_l[v][r] * fast_exp2(part_m[v][r] - top);
      weight += share_of[v];
    }
    const float each = weight == 0.f ? 0.f : 1.f / weight;
#pragma unroll
    for (int v = 0; v < kWarps; ++v) sum += reinterpret_cast<const float*>(smem + v * (kStages * STAGE))[at] * (share_of[v] * each);
    if (p.cluster == 1) {
      store(r, at % D, sum);
      continue;
    }
    const int to = at / share;
    cluster.map_shared_rank(inbox, to)[rank * share + at - to * share] = sum;
    if (at % D < p.cluster) {
      cluster.map_shared_rank(&inbox_m[rank][r], at % D)[0] = top;
      cluster.map_shared_rank(&inbox_l[rank][r], at % D)[0] = weight;
    }
  }
  if (p.cluster == 1) return;
  cluster.sync();
  for (int i = threadIdx.x; i < share && rank * share + i < nq * D; i += kWarps * 32) {
    const int at = rank * share + i, r = at / D;
    float top = kNothing, sum = 0.f, weight = 0.f, share_of[kMaxCluster];
#pragma unroll
    for (int v = 0; v < kMaxCluster; ++v)
      if (v < p.cluster) top = fmaxf(top, inbox_m[v][r]);
#pragma unroll
    for (int v = 0; v < kMaxCluster; ++v)
      if (v < p.cluster) {
        share_of[v] = inbox_l[v][r] * fast_exp2(inbox_m[v][r] - top);
        weight += share_of[v];
      }
    const float each = weight == 0.f ? 0.f : 1.f / weight;
#pragma unroll
    for (int v = 0; v < kMaxCluster; ++v)
      if (v < p.cluster) sum += inbox[v * share + i] * (share_of[v] * each);
    store(r, at % D, sum);
  }
}

template <typename T, int D, int GC, int NP> int launch(const AttnParams& p, int64_t groups, cudaStream_t stream) {
  constexpr int bytes = kWarps * kStages * NP * record_bytes(D);
  auto kernel = cache_attn_kernel<T, D, std::is_same_v<T, __half>, GC, NP>;
  static_assert(bytes + 9000 <= 48 * 1024, "shared memory that needs no opting in");
  const cudaError_t e = launch_kernel(kernel, static_cast<unsigned>(groups * p.cluster), kWarps * 32, bytes, stream, p, p.cluster);
  if (e == cudaSuccess) return BSP_OK;
  return fail(BSP_ERR_CUDA, "cache attention: %s", cudaGetErrorString(e));
}

template <typename T, int D, int GC> int pick(const AttnParams& p, int64_t groups, bool many, cudaStream_t stream) {
  return many ? launch<T, D, GC, 256 / D>(p, groups, stream) : launch<T, D, GC, 1>(p, groups, stream);
}
// As many groups of channels beside the queries in the products' columns as there are places (592 heads x 8192 keys of 128,
// bf16: one query with 4 groups 111 us, with 2 120, with 1 140; four queries with 2 groups 122, with 1 143).
template <typename T, int D> int pick(const AttnParams& p, int64_t groups, int queries, bool many, cudaStream_t stream) {
  if constexpr (D == 128)
    if (queries <= 2) return pick<T, D, 4>(p, groups, many, stream);
  return queries <= 4 ? pick<T, D, 2>(p, groups, many, stream) : pick<T, D, 1>(p, groups, many, stream);
}

}  // namespace
}  // namespace bsp

extern "C" int bsp_cache_attn_rows(const void* q, void* o, int dtype, int Z, int Hq, int Hk, int T, int D, int64_t q_sz, int64_t q_sh,
                                   int64_t q_st, int64_t o_sz, int64_t o_sh, int64_t o_st, const void* data, int num_pages, int page,
                                   const int32_t* pages, int64_t pages_sz, int slots, const int32_t* lengths, int block,
                                   const int32_t* meta_hdr, const int32_t* meta, int rows, float scale, void* stream) {
  using namespace bsp;
  if (dtype != BSP_F16 && dtype != BSP_BF16) return fail(BSP_ERR_INVALID, "cache attention: queries must be FP16 or BF16");
  if (Z < 0 || T < 0 || Hk < 1 || Hq < 0 || num_pages < 0 || slots < 0) return fail(BSP_ERR_INVALID, "cache attention: bad sizes (Z %d, heads %d over %d, T %d)", Z, Hq, Hk, T);
  if (Hq % Hk) return fail(BSP_ERR_INVALID, "cache attention: %d query heads cannot share %d heads of the cache", Hq, Hk);
  if (!valid_cache_dim(D)) return fail(BSP_ERR_UNSUPPORTED, "cache attention: head dimension %d (64 and 128 are supported)", D);
  if (!valid_page(page)) return fail(BSP_ERR_INVALID, "cache attention: pages of %d tokens (a power of two from 16 to 1024)", page);
  if (!valid_block(block)) return fail(BSP_ERR_INVALID, "cache attention: block must be 16, 32, 64 or 128 (got %d)", block);
  if (static_cast<int64_t>(slots) * page > INT32_MAX) return fail(BSP_ERR_UNSUPPORTED, "cache attention: sequences of up to 2^31 tokens");
  if (!meta_hdr || !meta) return fail(BSP_ERR_INVALID, "cache attention: NULL layout");
  if (meta_hdr[0] != BSP_META_MAGIC) return fail(BSP_ERR_INVALID, "cache attention: bad layout header (magic)");
  if (meta_hdr[2] != meta_hdr[3]) return fail(BSP_ERR_INVALID, "cache attention: the layout is not square");
  if (meta_hdr[1] != 1 && meta_hdr[1] != Hk) return fail(BSP_ERR_INVALID, "cache attention: layout of %d heads for a cache of %d", meta_hdr[1], Hk);
  if (rows < 0 || rows > meta_hdr[2]) return fail(BSP_ERR_INVALID, "cache attention: %d rows of a layout of %d", rows, meta_hdr[2]);
  if (static_cast<int64_t>(meta_hdr[2]) * block > INT32_MAX) return fail(BSP_ERR_UNSUPPORTED, "cache attention: sequences of up to 2^31 tokens");
  if (Z == 0 || T == 0 || Hq == 0) return BSP_OK;
  if (!q || !o || !lengths || (slots && !pages) || (num_pages && !data)) return fail(BSP_ERR_INVALID, "cache attention: NULL argument");
  if (reinterpret_cast<uintptr_t>(data) & 15) return fail(BSP_ERR_INVALID, "cache attention: the cache is not 16-byte aligned");
  if ((static_cast<int64_t>(num_pages) * Hk) << log2_of(page / kGranule) > INT32_MAX) return fail(BSP_ERR_UNSUPPORTED, "cache attention: caches of up to 2^31 times 16 tokens");
  uint64_t odd = reinterpret_cast<uintptr_t>(q) >> 1;    // queries are read two channels at a time
  if (Z > 1) odd |= q_sz;
  if (Hq > 1) odd |= q_sh;
  if (T > 1) odd |= q_st;
  if ((odd & 1) || (reinterpret_cast<uintptr_t>(q) & 1)) return fail(BSP_ERR_INVALID, "cache attention: queries need even strides and a base on 4 bytes");
  const Meta mt = meta_view(meta, meta_hdr[1], meta_hdr[2], meta_hdr[3], meta_hdr[4], meta_hdr[5], meta_hdr[6]);
  AttnParams p;
  p.q = q; p.o = o;
  p.q_sz = q_sz; p.q_sh = q_sh; p.q_st = q_st; p.o_sz = o_sz; p.o_sh = o_sh; p.o_st = o_st;
  p.data = static_cast<const uint8_t*>(data);
  p.pages = {pages, pages_sz, slots, num_pages, Hk, log2_of(page / kGranule)};
  p.lengths = lengths;
  p.row_ptr = mt.row_ptr; p.blk_col = mt.blk_col;
  p.layout_heads = mt.H; p.layout_rows = mt.Mb; p.rows = rows; p.block_shift = log2_of(block / kGranule);
  p.T = T; p.G = Hq / Hk;
  if (static_cast<int64_t>(T) * p.G > INT32_MAX / 2) return fail(BSP_ERR_UNSUPPORTED, "cache attention: too many queries");
  p.tiles = (T * p.G + kQueries - 1) / kQueries;
  p.scale_log2e = scale * 1.4426950408889634f;
  const int64_t groups = static_cast<int64_t>(Z) * Hk * p.tiles;
  // CTAs of a cluster: as many as fit the SMs at once (one sequence of 12 heads, rows of up to 19 blocks of 64: 8 CTAs 4.8 us,
  // one 5.8; 8 x 16 heads, 36 blocks: 4 CTAs 9.7 us, one 14.9, 8 CTAs, which do not fit, 14.4), and a granule of an average row
  // for every warp.  Two granules of 128 or four of 64 channels at a time where a warp has many (592 heads x 8192 keys of 128, one and eight
  // queries: 111 and 146 us, one at a time 120 and 160); fewer fill such steps badly (the 8 x 16 heads above, 9 granules a warp: 11.5 us, one at a time 9.7).
  const int64_t granules = (static_cast<int64_t>(mt.nnz) / std::max<int64_t>(1, static_cast<int64_t>(mt.H) * mt.Mb) + 1) << p.block_shift;
  p.cluster = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({kMaxCluster, kCtas * kSms / groups, granules / kWarps})));
  const bool many = granules > 16 * kWarps * p.cluster;
  if (Z > INT32_MAX / Hk / p.tiles / p.cluster) return fail(BSP_ERR_UNSUPPORTED, "cache attention: too many queries");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int queries = T * p.G;
  if (dtype == BSP_F16) return D == 64 ? pick<__half, 64>(p, groups, queries, many, s) : pick<__half, 128>(p, groups, queries, many, s);
  return D == 64 ? pick<__nv_bfloat16, 64>(p, groups, queries, many, s) : pick<__nv_bfloat16, 128>(p, groups, queries, many, s);
}

extern "C" int bsp_cache_attn(const void* q, void* o, int dtype, int Z, int Hq, int Hk, int T, int D, int64_t q_sz, int64_t q_sh,
                              int64_t q_st, int64_t o_sz, int64_t o_sh, int64_t o_st, const void* data, int num_pages, int page,
                              const int32_t* pages, int64_t pages_sz, int slots, const int32_t* lengths, int block,
                              const int32_t* meta_hdr, const int32_t* meta, float scale, void* stream) {
  return bsp_cache_attn_rows(q, o, dtype, Z, Hq, Hk, T, D, q_sz, q_sh, q_st, o_sz, o_sh, o_st, data, num_pages, page, pages, pages_sz, slots,
                             lengths, block, meta_hdr, meta, meta_hdr ? meta_hdr[2] : 0, scale, stream);
}
