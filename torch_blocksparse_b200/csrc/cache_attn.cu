// Attention of the newest tokens of every sequence over the 4-bit cache, along the rows of a sparse layout:
//
//   o = softmax(scale q K^T) V  over the keys j <= position in the nonzero blocks of the position's block-row,
//
// with K = s c and V = s c from codes c and a scale s for 32 channels (cache.cuh).  One launch, no workspace.
//
// Bound by memory (4.5 bits a value, each read once) if the codes reach the tensor cores in few enough
// instructions, which is what the format is for.  A warp takes 16 tokens (a granule) at a time:
//   S^T = K q^T   m16n8k16: 16 tokens x 16 channels by 16 channels x 8 queries.  The operand is a code word
//                 under a mask: c + 8 as a denormal half, 2^-24 each (16 * 2^-24 in the odd quarters, for which
//                 q is divided by 16), exact.  The + 8 leaves through the accumulator's start, -8 * sum(q).
//                 One multiply-add per group of 32 channels, token and query brings the scale in.
//   O^T = V^T P   16 channels x 16 tokens by 16 tokens x 8 queries, P = p * s for each group, so that the codes
//                 are used as they are here too; the + 8 leaves through one product with a matrix of eights for each
//                 group.  P comes out of S^T's accumulators by two transposes of 8 x 8 (movmatrix).
// Eight queries (query heads that share a head of the cache, times new tokens) ride along for one.  tcgen05 has no
// place here: its operands come from shared or tensor memory, and storing unpacked codes there would
// cost more than the products, which use a fraction of mma.sync's rate at this width.
//
// Numbers.  q is scaled by a power of two to the top of fp16's range and so keeps every bit of either type down to
// 2^-24 of the row's largest.  Scores, sums, maxima and accumulators are floats.  P is rounded to half:
// 2^-12 relative, an eighth of bf16's half step; for fp16 results a second product adds what the rounding
// cut off (SPLIT).  The largest scale seen so far of each group fixes a power of two that keeps P in
// half's range; maxima and those powers are renewed only when exceeded by 2^4 and 2^3 (exact, since
// everything is relative to them), so that a granule usually costs one vote.
//
// Work: a CTA's warps, times the CTAs of a cluster, take the granules of one (sequence, head, eight
// queries) in turn, each through a ring of its own (cp.async, no barriers), and join their sums
// once, in shared memory, then over the cluster in a fixed order: results do not depend on timing.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "cache.cuh"
#include "common.h"
#include "tile.cuh"

namespace bsp {
namespace {

namespace cg = cooperative_groups;

constexpr int kWarps = 8;
constexpr int kStages = 4;
constexpr int kQueries = 8;
constexpr float kLowest = -3e38f;  // a maximum that nothing has entered
constexpr float kSlack = 4.f;      // p <= 2^4
constexpr uint32_t kEights = 0x00080008u;

struct AttnParams {
  const void* q;
  void* o;
  int64_t q_sz, q_sh, q_st, o_sz, o_sh, o_st;
  const uint8_t* data;
  CachePages pages;
  const int32_t* lengths;
  const int32_t *row_ptr, *blk_col;
  int layout_heads, layout_rows, block_shift;   // block_shift: log2(granules of a block)
  int T, G, tiles, cluster;                     // G: query heads of a cache head; tiles of 8 queries
  float scale_log2e;
};

__device__ __forceinline__ void mma_half(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float exact_exp2(int e) { return __int_as_float((e + 127) << 23); }   // -126 <= e <= 127
__device__ __forceinline__ float bf16_at(uint32_t pair, int i) { return __uint_as_float(i ? pair & 0xffff0000u : pair << 16); }

// One stretch of a layout's row: granules of its blocks up to the last position that may be seen.
struct Segment {
  int begin, granules, last;       // first entry in blk_col; granules of all its blocks; last visible token
};

template <typename T, int D, bool SPLIT>
__global__ void __launch_bounds__(kWarps * 32, 2) cache_attn_kernel(const __grid_constant__ AttnParams p) {
  constexpr int REC = record_bytes(D), HALF = REC / 2, NC = D / 64, NG = D / kGroup, NK = D / 16;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int stage_token[kWarps][kStages];
  __shared__ float part_m[kWarps][kQueries], part_l[kWarps][kQueries], cta_m[kQueries], cta_l[kQueries];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t4 = lane % 4;
  uint8_t* ring = smem + warp * (kStages * REC);

  // ---- which queries, which rows of the layout
  const int rank = blockIdx.x % p.cluster;
  int w = blockIdx.x / p.cluster;
  const int tile = w % p.tiles;
  w /= p.tiles;
  const int hk = w % p.pages.heads, z = w / p.pages.heads;
  const int64_t len = p.lengths[z];
  const int r0 = tile * kQueries, nq = min(kQueries, p.T * p.G - r0);
  auto position = [&](int r) { return len - p.T + (r0 + r) / p.G; };     // of query r of the tile; negative: there is none
  Segment seg[2];
  const int64_t last_pos = position(nq - 1);
  int64_t first_pos = position(0);
  if (first_pos < 0) first_pos = 0;
  const int block_log2 = p.block_shift + 4;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    // the first query's row, and the last one's if that is another (8 queries span at most 8 positions, a block 16)
    const int64_t row = (s ? last_pos : first_pos) >> block_log2;
    seg[s] = {0, 0, -1};
    if (last_pos < 0 || row >= p.layout_rows || (s && row == first_pos >> block_log2)) continue;
    const int64_t at = static_cast<int64_t>(p.layout_heads > 1 ? hk : 0) * p.layout_rows + row;
    seg[s].begin = p.row_ptr[at];
    seg[s].granules = (p.row_ptr[at + 1] - seg[s].begin) << p.block_shift;
    seg[s].last = static_cast<int>(min(last_pos, ((row + 1) << block_log2) - 1));
  }
  // last visible token of this lane's two queries in each segment (-1: none), and what all queries see
  int limit[2][2], all_see[2] = {INT32_MAX, INT32_MAX};
#pragma unroll
  for (int r = 0; r < kQueries; ++r) {
    const int64_t pos = r < nq ? position(r) : -1;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int64_t row = (s ? last_pos : first_pos) >> block_log2;
      const int lim = pos >= 0 && pos >> block_log2 == row ? static_cast<int>(pos) : -1;
      if (r < nq) all_see[s] = min(all_see[s], lim);
      if (r / 2 == t4) limit[s][r % 2] = lim;
    }
  }

  // ---- q as operands: fp16 scaled by a power of two, and what the codes' offset adds up to
  uint32_t qf[NK][2];
  float start[NG][2], unscale[2];
  {
    const bool there = g < nq;
    const int r = r0 + g;
    const T* q = static_cast<const T*>(p.q) + z * p.q_sz + (hk * p.G + r % p.G) * p.q_sh + (r / p.G) * p.q_st;
    float x[NK][4], amax = 0.f;
#pragma unroll
    for (int n = 0; n < NK; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[n][i] = there ? static_cast<float>(q[n * 16 + t4 * 2 + i % 2 + i / 2 * 8]) : 0.f;
        amax = fmaxf(amax, fabsf(x[n][i]));
      }
    amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 2));
    // |q| < 2^(e + 1); q * 2^(13 - e) < 2^14, and a sixteenth of it in the odd quarters
    const int e = max(-100, min(100, static_cast<int>(__float_as_uint(amax) >> 23) - 127));
    const float up = exact_exp2(13 - e);
    float sum[NG] = {};
#pragma unroll
    for (int n = 0; n < NK; ++n) {
      const float f = n % 2 ? up * 0.0625f : up;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const __half2 h = __floats2half2_rn(x[n][2 * i] * f, x[n][2 * i + 1] * f);
        qf[n][i] = *reinterpret_cast<const uint32_t*>(&h);
        sum[n / 2] += (__half2float(h.x) + __half2float(h.y)) * (n % 2 ? 16.f : 1.f);
      }
    }
    const float down = p.scale_log2e * exact_exp2(e) * 2048.f;           // 2^24 * 2^(e - 13)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      unscale[i] = __shfl_sync(~0u, down, (2 * t4 + i) * 4);
#pragma unroll
      for (int k = 0; k < NG; ++k) {
        float s = sum[k];
        s += __shfl_xor_sync(~0u, s, 1);
        s += __shfl_xor_sync(~0u, s, 2);
        start[k][i] = __shfl_sync(~0u, s, (2 * t4 + i) * 4) * -0x1p-21f;
      }
    }
  }

  // ---- the warp's granules: number wid + n * nw of both segments, one after the other
  const int total = seg[0].granules + seg[1].granules, nw = kWarps * p.cluster, wid = rank * kWarps + warp;
  const int mine = total > wid ? (total - wid + nw - 1) / nw : 0;
  int n0 = 0;
  uint32_t found = 0;              // of the 32 last looked up, those that are not loaded yet
  int64_t my_at = 0;
  int my_token = 0;
  // Loads the next granule that has a page and a visible token into `stage`; token 16 k + segment, -1: no more.
  auto fetch = [&](int stage) {
    while (found == 0 && n0 < mine) {
      const int n = n0 + lane;
      my_at = -1;
      if (n < mine) {
        int i = wid + n * nw;
        const int s = i >= seg[0].granules;
        if (s) i -= seg[0].granules;
        const int begin = s ? seg[1].begin : seg[0].begin, last = s ? seg[1].last : seg[0].last;
        const int gran = (p.blk_col[begin + (i >> p.block_shift)] << p.block_shift) + (i & ((1 << p.block_shift) - 1));
        my_token = gran * kGranule + s;
        if (gran * kGranule <= last) my_at = p.pages.granule(z, hk, gran);
      }
      found = __ballot_sync(~0u, my_at >= 0);
      n0 += 32;
    }
    int token = -1;
    if (found) {
      const int src = __ffs(found) - 1;
      found &= found - 1;
      const int64_t at = __shfl_sync(~0u, my_at, src);
      token = __shfl_sync(~0u, my_token, src);
      const uint8_t* from = p.data + at * REC;
#pragma unroll
      for (int i = 0; i < (REC / 16 + 31) / 32; ++i)
        if (i * 32 + lane < REC / 16) cp_async16(ring + stage * REC + (i * 32 + lane) * 16, from + (i * 32 + lane) * 16, true);
    }
    if (lane == 0) stage_token[warp][stage] = token;
    cp_async_commit();
  };

  float acc[NK][4] = {}, eights[NG][4] = {};       // O^T: 16 channels each by the queries; sums of P times 8 * 2^-24
  float m[2] = {kLowest, kLowest}, l[2] = {0.f, 0.f};
  float boost[NG], ceiling[NG];                    // powers of two on P; scales that make a new one due
#pragma unroll
  for (int k = 0; k < NG; ++k) boost[k] = ceiling[k] = 0.f;

#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) fetch(s);
  for (int it = 0;; ++it) {
    cp_async_wait<kStages - 2>();
    __syncwarp();
    const int mark = stage_token[warp][it % kStages];
    if (mark < 0) break;
    fetch((it + kStages - 1) % kStages);
    const uint8_t* rec = ring + it % kStages * REC;
    const int token = mark & ~15, s = mark & 15;

    // scores of tokens token + g and token + g + 8 for queries 2 t4 and 2 t4 + 1
    uint32_t ks[2][NG / 2], vs[2][NG / 2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int k = 0; k < NG / 2; ++k) {
        ks[i][k] = reinterpret_cast<const uint32_t*>(rec + 8 * D)[(g + 8 * i) * (NG / 2) + k];
        vs[i][k] = reinterpret_cast<const uint32_t*>(rec + HALF + 8 * D)[(g + 8 * i) * (NG / 2) + k];
      }
    float sc[4] = {};
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      uint4 x = reinterpret_cast<const uint4*>(rec + c * 512)[lane];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int k = 2 * c + half, n = 4 * c + 2 * half;
        float a[4] = {start[k][0], start[k][1], start[k][0], start[k][1]};
        mma_half(a, x.x & 0x000f000fu, x.y & 0x000f000fu, x.z & 0x000f000fu, x.w & 0x000f000fu, qf[n][0], qf[n][1]);
        mma_half(a, x.x & 0x00f000f0u, x.y & 0x00f000f0u, x.z & 0x00f000f0u, x.w & 0x00f000f0u, qf[n + 1][0], qf[n + 1][1]);
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[i] = fmaf(a[i], bf16_at(ks[i / 2][k / 2], k % 2), sc[i]);
        x.x >>= 8; x.y >>= 8; x.z >>= 8; x.w >>= 8;
      }
    }
    float sv[2][NG];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int k = 0; k < NG; ++k) sv[i][k] = bf16_at(vs[i][k / 2], k % 2);
#pragma unroll
    for (int i = 0; i < 4; ++i) sc[i] *= unscale[i % 2];
    bool see[4] = {true, true, true, true};
    const bool masked = token + 15 > (s ? all_see[1] : all_see[0]);
    if (masked) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        see[i] = token + g + 8 * (i / 2) <= (s ? limit[1][i % 2] : limit[0][i % 2]);
        if (!see[i]) sc[i] = -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (!see[2 * i] && !see[2 * i + 1])
#pragma unroll
          for (int k = 0; k < NG; ++k) sv[i][k] = 0.f;
    }

    bool due = fmaxf(sc[0], sc[2]) > m[0] + kSlack || fmaxf(sc[1], sc[3]) > m[1] + kSlack;
#pragma unroll
    for (int k = 0; k < NG; ++k) due = due || fmaxf(sv[0][k], sv[1][k]) > ceiling[k];
    if (__any_sync(~0u, due)) {
      float f[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float x = fmaxf(sc[i], sc[i + 2]);
#pragma unroll
        for (int d = 4; d < 32; d *= 2) x = fmaxf(x, __shfl_xor_sync(~0u, x, d));
        x = fmaxf(x, m[i]);
        f[i] = fast_exp2(m[i] - x);
        m[i] = x;
        l[i] *= f[i];
      }
#pragma unroll
      for (int k = 0; k < NG; ++k) {
        float x = fmaxf(sv[0][k], sv[1][k]), ratio = 1.f;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) x = fmaxf(x, __shfl_xor_sync(~0u, x, d));
        if (x > ceiling[k]) {                      // the largest scale becomes 2^7 .. 2^8 in P
          const int e = max(-100, min(100, static_cast<int>(__float_as_uint(x) >> 23) - 127));
          const float b = exact_exp2(7 - e);
          ratio = boost[k] > 0.f ? b / boost[k] : 0.f;
          boost[k] = b;
          ceiling[k] = exact_exp2(e + 4);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          acc[2 * k][i] *= f[i % 2] * ratio;
          acc[2 * k + 1][i] *= f[i % 2] * ratio;
          eights[k][i] *= f[i % 2] * ratio;
        }
      }
    }

    float pr[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      pr[i] = fast_exp2(sc[i] - m[i % 2]);
      l[i % 2] += pr[i];
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      uint4 x = reinterpret_cast<const uint4*>(rec + HALF + c * 512)[lane];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int k = 2 * c + half, n = 4 * c + 2 * half;
        float pw[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          pw[i] = pr[i] * (sv[i / 2][k] * boost[k]);
          if (masked && !see[i]) pw[i] = 0.f;      // (a NaN scale of a token that this query does not see)
        }
        const uint32_t h0 = pack_half(pw[0], pw[1]), h1 = pack_half(pw[2], pw[3]);
        const uint32_t b0 = transpose8(h0), b1 = transpose8(h1);
        const uint4 lo = make_uint4(x.x & 0x000f000fu, x.y & 0x000f000fu, x.z & 0x000f000fu, x.w & 0x000f000fu);
        const uint4 hi = make_uint4(x.x & 0x00f000f0u, x.y & 0x00f000f0u, x.z & 0x00f000f0u, x.w & 0x00f000f0u);
        mma_half(acc[n], lo.x, lo.y, lo.z, lo.w, b0, b1);
        mma_half(acc[n + 1], hi.x, hi.y, hi.z, hi.w, b0, b1);
        mma_half(eights[k], kEights, kEights, kEights, kEights, b0, b1);
        if constexpr (SPLIT) {
          const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&h0)), f1 = __half22float2(*reinterpret_cast<const __half2*>(&h1));
          const uint32_t c0 = transpose8(pack_half(pw[0] - f0.x, pw[1] - f0.y)), c1 = transpose8(pack_half(pw[2] - f1.x, pw[3] - f1.y));
          mma_half(acc[n], lo.x, lo.y, lo.z, lo.w, c0, c1);
          mma_half(acc[n + 1], hi.x, hi.y, hi.z, hi.w, c0, c1);
          mma_half(eights[k], kEights, kEights, kEights, kEights, c0, c1);
        }
        x.x >>= 8; x.y >>= 8; x.z >>= 8; x.w >>= 8;
      }
    }
  }
  cp_async_wait<0>();
  __syncwarp();

  // ---- join: the warp's sums into its ring, then all warps', then all CTAs' of the cluster
  float* mine_o = reinterpret_cast<float*>(ring);  // [8 queries][D]
#pragma unroll
  for (int k = 0; k < NG; ++k) {
    const float back = boost[k] > 0.f ? 1.f / boost[k] : 0.f;
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float v = (acc[2 * k + half][i] * (half ? 0.0625f : 1.f) - eights[k][i]) * 0x1p24f * back;
        mine_o[(2 * t4 + i % 2) * D + (2 * k + half) * 16 + g + i / 2 * 8] = v;
      }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
#pragma unroll
    for (int d = 4; d < 32; d *= 2) l[i] += __shfl_xor_sync(~0u, l[i], d);
    if (g == 0) {
      part_m[warp][2 * t4 + i] = m[i];
      part_l[warp][2 * t4 + i] = l[i];
    }
  }
  __syncthreads();
  const bool alone = p.cluster == 1;
  T* o = static_cast<T*>(p.o) + z * p.o_sz;
  auto store = [&](int r, int d, float v) {
    const int q = r0 + r;
    o[(hk * p.G + q % p.G) * p.o_sh + (q / p.G) * p.o_st + d] = cvt_out<T>(v);
  };
  float* joined = reinterpret_cast<float*>(smem);
  constexpr int PER = kQueries * D / (kWarps * 32);
  float sums[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int at = i * kWarps * 32 + threadIdx.x, r = at / D;
    if (r >= nq) break;
    float top = kLowest, sum = 0.f, weight = 0.f;
#pragma unroll
    for (int v = 0; v < kWarps; ++v) top = fmaxf(top, part_m[v][r]);
#pragma unroll
    for (int v = 0; v < kWarps; ++v) {
      const float f = fast_exp2(part_m[v][r] - top);
      weight += part_l[v][r] * f;
      sum += reinterpret_cast<const float*>(smem + v * (kStages * REC))[at] * f;
    }
    if (alone) {
      store(r, at % D, weight > 0.f || weight != weight ? sum / weight : 0.f);
    } else {
      sums[i] = sum;
      if (at % D == 0) {
        cta_m[r] = top;
        cta_l[r] = weight;
      }
    }
  }
  if (alone) return;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int at = i * kWarps * 32 + threadIdx.x;
    if (at / D >= nq) break;
    joined[at] = sums[i];
  }
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  const int share = (nq * D + p.cluster - 1) / p.cluster;
  for (int at = rank * share + threadIdx.x; at < min((rank + 1) * share, nq * D); at += kWarps * 32) {
    const int r = at / D;
    float top = kLowest, sum = 0.f, weight = 0.f;
    for (int v = 0; v < p.cluster; ++v) top = fmaxf(top, *cluster.map_shared_rank(&cta_m[r], v));
    for (int v = 0; v < p.cluster; ++v) {
      const float f = fast_exp2(*cluster.map_shared_rank(&cta_m[r], v) - top);
      weight += *cluster.map_shared_rank(&cta_l[r], v) * f;
      sum += *cluster.map_shared_rank(&joined[at], v) * f;
    }
    store(r, at % D, weight > 0.f || weight != weight ? sum / weight : 0.f);
  }
  cluster.sync();                  // (nobody's shared memory goes before all have read it)
}

template <typename T, int D> int launch(const AttnParams& p, int64_t groups, cudaStream_t stream) {
  constexpr bool split = sizeof(T) == 2 && std::is_same_v<T, __half>;
  constexpr int bytes = kWarps * kStages * record_bytes(D);
  auto kernel = cache_attn_kernel<T, D, split>;
  static thread_local bool ready[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && !(dev < 64 && ready[dev])) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && dev < 64) ready[dev] = true;
  }
  if (e == cudaSuccess) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(groups * p.cluster));
    cfg.blockDim = dim3(kWarps * 32);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = p.cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, kernel, p);
  }
  if (e == cudaSuccess) return BSP_OK;
  (void)cudaGetLastError();
  return fail(BSP_ERR_CUDA, "cache attention: %s", cudaGetErrorString(e));
}

}  // namespace
}  // namespace bsp

extern "C" int bsp_cache_attn(const void* q, void* o, int dtype, int Z, int Hq, int Hk, int T, int D, int64_t q_sz, int64_t q_sh,
                              int64_t q_st, int64_t o_sz, int64_t o_sh, int64_t o_st, const void* data, int num_pages, int page,
                              const int32_t* pages, int64_t pages_sz, int slots, const int32_t* lengths, int block,
                              const int32_t* meta_hdr, const int32_t* meta, float scale, void* stream) {
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
  if (static_cast<int64_t>(meta_hdr[2]) * block > INT32_MAX) return fail(BSP_ERR_UNSUPPORTED, "cache attention: sequences of up to 2^31 tokens");
  if (Z == 0 || T == 0 || Hq == 0) return BSP_OK;
  if (!q || !o || !lengths || (slots && !pages) || (num_pages && !data)) return fail(BSP_ERR_INVALID, "cache attention: NULL argument");
  if (reinterpret_cast<uintptr_t>(data) & 15) return fail(BSP_ERR_INVALID, "cache attention: the cache is not 16-byte aligned");
  const Meta mt = meta_view(meta, meta_hdr[1], meta_hdr[2], meta_hdr[3], meta_hdr[4], meta_hdr[5], meta_hdr[6]);
  AttnParams p;
  p.q = q; p.o = o;
  p.q_sz = q_sz; p.q_sh = q_sh; p.q_st = q_st; p.o_sz = o_sz; p.o_sh = o_sh; p.o_st = o_st;
  p.data = static_cast<const uint8_t*>(data);
  p.pages = {pages, pages_sz, slots, num_pages, Hk, log2_of(page / kGranule)};
  p.lengths = lengths;
  p.row_ptr = mt.row_ptr; p.blk_col = mt.blk_col;
  p.layout_heads = mt.H; p.layout_rows = mt.Mb; p.block_shift = log2_of(block / kGranule);
  p.T = T; p.G = Hq / Hk;
  if (static_cast<int64_t>(T) * p.G > INT32_MAX / 2) return fail(BSP_ERR_UNSUPPORTED, "cache attention: too many queries");
  p.tiles = (T * p.G + kQueries - 1) / kQueries;
  p.scale_log2e = scale * 1.4426950408889634f;
  const int64_t groups = static_cast<int64_t>(Z) * Hk * p.tiles;
  // CTAs of a cluster: enough to fill two on every SM, no more than give every warp four granules of the longest row
  const int64_t granules = static_cast<int64_t>(mt.max_row) << p.block_shift;
  p.cluster = 1;
  while (p.cluster < 8 && groups * p.cluster < 2 * 148 && granules > 4 * kWarps * p.cluster) p.cluster *= 2;
  if (Z > INT32_MAX / Hk / p.tiles / p.cluster) return fail(BSP_ERR_UNSUPPORTED, "cache attention: too many queries");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == BSP_F16) return D == 64 ? launch<__half, 64>(p, groups, s) : launch<__half, 128>(p, groups, s);
  return D == 64 ? launch<__nv_bfloat16, 64>(p, groups, s) : launch<__nv_bfloat16, 128>(p, groups, s);
}
