// Writing keys and values into the 4-bit cache (quantised on the way) and reading them back.
// The format is described in cache.cuh.
//
// Both kernels give a warp one granule (16 tokens of one head).  Rows are read D / 8 lanes a token, 8 consecutive
// channels (one 16-byte access of a 16-bit type) each, so a warp reads 2 (D = 128) or 4 tokens at a time.  Lane
// `sub` of a token has channels 8 sub .. 8 sub + 7: chunk c = sub / 8 of 64, quarter n = sub / 2 % 4, half h = sub % 2.
//
// Bound by memory: 2 bytes in and 0.5625 out a value, or the other way round.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <type_traits>

#include "cache.cuh"
#include "common.h"
#include "launch.cuh"
#include "tile.cuh"

namespace bsp {
namespace {

constexpr int kWarps = 4;

// Byte of a granule's code area (K or V) at which the word for lane (g, t), register a of chunk c lies.
__device__ __forceinline__ int word_at(int c, int g, int t, int a) { return c * 512 + (g * 4 + t) * 16 + a * 4; }

struct WriteParams {
  const void* x[2];                // keys, values [Z, H, T, D]
  int64_t sz[2], sh[2], st[2];
  uint8_t* data;
  CachePages pages;
  const int32_t *start, *count;    // per sequence; count NULL: T
  int T, ctas;                     // ctas: for each head of each sequence
};

template <typename T> struct Two;
template <> struct Two<__half> { using t = __half2; };
template <> struct Two<__nv_bfloat16> { using t = __nv_bfloat162; };

// 8 consecutive channels.  !VEC: rows that start anywhere.
template <typename T, bool VEC> __device__ __forceinline__ uint4 load8(const T* p) {
  if constexpr (VEC) {
    return *reinterpret_cast<const uint4*>(p);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = reinterpret_cast<const uint16_t*>(p)[2 * i] | static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(p)[2 * i + 1]) << 16;
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}

__device__ __forceinline__ float2 to_f2(__half2 v) { return __half22float2(v); }
__device__ __forceinline__ float2 to_f2(__nv_bfloat162 v) { return __bfloat1622float2(v); }

// The scale of a group whose largest absolute value is `amax`, and how its codes are found.
//
// rint(x / s) without a division, and equal to it: with |x / s| < 8, r within 2^-23 of 1 / s and x of at
// most 11 significant bits, s of 8, a quotient that is no tie is at least 2^-13 away from one, x * r at most
// 2^-20 away from the quotient.  So x * r rounded to a multiple of 2^-16 (an FMA that adds 192, where
// floats are 2^-16 apart) lies on the same side of a tie, or on the tie itself if the quotient
// is one, and taking 192 off and adding 1.5 * 2^23 + 8 in one sum then rounds it to an even integer whose last 16
// bits are c + 8.  max / 7 is the rounded product with 1 / 7 and one step of correction by its exact remainder, which
// gives the rounded quotient (checked over both types' values, with the rest, by the tests).
struct Scale {
  float s, r;                      // r = 0: infinities, NaN, or a scale whose reciprocal a float does not hold; zeros: any other
  uint32_t bits;
  __device__ __forceinline__ explicit Scale(float amax) {
    constexpr float kSeventh = 1.f / 7.f;
    const float q = amax * kSeventh;
    __nv_bfloat16 b = __float2bfloat16_rn(__fmaf_rn(__fmaf_rn(-7.f, q, amax), kSeventh, q));
    r = 0.f;
    if (amax > 1e-29f && amax < INFINITY) asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(__bfloat162float(b)));
    else if (amax == 0.f) r = 1.f;
    else b = amax < INFINITY ? __float2bfloat16_rn(__fdiv_rn(amax, 7.f)) : __ushort_as_bfloat16(0x7fff);
    s = __bfloat162float(b);
    bits = __bfloat16_as_ushort(b);
  }
  // The codes + 8 of two channels in bits 0-3 and 16-19; FAST: r is known not to be 0.
  template <bool FAST, typename T2> __device__ __forceinline__ uint32_t codes(T2 v) const {
    const float2 x = to_f2(v);
    if (FAST || r > 0.f) {
      const float a = __fadd_rn(__fmaf_rn(x.x, r, 192.f), 12582912.f + 8.f - 192.f);
      const float b = __fadd_rn(__fmaf_rn(x.y, r, 192.f), 12582912.f + 8.f - 192.f);
      return __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x5410);
    }
    if (!(s > 0.f)) return 0x00080008u;
    const float a = fminf(fmaxf(rintf(__fdiv_rn(x.x, s)), -8.f), 7.f), b = fminf(fmaxf(rintf(__fdiv_rn(x.y, s)), -8.f), 7.f);
    return static_cast<uint32_t>(static_cast<int>(a) + 8) | static_cast<uint32_t>(static_cast<int>(b) + 8) << 16;
  }
};
template <typename T2> __device__ __forceinline__ T2 as_pair(uint32_t x) { return *reinterpret_cast<const T2*>(&x); }
template <typename T2> __device__ __forceinline__ uint32_t as_word(T2 x) { return *reinterpret_cast<const uint32_t*>(&x); }

// The codes + 8 of 8 channels, two in each word, and the scale of their group, which 4 neighbouring lanes hold together.
template <typename T> __device__ __forceinline__ uint32_t quantise8(uint4 raw, uint32_t (&pair)[4]) {
  using T2 = typename Two<T>::t;
  const T2 v[4] = {as_pair<T2>(raw.x), as_pair<T2>(raw.y), as_pair<T2>(raw.z), as_pair<T2>(raw.w)};
  T2 m = __hmax2_nan(__hmax2_nan(__habs2(v[0]), __habs2(v[1])), __hmax2_nan(__habs2(v[2]), __habs2(v[3])));
  m = __hmax2_nan(m, __shfl_xor_sync(~0u, m, 2));    // (lanes sub ^ 1, sub ^ 2 share the group)
  m = __hmax2_nan(m, __shfl_xor_sync(~0u, m, 1));
  const Scale s(static_cast<float>(__hmax_nan(m.x, m.y)));
  if (__all_sync(~0u, s.r > 0.f)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) pair[i] = s.codes<true>(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) pair[i] = s.codes<false>(v[i]);
  }
  return s.bits;
}

// The four quarters n of a chunk and half hold one 4-bit field each of four words; lane n is left with word n.
__device__ __forceinline__ uint32_t gather_fields(const uint32_t (&pair)[4], int n) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pair[i] << (4 * n);
  const bool hi = n & 2, odd = n & 1;               // quarters differ in lane bits 2 (hi) and 1 (odd)
  const uint32_t k0 = (hi ? w[2] : w[0]) | __shfl_xor_sync(~0u, hi ? w[0] : w[2], 4);
  const uint32_t k1 = (hi ? w[3] : w[1]) | __shfl_xor_sync(~0u, hi ? w[1] : w[3], 4);
  return place_fields((odd ? k1 : k0) | __shfl_xor_sync(~0u, odd ? k0 : k1, 2));
}

// What a lane of a token writes, by the token's place j in the granule: for every K or V one word (of K) or two half words (of V),
// and for one lane of each group the scale.
template <int D> struct Places {
  int sub, c, n, h;
  __device__ __forceinline__ explicit Places(int lane) : sub(lane % (D / 8)), c(sub / 8), n(sub / 2 % 4), h(sub % 2) {}
  __device__ __forceinline__ void put(uint8_t* granule, int kv, int j, uint32_t word, uint32_t scale) const {
    uint8_t* codes = granule + kv * (record_bytes(D) / 2);
    if (kv == 0) {                                  // word n: channels 16 n' + 8 h + 2 n, + 1 of all quarters n'
      *reinterpret_cast<uint32_t*>(codes + word_at(c, j % 8, n, j / 8 + 2 * h)) = word;
    } else {                                        // half words: channels 8 h + 2 n and 8 h + 2 n + 1
      uint8_t* q = codes + word_at(c, 2 * n, j % 8 / 2, h + 2 * (j / 8)) + 2 * (j % 2);
      *reinterpret_cast<uint16_t*>(q) = static_cast<uint16_t>(word);
      *reinterpret_cast<uint16_t*>(q + 64) = static_cast<uint16_t>(word >> 16);
    }
    if (sub % 4 == 0) *reinterpret_cast<uint16_t*>(codes + 8 * D + j * (2 * D / kGroup) + sub / 4 * 2) = static_cast<uint16_t>(scale);
  }
};

template <typename T, int D, bool VEC>
__global__ void __launch_bounds__(kWarps * 32) cache_write_kernel(const __grid_constant__ WriteParams p) {
  constexpr int REC = record_bytes(D);
  __shared__ __align__(16) T rows[kWarps][kGranule * (D + 8)];
  wait_for_earlier_kernels();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  // (a CTA's warps share a head: their number is found with one division of 32 bits for all)
  const uint32_t zh = blockIdx.x / static_cast<uint32_t>(p.ctas), z = zh / static_cast<uint32_t>(p.pages.heads);
  const int head = static_cast<int>(zh - z * p.pages.heads), nth = static_cast<int>(blockIdx.x - zh * p.ctas) * (blockDim.x / 32) + warp;
  const int64_t start = p.start[z];
  const int64_t count = min(p.count ? p.count[z] : p.T, p.T);
  // granules of positions from the one that `start` lies in; tokens t0 .. t0 + 15 of the operands
  const int64_t g = (start >> 4) + nth, t0 = g * kGranule - start;
  if (t0 >= count) return;
  const int64_t at = p.pages.granule(static_cast<int>(z), head, g);   // (negative positions have none)
  if (at < 0) return;
  uint8_t* record = p.data + at * REC;
  constexpr int LPT = D / 8, TPI = 32 / LPT, ITER = kGranule / TPI;
  const Places<D> to(lane);
  const int own = lane / LPT;
  const T* x[2];
#pragma unroll
  for (int kv = 0; kv < 2; ++kv)
    x[kv] = static_cast<const T*>(p.x[kv]) + static_cast<int64_t>(z) * p.sz[kv] + head * p.sh[kv] + (t0 + own) * p.st[kv] + to.sub * 8;
  if (t0 >= 0 && t0 + kGranule <= count) {
    // All 16 tokens.  Rows go through shared memory, and every lane (g, t) takes from there what its words of the
    // format are made of: channels 16 n + 8 h + 2 t, + 1 of tokens g and g + 8.  So a word is put together in one lane, and V's
    // words, two channels of a token in their halves, become two tokens of a channel by one transpose of 8 x 8 (movmatrix).
    // Bound by instructions, 78 % of the copy rate: 8 sequences of up to 8192 tokens, 16 heads of 64, 48 us; with the words gathered
    // over the lanes of a row by shuffles and stored in pieces 57.
    using T2 = typename Two<T>::t;
    constexpr int PITCH = D + 8;                    // rows 4 banks apart
    const int g = lane / 4, t4 = lane % 4;
    T* own_rows = rows[warp];
    uint4 raw[2][ITER];
#pragma unroll
    for (int kv = 0; kv < 2; ++kv)
#pragma unroll
      for (int it = 0; it < ITER; ++it) raw[kv][it] = load8<T, VEC>(x[kv] + it * TPI * p.st[kv]);
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
#pragma unroll
      for (int it = 0; it < ITER; ++it) *reinterpret_cast<uint4*>(own_rows + (it * TPI + own) * PITCH + to.sub * 8) = raw[kv][it];
      __syncwarp();
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          T2 v[4][2], m[2];
#pragma unroll
          for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) v[n][h] = *reinterpret_cast<const T2*>(own_rows + (g + 8 * i) * PITCH + 64 * c + 16 * n + 8 * h + 2 * t4);
#pragma unroll
          for (int k = 0; k < 2; ++k)
            m[k] = __hmax2_nan(__hmax2_nan(__habs2(v[2 * k][0]), __habs2(v[2 * k][1])), __hmax2_nan(__habs2(v[2 * k + 1][0]), __habs2(v[2 * k + 1][1])));
          // both groups' maxima in one pair, over the 4 lanes that share the token
          T2 top = __hmax2_nan(as_pair<T2>(__byte_perm(as_word(m[0]), as_word(m[1]), 0x5410)), as_pair<T2>(__byte_perm(as_word(m[0]), as_word(m[1]), 0x7632)));
          top = __hmax2_nan(top, __shfl_xor_sync(~0u, top, 1));
          top = __hmax2_nan(top, __shfl_xor_sync(~0u, top, 2));
          const Scale s0(static_cast<float>(top.x)), s1(static_cast<float>(top.y));
          if (t4 == 0) *reinterpret_cast<uint32_t*>(record + kv * (REC / 2) + 8 * D + (g + 8 * i) * (2 * D / kGroup) + c * 4) = s0.bits | s1.bits << 16;
          uint32_t word[2];
          auto encode = [&](auto fast) {
            constexpr bool F = decltype(fast)::value;
#pragma unroll
            for (int h = 0; h < 2; ++h)
              word[h] = s0.template codes<F>(v[0][h]) + (s0.template codes<F>(v[1][h]) << 4) + (s1.template codes<F>(v[2][h]) << 8) +
                        (s1.template codes<F>(v[3][h]) << 12);
          };
          if (__all_sync(~0u, s0.r > 0.f && s1.r > 0.f)) encode(std::true_type());
          else encode(std::false_type());
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            word[h] = place_fields(word[h]);
            if (kv) asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %0;\n" : "+r"(word[h]));
            w[kv ? h + 2 * i : i + 2 * h] = word[h];
          }
        }
        reinterpret_cast<uint4*>(record + kv * (REC / 2) + c * 512)[lane] = make_uint4(w[0], w[1], w[2], w[3]);
      }
      __syncwarp();
    }
  } else {
    // some of them (a single new token, most of the time): in the pieces that belong to one token
    const int end = static_cast<int>(min(count - t0, static_cast<int64_t>(kGranule)));
    for (int j = t0 < 0 ? static_cast<int>(-t0) : 0; j < end; j += TPI) {
      const bool there = j + own < end;
      const uint4 k = there ? load8<T, VEC>(x[0] + j * p.st[0]) : make_uint4(0, 0, 0, 0);
      const uint4 v = there ? load8<T, VEC>(x[1] + j * p.st[1]) : make_uint4(0, 0, 0, 0);
      uint32_t pair[4];
      uint32_t scale = quantise8<T>(k, pair), word = gather_fields(pair, to.n);
      if (there) to.put(record, 0, j + own, word, scale);
      scale = quantise8<T>(v, pair);
      word = gather_fields(pair, to.n);
      if (there) to.put(record, 1, j + own, word, scale);
    }
  }
}

// ---- reading -----------------------------------------------------------------------------------
struct ReadParams {
  void* y[2];                      // [Z, H, T, D]
  int64_t sz[2], sh[2], st[2];
  const uint8_t* data;
  CachePages pages;
  const int32_t *start, *count;
  int T, ctas;
};

// half (low or high of a pair) * f + c, in 32 bits: one instruction where a conversion and a sum are two
__device__ __forceinline__ float half_fma(uint32_t pair, int i, uint16_t f, float c) {
  float x;
  if (i) asm("{.reg .b16 l, h; mov.b32 {l, h}, %1; fma.rn.f32.f16 %0, h, %2, %3;}" : "=f"(x) : "r"(pair), "h"(f), "f"(c));
  else asm("{.reg .b16 l, h; mov.b32 {l, h}, %1; fma.rn.f32.f16 %0, l, %2, %3;}" : "=f"(x) : "r"(pair), "h"(f), "f"(c));
  return x;
}
__device__ __forceinline__ void put2(float* p, float a, float b) { *reinterpret_cast<float2*>(p) = make_float2(a, b); }
__device__ __forceinline__ void put2(__half* p, float a, float b) { *reinterpret_cast<__half2*>(p) = __floats2half2_rn(a, b); }
__device__ __forceinline__ void put2(__nv_bfloat16* p, float a, float b) { *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(a, b); }

// Every lane takes the words that a lane of the matrix instruction would: field n of a word under a mask, put
// beside the exponent of 128, is the half 128 + (c + 8) for n even; for n odd it is (c + 8) * 2^-17 as it is, of which
// 2^15 times less 2 makes c / 4, for scales times 4 (at most 2^127).  K's words hold two channels
// of a token; V's hold two tokens of a channel and become the same by a transpose of 8 x 8 (movmatrix).  Rows
// are put together in shared memory and stored 16 bytes at a time.  Against 8 channels of a token a lane, picked
// field by field (109 instructions for 8 values): 8 sequences of up to 8192 tokens, 16 heads of 64, 63 -> 55 us; 4 of 16384 tokens,
// 16 heads of 128, 112 -> 105 us, 95 % of the copy rate.
template <typename T, int D>
__global__ void __launch_bounds__(kWarps * 32) cache_read_kernel(const __grid_constant__ ReadParams p) {
  constexpr int REC = record_bytes(D), HALF = REC / 2, NC = D / 64, NG = D / kGroup;
  constexpr int PITCH = D + 32 / static_cast<int>(sizeof(T)) / (sizeof(T) == 4 ? 1 : 2);   // rows 4 (8: FP32) banks apart
  __shared__ __align__(16) T tile[kWarps][kGranule * PITCH];
  wait_for_earlier_kernels();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t4 = lane % 4;
  // (a CTA's warps share a head: their number is found with one division of 32 bits for all)
  const uint32_t zh = blockIdx.x / static_cast<uint32_t>(p.ctas), z = zh / static_cast<uint32_t>(p.pages.heads);
  const int head = static_cast<int>(zh - z * p.pages.heads), nth = static_cast<int>(blockIdx.x - zh * p.ctas) * (blockDim.x / 32) + warp;
  const int64_t start = p.start[z];
  const int64_t count = min(p.count ? p.count[z] : p.T, p.T);
  const int64_t gran = (start >> 4) + nth, t0 = gran * kGranule - start;
  if (t0 >= p.T) return;
  const int64_t at = t0 < count ? p.pages.granule(static_cast<int>(z), head, gran) : -1;
  uint4 w[2][NC] = {};
  uint32_t scale[2][2][NG / 2] = {};
  if (at >= 0) {
    const uint8_t* record = p.data + at * REC;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
#pragma unroll
      for (int c = 0; c < NC; ++c) w[kv][c] = reinterpret_cast<const uint4*>(record + kv * HALF + c * 512)[lane];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int k = 0; k < NG / 2; ++k)
          scale[kv][i][k] = reinterpret_cast<const uint32_t*>(record + kv * HALF + 8 * D)[(g + 8 * i) * (NG / 2) + k];
    }
  }
  T* own = tile[warp];
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      float s[2][4];                                 // by token half and field
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        s[i][0] = __uint_as_float(scale[kv][i][c] << 16);
        s[i][2] = __uint_as_float(scale[kv][i][c] & 0xffff0000u);
        s[i][1] = 4.f * s[i][0];
        s[i][3] = 4.f * s[i][2];
      }
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        // K: token half a % 2, channel half a / 2; V: the other way round
        const int i = kv ? a / 2 : a % 2, h = kv ? a % 2 : a / 2;
        uint32_t word = a == 0 ? w[kv][c].x : a == 1 ? w[kv][c].y : a == 2 ? w[kv][c].z : w[kv][c].w;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          uint32_t pair = n % 2 ? word & kHighField : (word & kLowField) | 0x58005800u;
          if (kv) asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %0;\n" : "+r"(pair));
          const uint16_t f = n % 2 ? 0x7800 : 0x3c00;               // 2^15, 1
          const float off = n % 2 ? -2.f : -136.f;
          put2(own + (g + 8 * i) * PITCH + 64 * c + 16 * n + 8 * h + 2 * t4, half_fma(pair, 0, f, off) * s[i][n], half_fma(pair, 1, f, off) * s[i][n]);
          if (n == 1) word = swap_bytes(word);
        }
      }
    }
    __syncwarp();
    T* y = static_cast<T*>(p.y[kv]) + static_cast<int64_t>(z) * p.sz[kv] + head * p.sh[kv];
    constexpr int PER = 16 / sizeof(T), PIECES = D / PER, ROWS = 32 / PIECES;
#pragma unroll
    for (int it = 0; it < kGranule / ROWS; ++it) {
      const int j = it * ROWS + lane / PIECES, d = lane % PIECES * PER;
      const int64_t t = t0 + j;
      if (t < 0 || t >= p.T) continue;
      const uint4 v = *reinterpret_cast<const uint4*>(own + j * PITCH + d);
      *reinterpret_cast<uint4*>(y + t * p.st[kv] + d) = at >= 0 && t < count ? v : make_uint4(0, 0, 0, 0);
    }
    __syncwarp();
  }
}

// Granules that `tokens` consecutive positions can touch.
int granules_of(int tokens) { return static_cast<int>((static_cast<int64_t>(tokens) + 2 * kGranule - 2) / kGranule); }

int check_cache(const char* what, int Z, int H, int T, int D, const void* data, int num_pages, int page, const int32_t* pages,
                int slots, const int32_t* start) {
  if (Z < 0 || H < 1 || T < 0 || num_pages < 0 || slots < 0) return fail(BSP_ERR_INVALID, "%s: bad sizes (Z %d, H %d, T %d, %d pages, %d slots)", what, Z, H, T, num_pages, slots);
  if (!valid_cache_dim(D)) return fail(BSP_ERR_UNSUPPORTED, "%s: head dimension %d (64 and 128 are supported)", what, D);
  if (!valid_page(page)) return fail(BSP_ERR_INVALID, "%s: pages of %d tokens (a power of two from 16 to 1024)", what, page);
  if (static_cast<int64_t>(slots) * page > INT32_MAX) return fail(BSP_ERR_UNSUPPORTED, "%s: sequences of up to 2^31 tokens", what);
  if (Z == 0 || T == 0) return BSP_OK;
  if ((num_pages && !data) || (slots && !pages) || !start) return fail(BSP_ERR_INVALID, "%s: NULL argument", what);
  if (reinterpret_cast<uintptr_t>(data) & 15) return fail(BSP_ERR_INVALID, "%s: the cache is not 16-byte aligned", what);
  return BSP_OK;
}

// CTAs for the granules that T tokens can touch: *warps each (fewer than kWarps where there are not as many), *ctas a head.
int grid_of(const char* what, int Z, int H, int T, unsigned* grid, int* warps, int* ctas) {
  const int granules = granules_of(T);
  *warps = granules < kWarps ? granules : kWarps;
  *ctas = (granules + kWarps - 1) / kWarps;
  if (static_cast<int64_t>(Z) * H > INT32_MAX / *ctas) return fail(BSP_ERR_UNSUPPORTED, "%s: too many tokens", what);
  *grid = static_cast<unsigned>(Z) * H * *ctas;
  return BSP_OK;
}

int launched(const char* what, cudaError_t e) {
  return e == cudaSuccess ? BSP_OK : fail(BSP_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

template <typename T, int D> int write(const WriteParams& p, bool vec, unsigned grid, int warps, cudaStream_t s) {
  return launched("cache write", launch_kernel(vec ? cache_write_kernel<T, D, true> : cache_write_kernel<T, D, false>, grid, warps * 32, 0, s, p));
}
template <typename T> int read(const ReadParams& p, int D, unsigned grid, int warps, cudaStream_t s) {
  return launched("cache read", launch_kernel(D == 64 ? cache_read_kernel<T, 64> : cache_read_kernel<T, 128>, grid, warps * 32, 0, s, p));
}

}  // namespace
}  // namespace bsp

extern "C" int64_t bsp_cache_page_bytes(int page, int D) {
  using namespace bsp;
  return valid_page(page) && valid_cache_dim(D) ? static_cast<int64_t>(page / kGranule) * record_bytes(D) : -1;
}

extern "C" int bsp_cache_write(const void* k, const void* v, int dtype, int Z, int H, int T, int D, int64_t k_sz, int64_t k_sh,
                               int64_t k_st, int64_t v_sz, int64_t v_sh, int64_t v_st, void* data, int num_pages, int page,
                               const int32_t* pages, int64_t pages_sz, int slots, const int32_t* start, const int32_t* count,
                               void* stream) {
  using namespace bsp;
  if (dtype != BSP_F16 && dtype != BSP_BF16) return fail(BSP_ERR_INVALID, "cache write: keys and values must be FP16 or BF16");
  if (const int rc = check_cache("cache write", Z, H, T, D, data, num_pages, page, pages, slots, start)) return rc;
  if (Z == 0 || T == 0) return BSP_OK;
  if (!k || !v) return fail(BSP_ERR_INVALID, "cache write: NULL argument");
  WriteParams p = {{k, v}, {k_sz, v_sz}, {k_sh, v_sh}, {k_st, v_st}, static_cast<uint8_t*>(data),
                   {pages, pages_sz, slots, num_pages, H, log2_of(page / kGranule)}, start, count, T, 0};
  uint64_t bits = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v);
  if (Z > 1) bits |= 2 * (k_sz | v_sz);
  if (H > 1) bits |= 2 * (k_sh | v_sh);
  if (T > 1) bits |= 2 * (k_st | v_st);
  unsigned grid;
  int warps;
  if (const int rc = grid_of("cache write", Z, H, T, &grid, &warps, &p.ctas)) return rc;
  const bool vec = bits % 16 == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == BSP_F16) return D == 64 ? write<__half, 64>(p, vec, grid, warps, s) : write<__half, 128>(p, vec, grid, warps, s);
  return D == 64 ? write<__nv_bfloat16, 64>(p, vec, grid, warps, s) : write<__nv_bfloat16, 128>(p, vec, grid, warps, s);
}

extern "C" int bsp_cache_read(void* k, void* v, int dtype, int Z, int H, int T, int D, int64_t k_sz, int64_t k_sh, int64_t k_st,
                              int64_t v_sz, int64_t v_sh, int64_t v_st, const void* data, int num_pages, int page,
                              const int32_t* pages, int64_t pages_sz, int slots, const int32_t* start, const int32_t* count,
                              void* stream) {
  using namespace bsp;
  if (!valid_dtype(dtype)) return fail(BSP_ERR_INVALID, "cache read: bad dtype %d", dtype);
  if (const int rc = check_cache("cache read", Z, H, T, D, data, num_pages, page, pages, slots, start)) return rc;
  if (Z == 0 || T == 0) return BSP_OK;
  if (!k || !v) return fail(BSP_ERR_INVALID, "cache read: NULL argument");
  uint64_t bits = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v);
  bits |= dtype_bytes(dtype) * (k_sz | k_sh | k_st | v_sz | v_sh | v_st);
  if (bits % 16) return fail(BSP_ERR_INVALID, "cache read: outputs need 16-byte aligned rows");
  ReadParams p = {{k, v}, {k_sz, v_sz}, {k_sh, v_sh}, {k_st, v_st}, static_cast<const uint8_t*>(data),
                  {pages, pages_sz, slots, num_pages, H, log2_of(page / kGranule)}, start, count, T, 0};
  unsigned grid;
  int warps;
  if (const int rc = grid_of("cache read", Z, H, T, &grid, &warps, &p.ctas)) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == BSP_F32) return read<float>(p, D, grid, warps, s);
  return dtype == BSP_F16 ? read<__half>(p, D, grid, warps, s) : read<__nv_bfloat16>(p, D, grid, warps, s);
}
