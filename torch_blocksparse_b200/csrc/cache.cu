// Writing keys and values into the 4-bit cache (quantised on the way) and reading them back.
// The format is described in cache.cuh.
//
// Both kernels give a warp one granule (16 tokens of one head).  A token takes D / 8 lanes, 8 consecutive
// channels (one 16-byte access of a 16-bit type) each, so a warp holds 2 (D = 128) or 4 tokens at a time.  Lane
// `sub` of a token has channels 8 sub .. 8 sub + 7: chunk c = sub / 8 of 64, quarter n = sub / 2 % 4, half h = sub % 2.
//
// Bound by memory: 2 bytes in and 0.5625 out a value, or the other way round.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "cache.cuh"
#include "common.h"
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
  int Z, T, granules;              // granules: most that T tokens can touch
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

// The codes + 8 of 8 channels, two in each word (bits 0-3 and 16-19), and the scale of their group, which 4
// neighbouring lanes hold together.
//
// rint(x / s) without a division, and equal to it: with |x / s| < 8, r within 2^-23 of 1 / s and x of at
// most 11 significant bits, s of 8, a quotient that is no tie is at least 2^-13 away from one, x * r at most
// 2^-20 away from the quotient.  So x * r rounded to a multiple of 2^-16 (an FMA that adds 192, where
// floats are 2^-16 apart) lies on the same side of a tie, or on the tie itself if the quotient
// is one, and taking 192 off and adding 1.5 * 2^23 + 8 in one sum then rounds it to an even integer that ends in c + 8.
// max / 7 is the rounded product with 1 / 7 and one step of correction by its exact remainder, which gives the
// rounded quotient (checked over both types' values, with the rest, by the tests).
template <typename T> __device__ __forceinline__ uint32_t quantise8(uint4 raw, uint32_t (&pair)[4]) {
  using T2 = typename Two<T>::t;
  const uint32_t in[4] = {raw.x, raw.y, raw.z, raw.w};
  T2 v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const T2*>(&in[i]);
  T2 m2 = __hmax2_nan(__hmax2_nan(__habs2(v[0]), __habs2(v[1])), __hmax2_nan(__habs2(v[2]), __habs2(v[3])));
  m2 = __hmax2_nan(m2, __shfl_xor_sync(~0u, m2, 2));    // (lanes sub ^ 1, sub ^ 2 share the group)
  m2 = __hmax2_nan(m2, __shfl_xor_sync(~0u, m2, 1));
  const float amax = static_cast<float>(__hmax_nan(m2.x, m2.y));
  constexpr float kSeventh = 1.f / 7.f;
  const float q0 = amax * kSeventh;
  const __nv_bfloat16 fast = __float2bfloat16_rn(__fmaf_rn(__fmaf_rn(-7.f, q0, amax), kSeventh, q0));
  if (amax > 1e-29f && amax < INFINITY) {
    const float s = __bfloat162float(fast);
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 x = to_f2(v[i]);
      const float a = __fadd_rn(__fmaf_rn(x.x, r, 192.f), 12582912.f + 8.f - 192.f);
      const float b = __fadd_rn(__fmaf_rn(x.y, r, 192.f), 12582912.f + 8.f - 192.f);
      pair[i] = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x5410) & 0x000f000fu;
    }
    return __bfloat16_as_ushort(fast);
  }
  // zeros, infinities, NaN, or scales whose reciprocal a float does not hold
  const __nv_bfloat16 sb = amax < INFINITY ? __float2bfloat16_rn(__fdiv_rn(amax, 7.f)) : __ushort_as_bfloat16(0x7fff);
  const float s = __bfloat162float(sb);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 x = to_f2(v[i]);
    float c[2] = {x.x, x.y};
#pragma unroll
    for (int j = 0; j < 2; ++j) c[j] = s > 0.f ? fminf(fmaxf(rintf(__fdiv_rn(c[j], s)), -8.f), 7.f) : 0.f;
    pair[i] = static_cast<uint32_t>(static_cast<int>(c[0]) + 8) | static_cast<uint32_t>(static_cast<int>(c[1]) + 8) << 16;
  }
  return __bfloat16_as_ushort(sb);
}

// The four quarters n of a chunk and half hold one 4-bit field each of four words; lane n is left with word n.
__device__ __forceinline__ uint32_t gather_fields(const uint32_t (&pair)[4], int n) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pair[i] << (4 * n);
  const bool hi = n & 2, odd = n & 1;               // quarters differ in lane bits 2 (hi) and 1 (odd)
  const uint32_t k0 = (hi ? w[2] : w[0]) | __shfl_xor_sync(~0u, hi ? w[0] : w[2], 4);
  const uint32_t k1 = (hi ? w[3] : w[1]) | __shfl_xor_sync(~0u, hi ? w[1] : w[3], 4);
  return (odd ? k1 : k0) | __shfl_xor_sync(~0u, odd ? k0 : k1, 2);
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
  __shared__ __align__(16) uint8_t image[kWarps][REC];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * kWarps + warp;
  const int64_t zh = id / p.granules;
  const int z = static_cast<int>(zh / p.pages.heads), head = static_cast<int>(zh % p.pages.heads);
  if (z >= p.Z) return;
  const int64_t start = p.start[z];
  const int64_t count = min(p.count ? p.count[z] : p.T, p.T);
  // granules of positions from the one that `start` lies in; tokens t0 .. t0 + 15 of the operands
  const int64_t g = (start >> 4) + id % p.granules, t0 = g * kGranule - start;
  if (t0 >= count) return;
  const int64_t at = p.pages.granule(z, head, g);   // (negative positions have none)
  if (at < 0) return;
  uint8_t* record = p.data + at * REC;
  constexpr int LPT = D / 8, TPI = 32 / LPT, ITER = kGranule / TPI;
  const Places<D> to(lane);
  const int own = lane / LPT;
  const T* x[2];
#pragma unroll
  for (int kv = 0; kv < 2; ++kv)
    x[kv] = static_cast<const T*>(p.x[kv]) + z * p.sz[kv] + head * p.sh[kv] + (t0 + own) * p.st[kv] + to.sub * 8;
  if (t0 >= 0 && t0 + kGranule <= count) {
    // all 16 tokens: put together in shared memory and stored 16 bytes at a time
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      uint4 raw[ITER];
#pragma unroll
      for (int it = 0; it < ITER; ++it) raw[it] = load8<T, VEC>(x[kv] + it * TPI * p.st[kv]);
      // (of a token's place only what depends on the lane is computed: steps of 8 / TPI go through places 0 .. 7)
      uint8_t* base = image[warp];
#pragma unroll
      for (int it = 0; it < ITER; ++it) {
        uint32_t pair[4];
        const uint32_t scale = quantise8<T>(raw[it], pair);
        const uint32_t word = gather_fields(pair, to.n);
        const int j = it * TPI;
        if (kv == 0) *reinterpret_cast<uint32_t*>(base + word_at(to.c, own, to.n, 2 * to.h) + word_at(0, j % 8, 0, j / 8)) = word;
        else {
          uint8_t* q = base + REC / 2 + word_at(to.c, 2 * to.n, own / 2, to.h) + 2 * (own % 2) + word_at(0, 0, j % 8 / 2, 2 * (j / 8));
          *reinterpret_cast<uint16_t*>(q) = static_cast<uint16_t>(word);
          *reinterpret_cast<uint16_t*>(q + 64) = static_cast<uint16_t>(word >> 16);
        }
        if (to.sub % 4 == 0)
          *reinterpret_cast<uint16_t*>(base + kv * (REC / 2) + 8 * D + own * (2 * D / kGroup) + to.sub / 4 * 2 + j * (2 * D / kGroup)) = static_cast<uint16_t>(scale);
      }
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < (REC / 16 + 31) / 32; ++i)
      if (i * 32 + lane < REC / 16) reinterpret_cast<uint4*>(record)[i * 32 + lane] = reinterpret_cast<const uint4*>(image[warp])[i * 32 + lane];
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
  int Z, T, granules;
};

template <typename T> __device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    typename Two<T>::t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      o[i].x = cvt_out<T>(v[2 * i]);
      o[i].y = cvt_out<T>(v[2 * i + 1]);
    }
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(o);
  }
}

// The value of a code + 8 in the lowest four bits: 2^23 + c + 8 as a float, less 2^23 + 8.
__device__ __forceinline__ float value_of(uint32_t code, float s) { return (__uint_as_float(0x4b000000u | (code & 15u)) - 8388616.f) * s; }

template <typename T, int D>
__global__ void __launch_bounds__(kWarps * 32) cache_read_kernel(const __grid_constant__ ReadParams p) {
  constexpr int LPT = D / 8, TPI = 32 / LPT, ITER = kGranule / TPI, REC = record_bytes(D), HALF = REC / 2;
  __shared__ __align__(16) uint8_t image[kWarps][REC];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * kWarps + warp;
  const int64_t zh = id / p.granules;
  const int z = static_cast<int>(zh / p.pages.heads), head = static_cast<int>(zh % p.pages.heads);
  if (z >= p.Z) return;
  const int64_t start = p.start[z];
  const int64_t count = min(p.count ? p.count[z] : p.T, p.T);
  const int64_t g = (start >> 4) + id % p.granules, t0 = g * kGranule - start;
  if (t0 >= p.T) return;
  const int64_t at = t0 < count ? p.pages.granule(z, head, g) : -1;
  if (at >= 0) {
    const uint4* record = reinterpret_cast<const uint4*>(p.data + at * REC);
#pragma unroll
    for (int i = 0; i < (REC / 16 + 31) / 32; ++i)
      if (i * 32 + lane < REC / 16) reinterpret_cast<uint4*>(image[warp])[i * 32 + lane] = record[i * 32 + lane];
  }
  __syncwarp();
  const int sub = lane % LPT, c = sub / 8, n = sub / 2 % 4, h = sub % 2;
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    T* y = static_cast<T*>(p.y[kv]) + z * p.sz[kv] + head * p.sh[kv] + sub * 8;
    const uint8_t* codes = image[warp] + kv * HALF;
#pragma unroll
    for (int it = 0; it < ITER; ++it) {
      const int j = it * TPI + lane / LPT;
      const int64_t t = t0 + j;
      if (t < 0 || t >= p.T) continue;
      float v[8];
      if (at >= 0 && t < count) {
        const float s = __bfloat162float(__ushort_as_bfloat16(*reinterpret_cast<const uint16_t*>(codes + 8 * D + (j * (D / kGroup) + sub / 4) * 2)));
        if (kv == 0) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(codes + word_at(c, j % 8, i, j / 8 + 2 * h)) >> (4 * n);
            v[2 * i] = value_of(w, s);
            v[2 * i + 1] = value_of(w >> 16, s);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            v[i] = value_of(*reinterpret_cast<const uint16_t*>(codes + word_at(c, i, j % 8 / 2, h + 2 * (j / 8)) + 2 * (j % 2)) >> (4 * n), s);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.f;
      }
      store8(y + t * p.st[kv], v);
    }
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

int grid_of(const char* what, int Z, int H, int granules, unsigned* grid) {
  const int64_t n = (static_cast<int64_t>(Z) * H * granules + kWarps - 1) / kWarps;
  if (static_cast<int64_t>(Z) * H > (1LL << 40) / granules || n > INT32_MAX) return fail(BSP_ERR_UNSUPPORTED, "%s: too many tokens", what);
  *grid = static_cast<unsigned>(n);
  return BSP_OK;
}

int launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? BSP_OK : fail(BSP_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

template <typename T, int D> int write(const WriteParams& p, bool vec, unsigned grid, cudaStream_t s) {
  if (vec) cache_write_kernel<T, D, true><<<grid, kWarps * 32, 0, s>>>(p);
  else cache_write_kernel<T, D, false><<<grid, kWarps * 32, 0, s>>>(p);
  return launched("cache write");
}
template <typename T> int read(const ReadParams& p, int D, unsigned grid, cudaStream_t s) {
  if (D == 64) cache_read_kernel<T, 64><<<grid, kWarps * 32, 0, s>>>(p);
  else cache_read_kernel<T, 128><<<grid, kWarps * 32, 0, s>>>(p);
  return launched("cache read");
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
                   {pages, pages_sz, slots, num_pages, H, log2_of(page / kGranule)}, start, count, Z, T, granules_of(T)};
  uint64_t bits = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v);
  if (Z > 1) bits |= 2 * (k_sz | v_sz);
  if (H > 1) bits |= 2 * (k_sh | v_sh);
  if (T > 1) bits |= 2 * (k_st | v_st);
  unsigned grid;
  if (const int rc = grid_of("cache write", Z, H, p.granules, &grid)) return rc;
  const bool vec = bits % 16 == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == BSP_F16) return D == 64 ? write<__half, 64>(p, vec, grid, s) : write<__half, 128>(p, vec, grid, s);
  return D == 64 ? write<__nv_bfloat16, 64>(p, vec, grid, s) : write<__nv_bfloat16, 128>(p, vec, grid, s);
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
                  {pages, pages_sz, slots, num_pages, H, log2_of(page / kGranule)}, start, count, Z, T, granules_of(T)};
  unsigned grid;
  if (const int rc = grid_of("cache read", Z, H, p.granules, &grid)) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == BSP_F32) return read<float>(p, D, grid, s);
  return dtype == BSP_F16 ? read<__half>(p, D, grid, s) : read<__nv_bfloat16>(p, D, grid, s);
}
