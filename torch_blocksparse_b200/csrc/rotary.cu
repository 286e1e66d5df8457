// Rotary positions: pairs of channels of queries and keys turned by angles that grow with the
// token's position along one or several axes (text; height and width; time, height and width).
//
//   y0 = x0 cos t - x1 sin t,   y1 = x1 cos t + x0 sin t,   t = position[axis(pair)] * freq(pair)
//
// and the gradient is the turn by -t (`inverse`).
//
// Angles.  A float loses the angle of a far position (2^20 times a frequency near 1 is off by up to
// 2^-5 rad), and doubles are slow.  The table holds each frequency as a 64-bit fraction of a whole
// turn, F = round(freq / 2 pi * 2^64); position * F modulo 2^64 is then the exact fraction of a turn of
// F (two's complement, so negative positions turn back).  Whole quarters of a turn are taken off it as integers, the rest,
// an eighth of a turn at most, goes to sincospif as a float, and the quarters come back as exchanges and signs.  So the float's
// rounding, 2^-24 of the rest, is no more than the last place of either result (as a float of up to half a turn the angle
// alone would be off by 9e-8 rad).
//
// Bound by memory: every element is read once and written once.  A CTA takes up to 8 tokens of all heads of
// q and k, computes the sines of its tokens once into shared memory (a pair's sine serves every
// head) and then moves rows in 16-byte pieces; both tensors in one launch.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "common.h"
#include "launch.cuh"
#include "tile.cuh"

namespace bsp {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 8;      // tokens of a CTA

struct RotaryTensor {
  const void* x;
  void* y;
  int64_t x_sz, x_sh, x_sl, y_sz, y_sh, y_sl;
};
struct RotaryParams {
  RotaryTensor t[2];
  int heads0, heads;               // heads of the first tensor, of both
  int Z, L, D, pairs;
  const int64_t* table;            // [2, pairs]: turns, axes
  int axes;
  const void* positions;
  int64_t p_sa, p_sz, p_sl;
  int pos_bytes;                   // 4, 8; 0: the token's index
  int inverse;
  int log_tokens, log_units;
};

template <typename T> __device__ __forceinline__ float to_f(T v) { return static_cast<float>(v); }

template <typename T, int VEC> struct alignas(sizeof(T) * VEC) Vec { T v[VEC]; };

// (through uint4: the compiler splits accesses of the struct itself, 51 -> 59 us for 8192 tokens x 2 x 32 heads of 128)
template <typename V> __device__ __forceinline__ V load_v(const void* p) {
  if constexpr (sizeof(V) == 16) {
    const uint4 x = *reinterpret_cast<const uint4*>(p);
    return *reinterpret_cast<const V*>(&x);
  } else {
    return *reinterpret_cast<const V*>(p);
  }
}
template <typename V> __device__ __forceinline__ void store_v(void* p, const V& v) {
  if constexpr (sizeof(V) == 16) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(&v);
  else *reinterpret_cast<V*>(p) = v;
}

// A unit is VEC elements of the first half and their partners in the second (!INTER), VEC neighbouring
// elements (INTER), or VEC elements behind the turned ones.
template <typename T, int VEC, bool INTER>
__global__ void __launch_bounds__(kThreads, VEC == 8 && !INTER ? 5 : 4) rotary_kernel(const __grid_constant__ RotaryParams p) {
  // Heads that a thread has under way at a time: with the sines of 8 pairs in registers, more warps do more than a second one
  // (8192 tokens x 2 x 32 heads of 128: one 51 us, two 58, four 75; with fewer sines the other way round: FP32, 3219 tokens x 15 heads of 80, 9.5 and 8.9 us).
  constexpr int kBatch = VEC == 8 && !INTER ? 1 : 2;
  extern __shared__ float2 cs[];                    // [tokens][pairs]
  wait_for_earlier_kernels();
  const int tid = threadIdx.x, tokens = 1 << p.log_tokens;
  const int64_t first = static_cast<int64_t>(blockIdx.x) << p.log_tokens, total = static_cast<int64_t>(p.Z) * p.L;
  // A thread keeps one unit of one token, and so its sines, for every head that it takes.
  const int u = tid & ((1 << p.log_units) - 1), tok = tid >> p.log_units & (tokens - 1);
  const int h0 = tid >> (p.log_units + p.log_tokens), step = kThreads >> (p.log_units + p.log_tokens);
  const int turned = INTER ? 2 * p.pairs / VEC : p.pairs / VEC, rest = (p.D - 2 * p.pairs) / VEC;
  const bool works = u < turned + rest && first + tok < total, tail = u >= turned;
  const int d = tail ? 2 * p.pairs + (u - turned) * VEC : u * VEC, far = INTER || tail ? 0 : p.pairs;
  const int64_t z = (first + tok) / p.L, l = (first + tok) - z * p.L;
  using V = Vec<T, VEC>;
  V a[kBatch], b[kBatch];
  auto load = [&](int h) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      int head = h + i * step;
      if (!works || head >= p.heads) continue;
      const RotaryTensor& t = p.t[head >= p.heads0];
      if (head >= p.heads0) head -= p.heads0;
      const T* x = static_cast<const T*>(t.x) + z * t.x_sz + l * t.x_sl + head * t.x_sh + d;
      a[i] = load_v<V>(x);
      if (far) b[i] = load_v<V>(x + far);
    }
  };

  for (int i = tid; i < p.pairs << p.log_tokens; i += kThreads) {
    const int n = i / p.pairs, pr = i - n * p.pairs;
    if (first + n >= total) break;
    const int64_t zn = (first + n) / p.L, ln = (first + n) - zn * p.L;
    const int64_t axis = max(static_cast<int64_t>(0), min(p.table[p.pairs + pr], static_cast<int64_t>(p.axes - 1)));
    int64_t pos = ln;
    if (p.pos_bytes) {
      const int64_t at = axis * p.p_sa + zn * p.p_sz + ln * p.p_sl;
      pos = p.pos_bytes == 4 ? static_cast<const int32_t*>(p.positions)[at] : static_cast<const int64_t*>(p.positions)[at];
    }
    const uint64_t turn = static_cast<uint64_t>(pos) * static_cast<uint64_t>(p.table[pr]);
    const uint32_t quarters = static_cast<uint32_t>((turn + (1ull << 61)) >> 62);
    float s, c;
    sincospif(__ll2float_rn(static_cast<int64_t>(turn - (static_cast<uint64_t>(quarters) << 62))) * 0x1p-63f, &s, &c);
    if (quarters & 1) {
      const float t = s;
      s = c;
      c = -t;
    }
    if (quarters & 2) {
      s = -s;
      c = -c;
    }
    cs[i] = make_float2(c, p.inverse ? -s : s);
  }
  __syncthreads();
  if (!works) return;
  constexpr int NCS = INTER ? (VEC + 1) / 2 : VEC;
  float2 w[NCS];
#pragma unroll
  for (int j = 0; j < NCS; ++j) w[j] = tail ? make_float2(1.f, 0.f) : cs[tok * p.pairs + (INTER ? d / 2 : d) + j];

  for (int h = h0; h < p.heads; h += kBatch * step) {
    load(h);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      int head = h + i * step;
      if (head >= p.heads) break;
      const RotaryTensor& t = p.t[head >= p.heads0];
      if (head >= p.heads0) head -= p.heads0;
      if (!tail) {
        if constexpr (INTER) {
#pragma unroll
          for (int j = 0; j < VEC / 2; ++j) {
            const float x0 = to_f(a[i].v[2 * j]), x1 = to_f(a[i].v[2 * j + 1]);
            a[i].v[2 * j] = cvt_out<T>(x0 * w[j].x - x1 * w[j].y);
            a[i].v[2 * j + 1] = cvt_out<T>(x1 * w[j].x + x0 * w[j].y);
          }
        } else {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const float x0 = to_f(a[i].v[j]), x1 = to_f(b[i].v[j]);
            a[i].v[j] = cvt_out<T>(x0 * w[j].x - x1 * w[j].y);
            b[i].v[j] = cvt_out<T>(x1 * w[j].x + x0 * w[j].y);
          }
        }
      }
      T* y = static_cast<T*>(t.y) + z * t.y_sz + l * t.y_sl + head * t.y_sh + d;
      store_v(y, a[i]);
      if (far) store_v(y + far, b[i]);
    }
  }
}

template <typename T, int VEC, bool INTER> int launch(RotaryParams& p, cudaStream_t stream) {
  const int units = (INTER ? 2 * p.pairs : p.pairs) / VEC + (p.D - 2 * p.pairs) / VEC;
  for (p.log_units = 0; (1 << p.log_units) < units; ++p.log_units) {}
  const int64_t total = static_cast<int64_t>(p.Z) * p.L;
  // more tokens a CTA while every SM still gets several
  for (p.log_tokens = 0; (2 << p.log_tokens) <= kMaxTokens && total >> p.log_tokens >= 2048 && p.log_units + p.log_tokens < 8; ++p.log_tokens) {}
  const int64_t grid = (total + (1 << p.log_tokens) - 1) >> p.log_tokens;
  if (grid > INT32_MAX) return fail(BSP_ERR_UNSUPPORTED, "rotary: too many tokens (%lld)", (long long)total);
  const cudaError_t e = launch_kernel(rotary_kernel<T, VEC, INTER>, static_cast<unsigned>(grid), kThreads, sizeof(float2) * p.pairs << p.log_tokens, stream, p);
  return e == cudaSuccess ? BSP_OK : fail(BSP_ERR_CUDA, "rotary: %s", cudaGetErrorString(e));
}

// Elements that can be moved together: everything that a unit's address is made of is a multiple of them.
int common_vec(const RotaryParams& p, int e, bool inter) {
  int64_t bits = (inter ? 2 * p.pairs : p.pairs) | (p.D - 2 * p.pairs);
  uint64_t at = 0;
  for (int i = 0; i < (p.heads > p.heads0 ? 2 : 1); ++i) {
    const RotaryTensor& t = p.t[i];
    const int heads = i ? p.heads - p.heads0 : p.heads0;
    if (p.Z > 1) bits |= t.x_sz | t.y_sz;
    if (heads > 1) bits |= t.x_sh | t.y_sh;
    if (p.L > 1) bits |= t.x_sl | t.y_sl;
    at |= reinterpret_cast<uintptr_t>(t.x) | reinterpret_cast<uintptr_t>(t.y);
  }
  int v = 16 / e;
  while (v > 1 && (bits % v || at % (v * e))) v /= 2;
  return v;
}

template <typename T, int VEC> int launch_vec(RotaryParams& p, int vec, bool inter, cudaStream_t stream) {
  if (vec >= VEC) return inter ? launch<T, VEC, true>(p, stream) : launch<T, VEC, false>(p, stream);
  if constexpr (VEC > 2) return launch_vec<T, VEC / 2>(p, vec, inter, stream);
  return inter ? fail(BSP_ERR_INVALID, "rotary: neighbouring pairs need even strides and pairs on a boundary of their size")
               : launch<T, 1, false>(p, stream);
}

}  // namespace
}  // namespace bsp

extern "C" int bsp_rotary(const void* q, void* q_out, int Hq, int64_t q_sz, int64_t q_sh, int64_t q_sl, int64_t qo_sz,
                          int64_t qo_sh, int64_t qo_sl, const void* k, void* k_out, int Hk, int64_t k_sz, int64_t k_sh,
                          int64_t k_sl, int64_t ko_sz, int64_t ko_sh, int64_t ko_sl, int dtype, int Z, int L, int D, int pairs,
                          int interleaved, const int64_t* table, int axes, const void* positions, int pos_bytes, int64_t p_sa,
                          int64_t p_sz, int64_t p_sl, int inverse, void* stream) {
  using namespace bsp;
  if (!valid_dtype(dtype)) return fail(BSP_ERR_INVALID, "rotary: bad dtype %d", dtype);
  if (Z < 0 || L < 0 || Hq < 0 || Hk < 0 || D < 2 || pairs < 1 || 2 * pairs > D || D > 256)
    return fail(BSP_ERR_INVALID, "rotary: bad sizes (Z %d, L %d, heads %d + %d, D %d, pairs %d)", Z, L, Hq, Hk, D, pairs);
  if (static_cast<int64_t>(Hq) + Hk > (1 << 20)) return fail(BSP_ERR_UNSUPPORTED, "rotary: too many heads");
  if (axes < 1 || (pos_bytes != 0 && pos_bytes != 4 && pos_bytes != 8) || (pos_bytes == 0 && axes != 1) || (pos_bytes && !positions))
    return fail(BSP_ERR_INVALID, "rotary: positions of %d bytes for %d axes", pos_bytes, axes);
  if (Z == 0 || L == 0 || Hq + Hk == 0) return BSP_OK;
  if (!table || (Hq && (!q || !q_out)) || (Hk && (!k || !k_out))) return fail(BSP_ERR_INVALID, "rotary: NULL argument");
  RotaryParams p;
  p.t[0] = {q, q_out, q_sz, q_sh, q_sl, qo_sz, qo_sh, qo_sl};
  p.t[1] = {k, k_out, k_sz, k_sh, k_sl, ko_sz, ko_sh, ko_sl};
  if (Hq == 0) p.t[0] = p.t[1];
  p.heads0 = Hq ? Hq : Hk;
  p.heads = Hq + Hk;
  p.Z = Z; p.L = L; p.D = D; p.pairs = pairs;
  p.table = table; p.axes = axes;
  p.positions = positions; p.pos_bytes = pos_bytes; p.p_sa = p_sa; p.p_sz = p_sz; p.p_sl = p_sl;
  p.inverse = inverse;
  const int e = dtype_bytes(dtype), vec = common_vec(p, e, interleaved != 0);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == BSP_F32) return launch_vec<float, 4>(p, vec, interleaved, s);
  return dtype == BSP_F16 ? launch_vec<__half, 8>(p, vec, interleaved, s) : launch_vec<__nv_bfloat16, 8>(p, vec, interleaved, s);
}
