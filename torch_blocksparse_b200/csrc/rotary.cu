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
// F (two's complement, so negative positions turn back), and its leading bits, as a float in [-1, 1)
// half turns, go to sincospif.  The float's rounding (2^-25 of half a turn: 9e-8 rad) is what remains.
//
// Bound by memory: every element is read once and written once.  A CTA takes up to 8 tokens of all heads of
// q and k, computes the sines of its tokens once into shared memory (a pair's sine serves every
// head) and then moves rows in 16-byte pieces; both tensors in one launch.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "common.h"
#include "tile.cuh"

namespace bsp {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 8;      // tokens of a CTA
constexpr int kBatch = 2;          // rows that a thread has under way at a time

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

// A unit is VEC elements of the first half and their partners in the second (!INTER), VEC neighbouring
// elements (INTER), or VEC elements behind the turned ones.
template <typename T, int VEC, bool INTER>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ RotaryParams p) {
  extern __shared__ float2 cs[];                    // [tokens][pairs]
  __shared__ int tz[kMaxTokens], tl[kMaxTokens];
  const int tid = threadIdx.x, tokens = 1 << p.log_tokens;
  const int64_t first = static_cast<int64_t>(blockIdx.x) << p.log_tokens, total = static_cast<int64_t>(p.Z) * p.L;
  if (tid < tokens) {
    const int64_t n = first + tid;
    tz[tid] = n < total ? static_cast<int>(n / p.L) : -1;
    tl[tid] = static_cast<int>(n % p.L);
  }
  __syncthreads();
  for (int i = tid; i < p.pairs << p.log_tokens; i += kThreads) {
    const int tok = i / p.pairs, pr = i - tok * p.pairs, z = tz[tok], l = tl[tok];
    if (z < 0) continue;
    const int64_t a = p.table[p.pairs + pr];
    const int64_t axis = a < 0 ? 0 : a < p.axes ? a : p.axes - 1;
    int64_t pos = l;
    if (p.pos_bytes) {
      const int64_t at = axis * p.p_sa + z * p.p_sz + l * p.p_sl;
      pos = p.pos_bytes == 4 ? static_cast<const int32_t*>(p.positions)[at] : static_cast<const int64_t*>(p.positions)[at];
    }
    const int64_t turn = static_cast<int64_t>(static_cast<uint64_t>(pos) * static_cast<uint64_t>(p.table[pr]));
    float s, c;
    sincospif(__ll2float_rn(turn) * 0x1p-63f, &s, &c);
    cs[i] = make_float2(c, p.inverse ? -s : s);
  }
  __syncthreads();

  const int units = 1 << p.log_units, u = tid & (units - 1), step = kThreads >> p.log_units;
  const int turned = INTER ? 2 * p.pairs / VEC : p.pairs / VEC, rest = (p.D - 2 * p.pairs) / VEC;
  if (u >= turned + rest) return;
  const int rows = p.heads << p.log_tokens;
  using V = Vec<T, VEC>;
  const bool tail = u >= turned;
  const int d = tail ? 2 * p.pairs + (u - turned) * VEC : u * VEC, far = INTER || tail ? 0 : p.pairs;
  // kBatch rows at a time: their loads are under way together
  for (int r0 = tid >> p.log_units; r0 < rows; r0 += kBatch * step) {
    V a[kBatch], b[kBatch];
    T* y[kBatch];
    int tok[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int r = r0 + i * step;
      tok[i] = r & (tokens - 1);
      y[i] = nullptr;
      if (r >= rows || tz[tok[i]] < 0) continue;
      const int64_t z = tz[tok[i]], l = tl[tok[i]];
      int h = r >> p.log_tokens;
      const RotaryTensor& t = p.t[h >= p.heads0];
      if (h >= p.heads0) h -= p.heads0;
      const T* x = static_cast<const T*>(t.x) + z * t.x_sz + h * t.x_sh + l * t.x_sl + d;
      y[i] = static_cast<T*>(t.y) + z * t.y_sz + h * t.y_sh + l * t.y_sl + d;
      a[i] = *reinterpret_cast<const V*>(x);
      if (far) b[i] = *reinterpret_cast<const V*>(x + far);
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (!y[i]) continue;
      const float2* w = cs + tok[i] * p.pairs;
      if (!tail) {
        if constexpr (INTER) {
#pragma unroll
          for (int j = 0; j < VEC / 2; ++j) {
            const float2 f = w[d / 2 + j];
            const float x0 = to_f(a[i].v[2 * j]), x1 = to_f(a[i].v[2 * j + 1]);
            a[i].v[2 * j] = cvt_out<T>(x0 * f.x - x1 * f.y);
            a[i].v[2 * j + 1] = cvt_out<T>(x1 * f.x + x0 * f.y);
          }
        } else {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const float2 f = w[d + j];
            const float x0 = to_f(a[i].v[j]), x1 = to_f(b[i].v[j]);
            a[i].v[j] = cvt_out<T>(x0 * f.x - x1 * f.y);
            b[i].v[j] = cvt_out<T>(x1 * f.x + x0 * f.y);
          }
        }
      }
      *reinterpret_cast<V*>(y[i]) = a[i];
      if (far) *reinterpret_cast<V*>(y[i] + far) = b[i];
    }
  }
}

template <typename T, int VEC, bool INTER> int launch(RotaryParams& p, cudaStream_t stream) {
  const int units = (INTER ? 2 * p.pairs : p.pairs) / VEC + (p.D - 2 * p.pairs) / VEC;
  for (p.log_units = 0; (1 << p.log_units) < units; ++p.log_units) {}
  const int64_t total = static_cast<int64_t>(p.Z) * p.L;
  // more tokens a CTA while every SM still gets several
  for (p.log_tokens = 0; (2 << p.log_tokens) <= kMaxTokens && total >> p.log_tokens >= 2048; ++p.log_tokens) {}
  const int64_t grid = (total + (1 << p.log_tokens) - 1) >> p.log_tokens;
  if (grid > INT32_MAX) return fail(BSP_ERR_UNSUPPORTED, "rotary: too many tokens (%lld)", (long long)total);
  rotary_kernel<T, VEC, INTER><<<static_cast<unsigned>(grid), kThreads, sizeof(float2) * p.pairs << p.log_tokens, stream>>>(p);
  const cudaError_t e = cudaGetLastError();
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
