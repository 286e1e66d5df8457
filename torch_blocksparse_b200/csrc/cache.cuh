// The 4-bit key / value cache: its format, shared by the kernels that write, read and attend over it.
//
// Values.  For every token, head and group of 32 channels s = bf16(max |x| / 7) and codes
// c = rint(x / s) in [-8, 7]; the cache stands for s * c.  A bf16 scale keeps the whole range of both 16-bit types
// (an fp16 one would overflow on bf16 values) and its rounding, 2^-9 of the value, is far below a code's
// half step.  A group with an infinity or a NaN gets a NaN scale: all of it reads back as NaN.
//
// Storage: [pages][heads][page / 16] granules of 16 tokens, 18 * D bytes each (4.5 bits a value):
//   K codes   8 D bytes  for every 64 channels the words of an m16n8k16 A operand (16 tokens x 16 channels)
//   K scales    D bytes  bf16 [token][D / 32]
//   V codes   8 D bytes  the same of V transposed (16 channels x 16 tokens)
//   V scales    D bytes
// A lane of the matrix instruction reads one uint4 for every 64 channels: word a of it is register a of
// the operand, with four 4-bit fields in each half for the four products n = 0 .. 3 over channels
// 64 c + 16 n .. + 15.  Fields n = 0 and 1 lie in bits 3-6 and 7-10 of a half, n = 2 and 3 do after its bytes are swapped
// (11-14; 15, 0, 1, 2).  So the codes go from memory to the tensor cores with one AND, and one byte permutation for
// four registers: c + 8 in bits 7-10 is the half (c + 8) * 2^-17, in bits 3-6 (c + 8) * 2^-21, exact both, since halves are
// evenly spaced up to 2^-13.  The higher a code lies, the more of a product the instruction keeps: it lines its
// addends up by the exponents of its operands, and what a denormal operand has in leading zeros is lost at the other end
// (fields at bits 0-3 and 4-7 left sums of few tokens at 2^-16 of their terms, these at 2^-19).
// A code word of K holds one token, a half word of V one token: a token is written without reading its neighbours.
#pragma once
#include <cstdint>

namespace bsp {

constexpr int kGranule = 16;       // tokens
constexpr int kGroup = 32;         // channels that share a scale
__host__ __device__ constexpr int record_bytes(int D) { return 18 * D; }

#ifdef __CUDACC__
// Four fields in bits 0-3, 4-7, 8-11 and 12-15 of each half, moved to where the format has them: a rotation by three.
__device__ __forceinline__ uint32_t place_fields(uint32_t word) { return ((word << 3) & 0xfff8fff8u) | ((word >> 13) & 0x00070007u); }
constexpr uint32_t kLowField = 0x00780078u, kHighField = 0x07800780u;   // products n even, n odd
__device__ __forceinline__ uint32_t swap_bytes(uint32_t word) { return __byte_perm(word, 0, 0x2301); }   // fields 2 and 3 to the front
#endif

inline bool valid_cache_dim(int D) { return D == 64 || D == 128; }
inline bool valid_page(int page) { return page >= 16 && page <= 1024 && (page & (page - 1)) == 0; }
inline int log2_of(int n) { int s = 0; while ((1 << s) < n) ++s; return s; }

// Where pages lie, and which of them a sequence has: every id and every slot is checked before use, so
// that a table may hold anything (-1: no page).
struct CachePages {
  const int32_t* table;            // [Z, slots]
  int64_t z_stride;
  int slots, num_pages, heads, shift;   // shift: log2(granules of a page)
  // Byte offset / record size of granule g of a sequence, or -1 where it has no page.
  __device__ __forceinline__ int64_t granule(int z, int head, int64_t g) const {
    const int64_t slot = g >> shift;
    if (g < 0 || slot >= slots) return -1;
    const int32_t id = table[z * z_stride + slot];
    if (id < 0 || id >= num_pages) return -1;
    return ((static_cast<int64_t>(id) * heads + head) << shift) + (g & ((1 << shift) - 1));
  }
};

}  // namespace bsp
