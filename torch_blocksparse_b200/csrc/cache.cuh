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
// the operand, its 4-bit fields (n, and n + 4 for the register's upper half) the four products n = 0 .. 3
// over channels 64 c + 16 n .. + 15.  So the codes go from memory to the tensor cores with one AND
// (n even) or a shift by 8 for two of them: a code c + 8 in the lowest bits of a half is the
// denormal (c + 8) * 2^-24, one four bits up is 16 times that, and both are exact operands.
// A code word of K holds one token, a half word of V one token: a token is written without reading its neighbours.
#pragma once
#include <cstdint>

namespace bsp {

constexpr int kGranule = 16;       // tokens
constexpr int kGroup = 32;         // channels that share a scale
__host__ __device__ constexpr int record_bytes(int D) { return 18 * D; }

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
