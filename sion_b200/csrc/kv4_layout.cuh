// Layout of the 4-bit paged cache of keys and values, shared by the kernels
// that write, read, attend over and move it.
//
// A pool is an array of pages. A page holds page_size tokens (a power of two
// >= 16) of every key/value head:
//
//   page  = [kv head][block of 16 tokens]
//   block = [K codes 16 x D/2 | V codes 16 x D/2 | K (scale, base) 16 x 2 fp16 |
//            V (scale, base) 16 x 2 fp16]                    16 * (D + 8) bytes
//
// A token's head vector x is held as x ~ base + scale * (code - 8), code in
// 0..15, one fp16 (scale, base) per token and head: 4 + 32/D bits a value.
//
// The codes stand in the order in which m16n8k16 matrix instructions take them
// from registers, so that attention loads them straight into operand order.
// A 32-bit word w holds nibbles 0..7; `w & 0x000f000f` is the fp16 pair of
// nibbles 0 and 4 as subnormals (code * 2^-24), `w & 0x00f000f0` that of
// nibbles 1 and 5 times 16, and the same of `w >> 8` gives 2, 6 and 3, 7: five
// logic operations turn eight codes into four operand registers, with no
// conversion.
//   K: token-major, natural order (even dimension in the low nibble). A lane
//      takes a quarter of a token's dimensions; the sum over dimensions may run
//      in any order, so q is permuted to match, once.
//   V: the pair in a register has to be two tokens of one dimension. With
//      token = 8h + 2t + o and dim = g * D/8 + 4w + i (i < 4), the code lies in
//      byte h*4D + g*D/2 + t*D/8 + 4w + 2o + i/2, nibble i % 2: lane (g, t) of a
//      warp reads its D/32 words of a half block as one vector, the warp 4D
//      consecutive bytes, and a byte never holds two tokens (so that tokens are
//      written one at a time without reading).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstddef>
#include <cstdint>

namespace felix_kv4 {

constexpr uint32_t kBlock = 16;        // tokens of a block
constexpr uint32_t kMaxPageSize = 4096;

__host__ __device__ constexpr uint32_t block_bytes(uint32_t D) { return kBlock * (D + 8); }
__host__ __device__ constexpr uint32_t v_codes_at(uint32_t D) { return kBlock * D / 2; }
__host__ __device__ constexpr uint32_t k_params_at(uint32_t D) { return kBlock * D; }
__host__ __device__ constexpr uint32_t v_params_at(uint32_t D) { return kBlock * D + 4 * kBlock; }

// What the kernels need of a cache. `table` [slots, width] names the pages of
// each slot, `lens` [slots] its tokens.
struct CacheView {
  unsigned char* pages;
  const int32_t* table;
  const int32_t* lens;
  uint64_t num_pages;
  size_t page_bytes;
  uint32_t slots, width, kv_heads, page_shift;  // page_size = 1 << page_shift
};

__device__ __forceinline__ int slot_length(const CacheView& c, uint32_t slot) {
  return max(c.lens[slot], 0);
}
// Tokens of a slot that its table row can name.
__device__ __forceinline__ int slot_reach(const CacheView& c, uint32_t slot) {
  const long long most = (long long)c.width << c.page_shift;
  const int n = slot_length(c, slot);
  return n > most ? int(most) : n;
}

// Address of the block of `token` (slot's position) for a head, nullptr where
// the table names no page of the pool.
__device__ __forceinline__ unsigned char* block_of(const CacheView& c, uint32_t slot, int token,
                                                   uint32_t head, uint32_t D) {
  const uint32_t at = uint32_t(token) >> c.page_shift;
  if (at >= c.width) return nullptr;
  const int page = c.table[size_t(slot) * c.width + at];
  if (page < 0 || uint64_t(page) >= c.num_pages) return nullptr;
  const uint32_t blocks = 1u << (c.page_shift - 4);
  const uint32_t in_page = (uint32_t(token) >> 4) & (blocks - 1);
  return c.pages + size_t(page) * c.page_bytes +
         (size_t(head) * blocks + in_page) * block_bytes(D);
}

}  // namespace felix_kv4
