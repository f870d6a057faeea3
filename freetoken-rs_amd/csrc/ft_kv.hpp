// ft_kv.hpp -- the layout of a quantised key-value cache, shared by what writes,
// reads and attends over it.
//
// A cache is n_pages pages of P tokens (a multiple of 16). A page holds a block
// per key head, one after the other:
//   keys    P x D bytes  [P/16 tiles][D/16][16 tokens][16 dimensions]
//   values  P x D bytes  [P/16 tiles][D/64][4 groups][64 dimensions][4 tokens]
//   P f32 scales of the keys, P f32 scales of the values
// A wavefront's 16-byte loads of a tile of 16 tokens are each 1 KB in a run, and
// what a lane gets is an operand of a 16x16x32 matrix instruction as it stands:
// 16 dimensions of a token's key, or 4 tokens' values of 4 dimensions each (the
// token axis is the one that is summed over, and lies in a lane). Stored row by
// row, values would have to be transposed each time they are read; so a new
// token's bytes are spread once, when it is written.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ft {

constexpr int KV_TILE = 16;  // tokens of a tile

// Bytes of one head's block in a page.
__host__ __device__ __forceinline__ int64_t kv_block_bytes(int64_t page_tokens, int64_t head_dim) {
    return page_tokens * (2 * head_dim + 8);
}

// Whether the sizes are ones that the kernels take.
inline bool kv_dims_fit(int64_t page_tokens, int64_t n_heads, int64_t head_dim) {
    return (page_tokens == 16 || page_tokens == 32 || page_tokens == 64 || page_tokens == 128 || page_tokens == 256) &&
           n_heads >= 1 && n_heads <= 256 && (head_dim == 64 || head_dim == 128 || head_dim == 256);
}

// Pages whose tokens are numbered in 31 bits.
inline bool kv_pages_fit(int64_t n_pages, int64_t page_tokens) {
    return n_pages >= 1 && n_pages <= INT32_MAX / page_tokens;
}

}  // namespace ft
