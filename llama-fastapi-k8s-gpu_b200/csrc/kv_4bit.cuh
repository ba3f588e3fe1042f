// The 4-bit form of a paged cache: where codes and scales lie, and what they stand for.
//   A group is 32 neighbouring entries of a head. scale = m / -8 in f16, m the group's entry of greatest magnitude (of m and -m the negative one), held to the largest f16;
//   code = round(entry / scale) + 8 held to 0 .. 15, 8 where the scale is 0; the value is scale * (code - 8). m itself comes back but for the scale's rounding, entries
//   near -m are held to 7/8 of it. A group with an entry that is no finite number has a NaN for its scale (0x7fff) and codes of 8; a scale of zero is positive.
// A pool is [pages][KV heads][blocks of 16 tokens][9 * head_dim bytes]: the block's codes (16 rows of head_dim / 2 bytes), then its scales. A block is one copy whatever the page's
// length, and its order is that of the attention kernels' fragments:
//   codes: word w of a row has entries 8 w .. 8 w + 7, the first lowest. Words that are 4 apart (those of one lane, one of every group) are neighbours, a chunk; chunks
//   are turned from row to row so that rows read together (16 keys of a key fragment, every other key of a value fragment) lie in different banks;
//   scales of keys: [token][group]; of values: [pair of tokens][group][those two, and the two 8 further on], for products over keys.
#pragma once
#include <stdint.h>

namespace b2 {

constexpr int Q4_GROUP = 32, Q4_TOKENS = 16;

#if defined(__CUDACC__)
#define Q4_HD __host__ __device__ __forceinline__
#else
#define Q4_HD inline
#endif

Q4_HD constexpr int q4_block(int dim) { return 9 * dim; }
// which chunk of a token's row has words w, w + 4, ... (dim 64 or 128; `w` below 4)
Q4_HD constexpr int q4_chunk(int dim, int token, int w) { return dim == 128 ? w ^ (token >> 1 & 3) : w ^ (token >> 1 & 2); }
// byte offsets in a block
Q4_HD constexpr int q4_word(int dim, int token, int w) { return token * (dim / 2) + (q4_chunk(dim, token, w & 3) * (dim / Q4_GROUP) + (w >> 2)) * 4; }
Q4_HD constexpr int q4_key_scale(int dim, int token, int group) { return 8 * dim + (token * (dim / Q4_GROUP) + group) * 2; }
Q4_HD constexpr int q4_value_scale(int dim, int token, int group) {
    return 8 * dim + ((token >> 1 & 3) * 4 * (dim / Q4_GROUP) + group * 4 + (token & 1) + 2 * (token >> 3)) * 2;
}

}  // namespace b2
