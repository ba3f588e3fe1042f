// The 4-bit form of a paged cache: where codes and scales lie, and what they stand for.
//   A group is 32 neighbouring entries of a head. scale = m / -8 in f16, m the group's entry of greatest magnitude (of m and -m the negative one), held to the largest f16;
//   code = round(entry / scale) + 8 held to 0 .. 15, 8 where the scale is 0; the value is scale * (code - 8). m itself comes back but for the scale's rounding, entries
//   near -m are held to 7/8 of it. A group with an entry that is no finite number has a NaN for its scale (0x7fff) and codes of 8; a scale of zero is positive.
// A pool is [pages][KV heads][blocks of 16 tokens][9 * head_dim bytes]: the block's codes (16 rows of head_dim / 2 bytes), then its scales. A block is one copy whatever the page's
// length, and its order is that of the attention kernels' fragments:
//   codes of keys: a row of head_dim / 2 bytes a token; word w has entries 8 w .. 8 w + 7, the first lowest. Words that are 4 apart (one of every group: those of one lane) are
//   neighbours, a chunk;
//   codes of values: a row a pair of tokens; a word has four entries 4 n .. 4 n + 3 of the even token in its lower half and of the odd one in its upper half, so that a mask
//   leaves an entry of both as two 16-bit numbers. Words of entries 32 apart are neighbours, a chunk;
//   chunks are turned from row to row so that what a fragment reads at once lies in different banks;
//   scales: [token][group].
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
// which chunk of a token's row has words w, w + 4, ... of its key (dim 64 or 128; `w` below 4)
Q4_HD constexpr int q4_key_chunk(int dim, int token, int w) { return dim == 128 ? w ^ (token >> 1 & 3) : w ^ (token >> 1 & 2); }
// which chunk of a pair's row has entries 4 n .. 4 n + 3, 32 further on, ... of its values (`n` below 8)
Q4_HD constexpr int q4_value_chunk(int dim, int pair, int n) { return dim == 128 ? n ^ (pair & 3) * 2 : n ^ (pair & 2) * 2; }
// byte offsets in a block: entries 8 w .. 8 w + 7 of a key, entries 4 n .. 4 n + 3 of a value (16 bits), scales
Q4_HD constexpr int q4_key(int dim, int token, int w) { return token * (dim / 2) + (q4_key_chunk(dim, token, w & 3) * (dim / Q4_GROUP) + (w >> 2)) * 4; }
Q4_HD constexpr int q4_value(int dim, int token, int n) {
    return (token >> 1) * dim + (q4_value_chunk(dim, token >> 1, n & 7) * (dim / Q4_GROUP) + (n >> 3)) * 4 + (token & 1) * 2;
}
Q4_HD constexpr int q4_scale(int dim, int token, int group) { return 8 * dim + (token * (dim / Q4_GROUP) + group) * 2; }

}  // namespace b2
