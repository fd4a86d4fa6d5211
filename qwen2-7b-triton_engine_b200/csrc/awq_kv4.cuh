// awq_kv4.cuh -- layout of the paged 4-bit key/value cache.
//
// cache[num_pages][kv_heads][page_size / 16] blocks of 16 tokens, block_bytes() each:
//   K codes   16 tokens x D/8 words.  With w = min(D/32, 4), word
//             (j / w) * 4w + t * w + j % w (t < 4) of a token holds channels
//             8 (4j + t) + p in nibble p: thread t of a quad of lanes reads its w words as
//             one vector and finds in word j an octet of channels [32 j, 32 j + 32).
//   V codes   8 token pairs x D/4 words.  Word (i / w) * 8w + h * w + i % w (h < 8) of a
//             pair holds channels 4 (8i + h) + p in nibbles p (even token) and 4 + p (odd
//             token): one AND of the word gives the half2 (even, odd) of a channel.
//   K params  16 tokens x D/group half2 (scale, minimum)
//   V params  the same
// value = code * scale + minimum.  One (page, head) is contiguous, and so is every run of
// its blocks, so a tile of 16 n tokens is one bulk copy.  Both layouts are the A operands
// of mma.m16n8k16 as they lie in memory: a masked word (c & 0x000F000F, c & 0x00F000F0) is
// a half2 of fp16 subnormals c * 2^-24 and c * 2^-20, exact, with no conversion.
#pragma once

#include <cuda_fp16.h>
#include <stdint.h>

namespace awq {
namespace kv4 {

constexpr int kBlockTokens = 16;

__host__ __device__ constexpr int block_bytes(int D, int group) {
  return 16 * D + 128 * (D / group);
}
__host__ __device__ constexpr int vec_words(int D) { return D / 32 < 4 ? D / 32 : 4; }
// word of octet o of a token's K row
__host__ __device__ constexpr int k_word(int D, int o) {
  const int w = vec_words(D), j = o / 4, t = o % 4;
  return (j / w) * 4 * w + t * w + j % w;
}
// word of quad c of a token pair's V row
__host__ __device__ constexpr int v_word(int D, int c) {
  const int w = vec_words(D), i = c / 8, h = c % 8;
  return (i / w) * 8 * w + h * w + i % w;
}
// byte offsets inside a block
__host__ __device__ constexpr int off_v(int D) { return 8 * D; }
__host__ __device__ constexpr int off_kp(int D) { return 16 * D; }
__host__ __device__ constexpr int off_vp(int D, int group) { return 16 * D + 64 * (D / group); }

}  // namespace kv4
}  // namespace awq
