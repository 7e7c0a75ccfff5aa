// What the two launches of a draft tree step share (tree_attn.hip, and the context part in
// paged_prefill.hip): how a sequence's keys are divided between them, and what a row sees.
#pragma once

#include "bvllm_device.h"

namespace bvllm {

// Whole 64-key tiles below the context length, inside the written keys and the table.
__device__ __forceinline__ int context_tiles(int ctx, int seq_len, int max_blocks) {
  return max(0, (int)min((int64_t)min(ctx, seq_len), (int64_t)16 * max_blocks)) >> 6;
}

// Their ranges: at most num_ranges, of `per` tiles each, as even as whole tiles allow (the last
// may hold fewer), and of at most split_tiles where num_ranges suffices for that.
struct ContextRanges {
  int per, count;
  __device__ __forceinline__ ContextRanges(int tiles, int split_tiles, int num_ranges) {
    const int n = max(1, min((tiles + split_tiles - 1) / split_tiles, num_ranges));
    per = max(1, (tiles + n - 1) / n);
    count = (tiles + per - 1) / per;
  }
};

// Keys that a sequence's rows can see at all: written ones (seq_len), up to its last
// drafted token, inside its table.
__device__ __forceinline__ int tree_keys(int seq_len, int ctx, int q_len, int max_blocks) {
  const int64_t last = min((int64_t)ctx + q_len, (int64_t)16 * max_blocks);
  return max(0, (int)min((int64_t)seq_len, last));
}

// Bits b = 0..31: whether a row sees key k0 + b, from its mask words (bit j: position ctx + j;
// word0 is row[0]).
__device__ __forceinline__ uint32_t seen_window(uint64_t word0, const int64_t* row, int words, int k0, int ctx,
                                                int keys) {
  const int j0 = k0 - ctx;
  uint64_t v;
  if (j0 >= 0) {
    const int w = j0 >> 6, s = j0 & 63;
    v = w == 0 ? word0 >> s : w < words ? (uint64_t)row[w] >> s : 0;
    if (s > 32 && w + 1 < words) v |= (uint64_t)row[w + 1] << (64 - s);
  } else if (j0 > -32) {
    v = (word0 << -j0) | ((1ull << -j0) - 1);
  } else {
    v = ~0ull;
  }
  uint32_t bits = (uint32_t)v;
  if (keys - k0 < 32) bits &= (1u << max(0, keys - k0)) - 1;
  return bits;
}

}  // namespace bvllm
