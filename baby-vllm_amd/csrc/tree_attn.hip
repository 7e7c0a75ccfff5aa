// Attention of drafted token trees over the paged cache: the drafted tokens of every
// sequence are verified in one step, each attending the sequence's cached context and
// its own branch.
//
// For row i of a sequence with context length ctx and drafted tokens at positions
// ctx + j:
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale·q_i·k_j - m_i)
// over the keys that row i sees: every position below ctx, and ctx + j where bit j of
// the row's mask words is set. A row that sees no key gives zeros.
//
// Short contexts take one launch over all keys (tree_attn_kernel). Long ones are cut: below the
// context length every row sees every key, so work-groups of the prefill kernel walk
// whole 64-key tiles without a mask, in ranges (paged_prefill.hip, CTX); on the same launch waves
// of their own take the rest, at most 63 context keys and the drafted ones, with the
// masks (the tail); all leave fp32 partials that a second launch adds. (The tail on the second
// launch, which then added the partials to its own walk, took 109 us for 16 trees of 64 tokens where
// the tail beside the ranges took 91, and 30 for 8 trees of 11 to 45 where it took 26; with what was
// changed since these are 81 and 22.5.)
//
// What bounds it: 48 chains of 2 to 7 tokens behind 200 to 4000 read 125 MB of keys in 35 us
// (3.6 TB/s) and 4 more on the second launch; 16 trees of 64 behind 1000 to 8000 multiply at 0.6
// PFLOP/s in 80 us (their 448 columns fill 3.5 of 4 blocks, and ranges are uneven); a few trees
// are bound by the chain of a range's round trips and tiles, and by the second launch (4.4 us).
//
// The walk with masks (tree_attn.h, tree_columns): a column is one of the sequence's (drafted token,
// query head) pairs of the KV head, numbered token first, so the GQA group shares every key.
// A wave holds 16 columns and takes 32-key steps. On the launch over all keys a work-group is
// (sequence, KV head, 16 columns, DS-th of the head's dims); its NW waves hold the same columns and
// take steps in turn, each with a running maximum and sum of its own, and their states
// meet once, through LDS. No wave waits for another inside the walk: a wave's K step goes from the
// cache straight into MFMA operand registers (a key's row is a lane's operand), its V step
// into a private double buffer in LDS by direct global->LDS loads, from where transpose reads
// form the operand.
//   S^T[32 keys x 16 cols] = K Q^T,  O^T[D/DS x 16 cols] += V^T P^T   (mfma 16x16x32)
// A walk of a few steps is a chain of round trips (metadata, table, keys, states), so waves
// are spent until the card is full (tree_shape): one tree of 8 behind 300 takes 5.3 us on 16 waves
// per 16 columns.
// Sums, maxima and outputs are fp32 up to the final rounding. In the walk with masks P meets its
// MFMA as two bf16 halves, 16 bits (one tree of 8 behind 300: 5.45 us with 8 bits, 5.57 with 16, and
// 1.25 times the output error of fp32 weights with 8, the same with 16). Over the context's whole
// tiles P is rounded to bf16 as in the prefill, and the row sum adds the rounded values, so a
// weight's error (at most 2^-8) cancels where one key dominates and averages out where many do: the
// output's error is 1.4 times that of fp32 weights, as large as its own rounding. A second half there
// takes the two launches of 48 chains from 32.0 to 33.5 us, of 8 trees from 23.8 to 25.2, of a tree behind 32,000
// from 33.2 to 38.2, of 16 trees of 64 from 80 to 105.
#include "bvllm_device.h"
#include "bvllm_abi_internal.h"
#include "tree_attn.h"

#include <algorithm>
#include <cmath>

namespace bvllm {

namespace {

template <int D, int DS, int NW>
__global__ __launch_bounds__(NW * 64, D == 128 && DS == 1 ? 2 : 3) void tree_attn_kernel(TreeArgs a, int n_pairs) {
  constexpr int DV = D / DS;
  constexpr int WALK = NW * 4 * kTreeStep * DV, MEET = NW * (16 * 4 * DV + 128);  // V buffers; the waves' states
  __shared__ __attribute__((aligned(1024))) unsigned char lds[WALK > MEET ? WALK : MEET];
  // Work-groups go round-robin over the 8 XCDs in the order of their number, x first: the
  // slices and column tiles (y) of one (sequence, KV head) follow each other on one XCD and
  // read its keys from one L2.
  const int pair = (int)blockIdx.z * 8 + (int)blockIdx.x;
  if (pair >= n_pairs) return;
  const int s = a.by_kv_heads(pair);
  tree_columns<D, DS, NW, false>(a, lds, wave_id(), s, pair - s * a.num_kv_heads, (int)blockIdx.y / DS * 16,
                                 (int)blockIdx.y % DS * DV);
}

// Adds the partials of every (token, head) of the sequences that have some: the ranges of its context
// and the tail's, out = sum_r 2^(m_r - M) o_r / sum_r 2^(m_r - M) l_r, in order, M the largest
// m_r, kept online over batches of kMergeBatch partials. One thread per 4 dims. Bound by its two
// round trips, and by the partials' bytes where there are many.
constexpr int kMergeBatch = 8;

template <int D>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeArgs a, int chunks) {
  constexpr int TPR = D / 4;  // threads per (token, head)
  const int s = (int)blockIdx.x / chunks;
  typedef ConstTreeI32 ConstI32;
  int q_start = ((ConstI32)a.query_start_loc)[s], q_end = ((ConstI32)a.query_start_loc)[s + 1];
  int ctx = ((ConstI32)a.context_lens)[s], seq_len = ((ConstI32)a.seq_lens)[s];
  asm volatile("" : "+s"(q_start), "+s"(q_end), "+s"(ctx), "+s"(seq_len));
  const int it = ((int)blockIdx.x - s * chunks) * 256 + (int)threadIdx.x;
  const int th = it / TPR, d = 4 * (it % TPR);  // th: (token of the sequence, head)
  if (th >= (q_end - q_start) * a.num_heads) return;
  const int tiles = context_tiles(ctx, seq_len, a.max_blocks);
  if (tiles == 0) return;  // the tail wrote the output
  const int n = ContextRanges(tiles, a.split_tiles, a.num_ranges).count + 1;
  const int64_t at = (int64_t)q_start * a.num_heads + th, step = (int64_t)a.num_tokens * a.num_heads;
  const float* const ml = a.part_ml + at * 2;
  const float* const po = a.part_out + at * D + d;
  float M = kNegInf, den = 0.f;
  f32x4_t num = {0.f, 0.f, 0.f, 0.f};
  for (int r0 = 0; r0 < n; r0 += kMergeBatch) {
    float2 x[kMergeBatch];
    f32x4_t o[kMergeBatch];
#pragma unroll
    for (int k = 0; k < kMergeBatch; ++k) {
      x[k] = make_float2(kNegInf, 0.f);
      o[k] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      if (r0 + k >= n) continue;  // uniform
      x[k] = *reinterpret_cast<const float2*>(ml + (r0 + k) * step * 2);
      o[k] = *reinterpret_cast<const f32x4_t*>(po + (r0 + k) * step * D);
    }
    float m_new = M;
#pragma unroll
    for (int k = 0; k < kMergeBatch; ++k) m_new = fmax_prop(m_new, x[k].x);
    const float keep = M == kNegInf ? 0.f : fast_exp2(M - m_new);
    M = m_new;
    num *= keep;
    den *= keep;
#pragma unroll
    for (int k = 0; k < kMergeBatch; ++k) {
      const float add = x[k].x == kNegInf ? 0.f : fast_exp2(x[k].x - M);
      den = __builtin_fmaf(x[k].y, add, den);
#pragma unroll
      for (int i = 0; i < 4; ++i) num[i] = __builtin_fmaf(o[k][i], add, num[i]);
    }
  }
  const float inv = den > 0.f ? 1.f / den : den;  // (0 without a visible key; a NaN stays)
  const int tok = a.by_heads(th);
  st8(reinterpret_cast<uint16_t*>(a.out) + (int64_t)(q_start + tok) * a.o_st + (int64_t)(th - tok * a.num_heads) * a.o_sh + d,
      make_uint2(pack_bf16x2_hw(num[0] * inv, num[1] * inv), pack_bf16x2_hw(num[2] * inv, num[3] * inv)));
}

template <int D, int DS, int NW>
hipError_t launch_tree(const TreeArgs& a, hipStream_t stream) {
  const int64_t col_tiles = ((int64_t)a.max_query_len * (a.num_heads / a.num_kv_heads) + 15) / 16;
  const int64_t pairs = (int64_t)a.num_seqs * a.num_kv_heads;
  if (col_tiles * DS > 65535 || (pairs + 7) / 8 > 65535) return hipErrorInvalidValue;
  hipLaunchKernelGGL((tree_attn_kernel<D, DS, NW>), dim3(8, (unsigned)(col_tiles * DS), (unsigned)((pairs + 7) / 8)),
                     dim3(NW * 64), 0, stream, a, (int)pairs);
  return hipGetLastError();
}

hipError_t launch_context_part(const TreeArgs& a, hipStream_t stream) {
  PrefillArgs p{};
  p.q = a.q; p.q_st = a.q_st; p.q_sh = a.q_sh;
  p.k_cache = a.k_cache; p.v_cache = a.v_cache;
  p.c_sb = a.c_sb; p.c_st = a.c_st; p.c_sh = a.c_sh;
  p.num_pages = a.num_pages;
  p.block_tables = a.block_tables; p.bt_stride = a.bt_stride; p.max_blocks = a.max_blocks;
  p.query_start_loc = a.query_start_loc; p.seq_lens = a.seq_lens; p.context_lens = a.context_lens;
  p.scale_log2 = a.scale_log2;
  p.num_seqs = a.num_seqs; p.num_tokens = a.num_tokens; p.max_query_len = a.max_query_len;
  p.num_heads = a.num_heads; p.num_kv_heads = a.num_kv_heads; p.head_dim = a.head_dim;
  p.split_tiles = a.split_tiles; p.num_ranges = a.num_ranges;
  p.part_out = a.part_out; p.part_ml = a.part_ml;
  return paged_prefill_context(p, a, stream);
}

// Slices and key waves of a 16-column tile on the launch over all keys, by the waves that each could
// have at two per SIMD of the whole card. Measured, us, n tokens a tree (7 / 2 heads of 64 and 28 / 4
// of 128), trees behind c; beside the chosen form those next to it:
//   D = 128, n = 9, c = 600: 64 waves (2 trees): <2,4> 10.6, <1,4> 11.7; 16 (8): 11.0, 12.0; 14 (9): 16.3, <1,4> 11.9,
//     <1,2> 15.4; 9 (14): <1,4> 12.4, <1,2> 15.7; 6.4 (20): 20.0, <1,2> 19.8, <1,1> 26.3; 4.3 (30): 21.1, 20.9, 27.1; 3.2
//     (40): 26.8, 26.7, 28.9
//   c = 250: 9 (14): <1,4> 9.3, <1,2> 10.1; 3.6 (36): 18.3, 15.3, <1,1> 15.7; n = 20, c = 300: 2.8 (20): 18.2, 15.7, 16.9;
//     2.4 (24): 21.7, 19.2, 18.0; 1.9 (30): 25.6, 24.1, 21.9
//   D = 64, n = 9, c = 600: 256 (1): <2,8> 7.4, <1,4> 8.2; 16 (16): 7.8, 8.7; 15 (17): 10.6, 8.7, <1,2> 11.4; 4.0 (64):
//     <1,4> 11.7, <1,2> 14.5; 3.6 (72): 15.8, 15.3, <1,1> 18.7; 2.0 (128): 20.1, 18.5, 20.7
//   n = 20, c = 300: 5.7 (20): <1,4> 8.5, <1,2> 9.2; 3.8 (30): 10.4, 9.7, <1,1> 11.2; 2.0 (56): 12.4, 11.5, 12.0;
//     1.8 (64): <1,2> 14.4, <1,1> 13.9; 1.2 (96): 17.5, 15.6
struct TreeShape {
  int slices, key_waves;
};
TreeShape tree_shape(const TreeArgs& a) {
  const int64_t tiles = ((int64_t)a.max_query_len * (a.num_heads / a.num_kv_heads) + 15) / 16;
  const int64_t waves = 8 * (int64_t)device_cus() / (a.num_seqs * tiles * a.num_kv_heads);
  const bool d64 = a.head_dim == 64;
  if (waves >= 16) return {2, d64 ? 8 : 4};
  if (waves >= (d64 ? 4 : 8)) return {1, 4};
  return {1, waves >= 2 ? 2 : 1};
}

template <int D>
hipError_t tree_for_dim(const TreeArgs& a, hipStream_t stream) {
  if (a.split_tiles > 0) {
    const int64_t chunks = ((int64_t)a.max_query_len * a.num_heads * (D / 4) + 255) / 256;
    if (chunks * a.num_seqs > 0x7fffffff || chunks * 256 > 0x7fffffff) return hipErrorInvalidValue;
    const hipError_t err = launch_context_part(a, stream);
    if (err != hipSuccess) return err;
    hipLaunchKernelGGL((tree_merge_kernel<D>), dim3((unsigned)(chunks * a.num_seqs)), dim3(256), 0, stream, a, (int)chunks);
    return hipGetLastError();
  }
  const TreeShape shape = tree_shape(a);
  if (shape.slices == 2) return launch_tree<D, 2, D == 64 ? 8 : 4>(a, stream);
  if (shape.key_waves == 4) return launch_tree<D, 1, 4>(a, stream);
  if (shape.key_waves == 2) return launch_tree<D, 1, 2>(a, stream);
  return launch_tree<D, 1, 1>(a, stream);
}

}  // namespace

hipError_t paged_tree_attention(const TreeArgs& args, hipStream_t stream) {
  TreeArgs a = args;
  a.by_kv_heads = fast_div(a.num_kv_heads);
  a.by_group = fast_div(a.num_heads / a.num_kv_heads);
  a.by_heads = fast_div(a.num_heads);
  return a.head_dim == 64 ? tree_for_dim<64>(a, stream) : tree_for_dim<128>(a, stream);
}

// Partials hold every token of the step for every range: at most this many bytes.
constexpr int64_t kMaxTreeBytes = 64ll << 20;

// Whether the context runs in ranges, their length and their blocks (negative: of 64 columns). Times in
// us as measured here, 1 to 48 sequences of up to 32 thousand tokens and 160 drafted ones:
//   one launch: 4.3 + 1.35 per 32-key step of a wave on the longest row, but at least 2.3 per
//     thousand steps of all waves;
//   two: 10.7 (11.8 at D = 64) + 0.4 per tile of a range in blocks of 64 columns (0.69 with more
//     than one work-group per CU), 0.7 and 1.9 of 128, + 0.17 per range of the longest row, + 7.1
//     per thousand 16-column tiles, the tail's.
// Blocks of 64 columns, whose waves share a tile's keys, walk a tile in half the time where
// work-groups are few and leave fewer columns empty (a tree of 25 behind 32,000, ranges of 16 tiles: 34.8 us, with
// 128 columns 37.3); they read the keys twice as often, which counts once there are more than 20
// 128-column tiles per CU (56 at D = 64): 26 trees of up to 53 behind 2100 to 6400 take 59.0 in ranges of 16, 53.9
// with 128 columns in ranges of 20.
// The range is as short as 1.63 work-groups per CU allow (1.8 of 128 columns; sequences end ranges
// early: half of one each), and not so short that adding partials outweighs the walk (a root of the
// longest row's tiles). Where that is more than 16 tiles (20), and more than a 10th (6th) of the longest
// row, it is cut shorter: long ranges leave CUs idle behind the last ones (the same 26: 100.9 us at
// 84 tiles, 53.9 at 20). Over 200 random steps the choice was 2.0% above the best of one launch and up to
// 22 ranges of either block on average, 15% at most; over 30 of 64 to 200 sequences, which it was not
// fitted to, 2.7% and 15%.
int32_t tree_split_tiles(const TreeArgs& a, int64_t key_tiles, int64_t longest_tiles) {
  const bool d64 = a.head_dim == 64;
  const int64_t cols = (int64_t)a.max_query_len * (a.num_heads / a.num_kv_heads);
  const int64_t table_tiles = ((int64_t)a.max_blocks + 3) / 4;
  const double longest = (double)(longest_tiles >= 0 ? std::min(table_tiles, longest_tiles) : table_tiles);
  const double total = key_tiles >= 0 ? (double)key_tiles : longest * a.num_seqs;
  const double max_ranges =
      (double)(kMaxTreeBytes / (prefill_range_floats(1, a.num_tokens, a.num_heads, a.head_dim) * 4) - 1);
  if (max_ranges < 1 || longest < 2) return 0;
  const double cus = device_cus();
  const bool narrow = cols <= 64 || total * (double)((cols + 127) / 128 * a.num_kv_heads) <= (d64 ? 56 : 20) * cus;
  const int64_t cb = narrow ? 64 : 128;
  const double blocks = (double)((cols + cb - 1) / cb * a.num_kv_heads);
  const double work = total * blocks, units = a.num_seqs * blocks, target = (narrow ? 1.63 : 1.8) * cus;
  const double rounds = 1.0 + std::floor(units / target);
  double range = std::max(work / (rounds * target - units / 2), std::sqrt((narrow ? 0.43 : 0.26) * longest));
  range = std::max(range, narrow ? 4.0 : 3.0);
  range = std::min(range, narrow ? std::max(16.0, longest / 10) : std::max(20.0, longest / 6.4));
  range = std::min({std::ceil(std::max(range, longest / max_ranges)), longest, (double)(1 << 20)});

  const TreeShape shape = tree_shape(a);
  const double col_tiles = (double)((cols + 15) / 16) * a.num_kv_heads;
  const double one = 4.3 + std::max(1.35 * std::ceil(2 * longest / shape.key_waves),
                                    1.13 * col_tiles * shape.slices * 2 * total / 1000);
  const double wgs = work / range + units / 2, alone = narrow ? 0.4 : 0.7, shared = narrow ? 0.69 : 1.9;
  const double two = (d64 ? 11.8 : 10.7) + (wgs < cus ? alone : shared) * range * std::max(1.0, wgs / (2 * cus)) +
                     0.17 * longest / range + 7.1 * a.num_seqs * col_tiles / 1000;
  return one <= two ? 0 : narrow ? -(int32_t)range : (int32_t)range;
}

}  // namespace bvllm
