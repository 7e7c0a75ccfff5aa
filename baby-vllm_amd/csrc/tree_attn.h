// The waves that walk a draft tree step's keys with masks (of tree_attn.hip, where the whole is
// described, and beside the context's work-groups in paged_prefill.hip), how a sequence's keys are
// divided between the two, and what a row sees.
#pragma once

#include "bvllm_abi_internal.h"
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

// Wave-wide: exclusive prefix sum, and the sum in `all`. Within the rows of 16 lanes, then the last
// lane of a row into the next, and of the first two rows into the others (ds_permutes instead took the
// step of a tree behind 32,000 from 32.7 to 33.9 us).
__device__ __forceinline__ int row_prefix(int mine, int& all) {
  int upto = mine;
  upto += __builtin_amdgcn_update_dpp(0, upto, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8
  upto += __builtin_amdgcn_update_dpp(0, upto, 0x112, 0xf, 0xf, false);
  upto += __builtin_amdgcn_update_dpp(0, upto, 0x114, 0xf, 0xf, false);
  upto += __builtin_amdgcn_update_dpp(0, upto, 0x118, 0xf, 0xf, false);
  upto += __builtin_amdgcn_update_dpp(0, upto, 0x142, 0xa, 0xf, false);  // row_bcast 15, 31
  upto += __builtin_amdgcn_update_dpp(0, upto, 0x143, 0xc, 0xf, false);
  all = __builtin_amdgcn_readlane(upto, 63);
  return upto - mine;
}

// Numbers below n that are x modulo 8.
__device__ __forceinline__ int congruent_below(int n, int x) { return (n + 7 - x) >> 3; }

// What the slot-th work-group of an XCD takes of the context. Teams are the work-groups of one
// (sequence, range, KV head), one per block of columns: numbered in that order, team t runs on
// XCD t mod 8, so that its blocks read their keys from one L2 and every sequence loads all XCDs.
// Only work there is has a number: the grid is larger, and work-groups without any, between the
// others, would hold them up, since each takes its LDS and two round trips before it ends (35
// sequences of 500 to 5000 with up to 64 tokens, 416 work-groups with work among 2304: 94 us, 62 with
// this numbering). seq < 0: the slot lies behind them, and slot is its number there. Sequences are looked at
// 64 at a time, a lane each.
struct ContextUnit {
  int seq = -1, kv_head, block, range, first_tile, tiles;
  int q_start, q_end, seq_len, ctx;
  __device__ __forceinline__ ContextUnit(const TreeArgs& a, int width, int xcd, int& slot) {
    const int group = a.num_heads / a.num_kv_heads;
    int teams = 0;
    for (int s0 = 0; s0 < a.num_seqs; s0 += 64) {
      const int i = min(s0 + lane_id(), a.num_seqs - 1);
      const int q0 = a.query_start_loc[i], q1 = a.query_start_loc[i + 1];
      const int c = a.context_lens[i], len = a.seq_lens[i];
      const int n_blocks = s0 + lane_id() < a.num_seqs ? max(0, ((q1 - q0) * group + width - 1) / width) : 0;
      const int all_tiles = context_tiles(c, len, a.max_blocks);
      const ContextRanges ranges(all_tiles, a.split_tiles, a.num_ranges);
      const int t = n_blocks > 0 && all_tiles > 0 ? ranges.count * a.num_kv_heads : 0;
      int all, all_slots;
      const int before = teams + row_prefix(t, all);
      const int slots = (congruent_below(before + t, xcd) - congruent_below(before, xcd)) * n_blocks;
      const int first = row_prefix(slots, all_slots);
      if (slot < all_slots) {
        const int l = (int)__builtin_ctzll(__builtin_amdgcn_ballot_w64(slot >= first && slot < first + slots));
        seq = s0 + l;
        const int b = __builtin_amdgcn_readlane(n_blocks, l), at = slot - __builtin_amdgcn_readlane(first, l);
        const int team0 = __builtin_amdgcn_readlane(before, l), k = at / b;
        block = at - k * b;
        const int in_seq = ((xcd - team0) & 7) + 8 * k;
        range = in_seq / a.num_kv_heads;
        kv_head = in_seq - range * a.num_kv_heads;
        first_tile = range * __builtin_amdgcn_readlane(ranges.per, l);
        tiles = min(__builtin_amdgcn_readlane(ranges.per, l), __builtin_amdgcn_readlane(all_tiles, l) - first_tile);
        q_start = __builtin_amdgcn_readlane(q0, l);
        q_end = __builtin_amdgcn_readlane(q1, l);
        seq_len = __builtin_amdgcn_readlane(len, l);
        ctx = __builtin_amdgcn_readlane(c, l);
        return;
      }
      slot -= all_slots;
      teams += all;
    }
  }
};

// The same for the tails, behind them: teams are the work-groups of one (sequence, KV head), each of
// `width` columns.
struct TailUnit {
  int seq = -1, kv_head, group;
  __device__ __forceinline__ TailUnit(const TreeArgs& a, int width, int xcd, int& slot) {
    for (int s0 = 0; s0 < a.num_seqs; s0 += 64) {
      const int i = min(s0 + lane_id(), a.num_seqs - 1);
      const int cols = (a.query_start_loc[i + 1] - a.query_start_loc[i]) * (a.num_heads / a.num_kv_heads);
      const int groups = s0 + lane_id() < a.num_seqs ? max(0, (cols + width - 1) / width) : 0;
      const int before = i * a.num_kv_heads;
      const int slots = (congruent_below(before + a.num_kv_heads, xcd) - congruent_below(before, xcd)) * groups;
      int all_slots;
      const int first = row_prefix(slots, all_slots);
      if (slot < all_slots) {
        const int l = (int)__builtin_ctzll(__builtin_amdgcn_ballot_w64(slot >= first && slot < first + slots));
        seq = s0 + l;
        const int g = __builtin_amdgcn_readlane(groups, l), at = slot - __builtin_amdgcn_readlane(first, l), k = at / g;
        group = at - k * g;
        kv_head = ((xcd - seq * a.num_kv_heads) & 7) + 8 * k;
        return;
      }
      slot -= all_slots;
    }
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

constexpr int kTreeStep = 32;  // keys per step of a walk: two 16-token pages

typedef const int32_t __attribute__((address_space(4)))* ConstTreeI32;

__device__ __forceinline__ bool not_finite2(uint32_t w) {
  return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
}

// Rows of a 32-key V tile in LDS (1 KB blocks of 64 lanes x 16 bytes) that hold an infinity
// or NaN: bit r for row r. Every lane gets them.
template <int D>
__device__ __forceinline__ uint32_t odd_rows_of(const unsigned char* tile) {
  constexpr int CPR = D / 8, RPB = 64 / CPR;
  uint32_t odd = 0;
#pragma unroll
  for (int e = 0; e < 32 / RPB; ++e) {
    const uint4 x = ld16(tile + e * 1024 + lane_id() * 16);
    const uint64_t hit = __builtin_amdgcn_ballot_w64(not_finite2(x.x) || not_finite2(x.y) || not_finite2(x.z) ||
                                                     not_finite2(x.w));
    if (hit != 0) {
#pragma unroll
      for (int r = 0; r < RPB; ++r)
        if ((hit >> (r * CPR)) & ((1ull << CPR) - 1)) odd |= 1u << (e * RPB + r);
    }
  }
  return odd;
}

// Masks that clear those rows in a lane's V operand (keys 4g + i and 16 + 4g + i).
__device__ __forceinline__ uint4 keep_mask(uint32_t odd) {
  const uint32_t o = ~odd >> (4 * (lane_id() >> 4));
  auto pair = [&](int b) { return ((o >> b) & 1 ? 0xffffu : 0u) | ((o >> (b + 1)) & 1 ? 0xffff0000u : 0u); };
  return make_uint4(pair(0), pair(2), pair(16), pair(18));
}

// Adds the drafted keys of a 32-key step whose V row is not finite to the columns that see
// them, their weights formed again from the cache: p = 2^(s·scale - m) with the final m. Taken
// only where such a row exists.
template <int D, int DV>
__device__ __forceinline__ void add_odd_keys(const unsigned char* kc, const unsigned char* vc, uint32_t page_bytes,
                                             uint32_t row_bytes, ConstTreeI32 table, int max_blocks, int num_pages, int k0,
                                             int ctx, int keys, float scale_log2, uint32_t seen,
                                             const uint4 (&q)[D / 32], float m, f32x4_t (&acc)[DV / 16]) {
  const int lane = lane_id(), g = lane >> 4;
#pragma unroll 1
  for (int r = 0; r < 32; ++r) {
    const int key = k0 + r;
    if (key < ctx || key >= keys) continue;
    const int page = min(max(table[min(key >> 4, max_blocks - 1)], 0), num_pages - 1);
    const uint64_t at = (uint64_t)page * page_bytes + (uint64_t)((key & 15) * row_bytes);
    const uint4 x = ld16(vc + at + 16 * (lane & (DV / 8 - 1)));
    if (__builtin_amdgcn_ballot_w64(not_finite2(x.x) || not_finite2(x.y) || not_finite2(x.z) || not_finite2(x.w)) == 0)
      continue;
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      const uint4 k = ld16(kc + at + 16 * (4 * c + g));
      const uint32_t kw[4] = {k.x, k.y, k.z, k.w}, qw[4] = {q[c].x, q[c].y, q[c].z, q[c].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s = __builtin_fmaf(lo_f32(kw[i]), lo_f32(qw[i]), s);
        s = __builtin_fmaf(hi_f32(kw[i]), hi_f32(qw[i]), s);
      }
    }
    const float p = fast_exp2(__builtin_fmaf(sum_across_groups(s), scale_log2, -m));
    if ((seen >> r) & 1) {
#pragma unroll
      for (int c = 0; c < DV / 16; ++c) {
        const uint2 v = ld8(vc + at + 32 * c + 8 * g);
        acc[c][0] = __builtin_fmaf(p, lo_f32(v.x), acc[c][0]);
        acc[c][1] = __builtin_fmaf(p, hi_f32(v.x), acc[c][1]);
        acc[c][2] = __builtin_fmaf(p, lo_f32(v.y), acc[c][2]);
        acc[c][3] = __builtin_fmaf(p, hi_f32(v.y), acc[c][3]);
      }
    }
  }
}

// A wave's share of 16 columns of (sequence s, KV head kvh), from column f0 on, dims d0 .. d0 + D/DS - 1:
// key steps first, first + NW, ..., with a running maximum and sum. TAIL: the keys behind the
// context's whole 64-key tiles, of one wave; its state is the sequence's last partial (its output,
// if the context has no whole tile). Else wave w of NW, all keys, whose states meet in lds.
template <int D, int DS, int NW, bool TAIL>
__device__ __forceinline__ void tree_columns(const TreeArgs& a, unsigned char* lds, int w, int s, int kvh, int f0,
                                             int d0) {
  static_assert(!TAIL || (DS == 1 && NW == 1), "a tail's columns are one wave's");
  constexpr int DV = D / DS;       // dims of the work-group's slice of V and of the output
  constexpr int RB = 2 * DV;       // bytes of one key's slice
  constexpr int TB = kTreeStep * RB;   // bytes of one V step
  constexpr int KC = D / 32, VD = DV / 16, CPR = DV / 8;
  constexpr int RPB = 1024 / RB;   // rows of one direct load (64 lanes × 16 B)
  constexpr int NB = kTreeStep / RPB;  // direct loads per V step
  constexpr int REC = 64 * VD * 16 + 128;  // a wave's state: accumulators, then m and sum

  // The sequence's metadata and, where the walk starts at key 0, the wave's first table
  // entries, requested together and waited for once: one round trip.
  typedef ConstTreeI32 ConstI32;
  const ConstI32 bts = (ConstI32)(a.block_tables + (int64_t)s * a.bt_stride);
  auto page_at = [&](int i) __attribute__((always_inline)) -> int { return bts[min(i, a.max_blocks - 1)]; };
  int q_start = ((ConstI32)a.query_start_loc)[s], q_end = ((ConstI32)a.query_start_loc)[s + 1];
  int ctx = ((ConstI32)a.context_lens)[s], seq_len = ((ConstI32)a.seq_lens)[s];
  int page0 = TAIL ? 0 : page_at(2 * w), page1 = TAIL ? 0 : page_at(2 * w + 1);
  asm volatile("" : "+s"(q_start), "+s"(q_end), "+s"(ctx), "+s"(seq_len), "+s"(page0), "+s"(page1));
  const int q_len = q_end - q_start;
  const int G = a.num_heads / a.num_kv_heads;
  const int n_cols = q_len * G;
  if (f0 >= n_cols) return;
  const int tiles = TAIL ? context_tiles(ctx, seq_len, a.max_blocks) : 0;  // of the context's work-groups
  ctx = max(0, ctx);
  const int keys = tree_keys(seq_len, ctx, q_len, a.max_blocks);
  const int last = (keys + kTreeStep - 1) / kTreeStep;
  const int first = TAIL ? 2 * tiles : w;
  if constexpr (TAIL) {
    page0 = page_at(2 * first);
    page1 = page_at(2 * first + 1);
  }

  // The column, its Q operand (lane n + 16g: elements 32c + 8g .. +7 of column n) and its
  // first mask word (trees of at most 64 nodes have no others).
  const int lane = lane_id(), n = lane & 15, g = lane >> 4;
  const bool valid = f0 + n < n_cols;
  const int f = min(f0 + n, n_cols - 1);
  const int qi = a.by_group(f), head = kvh * G + f - qi * G;
  const int64_t row = q_start + qi;
  uint4 qreg[KC];
  {
    const uint16_t* q = reinterpret_cast<const uint16_t*>(a.q) + row * a.q_st + (int64_t)head * a.q_sh;
#pragma unroll
    for (int c = 0; c < KC; ++c) qreg[c] = ld16(q + 8 * (4 * c + g));
  }
  const int64_t* const mask_row = a.tree_mask + row * a.mask_stride;
  const uint64_t word0 = (uint64_t)mask_row[0];

  const unsigned char* kc = reinterpret_cast<const unsigned char*>(a.k_cache) + (int64_t)kvh * a.c_sh * 2;
  const unsigned char* vc = reinterpret_cast<const unsigned char*>(a.v_cache) + ((int64_t)kvh * a.c_sh + d0) * 2;
  const uint32_t page_bytes = (uint32_t)a.c_sb * 2u;  // c_sb < 2^31, checked on the host
  const uint32_t row_bytes = (uint32_t)a.c_st * 2u;

  // K: lane (n, g) holds chunks 4c + g of keys 16t + n. V: block e of a step holds its
  // rows RPB·e .. +RPB-1, lane i the 16-byte chunk at position i mod CPR of row i / CPR;
  // chunk c of a row sits at c ^ 2·(row mod CPR/2), so that the transpose reads (32 bytes of
  // 16 rows each) spread over the banks. The swizzle of a lane is that of e's parity.
  const uint32_t k_off = (uint32_t)n * row_bytes + 16u * g;
  const int v_row = lane / CPR;
  uint32_t v_src[2];
#pragma unroll
  for (int p = 0; p < 2; ++p)
    v_src[p] = (uint32_t)v_row * row_bytes +
               16u * (uint32_t)((lane % CPR) ^ (2 * ((((p * RPB) & 15) + v_row) & (CPR / 2 - 1))));
  uint32_t v_off[VD];
  {
    const int tr_row = 4 * g + (n >> 2);
    const int sw = 2 * (tr_row & (CPR / 2 - 1));
#pragma unroll
    for (int c = 0; c < VD; ++c)
      v_off[c] = (uint32_t)(tr_row * RB + 16 * ((2 * c + ((n & 3) >> 1)) ^ sw) + 8 * (n & 1));
  }
  unsigned char* const vbuf = lds + w * 2 * TB;
  const uint32_t lds_wave = (uint32_t)(uintptr_t)((__attribute__((address_space(3))) unsigned char*)vbuf);

  uint4 kreg[2][KC];
  // Requests a step's K (into kreg) and V (into buffer buf); its two table entries are
  // clamped into the pool.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
  auto request = [&](int p0, int p1, int buf) __attribute__((always_inline)) {
    const uint64_t po[2] = {(uint64_t)(uint32_t)min(max(p0, 0), a.num_pages - 1) * page_bytes,
                            (uint64_t)(uint32_t)min(max(p1, 0), a.num_pages - 1) * page_bytes};
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int c = 0; c < KC; ++c) kreg[t][c] = ld16(kc + po[t] + k_off + 64 * c);
#pragma unroll
    for (int e = 0; e < NB; ++e) {
      const unsigned char* base = vc + po[(e * RPB) >> 4] + (uint64_t)(((e * RPB) & 15) * row_bytes);
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                   :
                   : "s"(lds_wave + (uint32_t)(buf * TB + e * 1024)), "v"(v_src[e & 1]), "s"(base)
                   : "memory", "m0");
    }
  };
#pragma clang diagnostic pop

  float m;
  f32x4_t acc[VD], lsum;
  const uint4 ones_bf16 = make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u);
  // The walk. A drafted token's V row that is not finite would reach the rows that do not see
  // it too, as their P of 0 times it: if some accumulator is not finite at the end, the walk is
  // repeated with such rows taken out of the products, and they are added where they are seen.
  for (bool careful = false;; careful = true) {
    if (first < last) request(page0, page1, 0);
    m = kNegInf;
    lsum = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < VD; ++c) acc[c] = f32x4_t{0.f, 0.f, 0.f, 0.f};

    bool any_odd = false;
    int buf = 0;
    for (int j = first; j < last; j += NW, buf ^= 1) {
      const int next0 = page_at(2 * (j + NW)), next1 = page_at(2 * (j + NW) + 1);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      f32x4_t S[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        S[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < KC; ++c) S[t] = mfma_16x16x32(kreg[t][c], qreg[c], S[t]);
      }
      if (j + NW < last) request(next0, next1, buf ^ 1);

      const unsigned char* const V = vbuf + buf * TB;
      const int k0 = j * kTreeStep;
      uint32_t odd = 0;  // V rows to leave out of the product
      const uint32_t not_finite = careful ? odd_rows_of<DV>(V) : 0;
      if (k0 + kTreeStep > ctx || k0 + kTreeStep > keys) {
        const uint32_t seen = seen_window(word0, mask_row, a.mask_words, k0, ctx, keys) >> (4 * g);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (!((seen >> (16 * t + i)) & 1)) S[t][i] = kNegInf;
        // Rows past the sequence's keys (unwritten slots may hold NaN, and 0·NaN would poison
        // the product).
        if (keys - k0 < 32) odd = ~0u << (keys - k0);
        if (careful) {
          // Of drafted keys only: the context's are seen by every row and stay in the product.
          const uint32_t drafted = ctx - k0 < 32 ? ~0u << max(0, ctx - k0) : 0;
          const uint32_t found = not_finite & drafted & ~odd;
          any_odd |= found != 0;
          odd |= found;
        }
      }

      // P = 2^(s·scale - m). The reference m is raised only when some P passes 2^8 or is not
      // a number (no key seen yet: m is -inf), so the common path has no cross-lane maximum.
      float p[2][4];
      auto form = [&](float ref) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) p[t][i] = fast_exp2(__builtin_fmaf(S[t][i], a.scale_log2, -ref));
      };
      form(m);
      float px = fmax_prop(fmax_prop(p[0][0], p[0][1]), p[0][2]);
      px = fmax_prop(fmax_prop(px, p[0][3]), p[1][0]);
      px = fmax_prop(fmax_prop(px, p[1][1]), p[1][2]);
      px = fmax_prop(px, p[1][3]);
      if (__builtin_amdgcn_ballot_w64(!(px <= 256.0f)) != 0) {
        float mx = fmax_prop(fmax_prop(S[0][0], S[0][1]), S[0][2]);
        mx = fmax_prop(fmax_prop(mx, S[0][3]), S[1][0]);
        mx = fmax_prop(fmax_prop(mx, S[1][1]), S[1][2]);
        mx = max_across_groups(fmax_prop(mx, S[1][3])) * a.scale_log2;
        const float m_new = fmax_prop(m, mx);
        const float alpha = m_new == kNegInf ? 0.f : fast_exp2(m - m_new);
        m = m_new;
#pragma unroll
        for (int c = 0; c < VD; ++c) acc[c] *= alpha;
        lsum *= alpha;
        form(m_new == kNegInf ? 0.f : m_new);
      }
      uint4 pb;
      pb.x = pack_bf16x2_hw(p[0][0], p[0][1]);
      pb.y = pack_bf16x2_hw(p[0][2], p[0][3]);
      pb.z = pack_bf16x2_hw(p[1][0], p[1][1]);
      pb.w = pack_bf16x2_hw(p[1][2], p[1][3]);
      // What the rounding left, as a second operand: P has 16 bits in the products.
      uint4 rest;
      rest.x = pack_bf16x2_hw(p[0][0] - lo_f32(pb.x), p[0][1] - hi_f32(pb.x));
      rest.y = pack_bf16x2_hw(p[0][2] - lo_f32(pb.y), p[0][3] - hi_f32(pb.y));
      rest.z = pack_bf16x2_hw(p[1][0] - lo_f32(pb.z), p[1][1] - hi_f32(pb.z));
      rest.w = pack_bf16x2_hw(p[1][2] - lo_f32(pb.w), p[1][3] - hi_f32(pb.w));

      const uint4 keep = keep_mask(odd), keep_rest = keep_mask(not_finite);
#pragma unroll
      for (int c = 0; c < VD; ++c) {
        const uint2 lo = ld_tr16(reinterpret_cast<const uint16_t*>(V + v_off[c]));
        const uint2 hi = ld_tr16(reinterpret_cast<const uint16_t*>(V + 16 * RB + v_off[c]));
        uint4 va = make_uint4(lo.x, lo.y, hi.x, hi.y);
        if (odd != 0) va = make_uint4(va.x & keep.x, va.y & keep.y, va.z & keep.z, va.w & keep.w);
        acc[c] = mfma_16x16x32(va, pb, acc[c]);
        // (An infinity meets P once: the rest may be 0 or below.)
        if (not_finite != 0) va = make_uint4(va.x & keep_rest.x, va.y & keep_rest.y, va.z & keep_rest.z, va.w & keep_rest.w);
        acc[c] = mfma_16x16x32(va, rest, acc[c]);
      }
      lsum = mfma_16x16x32(ones_bf16, pb, lsum);
      lsum = mfma_16x16x32(ones_bf16, rest, lsum);
    }

    if (careful) {
      if (any_odd)
#pragma unroll 1
        for (int j = first; j < last; j += NW)
          if ((j + 1) * kTreeStep > ctx)
            add_odd_keys<D, DV>(kc, vc, page_bytes, row_bytes, bts, a.max_blocks, a.num_pages, j * kTreeStep, ctx, keys,
                                a.scale_log2, seen_window(word0, mask_row, a.mask_words, j * kTreeStep, ctx, keys), qreg, m,
                                acc);
      break;
    }
    float largest = 0.f;
#pragma unroll
    for (int c = 0; c < VD; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) largest = fmax_prop(largest, fabsf(acc[c][i]));
    if (__builtin_amdgcn_ballot_w64(!(largest < __builtin_huge_valf())) == 0) break;
  }

  auto store = [&](int c, const f32x4_t& o, float den) __attribute__((always_inline)) {
    const float inv = den > 0.f ? 1.f / den : den;  // (0 without a visible key; a NaN stays)
    st8(reinterpret_cast<uint16_t*>(a.out) + row * a.o_st + (int64_t)head * a.o_sh + d0 + 16 * c + 4 * g,
        make_uint2(pack_bf16x2_hw(o[0] * inv, o[1] * inv), pack_bf16x2_hw(o[2] * inv, o[3] * inv)));
  };
  if (TAIL && tiles > 0) {  // (uniform)
    if (valid) {
      const int part = ContextRanges(tiles, a.split_tiles, a.num_ranges).count;
      const int64_t at = ((int64_t)part * a.num_tokens + row) * a.num_heads + head;
#pragma unroll
      for (int c = 0; c < VD; ++c) *reinterpret_cast<f32x4_t*>(a.part_out + at * D + 16 * c + 4 * g) = acc[c];
      if (g == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(m, lsum[0]);
    }
  } else if constexpr (NW == 1) {
    if (valid)
#pragma unroll
      for (int c = 0; c < VD; ++c) store(c, acc[c], lsum[0]);
  } else {
    // The waves' states meet: wave w adds dim blocks w, w + NW, ... of every state, in wave
    // order, each rescaled to the largest maximum.
    __syncthreads();
    unsigned char* rec = lds + w * REC;
#pragma unroll
    for (int c = 0; c < VD; ++c) *reinterpret_cast<f32x4_t*>(rec + (c * 64 + lane) * 16) = acc[c];
    if (g == 0) {
      reinterpret_cast<float*>(rec + 64 * VD * 16)[n] = m;
      reinterpret_cast<float*>(rec + 64 * VD * 16)[16 + n] = lsum[0];
    }
    __syncthreads();
    float M = kNegInf;
#pragma unroll
    for (int k = 0; k < NW; ++k) M = fmax_prop(M, reinterpret_cast<const float*>(lds + k * REC + 64 * VD * 16)[n]);
    float wgt[NW], den = 0.f;
#pragma unroll
    for (int k = 0; k < NW; ++k) {
      const float* ml = reinterpret_cast<const float*>(lds + k * REC + 64 * VD * 16);
      wgt[k] = ml[n] == kNegInf ? 0.f : fast_exp2(ml[n] - M);
      den = __builtin_fmaf(wgt[k], ml[16 + n], den);
    }
#pragma unroll
    for (int c0 = 0; c0 < VD; c0 += NW) {
      const int c = c0 + w;
      if (c >= VD || !valid) continue;
      f32x4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < NW; ++k) {
        const f32x4_t x = *reinterpret_cast<const f32x4_t*>(lds + k * REC + (c * 64 + lane) * 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = __builtin_fmaf(wgt[k], x[i], o[i]);
      }
      store(c, o, den);
    }
  }
}

}  // namespace bvllm
