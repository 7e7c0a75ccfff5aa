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
// Long contexts run on a launch of their own (paged_prefill.hip, CTX): there every row sees
// every key, so it walks whole 64-key tiles without a mask, in ranges, and leaves fp32
// partials. The kernel here takes the rest, at most 63 context keys and the drafted ones, with
// the masks, adds the partials and writes the output; short contexts it takes whole.
//
// Work-group = (sequence, KV head, 16 columns, DS-th of the head's dims). A column is one of
// the sequence's (drafted token, query head) pairs of the KV head, numbered token first, so
// the GQA group shares every key. The NW waves of a work-group hold the same columns and take
// 32-key steps (and partials) in turn, each with a running maximum and sum of its own; their
// states meet once, through LDS. No wave waits for another inside the walk: a wave's K step
// goes from the cache straight into MFMA operand registers (a key's row is a lane's operand),
// its V step into a private double buffer in LDS by direct global->LDS loads, from where
// transpose reads form the operand.
//   Sᵀ[32 keys × 16 cols] = K · Qᵀ,  Oᵀ[D/DS × 16 cols] += Vᵀ · Pᵀ   (mfma 16x16x32)
// A walk of a few steps is a chain of round trips (metadata, table, keys, states), so waves
// are spent until the card is full (tree_for_dim).
// Sums, maxima and outputs are fp32 up to the final rounding. P is rounded to bf16 for its
// MFMA, and the row sum adds the rounded values, so a weight's rounding error (at most 2^-8)
// cancels where one key dominates and averages out where many do.
#include "bvllm_device.h"
#include "bvllm_abi_internal.h"
#include "tree_attn.h"

#include <algorithm>
#include <cmath>

namespace bvllm {

namespace {

constexpr int kStep = 32;  // keys per step: two 16-token pages

typedef const int32_t __attribute__((address_space(4)))* ConstI32;

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
                                             uint32_t row_bytes, ConstI32 table, int max_blocks, int num_pages, int k0,
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

template <int D, int DS, int NW>
__global__ __launch_bounds__(NW * 64, D == 128 && DS == 1 ? 2 : 3) void tree_attn_kernel(TreeArgs a, FastDiv by_kv_heads,
                                                                            FastDiv by_group, int n_pairs) {
  constexpr int DV = D / DS;       // dims of the work-group's slice of V and of the output
  constexpr int RB = 2 * DV;       // bytes of one key's slice
  constexpr int TB = kStep * RB;   // bytes of one V step
  constexpr int KC = D / 32, VD = DV / 16, CPR = DV / 8;
  constexpr int RPB = 1024 / RB;   // rows of one direct load (64 lanes × 16 B)
  constexpr int NB = kStep / RPB;  // direct loads per V step
  constexpr int REC = 64 * VD * 16 + 128;  // a wave's state: accumulators, then m and sum
  constexpr int LDS = NW * 2 * TB > NW * REC ? NW * 2 * TB : NW * REC;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[LDS];

  // Work-groups go round-robin over the 8 XCDs in the order of their number, x first: the
  // slices and column tiles (y) of one (sequence, KV head) follow each other on one XCD and
  // read its keys from one L2.
  const int pair = (int)blockIdx.z * 8 + (int)blockIdx.x;
  if (pair >= n_pairs) return;
  const int s = by_kv_heads(pair), kvh = pair - s * a.num_kv_heads;
  const int f0 = (int)blockIdx.y / DS * 16;        // first column
  const int d0 = (int)blockIdx.y % DS * DV;        // first dim of the slice

  // The sequence's metadata and, where the walk starts at key 0, the wave's first table
  // entries, requested together and waited for once: one round trip.
  const int w = wave_id();
  const ConstI32 bts = (ConstI32)(a.block_tables + (int64_t)s * a.bt_stride);
  auto page_at = [&](int i) __attribute__((always_inline)) -> int { return bts[min(i, a.max_blocks - 1)]; };
  int q_start = ((ConstI32)a.query_start_loc)[s], q_end = ((ConstI32)a.query_start_loc)[s + 1];
  int ctx = ((ConstI32)a.context_lens)[s], seq_len = ((ConstI32)a.seq_lens)[s];
  int page0 = page_at(2 * w), page1 = page_at(2 * w + 1);
  asm volatile("" : "+s"(q_start), "+s"(q_end), "+s"(ctx), "+s"(seq_len), "+s"(page0), "+s"(page1));
  const int q_len = q_end - q_start;
  const int G = a.num_heads / a.num_kv_heads;
  const int n_cols = q_len * G;
  if (f0 >= n_cols) return;
  const int tiles = a.split_tiles > 0 ? context_tiles(ctx, seq_len, a.max_blocks) : 0;  // of the other launch
  const int n_parts = tiles > 0 ? ContextRanges(tiles, a.split_tiles, a.num_ranges).count : 0;
  ctx = max(0, ctx);
  const int keys = tree_keys(seq_len, ctx, q_len, a.max_blocks);
  const int last = (keys + kStep - 1) / kStep;
  const int first = 2 * tiles + w;
  if (tiles > 0) {
    page0 = page_at(2 * first);
    page1 = page_at(2 * first + 1);
  }

  // The column, its Q operand (lane n + 16g: elements 32c + 8g .. +7 of column n) and its
  // first mask word (trees of at most 64 nodes have no others).
  const int lane = lane_id(), n = lane & 15, g = lane >> 4;
  const bool valid = f0 + n < n_cols;
  const int f = min(f0 + n, n_cols - 1);
  const int qi = by_group(f), head = kvh * G + f - qi * G;
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
  // The walk. A V row that is not finite (a drafted token's that a row does not see) would
  // reach every row, as its P of 0 times it: if some accumulator is not finite at the end, the
  // walk is repeated with such rows taken out of the products, and they are added where they
  // are seen.
  for (bool careful = false;; careful = true) {
    if (first < last) request(page0, page1, 0);
    m = kNegInf;
    lsum = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < VD; ++c) acc[c] = f32x4_t{0.f, 0.f, 0.f, 0.f};

    // The wave's partials of the context, kBatch at a time: their loads go out together.
    constexpr int kBatch = VD >= 8 ? 1 : VD >= 4 ? 2 : 4;  // (by their registers)
    for (int r0 = w; r0 < n_parts; r0 += NW * kBatch) {
      float2 ml[kBatch];
      f32x4_t x[kBatch][VD];
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        ml[k] = make_float2(kNegInf, 0.f);
        if (r0 + k * NW >= n_parts) continue;  // uniform
        const int64_t at = ((int64_t)(r0 + k * NW) * a.num_tokens + row) * a.num_heads + head;
        ml[k] = *reinterpret_cast<const float2*>(a.part_ml + at * 2);
#pragma unroll
        for (int c = 0; c < VD; ++c) x[k][c] = *reinterpret_cast<const f32x4_t*>(a.part_out + at * D + d0 + 16 * c + 4 * g);
      }
      float m_new = m;
#pragma unroll
      for (int k = 0; k < kBatch; ++k) m_new = fmax_prop(m_new, ml[k].x);
      const float keep = m == kNegInf ? 0.f : fast_exp2(m - m_new);
      m = m_new;
      float total = lsum[0] * keep;
#pragma unroll
      for (int c = 0; c < VD; ++c) acc[c] *= keep;
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        if (r0 + k * NW >= n_parts) continue;
        const float add = ml[k].x == kNegInf ? 0.f : fast_exp2(ml[k].x - m_new);
        total = __builtin_fmaf(ml[k].y, add, total);
#pragma unroll
        for (int c = 0; c < VD; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[c][i] = __builtin_fmaf(x[k][c][i], add, acc[c][i]);
      }
      lsum = f32x4_t{total, total, total, total};
    }

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
      const int k0 = j * kStep;
      uint32_t odd = 0;  // V rows to leave out of the product
      if (k0 + kStep > ctx || k0 + kStep > keys) {
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
          const uint32_t found = odd_rows_of<DV>(V) & ~odd;
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

      const uint4 keep = keep_mask(odd);
#pragma unroll
      for (int c = 0; c < VD; ++c) {
        const uint2 lo = ld_tr16(reinterpret_cast<const uint16_t*>(V + v_off[c]));
        const uint2 hi = ld_tr16(reinterpret_cast<const uint16_t*>(V + 16 * RB + v_off[c]));
        uint4 va = make_uint4(lo.x, lo.y, hi.x, hi.y);
        if (odd != 0) va = make_uint4(va.x & keep.x, va.y & keep.y, va.z & keep.z, va.w & keep.w);
        acc[c] = mfma_16x16x32(va, pb, acc[c]);
      }
      lsum = mfma_16x16x32(ones_bf16, pb, lsum);
    }

    if (careful) {
      if (any_odd)
#pragma unroll 1
        for (int j = first; j < last; j += NW)
          if ((j + 1) * kStep > ctx)
            add_odd_keys<D, DV>(kc, vc, page_bytes, row_bytes, bts, a.max_blocks, a.num_pages, j * kStep, ctx, keys,
                                a.scale_log2, seen_window(word0, mask_row, a.mask_words, j * kStep, ctx, keys), qreg, m,
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
  if constexpr (NW == 1) {
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

template <int D, int DS, int NW>
hipError_t launch_tree(const TreeArgs& a, hipStream_t stream) {
  const int64_t col_tiles = ((int64_t)a.max_query_len * (a.num_heads / a.num_kv_heads) + 15) / 16;
  const int64_t pairs = (int64_t)a.num_seqs * a.num_kv_heads;
  if (col_tiles * DS > 65535 || (pairs + 7) / 8 > 65535) return hipErrorInvalidValue;
  hipLaunchKernelGGL((tree_attn_kernel<D, DS, NW>), dim3(8, (unsigned)(col_tiles * DS), (unsigned)((pairs + 7) / 8)),
                     dim3(NW * 64), 0, stream, a, fast_div(a.num_kv_heads), fast_div(a.num_heads / a.num_kv_heads),
                     (int)pairs);
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
  return paged_prefill_context(p, a.narrow, stream);
}

// Waves (slices times key waves) that each 16-column tile gets: what fills the card at two
// waves per SIMD.
int64_t waves_per_column_tile(const TreeArgs& a) {
  const int64_t tiles = ((int64_t)a.max_query_len * (a.num_heads / a.num_kv_heads) + 15) / 16;
  return std::min<int64_t>(16, std::max<int64_t>(1, 8 * (int64_t)device_cus() / (a.num_seqs * tiles * a.num_kv_heads)));
}

template <int D>
hipError_t tree_for_dim(const TreeArgs& a, hipStream_t stream) {
  if (a.split_tiles > 0) {
    const hipError_t err = launch_context_part(a, stream);
    if (err != hipSuccess) return err;
  }
  const int64_t waves = waves_per_column_tile(a);
  if (waves >= 16) return launch_tree<D, 2, 8>(a, stream);
  if (waves >= 8) return launch_tree<D, 2, 4>(a, stream);
  if (waves >= 4) return launch_tree<D, 1, 4>(a, stream);
  if (waves >= 2) return launch_tree<D, 1, 2>(a, stream);
  return launch_tree<D, 1, 1>(a, stream);
}

}  // namespace

hipError_t paged_tree_attention(const TreeArgs& a, hipStream_t stream) {
  return a.head_dim == 64 ? tree_for_dim<64>(a, stream) : tree_for_dim<128>(a, stream);
}

// Partials hold every token of the step for every range: at most this many bytes.
constexpr int64_t kMaxTreeBytes = 64ll << 20;

// Whether the context gets a launch of its own, its range and its blocks (negative: of 64 columns).
// Times in us as measured here, 1 to 48 sequences of up to 32 thousand tokens and 160 drafted ones:
//   one launch: 4.3 + 2.0 (1.3 at D = 64) per 32-key step of a wave on the longest row, but at
//     least 2.4 per thousand steps of all waves;
//   two: 13.2 (11.6 at D = 64) + 0.5 per tile of a range in blocks of 64 columns, 0.8 to 1.2
//     of 128 (with more than one work-group per CU), + 0.15 per partial that a 16-column
//     tile's waves add one after the other (of 16 waves).
// Blocks of 64 columns, whose waves share a tile's keys, walk a tile in half the time where
// work-groups are few and leave fewer columns empty (a tree of 25 behind 32,000: 34.4 us, with 128
// columns 38.9; 8 trees of 11 to 45: 29.3 and 32.6); they read the keys twice as often, which
// counts once there are more than 18 128-column tiles per CU (57 at D = 64): 21 trees of 5 to 18
// behind 4858: 71 and 61.
// The range is as short as about 1.5 work-groups per CU allow (sequences end ranges early: half
// of one each), and not so short that adding partials outweighs the walk (a third of the
// longest row's tiles, as a root). Where that is more than 20 tiles, and more than a 6th or 12th
// of the longest row, it is cut shorter: long ranges leave CUs idle behind the last ones (26
// sequences of 2100 to 6400 with up to 53 tokens: 118 us at 84 tiles, 69 at 28). Over 200 random
// steps the choice was 2.4% above the best of one launch and up to 22 ranges of either
// block on average, 35% at most.
int32_t tree_split_tiles(const TreeArgs& a, int64_t key_tiles, int64_t longest_tiles) {
  const bool d64 = a.head_dim == 64;
  const int64_t cols = (int64_t)a.max_query_len * (a.num_heads / a.num_kv_heads);
  const int64_t table_tiles = ((int64_t)a.max_blocks + 3) / 4;
  const double longest = (double)(longest_tiles >= 0 ? std::min(table_tiles, longest_tiles) : table_tiles);
  const double total = key_tiles >= 0 ? (double)key_tiles : longest * a.num_seqs;
  const double max_ranges =
      (double)(kMaxTreeBytes / (prefill_range_floats(1, a.num_tokens, a.num_heads, a.head_dim) * 4));
  if (max_ranges < 1 || longest < 2) return 0;
  const double cus = device_cus();
  const bool narrow = cols <= 64 || total * (double)((cols + 127) / 128 * a.num_kv_heads) <= (d64 ? 57 : 18) * cus;
  const int64_t cb = narrow ? 64 : 128;
  const double blocks = (double)((cols + cb - 1) / cb * a.num_kv_heads);
  const double work = total * blocks, units = a.num_seqs * blocks, target = (narrow ? 1.45 : 1.6) * cus;
  const double rounds = 1.0 + std::floor(units / target);
  double range = std::max({work / (rounds * target - units / 2), std::sqrt((narrow ? 0.27 : 0.33) * longest), 3.0});
  range = std::min(range, narrow ? std::max(20.0, longest / 12) : std::max(23.0, longest / 5.7));
  range = std::min({std::ceil(std::max(range, longest / max_ranges)), longest, (double)(1 << 20)});

  const double waves = (double)waves_per_column_tile(a), key_waves = waves >= 8 ? waves / 2 : waves;
  const double col_tiles = (double)((cols + 15) / 16) * a.num_kv_heads;
  const double one = 4.3 + std::max((d64 ? 1.3 : 2.0) * std::ceil(2 * longest / key_waves),
                                    1.2 * col_tiles * (waves >= 8 ? 2 : 1) * 2 * total / 1000);
  const double wgs = work / range + units / 2;
  const double two = (d64 ? 11.6 : 13.2) +
                     (narrow ? 0.5 : wgs < cus ? 0.8 : 1.2) * range * std::max(1.0, wgs / (2 * cus)) +
                     0.15 * longest / range * (16 / waves) + 2.55 * a.num_seqs * col_tiles * 3.5 / 1000;
  return one <= two ? 0 : narrow ? -(int32_t)range : (int32_t)range;
}

}  // namespace bvllm
