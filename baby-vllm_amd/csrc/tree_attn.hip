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
// Work-group = (sequence, KV head, block of CB = 16·QT columns, key range). A column is
// one of the sequence's (drafted token, query head) pairs of the KV head, numbered token
// first, so the GQA group shares every key. The NW waves of a work-group hold the same
// columns and take the range's 32-key steps in turn, each with a running maximum and sum
// of its own; their states meet once, through LDS. No wave waits for another inside the
// walk: a wave's K step goes from the cache straight into MFMA operand registers (a key's
// row is a lane's operand), its V step into a private double buffer in LDS by direct
// global->LDS loads, from where transpose reads form the operand.
//   Sᵀ[32 keys × 16 cols] = K · Qᵀ,  Oᵀ[D × 16 cols] += Vᵀ · Pᵀ   (mfma 16x16x32)
// Sums, maxima and outputs are fp32 up to the final rounding. P is rounded to bf16 for its
// MFMA, and the row sum adds the rounded values, so a weight's rounding error (2^-9 on
// average) cancels where one key dominates and averages out where many do.
#include "bvllm_device.h"
#include "bvllm_abi_internal.h"

#include <algorithm>

namespace bvllm {

namespace {

constexpr int kStep = 32;  // keys per step: two 16-token pages

// Keys that a sequence's rows can see at all: written ones (seq_len), up to its last
// drafted token, inside its table.
__device__ __forceinline__ int tree_keys(const TreeArgs& a, int seq_len, int ctx, int q_len) {
  const int64_t last = min((int64_t)ctx + q_len, (int64_t)16 * a.max_blocks);
  return max(0, (int)min((int64_t)seq_len, last));
}
__device__ __forceinline__ int tree_ranges(const TreeArgs& a, int keys) {
  const int steps = (keys + kStep - 1) / kStep;
  return max(1, min(a.num_ranges, (steps + a.range_steps - 1) / a.range_steps));
}

// Bits b = 0..31: whether a row sees key k0 + b, from its mask words (bit j: position ctx + j).
__device__ __forceinline__ uint32_t seen_window(const int64_t* row, int words, int k0, int ctx, int keys) {
  const int j0 = k0 - ctx;
  uint64_t v;
  if (j0 >= 0) {
    const int w = j0 >> 6, s = j0 & 63;
    v = w < words ? (uint64_t)row[w] >> s : 0;
    if (s > 32 && w + 1 < words) v |= (uint64_t)row[w + 1] << (64 - s);
  } else if (j0 > -32) {
    v = ((uint64_t)row[0] << -j0) | ((1ull << -j0) - 1);
  } else {
    v = ~0ull;
  }
  uint32_t bits = (uint32_t)v;
  if (keys - k0 < 32) bits &= (1u << max(0, keys - k0)) - 1;
  return bits;
}

__device__ __forceinline__ bool not_finite2(uint32_t w) {
  return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
}

template <int D, int QT, int NW>
__global__ __launch_bounds__(NW * 64, 2) void tree_attn_kernel(TreeArgs a, int n_triples, int col_blocks) {
  constexpr int RB = 2 * D;        // bytes of one key row
  constexpr int TB = kStep * RB;   // bytes of one V step
  constexpr int KC = D / 32, VD = D / 16, CPR = D / 8, CB = 16 * QT;
  constexpr int RPB = 1024 / RB;   // rows of one direct load (64 lanes × 16 B)
  constexpr int NB = kStep / RPB;  // direct loads per V step
  constexpr int REC = 64 * VD * 16 + 128;  // a wave's state of one column tile: accumulators, then m and sum
  constexpr int LDS = NW * 2 * TB > NW * REC ? NW * 2 * TB : NW * REC;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[LDS];

  // Work-groups go round-robin over the 8 XCDs: the column blocks of one (sequence, KV
  // head, range) follow each other on one XCD and read its keys from one L2.
  const int id = (int)blockIdx.x >> 3;
  const int triple = id / col_blocks * 8 + ((int)blockIdx.x & 7);
  const int cb = id % col_blocks;
  if (triple >= n_triples) return;
  const int kvh = triple % a.num_kv_heads;
  const int s = triple / a.num_kv_heads % a.num_seqs;
  const int range = triple / a.num_kv_heads / a.num_seqs;

  typedef const int32_t __attribute__((address_space(4)))* ConstI32;
  const int q_start = ((ConstI32)a.query_start_loc)[s];
  const int q_len = ((ConstI32)a.query_start_loc)[s + 1] - q_start;
  const int ctx = max(0, ((ConstI32)a.context_lens)[s]);
  const int keys = tree_keys(a, ((ConstI32)a.seq_lens)[s], ctx, q_len);
  const int G = a.num_heads / a.num_kv_heads;
  const int n_cols = q_len * G;
  const int n_ranges = tree_ranges(a, keys);
  if (cb * CB >= n_cols || range >= n_ranges) return;
  const int first = range * a.range_steps;
  const int steps = (keys + kStep - 1) / kStep;
  const int last = range == n_ranges - 1 ? steps : first + a.range_steps;

  const int lane = lane_id(), n = lane & 15, g = lane >> 4;
  const int w = wave_id();

  // The columns and their Q operands (lane n + 16g: elements 32c + 8g .. +7 of column n).
  int qi[QT], hl[QT];
  bool valid[QT];
  uint4 qreg[QT][KC];
#pragma unroll
  for (int ct = 0; ct < QT; ++ct) {
    const int f = cb * CB + 16 * ct + n;
    valid[ct] = f < n_cols;
    qi[ct] = valid[ct] ? f / G : q_len - 1;
    hl[ct] = valid[ct] ? f - qi[ct] * G : 0;
    const uint16_t* row = reinterpret_cast<const uint16_t*>(a.q) + (int64_t)(q_start + qi[ct]) * a.q_st +
                          (int64_t)(kvh * G + hl[ct]) * a.q_sh;
#pragma unroll
    for (int c = 0; c < KC; ++c) qreg[ct][c] = ld16(row + 8 * (4 * c + g));
  }

  float m[QT];
  f32x4_t acc[QT][VD], lsum[QT];
#pragma unroll
  for (int ct = 0; ct < QT; ++ct) {
    m[ct] = kNegInf;
    lsum[ct] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < VD; ++c) acc[ct][c] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  const uint4 ones_bf16 = make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u);

  const unsigned char* kc = reinterpret_cast<const unsigned char*>(a.k_cache) + (int64_t)kvh * a.c_sh * 2;
  const unsigned char* vc = reinterpret_cast<const unsigned char*>(a.v_cache) + (int64_t)kvh * a.c_sh * 2;
  const uint32_t page_bytes = (uint32_t)a.c_sb * 2u;  // c_sb < 2^31, checked on the host
  const uint32_t row_bytes = (uint32_t)a.c_st * 2u;
  const ConstI32 bts = (ConstI32)(a.block_tables + (int64_t)s * a.bt_stride);

  // K: lane (n, g) holds chunks 4c + g of keys 16t + n. V: block e of a step holds its
  // rows RPB·e .. +RPB-1, lane i the 16-byte chunk at position i mod CPR of row i / CPR;
  // chunk c of a row sits at c ^ 2·(row mod CPR/2), so that the transpose reads (32 bytes of
  // 16 rows each) meet no bank twice. The swizzle of a lane is that of e's parity.
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
  auto page_at = [&](int i) __attribute__((always_inline)) -> int { return bts[min(i, a.max_blocks - 1)]; };
  // Requests a step's K (into kreg) and V (into buffer buf); its two table entries are
  // clamped into the pool.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
  auto request = [&](int p0, int p1, int buf) __attribute__((always_inline)) {
    int64_t po[2];
    po[0] = (int64_t)((uint64_t)(uint32_t)min(max(p0, 0), a.num_pages - 1) * page_bytes);
    po[1] = (int64_t)((uint64_t)(uint32_t)min(max(p1, 0), a.num_pages - 1) * page_bytes);
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

  int j = first + w;
  if (j < last) request(page_at(2 * j), page_at(2 * j + 1), 0);
  int buf = 0;
  for (; j < last; j += NW, buf ^= 1) {
    const int next0 = page_at(2 * (j + NW)), next1 = page_at(2 * (j + NW) + 1);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    f32x4_t S[QT][2];
#pragma unroll
    for (int ct = 0; ct < QT; ++ct)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        S[ct][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < KC; ++c) S[ct][t] = mfma_16x16x32(kreg[t][c], qreg[ct][c], S[ct][t]);
      }
    if (j + NW < last) request(next0, next1, buf ^ 1);

    unsigned char* const V = vbuf + buf * TB;
    const int k0 = j * kStep;
    const bool masked = k0 + kStep > ctx || k0 + kStep > keys;
    uint32_t seen[QT];
    uint32_t odd_rows = 0;  // V rows of drafted tokens that hold an infinity or NaN
    if (masked) {
#pragma unroll
      for (int ct = 0; ct < QT; ++ct) {
        seen[ct] = seen_window(a.tree_mask + (int64_t)(q_start + qi[ct]) * a.mask_stride, a.mask_words, k0, ctx, keys);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (!((seen[ct] >> (16 * t + 4 * g + i)) & 1)) S[ct][t][i] = kNegInf;
      }
      // V rows past the sequence's keys become zeros (unwritten slots may hold NaN, and
      // 0·NaN would poison the product). So must a row inside that is not finite: another
      // branch does not see it, but its P of 0 would multiply it. Those are added below.
#pragma unroll
      for (int e = 0; e < NB; ++e) {
        const int row = e * RPB + v_row;
        uint4* at = reinterpret_cast<uint4*>(V + e * 1024 + lane * 16);
        if (k0 + row >= keys) *at = make_uint4(0u, 0u, 0u, 0u);
        const uint4 x = *at;
        const uint64_t odd = __builtin_amdgcn_ballot_w64(not_finite2(x.x) || not_finite2(x.y) || not_finite2(x.z) ||
                                                         not_finite2(x.w));
        if (odd != 0) {
#pragma unroll
          for (int r = 0; r < RPB; ++r)
            if ((odd >> (r * CPR)) & ((1ull << CPR) - 1)) odd_rows |= 1u << (e * RPB + r);
        }
      }
    }

    // P = 2^(s·scale - m). The reference m is raised only when some P passes 2^8 or is not
    // a number (no key seen yet: m is -inf), so the common path has no cross-lane maximum.
    uint4 pb[QT];
#pragma unroll
    for (int ct = 0; ct < QT; ++ct) {
      float p[2][4];
      auto form = [&](float ref) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) p[t][i] = fast_exp2(__builtin_fmaf(S[ct][t][i], a.scale_log2, -ref));
      };
      form(m[ct]);
      float px = fmax_prop(fmax_prop(p[0][0], p[0][1]), p[0][2]);
      px = fmax_prop(fmax_prop(px, p[0][3]), p[1][0]);
      px = fmax_prop(fmax_prop(px, p[1][1]), p[1][2]);
      px = fmax_prop(px, p[1][3]);
      if (__builtin_amdgcn_ballot_w64(!(px <= 256.0f)) != 0) {
        float mx = fmax_prop(fmax_prop(S[ct][0][0], S[ct][0][1]), S[ct][0][2]);
        mx = fmax_prop(fmax_prop(mx, S[ct][0][3]), S[ct][1][0]);
        mx = fmax_prop(fmax_prop(mx, S[ct][1][1]), S[ct][1][2]);
        mx = max_across_groups(fmax_prop(mx, S[ct][1][3])) * a.scale_log2;
        const float m_new = fmax_prop(m[ct], mx);
        const float alpha = m_new == kNegInf ? 0.f : fast_exp2(m[ct] - m_new);
        m[ct] = m_new;
#pragma unroll
        for (int c = 0; c < VD; ++c) acc[ct][c] *= alpha;
        lsum[ct] *= alpha;
        form(m_new == kNegInf ? 0.f : m_new);
      }
      pb[ct].x = pack_bf16x2_hw(p[0][0], p[0][1]);
      pb[ct].y = pack_bf16x2_hw(p[0][2], p[0][3]);
      pb[ct].z = pack_bf16x2_hw(p[1][0], p[1][1]);
      pb[ct].w = pack_bf16x2_hw(p[1][2], p[1][3]);
    }

    while (odd_rows != 0) {  // uniform; a drafted token whose V is not finite
      const int r = __builtin_ctz(odd_rows);
      odd_rows &= odd_rows - 1;
      const int sw = 2 * (r & (CPR / 2 - 1));
      const int src = n + 16 * ((r >> 2) & 3);  // lane holding the column's P of key r
#pragma unroll
      for (int ct = 0; ct < QT; ++ct) {
        const uint32_t x0 = pb[ct].x, x1 = pb[ct].y, x2 = pb[ct].z, x3 = pb[ct].w;
        const uint32_t pair0 = (r & 2) ? x1 : x0, pair1 = (r & 2) ? x3 : x2;
        const uint32_t pw = (uint32_t)__shfl((int)((r & 16) ? pair1 : pair0), src, 64);
        const float p = (r & 1) ? hi_f32(pw) : lo_f32(pw);
        if ((seen[ct] >> r) & 1) {
#pragma unroll
          for (int c = 0; c < VD; ++c) {
            const uint2 x = ld8(V + r * RB + 16 * ((2 * c + (g >> 1)) ^ sw) + 8 * (g & 1));
            acc[ct][c][0] = __builtin_fmaf(p, lo_f32(x.x), acc[ct][c][0]);
            acc[ct][c][1] = __builtin_fmaf(p, hi_f32(x.x), acc[ct][c][1]);
            acc[ct][c][2] = __builtin_fmaf(p, lo_f32(x.y), acc[ct][c][2]);
            acc[ct][c][3] = __builtin_fmaf(p, hi_f32(x.y), acc[ct][c][3]);
          }
        }
      }
      if (lane < CPR) *reinterpret_cast<uint4*>(V + r * RB + lane * 16) = make_uint4(0u, 0u, 0u, 0u);
    }

#pragma unroll
    for (int c = 0; c < VD; ++c) {
      const uint2 lo = ld_tr16(reinterpret_cast<const uint16_t*>(V + v_off[c]));
      const uint2 hi = ld_tr16(reinterpret_cast<const uint16_t*>(V + 16 * RB + v_off[c]));
      const uint4 va = make_uint4(lo.x, lo.y, hi.x, hi.y);
#pragma unroll
      for (int ct = 0; ct < QT; ++ct) acc[ct][c] = mfma_16x16x32(va, pb[ct], acc[ct][c]);
    }
#pragma unroll
    for (int ct = 0; ct < QT; ++ct) lsum[ct] = mfma_16x16x32(ones_bf16, pb[ct], lsum[ct]);
  }

  // The waves' states meet, one column tile at a time: wave w adds dim blocks w, w + NW, ...
  // of every state, in wave order, each rescaled to the largest maximum.
#pragma unroll
  for (int ct = 0; ct < QT; ++ct) {
    __syncthreads();
    unsigned char* rec = lds + w * REC;
#pragma unroll
    for (int c = 0; c < VD; ++c) *reinterpret_cast<f32x4_t*>(rec + (c * 64 + lane) * 16) = acc[ct][c];
    if (g == 0) {
      reinterpret_cast<float*>(rec + 64 * VD * 16)[n] = m[ct];
      reinterpret_cast<float*>(rec + 64 * VD * 16)[16 + n] = lsum[ct][0];
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
    for (int c = w; c < VD; c += NW) {
      f32x4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < NW; ++k) {
        const f32x4_t x = *reinterpret_cast<const f32x4_t*>(lds + k * REC + (c * 64 + lane) * 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = __builtin_fmaf(wgt[k], x[i], o[i]);
      }
      if (!valid[ct]) continue;
      const int64_t row = q_start + qi[ct];
      const int head = kvh * G + hl[ct];
      if (n_ranges == 1) {
        const float inv = den > 0.f ? 1.f / den : den;
        st8(reinterpret_cast<uint16_t*>(a.out) + row * a.o_st + (int64_t)head * a.o_sh + 16 * c + 4 * g,
            make_uint2(pack_bf16x2_hw(o[0] * inv, o[1] * inv), pack_bf16x2_hw(o[2] * inv, o[3] * inv)));
      } else {
        const int64_t at = ((int64_t)range * a.num_tokens + row) * a.num_heads + head;
        *reinterpret_cast<f32x4_t*>(a.part_out + at * D + 16 * c + 4 * g) = o;
        if (c == 0 && g == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(M, den);
      }
    }
  }
}

// Adds the ranges of every row that has more than one, in order: one thread per 4 dims.
template <int D>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeArgs a, int blocks_per_token) {
  constexpr int TPR = D / 4;
  const int t = (int)blockIdx.x / blocks_per_token;
  const int it = ((int)blockIdx.x - t * blocks_per_token) * 256 + (int)threadIdx.x;
  // The token's sequence: the sequences that start at or before it, less one.
  int s = -1;
  for (int s0 = 0; s0 < a.num_seqs; s0 += 64) {
    const int i = s0 + lane_id();
    const bool before = i < a.num_seqs && a.query_start_loc[i] <= t;
    s += __popcll(__builtin_amdgcn_ballot_w64(before));
  }
  const int head = it / TPR, d = 4 * (it - head * TPR);
  if (s < 0 || head >= a.num_heads) return;
  s = uniform(s);
  const int q_start = a.query_start_loc[s], q_len = a.query_start_loc[s + 1] - q_start;
  if (t >= q_start + q_len) return;
  const int nr = tree_ranges(a, tree_keys(a, a.seq_lens[s], max(0, a.context_lens[s]), q_len));
  if (nr == 1) return;  // written by its work-group
  const int64_t th = (int64_t)t * a.num_heads + head, step = (int64_t)a.num_tokens * a.num_heads;
  float M = kNegInf, den = 0.f;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  for (int r = 0; r < nr; ++r) {
    const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + (th + r * step) * 2);
    const f32x4_t x = *reinterpret_cast<const f32x4_t*>(a.part_out + (th + r * step) * D + d);
    const float m_new = fmax_prop(M, ml.x);
    const float keep = M == kNegInf ? 0.f : fast_exp2(M - m_new);
    const float wgt = ml.x == kNegInf ? 0.f : fast_exp2(ml.x - m_new);
    den = den * keep + ml.y * wgt;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = __builtin_fmaf(wgt, x[i], o[i] * keep);
    M = m_new;
  }
  const float inv = den > 0.f ? 1.f / den : den;
  st8(reinterpret_cast<uint16_t*>(a.out) + (int64_t)t * a.o_st + (int64_t)head * a.o_sh + d,
      make_uint2(pack_bf16x2_hw(o[0] * inv, o[1] * inv), pack_bf16x2_hw(o[2] * inv, o[3] * inv)));
}

template <int D, int QT, int NW>
hipError_t launch_tree(const TreeArgs& a, hipStream_t stream) {
  const int64_t cols = (int64_t)a.max_query_len * (a.num_heads / a.num_kv_heads);
  const int64_t col_blocks = (cols + 16 * QT - 1) / (16 * QT);
  const int64_t triples = (int64_t)a.num_seqs * a.num_kv_heads * a.num_ranges;
  const int64_t wgs = (triples + 7) / 8 * 8 * col_blocks;
  if (wgs > 0x7ffffff0) return hipErrorInvalidValue;
  hipLaunchKernelGGL((tree_attn_kernel<D, QT, NW>), dim3((unsigned)wgs), dim3(NW * 64), 0, stream, a, (int)triples,
                     (int)col_blocks);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess || a.num_ranges == 1) return err;
  const int per_token = (a.num_heads * (D / 4) + 255) / 256;
  const int64_t blocks = (int64_t)a.num_tokens * per_token;
  if (blocks > 0x7fffffff) return hipErrorInvalidValue;
  hipLaunchKernelGGL((tree_merge_kernel<D>), dim3((unsigned)blocks), dim3(256), 0, stream, a, per_token);
  return hipGetLastError();
}

template <int D>
hipError_t tree_for_dim(const TreeArgs& a, hipStream_t stream) {
  const int64_t cols = (int64_t)a.max_query_len * (a.num_heads / a.num_kv_heads);
  if (cols <= 16) return launch_tree<D, 1, 8>(a, stream);
  return launch_tree<D, 2, 8>(a, stream);
}

}  // namespace

hipError_t paged_tree_attention(const TreeArgs& a, hipStream_t stream) {
  return a.head_dim == 64 ? tree_for_dim<64>(a, stream) : tree_for_dim<128>(a, stream);
}

// Partials hold every token of the step for every range: at most this many bytes.
constexpr int64_t kMaxTreeBytes = 64ll << 20;

int32_t tree_range_steps(const TreeArgs& a, int64_t key_steps, int64_t longest_steps) {
  const int64_t cols = (int64_t)a.max_query_len * (a.num_heads / a.num_kv_heads);
  const int64_t cb = cols <= 16 ? 16 : 32;
  const int64_t blocks = (cols + cb - 1) / cb * a.num_kv_heads;
  const int64_t table_steps = ((int64_t)a.max_blocks + 1) / 2;
  const int64_t longest = longest_steps >= 0 ? std::min(table_steps, longest_steps) : table_steps;
  const int64_t total = (key_steps >= 0 ? key_steps : longest * a.num_seqs) * blocks;
  int64_t steps = (total + device_cus() - 1) / device_cus();
  steps = std::max<int64_t>(8, (steps + 7) / 8 * 8);
  const int64_t max_ranges = kMaxTreeBytes / tree_range_bytes(1, a.num_tokens, a.num_heads, a.head_dim);
  if (max_ranges < 2) return 0;
  steps = std::max(steps, ((longest + max_ranges - 1) / max_ranges + 7) / 8 * 8);
  return steps >= longest ? 0 : (int32_t)std::min<int64_t>(steps, 1 << 28);
}

}  // namespace bvllm
