// What a row of a windowed step sees, and the work-groups that compute its single rows (launched
// by window_attn.hip, and behind the prefill work-groups of a step with both by paged_prefill.hip).
//
// The row at position p of its sequence (context_lens[s] + its number among the sequence's
// rows) sees key j iff j <= p, j < seq_lens[s], j lies inside the table, and j > p - window or
// j < sinks. Softmax over the visible keys as elsewhere; a row without one gives zeros.
//
// The visible pages are those of the first tokens, [0, sink_pages), and those of the window,
// [first, end): walk step k is page k, or k + skip behind the first ones. Pages between are not
// touched, whatever the table says of them.
#pragma once

#include "paged_decode_wg.h"

namespace bvllm {

// A single row's view: keys [0, sinks) and [lo, limit), on `count` pages.
struct RowView {
  int lo, sinks, limit;
  int sink_pages, skip, count;
  __device__ __forceinline__ RowView(int64_t pos, int seq_len, int max_blocks, int window, int first_tokens) {
    limit = (int)max((int64_t)0, min(min(pos + 1, (int64_t)seq_len), (int64_t)16 * max_blocks));
    lo = (int)max((int64_t)0, min(pos - window + 1, (int64_t)limit));
    sinks = min(first_tokens, lo);
    sink_pages = (sinks + 15) >> 4;
    const int first = max(lo >> 4, sink_pages);
    skip = first - sink_pages;
    count = sink_pages + max(0, ((limit + 15) >> 4) - first);
  }
  __device__ __forceinline__ int page(int k) const { return k < sink_pages ? k : k + skip; }
  __device__ __forceinline__ bool sees(int tok) const { return tok < limit && (tok >= lo || tok < sinks); }
};

// The keys that some row of a block sees (rows q_first .. q_last of a sequence), as places in the walk
// over their pages: [0, sinks) and [first_place, end), in positions [0, sinks) and from `first` pages on.
struct BlockWalk {
  int sinks, first_place, end;
  int sink_end, skip;  // place behind the first tokens' pages, pages between them and the window's
  BlockWalk() = default;
  __device__ __forceinline__ BlockWalk(int ctx, int seq_len, int max_blocks, int window, int first_tokens, int q_first,
                                       int q_last) {
    const int limit = (int)max((int64_t)0, min(min((int64_t)ctx + q_last + 1, (int64_t)seq_len), (int64_t)16 * max_blocks));
    const int lo = (int)max((int64_t)0, (int64_t)ctx + q_first - window + 1);
    const int sink_pages = (int)(((int64_t)min(first_tokens, lo) + 15) >> 4);
    sinks = first_tokens;
    sink_end = 16 * sink_pages;
    skip = max(lo >> 4, sink_pages) - sink_pages;
    first_place = place(lo);
    end = place(limit);
  }
  __device__ __forceinline__ int page(int k) const { return 16 * k < sink_end ? k : k + skip; }
  // Of a position, 0 and up; the positions of no page of the walk have the place behind the first tokens'.
  __device__ __forceinline__ int place(int pos) const { return pos <= sink_end ? pos : max(sink_end, pos - 16 * skip); }
};

// What the launches of a step's single rows take (behind prefill work-groups: those of one query).
struct WindowRows {
  DecodeArgs rows;
  int32_t window, sinks;
};

// The prefill kernel on a step of windows (paged_prefill.hip), in blocks of 128, 64 or 32 columns, with the work-groups of
// `rows` where the step has sequences of one query; ranges of a.split_tiles tiles of the walk (> 0: in blocks of 128)
// leave partials that a second launch adds.
hipError_t paged_prefill_window(const PrefillArgs& a, const WindowRows& rows, int columns, hipStream_t stream);
// The prefill work-groups of a step in blocks of so many columns.
int64_t prefill_work_groups(const PrefillArgs& a, int columns);

// ---------------------------------------------------------------- single rows
//
// One work-group of NW waves per (single-query sequence, column group, split): the row's visible
// pages are cut into a.num_splits runs of equal length (the last ones may be shorter or
// missing), and the waves of a run take its pages in turn, each with a softmax state of its
// own, as the decode work-groups do (paged_decode_wg.h). The states meet in LDS: every wave
// writes its sums of the heads there are, and each (head, 4 dims) is added up in wave order.
// The result of a run that is not the whole row is an fp32 (o, lse), added by window_merge_kernel.
// Weights meet V as two bf16 operands, 16 bits: bound by memory, the rows have room for the second product
// (64 rows of 1028 keys, 28 / 4 heads of 128: 24.0 us with one operand, 24.1 with two, in one run; error against 64 bits
// 2.10e-3 -> 1.66e-3, as fp32 weights give; one row of 260 keys at D = 64 5.15 -> 5.31).

// Runs of a row of n pages: `per` pages each, `live` of them not empty (one of an empty row).
struct Runs {
  int per, live;
  __device__ __forceinline__ Runs(int n, int splits) {
    per = max(1, (n + splits - 1) / splits);
    live = max(1, (n + per - 1) / per);
  }
};

// LDS: the waves' K transpose tiles, and in their place later the states: m and l of wave w's head n
// at 2·(16 w + n), then its D sums, rows of D + 4 floats so that the heads' rows start in other banks.
template <int D>
constexpr int kStatePitch = D + 4;
template <int D, int NW>
constexpr size_t rows_lds_bytes(int heads) {
  const size_t tiles = (size_t)NW * kTileBytes<D>, states = (size_t)4 * NW * (32 + heads * kStatePitch<D>);
  return tiles > states ? tiles : states;
}

// The walk of one row by a work-group: steps k0 .. k1 - 1, step k on page page(k), keys as `view` sees them.
// store(head, d, o, ref, L) gets, of each head of the column group, the sums of dims d .. +3 divided by L, the sum of the
// weights 2^(score - ref) (0 where no key is seen: o is 0 then).
template <int D, int NW, typename Page, typename Store>
__device__ __forceinline__ void window_row(const DecodeArgs& a, int b, int row, const ColGroup& cg, const RowView& view, int k0,
                                           int k1, Page page, unsigned char* smem, Store store) {
  constexpr int KC = D / 32, VD = D / 16;
  const int lane = lane_id(), n = lane & 15, g = lane >> 4, w = wave_id();
  // The wave's pages are steps first, first + NW, ... of the walk; lane k holds the table entry of
  // its page number base + k.
  const int first = k0 + w, cnt = first < k1 ? (k1 - first + NW - 1) / NW : 0;
  const int32_t* bt = a.block_tables + (int64_t)b * a.bt_stride;
  auto entries = [&](int base) {
    const int e = bt[min(page(first + NW * (base + lane)), a.max_blocks - 1)];
    return min(max(e, 0), a.num_pages - 1);
  };
  int ent = entries(0);

  uint4 qb[KC];
  const uint16_t* qrow = reinterpret_cast<const uint16_t*>(a.q) + (int64_t)row * a.q_sb + (int64_t)(cg.head0 + n) * a.q_sh;
#pragma unroll
  for (int c = 0; c < KC; ++c) qb[c] = n < cg.cols ? ld16(qrow + 8 * (4 * c + g)) : make_uint4(0, 0, 0, 0);

  WaveState<D> st;
  st.m = kNegInf;
  st.l = 0.f;
#pragma unroll
  for (int c = 0; c < VD; ++c) st.acc[c] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  uint32_t off[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) off[j] = (uint32_t)((4 * g + j) * a.c_st + VD * n);
  unsigned char* tile = smem + w * kTileBytes<D>;
  const uint16_t* kc = reinterpret_cast<const uint16_t*>(a.k_cache) + (int64_t)cg.kvh * a.c_sh;
  const uint16_t* vc = reinterpret_cast<const uint16_t*>(a.v_cache) + (int64_t)cg.kvh * a.c_sh;
  auto page_work = [&](const PageRegs<D>& r, int k) __attribute__((always_inline)) {
    const f32x4_t scores = register_scores<D>(r, qb, tile, n, g);
    PagePv<D> ph;
    softmax_phase_if<D, true>(st, ph, scores, r.v, 16 * page(first + NW * k) + 4 * g,
                              [&](int tok) { return view.sees(tok); }, a.scale_log2);
    rescale_phase<D>(st, ph);
    pv_phase<D, true>(st, ph);
  };

  for (int base = 0; base < cnt; base += 64) {
    const int here = min(64, cnt - base);
    if (base > 0) ent = entries(base);
    auto page_at = [&](int k) -> int64_t { return (int64_t)__builtin_amdgcn_readlane(ent, k) * a.c_sb; };
    // One page in flight, the next requested as soon as it has landed, none past the wave's last.
    PageRegs<D> r[2];
    load_page<D>(r[0], kc + page_at(0), vc + page_at(0), off);
    for (int k = 0; k < here; k += 2) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (k + i < here) {
          wait_page<0, D>(r[i]);
          if (k + i + 1 < here) {
            const int64_t p = page_at(k + i + 1);
            load_page<D>(r[i ^ 1], kc + p, vc + p, off);
          }
          page_work(r[i], base + k + i);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) wait_page<0, D>(r[i]);
  }

  // (A NaN score: the sums hold it, and the maximum below, which passes over NaN, must not see none.)
  if (st.m != st.m) st.m = 0.f;
  const float l = sum_across_groups(st.l);
  __syncthreads();  // the tiles are no longer read
  float* ml = reinterpret_cast<float*>(smem);
  float* sums = ml + 32 * NW;
  if (n < cg.cols) {
    if (g == 0) *reinterpret_cast<float2*>(ml + 2 * (16 * w + n)) = make_float2(st.m, l);
    // acc[c][i] is dim VD·(4g + i) + c.
    float* dst = sums + (w * cg.cols + n) * kStatePitch<D> + 4 * VD * g;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int c = 0; c < VD; c += 4)
        *reinterpret_cast<f32x4_t*>(dst + VD * i + c) =
            f32x4_t{st.acc[c][i], st.acc[c + 1][i], st.acc[c + 2][i], st.acc[c + 3][i]};
  }
  __syncthreads();
  for (int it = (int)threadIdx.x; it < cg.cols * (D / 4); it += NW * 64) {
    const int h = it / (D / 4), d = 4 * (it - h * (D / 4));
    float M = kNegInf;
#pragma unroll
    for (int s = 0; s < NW; ++s) M = fmaxf(M, ml[2 * (16 * s + h)]);
    const float ref = M == kNegInf ? 0.f : M;
    float L = 0.f;
    f32x4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < NW; ++s) {
      const float2 x = *reinterpret_cast<const float2*>(ml + 2 * (16 * s + h));
      const f32x4_t v = *reinterpret_cast<const f32x4_t*>(sums + (s * cg.cols + h) * kStatePitch<D> + d);
      const float wgt = fast_exp2(x.x - ref);
      L = __builtin_fmaf(x.y, wgt, L);
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = __builtin_fmaf(v[i], wgt, o[i]);
    }
    o *= L == 0.f ? 0.f : 1.f / L;
    store(cg.head0 + h, d, o, ref, L);
  }
  __syncthreads();  // (a caller's next row writes its tiles there)
}

template <int D, int NW>
__device__ __forceinline__ void window_row_group(const DecodeArgs& a, int window, int first_tokens, int wg,
                                                 unsigned char* smem) {
  const int G = a.num_heads / a.num_kv_heads;
  const int ncg = a.num_kv_heads * col_groups_per_kv(G);
  const int unit = wg / a.num_splits, split = wg - unit * a.num_splits;
  const int b = unit / ncg;
  const ColGroup cg = col_group(G, unit - b * ncg);
  const int row = uniform(a.query_start_loc[b]), row_end = uniform(a.query_start_loc[b + 1]);
  const int seq_len = uniform(a.seq_lens[b]), ctx = uniform(a.context_lens[b]);
  if (row_end - row != 1) return;
  const RowView view(ctx, seq_len, a.max_blocks, window, first_tokens);
  const Runs runs(view.count, a.num_splits);
  if (split >= runs.live) return;
  window_row<D, NW>(a, b, row, cg, view, split * runs.per, min((split + 1) * runs.per, view.count),
                    [&](int k) { return view.page(k); }, smem, [&](int head, int d, f32x4_t o, float ref, float L) {
    if (runs.live == 1) {
      st8(reinterpret_cast<uint16_t*>(a.out) + (int64_t)row * a.o_sb + (int64_t)head * a.o_sh + d,
          make_uint2(pack_bf16x2_hw(o[0], o[1]), pack_bf16x2_hw(o[2], o[3])));
    } else {
      const int64_t part = ((int64_t)b * a.num_heads + head) * a.num_splits + split;
      *reinterpret_cast<f32x4_t*>(a.part_out + part * D + d) = o;
      if (d == 0) a.part_lse[part] = L == 0.f ? kNegInf : ref + __log2f(L);
    }
  });
}

}  // namespace bvllm
