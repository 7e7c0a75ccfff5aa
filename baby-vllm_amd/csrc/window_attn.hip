// Attention of a sliding window and a few first tokens over the paged cache.
//
// The row at position p of its sequence (context_lens[s] + its number among the sequence's
// rows) sees key j iff j <= p, j < seq_lens[s], j lies inside the table, and j > p - window or
// j < sinks. Softmax over the visible keys as elsewhere; a row without one gives zeros.
//
// A row's visible pages are those of its first tokens, [0, sink_pages), and those of its
// window, [first, end): walk step k is page k, or k + skip behind the first ones. Pages between
// are not touched, whatever the table says of them.
#include "paged_decode_wg.h"

#include <algorithm>

namespace bvllm {

namespace {

// What a row sees: keys [0, sinks) and [lo, limit), on `count` pages.
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

// One work-group per (row, column group): its four waves take the row's visible pages in turn
// and merge their states in LDS, as a decode row's.
template <int D>
__global__ __launch_bounds__(256) void window_rows_kernel(DecodeArgs a, int num_rows, int window, int first_tokens) {
  constexpr int NW = 4, KC = D / 32, VD = D / 16;
  __shared__ __attribute__((aligned(16))) unsigned char smem[decode_lds_bytes<D, NW>()];
  const int G = a.num_heads / a.num_kv_heads;
  const int ncg = a.num_kv_heads * col_groups_per_kv(G);
  const int row = (int)blockIdx.x / ncg;
  const ColGroup cg = col_group(G, (int)blockIdx.x - row * ncg);
  const int lane = lane_id(), n = lane & 15, g = lane >> 4, w = wave_id();

  // The row's sequence: the last one that starts at or before it.
  int s = -1;
  for (int s0 = 0; s0 < a.batch; s0 += 64) {
    const int i = s0 + lane;
    s += __popcll(__builtin_amdgcn_ballot_w64(i < a.batch && a.query_start_loc[i] <= row));
  }
  s = uniform(s);
  if (s < 0 || row >= uniform(a.query_start_loc[s + 1])) return;
  const int64_t pos = (int64_t)uniform(a.context_lens[s]) + (row - uniform(a.query_start_loc[s]));
  const RowView view(pos, uniform(a.seq_lens[s]), a.max_blocks, window, first_tokens);

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
  const int32_t* bt = a.block_tables + (int64_t)s * a.bt_stride;

  for (int k = w; k < view.count; k += NW) {
    const int page = view.page(k);
    const int64_t p = (int64_t)min(max(uniform(bt[page]), 0), a.num_pages - 1) * a.c_sb;
    PageRegs<D> r;
    load_page<D>(r, kc + p, vc + p, off);
    wait_page<0, D>(r);
    const f32x4_t scores = register_scores<D>(r, qb, tile, n, g);
    PagePv<D> ph;
    softmax_phase_if<D>(st, ph, scores, r.v, 16 * page + 4 * g, [&](int tok) { return view.sees(tok); }, a.scale_log2);
    rescale_phase<D>(st, ph);
    pv_phase<D>(st, ph);
  }
  float* merge = reinterpret_cast<float*>(smem + NW * kTileBytes<D>);
  // (A NaN score: the sums hold it, and the merge's maximum, which passes over NaN, must not see none.)
  if (st.m != st.m) st.m = 0.f;
  save_state<D>(merge, st, w, lane);
  __syncthreads();
  merge_states<D>(a, merge, w, cg.cols, row, cg.head0, lane);
}

}  // namespace

template <int D>
static hipError_t launch_window(const WindowArgs& w, hipStream_t stream) {
  DecodeArgs a{};
  a.q = w.q; a.q_sb = w.q_st; a.q_sh = w.q_sh;
  a.k_cache = w.k_cache; a.v_cache = w.v_cache;
  a.c_sb = w.c_sb; a.c_st = w.c_st; a.c_sh = w.c_sh;
  a.num_pages = w.num_pages;
  a.block_tables = w.block_tables; a.bt_stride = w.bt_stride; a.max_blocks = w.max_blocks;
  a.seq_lens = w.seq_lens; a.query_start_loc = w.query_start_loc; a.context_lens = w.context_lens;
  a.scale_log2 = w.scale_log2;
  a.out = w.out; a.o_sb = w.o_st; a.o_sh = w.o_sh;
  a.batch = w.num_seqs; a.num_heads = w.num_heads; a.num_kv_heads = w.num_kv_heads; a.head_dim = w.head_dim;
  const int64_t wgs = (int64_t)w.num_tokens * decode_col_groups(a);
  if (wgs > 0x7fffffff) return hipErrorInvalidValue;
  hipLaunchKernelGGL((window_rows_kernel<D>), dim3((unsigned)wgs), dim3(256), 0, stream, a, w.num_tokens, w.window, w.sinks);
  return hipGetLastError();
}

int64_t window_workspace_bytes(const WindowArgs&) { return 0; }

hipError_t paged_window_attention(const WindowArgs& a, hipStream_t stream) {
  switch (a.head_dim) {
    case 64: return launch_window<64>(a, stream);
    case 128: return launch_window<128>(a, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace bvllm
