// Attention of a sliding window and a few first tokens over the paged cache: the launches of single rows
// and the sum of their runs (window_attn.h); prompts run on the prefill kernel (paged_prefill.hip).
#include "window_attn.h"

#include <algorithm>

namespace bvllm {

template <int D, int NW>
__global__ __launch_bounds__(NW * 64) void window_rows_kernel(WindowRows w) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  window_row_group<D, NW>(w.rows, w.window, w.sinks, (int)blockIdx.x, smem);
}

// Adds a row's runs: out = Σ 2^(lse_r − M)·o_r / Σ 2^(lse_r − M) in their order, one thread per 4 dims,
// kMergeBatch runs' loads at once.
constexpr int kMergeBatch = 8;

template <int D>
__global__ __launch_bounds__(256) void window_merge_kernel(WindowRows w, int per_row) {
  const DecodeArgs& a = w.rows;
  const int b = (int)blockIdx.x / per_row;
  const int it = ((int)blockIdx.x - b * per_row) * 256 + (int)threadIdx.x;
  const int row = uniform(a.query_start_loc[b]), row_end = uniform(a.query_start_loc[b + 1]);
  const int seq_len = uniform(a.seq_lens[b]), ctx = uniform(a.context_lens[b]);
  if (row_end - row != 1) return;
  const Runs runs(RowView(ctx, seq_len, a.max_blocks, w.window, w.sinks).count, a.num_splits);
  const int head = it / (D / 4), d = 4 * (it - head * (D / 4));
  if (runs.live == 1 || head >= a.num_heads) return;
  const int64_t part = ((int64_t)b * a.num_heads + head) * a.num_splits;
  float M = kNegInf, den = 0.f;
  f32x4_t num = {0.f, 0.f, 0.f, 0.f};
  for (int r0 = 0; r0 < runs.live; r0 += kMergeBatch) {
    float lse[kMergeBatch];
    f32x4_t o[kMergeBatch];
#pragma unroll
    for (int k = 0; k < kMergeBatch; ++k) {
      const int64_t p = part + min(r0 + k, runs.live - 1);
      lse[k] = a.part_lse[p];
      o[k] = *reinterpret_cast<const f32x4_t*>(a.part_out + p * D + d);
    }
    float Mb = M;
#pragma unroll
    for (int k = 0; k < kMergeBatch; ++k) Mb = fmaxf(Mb, lse[k]);
    const float ref = Mb == kNegInf ? 0.f : Mb;
    const float alpha = fast_exp2(M - ref);
    den *= alpha;
    num *= alpha;
    M = Mb;
#pragma unroll
    for (int k = 0; k < kMergeBatch; ++k) {
      const float wgt = r0 + k < runs.live ? fast_exp2(lse[k] - ref) : 0.f;
      den += wgt;
      if (r0 + k < runs.live) {
#pragma unroll
        for (int i = 0; i < 4; ++i) num[i] = __builtin_fmaf(wgt, o[k][i], num[i]);
      }
    }
  }
  const float inv = den == 0.f ? 0.f : 1.f / den;
  st8(reinterpret_cast<uint16_t*>(a.out) + (int64_t)row * a.o_sb + (int64_t)head * a.o_sh + d,
      make_uint2(pack_bf16x2_hw(num[0] * inv, num[1] * inv), pack_bf16x2_hw(num[2] * inv, num[3] * inv)));
}

// The runs of a step of single rows, work-groups of `waves` waves each. Times (us) as measured here, rows of equal length: 5
// of start, with 0.18 per page of a work-group at D = 128 (the waves of a work-group share what a CU takes: 4, 8 or 16
// of them make no difference) and 0.09 at D = 64 (0.14 on four waves), and 2.3 of the second launch. So rows are cut until
// every CU has a work-group, into runs of 8 pages at least, where that saves more than the second launch costs (one row
// of 7B, 4097 keys: 46.4 whole, 11.2 in 32 runs; 1025: 14.2 and 8.7; 257: 6.0 and 7.4. 32 rows, 1025:
// 18.6 and 18.3. 48 rows, 4097, where 64 CUs are idle: 70.3 and 76.2). Eight waves at D = 64 but for
// a few pages (64 keys: 4.5 against 4.4), and at D = 128 while half of the CUs are idle (one row, 1025
// keys: 8.7 against 9.0); else four (64 rows, 1025: 24.8 against 25.1, 96 rows: 39.4 against 41.2).
constexpr int64_t kMaxRowBytes = 64ll << 20;  // of their partials

// The pages that a row can see at most.
static int64_t max_row_pages(const WindowArgs& a) {
  return std::min<int64_t>(a.max_blocks, ((int64_t)a.window + 15) / 16 + 1 + ((int64_t)a.sinks + 15) / 16);
}
// (Row, column group) pairs of so many rows.
static int64_t row_units(const WindowArgs& a, int64_t rows) {
  const int G = a.num_heads / a.num_kv_heads;
  return std::max<int64_t>(1, rows * a.num_kv_heads * ((G + 15) / 16));
}

static int32_t runs_of_rows(const WindowArgs& a) {
  const int64_t pages = max_row_pages(a), units = row_units(a, std::min(a.num_tokens, a.num_seqs));
  const int64_t room = kMaxRowBytes / ((int64_t)a.num_seqs * a.num_heads * (a.head_dim + 1) * 4);
  const int64_t runs = std::min({device_cus() / units, pages / 8, room});
  const bool pays = runs > 1 && (a.head_dim == 128 ? 0.18 : 0.09) * (double)(pages - (pages + runs - 1) / runs) > 3.5;
  return pays ? (int32_t)runs : 1;
}

static int waves_of_rows(const WindowArgs& a, int32_t runs) {
  if (a.head_dim == 64) return max_row_pages(a) < 8 ? 4 : 8;
  return 2 * row_units(a, std::min(a.num_tokens, a.num_seqs)) * runs <= device_cus() ? 8 : 4;
}

static DecodeArgs rows_of_step(const WindowArgs& w) {
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
  return a;
}

template <int D, int NW>
static hipError_t launch_rows(const WindowRows& w, hipStream_t stream) {
  const DecodeArgs& a = w.rows;
  const int G = a.num_heads / a.num_kv_heads;
  const int64_t wgs = (int64_t)a.batch * decode_col_groups(a) * a.num_splits;
  if (wgs > 0x7fffffff) return hipErrorInvalidValue;
  static std::atomic<bool> done[64] = {};
  hipError_t err = allow_lds(&window_rows_kernel<D, NW>, done, (int)rows_lds_bytes<D, NW>(16));
  if (err != hipSuccess) return err;
  const size_t lds = rows_lds_bytes<D, NW>(std::min(G, 16));
  hipLaunchKernelGGL((window_rows_kernel<D, NW>), dim3((unsigned)wgs), dim3(NW * 64), lds, stream, w);
  return hipGetLastError();
}

static PrefillArgs blocks_of_step(const WindowArgs& w) {
  PrefillArgs a{};
  a.q = w.q; a.q_st = w.q_st; a.q_sh = w.q_sh;
  a.k_cache = w.k_cache; a.v_cache = w.v_cache;
  a.c_sb = w.c_sb; a.c_st = w.c_st; a.c_sh = w.c_sh;
  a.num_pages = w.num_pages;
  a.block_tables = w.block_tables; a.bt_stride = w.bt_stride; a.max_blocks = w.max_blocks;
  a.query_start_loc = w.query_start_loc; a.seq_lens = w.seq_lens; a.context_lens = w.context_lens;
  a.scale_log2 = w.scale_log2;
  a.out = w.out; a.o_st = w.o_st; a.o_sh = w.o_sh;
  a.num_seqs = w.num_seqs; a.num_tokens = w.num_tokens; a.max_query_len = w.max_query_len;
  a.num_heads = w.num_heads; a.num_kv_heads = w.num_kv_heads; a.head_dim = w.head_dim;
  a.single_query_seqs = w.single_query_seqs;
  return a;
}

// What a launch of the blocks takes (us), fitted to 9,232 random steps (prompts of 2 to 8192 tokens of up to 64 sequences
// behind up to 16,000, windows of 32 to 8192, 7B and 0.5B heads; rms 19%): a start, and per tile of a walk less with one
// work-group per CU than with two; every further round of two per CU has its own start. Ranges
// add a launch and their partials' bytes. With ranges of 4, 8, 12, 16, 24 or 32 tiles, the best form by these takes 1.02 times
// the best as measured on average, 1.24 in one step of 100 (128 columns without ranges always: 1.18, 64 or 32: 1.25). Cuts into
// ranges about as long as each other take 0.96 times as long as those, over 8914 random steps of 2 to 400 new tokens behind
// 1000 to 16,000 (0.83 in one step of 100, 1.12 in another).
struct BlockCost {
  double start, tile_one, tile_two, round;
};
constexpr BlockCost kBlockCost[2][3] = {
    {{5.8, 1.20, 1.43, 3.6}, {7.2, 0.64, 0.73, 4.9}, {6.5, 0.50, 0.53, 4.0}},   // D = 64: 128, 64, 32 columns
    {{7.0, 1.41, 1.93, 5.9}, {9.0, 0.83, 1.03, 6.9}, {7.5, 0.65, 0.69, 5.3}}};  // D = 128
constexpr double kRangeLaunch = 4.9, kRangeBytesPerUs = 16e6;
constexpr int64_t kMaxRangeBytes = 64ll << 20;  // of the ranges' partials

// The step's single rows run beside the blocks, on four waves a run: 5 us and 0.18 (D = 128) or 0.14 per page. Where they
// would take longer than the blocks they are cut, for a launch that adds their runs (4.5 us with its partials; 6 rows of
// 2140 to 8560 keys beside prompts of 3 to 5 tokens 87 -> 33 us). Where a CU has no place for them beside the blocks, their
// last work-groups start as blocks end, of which some end early: half a row's time more. (Over 4136 random steps in which it
// matters, the form chosen takes 1.04 times the best tried; 1.07 with a quarter of a row's time, 1.16 with none,
// 1.04 with all of it. Rows in turn on as many work-groups as find a place: 1.02 times as long, a row beside a block is slow.)
constexpr double kRunLaunch = 4.5, kLateRows = 0.5;

static WindowPlan plan_blocks(const WindowArgs& w) {
  const PrefillArgs a = blocks_of_step(w);
  const int64_t group = a.num_heads / a.num_kv_heads, cus = device_cus();
  const int64_t range_bytes = prefill_range_floats(1, a.num_tokens, a.num_heads, a.head_dim) * 4;
  const int64_t row_pages = max_row_pages(w);
  const int64_t rows = w.single_query_seqs >= 0 ? w.single_query_seqs : w.num_seqs;
  const int64_t units = row_units(w, rows);
  const int64_t row_bytes = (int64_t)a.num_seqs * a.num_heads * (a.head_dim + 1) * 4;
  double row_us[5];  // a row's work-group, in 1, 2, .. 16 runs
  for (int i = 0; i < 5; ++i) row_us[i] = 5 + (a.head_dim == 128 ? 0.18 : 0.14) * (double)((row_pages + (1 << i) - 1) >> i);
  WindowPlan p{128, 0, 0, 1};
  double best = 0;
  for (int form = 0; form < 3; ++form) {
    const int columns = 128 >> form;
    const BlockCost& c = kBlockCost[a.head_dim == 128][form];
    // The longest walk that there can be: the window of a block's rows, the first tokens' pages, inside the table.
    const int64_t span = std::min<int64_t>(a.max_query_len, (columns + group - 1) / group + 1);
    const int64_t pages = std::min<int64_t>(a.max_blocks, ((int64_t)w.window + span + 15) / 16 + 1 + ((int64_t)w.sinks + 15) / 16);
    const int64_t tiles = (pages + 3) / 4, blocks = prefill_work_groups(a, columns);
    for (int64_t most : {0, 4, 5, 6, 7, 8, 10, 12, 14, 16, 20, 24, 28, 32}) {
      if (most >= tiles) break;
      // As few ranges as of so many tiles at most, all about as long.
      const int64_t ranges = most > 0 ? (tiles + most - 1) / most : 1, split = most > 0 ? (tiles + ranges - 1) / ranges : 0;
      if (ranges > 1 && ranges * range_bytes > kMaxRangeBytes) continue;
      const double walk = (double)(split > 0 ? split : tiles);
      const int64_t full = blocks * ranges / (2 * cus), rest = blocks * ranges - full * 2 * cus;
      double t = c.start - c.round + (double)full * (c.round + c.tile_two * walk);
      if (rest > 0) t += c.round + (rest > cus ? c.tile_two : c.tile_one) * walk;
      if (split > 0) t += kRangeLaunch + 2.0 * (double)(ranges * range_bytes) / kRangeBytesPerUs;
      const int64_t places = rest > 0 ? 2 * cus - rest : 0;  // beside the last round
      for (int i = 0; i < 5; ++i) {
        const int64_t runs = 1 << i;
        if (i > 0 && (units * runs + blocks * ranges > 2 * cus || row_pages < 8 * runs || runs * row_bytes > kMaxRowBytes)) break;
        // How long the rows outlast the blocks.
        const double after = units * runs <= places ? std::max(0.0, row_us[i] - c.round - c.tile_two * walk) : kLateRows * row_us[i];
        const double both = t + (rows > 0 ? after : 0) + (runs > 1 ? kRunLaunch : 0);
        if (best == 0 || both < best) {
          best = both;
          p = {columns, (int32_t)split, split > 0 ? (int32_t)ranges : 0, (int32_t)runs};
        }
        if (rows == 0) break;
      }
    }
  }
  return p;
}

WindowPlan window_plan(const WindowArgs& a) {
  return a.max_query_len == 1 ? WindowPlan{128, 0, 0, runs_of_rows(a)} : plan_blocks(a);
}

template <int D>
static hipError_t launch_window(const WindowArgs& w, const WindowPlan& p, float* workspace, hipStream_t stream) {
  WindowRows r{rows_of_step(w), w.window, w.sinks};
  r.rows.num_splits = p.row_runs;
  r.rows.part_out = workspace;
  r.rows.part_lse = workspace + (int64_t)w.num_seqs * w.num_heads * p.row_runs * D;
  hipError_t err;
  if (w.max_query_len == 1) {
    err = waves_of_rows(w, p.row_runs) == 4 ? launch_rows<D, 4>(r, stream) : launch_rows<D, 8>(r, stream);
  } else {
    PrefillArgs a = blocks_of_step(w);
    a.split_tiles = p.split_tiles;
    a.num_ranges = p.num_ranges;
    a.part_out = workspace + window_row_floats(w.num_seqs, w.num_heads, D, p.row_runs);
    a.part_ml = a.part_out + (int64_t)p.num_ranges * w.num_tokens * w.num_heads * D;
    err = paged_prefill_window(a, r, p.columns, stream);
  }
  // (Steps of one row a sequence run on the rows' work-groups whatever the count says; longer ones with a count of 0 have none.)
  const bool has_rows = w.max_query_len == 1 || w.single_query_seqs != 0;
  if (err != hipSuccess || p.row_runs == 1 || !has_rows) return err;
  const int per_row = (w.num_heads * (D / 4) + 255) / 256;
  if ((int64_t)w.num_seqs * per_row > 0x7fffffff) return hipErrorInvalidValue;
  hipLaunchKernelGGL((window_merge_kernel<D>), dim3((unsigned)(w.num_seqs * per_row)), dim3(256), 0, stream, r, per_row);
  return hipGetLastError();
}

hipError_t paged_window_attention(const WindowArgs& a, const WindowPlan& p, float* workspace, hipStream_t stream) {
  switch (a.head_dim) {
    case 64: return launch_window<64>(a, p, workspace, stream);
    case 128: return launch_window<128>(a, p, workspace, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace bvllm
