// Block tables, row offsets and slot maps of a step from its requests' lengths.
//
// Request s has c tokens in the cache and n new ones; its pages stand in the list one
// request after another, those of request s from start_s on. With P = ceil((c + n) / 16),
// of a windowed cache the entries i < P with kept <= i < kept + gone are not in the list (kept the
// pages of the first tokens that stay; kept + gone the page of the earliest position in the
// window of the request's first new token), so that entry i < kept stands at start_s + i, entry
// i >= kept + gone at start_s + i - gone, and start_s is the sum of P - gone over the requests
// before it. Row t of request s is position c + t - (sum of n over the requests before it).
//
// Every work-group sums the requests' lengths (kChunk at a time: one round trip and a scan by lane
// swaps), then writes its share of the step's rows (the first work-groups, one row a thread: a search and
// a list entry each) or of the table's entries; the first one writes the per-request results. Nothing is shared between work-groups, so there is no order
// between them to wait for. Bound by the chain of launch, lengths, scan, list and stores: one request
// takes 4 us, and the entries go out four to a store so that a table of some MB adds little to that.
#include "bvllm_abi_internal.h"
#include "bvllm_device.h"

namespace bvllm {

namespace {

constexpr int kThreads = 256;
constexpr int kPerThread = 4;
constexpr int kChunk = kThreads * kPerThread;  // requests per scan
constexpr int kShare = 4 * kThreads;           // table entries of a work-group: four a thread

// x of the lane that DPP control CTRL names where the row mask has the lane's row, else 0; both halves.
template <int CTRL, int ROWS>
__device__ __forceinline__ int64_t lane_shift(int64_t x) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, CTRL, ROWS, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)((uint64_t)x >> 32), CTRL, ROWS, 0xf, false);
  return (int64_t)((uint64_t)hi << 32 | lo);
}
// Sum over the lanes up to this one: within the rows of 16, then a row's last lane into the next, and the second
// row's into the upper two.
__device__ __forceinline__ int64_t prefix_sum(int64_t x) {
  x += lane_shift<0x111, 0xf>(x);  // row_shr 1, 2, 4, 8
  x += lane_shift<0x112, 0xf>(x);
  x += lane_shift<0x114, 0xf>(x);
  x += lane_shift<0x118, 0xf>(x);
  x += lane_shift<0x142, 0xa>(x);  // row_bcast 15, 31
  x += lane_shift<0x143, 0xc>(x);
  return x;
}

struct Lengths {
  int64_t tokens, pages;  // sums
};

__global__ __launch_bounds__(kThreads) void step_tables_kernel(StepTablesArgs a, int64_t entries, FastDiv by_width,
                                                               int row_groups) {
  __shared__ int64_t list_start[kChunk];
  __shared__ int32_t row_start[kChunk], ctx[kChunk], pages[kChunk], gone[kChunk];
  __shared__ Lengths wave_sum[kThreads / 64];

  const int tid = (int)threadIdx.x, lane = lane_id(), wave = wave_id();
  const bool writes_lens = blockIdx.x == 0, writes_rows = (int)blockIdx.x < row_groups;
  const int64_t t = (int64_t)blockIdx.x * kThreads + tid;  // the thread's row
  // The thread's four entries: the first one's row and column.
  const int64_t e = writes_rows ? entries : ((int64_t)blockIdx.x - row_groups) * kShare + 4 * tid;
  const int row0 = entries <= 0x7fffffff ? by_width((int)min(e, (int64_t)0x7fffffff)) : (int)(e / a.width);
  const int col0 = (int)(e - (int64_t)row0 * a.width);

  // Place of a request's entry behind its first one in the list, -1: not in it.
  auto place = [&](int32_t entry, int32_t n_pages, int32_t n_gone) {
    const int32_t at = entry < a.kept_pages ? entry : entry - a.kept_pages >= n_gone ? entry - n_gone : -1;
    return entry < n_pages ? at : -1;
  };
  auto listed = [&](int64_t start, int32_t rel, int32_t none) {
    const int64_t i = start + rel;
    return rel >= 0 && i < a.num_listed ? a.pages[i] : none;
  };

  Lengths before = {0, 0};
  for (int s0 = 0; s0 < a.num_seqs; s0 += kChunk) {
    const int here = min(kChunk, a.num_seqs - s0);
    int32_t c[kPerThread], n[kPerThread], p[kPerThread], g[kPerThread];
#pragma unroll
    for (int k = 0; k < kPerThread; ++k) {
      const int i = tid * kPerThread + k;
      c[k] = i < here ? a.context_lens[s0 + i] : 0;
      n[k] = i < here ? a.query_lens[s0 + i] : 0;
    }
    Lengths mine = {0, 0};
#pragma unroll
    for (int k = 0; k < kPerThread; ++k) {
      c[k] = max(c[k], 0);
      n[k] = min(max(n[k], 0), 0x7fffffff - c[k]);  // (positions are 32-bit everywhere else)
      p[k] = (int32_t)(((uint32_t)(c[k] + n[k]) + 15) >> 4);
      g[k] = a.window > 0 && c[k] >= a.window ? max(0, ((c[k] - a.window + 1) >> 4) - a.kept_pages) : 0;
      mine.tokens += n[k];
      mine.pages += p[k] - g[k];
    }
    const Lengths upto = {prefix_sum(mine.tokens), prefix_sum(mine.pages)};
    if (s0 > 0) __syncthreads();  // (the chunk before is no longer read)
    if (lane == 63) wave_sum[wave] = upto;
    __syncthreads();
    Lengths at = {before.tokens + upto.tokens - mine.tokens, before.pages + upto.pages - mine.pages};
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) {
      const Lengths x = wave_sum[w];
      if (w < wave) {
        at.tokens += x.tokens;
        at.pages += x.pages;
      }
      before.tokens += x.tokens;
      before.pages += x.pages;
    }
#pragma unroll
    for (int k = 0; k < kPerThread; ++k) {
      const int i = tid * kPerThread + k;
      const int32_t start = (int32_t)min(at.tokens, (int64_t)a.num_tokens);
      row_start[i] = start;
      list_start[i] = at.pages;
      ctx[i] = c[k];
      pages[i] = p[k];
      gone[i] = g[k];
      if (writes_lens && i < here) {
        a.query_start_loc[s0 + i] = start;
        a.seq_lens[s0 + i] = c[k] + n[k];
      }
      at.tokens += n[k];
      at.pages += p[k] - g[k];
    }
    const int32_t rows_end = (int32_t)min(before.tokens, (int64_t)a.num_tokens);
    __syncthreads();

    // The thread's table entries, of one or of several rows, as far as they lie in the chunk.
    if (e < entries) {
      int32_t page[4];
      bool mine_here[4];
      int s = row0, col = col0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = min(max(s - s0, 0), kChunk - 1);
        mine_here[k] = s >= s0 && s < s0 + here && e + k < entries;
        page[k] = mine_here[k] ? listed(list_start[i], place(col, pages[i], gone[i]), a.pad_page) : 0;
        if (++col == a.width) {
          col = 0;
          ++s;
        }
      }
      // (The table is contiguous and e a multiple of 4: 16-byte aligned, where the table is.)
      if (mine_here[0] && mine_here[1] && mine_here[2] && mine_here[3] && a.vec_ok) {
        st16(a.block_tables + e, make_uint4(page[0], page[1], page[2], page[3]));
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (mine_here[k]) a.block_tables[e + k] = page[k];
      }
    }
    // The thread's row, if it is one of the chunk's requests.
    if (writes_rows && t < rows_end && t >= row_start[0]) {
      int lo = 0, hi = here;  // the last request that starts at or before t: it has rows
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (row_start[mid] <= t) lo = mid;
        else hi = mid;
      }
      const int32_t pos = ctx[lo] + (int32_t)(t - row_start[lo]), entry = pos >> 4;
      const int32_t page = listed(list_start[lo], entry < a.width ? place(entry, pages[lo], gone[lo]) : -1, -1);
      a.positions[t] = pos;
      a.slot_mapping[t] = page >= 0 ? (int64_t)page * 16 + (pos & 15) : -1;
    }
  }
  const int64_t rows = min(before.tokens, (int64_t)a.num_tokens);
  if (writes_lens && tid == 0) a.query_start_loc[a.num_seqs] = (int32_t)rows;
  if (writes_rows && t >= rows && t < a.num_tokens) {  // behind the last request's
    a.positions[t] = 0;
    a.slot_mapping[t] = -1;
  }
}

}  // namespace

hipError_t build_step_tables(const StepTablesArgs& a, hipStream_t stream) {
  const int64_t entries = (int64_t)a.num_seqs * a.width;
  const int64_t row_groups = a.num_tokens > 0 ? ((int64_t)a.num_tokens + kThreads - 1) / kThreads : 1;
  const int64_t wgs = row_groups + (entries + kShare - 1) / kShare;
  if (wgs > 0x7fffffff) return hipErrorInvalidValue;
  hipLaunchKernelGGL(step_tables_kernel, dim3((unsigned)wgs), dim3(kThreads), 0, stream, a, entries, fast_div(a.width),
                     (int)row_groups);
  return hipGetLastError();
}

}  // namespace bvllm
