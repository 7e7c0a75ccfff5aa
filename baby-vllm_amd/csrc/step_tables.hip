// Block tables, row offsets and slot maps of a step from its requests' lengths.
//
// Request s has c tokens in the cache and n new ones; its pages stand in the list one
// request after another, those of request s from start_s on. With P = ceil((c + n) / 16),
// of a windowed cache the entries i < P with kept <= i < first are not in the list (kept the
// pages of the first tokens that stay, first the page of the earliest position in the window
// of the request's first new token), so that entry i < kept stands at start_s + i, entry
// i >= max(kept, first) at start_s + i - gone, gone = max(0, min(first, P) - kept), and
// start_s is the sum of P - gone over the requests before it. Row t of request s is
// position c + t - (sum of n over the requests before it).
//
// Every work-group sums the requests' lengths (kChunk at a time: one round trip and a scan in
// LDS), then writes its share of the table's entries and of the step's rows; the first one
// writes the per-request results. Nothing is shared between work-groups, so there is no order
// between them to wait for.
#include "bvllm_abi_internal.h"
#include "bvllm_device.h"

namespace bvllm {

namespace {

constexpr int kThreads = 256;
constexpr int kPerThread = 4;
constexpr int kChunk = kThreads * kPerThread;  // requests per scan
constexpr int kShare = 4 * kThreads;           // table entries, and rows, of a work-group

struct Lengths {
  int64_t tokens, pages;  // sums
};

__global__ __launch_bounds__(kThreads) void step_tables_kernel(StepTablesArgs a, int64_t entries) {
  __shared__ int32_t tok_start[kChunk + 1];   // first row of each request of the chunk, at most num_tokens
  __shared__ int64_t list_start[kChunk];      // its first place in the list
  __shared__ int32_t ctx[kChunk], total[kChunk];  // its cached tokens, and with the new ones
  __shared__ Lengths wave_sum[kThreads / 64];

  const int tid = (int)threadIdx.x, lane = lane_id(), wave = wave_id();
  const int64_t e0 = (int64_t)blockIdx.x * kShare, e1 = min(e0 + kShare, entries);
  const int64_t t0 = (int64_t)blockIdx.x * kShare, t1 = min(t0 + kShare, (int64_t)a.num_tokens);
  const int first_row = e0 < e1 ? (int)(e0 / a.width) : 0;            // table row and column of the first entry
  const int first_col = e0 < e1 ? (int)(e0 - (int64_t)first_row * a.width) : 0;
  const bool writes_lens = blockIdx.x == 0;

  // Of request (c, n): pages before `first` that are in the window of none of its rows.
  auto pages_of = [&](int64_t c, int64_t n, int64_t& gone) {
    const int64_t p = (c + n + 15) >> 4;
    gone = 0;
    if (a.window > 0 && c >= a.window) gone = max((int64_t)0, ((c - a.window + 1) >> 4) - a.kept_pages);
    return p;
  };
  // Place in the list of a request's entry (relative to its first), -1: not in it.
  auto place = [&](int64_t c, int64_t len, int64_t entry) -> int64_t {
    int64_t gone;
    const int64_t p = pages_of(c, len - c, gone);
    if (entry >= p) return -1;
    if (entry < a.kept_pages) return entry;
    return entry - a.kept_pages >= gone ? entry - gone : -1;
  };
  auto page_at = [&](int64_t start, int64_t rel) -> int32_t {
    const int64_t i = start + rel;
    return rel >= 0 && i < a.num_listed ? a.pages[i] : a.pad_page;
  };

  Lengths before = {0, 0};
  for (int s0 = 0; s0 < a.num_seqs; s0 += kChunk) {
    const int here = min(kChunk, a.num_seqs - s0);
    int64_t c[kPerThread], n[kPerThread], held[kPerThread];
    Lengths mine = {0, 0};
#pragma unroll
    for (int k = 0; k < kPerThread; ++k) {
      const int i = tid * kPerThread + k;
      c[k] = i < here ? max(a.context_lens[s0 + i], 0) : 0;
      n[k] = i < here ? max(a.query_lens[s0 + i], 0) : 0;
      n[k] = min(n[k], (int64_t)0x7fffffff - c[k]);  // (positions are 32-bit everywhere else)
      int64_t gone;
      held[k] = pages_of(c[k], n[k], gone);
      held[k] -= gone;
      mine.tokens += n[k];
      mine.pages += held[k];
    }
    Lengths upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int64_t t = __shfl_up(upto.tokens, d, 64), p = __shfl_up(upto.pages, d, 64);
      if (lane >= d) {
        upto.tokens += t;
        upto.pages += p;
      }
    }
    __syncthreads();  // (the chunk before is no longer read)
    if (lane == 63) wave_sum[wave] = upto;
    __syncthreads();
    Lengths at = before;
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) {
      if (w < wave) {
        at.tokens += wave_sum[w].tokens;
        at.pages += wave_sum[w].pages;
      }
      before.tokens += wave_sum[w].tokens;
      before.pages += wave_sum[w].pages;
    }
    at.tokens += upto.tokens - mine.tokens;
    at.pages += upto.pages - mine.pages;
#pragma unroll
    for (int k = 0; k < kPerThread; ++k) {
      const int i = tid * kPerThread + k;
      const int32_t start = (int32_t)min(at.tokens, (int64_t)a.num_tokens);
      tok_start[i] = start;
      list_start[i] = at.pages;
      ctx[i] = (int32_t)c[k];
      total[i] = (int32_t)(c[k] + n[k]);
      if (writes_lens && i < here) {
        a.query_start_loc[s0 + i] = start;
        a.seq_lens[s0 + i] = (int32_t)(c[k] + n[k]);
      }
      at.tokens += n[k];
      at.pages += held[k];
    }
    const int32_t chunk_rows_end = (int32_t)min(before.tokens, (int64_t)a.num_tokens);
    if (tid == 0) tok_start[kChunk] = chunk_rows_end;
    __syncthreads();

    // Table entries of the share that lie in the chunk's rows.
#pragma unroll
    for (int k = 0; k < kShare / kThreads; ++k) {
      const int l = k * kThreads + tid;
      const int down = (first_col + l) / a.width;
      const int s = first_row + down, col = first_col + l - down * a.width;
      if (e0 + l < e1 && s >= s0 && s < s0 + here)
        a.block_tables[e0 + l] = page_at(list_start[s - s0], place(ctx[s - s0], total[s - s0], col));
    }
    // Rows of the share that belong to the chunk's requests.
#pragma unroll
    for (int k = 0; k < kShare / kThreads; ++k) {
      const int64_t t = t0 + k * kThreads + tid;
      if (t >= t1 || t < tok_start[0] || t >= chunk_rows_end) continue;
      int lo = 0, hi = here;  // the last request that starts at or before t: it has rows
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (tok_start[mid] <= t) lo = mid;
        else hi = mid;
      }
      const int64_t pos = (int64_t)ctx[lo] + (t - tok_start[lo]), entry = pos >> 4;
      const int64_t rel = entry < a.width ? place(ctx[lo], total[lo], entry) : -1;
      const int64_t i = list_start[lo] + rel;
      const int32_t page = rel >= 0 && i < a.num_listed ? a.pages[i] : -1;
      a.positions[t] = pos;
      a.slot_mapping[t] = page >= 0 ? (int64_t)page * 16 + (pos & 15) : -1;
    }
  }
  const int64_t rows = min(before.tokens, (int64_t)a.num_tokens);
  if (writes_lens && tid == 0) a.query_start_loc[a.num_seqs] = (int32_t)rows;
#pragma unroll
  for (int k = 0; k < kShare / kThreads; ++k) {
    const int64_t t = t0 + k * kThreads + tid;
    if (t < t1 && t >= rows) {
      a.positions[t] = 0;
      a.slot_mapping[t] = -1;
    }
  }
}

}  // namespace

hipError_t build_step_tables(const StepTablesArgs& a, hipStream_t stream) {
  const int64_t entries = (int64_t)a.num_seqs * a.width;
  const int64_t most = entries > a.num_tokens ? entries : (int64_t)a.num_tokens;
  const int64_t wgs = most > 0 ? (most + kShare - 1) / kShare : 1;
  if (wgs > 0x7fffffff) return hipErrorInvalidValue;
  hipLaunchKernelGGL(step_tables_kernel, dim3((unsigned)wgs), dim3(kThreads), 0, stream, a, entries);
  return hipGetLastError();
}

}  // namespace bvllm
