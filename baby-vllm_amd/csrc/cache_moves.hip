// The paged cache after several candidates were tried: a verified draft tree's path moves
// behind the context, and beams take over their parents' pages. Every layer's K and V in
// one launch.
//
// Both read and write a few token rows per layer (a row is 256 or 1024 bytes at the
// presets' shapes) and are bound by the chain of dependent loads in front of the rows and,
// for full batches, by HBM: one thread per 16 bytes of a row, which moves that column
// for every row that it depends on, so that reads come before the writes that would
// overwrite them and no thread waits for another. Measured: the commit of one tree of 8 in 24
// layers 2.3 us, of 48 trees of 20 to 64 in 28 layers 7 to 8 (8 MB out and in); beams of one request at
// 1003 tokens 3.7 us, 16 groups of 8 beams 13 (67 MB read and written, 5.2 TB/s).
#include "bvllm_device.h"
#include "bvllm_abi_internal.h"

#include <algorithm>

namespace bvllm {

namespace {

typedef const int32_t __attribute__((address_space(4)))* ConstI32;
typedef const int64_t __attribute__((address_space(4)))* ConstI64;

// Address of a 16-byte column of token rows, at page 0, token 0: `chunk` of the row of layer
// half / 2's K (even) or V (odd).
__device__ __forceinline__ unsigned char* column_at(const CacheSet& c, const CacheShape& s, int half, int chunk) {
  const int per_head = s.head_dim / 8, head = chunk / per_head;
  void* cache = (half & 1) ? c.v[half >> 1] : c.k[half >> 1];
  return reinterpret_cast<unsigned char*>(cache) +
         ((int64_t)head * s.stride_head + 8 * (chunk - head * per_head)) * 2;
}

// The path of sequence s: from node 0, always the first child whose drafted token is the
// answer at the node. Children come after their parent, so the walk ends. path is filled by
// lane 0 of every wave with the same values; returns its length and the last node's answer.
__device__ __forceinline__ int walk(const CommitArgs& a, int start, int n, int* path, int64_t& following) {
  const int lane = lane_id();
  const int32_t* parents = a.parents + start;
  const int64_t* draft = a.draft_tokens + start;
  const int64_t* target = a.target_tokens + start;
  // The first 64 nodes stay in registers.
  const bool mine = lane < n;
  const int par0 = mine ? parents[lane] : -2;
  const int64_t draft0 = mine ? draft[lane] : 0, target0 = mine ? target[lane] : 0;
  int cur = 0, len = 1;
  if (lane == 0) path[0] = 0;
  for (;;) {
    const int64_t answer = cur < 64 ? __shfl(target0, cur, 64) : target[cur];
    following = answer;
    if (len >= a.max_path) return len;
    int next = -1;
    for (int c0 = (cur + 1) & ~63; c0 < n && next < 0; c0 += 64) {
      const int c = c0 + lane;
      const int par = c0 == 0 ? par0 : c < n ? parents[c] : -2;
      const int64_t tok = c0 == 0 ? draft0 : c < n ? draft[c] : 0;
      const uint64_t hit = __builtin_amdgcn_ballot_w64(c > cur && par == cur && tok == answer);
      if (hit != 0) next = c0 + (int)__builtin_ctzll(hit);
    }
    if (next < 0) return len;
    cur = uniform(next);
    if (lane == 0) path[len] = cur;
    ++len;
  }
}

__global__ __launch_bounds__(256) void commit_tree_kernel(CommitArgs a, CacheSet caches, int items, int outputs) {
  extern __shared__ int path[];
  const int s = (int)blockIdx.y;
  const int start = ((ConstI32)a.query_start_loc)[s];
  const int n = ((ConstI32)a.query_start_loc)[s + 1] - start;
  const int ctx = ((ConstI32)a.context_lens)[s];
  int64_t following = -1;
  const int len = n > 0 ? walk(a, start, n, path, following) : 0;
  __syncthreads();
  if (outputs && blockIdx.x == 0) {
    for (int i = (int)threadIdx.x; i < a.max_path; i += 256) a.path[(int64_t)s * a.max_path + i] = i < len ? path[i] : -1;
    if (threadIdx.x == 0) {
      a.accepted[s] = len;
      a.following[s] = following;
    }
  }
  const int item = (int)blockIdx.x * 256 + (int)threadIdx.x;
  if (item >= items || ctx < 0) return;
  const int per_row = a.cache.num_kv_heads * (a.cache.head_dim / 8), half = item / per_row;
  unsigned char* const col = column_at(caches, a.cache, half, item - half * per_row);
  const int32_t* table = a.block_tables + (int64_t)s * a.bt_stride;
  // Byte offset of the row at position ctx + i, or -1 outside the table or the pool.
  auto row_at = [&](int i) -> int64_t {
    const int64_t pos = (int64_t)ctx + i;
    if (pos >> 4 >= a.max_blocks) return -1;
    const int page = table[pos >> 4];
    if (page < 0 || page >= a.cache.num_pages) return -1;
    return ((int64_t)page * a.cache.stride_page + (pos & 15) * a.cache.stride_token) * 2;
  };
  // Rows move towards the front (path[i] >= i, ascending), so a batch that is read whole
  // before it is written never overwrites a row that a later batch reads.
  constexpr int kBatch = 8;
  for (int i0 = 1; i0 < len; i0 += kBatch) {
    uint4 v[kBatch];
    int64_t to[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      to[k] = -1;
      const int i = i0 + k;
      if (i < len && path[i] != i) {
        const int64_t from = row_at(path[i]);
        if (from >= 0) {
          to[k] = row_at(i);
          v[k] = ld16(col + from);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k)
      if (to[k] >= 0) st16(col + to[k], v[k]);
  }
}

// Beams: thread = (row of the partial page, column); it holds that column of every beam
// that takes another's, all read before any is written. The work-groups behind those
// permute the full pages' table entries in the same way, a thread per table column. (The
// partial page's own entry is not among them, so no work-group reads what another writes.)
template <int KB>
__global__ __launch_bounds__(256) void reorder_beams_kernel(ReorderArgs a, CacheSet caches, int halves, int data_wgs) {
  const int K = a.num_beams;
  const int64_t row0 = (int64_t)blockIdx.y * K;
  const int len = ((ConstI32)a.seq_lens)[row0];
  const int full = max(0, len) >> 4, partial = max(0, len) & 15;
  // The beam's parent; itself where the index is not one of the group.
  auto parent = [&](int b) __attribute__((always_inline)) -> int {
    const int64_t p = ((ConstI64)a.beams)[row0 + b];
    return p >= 0 && p < K ? (int)p : b;
  };
  if ((int)blockIdx.x >= data_wgs) {
    const int c = ((int)blockIdx.x - data_wgs) * 256 + (int)threadIdx.x;
    if (c >= min(full, a.max_blocks)) return;
    int32_t* t = a.block_tables + row0 * a.bt_stride + c;
    int32_t e[KB];
#pragma unroll
    for (int b = 0; b < KB; ++b)
      if (b < K) e[b] = t[(int64_t)parent(b) * a.bt_stride];
#pragma unroll
    for (int b = 0; b < KB; ++b)
      if (b < K && parent(b) != b) t[(int64_t)b * a.bt_stride] = e[b];
    return;
  }
  if (full >= a.max_blocks) return;
  const int item = (int)blockIdx.x * 256 + (int)threadIdx.x;
  const int per_row = a.cache.num_kv_heads * (a.cache.head_dim / 8);
  const int half_row = item / per_row, row = half_row & 15;  // 16 rows of each half, their chunks together
  if (row >= partial || (half_row >> 4) >= halves) return;
  unsigned char* const at = column_at(caches, a.cache, half_row >> 4, item - half_row * per_row) +
                            (int64_t)row * a.cache.stride_token * 2;
  const ConstI32 table = (ConstI32)(a.block_tables + row0 * a.bt_stride + full);
  uint4 v[KB];
  uint32_t taken = 0;  // beams whose parent's page is one of the pool
#pragma unroll
  for (int b = 0; b < KB; ++b)
    if (b < K) {
      const int p = parent(b), entry = table[(int64_t)p * a.bt_stride];
      const int page = min(max(entry, 0), a.cache.num_pages - 1);
      if (p != b) v[b] = ld16(at + (int64_t)page * a.cache.stride_page * 2);
      taken |= (uint32_t)(p != b && page == entry) << b;
    }
#pragma unroll
  for (int b = 0; b < KB; ++b)
    if ((taken >> b) & 1) {
      const int page = table[(int64_t)b * a.bt_stride];
      if (page >= 0 && page < a.cache.num_pages) st16(at + (int64_t)page * a.cache.stride_page * 2, v[b]);
    }
}

CacheSet cache_set(void* const* k, void* const* v, int first, int count) {
  CacheSet c{};
  for (int i = 0; i < count; ++i) {
    c.k[i] = k[first + i];
    c.v[i] = v[first + i];
  }
  return c;
}

}  // namespace

hipError_t commit_draft_tree(const CommitArgs& a, void* const* k, void* const* v, int layers, hipStream_t stream) {
  for (int first = 0; first == 0 || first < layers; first += kCacheSetLayers) {
    const int count = std::min(kCacheSetLayers, layers - first);
    const int items = count * 2 * a.cache.num_kv_heads * (a.cache.head_dim / 8);
    hipLaunchKernelGGL(commit_tree_kernel, dim3((unsigned)std::max(1, (items + 255) / 256), (unsigned)a.num_seqs),
                       dim3(256), (size_t)a.max_path * sizeof(int), stream, a, cache_set(k, v, first, count), items,
                       first == 0 ? 1 : 0);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
  }
  return hipSuccess;
}

template <int KB>
static hipError_t launch_reorder(const ReorderArgs& a, void* const* k, void* const* v, int layers, hipStream_t stream) {
  const int table_wgs = (a.max_blocks + 255) / 256;
  for (int first = 0; first == 0 || first < layers; first += kCacheSetLayers) {
    const int count = std::min(kCacheSetLayers, layers - first);
    const int64_t items = (int64_t)count * 2 * 16 * a.cache.num_kv_heads * (a.cache.head_dim / 8);
    const int data_wgs = (int)((items + 255) / 256);
    // The tables are permuted once, by the last launch.
    const int wgs = data_wgs + (first + count >= layers ? table_wgs : 0);
    hipLaunchKernelGGL((reorder_beams_kernel<KB>), dim3((unsigned)wgs, (unsigned)a.num_groups), dim3(256), 0, stream,
                       a, cache_set(k, v, first, count), 2 * count, data_wgs);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
  }
  return hipSuccess;
}

hipError_t reorder_beams(const ReorderArgs& a, void* const* k, void* const* v, int layers, hipStream_t stream) {
  if (a.num_beams <= 4) return launch_reorder<4>(a, k, v, layers, stream);
  if (a.num_beams <= 8) return launch_reorder<8>(a, k, v, layers, stream);
  if (a.num_beams <= 16) return launch_reorder<16>(a, k, v, layers, stream);
  return launch_reorder<32>(a, k, v, layers, stream);
}

}  // namespace bvllm
