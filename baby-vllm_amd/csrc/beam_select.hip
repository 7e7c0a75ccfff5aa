// Beam search's selection: the n best continuations of a group of K beams over the
// vocabulary,
//   total(b, v) = score_b + logit_bv - lse_b,  lse_b = log sum_v exp(logit_bv),
// in descending order, equal totals by their flat index b·V + v.
//
// Bound by one pass over the logits (16 groups of 8 beams over 152,064 bf16 tokens are
// 39 MB). Stage 1, one wave per piece of 2048 columns: the piece's maximum and its sum of
// exponentials relative to it, nothing else. Stage 2, one work-group per group: the rows'
// lse from the pieces; then the n best pieces by (total of the maximum, index) hold the n
// best tokens (each of n better pieces has a better token), so only those are read again,
// and of them only tokens that reach the n-th piece's maximum compete.
//
// Pieces are cut by column, whatever a row's alignment, so equal rows get equal bits. Sums
// of exponentials are fp32 within a piece (32 terms per lane) and fp64 across; totals are
// formed and compared in fp64, so that two tokens of one beam keep the order of their
// logits, and rounded once to fp32 on output.
//
// A beam whose score is not finite, or whose logits hold a NaN, a +inf or no finite value,
// has no distribution: all its totals are -inf.
#include "bvllm_device.h"
#include "bvllm_abi_internal.h"

namespace bvllm {

namespace {

constexpr int kPiece = kBeamPiece;   // columns per piece: 32 per lane
constexpr int kScanWaves = 4;
constexpr int kPickWaves = 16;
constexpr int kPickThreads = 64 * kPickWaves;
constexpr int kMaxPick = kBeamMaxCandidates;  // n at most: the wave-wide steps hold one per lane
static_assert(kMaxPick == 64, "one candidate per lane");

typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

// The lane's elements of a piece as fp32: vector k (16 bytes) of lane l starts at column
// (64·k + l)·VEC of the piece. Columns past `left` read as -inf. Rows need not be aligned.
template <typename T>
struct Piece {
  static constexpr int VEC = 16 / sizeof(T), LOADS = 32 / VEC;
  float v[32];
  static __device__ __forceinline__ int column(int e) { return ((e / VEC) * 64 + lane_id()) * VEC + e % VEC; }
  __device__ __forceinline__ void load(const T* x, int left) {
    u32x4_any raw[LOADS];
#pragma unroll
    for (int k = 0; k < LOADS; ++k) {
      const int c = column(k * VEC);
      if (c + VEC <= left) {
        raw[k] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_any*>(x + c));
      } else if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t lo = c + 2 * j < left ? (uint32_t)x[c + 2 * j] : 0xff80u;
          const uint32_t hi = c + 2 * j + 1 < left ? (uint32_t)x[c + 2 * j + 1] : 0xff80u;
          raw[k][j] = lo | (hi << 16);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) raw[k][j] = c + j < left ? __float_as_uint(x[c + j]) : 0xff800000u;
      }
    }
#pragma unroll
    for (int e = 0; e < 32; ++e) {
      const uint32_t w = raw[e / VEC][sizeof(T) == 2 ? (e % VEC) / 2 : e % VEC];
      v[e] = sizeof(T) == 4 ? __uint_as_float(w) : (e & 1) ? hi_f32(w) : lo_f32(w);
    }
  }
};

__device__ __forceinline__ float wave_max(float x) {
  x = fmax_prop(x, __uint_as_float(dpp<kQuadSwap1>(__float_as_uint(x))));
  x = fmax_prop(x, __uint_as_float(dpp<kQuadSwap2>(__float_as_uint(x))));
  x = fmax_prop(x, __uint_as_float(dpp<kRowHalfMirror>(__float_as_uint(x))));
  x = fmax_prop(x, __uint_as_float(dpp<kRowMirror>(__float_as_uint(x))));
  return max_across_groups(x);
}
__device__ __forceinline__ float wave_sum(float x) {
  x += __uint_as_float(dpp<kQuadSwap1>(__float_as_uint(x)));
  x += __uint_as_float(dpp<kQuadSwap2>(__float_as_uint(x)));
  x += __uint_as_float(dpp<kRowHalfMirror>(__float_as_uint(x)));
  x += __uint_as_float(dpp<kRowMirror>(__float_as_uint(x)));
  return sum_across_groups(x);
}

// ------------------------------------------------------------- stage 1

template <typename T>
__global__ __launch_bounds__(64 * kScanWaves) void beam_scan_kernel(BeamSelectArgs a, int pieces, int groups_per_row) {
  const int row = (int)blockIdx.x / groups_per_row;
  const int piece = ((int)blockIdx.x - row * groups_per_row) * kScanWaves + wave_id();
  if (piece >= pieces) return;
  Piece<T> p;
  p.load(reinterpret_cast<const T*>(a.logits) + (int64_t)row * a.row_stride + (int64_t)piece * kPiece,
         a.vocab - piece * kPiece);
  float mx[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) mx[e] = fmax_prop(p.v[e], p.v[e + 16]);
#pragma unroll
  for (int s = 8; s >= 1; s /= 2)
#pragma unroll
    for (int e = 0; e < s; ++e) mx[e] = fmax_prop(mx[e], mx[e + s]);
  const float m = wave_max(mx[0]);
  // (A piece of -inf alone adds nothing; one with a NaN or +inf leaves its mark in m.)
  const float ref = m == kNegInf ? 0.f : m;
  float sum = 0.f;
#pragma unroll
  for (int e = 0; e < 32; ++e) sum += fast_exp2((p.v[e] - ref) * kLog2e);
  sum = wave_sum(sum);
  if (lane_id() == 0) *reinterpret_cast<float2*>(a.stats + ((int64_t)row * pieces + piece) * 2) = make_float2(m, sum);
}

// ------------------------------------------------------------- stage 2

// A total as an integer of the same order.
__device__ __forceinline__ uint64_t order_of(double x) {
  const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);
  return u >> 63 ? ~u : u | (1ull << 63);
}
__device__ __forceinline__ double total_of(uint64_t k) {
  return __longlong_as_double((long long)(k >> 63 ? k & ~(1ull << 63) : ~k));
}

__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u >> 31 ? ~u : u | (1u << 31);
}

constexpr double kNegInf64 = -__builtin_huge_val();

template <typename T>
__global__ __launch_bounds__(kPickThreads) void beam_pick_kernel(BeamSelectArgs a, int pieces) {
  constexpr int kMaxKeys = kBeamMaxPieces;
  // Keys of the pieces, later the competing tokens (key and flat index).
  __shared__ __attribute__((aligned(16))) uint64_t store[kMaxKeys];
  static_assert(kMaxKeys >= 2 * kMaxPick * kMaxPick, "n tokens of n pieces");
  __shared__ uint16_t ahead[kMaxKeys];  // pieces that reach the lane threshold
  __shared__ double base[kBeamMaxBeams];
  __shared__ uint64_t lane_key[64];
  __shared__ int lane_piece[64], lane_rank[64], chosen[kMaxPick], counts[2];
  uint64_t* keys = store;

  const int tid = (int)threadIdx.x, lane = lane_id(), w = wave_id();
  const int K = a.num_beams, n = a.num_candidates, M = K * pieces;
  const int64_t row0 = (int64_t)blockIdx.x * K;
  const float2* stats = reinterpret_cast<const float2*>(a.stats) + row0 * pieces;
  if (tid < 2) counts[tid] = 0;
  if (tid < 64) lane_rank[tid] = 0;

  // base_b = score_b - lse_b, in fp64 from the largest piece maximum on.
  for (int b = w; b < K; b += kPickWaves) {
    float m = kNegInf;
    for (int i = lane; i < pieces; i += 64) m = fmax_prop(m, stats[b * pieces + i].x);
    m = wave_max(m);
    double sum = 0.0;
    for (int i = lane; i < pieces; i += 64) {
      const float2 x = stats[b * pieces + i];
      if (x.x != kNegInf) sum += (double)x.y * exp((double)x.x - (double)m);
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d, 64);
    if (lane == 0) {
      const float score = a.scores[row0 + b];
      const bool live = fabsf(m) < __builtin_huge_valf() && fabsf(score) < __builtin_huge_valf();
      base[b] = live ? (double)score - ((double)m + log(sum)) : kNegInf64;
    }
  }
  __syncthreads();
  // (base is -inf for a beam without a distribution, whatever its logits.)
  auto total = [&](int b, float x) { return base[b] == kNegInf64 ? kNegInf64 : (double)x + base[b]; };
  for (int i = tid; i < M; i += kPickThreads) keys[i] = order_of(total(i / pieces, stats[i].x));
  __syncthreads();

  // A threshold that at least n pieces reach and few others: lane l of a wave takes the best
  // of pieces l, l + 64, ...; the n-th best of those 64.
  int n_chosen = M;
  if (M > n) {
    n_chosen = n;
    if (w == 0) {
      uint64_t k = 0;
      int at = 0x7fffffff;
      for (int i = lane; i < M; i += 64)
        if (at == 0x7fffffff || keys[i] > k) {
          k = keys[i];
          at = i;
        }
      lane_key[lane] = k;
      lane_piece[lane] = at;
    }
    __syncthreads();
    {
      const uint64_t k = lane_key[lane];
      const int at = lane_piece[lane];
      int better = 0;
#pragma unroll
      for (int q = 0; q < 64 / kPickWaves; ++q) {
        const int o = w * (64 / kPickWaves) + q;
        better += lane_key[o] > k || (lane_key[o] == k && lane_piece[o] < at);
      }
      if (better) atomicAdd(&lane_rank[lane], better);
    }
    __syncthreads();
    const uint64_t at_rank = __builtin_amdgcn_ballot_w64(lane_rank[lane] == n - 1);
    const int tl = (int)__builtin_ctzll(at_rank);
    const uint64_t tk = lane_key[tl];
    const int tp = lane_piece[tl];
    for (int i = tid; i < M; i += kPickThreads)
      if (keys[i] > tk || (keys[i] == tk && i <= tp)) ahead[atomicAdd(&counts[0], 1)] = (uint16_t)i;
    __syncthreads();
    const int c = counts[0];
    for (int e = tid; e < c; e += kPickThreads) {
      const int i = ahead[e];
      const uint64_t k = keys[i];
      int rank = 0;
      for (int o = 0; o < c; ++o) {
        const int p = ahead[o];
        rank += keys[p] > k || (keys[p] == k && p < i);
      }
      if (rank < n) chosen[rank] = i;
    }
  } else if (tid < M) {
    chosen[tid] = tid;
  }
  __syncthreads();
  // With n pieces a token has to reach the n-th one's maximum.
  const uint64_t bar = M > n ? keys[chosen[n - 1]] : 0;
  __syncthreads();

  // The chosen pieces' tokens that reach the bar: (key, flat index) pairs. At most n of a
  // piece, its best ones.
  uint64_t* cand = store;
  for (int e = w; e < n_chosen; e += kPickWaves) {
    const int b = chosen[e] / pieces, piece = chosen[e] - b * pieces;
    Piece<T> p;
    p.load(reinterpret_cast<const T*>(a.logits) + (row0 + b) * a.row_stride + (int64_t)piece * kPiece,
           a.vocab - piece * kPiece);
    const int left = a.vocab - piece * kPiece;
    if (base[b] == kNegInf64) {  // no distribution: all alike, whatever they hold
#pragma unroll
      for (int i = 0; i < 32; ++i) p.v[i] = kNegInf;
    }
    uint32_t over = 0, even = 0;  // the lane's elements above the bar, and at it
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      if (Piece<T>::column(i) < left) {
        const uint64_t k = order_of(total(b, p.v[i]));
        over |= (uint32_t)(k > bar) << i;
        even |= (uint32_t)(k == bar) << i;
      }
    }
    auto wave_count = [&](uint32_t bits) {
      return wave_reduce(__builtin_popcount(bits), [](int x, int y) { return x + y; });
    };
    int n_over = wave_count(over);
    if (n_over > n) {
      // The piece alone holds more than n above the bar: its own bar is its n-th logit, found
      // bit by bit from the top (the largest value that at least n reach).
      const uint32_t open = over;
      uint32_t nth = 0;
      for (int bit = 31; bit >= 0; --bit) {
        const uint32_t probe = nth | (1u << bit);
        int mine = 0;
#pragma unroll
        for (int i = 0; i < 32; ++i) mine += ((open >> i) & 1) && order_of(p.v[i]) >= probe;
        const int reach = wave_reduce(mine, [](int x, int y) { return x + y; });
        if (reach >= n) nth = probe;
        if (reach == n) break;
      }
      over = even = 0;
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        over |= (uint32_t)(((open >> i) & 1) && order_of(p.v[i]) > nth) << i;
        even |= (uint32_t)(((open >> i) & 1) && order_of(p.v[i]) == nth) << i;
      }
      n_over = wave_count(over);
      if (n_over == n) even = 0;
    }
    // Elements at the bar are equal: the first of them by column, as many as could be taken.
    int want_even = n_over >= n ? 0 : n - n_over;
    if (wave_count(even) > want_even) {
      // Vectors in order, lanes in order within one.
      uint32_t keep = 0;
#pragma unroll
      for (int k = 0; k < Piece<T>::LOADS; ++k) {
        constexpr int VEC = Piece<T>::VEC;
        uint32_t bits = (even >> (k * VEC)) & ((1u << VEC) - 1);
        const int mine = __builtin_popcount(bits);
        int before = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
          const int t = __shfl_up(before, d, 64);
          if (lane >= d) before += t;
        }
        const int all = __shfl(before, 63, 64);
        before -= mine;
        int room = max(0, want_even - before);
        while (bits != 0 && room > 0) {
          keep |= (bits & -bits) << (k * VEC);
          bits &= bits - 1;
          --room;
        }
        want_even = max(0, want_even - all);
      }
      even = keep;
    }
    const uint32_t taken = over | even;
    const int mine = __builtin_popcount(taken);
    int before = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int t = __shfl_up(before, d, 64);
      if (lane >= d) before += t;
    }
    int at = 0;
    if (lane == 63) at = atomicAdd(&counts[1], before);
    at = __shfl(at, 63, 64) + before - mine;
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if ((taken >> i) & 1) {
        cand[2 * at] = order_of(total(b, p.v[i]));
        cand[2 * at + 1] = (uint64_t)((int64_t)b * a.vocab + (int64_t)piece * kPiece + Piece<T>::column(i));
        ++at;
      }
  }
  __syncthreads();
  const int c = counts[1];
  const int64_t out0 = (int64_t)blockIdx.x * n;
  for (int e = tid; e < c; e += kPickThreads) {
    const uint64_t k = cand[2 * e], flat = cand[2 * e + 1];
    int rank = 0;
    for (int o = 0; o < c; ++o) rank += cand[2 * o] > k || (cand[2 * o] == k && cand[2 * o + 1] < flat);
    if (rank < n) {
      const int64_t beam = (int64_t)(flat / (uint64_t)a.vocab);
      a.out_scores[out0 + rank] = (float)total_of(k);
      a.out_beams[out0 + rank] = beam;
      a.out_tokens[out0 + rank] = (int64_t)flat - beam * a.vocab;
    }
  }
}

template <typename T>
hipError_t launch_select(const BeamSelectArgs& a, hipStream_t stream) {
  const int pieces = (a.vocab + kPiece - 1) / kPiece;
  const int per_row = (pieces + kScanWaves - 1) / kScanWaves;
  const int64_t wgs = (int64_t)a.num_groups * a.num_beams * per_row;
  if (wgs > 0x7fffffff) return hipErrorInvalidValue;
  hipLaunchKernelGGL((beam_scan_kernel<T>), dim3((unsigned)wgs), dim3(64 * kScanWaves), 0, stream, a, pieces, per_row);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  hipLaunchKernelGGL((beam_pick_kernel<T>), dim3((unsigned)a.num_groups), dim3(kPickThreads), 0, stream, a, pieces);
  return hipGetLastError();
}

}  // namespace

hipError_t beam_select(const BeamSelectArgs& a, hipStream_t stream) {
  return a.fp32 ? launch_select<float>(a, stream) : launch_select<uint16_t>(a, stream);
}

}  // namespace bvllm
