// Beam search's selection: the n best continuations of a group of K beams over the
// vocabulary,
//   total(b, v) = score_b + logit_bv - lse_b,  lse_b = log sum_v exp(logit_bv),
// in descending order, equal totals by their flat index b·V + v.
//
// Stage 1, one wave per piece of 2048 columns: the piece's maximum and its sum of
// exponentials relative to it, nothing else. It is one pass over the logits (16 groups of 8
// beams over 152,064 bf16 tokens, 39 MB: 7.7-9.5 us, 4.1-5.1 TB/s). Stage 2, one work-group
// per group: the rows' lse from the pieces; then a bar that n pieces' maxima reach, so that a
// token has to reach it too. Only pieces that do are read again, some more than n of them, and
// few tokens in them compete: each counts the better ones. It is bound by its chain of loads
// and barriers (1 group of 4 beams, 8 candidates: 6.8 us; 16 groups of 8, 16 candidates: 9).
// Choosing the n best of each piece in stage 1 instead took 24.4 us there, most of it in
// counting that no later choice needed.
//
// Crowds of equal totals, of masks that leave fewer tokens than candidates among them, take the
// exact choice (the same two sizes with one token of a row left: 19.4 and 30.1 us in all, with 20
// tokens 9.8 and 16.7, with all 9.1 and 16.8).
//
// Pieces are cut by column, whatever a row's alignment, so equal rows get equal bits. Sums
// of exponentials are fp32 within a piece (32 terms per lane) and fp64 across, so a row's lse is off by
// less than 2^-17: exponents and their arguments by 2^-23 per unit of distance from the maximum, whose
// average by weight is below ln V = 12 or so, sums of 32 and 64 terms by 38 * 2^-24 (as measured, 3e-7 at
// most over 9600 rows of 1000 to 151,936 tokens). Totals of different beams that are closer than
// that can come in either order. Totals are formed and compared in fp64, so that two
// tokens of one beam keep the order of their logits, and rounded once to fp32 on output.
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
        raw[k] = *reinterpret_cast<const u32x4_any*>(x + c);
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

// Candidates: more than this many send the group to the exact choice.
constexpr int kMaxCand = kMaxPick * kMaxPick;
static_assert(kMaxCand >= kMaxPick * kMaxPick, "the exact choice: n tokens of n pieces");
static_assert(kBeamMaxPieces >= 64 * kMaxPick, "a key for each lane's share of up to n pieces");
constexpr int kSets = 128;
constexpr int kRankDirect = 128;  // items that count the better ones among all of them

struct PickShared {
  uint64_t keys[kBeamMaxPieces];  // maxima as totals: of the pieces, or of the lanes' shares of few pieces
  uint64_t cand_key[kMaxCand];
  uint32_t cand[kMaxCand];        // b * vocab + v < 2^24 (at most 8192 pieces of 2048)
  uint64_t part_key[kPickThreads], set_key[kSets];
  uint32_t part_index[kPickThreads], set_index[kSets];
  double base[kBeamMaxBeams];
  int rank[kSets];
  uint64_t bar_key;
  uint32_t bar_index;
  uint16_t near[kMaxCand];        // items that reach the threshold
  uint16_t best[kMaxPick];        // the n best, in order
  int count, n_near;
};

// (key, index) pairs: larger keys first, equal ones by index.
__device__ __forceinline__ bool ahead(uint64_t k, uint32_t i, uint64_t l, uint32_t j) {
  return k > l || (k == l && i < j);
}

// A pair that at least n of the items reach and few others, into bar_key and bar_index (0 and
// ~0, reached by all, with fewer): the items are dealt to 128 sets, and it is the n-th best of the
// sets' best. With n at most half the sets, about 1.4 n items reach it.
template <typename Key, typename Index>
__device__ __forceinline__ void near_best(PickShared& sh, int n_items, int n, Key key, Index index) {
  const int tid = (int)threadIdx.x, set = tid & (kSets - 1), slice = tid / kSets;
  uint64_t k = 0;
  uint32_t x = ~0u;
  for (int i = tid; i < n_items; i += kPickThreads)
    if (ahead(key(i), index(i), k, x)) {
      k = key(i);
      x = index(i);
    }
  sh.part_key[tid] = k;
  sh.part_index[tid] = x;
  if (tid < kSets) sh.rank[tid] = 0;
  if (tid == 0) {
    sh.bar_key = 0;
    sh.bar_index = ~0u;
    sh.n_near = 0;
  }
  __syncthreads();
  if (tid < kSets) {
#pragma unroll
    for (int q = 1; q < kPickThreads / kSets; ++q)
      if (ahead(sh.part_key[tid + q * kSets], sh.part_index[tid + q * kSets], k, x)) {
        k = sh.part_key[tid + q * kSets];
        x = sh.part_index[tid + q * kSets];
      }
    sh.set_key[tid] = k;
    sh.set_index[tid] = x;
  }
  __syncthreads();
  k = sh.set_key[set];
  x = sh.set_index[set];
  int better = 0;
  constexpr int kEach = kSets * kSets / kPickThreads;
#pragma unroll
  for (int q = 0; q < kEach; ++q) {
    const int o = slice * kEach + q;
    better += ahead(sh.set_key[o], sh.set_index[o], k, x);
  }
  if (better != 0) atomicAdd(&sh.rank[set], better);
  __syncthreads();
  // (An empty set's pair ranks behind every item's, as all empty sets do together.)
  if (tid < kSets && sh.rank[tid] == n - 1 && k != 0) {
    sh.bar_key = k;
    sh.bar_index = x;
  }
  __syncthreads();
}

// The n best items in order, into sh.best (there are at least n with a key).
template <typename Key, typename Index>
__device__ __forceinline__ void best_items(PickShared& sh, int n_items, int n, Key key, Index index) {
  const int tid = (int)threadIdx.x;
  int m = n_items;
  const bool all = n_items <= kRankDirect;
  if (!all) {
    near_best(sh, n_items, n, key, index);
    for (int i = tid; i < n_items; i += kPickThreads)
      if (!ahead(sh.bar_key, sh.bar_index, key(i), index(i))) sh.near[atomicAdd(&sh.n_near, 1)] = (uint16_t)i;
    __syncthreads();
    m = sh.n_near;
  }
  // Eight lanes per item count the better ones among an eighth of them each (107 items: 6.4 us
  // with one).
  for (int e = tid >> 3; e < m; e += kPickThreads / 8) {
    const int i = all ? e : sh.near[e];
    const uint64_t k = key(i);
    const uint32_t x = index(i);
    int rank = 0;
#pragma unroll 2
    for (int f = tid & 7; f < m; f += 8) {
      const int o = all ? f : sh.near[f];
      rank += ahead(key(o), index(o), k, x);
    }
    rank += (int)dpp<kQuadSwap1>((uint32_t)rank);
    rank += (int)dpp<kQuadSwap2>((uint32_t)rank);
    rank += (int)dpp<kRowHalfMirror>((uint32_t)rank);
    if ((tid & 7) == 0 && rank < n && k != 0) sh.best[rank] = (uint16_t)i;
  }
  __syncthreads();
}

// Totals of beam b; -inf for a beam without a distribution (base -inf), whatever its logits.
__device__ __forceinline__ double total_of_logit(double base, float x) {
  return base == kNegInf64 ? kNegInf64 : (double)x + base;
}

// A beam without a distribution holds nothing but -inf.
template <typename T>
__device__ __forceinline__ void load_piece(const BeamSelectArgs& a, int64_t row, int piece, bool live, Piece<T>& p) {
  p.load(reinterpret_cast<const T*>(a.logits) + row * a.row_stride + (int64_t)piece * kPiece, a.vocab - piece * kPiece);
  if (!live) {
#pragma unroll
    for (int i = 0; i < 32; ++i) p.v[i] = kNegInf;
  }
}

// Wave-wide: exclusive prefix sum, and the sum in `all`.
__device__ __forceinline__ int wave_prefix(int mine, int& all) {
  int upto = mine;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int t = __shfl_up(upto, d, 64);
    if (lane_id() >= d) upto += t;
  }
  all = __shfl(upto, 63, 64);
  return upto - mine;
}

// The piece's n best tokens that reach the bar, whatever there is of equal ones. The lane's
// elements to take, as bits.
template <typename T>
__device__ __forceinline__ uint32_t best_of_piece(const Piece<T>& p, double base, uint64_t bar, int left, int n) {
  uint32_t over = 0, even = 0;  // the lane's elements above the bar, and at it
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    if (Piece<T>::column(i) < left) {
      const uint64_t k = order_of(total_of_logit(base, p.v[i]));
      over |= (uint32_t)(k > bar) << i;
      even |= (uint32_t)(k == bar) << i;
    }
  }
  auto wave_count = [&](uint32_t bits) {
    return wave_reduce(__builtin_popcount(bits), [](int x, int y) { return x + y; });
  };
  int n_over = wave_count(over);
  if (n_over > n) {
    // The piece alone holds more than n above the bar: its own bar is the total of its n-th logit,
    // which is found bit by bit from the top (the largest value that at least n reach).
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
    uint32_t least = ~0u;  // (the search ends early at a value between two logits)
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (((open >> i) & 1) && order_of(p.v[i]) >= nth) least = min(least, order_of(p.v[i]));
    least = wave_reduce(least, [](uint32_t x, uint32_t y) { return min(x, y); });
    double again = base;
    asm volatile("" : "+v"(again));  // (the totals are formed again, not kept in registers meanwhile)
    const uint64_t own = order_of(total_of_logit(base, __uint_as_float(least >> 31 ? least & ~(1u << 31) : ~least)));
    over = even = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const uint64_t k = order_of(total_of_logit(again, p.v[i]));
      over |= (uint32_t)(((open >> i) & 1) && k > own) << i;
      even |= (uint32_t)(((open >> i) & 1) && k == own) << i;
    }
    n_over = wave_count(over);
  }
  // Elements at the bar are equal: the first of them by column, as many as could be taken
  // (vectors in order, lanes in order within one).
  int want = max(0, n - n_over);
  if (wave_count(even) > want) {
    constexpr int VEC = Piece<T>::VEC;
    uint32_t keep = 0;
    for (int k = 0; k < Piece<T>::LOADS; ++k) {
      uint32_t bits = (even >> (k * VEC)) & ((1u << VEC) - 1);
      int all;
      int room = max(0, want - wave_prefix(__builtin_popcount(bits), all));
      while (bits != 0 && room > 0) {
        keep |= (bits & -bits) << (k * VEC);
        bits &= bits - 1;
        --room;
      }
      want = max(0, want - all);
    }
    even = keep;
  }
  return over | even;
}

// The exact choice of pieces and tokens, for groups with too many candidates: many equal
// totals at the bar (masked vocabularies, few distinct logits), or many good tokens in one
// piece. The n best pieces by maximum and index (all of fewer), and of each its n best tokens.
template <typename T>
__device__ __forceinline__ void pick_exact(const BeamSelectArgs& a, int pieces, PickShared& sh) {
  const int lane = lane_id(), w = wave_id();
  const int n = a.num_candidates, M = a.num_beams * pieces;
  const int64_t row0 = (int64_t)blockIdx.x * a.num_beams;
  uint64_t bar = 0;
  if (M > n) {
    best_items(sh, M, n, [&](int i) { return sh.keys[i]; }, [&](int i) { return (uint32_t)i; });
    bar = sh.keys[sh.best[n - 1]];
  }
  for (int e = w; e < min(n, M); e += kPickWaves) {
    const int i = M > n ? sh.best[e] : e, b = i / pieces, piece = i - b * pieces;
    Piece<T> p;
    load_piece(a, row0 + b, piece, sh.base[b] != kNegInf64, p);
    const uint32_t taken = best_of_piece(p, sh.base[b], bar, a.vocab - piece * kPiece, n);
    int all;
    int at = wave_prefix(__builtin_popcount(taken), all);
    int start = 0;
    if (lane == 0) start = atomicAdd(&sh.count, all);
    at += __shfl(start, 0, 64);
#pragma unroll
    for (int q = 0; q < 32; ++q)
      if ((taken >> q) & 1) {
        sh.cand_key[at] = order_of(total_of_logit(sh.base[b], p.v[q]));
        sh.cand[at++] = (uint32_t)(b * a.vocab + piece * kPiece + Piece<T>::column(q));
      }
  }
  __syncthreads();
}

template <typename T>
__global__ __launch_bounds__(kPickThreads) void beam_pick_kernel(BeamSelectArgs a, int pieces) {
  __shared__ PickShared sh;
  const int tid = (int)threadIdx.x, lane = lane_id(), w = wave_id();
  const int K = a.num_beams, n = a.num_candidates, M = K * pieces;
  const int64_t row0 = (int64_t)blockIdx.x * K;
  const float2* stats = reinterpret_cast<const float2*>(a.stats) + row0 * pieces;
  if (tid == 0) sh.count = 0;
  if (tid < 64) sh.rank[tid] = 0;

  // A wave per beam: base_b = score_b - lse_b, in fp64 from the pieces' sums on, and the keys
  // of its pieces, or of the lanes' shares of them where the pieces alone are too few for a bar.
  const bool shares = M <= n;
  const int share_lanes = min(64, (a.vocab + Piece<T>::VEC - 1) / Piece<T>::VEC);  // that hold a token of some piece
  for (int b = w; b < K; b += kPickWaves) {
    const float score = a.scores[row0 + b];
    // (Up to 256 pieces are read once: 4 beams of 75 pieces 0.3 us less.)
    constexpr int kHeld = 4;
    float2 held[kHeld];
#pragma unroll
    for (int q = 0; q < kHeld; ++q)
      held[q] = lane + 64 * q < pieces ? stats[b * pieces + lane + 64 * q] : make_float2(kNegInf, 0.f);
    float m = fmax_prop(fmax_prop(held[0].x, held[1].x), fmax_prop(held[2].x, held[3].x));
    for (int i = lane + 64 * kHeld; i < pieces; i += 64) m = fmax_prop(m, stats[b * pieces + i].x);
    m = wave_max(m);
    double sum = 0.0;
    auto add = [&](float2 x) __attribute__((always_inline)) {
      if (x.x != kNegInf) sum += (double)(x.y * fast_exp2((x.x - m) * kLog2e));
    };
#pragma unroll
    for (int q = 0; q < kHeld; ++q) add(held[q]);
    for (int i = lane + 64 * kHeld; i < pieces; i += 64) add(stats[b * pieces + i]);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d, 64);
    const bool live = fabsf(m) < __builtin_huge_valf() && fabsf(score) < __builtin_huge_valf();
    const double base = live ? (double)score - ((double)m + log(sum)) : kNegInf64;
    if (lane == 0) sh.base[b] = base;
    if (!shares) {
#pragma unroll
      for (int q = 0; q < kHeld; ++q)
        if (lane + 64 * q < pieces) sh.keys[b * pieces + lane + 64 * q] = order_of(total_of_logit(base, held[q].x));
      for (int i = lane + 64 * kHeld; i < pieces; i += 64)
        sh.keys[b * pieces + i] = order_of(total_of_logit(base, stats[b * pieces + i].x));
    } else {
      for (int piece = 0; piece < pieces; ++piece) {
        Piece<T> p;
        load_piece(a, row0 + b, piece, live, p);
        float x = kNegInf;
#pragma unroll
        for (int e = 0; e < 32; ++e) x = fmax_prop(x, p.v[e]);
        // (A share behind the row's end holds no token: key 0.)
        const bool any = Piece<T>::column(0) < a.vocab - piece * kPiece;
        if (lane < share_lanes)
          sh.keys[(b * pieces + piece) * share_lanes + lane] = any ? order_of(total_of_logit(base, x)) : 0;
      }
    }
  }
  __syncthreads();

  // The bar: a total that at least n tokens reach, and few others. Up to 24 candidates: lane l takes the best of
  // pieces l, l + 64, ... and the bar is the n-th best of those 64. More: of 128 sets of all the
  // work-group's threads, which leaves fewer tokens above it but takes more steps. In us, both launches, lanes
  // and sets: 1 group of 4 beams, 300 pieces: 9.6 and 10.9 at n = 8, 11.5 and 12.9 at 24, 13.3 and 14.8 at
  // 40, 25.6 and 19.9 at 64; 16 of 8, 600 pieces each: 15.5 and 16.6, 17.7 and 18.8, 21.9 and 20.6, 55.0 and
  // 26.1; 4 of 32, 800 pieces: 14.7 and 15.5, 17.2 and 17.5, 20.5 and 19.9, 47.8 and 24.8; 1 of 30, 2250
  // pieces: 15.4 and 14.9, 17.3 and 17.0, 20.6 and 19.7, 50.8 and 23.7; 8 of 2, 32 pieces: 9.7 and 11.1
  // at n = 8, 15.7 and 18.5 at 24.
  uint64_t bar = 0;
  if (!shares && n <= 24) {
    uint64_t best = 0;
    for (int i = lane; i < M; i += 64) best = max(best, sh.keys[i]);
    // Each wave compares every lane's best with a few of them.
    int better = 0;
#pragma unroll
    for (int q = 0; q < 64 / kPickWaves; ++q) {
      const int o = w * (64 / kPickWaves) + q;
      const uint64_t other = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(best >> 32), o) << 32) |
                             (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)best, o);
      better += other > best || (other == best && o < lane);
    }
    if (better != 0) atomicAdd(&sh.rank[lane], better);
    __syncthreads();
    const int l = (int)__builtin_ctzll(__builtin_amdgcn_ballot_w64(sh.rank[lane] == n - 1));
    bar = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(best >> 32), l) << 32) |
          (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)best, l);
  } else {
    near_best(sh, shares ? share_lanes * M : M, n, [&](int i) { return sh.keys[i]; }, [&](int i) { return (uint32_t)i; });
    bar = sh.bar_key;
  }
  // Totals of -inf (masked tokens) are no candidates: where fewer than n others are found, the
  // exact choice is taken.
  bar = max(bar, order_of(kNegInf64) + 1);

  // The pieces that reach it (all, if the bar comes from shares), dealt to the waves.
  if (tid == 0) sh.n_near = 0;
  __syncthreads();
  for (int i = tid; i < M; i += kPickThreads)
    if (shares || sh.keys[i] >= bar) {
      const int at = atomicAdd(&sh.n_near, 1);
      if (at < kMaxCand) sh.near[at] = (uint16_t)i;
    }
  __syncthreads();
  const int n_reach = sh.n_near;
  // Far more pieces than candidates: equal maxima at the bar, and the exact choice reads fewer. In us,
  // both launches, all of them read and the exact choice, 1 group of 8 beams of 75 pieces: n = 2, 40 pieces that
  // reach it: 12.2 and 14.4, 72: 15.5 and 14.4; n = 8, 48: 13.2 and 15.2, 96: 19.0 and 15.2; n = 16, 64: 15.1
  // and 18.1, 128: 22.6 and 18.2; n = 64, 160: 28.1 and 39.0, 320: 43.5 and 39.0. With 1 to 32 beams in 1 to 16
  // groups the two are even at 45 to 61, 51 to 65, 75 to 91 and 248 to 274 pieces.
  const bool too_many = n_reach > 4 * n + 32;
  // Their tokens that reach it are candidates: a conservative fp32 threshold sorts out nearly
  // all others. (A wave's next piece on its way meanwhile took registers that spilled: 1 group of
  // 23 fp32 beams, 46 candidates 31.4 us in all, now 20.6; 16 groups of 8 bf16 beams 19.9 and 18.6.)
  const double bar_total = total_of(bar);
  for (int e = w; e < n_reach && !too_many; e += kPickWaves) {
    const int i = uniform((int)sh.near[e]), b = i / pieces, piece = i - b * pieces;
    const double base = sh.base[b];
    Piece<T> p;
    load_piece(a, row0 + b, piece, base != kNegInf64, p);
    const float at_bar = base == kNegInf64 ? kNegInf : (float)(bar_total - base);
    // (The second term: scores so large that a total's own rounding hides logits.)
    float threshold =
        at_bar - fabsf(at_bar) * 0x1p-22f - (base == kNegInf64 ? 0.f : (float)(fabs(base) * 0x1p-51)) - 0x1p-126f;
    if (!(threshold >= -3.402823466e38f)) threshold = at_bar > 0.f ? at_bar : -3.402823466e38f;  // (nothing; all but -inf)
    // Few do: only groups of 8 elements whose maximum reaches it are looked into (4 groups of 32
    // beams, 83 pieces, element by element: 2.7 us more).
    bool full = false;
#pragma unroll
    for (int h = 0; h < 32; h += 8) {
      float top = p.v[h];
#pragma unroll
      for (int q = 1; q < 8; ++q) top = fmaxf(top, p.v[h + q]);
      if (full || __builtin_amdgcn_ballot_w64(top >= threshold) == 0) continue;
#pragma unroll
      for (int q = h; q < h + 8; ++q) {
        const uint64_t hit = __builtin_amdgcn_ballot_w64(p.v[q] >= threshold);
        if (hit == 0 || full) continue;
        int at = 0;
        if (lane == 0) at = atomicAdd(&sh.count, (int)__popcll(hit));
        at = uniform(at);
        full = at + (int)__popcll(hit) > kMaxCand;  // (the count tells everybody)
        if (!full && ((hit >> lane) & 1)) {
          int l = lane;
          asm volatile("" : "+v"(l));  // (formed here, not for all 32 elements ahead)
          const int slot = at + __popcll(hit & ((1ull << l) - 1));
          sh.cand_key[slot] = (uint64_t)b << 32 | __float_as_uint(p.v[q]);
          sh.cand[slot] = (uint32_t)(b * a.vocab + piece * kPiece + (q / Piece<T>::VEC * 64 + l) * Piece<T>::VEC + q % Piece<T>::VEC);
        }
      }
    }
    if (full) break;
  }
  __syncthreads();
  if (too_many || sh.count > kMaxCand || sh.count < n) {
    __syncthreads();
    if (tid == 0) sh.count = 0;
    __syncthreads();
    pick_exact<T>(a, pieces, sh);
  } else {
    for (int c = tid; c < sh.count; c += kPickThreads) {
      const uint64_t x = sh.cand_key[c];
      const uint64_t k = order_of(total_of_logit(sh.base[x >> 32], __uint_as_float((uint32_t)x)));
      sh.cand_key[c] = k >= bar ? k : 0;  // (just below the bar: no candidate)
    }
    __syncthreads();
  }

  // The n best candidates by key, equal ones by index.
  best_items(sh, sh.count, n, [&](int i) { return sh.cand_key[i]; }, [&](int i) { return sh.cand[i]; });
  if (tid < n) {
    const int e = sh.best[tid];
    const int64_t at = (int64_t)blockIdx.x * n + tid;
    const uint32_t flat = sh.cand[e], beam = flat / (uint32_t)a.vocab;
    a.out_scores[at] = (float)total_of(sh.cand_key[e]);
    a.out_beams[at] = beam;
    a.out_tokens[at] = flat - beam * (uint32_t)a.vocab;
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
