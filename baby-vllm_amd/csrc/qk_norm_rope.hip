// RMS norm of every query and key head, rotate-half RoPE of both, and the append of k and v to
// the paged cache, in one pass over the step's projection.
//
//   r = 1 / sqrt(mean(x²) + eps),  y = x·r·w
//   o[:D/2] = y[:D/2]·cos[:D/2] − y[D/2:]·sin[:D/2]
//   o[D/2:] = y[D/2:]·cos[D/2:] + y[:D/2]·sin[D/2:]
// all in fp32, rounded once to bf16. (The RoPE kernel rounds every product and the RMSNorm its
// quotient, since both reproduce torch's bf16 operations bit by bit; here is no such form to
// follow, and every rounding left out is an error less.)
//
// Bound by memory: each row is read once and written once. q goes to the output, rotated k and v
// go to the cache only. One wave takes one unit: 64 / (D/16) rows of q or k of a token (lane =
// row and chunk c: 8 elements of the first half at 8c and the 8 that rotate with them at
// D/2 + 8c, so that a head's sum takes log2(D/16) lane swaps and the rotation none), or
// 64 / (D/8) rows of v. Rows that are not 16-byte aligned are loaded and stored element by
// element (ALIGNED = false), with the same arithmetic.
#include "bvllm_abi_internal.h"
#include "bvllm_device.h"

namespace bvllm {

namespace {

template <bool ALIGNED>
__device__ __forceinline__ uint4 load8(const uint16_t* p) {
  if constexpr (ALIGNED) return ld16_nt(p);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = (uint32_t)p[2 * i] | ((uint32_t)p[2 * i + 1] << 16);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <bool ALIGNED>
__device__ __forceinline__ void store8(uint16_t* p, const uint4& v) {
  if constexpr (ALIGNED) {
    st16_nt(p, v);
  } else {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      p[2 * i] = (uint16_t)w[i];
      p[2 * i + 1] = (uint16_t)(w[i] >> 16);
    }
  }
}

__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// 8 values as they lie in memory, bf16 or fp32, widened where they are used. (The type is the kernel's: a branch on it
// around the loads waited for each of them by itself, 8192 tokens of 7B with bf16 rows and weights 37.8 us.)
template <bool FP32>
struct Eight {
  uint4 w[FP32 ? 2 : 1];
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (FP32) return __uint_as_float(word(w[i / 4], i % 4));
    else return i & 1 ? hi_f32(word(w[0], i / 2)) : lo_f32(word(w[0], i / 2));
  }
};

// Of a row of cos, sin or a weight.
template <bool ALIGNED, bool FP32>
__device__ __forceinline__ Eight<FP32> load_eight(const void* base, int64_t at) {
  Eight<FP32> r;
  if constexpr (FP32) {
    const float* p = reinterpret_cast<const float*>(base) + at;
    if constexpr (ALIGNED) {
      r.w[0] = ld16(p);
      r.w[1] = ld16(p + 4);
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        r.w[i] = make_uint4(__float_as_uint(p[4 * i]), __float_as_uint(p[4 * i + 1]), __float_as_uint(p[4 * i + 2]),
                            __float_as_uint(p[4 * i + 3]));
    }
  } else {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(base) + at;
    if constexpr (ALIGNED) {
      r.w[0] = ld16(p);
    } else {
      uint32_t x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = (uint32_t)p[2 * i] | ((uint32_t)p[2 * i + 1] << 16);
      r.w[0] = make_uint4(x[0], x[1], x[2], x[3]);
    }
  }
  return r;
}

// Sum over groups of N lanes: pairs, quads, then mirrors, which exchange lanes that hold the same.
template <int N>
__device__ __forceinline__ float row_sum(float x) {
  x += __uint_as_float(dpp<kQuadSwap1>(__float_as_uint(x)));
  x += __uint_as_float(dpp<kQuadSwap2>(__float_as_uint(x)));
  if constexpr (N > 4) x += __uint_as_float(dpp<kRowHalfMirror>(__float_as_uint(x)));
  if constexpr (N > 8) x += __uint_as_float(dpp<kRowMirror>(__float_as_uint(x)));
  return x;
}

__device__ __forceinline__ uint4 narrow(const float (&f)[8]) {
  return make_uint4(pack_bf16x2_hw(f[0], f[1]), pack_bf16x2_hw(f[2], f[3]), pack_bf16x2_hw(f[4], f[5]),
                    pack_bf16x2_hw(f[6], f[7]));
}

template <int D, bool ALIGNED, bool ROWS_FP32, bool WEIGHT_FP32>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(QkNormRopeArgs a, int32_t units) {
  constexpr int HALF = D / 2;
  constexpr int RC = D / 16, RPU = 64 / RC;  // lanes per rotated row, rows per unit
  constexpr int VC = D / 8, VPU = 64 / VC;   // lanes per v row, rows per unit
  const int64_t wave = (int64_t)blockIdx.x * (blockDim.x / 64) + wave_id();
  const int64_t t = wave / units;
  if (t >= a.num_tokens) return;
  const int u = (int)(wave - t * units);
  const int lane = lane_id();
  const int rows = a.num_heads + a.num_kv_heads;
  const int rot_units = (rows + RPU - 1) / RPU;
  const int64_t slot = a.slot_mapping[t];
  const bool stored = slot >= 0 && slot < a.num_slots;  // slots outside the cache are not written

  if (u >= rot_units) {
    const int h = (u - rot_units) * VPU + lane / VC, c = lane % VC;
    if (h < a.num_kv_heads && stored) {
      const uint16_t* src = reinterpret_cast<const uint16_t*>(a.v) + t * a.v_st + h * a.v_sh;
      uint16_t* dst = reinterpret_cast<uint16_t*>(a.v_cache) + slot * a.c_slot + h * a.c_head;
      store8<ALIGNED>(dst + 8 * c, load8<ALIGNED>(src + 8 * c));
    }
    return;
  }
  // (Lanes past the last row take part in the swaps on a row of their own group: nothing of them is written.)
  const int row = u * RPU + lane / RC, c = lane % RC;
  const bool live = row < rows, is_k = row >= a.num_heads;
  const int head = live ? (is_k ? row - a.num_heads : row) : 0;
  const uint16_t* src = is_k ? reinterpret_cast<const uint16_t*>(a.k) + t * a.k_st + head * a.k_sh
                             : reinterpret_cast<const uint16_t*>(a.q) + t * a.q_st + head * a.q_sh;
  // All loads of the lane, then the sums.
  const Eight<false> a1 = {{load8<ALIGNED>(src + 8 * c)}}, a2 = {{load8<ALIGNED>(src + HALF + 8 * c)}};
  const void* weight = is_k ? a.k_weight : a.q_weight;
  const Eight<WEIGHT_FP32> w1 = load_eight<ALIGNED, WEIGHT_FP32>(weight, 8 * c);
  const Eight<WEIGHT_FP32> w2 = load_eight<ALIGNED, WEIGHT_FP32>(weight, HALF + 8 * c);
  const int64_t cs = t * a.cs_st + 8 * c, sn = t * a.sn_st + 8 * c;
  const Eight<ROWS_FP32> c1 = load_eight<ALIGNED, ROWS_FP32>(a.cos, cs), c2 = load_eight<ALIGNED, ROWS_FP32>(a.cos, cs + HALF);
  const Eight<ROWS_FP32> s1 = load_eight<ALIGNED, ROWS_FP32>(a.sin, sn), s2 = load_eight<ALIGNED, ROWS_FP32>(a.sin, sn + HALF);
  __builtin_amdgcn_sched_barrier(0);
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) sum = __builtin_fmaf(a1[i], a1[i], __builtin_fmaf(a2[i], a2[i], sum));
  sum = row_sum<RC>(sum);
  const float r = 1.f / sqrtf(sum * (1.f / D) + a.eps);
  float x1[8], x2[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float y1 = a1[i] * r * w1[i], y2 = a2[i] * r * w2[i];
    x1[i] = y1 * c1[i] - y2 * s1[i];
    x2[i] = y2 * c2[i] + y1 * s2[i];
  }
  if (!live || (is_k && !stored)) return;
  uint16_t* dst = is_k ? reinterpret_cast<uint16_t*>(a.k_cache) + slot * a.c_slot + head * a.c_head
                       : reinterpret_cast<uint16_t*>(a.out) + t * a.o_st + head * a.o_sh;
  store8<ALIGNED>(dst + 8 * c, narrow(x1));
  store8<ALIGNED>(dst + HALF + 8 * c, narrow(x2));
}

template <int D, bool ALIGNED, bool ROWS_FP32>
void launch(const QkNormRopeArgs& a, unsigned blocks, int32_t units, hipStream_t stream) {
  if (a.weight_fp32)
    hipLaunchKernelGGL((qk_norm_rope_kernel<D, ALIGNED, ROWS_FP32, true>), dim3(blocks), dim3(256), 0, stream, a, units);
  else
    hipLaunchKernelGGL((qk_norm_rope_kernel<D, ALIGNED, ROWS_FP32, false>), dim3(blocks), dim3(256), 0, stream, a, units);
}

template <int D>
hipError_t launch(const QkNormRopeArgs& a, hipStream_t stream) {
  constexpr int RPU = 64 / (D / 16), VPU = 64 / (D / 8);
  const int64_t units = ((int64_t)a.num_heads + a.num_kv_heads + RPU - 1) / RPU + (a.num_kv_heads + VPU - 1) / VPU;
  const int64_t blocks = (a.num_tokens * units + 3) / 4;
  if (units > 0x7fffffff || blocks > 0x7fffffff) return hipErrorInvalidValue;
  if (a.vec_ok && a.rows_fp32) launch<D, true, true>(a, (unsigned)blocks, (int32_t)units, stream);
  else if (a.vec_ok) launch<D, true, false>(a, (unsigned)blocks, (int32_t)units, stream);
  else if (a.rows_fp32) launch<D, false, true>(a, (unsigned)blocks, (int32_t)units, stream);
  else launch<D, false, false>(a, (unsigned)blocks, (int32_t)units, stream);
  return hipGetLastError();
}

}  // namespace

hipError_t qk_norm_rope_append(const QkNormRopeArgs& a, hipStream_t stream) {
  switch (a.head_dim) {
    case 64: return launch<64>(a, stream);
    case 128: return launch<128>(a, stream);
    case 256: return launch<256>(a, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace bvllm
