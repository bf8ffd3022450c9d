// What the two forms of attention over the 8-bit cache share (cache_attn.cu, cache_attn_tiles.cu).
#pragma once
#include <cuda_runtime.h>

#include "../../include/iflb200.h"
#include "launch.cuh"
#include "rowmath.cuh"

namespace iflb200 {

struct AttendArgs {
  const void* q;
  int64_t q_b, q_t, q_h;
  void* out;
  int64_t o_b, o_t, o_h;
  const uint8_t* k;
  const uint8_t* v;
  const float* ks;
  const float* vs;
  const int32_t* table;
  int64_t ld_table;
  const int32_t* lens;
  const int32_t* q_lens;
  const int32_t* prefix;
  const float* slopes;
  float scale, cap;
  int B, T, HQ, H, G, P, pages, max_pages, causal;
  int row_tiles, chunk, splits;     // keys of a chunk; most chunks a sequence can have
  uint32_t* tickets;                // one for each (sequence, head and row tile), zero between calls
  float* partial;                   // [ticket][chunk][rows][D], then [ticket][chunk][rows][2]
  int64_t partial_ml;               // floats ahead of the second part
};

constexpr float kLog2e = 1.4426950408889634f;
// The value scale is part of the exponent.  A scale of zero counts as 2^-60 there, so that its weights, whose values are zeros, take
// no bits from others'.
constexpr float kNilLog2 = -60.0f, kNilInverse = 1152921504606846976.0f;
// Weights enter the product as f16.  The running maximum's is 2^10: a weight keeps eleven bits down to 2^-24 of it and half a step of
// f16's subnormals, 2^-35 of it, below (with the maximum at 1 a tail of 2^-22 came out wrong in its third digit, one of 2^-26 was
// lost).  A page with a large value scale would take these bits from the other pages', which still are all there is in columns where
// it has zeros.  So units whose scale is more than 2^6 below the largest one so far get weights with a maximum of their own (few
// rows), or a pass over the keys for each 2^6 of scales, from the lowest up (row tiles): no weight is off by more than 2^-11 of it or
// 2^-28 of its row's largest probability, whatever the scales.
constexpr float kWeightTop = 10.0f;
constexpr float kLazy = 5.0f;  // base-2 exponent by which a score may pass the running maximum before it moves: to 2^15
constexpr float kFar = 6.0f;

// cap * tanh(s / cap).  tanh(x) = 1 - 2 / (1 + e^2x) is off by 1e-7 of 1; near zero, where that is more than fp32 keeps
// of the result, the series (next term below 1e-7 of x at 1/4).
__device__ __forceinline__ float soft_cap(float s, float cap, float inv_cap) {
  const float x = s * inv_cap;
  const float y = x * x;
  const float near = x + x * y * (-0.33333333f + y * (0.13333333f + y * (-0.053968254f + y * 0.021869489f)));
  const float far = 1.0f - 2.0f * rcp_approx_ftz(1.0f + ex2_approx_ftz(2.0f * kLog2e * x));
  return cap * (fabsf(x) < 0.25f ? near : far);
}

__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float as_float(__half x) { return __half2float(x); }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }

__device__ __forceinline__ float log2_approx(float a) {
  float r;
  asm("lg2.approx.f32 %0, %1;" : "=f"(r) : "f"(a));
  return r;
}
// Two e4m3 codes in the low half of `two` as two f16 (exact).
__device__ __forceinline__ uint32_t e4m3x2_f16x2(uint32_t two) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)two));
  return r;
}
__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// The form for many rows: (query token, head of the group) rows in tiles on tcgen05.  splits: key ranges, as in AttendArgs.
int attend_tiles_rows(int head_dim);  // rows of a CTA
template <typename T>
int launch_attend_tiles(const AttendArgs& a, int head_dim, cudaStream_t s);

}  // namespace iflb200
