// Quantisers with a scale for a block: activations for each row and 128 columns (the operand of gemm_block.cu),
// keys and values for each page and head of a paged cache (the operand of cache_attn.cu).
//
// Both are bound by memory: two (four, gated) bytes a value in, one code out, 4 / 128 bytes of scales.
#include <cuda_runtime.h>

#include "../../include/iflb200.h"
#include "launch.cuh"
#include "rowmath.cuh"

namespace iflb200 {

constexpr int kQuantBlock = 128;
constexpr int kQuantThreads = 256;

// Eight values from memory: 16-byte loads where rows allow them, one by one up to `valid` otherwise.
template <bool VEC>
__device__ __forceinline__ void load_eight(const float* p, int valid, float (&v)[8]) {
  if (VEC) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < valid ? p[i] : 0.0f;
  }
}
template <bool VEC>
__device__ __forceinline__ void load_eight(const __nv_bfloat16* p, int valid, float (&v)[8]) {
  if (VEC) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < valid ? __bfloat162float(p[i]) : 0.0f;
  }
}
template <bool VEC>
__device__ __forceinline__ void load_eight(const __half* p, int valid, float (&v)[8]) {
  if (VEC) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < valid ? __half2float(p[i]) : 0.0f;
  }
}

struct BlockQuantArgs {
  const void* x;
  int64_t ld_x;
  int M, K, blocks;
  uint8_t* q;
  int64_t ld_q;
  float* qs;
  int64_t qs_row, qs_block;
};

// Sixteen lanes take a block of 128 columns, eight values each.  The maximum is taken of the bits of |v|: they order
// as the values do and put NaN on top, so that a block with a NaN gets the scale NaN.  Divisions are IEEE ones.
template <typename T, int ACT, bool VEC>
__global__ void __launch_bounds__(kQuantThreads) block_quant_kernel(const BlockQuantArgs a) {
  grid_dependency_wait();
  const int lane = threadIdx.x & 15;
  const int64_t groups = (int64_t)a.M * a.blocks;
  const int64_t g0 = ((int64_t)blockIdx.x * kQuantThreads + threadIdx.x) >> 4;
  const int64_t step = (int64_t)gridDim.x * (kQuantThreads / 16);
  // (whole warps stay in the loop: the exchange below is among sixteen lanes of a warp)
  for (int64_t g = g0; g - (threadIdx.x >> 4 & 1) < groups; g += step) {
    const bool in = g < groups;
    const int m = in ? (int)(g / a.blocks) : 0, b = in ? (int)(g - (int64_t)m * a.blocks) : 0;
    const int k = b * kQuantBlock + lane * 8;
    const int valid = in ? min(8, max(0, a.K - k)) : 0;
    float v[8] = {};
    if (VEC ? valid == 8 : valid > 0) {
      const T* row = reinterpret_cast<const T*>(a.x) + (int64_t)m * a.ld_x + k;
      load_eight<VEC>(row, valid, v);
      if (ACT >= 0) {
        float u[8];
        load_eight<VEC>(row + a.K, valid, u);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (ACT == IFLB200_ACT_SILU ? silu_ref(v[i]) : gelu_tanh_ref(v[i])) * u[i];
      }
    }
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
#pragma unroll
    for (int d = 8; d > 0; d >>= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
    const float amax = __uint_as_float(max(top, 0x322BCC77u));  // 1e-8
    const float inv = __fdiv_rn(448.0f, amax);
    if (valid > 0) {
      uint8_t* q = a.q + (int64_t)m * a.ld_q + k;
      const uint32_t lo = cvt_e4m3x4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
      const uint32_t hi = cvt_e4m3x4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
      if (VEC) {
        *reinterpret_cast<uint2*>(q) = make_uint2(lo, hi);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i < valid) q[i] = (uint8_t)((i < 4 ? lo : hi) >> (8 * (i & 3)));
      }
      if (lane == 0) a.qs[m * a.qs_row + b * a.qs_block] = __fdiv_rn(amax, 448.0f);
    }
  }
  grid_launch_dependents();
}

template <typename T, int ACT>
static int launch_block_quant(const BlockQuantArgs& a, cudaStream_t s) {
  const uintptr_t bytes = reinterpret_cast<uintptr_t>(a.x) | (uintptr_t)(a.ld_x * sizeof(T)) | (uintptr_t)(a.K * sizeof(T));
  const bool vec = a.K % 8 == 0 && bytes % 16 == 0 && (reinterpret_cast<uintptr_t>(a.q) | (uintptr_t)a.ld_q) % 8 == 0;
  const int64_t groups = (int64_t)a.M * a.blocks;
  const int sms = device_sm_count();
  if (sms == 0) return IFLB200_ERR_DEVICE;
  const int64_t want = (groups + kQuantThreads / 16 - 1) / (kQuantThreads / 16), most = (int64_t)sms * 8;
  const dim3 grid((unsigned)(want < most ? want : most));
  const bool dep = dependent_launch_for(a.M);
  const cudaError_t e = vec ? launch_dep(block_quant_kernel<T, ACT, true>, grid, dim3(kQuantThreads), 0, s, 1, dep, a)
                            : launch_dep(block_quant_kernel<T, ACT, false>, grid, dim3(kQuantThreads), 0, s, 1, dep, a);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

template <typename T>
static int launch_block_quant(const BlockQuantArgs& a, int act, cudaStream_t s) {
  if (act == IFLB200_ACT_GELU_TANH) return launch_block_quant<T, IFLB200_ACT_GELU_TANH>(a, s);
  if (act == IFLB200_ACT_SILU) return launch_block_quant<T, IFLB200_ACT_SILU>(a, s);
  return launch_block_quant<T, -1>(a, s);
}

// ---------------------------------------------------------------------------------------------
// New keys and values into the pages of an 8-bit cache.
//
// One CTA takes what falls into one page of one head of K or of V.  The scale is a power of two, the least one that
// brings the largest finite value to 448 or below, and never less than what the page had: e4m3 is a floating type, so
// a power of two costs no precision above its subnormals, and codes that are in the page already move to a larger
// scale without rounding (again above the subnormals).
// ---------------------------------------------------------------------------------------------
constexpr int kAppendThreads = 256;

struct AppendArgs {
  const void* src[2];
  int64_t sb[2], st[2], sh[2];  // strides of the new keys / values in elements
  uint8_t* codes[2];
  float* scale[2];
  const int32_t* table;
  int64_t ld_table;
  int max_pages, pages, heads, page_tokens, head_dim, T;
  const int32_t* start;
  const int32_t* counts;
};

// The least power of two that brings amax (>= 1e-8) to 448 = 1.75 * 2^8 or below.
__device__ __forceinline__ float page_scale(uint32_t amax_bits) {
  const uint32_t bits = max(amax_bits, 0x322BCC77u);  // 1e-8
  return __uint_as_float(((bits >> 23) - ((bits & 0x7FFFFFu) <= 0x600000u ? 8 : 7)) << 23);
}

__device__ __forceinline__ float2 e4m3x2_to_f32(uint32_t two) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)two));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kAppendThreads) cache_append_kernel(const AppendArgs a) {
  grid_dependency_wait();
  const int b = blockIdx.z, h = blockIdx.y, which = blockIdx.x & 1, span = blockIdx.x >> 1;
  const int P = a.page_tokens, D = a.head_dim;
  const int64_t start = a.start[b];
  const int count = a.counts ? min(max(a.counts[b], 0), a.T) : a.T;
  if (start < 0) return;
  const int64_t slot = start / P + span, at = slot * P;
  const int lo = (int)max((int64_t)0, start - at), hi = (int)min((int64_t)P, start + count - at);
  if (lo >= hi || slot >= a.max_pages) return;
  const int page = a.table[b * a.ld_table + slot];
  if (page < 0 || page >= a.pages) return;
  float* scale = a.scale[which] + (int64_t)page * a.heads + h;
  const float old = lo > 0 ? *scale : 0.0f;
  const T* src = reinterpret_cast<const T*>(a.src[which]) + b * a.sb[which] + (at - start) * a.st[which] + h * a.sh[which];
  const int64_t st = a.st[which];
  const int vecs = D / 8, n = (hi - lo) * vecs;
  uint32_t top = 0;
  for (int i = threadIdx.x; i < n; i += kAppendThreads) {
    float v[8];
    const int j = lo + i / vecs;
    load_eight<VEC>(src + j * st + (i - (i / vecs) * vecs) * 8, 8, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t bits = __float_as_uint(v[e]) & 0x7FFFFFFFu;
      top = max(top, bits < 0x7F800000u ? bits : 0u);
    }
  }
  __shared__ uint32_t tops[kAppendThreads / 32];
  top = __reduce_max_sync(0xFFFFFFFFu, top);
  if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kAppendThreads / 32; ++w) top = max(top, tops[w]);
  const float now = fmaxf(old, page_scale(top));
  uint8_t* codes = a.codes[which] + ((int64_t)page * a.heads + h) * P * D;
  const bool two = (__float_as_uint(now) & 0x7FFFFFu) == 0;  // (a scale of another origin need not be a power of two)
  const float inv = __fdiv_rn(1.0f, now);
  for (int i = threadIdx.x; i < n; i += kAppendThreads) {
    float v[8];
    const int j = lo + i / vecs, d = (i - (i / vecs) * vecs) * 8;
    load_eight<VEC>(src + j * st + d, 8, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = two ? v[e] * inv : __fdiv_rn(v[e], now);
      if (fabsf(v[e]) > 3e38f) v[e] = __uint_as_float(0x7FC00000u);  // an infinity is no e4m3 value: NaN
    }
    *reinterpret_cast<uint2*>(codes + j * D + d) =
        make_uint2(cvt_e4m3x4(v[0], v[1], v[2], v[3]), cvt_e4m3x4(v[4], v[5], v[6], v[7]));
  }
  if (lo > 0 && now > old) {
    const float ratio = __fdiv_rn(old, now);
    for (int i = threadIdx.x; i < lo * vecs; i += kAppendThreads) {
      uint2* at8 = reinterpret_cast<uint2*>(codes) + i;
      const uint2 u = *at8;
      const float2 p0 = e4m3x2_to_f32(u.x & 0xFFFF), p1 = e4m3x2_to_f32(u.x >> 16), p2 = e4m3x2_to_f32(u.y & 0xFFFF),
                   p3 = e4m3x2_to_f32(u.y >> 16);
      *at8 = make_uint2(cvt_e4m3x4(p0.x * ratio, p0.y * ratio, p1.x * ratio, p1.y * ratio),
                        cvt_e4m3x4(p2.x * ratio, p2.y * ratio, p3.x * ratio, p3.y * ratio));
    }
  }
  if (threadIdx.x == 0 && now != old) *scale = now;
  grid_launch_dependents();
}

template <typename T>
static int launch_append(const AppendArgs& a, int B, cudaStream_t s) {
  uintptr_t bytes = 0;
  for (int i = 0; i < 2; ++i)
    bytes |= reinterpret_cast<uintptr_t>(a.src[i]) | (uintptr_t)((a.sb[i] | a.st[i] | a.sh[i]) * (int64_t)sizeof(T));
  const int64_t spans = ((int64_t)a.T + a.page_tokens - 2) / a.page_tokens + 1;
  const dim3 grid((unsigned)(2 * spans), (unsigned)a.heads, (unsigned)B);
  const bool dep = dependent_launch_for((int64_t)B * a.T);
  const cudaError_t e = bytes % 16 == 0 ? launch_dep(cache_append_kernel<T, true>, grid, dim3(kAppendThreads), 0, s, 1, dep, a)
                                        : launch_dep(cache_append_kernel<T, false>, grid, dim3(kAppendThreads), 0, s, 1, dep, a);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

}  // namespace iflb200

using namespace iflb200;

extern "C" int iflb200_block_quant(const void* x, int x_dtype, int64_t ld_x, int M, int K, int act, void* q, int64_t ld_q,
                                   float* qs, int64_t qs_row, int64_t qs_block, void* stream) {
  if (M < 0 || K < 0) return IFLB200_ERR_ARG;
  if (act < -1 || act > IFLB200_ACT_SILU) return IFLB200_ERR_ARG;
  if (x_dtype != IFLB200_F32 && x_dtype != IFLB200_BF16 && x_dtype != IFLB200_F16) return IFLB200_ERR_DTYPE;
  if (M == 0 || K == 0) return IFLB200_OK;
  if (K > (1 << 29)) return IFLB200_ERR_SHAPE;
  if (!x || !q || !qs) return IFLB200_ERR_ARG;
  if (ld_x < (int64_t)K * (act >= 0 ? 2 : 1) || ld_q < K || qs_row < 0 || qs_block < 0) return IFLB200_ERR_ARG;
  BlockQuantArgs a = {x, ld_x, M, K, (K + kQuantBlock - 1) / kQuantBlock, reinterpret_cast<uint8_t*>(q), ld_q, qs, qs_row, qs_block};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (x_dtype == IFLB200_F32) return launch_block_quant<float>(a, act, s);
  if (x_dtype == IFLB200_BF16) return launch_block_quant<__nv_bfloat16>(a, act, s);
  return launch_block_quant<__half>(a, act, s);
}

extern "C" int iflb200_cache_append(const void* k, int64_t k_b, int64_t k_t, int64_t k_h, const void* v, int64_t v_b,
                                    int64_t v_t, int64_t v_h, int dtype, int B, int T, int heads, int head_dim, void* k_codes,
                                    void* v_codes, float* k_scale, float* v_scale, int pages, int page_tokens,
                                    const int32_t* table, int64_t ld_table, int max_pages, const int32_t* start,
                                    const int32_t* counts, void* stream) {
  if (B < 0 || T < 0 || heads < 1 || pages < 0 || max_pages < 0) return IFLB200_ERR_ARG;
  if (dtype != IFLB200_F32 && dtype != IFLB200_BF16 && dtype != IFLB200_F16) return IFLB200_ERR_DTYPE;
  if ((head_dim != 64 && head_dim != 128 && head_dim != 256) || page_tokens < 16 || page_tokens > 256 || page_tokens % 16 ||
      heads > 65535 || B > 65535 || T > (1 << 30))
    return IFLB200_ERR_SHAPE;
  if (B == 0 || T == 0 || pages == 0 || max_pages == 0) return IFLB200_OK;
  if (!k || !v || !k_codes || !v_codes || !k_scale || !v_scale || !table || !start) return IFLB200_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(k_codes) | reinterpret_cast<uintptr_t>(v_codes)) % 16) return IFLB200_ERR_ALIGN;
  AppendArgs a = {{k, v}, {k_b, v_b}, {k_t, v_t}, {k_h, v_h}, {reinterpret_cast<uint8_t*>(k_codes), reinterpret_cast<uint8_t*>(v_codes)},
                  {k_scale, v_scale}, table, ld_table, max_pages, pages, heads, page_tokens, head_dim, T, start, counts};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == IFLB200_F32) return launch_append<float>(a, B, s);
  if (dtype == IFLB200_BF16) return launch_append<__nv_bfloat16>(a, B, s);
  return launch_append<__half>(a, B, s);
}
