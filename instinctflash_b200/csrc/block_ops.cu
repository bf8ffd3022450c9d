// Quantisers with a scale for a block: activations for each row and 128 columns (the operand of gemm_block.cu),
// keys and values for each page and head of a paged cache (the operand of cache_attn.cu).
//
// Both are bound by memory: two (four, gated) bytes a value in, one code out, 4 / 128 bytes of scales.
#include <cuda_runtime.h>
#include <string.h>

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

// silu(g) * u for two elements, with ex2 and the reciprocal to an ulp or two.
__device__ __forceinline__ void silu_mul2(float& g0, float& g1, float u0, float u1) {
  float z0, z1;
  unpack2(mul2(pack2(g0, g1), pack2(-1.4426950408889634f, -1.4426950408889634f)), z0, z1);
  float d0, d1;
  unpack2(add2(pack2(ex2_approx_ftz(z0), ex2_approx_ftz(z1)), pack2(1.0f, 1.0f)), d0, d1);
  unpack2(mul2(mul2(pack2(g0, g1), pack2(rcp_approx_ftz(d0), rcp_approx_ftz(d1))), pack2(u0, u1)), g0, g1);
}

// Eight lanes take a block of 128 columns, twice eight neighbouring values each, so that every load and store of the eight
// is one piece of memory.  The maximum is taken of the bits of |v|: they order as the values do and put NaN on top, so
// that a block with a NaN gets the scale NaN.  Divisions are IEEE ones.
//
// B200, 816 x [16384 | 16384] bf16: 21.0 us with sixteen lanes a block and 64-bit index arithmetic, 13.7 us like this (66 MB:
// 10.3 at the copy rate); what is left is the activation, some 20 instructions a value.
template <typename T, int ACT, bool VEC>
__global__ void __launch_bounds__(kQuantThreads) block_quant_kernel(const BlockQuantArgs a) {
  grid_dependency_wait();
  const int lane = threadIdx.x & 7;
  const int groups = a.M * a.blocks, step = (int)gridDim.x * (kQuantThreads / 8);  // (checked on the host)
  // (whole warps stay in the loop: the exchange below is among eight lanes of a warp)
  for (int g = (int)blockIdx.x * (kQuantThreads / 8) + (threadIdx.x >> 3); g - (int)(threadIdx.x >> 3 & 3) < groups; g += step) {
    const bool in = g < groups;
    const int m = in ? (int)((unsigned)g / (unsigned)a.blocks) : 0, b = in ? g - m * a.blocks : 0;
    const int k = b * kQuantBlock + lane * 8;
    float v[2][8];
    int valid[2];
    const T* row = reinterpret_cast<const T*>(a.x) + (int64_t)m * a.ld_x;
#pragma unroll
    for (int z = 0; z < 2; ++z) {
      valid[z] = in ? min(8, max(0, a.K - k - 64 * z)) : 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) v[z][i] = 0.0f;
      if (VEC ? valid[z] == 8 : valid[z] > 0) load_eight<VEC>(row + k + 64 * z, valid[z], v[z]);
    }
    if (ACT >= 0) {
      float u[2][8];
#pragma unroll
      for (int z = 0; z < 2; ++z) {
#pragma unroll
        for (int i = 0; i < 8; ++i) u[z][i] = 0.0f;
        if (VEC ? valid[z] == 8 : valid[z] > 0) load_eight<VEC>(row + a.K + k + 64 * z, valid[z], u[z]);
      }
#pragma unroll
      for (int z = 0; z < 2; ++z) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          if (ACT == IFLB200_ACT_SILU) {
            silu_mul2(v[z][i], v[z][i + 1], u[z][i], u[z][i + 1]);
          } else {
            gelu_tanh_ref2(v[z][i], v[z][i + 1]);
            v[z][i] *= u[z][i];
            v[z][i + 1] *= u[z][i + 1];
          }
        }
      }
    }
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) top = max(top, __float_as_uint(v[i >> 3][i & 7]) & 0x7FFFFFFFu);
#pragma unroll
    for (int d = 4; d > 0; d >>= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
    const float amax = __uint_as_float(max(top, 0x322BCC77u));  // 1e-8
    const float inv = __fdiv_rn(448.0f, amax);
    const uint64_t inv2 = pack2(inv, inv);
#pragma unroll
    for (int z = 0; z < 2; ++z) {
      if (valid[z] > 0) {
        float c[8];
#pragma unroll
        for (int i = 0; i < 8; i += 2) unpack2(mul2(pack2(v[z][i], v[z][i + 1]), inv2), c[i], c[i + 1]);
        uint8_t* q = a.q + (int64_t)m * a.ld_q + k + 64 * z;
        const uint32_t lo = cvt_e4m3x4(c[0], c[1], c[2], c[3]), hi = cvt_e4m3x4(c[4], c[5], c[6], c[7]);
        if (VEC) {
          *reinterpret_cast<uint2*>(q) = make_uint2(lo, hi);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (i < valid[z]) q[i] = (uint8_t)((i < 4 ? lo : hi) >> (8 * (i & 3)));
        }
      }
    }
    if (lane == 0 && in) a.qs[m * a.qs_row + b * a.qs_block] = __fdiv_rn(amax, 448.0f);
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
  const int64_t want = (groups + kQuantThreads / 8 - 1) / (kQuantThreads / 8), most = (int64_t)sms * 8;
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

// Eight values as they lie in memory.
template <typename T>
struct Piece {
  uint4 w[sizeof(T) / 2];
  template <bool VEC>
  __device__ __forceinline__ void load(const T* p) {
    if (VEC) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = reinterpret_cast<const uint4*>(p)[i];
    } else {
      T x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = p[i];
      memcpy(w, x, sizeof(w));
    }
  }
  __device__ __forceinline__ void values(float (&v)[8]) const { load_eight<true>(reinterpret_cast<const T*>(w), 8, v); }
};

// Pieces stay in registers between the maximum and the codes, up to four a thread; a larger page reads the rest again.
template <typename T, int D, bool VEC>
__global__ void __launch_bounds__(kAppendThreads) cache_append_kernel(const AppendArgs a) {
  constexpr int VECS = D / 8, KEEP = 4;
  grid_dependency_wait();
  const int b = blockIdx.z, h = blockIdx.y, which = blockIdx.x & 1, span = blockIdx.x >> 1;
  const int P = a.page_tokens;
  const int64_t start = a.start[b];
  const int count = a.counts ? min(max(a.counts[b], 0), a.T) : a.T;
  if (start < 0) return;
  const int64_t slot = start / P + span, at = slot * P;
  const int lo = (int)max((int64_t)0, start - at), hi = (int)min((int64_t)P, start + count - at);
  if (lo >= hi || slot >= a.max_pages) return;
  const int page = a.table[b * a.ld_table + slot];
  const T* src = reinterpret_cast<const T*>(a.src[which]) + b * a.sb[which] + (at - start + lo) * a.st[which] + h * a.sh[which];
  const int64_t st = a.st[which];
  const int n = (hi - lo) * VECS;
  Piece<T> v[KEEP];
  uint32_t top = 0;
  auto highest = [&](const float (&x)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t bits = __float_as_uint(x[e]) & 0x7FFFFFFFu;
      top = max(top, bits < 0x7F800000u ? bits : 0u);
    }
  };
#pragma unroll
  for (int z = 0; z < KEEP; ++z) {
    const int i = threadIdx.x + z * blockDim.x;
    if (i < n) v[z].template load<VEC>(src + (i / VECS) * st + i % VECS * 8);
  }
  if (page < 0 || page >= a.pages) return;
  float* scale = a.scale[which] + (int64_t)page * a.heads + h;
  const float old = lo > 0 ? *scale : 0.0f;
#pragma unroll
  for (int z = 0; z < KEEP; ++z)
    if ((int)(threadIdx.x + z * blockDim.x) < n) {
      float x[8];
      v[z].values(x);
      highest(x);
    }
  for (int i = threadIdx.x + KEEP * blockDim.x; i < n; i += blockDim.x) {
    float x[8];
    load_eight<VEC>(src + (i / VECS) * st + i % VECS * 8, 8, x);
    highest(x);
  }
  __shared__ uint32_t tops[kAppendThreads / 32];
  top = __reduce_max_sync(0xFFFFFFFFu, top);
  if (blockDim.x > 32) {
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
    for (int w = 0; w < (int)blockDim.x / 32; ++w) top = max(top, tops[w]);
  } else {
    __syncwarp();  // (every lane has read the old scale before the first one writes the new)
  }
  const float now = fmaxf(old, page_scale(top));
  uint8_t* codes = a.codes[which] + ((int64_t)page * a.heads + h) * P * D;
  const bool two = (__float_as_uint(now) & 0x7FFFFFu) == 0;  // (a scale of another origin need not be a power of two)
  const float inv = __fdiv_rn(1.0f, now);
  auto write = [&](int i, float (&x)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = two ? x[e] * inv : __fdiv_rn(x[e], now);
      if (fabsf(x[e]) > 3e38f) x[e] = __uint_as_float(0x7FC00000u);  // an infinity is no e4m3 value: NaN
    }
    *reinterpret_cast<uint2*>(codes + lo * D + i * 8) = make_uint2(cvt_e4m3x4(x[0], x[1], x[2], x[3]), cvt_e4m3x4(x[4], x[5], x[6], x[7]));
  };
#pragma unroll
  for (int z = 0; z < KEEP; ++z) {
    const int i = threadIdx.x + z * blockDim.x;
    if (i < n) {
      float x[8];
      v[z].values(x);
      write(i, x);
    }
  }
  for (int i = threadIdx.x + KEEP * blockDim.x; i < n; i += blockDim.x) {
    float x[8];
    load_eight<VEC>(src + (i / VECS) * st + i % VECS * 8, 8, x);
    write(i, x);
  }
  if (lo > 0 && now > old) {
    const float ratio = __fdiv_rn(old, now);
    for (int i = threadIdx.x; i < lo * VECS; i += blockDim.x) {
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

template <typename T, int D>
static cudaError_t launch_append(const AppendArgs& a, bool vec, const dim3& grid, int threads, bool dep, cudaStream_t s) {
  return vec ? launch_dep(cache_append_kernel<T, D, true>, grid, dim3(threads), 0, s, 1, dep, a)
             : launch_dep(cache_append_kernel<T, D, false>, grid, dim3(threads), 0, s, 1, dep, a);
}

template <typename T>
static int launch_append(const AppendArgs& a, int B, cudaStream_t s) {
  uintptr_t bytes = 0;
  for (int i = 0; i < 2; ++i)
    bytes |= reinterpret_cast<uintptr_t>(a.src[i]) | (uintptr_t)((a.sb[i] | a.st[i] | a.sh[i]) * (int64_t)sizeof(T));
  const int64_t spans = ((int64_t)a.T + a.page_tokens - 2) / a.page_tokens + 1;
  const dim3 grid((unsigned)(2 * spans), (unsigned)a.heads, (unsigned)B);
  const bool dep = dependent_launch_for((int64_t)B * a.T), vec = bytes % 16 == 0;
  // as many threads as a page gets pieces of eight values; one warp needs no barrier
  const int pieces = (a.T < a.page_tokens ? a.T : a.page_tokens) * a.head_dim / 8;
  const int threads = pieces >= kAppendThreads ? kAppendThreads : (pieces + 31) / 32 * 32;
  const cudaError_t e = a.head_dim == 64 ? launch_append<T, 64>(a, vec, grid, threads, dep, s)
                                         : (a.head_dim == 128 ? launch_append<T, 128>(a, vec, grid, threads, dep, s)
                                                              : launch_append<T, 256>(a, vec, grid, threads, dep, s));
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
  if (K > (1 << 29) || (int64_t)M * ((K + kQuantBlock - 1) / kQuantBlock) > (1ll << 31) - (1 << 24)) return IFLB200_ERR_SHAPE;
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
