// Attention over the paged 8-bit cache for many rows: row tiles of 128 (query token x head of a group) on tcgen05.
//
// One CTA has NQ row tiles of one key/value head and walks its keys BN at a time.  Per step and row tile
//
//   S = Q K^T            128 x BN x D, operands f16 in shared memory, S fp32 in tensor memory
//   y = S * (factor of the row * ks) + log2 vs       base-2 exponents, masked at the edge
//   P = 2^(y - M + 10) as f16 into tensor memory     M: the row's running maximum of y, 10: kWeightTop
//   O += P V             128 x D x BN, P from tensor memory, V f16 in shared memory, O fp32 in tensor memory
//
// The value scale of a page is part of the exponent, so that O needs no scale of its own: with l = sum 2^(y - M + 10) / vs
// the output is O / l.  M moves only when a score passes it by more than 2^5, which is what f16 has room for, since O in tensor
// memory has to be multiplied then.
//
// Codes become f16 on the way into shared memory (exact): a 16-bit operand of the same MMA rate as two 8-bit halves of q
// and P would have, with 11 bits of P and no work on P but its rounding.  The MMA takes the values [key][D] as they lie
// (transposed B operand).
//
//   warp 0               MMA issuer, tensor memory (the first warp: behind the others' work it issued an MMA every 300 clocks)
//   warps 4..7, 8..11    softmax, one row a thread, and the output (D 256 has one row tile, whose S has two buffers instead)
//   warps 12..19         codes from global memory through registers to f16 tiles, one tile ahead; a step's scales
#include "bounded_wait.cuh"
#include "cache_attn.cuh"

namespace iflb200 {

namespace {

constexpr int kConvert = 8;  // converter warps
constexpr int kThreads = 32 * (12 + kConvert);

template <int D>
struct Tiles {
  static constexpr int BN = D == 256 ? 64 : 128;   // keys of a step
  static constexpr int NQ = D == 256 ? 1 : 2;      // row tiles of a CTA
  static constexpr int ROWS = 128 * NQ;
  static constexpr int GR = BN / 16;               // units of sixteen keys, which lie in one page
  // Tensor memory: scores of the two slots (row tiles, or every other step), weights, output.  Products are only ordered among
  // those of one shape into one accumulator, so the scores that follow must not be written over weights that a product may still
  // be reading: they have columns of their own, but for D 128, where the MMA issuer waits for the product instead.
  static constexpr bool kOver = D == 128;
  static constexpr uint32_t kS = 0, kO = 256, kP = D == 64 ? 384 : (D == 256 ? 128 : 0), kPStride = kOver ? BN : BN / 2;
  static constexpr int kQ = 128 * D * 2, kTile = BN * D * 2;  // bytes
  static constexpr int kMeta = NQ * kQ + 4 * kTile;
  static constexpr int kNan = kMeta + 4 * GR * 16;
  static constexpr int kOff = kNan + D * 4 + 16;          // each converter warp's units of two steps: offset of the codes
  static constexpr int kHole = kOff + kConvert * 2 * GR * 8;  // of four steps: whether a unit has no page
  static constexpr int kFactor = kHole + 16;              // of each row of q
  static constexpr int kBar = kFactor + ROWS * 4;         // barriers, address of the tensor memory, abort, bands of value scales
  static constexpr int kSmem = kBar + 24 * 8 + 16 + 1024;
};

__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_16c(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// f16 operands, fp32 result; `mn_b`: the B operand lies with its N side contiguous
__host__ __device__ constexpr uint32_t idesc_f16(int m, int n, bool mn_b) {
  return (1u << 4) | (mn_b ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// An operand whose N side is contiguous: rows (one for each k) of 64 f16 under the 128-byte swizzle, eight rows an atom; the
// next eight rows 1024 bytes on, the next 64 columns `step` bytes on.
__device__ __forceinline__ uint64_t make_mnmajor_desc(uint32_t smem_addr, uint32_t step) {
  return make_kmajor_sw128_desc(smem_addr) | ((uint64_t)(step >> 4) << 16);
}
__device__ __forceinline__ void sts128(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ float4 lds_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float row_value(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float row_value(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ uint32_t pack_out(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack_out<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack_out<__half>(float a, float b) {
  return pack_half2(a, b);
}

// Sixteen codes of key `key` without their NaNs, whose columns learn of the first key that has one.  (Out of line: it is
// hardly ever run.)
__device__ __noinline__ uint4 without_nans(uint4 codes, int* first_nan, int key) {
  uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll 1
  for (int e = 0; e < 16; ++e) {
    const uint32_t at = e >> 2, shift = 8 * (e & 3);
    const uint32_t word = at == 0 ? w[0] : (at == 1 ? w[1] : (at == 2 ? w[2] : w[3]));
    if ((word >> shift & 0x7F) == 0x7F) {
      atomicMin(first_nan + e, key);
#pragma unroll
      for (uint32_t z = 0; z < 4; ++z)
        if (z == at) w[z] &= ~(0xFFu << shift);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// CAP, SLOPES: whether the scores are capped, and get a bias by distance; kernels of their own, for the size of the code.
template <int D, typename T, bool CAP, bool SLOPES>
__global__ void __launch_bounds__(kThreads, 1) cache_attend_tiles_kernel(const __grid_constant__ AttendArgs a, const int vec) {
  using L = Tiles<D>;
  constexpr int BN = L::BN, NQ = L::NQ, GR = L::GR;
  constexpr uint32_t kS = L::kS, kO = L::kO;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t base = (raw_addr + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw_addr);
  const uint32_t q_at = base, k_at = base + NQ * L::kQ, v_at = k_at + 2 * L::kTile, meta = base + L::kMeta, bar0 = base + L::kBar;
  int* nan_at = reinterpret_cast<int*>(smem + L::kNan);  // for each element of D the first key whose value is a NaN there
  volatile int* nan_any = nan_at + D;
  float* row_factor = reinterpret_cast<float*>(smem + L::kFactor);
  enum { KFULL = 0, KEMPTY = 2, VFULL = 4, VEMPTY = 6, SFULL = 8, PFULL = 10, PV = 12, QFULL = 14 };
  auto bar = [&](int kind, int i) { return bar0 + 8u * (kind + i); };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kBar + 24 * 8);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  volatile uint32_t* far_bands = tmem_slot + 2;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // (the last row tiles first: under a causal mask they have the most keys)
  const int split = blockIdx.x, y = gridDim.y - 1 - blockIdx.y, b = blockIdx.z;
  const int h = y / a.row_tiles, row0 = (y - h * a.row_tiles) * L::ROWS;
  grid_dependency_wait();
  const int len = min(max(a.lens[b], 0), (int)min((int64_t)a.max_pages * a.P, (int64_t)INT32_MAX));
  const int nq = a.q_lens ? min(max(a.q_lens[b], 0), a.T) : a.T;
  const int rows = min(L::ROWS, nq * a.G - row0);
  if (rows <= 0) return;
  const int prefix = a.prefix ? a.prefix[b] : 0;
  auto limit_of = [&](int r) { return a.causal ? min(len, max(len - nq + r / a.G + 1, prefix)) : len; };
  const int most = max(0, limit_of(row0 + rows - 1));
  const int chunks = max(1, (most + a.chunk - 1) / a.chunk);
  if (split >= chunks) return;
  const int key0 = split * a.chunk, key1 = min(most, key0 + a.chunk);
  const int steps = (key1 - key0 + BN - 1) / BN;
  // With slopes steps go from the last keys to the first: the maximum is among the nearest keys, and stays (from the first key on it
  // moved at every step: 2048 tokens behind 6144, 32 heads, 507 us, 420 like this).  Without them from the first keys on: a row that
  // sees few keys of its first step has its maximum moved within the next one (from the last on 381 us, 367 like this; 1024 tokens,
  // 16 heads of 64 over 4096 keys 67.6 and 63.5).  Head dim 256 goes from the last on all the same (four times 256 tokens over 4096
  // keys: 174 us, 181 from the first on).
  constexpr bool kBackward = SLOPES || D == 256;
  auto key_of = [&](int step) { return key0 + (kBackward ? steps - 1 - step : step) * BN; };

  auto start_barriers = [&]() {
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(KFULL, i), kConvert);
      mbar_init(bar(KEMPTY, i), 1);
      mbar_init(bar(VFULL, i), kConvert);
      mbar_init(bar(VEMPTY, i), 1);
      mbar_init(bar(SFULL, i), 1);
      mbar_init(bar(PFULL, i), 4);
      mbar_init(bar(PV, i), 1);
    }
  };
  if (threadIdx.x == 0) {
    start_barriers();
    mbar_init(bar(QFULL, 0), 8);
    tmem_slot[1] = 0;
    *far_bands = 0;
    *nan_any = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  for (int i = threadIdx.x; i < D; i += kThreads) nan_at[i] = INT32_MAX;
  __syncwarp();
  if (warp == 0) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // Passes over the keys.  The first one takes all; where it found value scales more than 2^kFar apart it is forgotten, and there is
  // one for each band of 2^kFar that has a scale, from the lowest up, into the same sums (see kWeightTop).  Between passes no MMA and
  // no arrival is on its way: the last product has been waited for, and a slot is only given back where a later step waits for it.
  // 2048 tokens behind 6144, 32 heads: 395 us, 1245 with a third of the pages 2^8 or 2^27 below the rest (three passes); few rows
  // lose 2 % by it (32 sequences of up to 8192 keys, one token: 88 and 90 us).
  int band = -1;            // of value scales; -1: all
  uint32_t bands = 0;       // that are still to come
  auto band_of = [](float log2_scale) { return min(max((int)floorf((log2_scale + 96.0f) * (1.0f / kFar)), 0), 31); };
  auto next_pass = [&]() {  // every warp, converged; the same answer for all
    tc_fence_before();
    named_bar_sync(2, kThreads);
    if (band < 0) bands = *far_bands;
    if (bands == 0 || *abort_flag) return false;
    band = __ffs(bands) - 1;
    bands &= bands - 1;
    if (threadIdx.x == 0) {
      for (int i = 0; i < QFULL; ++i) mbar_inval(bar(i, 0));
      start_barriers();
      fence_barrier_init();
      fence_proxy_async_smem();
    }
    named_bar_sync(2, kThreads);
    tc_fence_after();
    return true;
  };

  if (warp >= 4 && warp < 12) {
    // The rows of q as f16, each row's largest element near 2^15: eight warps, LR lanes a row, eight loads in flight.
    constexpr int LR = D / 8, RI = 32 / LR, RW = L::ROWS / 8;
    const int piece = lane % LR, from = (warp - 4) * RW;
#pragma unroll 1
    for (int i0 = 0; i0 < RW; i0 += 8 * RI) {
      uint4 x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int rr = from + i0 + i * RI + lane / LR, row = row0 + (rr < rows ? rr : 0);
        const int t = row / a.G;
        const T* q = reinterpret_cast<const T*>(a.q) + b * a.q_b + t * a.q_t + (h * a.G + row - t * a.G) * a.q_h + 8 * piece;
        if (vec) {
          x[i] = *reinterpret_cast<const uint4*>(q);
        } else {
          const uint16_t* u = reinterpret_cast<const uint16_t*>(q);
          x[i] = make_uint4(u[0] | (uint32_t)u[1] << 16, u[2] | (uint32_t)u[3] << 16, u[4] | (uint32_t)u[5] << 16, u[6] | (uint32_t)u[7] << 16);
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float v[8], top = 0.0f;
        const T* e8 = reinterpret_cast<const T*>(&x[i]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[e] = row_value(e8[e]);
          if (fabsf(v[e]) < 3.39e38f) top = fmaxf(top, fabsf(v[e]));
        }
        if (LR == 32) {
          top = __uint_as_float(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(top)));
        } else {
#pragma unroll
          for (int z = 1; z < LR; z <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, z));
        }
        const int e2 = max((int)(__float_as_uint(top) >> 23), 16);  // (as in cache_attn.cu)
        const float down = __uint_as_float((uint32_t)(269 - e2) << 23);
        const int rr = from + i0 + i * RI + lane / LR, r128 = rr & 127;
        if (piece == 0) row_factor[rr] = __uint_as_float((uint32_t)(e2 - 15) << 23) * a.scale;
        sts128(q_at + (rr >> 7) * L::kQ + (piece >> 3) * 128 * 128 + r128 * 128 + (((piece & 7) ^ (r128 & 7)) << 4),
               pack_half2(v[0] * down, v[1] * down), pack_half2(v[2] * down, v[3] * down), pack_half2(v[4] * down, v[5] * down),
               pack_half2(v[6] * down, v[7] * down));
      }
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(QFULL, 0));
    named_bar_sync(1, 256);
  }
  if (warp >= 4 && warp < 4 + 4 * NQ) {
    // ------------------------------------------------------------------ softmax and output
    const int slot = (warp >> 2) - 1;
    const int r = slot * 128 + (warp & 3) * 32 + lane;
    const bool in = r < rows;
    const int tok = (row0 + (in ? r : 0)) / a.G, hq = h * a.G + (row0 + (in ? r : 0)) - tok * a.G;
    const int limit = in ? limit_of(row0 + r) : INT32_MAX;  // (a row that is not there needs no mask)
    const int least = __reduce_min_sync(0xFFFFFFFFu, limit);
    const int pos = len - nq + tok;
    const float slope = SLOPES ? a.slopes[hq] * kLog2e : 0.0f;
    const float inv_cap = CAP ? 1.0f / a.cap : 0.0f;
    const float factor = row_factor[r];
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t o_at = tmem + lanes + kO + slot * D;
    float top_run = -INFINITY, l = 0.0f;
    bool ok = true, fresh = true;  // fresh: nothing in O yet
    for (;;) {
      for (int j = 0; j < steps; ++j) {
        float drop = 1.0f;   // what O has to be multiplied by ahead of this step's product: a power of two
        const int buf = NQ == 2 ? slot : j & 1;
        const uint32_t phase = NQ == 2 ? j & 1u : (j >> 1) & 1u;
        const uint32_t s_at = tmem + lanes + kS + buf * BN, p_at = tmem + lanes + L::kP + buf * L::kPStride;
        ok = wait_warp(bar(SFULL, buf), phase, abort_flag, (1u << 24) | (1u << 16) | (j & 0xFFFF));
        if (!ok) break;
        tc_fence_after();
        const uint32_t m_at = meta + (j & 3) * GR * 16;  // of each unit: ks, log2 vs, 1 / vs, 0 where there is no page
        const int key = key_of(j);
        const bool edge = key + BN > least || *reinterpret_cast<volatile int*>(smem + L::kHole + (j & 3) * 4) != 0;
        float4 m0, m1;
        // Exponents of 32 columns (two units).  Everything here is a loop over 32 columns that is not unrolled: the parts of this
        // kernel that run at the same time have to fit the instruction cache together.  With 128 columns unrolled an MMA was
        // issued every 300 clocks (2048 tokens behind 6144, 32 heads: 746 us then, 495 rolled up; 383 with the steps since).
        auto exponents = [&](int i, uint32_t (&v)[32]) {
          tmem_ld_32x32b_x32(s_at + 32 * i, v);
          m0 = lds_f4(m_at + 32 * i);
          m1 = lds_f4(m_at + 32 * i + 16);
          const float f0 = factor * m0.x * (CAP ? 1.0f : kLog2e), f1 = factor * m1.x * (CAP ? 1.0f : kLog2e);
          const float base = (top_run == -INFINITY ? 0.0f : top_run) - kWeightTop, c0 = m0.y - base, c1 = m1.y - base;
          tmem_ld_wait();
          if (CAP) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              v[e] = __float_as_uint(fmaf(soft_cap(__uint_as_float(v[e]) * (e < 16 ? f0 : f1), a.cap, inv_cap), kLog2e, e < 16 ? c0 : c1));
          } else {
            const uint64_t f[2] = {pack2(f0, f0), pack2(f1, f1)}, c[2] = {pack2(c0, c0), pack2(c1, c1)};
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              float p0, p1;
              unpack2(fma2(pack2(__uint_as_float(v[e]), __uint_as_float(v[e + 1])), f[e >> 4], c[e >> 4]), p0, p1);
              v[e] = __float_as_uint(p0);
              v[e + 1] = __float_as_uint(p1);
            }
          }
          if (SLOPES) {
            const float from = (float)(pos - key - 32 * i);  // (whole numbers first: beyond 2^24 positions are no floats)
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(fmaf(-slope, fabsf(from - (float)e), __uint_as_float(v[e])));
          }
          if (edge) {
            const int n = limit - key - 32 * i, n0 = m0.w == 0.0f ? 0 : n, n1 = m1.w == 0.0f ? 0 : n;
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (e >= (e < 16 ? n0 : n1)) v[e] = 0xFF800000u;
          }
          float high[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int e = 0; e < 32; e += 2) high[e >> 1 & 3] = max3(high[e >> 1 & 3], __uint_as_float(v[e]), __uint_as_float(v[e + 1]));
          return fmaxf(max3(high[0], high[1], high[2]), high[3]);
        };
        // O may change once the product of the step before is complete, and every phase of its barrier is waited for in turn.
        auto settle = [&]() {
          if (j > 0) ok = wait_warp(bar(PV, slot), (j - 1) & 1u, abort_flag, (1u << 24) | (2u << 16) | (j & 0xFFFF));
          tc_fence_after();
          if (ok && __any_sync(0xFFFFFFFFu, drop != 1.0f)) {
            if (j > 0 || !fresh) {
#pragma unroll 1
              for (int i = 0; i < D / 16; ++i) {
                uint32_t o[16];
                tmem_ld_16c(o_at + 16 * i, o);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * drop);
                tmem_st_16(o_at + 16 * i, o);
              }
              tmem_st_wait();
            }
            drop = 1.0f;
          }
        };
        // A row without a maximum yet gets that of these scores.
        if (__any_sync(0xFFFFFFFFu, top_run == -INFINITY)) {
          float first = -INFINITY;
          const bool none = top_run == -INFINITY;
#pragma unroll 1
          for (int i = 0; i < BN / 32; ++i) {
            uint32_t v[32];
            first = fmaxf(first, exponents(i, v));
          }
          if (none) top_run = first - kWeightTop;
        }
        // The weights, relative to the maximum of the steps before.
#pragma unroll 1
        for (int i = 0; i < BN / 32; ++i) {
          uint32_t v[32];
          float now = exponents(i, v);
          uint32_t w[16];
          uint64_t t[2];
          for (;;) {  // (as a rule once; the exponentials do not wait for the vote: without slopes 377 us with it ahead, 362 like this)
            t[0] = t[1] = 0;
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              const float p0 = ex2_approx_ftz(__uint_as_float(v[e])), p1 = ex2_approx_ftz(__uint_as_float(v[e + 1]));
              t[e >> 4] = add2(t[e >> 4], pack2(p0, p1));
              w[e / 2] = pack_half2(p0, p1);
            }
            if (__builtin_expect(!__any_sync(0xFFFFFFFFu, now > kWeightTop + kLazy), 1)) break;
            // more than f16 has: the maximum moves by a whole power of two, and all there is down, the weights of this step that are
            // stored already too (in fp32: f16 may not have the factor)
            const float by = now > kWeightTop + kLazy ? ceilf(now - kWeightTop) : 0.0f, f = ex2_approx_ftz(-by);
            if (by > 0.0f) top_run += by;
            now -= by;
            l *= f;
            drop *= f;
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) - by);
            tmem_st_wait();
#pragma unroll 1
            for (int z = 0; z < i; ++z) {
              uint32_t u[16];
              tmem_ld_16c(p_at + 16 * z, u);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&u[e]));
                u[e] = pack_half2(p.x * f, p.y * f);
              }
              tmem_st_16(p_at + 16 * z, u);
            }
          }
          float t0, t1;
          unpack2(t[0], t0, t1);
          l = fmaf(t0 + t1, m0.z, l);
          unpack2(t[1], t0, t1);
          l = fmaf(t0 + t1, m1.z, l);
          // (over scores that have been read, where the weights have no columns of their own)
          tmem_st_16(p_at + 16 * i, w);
        }
        settle();
        if (!ok) break;
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(PFULL, buf));
      }
      if (ok && steps > 0) ok = wait_warp(bar(PV, slot), (steps - 1) & 1u, abort_flag, (1u << 24) | (3u << 16));
      fresh = band < 0;
      if (!next_pass()) break;
      if (fresh) top_run = -INFINITY, l = 0.0f;
    }
    tc_fence_after();
    // The output through shared memory (this row tile of q is done with), 2 D bytes of each row at a time: whole rows go to
    // memory, where a row a thread would write half sectors.
    const bool any_nan = *nan_any != 0, partial = chunks > 1;
    const float inv = partial ? 1.0f : (l == 0.0f ? 0.0f : 1.0f / l);
    const uint32_t stage = q_at + slot * L::kQ + (warp & 3) * 32 * 2 * D;
    const int64_t at = ((int64_t)(b * a.H * a.row_tiles + y) * a.splits + split) * L::ROWS;
    constexpr int PR = D / 8;  // 16-byte pieces of a row
#pragma unroll 1
    for (int pass = 0; pass < (partial ? 2 : 1); ++pass) {
      __syncwarp();
#pragma unroll 1
      for (int i = 0; i < (partial ? D / 32 : D / 16); ++i) {
        const int col = pass * (D / 2) + 16 * i;
        uint32_t o[16];
        if (steps > 0) {
          tmem_ld_16c(o_at + col, o);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = 0;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float x = __uint_as_float(o[e]) * inv;
          if (any_nan && nan_at[col + e] < limit) x = __uint_as_float(0x7FC00000u);
          o[e] = __float_as_uint(x);
        }
        const uint32_t row_at = stage + lane * 2 * D;
        if (partial) {
#pragma unroll
          for (int z = 0; z < 4; ++z) sts128(row_at + (((4 * i + z) ^ (lane & 7)) << 4), o[4 * z], o[4 * z + 1], o[4 * z + 2], o[4 * z + 3]);
        } else {
          uint32_t w[8];
#pragma unroll
          for (int z = 0; z < 8; ++z) w[z] = pack_out<T>(__uint_as_float(o[2 * z]), __uint_as_float(o[2 * z + 1]));
#pragma unroll
          for (int z = 0; z < 2; ++z) sts128(row_at + (((2 * i + z) ^ (lane & 7)) << 4), w[4 * z], w[4 * z + 1], w[4 * z + 2], w[4 * z + 3]);
        }
      }
      __syncwarp();
#pragma unroll 4
      for (int i = lane; i < 32 * PR; i += 32) {
        const int rw = i / PR, piece = i % PR, rr = slot * 128 + (warp & 3) * 32 + rw;
        const float4 f = lds_f4(stage + rw * 2 * D + ((piece ^ (rw & 7)) << 4));
        if (rr < rows && ok) {
          if (partial) {
            *reinterpret_cast<float4*>(a.partial + (at + rr) * D + pass * (D / 2) + piece * 4) = f;
          } else {
            const int t = (row0 + rr) / a.G;
            T* dst = reinterpret_cast<T*>(a.out) + b * a.o_b + t * a.o_t + (h * a.G + row0 + rr - t * a.G) * a.o_h + piece * 8;
            if (vec) {
              *reinterpret_cast<float4*>(dst) = f;
            } else {
              const T* e8 = reinterpret_cast<const T*>(&f);
#pragma unroll
              for (int e = 0; e < 8; ++e) dst[e] = e8[e];
            }
          }
        }
      }
    }
    if (partial && in) *reinterpret_cast<float2*>(a.partial + a.partial_ml + (at + r) * 2) = make_float2(top_run, l);
  } else if (warp >= 12) {
    // ------------------------------------------------------------------ codes to f16 tiles
    constexpr int CH = D / 16, UN = BN * CH / (32 * kConvert), TPI = 32 * kConvert / CH;  // chunks of a key, chunks a thread, keys apart
    // Eight lanes store four pieces of one key and four of the next, which the swizzle puts on other banks.
    const int tid = threadIdx.x - 384, chunk = (tid & 3) | ((tid >> 3) & (CH / 4 - 1)) << 2, first = (tid >> 2 & 1) | (tid >> 3) / (CH / 4) << 1;
    const int32_t* table = a.table + b * a.ld_table;
    auto raw_page = [&](int step) {  // of this lane's unit of the step
      const int key = key_of(step) + 16 * lane;
      return lane < GR && step < steps && key < key1 ? __ldg(table + key / a.P) : -1;
    };
    int page = raw_page(0), page_next = raw_page(1);
    float ks = 0.0f, vs = 0.0f;
    bool there = false, fresh = true;  // fresh: no band has been taken yet
    float lowest = INFINITY, highest = -INFINITY;  // of this lane's units' value scales, to base 2
    uint32_t seen = 0;                             // their bands
    // Where the units of a step lie, through shared memory to the warp's lanes; -1: no page.
    int64_t* offs = reinterpret_cast<int64_t*>(smem + L::kOff) + (warp - 12) * 2 * GR;
    auto look_up = [&](int step) {
      there = page >= 0 && page < a.pages;
      const int key = key_of(step) + 16 * lane;
      if (band >= 0 && there) {  // what is not of the band counts as no page (zero scales: of the first one)
        const float scale = __ldg(a.vs + (int64_t)page * a.H + h);
        there = scale == 0.0f ? fresh : band_of(log2_approx(scale)) == band;
      }
      if (lane < GR) offs[(step & 1) * GR + lane] = there ? (((int64_t)page * a.H + h) * a.P + key % a.P) * D : -1;
      ks = there ? __ldg(a.ks + (int64_t)page * a.H + h) : 0.0f;
      vs = there ? __ldg(a.vs + (int64_t)page * a.H + h) : 0.0f;
      __syncwarp();
    };
    uint4 kr[UN], vr[UN];
    // (what is not there is read at the cache's beginning and made zero: no branch around a load)
    auto load = [&](const uint8_t* codes, int step, uint4 (&r)[UN]) {
#pragma unroll
      for (int i = 0; i < UN; ++i) {
        const int t = i * TPI + first;
        const int64_t o = offs[(step & 1) * GR + (t >> 4)];
        const bool in = o >= 0 && key_of(step) + t < key1;
        r[i] = __ldg(reinterpret_cast<const uint4*>(codes + (in ? o + (t & 15) * D : 0) + chunk * 16));
        if (!in) r[i] = make_uint4(0, 0, 0, 0);
      }
    };
    auto write = [&](uint32_t tile, const uint4 (&r)[UN]) {
#pragma unroll
      for (int i = 0; i < UN; ++i) {
        const int t = i * TPI + first;
        const uint32_t at = tile + (chunk >> 2) * BN * 128 + t * 128;
        const uint32_t c0 = (chunk & 3) * 2;
        const uint32_t w[4] = {r[i].x, r[i].y, r[i].z, r[i].w};
        uint32_t f[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          f[2 * e] = e4m3x2_f16x2(w[e]);
          f[2 * e + 1] = e4m3x2_f16x2(w[e] >> 16);
        }
        sts128(at + ((c0 ^ (t & 7)) << 4), f[0], f[1], f[2], f[3]);
        sts128(at + (((c0 + 1) ^ (t & 7)) << 4), f[4], f[5], f[6], f[7]);
      }
      fence_proxy_async_smem();
      __syncwarp();
    };
    bool ok = true;
    uint32_t zero_units = 0;
    for (;;) {
      for (int j = -1; j < steps; ++j) {  // (-1: loads only)
        if (j >= 0) {
        const int s = j & 1;
        const uint32_t phase = (j >> 1) & 1u;
        // pages with a value scale of zero: their weights count, their values are zeros
        const float vs_now = vs;
        zero_units = __ballot_sync(0xFFFFFFFFu, vs_now == 0.0f);
        const uint32_t holes = __ballot_sync(0xFFFFFFFFu, lane < GR && !there);
        if (warp == 12 && lane == 0) *reinterpret_cast<int*>(smem + L::kHole + (j & 3) * 4) = holes != 0;
        if (warp == 12 && lane < GR) {
          const float lv = vs_now == 0.0f ? kNilLog2 : log2_approx(vs_now);
          if (vs_now != 0.0f) {
            lowest = fminf(lowest, lv);
            highest = fmaxf(highest, lv);
            seen |= 1u << band_of(lv);
          }
          *reinterpret_cast<float4*>(smem + L::kMeta + (j & 3) * GR * 16 + lane * 16) =
              make_float4(ks, lv, vs_now == 0.0f ? kNilInverse : 1.0f / vs_now, there ? 1.0f : 0.0f);
        }
        ok = wait_warp(bar(KEMPTY, s), phase ^ 1u, abort_flag, (2u << 24) | (4u << 16) | (j & 0xFFFF));
        if (!ok) break;
        write(k_at + s * L::kTile, kr);
        if (lane == 0) mbar_arrive(bar(KFULL, s));
        // (zero_units: of this step, the look-up below is the next one's)
        }
        if (j + 1 < steps) {
          if (j >= 0) {
            page = page_next;
            page_next = raw_page(j + 2);
          }
          look_up(j + 1);
          load(a.k, j + 1, kr);
        }
        if (j >= 0) {
        const int s = j & 1;
        const uint32_t phase = (j >> 1) & 1u;
        // NaN codes become zeros, and where the first one of a column is goes to the output's warps
#pragma unroll
        for (int i = 0; i < UN; ++i) {
          const int t = i * TPI + first;
          uint32_t* w = reinterpret_cast<uint32_t*>(&vr[i]);
          const uint32_t hit = __vcmpeq4(w[0] & 0x7F7F7F7Fu, 0x7F7F7F7Fu) | __vcmpeq4(w[1] & 0x7F7F7F7Fu, 0x7F7F7F7Fu) |
                               __vcmpeq4(w[2] & 0x7F7F7F7Fu, 0x7F7F7F7Fu) | __vcmpeq4(w[3] & 0x7F7F7F7Fu, 0x7F7F7F7Fu);
          if (hit) {
            *nan_any = 1;
            vr[i] = without_nans(vr[i], nan_at + chunk * 16, key_of(j) + t);
          }
          if (zero_units >> (t >> 4) & 1u) w[0] = w[1] = w[2] = w[3] = 0;
        }
        ok = wait_warp(bar(VEMPTY, s), phase ^ 1u, abort_flag, (2u << 24) | (5u << 16) | (j & 0xFFFF));
        if (!ok) break;
        write(v_at + s * L::kTile, vr);
        if (lane == 0) mbar_arrive(bar(VFULL, s));
        }
        if (j + 1 < steps) load(a.v, j + 1, vr);
      }
      if (warp == 12 && band < 0) {
#pragma unroll
        for (int z = 16; z > 0; z >>= 1) {
          lowest = fminf(lowest, __shfl_xor_sync(0xFFFFFFFFu, lowest, z));
          highest = fmaxf(highest, __shfl_xor_sync(0xFFFFFFFFu, highest, z));
        }
        seen = __reduce_or_sync(0xFFFFFFFFu, seen);
        if (lane == 0 && highest - lowest > kFar) *far_bands = seen;
      }
      fresh = band < 0;
      if (!next_pass()) break;
      page = raw_page(0);
      page_next = raw_page(1);
    }
    grid_launch_dependents();
  } else {
    // ------------------------------------------------------------------ MMA issuer (warps without a part only keep the passes)
    bool fresh = true;
    for (;;) {
      if (warp == 0 && elect_one() && steps > 0) {
        constexpr uint32_t id_s = idesc_f16(128, BN, false), id_o = idesc_f16(128, D, true);
        auto scores = [&](int j, int slot, int buf) {
          const uint64_t dq = make_kmajor_sw128_desc(q_at + slot * L::kQ), dk = make_kmajor_sw128_desc(k_at + (j & 1) * L::kTile);
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            mma_f16_ss(tmem + kS + buf * BN, dq + ((k >> 2) * 128 * 128 + (k & 3) * 32) / 16, dk + ((k >> 2) * BN * 128 + (k & 3) * 32) / 16,
                       id_s, k > 0);
          mma_commit(bar(SFULL, buf));
        };
        auto product = [&](int j, int slot, int buf) {
          const uint64_t dv = make_mnmajor_desc(v_at + (j & 1) * L::kTile, BN * 128);
#pragma unroll
          for (int k = 0; k < BN / 16; ++k)
            mma_f16_ts(tmem + kO + slot * D, tmem + L::kP + buf * L::kPStride + 8 * k, dv + k * 2048 / 16, id_o, j > 0 || k > 0 || !fresh);
          mma_commit(bar(PV, slot));
        };
        // Scores are AHEAD steps ahead of products: one with two row tiles in turn, two with two buffers.
        constexpr int AHEAD = NQ == 2 ? 1 : 2;
        bool ok = wait_one(bar(QFULL, 0), 0, abort_flag, (3u << 24) | (6u << 16));  // (of the first pass)
#pragma unroll 1
        for (int j = -AHEAD; ok && j < steps; ++j) {
          const int n = j + AHEAD;  // whose scores are next
#pragma unroll 1
          for (int slot = 0; ok && slot < NQ; ++slot) {
            const int buf = NQ == 2 ? slot : j & 1;
            if (j >= 0) {
              if (slot == 0) ok = wait_one(bar(VFULL, j & 1), (j >> 1) & 1u, abort_flag, (3u << 24) | (8u << 16) | (j & 0xFFFF));
              ok = ok && wait_one(bar(PFULL, buf), NQ == 2 ? j & 1u : (j >> 1) & 1u, abort_flag, (3u << 24) | (9u << 16) | (j & 0xFFFF));
              if (!ok) break;
              tc_fence_after();
              product(j, slot, buf);
            }
            if (n < steps) {
              if (slot == 0) ok = wait_one(bar(KFULL, n & 1), (n >> 1) & 1u, abort_flag, (3u << 24) | (7u << 16) | (n & 0xFFFF));
              if (L::kOver && j >= 0) ok = ok && wait_one(bar(PV, slot), j & 1u, abort_flag, (3u << 24) | (10u << 16) | (j & 0xFFFF));
              if (!ok) break;
              tc_fence_after();
              scores(n, slot, buf);
            }
          }
          // given back only where a later step waits for it
          if (ok && j >= 0 && j + 2 < steps) mma_commit(bar(VEMPTY, j & 1));
          if (ok && n + 2 < steps) mma_commit(bar(KEMPTY, n & 1));
        }
      }
      __syncwarp();
      fresh = band < 0;
      if (!next_pass()) break;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Adds the key ranges of a row tile up, in their order: a warp a row, all of a row's loads of eight ranges in flight.
template <int D, typename T>
__global__ void __launch_bounds__(256) cache_attend_combine_kernel(const __grid_constant__ AttendArgs a, const int vec) {
  constexpr int ROWS = Tiles<D>::ROWS, PL = D / 128 > 0 ? D / 128 : 1;  // four elements a lane and load
  const int lane = threadIdx.x & 31, y = blockIdx.y, b = blockIdx.z;
  const int h = y / a.row_tiles, row0 = (y - h * a.row_tiles) * ROWS, r = blockIdx.x * 8 + (threadIdx.x >> 5);
  grid_dependency_wait();
  const int len = min(max(a.lens[b], 0), a.max_pages * a.P);
  const int nq = a.q_lens ? min(max(a.q_lens[b], 0), a.T) : a.T;
  const int rows = min(ROWS, nq * a.G - row0);
  const int prefix = a.prefix ? a.prefix[b] : 0;
  const int last = row0 + rows - 1;
  const int most = rows <= 0 ? 0 : max(0, a.causal ? min(len, max(len - nq + last / a.G + 1, prefix)) : len);
  const int chunks = max(1, (most + a.chunk - 1) / a.chunk);
  if (r >= rows || chunks == 1) return;   // (one range: written by its CTA)
  const int64_t from = (int64_t)(b * a.H * a.row_tiles + y) * a.splits * ROWS + r;
  const float2* ml = reinterpret_cast<const float2*>(a.partial + a.partial_ml) + from;
  const float* po = a.partial + from * D;
  const bool on = 4 * lane < D;
  float m = -INFINITY, l = 0.0f;
  for (int s = lane; s < chunks; s += 32) m = fmaxf(m, __ldcg(ml + (int64_t)s * ROWS).x);
#pragma unroll
  for (int z = 16; z > 0; z >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, z));
  float4 o[PL] = {};
#pragma unroll 1
  for (int s0 = 0; s0 < chunks; s0 += 8) {
    float4 u[8][PL];
    float2 x[8];
#pragma unroll
    for (int z = 0; z < 8; ++z) {
      if (s0 + z < chunks) {
        x[z] = __ldcg(ml + (int64_t)(s0 + z) * ROWS);
#pragma unroll
        for (int p = 0; p < PL; ++p)
          if (on) u[z][p] = __ldcg(reinterpret_cast<const float4*>(po + (int64_t)(s0 + z) * ROWS * D + 128 * p) + lane);
      }
    }
#pragma unroll
    for (int z = 0; z < 8; ++z) {
      if (s0 + z < chunks) {
        const float f = x[z].x == -INFINITY ? 1.0f : ex2_approx_ftz(x[z].x - m);
        l = fmaf(f, x[z].y, l);
#pragma unroll
        for (int p = 0; p < PL; ++p) {
          o[p].x = fmaf(f, u[z][p].x, o[p].x);
          o[p].y = fmaf(f, u[z][p].y, o[p].y);
          o[p].z = fmaf(f, u[z][p].z, o[p].z);
          o[p].w = fmaf(f, u[z][p].w, o[p].w);
        }
      }
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const int t = (row0 + r) / a.G;
  T* out = reinterpret_cast<T*>(a.out) + b * a.o_b + t * a.o_t + (h * a.G + row0 + r - t * a.G) * a.o_h;
#pragma unroll
  for (int p = 0; p < PL; ++p) {
    if (!on) break;
    const uint32_t w0 = pack_out<T>(o[p].x * inv, o[p].y * inv), w1 = pack_out<T>(o[p].z * inv, o[p].w * inv);
    T* dst = out + 128 * p + 4 * lane;
    if (vec) {
      *reinterpret_cast<uint2*>(dst) = make_uint2(w0, w1);
    } else {
      const T *p0 = reinterpret_cast<const T*>(&w0), *p1 = reinterpret_cast<const T*>(&w1);
      dst[0] = p0[0];
      dst[1] = p0[1];
      dst[2] = p1[0];
      dst[3] = p1[1];
    }
  }
}

template <int D, typename T, bool CAP, bool SLOPES>
int launch_tiles(const AttendArgs& a, int vec, cudaStream_t s) {
  static bool attr_set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return IFLB200_ERR_DEVICE;
  if (!attr_set[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(cache_attend_tiles_kernel<D, T, CAP, SLOPES>, cudaFuncAttributeMaxDynamicSharedMemorySize, Tiles<D>::kSmem);
    if (e != cudaSuccess) return (int)e;
    attr_set[dev] = true;
  }
  const bool dep = dependent_launch_for((int64_t)a.B * a.T);
  const unsigned tiles = (unsigned)(a.H * a.row_tiles);
  cudaError_t e = launch_dep(cache_attend_tiles_kernel<D, T, CAP, SLOPES>, dim3((unsigned)a.splits, tiles, (unsigned)a.B), dim3(kThreads),
                             Tiles<D>::kSmem, s, 1, dep, a, vec);
  if (e == cudaSuccess && a.splits > 1)
    e = launch_dep(cache_attend_combine_kernel<D, T>, dim3((unsigned)Tiles<D>::ROWS / 8, tiles, (unsigned)a.B), dim3(256), 0, s, 1, dep, a, vec);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

template <int D, typename T>
int launch_tiles(const AttendArgs& a, int vec, cudaStream_t s) {
  if (a.cap > 0.0f) return a.slopes ? launch_tiles<D, T, true, true>(a, vec, s) : launch_tiles<D, T, true, false>(a, vec, s);
  return a.slopes ? launch_tiles<D, T, false, true>(a, vec, s) : launch_tiles<D, T, false, false>(a, vec, s);
}

}  // namespace

int attend_tiles_rows(int head_dim) { return head_dim == 256 ? Tiles<256>::ROWS : Tiles<128>::ROWS; }

template <typename T>
int launch_attend_tiles(const AttendArgs& a, int head_dim, cudaStream_t s) {
  const uintptr_t bits = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.out) |
                         (uintptr_t)((a.q_b | a.q_t | a.q_h | a.o_b | a.o_t | a.o_h) * (int64_t)sizeof(T));
  const int vec = bits % 16 == 0;
  if (head_dim == 64) return launch_tiles<64, T>(a, vec, s);
  if (head_dim == 128) return launch_tiles<128, T>(a, vec, s);
  return launch_tiles<256, T>(a, vec, s);
}
template int launch_attend_tiles<__nv_bfloat16>(const AttendArgs&, int, cudaStream_t);
template int launch_attend_tiles<__half>(const AttendArgs&, int, cudaStream_t);

int set_attend_wait_budget_ns(uint64_t ns) { return set_budget_ns(ns); }
int take_attend_timeout_record(uint32_t* record, cudaStream_t s) { return take_record(record, s); }

}  // namespace iflb200
