// Attention over the paged 8-bit cache for many rows: row tiles of 128 (query token x head of a group) on tcgen05.
//
// One CTA has NQ row tiles of one key/value head and walks its keys BN at a time.  Per step and row tile
//
//   S = Q K^T            128 x BN x D, operands f16 in shared memory, S fp32 in tensor memory
//   y = S * (factor of the row * ks) + log2 vs       base-2 exponents, masked at the edge
//   P = 2^(y - M) as f16 into tensor memory          M: the row's running maximum of y
//   O += P V             128 x D x BN, P from tensor memory, V f16 in shared memory, O fp32 in tensor memory
//
// The value scale of a page is part of the exponent, so that O needs no scale of its own: with l = sum 2^(y - M) / vs
// the output is O / l.  M moves only when a score passes it by more than 2^5, since O in tensor memory has to be
// multiplied then.
//
// Codes become f16 on the way into shared memory (exact): a 16-bit operand of the same MMA rate as two 8-bit halves of q
// and P would have, with 11 bits of P and no work on P but its rounding.  The MMA takes the values [key][D] as they lie
// (transposed B operand).
//
//   warps 0..3, 4..7   softmax, one row a thread, and the output (D 256 has one row tile, whose S has two buffers instead)
//   warps 8..11        codes from global memory through registers to f16 tiles, one tile ahead; a step's scales
//   warp 12            MMA issuer, tensor memory
#include "bounded_wait.cuh"
#include "cache_attn.cuh"

namespace iflb200 {

namespace {

constexpr int kThreads = 512;

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
  static constexpr int kBar = kNan + D * 4 + 16;
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
__device__ __forceinline__ void tmem_st_32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
      "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
      "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
template <int REGS>
__device__ __forceinline__ void more_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS));
}
template <int REGS>
__device__ __forceinline__ void fewer_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS));
}

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
__device__ __forceinline__ float log2_approx(float a) {
  float r;
  asm("lg2.approx.f32 %0, %1;" : "=f"(r) : "f"(a));
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

// D elements of a row of q: 16 bytes at a time where they are aligned.
template <typename T, bool VEC>
__device__ __forceinline__ void load_row8(const T* q, float (&x)[8]) {
  if (VEC) {
    const uint4 u = *reinterpret_cast<const uint4*>(q);
    const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = row_value(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = row_value(q[i]);
  }
}

template <int D, typename T>
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
  volatile int* last_one = nan_at + D + 1;
  enum { KFULL = 0, KEMPTY = 2, VFULL = 4, VEMPTY = 6, SFULL = 8, PFULL = 10, PV = 12, QFULL = 14 };
  auto bar = [&](int kind, int i) { return bar0 + 8u * (kind + i); };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kBar + 24 * 8);
  volatile uint32_t* abort_flag = tmem_slot + 1;

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

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(KFULL, i), 4);
      mbar_init(bar(KEMPTY, i), 1);
      mbar_init(bar(VFULL, i), 4);
      mbar_init(bar(VEMPTY, i), 1);
      mbar_init(bar(SFULL, i), 1);
      mbar_init(bar(PFULL, i), 4);
      mbar_init(bar(PV, i), 1);
    }
    mbar_init(bar(QFULL, 0), 4 * NQ);
    tmem_slot[1] = 0;
    *nan_any = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  for (int i = threadIdx.x; i < D; i += kThreads) nan_at[i] = INT32_MAX;
  __syncwarp();
  if (warp == 12) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp < 4 * NQ) {
    // ------------------------------------------------------------------ softmax and output
    more_registers<184>();
    const int slot = warp >> 2;
    const int r = slot * 128 + (warp & 3) * 32 + lane;
    const bool in = r < rows;
    const int tok = (row0 + (in ? r : 0)) / a.G, hq = h * a.G + (row0 + (in ? r : 0)) - tok * a.G;
    const int limit = in ? limit_of(row0 + r) : INT32_MAX;  // (a row that is not there needs no mask)
    const int least = __reduce_min_sync(0xFFFFFFFFu, limit);
    const float pos = (float)(len - nq + tok);
    const float slope = a.slopes ? a.slopes[hq] * kLog2e : 0.0f;
    const float inv_cap = a.cap > 0.0f ? 1.0f / a.cap : 0.0f;
    float factor;
    {
      // the row of q as f16, its largest element near 1
      const T* q = reinterpret_cast<const T*>(a.q) + b * a.q_b + tok * a.q_t + hq * a.q_h;
      float top = 0.0f;
      for (int i = 0; i < D / 8; ++i) {
        float x[8];
        if (vec) load_row8<T, true>(q + 8 * i, x);
        else load_row8<T, false>(q + 8 * i, x);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (fabsf(x[e]) < 3.39e38f) top = fmaxf(top, fabsf(x[e]));
      }
      const int e2 = min(max((int)(__float_as_uint(top) >> 23), 2), 252);
      const float down = __uint_as_float((uint32_t)(254 - e2) << 23);
      factor = __uint_as_float((uint32_t)e2 << 23) * a.scale;
      const uint32_t at = q_at + slot * L::kQ + (r & 127) * 128;
      for (int i = 0; i < D / 8; ++i) {
        float x[8];
        if (vec) load_row8<T, true>(q + 8 * i, x);
        else load_row8<T, false>(q + 8 * i, x);
        sts128(at + (i >> 3) * 128 * 128 + (((i & 7) ^ (r & 7)) << 4), pack_half2(x[0] * down, x[1] * down),
               pack_half2(x[2] * down, x[3] * down), pack_half2(x[4] * down, x[5] * down), pack_half2(x[6] * down, x[7] * down));
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(QFULL, 0));
    }
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t o_at = tmem + lanes + kO + slot * D;
    float top_run = -INFINITY, l = 0.0f;
    bool ok = true;
    for (int j = 0; j < steps; ++j) {
      const int buf = NQ == 2 ? slot : j & 1;
      const uint32_t phase = NQ == 2 ? j & 1u : (j >> 1) & 1u;
      const uint32_t s_at = tmem + lanes + kS + buf * BN;
      ok = wait_warp(bar(SFULL, buf), phase, abort_flag, (1u << 24) | (1u << 16) | (j & 0xFFFF));
      if (!ok) break;
      tc_fence_after();
      uint32_t v[BN];
#pragma unroll
      for (int i = 0; i < BN / 32; ++i) tmem_ld_32x32b_x32(s_at + 32 * i, *reinterpret_cast<uint32_t(*)[32]>(v + 32 * i));
      const uint32_t m_at = meta + (j & 3) * GR * 16;
      const int key = key0 + j * BN;
      // The product of the step before has to be complete ahead of a change of O, and every phase of its barrier is waited
      // for in turn.  With two row tiles it was ahead of these scores; else it may run until the weights are ready.
      bool waited = j == 0;
      auto product_done = [&]() {
        if (!waited) ok = wait_warp(bar(PV, slot), (j - 1) & 1u, abort_flag, (1u << 24) | (2u << 16) | (j & 0xFFFF));
        waited = true;
        tc_fence_after();
      };
      if (NQ == 2) product_done();
      tmem_ld_wait();
      float top = -INFINITY;
      bool broken = false;
#pragma unroll
      for (int g = 0; g < GR; ++g) {
        const float4 m = lds_f4(m_at + 16 * g);  // ks, log2 vs, 1 / vs, 0 where there is no page
        broken |= m.w == 0.0f;
        const float f = factor * m.x;
        if (a.cap > 0.0f) {
#pragma unroll
          for (int e = 0; e < 16; ++e)
            v[16 * g + e] = __float_as_uint(fmaf(soft_cap(__uint_as_float(v[16 * g + e]) * f, a.cap, inv_cap), kLog2e, m.y));
        } else {
          const uint64_t f2 = pack2(f * kLog2e, f * kLog2e), y2 = pack2(m.y, m.y);
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            float p0, p1;
            unpack2(fma2(pack2(__uint_as_float(v[16 * g + e]), __uint_as_float(v[16 * g + e + 1])), f2, y2), p0, p1);
            v[16 * g + e] = __float_as_uint(p0);
            v[16 * g + e + 1] = __float_as_uint(p1);
          }
        }
      }
      if (a.slopes) {
        const float from = pos - (float)key;
#pragma unroll
        for (int e = 0; e < BN; ++e) v[e] = __float_as_uint(fmaf(-slope, fabsf(from - (float)e), __uint_as_float(v[e])));
      }
      if (key + BN > least || broken) {
        const int n = limit - key;
#pragma unroll
        for (int g = 0; g < GR; ++g) {
          const bool gone = lds_f4(m_at + 16 * g).w == 0.0f;
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (16 * g + e >= n || gone) v[16 * g + e] = 0xFF800000u;
        }
      }
#pragma unroll
      for (int e = 0; e < BN; e += 2) top = max3(top, __uint_as_float(v[e]), __uint_as_float(v[e + 1]));
      if (__any_sync(0xFFFFFFFFu, top > top_run + kLazy)) {
        const float now = fmaxf(top_run, top);
        const float f = top_run == -INFINITY ? 0.0f : ex2_approx_ftz(top_run - now);
        top_run = now;
        l *= f;
        if (j > 0) {
          if (NQ == 1) product_done();
#pragma unroll 1
          for (int i = 0; i < D / 32; ++i) {
            uint32_t o[32];
            tmem_ld_32x32b_x32(o_at + 32 * i, o);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            tmem_st_32(o_at + 32 * i, o);
          }
          tmem_st_wait();
        }
      }
      const float m = top_run == -INFINITY ? 0.0f : top_run;
#pragma unroll
      for (int g = 0; g < GR; ++g) {
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          const float p0 = ex2_approx_ftz(__uint_as_float(v[16 * g + e]) - m), p1 = ex2_approx_ftz(__uint_as_float(v[16 * g + e + 1]) - m);
          s += p0 + p1;
          v[8 * g + e / 2] = pack_half2(p0, p1);
        }
        l = fmaf(s, lds_f4(m_at + 16 * g).z, l);
      }
      product_done();
      if (!ok) break;
#pragma unroll
      for (int i = 0; i < BN / 64; ++i) tmem_st_32(tmem + lanes + L::kP + buf * L::kPStride + 32 * i, v + 32 * i);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(PFULL, buf));
    }
    if (ok && steps > 0) ok = wait_warp(bar(PV, slot), (steps - 1) & 1u, abort_flag, (1u << 24) | (3u << 16));
    tc_fence_after();
    const int ticket = b * a.H * a.row_tiles + y;
    const bool any_nan = *nan_any != 0;
    const float inv = chunks > 1 ? 1.0f : (l == 0.0f ? 0.0f : 1.0f / l);
    T* out = reinterpret_cast<T*>(a.out) + b * a.o_b + tok * a.o_t + hq * a.o_h;
    const int64_t at = ((int64_t)ticket * a.splits + split) * L::ROWS + r;
    float* part = a.partial + at * D;
#pragma unroll 1
    for (int i = 0; i < D / 32; ++i) {
      uint32_t o[32];
      if (steps > 0) {
        tmem_ld_32x32b_x32(o_at + 32 * i, o);
        tmem_ld_wait();
      } else {
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = 0;
      }
      if (in && ok) {
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          float x = __uint_as_float(o[e]) * inv;
          if (any_nan && nan_at[32 * i + e] < limit) x = __uint_as_float(0x7FC00000u);
          o[e] = __float_as_uint(x);
        }
        if (chunks > 1) {
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            *reinterpret_cast<uint4*>(part + 32 * i + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        } else if (vec) {
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            uint4 u;
            uint32_t* w = reinterpret_cast<uint32_t*>(&u);
#pragma unroll
            for (int z = 0; z < 4; ++z) w[z] = pack_out<T>(__uint_as_float(o[e + 2 * z]), __uint_as_float(o[e + 2 * z + 1]));
            *reinterpret_cast<uint4*>(out + 32 * i + e) = u;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const uint32_t w = pack_out<T>(__uint_as_float(o[e]), __uint_as_float(o[e + 1]));
            const T* two = reinterpret_cast<const T*>(&w);
            out[32 * i + e] = two[0];
            out[32 * i + e + 1] = two[1];
          }
        }
      }
      __syncwarp();  // (the next load is the whole warp's)
    }
    if (chunks > 1) {
      if (in) *reinterpret_cast<float2*>(a.partial + a.partial_ml + at * 2) = make_float2(top_run, l);
      // the last CTA of the chunks adds them up, in their order
      __threadfence();
      named_bar_sync(1, 128 * NQ);
      if (threadIdx.x == 0) *last_one = atomicAdd(a.tickets + ticket, 1u) == (uint32_t)chunks - 1;
      named_bar_sync(1, 128 * NQ);
      if (*last_one) {
        __threadfence();
        if (threadIdx.x == 0) a.tickets[ticket] = 0;
        const int64_t from = (int64_t)ticket * a.splits * L::ROWS;
        const float2* ml = reinterpret_cast<const float2*>(a.partial + a.partial_ml) + from;
        const float* po = a.partial + from * D;
        for (int i = threadIdx.x; i < rows * (D / 4); i += 128 * NQ) {
          const int rr = i / (D / 4), d = (i - rr * (D / 4)) * 4;
          float mm = -INFINITY;
          for (int s = 0; s < chunks; ++s) mm = fmaxf(mm, __ldcg(ml + s * L::ROWS + rr).x);
          float ll = 0.0f;
          float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          for (int s = 0; s < chunks; ++s) {
            const float2 x = __ldcg(ml + s * L::ROWS + rr);
            const float f = x.x == -INFINITY ? 1.0f : ex2_approx_ftz(x.x - mm);
            const float4 u = __ldcg(reinterpret_cast<const float4*>(po + ((int64_t)s * L::ROWS + rr) * D + d));
            ll += f * x.y;
            o.x += f * u.x;
            o.y += f * u.y;
            o.z += f * u.z;
            o.w += f * u.w;
          }
          const float w = ll == 0.0f ? 0.0f : 1.0f / ll;
          const int t2 = (row0 + rr) / a.G, h2 = h * a.G + (row0 + rr) - t2 * a.G;
          T* dst = reinterpret_cast<T*>(a.out) + b * a.o_b + t2 * a.o_t + h2 * a.o_h + d;
          const uint32_t w0 = pack_out<T>(o.x * w, o.y * w), w1 = pack_out<T>(o.z * w, o.w * w);
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
    }
  } else if (warp < 8) {
    fewer_registers<40>();
  } else if (warp < 12) {
    // ------------------------------------------------------------------ codes to f16 tiles
    fewer_registers<96>();
    constexpr int CH = D / 16, UN = BN * CH / 128, TPI = 128 / CH;  // chunks of a key, chunks a thread, keys apart
    const int tid = threadIdx.x - 256, chunk = tid % CH, first = tid / CH;
    const int32_t* table = a.table + b * a.ld_table;
    auto raw_page = [&](int step) {  // of this lane's unit of the step
      const int key = key0 + step * BN + 16 * lane;
      return lane < GR && key < key1 ? __ldg(table + key / a.P) : -1;
    };
    int page = raw_page(0), page_next = raw_page(1);
    float ks = 0.0f, vs = 0.0f;
    int64_t off = -1;
    auto look_up = [&](int step) {  // where this lane's unit lies, and its scales
      const bool there = page >= 0 && page < a.pages;
      const int key = key0 + step * BN + 16 * lane;
      off = there ? (((int64_t)page * a.H + h) * a.P + key % a.P) * D : -1;
      ks = there ? __ldg(a.ks + (int64_t)page * a.H + h) : 0.0f;
      vs = there ? __ldg(a.vs + (int64_t)page * a.H + h) : 0.0f;
    };
    uint4 kr[UN], vr[UN];
    auto load = [&](const uint8_t* codes, int step, uint4 (&r)[UN]) {
#pragma unroll
      for (int i = 0; i < UN; ++i) {
        const int t = i * TPI + first;
        const int64_t o = __shfl_sync(0xFFFFFFFFu, off, t >> 4);
        r[i] = make_uint4(0, 0, 0, 0);
        if (o >= 0 && key0 + step * BN + t < key1) r[i] = __ldg(reinterpret_cast<const uint4*>(codes + o + (t & 15) * D + chunk * 16));
      }
    };
    auto write = [&](uint32_t tile, const uint4 (&r)[UN]) {
#pragma unroll
      for (int i = 0; i < UN; ++i) {
        const int t = i * TPI + first;
        const uint32_t at = tile + (chunk >> 2) * BN * 128 + t * 128;
        const uint32_t c0 = (chunk & 3) * 2, odd = chunk >> 2 & 1;  // (halves of a key store in turn: no bank twice)
        const uint32_t w[4] = {r[i].x, r[i].y, r[i].z, r[i].w};
        uint32_t f[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          f[2 * e] = e4m3x2_f16x2(w[e]);
          f[2 * e + 1] = e4m3x2_f16x2(w[e] >> 16);
        }
        const uint32_t lo = at + ((c0 ^ (t & 7)) << 4), hi = at + (((c0 + 1) ^ (t & 7)) << 4);
        if (odd) {
          sts128(hi, f[4], f[5], f[6], f[7]);
          sts128(lo, f[0], f[1], f[2], f[3]);
        } else {
          sts128(lo, f[0], f[1], f[2], f[3]);
          sts128(hi, f[4], f[5], f[6], f[7]);
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
    };
    bool ok = true;
    if (steps > 0) {
      look_up(0);
      load(a.k, 0, kr);
      load(a.v, 0, vr);
    }
    for (int j = 0; j < steps; ++j) {
      const int s = j & 1;
      const uint32_t phase = (j >> 1) & 1u;
      // pages with a value scale of zero: their weights count, their values are zeros
      const float vs_now = vs;
      const uint32_t zero_units = __ballot_sync(0xFFFFFFFFu, vs_now == 0.0f);
      if (warp == 8 && lane < GR) {
        const float lv = vs_now == 0.0f ? 0.0f : log2_approx(vs_now);
        *reinterpret_cast<float4*>(smem + L::kMeta + (j & 3) * GR * 16 + lane * 16) =
            make_float4(ks, lv, vs_now == 0.0f ? 1.0f : 1.0f / vs_now, off >= 0 ? 1.0f : 0.0f);
      }
      ok = wait_warp(bar(KEMPTY, s), phase ^ 1u, abort_flag, (2u << 24) | (4u << 16) | (j & 0xFFFF));
      if (!ok) break;
      write(k_at + s * L::kTile, kr);
      if (lane == 0) mbar_arrive(bar(KFULL, s));
      page = page_next;
      if (j + 1 < steps) {
        page_next = raw_page(j + 2);
        look_up(j + 1);
        load(a.k, j + 1, kr);
      }
      // NaN codes become zeros, and where the first one of a column is goes to the output's warps
#pragma unroll
      for (int i = 0; i < UN; ++i) {
        const int t = i * TPI + first;
        uint32_t* w = reinterpret_cast<uint32_t*>(&vr[i]);
        if (zero_units >> (t >> 4) & 1u) w[0] = w[1] = w[2] = w[3] = 0;
        const uint32_t hit = __vcmpeq4(w[0] & 0x7F7F7F7Fu, 0x7F7F7F7Fu) | __vcmpeq4(w[1] & 0x7F7F7F7Fu, 0x7F7F7F7Fu) |
                             __vcmpeq4(w[2] & 0x7F7F7F7Fu, 0x7F7F7F7Fu) | __vcmpeq4(w[3] & 0x7F7F7F7Fu, 0x7F7F7F7Fu);
        if (hit) {
          *nan_any = 1;
          for (int e = 0; e < 16; ++e) {
            if ((w[e >> 2] >> (8 * (e & 3)) & 0x7F) == 0x7F) {
              atomicMin(nan_at + chunk * 16 + e, key0 + j * BN + t);
              w[e >> 2] &= ~(0xFFu << (8 * (e & 3)));
            }
          }
        }
      }
      ok = wait_warp(bar(VEMPTY, s), phase ^ 1u, abort_flag, (2u << 24) | (5u << 16) | (j & 0xFFFF));
      if (!ok) break;
      write(v_at + s * L::kTile, vr);
      if (lane == 0) mbar_arrive(bar(VFULL, s));
      if (j + 1 < steps) load(a.v, j + 1, vr);
    }
    grid_launch_dependents();
  } else {
    fewer_registers<40>();
    // ------------------------------------------------------------------ MMA issuer
    if (warp == 12 && elect_one() && steps > 0) {
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
          mma_f16_ts(tmem + kO + slot * D, tmem + L::kP + buf * L::kPStride + 8 * k, dv + k * 2048 / 16, id_o, j > 0 || k > 0);
        mma_commit(bar(PV, slot));
      };
      bool ok = wait_one(bar(QFULL, 0), 0, abort_flag, (3u << 24) | (6u << 16));
      auto keys = [&](int j) {
        ok = ok && wait_one(bar(KFULL, j & 1), (j >> 1) & 1u, abort_flag, (3u << 24) | (7u << 16) | (j & 0xFFFF));
        tc_fence_after();
      };
      keys(0);
      if (ok) {
        scores(0, 0, 0);
        if (NQ == 2) scores(0, 1, 1);
        if (steps > 2) mma_commit(bar(KEMPTY, 0));  // (here and below: only where a later tile waits for it)
      }
      if (NQ == 1 && steps > 1) {
        keys(1);
        if (ok) {
          scores(1, 0, 1);
          if (steps > 3) mma_commit(bar(KEMPTY, 1));
        }
      }
      for (int j = 0; ok && j < steps; ++j) {
        ok = wait_one(bar(VFULL, j & 1), (j >> 1) & 1u, abort_flag, (3u << 24) | (8u << 16) | (j & 0xFFFF));
        if (NQ == 2) {
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            ok = ok && wait_one(bar(PFULL, s), j & 1u, abort_flag, (3u << 24) | (9u << 16) | (j & 0xFFFF));
            if (!ok) break;
            tc_fence_after();
            product(j, s, s);
            if (j + 1 < steps) {
              if (s == 0) keys(j + 1);
              if (L::kOver) ok = ok && wait_one(bar(PV, s), j & 1u, abort_flag, (3u << 24) | (10u << 16) | (j & 0xFFFF));
              if (ok) scores(j + 1, s, s);
            }
          }
          if (!ok) break;
          if (j + 2 < steps) mma_commit(bar(VEMPTY, j & 1));
          if (j + 3 < steps) mma_commit(bar(KEMPTY, (j + 1) & 1));
        } else {
          ok = ok && wait_one(bar(PFULL, j & 1), (j >> 1) & 1u, abort_flag, (3u << 24) | (9u << 16) | (j & 0xFFFF));
          if (!ok) break;
          tc_fence_after();
          product(j, 0, j & 1);
          if (j + 2 < steps) mma_commit(bar(VEMPTY, j & 1));
          if (j + 2 < steps) {
            keys(j + 2);
            if (!ok) break;
            scores(j + 2, 0, j & 1);
            if (j + 4 < steps) mma_commit(bar(KEMPTY, j & 1));
          }
        }
      }
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int D, typename T>
int launch_tiles(const AttendArgs& a, int vec, cudaStream_t s) {
  static bool attr_set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return IFLB200_ERR_DEVICE;
  if (!attr_set[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(cache_attend_tiles_kernel<D, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, Tiles<D>::kSmem);
    if (e != cudaSuccess) return (int)e;
    attr_set[dev] = true;
  }
  const dim3 grid((unsigned)a.splits, (unsigned)(a.H * a.row_tiles), (unsigned)a.B);
  const cudaError_t e = launch_dep(cache_attend_tiles_kernel<D, T>, grid, dim3(kThreads), Tiles<D>::kSmem, s, 1,
                                   dependent_launch_for((int64_t)a.B * a.T), a, vec);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
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
