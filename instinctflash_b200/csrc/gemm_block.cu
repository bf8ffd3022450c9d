// FP8 GEMM whose operands have a scale for each block of 128: activations for each row and 128 columns, weights for
// each 128 x 128 block.
//
//   out[t, n] = out_type( sum_b sa[t, b] sw[n / 128, b] * ( sum_{k in block b} A[t, k] W[n, k] )  (+ bias[n]) )
//
// The inner sums run on tcgen05 (fp32 accumulators in tensor memory).  A scale changes from one K step of 128 to the
// next, so the accumulator of every step is taken out of tensor memory, multiplied and added to a sum in the epilogue
// warps' registers (fp32 throughout), while the MMAs of the next step run into another accumulator.
//
// Weights are on the MMA's M side (128 rows a CTA: one row of weight blocks, so one weight scale a step), tokens on its
// N side in tiles of any multiple of 16 up to 128: the accumulator is the tile transposed.  Sixteen warps take it out in the
// 16 x 256-bit shape, where a thread holds four weight rows of two neighbouring tokens: one 8-byte read of the tokens'
// scales serves four packed fused multiply-adds.
//
//   warp 0      TMA producer of W         warp 1   MMA issuer, tensor memory
//   warp 2      TMA producer of A         warp 3   scales: sa * sw into shared memory, eight K steps at a time
//   warps 4..19 promotion and epilogue: a quadrant of tensor memory and 32 tokens each
//
// CG 2 works on CTA pairs (256 weight rows), CG 1 on single CTAs, whose K range a cluster of up to eight may share:
// the partial sums meet in distributed shared memory and are added in the order of the ranges.  A stage is two K steps
// with an accumulator each, two stages fill tensor memory.
//
// What it took (4680 x 14336 x 5120, B200): 872 us with release semantics on the arrivals that free an accumulator in the
// pair's other CTA (a memory barrier each), 568 without; 527 with a ring of scales in place of two steps'; 380 with
// branch-free stages (the sums then stay in their registers) of two K steps.  The epilogue's work without the
// sums takes 300, and a GEMM of the same size with one scale a row 240: both run at the 1000 W limit.
#include <cuda.h>
#include <cuda_runtime.h>

#include <type_traits>

#include "../../include/iflb200.h"
#include "bounded_wait.cuh"
#include "launch.cuh"
#include "rowmath.cuh"

namespace iflb200 {

namespace {

constexpr int kStep = 128;  // bytes of K and weight rows: a block of the weight
constexpr int kEpi = 16;    // epilogue warps
constexpr int kThreads = 32 * (4 + kEpi);
constexpr int kMaxStages = 8;
constexpr int SL = 2;           // K steps of a stage
constexpr int kAcc = 128;       // tensor-memory columns of an accumulator
constexpr int kBatch = 8;       // K steps of a batch of scales; two batches in shared memory
constexpr int kBars = 2 * kMaxStages + 2 + 4;
constexpr int kMaxSmem = 227 * 1024;

struct BlockParams {
  int M, N, K;
  int bt;                                // tokens of a tile
  int num_m, num_n, num_k, units, group_m;
  int splits;                            // CG 1: CTAs of a cluster that share a tile's K range
  int stages;
  uint32_t idesc;
  const float* sa;
  int64_t sa_row, sa_block;
  int blocks;                            // of K; num_k: rounded up to whole stages
  const float* sw;                       // [ceil(N / 128)][blocks]
  const void* bias;
  int bias_dtype;
  uint8_t* out;
  int64_t ld_out;                        // bytes
  int out_dtype;
  int staging;                           // bytes a warp: 16 tokens x 32 columns
  int early;                             // the first weights may be read ahead of the dependency wait
};

// Thirty-two token columns of sixteen lanes: r[4 j + {0, 1}] = weight row t/4, tokens 8 j + 2 (t % 4) + {0, 1};
// r[4 j + {2, 3}] = row t/4 + 8.
__device__ __forceinline__ void tmem_ld_32(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void store_transposed(uint32_t addr, const uint32_t (&v)[4]) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v[0]), "r"(v[1]),
               "r"(v[2]), "r"(v[3])
               : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint64_t lds64(uint32_t addr) {
  uint64_t v;
  asm volatile("ld.shared.b64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void sts32(uint32_t addr, float v) {
  asm volatile("st.shared.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
__device__ __forceinline__ void st_cluster_64x2(uint32_t addr, uint32_t rank, uint64_t a, uint64_t b) {
  asm volatile(
      "{\n\t.reg .b32 ra;\n\t"
      "mapa.shared::cluster.u32 ra, %0, %1;\n\t"
      "st.shared::cluster.v2.b64 [ra], {%2, %3};\n\t}"
      ::"r"(addr), "r"(rank), "l"(a), "l"(b)
      : "memory");
}

// Arrival at the leader's barrier.  It publishes no memory: what it stands for is that tensor memory has been read, into
// registers, as tcgen05.wait::ld ahead of it has seen; the MMA that follows writes what nobody reads any more.  That is an order of
// the hardware's: by the words of the memory model the arrival would need release semantics, which at cluster scope is a memory
// barrier that the epilogue warps waited for longer than for anything else (4680 x 14336 x 5120: 872 us with it, 568 without).
__device__ __forceinline__ void arrive_relaxed_cluster(uint32_t bar, uint32_t rank) {
  asm volatile(
      "{\n\t.reg .b32 ra;\n\t"
      "mapa.shared::cluster.u32 ra, %0, %1;\n\t"
      "mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [ra];\n\t}"
      ::"r"(bar), "r"(rank)
      : "memory");
}

__device__ __forceinline__ uint32_t pair_bf16(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pair_f16(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <int CG>
struct Layout {
  static constexpr int kScales = 2 * kBatch * kAcc * 4;  // bytes
  __host__ __device__ static int slab(int bt) { return kStep * kStep + bt / CG * kStep; }
  static int blocks_of(int bt, int splits) { return (bt / 16 + splits - 1) / splits; }  // token blocks that a rank adds up
  static int meeting(int bt, int splits) { return splits > 1 ? blocks_of(bt, splits) * splits * 4 * 2048 : 0; }
  static int fixed(int bt, int splits, int staging) {
    return 1024 + kEpi * staging + kScales + meeting(bt, splits) + kBars * 8 + 16;
  }
  static int stages(int bt, int splits, int staging) {
    const int n = (kMaxSmem - fixed(bt, splits, staging)) / (SL * slab(bt));
    return n < kMaxStages ? n : kMaxStages;
  }
};

template <int CG>
__global__ void __launch_bounds__(kThreads, 1)
gemm_fp8_block_kernel(const __grid_constant__ CUtensorMap tm_t, const __grid_constant__ CUtensorMap tm_w,
                      const __grid_constant__ BlockParams p) {
  using L = Layout<CG>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t base = (raw_addr + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw_addr);
  const int stages = p.stages;
  const uint32_t w_bytes = kStep * kStep, t_bytes = (uint32_t)(p.bt / CG) * kStep, slab_bytes = w_bytes + t_bytes;
  const uint32_t staging0 = base + stages * SL * slab_bytes;
  const uint32_t scales0 = staging0 + kEpi * p.staging;
  const uint32_t meeting0 = scales0 + L::kScales;
  const int own_blocks = CG == 1 && p.splits > 1 ? (p.bt / 16 + p.splits - 1) / p.splits : 0;
  const uint32_t bar0 = meeting0 + (uint32_t)(own_blocks * p.splits) * 4 * 2048;
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto done_bar = [&](int s) { return bar0 + 8u * (kMaxStages + s); };      // MMAs of the stage complete: slabs free, accumulators full
  auto tempty_bar = [&](int a) { return bar0 + 8u * (2 * kMaxStages + a); };
  auto sfull_bar = [&](int i) { return bar0 + 8u * (2 * kMaxStages + 2 + i); };
  auto sempty_bar = [&](int i) { return bar0 + 8u * (2 * kMaxStages + 4 + i); };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + (bar0 - base) + kBars * 8);
  volatile uint32_t* abort_flag = tmem_slot + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = CG == 1 || rank == 0;
  const int splits = CG == 1 ? p.splits : 1;
  const int width = CG == 1 ? splits : 2;
  const int first_unit = blockIdx.x / width, unit_stride = gridDim.x / width;
  // this CTA's K range, in blocks: whole stages (past the operands' last columns TMA reads zeros)
  const int kb0 = CG == 1 ? (int)((int64_t)(p.num_k / SL) * rank / splits) * SL : 0;
  const int kb1 = CG == 1 ? (int)((int64_t)(p.num_k / SL) * (rank + 1) / splits) * SL : p.num_k;
  auto place = [&](int unit, int& t_blk, int& w_blk) {
    const int band = p.group_m * p.num_n, g = unit / band;
    const int first = g * p.group_m, size = min(p.num_m - first, p.group_m), r = unit - g * band;
    t_blk = first + r % size;
    w_blk = r / size;
  };

  if (threadIdx.x == 0) {
    prefetch_tensormap(&tm_w);
    prefetch_tensormap(&tm_t);
    for (int i = 0; i < stages; ++i) {
      mbar_init(full_bar(i), 2);
      mbar_init(done_bar(i), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tempty_bar(a), CG * kEpi);
      mbar_init(sfull_bar(a), 1);
      mbar_init(sempty_bar(a), kEpi);
    }
    tmem_slot[1] = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  __syncwarp();
  cluster_arrive();
  if (warp == 1) {
    if (CG == 2) {
      tmem_alloc_pair(smem_u32(tmem_slot), 512);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(smem_u32(tmem_slot), 512);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  cluster_wait();

  const int quad = warp & 3, part = (warp - 4) >> 2;
  const int r4 = lane >> 2, c4 = lane & 3;

  if (warp == 0 || warp == 2) {
    // ------------------------------------------------------------------ TMA producers
    const bool weights = warp == 0;
    if (elect_one()) {
      bool waited = weights && p.early, ok = true;
      int stage = 0;
      uint32_t phase = 0;
      for (int unit = first_unit; ok && unit < p.units; unit += unit_stride) {
        int t_blk, w_blk;
        place(unit, t_blk, w_blk);
        const int w_row = (w_blk * CG + (CG == 2 ? (int)rank : 0)) * kStep;
        const int t_row = t_blk * p.bt + (CG == 2 ? (int)rank * (p.bt / 2) : 0);
        for (int kb = kb0; kb < kb1; kb += SL) {
          ok = wait_one(done_bar(stage), phase ^ 1, abort_flag, (1u << 24) | (1u << 16) | (uint32_t)(kb & 0xFFFF));
          if (!ok) break;
          const uint32_t bar = full_bar(stage), dst = base + stage * SL * slab_bytes + (weights ? 0u : w_bytes);
          if (leader) mbar_arrive_expect_tx(bar, (uint32_t)(CG * SL) * (weights ? w_bytes : t_bytes));
          if (!waited) grid_dependency_wait();
          waited = true;
#pragma unroll
          for (int h = 0; h < SL; ++h) {
            const int x = (kb + h) * kStep;
            if (CG == 2) {
              tma_load_2d_pair(dst + h * slab_bytes, weights ? &tm_w : &tm_t, bar & kPeerBitMask, x, weights ? w_row : t_row);
            } else {
              tma_load_2d(dst + h * slab_bytes, weights ? &tm_w : &tm_t, bar, x, weights ? w_row : t_row);
            }
          }
          if (++stage == stages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      if (!weights) {
        grid_dependency_wait();
        grid_launch_dependents();
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    if (leader && elect_one()) {
      bool ok = true;
      int stage = 0;
      uint32_t phase = 0, it = 0;
      const uint64_t dw0 = make_kmajor_sw128_desc(base), dt0 = make_kmajor_sw128_desc(base + w_bytes);
      for (int unit = first_unit; ok && unit < p.units; unit += unit_stride) {
        for (int kb = kb0; kb < kb1; kb += SL, ++it) {
          const uint32_t a = it & 1u;
          ok = wait_one(tempty_bar(a), ((it >> 1) & 1u) ^ 1u, abort_flag, (2u << 24) | (2u << 16) | (it & 0xFFFF)) &&
               wait_one(full_bar(stage), phase, abort_flag, (2u << 24) | (3u << 16) | (it & 0xFFFF));
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int h = 0; h < SL; ++h) {
            const uint64_t at = (uint64_t)(((stage * SL + h) * slab_bytes) >> 4);
            const uint32_t d = tmem_base + (a * SL + h) * kAcc;
#pragma unroll
            for (int j = 0; j < kStep / 32; ++j) {
              if (CG == 2) mma_f8f6f4_pair(d, dw0 + at + 2 * j, dt0 + at + 2 * j, p.idesc, j > 0);
              else mma_f8f6f4(d, dw0 + at + 2 * j, dt0 + at + 2 * j, p.idesc, j > 0);
            }
          }
          if (CG == 2) mma_commit_pair(done_bar(stage), 3);
          else mma_commit(done_bar(stage));
          if (++stage == stages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == 3) {
    // ------------------------------------------------------------------ scales
    // 32 values a lane in flight: one trip to L2 for eight K steps.
    constexpr int TPL = kAcc / 32;
    bool ok = true;
    uint32_t batch = 0;
    grid_dependency_wait();
    for (int unit = first_unit; ok && unit < p.units; unit += unit_stride) {
      int t_blk, w_blk;
      place(unit, t_blk, w_blk);
      const int nb = min(w_blk * CG + (CG == 2 ? (int)rank : 0), (p.N - 1) / kStep);
      const float* sw = p.sw + (int64_t)nb * p.blocks;
      for (int kb = kb0; kb < kb1; kb += kBatch, ++batch) {
        float v[kBatch][TPL];
#pragma unroll
        for (int i = 0; i < TPL; ++i) {
          const float* sa = p.sa + (int64_t)min(t_blk * p.bt + 32 * i + lane, p.M - 1) * p.sa_row + (int64_t)kb * p.sa_block;
#pragma unroll
          for (int j = 0; j < kBatch; ++j) v[j][i] = kb + j < p.blocks && 32 * i < p.bt ? __ldg(sa + j * p.sa_block) : 0.0f;
        }
        const float w = lane < kBatch && kb + lane < p.blocks ? __ldg(sw + kb + lane) : 0.0f;
        const uint32_t half = batch & 1u;
        ok = wait_warp(sempty_bar(half), ((batch >> 1) & 1u) ^ 1u, abort_flag, (4u << 24) | (5u << 16) | (batch & 0xFFFF));
        if (!ok) break;
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          const float wj = __shfl_sync(0xFFFFFFFFu, w, j);
#pragma unroll
          for (int i = 0; i < TPL; ++i) sts32(scales0 + ((half * kBatch + j) * kAcc + 32 * i + lane) * 4, v[j][i] * wj);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(sfull_bar(half));
      }
    }
  } else {
    // ------------------------------------------------------------------ promotion, epilogue
    bool ok = true;
    int stage = 0;
    uint32_t phase = 0, it = 0, batch = 0;
    const uint32_t staging = staging0 + (uint32_t)(warp - 4) * p.staging;
    // bias and stores of one block of 16 tokens
    auto store = [&](const uint64_t* s, int tok, int n0, const float (&bs)[4]) {
      __syncwarp();  // the block before this one has left the staging buffer
      if (p.out_dtype == IFLB200_F32) {
        // 128-byte rows of 32 columns, 16-byte pieces swizzled by the token
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int half = i >> 2, j = (i >> 1) & 1, sub = i & 1;
          float v[2];
          unpack2(s[i], v[0], v[1]);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t chunk = (uint32_t)(4 * half + 2 * sub + (lane >> 4)) ^ (uint32_t)(2 * c4 + e);
            sts32(staging + (8 * j + 2 * c4 + e) * 128 + chunk * 16 + (r4 & 3) * 4, v[e] + bs[2 * half + sub]);
          }
        }
        __syncwarp();
        uint8_t* o = p.out + (int64_t)(tok + (lane >> 3)) * p.ld_out + (int64_t)n0 * 4 + (lane & 7) * 16;
        const bool in = n0 + 4 * (lane & 7) < p.N;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int t = 4 * i + (lane >> 3);
          const uint4 v = lds128(staging + t * 128 + (((lane & 7) ^ (t & 7)) << 4));
          if (in && tok + t < p.M) *reinterpret_cast<uint4*>(o + 4 * i * p.ld_out) = v;
        }
      } else {
        // 64-byte rows of 32 columns, pieces swizzled by the token pair: four 8 x 8 matrices a store, transposed on the way
        const uint32_t row = (uint32_t)(lane & 7), chunk = (uint32_t)(lane >> 3) ^ (row >> 1 & 3);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint32_t v[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float a, b;
            unpack2(s[(i >> 1) * 4 + j * 2 + (i & 1)], a, b);
            a += bs[i];
            b += bs[i];
            v[i] = p.out_dtype == IFLB200_F16 ? pair_f16(a, b) : pair_bf16(a, b);
          }
          store_transposed(staging + (8 * j + row) * 64 + chunk * 16, v);
        }
        __syncwarp();
        uint8_t* o = p.out + (int64_t)(tok + r4) * p.ld_out + (int64_t)n0 * 2 + c4 * 16;
        const bool in = n0 + c4 * 8 < p.N;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint4 v = lds128(staging + (8 * i + r4) * 64 + ((c4 ^ (r4 >> 1 & 3)) << 4));
          if (in && tok + 8 * i + r4 < p.M) *reinterpret_cast<uint4*>(o + 8 * i * p.ld_out) = v;
        }
      }
    };
    grid_dependency_wait();
    for (int unit = first_unit; ok && unit < p.units; unit += unit_stride) {
      int t_blk, w_blk;
      place(unit, t_blk, w_blk);
      const int tok_base = t_blk * p.bt;
      const int n0 = (w_blk * CG + (CG == 2 ? (int)rank : 0)) * kStep + quad * 32;
      const int blocks = n0 < p.N ? min(p.bt, p.M - tok_base + 15) / 16 : 0;
      float bs[4] = {-0.0f, -0.0f, -0.0f, -0.0f};  // an addend of -0 changes nothing
      if (p.bias) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int n = n0 + 8 * i + r4;
          if (n < p.N)
            bs[i] = p.bias_dtype == IFLB200_F32 ? __ldg(reinterpret_cast<const float*>(p.bias) + n)
                                                : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.bias)[n]);
        }
      }
      // sums: block of 16 tokens, then half of the lanes * 4 + eight tokens * 2 + row of 8
      uint64_t acc[2][8];
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[i >> 3][i & 7] = 0;
      // A warp whose tokens are all past the tile's end only keeps the barriers in step.  (A loop of its own, and no branch in
      // the other's body: there the compiler moves the sums from register to register on every path.)
      auto step = [&](auto active) {
        for (int kb = kb0; kb < kb1; kb += SL, ++it) {
          const uint32_t a = it & 1u;
          const int in_batch = (kb - kb0) & (kBatch - 1);
          if (in_batch == 0)
            ok = wait_warp(sfull_bar(batch & 1u), (batch >> 1) & 1u, abort_flag, (3u << 24) | (6u << 16) | (it & 0xFFFF));
          ok = ok && wait_warp(done_bar(stage), phase, abort_flag, (3u << 24) | (4u << 16) | (it & 0xFFFF));
          if (!ok) break;
          tc_fence_after();
          const uint32_t t_acc = tmem_base + ((uint32_t)(quad * 32) << 16) + a * SL * kAcc + 32 * part;
          const uint32_t s_at = scales0 + (((batch & 1u) * kBatch + in_batch) * kAcc + 32 * part + 2 * c4) * 4;
#pragma unroll
          for (int h = 0; h < SL; ++h) {
            // (tokens past the tile's end inside a group are taken too: their sums are never stored)
            uint32_t r[2][16];
            uint64_t sc[4];
            if constexpr (decltype(active)::value) {
              tmem_ld_32(t_acc + h * kAcc, r[0]);
              tmem_ld_32(t_acc + h * kAcc + (16u << 16), r[1]);
#pragma unroll
              for (int j = 0; j < 4; ++j) sc[j] = lds64(s_at + (h * kAcc + 8 * j) * 4);
              tmem_ld_wait();
            }
            if (h == SL - 1) {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) {
                if (CG == 2) arrive_relaxed_cluster(tempty_bar(a), 0);
                else mbar_arrive(tempty_bar(a));
              }
            }
            if constexpr (decltype(active)::value) {
#pragma unroll
              for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int i = 0; i < 8; ++i)  // i: eight tokens * 2 + row of 8
                  acc[i >> 2][half * 4 + (i & 3)] = fma2(pack2(__uint_as_float(r[half][2 * i]), __uint_as_float(r[half][2 * i + 1])),
                                                         sc[i >> 1], acc[i >> 2][half * 4 + (i & 3)]);
            }
          }
          if (++stage == stages) {
            stage = 0;
            phase ^= 1;
          }
          if (in_batch + SL == kBatch || kb + SL >= kb1) {
            __syncwarp();
            if (lane == 0) mbar_arrive(sempty_bar(batch & 1u));
            ++batch;
          }
        }
      };
      if (32 * part < p.bt) step(std::true_type());
      else step(std::false_type());
      if (!ok) break;
      if (CG == 1 && splits > 1) {
        // to the rank that adds the block up: [own block][source rank][quadrant][piece][lane]
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int block = 2 * part + b;
          if (block < blocks) {
            const uint32_t at = meeting0 + (uint32_t)(((block / splits) * splits + (int)rank) * 4 + quad) * 2048 + lane * 16;
            const uint64_t* v = acc[b];
#pragma unroll
            for (int i = 0; i < 4; ++i) st_cluster_64x2(at + i * 512, (uint32_t)(block % splits), v[2 * i], v[2 * i + 1]);
          }
        }
      } else {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int block = 2 * part + b;
          if (block < blocks) store(acc[b], tok_base + 16 * block, n0, bs);
        }
      }
    }
    if (CG == 1 && splits > 1) {
      __syncwarp();
      cluster_arrive();
      cluster_wait();
      int t_blk, w_blk;
      place(first_unit, t_blk, w_blk);
      const int tok_base = t_blk * p.bt, n0 = w_blk * kStep + quad * 32;
      const int blocks = n0 < p.N ? min(p.bt, p.M - tok_base + 15) / 16 : 0;
      float bs[4] = {-0.0f, -0.0f, -0.0f, -0.0f};
      if (p.bias) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int n = n0 + 8 * i + r4;
          if (n < p.N)
            bs[i] = p.bias_dtype == IFLB200_F32 ? __ldg(reinterpret_cast<const float*>(p.bias) + n)
                                                : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.bias)[n]);
        }
      }
      for (int own = part; own < own_blocks; own += 4) {
        const int block = own * splits + (int)rank;
        if (ok && block < blocks) {
          uint64_t s[8] = {};
          for (int src = 0; src < splits; ++src) {
            const uint32_t at = meeting0 + (uint32_t)((own * splits + src) * 4 + quad) * 2048 + lane * 16;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint4 v = lds128(at + i * 512);
              s[2 * i] = add2(s[2 * i], (uint64_t)v.x | ((uint64_t)v.y << 32));
              s[2 * i + 1] = add2(s[2 * i + 1], (uint64_t)v.z | ((uint64_t)v.w << 32));
            }
          }
          store(s, tok_base + 16 * block, n0, bs);
        }
      }
    }
  }
  if (CG == 1 && splits > 1 && warp < 4) {
    __syncwarp();
    cluster_arrive();
    cluster_wait();
  }

  // Neither CTA of a pair leaves while the other's MMAs, commits or arrivals can still reach it.
  if (*abort_flag) {
    for (int i = 0; i < 64; ++i) __nanosleep(1000);
  }
  tc_fence_before();
  if (CG == 2) {
    __syncwarp();
    cluster_arrive();
    cluster_wait();
  } else {
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    if (CG == 2) tmem_dealloc_pair(tmem_base, 512);
    else tmem_dealloc(tmem_base, 512);
  }
}

// --------------------------------------------------------------------------------------------
// Host side
// --------------------------------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                  CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                  CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeTiledFn>(p);
  }();
  return fn;
}

// [rows, K] e4m3, box 128 bytes x box_rows with the 128-byte swizzle, zeros outside.
int operand_map(CUtensorMap* tm, const void* ptr, int rows, int K, int64_t ld, int box_rows) {
  EncodeTiledFn enc = encode_fn();
  if (!enc) return IFLB200_ERR_DRIVER;
  const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld};
  const cuuint32_t box[2] = {(cuuint32_t)kStep, (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  return enc(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? IFLB200_OK
             : IFLB200_ERR_DRIVER;
}

// iflb200_block_linear_set_form; zeros: by rule
int g_form = 0, g_tokens = 0, g_splits = 0;

// Form, tokens of a tile and CTAs to a K range of least estimated time; what is given (not 0) stays.
//
// In microseconds, fitted to shapes of 1 to 4680 tokens, 1024 to 32768 columns, 512 to 16384 deep, in every width and split: a stage takes 0.30 + 0.0016 a token on single CTAs up to 64 tokens and 0.005 a token more above (both operands come
// through one SM), 0.45 on pairs up to 64 tokens and 0.0025 a token more up to 0.575; a quarter less where the GPU is empty.
// A tile's end is 0.4 + 0.006 a token.  Handing partial sums over is 0.4 + 0.25 a CTA; 33 clusters of four and 16 of eight fit
// the GPU.  Over 24 drawn shapes of 1 to 2606 tokens the chosen form took 1.04 times the fastest of all on average, 1.15 at most.
void choose(int M, int N, int stages, int out_dtype, int sms, int& form, int& bt, int& splits) {
  const int staging = out_dtype == IFLB200_F32 ? 2048 : 1024;
  const int form0 = form, bt0 = bt, splits0 = splits;
  double best = 1e30;
  int before = 0;
  for (int t = bt0 ? bt0 : 16; t <= (bt0 ? bt0 : kAcc); t += 16) {
    const int blocks = (M + t - 1) / t;
    if (!bt0 && blocks == before) continue;  // no fewer tiles than the narrower ones
    before = blocks;
    const double end = 0.4 + 0.006 * t, over = t > 64 ? t - 64 : 0;
    for (int f = form0 ? form0 : 1; f <= (form0 ? form0 : 2); ++f) {
      for (int k = splits0 && f == 1 ? splits0 : 1; k <= (f == 2 ? 1 : (splits0 ? splits0 : 8)); k *= 2) {
        if (k > 1 && (k > stages || Layout<1>::stages(t, k, staging) < 2)) continue;  // (a stage in flight needs a second beside it)
        const int64_t units = (int64_t)blocks * ((N + f * kStep - 1) / (f * kStep)) * k;
        const int64_t room = f == 2 ? sms / 2 : (k == 8 ? 128 : (k == 4 ? sms - 16 : sms));
        const int64_t waves = (units + room - 1) / room;
        if (k > 1 && waves > 1 && !splits0) continue;
        const double load = waves == 1 ? (double)units / room : 1.0;
        const double stage = (f == 1 ? 0.30 + 0.0016 * t + 0.0034 * over : (0.45 + 0.0025 * over < 0.575 ? 0.45 + 0.0025 * over : 0.575)) * (0.75 + 0.25 * load);
        const double time = waves * ((stages + k - 1) / k * stage + end) + (k > 1 ? 0.4 + 0.25 * k : 0.0);
        if (time < best) {
          best = time;
          form = f;
          bt = t;
          splits = k;
        }
      }
    }
  }
  if (best == 1e30) {  // (only with a given split that does not fit)
    form = form0 ? form0 : 1;
    bt = bt0 ? bt0 : (M < kAcc ? (M + 15) / 16 * 16 : kAcc);
    splits = 1;
  }
}

template <int CG>
int launch_form(const void* a, int64_t ld_a, const void* w, int64_t ld_w, BlockParams p, int bt, int splits, int sms, cudaStream_t s) {
  using L = Layout<CG>;
  static bool attr_set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return IFLB200_ERR_DEVICE;
  if (!attr_set[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(gemm_fp8_block_kernel<CG>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
    if (e != cudaSuccess) return (int)e;
    attr_set[dev] = true;
  }
  p.bt = bt;
  p.splits = splits;
  p.num_m = (p.M + bt - 1) / bt;
  p.num_n = (p.N + CG * kStep - 1) / (CG * kStep);
  p.blocks = (p.K + kStep - 1) / kStep;
  p.num_k = (p.blocks + SL - 1) / SL * SL;
  p.units = p.num_m * p.num_n;
  p.group_m = p.num_m <= 24 ? p.num_m : 16;
  p.staging = p.out_dtype == IFLB200_F32 ? 2048 : 1024;
  p.stages = L::stages(bt, splits, p.staging);
  p.idesc = make_idesc_e4m3_f32(CG * kStep, bt);
  CUtensorMap tt, tw;
  int st = operand_map(&tt, a, p.M, p.K, ld_a, bt / CG);
  if (st == IFLB200_OK) st = operand_map(&tw, w, p.N, p.K, ld_w, kStep);
  if (st != IFLB200_OK) return st;
  const int most = CG == 2 ? sms / 2 : sms;
  const unsigned ctas = CG == 1 && splits > 1 ? (unsigned)(p.units * splits) : (unsigned)(CG * (p.units < most ? p.units : most));
  const size_t smem = (size_t)L::fixed(bt, splits, p.staging) + (size_t)p.stages * SL * L::slab(bt);
  const cudaError_t e = launch_dep(gemm_fp8_block_kernel<CG>, dim3(ctas), dim3(kThreads), smem, s, CG == 2 ? 2 : splits,
                                   dependent_launch_for(p.M, true), tt, tw, p);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

}  // namespace

int set_block_wait_budget_ns(uint64_t ns) { return set_budget_ns(ns); }
int take_block_timeout_record(uint32_t* record, cudaStream_t s) { return take_record(record, s); }

}  // namespace iflb200

using namespace iflb200;

extern "C" int iflb200_block_linear_set_form(int form, int tokens, int splits) {
  if (form < 0 || form > 2 || tokens < 0 || tokens > kAcc || tokens % 16 || splits < 0 || splits > 8) return IFLB200_ERR_ARG;
  if (form != 1 && splits > 1) return IFLB200_ERR_ARG;
  g_form = form;
  g_tokens = tokens;
  g_splits = splits;
  return IFLB200_OK;
}

extern "C" int iflb200_block_linear(const void* a, int64_t ld_a, const void* w, int64_t ld_w, int M, int N, int K,
                                    const float* a_scale, int64_t a_scale_row, int64_t a_scale_block, const float* w_scale,
                                    const void* bias, int bias_dtype, void* out, int out_dtype, int64_t ld_out, void* stream) {
  if (M < 0 || N < 0 || K < 0) return IFLB200_ERR_ARG;
  if (out_dtype != IFLB200_F32 && out_dtype != IFLB200_BF16 && out_dtype != IFLB200_F16) return IFLB200_ERR_DTYPE;
  if (bias && bias_dtype != IFLB200_F32 && bias_dtype != IFLB200_BF16) return IFLB200_ERR_DTYPE;
  if (K % 16 || N % 16) return IFLB200_ERR_SHAPE;
  if (M == 0 || N == 0) return IFLB200_OK;
  if (K < 16) return IFLB200_ERR_SHAPE;
  if (!a || !w || !out || !a_scale || !w_scale) return IFLB200_ERR_ARG;
  if (ld_a < K || ld_w < K || ld_out < N || a_scale_row < 0 || a_scale_block < 0) return IFLB200_ERR_ARG;
  const int es = out_dtype == IFLB200_F32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(out) | (uintptr_t)ld_a |
       (uintptr_t)ld_w | (uintptr_t)(ld_out * es)) & 15)
    return IFLB200_ERR_ALIGN;
  const int sms = device_sm_count();
  if (sms == 0) return IFLB200_ERR_DEVICE;
  BlockParams p = {};
  p.M = M; p.N = N; p.K = K;
  p.sa = a_scale; p.sa_row = a_scale_row; p.sa_block = a_scale_block;
  p.sw = w_scale;
  p.bias = bias; p.bias_dtype = bias_dtype;
  p.out = reinterpret_cast<uint8_t*>(out);
  p.ld_out = ld_out * es;
  p.out_dtype = out_dtype;
  p.early = M <= kEarlyWeightsMaxRows;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int steps = (K + SL * kStep - 1) / (SL * kStep);  // stages
  int form = g_form, bt = g_tokens, splits = g_splits;
  choose(M, N, steps, out_dtype, sms, form, bt, splits);
  if (form == 2) return launch_form<2>(a, ld_a, w, ld_w, p, bt, 1, sms, s);
  return launch_form<1>(a, ld_a, w, ld_w, p, bt, splits, sms, s);
}
