// Attention over a paged 8-bit cache with a scale for each page and head.
//
//   s[r, j] = scale * ks[page(j)] * sum_d q[r, d] K[j, d];  s = cap tanh(s / cap) where a cap is given;  s -= slope |p_r - j|
//   out[r]  = sum_j exp(s[r, j] - m_r) vs[page(j)] V[j] / sum_j exp(s[r, j] - m_r)          over the keys j < limit_r
//
// Every mask here leaves a row the keys below a limit of its own: the sequence's length, or with a causal mask
// max(position + 1, prefix).
#include "cache_attn.cuh"

namespace iflb200 {

namespace {

constexpr int kWarps = 4;
constexpr int kTile = 32;    // keys a warp takes at a time
constexpr int kStages = 3;

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// 1.0 in each half of x that is a NaN (all bits below the sign set: what a NaN code converts to), else 0.
__device__ __forceinline__ uint32_t nan_halves(uint32_t x) {
  return ((x & 0x7FFF) > 0x7C00 ? 0x3C00u : 0u) | ((x & 0x7FFF0000u) > 0x7C000000u ? 0x3C000000u : 0u);
}
__device__ __forceinline__ uint32_t without_nan(uint32_t x) {
  return ((x & 0x7FFF) > 0x7C00 ? 0u : x & 0xFFFF) | ((x & 0x7FFF0000u) > 0x7C000000u ? 0u : x & 0xFFFF0000u);
}

// ---------------------------------------------------------------------------------------------
// Few rows (query token x head of a group): bound by the cache's bytes.
//
// Keys on the MMA's M side, 8 rows on its N side.  Every warp walks key tiles of its own with a softmax state of its
// own, loads (cp.async, three tiles ahead, 16-byte pieces swizzled for ldmatrix) and all: no barrier until the end.
// Codes become f16 in registers, which is exact; q is f16 too, its row brought near 1 by a power of two (a bf16 row keeps
// all its bits down to 2^-14 of its largest element); weights are f16 relative to the row's running maximum.  All sums
// and the softmax state are fp32.  The two scales of a page are uniform over 16 keys: ks goes into the factor of the
// scores, vs / (the scale that the output is kept in) into the weights ahead of their rounding.
// ---------------------------------------------------------------------------------------------
template <int D, int NT, typename T>
__global__ void __launch_bounds__(32 * kWarps) cache_attend_rows_kernel(const __grid_constant__ AttendArgs a) {
  constexpr int ROWS = 8 * NT, CH = D / 16, KB = kTile * D;  // 16-byte chunks of a key, bytes of a tile of K or V
  constexpr int LPR = CH, RPI = 32 / LPR;                    // lanes a key, keys an instruction of cp.async
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float m_of[kWarps][ROWS], l_of[kWarps][ROWS];
  __shared__ uint32_t last_one;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int split = blockIdx.x, y = blockIdx.y, b = blockIdx.z;
  const int h = y / a.row_tiles, row0 = (y - h * a.row_tiles) * ROWS;
  grid_dependency_wait();
  const int len = min(max(a.lens[b], 0), (int)min((int64_t)a.max_pages * a.P, (int64_t)INT32_MAX));
  const int nq = a.q_lens ? min(max(a.q_lens[b], 0), a.T) : a.T;
  const int rows = min(ROWS, nq * a.G - row0);
  if (rows <= 0) return;
  const int prefix = a.prefix ? a.prefix[b] : 0;
  auto limit_of = [&](int r) { return a.causal ? min(len, max(len - nq + r / a.G + 1, prefix)) : len; };
  // limits grow with the row: the last row's is the largest, the first one's the smallest
  const int most = max(0, limit_of(row0 + rows - 1)), least = limit_of(row0);
  const int chunks = max(1, (most + a.chunk - 1) / a.chunk);
  if (split >= chunks) return;
  const int key0 = split * a.chunk, key1 = min(most, key0 + a.chunk);

  // this thread's columns of the scores: rows 8 n + 2 c + e
  float factor[NT][2], slope[NT][2], pos[NT][2];
  int limit[NT][2];
  uint32_t qf[NT][CH][2];  // q fragments: row 8 n + g, elements 16 i + 4 c .. + 3
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = 8 * n + g;
    const bool in = r < rows;
    const int t = (row0 + (in ? r : 0)) / a.G, hq = h * a.G + (row0 + (in ? r : 0)) - t * a.G;
    const T* q = reinterpret_cast<const T*>(a.q) + b * a.q_b + t * a.q_t + hq * a.q_h;
    float top = 0.0f;
    float x[CH][4];
#pragma unroll
    for (int i = 0; i < CH; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[i][e] = in ? as_float(q[16 * i + 4 * c + e]) : 0.0f;
        if (fabsf(x[i][e]) < 3.39e38f) top = fmaxf(top, fabsf(x[i][e]));
      }
    }
    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
    // 2^-e of the largest finite element's exponent e, within what has a normal reciprocal
    const int e2 = min(max((int)(__float_as_uint(top) >> 23), 2), 252);
    const float down = __uint_as_float((uint32_t)(254 - e2) << 23), up = __uint_as_float((uint32_t)e2 << 23);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      qf[n][i][0] = pack_half2(x[i][0] * down, x[i][1] * down);
      qf[n][i][1] = pack_half2(x[i][2] * down, x[i][3] * down);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      factor[n][e] = __shfl_sync(0xFFFFFFFFu, up, (2 * c + e) * 4) * a.scale;
      const int rr = 8 * n + 2 * c + e, tt = (row0 + rr) / a.G;
      limit[n][e] = rr < rows ? limit_of(row0 + rr) : 0;
      pos[n][e] = (float)(len - nq + tt);
      slope[n][e] = a.slopes && rr < rows ? a.slopes[h * a.G + row0 + rr - tt * a.G] * kLog2e : 0.0f;
    }
  }
  const float inv_cap = a.cap > 0.0f ? 1.0f / a.cap : 0.0f;

  const uint32_t ring = smem_u32(smem) + warp * kStages * 2 * KB;
  const int32_t* table = a.table + b * a.ld_table;
  auto page_of = [&](int key) {  // -1: no such page
    if (key >= key1) return -1;
    const int page = __ldg(table + key / a.P);
    return page >= 0 && page < a.pages ? page : -1;
  };
  const int64_t head_bytes = (int64_t)a.P * D;
  auto load = [&](int key, int slot, int p0, int p1) {
    // keys key .. key + 31, of pages p0 (first sixteen) and p1
    const uint32_t dst = ring + slot * 2 * KB;
#pragma unroll
    for (int i = 0; i < kTile / RPI; ++i) {
      const int row = i * RPI + lane / LPR, chunk = lane % LPR, kk = key + row;
      const int page = row < 16 ? p0 : p1;
      const bool in = kk < key1 && page >= 0;
      const int64_t off = in ? ((int64_t)page * a.H + h) * head_bytes + (int64_t)(kk % a.P) * D + chunk * 16 : 0;
      const int sw = D == 64 ? chunk ^ (row >> 1 & 3) : chunk ^ (row & 7);
      cp_async_16(dst + row * D + sw * 16, a.k + off, in ? 16 : 0);
      cp_async_16(dst + KB + row * D + sw * 16, a.v + off, in ? 16 : 0);
    }
  };

  float acc[NT][CH][4] = {};  // output, transposed: elements 16 i + 2 g (c0, c1) and + 1 (c2, c3) of rows 2 c, 2 c + 1
  float run[NT][2], sum[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      run[n][e] = -INFINITY;
      sum[n][e] = 0.0f;
    }
  float vref = 0.0f;
  constexpr int STEP = kWarps * kTile;
  int pages[kStages][2];
  float kss[kStages][2], vss[kStages][2];
  auto fetch = [&](int key, int s) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int page = page_of(key + 16 * u);
      pages[s][u] = page;
      kss[s][u] = page >= 0 ? __ldg(a.ks + (int64_t)page * a.H + h) : 0.0f;
      vss[s][u] = page >= 0 ? __ldg(a.vs + (int64_t)page * a.H + h) : 0.0f;
    }
    if (key < key1) load(key, s, pages[s][0], pages[s][1]);
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  const int first = key0 + warp * kTile;
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) fetch(first + s * STEP, s);
  for (int base = first; base < key1; base += kStages * STEP) {
#pragma unroll
    for (int s = 0; s < kStages; ++s) {
      const int key = base + s * STEP;
      if (key >= key1) break;
      fetch(key + (kStages - 1) * STEP, (s + kStages - 1) % kStages);
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
      __syncwarp();
      const uint32_t kt = ring + s * 2 * KB, vt = kt + KB;
      // scores of two 16-key units
      float sc[2][NT][4];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int n = 0; n < NT; ++n) sc[u][n][0] = sc[u][n][1] = sc[u][n][2] = sc[u][n][3] = 0.0f;
        const int row = 16 * u + (lane & 15);
#pragma unroll
        for (int i = 0; i < CH; i += 2) {
          uint32_t r[4];
          const int chunk = i + (lane >> 4), sw = D == 64 ? chunk ^ (row >> 1 & 3) : chunk ^ (row & 7);
          ldsm_x4(kt + row * D + sw * 16, r);
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const uint32_t f[4] = {e4m3x2_f16x2(r[2 * x]), e4m3x2_f16x2(r[2 * x + 1]), e4m3x2_f16x2(r[2 * x] >> 16),
                                   e4m3x2_f16x2(r[2 * x + 1] >> 16)};
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_f16(sc[u][n], f, qf[n][i + x][0], qf[n][i + x][1]);
          }
        }
      }
      // to base-2 exponents; masked where a row does not reach
      const bool edge = key + kTile > least || pages[s][0] < 0 || pages[s][1] < 0;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int j = key + 16 * u + g + (e >> 1) * 8;
            float x = sc[u][n][e] * (factor[n][e & 1] * kss[s][u]);
            if (a.cap > 0.0f) x = soft_cap(x, a.cap, inv_cap);
            x *= kLog2e;
            if (a.slopes) x -= slope[n][e & 1] * fabsf(pos[n][e & 1] - (float)j);
            if (edge && (j >= limit[n][e & 1] || pages[s][u] < 0)) x = -INFINITY;
            sc[u][n][e] = x;
          }
        }
      }
      // the running maximum moves only when a score passes it by more than kLazy
      float top[NT][2];
      bool moves = false;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          top[n][e] = fmaxf(fmaxf(sc[0][n][e], sc[0][n][e + 2]), fmaxf(sc[1][n][e], sc[1][n][e + 2]));
          moves |= top[n][e] > run[n][e] + kLazy;
        }
      }
      if (__any_sync(0xFFFFFFFFu, moves)) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float f[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float t = top[n][e];
            t = fmaxf(t, __shfl_xor_sync(0xFFFFFFFFu, t, 4));
            t = fmaxf(t, __shfl_xor_sync(0xFFFFFFFFu, t, 8));
            t = fmaxf(t, __shfl_xor_sync(0xFFFFFFFFu, t, 16));
            t = fmaxf(t, run[n][e]);
            f[e] = run[n][e] == -INFINITY ? 0.0f : ex2_approx_ftz(run[n][e] - t);
            run[n][e] = t;
            sum[n][e] *= f[e];
          }
#pragma unroll
          for (int i = 0; i < CH; ++i) {
            acc[n][i][0] *= f[0];
            acc[n][i][1] *= f[1];
            acc[n][i][2] *= f[0];
            acc[n][i][3] *= f[1];
          }
        }
      }
      // weights
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float m = run[n][e & 1];
            sc[u][n][e] = ex2_approx_ftz(sc[u][n][e] - (m == -INFINITY ? 0.0f : m));
            sum[n][e & 1] += sc[u][n][e];
          }
        }
      }
      uint32_t seen[2][NT][2];
      // A NaN among the values of a tile that some row sees only in part: it belongs to the rows that see it alone
      bool nan_here = false;
      if (edge) {
        for (int i = lane; i < KB / 16; i += 32) {
          uint4 x;
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(vt + i * 16));
          const uint32_t z[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) nan_here |= __vcmpeq4(z[e] & 0x7F7F7F7Fu, 0x7F7F7F7Fu) != 0;
        }
        nan_here = __any_sync(0xFFFFFFFFu, nan_here);
        if (nan_here) {
#pragma unroll
          for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              float see[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) see[e] = key + 16 * u + g + (e >> 1) * 8 < limit[n][e & 1] ? 1.0f : 0.0f;
              seen[u][n][0] = transpose8x8(pack_half2(see[0], see[1]));
              seen[u][n][1] = transpose8x8(pack_half2(see[2], see[3]));
            }
          }
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        // the output is kept in units of vref: another page's scale goes into the weights, within what f16 takes
        float ratio = 0.0f;
        if (pages[s][u] >= 0) {
          if (vref == 0.0f) vref = vss[s][u];
          ratio = vref == 0.0f ? 0.0f : __fdividef(vss[s][u], vref);
          if (ratio != 0.0f && (ratio > 64.0f || ratio < 0.015625f)) {
            const float f = fminf(vref / vss[s][u], 1e38f);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int i = 0; i < CH; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[n][i][e] *= f;
            vref = vss[s][u];
            ratio = 1.0f;
          }
        }
        // 16 keys x 8 rows transposed into the MMA's B fragments
        uint32_t w[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          w[n][0] = transpose8x8(pack_half2(sc[u][n][0] * ratio, sc[u][n][1] * ratio));
          w[n][1] = transpose8x8(pack_half2(sc[u][n][2] * ratio, sc[u][n][3] * ratio));
        }
        const int row = 16 * u + (lane & 15);
#pragma unroll
        for (int i = 0; i < CH; i += 2) {
          uint32_t r[4];
          const int chunk = i + (lane >> 4), sw = D == 64 ? chunk ^ (row >> 1 & 3) : chunk ^ (row & 7);
          ldsm_x4_trans(vt + row * D + sw * 16, r);
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            // a register has two elements of two neighbouring keys: pair the keys
            const uint32_t lo = __byte_perm(r[2 * x], 0, 0x3120), hi = __byte_perm(r[2 * x + 1], 0, 0x3120);
            uint32_t f[4] = {e4m3x2_f16x2(lo), e4m3x2_f16x2(lo >> 16), e4m3x2_f16x2(hi), e4m3x2_f16x2(hi >> 16)};
            if (nan_here) {
              const uint32_t at[4] = {nan_halves(f[0]), nan_halves(f[1]), nan_halves(f[2]), nan_halves(f[3])};
#pragma unroll
              for (int z = 0; z < 4; ++z) f[z] = without_nan(f[z]);
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                float hits[4] = {};
                mma_f16(hits, at, seen[u][n][0], seen[u][n][1]);
#pragma unroll
                for (int z = 0; z < 4; ++z)
                  if (hits[z] > 0.0f) acc[n][i + x][z] = __uint_as_float(0x7FC00000u);
              }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_f16(acc[n][i + x], f, w[n][0], w[n][1]);
          }
        }
      }
      __syncwarp();
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  grid_launch_dependents();

  // the warps' states meet in shared memory: [warp][row][D], rows padded by eight floats
  __syncthreads();
  float* part = reinterpret_cast<float*>(smem);
  constexpr int LD = D + 8;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float l = sum[n][e];
      l += __shfl_xor_sync(0xFFFFFFFFu, l, 4);
      l += __shfl_xor_sync(0xFFFFFFFFu, l, 8);
      l += __shfl_xor_sync(0xFFFFFFFFu, l, 16);
      const int r = 8 * n + 2 * c + e;
      if (g == 0) {
        m_of[warp][r] = run[n][e];
        l_of[warp][r] = l;
      }
#pragma unroll
      for (int i = 0; i < CH; ++i)
        *reinterpret_cast<float2*>(part + (warp * ROWS + r) * LD + 16 * i + 2 * g) =
            make_float2(acc[n][i][e] * vref, acc[n][i][e + 2] * vref);
    }
  }
  __syncthreads();
  const int ticket = b * a.H * a.row_tiles + y;
  T* out = reinterpret_cast<T*>(a.out);
  auto out_row = [&](int r) {
    const int t = (row0 + r) / a.G, hq = h * a.G + (row0 + r) - t * a.G;
    return out + b * a.o_b + t * a.o_t + hq * a.o_h;
  };
  for (int i = threadIdx.x; i < rows * D; i += 32 * kWarps) {
    const int r = i / D, d = i - r * D;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m = fmaxf(m, m_of[w][r]);
    float l = 0.0f, o = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = m_of[w][r] == -INFINITY ? 0.0f : ex2_approx_ftz(m_of[w][r] - m);
      l += m_of[w][r] == -INFINITY ? l_of[w][r] : f * l_of[w][r];
      o += m_of[w][r] == -INFINITY ? part[(w * ROWS + r) * LD + d] : f * part[(w * ROWS + r) * LD + d];
    }
    if (chunks == 1) {
      put(out_row(r) + d, l == 0.0f ? 0.0f : o / l);
    } else {
      const int64_t at = ((int64_t)ticket * a.splits + split) * ROWS + r;
      a.partial[at * D + d] = o;
      if (d == 0) *reinterpret_cast<float2*>(a.partial + a.partial_ml + at * 2) = make_float2(m, l);
    }
  }
  if (chunks == 1) return;
  // the last CTA of the chunks adds them up, in their order
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last_one = atomicAdd(a.tickets + ticket, 1u) == (uint32_t)chunks - 1 ? 1u : 0u;
  __syncthreads();
  if (!last_one) return;
  __threadfence();
  if (threadIdx.x == 0) a.tickets[ticket] = 0;
  const float2* ml = reinterpret_cast<const float2*>(a.partial + a.partial_ml) + (int64_t)ticket * a.splits * ROWS;
  const float* po = a.partial + (int64_t)ticket * a.splits * ROWS * D;
  for (int i = threadIdx.x; i < rows * D; i += 32 * kWarps) {
    const int r = i / D, d = i - r * D;
    float m = -INFINITY;
    for (int s = 0; s < chunks; ++s) m = fmaxf(m, __ldcg(ml + s * ROWS + r).x);
    float l = 0.0f, o = 0.0f;
    for (int s = 0; s < chunks; ++s) {
      const float2 x = __ldcg(ml + s * ROWS + r);
      const float f = x.x == -INFINITY ? 1.0f : ex2_approx_ftz(x.x - m);
      l += f * x.y;
      o += f * __ldcg(po + ((int64_t)s * ROWS + r) * D + d);
    }
    put(out_row(r) + d, l == 0.0f ? 0.0f : o / l);
  }
}

template <int D, int NT, typename T>
int launch_rows(const AttendArgs& a, cudaStream_t s) {
  constexpr int ring = kWarps * kStages * 2 * kTile * D, meet = kWarps * 8 * NT * (D + 8) * 4;
  constexpr int smem = ring > meet ? ring : meet;
  static bool attr_set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return IFLB200_ERR_DEVICE;
  if (!attr_set[dev]) {
    const cudaError_t e =
        cudaFuncSetAttribute(cache_attend_rows_kernel<D, NT, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return (int)e;
    attr_set[dev] = true;
  }
  const dim3 grid((unsigned)a.splits, (unsigned)(a.H * a.row_tiles), (unsigned)a.B);
  const cudaError_t e = launch_dep(cache_attend_rows_kernel<D, NT, T>, grid, dim3(32 * kWarps), smem, s, 1,
                                   dependent_launch_for((int64_t)a.B * a.T), a);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

// iflb200_cache_attention_set_form; 0: by rule
int g_form = 0;
constexpr int64_t kFewRows = 32;

template <typename T>
int attend(AttendArgs a, int D, void* workspace, int64_t bytes, cudaStream_t s) {
  const int64_t rows = (int64_t)a.T * a.G;
  const bool many = g_form == 2 || (g_form == 0 && rows > kFewRows);
  const int nt = D == 256 || rows <= 8 ? 1 : 2, per = many ? attend_tiles_rows(D) : 8 * nt;
  const int64_t tiles = (rows + per - 1) / per;
  if (tiles * a.H > 65535) return IFLB200_ERR_SHAPE;
  a.row_tiles = (int)tiles;
  const int sms = device_sm_count();
  if (sms == 0) return IFLB200_ERR_DEVICE;
  // Chunks of keys: enough for two waves of CTAs, none shorter than a step of all warps, as many as the workspace takes.
  const int64_t keys = (int64_t)a.max_pages * a.P, units = (int64_t)a.B * a.H * tiles;
  constexpr int64_t kLeast = kWarps * kTile;
  const int64_t want = ((many ? 1ll : 4ll) * sms + units - 1) / units;
  // The tickets have a place of their own whatever the geometry: they are zero between calls, partial results are not.
  // (Sequences are only shared where there are fewer units than CTAs wanted.)
  constexpr int64_t head = 4096;
  const int64_t each = units * per * (D + 2) * 4;
  const int64_t room = workspace && bytes > head ? (bytes - head) / each : 0;
  int64_t splits = units * 4 > head ? 1 : (want < room ? want : room);
  if (splits < 1) splits = 1;
  int64_t chunk = ((keys + splits - 1) / splits + kLeast - 1) / kLeast * kLeast;
  if (chunk < kLeast) chunk = kLeast;
  if (chunk > (1 << 30)) chunk = 1 << 30;
  a.chunk = (int)chunk;
  a.splits = (int)((keys + chunk - 1) / chunk);
  if (a.splits < 1) a.splits = 1;
  a.tickets = reinterpret_cast<uint32_t*>(workspace);
  a.partial = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(workspace) + head);
  a.partial_ml = units * a.splits * per * D;
  if (many) return launch_attend_tiles<T>(a, D, s);
  if (D == 64) return nt == 1 ? launch_rows<64, 1, T>(a, s) : launch_rows<64, 2, T>(a, s);
  if (D == 128) return nt == 1 ? launch_rows<128, 1, T>(a, s) : launch_rows<128, 2, T>(a, s);
  return launch_rows<256, 1, T>(a, s);
}

}  // namespace

}  // namespace iflb200

using namespace iflb200;

extern "C" int iflb200_cache_attention_set_form(int form) {
  if (form < 0 || form > 2) return IFLB200_ERR_ARG;
  g_form = form;
  return IFLB200_OK;
}

extern "C" int iflb200_cache_attention(const void* q, int dtype, int64_t q_b, int64_t q_t, int64_t q_h, const void* k_codes,
                                       const void* v_codes, const float* k_scale, const float* v_scale, int pages,
                                       int page_tokens, int head_dim, const int32_t* table, int64_t ld_table, int max_pages,
                                       const int32_t* lens, const int32_t* q_lens, const int32_t* prefix, const float* slopes,
                                       int B, int T, int heads_q, int heads_kv, float scale, float softcap, int causal, void* out,
                                       int64_t o_b, int64_t o_t, int64_t o_h, void* workspace, int64_t workspace_bytes,
                                       void* stream) {
  if (B < 0 || T < 0 || heads_q < 1 || heads_kv < 1 || pages < 0 || max_pages < 0 || workspace_bytes < 0) return IFLB200_ERR_ARG;
  if (dtype != IFLB200_BF16 && dtype != IFLB200_F16) return IFLB200_ERR_DTYPE;
  if ((head_dim != 64 && head_dim != 128 && head_dim != 256) || page_tokens < 16 || page_tokens > 256 || page_tokens % 16 ||
      heads_q % heads_kv || B > 65535)
    return IFLB200_ERR_SHAPE;
  if (!(softcap >= 0.0f) || !(scale == scale) || (prefix && !causal)) return IFLB200_ERR_ARG;
  if (B == 0 || T == 0) return IFLB200_OK;
  if (!q || !out || !lens) return IFLB200_ERR_ARG;
  if (pages > 0 && max_pages > 0 && (!k_codes || !v_codes || !k_scale || !v_scale || !table)) return IFLB200_ERR_ARG;
  if ((int64_t)max_pages * page_tokens > (1 << 30) || (int64_t)T * (heads_q / heads_kv) > (1 << 30)) return IFLB200_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(k_codes) | reinterpret_cast<uintptr_t>(v_codes) | reinterpret_cast<uintptr_t>(workspace)) % 16)
    return IFLB200_ERR_ALIGN;
  AttendArgs a = {};
  a.q = q; a.q_b = q_b; a.q_t = q_t; a.q_h = q_h;
  a.out = out; a.o_b = o_b; a.o_t = o_t; a.o_h = o_h;
  a.k = reinterpret_cast<const uint8_t*>(k_codes);
  a.v = reinterpret_cast<const uint8_t*>(v_codes);
  a.ks = k_scale; a.vs = v_scale;
  a.table = table; a.ld_table = ld_table;
  a.lens = lens; a.q_lens = q_lens; a.prefix = prefix; a.slopes = slopes;
  a.scale = scale; a.cap = softcap;
  a.B = B; a.T = T; a.HQ = heads_q; a.H = heads_kv; a.G = heads_q / heads_kv;
  a.P = page_tokens; a.pages = pages; a.max_pages = pages > 0 ? max_pages : 0; a.causal = causal;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return dtype == IFLB200_BF16 ? attend<__nv_bfloat16>(a, head_dim, workspace, workspace_bytes, s)
                               : attend<__half>(a, head_dim, workspace, workspace_bytes, s);
}
