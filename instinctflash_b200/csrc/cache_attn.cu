// Attention over a paged 8-bit cache with a scale for each page and head.
//
//   s[r, j] = scale * ks[page(j)] * sum_d q[r, d] K[j, d];  s = cap tanh(s / cap) where a cap is given;  s -= slope |p_r - j|
//   out[r]  = sum_j exp(s[r, j] - m_r) vs[page(j)] V[j] / sum_j exp(s[r, j] - m_r)          over the keys j < limit_r
//
// Every mask here leaves a row the keys below a limit of its own: the sequence's length, or with a causal mask
// max(position + 1, prefix).
#include "cache_attn.cuh"

#include <float.h>

namespace iflb200 {

namespace {

constexpr int kWarps = 4;
constexpr int kTile = 32;    // keys a warp takes at a time
constexpr int kStages = 2;

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
// Four elements of a row; `vec`: rows are 8-byte aligned.
template <typename T>
__device__ __forceinline__ void put4(T* p, float a, float b, float c, float d, int vec) {
  T x[4];
  put(x, a);
  put(x + 1, b);
  put(x + 2, c);
  put(x + 3, d);
  if (vec) {
    uint2 u;
    u.x = *reinterpret_cast<const uint16_t*>(x) | (uint32_t)*reinterpret_cast<const uint16_t*>(x + 1) << 16;
    u.y = *reinterpret_cast<const uint16_t*>(x + 2) | (uint32_t)*reinterpret_cast<const uint16_t*>(x + 3) << 16;
    *reinterpret_cast<uint2*>(p) = u;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = x[i];
  }
}

// ---------------------------------------------------------------------------------------------
// Few rows (query token x head of a group): bound by the cache's bytes.
//
// Keys on the MMA's M side, 8 rows on its N side.  Every warp walks key tiles of its own with a softmax state of its
// own, loads (cp.async, one tile ahead, 16-byte pieces swizzled for ldmatrix) and all: no barrier until the end.
// Codes become f16 in registers, which is exact; q is f16 too, its row brought by a power of two to where f16 ends (a bf16 element
// keeps all its bits down to 2^-32 of the row's largest, 2^-17 with that at 1; an f16 row loses nothing); weights are f16 with the row's running maximum at 2^10 (kWeightTop).  All sums
// and the softmax state are fp32.
//
// The scales of a page are uniform over 16 keys: ks is part of the scores' factor, vs part of the exponent, as in
// cache_attn_tiles.cu: weights 2^(y - M + 10) with y = x + log2 vs, l = sum 2^(y - M + 10) / vs, output = (sum of weights times
// codes) / l.  Sixteen tiles' pages and scales are looked up at a time, one unit of sixteen keys a lane.
//
// The code is kept short (loops over stages are not unrolled, what is rare is out of the way): a step of few rows is as much
// instruction fetch as memory (32 sequences up to 8192 long, 8 heads of 128 with four rows each: 248 -> 80 us when it was made short).
// ---------------------------------------------------------------------------------------------

// NaN codes of a tile's values: the first key that has one, by column, and zeros in their place.
__device__ __noinline__ void take_nans(uint32_t vt, int bytes, int D, int key, int lane, int* first_nan) {
#pragma unroll 1
  for (int i = lane; i < bytes / 4; i += 32) {
    uint32_t w;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(vt + 4 * i));
    if (__vcmpeq4(w & 0x7F7F7F7Fu, 0x7F7F7F7Fu) == 0) continue;
    const int row = 4 * i / D, at = 4 * i % D, chunk = at >> 4;
    const int d = (D == 64 ? chunk ^ (row >> 1 & 3) : chunk ^ (row & 7)) * 16 + (at & 15);
#pragma unroll 1
    for (int e = 0; e < 4; ++e) {
      if ((w >> (8 * e) & 0x7F) == 0x7F) {
        atomicMin(first_nan + d + e, key + row);
        w &= ~(0xFFu << (8 * e));
      }
    }
    asm volatile("st.shared.b32 [%0], %1;" ::"r"(vt + 4 * i), "r"(w) : "memory");
  }
  __syncwarp();
}

template <int D, int NT, typename T, bool CAP>
__global__ void __launch_bounds__(32 * kWarps) cache_attend_rows_kernel(const __grid_constant__ AttendArgs a, const int vec) {
  constexpr int ROWS = 8 * NT, CH = D / 16, KB = kTile * D;  // 16-byte chunks of a key, bytes of a tile of K or V
  constexpr int LPR = CH, RPI = 32 / LPR;                    // lanes a key, keys an instruction of cp.async
  constexpr int STEP = kWarps * kTile;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float m_of[kWarps][ROWS], l_of[kWarps][ROWS];
  __shared__ int first_nan[D];
  __shared__ int limits[ROWS];
  __shared__ float4 unit[kWarps][kStages][2];  // of a stage's units: ks, log2 vs, 1 / vs, weight in the product (-1: no page)
  __shared__ uint32_t last_one;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int split = blockIdx.x, y = blockIdx.y, b = blockIdx.z;
  const int h = y / a.row_tiles, row0 = (y - h * a.row_tiles) * ROWS;
  for (int i = threadIdx.x; i < D; i += 32 * kWarps) first_nan[i] = INT32_MAX;
  grid_dependency_wait();
  const int room = a.max_pages * a.P;   // (at most 2^30)
  const int key0 = split * a.chunk, first = key0 + warp * kTile;
  const int32_t* table = a.table + b * a.ld_table;
  // this lane's unit of the sixteen tiles from `tile` on
  auto raw_page = [&](int tile) {
    const int key = first + (tile + (lane >> 1)) * STEP + 16 * (lane & 1);
    return key < room ? __ldg(table + key / a.P) : -1;
  };
  int page = raw_page(0), page_next = -1;
  const int len = min(max(a.lens[b], 0), room);
  const int nq = a.q_lens ? min(max(a.q_lens[b], 0), a.T) : a.T;
  const int prefix = a.prefix ? a.prefix[b] : 0;
  const int rows = min(ROWS, nq * a.G - row0);
  if (rows <= 0) return;
  auto limit_of = [&](int r) { return a.causal ? min(len, max(len - nq + r / a.G + 1, prefix)) : len; };
  // limits grow with the row: the last row's is the largest, the first one's the smallest
  const int most = max(0, limit_of(row0 + rows - 1)), least = limit_of(row0);
  const int chunks = max(1, (most + a.chunk - 1) / a.chunk);
  if (split >= chunks) return;
  const int key1 = min(most, key0 + a.chunk);
  if (threadIdx.x < ROWS) limits[threadIdx.x] = (int)threadIdx.x < rows ? limit_of(row0 + threadIdx.x) : 0;
  __syncthreads();

  const uint32_t ring = smem_u32(smem) + warp * kStages * 2 * KB;
  const int64_t head_bytes = (int64_t)a.P * D;
  float ks = 0.0f, vs = 0.0f;
  int in_page = 0;  // of this lane's unit: its first key in the page
  auto look_up = [&](int tile) {
    const int key = first + (tile + (lane >> 1)) * STEP + 16 * (lane & 1);
    if (page < 0 || page >= a.pages || key >= key1) page = -1;
    in_page = key % a.P;
    ks = page >= 0 ? __ldg(a.ks + (int64_t)page * a.H + h) : 0.0f;
    vs = page >= 0 ? __ldg(a.vs + (int64_t)page * a.H + h) : 0.0f;
  };
  // Tile `tile` into its stage; its units are lanes 2 (tile % 16) and the next.  What is not there becomes zeros.
  const int load_row = lane / LPR, load_chunk = lane % LPR;
  auto fetch = [&](int tile, int stage) {
    const int key = first + tile * STEP;
    if (key < key1) {
      const int src = 2 * (tile & 15);
      if (src == 0) {
        if (tile > 0) page = page_next;
        look_up(tile);
      } else if (src == 16) {
        page_next = raw_page(tile + 8);
      }
      if ((lane >> 1) == (tile & 15)) {
        // (a value scale of zero: the weights count, their product is nothing)
        const bool nil = vs == 0.0f;
        unit[warp][stage][lane & 1] = make_float4(ks, nil ? kNilLog2 : log2_approx(vs), nil ? kNilInverse : 1.0f / vs, page < 0 ? -1.0f : (nil ? 0.0f : 1.0f));
      }
      const int p0 = __shfl_sync(0xFFFFFFFFu, page, src), p1 = __shfl_sync(0xFFFFFFFFu, page, src + 1);
      const int i0 = __shfl_sync(0xFFFFFFFFu, in_page, src), i1 = __shfl_sync(0xFFFFFFFFu, in_page, src + 1);
      const int64_t o0 = ((int64_t)max(p0, 0) * a.H + h) * head_bytes + i0 * D, o1 = ((int64_t)max(p1, 0) * a.H + h) * head_bytes + i1 * D;
      const uint32_t dst = ring + stage * 2 * KB;
#pragma unroll
      for (int i = 0; i < kTile / RPI; ++i) {
        const int row = i * RPI + load_row;
        const bool in = key + row < key1 && (i < kTile / RPI / 2 ? p0 : p1) >= 0;
        const int64_t off = in ? (i < kTile / RPI / 2 ? o0 : o1) + (row & 15) * D + load_chunk * 16 : 0;
        const uint32_t at = dst + row * D + (D == 64 ? load_chunk ^ (row >> 1 & 3) : load_chunk ^ (row & 7)) * 16;
        cp_async_16(at, a.k + off, in ? 16 : 0);
        cp_async_16(at + KB, a.v + off, in ? 16 : 0);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll 1
  for (int s = 0; s < kStages - 1; ++s) fetch(s, s);

  // this thread's columns of the scores: rows 8 n + 2 c + e
  float factor[NT][2], slope[NT][2];
  int limit[NT][2], pos[NT][2];  // pos: the row's position, less the thread's first key in a tile
  uint32_t qf[NT][CH][2];  // q fragments: row 8 n + g, elements 16 i + 4 c .. + 3
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = 8 * n + g;
    const bool in = r < rows;
    const int t = (row0 + (in ? r : 0)) / a.G, hq = h * a.G + (row0 + (in ? r : 0)) - t * a.G;
    const T* q = reinterpret_cast<const T*>(a.q) + b * a.q_b + t * a.q_t + hq * a.q_h + 4 * c;
    uint2 x[CH];
    if (vec) {
#pragma unroll
      for (int i = 0; i < CH; ++i) x[i] = *reinterpret_cast<const uint2*>(q + 16 * i);
    } else {
      const uint16_t* u = reinterpret_cast<const uint16_t*>(q);
#pragma unroll
      for (int i = 0; i < CH; ++i)
        x[i] = make_uint2(u[16 * i] | (uint32_t)u[16 * i + 1] << 16, u[16 * i + 2] | (uint32_t)u[16 * i + 3] << 16);
    }
    float top = 0.0f;
    auto value = [&](uint32_t w, int half) {
      const uint16_t bits = (uint16_t)(w >> (16 * half));
      return as_float(*reinterpret_cast<const T*>(&bits));
    };
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      if (!in) x[i] = make_uint2(0, 0);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float z = fabsf(value(e < 2 ? x[i].x : x[i].y, e & 1));
        if (z < 3.39e38f) top = fmaxf(top, z);
      }
    }
    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
    // the largest finite element to 2^15 .. 2^16, within what has a normal reciprocal
    const int e2 = max((int)(__float_as_uint(top) >> 23), 16);
    const float down = __uint_as_float((uint32_t)(269 - e2) << 23), up = __uint_as_float((uint32_t)(e2 - 15) << 23);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      qf[n][i][0] = pack_half2(value(x[i].x, 0) * down, value(x[i].x, 1) * down);
      qf[n][i][1] = pack_half2(value(x[i].y, 0) * down, value(x[i].y, 1) * down);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      factor[n][e] = __shfl_sync(0xFFFFFFFFu, up, (2 * c + e) * 4) * a.scale * (CAP ? 1.0f : kLog2e);
      const int rr = 8 * n + 2 * c + e, tt = (row0 + rr) / a.G;
      limit[n][e] = rr < rows ? limit_of(row0 + rr) : 0;
      pos[n][e] = len - nq + tt - g;
      slope[n][e] = a.slopes && rr < rows ? a.slopes[h * a.G + row0 + rr - tt * a.G] * kLog2e : 0.0f;
    }
  }
  const float inv_cap = CAP ? 1.0f / a.cap : 0.0f;

  float acc[NT][CH][4] = {};  // output, transposed: elements 16 i + 2 g (c0, c1) and + 1 (c2, c3) of rows 2 c, 2 c + 1
  float run[NT][2], sum[NT][2];
  float top_scale = -INFINITY;  // the largest value scale so far, to base 2
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      run[n][e] = -INFINITY;
      sum[n][e] = 0.0f;
    }
  int stage = 0, ahead = kStages - 1;
#pragma unroll 1
  for (int tile = 0; first + tile * STEP < key1; ++tile) {
    const int key = first + tile * STEP;
    fetch(tile + kStages - 1, ahead);
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
    __syncwarp();
    const uint32_t kt = ring + stage * 2 * KB, vt = kt + KB;
    const float4 un[2] = {unit[warp][stage][0], unit[warp][stage][1]};
    if (++stage == kStages) stage = 0;
    if (++ahead == kStages) ahead = 0;
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
    // to base-2 exponents with the value scale; masked where a row does not reach
    const bool edge = key + kTile > least || un[0].w < 0.0f || un[1].w < 0.0f;
    float top[NT][2];
    bool moves = false;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x = sc[u][n][e] * (factor[n][e & 1] * un[u].x);
          if (CAP) x = soft_cap(x, a.cap, inv_cap) * kLog2e;
          sc[u][n][e] = x + un[u].y;
        }
      }
      if (a.slopes) {
        // (whole numbers first: beyond 2^24 positions are no floats)
        const float from[2] = {(float)(pos[n][0] - key), (float)(pos[n][1] - key)};
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[u][n][e] = fmaf(-slope[n][e & 1], fabsf(from[e & 1] - (float)(16 * u + (e >> 1) * 8)), sc[u][n][e]);
      }
      if (edge) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (key + 16 * u + g + (e >> 1) * 8 >= limit[n][e & 1] || un[u].w < 0.0f) sc[u][n][e] = -INFINITY;
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        top[n][e] = fmaxf(fmaxf(sc[0][n][e], sc[0][n][e + 2]), fmaxf(sc[1][n][e], sc[1][n][e + 2]));
        moves |= top[n][e] > run[n][e] + kLazy;
      }
    }
    // the running maximum moves only when a score passes it by more than kLazy
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
    // A NaN among the values of a tile that some row sees only in part belongs to the rows that see it alone.
    if (edge) {
      bool nan_here = false;
#pragma unroll 1
      for (int i = lane; i < KB / 16; i += 32) {
        uint4 x;
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(vt + i * 16));
        nan_here |= (__vcmpeq4(x.x & 0x7F7F7F7Fu, 0x7F7F7F7Fu) | __vcmpeq4(x.y & 0x7F7F7F7Fu, 0x7F7F7F7Fu) |
                     __vcmpeq4(x.z & 0x7F7F7F7Fu, 0x7F7F7F7Fu) | __vcmpeq4(x.w & 0x7F7F7F7Fu, 0x7F7F7F7Fu)) != 0;
      }
      if (__any_sync(0xFFFFFFFFu, nan_here)) take_nans(vt, KB, D, key, lane, first_nan);
    }
    // weights, 16 keys x 8 rows transposed into the MMA's B fragments, and their product with the codes
    uint32_t w[2][NT][2];
    auto weights = [&](int u, int n, float m0, float m1, float inverse0, float inverse1) {
      float p[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        p[e] = ex2_approx_ftz(sc[u][n][e] - (e & 1 ? m1 : m0));
        sum[n][e & 1] = fmaf(p[e], e & 1 ? inverse1 : inverse0, sum[n][e & 1]);
      }
      const bool nil = un[u].w == 0.0f;
      w[u][n][0] = transpose8x8(nil ? 0u : pack_half2(p[0], p[1]));
      w[u][n][1] = transpose8x8(nil ? 0u : pack_half2(p[2], p[3]));
    };
    // Values 16 i .. + 31 of a unit's keys as A fragments.
    auto values = [&](int u, int i, uint32_t (&f)[2][4]) {
      uint32_t r[4];
      const int row = 16 * u + (lane & 15), chunk = i + (lane >> 4), sw = D == 64 ? chunk ^ (row >> 1 & 3) : chunk ^ (row & 7);
      ldsm_x4_trans(vt + row * D + sw * 16, r);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        // a register has two elements of two neighbouring keys: pair the keys
        const uint32_t lo = __byte_perm(r[2 * x], 0, 0x3120), hi = __byte_perm(r[2 * x + 1], 0, 0x3120);
        f[x][0] = e4m3x2_f16x2(lo);
        f[x][1] = e4m3x2_f16x2(lo >> 16);
        f[x][2] = e4m3x2_f16x2(hi);
        f[x][3] = e4m3x2_f16x2(hi >> 16);
      }
    };
    const float scale0 = un[0].w > 0.0f ? un[0].y : INFINITY, scale1 = un[1].w > 0.0f ? un[1].y : INFINITY;
    if (scale0 < INFINITY) top_scale = fmaxf(top_scale, scale0);
    if (scale1 < INFINITY) top_scale = fmaxf(top_scale, scale1);
    if (__builtin_expect(fminf(scale0, scale1) >= top_scale - kFar, 1)) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float m0 = (run[n][0] == -INFINITY ? 0.0f : run[n][0]) - kWeightTop, m1 = (run[n][1] == -INFINITY ? 0.0f : run[n][1]) - kWeightTop;
#pragma unroll
        for (int u = 0; u < 2; ++u) weights(u, n, m0, m1, un[u].z, un[u].z);
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int i = 0; i < CH; i += 2) {
          uint32_t f[2][4];
          values(u, i, f);
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_f16(acc[n][i + x], f[x], w[u][n][0], w[u][n][1]);
        }
      }
    } else {
      // a scale far below another: every unit's and row's largest weight moves to 2^10, and the product back by as much
      float back[2][NT][2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float m[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float t = fmaxf(sc[u][n][e], sc[u][n][e + 2]);
            t = fmaxf(t, __shfl_xor_sync(0xFFFFFFFFu, t, 4));
            t = fmaxf(t, __shfl_xor_sync(0xFFFFFFFFu, t, 8));
            t = fmaxf(t, __shfl_xor_sync(0xFFFFFFFFu, t, 16));
            const float lift = t == -INFINITY ? 0.0f : fminf(floorf(run[n][e] - t), 120.0f);
            m[e] = (run[n][e] == -INFINITY ? 0.0f : run[n][e]) - kWeightTop - lift;
            back[u][n][e] = ex2_approx_ftz(-lift);
          }
          weights(u, n, m[0], m[1], un[u].z * back[u][n][0], un[u].z * back[u][n][1]);
        }
      }
#pragma unroll 1
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int i = 0; i < CH; i += 2) {
          uint32_t f[2][4];
          values(u, i, f);
#pragma unroll
          for (int x = 0; x < 2; ++x) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              float t[4] = {0.0f, 0.0f, 0.0f, 0.0f};
              mma_f16(t, f[x], u ? w[1][n][0] : w[0][n][0], u ? w[1][n][1] : w[0][n][1]);
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[n][i + x][e] = fmaf(t[e], u ? back[1][n][e & 1] : back[0][n][e & 1], acc[n][i + x][e]);
            }
          }
        }
      }
    }
    __syncwarp();
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
        *reinterpret_cast<float2*>(part + (warp * ROWS + r) * LD + 16 * i + 2 * g) = make_float2(acc[n][i][e], acc[n][i][e + 2]);
    }
  }
  __syncthreads();
  const int ticket = b * a.H * a.row_tiles + y;
  T* out = reinterpret_cast<T*>(a.out) + b * a.o_b;
  auto out_row = [&](int r) {
    const int t = (row0 + r) / a.G, hq = h * a.G + (row0 + r) - t * a.G;
    return out + t * a.o_t + hq * a.o_h;
  };
  // four elements of a row a thread
#pragma unroll 1
  for (int i = threadIdx.x; i < rows * (D / 4); i += 32 * kWarps) {
    const int r = i / (D / 4), d = (i - r * (D / 4)) * 4;
    float m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m = fmaxf(m, m_of[w][r]);
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = m_of[w][r] == -INFINITY ? 1.0f : ex2_approx_ftz(m_of[w][r] - m);
      const float4 x = *reinterpret_cast<const float4*>(part + (w * ROWS + r) * LD + d);
      l = fmaf(f, l_of[w][r], l);
      o.x = fmaf(f, x.x, o.x);
      o.y = fmaf(f, x.y, o.y);
      o.z = fmaf(f, x.z, o.z);
      o.w = fmaf(f, x.w, o.w);
    }
    const int lim = limits[r];
    const float nan = __uint_as_float(0x7FC00000u);
    if (first_nan[d] < lim) o.x = nan;
    if (first_nan[d + 1] < lim) o.y = nan;
    if (first_nan[d + 2] < lim) o.z = nan;
    if (first_nan[d + 3] < lim) o.w = nan;
    if (chunks == 1) {
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      put4(out_row(r) + d, o.x * inv, o.y * inv, o.z * inv, o.w * inv, vec);
    } else {
      const int64_t at = ((int64_t)ticket * a.splits + split) * ROWS + r;
      *reinterpret_cast<float4*>(a.partial + at * D + d) = o;
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
  // every row's share of each chunk first, then the sums, four elements a thread and several chunks in flight
  const float2* ml = reinterpret_cast<const float2*>(a.partial + a.partial_ml) + (int64_t)ticket * a.splits * ROWS;
  const float* po = a.partial + (int64_t)ticket * a.splits * ROWS * D;
  float* share = part;  // [chunk][row]
  if (threadIdx.x < 8 * ROWS) {  // eight lanes a row
    const int r = threadIdx.x >> 3, at = threadIdx.x & 7;
    float m = -INFINITY, l = 0.0f;
#pragma unroll 4
    for (int s = at; s < chunks; s += 8) m = fmaxf(m, __ldcg(ml + s * ROWS + r).x);
#pragma unroll
    for (int d = 1; d < 8; d <<= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, d));
#pragma unroll 4
    for (int s = at; s < chunks; s += 8) {
      const float2 x = __ldcg(ml + s * ROWS + r);
      const float f = x.x == -INFINITY ? 1.0f : ex2_approx_ftz(x.x - m);
      share[s * ROWS + r] = f;
      l = fmaf(f, x.y, l);
    }
#pragma unroll
    for (int d = 1; d < 8; d <<= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, d);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    for (int s = at; s < chunks; s += 8) share[s * ROWS + r] *= inv;
  }
  __syncthreads();
#pragma unroll 1
  for (int i = threadIdx.x; i < rows * (D / 4); i += 32 * kWarps) {
    const int r = i / (D / 4), d = (i - r * (D / 4)) * 4;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
    for (int s0 = 0; s0 < chunks; s0 += 8) {
      float4 u[8];
#pragma unroll
      for (int z = 0; z < 8; ++z)
        if (s0 + z < chunks) u[z] = __ldcg(reinterpret_cast<const float4*>(po + ((int64_t)(s0 + z) * ROWS + r) * D + d));
#pragma unroll
      for (int z = 0; z < 8; ++z) {
        if (s0 + z < chunks) {
          const float f = share[(s0 + z) * ROWS + r];
          o.x = fmaf(f, u[z].x, o.x);
          o.y = fmaf(f, u[z].y, o.y);
          o.z = fmaf(f, u[z].z, o.z);
          o.w = fmaf(f, u[z].w, o.w);
        }
      }
    }
    put4(out_row(r) + d, o.x, o.y, o.z, o.w, vec);
  }
}

template <int D, int NT, typename T, bool CAP>
int launch_rows(const AttendArgs& a, int vec, cudaStream_t s) {
  constexpr int ring = kWarps * kStages * 2 * kTile * D, meet = kWarps * 8 * NT * (D + 8) * 4;
  constexpr int smem = ring > meet ? ring : meet;
  static bool attr_set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return IFLB200_ERR_DEVICE;
  if (!attr_set[dev]) {
    const cudaError_t e =
        cudaFuncSetAttribute(cache_attend_rows_kernel<D, NT, T, CAP>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return (int)e;
    attr_set[dev] = true;
  }
  const dim3 grid((unsigned)a.splits, (unsigned)(a.H * a.row_tiles), (unsigned)a.B);
  const cudaError_t e = launch_dep(cache_attend_rows_kernel<D, NT, T, CAP>, grid, dim3(32 * kWarps), smem, s, 1,
                                   dependent_launch_for((int64_t)a.B * a.T), a, vec);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

template <int D, int NT, typename T>
int launch_rows(const AttendArgs& a, cudaStream_t s) {
  const uintptr_t bits = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.out) |
                         (uintptr_t)((a.q_b | a.q_t | a.q_h | a.o_b | a.o_t | a.o_h) * (int64_t)sizeof(T));
  const int vec = bits % 8 == 0;
  return a.cap > 0.0f ? launch_rows<D, NT, T, true>(a, vec, s) : launch_rows<D, NT, T, false>(a, vec, s);
}

// iflb200_cache_attention_set_form; 0: by rule
int g_form = 0;

// Few rows take 16 rows (8 of 256 elements) at a time and are faster up to 64 rows of one head (32): row tiles cost the same
// up to 256 (128) rows.  Few rows / tiles, 4 sequences of 16384 keys, 8 heads of 128: 63 / 118 us with 32 rows, 108 / 118 with
// 64, 150 / 118 with 96; 16 of 4096, two heads of 256: 35 / 62 with 16, 66 / 64 with 32, 80 / 64 with 40.
template <typename T>
int attend(AttendArgs a, int D, void* workspace, int64_t bytes, cudaStream_t s) {
  const int64_t rows = (int64_t)a.T * a.G;
  const bool many = g_form == 2 || (g_form == 0 && rows > (D == 256 ? 32 : 64));
  const int nt = D == 256 || rows <= 8 ? 1 : 2, per = many ? attend_tiles_rows(D) : 8 * nt;
  const int64_t tiles = (rows + per - 1) / per;
  if (tiles * a.H > 65535) return IFLB200_ERR_SHAPE;
  a.row_tiles = (int)tiles;
  const int sms = device_sm_count();
  if (sms == 0) return IFLB200_ERR_DEVICE;
  // Ranges of keys, of whole steps of all warps, as many as the workspace takes and no more than fill the GPU once (few rows:
  // as many CTAs an SM as share its issue slots without loss), where that is two or more.  Where it is not, sequences of
  // different lengths are evened out: few rows over eight CTAs an SM, row tiles over two ranges while there are fewer than SMs.
  //   16384 keys, 8 heads of 256, 8 rows, two sequences: 84.6 us with 74 ranges, 43.0 with 9, 86.0 with 2
  //   32 sequences of 2048 to 8192 keys, 8 heads of 128, 4 rows: 67 us with five, 76 with three
  //   the same of 1 to 8192 keys: 65 us with five, 59.4 with three, 77.8 unshared
  //   row tiles, 16384 keys, 8 heads of 128, one sequence: 58.0 us with 19 (152 CTAs), 44.1 with 16
  const int64_t keys = (int64_t)a.max_pages * a.P, units = (int64_t)a.B * a.H * tiles;
  constexpr int64_t kLeast = kWarps * kTile;
  const int64_t fill = (many ? 1 : (D == 64 ? 3 : (D == 128 ? 2 : 1))) * (int64_t)sms / units;
  const int64_t even = many ? (units < sms ? 2 : 1) : (8ll * sms + units - 1) / units;
  const int64_t want = fill >= 2 ? fill : even;
  // The tickets have a place of their own whatever the geometry: they are zero between calls, partial results are not.
  // (Sequences are only shared where there are fewer units than CTAs wanted.)
  constexpr int64_t head = 4096;
  const int64_t each = units * per * (D + 2) * 4;
  const int64_t room = workspace && bytes > head ? (bytes - head) / each : 0;
  int64_t splits = units * 4 > head ? 1 : (want < room ? want : room);
  if (splits > 512) splits = 512;  // (shares of the chunks are worked out in shared memory)
  if (splits < 1) splits = 1;
  const int64_t steps = (keys + kLeast - 1) / kLeast;
  int64_t per_range = (steps + splits - 1) / splits;
  if (per_range < 1) per_range = 1;
  // The last CTA of few rows reads every range's result: five ranges cost about a step (16384 keys of one head of 256: 47 us
  // with 128 ranges, 25.4 with 16 or 24, 51 with 4).
  for (int64_t n = per_range + 1, best = 5 * per_range + (steps + per_range - 1) / per_range; !many && 5 * n < best; ++n) {
    const int64_t cost = 5 * n + (steps + n - 1) / n;
    if (cost < best) best = cost, per_range = n;
  }
  int64_t chunk = per_range * kLeast;
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
  // (a cap needs a reciprocal, and infinity times tanh(0) is none)
  if (!(softcap == 0.0f || (softcap >= FLT_MIN && softcap <= FLT_MAX)) || !(fabsf(scale) <= FLT_MAX) || (prefix && !causal)) return IFLB200_ERR_ARG;
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
