// Products of few token rows with weights that stream through the chip, and
// their launch rules: bf16 and fp32 (proj.hip) and int8 codes (int8.hip).
#pragma once

#include "front.h"

#include <climits>
#include <type_traits>

namespace coda {

// dword 3 of a raw buffer resource on gfx9 (32-bit data format, no swizzle)
static constexpr int kProjBufWord3 = 0x00020000;

// Few token rows (M <= 128): the weights are the traffic.  A workgroup owns
// 16 RB features over all of K: its 8 waves split K and stream their weight
// rows and the token rows of that range straight from memory into MFMA
// fragments, one 16 x 16 accumulator per 16 features and 16 tokens; the
// partials meet in LDS and are summed in wave order (deterministic), then
// the epilogue.  No workspace, no cross-workgroup exchange.  Weights cross
// HBM once; the token rows are read by every workgroup from L2.
// K goes in pairs of 64-byte steps: a lane's two 16-byte pieces of a row
// come from the two halves of one 128-byte line, requested back to back.
// Measured (bf16, tiles, weights not in cache): 6177 x 4096 M = 1 12.2 us, M
// = 16 13.3 us (4.1 / 3.8 TB/s), 10305 x 8192 M = 1 31.3 us (5.4 TB/s).
// The weights: in fragment tiles (TileRows; coda_project_pack), where the
// operand of row block fb at k-step ks is the KiB at (fb D/32 + ks) 512
// elements (bf16), lane l's 16 bytes at 16 l; or rows as they lie (MatRows:
// one matrix; ParamRows: the layer's own parameters), at any element address.
// A load of tiles is a KiB in one piece, one of rows 16 pieces of 64 bytes:
// 6177 x 4096 M = 1 13.3 us (tiles 12.2), M = 64 22.3 (18.2), 10305 x 8192 M =
// 128 63.3 (53.7), 4096 x 4096 M = 1 8.7 (7.9; the library 14.9).
template <typename T>
struct TileRows {
  static constexpr bool kTiles = true;
  const T* w;
};
template <typename T>
struct MatRows {
  const T* w;
  int64_t sm;
  __device__ __forceinline__ const T* row16(int f0, int r16, int last) const { return w + min(f0 + r16, last) * sm; }
};
template <typename Src>
struct IsTiles : std::false_type {};
template <typename T>
struct IsTiles<TileRows<T>> : std::true_type {};
// a row's 16 bytes at any element address
typedef uint32_t pu32x4u __attribute__((ext_vector_type(4), aligned(2)));
// accumulators: fp32, of int8 codes int32 (exact)
typedef int32_t pi32x4 __attribute__((ext_vector_type(4)));
template <typename T>
using RowsAcc = typename std::conditional<sizeof(T) == 1, pi32x4, pf32x4>::type;
template <typename T>
__device__ __forceinline__ RowsAcc<T> rows_mfma(const pu32x4& a, const pu32x4& b, RowsAcc<T> c) {
  if constexpr (sizeof(T) == 1) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(pi32x4, a), __builtin_bit_cast(pi32x4, b), c, 0, 0, 0);
  } else if constexpr (sizeof(T) == 2) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pbf16x8_t, a), __builtin_bit_cast(pbf16x8_t, b),
                                                   c, 0, 0, 0);
  } else {
    const pf32x4 x = __builtin_bit_cast(pf32x4, a), y = __builtin_bit_cast(pf32x4, b);
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], c, 0, 0, 0);
    return c;
  }
}
// waves whose partials meet in LDS at once: all 8, or 4 after the upper 4
// have handed theirs to the lower 4
template <int MT, int RB>
struct RowsLds {
  static constexpr int kWaves = RB * MT <= 8 ? 8 : 4;
  static constexpr size_t kBytes = (size_t)kWaves * RB * MT * 64 * sizeof(pf32x4);
};
// One dword of each 64 bytes of the epilogue's arguments, read before the
// products: the compiler loads them where they are used, after the products,
// in several dependent rounds, each a miss of the scalar cache then
template <typename V>
__device__ __forceinline__ void touch_args(const V& v) {
  const int* p = reinterpret_cast<const int*>(&v);
#pragma unroll
  for (int i = 0; i < (int)(sizeof(V) / 4); i += 16) asm volatile("" ::"s"(p[i]));
}
// The waves' partials (accumulators of 16 features x 16 tokens each), summed in
// wave order, and the epilogue
template <int MT, int RB, typename Acc, typename Src, typename Epi>
__device__ __forceinline__ void rows_finish(Acc (&acc)[RB][MT], char* smem, int n_feat, int M, const Src& W,
                                            const Epi& epi) {
  Acc* part = reinterpret_cast<Acc*>(smem);
  const int t = threadIdx.x, lane = t & 63, wv = __builtin_amdgcn_readfirstlane(t >> 6), f0 = blockIdx.x * 16 * RB;
  constexpr int NWv = RowsLds<MT, RB>::kWaves;
  if constexpr (NWv == 4) {
    if (wv >= 4)
#pragma unroll
      for (int i = 0; i < RB; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) part[(((wv - 4) * RB + i) * MT + j) * 64 + lane] = acc[i][j];
    __syncthreads();
    if (wv < 4)
#pragma unroll
      for (int i = 0; i < RB; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[i][j] += part[((wv * RB + i) * MT + j) * 64 + lane];
    __syncthreads();
  }
  if (wv < NWv)
#pragma unroll
    for (int i = 0; i < RB; ++i)
#pragma unroll
      for (int j = 0; j < MT; ++j) part[((wv * RB + i) * MT + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  if (blockIdx.x == 0) epi.once(t);
  // item 64 (MT i + j) + l: features f0 + 16 i + 4 (l / 16) .. + 3 of token
  // 16 j + l % 16
  for (int item = t; item < 64 * MT * RB; item += 512) {
    const int ij = item >> 6, l = item & 63;
    Acc sum = part[ij * 64 + l];
#pragma unroll
    for (int w = 1; w < NWv; ++w) sum += part[(w * RB * MT + ij) * 64 + l];
    const int m = 16 * (ij % MT) + (l & 15), f = f0 + 16 * (ij / MT) + 4 * (l >> 4);
    if (m < M && f < n_feat) epi(W, f, m, sum);
  }
}

template <typename T, int MT, int RB, typename Src, typename Epi>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2))) void proj_rows(
    const Src W, int n_feat, int D, const T* __restrict__ X, int64_t x_sm, int M, const Epi epi) {
  constexpr bool TILED = IsTiles<Src>::value;
  extern __shared__ __attribute__((aligned(16))) char rows_smem[];
  // pairs of k-steps in flight ahead of the products
  constexpr int LP = RB * MT <= 3 ? 4 : RB * MT <= 12 ? 2 : 1;
  const int f0 = blockIdx.x * 16 * RB;
  const int t = threadIdx.x, lane = t & 63, wv = __builtin_amdgcn_readfirstlane(t >> 6), r16 = lane & 15, kq = lane >> 4;
  const int pairs = D * (int)sizeof(T) / 128, p0 = pairs * wv / 8, np = pairs * (wv + 1) / 8 - p0;
  // byte addresses of this lane's first piece of pair 0; WP / WH: bytes from
  // a pair to the next, from its first half to its second
  constexpr int WP = TILED ? 2048 : 128, WH = TILED ? 1024 : 64;
  const char* wr[RB];
#pragma unroll
  for (int i = 0; i < RB; ++i)
    if constexpr (TILED)
      wr[i] = (const char*)W.w + ((int64_t)min(f0 / 16 + i, (n_feat + 15) / 16 - 1) * pairs + p0) * 2048 + 16 * lane;
    else
      wr[i] = (const char*)W.row16(f0 + 16 * i, r16, n_feat - 1) + 128 * p0 + 16 * kq;
  const char* xr[MT];
#pragma unroll
  for (int j = 0; j < MT; ++j) xr[j] = (const char*)(X + (int64_t)min(16 * j + r16, M - 1) * x_sm) + 128 * p0 + 16 * kq;
  pu32x4 a[LP][RB][2], b[LP][MT][2];
  auto load = [&](int u, int p) {
#pragma unroll
    for (int i = 0; i < RB; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        a[u][i][h] = *reinterpret_cast<const typename std::conditional<TILED, pu32x4, pu32x4u>::type*>(wr[i] + WP * p + WH * h);
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) b[u][j][h] = *reinterpret_cast<const pu32x4*>(xr[j] + 128 * p + 64 * h);
  };
  RowsAcc<T> acc[RB][MT];
#pragma unroll
  for (int i = 0; i < RB; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = RowsAcc<T>{0, 0, 0, 0};
#pragma unroll
  for (int u = 0; u < LP; ++u)
    if (u < np) load(u, u);
  touch_args(epi);
  auto products = [&](const pu32x4 (&as)[RB][2], const pu32x4 (&bs)[MT][2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < RB; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[i][j] = rows_mfma<T>(as[i][h], bs[j][h], acc[i][j]);
  };
  int p = 0;
  for (; p + 2 * LP <= np; p += LP) {
#pragma unroll
    for (int u = 0; u < LP; ++u) {
      products(a[u], b[u]);
      load(u, p + u + LP);
    }
  }
#pragma unroll
  for (int u = 0; u < 2 * LP; ++u) {
    if (p + u >= np) break;
    products(a[u % LP], b[u % LP]);
    if (p + u + LP < np) load(u % LP, p + u + LP);
  }
  rows_finish<MT, RB>(acc, rows_smem, n_feat, M, W, epi);
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const char* p, int nbytes) {
  const uint64_t v = (uint64_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
  return __builtin_amdgcn_make_buffer_rsrc((void*)(((uint64_t)hi << 32) | lo), (short)0,
                                           __builtin_amdgcn_readfirstlane(nbytes), kProjBufWord3);
}
// The same for 17 .. 128 rows and K in whole chunks (8 waves x CS steps of 64
// bytes): the token rows pass through LDS.  Operand loads straight from
// memory take 16 rows' 64-byte pieces at a power-of-two stride, a quarter of
// the rate of contiguous ones, and with 64 rows they outweigh the weights
// (6184 x 4096, M = 64: 23.7 us with them, 18.8 us here; 10305 x 8192, M =
// 128: 83 against 52.7 us; 4096 x 4096, M = 32: 12.1 against 11.1 us).  Per chunk and 16
// tokens a wave loads its own part of the rows as CS * 64 contiguous bytes a
// row into registers (two such slabs in flight), writes it to its LDS slab
// and reads the operands back; 16-byte pieces are swizzled by the row, so
// writes and reads spread over the banks.  The slab is the wave's alone and
// LDS serves a wave in order: no barrier.  The next chunk's weights load
// while this chunk's products run.  Same sums in the same order as proj_rows.
template <typename T, int MT, int RB, int CS, typename Src, typename Epi>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2))) void proj_rows_lds(
    const Src W, int n_feat, int D, const T* __restrict__ X, int64_t x_sm, int M, const Epi epi) {
  constexpr bool TILED = IsTiles<Src>::value;
  extern __shared__ __attribute__((aligned(16))) char rows_smem[];
  constexpr int RBY = CS * 64, PCS = RBY / 16, NI = 16 * PCS / 64, RPI = 64 / PCS;  // row bytes, pieces; loads a slab, rows a load
  const int f0 = blockIdx.x * 16 * RB;
  const int t = threadIdx.x, lane = t & 63, wv = __builtin_amdgcn_readfirstlane(t >> 6), r16 = lane & 15, kq = lane >> 4;
  const int steps = D * (int)sizeof(T) / 64, nc = steps / (8 * CS), s0 = nc * CS * wv;
  char* slab = rows_smem + wv * 16 * RBY;
  // tiles and token rows through raw buffer resources: 32-bit offsets, and
  // token rows past the last read 0 without touching memory
  const int nfb = (n_feat + 15) / 16;
  const __amdgpu_buffer_rsrc_t rx = rows_rsrc((const char*)X, (int)(((M - 1) * x_sm + D) * (int)sizeof(T)));
  __amdgpu_buffer_rsrc_t rw;
  int wo[RB];
  const char* wr[RB];
  if constexpr (TILED) {
    rw = rows_rsrc((const char*)W.w + (int64_t)(f0 / 16) * steps * 1024, RB * steps * 1024);
#pragma unroll
    for (int i = 0; i < RB; ++i) wo[i] = (min(f0 / 16 + i, nfb - 1) - f0 / 16) * steps * 1024 + s0 * 1024;
  } else {
#pragma unroll
    for (int i = 0; i < RB; ++i)
      wr[i] = (const char*)W.row16(f0 + 16 * i, r16, n_feat - 1) + 64 * s0 + 16 * kq;
  }
  const int lr = lane / PCS, lp = lane % PCS, xrow = (int)x_sm * (int)sizeof(T);
  const int xo = 64 * s0 + 16 * lp + lr * xrow;
  pu32x4 a0[CS][RB], a1[CS][RB], x0[NI], x1[NI];
  auto load_w = [&](pu32x4 (&w)[CS][RB], int c) {
#pragma unroll
    for (int s = 0; s < CS; ++s)
#pragma unroll
      for (int i = 0; i < RB; ++i) {
        if constexpr (TILED) w[s][i] = __builtin_amdgcn_raw_buffer_load_b128(rw, 16 * lane, wo[i] + (c * CS + s) * 1024, 0);
        else w[s][i] = *reinterpret_cast<const pu32x4u*>(wr[i] + c * RBY + 64 * s);
      }
  };
  // slab (chunk c, tokens 16 j ..)
  auto load_x = [&](pu32x4 (&v)[NI], int c, int j) {
    const int cb = xo + c * RBY;
#pragma unroll
    for (int i = 0; i < NI; ++i) v[i] = __builtin_amdgcn_raw_buffer_load_b128(rx, cb + (16 * j + RPI * i) * xrow, 0, 0);
  };
  RowsAcc<T> acc[RB][MT];
#pragma unroll
  for (int i = 0; i < RB; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = RowsAcc<T>{0, 0, 0, 0};
  auto tokens = [&](int c, int j, pu32x4 (&v)[NI], const pu32x4 (&w)[CS][RB], RowsAcc<T> (&ac)[RB][MT]) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int row = RPI * i + lr;
      *reinterpret_cast<pu32x4*>(slab + row * RBY + ((lp ^ row) & (PCS - 1)) * 16) = v[i];
    }
    // slab j + 2 of the walk over (chunk, tokens); past the end: the last again
    load_x(v, j + 2 < MT ? c : min(c + 1, nc - 1), (j + 2) % MT);
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int s = 0; s < CS; ++s) {
      const pu32x4 b = *reinterpret_cast<const pu32x4*>(slab + r16 * RBY + (((4 * s + kq) ^ r16) & (PCS - 1)) * 16);
#pragma unroll
      for (int i = 0; i < RB; ++i) ac[i][j] = rows_mfma<T>(w[s][i], b, ac[i][j]);
    }
    __builtin_amdgcn_wave_barrier();
  };
  auto chunk = [&](int c, pu32x4 (&w)[CS][RB], pu32x4 (&wn)[CS][RB]) {
    load_w(wn, min(c + 1, nc - 1));
#pragma unroll
    for (int j = 0; j < MT; j += 2) {
      tokens(c, j, x0, w, acc);
      tokens(c, j + 1, x1, w, acc);
    }
  };
  static_assert(MT % 2 == 0, "slabs alternate between two register sets");
  load_w(a0, 0);
  load_x(x0, 0, 0);
  load_x(x1, 0, 1);
  touch_args(epi);
  int c = 0;
  for (; c + 1 < nc; c += 2) {
    chunk(c, a0, a1);
    chunk(c + 1, a1, a0);
  }
  if (c < nc) chunk(c, a0, a1);
  __syncthreads();
  rows_finish<MT, RB>(acc, rows_smem, n_feat, M, W, epi);
}

template <typename T, int MT, int RB, typename Src, typename Epi>
static int launch_rows_k(const Src& W, int n_feat, int D, const T* X, int64_t x_sm, int M, const Epi& epi,
                         hipStream_t st, const char* who) {
  constexpr size_t lds = RowsLds<MT, RB>::kBytes;
  const int rc = lds_limit<proj_rows<T, MT, RB, Src, Epi>>(lds, who);
  if (rc) return rc;
  hipLaunchKernelGGL((proj_rows<T, MT, RB, Src, Epi>), dim3((n_feat + 16 * RB - 1) / (16 * RB)), dim3(512), lds, st, W,
                     n_feat, D, X, x_sm, M, epi);
  return check_launch("proj_rows");
}
// Features a workgroup: the RB (1 .. 3) of the fewest 16-feature turns, ceil
// (workgroups / CUs) * RB, and of these the largest (it reads the token rows
// least often)
static int rows_rb(int n_feat) {
  const int cus = device_cus(), fb = (n_feat + 15) / 16;
  int best = 1, turns = INT_MAX;
  for (int rb = 1; rb <= 3; ++rb) {
    const int n = ((fb + rb - 1) / rb + cus - 1) / cus * rb;
    if (n <= turns) {
      turns = n;
      best = rb;
    }
  }
  return best;
}
template <typename T, int MT, int RB, typename Src, typename Epi>
static int launch_rows_lds(const Src& W, int n_feat, int D, const T* X, int64_t x_sm, int M, const Epi& epi,
                           hipStream_t st, const char* who) {
  // steps a chunk: as many as the accumulators (and the row addresses of
  // weights that are not tiles) leave registers for
  constexpr int CS = RB * MT <= (IsTiles<Src>::value ? 4 : 3) || RB == 1 && MT == 4 ? 8 : RB * MT <= 16 ? 4 : 2;
  constexpr size_t slabs = (size_t)8 * 16 * CS * 64;
  constexpr size_t lds = slabs > RowsLds<MT, RB>::kBytes ? slabs : RowsLds<MT, RB>::kBytes;
  const int rc = lds_limit<proj_rows_lds<T, MT, RB, CS, Src, Epi>>(lds, who);
  if (rc) return rc;
  hipLaunchKernelGGL((proj_rows_lds<T, MT, RB, CS, Src, Epi>), dim3((n_feat + 16 * RB - 1) / (16 * RB)), dim3(512), lds,
                     st, W, n_feat, D, X, x_sm, M, epi);
  return check_launch("proj_rows_lds");
}
template <typename T, int MT, typename Src, typename Epi>
static int launch_rows_mt(const Src& W, int n_feat, int D, const T* X, int64_t x_sm, int M, const Epi& epi,
                          hipStream_t st, const char* who) {
  if constexpr (MT > 1) {
    // (token rows within a 31-bit offset)
    if (D * sizeof(T) % 4096 == 0 && x_sm >= 0 && (M * x_sm + D) * (int64_t)sizeof(T) < INT_MAX) {
      switch (rows_rb(n_feat)) {
        case 1: return launch_rows_lds<T, MT, 1>(W, n_feat, D, X, x_sm, M, epi, st, who);
        case 2: return launch_rows_lds<T, MT, 2>(W, n_feat, D, X, x_sm, M, epi, st, who);
        default: return launch_rows_lds<T, MT, 3>(W, n_feat, D, X, x_sm, M, epi, st, who);
      }
    }
  }
  switch (rows_rb(n_feat)) {
    case 1: return launch_rows_k<T, MT, 1>(W, n_feat, D, X, x_sm, M, epi, st, who);
    case 2: return launch_rows_k<T, MT, 2>(W, n_feat, D, X, x_sm, M, epi, st, who);
    default: return launch_rows_k<T, MT, 3>(W, n_feat, D, X, x_sm, M, epi, st, who);
  }
}
template <typename T, typename Src, typename Epi>
static int launch_rows(const Src& W, int n_feat, int D, const T* X, int64_t x_sm, int M, const Epi& epi,
                       hipStream_t st, const char* who) {
  if (M <= 16) return launch_rows_mt<T, 1>(W, n_feat, D, X, x_sm, M, epi, st, who);
  if (M <= 32) return launch_rows_mt<T, 2>(W, n_feat, D, X, x_sm, M, epi, st, who);
  if (M <= 64) return launch_rows_mt<T, 4>(W, n_feat, D, X, x_sm, M, epi, st, who);
  return launch_rows_mt<T, 8>(W, n_feat, D, X, x_sm, M, epi, st, who);
}

}  // namespace coda
