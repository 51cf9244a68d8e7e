// Rows in 8 bits on gfx950: their making (with or without a norm), and the
// product of two sets of them.
//
// A set of rows is int8 codes in [-127, 127] with one fp32 scale a row, the
// value of a code being code * scale.  A row's codes lie at a 16-byte address
// and are followed by zeros up to a multiple of kPad bytes, so that the
// product runs over whole 128-byte steps and has no ragged end.
#include "rows.h"

#include <algorithm>
#include <climits>
#include <utility>

namespace coda {

static constexpr int kPad = 128;
// the longest sum of products of int8 that int32 holds: 128 * 128 * K < 2^31
static constexpr int kMaxK = (1 << 17) - kPad;
// the largest row stride: a tile's rows lie within 32-bit offsets of its first
static constexpr int64_t kMaxStride = 1 << 24;
// elements of the longest row that the making of codes keeps in registers
static constexpr int kMaxRow = 32768;
// rows of a launch of a row a workgroup (a grid has less than 2^32 threads)
static constexpr int64_t kLaunchRows = 1 << 21;
// rows of a product's operand (their numbers, up to a whole tile, are 32 bits)
static constexpr int kMaxRows = 1 << 30;

// ------------------------------------------------------------ making codes
__device__ __forceinline__ double wave_reduce(double v, bool max) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const double o = __shfl_xor(v, d);
    v = max ? fmax(v, o) : v + o;
  }
  return v;
}

// a run of 8 elements, at any element address
template <typename T>
struct Run8 {
  T v[8];
};
template <typename T>
__device__ __forceinline__ Run8<T> run_ld(const T* p, int n) {  // elements past n: 0
  Run8<T> r;
  if (n >= 8) {
    constexpr int N = sizeof(Run8<T>) / 16;
    pu32x4 w[N];
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = reinterpret_cast<const pu32x4u*>(p)[i];
    __builtin_memcpy(&r, w, sizeof(r));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) r.v[e] = e < n ? p[e] : Elt<T>::st(0.f);
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void run_st(T* p, int n, const Run8<T>& r) {
  if (n >= 8) {
    constexpr int N = sizeof(Run8<T>) / 16;
    pu32x4 w[N];
    __builtin_memcpy(w, &r, sizeof(r));
#pragma unroll
    for (int i = 0; i < N; ++i) reinterpret_cast<pu32x4u*>(p)[i] = w[i];
  } else {
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (e < n) p[e] = r.v[e];
  }
}

// Codes of a row whose largest magnitude is P: code(p) = rint(127 p / P), the
// quotient to the last bit: n = 127 p, times the reciprocal, then its
// remainder's share.  In fp32 P is brought to [1, 2) (p by the same power of
// two), where neither leaves the range.
template <typename R>
struct Coder {
  // leaves a quotient's nearest integer (ties to even) in its low bits: 1.5
  // times 2^23 or 2^52
  static constexpr R kShift = sizeof(R) == 4 ? (R)12582912. : (R)6755399441055744.;
  R k, Q, inv;
  __device__ __forceinline__ Coder(double P, bool fine) : k(127), Q((R)P), inv(0) {
    if (!fine) return;
    if constexpr (sizeof(R) == 4) {
      int ex;
      Q = (float)(2. * frexp(P, &ex));
      k = (float)ldexp(127., min(1 - ex, 119));
      Q = (float)ldexp((double)Q, min(1 - ex, 119) - (1 - ex));
    }
    inv = (R)1 / Q;
  }
  __device__ __forceinline__ uint32_t operator()(R p) const {  // in the low byte
    const R n = p * k, q0 = n * inv;
    const R q = __builtin_elementwise_fma(__builtin_elementwise_fma(-q0, Q, n), inv, q0) + kShift;
    if constexpr (sizeof(R) == 4) return __builtin_bit_cast(uint32_t, q);
    else return (uint32_t)__builtin_bit_cast(uint64_t, q);
  }
};
// the low bytes of eight
__device__ __forceinline__ uint2 pack8(const uint32_t (&c)[8]) {
  const auto four = [](uint32_t a, uint32_t b, uint32_t d, uint32_t e) {
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(e, d, 0x0c0c0400u), __builtin_amdgcn_perm(b, a, 0x0c0c0400u),
                                 0x05040100u);
  };
  return uint2{four(c[0], c[1], c[2], c[3]), four(c[4], c[5], c[6], c[7])};
}
// the type that p and P of plain rows need
template <typename T>
using PlainR = typename std::conditional<sizeof(T) == 2, float, double>::type;

// Rows in 8 bits, with p_i = x_i (plain) or p_i = s_i w_i (norm; s = x +
// residual, rounded to T and written):
//   P = max |p|, code_i = rint(127 p_i / P),
//   scale = P / 127, with the norm P / (127 sqrt(mean(s^2) + eps)):
// the norm is the same factor for the whole row, so the codes need not wait
// for it.  p, P, the sum and the quotient are held in 64 bits: a product of
// two floats is exact there, and a quotient that falls on a half is rounded
// to even as the formula says, whatever the order of the sums.  (Plain rows
// of 16 bits: p and P need no more than fp32, and the quotient's remainder,
// of at most 18 bits, is exact in it.)  A row that holds an infinity or a
// NaN (its weight's count too) gets scale NaN and codes 0; a row of zeros
// scale 0.
// TPR threads keep a row in registers (IT runs of 8 elements each) between
// the row's maximum and its codes, so that memory is read once.  It is bound
// by memory where rows are many: 16384 x 8192 bf16 with a residual 164-180 us
// (5.2-5.7 TB/s), plain 76 us (5.3); 1 x 4096 with a residual 3.2 us, a
// launch.  A wave for a row of up to 1024 elements needs no barrier; longer
// ones share it, 16 elements a thread (1024 threads: up to 32).
template <typename T, bool NORM, bool RES, int TPR, int IT>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void codes_kernel(
    const T* __restrict__ x, int64_t x_sm, const T* __restrict__ res, int64_t r_sm, const T* __restrict__ w, int rows,
    int D, float eps, T* __restrict__ sum_out, int64_t s_sm, int8_t* __restrict__ codes, int64_t c_sm,
    float* __restrict__ scales) {
  using E = Elt<T>;
  typedef typename std::conditional<NORM, double, PlainR<T>>::type R;
  constexpr int NT = TPR < 256 ? 256 : TPR, RPB = NT / TPR;
  const int t = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
  if (TPR == 64 && row >= rows) return;  // (whole waves; else a workgroup is a row)
  const T* xr = x + row * x_sm;
  R p[IT * 8];
  double ss = 0.;
  R top = 0, bad = 0;
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int at = (i * TPR + t) * 8, n = D - at;
#pragma unroll
    for (int e = 0; e < 8; ++e) p[i * 8 + e] = 0;
    if (n <= 0) continue;
    Run8<T> a = run_ld(xr + at, n);
    if constexpr (NORM) {
      const Run8<T> g = run_ld(w + at, n);
      if constexpr (RES) {
        const Run8<T> r = run_ld(res + row * r_sm + at, n);
#pragma unroll
        for (int e = 0; e < 8; ++e) a.v[e] = E::st(E::ld(a.v[e]) + E::ld(r.v[e]));
        run_st(sum_out + row * s_sm + at, n, a);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const double s = (double)E::ld(a.v[e]);
        ss = fma(s, s, ss);
        p[i * 8 + e] = s * (double)E::ld(g.v[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) p[i * 8 + e] = (R)E::ld(a.v[e]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      top = __builtin_elementwise_max(top, __builtin_elementwise_abs(p[i * 8 + e]));
      bad = __builtin_elementwise_fma(p[i * 8 + e], (R)0, bad);  // NaN from an infinity or a NaN
    }
  }
  ss += bad;
  ss = wave_reduce(ss, false);
  double P = wave_reduce((double)top, true);
  if constexpr (TPR > 64) {
    constexpr int NW = TPR / 64;
    __shared__ double red[2][NW];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    if (lane == 0) {
      red[0][wv] = ss;
      red[1][wv] = P;
    }
    __syncthreads();
    ss = red[0][0];
    P = red[1][0];
#pragma unroll
    for (int i = 1; i < NW; ++i) {
      ss += red[0][i];
      P = fmax(P, red[1][i]);
    }
  }
  const bool fine = ss == ss && P > 0.;
  if (t == 0) {
    double sc = P / 127.;
    if constexpr (NORM) sc /= sqrt(ss / (double)D + (double)eps);
    scales[row] = ss != ss ? __builtin_nanf("") : P > 0. ? (float)sc : 0.f;
  }
  const Coder<R> code(P, fine);
  int8_t* cr = codes + row * c_sm;
  // (the row's tail: zeros up to a whole 128 bytes)
  const int padded = (D + kPad - 1) / kPad * kPad;
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int at = (i * TPR + t) * 8;
    if (at >= padded) continue;
    uint32_t c[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) c[e] = code(p[i * 8 + e]);
    const uint2 v = fine ? pack8(c) : uint2{0u, 0u};
    *reinterpret_cast<uint2*>(cr + at) = v;
  }
}

template <typename T, bool NORM, bool RES, int TPR, int IT>
static int launch_codes(const T* x, int64_t x_sm, const T* res, int64_t r_sm, const T* w, int rows, int D, float eps,
                        T* sum_out, int64_t s_sm, int8_t* codes, int64_t c_sm, float* scales, hipStream_t st) {
  constexpr int NT = TPR < 256 ? 256 : TPR, RPB = NT / TPR;
  for (int64_t r = 0; r < rows; r += kLaunchRows) {
    const int n = (int)std::min(kLaunchRows, rows - r);
    hipLaunchKernelGGL((codes_kernel<T, NORM, RES, TPR, IT>), dim3((n + RPB - 1) / RPB), dim3(NT), 0, st, x + r * x_sm, x_sm,
                       RES ? res + r * r_sm : res, r_sm, w, n, D, eps, RES ? sum_out + r * s_sm : sum_out, s_sm,
                       codes + r * c_sm, c_sm, scales + r);
    const int rc = check_launch("codes_kernel");
    if (rc) return rc;
  }
  return CODA_OK;
}

// threads and runs of a row of D elements (up to a multiple of 128)
template <typename T, bool NORM, bool RES>
static int run_codes(const void* x, int64_t x_sm, const void* res, int64_t r_sm, const void* w, int rows, int D, float eps,
                     void* sum, int64_t s_sm, int8_t* codes, int64_t c_sm, float* scales, hipStream_t st) {
  const int P = (D + kPad - 1) / kPad * kPad;
#define CODES(TPR, IT)                                                                                                   \
  return launch_codes<T, NORM, RES, TPR, IT>((const T*)x, x_sm, (const T*)res, r_sm, (const T*)w, rows, D, eps, (T*)sum, \
                                             s_sm, codes, c_sm, scales, st)
  if (P <= 512) CODES(64, 1);
  if (P <= 1024) CODES(64, 2);
  if (P <= 2048) CODES(256, 1);
  if (P <= 4096) CODES(256, 2);
  if (P <= 8192) CODES(512, 2);
  if (P <= 16384) CODES(1024, 2);
  CODES(1024, 4);
#undef CODES
}

// values of codes: out = code * scale, one rounding to T.  TPR threads a row
// and workgroup, 8 codes each; out rows of any element address.  Bound by
// memory: 16384 x 8192 to bf16 70-74 us (5.4-5.7 TB/s).
template <typename T, int TPR>
__global__ __launch_bounds__(256) void values_kernel(const int8_t* __restrict__ codes, int64_t c_sm,
                                                     const float* __restrict__ scales, int rows, int D,
                                                     T* __restrict__ out, int64_t o_sm) {
  const int64_t row = (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
  const int at = (blockIdx.y * TPR + threadIdx.x % TPR) * 8;
  if (row >= rows || at >= D) return;
  int8_t c[8];
  const uint2 raw = *reinterpret_cast<const uint2*>(codes + row * c_sm + at);
  __builtin_memcpy(c, &raw, 8);
  const float sc = scales[row];
  T* o = out + row * o_sm + at;
  Run8<T> v;
#pragma unroll
  for (int e = 0; e < 8; ++e) v.v[e] = Elt<T>::st((float)c[e] * sc);
  run_st(o, D - at, v);
}
template <typename T>
static int run_values(const int8_t* codes, int64_t c_sm, const float* scales, int rows, int D, void* out, int64_t o_sm,
                      hipStream_t st) {
  // (a row of up to 512 elements leaves most of 256 threads idle)
  for (int64_t r = 0; r < rows; r += kLaunchRows) {
    const int n = (int)std::min(kLaunchRows, rows - r);
    const int8_t* c = codes + r * c_sm;
    T* o = (T*)out + r * o_sm;
    if (D <= 512)
      hipLaunchKernelGGL((values_kernel<T, 64>), dim3((n + 3) / 4), dim3(256), 0, st, c, c_sm, scales + r, n, D, o, o_sm);
    else
      hipLaunchKernelGGL((values_kernel<T, 256>), dim3(n, (D + 2047) / 2048), dim3(256), 0, st, c, c_sm, scales + r, n, D, o,
                         o_sm);
    const int rc = check_launch("values_kernel");
    if (rc) return rc;
  }
  return CODA_OK;
}

// ------------------------------------------------------------ product
//   y[m, f] = round_T((sum_k x[m, k] w[f, k]) sx[m] sw[f] + bias[f])
// with the sum exact in int32 (so that neither the tile nor a split of K
// shows in the result).  MFMA rows (operand A) are the features, columns (B)
// the tokens: a lane holds four consecutive features of a token.
typedef pi32x4 i32x4;
typedef int32_t i32x16 __attribute__((ext_vector_type(16)));

struct Int8Mat {
  const int8_t* p;
  int64_t sm;  // bytes
  const float* scales;
  int rows;
};

// N features of a token, rounded to T
template <typename T, int N>
struct alignas(N * sizeof(T)) Feats {
  T v[N];
};

// Where the values of a product go: bias1(f) is added to feature f; lane(f) is
// what a lane that writes features f .. f + N - 1 of several tokens needs to
// know once, put() writes them for tokens m, m + step, .. below rows (N = 4,
// or kRun; f a multiple).
template <typename T>
struct LinearSink {
  typedef T Out;
  static constexpr int kRun = 16 / sizeof(T);
  T* out;
  const T* bias;  // or null
  int64_t o_sm;
  int n_feat;
  struct Lane {
    T* p;
    int n;
  };
  __device__ __forceinline__ void once(int) const {}
  __device__ __forceinline__ float bias1(int f) const { return bias ? Elt<T>::ld(bias[f]) : 0.f; }
  __device__ __forceinline__ Lane lane(int f) const { return Lane{out + f, n_feat - f}; }
  template <int N, int R>
  __device__ __forceinline__ void put(const Lane& l, int m, int step, int rows, const Feats<T, N> (&v)[R]) const {
    // (rows of any element address)
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2), aligned(2)));
    typedef typename std::conditional<sizeof(v[0]) == 8, u32x2, pu32x4u>::type V;
    T* row = l.p + (int64_t)m * o_sm;
    const int64_t next = step * o_sm;
    if (l.n >= N) {
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (m + r * step < rows) *reinterpret_cast<V*>(row + r * next) = __builtin_bit_cast(V, v[r]);
    } else {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int e = 0; e < N - 1; ++e)
          if (e < l.n && m + r * step < rows) row[r * next + e] = v[r].v[e];
    }
  }
};

// n / d for n below 2^31 without a division (d's reciprocal of 33 bits, from
// the host)
struct FastDiv {
  uint32_t d, mul, shift;
  explicit FastDiv(int div) : d((uint32_t)div) {
    shift = 0;
    while ((1u << shift) < d) ++shift;
    mul = (uint32_t)(((uint64_t)1 << 32) * (((uint64_t)1 << shift) - d) / d + 1);
  }
  __device__ __forceinline__ uint32_t mod(uint32_t n) const {
    const uint32_t h = __umulhi(mul, n), q = shift ? (h + ((n - h) >> 1)) >> (shift - 1) : n;
    return n - q * d;
  }
};

// The projection front end: the sections and roundings of FrontEpilogue (a
// value is rounded to T before the RoPE or the sigmoid), with all that does
// not change from token to token found once.  TABLES: angles that the launch
// makes itself where tab says so.  N: features of a run: 8 where heads and
// rows allow 16-byte pieces, else 4.
template <typename T, bool TABLES, int N>
struct FrontSink {
  typedef T Out;
  typedef Elt<T> E;
  static constexpr int kRun = N;
  coda_proj_desc d;
  FrontTables tab;
  FastDiv len;  // of a sequence: table row = token % L
  int n_feat;
  // Where a run of features goes: q or v (kind 0), k (1), single lambdas / gates
  // (2); at: of a token 0's first channel (kind 1: of its head), c: that
  // channel (kind 2: the feature)
  struct Lane {
    int kind, c;
    T* at;
    int64_t sm;
  };
  __device__ __forceinline__ float bias1(int f) const { return d.bias[f]; }
  __device__ __forceinline__ Lane lane(int f) const {
    const int Fq = d.H * d.Dh, Fk = d.Hkv * d.Dh;
    if (f < Fq) return Lane{0, 0, (T*)d.q + f, d.q_sm};
    if (f < Fq + Fk) {
      const int c = (f - Fq) % d.Dh;
      return Lane{1, c, (T*)d.k + (f - Fq - c), d.k_sm};
    }
    if (f < Fq + 2 * Fk) return Lane{0, 0, (T*)d.v + (f - Fq - Fk), d.v_sm};
    return Lane{2, f, nullptr, 0};
  }
  // Of 16-bit values by the hardware's exponential and reciprocal, off by some
  // 2^-22 where the result is rounded to 2^-9 (the lambdas of a tile are few
  // lanes' work and hold up the whole launch: 35 instructions against 4).
  static __device__ __forceinline__ float sigmoid(float x) {
    if constexpr (sizeof(T) == 4) return proj_sigmoid(x);
    else return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504f * x));
  }
  // a row's runs of n T's: at 8-byte addresses at least (the entry's checks)
  template <int n>
  static __device__ __forceinline__ void st(T* p, const Feats<T, n>& v) {
    typedef uint32_t V __attribute__((ext_vector_type(sizeof(v) / 4), aligned(sizeof(v) == 4 ? 4 : 8)));
    *reinterpret_cast<V*>(p) = __builtin_bit_cast(V, v);
  }
  template <int M, int R>
  __device__ __forceinline__ void put(const Lane& l, int m, int step, int rows, const Feats<T, M> (&v)[R]) const {
    T* row = l.at + (int64_t)m * l.sm;
    const int64_t next = step * l.sm;
    if (l.kind == 0) {
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (m + r * step < rows) st(row + r * next, v[r]);
    } else if (l.kind == 1) {
      typedef Feats<T, M / 2> Half;  // a table's entries of M / 2 pairs, at any element address
      struct Any {
        T v[M / 2];
      };
      const int half = d.Dh / 2, p = l.c / 2;
      const bool inter = d.rope_interleaved != 0;
      Any cs[R], sn[R];
      int prow[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        prow[r] = (int)len.mod((uint32_t)min(m + r * step, rows - 1));
        if (!(TABLES && tab.inv_freq)) {
          typedef uint16_t U __attribute__((ext_vector_type(sizeof(Any) / 2), aligned(2)));
          const int64_t at = (int64_t)prow[r] * half + p;
          cs[r] = __builtin_bit_cast(Any, *reinterpret_cast<const U*>((const T*)d.rope_cos + at));
          sn[r] = __builtin_bit_cast(Any, *reinterpret_cast<const U*>((const T*)d.rope_sin + at));
        }
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (m + r * step >= rows) continue;
        Feats<T, M> o;  // pair by pair
        Half first, second;
#pragma unroll
        for (int pp = 0; pp < M / 2; ++pp) {
          const float2 a = TABLES && tab.inv_freq ? rope_angle<T>(tab.inv_freq, tab.inv_dtype, tab.p0 + prow[r], p + pp)
                                                  : float2{E::ld(cs[r].v[pp]), E::ld(sn[r].v[pp])};
          float o0, o1;
          rope_pair_t<T>(E::ld(v[r].v[2 * pp]), E::ld(v[r].v[2 * pp + 1]), a.x, a.y, inter, o0, o1);
          o.v[2 * pp] = first.v[pp] = E::st(o0);
          o.v[2 * pp + 1] = second.v[pp] = E::st(o1);
        }
        T* at = row + r * next;
        if (inter) {
          st(at + l.c, o);
        } else {  // pairs (p, p + half): channels p .. and the same + half
          st(at + p, first);
          st(at + p + half, second);
        }
      }
    } else {
      const int o_l = d.H * d.Dh + 2 * d.Hkv * d.Dh, o_g = o_l + d.H;
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int e = 0; e < M; ++e) {
          const int f = l.c + e;
          const int64_t mr = m + r * step;
          if (f >= n_feat || mr >= rows) continue;
          const float sg = E::rnd(sigmoid(E::ld(v[r].v[e])));
          if (f < o_g) ((T*)d.lam)[mr * d.lam_sm + (f - o_l)] = E::st(sg);
          else d.g[mr] = sg;
        }
    }
  }
  __device__ __forceinline__ void once(int t) const {
    if constexpr (TABLES) leave_tables<T>(tab, d.L, d.Dh / 2, t);
  }
};

// three roundings to fp32 (the sum, times the token's scale, times the
// channel's plus bias) and the one to T
template <typename T>
__device__ __forceinline__ Feats<T, 4> int8_value(const i32x4& a, float sx, const pf32x4& sw, const pf32x4& bias) {
  Feats<T, 4> v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v.v[e] = Elt<T>::st(fmaf((float)a[e] * sx, sw[e], bias[e]));
  return v;
}

// ---- tiles
// 16 bytes a lane, global -> LDS at lds + 16 lane (counted in vmcnt)
__device__ __forceinline__ void tile_load16(const void* g, void* lds) {
  __builtin_amdgcn_global_load_lds(g, (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
}
__device__ __forceinline__ uint32_t tile_lds(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)p;
}
// LDS read by hand: the compiler would wait for every load to LDS in flight
// before its own (it cannot tell the stages apart)
template <int OFF>
__device__ __forceinline__ i32x4 tile_read(uint32_t addr) {
  static_assert(OFF >= 0 && OFF < 65536, "ds offset is 16 bits");
  i32x4 r;
  asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(r) : "v"(addr), "i"(OFF));
  return r;
}
// all of its reads have landed
template <int N>
__device__ __forceinline__ void tile_landed(i32x4 (&a)[N]) {
  if constexpr (N == 2) asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(a[0]), "+v"(a[1]));
  if constexpr (N == 3) asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(a[0]), "+v"(a[1]), "+v"(a[2]));
  if constexpr (N == 4) asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(a[0]), "+v"(a[1]), "+v"(a[2]), "+v"(a[3]));
  if constexpr (N == 5)
    asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(a[0]), "+v"(a[1]), "+v"(a[2]), "+v"(a[3]), "+v"(a[4]));
  if constexpr (N == 6)
    asm volatile("s_waitcnt lgkmcnt(0)"
                 : "+v"(a[0]), "+v"(a[1]), "+v"(a[2]), "+v"(a[3]), "+v"(a[4]), "+v"(a[5]));
  if constexpr (N == 8)
    asm volatile("s_waitcnt lgkmcnt(0)"
                 : "+v"(a[0]), "+v"(a[1]), "+v"(a[2]), "+v"(a[3]), "+v"(a[4]), "+v"(a[5]), "+v"(a[6]), "+v"(a[7]));
}
template <class F, int... I>
__device__ __forceinline__ void each_impl(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void each(F&& f) {
  each_impl(f, std::make_integer_sequence<int, N>{});
}

// An accumulator out of its AGPR, here and not earlier: the compiler would
// move all 256 at once, over registers that the loop then lacks.  (The
// caller is a barrier behind the last product: no hazard is left.)
__device__ __forceinline__ int32_t acc_read(int32_t a) {
  int32_t v;
  asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(v) : "a"(a));
  return v;
}

struct TileAt {
  int f, m;
};
// Workgroups go round the 8 XCDs; each XCD takes a run of tiles of its own, t0
// .. end, in groups of 4 token tiles, so that what it has at a time shares rows
// in its L2; its workgroups take them in turn.
struct TileOrder {
  int ntf, ntm, t0, end;
  __device__ __forceinline__ TileOrder(int ntf_, int ntm_) : ntf(ntf_), ntm(ntm_) {
    const int n = ntf * ntm, xcd = blockIdx.x & 7, base = n >> 3, rem = n & 7;
    t0 = xcd * base + min(xcd, rem);
    end = t0 + base + (xcd < rem ? 1 : 0);
  }
  template <int BF, int BM>
  __device__ __forceinline__ TileAt at(int t) const {
    const int group = t / (4 * ntf), in = t - group * 4 * ntf, gm = min(4, ntm - 4 * group);
    return TileAt{in / gm * BF, (4 * group + in % gm) * BM};
  }
};

// A wave's values out: through LDS (at mine, rows of ROW bytes, its own) from
// four features of 32 tokens a lane to runs of a token's features, FEATS of
// them at a time.  sw, sb, sx: in LDS, of its first feature and token (f0, m0).
template <int SF, int SM, int FEATS, int ROW, typename Sink>
__device__ __forceinline__ void tile_out(const i32x16 (&acc)[SF][SM], char* mine, const float* sw, const float* sb,
                                         const float* sx, int le, int f0, int m0, int n_feat, int rows, const Sink& sink) {
  typedef typename Sink::Out T;
  constexpr int N = Sink::kRun, PR = FEATS / N, NF = FEATS / 32;  // runs of a row, blocks of 32 features
  const int fq = le % PR * N, four = 4 * (le >> 5);
  each<SM>([&](auto jc) {
    constexpr int j = decltype(jc)::value;
    const float x = sx[32 * j + (le & 31)];
    each<SF / NF>([&](auto pc) {
      constexpr int part = decltype(pc)::value;
      each<4 * NF>([&](auto gc) {
        constexpr int q = decltype(gc)::value, i = part * NF + q / 4, r = q % 4, f = 32 * i + 8 * r;
        const pf32x4 w = *reinterpret_cast<const pf32x4*>(sw + four + f), b = *reinterpret_cast<const pf32x4*>(sb + four + f);
        i32x4 v;
        each<4>([&](auto ec) {
          constexpr int e = decltype(ec)::value;
          v[e] = SF == 4 ? acc_read(acc[i][j][4 * r + e]) : acc[i][j][4 * r + e];
        });
        *reinterpret_cast<Feats<T, 4>*>(mine + (le & 31) * ROW + (32 * (q / 4) + 8 * r + four) * sizeof(T)) =
            int8_value<T>(v, x, w, b);
      });
      __builtin_amdgcn_wave_barrier();
      const int f = f0 + part * FEATS + fq;
      const typename Sink::Lane to = sink.lane(min(f, n_feat - 1));
      constexpr int R = PR / 2;  // of 32 tokens: 64 / PR a turn
      Feats<T, N> v[R];
#pragma unroll
      for (int r = 0; r < R; ++r)
        v[r] = *reinterpret_cast<const Feats<T, N>*>(mine + (r * (64 / PR) + le / PR) * ROW + fq * sizeof(T));
      if (f < n_feat) sink.put(to, m0 + 32 * j + le / PR, 64 / PR, rows, v);
      __builtin_amdgcn_wave_barrier();
    });
  });
}

// 4 waves (2 x 2) make 64 SF features x 64 SM tokens, a wave 32 SF x 32 SM in
// SF x SM accumulators of 32 x 32.  K passes through LDS in steps of 128 bytes
// (whole lines: rows of 64 bytes come out of L2 at 70 GB/s a CU, of 128 at
// 120), ST stages.  A step is four quarters of 32 bytes of K.  Beside a
// quarter's products the next one's operands are read, so that none waits for
// LDS.  The one barrier of a step is before its last quarter: by then every
// wave has read all of the step, whose stage is loaded anew (step + ST) beside
// that quarter and the next two, and the next step, whose first operands are
// read now, has landed.  Where a quarter is a product or two (SF = 1),
// all operands of a step are read beside the products of the one before, and
// the barrier is at a step's start.  A stage holds a row's eight 16-byte pieces in the
// order slot = piece ^ (row / 2) % 8, by which the 16 lanes that LDS serves at
// once (of 32 rows: 0-3, 12-15, 20-27 and the rest) touch every bank once.
// KS = 2: two sets of four waves, a half of K and a ring of stages each; the
// second set's sums pass through LDS at the end.
// A workgroup of the largest tiles goes from tile to tile; the stages run on
// over the border, so that the next tile's first steps are in LDS when this
// one's values have been written, and the writes are on their way while its
// products run.  Those are bound by the matrix pipe, whose clock falls to 1.25
// to 1.6 GHz under it: 16384 x 8192 x 8192 880-900 us = 2440-2500 TOP/s, 32768
// x 4096 x 6177 767 us; the smaller ones by what L2 and LDS deliver beside few
// products: 1999 x 4096 x 4096 41 us, 128 x 8192 x 10305 33.
template <int SF, int SM, int ST, int KS, typename T>
struct TileLds {
  static constexpr int kRows = 64 * (SF + SM);  // features, then tokens
  static constexpr int kStage = kRows * 128;    // bytes
  static constexpr bool kWalk = SF * SM == 16;
  // a wave's values on their way out: 32 tokens x kFeats features
  static constexpr int kFeats = kWalk ? 128 / (int)sizeof(T) : 32 * SF;
  static constexpr int kRow = kFeats * sizeof(T) + 16;
  static constexpr int kScales = 64 * (2 * SF + SM) * sizeof(float);  // features' scales, biases, tokens' scales
  static constexpr int kOut = kWalk ? ST * kStage : 0;         // (smaller tiles: over the stages)
  static constexpr size_t kSums = kOut + kScales + 4 * 32 * kRow;  // of the second half of K
  static constexpr size_t kEnd = kSums + (KS - 1) * SF * SM * 16 * 256 * sizeof(int32_t);
  static constexpr size_t kBytes = kEnd > KS * ST * kStage ? kEnd : KS * ST * kStage;
};
template <int SF, int SM, int ST, int KS, typename Sink>
__global__ __launch_bounds__(256 * KS) __attribute__((amdgpu_waves_per_eu(SF == 4 ? 1 : 2))) void int8_tile(
    const Int8Mat X, const Int8Mat W, int K, int ntf, int ntm, const Sink sink) {
  typedef typename Sink::Out T;
  typedef TileLds<SF, SM, ST, KS, T> L;
  static_assert(KS == 1 || SF == 1, "tiles of more products a step are not split");
  extern __shared__ __attribute__((aligned(128))) char smem[];
  constexpr int BF = 64 * SF, BM = 64 * SM, NO = SF + SM, NL = 2 * NO;  // NO operands a quarter, NL loads a thread and step
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wv = wave & 3, part_k = KS == 1 ? 0 : wave >> 2;  // the share of K
  char* const stages = smem + part_k * (ST * L::kStage);
  const TileOrder order(ntf, ntm);
  const int t0 = order.t0, end = order.end, turn = ((int)gridDim.x - (int)(blockIdx.x & 7) + 7) >> 3;
  const auto place = [&](int t) { return order.at<BF, BM>(t); };
  // this lane's pieces, as offsets from a tile's first rows: a load is 8 rows
  // of eight pieces, the first 2 SF of them features
  uint32_t src[NL];
  const int8_t *wsrc, *xsrc;
  auto aim = [&](const TileAt& a) {
    int l = lane;
    asm volatile("" : "+v"(l));  // (nothing of this is worth a register between tiles)
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int r = (4 * (i < 2 * SF ? i : i - 2 * SF) + wv) * 8 + (l >> 3), piece = (l & 7) ^ ((r >> 1) & 7);
      src[i] = 16 * piece + (i < 2 * SF ? (uint32_t)min(r, W.rows - 1 - a.f) * (uint32_t)W.sm
                                        : (uint32_t)min(r, X.rows - 1 - a.m) * (uint32_t)X.sm);
    }
    wsrc = W.p + a.f * W.sm + part_k * (K / KS);
    xsrc = X.p + a.m * X.sm + part_k * (K / KS);
  };
  // the loads: tile lt's step lk, the ls-th of all, to stage lat; on to the next
  // tile at its end
  const int steps = K / (128 * KS);
  int tile = t0 + (int)(blockIdx.x >> 3), lt = tile, lk = 0, ls = 0, lat = 0;
  auto load1 = [&](auto c) {
    constexpr int i = decltype(c)::value;
    tile_load16((i < 2 * SF ? wsrc : xsrc) + src[i], stages + lat + wv * 1024 + i * 4096);
  };
  auto next_stage = [](int at) { return at + L::kStage == ST * L::kStage ? 0 : at + L::kStage; };
  auto loaded = [&]() {
    ++ls;
    lat = next_stage(lat);
    wsrc += 128;
    xsrc += 128;
    if (++lk == steps) {
      lk = 0;
      lt = L::kWalk ? lt + turn : end;
      if (lt < end) aim(place(lt));
    }
  };
  i32x16 acc[SF][SM];
  // operands of quarter h of a step: pieces 2 h + lane / 32
  const int wf = wv >> 1, wm = wv & 1, r32 = lane & 31;
  const uint32_t at = tile_lds(stages) + r32 * 128 + (((lane >> 5) ^ ((r32 >> 1) & 7)) << 4);
  constexpr bool kAhead = SF == 1;  // a whole step's operands are read ahead
  i32x4 op[kAhead ? 8 : 2][NO];
  auto read = [&](auto c, i32x4 (&o)[NO], uint32_t a) {  // operand c: SF of features, SM of tokens
    constexpr int i = decltype(c)::value;
    if constexpr (i < SF) o[i] = tile_read<i * 4096>(a + wf * (SF * 4096));
    else o[i] = tile_read<BF * 128 + (i - SF) * 4096>(a + wm * (SM * 4096));
  };
  // The products of a quarter; beside the first of them the reads of the next
  // one's operands, at address a; beside the last loads from .. to of the step
  // that is asked for (asked for all at once, they hold the wave up).
  auto quarter = [&](auto from, auto to, bool some, i32x4 (&now)[NO], i32x4 (&next)[NO], uint32_t a) {
    constexpr int n = SF * SM, lo = decltype(from)::value, hi = decltype(to)::value;
    constexpr int reads = n >= 2 * NO ? 1 : 2, first = n / 2, loads = (hi - lo + n - first - 1) / (n - first);
    each<n>([&](auto c) {
      constexpr int q = decltype(c)::value, i = q / SM, j = q % SM;
      each<reads>([&](auto d) {
        constexpr int o = q * reads + decltype(d)::value;
        if constexpr (o < NO) read(std::integral_constant<int, o>{}, next, a);
      });
      if constexpr (q >= first && lo + (q - first) * loads < hi)
        if (some)
          each<loads>([&](auto d) {
            constexpr int o = lo + (q - first) * loads + decltype(d)::value;
            if constexpr (o < hi) load1(std::integral_constant<int, o>{});
          });
      acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(now[i], now[SF + j], acc[i][j], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    });
    tile_landed(next);
  };
  // steps up to n have landed: those asked for behind it may be on their way
  auto landed = [&](int n) {
    const int behind = ls - 1 - n;
    if (behind <= 0) __builtin_amdgcn_s_waitcnt(0x0f70);
    each<ST - 1>([&](auto c) {
      constexpr int v = (decltype(c)::value + 1) * NL;
      static_assert(v < 64, "vmcnt is 6 bits");
      if (behind == decltype(c)::value + 1) __builtin_amdgcn_s_waitcnt((v & 15) | (v >> 4) << 14 | 0x0f70);
    });
  };
  // Step g, in stage rat.  asked: a third of a step was asked for at the end of
  // the last one.
  int g = 0, rat = 0;
  bool asked = false;
  auto step = [&]() {
    constexpr int third = (NL + 2) / 3;
    constexpr std::integral_constant<int, 0> none{};
    constexpr std::integral_constant<int, third> one{};
    constexpr std::integral_constant<int, 2 * third> two{};
    constexpr std::integral_constant<int, NL> all{};
    const uint32_t here = at + rat;
    rat = next_stage(rat);
    quarter(one, two, asked, op[0], op[1], here ^ 32);
    quarter(two, all, asked, op[1], op[0], here ^ 64);
    if (asked) loaded();
    quarter(none, none, false, op[0], op[1], here ^ 96);
    landed(g + 1);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    asked = lt < end;
    quarter(none, one, asked, op[1], op[0], at + rat);
    ++g;
  };
  // The same with all operands read ahead, of set now (0 or 4), the next
  // step's to the other; loads beside the products.
  auto step_ahead = [&](auto set) {
    constexpr int now = decltype(set)::value, next = 4 - now, n = 4 * SF * SM, reads = 4 * NO / n + 1, loads = (NL + n - 1) / n;
    landed(g + 1);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    rat = next_stage(rat);
    const uint32_t then = at + rat;
    const bool ask = lt < end;
    each<n>([&](auto c) {
      constexpr int p = decltype(c)::value, h = p / (SF * SM), i = p % (SF * SM) / SM, j = p % SM;
      each<reads>([&](auto d) {
        constexpr int o = p * reads + decltype(d)::value;
        if constexpr (o < 4 * NO) read(std::integral_constant<int, o % NO>{}, op[next + o / NO], then ^ (32 * (o / NO)));
      });
      if constexpr (p * loads < NL)
        if (ask)
          each<loads>([&](auto d) {
            constexpr int o = p * loads + decltype(d)::value;
            if constexpr (o < NL) load1(std::integral_constant<int, o>{});
          });
      acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(op[now + h][i], op[now + h][SF + j], acc[i][j], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    });
    each<4>([&](auto h) { tile_landed(op[next + decltype(h)::value]); });
    if (ask) loaded();
    ++g;
  };
  aim(place(tile));
  for (int s = 0; s < ST && lt < end; ++s) {
    each<NL>([&](auto c) { load1(c); });
    loaded();
  }
  __builtin_amdgcn_sched_barrier(0);
  landed(0);
  __builtin_amdgcn_s_barrier();
  each<kAhead ? 4 : 1>([&](auto hc) {
    constexpr int h = decltype(hc)::value;
    each<NO>([&](auto c) { read(c, op[h], at ^ (32 * h)); });
    tile_landed(op[h]);
  });
  for (;;) {
    const TileAt a = place(tile);
    float scale[3] = {0.f, 0.f, 0.f};
    const int own = (int)threadIdx.x & 255;
    if (own < BF) {
      const int f = min(a.f + own, W.rows - 1);
      scale[0] = W.scales[f];
      scale[1] = sink.bias1(f);
    }
    if (own < BM) scale[2] = X.scales[min(a.m + own, X.rows - 1)];
#pragma unroll
    for (int i = 0; i < SF; ++i)
#pragma unroll
      for (int j = 0; j < SM; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;
    if constexpr (kAhead) {
      int k = 0;
      for (; k + 1 < steps; k += 2) {
        step_ahead(std::integral_constant<int, 0>{});
        step_ahead(std::integral_constant<int, 4>{});
      }
      if (k < steps) step_ahead(std::integral_constant<int, 0>{});
    } else {
      for (int k = 0; k < steps; ++k) step();
    }
    int le = lane;
    asm volatile("" : "+v"(le));  // (nor are these addresses)
    if (!L::kWalk) __builtin_amdgcn_s_barrier();  // every wave has read its last operands
    float* fs = reinterpret_cast<float*>(smem + L::kOut);
    if (own < BF) {
      fs[own] = scale[0];
      fs[BF + own] = scale[1];
    }
    if (own < BM) fs[2 * BF + own] = scale[2];
    i32x4* sums = reinterpret_cast<i32x4*>(smem + L::kSums) + own;
    if (KS == 2 && part_k)
      each<SF * SM * 4>([&](auto c) {
        constexpr int i = decltype(c)::value / 4, r = decltype(c)::value % 4;
        const i32x16& s = acc[i / SM][i % SM];
        sums[256 * decltype(c)::value] = i32x4{s[4 * r], s[4 * r + 1], s[4 * r + 2], s[4 * r + 3]};
      });
    // (the loads too: the writes below do not stand before them)
    __builtin_amdgcn_s_waitcnt(0x0070);
    __builtin_amdgcn_s_barrier();
    if constexpr (KS == 2) {
      if (part_k) return;
      each<SF * SM * 4>([&](auto c) {
        constexpr int i = decltype(c)::value / 4, r = decltype(c)::value % 4;
        const i32x4 s = sums[256 * decltype(c)::value];
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i / SM][i % SM][4 * r + e] += s[e];
      });
    }
    const int fw = 32 * SF * wf, mw = 32 * SM * wm;
    tile_out<SF, SM, L::kFeats, L::kRow>(acc, smem + L::kOut + L::kScales + wv * 32 * L::kRow, fs + fw, fs + BF + fw,
                                         fs + 2 * BF + mw, le, a.f + fw, a.m + mw, W.rows, X.rows, sink);
    if (!L::kWalk) break;
    tile += turn;
    if (tile >= end) break;
  }
}

// A tile of 32 FB features x 64 tokens of whose K each of 4 waves takes a quarter, in steps of 128
// bytes through two LDS stages of its own: no wave waits for another, and every
// operand passes LDS once (in int8_tile twice).  Beside the first half of a
// step's 8 FB products the step after next is asked for, into the stage whose
// operands are in registers by now; beside the second half the next step's
// operands are read.  Then the waves exchange sums and write blocks of 32 x 32.
// Bound by a CU's loads (a MiB in 14 us at 128 x 8192 x 4096).  us, weights in
// cache | not, beside int8_tile<1, 1, 4, 1>: 128 x 8192 x 8192 17.4 | 22.7 and
// 25.5 | 26.1, 128 x 8192 x 4096 15.2 | 20.1 and 24.1 | 23.1, 256 x 4096 x 4096
// 10.6 | 11.4 and 14.8 | 13.5, 200 x 512 x 1024 4.2 both.  With two sets of four
// waves and halves of K 24.0, 21.6 and 12.4 (weights not in cache), with eight
// waves of a stage each 24.0, 21.1 and 11.8.
template <int FB, typename Sink>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1))) void int8_quarters(
    const Int8Mat X, const Int8Mat W, int K, int ntf, int ntm, const Sink sink) {
  typedef typename Sink::Out T;
  extern __shared__ __attribute__((aligned(128))) char smem[];
  constexpr int BF = 32 * FB, NO = FB + 2, NL = 4 * NO, NP = 8 * FB, kStage = (BF + 64) * 128;
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const TileOrder order(ntf, ntm);
  const TileAt a = order.at<BF, 64>(order.t0 + (int)(blockIdx.x >> 3));
  // of a ring: a wave's sums, then (at kOut) its values
  constexpr int kSums = FB * 2 * 4096, kRow = 32 * sizeof(T) + 16, kOut = kSums + 4 * (2 * BF + 64);
  static_assert(kOut + 32 * kRow <= 2 * kStage, "the exchange lies in the rings");
  char* const mine = smem + wv * (2 * kStage);
  const int steps = K / 128, first = steps * wv / 4, np = steps * (wv + 1) / 4 - first;
  uint32_t src[NL];  // a load: 8 rows of eight pieces (their order in LDS as in int8_tile)
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int r = 8 * (i < 4 * FB ? i : i - 4 * FB) + (lane >> 3), piece = (lane & 7) ^ ((r >> 1) & 7);
    src[i] = 16 * piece + (i < 4 * FB ? (uint32_t)min(r, W.rows - 1 - a.f) * (uint32_t)W.sm
                                 : (uint32_t)min(r, X.rows - 1 - a.m) * (uint32_t)X.sm);
  }
  const int8_t *wsrc = W.p + a.f * W.sm + first * 128, *xsrc = X.p + a.m * X.sm + first * 128;
  auto load1 = [&](auto c, int stage) {
    constexpr int i = decltype(c)::value;
    tile_load16((i < 4 * FB ? wsrc : xsrc) + src[i], mine + stage * kStage + i * 1024);
  };
  auto loaded = [&]() {
    wsrc += 128;
    xsrc += 128;
  };
  // operands of quarter h of a step: pieces 2 h + lane / 32; FB of features,
  // two of tokens
  const int r32 = lane & 31;
  const uint32_t at = tile_lds(mine) + r32 * 128 + (((lane >> 5) ^ ((r32 >> 1) & 7)) << 4);
  i32x4 op[8][NO];
  i32x16 acc[FB][2];
#pragma unroll
  for (int i = 0; i < 2 * FB; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[i / 2][i % 2][e] = 0;
  auto read = [&](auto c, auto set) {  // operand c of NL, of the step in stage set
    constexpr int h = decltype(c)::value / NO, i = decltype(c)::value % NO, st = decltype(set)::value;
    op[4 * st + h][i] = tile_read<st * kStage + i * 4096>(at ^ (32 * h));
  };
  auto step = [&](auto set, int behind) {  // behind: steps left after this one
    constexpr int now = decltype(set)::value, next = 1 - now;
    const bool ask = behind >= 2;
    each<NP>([&](auto c) {
      constexpr int p = decltype(c)::value, h = p / (2 * FB), i = p % (2 * FB) / 2, j = p % 2, late = p - NP / 2;
      if constexpr (2 * p < NL)
        if (ask) {
          load1(std::integral_constant<int, 2 * p>{}, now);
          load1(std::integral_constant<int, 2 * p + 1>{}, now);
        }
      if constexpr (late == 0) {  // the next step has landed
        if (ask) __builtin_amdgcn_s_waitcnt((NL & 15) | (NL >> 4) << 14 | 0x0f70);
        else __builtin_amdgcn_s_waitcnt(0x0f70);
        __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (late >= 0 && 2 * late < NL) {
        read(std::integral_constant<int, 2 * late>{}, std::integral_constant<int, next>{});
        read(std::integral_constant<int, 2 * late + 1>{}, std::integral_constant<int, next>{});
      }
      acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(op[4 * now + h][i], op[4 * now + h][FB + j], acc[i][j], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    });
    each<4>([&](auto h) { tile_landed(op[4 * next + decltype(h)::value]); });
    if (ask) loaded();
  };
  // (the values and the scales over the ends of rings)
  float* fs = reinterpret_cast<float*>(smem + kOut - 4 * (2 * BF + 64));  // of features, their biases, of tokens
  float scale[3] = {0.f, 0.f, 0.f};
  const int own = (int)threadIdx.x;
  if (own < BF) {
    const int f = min(a.f + own, W.rows - 1);
    scale[0] = W.scales[f];
    scale[1] = sink.bias1(f);
  }
  if (own < 64) scale[2] = X.scales[min(a.m + own, X.rows - 1)];
  __builtin_amdgcn_sched_barrier(0);
  for (int s = 0; s < 2 && s < np; ++s) {
    each<NL>([&](auto c) { load1(c, s); });
    loaded();
  }
  __builtin_amdgcn_sched_barrier(0);
  if (np > 1) __builtin_amdgcn_s_waitcnt((NL & 15) | (NL >> 4) << 14 | 0x0f70);
  else __builtin_amdgcn_s_waitcnt(0x0f70);
  __builtin_amdgcn_sched_barrier(0);
  each<NL>([&](auto c) { read(c, std::integral_constant<int, 0>{}); });
  each<4>([&](auto h) { tile_landed(op[decltype(h)::value]); });
  int k = 0;
  for (; k + 1 < np; k += 2) {
    step(std::integral_constant<int, 0>{}, np - 1 - k);
    step(std::integral_constant<int, 1>{}, np - 2 - k);
  }
  if (k < np) step(std::integral_constant<int, 0>{}, 0);
  i32x4* sums = reinterpret_cast<i32x4*>(smem) + lane;
  constexpr int kWave = 2 * kStage / 16;  // from wave to wave
  each<NP>([&](auto c) {
    constexpr int b = decltype(c)::value / 4, r = decltype(c)::value % 4;
    const i32x16& s = acc[b / 2][b % 2];
    sums[wv * kWave + 64 * decltype(c)::value] = i32x4{s[4 * r], s[4 * r + 1], s[4 * r + 2], s[4 * r + 3]};
  });
  // (the scales lie in wave 0's ring: behind its loop only by a barrier)
  __syncthreads();
  if (own < BF) {
    fs[own] = scale[0];
    fs[BF + own] = scale[1];
  }
  if (own < 64) fs[2 * BF + own] = scale[2];
  __syncthreads();
  for (int b = wv; b < 2 * FB; b += 4) {
    i32x16 total[1][1];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      i32x4 t = sums[64 * (4 * b + r)];
#pragma unroll
      for (int o = 1; o < 4; ++o) t += sums[o * kWave + 64 * (4 * b + r)];
#pragma unroll
      for (int e = 0; e < 4; ++e) total[0][0][4 * r + e] = t[e];
    }
    const int fw = 32 * (b >> 1), mw = 32 * (b & 1);
    tile_out<1, 1, 32, kRow>(total, mine + kOut, fs + fw, fs + BF + fw, fs + 2 * BF + mw, lane, a.f + fw, a.m + mw, W.rows,
                             X.rows, sink);
  }
}

template <int FB, typename Sink>
static int launch_quarters(const Int8Mat& X, const Int8Mat& W, int K, const Sink& sink, hipStream_t st, const char* who) {
  constexpr size_t kBytes = 4 * 2 * (32 * FB + 64) * 128;
  const int ntf = (W.rows + 32 * FB - 1) / (32 * FB), ntm = (X.rows + 63) / 64;
  if ((int64_t)ntf * ntm >= 1 << 24) return fail(CODA_EUNSUP, "%s: %lld tiles", who, (long long)ntf * ntm);
  const int rc = lds_limit<int8_quarters<FB, Sink>>(kBytes, who);
  if (rc) return rc;
  hipLaunchKernelGGL((int8_quarters<FB, Sink>), dim3(ntf * ntm), dim3(256), kBytes, st, X, W, K, ntf, ntm, sink);
  return check_launch("int8_quarters");
}

template <int SF, int SM, int ST, int KS, typename Sink>
static int launch_tile(const Int8Mat& X, const Int8Mat& W, int K, const Sink& sink, hipStream_t st, const char* who) {
  typedef TileLds<SF, SM, ST, KS, typename Sink::Out> L;
  const int64_t ntf = ((int64_t)W.rows + 64 * SF - 1) / (64 * SF), ntm = ((int64_t)X.rows + 64 * SM - 1) / (64 * SM);
  const int64_t n = ntf * ntm;
  // (a grid has less than 2^32 threads; a walk's tiles are counted in 32 bits)
  if (n >= (L::kWalk ? INT_MAX / 8 : 1 << 24)) return fail(CODA_EUNSUP, "%s: %lld tiles", who, (long long)n);
  const int rc = lds_limit<int8_tile<SF, SM, ST, KS, Sink>>(L::kBytes, who);
  if (rc) return rc;
  const int64_t grid = L::kWalk && n > device_cus() ? device_cus() : n;
  hipLaunchKernelGGL((int8_tile<SF, SM, ST, KS, Sink>), dim3((unsigned)grid), dim3(256 * KS), L::kBytes, st, X, W, K, (int)ntf, (int)ntm,
                     sink);
  return check_launch("int8_tile");
}

// ---- few token rows: the row kernels of the float projections on codes
template <typename Sink>
struct RowsSink {
  Sink sink;
  const float* sx;
  const float* sw;
  int n_feat;
  template <typename Src>
  __device__ __forceinline__ void operator()(const Src&, int f, int m, const i32x4& a) const {
    pf32x4 s, b;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int g = min(f + e, n_feat - 1);
      s[e] = sw[g];
      b[e] = sink.bias1(g);
    }
    const Feats<typename Sink::Out, 4> v[1] = {int8_value<typename Sink::Out>(a, sx[m], s, b)};
    sink.put(sink.lane(f), m, 1, m + 1, v);
  }
  __device__ __forceinline__ void once(int t) const { sink.once(t); }
};

static constexpr int kFloatRows = 4;
// Up to 4 tokens as they come, quantised by every workgroup while its first
// weights are on their way: the codes and scales of codes_kernel, the sums of
// proj_rows.  The codes lie in LDS, rows of K + 16 bytes; two waves or more
// share a row, which they read twice (the second time from cache).  K: of the
// weights, D <= K.  One launch against two, us, bf16: 4096 x 6177 10.1 and
// 11.3 at 1 row, 11.3 and 11.6 at 4, 13.8 and 12.0 at 8; 4096 x 4096 7.3 and
// 8.8, 512 x 649 4.1 and 4.9 at 1 row.
template <typename T, int RB, typename Sink>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2))) void int8_rows_of(
    const T* __restrict__ X, int64_t x_sm, int M, int D, const Int8Mat W, int K, const Sink sink) {
  using E = Elt<T>;
  typedef PlainR<T> R;
  extern __shared__ __attribute__((aligned(16))) char rows_smem[];
  __shared__ double tops[8];
  __shared__ float scales[kFloatRows];
  constexpr int LP = 4;  // pairs of k-steps in flight ahead of the products
  const int f0 = blockIdx.x * 16 * RB;
  const int t = threadIdx.x, lane = t & 63, wv = __builtin_amdgcn_readfirstlane(t >> 6), r16 = lane & 15, kq = lane >> 4;
  const int pairs = K / 128, p0 = pairs * wv / 8, np = pairs * (wv + 1) / 8 - p0;
  const int8_t* wr[RB];
#pragma unroll
  for (int i = 0; i < RB; ++i) wr[i] = W.p + (int64_t)min(f0 + 16 * i + r16, W.rows - 1) * W.sm + 128 * p0 + 16 * kq;
  pu32x4 a[LP][RB][2];
  auto load = [&](int u, int p) {
#pragma unroll
    for (int i = 0; i < RB; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) a[u][i][h] = *reinterpret_cast<const pu32x4*>(wr[i] + 128 * p + 64 * h);
  };
#pragma unroll
  for (int u = 0; u < LP; ++u)
    if (u < np) load(u, u);
  const int share = M == 1 ? 8 : M == 2 ? 4 : 2, step = 512 * share;  // waves a row; elements a turn
  const int m = wv / share, first = (wv % share * 64 + lane) * 8;
  const T* xr = X + (int64_t)min(m, M - 1) * x_sm;
  R top = 0, bad = 0;
  for (int k = first; k < D; k += step) {
    const Run8<T> v = run_ld(xr + k, D - k);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const R p = (R)E::ld(v.v[e]);
      top = __builtin_elementwise_max(top, __builtin_elementwise_abs(p));
      bad = __builtin_elementwise_fma(p, (R)0, bad);
    }
  }
  double P = wave_reduce((double)top, true) + wave_reduce((double)bad, false);  // NaN: no number in the row
  if (lane == 0) tops[wv] = P;
  __syncthreads();
  P = tops[m * share];
  for (int i = 1; i < share; ++i) {
    const double o = tops[m * share + i];
    P = P != P || o != o ? P + o : fmax(P, o);
  }
  const bool fine = P == P && P > 0.;
  if (m < M) {
    if (lane == 0) scales[m] = fine || P != P ? (float)(P / 127.) : 0.f;
    const Coder<R> code(P, fine);
    for (int k = first; k < K; k += step) {
      const Run8<T> v = run_ld(xr + k, D - k);
      uint32_t c[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) c[e] = code((R)E::ld(v.v[e]));
      *reinterpret_cast<uint2*>(rows_smem + m * (K + 16) + k) = fine ? pack8(c) : uint2{0u, 0u};
    }
  }
  __syncthreads();
  i32x4 acc[RB][1];
#pragma unroll
  for (int i = 0; i < RB; ++i) acc[i][0] = i32x4{0, 0, 0, 0};
  const char* br = rows_smem + min(r16, M - 1) * (K + 16) + 128 * p0 + 16 * kq;
  for (int p = 0; p < np; p += LP)
#pragma unroll
    for (int u = 0; u < LP; ++u) {
      if (p + u >= np) break;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const pu32x4 b = *reinterpret_cast<const pu32x4*>(br + 128 * (p + u) + 64 * h);
#pragma unroll
        for (int i = 0; i < RB; ++i) acc[i][0] = rows_mfma<int8_t>(a[u][i][h], b, acc[i][0]);
      }
      if (p + u + LP < np) load(u, p + u + LP);
    }
  __syncthreads();
  rows_finish<1, RB>(acc, rows_smem, W.rows, M, 0, RowsSink<Sink>{sink, scales, W.scales, W.rows});
}
template <typename T, int RB, typename Sink>
static int launch_rows_of(const T* X, int64_t x_sm, int M, int D, const Int8Mat& W, int K, const Sink& sink,
                          hipStream_t st, const char* who) {
  const size_t codes = (size_t)M * (K + 16), lds = codes > RowsLds<1, RB>::kBytes ? codes : RowsLds<1, RB>::kBytes;
  const int rc = lds_limit<int8_rows_of<T, RB, Sink>>(lds, who);
  if (rc) return rc;
  hipLaunchKernelGGL((int8_rows_of<T, RB, Sink>), dim3((W.rows + 16 * RB - 1) / (16 * RB)), dim3(512), lds, st, X, x_sm, M,
                     D, W, K, sink);
  return check_launch("int8_rows_of");
}
template <typename T, typename Sink>
static int launch_of(const void* x, int64_t x_sm, int M, int D, const Int8Mat& W, int K, const Sink& sink,
                     hipStream_t st, const char* who) {
  switch (rows_rb(W.rows)) {
    case 1: return launch_rows_of<T, 1>((const T*)x, x_sm, M, D, W, K, sink, st, who);
    case 2: return launch_rows_of<T, 2>((const T*)x, x_sm, M, D, W, K, sink, st, who);
    default: return launch_rows_of<T, 3>((const T*)x, x_sm, M, D, W, K, sink, st, who);
  }
}

static constexpr int kFewRows = 128;  // of the row kernels
template <typename Sink>
static int launch_few(const Int8Mat& X, const Int8Mat& W, int K, const Sink& sink, hipStream_t st, const char* who) {
  return launch_rows<int8_t>(MatRows<int8_t>{W.p, W.sm}, W.rows, K, X.p, X.sm, X.rows,
                             RowsSink<Sink>{sink, X.scales, W.scales, W.rows}, st, who);
}
static int64_t tiles_of(const Int8Mat& X, const Int8Mat& W, int f, int m) {
  return ((int64_t)W.rows + f - 1) / f * (((int64_t)X.rows + m - 1) / m);
}
// The row kernels or tiles: the former up to 32 rows, and up to 64 where there
// are few features (us, rows and tiles, weights not in cache | in cache: 32 x
// 4096 x 4096 7.6 | 7.3 and 10.8 | 9.2, 32 x 8192 x 8192 21.5 | 19.5 and 23.7 |
// 15.1, 64 x 4096 x 4096 9.5 | 9.0 and 12.0 | 9.2, 64 x 4096 x 6177 14.7 | 12.7
// and 13.8 | 9.7, 64 x 8192 x 8192 24.5 | 22.0 and 25.4 | 16.4, 64 x 8192 x
// 10305 31.8 | 26.6 and 28.3 | 18.2).
static bool few_rows(const Int8Mat& X, const Int8Mat& W) { return X.rows <= (W.rows < 6144 ? 64 : 32); }
// Whether tiles of 96 x 64 save a second round of 64 x 64 (weights not in cache |
// in cache, us, the best of the others and this: 128 x 8192 x 10305 33.9 | 24.0
// and 30.8 | 21.0, 250 x 4096 x 6000 16.9 | 15.4 and 15.8 | 13.2, 128 x 1024 x
// 9000 7.1 | 7.8 and 7.5 | 8.0)
static bool one_round_of_96(const Int8Mat& X, const Int8Mat& W, int K) {
  return K >= 2048 && tiles_of(X, W, 64, 64) > device_cus() && tiles_of(X, W, 96, 64) <= device_cus();
}
// The tile by the time that its rounds take, us a round of one tile (64 x 64:
// two) a CU at K = 4096.  Measured, 256 x 256 | 256 x 128 | 128 x 128 | 64 x
// 128 | 64 x 64 (features x tokens): 1999 x 4096 x 4096 55 41 50 - 75, 1999 x
// 4096 x 6177 58 68 81 - 107, 1000 x 4096 x 4096 52 31 24 35 38, 300 x 4096 x
// 6177 - 37 20 32 21, 500 x 2048 x 3105 - 19 12.5 10.6 10.8, 128 x 8192 x
// 10305 - - 43 33 41, 128 x 8192 x 8192 - - 42 31 23, 4096 x 4096 x 6177 112
// 130 157 - -, 2000 x 1024 x 1024 - - 9.3 - 8.1.
template <typename Sink>
static int launch_many(const Int8Mat& X, const Int8Mat& W, int K, const Sink& sink, hipStream_t st, const char* who) {
  const int64_t cus = device_cus(), n1 = tiles_of(X, W, 64, 64);
  const auto rounds = [&](int f, int m) { return (tiles_of(X, W, f, m) + cus - 1) / cus; };
  const int64_t t44 = 56 * rounds(256, 256), t42 = 39 * rounds(256, 128), t22 = 23 * rounds(128, 128);
  const int64_t t12 = 17 * rounds(64, 128), t11 = n1 <= cus ? 12 : 19 * ((n1 + 2 * cus - 1) / (2 * cus));
  const int64_t t31 = one_round_of_96(X, W, K) ? 15 : INT_MAX;
  const int64_t least = std::min({t44, t42, t22, t12, t31, t11});
  if (t31 == least) return launch_quarters<3>(X, W, K, sink, st, who);
  if (t44 == least) return launch_tile<4, 4, 2, 1>(X, W, K, sink, st, who);
  if (t42 == least) return launch_tile<4, 2, 3, 1>(X, W, K, sink, st, who);
  if (t22 == least) return launch_tile<2, 2, 4, 1>(X, W, K, sink, st, who);
  // (64 x 128 in one round: a workgroup a CU anyway, so with a second set of
  // waves for half of K, if it has halves of whole steps: 250 x 4096 x 6177 18.6
  // -> 17.0, 128 x 8192 x 10305 33.6 -> 33.1)
  const bool halves = K % 256 == 0;
  if (t12 == least)
    return halves && tiles_of(X, W, 64, 128) <= cus ? launch_tile<1, 2, 3, 2>(X, W, K, sink, st, who)
                                                    : launch_tile<1, 2, 4, 1>(X, W, K, sink, st, who);
  return n1 <= cus ? launch_quarters<2>(X, W, K, sink, st, who) : launch_tile<1, 1, 4, 1>(X, W, K, sink, st, who);
}

static int check_codes_out(const int8_t* codes, int64_t c_sm, const float* scales, int rows, int D, const char* who) {
  CODA_REQUIRE(rows >= 0 && D > 0, "%s: bad sizes rows=%d D=%d", who, rows, D);
  if (D > kMaxRow) return fail(CODA_EUNSUP, "%s: rows of %d elements (at most %d)", who, D, kMaxRow);
  if (rows == 0) return CODA_OK;
  CODA_REQUIRE(codes && scales, "%s: null pointer", who);
  CODA_REQUIRE((uintptr_t)codes % 16 == 0 && c_sm % 16 == 0 && c_sm >= (D + kPad - 1) / kPad * kPad,
               "%s: rows of codes must lie at 16-byte addresses and hold D=%d up to a multiple of %d", who, D, kPad);
  return CODA_OK;
}
static bool int8_dtype(int t) { return t == CODA_F32 || t == CODA_BF16 || t == CODA_F16; }

// The two operands of a product: of X codes, or (no scales) D elements a row
static int check_mats(const Int8Mat& X, int D, const Int8Mat& W, int K, const char* who) {
  CODA_REQUIRE(X.rows >= 0 && W.rows > 0 && K > 0 && K % kPad == 0 && K <= kMaxK,
               "%s: bad sizes rows=%d features=%d K=%d (K a multiple of %d, at most %d: int32 holds the sum)", who, X.rows,
               W.rows, K, kPad, kMaxK);
  if (X.rows > kMaxRows || W.rows > kMaxRows)
    return fail(CODA_EUNSUP, "%s: %d rows times %d (at most 2^30)", who, X.rows, W.rows);
  CODA_REQUIRE(W.p && W.scales && (X.rows == 0 || X.p), "%s: null pointer", who);
  const char* lie = "%s: rows of codes must lie at 16-byte addresses, %lld bytes apart at most";
  CODA_REQUIRE((uintptr_t)W.p % 16 == 0 && W.sm % 16 == 0 && W.sm >= 0 && W.sm <= kMaxStride, lie, who,
               (long long)kMaxStride);
  if (X.scales || X.rows == 0) {
    CODA_REQUIRE((uintptr_t)X.p % 16 == 0 && X.sm % 16 == 0 && X.sm >= 0 && X.sm <= kMaxStride, lie, who,
                 (long long)kMaxStride);
  } else {
    CODA_REQUIRE(X.rows <= kFloatRows, "%s: %d token rows without scales (at most %d are quantised by the launch)", who,
                 X.rows, kFloatRows);
    CODA_REQUIRE(D > 0 && D <= K && X.sm >= 0, "%s: rows of %d elements for K=%d", who, D, K);
  }
  return CODA_OK;
}

}  // namespace coda

using namespace coda;

extern "C" int coda_quantize_rows(int dtype, const void* x, int64_t x_sm, int rows, int D, int8_t* codes, int64_t c_sm,
                                  float* scales, void* stream) {
  const char* who = "coda_quantize_rows";
  CODA_REQUIRE(int8_dtype(dtype), "%s: dtype must be CODA_F32, CODA_BF16 or CODA_F16", who);
  const int rc = check_codes_out(codes, c_sm, scales, rows, D, who);
  if (rc || rows == 0) return rc;
  CODA_REQUIRE(x, "%s: null pointer", who);
  const hipStream_t st = (hipStream_t)stream;
#define RUN(T) run_codes<T, false, false>(x, x_sm, nullptr, 0, nullptr, rows, D, 0.f, nullptr, 0, codes, c_sm, scales, st)
  return dtype == CODA_F32 ? RUN(float) : dtype == CODA_BF16 ? RUN(bf16_t) : RUN(f16_t);
#undef RUN
}

extern "C" int coda_rms_norm_int8(int dtype, const void* x, int64_t x_sm, const void* residual, int64_t r_sm,
                                  const void* weight, int rows, int D, float eps, void* sum_out, int64_t s_sm,
                                  int8_t* codes, int64_t c_sm, float* scales, void* stream) {
  const char* who = "coda_rms_norm_int8";
  CODA_REQUIRE(int8_dtype(dtype), "%s: dtype must be CODA_F32, CODA_BF16 or CODA_F16", who);
  const int rc = check_codes_out(codes, c_sm, scales, rows, D, who);
  if (rc || rows == 0) return rc;
  CODA_REQUIRE(x && weight && (!residual || sum_out), "%s: null pointer", who);
  CODA_REQUIRE(eps >= 0.f, "%s: eps=%g is negative", who, (double)eps);
  const hipStream_t st = (hipStream_t)stream;
#define RUN(T, RES) \
  run_codes<T, true, RES>(x, x_sm, residual, r_sm, weight, rows, D, eps, sum_out, s_sm, codes, c_sm, scales, st)
  if (residual) return dtype == CODA_F32 ? RUN(float, true) : dtype == CODA_BF16 ? RUN(bf16_t, true) : RUN(f16_t, true);
  return dtype == CODA_F32 ? RUN(float, false) : dtype == CODA_BF16 ? RUN(bf16_t, false) : RUN(f16_t, false);
#undef RUN
}

extern "C" int coda_dequantize_rows(int dtype, const int8_t* codes, int64_t c_sm, const float* scales, int rows, int D,
                                    void* out, int64_t o_sm, void* stream) {
  const char* who = "coda_dequantize_rows";
  CODA_REQUIRE(int8_dtype(dtype), "%s: dtype must be CODA_F32, CODA_BF16 or CODA_F16", who);
  CODA_REQUIRE(rows >= 0 && D > 0, "%s: bad sizes rows=%d D=%d", who, rows, D);
  if (rows == 0) return CODA_OK;
  CODA_REQUIRE(codes && scales && out, "%s: null pointer", who);
  CODA_REQUIRE((uintptr_t)codes % 16 == 0 && c_sm % 16 == 0 && c_sm >= (D + kPad - 1) / kPad * kPad && D <= kMaxK,
               "%s: rows of codes must lie at 16-byte addresses and hold D=%d up to a multiple of %d", who, D, kPad);
  const hipStream_t st = (hipStream_t)stream;
#define RUN(T) run_values<T>(codes, c_sm, scales, rows, D, out, o_sm, st)
  return dtype == CODA_F32 ? RUN(float) : dtype == CODA_BF16 ? RUN(bf16_t) : RUN(f16_t);
#undef RUN
}

extern "C" int coda_linear_int8(int dtype, const void* x, int64_t x_sm, const float* x_scales, int M, int D,
                                const int8_t* w, int64_t w_sm, const float* w_scales, int n_feat, int K, const void* bias,
                                void* out, int64_t o_sm, void* stream) {
  const char* who = "coda_linear_int8";
  CODA_REQUIRE(int8_dtype(dtype), "%s: dtype must be CODA_F32, CODA_BF16 or CODA_F16", who);
  const Int8Mat X{(const int8_t*)x, x_sm, x_scales, M}, W{w, w_sm, w_scales, n_feat};
  const int rc = check_mats(X, D, W, K, who);
  if (rc || M == 0) return rc;
  CODA_REQUIRE(out && o_sm >= n_feat, "%s: no output, or its rows shorter than %d features", who, n_feat);
  const hipStream_t st = (hipStream_t)stream;
  const auto run = [&](auto t) {
    typedef decltype(t) T;
    const LinearSink<T> sink{(T*)out, (const T*)bias, o_sm, n_feat};
    if (!x_scales) return launch_of<T>(x, x_sm, M, D, W, K, sink, st, who);
    return few_rows(X, W) ? launch_few(X, W, K, sink, st, who) : launch_many(X, W, K, sink, st, who);
  };
  return dtype == CODA_F32 ? run(float{}) : dtype == CODA_BF16 ? run(bf16_t{}) : run(f16_t{});
}

extern "C" int coda_project_int8(const coda_proj_desc* d, const float* x_scales, const float* w_scales, int64_t w_sm,
                                 int K, const coda_proj_params* p, void* stream) {
  const char* who = "coda_project_int8";
  CODA_REQUIRE(d != nullptr, "%s: null descriptor", who);
  CODA_REQUIRE(d->dtype == CODA_BF16 || d->dtype == CODA_F32, "%s: dtype must be CODA_F32 or CODA_BF16", who);
  CODA_REQUIRE(d->H > 0 && d->Hkv > 0 && d->Dh > 0 && d->Dh % 4 == 0 && d->L > 0 && d->M >= 0,
               "%s: bad sizes M=%d H=%d Hkv=%d Dh=%d L=%d", who, d->M, d->H, d->Hkv, d->Dh, d->L);
  const int n_feat = d->H * d->Dh + 2 * d->Hkv * d->Dh + d->H + (d->gate ? 1 : 0);
  const Int8Mat X{(const int8_t*)d->x, d->x_sm, x_scales, d->M}, W{(const int8_t*)d->w, w_sm, w_scales, n_feat};
  const int rc = check_mats(X, d->D, W, K, who);
  if (rc || d->M == 0) return rc;
  const bool own = p && p->inv_freq;
  CODA_REQUIRE(d->bias && (own || (d->rope_cos && d->rope_sin)) && d->q && d->k && d->v && d->lam && (d->g || !d->gate),
               "%s: pointer missing", who);
  CODA_REQUIRE(((uintptr_t)d->bias % 16) == 0, "%s: bias must be 16-byte aligned", who);
  CODA_REQUIRE(d->q_sm % 4 == 0 && d->k_sm % 4 == 0 && d->v_sm % 4 == 0 && ((uintptr_t)d->q % 8) == 0 &&
                   ((uintptr_t)d->k % 8) == 0 && ((uintptr_t)d->v % 8) == 0,
               "%s: q / k / v rows must be 8-byte aligned", who);
  FrontTables tab{};
  if (p) {
    const auto angle = [](int t) { return t == CODA_F32 || t == CODA_BF16; };
    CODA_REQUIRE(!own || (p->rope_cos && p->rope_sin && angle(p->inv_dtype) && p->p0 >= 0 && p->p0 + d->L <= 1 << 24),
                 "%s: RoPE tables missing, or positions past 2^24", who);
    CODA_REQUIRE(!p->theta || (p->theta_cos && p->theta_sin && angle(p->theta_dtype)), "%s: theta tables missing", who);
    CODA_REQUIRE(d->M <= kFewRows, "%s: a launch makes the tables of at most %d token rows, not of %d", who, kFewRows,
                 d->M);
    tab = FrontTables{p->inv_freq,   p->inv_dtype, p->p0,        p->rope_cos, p->rope_sin, p->theta,
                      p->theta_dtype, d->H * (d->Dh / 2), p->theta_cos, p->theta_sin};
  }
  const hipStream_t st = (hipStream_t)stream;
  const FastDiv len(d->L);
  const auto run = [&](auto t) {
    typedef decltype(t) T;
    const FrontSink<T, true, 4> few{*d, tab, len, n_feat};
    if (!x_scales) return launch_of<T>(d->x, d->x_sm, d->M, d->D, W, K, few, st, who);
    // (tiles that do not go round in one wait for their tokens' RoPE rows too
    // often: 128 x 8192 x 10305 37.4 us against 33.8; in one of 96 x 64 25.8)
    if (p || few_rows(X, W) ||
        (d->M <= kFewRows && tiles_of(X, W, 64, 64) > device_cus() && !one_round_of_96(X, W, K)))
      return launch_few(X, W, K, few, st, who);
    if constexpr (sizeof(T) == 2)
      if (d->Dh % 8 == 0) return launch_many(X, W, K, FrontSink<T, false, 8>{*d, tab, len, n_feat}, st, who);
    return launch_many(X, W, K, FrontSink<T, false, 4>{*d, tab, len, n_feat}, st, who);
  };
  return d->dtype == CODA_BF16 ? run(bf16_t{}) : run(float{});
}
