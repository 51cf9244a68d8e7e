// Rows in 8 bits on gfx950: their making (with or without a norm), and the
// product of two sets of them.
//
// A set of rows is int8 codes in [-127, 127] with one fp32 scale a row, the
// value of a code being code * scale.  A row's codes lie at a 16-byte address
// and are followed by zeros up to a multiple of kPad bytes, so that the
// product runs over whole 128-byte steps and has no ragged end.
#include "front.h"

#include <climits>
#include <type_traits>

namespace coda {

static constexpr int kPad = 128;
// the longest sum of products of int8 that int32 holds: 128 * 128 * K < 2^31
static constexpr int kMaxK = (1 << 17) - kPad;
// elements of the longest row that the making of codes keeps in registers
static constexpr int kMaxRow = 32768;

// ------------------------------------------------------------ making codes
__device__ __forceinline__ double wave_reduce(double v, bool max) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const double o = __shfl_xor(v, d);
    v = max ? fmax(v, o) : v + o;
  }
  return v;
}

// Rows in 8 bits, with p_i = x_i (plain) or p_i = s_i w_i (norm; s = x +
// residual, rounded to T and written):
//   P = max |p|, code_i = rint(127 p_i / P),
//   scale = P / 127, with the norm P / (127 sqrt(mean(s^2) + eps)):
// the norm is the same factor for the whole row, so the codes need not wait
// for it.  p, P, the sum and the quotient are held in 64 bits: a product of
// two floats is exact there, and a quotient that falls on a half is rounded
// to even as the formula says, whatever the order of the sums.  A row that
// holds an infinity or a NaN (its weight's counts too) gets scale NaN and
// codes 0; a row of zeros scale 0.
// TPR threads keep a row in registers (IT runs of VEC elements each) between
// the row's maximum and its codes, so that memory is read once.
template <typename T, bool NORM, bool RES, int VEC, int TPR, int IT>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void codes_kernel(
    const T* __restrict__ x, int64_t x_sm, const T* __restrict__ res, int64_t r_sm, const T* __restrict__ w, int rows,
    int D, float eps, T* __restrict__ sum_out, int64_t s_sm, int8_t* __restrict__ codes, int64_t c_sm,
    float* __restrict__ scales) {
  using E = Elt<T>;
  constexpr int NT = TPR < 256 ? 256 : TPR, RPB = NT / TPR;
  struct alignas(sizeof(T) * VEC) Run { T v[VEC]; };
  const int t = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
  if (TPR == 64 && row >= rows) return;  // (whole waves; else a workgroup is a row)
  const T* xr = x + row * x_sm;
  double p[IT * VEC];
  double ss = 0., top = 0., bad = 0.;
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int at = (i * TPR + t) * VEC;
#pragma unroll
    for (int e = 0; e < VEC; ++e) p[i * VEC + e] = 0.;
    if (at >= D) continue;
    Run a = *reinterpret_cast<const Run*>(xr + at);
    if constexpr (NORM) {
      const Run g = *reinterpret_cast<const Run*>(w + at);
      if constexpr (RES) {
        const Run r = *reinterpret_cast<const Run*>(res + row * r_sm + at);
#pragma unroll
        for (int e = 0; e < VEC; ++e) a.v[e] = E::st(E::ld(a.v[e]) + E::ld(r.v[e]));
        *reinterpret_cast<Run*>(sum_out + row * s_sm + at) = a;
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const double s = (double)E::ld(a.v[e]);
        ss = fma(s, s, ss);
        p[i * VEC + e] = s * (double)E::ld(g.v[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) p[i * VEC + e] = (double)E::ld(a.v[e]);
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      top = fmax(top, fabs(p[i * VEC + e]));
      bad = fma(p[i * VEC + e], 0., bad);  // NaN from an infinity or a NaN
    }
  }
  ss += bad;
  ss = wave_reduce(ss, false);
  top = wave_reduce(top, true);
  if constexpr (TPR > 64) {
    constexpr int NW = TPR / 64;
    __shared__ double red[2][NW];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    if (lane == 0) {
      red[0][wv] = ss;
      red[1][wv] = top;
    }
    __syncthreads();
    ss = red[0][0];
    top = red[1][0];
#pragma unroll
    for (int i = 1; i < NW; ++i) {
      ss += red[0][i];
      top = fmax(top, red[1][i]);
    }
  }
  const bool fine = ss == ss && top > 0.;
  const double r = fine ? 1. / top : 0.;
  if (t == 0) {
    double sc = top / 127.;
    if constexpr (NORM) sc /= sqrt(ss / (double)D + (double)eps);
    scales[row] = ss != ss ? __builtin_nanf("") : top > 0. ? (float)sc : 0.f;
  }
  int8_t* cr = codes + row * c_sm;
  // (the row's tail: zeros up to a whole 128 bytes)
  const int padded = (D + kPad - 1) / kPad * kPad;
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int at = (i * TPR + t) * VEC;
    if (at >= padded) continue;
    int8_t c[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      // 127 p / P to the last bit: the quotient by the reciprocal, then its
      // remainder's share
      const double n = p[i * VEC + e] * 127., q0 = n * r, q = fma(fma(-q0, top, n), r, q0);
      c[e] = fine ? (int8_t)(int)rint(q) : (int8_t)0;
    }
    if constexpr (VEC == 8) {
      uint2 v;
      __builtin_memcpy(&v, c, 8);
      *reinterpret_cast<uint2*>(cr + at) = v;
    } else {
      cr[at] = c[0];
    }
  }
}

template <typename T, bool NORM, bool RES, int VEC, int TPR, int IT>
static int launch_codes(const T* x, int64_t x_sm, const T* res, int64_t r_sm, const T* w, int rows, int D, float eps,
                        T* sum_out, int64_t s_sm, int8_t* codes, int64_t c_sm, float* scales, hipStream_t st) {
  constexpr int NT = TPR < 256 ? 256 : TPR, RPB = NT / TPR;
  hipLaunchKernelGGL((codes_kernel<T, NORM, RES, VEC, TPR, IT>), dim3((unsigned)(((int64_t)rows + RPB - 1) / RPB)),
                     dim3(NT), 0, st, x, x_sm, res, r_sm, w, rows, D, eps, sum_out, s_sm, codes, c_sm, scales);
  return check_launch("codes_kernel");
}

// threads and runs of a row of D elements (up to a multiple of 128)
template <typename T, bool NORM, bool RES>
static int run_codes(const void* x_, int64_t x_sm, const void* res_, int64_t r_sm, const void* w_, int rows, int D,
                     float eps, void* sum_, int64_t s_sm, int8_t* codes, int64_t c_sm, float* scales, hipStream_t st) {
  const T *x = (const T*)x_, *res = (const T*)res_, *w = (const T*)w_;
  T* so = (T*)sum_;
  const int P = (D + kPad - 1) / kPad * kPad;
  constexpr uintptr_t run = 8 * sizeof(T);
  bool vec = D % 8 == 0 && x_sm % 8 == 0 && (uintptr_t)x % run == 0;
  if (NORM) vec = vec && (uintptr_t)w % run == 0;
  if (RES) vec = vec && r_sm % 8 == 0 && s_sm % 8 == 0 && (uintptr_t)res % run == 0 && (uintptr_t)so % run == 0;
#define CODES(V, TPR, IT) \
  return launch_codes<T, NORM, RES, V, TPR, IT>(x, x_sm, res, r_sm, w, rows, D, eps, so, s_sm, codes, c_sm, scales, st)
  if (vec) {
    if (P <= 1024) CODES(8, 64, 2);
    if (P <= 2048) CODES(8, 256, 1);
    if (P <= 4096) CODES(8, 256, 2);
    if (P <= 8192) CODES(8, 512, 2);
    CODES(8, 1024, 4);
  }
  if (P <= 1024) CODES(1, 64, 16);
  if (P <= 8192) CODES(1, 512, 16);
  CODES(1, 1024, 32);
#undef CODES
}

// values of codes: out = code * scale, one rounding
template <typename T>
__global__ __launch_bounds__(256) void values_kernel(const int8_t* __restrict__ codes, int64_t c_sm,
                                                     const float* __restrict__ scales, int D, T* __restrict__ out,
                                                     int64_t o_sm) {
  const int64_t row = blockIdx.x;
  const float sc = scales[row];
  for (int i = threadIdx.x; i < D; i += 256) out[row * o_sm + i] = Elt<T>::st((float)codes[row * c_sm + i] * sc);
}

// ------------------------------------------------------------ product
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));

// Epilogue of a plain product: out = value + bias, one rounding
template <typename T>
struct Int8Out {
  T* out;
  const T* bias;  // or null
  int64_t o_sm;
  int n_feat;
  __device__ __forceinline__ void operator()(const int&, int f, int m, pf32x4 v) const {
    T* row = out + (int64_t)m * o_sm;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (f + e < n_feat) row[f + e] = Elt<T>::st(bias ? v[e] + Elt<T>::ld(bias[f + e]) : v[e]);
  }
};

struct Int8Mat {
  const int8_t* p;
  int64_t sm;  // bytes
  const float* scales;
  int rows;
};

// y[m, f] = (sum_k x[m, k] w[f, k]) sx[m] sw[f], the sum exact in int32, then
// the epilogue.  A workgroup of 4 waves makes 64 features x 64 tokens, a wave
// 16 x 64; the MFMA's rows are the features, so a lane holds four consecutive
// ones of a token.
template <typename Epi>
__global__ __launch_bounds__(256) void int8_tile64(const Int8Mat X, const Int8Mat W, int K, int ntf, const Epi epi) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, r16 = lane & 15, kq = lane >> 4;
  const int f0 = (blockIdx.x % ntf) * 64 + 16 * wv, m0 = (int)(blockIdx.x / ntf) * 64;
  const int8_t* wr = W.p + (int64_t)min(f0 + r16, W.rows - 1) * W.sm + 16 * kq;
  const int8_t* xr[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) xr[j] = X.p + (int64_t)min(m0 + 16 * j + r16, X.rows - 1) * X.sm + 16 * kq;
  i32x4 acc[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) acc[j] = i32x4{0, 0, 0, 0};
  for (int k = 0; k < K; k += 64) {
    const i32x4 a = *reinterpret_cast<const i32x4*>(wr + k);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, *reinterpret_cast<const i32x4*>(xr[j] + k), acc[j], 0, 0, 0);
  }
  const int f = f0 + 4 * kq;
  if (f >= W.rows) return;
  float sw[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) sw[e] = W.scales[min(f + e, W.rows - 1)];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int m = m0 + 16 * j + r16;
    if (m >= X.rows) continue;
    const float sx = X.scales[m];
    pf32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (float)acc[j][e] * sx * sw[e];
    epi(0, f, m, v);
  }
}

template <typename Epi>
static int launch_int8(const Int8Mat& X, const Int8Mat& W, int K, const Epi& epi, hipStream_t st) {
  const int ntf = (W.rows + 63) / 64;
  const int64_t n = (int64_t)ntf * ((X.rows + 63) / 64);
  if (n > INT_MAX) return fail(CODA_EUNSUP, "int8 product: %lld tiles", (long long)n);
  hipLaunchKernelGGL((int8_tile64<Epi>), dim3((unsigned)n), dim3(256), 0, st, X, W, K, ntf, epi);
  return check_launch("int8_tile64");
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

// The two operands of a product
static int check_mats(const Int8Mat& X, const Int8Mat& W, int K, const char* who) {
  CODA_REQUIRE(X.rows >= 0 && W.rows > 0 && K > 0 && K % kPad == 0 && K <= kMaxK,
               "%s: bad sizes rows=%d features=%d K=%d (K a multiple of %d, at most %d: int32 holds the sum)", who, X.rows,
               W.rows, K, kPad, kMaxK);
  CODA_REQUIRE(W.p && W.scales && (X.rows == 0 || (X.p && X.scales)), "%s: null pointer", who);
  CODA_REQUIRE((uintptr_t)X.p % 16 == 0 && (uintptr_t)W.p % 16 == 0 && X.sm % 16 == 0 && W.sm % 16 == 0 &&
                   X.sm >= 0 && W.sm >= 0,
               "%s: rows of codes must lie at 16-byte addresses", who);
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
  const hipStream_t st = (hipStream_t)stream;
#define RUN(T)                                                                                                      \
  hipLaunchKernelGGL((values_kernel<T>), dim3((unsigned)rows), dim3(256), 0, st, codes, c_sm, scales, D, (T*)out, o_sm)
  if (dtype == CODA_F32) RUN(float);
  else if (dtype == CODA_BF16) RUN(bf16_t);
  else RUN(f16_t);
#undef RUN
  return check_launch("values_kernel");
}

extern "C" int coda_linear_int8(int dtype, const int8_t* x, int64_t x_sm, const float* x_scales, int M, const int8_t* w,
                                int64_t w_sm, const float* w_scales, int n_feat, int K, const void* bias, void* out,
                                int64_t o_sm, void* stream) {
  const char* who = "coda_linear_int8";
  CODA_REQUIRE(int8_dtype(dtype), "%s: dtype must be CODA_F32, CODA_BF16 or CODA_F16", who);
  const Int8Mat X{x, x_sm, x_scales, M}, W{w, w_sm, w_scales, n_feat};
  const int rc = check_mats(X, W, K, who);
  if (rc || M == 0) return rc;
  CODA_REQUIRE(out && o_sm >= n_feat, "%s: no output, or its rows shorter than %d features", who, n_feat);
  const hipStream_t st = (hipStream_t)stream;
#define RUN(T) launch_int8(X, W, K, Int8Out<T>{(T*)out, (const T*)bias, o_sm, n_feat}, st)
  return dtype == CODA_F32 ? RUN(float) : dtype == CODA_BF16 ? RUN(bf16_t) : RUN(f16_t);
#undef RUN
}

extern "C" int coda_project_int8(const coda_proj_desc* d, const float* x_scales, const float* w_scales, int64_t w_sm,
                                 int K, void* stream) {
  const char* who = "coda_project_int8";
  CODA_REQUIRE(d != nullptr, "%s: null descriptor", who);
  CODA_REQUIRE(d->dtype == CODA_BF16 || d->dtype == CODA_F32, "%s: dtype must be CODA_F32 or CODA_BF16", who);
  CODA_REQUIRE(d->H > 0 && d->Hkv > 0 && d->Dh > 0 && d->Dh % 4 == 0 && d->L > 0 && d->M >= 0,
               "%s: bad sizes M=%d H=%d Hkv=%d Dh=%d L=%d", who, d->M, d->H, d->Hkv, d->Dh, d->L);
  const int n_feat = d->H * d->Dh + 2 * d->Hkv * d->Dh + d->H + (d->gate ? 1 : 0);
  const Int8Mat X{(const int8_t*)d->x, d->x_sm, x_scales, d->M}, W{(const int8_t*)d->w, w_sm, w_scales, n_feat};
  const int rc = check_mats(X, W, K, who);
  if (rc || d->M == 0) return rc;
  CODA_REQUIRE(d->bias && d->rope_cos && d->rope_sin && d->q && d->k && d->v && d->lam && (d->g || !d->gate),
               "%s: pointer missing", who);
  CODA_REQUIRE(((uintptr_t)d->bias % 16) == 0, "%s: bias must be 16-byte aligned", who);
  CODA_REQUIRE(d->q_sm % 4 == 0 && d->k_sm % 4 == 0 && d->v_sm % 4 == 0 && ((uintptr_t)d->q % 8) == 0 &&
                   ((uintptr_t)d->k % 8) == 0 && ((uintptr_t)d->v % 8) == 0,
               "%s: q / k / v rows must be 8-byte aligned", who);
  const hipStream_t st = (hipStream_t)stream;
  return d->dtype == CODA_BF16 ? launch_int8(X, W, K, FrontEpilogue<bf16_t, false>{*d, FrontTables{}}, st)
                               : launch_int8(X, W, K, FrontEpilogue<float, false>{*d, FrontTables{}}, st);
}
