// Epilogue of the projection front end: what becomes of four features of
// one token (q / k with RoPE / v / lambda / gate), shared by the kernels of
// proj.hip and int8.hip.
#pragma once

#include "common.h"

namespace coda {

typedef __bf16 pbf16x8_t __attribute__((ext_vector_type(8)));
typedef float pf32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t pu32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float proj_sigmoid(float x) { return 1.f / (1.f + expf(-x)); }

// Four consecutive elements to memory: one 8-byte (bf16) or 16-byte (fp32,
// any 4-byte address) store
typedef float pf4u __attribute__((ext_vector_type(4), aligned(4)));
__device__ __forceinline__ void proj_put4(bf16_t* p, const pf32x4& v) {
  using E = Elt<bf16_t>;
  uint2 w;
  w.x = (uint32_t)E::st(v[0]) | ((uint32_t)E::st(v[1]) << 16);
  w.y = (uint32_t)E::st(v[2]) | ((uint32_t)E::st(v[3]) << 16);
  *reinterpret_cast<uint2*>(p) = w;
}
__device__ __forceinline__ void proj_put4(float* p, const pf32x4& v) { *reinterpret_cast<pf4u*>(p) = v; }

// Angle tables made by the launch itself (pointers null: given in the
// descriptor, or not asked for)
struct FrontTables {
  const void* inv_freq;
  int inv_dtype;
  int64_t p0;
  void* rope_cos;
  void* rope_sin;
  const void* theta;
  int theta_dtype, n_theta;
  void* theta_cos;
  void* theta_sin;
};

// What a launch leaves of its own tables, by 512 threads
template <typename T>
__device__ __forceinline__ void leave_tables(const FrontTables& tab, int L, int half, int t) {
  if (tab.inv_freq)
    for (int i = t; i < L * half; i += 512) {
      const float2 a = rope_angle<T>(tab.inv_freq, tab.inv_dtype, tab.p0 + i / half, i % half);
      ((T*)tab.rope_cos)[i] = Elt<T>::st(a.x);
      ((T*)tab.rope_sin)[i] = Elt<T>::st(a.y);
    }
  if (tab.theta)
    for (int i = t; i < tab.n_theta; i += 512) {
      const float2 a = cos_sin_of<T>(angle_ld(tab.theta, tab.theta_dtype, i), tab.theta_dtype);
      ((T*)tab.theta_cos)[i] = Elt<T>::st(a.x);
      ((T*)tab.theta_sin)[i] = Elt<T>::st(a.y);
    }
}

// Epilogue of features f .. f + 3 (f a multiple of 4) of token row m:
// the fp32 accumulators plus bias, rounded and routed to q / k (RoPE) / v /
// lambda / gate
// PARAMS: biases from the parameters, the launch's own tables; else one
// packed fp32 bias vector (zero where a linear has none) and given tables
template <typename T, bool PARAMS>
struct FrontEpilogue {
  coda_proj_desc d;
  FrontTables tab;
  template <typename Src>
  __device__ __forceinline__ pf32x4 bias4(const Src& W, int f, int last) const {
    if constexpr (PARAMS) {
      return W.bias4(f, last);
    } else {
      if (f + 3 <= last) {
        const float4 v = *reinterpret_cast<const float4*>(d.bias + f);
        return pf32x4{v.x, v.y, v.z, v.w};
      }
      return pf32x4{d.bias[f], d.bias[min(f + 1, last)], d.bias[min(f + 2, last)], d.bias[min(f + 3, last)]};
    }
  }
  template <typename Src>
  __device__ __forceinline__ void operator()(const Src& W, int f, int m, pf32x4 v) const {
    using E = Elt<T>;
    const int Fq = d.H * d.Dh, Fk = d.Hkv * d.Dh, half = d.Dh / 2;
    const int o_k = Fq, o_v = Fq + Fk, o_l = Fq + 2 * Fk, o_g = o_l + d.H;
    v += bias4(W, f, o_g - (d.gate ? 0 : 1));
    if (f + 3 < o_k) {  // q
      proj_put4((T*)d.q + (int64_t)m * d.q_sm + f, v);
    } else if (f >= o_k && f + 3 < o_v) {  // k: two RoPE pairs
      const int kf = f - o_k, hk = kf / d.Dh, c = kf % d.Dh, prow = m % d.L;
      const bool inter = d.rope_interleaved != 0;
      const T* cs = (const T*)d.rope_cos;
      const T* sn = (const T*)d.rope_sin;
      T* krow = (T*)d.k + (int64_t)m * d.k_sm + (int64_t)hk * d.Dh;
      float r[4];
#pragma unroll
      for (int pp = 0; pp < 2; ++pp) {
        const int p = c / 2 + pp;  // pair index
        float cc, ss;
        if constexpr (!PARAMS) {
          cc = E::ld(cs[(int64_t)prow * half + p]);
          ss = E::ld(sn[(int64_t)prow * half + p]);
        } else if (tab.inv_freq) {
          const float2 t = rope_angle<T>(tab.inv_freq, tab.inv_dtype, tab.p0 + prow, p);
          cc = t.x;
          ss = t.y;
        } else {
          cc = E::ld(cs[(int64_t)prow * half + p]);
          ss = E::ld(sn[(int64_t)prow * half + p]);
        }
        rope_pair_t<T>(E::rnd(v[2 * pp]), E::rnd(v[2 * pp + 1]), cc, ss, inter, r[2 * pp], r[2 * pp + 1]);
      }
      if (inter) {
        proj_put4(krow + c, pf32x4{r[0], r[1], r[2], r[3]});
      } else {  // packed pairs (p, p + half): channels c/2, c/2 + 1 and the same + half
        const int p = c / 2;
        krow[p] = E::st(r[0]);
        krow[p + 1] = E::st(r[2]);
        krow[p + half] = E::st(r[1]);
        krow[p + half + 1] = E::st(r[3]);
      }
    } else if (f >= o_v && f + 3 < o_l) {  // v
      proj_put4((T*)d.v + (int64_t)m * d.v_sm + (f - o_v), v);
    } else {  // lambda / write gate, one feature at a time
#pragma unroll
      for (int rr = 0; rr < 4; ++rr) {
        const int ff = f + rr;
        if (ff < o_l || ff >= o_g + (d.gate ? 1 : 0)) continue;
        const float lin = E::rnd(v[rr]);
        const float sg = E::rnd(proj_sigmoid(lin));
        if (ff < o_g) ((T*)d.lam)[(int64_t)m * d.lam_sm + (ff - o_l)] = E::st(sg);
        else d.g[m] = sg;
      }
    }
  }
  // no gate column: the gate is 1; the tables that the launch leaves
  __device__ __forceinline__ void once(int t) const {
    if (!d.gate && t < d.M) d.g[t] = 1.f;
    if constexpr (PARAMS) leave_tables<T>(tab, d.L, d.Dh / 2, t);
  }
};

}  // namespace coda
