// Projection front end of the bounded layer on gfx950: one GEMM of the
// token rows against the packed [q | k | v | lambda | write-gate] weights
// (bf16 MFMA, fp32 accumulation), with the epilogues of the reference's
// eager ops fused into the tile's store (attention.py:396-410, 592-608):
//   q, v    (+ bias) rounded to bf16;
//   k       (+ bias) rounded to bf16, then RoPE with the tables of the row's
//           position, one bf16 rounding per op (primitives.py:83-113);
//   lambda  sigmoid(bf16(acc + bias)) in bf16;
//   gate    sigmoid(bf16(acc + bias)) in bf16, stored as float32.
// The tile computes C^T = W X^T: MFMA A operand = weight rows (features), B
// operand = token rows, so each lane holds 4 consecutive features of one
// token (the RoPE pairs of a head sit in one lane; the half-split layout
// is packed with each pair (i, i + Dh/2) on adjacent weight rows).
#include "rows.h"

#include <climits>

namespace coda {

static constexpr int kProjKT = 64;        // D of coda_project: whole multiples

// The layer's own parameters (coda_proj_params) as sections of the packed
// feature order: q, k, v, lambda, gate
template <typename T>
struct ParamRows {
  const T* w[5];
  const T* b[5];
  int64_t sm[5];
  int start[5];  // first feature of a section; INT_MAX: not there
  int Dh;
  int halves;  // k rows of a head in the order (0, half, 1, half + 1, ..): half-split RoPE
  __device__ __forceinline__ int section(int f) const {
    int s = 0;
#pragma unroll
    for (int i = 1; i < 5; ++i) s = f >= start[i] ? i : s;
    return s;
  }
  // a[s], from registers
  template <typename V>
  __device__ __forceinline__ V pick(const V (&a)[5], int s) const {
    V v = a[0];
#pragma unroll
    for (int i = 1; i < 5; ++i) v = s == i ? a[i] : v;
    return v;
  }
  // row of section s that feature f is
  __device__ __forceinline__ int row_in(int s, int f) const {
    int r = f - pick(start, s);
    if (halves && s == 1) {
      const int c = r % Dh;
      r = r - c + (c >> 1) + (c & 1) * (Dh / 2);
    }
    return r;
  }
  // row of feature f0 + r16, at most last; f0, last the same in every lane:
  // in most blocks of 16 the section is too (200 vector instructions before
  // the first load cost 0.4 us)
  __device__ __forceinline__ const T* row16(int f0, int r16, int last) const {
    const int s0 = section(min(f0, last)), f = min(f0 + r16, last);
    if (s0 == section(min(f0 + 15, last))) return pick(w, s0) + row_in(s0, f) * pick(sm, s0);
    const int s = section(f);
    return pick(w, s) + row_in(s, f) * pick(sm, s);
  }
  __device__ __forceinline__ float bias1(int f) const {
    const int s = section(f);
    const T* p = pick(b, s);
    return p ? Elt<T>::ld(p[row_in(s, f)]) : 0.f;
  }
  // biases of features f .. f + 3 (f a multiple of 4; past the last: any)
  __device__ __forceinline__ pf32x4 bias4(int f, int last) const {
    const int s = section(f);
    pf32x4 v{0.f, 0.f, 0.f, 0.f};
    if (s < 3) {
      const T* p = pick(b, s);
      if (!p) return v;
      const int r = row_in(s, f), hs = halves && s == 1 ? Dh / 2 : 0;
      const int o1 = hs ? hs : 1, o2 = hs ? 1 : 2, o3 = hs ? hs + 1 : 3;
      return pf32x4{Elt<T>::ld(p[r]), Elt<T>::ld(p[r + o1]), Elt<T>::ld(p[r + o2]), Elt<T>::ld(p[r + o3])};
    }
    const T* lb = b[3];
    const T* gb = b[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int ff = min(f + e, last);
      const bool gate = ff >= start[4];
      const T* p = gate ? gb : lb;
      if (p) v[e] = Elt<T>::ld(p[ff - (gate ? start[4] : start[3])]);
    }
    return v;
  }
};
// Epilogue of a plain linear layer: out = acc + bias, one rounding
template <typename T, typename BT>
struct LinearEpilogue {
  T* out;
  const BT* bias;  // or null
  int64_t o_sm;
  int n_feat;
  template <typename Src>
  __device__ __forceinline__ void operator()(const Src&, int f, int m, pf32x4 v) const {
    T* row = out + (int64_t)m * o_sm;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += bias && f + e < n_feat ? Elt<BT>::ld(bias[f + e]) : 0.f;
    if (f + 3 < n_feat) {
      proj_put4(row + f, v);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (f + e < n_feat) row[f + e] = Elt<T>::st(v[e]);
    }
  }
  __device__ __forceinline__ void once(int) const {}
};

// one thread per 16-byte piece of the tiled copy; row_pieces: 16-byte pieces
// of a row
__global__ __launch_bounds__(256) void proj_pack_kernel(const char* __restrict__ w, int n_feat, int row_pieces,
                                                        int64_t row_bytes, uint4* __restrict__ out, int64_t n_pieces) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n_pieces) return;
  const int l = (int)(i & 63), r = l & 15, q = l >> 4;
  const int64_t tile = i >> 6;
  const int ksteps = row_pieces / 4;
  const int64_t fb = tile / ksteps;
  const int ks = (int)(tile % ksteps);
  const int64_t f = fb * 16 + r;
  uint4 v = make_uint4(0u, 0u, 0u, 0u);
  if (f < n_feat) v = *reinterpret_cast<const uint4*>(w + f * row_bytes + 64 * ks + 16 * q);
  out[i] = v;
}
static int launch_pack(int esz, const void* w, int n_feat, int D, int64_t w_sm, void* out, hipStream_t st) {
  // (rows padded to a multiple of 64)
  const int row_pieces = D * esz / 16;
  const int64_t n_pieces = (int64_t)((n_feat + 63) / 64) * 64 * row_pieces;
  hipLaunchKernelGGL(proj_pack_kernel, dim3((unsigned)((n_pieces + 255) / 256)), dim3(256), 0, st, (const char*)w, n_feat,
                     row_pieces, w_sm * esz, (uint4*)out, n_pieces);
  return check_launch("proj_pack_kernel");
}

// D of the tiled weights that coda_project_pack makes
static bool rows_path(int D) {
  return D >= 512 && D <= 8192 && D % 256 == 0 && ((D / 256) & (D / 256 - 1)) == 0;
}

// What the front-end entries ask of a descriptor (packed: of its w and bias too)
static int check_project(const coda_proj_desc* d, const char* who, bool packed) {
  CODA_REQUIRE(d->D > 0 && d->D % kProjKT == 0, "%s: D=%d must be a positive multiple of %d", who, d->D, kProjKT);
  CODA_REQUIRE(d->H > 0 && d->Hkv > 0 && d->Dh > 0 && d->Dh % 4 == 0 && d->L > 0,
               "%s: bad sizes H=%d Hkv=%d Dh=%d L=%d", who, d->H, d->Hkv, d->Dh, d->L);
  CODA_REQUIRE(d->x && d->q && d->k && d->v && d->lam && d->g, "%s: pointer missing", who);
  CODA_REQUIRE(!packed || (d->w && d->bias && d->rope_cos && d->rope_sin), "%s: pointer missing", who);
  CODA_REQUIRE(!packed || ((uintptr_t)d->bias % 16) == 0, "%s: bias must be 16-byte aligned", who);
  const int pc = d->dtype == CODA_BF16 ? 8 : 4;  // elements of a 16-byte piece
  CODA_REQUIRE(d->x_sm % pc == 0 && ((uintptr_t)d->x % 16) == 0 && (!packed || ((uintptr_t)d->w % 16) == 0),
               "%s: x / w rows must be 16-byte aligned", who);
  CODA_REQUIRE(d->q_sm % 4 == 0 && d->k_sm % 4 == 0 && d->v_sm % 4 == 0 && ((uintptr_t)d->q % 8) == 0 &&
                   ((uintptr_t)d->k % 8) == 0 && ((uintptr_t)d->v % 8) == 0,
               "%s: q / k / v rows must be 8-byte aligned", who);
  return CODA_OK;
}
static int front_features(const coda_proj_desc* d) {
  return d->H * d->Dh + 2 * d->Hkv * d->Dh + d->H + (d->gate ? 1 : 0);
}
template <typename T>
static int run_project(const coda_proj_desc* d, hipStream_t st, const char* who) {
  const FrontEpilogue<T, false> epi{*d, FrontTables{}};
  const T *w = (const T*)d->w, *x = (const T*)d->x;
  const int n = front_features(d);
  return d->w_layout ? launch_rows<T>(TileRows<T>{w}, n, d->D, x, d->x_sm, d->M, epi, st, who)
                     : launch_rows<T>(MatRows<T>{w, d->D}, n, d->D, x, d->x_sm, d->M, epi, st, who);
}
template <typename T>
static ParamRows<T> param_rows(const coda_proj_desc* d, const coda_proj_params* p) {
  ParamRows<T> r;
  const int sizes[5] = {d->H * d->Dh, d->Hkv * d->Dh, d->Hkv * d->Dh, d->H, d->gate ? 1 : 0};
  int f = 0;
  for (int i = 0; i < 5; ++i) {
    r.w[i] = (const T*)p->w[i];
    r.b[i] = (const T*)p->b[i];
    r.sm[i] = p->w_sm[i];
    r.start[i] = sizes[i] ? f : INT_MAX;
    f += sizes[i];
  }
  r.Dh = d->Dh;
  r.halves = !d->rope_interleaved;
  return r;
}
template <typename T>
static int run_project_params(const coda_proj_desc* d, const coda_proj_params* p, hipStream_t st, const char* who) {
  const ParamRows<T> r = param_rows<T>(d, p);
  const FrontTables t{p->inv_freq,  p->inv_dtype, p->p0,        p->rope_cos, p->rope_sin,
                      p->theta, p->theta_dtype, d->H * (d->Dh / 2), p->theta_cos, p->theta_sin};
  return launch_rows<T>(r, front_features(d), d->D, (const T*)d->x, d->x_sm, d->M, FrontEpilogue<T, true>{*d, t}, st,
                        who);
}
// The packed form of a layer's parameters, tiles and fp32 biases, in one
// launch: one thread per 16-byte piece of the tiles (a concatenation and its
// packing moved the weights twice and took a dozen launches of a layer's
// first token)
template <typename T>
__global__ __launch_bounds__(256) void proj_pack_params_kernel(const ParamRows<T> W, int n_feat, int row_pieces,
                                                               uint4* __restrict__ out, int64_t n_pieces,
                                                               float* __restrict__ bias) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < (n_feat + 3) / 4 * 4) bias[i] = i < n_feat ? W.bias1((int)i) : 0.f;
  if (i >= n_pieces) return;
  const int l = (int)(i & 63), ksteps = row_pieces / 4;
  const int64_t tile = i >> 6, fb = tile / ksteps;
  const int ks = (int)(tile % ksteps);
  pu32x4 v{0u, 0u, 0u, 0u};
  if (fb * 16 + (l & 15) < n_feat)
    v = *reinterpret_cast<const pu32x4u*>((const char*)W.row16((int)fb * 16, l & 15, n_feat - 1) + 64 * ks + 16 * (l >> 4));
  out[i] = make_uint4(v[0], v[1], v[2], v[3]);
}
template <typename T>
static int run_pack_params(const coda_proj_desc* d, const coda_proj_params* p, void* out, float* bias, hipStream_t st) {
  const int n = front_features(d), row_pieces = d->D * (int)sizeof(T) / 16;
  const int64_t n_pieces = (int64_t)((n + 63) / 64) * 64 * row_pieces;
  hipLaunchKernelGGL(proj_pack_params_kernel<T>, dim3((unsigned)((n_pieces + 255) / 256)), dim3(256), 0, st,
                     param_rows<T>(d, p), n, row_pieces, (uint4*)out, n_pieces, bias);
  return check_launch("proj_pack_params_kernel");
}

}  // namespace coda

using namespace coda;

extern "C" int coda_project(const coda_proj_desc* d, void* stream) {
  CODA_REQUIRE(d != nullptr, "coda_project: null descriptor");
  CODA_REQUIRE(d->dtype == CODA_BF16, "coda_project: bf16 only");
  CODA_REQUIRE(d->M >= 0 && d->M <= 64, "coda_project: %d token rows; the front end serves decode-shaped inputs "
               "(at most 64 rows), many rows are library GEMMs", d->M);
  const int rc = check_project(d, "coda_project", true);
  if (rc) return rc;
  if (d->M == 0) return CODA_OK;
  CODA_REQUIRE(d->w_layout == 0 || (d->w_layout == 1 && rows_path(d->D)),
               "coda_project: weight layout %d with D=%d (tiles serve the row kernel's D only)", d->w_layout, d->D);
  return run_project<bf16_t>(d, (hipStream_t)stream, "coda_project");
}

extern "C" int coda_project_rows(const coda_proj_desc* d, void* stream) {
  CODA_REQUIRE(d != nullptr, "coda_project_rows: null descriptor");
  CODA_REQUIRE(d->dtype == CODA_BF16 || d->dtype == CODA_F32, "coda_project_rows: dtype must be CODA_F32 or CODA_BF16");
  CODA_REQUIRE(d->M >= 0 && d->M <= 128, "coda_project_rows: %d token rows (at most 128)", d->M);
  const int rc = check_project(d, "coda_project_rows", true);
  if (rc) return rc;
  if (d->M == 0) return CODA_OK;
  CODA_REQUIRE(d->w_layout == 0 || d->w_layout == 1, "coda_project_rows: weight layout %d", d->w_layout);
  return d->dtype == CODA_BF16 ? run_project<bf16_t>(d, (hipStream_t)stream, "coda_project_rows")
                               : run_project<float>(d, (hipStream_t)stream, "coda_project_rows");
}

// What both entries on parameters ask of them
static int check_params(const coda_proj_desc* d, const coda_proj_params* p, const char* who) {
  const size_t esz = d->dtype == CODA_BF16 ? 2 : 4;
  for (int i = 0; i < (d->gate ? 5 : 4); ++i) {
    CODA_REQUIRE(p->w[i] && p->w_sm[i] >= d->D, "%s: weight %d missing or its rows shorter than D", who, i);
    CODA_REQUIRE((uintptr_t)p->w[i] % esz == 0 && (uintptr_t)p->b[i] % esz == 0, "%s: weight or bias %d off its type",
                 who, i);
  }
  return CODA_OK;
}

extern "C" int coda_project_pack_params(const coda_proj_desc* d, const coda_proj_params* p, void* out, float* bias,
                                        void* stream) {
  const char* who = "coda_project_pack_params";
  CODA_REQUIRE(d != nullptr && p != nullptr && out && bias, "%s: null pointer", who);
  CODA_REQUIRE(d->dtype == CODA_BF16 || d->dtype == CODA_F32, "%s: dtype must be CODA_F32 or CODA_BF16", who);
  CODA_REQUIRE(d->D > 0 && d->D % kProjKT == 0 && d->H > 0 && d->Hkv > 0 && d->Dh > 0 && d->Dh % 4 == 0,
               "%s: bad sizes D=%d H=%d Hkv=%d Dh=%d", who, d->D, d->H, d->Hkv, d->Dh);
  CODA_REQUIRE((uintptr_t)out % 16 == 0 && (uintptr_t)bias % 16 == 0, "%s: outputs must be 16-byte aligned", who);
  const int rc = check_params(d, p, who);
  if (rc) return rc;
  return d->dtype == CODA_BF16 ? run_pack_params<bf16_t>(d, p, out, bias, (hipStream_t)stream)
                               : run_pack_params<float>(d, p, out, bias, (hipStream_t)stream);
}

extern "C" int coda_project_params(const coda_proj_desc* d, const coda_proj_params* p, void* stream) {
  const char* who = "coda_project_params";
  CODA_REQUIRE(d != nullptr && p != nullptr, "%s: null descriptor", who);
  CODA_REQUIRE(d->dtype == CODA_BF16 || d->dtype == CODA_F32, "%s: dtype must be CODA_F32 or CODA_BF16", who);
  CODA_REQUIRE(d->M >= 0 && d->M <= 128, "%s: %d token rows (at most 128)", who, d->M);
  int rc = check_project(d, who, false);
  if (!rc) rc = check_params(d, p, who);
  if (rc) return rc;
  const auto angle = [](int t) { return t == CODA_F32 || t == CODA_BF16; };
  CODA_REQUIRE(p->inv_freq ? p->rope_cos && p->rope_sin && angle(p->inv_dtype) && p->p0 >= 0 && p->p0 + d->L <= 1 << 24
                           : d->rope_cos && d->rope_sin,
               "%s: RoPE tables missing, or positions past 2^24", who);
  CODA_REQUIRE(!p->theta || (p->theta_cos && p->theta_sin && angle(p->theta_dtype)), "%s: theta tables missing", who);
  if (d->M == 0) return CODA_OK;
  return d->dtype == CODA_BF16 ? run_project_params<bf16_t>(d, p, (hipStream_t)stream, who)
                               : run_project_params<float>(d, p, (hipStream_t)stream, who);
}

static int check_linear(int dtype, const void* x, int64_t x_sm, int M, const void* w, int n_feat, int D, const void* out,
                        int64_t o_sm, const char* who) {
  CODA_REQUIRE(dtype == CODA_BF16 || dtype == CODA_F32, "%s: dtype must be CODA_F32 or CODA_BF16", who);
  CODA_REQUIRE(M >= 0 && M <= 128 && n_feat > 0 && D > 0 && D % kProjKT == 0,
               "%s: bad sizes M=%d n_feat=%d D=%d (at most 128 rows, D a multiple of %d)", who, M, n_feat, D, kProjKT);
  CODA_REQUIRE(x && w && out, "%s: null pointer", who);
  const int pc = dtype == CODA_BF16 ? 8 : 4;
  CODA_REQUIRE(x_sm % pc == 0 && ((uintptr_t)x % 16) == 0, "%s: x / w rows must be 16-byte aligned", who);
  CODA_REQUIRE(o_sm % 4 == 0 && ((uintptr_t)out % 8) == 0, "%s: out rows must be 8-byte aligned", who);
  return CODA_OK;
}
template <typename T, typename BT, typename Src>
static int run_linear(const Src& w, const void* x, int64_t x_sm, int M, int n_feat, int D, const void* bias, void* out,
                      int64_t o_sm, void* stream, const char* who) {
  return launch_rows<T>(w, n_feat, D, (const T*)x, x_sm, M,
                        LinearEpilogue<T, BT>{(T*)out, (const BT*)bias, o_sm, n_feat}, (hipStream_t)stream, who);
}

extern "C" int coda_linear_rows(int dtype, const void* x, int64_t x_sm, int M, const void* w, int n_feat, int D,
                                const float* bias, void* out, int64_t o_sm, void* stream) {
  const char* who = "coda_linear_rows";
  const int rc = check_linear(dtype, x, x_sm, M, w, n_feat, D, out, o_sm, who);
  if (rc) return rc;
  CODA_REQUIRE(((uintptr_t)w % 16) == 0, "%s: x / w rows must be 16-byte aligned", who);
  if (M == 0) return CODA_OK;
  return dtype == CODA_BF16
             ? run_linear<bf16_t, float>(TileRows<bf16_t>{(const bf16_t*)w}, x, x_sm, M, n_feat, D, bias, out, o_sm, stream, who)
             : run_linear<float, float>(TileRows<float>{(const float*)w}, x, x_sm, M, n_feat, D, bias, out, o_sm, stream, who);
}

extern "C" int coda_linear_params(int dtype, const void* x, int64_t x_sm, int M, const void* w, int64_t w_sm, int n_feat,
                                  int D, const void* bias, void* out, int64_t o_sm, void* stream) {
  const char* who = "coda_linear_params";
  const int rc = check_linear(dtype, x, x_sm, M, w, n_feat, D, out, o_sm, who);
  if (rc) return rc;
  const size_t esz = dtype == CODA_BF16 ? 2 : 4;
  CODA_REQUIRE(w_sm >= D && (uintptr_t)w % esz == 0 && (uintptr_t)bias % esz == 0,
               "%s: weight rows shorter than D, or off their type", who);
  if (M == 0) return CODA_OK;
  return dtype == CODA_BF16
             ? run_linear<bf16_t, bf16_t>(MatRows<bf16_t>{(const bf16_t*)w, w_sm}, x, x_sm, M, n_feat, D, bias, out, o_sm, stream, who)
             : run_linear<float, float>(MatRows<float>{(const float*)w, w_sm}, x, x_sm, M, n_feat, D, bias, out, o_sm, stream, who);
}

extern "C" int coda_rows_pack(int dtype, const void* w, int n_feat, int D, int64_t w_sm, void* out, void* stream) {
  CODA_REQUIRE(dtype == CODA_BF16 || dtype == CODA_F32, "coda_rows_pack: dtype must be CODA_F32 or CODA_BF16");
  CODA_REQUIRE(w && out && n_feat > 0 && D > 0 && D % kProjKT == 0 && w_sm >= D, "coda_rows_pack: bad arguments");
  const int esz = dtype == CODA_BF16 ? 2 : 4;
  CODA_REQUIRE(w_sm * esz % 16 == 0 && ((uintptr_t)w % 16) == 0 && ((uintptr_t)out % 16) == 0,
               "coda_rows_pack: rows must be 16-byte aligned");
  return launch_pack(esz, w, n_feat, D, w_sm, out, (hipStream_t)stream);
}

extern "C" int coda_project_pack(const void* w, int n_feat, int D, int64_t w_sm, void* out, void* stream) {
  CODA_REQUIRE(w && out && n_feat > 0 && D > 0 && w_sm >= D, "coda_project_pack: bad arguments");
  if (!rows_path(D)) return fail(CODA_EUNSUP, "coda_project_pack: D=%d does not take the tiled weights", D);
  CODA_REQUIRE(w_sm % 8 == 0 && ((uintptr_t)w % 16) == 0 && ((uintptr_t)out % 16) == 0,
               "coda_project_pack: rows must be 16-byte aligned");
  return launch_pack(2, w, n_feat, D, w_sm, out, (hipStream_t)stream);
}

extern "C" int coda_project_workspace_bytes(const coda_proj_desc* d, size_t* bytes) {
  CODA_REQUIRE(d != nullptr && bytes != nullptr, "coda_project_workspace_bytes: null pointer");
  *bytes = 0;
  return CODA_OK;
}
