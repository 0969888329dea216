// Products of a gated layer on bfloat16 parts (gated_tc.cu), as gated.cu calls them.
#pragma once
#include "common.cuh"

namespace b200 {

enum GatedActivation { kLinear = 0, kLogistic, kRelu, kSilu, kGelu, kActivations };

#ifdef __CUDACC__
// act(g) and its slope.
template <int kAct>
__device__ __forceinline__ float activate(float g, float& slope) {
  if (kAct == kLogistic || kAct == kSilu) {
    const float p = sigmoid_accurate(g), q = sigmoid_accurate(-g);     // (1 - p loses what is left of it)
    slope = kAct == kLogistic ? p * q : p * (1.0f + g * q);
    return kAct == kLogistic ? p : g * p;
  }
  if (kAct == kRelu) {
    slope = g > 0.0f ? 1.0f : g == g ? 0.0f : g;                       // (NaN stays)
    return g > 0.0f || g != g ? g : 0.0f;
  }
  if (kAct == kGelu) {
    const float cdf = 0.5f * erfcf(-0.70710678118654752f * g);
    slope = cdf + g * (0.39894228040143268f * expf(-0.5f * g * g));
    return g * cdf;
  }
  slope = 1.0f;
  return g;
}

// kVec consecutive floats (4, 8: the address is on 16 bytes).
template <int kVec>
__device__ __forceinline__ void load(const float* p, float (&v)[kVec]) {
  if constexpr (kVec % 4 == 0) {
#pragma unroll
    for (int j = 0; j < kVec; j += 4) {
      const float4 x = *reinterpret_cast<const float4*>(p + j);
      v[j] = x.x; v[j + 1] = x.y; v[j + 2] = x.z; v[j + 3] = x.w;
    }
  } else {
    v[0] = *p;
  }
}
template <int kVec>
__device__ __forceinline__ void store(float* p, const float (&v)[kVec]) {
  if constexpr (kVec == 4) *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  else *p = v[0];
}

// x = hi + mid + lo, each the bfloat16 (a float's upper half) nearest to what is left, hi the largest finite one at most: 24 bits in
// three times eight, exact from magnitudes of 2^-103 on (below, lo is no normal number).  Infinities and NaN are in hi alone.
__device__ __forceinline__ void split_parts(float x, uint32_t& lo, uint32_t& mid, uint32_t& hi) {
  const uint32_t u = __float_as_uint(x);
  hi = (u + 0x8000u) & 0xffff0000u;
  float rest = x - __uint_as_float(hi);
  if ((u & 0x7fffffffu) >= 0x7f7f8000u) {            // would round to infinity, is infinite, or NaN
    const bool finite = fabsf(x) <= 3.4028234e38f;
    hi = finite || x == x ? u & 0xffff0000u : 0x7fff0000u;
    rest = finite ? x - __uint_as_float(hi) : 0.0f;
  }
  mid = (__float_as_uint(rest) + 0x8000u) & 0xffff0000u;
  lo = __float_as_uint(rest - __uint_as_float(mid));
}
#endif

// A rows x cols matrix as three bfloat16 parts of its elements.  p: mid and hi, in an aux matrix's layout (common.cuh; plane 0, 1);
// low: columns of lo, low_ld apart (a multiple of 8).
struct Planes {
  uint16_t *p, *low;
  int low_ld, rows, cols;
};
inline size_t planes_bytes(int rows, int cols) { return (size_t)aux_rows(rows) * cols * 6; }
inline Planes planes_at(void* at, int rows, int cols) {          // on 16 bytes
  uint16_t* p = (uint16_t*)at;
  return {p, p + (size_t)2 * aux_rows(rows) * cols, aux_rows(rows), rows, cols};
}
struct SplitJob {
  const float* x;
  Planes to;
};
// Up to three matrices of the same number of rows, in one launch.
int split_columns(const SplitJob* jobs, int njobs, int rows);

#ifdef __CUDACC__
// Elements r .. of column c (kVec 4, 8: r is a multiple of it).
template <int kVec>
__device__ __forceinline__ void store_parts(const Planes& to, int r, long c, const float (&v)[kVec]) {
  const int lda = aux_rows(to.rows);
  uint32_t l[kVec], m[kVec], h[kVec];
  uint16_t *at = to.p + c * 2 * lda + r, *low = to.low + c * to.low_ld + r;
#pragma unroll
  for (int j = 0; j < kVec; j++) split_parts(v[j], l[j], m[j], h[j]);
  auto put = [](uint16_t* p, const uint32_t (&x)[kVec]) {
    if constexpr (kVec == 1) {
      *p = (uint16_t)(x[0] >> 16);
    } else {
      uint32_t two[kVec / 2];                          // upper halves, side by side
#pragma unroll
      for (int j = 0; j < kVec; j += 2) two[j / 2] = __byte_perm(x[j], x[j + 1], 0x7632);
      if constexpr (kVec == 8) *reinterpret_cast<uint4*>(p) = make_uint4(two[0], two[1], two[2], two[3]);
      else *reinterpret_cast<uint2*>(p) = make_uint2(two[0], two[1]);
    }
  };
  put(low, l);
  put(at, m);
  put(at + lda, h);
}
#endif

// y = act(Wg' x + bg) * (Wu' x + bu)
struct GatedForward {
  Planes wg, wu, x;
  const float *bg, *bu;
  float *gate, *up, *y;
  int activation;
};
int gated_tc(const GatedForward& f);

// out = sum over the pairs (a, b) of a . op(b): a as stored (its rows are the output's), b as stored (its columns are the output's, `trans`
// false, up to two pairs) or transposed (its rows are; one pair, and with a second b a second out, for the same a).
struct PlaneProduct {
  int npairs;
  Planes a[2], b[2];
  bool trans;
  int nout;
  float* out[2];
};
// One or two in one launch: the inputs' gradient (two pairs) and the weights' (transposed), of a layer of V inputs and H units.
int plane_products(const PlaneProduct* f, int nproducts, int V, int H, int cases);

// gate, up = their gradients dG, dU from dy; with parts_g.p these as parts too.  part: sums of dG and dU over the cases of a block, blocks
// of `cases` x 2 x H, or null.
struct GatedDeriv {
  const float* dy;
  float *gate, *up;
  int H, N, activation;
  Planes parts_g, parts_u;
  float* part;
  int cases;                // of a block
};
int gated_deriv_cases(int N);
int gated_deriv(const GatedDeriv& d);

}  // namespace b200
