// Products of a gated layer on scaled half-precision planes (gated_tc.cu), as gated.cu calls them.
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
#endif

// A rows x cols matrix as planes, in an aux matrix's layout (common.cuh): column c times 2^e(c), split into two half-precision
// numbers; inv[c * inv_stride] = 2^-e(c).  e puts the column's largest finite magnitude into (2^12, 2^13].
struct Planes {
  const uint16_t* p;
  int rows, cols;
  long bytes() const { return (long)aux_rows(rows) * cols * 4; }
};
struct SplitJob {
  const float* x;
  uint16_t* planes;
  float* inv;
  int inv_stride, cols;
};
// Up to three matrices of the same number of rows, in one launch, which sets nzero words to zero too.
int split_columns(const SplitJob* jobs, int njobs, int rows, uint32_t* zero = nullptr, int nzero = 0);

// y = act(Wg' x + bg) * (Wu' x + bu); w_inv: 2 x H, gate's and up's
struct GatedForward {
  Planes wg, wu, x;
  const float *w_inv, *x_inv, *bg, *bu;
  float *gate, *up, *y;
  int activation;
};
int gated_tc(const GatedForward& f);

// out[:, n] = inv(n) sum over the pairs (a, b) of a . op(b): planes of a as stored (their rows are the output's), of b as stored
// (its columns are the output's, `trans` false, up to two pairs) or transposed (its rows are; one pair, and with a second b a second
// out, for the same a).
struct PlaneProduct {
  int npairs;
  Planes a[2], b[2];
  bool trans;
  int nout;
  float* out[2];
  const float* inv[2];      // of out's columns; stride inv_stride
  int inv_stride;
};
int plane_products(const PlaneProduct* f, int nproducts);      // one or two, in one launch

// gate, up = their gradients dG, dU from dy; with `maxima` the largest |dG| w_inv, |dU| w_inv of each case (token_max) and the largest
// |dG| x_inv, |dU| x_inv of each unit (unit_max, gate's and up's): bits of floats, all zero before.  part: sums of dG and dU over the
// cases of a block, blocks of `cases` x 2 x H, or null.
struct GatedDeriv {
  const float* dy;
  float *gate, *up;
  int H, N, activation;
  const float *w_inv, *x_inv;
  uint32_t *token_max, *unit_max;
  float* part;
  int cases;                // of a block
};
int gated_deriv_cases(int N);
int gated_deriv(const GatedDeriv& d);
// Sums over the blocks of `part` (GatedDeriv): of dG and dU over all cases.
struct BiasSums {
  const float* part;
  int blocks, H;
  float *gate, *up;
};
// dG and dU as planes: with the weights' scales divided out and one of their own a case (by_case: gate's, up's; inverses case_inv),
// and with the inputs' scales divided out and one of their own a unit (by_unit; unit_inv 2 x H).  Either may be null.
struct GradientPlanes {
  const float *gate, *up;
  int H, N;
  const float *w_inv, *x_inv;
  const uint32_t *token_max, *unit_max;
  uint16_t *by_case[2], *by_unit[2];
  float *case_inv, *unit_inv;
  int cases, grid;          // set by the call
  BiasSums biases;          // part not null: summed by the same launch
};
int gradient_planes(const GradientPlanes& g);

}  // namespace b200
