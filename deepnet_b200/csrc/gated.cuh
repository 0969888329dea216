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
// Up to three matrices of the same number of rows, in one launch.
int split_columns(const SplitJob* jobs, int njobs, int rows);

// y = act(Wg' x + bg) * (Wu' x + bu); w_inv: 2 x H, gate's and up's
struct GatedForward {
  Planes wg, wu, x;
  const float *w_inv, *x_inv, *bg, *bu;
  float *gate, *up, *y;
  int activation;
};
int gated_tc(const GatedForward& f);

}  // namespace b200
