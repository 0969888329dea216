// Sampling operations of the C ABI (cudamat/cudamat.cu:437-590) on a counter-based
// Philox4x32-10 stream instead of the reference's table of 12288 multiply-with-carry
// generators: no state arrays, any number of threads, and the number drawn for a
// matrix element depends only on (seed, call number, row, global column).
// One thread produces the four columns {4j..4j+3} of one row from one Philox block;
// consecutive threads take consecutive rows, so every store is coalesced.
#include "common.cuh"

using namespace b200;

namespace {

enum RngOp { kUniform = 0, kNormal, kBernoulli, kBernoulliTanh, kGaussianAdd, kPerturbProb, kPerturbEnergy, kDropout };

template <int kOp>
__global__ void __launch_bounds__(256) k_rng(const float* src, float* dst, int h, int w, int col0, PhiloxKey key,
                                             float p0, float p1) {
  grid_dependents_launch();
  grid_dependency_wait();
  // global column blocks covered by this matrix: [col0 >> 2, (col0 + w - 1) >> 2]
  const int blk0 = col0 >> 2;
  const int nblk = ((col0 + w - 1) >> 2) - blk0 + 1;
  const long items = (long)h * nblk;
  for (long it = (long)blockIdx.x * blockDim.x + threadIdx.x; it < items; it += (long)gridDim.x * blockDim.x) {
    const int b = (int)(it / h), r = (int)(it - (long)b * h);
    const uint4 wd = philox4x32_10((uint32_t)r, (uint32_t)(blk0 + b), key);
    float z[4];
    if (kOp == kNormal || kOp == kGaussianAdd) {
      // Box-Muller on word pairs (0,1) and (2,3), as cudamat_kernels.cu:125-143 pairs its draws
      const float u0 = word_to_uniform(wd.x), u1 = word_to_uniform(wd.y);
      const float u2 = word_to_uniform(wd.z), u3 = word_to_uniform(wd.w);
      const float r0 = sqrtf(-2.0f * logf(u0)), r1 = sqrtf(-2.0f * logf(u2));
      const float a0 = 6.283185307179586f * u1, a1 = 6.283185307179586f * u3;
      z[0] = r0 * cosf(a0); z[1] = r0 * sinf(a0); z[2] = r1 * cosf(a1); z[3] = r1 * sinf(a1);
    } else {
      z[0] = word_to_uniform(wd.x); z[1] = word_to_uniform(wd.y);
      z[2] = word_to_uniform(wd.z); z[3] = word_to_uniform(wd.w);
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int c = ((blk0 + b) << 2) + j - col0;  // local column
      if (c < 0 || c >= w) continue;
      const long idx = (long)c * h + r;
      const float u = z[j];
      float out;
      if (kOp == kUniform || kOp == kNormal) out = u;
      else if (kOp == kBernoulli) out = u < src[idx] ? 1.0f : 0.0f;
      else if (kOp == kBernoulliTanh) out = u < (1.0f + src[idx]) * 0.5f ? 1.0f : -1.0f;
      else if (kOp == kGaussianAdd) out = src[idx] + p0 * u;
      else if (kOp == kPerturbProb) out = -src[idx] / logf(u);
      else if (kOp == kPerturbEnergy) out = src[idx] - logf(-logf(u));
      else out = u > p0 ? src[idx] : p1;  // dropout
      dst[idx] = out;
    }
  }
}

template <int kOp>
int launch(rnd_struct* rnd, cudamat* mat, cudamat* target, float p0 = 0, float p1 = 0) {
  if (!mat->on_device || !target->on_device) return ERROR_NOT_ON_DEVICE;
  if (!same_shape(mat, target)) return ERROR_INCOMPATIBLE_DIMENSIONS;
  const PhiloxKey key = make_philox_key(rnd->seed, rnd->calls);
  rnd->calls += 1;
  // A transposed handle shares its parent's storage; numbers are assigned by stored position.
  const int h = mat->size[0], w = mat->size[1];
  if ((long)h * w == 0) return 0;
  const int col0 = rng_col0();
  const long items = (long)h * (((col0 + w - 1) >> 2) - (col0 >> 2) + 1);
  long blocks = (items + 255) / 256;
  if (blocks > (long)sm_count() * 8) blocks = (long)sm_count() * 8;
  (void)launch_dependent(k_rng<kOp>, dim3((unsigned)blocks), dim3(256), 0, stream(), mat->data_device, target->data_device, h, w,
                         col0, key, p0, p1);
  return check_launch();
}

// target = add + (u > p ? mat * scale : 0).  The comparison is made on the random word itself: its uniform grows with it, so
// `last`, the largest word that is dropped, decides as u > p does.  A thread takes kRows rows of four columns.
// Bound by HBM (8 bytes an element, 12 with `add`) with the Philox rounds close behind: they and the mask take about 25
// instructions an element of the 40 or so that fit beside 8 bytes.  4096 x 8192 with `add`, and back: 112 us, 6.0 TB/s.
template <int kRows, bool kAdd>
__global__ void __launch_bounds__(256) k_dropout_scaled(const float* src, const float* add, float* dst, int h, int w, int col0,
                                                        PhiloxKey key, uint32_t last, bool all, float scale) {
  grid_dependents_launch();
  grid_dependency_wait();
  const int groups = h / kRows, blk0 = col0 >> 2;
  const long it = (long)blockIdx.x * blockDim.x + threadIdx.x;
  const int b = (int)(it / groups), r = kRows * (int)(it - (long)b * groups);
  const int c0 = ((blk0 + b) << 2) - col0;         // first local column (below 0, or the last beyond w, at a shard's ends)
  if (c0 >= w) return;
  float x[4][kRows], y[4][kRows];
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const int c = c0 + j;
    if (c < 0 || c >= w) continue;
    const long idx = (long)c * h + r;
    if constexpr (kRows == 4) {
      const float4 v = *reinterpret_cast<const float4*>(src + idx);
      x[j][0] = v.x; x[j][1] = v.y; x[j][2] = v.z; x[j][3] = v.w;
      if (kAdd) {
        const float4 a = *reinterpret_cast<const float4*>(add + idx);
        y[j][0] = a.x; y[j][1] = a.y; y[j][2] = a.z; y[j][3] = a.w;
      }
    } else {
      x[j][0] = src[idx];
      if (kAdd) y[j][0] = add[idx];
    }
  }
#pragma unroll
  for (int i = 0; i < kRows; i++) {
    const uint4 wd = philox4x32_10((uint32_t)(r + i), (uint32_t)(blk0 + b), key);
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const float kept = pick_word(wd, j) > last || all ? x[j][i] * scale : 0.0f;
      y[j][i] = kAdd ? y[j][i] + kept : kept;
    }
  }
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const int c = c0 + j;
    if (c < 0 || c >= w) continue;
    const long idx = (long)c * h + r;
    if constexpr (kRows == 4) *reinterpret_cast<float4*>(dst + idx) = make_float4(y[j][0], y[j][1], y[j][2], y[j][3]);
    else dst[idx] = y[j][0];
  }
}

// The uniform of a word as the device computes it.
float uniform_of(uint32_t word) {
  const volatile float f = (float)word;
  const volatile float g = f + 1.0f;
  return g * 2.3283064365386963e-10f;
}

}  // namespace

extern "C" {

int dropout_scaled(rnd_struct* rnd_state, cudamat* mat, cudamat* add, cudamat* target, float dropprob) {
  if (!mat->on_device || !target->on_device || (add && !add->on_device)) return ERROR_NOT_ON_DEVICE;
  if (mat->is_trans || target->is_trans || (add && add->is_trans)) return ERROR_TRANSPOSED;
  if (!same_shape(mat, target) || (add && !same_shape(mat, add))) return ERROR_INCOMPATIBLE_DIMENSIONS;
  if (!(dropprob >= 0.0f && dropprob <= 1.0f)) {
    set_error("the probability has to lie in 0 .. 1");
    return ERROR_UNSUPPORTED;
  }
  if (overlapping({target, unless_in_place(mat, target), unless_in_place(add, target)}, 1)) return ERROR_UNSUPPORTED;
  const PhiloxKey key = make_philox_key(rnd_state->seed, rnd_state->calls);
  rnd_state->calls += 1;
  const int h = mat->size[0], w = mat->size[1], col0 = rng_col0();
  if ((long)h * w == 0) return 0;
  // largest word whose uniform is not above dropprob (word 0 is above 0 already: then everything is kept)
  uint32_t last = 0;
  const bool all = uniform_of(0) > dropprob;
  for (uint32_t bit = 1u << 31; bit && !all; bit >>= 1)
    if (!(uniform_of(last | bit) > dropprob)) last |= bit;
  const float scale = dropprob < 1.0f ? (float)(1.0 / (1.0 - (double)dropprob)) : 0.0f;
  const float *x = mat->data_device, *a = add ? add->data_device : nullptr;
  float* y = target->data_device;
  const bool vec = h % 4 == 0 && (((uintptr_t)x | (uintptr_t)a | (uintptr_t)y) & 15) == 0;
  const long items = (long)(vec ? h / 4 : h) * (((col0 + (long)w - 1) >> 2) - (col0 >> 2) + 1);
  const dim3 grid((unsigned)((items + 255) / 256));
#define DROP(ROWS, ADD) \
  (void)launch_dependent(k_dropout_scaled<ROWS, ADD>, grid, dim3(256), 0, stream(), x, a, y, h, w, col0, key, last, all, scale)
  if (vec && a) DROP(4, true);
  else if (vec) DROP(4, false);
  else if (a) DROP(1, true);
  else DROP(1, false);
#undef DROP
  return check_launch();
}

}  // extern "C"

extern "C" {

// cudamat/cudamat.cu:437-467.
int fill_with_rand(rnd_struct* rnd_state, cudamat* mat) { return launch<kUniform>(rnd_state, mat, mat); }
int fill_with_randn(rnd_struct* rnd_state, cudamat* mat) { return launch<kNormal>(rnd_state, mat, mat); }
// cudamat/cudamat.cu:469-501: target = (u < mat) ? 1 : 0 (strict, u in (0, 1]).
int sample_bernoulli(rnd_struct* rnd_state, cudamat* mat, cudamat* target) {
  return launch<kBernoulli>(rnd_state, mat, target);
}
int sample_bernoulli_tanh(rnd_struct* rnd_state, cudamat* mat, cudamat* target) {
  return launch<kBernoulliTanh>(rnd_state, mat, target);
}
// cudamat/cudamat.cu:520-536.
int sample_gaussian(rnd_struct* rnd_state, cudamat* mat, cudamat* target, float mult) {
  return launch<kGaussianAdd>(rnd_state, mat, target, mult);
}
// cudamat/cudamat.cu:538-572.
int perturb_energy(rnd_struct* rnd_state, cudamat* mat, cudamat* target) {
  return launch<kPerturbEnergy>(rnd_state, mat, target);
}
int perturb_prob(rnd_struct* rnd_state, cudamat* mat, cudamat* target) {
  return launch<kPerturbProb>(rnd_state, mat, target);
}
// cudamat/cudamat.cu:574-590.
int dropout(rnd_struct* rnd_state, cudamat* mat, float dropprob, float val) {
  return launch<kDropout>(rnd_state, mat, mat, dropprob, val);
}

}  // extern "C"
