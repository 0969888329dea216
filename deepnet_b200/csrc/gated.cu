// Gated layers: target = act(Wg' x + bg) * (Wu' x + bu), both products, the activation and the product of the two in one kernel,
// and the derivative.  Weights are inputs x units, as an edge's; x is inputs x cases.
//   G = Wg' x + bg,  U = Wu' x + bu,  y = act(G) U
//   dU = dy act(G),  dG = dy U act'(G),  dx = Wg dG + Wu dU,  dWg = x dG',  dWu = x dU',  dbg, dbu: row sums of dG, dU
#include "common.cuh"

using namespace b200;

extern "C" {
int dot(cudamat* mat1, cudamat* mat2, cudamat* target, float beta, float alpha);
int sum_by_axis(cudamat* mat, cudamat* target, int axis);
}

namespace {

enum { kLinear = 0, kLogistic, kRelu, kSilu, kGelu, kActivations };

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

struct GatedArgs {
  const float *wg, *wu, *x, *bg, *bu;
  float *gate, *up, *y;
  int V, H, N;
};

// 64 units by 64 cases a block of 256 threads, four by four of both products a thread, full fp32 multiply-adds.
template <int kAct>
__global__ void __launch_bounds__(256) k_gated_simt(const GatedArgs a) {
  constexpr int T = 64, K = 16;
  __shared__ float sg[K][T + 4], su[K][T + 4], sx[K][T + 4];
  grid_dependents_launch();
  grid_dependency_wait();
  const int tiles_u = (a.H + T - 1) / T, u0 = (int)(blockIdx.x % tiles_u) * T, n0 = (int)(blockIdx.x / tiles_u) * T, tu = threadIdx.x & 15, tn = threadIdx.x >> 4;
  float g[4][4] = {}, u[4][4] = {};
  for (int k0 = 0; k0 < a.V; k0 += K) {
    for (int i = threadIdx.x; i < K * T; i += 256) {
      const int k = i % K, r = i / K;
      const bool in = k0 + k < a.V;
      sg[k][r] = in && u0 + r < a.H ? a.wg[(long)(u0 + r) * a.V + k0 + k] : 0.0f;
      su[k][r] = in && u0 + r < a.H ? a.wu[(long)(u0 + r) * a.V + k0 + k] : 0.0f;
      sx[k][r] = in && n0 + r < a.N ? a.x[(long)(n0 + r) * a.V + k0 + k] : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; k++)
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
          g[i][j] = fmaf(sg[k][tu + 16 * i], sx[k][tn + 16 * j], g[i][j]);
          u[i][j] = fmaf(su[k][tu + 16 * i], sx[k][tn + 16 * j], u[i][j]);
        }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int r = u0 + tu + 16 * i, c = n0 + tn + 16 * j;
      if (r >= a.H || c >= a.N) continue;
      const long at = (long)c * a.H + r;
      const float gv = g[i][j] + (a.bg ? a.bg[r] : 0.0f), uv = u[i][j] + (a.bu ? a.bu[r] : 0.0f);
      if (a.gate) {
        a.gate[at] = gv;
        a.up[at] = uv;
      }
      float slope;
      a.y[at] = activate<kAct>(gv, slope) * uv;
    }
}

// gate, up = dG, dU
template <int kAct, bool kVec>
__global__ void __launch_bounds__(256) k_gated_deriv(const float* dy, float* gate, float* up, long n) {
  grid_dependents_launch();
  grid_dependency_wait();
  const long step = (long)gridDim.x * blockDim.x;
  auto one = [](float d, float& g, float& u) {
    float slope;
    const float act = activate<kAct>(g, slope);
    g = d * u * slope;
    u = d * act;
  };
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < (kVec ? n / 4 : n); i += step) {
    if (kVec) {
      const float4 d = reinterpret_cast<const float4*>(dy)[i];
      float4 g = reinterpret_cast<float4*>(gate)[i], u = reinterpret_cast<float4*>(up)[i];
      one(d.x, g.x, u.x);
      one(d.y, g.y, u.y);
      one(d.z, g.z, u.z);
      one(d.w, g.w, u.w);
      reinterpret_cast<float4*>(gate)[i] = g;
      reinterpret_cast<float4*>(up)[i] = u;
    } else {
      one(dy[i], gate[i], up[i]);
    }
  }
}

bool on16(const void* p) { return ((uintptr_t)p & 15) == 0; }
int bias_ok(const cudamat* v, int h) {
  if (!v) return 0;
  if (!v->on_device) return ERROR_NOT_ON_DEVICE;
  return numel(v) == h && (v->size[0] == 1 || v->size[1] == 1) ? 0 : ERROR_INCOMPATIBLE_DIMENSIONS;
}
bool is(const cudamat* m, int rows, int cols) { return m->size[0] == rows && m->size[1] == cols; }
bool is_planes(const cudamat* m, int rows, int cols) { return m->on_device && !m->is_trans && is(m, aux_rows(rows), cols); }
int weights_ok(const cudamat* gate_w, const cudamat* up_w) {
  if (!gate_w->on_device || !up_w->on_device) return ERROR_NOT_ON_DEVICE;
  if (gate_w->is_trans || up_w->is_trans) return ERROR_TRANSPOSED;
  return same_shape(gate_w, up_w) ? 0 : ERROR_INCOMPATIBLE_DIMENSIONS;
}

}  // namespace

extern "C" {

int gated_product(cudamat* gate_w, cudamat* up_w, cudamat* mat, cudamat* gate_bias, cudamat* up_bias, int activation, cudamat* gate,
                  cudamat* up, cudamat* target) {
  int err = weights_ok(gate_w, up_w);
  if (err) return err;
  if (!mat->on_device || !target->on_device || (gate && !gate->on_device) || (up && !up->on_device)) return ERROR_NOT_ON_DEVICE;
  if (mat->is_trans || target->is_trans || (gate && gate->is_trans) || (up && up->is_trans)) return ERROR_TRANSPOSED;
  const int V = gate_w->size[0], H = gate_w->size[1], N = mat->size[1];
  if (mat->size[0] != V || !is(target, H, N) || !gate != !up || (gate && (!is(gate, H, N) || !is(up, H, N))))
    return ERROR_INCOMPATIBLE_DIMENSIONS;
  if ((err = bias_ok(gate_bias, H)) || (err = bias_ok(up_bias, H))) return err;
  if (activation < 0 || activation >= kActivations) {
    set_error("no such activation");
    return ERROR_UNSUPPORTED;
  }
  if (H == 0 || N == 0) return 0;
  auto at = [](cudamat* m) { return m ? m->data_device : nullptr; };
  const GatedArgs a = {gate_w->data_device, up_w->data_device, mat->data_device, at(gate_bias), at(up_bias),
                       at(gate),            at(up),            target->data_device, V, H, N};
  const long tiles = (long)((H + 63) / 64) * ((N + 63) / 64);
  if (tiles > 0x7fffffffL) return ERROR_UNSUPPORTED;
  const dim3 grid((unsigned)tiles);
#define SIMT(ACT) case ACT: (void)launch_dependent(k_gated_simt<ACT>, grid, dim3(256), 0, stream(), a); break
  switch (activation) { SIMT(kLinear); SIMT(kLogistic); SIMT(kRelu); SIMT(kSilu); SIMT(kGelu); }
#undef SIMT
  return check_launch();
}

int gated_product_deriv(cudamat* deriv, cudamat* gate, cudamat* up, cudamat* gate_w, cudamat* up_w, cudamat* mat, int activation,
                        cudamat* grad_mat, cudamat* grad_gate_w, cudamat* grad_up_w, cudamat* grad_gate_bias, cudamat* grad_up_bias) {
  int err = weights_ok(gate_w, up_w);
  if (err) return err;
  const int V = gate_w->size[0], H = gate_w->size[1], N = mat->size[1];
  struct { cudamat* m; int rows, cols; } want[] = {{deriv, H, N}, {gate, H, N}, {up, H, N}, {mat, V, N}, {grad_mat, V, N},
                                                   {grad_gate_w, V, H}, {grad_up_w, V, H}};
  for (auto& w : want) {
    if (!w.m) continue;
    if (!w.m->on_device) return ERROR_NOT_ON_DEVICE;
    if (w.m->is_trans) return ERROR_TRANSPOSED;
    if (!is(w.m, w.rows, w.cols)) return ERROR_INCOMPATIBLE_DIMENSIONS;
  }
  if ((err = bias_ok(grad_gate_bias, H)) || (err = bias_ok(grad_up_bias, H))) return err;
  if (activation < 0 || activation >= kActivations) {
    set_error("no such activation");
    return ERROR_UNSUPPORTED;
  }
  const long n = (long)H * N;
  if (N == 0 && H > 0) {            // sums over no cases
    for (cudamat* m : {grad_gate_bias, grad_up_bias})
      if (m && cudaMemsetAsync(m->data_device, 0, sizeof(float) * H, stream()) != cudaSuccess)
        return set_error(cudaGetErrorString(cudaGetLastError()));
  }
  if (n > 0) {
    const float* dy = deriv->data_device;
    float *g = gate->data_device, *u = up->data_device;
    const bool vec = n % 4 == 0 && on16(dy) && on16(g) && on16(u);
    long blocks = ((vec ? n / 4 : n) + 255) / 256;
    if (blocks > 16L * sm_count()) blocks = 16L * sm_count();
#define DERIV(ACT)                                                                                                               \
  case ACT:                                                                                                                      \
    if (vec) (void)launch_dependent(k_gated_deriv<ACT, true>, dim3((unsigned)blocks), dim3(256), 0, stream(), dy, g, u, n);       \
    else (void)launch_dependent(k_gated_deriv<ACT, false>, dim3((unsigned)blocks), dim3(256), 0, stream(), dy, g, u, n);          \
    break
    switch (activation) { DERIV(kLinear); DERIV(kLogistic); DERIV(kRelu); DERIV(kSilu); DERIV(kGelu); }
#undef DERIV
    if ((err = check_launch())) return err;
  }
  if (grad_gate_bias && n && (err = sum_by_axis(gate, grad_gate_bias, 1))) return err;
  if (grad_up_bias && n && (err = sum_by_axis(up, grad_up_bias, 1))) return err;
  cudamat dg = *gate, du = *up;
  dg.is_trans = du.is_trans = 1;
  dg.owns_data = du.owns_data = 0;
  if (grad_gate_w && (err = dot(mat, &dg, grad_gate_w, 0.0f, 1.0f))) return err;
  if (grad_up_w && (err = dot(mat, &du, grad_up_w, 0.0f, 1.0f))) return err;
  if (grad_mat) {
    if ((err = dot(gate_w, gate, grad_mat, 0.0f, 1.0f))) return err;
    if ((err = dot(up_w, up, grad_mat, 1.0f, 1.0f))) return err;
  }
  return 0;
}

}  // extern "C"
