// Gated layers: target = act(Wg' x + bg) * (Wu' x + bu), both products, the activation and the product of the two in one kernel,
// and the derivative.  Weights are inputs x units, as an edge's; x is inputs x cases.
//   G = Wg' x + bg,  U = Wu' x + bu,  y = act(G) U
//   dU = dy act(G),  dG = dy U act'(G),  dx = Wg dG + Wu dU,  dWg = x dG',  dWu = x dU',  dbg, dbu: row sums of dG, dU
#include "gated.cuh"
#include "gemm.cuh"

using namespace b200;

extern "C" {
int dot(cudamat* mat1, cudamat* mat2, cudamat* target, float beta, float alpha);
int sum_by_axis(cudamat* mat, cudamat* target, int axis);
}

namespace {

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
constexpr long kTensorWork = 1L << 21;      // multiply-adds of one of the products from which the tensor cores take both
int weights_ok(const cudamat* gate_w, const cudamat* up_w) {
  if (!gate_w->on_device || !up_w->on_device) return ERROR_NOT_ON_DEVICE;
  if (gate_w->is_trans || up_w->is_trans) return ERROR_TRANSPOSED;
  return same_shape(gate_w, up_w) ? 0 : ERROR_INCOMPATIBLE_DIMENSIONS;
}
// Planes of both weights: all three, on 16 bytes.
int planes_ok(const cudamat* w, const cudamat* gate_planes, const cudamat* up_planes, const cudamat* scales) {
  if (!gate_planes || !up_planes || !scales) return ERROR_INCOMPATIBLE_DIMENSIONS;
  if (!gate_planes->on_device || !up_planes->on_device || !scales->on_device) return ERROR_NOT_ON_DEVICE;
  if (gate_planes->is_trans || up_planes->is_trans || scales->is_trans) return ERROR_TRANSPOSED;
  const int lda = aux_rows(w->size[0]), H = w->size[1];
  if (!is(gate_planes, lda, H) || !is(up_planes, lda, H) || !is(scales, 2, H)) return ERROR_INCOMPATIBLE_DIMENSIONS;
  if (!on16(gate_planes->data_device) || !on16(up_planes->data_device)) {
    set_error("planes have to start on 16 bytes");
    return ERROR_UNSUPPORTED;
  }
  return 0;
}

}  // namespace

extern "C" {

int gated_planes(cudamat* gate_w, cudamat* up_w, cudamat* gate_planes, cudamat* up_planes, cudamat* scales) {
  int err = weights_ok(gate_w, up_w);
  if (!err) err = planes_ok(gate_w, gate_planes, up_planes, scales);
  if (err) return err;
  const int V = gate_w->size[0], H = gate_w->size[1];
  if (V == 0 || H == 0) return 0;
  const SplitJob jobs[2] = {{gate_w->data_device, (uint16_t*)gate_planes->data_device, scales->data_device, 2, H},
                            {up_w->data_device, (uint16_t*)up_planes->data_device, scales->data_device + 1, 2, H}};
  return split_columns(jobs, 2, V);
}

int gated_product(cudamat* gate_w, cudamat* up_w, cudamat* mat, cudamat* gate_bias, cudamat* up_bias, int activation,
                  cudamat* gate_planes, cudamat* up_planes, cudamat* scales, cudamat* gate, cudamat* up, cudamat* target) {
  int err = weights_ok(gate_w, up_w);
  if (err) return err;
  if ((gate_planes || up_planes || scales) && (err = planes_ok(gate_w, gate_planes, up_planes, scales))) return err;
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
  // Tensor cores, behind a launch or two that split the operands: where the products are more than those cost.
  const bool large = (long)V * H * N >= kTensorWork;
  if (V > 0 && gemm_path() != 2 && (large || gemm_path() == 1) && tma_available()) {
    const long px = (long)aux_rows(V) * N * 4, pw = gate_planes ? 0 : (long)aux_rows(V) * H * 4;
    const long inv = ((long)(N + 2L * H) * 4 + 255) / 256 * 256;
    CallScratch room(6, (size_t)(px + 2 * pw + inv));
    if (!room.p) return CUDA_ERROR;
    uint16_t* xp = (uint16_t*)((char*)room.p + inv);
    float* x_inv = (float*)room.p;
    GatedForward f;
    f.x = {xp, V, N};
    f.wg = {gate_planes ? (uint16_t*)gate_planes->data_device : xp + px / 2, V, H};
    f.wu = {gate_planes ? (uint16_t*)up_planes->data_device : xp + (px + pw) / 2, V, H};
    float* w_inv = gate_planes ? scales->data_device : x_inv + N;
    const SplitJob jobs[3] = {{mat->data_device, xp, x_inv, 1, N},
                              {gate_w->data_device, (uint16_t*)f.wg.p, w_inv, 2, H},
                              {up_w->data_device, (uint16_t*)f.wu.p, w_inv + 1, 2, H}};
    if ((err = split_columns(jobs, gate_planes ? 1 : 3, V))) return err;
    f.w_inv = w_inv;
    f.x_inv = x_inv;
    f.bg = at(gate_bias);
    f.bu = at(up_bias);
    f.gate = at(gate);
    f.up = at(up);
    f.y = target->data_device;
    f.activation = activation;
    return gated_tc(f);
  }
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
