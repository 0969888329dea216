// Gated layers: target = act(Wg' x + bg) * (Wu' x + bu), both products, the activation and the product of the two in one kernel,
// and the derivative.  Weights are inputs x units, as an edge's; x is inputs x cases.
//   G = Wg' x + bg,  U = Wu' x + bu,  y = act(G) U
//   dU = dy act(G),  dG = dy U act'(G),  dx = Wg dG + Wu dU,  dWg = x dG',  dWu = x dU',  dbg, dbu: row sums of dG, dU
#include "gated.cuh"
#include "gemm.cuh"

using namespace b200;

extern "C" {
int dot(cudamat* mat1, cudamat* mat2, cudamat* target, float beta, float alpha);
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

// Up to kN cases: every weight is read once, by a warp a unit (kWarps 1) or a block's eight, which both products of a unit share;
// the cases come from L1.  Full fp32 multiply-adds.  Bound by HBM: 8 bytes a weight pair.
constexpr int kFewCases = 8;
template <int kN, int kVec, int kWarps>
__global__ void __launch_bounds__(256) k_gated_few(const GatedArgs a, int activation) {
  __shared__ float red[kWarps > 1 ? kWarps : 1][2 * kN];
  grid_dependents_launch();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const long u = kWarps > 1 ? (long)blockIdx.x : (long)blockIdx.x * 8 + wid;
  if (u >= a.H) return;
  // groups on their way: what the registers of kN cases leave (2048 x 8192, 8 cases: 4 groups 83 us, 1 group 52)
  constexpr int kBatch = kN <= 2 ? (kVec == 4 ? 4 : 8) : kN == 4 ? (kVec == 4 ? 2 : 8) : (kVec == 4 ? 1 : 4);
  const float *wg = a.wg + u * a.V, *wu = a.wu + u * a.V;
  const float* xs[kN];
#pragma unroll
  for (int n = 0; n < kN; n++) xs[n] = a.x + (n < a.N ? (long)n * a.V : 0);
  float sum[2 * kN];
#pragma unroll
  for (int i = 0; i < 2 * kN; i++) sum[i] = 0.0f;
  const int step = 32 * kWarps, items = a.V / kVec;
  for (int base = (kWarps > 1 ? wid * 32 : 0) + lane; base < items; base += kBatch * step) {
    float g[kBatch][kVec], w[kBatch][kVec];
#pragma unroll
    for (int b = 0; b < kBatch; b++) {
      const int i = base + b * step;
      if (i < items) {
        load<kVec>(wg + (long)i * kVec, g[b]);
        load<kVec>(wu + (long)i * kVec, w[b]);
      } else {
#pragma unroll
        for (int j = 0; j < kVec; j++) g[b][j] = w[b][j] = 0.0f;
      }
    }
    // (no branch around a load: cases beyond the last read the first again, a group beyond the last is 0)
#pragma unroll
    for (int b = 0; b < kBatch; b++) {
      const int i = base + b * step;
      float x[kN][kVec];
#pragma unroll
      for (int n = 0; n < kN; n++) {
        if (i < items) {
          load<kVec>(xs[n] + (long)i * kVec, x[n]);
        } else {
#pragma unroll
          for (int j = 0; j < kVec; j++) x[n][j] = 0.0f;
        }
      }
#pragma unroll
      for (int n = 0; n < kN; n++)
#pragma unroll
        for (int j = 0; j < kVec; j++) {
          sum[2 * n] = fmaf(g[b][j], x[n][j], sum[2 * n]);
          sum[2 * n + 1] = fmaf(w[b][j], x[n][j], sum[2 * n + 1]);
        }
    }
  }
#pragma unroll
  for (int i = 0; i < 2 * kN; i++)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], o);
  if (kWarps > 1) {
    if (lane == 0)
#pragma unroll
      for (int i = 0; i < 2 * kN; i++) red[wid][i] = sum[i];
    __syncthreads();
    if (wid) return;
#pragma unroll
    for (int i = 0; i < 2 * kN; i++) {
      sum[i] = red[0][i];
#pragma unroll
      for (int k = 1; k < kWarps; k++) sum[i] += red[k][i];
    }
  }
  float gv = 0.0f, uv = 0.0f;      // lane n finishes case n
#pragma unroll
  for (int n = 0; n < kN; n++)
    if (lane == n) {
      gv = sum[2 * n];
      uv = sum[2 * n + 1];
    }
  if (lane >= kN || lane >= a.N) return;
  if (a.bg) gv += a.bg[u];
  if (a.bu) uv += a.bu[u];
  const long at = (long)lane * a.H + u;
  if (a.gate) {
    a.gate[at] = gv;
    a.up[at] = uv;
  }
  float slope;
  switch (activation) {
    case kLogistic: gv = activate<kLogistic>(gv, slope); break;
    case kRelu: gv = activate<kRelu>(gv, slope); break;
    case kSilu: gv = activate<kSilu>(gv, slope); break;
    case kGelu: gv = activate<kGelu>(gv, slope); break;
  }
  a.y[at] = gv * uv;
}

// ---- the derivative's elementwise part ------------------------------------------------------
// A thread takes kVec units of some cases, one case after another: the units' sums stay in registers.  Bound by HBM: 20 bytes a unit and
// case for the gradients, 12 more for their parts.
constexpr int kMostCases = 64, kDerivThreads = 128;

template <int kAct, int kVec>
__global__ void __launch_bounds__(kDerivThreads) k_gated_deriv(const GatedDeriv a) {
  grid_dependents_launch();
  grid_dependency_wait();
  const int blocks_u = (a.H + kDerivThreads * kVec - 1) / (kDerivThreads * kVec), ub = blockIdx.x % blocks_u, cb = blockIdx.x / blocks_u;
  const int r = (ub * kDerivThreads + threadIdx.x) * kVec;
  if (r >= a.H) return;
  const int c1 = min(a.N, (cb + 1) * a.cases);
  float sg[kVec] = {}, su[kVec] = {};
#pragma unroll 2
  for (int c = cb * a.cases; c < c1; c++) {
    const long at = (long)c * a.H + r;
    float d[kVec], g[kVec], u[kVec];
    load<kVec>(a.dy + at, d);
    load<kVec>(a.gate + at, g);
    load<kVec>(a.up + at, u);
#pragma unroll
    for (int j = 0; j < kVec; j++) {
      float slope;
      const float act = activate<kAct>(g[j], slope);
      g[j] = d[j] * u[j] * slope;
      u[j] = d[j] * act;
      sg[j] += g[j];
      su[j] += u[j];
    }
    store<kVec>(a.gate + at, g);
    store<kVec>(a.up + at, u);
    if (a.parts_g.p) {
      store_parts<kVec>(a.parts_g, r, c, g);
      store_parts<kVec>(a.parts_u, r, c, u);
    }
  }
  if (!a.part) return;
#pragma unroll
  for (int j = 0; j < kVec; j++) {
    a.part[2L * cb * a.H + r + j] = sg[j];
    a.part[(2L * cb + 1) * a.H + r + j] = su[j];
  }
}

// Sums of dG and dU over all cases: the blocks' of `part` (GatedDeriv) in order, 32 values a block, four threads a value.
__global__ void __launch_bounds__(kDerivThreads) k_gated_biases(const float* part, int blocks, int H, float* gate, float* up) {
  __shared__ float red[kDerivThreads / 32][33];
  grid_dependents_launch();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const long v = (long)blockIdx.x * 32 + lane;
  float s = 0.0f;
  if (v < 2L * H) {
#pragma unroll 8
    for (int b = wid; b < blocks; b += kDerivThreads / 32) s += part[2L * b * H + v];
  }
  red[wid][lane] = s;
  __syncthreads();
  if (wid || v >= 2L * H) return;
#pragma unroll
  for (int k = 1; k < kDerivThreads / 32; k++) s += red[k][lane];
  if (v < H) {
    if (gate) gate[v] = s;
  } else if (up) {
    up[v - H] = s;
  }
}

bool on16(const void* p) { return ((uintptr_t)p & 15) == 0; }
int bias_ok(const cudamat* v, int h) {
  if (!v) return 0;
  if (!v->on_device) return ERROR_NOT_ON_DEVICE;
  return numel(v) == h && (v->size[0] == 1 || v->size[1] == 1) ? 0 : ERROR_INCOMPATIBLE_DIMENSIONS;
}
bool is(const cudamat* m, int rows, int cols) { return m->size[0] == rows && m->size[1] == cols; }
constexpr long kTensorWork = 1L << 18;      // multiply-adds of one of the products from which the tensor cores take both
int weights_ok(const cudamat* gate_w, const cudamat* up_w) {
  if (!gate_w->on_device || !up_w->on_device) return ERROR_NOT_ON_DEVICE;
  if (gate_w->is_trans || up_w->is_trans) return ERROR_TRANSPOSED;
  return same_shape(gate_w, up_w) ? 0 : ERROR_INCOMPATIBLE_DIMENSIONS;
}
// Parts of both weights: all three matrices, on 16 bytes.
int planes_ok(const cudamat* w, const cudamat* gate_planes, const cudamat* up_planes, const cudamat* low_planes) {
  const cudamat* const all[3] = {gate_planes, up_planes, low_planes};
  for (const cudamat* m : all)
    if (!m) return ERROR_INCOMPATIBLE_DIMENSIONS;
  for (const cudamat* m : all)
    if (!m->on_device) return ERROR_NOT_ON_DEVICE;
  for (const cudamat* m : all)
    if (m->is_trans) return ERROR_TRANSPOSED;
  for (const cudamat* m : all)
    if (!on16(m->data_device)) {
      set_error("planes have to start on 16 bytes");
      return ERROR_UNSUPPORTED;
    }
  for (const cudamat* m : all)
    if (!is(m, aux_rows(w->size[0]), w->size[1])) return ERROR_INCOMPATIBLE_DIMENSIONS;
  return 0;
}
// Gate's or up's (`which` 1) parts among them.
Planes weight_planes(const cudamat* w, const cudamat* planes, const cudamat* low_planes, int which) {
  const int lda = aux_rows(w->size[0]);
  return {(uint16_t*)planes->data_device, (uint16_t*)low_planes->data_device + which * lda, 2 * lda, w->size[0], w->size[1]};
}

}  // namespace

namespace b200 {
// A block's cases are worked on one after another (0.35 us each).  About 48 blocks of cases.
int gated_deriv_cases(int N) {
  const int cases = (N + 47) / 48;
  return cases > kMostCases ? kMostCases : cases;
}
static long deriv_grid(int H, int N, int cases, bool vec) {
  const int units = kDerivThreads * (vec ? 4 : 1);
  return (long)((N + cases - 1) / cases) * ((H + units - 1) / units);
}
int gated_deriv(const GatedDeriv& d) {
  const bool vec = d.H % 4 == 0 && on16(d.dy) && on16(d.gate) && on16(d.up);
  const long blocks = deriv_grid(d.H, d.N, d.cases, vec);
  if (blocks > 0x7fffffffL) return ERROR_UNSUPPORTED;
#define DERIV(ACT)                                                                                                  \
  case ACT:                                                                                                         \
    if (vec) (void)launch_dependent(k_gated_deriv<ACT, 4>, dim3((unsigned)blocks), dim3(kDerivThreads), 0, stream(), d);       \
    else (void)launch_dependent(k_gated_deriv<ACT, 1>, dim3((unsigned)blocks), dim3(kDerivThreads), 0, stream(), d);           \
    break
  switch (d.activation) { DERIV(kLinear); DERIV(kLogistic); DERIV(kRelu); DERIV(kSilu); DERIV(kGelu); }
#undef DERIV
  return check_launch();
}
}  // namespace b200

extern "C" {

int gated_planes(cudamat* gate_w, cudamat* up_w, cudamat* gate_planes, cudamat* up_planes, cudamat* low_planes) {
  int err = weights_ok(gate_w, up_w);
  if (!err) err = planes_ok(gate_w, gate_planes, up_planes, low_planes);
  if (err) return err;
  const int V = gate_w->size[0], H = gate_w->size[1];
  if (V == 0 || H == 0) return 0;
  if (overlapping({gate_planes, up_planes, low_planes, gate_w, up_w}, 3)) return ERROR_UNSUPPORTED;
  const SplitJob jobs[2] = {{gate_w->data_device, weight_planes(gate_w, gate_planes, low_planes, 0)},
                            {up_w->data_device, weight_planes(up_w, up_planes, low_planes, 1)}};
  return split_columns(jobs, 2, V);
}

int gated_product(cudamat* gate_w, cudamat* up_w, cudamat* mat, cudamat* gate_bias, cudamat* up_bias, int activation,
                  cudamat* gate_planes, cudamat* up_planes, cudamat* low_planes, cudamat* gate, cudamat* up, cudamat* target) {
  int err = weights_ok(gate_w, up_w);
  if (err) return err;
  if ((gate_planes || up_planes || low_planes) && (err = planes_ok(gate_w, gate_planes, up_planes, low_planes))) return err;
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
  if (overlapping({target, gate, up, mat, gate_w, up_w, gate_bias, up_bias, gate_planes, up_planes, low_planes}, 3)) return ERROR_UNSUPPORTED;
  auto at = [](cudamat* m) { return m ? m->data_device : nullptr; };
  // Of large layers the tensor cores read planes faster from five cases on: 2048 x 8192, 8 cases 38 us, 50 without planes (94 with the
  // split before them), 5 cases 38 and 41, 4 cases 38 and 34.
  const bool on_groups = V % 4 == 0 && on16(gate_w->data_device) && on16(up_w->data_device) && on16(mat->data_device);
  const bool planes_first = gate_planes && N > 4 && (long)V * H >= 1L << 22;
  if (N <= kFewCases && gemm_path() == 0 && !planes_first) {
    const GatedArgs a = {gate_w->data_device, up_w->data_device, mat->data_device, at(gate_bias), at(up_bias),
                         at(gate),            at(up),            target->data_device, V, H, N};
    const bool vec = on_groups, block = H < 16L * sm_count() && V >= 512;
    const dim3 grid(block ? H : (H + 7) / 8);
#define FEW(CASES)                                                                                                                \
  do {                                                                                                                            \
    if (vec && block) (void)launch_dependent(k_gated_few<CASES, 4, 8>, grid, dim3(256), 0, stream(), a, activation);               \
    else if (vec) (void)launch_dependent(k_gated_few<CASES, 4, 1>, grid, dim3(256), 0, stream(), a, activation);                   \
    else if (block) (void)launch_dependent(k_gated_few<CASES, 1, 8>, grid, dim3(256), 0, stream(), a, activation);                 \
    else (void)launch_dependent(k_gated_few<CASES, 1, 1>, grid, dim3(256), 0, stream(), a, activation);                            \
  } while (0)
    if (N == 1) FEW(1);
    else if (N == 2) FEW(2);
    else if (N <= 4) FEW(4);
    else FEW(8);
#undef FEW
    return check_launch();
  }
  // Tensor cores, behind a launch or two that split the operands: where the products are more than those cost.
  const bool large = (long)V * H * N >= kTensorWork;
  if (V > 0 && gemm_path() != 2 && (large || gemm_path() == 1) && tma_available()) {
    const size_t px = (planes_bytes(V, N) + 255) / 256 * 256, pw = gate_planes ? 0 : (planes_bytes(V, H) + 255) / 256 * 256;
    CallScratch room(6, px + 2 * pw);
    char* const p = (char*)room.p;
    if (!p) return CUDA_ERROR;
    GatedForward f;
    f.x = planes_at(p, V, N);
    f.wg = gate_planes ? weight_planes(gate_w, gate_planes, low_planes, 0) : planes_at(p + px, V, H);
    f.wu = gate_planes ? weight_planes(up_w, up_planes, low_planes, 1) : planes_at(p + px + pw, V, H);
    const SplitJob jobs[3] = {{mat->data_device, f.x}, {gate_w->data_device, f.wg}, {up_w->data_device, f.wu}};
    if ((err = split_columns(jobs, gate_planes ? 1 : 3, V))) return err;
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
                        cudamat* gate_planes, cudamat* up_planes, cudamat* low_planes, cudamat* grad_mat, cudamat* grad_gate_w, cudamat* grad_up_w, cudamat* grad_gate_bias, cudamat* grad_up_bias) {
  int err = weights_ok(gate_w, up_w);
  if (err) return err;
  if ((gate_planes || up_planes || low_planes) && (err = planes_ok(gate_w, gate_planes, up_planes, low_planes))) return err;
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
  if (overlapping({gate, up, grad_mat, grad_gate_w, grad_up_w, grad_gate_bias, grad_up_bias, deriv, gate_w, up_w, mat, gate_planes, up_planes,
                   low_planes}, 7))
    return ERROR_UNSUPPORTED;
  if (N == 0 || H == 0) {           // sums over no cases, or no units
    for (cudamat* m : {grad_gate_bias, grad_up_bias, grad_gate_w, grad_up_w, grad_mat})
      if (m && numel(m) && cudaMemsetAsync(m->data_device, 0, sizeof(float) * numel(m), stream()) != cudaSuccess)
        return set_error(cudaGetErrorString(cudaGetLastError()));
    return 0;
  }
  const bool biases = grad_gate_bias || grad_up_bias, weights = grad_gate_w || grad_up_w;
  // On parts, or as four products of the matrices themselves (`dot`), which for layers this small take one launch each and no scratch.
  // (Beyond, parts are at least as fast, or 11 % slower where few cases meet large weights: 784 x 500, 100 cases 22 us and 42; 2048 x
  // 8192, 8 cases 154 and 138, 256 cases 238 and 236, 4096 cases 2471 and 2777.  They need nothing that a capture does not allow.)
  const bool large = (long)V * H * N >= 1L << 16;
  const bool tc = V > 0 && (weights || grad_mat) && gemm_path() != 2 && (large || gemm_path() == 1) && tma_available();
  const int cases = gated_deriv_cases(N), blocks = (N + cases - 1) / cases;
  const bool split_w = tc && grad_mat && !gate_planes;
  // scratch, each part on 256 bytes
  size_t room_bytes = 0;
  auto take = [&](bool wanted, size_t bytes) {
    const size_t at = room_bytes;
    if (wanted) room_bytes += (bytes + 255) / 256 * 256;
    return at;
  };
  const size_t at_part = take(biases, sizeof(float) * 2 * (size_t)H * blocks), at_x = take(tc && weights, planes_bytes(V, N));
  const size_t at_wg = take(split_w, planes_bytes(V, H)), at_wu = take(split_w, planes_bytes(V, H));
  const size_t at_g = take(tc, planes_bytes(H, N)), at_u = take(tc, planes_bytes(H, N));
  CallScratch room(6, room_bytes);
  char* const p = (char*)room.p;
  if (room_bytes && !p) return CUDA_ERROR;
  GatedDeriv d = {};
  d.dy = deriv->data_device;
  d.gate = gate->data_device;
  d.up = up->data_device;
  d.H = H;
  d.N = N;
  d.activation = activation;
  d.cases = cases;
  d.part = biases ? (float*)(p + at_part) : nullptr;
  Planes xp = {}, wgp = {}, wup = {};
  if (tc) {
    SplitJob jobs[3];
    int njobs = 0;
    if (weights) jobs[njobs++] = {mat->data_device, xp = planes_at(p + at_x, V, N)};
    if (split_w) {
      jobs[njobs++] = {gate_w->data_device, wgp = planes_at(p + at_wg, V, H)};
      jobs[njobs++] = {up_w->data_device, wup = planes_at(p + at_wu, V, H)};
    } else if (grad_mat) {
      wgp = weight_planes(gate_w, gate_planes, low_planes, 0);
      wup = weight_planes(up_w, up_planes, low_planes, 1);
    }
    if (njobs && (err = split_columns(jobs, njobs, V))) return err;
    d.parts_g = planes_at(p + at_g, H, N);
    d.parts_u = planes_at(p + at_u, H, N);
  }
  if ((err = gated_deriv(d))) return err;
  if (biases) {
    (void)launch_dependent(k_gated_biases, dim3((2 * (unsigned)H + 31) / 32), dim3(kDerivThreads), 0, stream(), d.part, blocks, H,
                           grad_gate_bias ? grad_gate_bias->data_device : nullptr, grad_up_bias ? grad_up_bias->data_device : nullptr);
    if ((err = check_launch())) return err;
  }
  if (!tc) {
    cudamat dg = *gate, du = *up;
    dg.is_trans = du.is_trans = 1;
    dg.owns_data = du.owns_data = 0;
    if (grad_gate_w && V && (err = dot(mat, &dg, grad_gate_w, 0.0f, 1.0f))) return err;
    if (grad_up_w && V && (err = dot(mat, &du, grad_up_w, 0.0f, 1.0f))) return err;
    if (grad_mat && V) {
      if ((err = dot(gate_w, gate, grad_mat, 0.0f, 1.0f))) return err;
      if ((err = dot(up_w, up, grad_mat, 1.0f, 1.0f))) return err;
    }
    return 0;
  }
  PlaneProduct f[2] = {};
  int products = 0;
  if (grad_mat) {
    PlaneProduct& x = f[products++];
    x.npairs = 2;
    x.a[0] = wgp;
    x.a[1] = wup;
    x.b[0] = d.parts_g;
    x.b[1] = d.parts_u;
    x.nout = 1;
    x.out[0] = grad_mat->data_device;
  }
  if (weights) {
    PlaneProduct& w = f[products++];
    w.npairs = 1;
    w.trans = true;
    w.a[0] = xp;
    cudamat* const out[2] = {grad_gate_w, grad_up_w};
    for (int k = 0; k < 2; k++) {
      if (!out[k]) continue;
      w.b[w.nout] = k ? d.parts_u : d.parts_g;
      w.out[w.nout++] = out[k]->data_device;
    }
  }
  return plane_products(f, products, V, H, N);
}

}  // extern "C"
