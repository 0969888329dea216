// Gated layers: target = act(Wg' x + bg) * (Wu' x + bu), both products, the activation and the product of the two in one kernel,
// and the derivative.  Weights are inputs x units, as an edge's; x is inputs x cases.
//   G = Wg' x + bg,  U = Wu' x + bu,  y = act(G) U
//   dU = dy act(G),  dG = dy U act'(G),  dx = Wg dG + Wu dU,  dWg = x dG',  dWu = x dU',  dbg, dbu: row sums of dG, dU
#include <initializer_list>

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

template <int kVec>
__device__ __forceinline__ void load(const float* p, float (&v)[kVec]) {
  if constexpr (kVec == 4) {
    const float4 x = *reinterpret_cast<const float4*>(p);
    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
  } else {
    v[0] = *p;
  }
}
template <int kVec>
__device__ __forceinline__ void store(float* p, const float (&v)[kVec]) {
  if constexpr (kVec == 4) *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  else *p = v[0];
}
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
// A thread takes kVec units of some cases, one case after another: the units' sums and maxima stay in registers.  Bound by HBM:
// 20 bytes a unit and case for the gradients, 8 + 16 for their planes.
constexpr int kMostCases = 64, kDerivThreads = 128;

__device__ __forceinline__ uint32_t magnitude(float v) {      // bits of finite magnitudes, in their order
  const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}

template <int kAct, int kVec>
__global__ void __launch_bounds__(kDerivThreads) k_gated_deriv(const GatedDeriv a) {
  grid_dependents_launch();
  grid_dependency_wait();
  const int blocks_u = (a.H + kDerivThreads * kVec - 1) / (kDerivThreads * kVec), ub = blockIdx.x % blocks_u, cb = blockIdx.x / blocks_u;
  const int r = (ub * kDerivThreads + threadIdx.x) * kVec;
  const bool in = r < a.H;
  const int c1 = min(a.N, (cb + 1) * a.cases);
  float sg[kVec] = {}, su[kVec] = {}, wg[kVec], wu[kVec];
  uint32_t mg[kVec] = {}, mu[kVec] = {};
#pragma unroll
  for (int j = 0; j < kVec; j++) {
    wg[j] = in && a.w_inv ? a.w_inv[2L * (r + j)] : 0.0f;
    wu[j] = in && a.w_inv ? a.w_inv[2L * (r + j) + 1] : 0.0f;
  }
#pragma unroll 2
  for (int c = cb * a.cases; c < c1; c++) {
    const long at = (long)c * a.H + r;
    float d[kVec] = {}, g[kVec] = {}, u[kVec] = {};
    if (in) {
      load<kVec>(a.dy + at, d);
      load<kVec>(a.gate + at, g);
      load<kVec>(a.up + at, u);
    }
#pragma unroll
    for (int j = 0; j < kVec; j++) {
      float slope;
      const float act = activate<kAct>(g[j], slope);
      g[j] = d[j] * u[j] * slope;
      u[j] = d[j] * act;
      sg[j] += g[j];
      su[j] += u[j];
    }
    if (in) {
      store<kVec>(a.gate + at, g);
      store<kVec>(a.up + at, u);
    }
    if (a.token_max) {
      const float xi = a.x_inv[c];
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < kVec; j++) {
        m = max(m, max(magnitude(g[j] * wg[j]), magnitude(u[j] * wu[j])));
        mg[j] = max(mg[j], magnitude(g[j] * xi));
        mu[j] = max(mu[j], magnitude(u[j] * xi));
      }
      m = __reduce_max_sync(0xffffffffu, m);
      if ((threadIdx.x & 31) == 0 && m) atomicMax(a.token_max + c, m);
    }
  }
  if (!in) return;
  // Maxima, which are the same in any order.  Most blocks come too late to raise one: a look first, at all of them at once.
  uint32_t seen[2 * kVec];
#pragma unroll
  for (int j = 0; j < 2 * kVec; j++) seen[j] = a.token_max ? __ldcg(a.unit_max + 2L * r + j) : 0u;
#pragma unroll
  for (int j = 0; j < kVec; j++) {
    if (a.part) {
      a.part[2L * cb * a.H + r + j] = sg[j];
      a.part[(2L * cb + 1) * a.H + r + j] = su[j];
    }
    if (a.token_max) {
      if (mg[j] > seen[2 * j]) atomicMax(a.unit_max + 2L * (r + j), mg[j]);
      if (mu[j] > seen[2 * j + 1]) atomicMax(a.unit_max + 2L * (r + j) + 1, mu[j]);
    }
  }
}

// The blocks' sums, in order: 32 values a block, four threads a value.
__device__ __forceinline__ void sum_biases(const BiasSums& a, int block) {
  __shared__ float red[kDerivThreads / 32][33];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const long v = (long)block * 32 + lane;
  float s = 0.0f;
  if (v < 2L * a.H) {
#pragma unroll 8
    for (int b = wid; b < a.blocks; b += kDerivThreads / 32) s += a.part[2L * b * a.H + v];
  }
  red[wid][lane] = s;
  __syncthreads();
  if (wid || v >= 2L * a.H) return;
#pragma unroll
  for (int k = 1; k < kDerivThreads / 32; k++) s += red[k][lane];
  if (v < a.H) {
    if (a.gate) a.gate[v] = s;
  } else if (a.up) {
    a.up[v - a.H] = s;
  }
}
__global__ void __launch_bounds__(kDerivThreads) k_gated_biases(const BiasSums a) {
  grid_dependents_launch();
  grid_dependency_wait();
  sum_biases(a, blockIdx.x);
}

__device__ __forceinline__ float power_of(uint32_t max_bits, float* inv) {
  const int e = (int)f16_exponent(__uint_as_float(max_bits));
  if (inv) *inv = __int_as_float((127 - e) << 23);
  return __int_as_float((127 + e) << 23);
}

template <int kVec>
__global__ void __launch_bounds__(kDerivThreads) k_gradient_planes(const GradientPlanes a) {
  grid_dependents_launch();
  grid_dependency_wait();
  if ((int)blockIdx.x >= a.grid) {           // the biases' sums ride along
    sum_biases(a.biases, blockIdx.x - a.grid);
    return;
  }
  const int blocks_u = (a.H + kDerivThreads * kVec - 1) / (kDerivThreads * kVec), ub = blockIdx.x % blocks_u, cb = blockIdx.x / blocks_u;
  const int r = (ub * kDerivThreads + threadIdx.x) * kVec, lda = aux_rows(a.H);
  if (r >= a.H) return;
  const int c1 = min(a.N, (cb + 1) * a.cases);
  float w[2][kVec], s[2][kVec];
#pragma unroll
  for (int k = 0; k < 2; k++)
#pragma unroll
    for (int j = 0; j < kVec; j++) {
      const long i = 2L * (r + j) + k;
      w[k][j] = a.w_inv[i];
      s[k][j] = power_of(a.unit_max[i], cb == 0 && a.by_unit[0] ? a.unit_inv + i : nullptr);
    }
#pragma unroll 2
  for (int c = cb * a.cases; c < c1; c++) {
    const float xi = a.x_inv[c], sc = power_of(a.token_max[c], r == 0 && a.by_case[0] ? a.case_inv + c : nullptr);
#pragma unroll
    for (int k = 0; k < 2; k++) {
      float v[kVec];
      load<kVec>((k ? a.up : a.gate) + (long)c * a.H + r, v);
      auto write = [&](uint16_t* planes, const float (&f)[kVec], const float (&scale)[kVec]) {
        uint16_t lo[kVec], hi[kVec], *at = planes + (long)c * 2 * lda + r;
#pragma unroll
        for (int j = 0; j < kVec; j++) split_f16(v[j] * f[j], scale[j], lo[j], hi[j]);
        if constexpr (kVec == 4) {
          *reinterpret_cast<ushort4*>(at) = make_ushort4(lo[0], lo[1], lo[2], lo[3]);
          *reinterpret_cast<ushort4*>(at + lda) = make_ushort4(hi[0], hi[1], hi[2], hi[3]);
        } else {
          at[0] = lo[0];
          at[lda] = hi[0];
        }
      };
      float one[kVec];
#pragma unroll
      for (int j = 0; j < kVec; j++) one[j] = sc;
      if (a.by_case[0]) write(a.by_case[k], w[k], one);
#pragma unroll
      for (int j = 0; j < kVec; j++) one[j] = xi;
      if (a.by_unit[0]) write(a.by_unit[k], one, s[k]);
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
constexpr long kTensorWork = 1L << 18;      // multiply-adds of one of the products from which the tensor cores take both
int weights_ok(const cudamat* gate_w, const cudamat* up_w) {
  if (!gate_w->on_device || !up_w->on_device) return ERROR_NOT_ON_DEVICE;
  if (gate_w->is_trans || up_w->is_trans) return ERROR_TRANSPOSED;
  return same_shape(gate_w, up_w) ? 0 : ERROR_INCOMPATIBLE_DIMENSIONS;
}
// Whether something that is written lies over anything else: the first `written` matrices may lie over none.
bool overlapping(std::initializer_list<const cudamat*> mats, int written) {
  for (int i = 0; i < written; i++)
    for (int j = i + 1; j < (int)mats.size(); j++) {
      const cudamat *a = mats.begin()[i], *b = mats.begin()[j];
      if (!a || !b || numel(a) == 0 || numel(b) == 0) continue;
      const uintptr_t x = (uintptr_t)a->data_device, y = (uintptr_t)b->data_device;
      if (x < y + 4 * numel(b) && y < x + 4 * numel(a)) {
        set_error("a result may not lie over another argument");
        return true;
      }
    }
  return false;
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

namespace b200 {
// A block's cases are worked on one after another (0.35 us each), its units' maxima raised at the end: up to 0.09 us for each block
// that raises the same one.  About 48 blocks of cases.
int gated_deriv_cases(int N) {
  const int cases = (N + 47) / 48;
  return cases > kMostCases ? kMostCases : cases;
}
// As many as leave the device eight blocks an SM.
static int planes_cases(int H, int N) {
  const long cases = (long)((H + 511) / 512) * N / (8L * sm_count());
  return cases < 1 ? 1 : cases > kMostCases ? kMostCases : (int)cases;
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
int gradient_planes(const GradientPlanes& planes) {
  GradientPlanes g = planes;
  g.cases = planes_cases(g.H, g.N);
  const bool vec = g.H % 4 == 0 && on16(g.gate) && on16(g.up);
  const long blocks = deriv_grid(g.H, g.N, g.cases, vec);
  const long extra = g.biases.part ? (2L * g.H + 31) / 32 : 0;
  if (blocks + extra > 0x7fffffffL) return ERROR_UNSUPPORTED;
  g.grid = (int)blocks;
  if (vec) (void)launch_dependent(k_gradient_planes<4>, dim3((unsigned)(blocks + extra)), dim3(kDerivThreads), 0, stream(), g);
  else (void)launch_dependent(k_gradient_planes<1>, dim3((unsigned)(blocks + extra)), dim3(kDerivThreads), 0, stream(), g);
  return check_launch();
}
}  // namespace b200

extern "C" {

int gated_planes(cudamat* gate_w, cudamat* up_w, cudamat* gate_planes, cudamat* up_planes, cudamat* scales) {
  int err = weights_ok(gate_w, up_w);
  if (!err) err = planes_ok(gate_w, gate_planes, up_planes, scales);
  if (err) return err;
  const int V = gate_w->size[0], H = gate_w->size[1];
  if (V == 0 || H == 0) return 0;
  if (overlapping({gate_planes, up_planes, scales, gate_w, up_w}, 3)) return ERROR_UNSUPPORTED;
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
  if (overlapping({target, gate, up, mat, gate_w, up_w, gate_bias, up_bias, gate_planes, up_planes, scales}, 3)) return ERROR_UNSUPPORTED;
  auto at = [](cudamat* m) { return m ? m->data_device : nullptr; };
  // Of large layers the tensor cores read planes faster from five cases on: 2048 x 8192, 8 cases 34 us, 52 without planes (83 with the
  // split before them), 4 cases 33 and 35.
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
                        cudamat* gate_planes, cudamat* up_planes, cudamat* scales, cudamat* grad_mat, cudamat* grad_gate_w, cudamat* grad_up_w, cudamat* grad_gate_bias, cudamat* grad_up_bias) {
  int err = weights_ok(gate_w, up_w);
  if (err) return err;
  if ((gate_planes || up_planes || scales) && (err = planes_ok(gate_w, gate_planes, up_planes, scales))) return err;
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
                   scales}, 7))
    return ERROR_UNSUPPORTED;
  if (N == 0 || H == 0) {           // sums over no cases, or no units
    for (cudamat* m : {grad_gate_bias, grad_up_bias, grad_gate_w, grad_up_w, grad_mat})
      if (m && numel(m) && cudaMemsetAsync(m->data_device, 0, sizeof(float) * numel(m), stream()) != cudaSuccess)
        return set_error(cudaGetErrorString(cudaGetLastError()));
    return 0;
  }
  const bool biases = grad_gate_bias || grad_up_bias, weights = grad_gate_w || grad_up_w;
  // On planes, or as four products of the matrices themselves (`dot`), which read large weights faster for few cases but take
  // matrices that TMA cannot address behind copies.  Microseconds, planes / dot: 256 x 256, 32 cases 18 / 28; 784 x 500, 100 cases
  // 27 / 40; 1024 x 1024, 128 cases 34 / 52; 2048 x 8192, 64 cases 167 / 149, 256 cases 209 / 233, 4096 cases 1385 / 2462; 301 x 301,
  // 301 cases 25 / 61; 1357 x 601, 203 cases 31 / 103.
  const bool aligned = V % 4 == 0 && H % 4 == 0 && on16(gate_w->data_device) && on16(up_w->data_device) && on16(mat->data_device) &&
                       on16(gate->data_device) && on16(up->data_device);
  const bool few = aligned && !gate_planes && N < 128 && (long)V * H >= 1L << 22;
  const bool large = (long)V * H * N >= 1L << 16 && !few;
  const bool tc = V > 0 && (weights || grad_mat) && gemm_path() != 2 && (large || gemm_path() == 1) && tma_available();
  const int cases = gated_deriv_cases(N), blocks = (N + cases - 1) / cases;
  const bool split_w = tc && !gate_planes;
  // scratch, each part on 256 bytes
  size_t room_bytes = 0;
  auto take = [&](bool wanted, size_t bytes) {
    const size_t at = room_bytes;
    if (wanted) room_bytes += (bytes + 255) / 256 * 256;
    return at;
  };
  const size_t unit = sizeof(float) * 2 * (size_t)H, each = sizeof(float) * (size_t)N, hn = (size_t)aux_rows(H) * N * 4;
  const size_t at_part = take(biases, unit * blocks), at_tmax = take(tc, each), at_umax = take(tc, unit), after_max = room_bytes;
  const size_t at_xi = take(tc, each), at_wi = take(split_w, unit), at_ci = take(tc, each), at_ui = take(tc, unit);
  const size_t at_x = take(tc, (size_t)aux_rows(V) * N * 4), vh = (size_t)aux_rows(V) * H * 4, at_wg = take(split_w, vh), at_wu = take(split_w, vh);
  const size_t at_cg = take(tc && grad_mat, hn), at_cu = take(tc && grad_mat, hn), at_ug = take(tc && weights, hn), at_uu = take(tc && weights, hn);
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
    d.token_max = (uint32_t*)(p + at_tmax);
    d.unit_max = (uint32_t*)(p + at_umax);
    d.x_inv = (float*)(p + at_xi);
    d.w_inv = split_w ? (float*)(p + at_wi) : scales->data_device;
    xp = {(uint16_t*)(p + at_x), V, N};
    wgp = {split_w ? (uint16_t*)(p + at_wg) : (uint16_t*)gate_planes->data_device, V, H};
    wup = {split_w ? (uint16_t*)(p + at_wu) : (uint16_t*)up_planes->data_device, V, H};
    const SplitJob jobs[3] = {{mat->data_device, (uint16_t*)xp.p, (float*)d.x_inv, 1, N},
                              {gate_w->data_device, (uint16_t*)wgp.p, (float*)d.w_inv, 2, H},
                              {up_w->data_device, (uint16_t*)wup.p, (float*)d.w_inv + 1, 2, H}};
    if ((err = split_columns(jobs, split_w ? 3 : 1, V, d.token_max, (int)((after_max - at_tmax) / 4)))) return err;
  }
  if ((err = gated_deriv(d))) return err;
  const BiasSums sums = {d.part, blocks, H, grad_gate_bias ? grad_gate_bias->data_device : nullptr,
                         grad_up_bias ? grad_up_bias->data_device : nullptr};
  if (biases && !tc) {
    (void)launch_dependent(k_gated_biases, dim3((2 * (unsigned)H + 31) / 32), dim3(kDerivThreads), 0, stream(), sums);
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
  GradientPlanes g = {};
  if (biases) g.biases = sums;
  g.gate = d.gate;
  g.up = d.up;
  g.H = H;
  g.N = N;
  g.w_inv = d.w_inv;
  g.x_inv = d.x_inv;
  g.token_max = d.token_max;
  g.unit_max = d.unit_max;
  g.case_inv = (float*)(p + at_ci);
  g.unit_inv = (float*)(p + at_ui);
  if (grad_mat) {
    g.by_case[0] = (uint16_t*)(p + at_cg);
    g.by_case[1] = (uint16_t*)(p + at_cu);
  }
  if (weights) {
    g.by_unit[0] = (uint16_t*)(p + at_ug);
    g.by_unit[1] = (uint16_t*)(p + at_uu);
  }
  if ((err = gradient_planes(g))) return err;
  PlaneProduct f[2] = {};
  int products = 0;
  if (grad_mat) {
    PlaneProduct& x = f[products++];
    x.npairs = 2;
    x.a[0] = wgp;
    x.a[1] = wup;
    x.b[0] = {g.by_case[0], H, N};
    x.b[1] = {g.by_case[1], H, N};
    x.nout = 1;
    x.out[0] = grad_mat->data_device;
    x.inv[0] = g.case_inv;
    x.inv_stride = 1;
  }
  if (weights) {
    PlaneProduct& w = f[products++];
    w.npairs = 1;
    w.trans = true;
    w.a[0] = xp;
    w.inv_stride = 2;
    cudamat* const out[2] = {grad_gate_w, grad_up_w};
    for (int k = 0; k < 2; k++) {
      if (!out[k]) continue;
      w.b[w.nout] = {g.by_unit[k], H, N};
      w.out[w.nout] = out[k]->data_device;
      w.inv[w.nout++] = g.unit_inv + k;
    }
  }
  return plane_products(f, products);
}

}  // extern "C"
