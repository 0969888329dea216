// Layer normalisation of columns (one case a column) and its derivative.
//   m = mean(x), r = 1 / sqrt(mean((x - m)^2) + eps), xh = (x - m) r, y = gain xh + bias
//   a = gain dy:  dx = r (a - mean(a) - xh mean(a xh)),  dgain = sum over columns of dy xh,  dbias = sum over columns of dy
// Bound by HBM: 8 bytes an element forward, 12 back.  A column is read once into registers (the variance is that of the centred
// values).  Forward, columns that all start on 16 bytes: by a warp up to 1024 rows, by a block up to 32768 (k_layer_norm); others by a
// warp up to 512, by a block up to 4096 (k_layer_norm_ring), or value by value, where the result lies differently to 16 bytes or a
// column is longer, by a warp up to 256 and by a block up to 8192.  Back by a warp up to 512, by a block up to 8192.  The ring and the derivative have the next columns on
// their way meanwhile.  What is longer, or back lies differently, is read again and again (k_layer_norm_long, k_layer_norm_deriv_long).
// Back, a block walks columns and keeps its share of both parameters' gradients in registers; the blocks' shares are added by
// a second launch in a fixed order, so results do not change from run to run.  4096 x 8192: forward 45 us (6.0 TB/s), back 80
// (5.0 TB/s: one barrier a column at two blocks an SM; instructions issue in 58 % of the cycles, and of the 13.3 cycles a warp takes
// for one it waits 4.4 for loads, 1.8 for shared memory and 1.5 at the barrier).
#include <map>
#include <mutex>
#include <tuple>

#include "common.cuh"

using namespace b200;

namespace {

constexpr int kWarpsPerBlock = 8;        // columns a block works on side by side where a warp holds one

// Sum over the threads of a column: the warp, or with `block` the whole block (red: 32 floats, free again on return
// of the next call but one: the callers alternate between two).
template <bool kBlock>
__device__ __forceinline__ float column_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (kBlock) {
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, nw = blockDim.x >> 5;
    if (lane == 0) red[wid] = v;
    __syncthreads();
    v = lane < nw ? red[lane] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  }
  return v;
}
// Both sums of a pair, with one barrier.
template <bool kBlock>
__device__ __forceinline__ float2 column_sum2(float2 v, float2* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  if (kBlock) {
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, nw = blockDim.x >> 5;
    if (lane == 0) red[wid] = v;
    __syncthreads();
    v = lane < nw ? red[lane] : make_float2(0.0f, 0.0f);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
      v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
  }
  return v;
}

// kVec consecutive floats (4: the address is on 16 bytes).
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

// kPer groups of kVec values a thread; h / kVec <= kPer * threads of a column.
template <int kVec, int kPer, bool kBlock>
__global__ void __launch_bounds__(kBlock ? 1024 : 32 * kWarpsPerBlock)
    k_layer_norm(const float* x, const float* gain, const float* bias, float* y, float* stats, int h, int w, float eps) {
  __shared__ float red[2][32];
  grid_dependents_launch();
  grid_dependency_wait();
  const int threads = kBlock ? blockDim.x : 32, t = kBlock ? threadIdx.x : threadIdx.x & 31;
  const int c = kBlock ? blockIdx.x : blockIdx.x * kWarpsPerBlock + (threadIdx.x >> 5);
  if (c >= w) return;
  const float* col = x + (long)c * h;
  float v[kPer][kVec], s = 0.0f;
#pragma unroll
  for (int i = 0; i < kPer; i++) {
    const int r = kVec * (t + i * threads);
    if (r < h) {
      load<kVec>(col + r, v[i]);
    } else {
#pragma unroll
      for (int j = 0; j < kVec; j++) v[i][j] = 0.0f;
    }
  }
#pragma unroll
  for (int i = 0; i < kPer; i++)
#pragma unroll
    for (int j = 0; j < kVec; j++) s += v[i][j];
  const float m = column_sum<kBlock>(s, red[0]) / h;
  s = 0.0f;
#pragma unroll
  for (int i = 0; i < kPer; i++)
    if (kVec * (t + i * threads) < h) {
#pragma unroll
      for (int j = 0; j < kVec; j++) s += (v[i][j] - m) * (v[i][j] - m);
    }
  const float rs = 1.0f / sqrtf(column_sum<kBlock>(s, red[1]) / h + eps);
  float* out = y + (long)c * h;
#pragma unroll
  for (int i = 0; i < kPer; i++) {
    const int r = kVec * (t + i * threads);
    if (r >= h) continue;
    float g[kVec], b[kVec];
    if (gain) load<kVec>(gain + r, g);
    if (bias) load<kVec>(bias + r, b);
#pragma unroll
    for (int j = 0; j < kVec; j++) {
      float xh = (v[i][j] - m) * rs;
      if (gain) xh *= g[j];
      v[i][j] = bias ? xh + b[j] : xh;
    }
    store<kVec>(out + r, v[i]);
  }
  if (stats && t == 0) {
    stats[2L * c] = m;
    stats[2L * c + 1] = rs;
  }
}

// Columns too long for registers: one block a column, which reads it three times (twice from L2).
__global__ void __launch_bounds__(1024) k_layer_norm_long(const float* x, const float* gain, const float* bias, float* y, float* stats,
                                                          int h, int w, float eps) {
  __shared__ float red[2][32];
  grid_dependents_launch();
  grid_dependency_wait();
  const int c = blockIdx.x;
  const float* col = x + (long)c * h;
  float* out = y + (long)c * h;
  float s = 0.0f;
#pragma unroll 8
  for (int r = threadIdx.x; r < h; r += blockDim.x) s += col[r];
  const float m = column_sum<true>(s, red[0]) / h;
  s = 0.0f;
#pragma unroll 8
  for (int r = threadIdx.x; r < h; r += blockDim.x) s += (col[r] - m) * (col[r] - m);
  const float rs = 1.0f / sqrtf(column_sum<true>(s, red[1]) / h + eps);
#pragma unroll 4
  for (int r = threadIdx.x; r < h; r += blockDim.x) {
    float xh = (col[r] - m) * rs;
    if (gain) xh *= gain[r];
    out[r] = bias ? xh + bias[r] : xh;
  }
  if (stats && threadIdx.x == 0) {
    stats[2L * c] = m;
    stats[2L * c + 1] = rs;
  }
}

// Columns on the move.  A thread holds kPer groups of four values, on 16 bytes whatever the column's length: group q holds rows
// 4 q - o .. of a column that starts o floats behind a 16-byte boundary, and only a column's first and last group may be partial.
// A block's (or warp's) columns lie a multiple of four apart, so that o, and with it a thread's rows, stay the same.  The next
// columns are on their way into shared memory while one is worked on: a thread copies what it will read itself, so its own copies
// are all it waits for.  1357 x 20003, back: 154 us value by value and without, 79 so.
constexpr int kAhead = 2;                 // columns on their way
constexpr int kMostThreads = 512;
constexpr int kMostSmem = (kAhead + 1) * 2 * 4 * kMostThreads * 16;      // of the largest block

template <int kPer, int kSources>
struct Ring {
  float* mem;                             // [stage][source][group][thread of the block][4]
  int all, o, h, t, threads;
  uint32_t at;

  __device__ __forceinline__ Ring(float* shared, int t_, int threads_, int o_, int h_) : all(blockDim.x), o(o_), h(h_), t(t_), threads(threads_) {
    mem = shared + threadIdx.x * 4;
    at = (uint32_t)__cvta_generic_to_shared(mem);
  }
  __device__ __forceinline__ int row(int i) const { return 4 * (t + i * threads) - o; }
  __device__ __forceinline__ bool whole(int r) const { return r >= 0 && r + 4 <= h; }
  __device__ __forceinline__ long slot(int stage, int source, int i) const { return ((long)(stage * kSources + source) * kPer + i) * all * 4; }
  // column: its first value
  __device__ __forceinline__ void fetch(int stage, int source, const float* column) {
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      const int r = row(i);
      const uint32_t to = at + (uint32_t)slot(stage, source, i) * 4u;
      if (whole(r)) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(column + r) : "memory");
      } else if (r < h) {
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (r + j >= 0 && r + j < h)
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to + 4u * j), "l"(column + r + j) : "memory");
      }
    }
  }
  __device__ __forceinline__ void read(int stage, int source, float none, float (&v)[kPer][4]) {
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      const int r = row(i);
      load<4>(mem + slot(stage, source, i), v[i]);
      if (!whole(r))
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (r + j < 0 || r + j >= h) v[i][j] = none;
    }
  }
  __device__ __forceinline__ void write(float* column, const float (&v)[kPer][4]) {
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      const int r = row(i);
      if (whole(r)) {
        store<4>(column + r, v[i]);
      } else if (r < h) {
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (r + j >= 0 && r + j < h) column[r + j] = v[i][j];
      }
    }
  }
  __device__ __forceinline__ void constants(const float* p, float none, float (&v)[kPer][4]) {
#pragma unroll
    for (int i = 0; i < kPer; i++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int r = row(i) + j;
        v[i][j] = p && r >= 0 && r < h ? p[r] : none;
      }
  }
};

template <int kPer, bool kBlock>
__global__ void __launch_bounds__(kBlock ? kMostThreads : 32 * kWarpsPerBlock, 2)
    k_layer_norm_ring(const float* x, const float* gain, const float* bias, float* y, float* stats, int h, int w, float eps, int offset) {
  extern __shared__ __align__(16) float shares[];
  __shared__ float red[2][32];
  grid_dependents_launch();
  grid_dependency_wait();
  const int threads = kBlock ? blockDim.x : 32, t = kBlock ? threadIdx.x : threadIdx.x & 31;
  const int first = kBlock ? blockIdx.x : blockIdx.x * kWarpsPerBlock + (threadIdx.x >> 5);
  const int step = kBlock ? gridDim.x : gridDim.x * kWarpsPerBlock;
  if (first >= w) return;
  Ring<kPer, 1> ring(shares, t, threads, (int)((offset + (long)first * h) & 3), h);
  float g[kPer][4], b[kPer][4];
  ring.constants(gain, 1.0f, g);
  ring.constants(bias, 0.0f, b);
  auto fetch = [&](long c, int stage) {
    if (c < w) ring.fetch(stage, 0, x + c * h);
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int k = 0; k < kAhead; k++) fetch(first + (long)k * step, k);
  int stage = 0;
  for (long c = first; c < w; c += step) {
    fetch(c + (long)kAhead * step, stage > 0 ? stage - 1 : kAhead);      // (stage + kAhead modulo kAhead + 1)
    asm volatile("cp.async.wait_group %0;" ::"n"(kAhead) : "memory");
    float v[kPer][4], s = 0.0f;
    ring.read(stage, 0, 0.0f, v);
    stage = stage == kAhead ? 0 : stage + 1;
#pragma unroll
    for (int i = 0; i < kPer; i++)
#pragma unroll
      for (int j = 0; j < 4; j++) s += v[i][j];
    const float m = column_sum<kBlock>(s, red[0]) / h;
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; i++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int r = ring.row(i) + j;
        const float d = v[i][j] - m;
        s += r >= 0 && r < h ? d * d : 0.0f;
      }
    const float rs = 1.0f / sqrtf(column_sum<kBlock>(s, red[1]) / h + eps);
#pragma unroll
    for (int i = 0; i < kPer; i++)
#pragma unroll
      for (int j = 0; j < 4; j++) v[i][j] = fmaf((v[i][j] - m) * rs, g[i][j], b[i][j]);
    ring.write(y + c * h, v);
    if (stats && t == 0) {
      stats[2 * c] = m;
      stats[2 * c + 1] = rs;
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// Back.  part: blocks x 2 x h, this block's sums of dy xh and of dy (or null: no parameter's gradient is wanted).
template <int kPer, bool kBlock>
__global__ void __launch_bounds__(kBlock ? kMostThreads : 32 * kWarpsPerBlock, kBlock && kPer == 4 ? 1 : 2)
    k_layer_norm_deriv(const float* dy, const float* x, const float* stats, const float* gain, float* dx, float* part, int h, int w,
                       int offset) {
  extern __shared__ __align__(16) float shares[];
  __shared__ float2 red[2][32];
  grid_dependents_launch();
  grid_dependency_wait();
  const int threads = kBlock ? blockDim.x : 32, t = kBlock ? threadIdx.x : threadIdx.x & 31;
  const int first = kBlock ? blockIdx.x : blockIdx.x * kWarpsPerBlock + (threadIdx.x >> 5);
  const int step = kBlock ? gridDim.x : gridDim.x * kWarpsPerBlock;
  const float inv = 1.0f / h;
  Ring<kPer, 2> ring(shares, t, threads, (int)((offset + (long)first * h) & 3), h);
  float dg[kPer][4], db[kPer][4], gains[kPer][4];
  ring.constants(gain, 1.0f, gains);
  auto fetch = [&](long c, int stage) {
    if (c < w) {
      ring.fetch(stage, 0, x + c * h);
      ring.fetch(stage, 1, dy + c * h);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kPer; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) dg[i][j] = db[i][j] = 0.0f;
#pragma unroll
  for (int k = 0; k < kAhead; k++) fetch(first + (long)k * step, k);
  int turn = 0, stage = 0;
  for (long c = first; c < w; c += step, turn ^= 1) {
    fetch(c + (long)kAhead * step, stage > 0 ? stage - 1 : kAhead);
    const float m = stats[2 * c], rs = stats[2 * c + 1];
    asm volatile("cp.async.wait_group %0;" ::"n"(kAhead) : "memory");
    float v[kPer][4], d[kPer][4];
    ring.read(stage, 0, m, v);
    ring.read(stage, 1, 0.0f, d);
    stage = stage == kAhead ? 0 : stage + 1;
    float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < kPer; i++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float xh = (v[i][j] - m) * rs;
        v[i][j] = xh;
        dg[i][j] += d[i][j] * xh;
        db[i][j] += d[i][j];
        d[i][j] *= gains[i][j];
        s.x += d[i][j];
        s.y += d[i][j] * xh;
      }
    s = column_sum2<kBlock>(s, red[turn]);
    const float ma = s.x * inv, mx = s.y * inv;
#pragma unroll
    for (int i = 0; i < kPer; i++)
#pragma unroll
      for (int j = 0; j < 4; j++) d[i][j] = rs * (d[i][j] - ma - v[i][j] * mx);
    ring.write(dx + c * h, d);
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (!part) return;
  float* out = part + 2L * blockIdx.x * h;
  if (kBlock) {
#pragma unroll
    for (int i = 0; i < kPer; i++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int r = ring.row(i) + j;
        if (r < 0 || r >= h) continue;
        out[r] = dg[i][j];
        out[h + r] = db[i][j];
      }
    return;
  }
  // the block's warps one after another (in the ring's place)
  __syncthreads();
  for (int k = 0; k < kWarpsPerBlock; k++) {
    if ((threadIdx.x >> 5) == k) {
#pragma unroll
      for (int i = 0; i < kPer; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int r = ring.row(i) + j;
          if (r < 0 || r >= h) continue;
          shares[r] = k ? shares[r] + dg[i][j] : dg[i][j];
          shares[h + r] = k ? shares[h + r] + db[i][j] : db[i][j];
        }
    }
    __syncthreads();
  }
  for (int r = threadIdx.x; r < 2 * h; r += blockDim.x) out[r] = shares[r];
}

// Long columns: dx as above with the columns read twice, and the shares of the parameters' gradients by rows.
__global__ void __launch_bounds__(1024) k_layer_norm_deriv_long(const float* dy, const float* x, const float* stats, const float* gain,
                                                                float* dx, int h, int w) {
  __shared__ float2 red[32];
  grid_dependents_launch();
  grid_dependency_wait();
  const long c = blockIdx.x;
  const float m = stats[2 * c], rs = stats[2 * c + 1], inv = 1.0f / h;
  float2 s = make_float2(0.0f, 0.0f);
#pragma unroll 4
  for (int r = threadIdx.x; r < h; r += blockDim.x) {
    const float a = dy[c * h + r] * (gain ? gain[r] : 1.0f);
    s.x += a;
    s.y += a * ((x[c * h + r] - m) * rs);
  }
  s = column_sum2<true>(s, red);
  const float ma = s.x * inv, mx = s.y * inv;
#pragma unroll 4
  for (int r = threadIdx.x; r < h; r += blockDim.x) {
    const float a = dy[c * h + r] * (gain ? gain[r] : 1.0f), xh = (x[c * h + r] - m) * rs;
    dx[c * h + r] = rs * (a - ma - xh * mx);
  }
}
// grid: (blocks of 256 rows, parts of the columns)
__global__ void __launch_bounds__(256) k_layer_norm_shares(const float* dy, const float* x, const float* stats, float* part, int h, int w) {
  grid_dependents_launch();
  grid_dependency_wait();
  const int r = blockIdx.x * 256 + threadIdx.x;
  if (r >= h) return;
  const long c0 = (long)w * blockIdx.y / gridDim.y, c1 = (long)w * (blockIdx.y + 1) / gridDim.y;
  float dg = 0.0f, db = 0.0f;
#pragma unroll 4
  for (long c = c0; c < c1; c++) {
    const float d = dy[c * h + r];
    dg += d * ((x[c * h + r] - stats[2 * c]) * stats[2 * c + 1]);
    db += d;
  }
  part[2L * blockIdx.y * h + r] = dg;
  part[(2L * blockIdx.y + 1) * h + r] = db;
}

// The blocks' shares, in order: 32 values a block, 32 threads a value.
__global__ void __launch_bounds__(1024) k_layer_norm_params(const float* part, int blocks, float* dgain, float* dbias, int h) {
  __shared__ float red[32][33];
  grid_dependents_launch();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const long v = (long)blockIdx.x * 32 + lane;
  float s = 0.0f;
  if (v < 2L * h) {
#pragma unroll 8
    for (int b = wid; b < blocks; b += 32) s += part[2L * b * h + v];
  }
  red[wid][lane] = s;
  __syncthreads();
  s = red[lane][wid];                 // the shares of value `wid` of the block
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const long mine = (long)blockIdx.x * 32 + wid;
  if (lane || mine >= 2L * h) return;
  if (mine < h) {
    if (dgain) dgain[mine] = s;
  } else if (dbias) {
    dbias[mine - h] = s;
  }
}

bool on16(const void* p) { return ((uintptr_t)p & 15) == 0; }
int round32(int n) { return (n + 31) & ~31; }

int offset_of(const void* p) { return (int)((uintptr_t)p >> 2 & 3); }      // floats behind a 16-byte boundary

// Blocks of a kernel that the device keeps resident: a multiple of four (Ring), looked up once a kernel, size and device.
template <class K>
int resident_blocks(K kernel, int threads, int smem, int& err) {
  static std::mutex mu;
  static std::map<std::tuple<int, const void*, int, int>, int> known;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    err = set_error(cudaGetErrorString(cudaGetLastError()));
    return 0;
  }
  std::lock_guard<std::mutex> lock(mu);
  int& n = known[std::make_tuple(dev, (const void*)kernel, threads, smem)];
  if (n == 0) {
    // (each takes what the largest block of it needs: the attribute is the kernel's, not the launch's)
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSmem) != cudaSuccess ||
        cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, 100) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, smem) != cudaSuccess || n < 1) {
      n = 0;
      err = set_error(cudaGetErrorString(cudaGetLastError()));
      return 0;
    }
  }
  return (n * sm_count() + 3) & ~3;
}

int vector_ok(const cudamat* v, int h) {
  if (!v) return 0;
  if (!v->on_device) return ERROR_NOT_ON_DEVICE;
  return numel(v) == h && (v->size[0] == 1 || v->size[1] == 1) ? 0 : ERROR_INCOMPATIBLE_DIMENSIONS;
}

}  // namespace

extern "C" {

int layer_norm(cudamat* mat, cudamat* gain, cudamat* bias, cudamat* target, cudamat* stats, float eps) {
  if (!mat->on_device || !target->on_device || (stats && !stats->on_device)) return ERROR_NOT_ON_DEVICE;
  if (mat->is_trans || target->is_trans || (stats && stats->is_trans)) return ERROR_TRANSPOSED;
  const int h = mat->size[0], w = mat->size[1];
  if (!same_shape(mat, target) || (stats && (stats->size[0] != 2 || stats->size[1] != w))) return ERROR_INCOMPATIBLE_DIMENSIONS;
  int err = vector_ok(gain, h);
  if (!err) err = vector_ok(bias, h);
  if (err) return err;
  if (!(eps >= 0.0f)) {
    set_error("eps has to be at least 0");
    return ERROR_UNSUPPORTED;
  }
  if (overlapping({target, stats, unless_in_place(mat, target), gain, bias}, 2)) return ERROR_UNSUPPORTED;
  if (h == 0 || w == 0) return 0;
  const float *x = mat->data_device, *g = gain ? gain->data_device : nullptr, *b = bias ? bias->data_device : nullptr;
  float *y = target->data_device, *st = stats ? stats->data_device : nullptr;
  const bool vec = h % 4 == 0 && on16(x) && on16(y) && on16(g) && on16(b);
  const int offset = offset_of(x), groups = (h + 2) / 4 + 1;
  // Columns that do not start on 16 bytes: groups of four values all the same (Ring), where the result lies as the input does.
  // 1357 x 20003: 74 us value by value, 58 so; where all columns start on 16 bytes, and beyond 4096 rows, a block a column is the
  // faster one (4096 x 8192: 62 us with the ring, 51 without; 8191 x 4096: 101 and 81).
  if (!vec && offset == offset_of(y) && groups <= 2 * kMostThreads) {
    int err = 0;
    auto run = [&](auto kernel, int per, int threads, bool block) {
      const int smem = (kAhead + 1) * per * threads * 16, columns = block ? w : (w + kWarpsPerBlock - 1) / kWarpsPerBlock;
      int blocks = resident_blocks(kernel, threads, smem, err);
      if (err) return;
      if (blocks > columns) blocks = columns;
      (void)launch_dependent(kernel, dim3(blocks), dim3(threads), (size_t)smem, stream(), x, g, b, y, st, h, w, eps, offset);
    };
    if (groups <= 32) run(k_layer_norm_ring<1, false>, 1, 32 * kWarpsPerBlock, false);
    else if (groups <= 64) run(k_layer_norm_ring<2, false>, 2, 32 * kWarpsPerBlock, false);
    else if (groups <= 128) run(k_layer_norm_ring<4, false>, 4, 32 * kWarpsPerBlock, false);
    else run(k_layer_norm_ring<2, true>, 2, round32((groups + 1) / 2), true);
    return err ? err : check_launch();
  }
  const int items = vec ? h / 4 : h;
#define NORM(VEC, PER, BLOCK, GRID, THREADS) \
  (void)launch_dependent(k_layer_norm<VEC, PER, BLOCK>, dim3(GRID), dim3(THREADS), 0, stream(), x, g, b, y, st, h, w, eps)
#define NORM_PER(PER, BLOCK, GRID, THREADS)                \
  do {                                                     \
    if (vec) NORM(4, PER, BLOCK, GRID, THREADS);           \
    else NORM(1, PER, BLOCK, GRID, THREADS);               \
  } while (0)
  const int warps = (w + kWarpsPerBlock - 1) / kWarpsPerBlock;
  if (items <= 32) NORM_PER(1, false, warps, 32 * kWarpsPerBlock);
  else if (items <= 64) NORM_PER(2, false, warps, 32 * kWarpsPerBlock);
  else if (items <= 128) NORM_PER(4, false, warps, 32 * kWarpsPerBlock);
  else if (items <= 256) NORM_PER(8, false, warps, 32 * kWarpsPerBlock);
  else if (items <= 4 * 1024) NORM_PER(4, true, w, round32((items + 3) / 4));
  else if (items <= 8 * 1024) NORM_PER(8, true, w, 1024);
  else (void)launch_dependent(k_layer_norm_long, dim3(w), dim3(1024), 0, stream(), x, g, b, y, st, h, w, eps);
#undef NORM_PER
#undef NORM
  return check_launch();
}

int layer_norm_deriv(cudamat* deriv, cudamat* mat, cudamat* stats, cudamat* gain, cudamat* target, cudamat* grad_gain,
                     cudamat* grad_bias) {
  if (!deriv->on_device || !mat->on_device || !stats->on_device || !target->on_device) return ERROR_NOT_ON_DEVICE;
  if (deriv->is_trans || mat->is_trans || stats->is_trans || target->is_trans) return ERROR_TRANSPOSED;
  const int h = mat->size[0], w = mat->size[1];
  if (!same_shape(mat, deriv) || !same_shape(mat, target) || stats->size[0] != 2 || stats->size[1] != w)
    return ERROR_INCOMPATIBLE_DIMENSIONS;
  int err = vector_ok(gain, h);
  if (!err) err = vector_ok(grad_gain, h);
  if (!err) err = vector_ok(grad_bias, h);
  if (err) return err;
  // (the parameters' gradients are written when gain has been read)
  if (overlapping({target, grad_gain, grad_bias, unless_in_place(deriv, target), unless_in_place(mat, target), stats,
                   unless_in_place(unless_in_place(gain, grad_gain), grad_bias)}, 3))
    return ERROR_UNSUPPORTED;
  if (h == 0) return 0;
  float *dgain = grad_gain ? grad_gain->data_device : nullptr, *dbias = grad_bias ? grad_bias->data_device : nullptr;
  if (w == 0) {            // sums over no columns
    for (float* p : {dgain, dbias})
      if (p && cudaMemsetAsync(p, 0, sizeof(float) * h, stream()) != cudaSuccess) return set_error(cudaGetErrorString(cudaGetLastError()));
    return 0;
  }
  const float *dy = deriv->data_device, *x = mat->data_device, *st = stats->data_device, *g = gain ? gain->data_device : nullptr;
  float* dx = target->data_device;
  const int offset = offset_of(x), groups = h % 4 == 0 && offset == 0 ? h / 4 : (h + 2) / 4 + 1;
  const bool params = dgain || dbias, by_warp = groups <= 128, is_long = offset != offset_of(dy) || offset != offset_of(dx) || groups > 4 * kMostThreads;
  // how many blocks the columns are spread over: each adds 8 h bytes of shares, written and read again
  const int per = groups <= 32 ? 1 : groups <= 64 ? 2 : groups <= 128 ? 4 : groups <= 2 * 512 ? 2 : 4;
  const int threads = by_warp ? 32 * kWarpsPerBlock : round32((groups + per - 1) / per), smem = (kAhead + 1) * 2 * per * threads * 16;
  const int columns = by_warp ? (w + kWarpsPerBlock - 1) / kWarpsPerBlock : w;
  int blocks = (16 * sm_count() * 256 + h - 1) / h;
  err = 0;
  auto count = [&](auto kernel) { blocks = resident_blocks(kernel, threads, smem, err); };
#define EACH(F)                                              \
  do {                                                       \
    if (groups <= 32) F(k_layer_norm_deriv<1, false>);       \
    else if (groups <= 64) F(k_layer_norm_deriv<2, false>);  \
    else if (groups <= 128) F(k_layer_norm_deriv<4, false>); \
    else if (groups <= 2 * 512) F(k_layer_norm_deriv<2, true>); \
    else F(k_layer_norm_deriv<4, true>);                     \
  } while (0)
  if (!is_long) EACH(count);
  if (err) return err;
  if (blocks > columns) blocks = columns;
  if (is_long && blocks > 32768) blocks = 32768;
  if (blocks < 1) blocks = 1;
  CallScratch room(5, params ? 2 * sizeof(float) * (size_t)h * blocks : 0);
  float* part = params ? (float*)room.p : nullptr;
  if (params && !part) return CUDA_ERROR;
  if (is_long) {
    if (params)
      (void)launch_dependent(k_layer_norm_shares, dim3((h + 255) / 256, blocks), dim3(256), 0, stream(), dy, x, st, part, h, w);
    (void)launch_dependent(k_layer_norm_deriv_long, dim3(w), dim3(1024), 0, stream(), dy, x, st, g, dx, h, w);
  } else {
    auto run = [&](auto kernel) {
      (void)launch_dependent(kernel, dim3(blocks), dim3(threads), (size_t)smem, stream(), dy, x, st, g, dx, part, h, w, offset);
    };
    EACH(run);
  }
#undef EACH
  if (params)
    (void)launch_dependent(k_layer_norm_params, dim3((2 * (unsigned)h + 31) / 32), dim3(1024), 0, stream(), part, blocks, dgain, dbias, h);
  return check_launch();
}

}  // extern "C"
