// A gated layer's products on the tensor cores: operands as two half-precision planes (hi, lo) scaled by a power of two a
// column, three products hi.lo + lo.hi + hi.hi into one fp32 accumulator, 22 bits of an operand and 2^-21 of |a||b| a term.
// The scale is one a column (a unit's weights, a case's inputs), so that neither a large unit nor a large case costs the
// others bits; the epilogue divides it out, exactly.
//
// Both products of the forward pass share the tile: of a pair of CTAs, each multiplies 64 units' gate weights and the same
// units' up weights (128 rows of A, rows 0-63 gate, 64-127 up) with the same BN cases.  A unit's two sums then lie 64 lanes
// apart in tensor memory, which other warps read: pairs of epilogue warps hand each other half their columns through
// shared memory, and each finishes the other half: bias, activation, product, coalesced stores.  Against two tiles of half the
// width (A twice, B once) this reads a quarter less shared memory a multiply-add and keeps the widest instruction.
//
// Persistent pairs of CTAs, 384 threads: warp 0 copies (TMA), warp 1 issues, warps 4-11 drain.  The accumulator truncates
// at every instruction, so sums are folded into registers every 128 products (two buffers in tensor memory).  Every wait is
// bounded; on expiry the kernel records a status word, drains and returns.
#include <cuda.h>

#include <mutex>
#include <type_traits>

#include "gated.cuh"
#include "gemm.cuh"
#include "tcgen05.cuh"

namespace b200 {

namespace {

constexpr int kK = 64;                       // products of a stage: 128 bytes of a plane
constexpr int kRing = 192 * 1024;
constexpr int kExchange = 32 * 1024;         // two buffers of 16 columns each way for four pairs of warps
constexpr int kSmem = kRing + kExchange + 1024 /*alignment*/ + 256 /*barriers*/;
constexpr int kThreads = 384, kEpiThreads = 256;
constexpr int kStages = 6;                   // most of any tile width
constexpr int kChunk = 128 / kK;             // stages an accumulator sums
constexpr int kDrainRegs = 208, kRestRegs = 80;      // 128 x 80 + 256 x 208 of the 384 x 168 the block starts with
constexpr uint32_t kDescK = (1024u >> 4) | (1u << 14) | (2u << 29);   // K-major: rows of 128 bytes, groups of eight 1024 apart

struct GatedParams {
  CUtensorMap maps[6];                       // gate hi, lo, up hi, lo, x hi, lo
  int M, N, K, tiles_m, tiles_n, activation;
  const float *w_inv, *x_inv, *bg, *bu;
  float *gate, *up, *y;
  int* status;
  uint32_t spin_limit;
  uint32_t stage_tx;                         // bytes that both CTAs' copies of a stage bring
};

__device__ __forceinline__ float act_of(int activation, float g) {
  float slope;
  switch (activation) {
    case kLogistic: return activate<kLogistic>(g, slope);
    case kRelu: return activate<kRelu>(g, slope);
    case kSilu: return activate<kSilu>(g, slope);
    case kGelu: return activate<kGelu>(g, slope);
  }
  return g;
}

// v / (2^a 2^b) for the factors r = 2^-a, c = 2^-b: one product where theirs is a normal number.
__device__ __forceinline__ float unscale(float v, float r, float c) {
  const float s = r * c;
  return s >= 1.17549435e-38f && s <= 3.4028234e38f ? v * s : (v * r) * c;
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

// Whether `ok` holds in all of 64 threads, which wait for each other at barrier `id`.
__device__ __forceinline__ bool all_ok(int id, bool ok) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 q, %2, 0;\n\t"
      "bar.red.and.pred p, %1, 64, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r)
      : "r"(id), "r"((uint32_t)ok)
      : "memory");
  return r != 0;
}

template <int BN>
struct Tile {
  static constexpr int kStageBytes = 32 * 1024 + BN * 128;      // A: two planes of 128 rows; B: two planes of BN / 2 rows
  static constexpr int kNumStages = kRing / kStageBytes < kStages ? kRing / kStageBytes : kStages;
  static constexpr int kTmemCols = 2 * BN < 32 ? 32 : 2 * BN;
  static constexpr int kCols = BN / 2;                          // columns a drain warp holds
};

template <int BN>
__global__ void __launch_bounds__(kThreads, 1) k_gated_tc(const __grid_constant__ GatedParams p) {
  using T = Tile<BN>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u, exchange = base + kRing, bars = exchange + kExchange;
  auto full = [&](int s) { return bars + 8u * s; };                 // the stage's copies, of both CTAs, in the leader
  auto empty = [&](int s) { return bars + 8u * (kStages + s); };    // the stage has been multiplied
  auto done = [&](int a) { return bars + 8u * (2 * kStages + a); }; // the accumulator holds its chunk
  auto free_ = [&](int a) { return bars + 8u * (2 * kStages + 2 + a); };
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  grid_dependents_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const uint32_t limit = p.spin_limit;
  const int tiles = p.tiles_m * p.tiles_n, first = blockIdx.x >> 1, step = gridDim.x >> 1;
  const int k_iters = (p.K + kK - 1) / kK;
  if (warp == 2 && lane < 6) asm volatile("prefetch.tensormap [%0];" ::"l"(&p.maps[lane]) : "memory");
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < kStages; s++) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    for (int a = 0; a < 2; a++) {
      mbar_init(done(a), 1);
      mbar_init(free_(a), 2 * kEpiThreads / 32);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    tmem_alloc2(smem_u32(&tmem_slot), T::kTmemCols);
    tmem_relinquish2();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  grid_dependency_wait();

  auto gave_up = [&](int code) {
    if (!*(volatile int*)&abort_flag) atomicCAS(p.status, 0, code);
    *(volatile int*)&abort_flag = 1;
  };
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRestRegs));
    if (warp == 0) {
      // copies: lanes 0-3 a plane of gate's or up's 64 rows, lanes 4, 5 a plane of this CTA's half of the cases
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      const bool is_a = lane < 4;
      const uint32_t to = is_a ? (lane & 1) * 16384u + (lane >> 1) * 8192u : 32768u + (lane & 1) * (uint32_t)(BN * 64);
      for (int t = first; t < tiles && ok; t += step) {
        int tm, tn;
        tile_coords_g<8>(t, p.tiles_m, p.tiles_n, tm, tn);
        const int row = is_a ? tm * 128 + (int)rank * 64 : tn * BN + (int)rank * (BN / 2);
        for (int kb = 0; kb < k_iters; kb++) {
          if (!mbar_wait(empty(stage), phase ^ 1u, &abort_flag, limit)) {
            gave_up(31);
            ok = false;
            break;
          }
          const uint32_t bar = full(stage);
          if (lane == 0 && rank == 0) mbar_expect_tx(bar, p.stage_tx);
          if (lane < 6) tma_load_2d_pair(base + stage * T::kStageBytes + to, &p.maps[lane], kb * kK, row, bar);
          if (++stage == T::kNumStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      // copies already issued land before the CTA leaves: they have had the wait's limit, and some more
      if (!ok)
        for (int i = 0; i < 1024; i++) __nanosleep(100);
    } else if (warp == 1 && rank == 0) {
      const bool elected = elect_one();
      // fp32 accumulator, half-precision operands, both K-major, BN wide, 256 rows
      const uint32_t idesc = (1u << 4) | ((uint32_t)(BN >> 3) << 17) | ((256u >> 4) << 24);
      int stage = 0;
      uint32_t phase = 0, chunk = 0;
      bool ok = true;
      for (int t = first; t < tiles && ok; t += step) {
        int in_chunk = 0;
        for (int kb = 0; kb < k_iters; kb++) {
          const int acc = chunk & 1;
          if (in_chunk == 0) {
            if (!mbar_wait(free_(acc), ((chunk >> 1) & 1u) ^ 1u, &abort_flag, limit)) {
              gave_up(32);
              ok = false;
              break;
            }
            tc_fence_after();
          }
          if (!mbar_wait(full(stage), phase, &abort_flag, limit)) {
            gave_up(33);
            ok = false;
            break;
          }
          const uint32_t sb = (base + stage * T::kStageBytes) >> 4;
          const uint32_t a_hi = sb, a_lo = sb + (16384u >> 4), b_hi = sb + (32768u >> 4), b_lo = b_hi + ((uint32_t)(BN * 64) >> 4);
#pragma unroll
          for (int i = 0; i < 3; i++) {                   // the small products first
            const uint32_t a = i == 1 ? a_lo : a_hi, b = i == 0 ? b_lo : b_hi;
#pragma unroll
            for (int j = 0; j < kK / 16; j++) {
              const uint64_t da = ((uint64_t)kDescK << 32) | (uint64_t)((1u << 16) + a + 2 * j);
              const uint64_t db = ((uint64_t)kDescK << 32) | (uint64_t)((1u << 16) + b + 2 * j);
              if (elected) mma_f16_pair(tmem + acc * BN, da, db, idesc, i + j > 0 || in_chunk > 0);
            }
          }
          if (elected) mma_commit_pair(empty(stage), 3);
          if (++stage == T::kNumStages) {
            stage = 0;
            phase ^= 1u;
          }
          if (++in_chunk == kChunk || kb == k_iters - 1) {
            if (elected) mma_commit_pair(done(acc), 3);
            chunk++;
            in_chunk = 0;
          }
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kDrainRegs));
    // Warp: lanes 32 q .. of the accumulator (q 0, 1 gate, 2, 3 up of units 32 (q & 1) ..), half the columns.
    constexpr int kCols = T::kCols, kMine = kCols / 2, kRound = kMine < 16 ? kMine : 16;
    const int ew = warp - 4, q = warp & 3, half = ew >> 2, which = q >> 1;
    const uint32_t give = exchange + (uint32_t)(((q & 1) * 2 + half) * 8192 + which * 4096 + lane * 4);
    const uint32_t take = exchange + (uint32_t)(((q & 1) * 2 + half) * 8192 + (1 - which) * 4096 + lane * 4);
    uint32_t chunk = 0;
    const int chunks = (k_iters + kChunk - 1) / kChunk;
    bool ok = true;
    for (int t = first; t < tiles && ok; t += step) {
      int tm, tn;
      tile_coords_g<8>(t, p.tiles_m, p.tiles_n, tm, tn);
      const int unit = tm * 128 + (int)rank * 64 + (q & 1) * 32 + lane, n0 = tn * BN + half * kCols;
      float sum[kCols];
#pragma unroll
      for (int j = 0; j < kCols; j++) sum[j] = 0.0f;
      for (int c = 0; c < chunks; c++, chunk++) {
        const int acc = chunk & 1;
        if (!mbar_wait(done(acc), (chunk >> 1) & 1u, &abort_flag, limit)) {
          gave_up(34);
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t from = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * BN + half * kCols);
#pragma unroll
        for (int j = 0; j < kCols; j += 16) {
          float v[16];
          tmem_ld16(from + j, v);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; i++) sum[j + i] += v[i];
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_leader(free_(acc), 0);
      }
      // both warps of a pair go on, or neither: they wait for each other below
      ok = all_ok(1 + (q & 1) * 2 + half, ok);
      if (!ok) break;
      const bool in = unit < p.M;
      const float r = in ? p.w_inv[2L * unit + which] : 0.0f;
      const float* b = which ? p.bu : p.bg;
      const float bias = in && b ? b[unit] : 0.0f;
      // the pair's first warp finishes the first half of the columns, its second the second
      auto finish = [&](auto second) {
        constexpr bool kSecond = decltype(second)::value;
#pragma unroll
        for (int j0 = 0, round = 0; j0 < kMine; j0 += kRound, round++) {
          const uint32_t buf = (uint32_t)(round & 1) * 2048u;
#pragma unroll
          for (int i = 0; i < kRound; i++) {
            const int j = (kSecond ? 0 : kMine) + j0 + i, n = n0 + j;
            const float v = unscale(sum[j], r, n < p.N ? p.x_inv[n] : 1.0f) + bias;
            asm volatile("st.shared.f32 [%0], %1;" ::"r"(give + buf + i * 128), "f"(v) : "memory");
          }
          named_bar_sync(1 + (q & 1) * 2 + half, 64);
#pragma unroll
          for (int i = 0; i < kRound; i++) {
            const int j = (kSecond ? kMine : 0) + j0 + i, n = n0 + j;
            float other;
            asm volatile("ld.shared.f32 %0, [%1];" : "=f"(other) : "r"(take + buf + i * 128) : "memory");
            if (!in || n >= p.N) continue;
            const float mine = unscale(sum[j], r, p.x_inv[n]) + bias;
            const float g = kSecond ? other : mine, u = kSecond ? mine : other;
            const long at = (long)n * p.M + unit;
            if (p.gate) {
              p.gate[at] = g;
              p.up[at] = u;
            }
            p.y[at] = act_of(p.activation, g) * u;
          }
        }
        if (kMine / kRound % 2) named_bar_sync(1 + (q & 1) * 2 + half, 64);   // (the next tile starts with the buffer just read)
      };
      if (which) finish(std::integral_constant<bool, true>{});
      else finish(std::integral_constant<bool, false>{});
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc2(tmem, T::kTmemCols);
  }
}

template <int BN>
int launch(GatedParams& p) {
  static std::mutex mu;
  static bool ready[64] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return set_error("cudaGetDevice failed");
  {
    std::lock_guard<std::mutex> lock(mu);
    if (!ready[dev] && cudaFuncSetAttribute(k_gated_tc<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess)
      return set_error("cudaFuncSetAttribute(max dynamic shared memory) failed");
    ready[dev] = true;
  }
  p.stage_tx = 2 * Tile<BN>::kStageBytes + (uint32_t)take_injected_bytes();
  const int tiles = p.tiles_m * p.tiles_n;
  int pairs = sm_count() / 2;
  if (pairs > tiles) pairs = tiles;
  if (pairs < 1) pairs = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * pairs);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = stream();
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = 2;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = dependent_launch_enabled() ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, k_gated_tc<BN>, p) != cudaSuccess) return set_error(cudaGetErrorString(cudaGetLastError()));
  return check_launch();
}

// ---- matrices as planes --------------------------------------------------------------------
struct SplitJobs {
  SplitJob job[3];
  int first[4];          // blocks
  int h, lda, per_block; // columns of a block: one (all its warps) or one a warp
  bool vec[3];
};

// One column by `threads` threads: its largest finite magnitude, then the planes (the second read comes from L1 or L2).
template <bool kBlock>
__global__ void __launch_bounds__(256) k_split_columns(const SplitJobs a) {
  __shared__ uint32_t red[8];
  grid_dependents_launch();
  grid_dependency_wait();
  const int which = blockIdx.x >= a.first[2] ? 2 : blockIdx.x >= a.first[1] ? 1 : 0;
  const SplitJob j = a.job[which];
  const int threads = kBlock ? 256 : 32, t = kBlock ? threadIdx.x : threadIdx.x & 31, h = a.h;
  const long c = (long)(blockIdx.x - a.first[which]) * (kBlock ? 1 : 8) + (kBlock ? 0 : threadIdx.x >> 5);
  if (c >= j.cols) return;
  const float* x = j.x + c * h;
  const bool vec = a.vec[which];
  uint32_t m = 0;                                     // bits of a magnitude: in the magnitudes' order
  auto see = [&](float v) {
    const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
    if (b < 0x7f800000u) m = max(m, b);
  };
  if (vec) {
#pragma unroll 4
    for (int i = t; i < h / 4; i += threads) {
      const float4 v = reinterpret_cast<const float4*>(x)[i];
      see(v.x); see(v.y); see(v.z); see(v.w);
    }
  } else {
#pragma unroll 8
    for (int i = t; i < h; i += threads) see(x[i]);
  }
  m = __reduce_max_sync(0xffffffffu, m);
  if (kBlock) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
    __syncthreads();
    m = __reduce_max_sync(0xffffffffu, red[threadIdx.x & 7]);
  }
  const int e = (int)f16_exponent(__uint_as_float(m));
  const float scale = __int_as_float((127 + e) << 23);
  if (t == 0) j.inv[c * j.inv_stride] = __int_as_float((127 - e) << 23);
  uint16_t *lo = j.planes + c * 2 * a.lda, *hi = lo + a.lda;
  if (vec) {
#pragma unroll 4
    for (int i = t; i < h / 4; i += threads) {
      const float4 v = reinterpret_cast<const float4*>(x)[i];
      ushort4 l, g;
      split_f16(v.x, scale, l.x, g.x);
      split_f16(v.y, scale, l.y, g.y);
      split_f16(v.z, scale, l.z, g.z);
      split_f16(v.w, scale, l.w, g.w);
      reinterpret_cast<ushort4*>(lo)[i] = l;
      reinterpret_cast<ushort4*>(hi)[i] = g;
    }
  } else {
#pragma unroll 4
    for (int i = t; i < h; i += threads) split_f16(x[i], scale, lo[i], hi[i]);
  }
}

}  // namespace

int split_columns(const SplitJob* jobs, int njobs, int rows) {
  SplitJobs a = {};
  a.h = rows;
  a.lda = aux_rows(rows);
  const bool block = rows > 1024;
  int at = 0;
  for (int i = 0; i < 3; i++) {
    a.first[i] = at;
    if (i >= njobs) continue;
    a.job[i] = jobs[i];
    a.vec[i] = rows % 4 == 0 && ((uintptr_t)jobs[i].x & 15) == 0;
    at += block ? jobs[i].cols : (jobs[i].cols + 7) / 8;
  }
  a.first[3] = at;
  if (at == 0) return 0;
  if (block) (void)launch_dependent(k_split_columns<true>, dim3(at), dim3(256), 0, stream(), a);
  else (void)launch_dependent(k_split_columns<false>, dim3(at), dim3(256), 0, stream(), a);
  return check_launch();
}

int gated_tc(const GatedForward& f) {
  GatedParams p = {};
  p.M = f.wg.cols;
  p.N = f.x.cols;
  p.K = f.wg.rows;
  p.activation = f.activation;
  p.w_inv = f.w_inv;
  p.x_inv = f.x_inv;
  p.bg = f.bg;
  p.bu = f.bu;
  p.gate = f.gate;
  p.up = f.up;
  p.y = f.y;
  p.status = status_word();
  p.spin_limit = wait_limit();
  p.tiles_m = (p.M + 127) / 128;
  // The tile's width: what the pairs of CTAs need for their share of the tiles, a stage taking as long as its twelve
  // instructions (half a cycle a column) or, below that, as its copies.
  const int widths[4] = {256, 128, 64, 32};
  int bn = 256;
  double best = 0;
  for (int w : widths) {
    const long tiles = (long)p.tiles_m * ((p.N + w - 1) / w), pairs = sm_count() / 2 > 0 ? sm_count() / 2 : 1;
    const double stage = 6.0 * w > 500.0 ? 6.0 * w : 500.0;
    const double cost = (double)((tiles + pairs - 1) / pairs) * (stage * ((p.K + kK - 1) / kK) + 2000.0 + 8.0 * w);
    if (w == 256 || cost < 0.98 * best) {
      best = cost;
      bn = w;
    }
  }
  p.tiles_n = (p.N + bn - 1) / bn;
  const Planes* src[3] = {&f.wg, &f.wu, &f.x};
  for (int i = 0; i < 6; i++) {
    const Planes& m = *src[i >> 1];
    const int lda = aux_rows(m.rows);
    // (plane 1 is hi)
    if (!plane_map(&p.maps[i], m.p + ((i & 1) ? 0 : lda), (uint64_t)m.rows, (uint64_t)m.cols, 2 * (uint64_t)lda, kK, i < 4 ? 64 : bn / 2))
      return set_error("cuTensorMapEncodeTiled failed for a plane");
  }
  switch (bn) {
    case 256: return launch<256>(p);
    case 128: return launch<128>(p);
    case 64: return launch<64>(p);
  }
  return launch<32>(p);
}

}  // namespace b200
