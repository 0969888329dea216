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
// at every instruction, so sums are folded into registers every 128 products (two buffers in tensor memory; 256 products: 5 %
// faster on 2048 x 8192, 4096 cases, and twice the error of a plain fp32 product).  Every wait is bounded; on expiry the kernel
// records a status word, drains and returns.  2048 x 8192, 4096 cases: 580 to 610 us, 450 to 475 TFLOP/s (three terms: 1350 to 1420
// of the tensor pipe's), the pipe 75 % active at the clock the power cap allows; the rest is the end of a tile, which two
// buffers do not cover.  Tried and taken back: stages of 32 products (as fast, few tiles 1.3 times slower), sixteen drain warps.
#include <cuda.h>

#include <type_traits>

#include "gated.cuh"
#include "gemm.cuh"
#include "tcgen05.cuh"

namespace b200 {

namespace {

constexpr int kK = 64;                       // products of a stage: 128 bytes of a plane
constexpr int kRing = 192 * 1024;
constexpr int kExchange = 32 * 1024;         // two buffers of 16 columns each way for four pairs of warps
constexpr int kSmem = kRing + kExchange + 1024 /*alignment*/ + 1024 /*scales*/ + 256 /*barriers*/;
constexpr int kThreads = 384, kEpiThreads = 256;
constexpr int kStages = 6;                   // most of any tile width
constexpr int kChunk = 128 / kK;             // stages an accumulator sums
constexpr int kDrainRegs = 208, kRestRegs = 80;      // 128 x 80 + 256 x 208 of the 384 x 168 the block starts with
constexpr uint32_t kDescK = (1024u >> 4) | (1u << 14) | (2u << 29);   // K-major: rows of 128 bytes, groups of eight 1024 apart

struct GatedParams {
  CUtensorMap maps[6];                       // gate hi, lo, up hi, lo, x hi, lo
  int M, N, K, tiles_m, tiles_n, activation;
  int splits;                                // > 1: each tile's stages are shared out; split s leaves its sums in part + s * 2 * M * N
  float* part;                               // (gate's, then up's)
  const float *w_inv, *x_inv, *bg, *bu;
  float *gate, *up, *y;
  int* status;
  uint32_t spin_limit;
  uint32_t stage_tx;                         // bytes that both CTAs' copies of a stage bring
};

template <int kAct>
__device__ __forceinline__ void activate_times(float (&g)[8], const float (&u)[8]) {
  float slope;
#pragma unroll
  for (int i = 0; i < 8; i++) g[i] = activate<kAct>(g[i], slope) * u[i];
}
// g = act(g) * u
__device__ __forceinline__ void activate_times(int activation, float (&g)[8], const float (&u)[8]) {
  switch (activation) {
    case kLogistic: activate_times<kLogistic>(g, u); break;
    case kRelu: activate_times<kRelu>(g, u); break;
    case kSilu: activate_times<kSilu>(g, u); break;
    case kGelu: activate_times<kGelu>(g, u); break;
    default: activate_times<kLinear>(g, u);
  }
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

// Whether two scales multiply to a normal number.
__device__ __forceinline__ bool tame(float scale) { return scale >= 8.6736174e-19f && scale <= 1.1529215e18f; }      // 2^-60, 2^60
__device__ __forceinline__ float4 lds_f4(uint32_t at) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at));
  return v;
}
// Whether `ok` holds in all of `threads` threads, which wait for each other at barrier `id`.
__device__ __forceinline__ bool all_ok(int id, int threads, bool ok) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 q, %3, 0;\n\t"
      "bar.red.and.pred p, %1, %2, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r)
      : "r"(id), "r"(threads), "r"((uint32_t)ok)
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
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u, exchange = base + kRing, scales = exchange + kExchange, bars = scales + 1024;
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
  const int splits = p.splits, items = p.tiles_m * p.tiles_n * splits, first = blockIdx.x >> 1, step = gridDim.x >> 1;
  const int k_iters = (p.K + kK - 1) / kK;
  auto of_split = [&](int s) { return (int)((long)k_iters * s / splits); };       // its first stage
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
      for (int w = first; w < items && ok; w += step) {
        int tm, tn;
        tile_coords_g<8>(w / splits, p.tiles_m, p.tiles_n, tm, tn);
        const int row = is_a ? tm * 128 + (int)rank * 64 : tn * BN + (int)rank * (BN / 2);
        const int last = of_split(w % splits + 1);
        for (int kb = of_split(w % splits); kb < last; kb++) {
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
      for (int w = first; w < items && ok; w += step) {
        int in_chunk = 0;
        const int last = of_split(w % splits + 1);
        for (int kb = of_split(w % splits); kb < last; kb++) {
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
          if (++in_chunk == kChunk || kb == last - 1) {
            if (elected) mma_commit_pair(done(acc), 3);
            chunk++;
            in_chunk = 0;
          }
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kDrainRegs));
    // Warp: lanes 32 q .. of the accumulator (q 0, 1 gate, 2, 3 up of units 32 (q & 1) ..), half the columns.  The two warps that
    // hold a unit's sums stage sixteen columns of both, then each finishes eight of them.  The code of a column is there once,
    // not once a column: it runs seldom, and unrolled over the columns and the activations it would be fetched from memory each time.
    constexpr int kCols = T::kCols, kLoad = kCols < 32 ? kCols : 32;
    const int ew = warp - 4, q = warp & 3, half = ew >> 2, which = q >> 1, pair = (q & 1) * 2 + half;
    const uint32_t stage_at = exchange + (uint32_t)(pair * 8192 + lane * 4);
    uint32_t chunk = 0;
    bool ok = true;
    for (int w = first; w < items && ok; w += step) {
      int tm, tn;
      tile_coords_g<8>(w / splits, p.tiles_m, p.tiles_n, tm, tn);
      const int unit = tm * 128 + (int)rank * 64 + (q & 1) * 32 + lane, n0 = tn * BN + half * kCols;
      // (asked for here, wanted behind the sums)
      const float2 r = unit < p.M ? make_float2(p.w_inv[2L * unit], p.w_inv[2L * unit + 1]) : make_float2(1.0f, 1.0f);
      const float bg = unit < p.M && p.bg ? p.bg[unit] : 0.0f, bu = unit < p.M && p.bu ? p.bu[unit] : 0.0f;
      const int case_of_mine = tn * BN + (int)threadIdx.x - 128;
      const float c = (int)threadIdx.x - 128 < BN && case_of_mine < p.N ? p.x_inv[case_of_mine] : 1.0f;
      const int sp = w % splits, chunks = (of_split(sp + 1) - of_split(sp) + kChunk - 1) / kChunk;
      float sum[kCols];
#pragma unroll
      for (int j = 0; j < kCols; j++) sum[j] = 0.0f;
      for (int k = 0; k < chunks; k++, chunk++) {
        const int acc = chunk & 1;
        if (!mbar_wait(done(acc), (chunk >> 1) & 1u, &abort_flag, limit)) {
          gave_up(34);
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t from = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * BN + half * kCols);
#pragma unroll
        for (int j = 0; j < kCols; j += kLoad) {
          float v[kLoad];
          if constexpr (kLoad == 32) tmem_ld32(from + j, v);
          else tmem_ld16(from + j, v);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < kLoad; i++) sum[j + i] += v[i];
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_leader(free_(acc), 0);
      }
      if (splits > 1) {
        if (!ok) break;
        float* to = p.part + ((long)(sp * 2 + which) * p.N + n0) * p.M + unit;
        const int live = unit < p.M ? p.N - n0 : 0;
#pragma unroll
        for (int j = 0; j < kCols; j++)
          if (j < live) to[(long)j * p.M] = sum[j];
        continue;
      }
      // All drain warps go on, or none: they wait for each other here and below.  The cases' scales are there for all of them; where no
      // product of two scales leaves the range of normal numbers, one multiplication takes both.
      const bool in = unit < p.M;
      ok = all_ok(5, kEpiThreads, ok);
      if (!ok) break;
      // (everybody is done with the last tile's)
      if ((int)threadIdx.x - 128 < BN) asm volatile("st.shared.f32 [%0], %1;" ::"r"(scales + (threadIdx.x - 128) * 4u), "f"(c) : "memory");
      const bool plain = all_ok(5, kEpiThreads, tame(c) && tame(r.x) && tame(r.y));
      float *yo = p.y + unit, *go = p.gate + unit, *uo = p.up + unit;
#pragma unroll 1
      for (int round = 0; round < kCols / 16; round++) {
        const uint32_t buf = stage_at + (uint32_t)(round & 1) * 4096u;
        const int first_n = n0 + 16 * round + 8 * which;
#pragma unroll
        for (int x = 0; x < kCols / 16; x++)
          if (x == round) {
#pragma unroll
            for (int i = 0; i < 16; i++)
              asm volatile("st.shared.f32 [%0], %1;" ::"r"(buf + (uint32_t)which * 2048u + i * 128), "f"(sum[16 * x + i]));
          }
        named_bar_sync(1 + pair, 64);
        float gs[8], us[8], c8[8];
        const uint32_t scale_at = scales + (uint32_t)(half * kCols + 16 * round + 8 * which) * 4u;
        const float4 c0 = lds_f4(scale_at), c1 = lds_f4(scale_at + 16);
        c8[0] = c0.x; c8[1] = c0.y; c8[2] = c0.z; c8[3] = c0.w; c8[4] = c1.x; c8[5] = c1.y; c8[6] = c1.z; c8[7] = c1.w;
#pragma unroll
        for (int i = 0; i < 8; i++) {
          asm volatile("ld.shared.f32 %0, [%1];" : "=f"(gs[i]) : "r"(buf + (uint32_t)(8 * which + i) * 128u));
          asm volatile("ld.shared.f32 %0, [%1];" : "=f"(us[i]) : "r"(buf + 2048u + (uint32_t)(8 * which + i) * 128u));
        }
        if (plain) {
#pragma unroll
          for (int i = 0; i < 8; i++) {
            gs[i] = fmaf(gs[i], r.x * c8[i], bg);
            us[i] = fmaf(us[i], r.y * c8[i], bu);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; i++) {
            gs[i] = unscale(gs[i], r.x, c8[i]) + bg;
            us[i] = unscale(us[i], r.y, c8[i]) + bu;
          }
        }
        const int live = in ? min(8, p.N - first_n) : 0;
        if (p.gate) {
#pragma unroll
          for (int i = 0; i < 8; i++)
            if (i < live) {
              go[(long)(first_n + i) * p.M] = gs[i];
              uo[(long)(first_n + i) * p.M] = us[i];
            }
        }
        activate_times(p.activation, gs, us);
#pragma unroll
        for (int i = 0; i < 8; i++)
          if (i < live) yo[(long)(first_n + i) * p.M] = gs[i];
      }
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

// The splits' sums in order, and what the epilogue does with them.
template <int kAct>
__global__ void __launch_bounds__(256) k_gated_finish(const __grid_constant__ GatedParams p) {
  grid_dependents_launch();
  grid_dependency_wait();
  const long all = (long)p.M * p.N;
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < all; i += (long)gridDim.x * blockDim.x) {
    const int n = (int)(i / p.M), unit = (int)(i - (long)n * p.M);
    float g = 0.0f, u = 0.0f;
#pragma unroll 8
    for (int k = 0; k < p.splits; k++) {
      g += p.part[2 * all * k + i];
      u += p.part[2 * all * k + all + i];
    }
    const float c = p.x_inv[n];
    g = unscale(g, p.w_inv[2L * unit], c) + (p.bg ? p.bg[unit] : 0.0f);
    u = unscale(u, p.w_inv[2L * unit + 1], c) + (p.bu ? p.bu[unit] : 0.0f);
    if (p.gate) {
      p.gate[i] = g;
      p.up[i] = u;
    }
    float slope;
    p.y[i] = activate<kAct>(g, slope) * u;
  }
}

// Pairs of CTAs for `tiles` tiles.
template <class Params>
int launch_pairs(void (*kernel)(Params), const Params& p, long tiles) {
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess)
    return set_error("cudaFuncSetAttribute(max dynamic shared memory) failed");
  long pairs = sm_count() / 2;
  if (pairs > tiles) pairs = tiles;
  if (pairs < 1) pairs = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * pairs));
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
  if (cudaLaunchKernelEx(&cfg, kernel, p) != cudaSuccess) return set_error(cudaGetErrorString(cudaGetLastError()));
  return check_launch();
}

// ---- products of planes as they are stored --------------------------------------------------
// The derivative's products: of the weights and the gradients (K runs over units), of the inputs and the gradients (K over cases).
// One operand's K is its columns, so its tiles arrive with M or N contiguous (boxes of 64 x 64) and tcgen05 reads them so; the
// scales that lie along K are divided out of the other operand when its planes are written.  Tiles of 256 rows by BN columns a
// pair of CTAs; the rest as above.
// Two products share a launch, so that few tiles of either leave fewer SMs without work.
struct ProductPart {
  int M, N, tiles_m, tiles_n, npairs, nout, trans, k_iters, inv_stride;
  int a_map, b_map;                          // first of its tensor maps: a0 hi, lo, (a1 hi, lo); b0 hi, lo, (b1 hi, lo)
  int splits;                                // > 1: each tile's stages are shared out; split s leaves its sums in part + s * nout * M * N
  int items;                                 // tiles times splits
  float* part;
  float* out[2];
  const float* inv[2];
};
struct ProductParams {
  CUtensorMap maps[14];
  ProductPart product[2];
  int nmaps, items;
  int* status;
  uint32_t spin_limit, stage_tx;
};
// Where item w belongs.
struct ProductItem {
  int which, out, tm, tn, split, first, last;     // first, last: stages
  __device__ __forceinline__ ProductItem(const ProductParams& p, int w) {
    which = w >= p.product[0].items;
    const ProductPart& q = p.product[which];
    w -= which ? p.product[0].items : 0;
    split = w % q.splits;
    tile_coords_g<8>(w / q.splits, q.tiles_m, q.tiles_n * q.nout, tm, tn);
    out = tn >= q.tiles_n;
    tn -= out * q.tiles_n;
    const long all = (long)q.k_iters * q.npairs;
    first = (int)(all * split / q.splits);
    last = (int)(all * (split + 1) / q.splits);
  }
};

// The splits' sums in order, times the columns' scales.
__global__ void __launch_bounds__(256) k_plane_finish(const __grid_constant__ ProductParams p) {
  grid_dependents_launch();
  grid_dependency_wait();
#pragma unroll 1
  for (int which = 0; which < 2; which++) {
    const ProductPart& q = p.product[which];
    if (q.items == 0 || q.splits == 1) continue;
    const long n = (long)q.M * q.N, all = n * q.nout;
    for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < all; i += (long)gridDim.x * blockDim.x) {
      float s = 0.0f;
#pragma unroll 8
      for (int k = 0; k < q.splits; k++) s += q.part[all * k + i];
      const int o = i >= n;
      const long at = i - o * n;
      q.out[o][at] = s * q.inv[o][at / q.M * q.inv_stride];
    }
  }
}

template <int BN>
__global__ void __launch_bounds__(kThreads, 1) k_plane_product(const __grid_constant__ ProductParams p) {
  using T = Tile<BN>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u, bars = base + kRing;
  auto full = [&](int s) { return bars + 8u * s; };
  auto empty = [&](int s) { return bars + 8u * (kStages + s); };
  auto done = [&](int a) { return bars + 8u * (2 * kStages + a); };
  auto free_ = [&](int a) { return bars + 8u * (2 * kStages + 2 + a); };
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  grid_dependents_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const uint32_t limit = p.spin_limit;
  const int items = p.items, first = blockIdx.x >> 1, step = gridDim.x >> 1;
  if (warp == 2 && lane < p.nmaps) asm volatile("prefetch.tensormap [%0];" ::"l"(&p.maps[lane]) : "memory");
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
      // copies: lanes 0-3 a plane of 64 of this CTA's 128 rows, lanes 4 on a plane of its half of the columns (64 at a time where
      // they are contiguous)
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      const bool is_a = lane < 4;
      const int plane = lane & 1, box = is_a ? lane >> 1 : (lane - 4) >> 1;
      const uint32_t to = is_a ? plane * 16384u + box * 8192u : 32768u + plane * (uint32_t)(BN * 64) + box * 8192u;
      for (int w = first; w < items && ok; w += step) {
        const ProductItem at(p, w);
        const ProductPart& part = p.product[at.which];
        const int row = (is_a ? at.tm * 256 + (int)rank * 128 : at.tn * BN + (int)rank * (BN / 2)) + 64 * box;
        const int per = part.k_iters, trans = part.trans;
        const bool mine = is_a || lane < 4 + (trans ? 2 * (BN / 128) : 2);
        int q = at.first / per, kb = at.first - q * per;
        for (int it = at.first; it < at.last; it++) {
          const CUtensorMap* map = &p.maps[(is_a ? part.a_map + 2 * q : part.b_map + 2 * (trans ? at.out : q)) + plane];
          if (!mbar_wait(empty(stage), phase ^ 1u, &abort_flag, limit)) {
            gave_up(35);
            ok = false;
            break;
          }
          const uint32_t bar = full(stage), dst = base + stage * T::kStageBytes + to;
          if (lane == 0 && rank == 0) mbar_expect_tx(bar, p.stage_tx);
          if (mine) {
            const bool along = is_a || trans;            // rows are the contiguous dimension
            tma_load_2d_pair(dst, map, along ? row : kb * kK, along ? kb * kK : row, bar);
          }
          if (++stage == T::kNumStages) {
            stage = 0;
            phase ^= 1u;
          }
          if (++kb == per) {
            kb = 0;
            q++;
          }
        }
      }
      if (!ok)
        for (int i = 0; i < 1024; i++) __nanosleep(100);
    } else if (warp == 1 && rank == 0) {
      const bool elected = elect_one();
      // M or N contiguous: blocks of 64 (a row of 128 bytes an element of K) 64 rows apart; sixteen rows a step.  K-major as above.
      constexpr uint32_t kMn = ((uint32_t)(kK * 128) >> 4) << 16, kStepMn = 2048u >> 4;
      int stage = 0;
      uint32_t phase = 0, chunk = 0;
      bool ok = true;
      for (int w = first; w < items && ok; w += step) {
        int in_chunk = 0;
        const ProductItem at(p, w);
        const int iters = at.last - at.first;
        const uint32_t trans = (uint32_t)p.product[at.which].trans;
        const uint32_t idesc = (1u << 4) | (1u << 15) | (trans << 16) | ((uint32_t)(BN >> 3) << 17) | ((256u >> 4) << 24);
        const uint32_t b_lead = trans ? kMn : 1u << 16, b_step = trans ? kStepMn : 2u;
        for (int kb = 0; kb < iters; kb++) {
          const int acc = chunk & 1;
          if (in_chunk == 0) {
            if (!mbar_wait(free_(acc), ((chunk >> 1) & 1u) ^ 1u, &abort_flag, limit)) {
              gave_up(36);
              ok = false;
              break;
            }
            tc_fence_after();
          }
          if (!mbar_wait(full(stage), phase, &abort_flag, limit)) {
            gave_up(37);
            ok = false;
            break;
          }
          const uint32_t sb = (base + stage * T::kStageBytes) >> 4;
          const uint32_t a_hi = sb, a_lo = sb + (16384u >> 4), b_hi = sb + (32768u >> 4), b_lo = b_hi + ((uint32_t)(BN * 64) >> 4);
#pragma unroll
          for (int i = 0; i < 3; i++) {
            const uint32_t a = i == 1 ? a_lo : a_hi, b = i == 0 ? b_lo : b_hi;
#pragma unroll
            for (int j = 0; j < kK / 16; j++) {
              const uint64_t da = ((uint64_t)kDescK << 32) | (uint64_t)(kMn + a + kStepMn * j);
              const uint64_t db = ((uint64_t)kDescK << 32) | (uint64_t)(b_lead + b + b_step * j);
              if (elected) mma_f16_pair(tmem + acc * BN, da, db, idesc, i + j > 0 || in_chunk > 0);
            }
          }
          if (elected) mma_commit_pair(empty(stage), 3);
          if (++stage == T::kNumStages) {
            stage = 0;
            phase ^= 1u;
          }
          if (++in_chunk == kChunk || kb == iters - 1) {
            if (elected) mma_commit_pair(done(acc), 3);
            chunk++;
            in_chunk = 0;
          }
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kDrainRegs));
    constexpr int kCols = T::kCols, kLoad = kCols < 32 ? kCols : 32;
    const int ew = warp - 4, q = warp & 3, half = ew >> 2;
    uint32_t chunk = 0;
    bool ok = true;
    for (int w = first; w < items && ok; w += step) {
      const ProductItem at(p, w);
      const ProductPart& part = p.product[at.which];
      const int o = at.out, n0 = at.tn * BN + half * kCols, m = at.tm * 256 + (int)rank * 128 + q * 32 + lane;
      const int chunks = (at.last - at.first + kChunk - 1) / kChunk;
      // the columns' scales, one a lane (asked for here, wanted behind the sums)
      float scales[(kCols + 31) / 32];
#pragma unroll
      for (int g = 0; g < (kCols + 31) / 32; g++) {
        const int n = n0 + 32 * g + lane;
        scales[g] = n < part.N ? part.inv[o][(long)n * part.inv_stride] : 0.0f;
      }
      float sum[kCols];
#pragma unroll
      for (int j = 0; j < kCols; j++) sum[j] = 0.0f;
      for (int c = 0; c < chunks; c++, chunk++) {
        const int acc = chunk & 1;
        if (!mbar_wait(done(acc), (chunk >> 1) & 1u, &abort_flag, limit)) {
          gave_up(38);
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t from = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * BN + half * kCols);
#pragma unroll
        for (int j = 0; j < kCols; j += kLoad) {
          float v[kLoad];
          if constexpr (kLoad == 32) tmem_ld32(from + j, v);
          else tmem_ld16(from + j, v);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < kLoad; i++) sum[j + i] += v[i];
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_leader(free_(acc), 0);
      }
      if (!ok) break;
      const long M = part.M;
      const int live = m < part.M ? part.N - n0 : 0;
      if (part.splits > 1) {
        float* to = part.part + ((long)at.split * part.nout + o) * M * part.N + n0 * M + m;
#pragma unroll
        for (int j = 0; j < kCols; j++)
          if (j < live) to[j * M] = sum[j];
        continue;
      }
      float* out = part.out[o] + n0 * M + m;
#pragma unroll
      for (int j = 0; j < kCols; j++) {
        const float c = __shfl_sync(0xffffffffu, scales[j / 32], j % 32);
        if (j < live) out[j * M] = sum[j] * c;
      }
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

// ---- matrices as planes --------------------------------------------------------------------
struct SplitJobs {
  SplitJob job[3];
  int first[3];          // each one's first block: of eight columns, or of one
  int h, lda;
  uint32_t* zero;        // words that later launches count in
  int nzero;
};

// A column's exponent from its largest finite magnitude (m: its bits), and its inverse scale written.
__device__ __forceinline__ float scale_of(uint32_t m, float* inv) {
  const int e = (int)f16_exponent(__uint_as_float(m));
  if (inv) *inv = __int_as_float((127 - e) << 23);
  return __int_as_float((127 + e) << 23);
}
__device__ __forceinline__ uint32_t magnitude(float v) {      // bits of finite magnitudes, in their order
  const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}
template <int kVec>
__device__ __forceinline__ void store_planes(uint16_t* lo, uint16_t* hi, long i, const float (&v)[kVec], float scale) {
  uint16_t l[kVec], g[kVec];
#pragma unroll
  for (int j = 0; j < kVec; j++) split_f16(v[j], scale, l[j], g[j]);
  if constexpr (kVec == 4) {
    reinterpret_cast<ushort4*>(lo)[i] = make_ushort4(l[0], l[1], l[2], l[3]);
    reinterpret_cast<ushort4*>(hi)[i] = make_ushort4(g[0], g[1], g[2], g[3]);
  } else {
    lo[i] = l[0];
    hi[i] = g[0];
  }
}

// A warp (or block) a column, which it holds in registers: kPer groups of kVec values a thread.  Bound by HBM: 8 bytes a value.
template <int kVec, int kPer, bool kBlock>
__global__ void __launch_bounds__(256) k_split_columns(const __grid_constant__ SplitJobs a) {
  __shared__ uint32_t red[8];
  grid_dependents_launch();
  grid_dependency_wait();
  for (int i = blockIdx.x * 256 + threadIdx.x; i < a.nzero; i += gridDim.x * 256) a.zero[i] = 0;
  const int which = blockIdx.x >= a.first[2] ? 2 : blockIdx.x >= a.first[1] ? 1 : 0;
  const float* src = which == 2 ? a.job[2].x : which ? a.job[1].x : a.job[0].x;
  uint16_t* planes = which == 2 ? a.job[2].planes : which ? a.job[1].planes : a.job[0].planes;
  float* inv = which == 2 ? a.job[2].inv : which ? a.job[1].inv : a.job[0].inv;
  const int stride = which == 2 ? a.job[2].inv_stride : which ? a.job[1].inv_stride : a.job[0].inv_stride;
  const int cols = which == 2 ? a.job[2].cols : which ? a.job[1].cols : a.job[0].cols;
  const int at = blockIdx.x - (which == 2 ? a.first[2] : which ? a.first[1] : a.first[0]);
  const int threads = kBlock ? 256 : 32, t = kBlock ? threadIdx.x : threadIdx.x & 31, items = a.h / kVec;
  const long c = (long)at * (kBlock ? 1 : 8) + (kBlock ? 0 : threadIdx.x >> 5);
  if (c >= cols) return;
  const float* x = src + c * a.h;
  float v[kPer][kVec];
  uint32_t m = 0;
  auto load = [&](int i, float (&to)[kVec]) {
    if constexpr (kVec == 4) {
      const float4 f = reinterpret_cast<const float4*>(x)[i];
      to[0] = f.x; to[1] = f.y; to[2] = f.z; to[3] = f.w;
    } else {
      to[0] = x[i];
    }
  };
#pragma unroll
  for (int i = 0; i < kPer; i++) {
    if (t + i * threads < items) {
      load(t + i * threads, v[i]);
    } else {
#pragma unroll
      for (int j = 0; j < kVec; j++) v[i][j] = 0.0f;
    }
  }
#pragma unroll
  for (int i = 0; i < kPer; i++)
#pragma unroll
    for (int j = 0; j < kVec; j++) m = max(m, magnitude(v[i][j]));
  if (kBlock)        // (columns longer than that are read again below)
    for (int i = t + kPer * threads; i < items; i += threads) {
      float w[kVec];
      load(i, w);
#pragma unroll
      for (int j = 0; j < kVec; j++) m = max(m, magnitude(w[j]));
    }
  m = __reduce_max_sync(0xffffffffu, m);
  if (kBlock) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
    __syncthreads();
    m = __reduce_max_sync(0xffffffffu, red[threadIdx.x & 7]);
  }
  const float scale = scale_of(m, t == 0 ? inv + c * stride : nullptr);
  uint16_t *lo = planes + c * 2 * a.lda, *hi = lo + a.lda;
#pragma unroll
  for (int i = 0; i < kPer; i++)
    if (t + i * threads < items) store_planes<kVec>(lo, hi, t + i * threads, v[i], scale);
  if (kBlock)
    for (int i = t + kPer * threads; i < items; i += threads) {
      float w[kVec];
      load(i, w);
      store_planes<kVec>(lo, hi, i, w, scale);
    }
}

}  // namespace

int split_columns(const SplitJob* jobs, int njobs, int rows, uint32_t* zero, int nzero) {
  SplitJobs a = {};
  a.zero = zero;
  a.nzero = nzero;
  a.h = rows;
  a.lda = aux_rows(rows);
  bool vec = rows % 4 == 0;
  for (int i = 0; i < njobs; i++) vec = vec && ((uintptr_t)jobs[i].x & 15) == 0;
  const int items = vec ? rows / 4 : rows;
  const bool block = items > 32 * 16;
  int at = 0;
  for (int i = 0; i < 3; i++) {
    a.first[i] = at;
    if (i >= njobs) continue;
    a.job[i] = jobs[i];
    at += block ? jobs[i].cols : (jobs[i].cols + 7) / 8;
  }
  if (at == 0) return 0;
#define SPLIT(VEC, PER, BLOCK) (void)launch_dependent(k_split_columns<VEC, PER, BLOCK>, dim3(at), dim3(256), 0, stream(), a)
#define SPLIT_PER(PER, BLOCK)          \
  do {                                 \
    if (vec) SPLIT(4, PER, BLOCK);     \
    else SPLIT(1, PER, BLOCK);         \
  } while (0)
  if (items <= 32 * 4) SPLIT_PER(4, false);
  else if (items <= 32 * 8) SPLIT_PER(8, false);
  else if (items <= 32 * 16) SPLIT_PER(16, false);
  else if (items <= 256 * 4) SPLIT_PER(4, true);
  else SPLIT_PER(8, true);
#undef SPLIT_PER
#undef SPLIT
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
  // The tile's width, and whether the sums are shared out: what the pairs of CTAs need for their share of the work, in cycles.  A
  // stage takes as long as its instructions (6 BN) or the rows its copies bring (3.6 each: 4096 x 64, 64 cases, a single tile, 0.55
  // us a stage at any width); sums that are shared out cost a launch and their way through memory.
  const long pairs = sm_count() / 2 > 0 ? sm_count() / 2 : 1, stages = (p.K + kK - 1) / kK;
  int bn = 256;
  double best = 0;
  for (int w = 256; w >= 32; w /= 2) {
    const long tiles = (long)p.tiles_m * ((p.N + w - 1) / w);
    for (long s = 1; s <= 16 && s * 2 <= (stages > 2 ? stages : 2); s++) {
      const long turns = (tiles * s + pairs - 1) / pairs;
      if (s > 1 && turns > 1) break;
      const double stage = 6.0 * w > 3.6 * (256 + w) ? 6.0 * w : 3.6 * (256 + w);
      const double cost = turns * (stage * ((stages + s - 1) / s) + 2500.0 + 10.0 * w) +
                          (s > 1 ? 12000.0 + (double)s * p.M * p.N * 8.0 / 1500.0 : 0.0);
      if (best == 0 || cost < 0.97 * best) {
        best = cost;
        bn = w;
        p.splits = (int)s;
      }
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
  const long tiles = (long)p.tiles_m * p.tiles_n * p.splits;
  if (tiles > 0x7fffffffL) return ERROR_UNSUPPORTED;
  CallScratch room(2, p.splits > 1 ? (size_t)p.splits * 2 * p.M * p.N * sizeof(float) : 0);
  p.part = (float*)room.p;
  if (p.splits > 1 && !p.part) return CUDA_ERROR;
  p.stage_tx = 2 * (32 * 1024 + bn * 128) + (uint32_t)take_injected_bytes();
  int err;
  switch (bn) {
    case 256: err = launch_pairs(k_gated_tc<256>, p, tiles); break;
    case 128: err = launch_pairs(k_gated_tc<128>, p, tiles); break;
    case 64: err = launch_pairs(k_gated_tc<64>, p, tiles); break;
    default: err = launch_pairs(k_gated_tc<32>, p, tiles);
  }
  if (err || p.splits == 1) return err;
  long blocks = ((long)p.M * p.N + 255) / 256;
  if (blocks > 8L * sm_count()) blocks = 8L * sm_count();
#define FINISH(ACT) case ACT: (void)launch_dependent(k_gated_finish<ACT>, dim3((unsigned)blocks), dim3(256), 0, stream(), p); break
  switch (p.activation) { FINISH(kLinear); FINISH(kLogistic); FINISH(kRelu); FINISH(kSilu); FINISH(kGelu); }
#undef FINISH
  return check_launch();
}

int plane_products(const PlaneProduct* f, int nproducts) {
  ProductParams p = {};
  p.status = status_word();
  p.spin_limit = wait_limit();
  const long pairs = sm_count() / 2 > 0 ? sm_count() / 2 : 1;
  // The wider tile reads less shared memory a multiply-add; the narrower one where it needs fewer turns of the pairs.  Work counted in
  // stages of a tile.
  auto stages = [&](int w) {
    long n = 0;
    for (int i = 0; i < nproducts; i++) {
      const long N = f[i].trans ? f[i].b[0].rows : f[i].b[0].cols;
      n += (long)((f[i].a[0].rows + 255) / 256) * f[i].nout * ((N + w - 1) / w) * f[i].npairs * ((f[i].a[0].cols + kK - 1) / kK);
    }
    return n;
  };
  const int bn = 2 * ((stages(256) + pairs - 1) / pairs) <= 1.1 * ((stages(128) + pairs - 1) / pairs) ? 256 : 128;
  const long share = (stages(bn) + pairs - 1) / pairs;       // stages a pair has to do at least
  size_t bytes = 0;
  long items = 0;
  for (int i = 0; i < nproducts; i++) {
    ProductPart& q = p.product[i];
    q.M = f[i].a[0].rows;
    q.N = f[i].trans ? f[i].b[0].rows : f[i].b[0].cols;
    q.npairs = f[i].npairs;
    q.nout = f[i].nout;
    q.trans = f[i].trans;
    q.k_iters = (f[i].a[0].cols + kK - 1) / kK;
    q.inv_stride = f[i].inv_stride;
    q.tiles_m = (q.M + 255) / 256;
    q.tiles_n = (q.N + bn - 1) / bn;
    // a sum that is longer than a pair's share is shared out, eight stages or more to a pair
    const long all = (long)q.k_iters * q.npairs, least = share > 8 ? share : 8;
    long splits = (all + least / 2) / least;
    if (splits > 64) splits = 64;
    q.splits = splits < 1 ? 1 : (int)splits;
    const long n = (long)q.tiles_m * q.tiles_n * q.nout * q.splits;
    items += n;
    if (items > 0x3fffffffL) return ERROR_UNSUPPORTED;
    q.items = (int)n;
    if (q.splits > 1) bytes += (size_t)q.splits * q.nout * q.M * q.N * sizeof(float);
    q.a_map = p.nmaps;
    for (int side = 0; side < 2; side++) {
      const int count = side == 0 ? q.npairs : f[i].trans ? q.nout : q.npairs;
      if (side) q.b_map = p.nmaps;
      for (int m = 0; m < 2 * count; m++) {
        const Planes& x = side ? f[i].b[m >> 1] : f[i].a[m >> 1];
        const int lda = aux_rows(x.rows);
        if (!plane_map(&p.maps[p.nmaps++], x.p + ((m & 1) ? 0 : lda), (uint64_t)x.rows, (uint64_t)x.cols, 2 * (uint64_t)lda, kK,
                       side == 0 || f[i].trans ? kK : bn / 2))
          return set_error("cuTensorMapEncodeTiled failed for a plane");
      }
    }
    for (int o = 0; o < q.nout; o++) {
      q.out[o] = f[i].out[o];
      q.inv[o] = f[i].inv[o];
    }
  }
  p.items = (int)items;
  CallScratch room(2, bytes);
  if (bytes && !room.p) return CUDA_ERROR;
  float* at = (float*)room.p;
  long finished = 0;
  for (int i = 0; i < nproducts; i++) {
    ProductPart& q = p.product[i];
    if (q.splits == 1) continue;
    q.part = at;
    at += (size_t)q.splits * q.nout * q.M * q.N;
    finished += (long)q.nout * q.M * q.N;
  }
  p.stage_tx = 2 * (32 * 1024 + bn * 128) + (uint32_t)take_injected_bytes();
  const int err = bn == 256 ? launch_pairs(k_plane_product<256>, p, items) : launch_pairs(k_plane_product<128>, p, items);
  if (err || !bytes) return err;
  long blocks = (finished + 255) / 256;
  if (blocks > 8L * sm_count()) blocks = 8L * sm_count();
  (void)launch_dependent(k_plane_finish, dim3((unsigned)blocks), dim3(256), 0, stream(), p);
  return check_launch();
}

}  // namespace b200
