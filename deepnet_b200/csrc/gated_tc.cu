// A gated layer's products on the tensor cores, at float32's range and to its last bits: operands as three bfloat16 parts (hi, mid,
// lo) that add up to them, six products of parts (mid.mid + lo.hi + hi.lo + hi.mid + mid.hi + hi.hi) into one fp32 accumulator; what is
// left out is below 2^-26 of |a||b| a term, whatever else a column holds.  (Half-precision planes under a power of two a column took
// half the time and lost what lay 2^-16 below a column's largest: features or gradients of other scales are no exception.)
//
// Both products of the forward pass share the tile: of a pair of CTAs, each multiplies 64 units' gate weights and the same
// units' up weights (128 rows of A, rows 0-63 gate, 64-127 up) with the same BN cases.  A unit's two sums then lie 64 lanes
// apart in tensor memory, which other warps read: pairs of epilogue warps hand each other half their columns through
// shared memory, and each finishes the other half: bias, activation, product, coalesced stores.  Against two tiles of half the
// width (A twice, B once) this reads a quarter less shared memory a multiply-add and keeps the widest instruction.
//
// Persistent pairs of CTAs, 384 threads: warp 0 copies (TMA), warp 1 issues, warps 4-11 drain.  A slot of the ring holds one part of
// both operands, 64 products deep, and is free again behind its last instruction, so that two stages of 256 columns are enough.  The
// accumulator truncates at every instruction, so sums are folded into registers every 64 products (two buffers in tensor memory), the
// small products first.  Every wait is bounded; on expiry the kernel records a status word, drains and returns.  2048 x 8192,
// 4096 cases: 1030 us, 267 TFLOP/s (six terms: 1600 of the tensor pipe's).
#include <cuda.h>

#include "gated.cuh"
#include "gemm.cuh"
#include "tcgen05.cuh"

namespace b200 {

namespace {

constexpr int kK = 64;                       // products of a stage: 128 bytes of a part
constexpr int kRing = 192 * 1024;
constexpr int kExchange = 32 * 1024;         // two buffers of 16 columns each way for four pairs of warps
constexpr int kSmem = kRing + kExchange + 1024 /*alignment*/ + 256 /*barriers*/;
constexpr int kThreads = 384, kEpiThreads = 256;
constexpr int kMostSlots = 10;               // of any tile width
constexpr int kDrainRegs = 208, kRestRegs = 80;      // 128 x 80 + 256 x 208 of the 384 x 168 the block starts with
constexpr uint32_t kDescK = (1024u >> 4) | (1u << 14) | (2u << 29);   // K-major: rows of 128 bytes, groups of eight 1024 apart

struct GatedParams {
  CUtensorMap maps[9];                       // a part's gate, up and x: lo, mid, hi
  int M, N, K, tiles_m, tiles_n, activation;
  int splits;                                // > 1: each tile's stages are shared out; split s leaves its sums in part + s * 2 * M * N
  float* part;                               // (gate's, then up's)
  const float *bg, *bu;
  float *gate, *up, *y;
  int* status;
  uint32_t spin_limit;
  uint32_t slot_tx;                          // bytes that both CTAs' copies of a slot bring
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

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
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
  static constexpr int kSlotBytes = 16 * 1024 + BN * 64;        // 128 rows of A, BN / 2 rows of B
  static constexpr int kSlots = kRing / kSlotBytes < kMostSlots ? kRing / kSlotBytes : kMostSlots;
  static constexpr int kTmemCols = 2 * BN < 32 ? 32 : 2 * BN;
  static constexpr int kCols = BN / 2;                          // columns a drain warp holds
};

// What the roles of a kernel share: the ring of slots, the two accumulators, the barriers between them.  A stage takes three slots.
enum Part { kLo, kMid, kHi };
template <int BN>
struct Machine {
  using T = Tile<BN>;
  uint32_t ring, bars, tmem, rank, limit;
  int *abort_flag, *status;

  __device__ __forceinline__ uint32_t full(int s) const { return bars + 8u * s; }                   // the slot's copies, of both CTAs, in the leader
  __device__ __forceinline__ uint32_t empty(int s) const { return bars + 8u * (kMostSlots + s); }   // the slot has been multiplied
  __device__ __forceinline__ uint32_t done(int a) const { return bars + 8u * (2 * kMostSlots + a); }      // the accumulator holds its stage
  __device__ __forceinline__ uint32_t free_(int a) const { return bars + 8u * (2 * kMostSlots + 2 + a); }
  __device__ __forceinline__ uint32_t slot_at(int s) const { return ring + (uint32_t)s * T::kSlotBytes; }
  __device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, int code) const {
    if (mbar_wait(bar, parity, abort_flag, limit)) return true;
    if (!*(volatile int*)abort_flag) atomicCAS(status, 0, code);
    *(volatile int*)abort_flag = 1;
    return false;
  }

  // All threads; behind it what earlier launches wrote is there.
  __device__ __forceinline__ void start(uint32_t at, uint32_t barriers, uint32_t* tmem_slot, int* flag, int* status_word, uint32_t spin_limit,
                                        const CUtensorMap* maps, int nmaps) {
    grid_dependents_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    ring = at;
    bars = barriers;
    rank = cluster_ctarank();
    limit = spin_limit;
    abort_flag = flag;
    status = status_word;
    if (warp == 2 && lane < nmaps) asm volatile("prefetch.tensormap [%0];" ::"l"(maps + lane) : "memory");
    if (threadIdx.x == 0) {
      *flag = 0;
      for (int s = 0; s < T::kSlots; s++) {
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
      tmem_alloc2(smem_u32(tmem_slot), T::kTmemCols);
      tmem_relinquish2();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    tmem = *tmem_slot;
    grid_dependency_wait();
  }
  __device__ __forceinline__ void end() {
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    if (threadIdx.x >> 5 == 1) {
      tc_fence_after();
      tmem_dealloc2(tmem, T::kTmemCols);
    }
  }

  struct Place {
    int slot = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void next() {
      if (++slot == T::kSlots) {
        slot = 0;
        phase ^= 1u;
      }
    }
  };
  // The copying warp: load(part, shared address, barrier) issues this CTA's copies.
  template <class Load>
  __device__ __forceinline__ bool copy_stage(Place& at, uint32_t tx, int code, Load load) const {
#pragma unroll
    for (int part = kLo; part <= kHi; part++) {
      if (!wait(empty(at.slot), at.phase ^ 1u, code)) return false;
      const uint32_t bar = full(at.slot);
      if ((threadIdx.x & 31) == 0 && rank == 0) mbar_expect_tx(bar, tx);
      load(part, slot_at(at.slot), bar);
      at.next();
    }
    return true;
  }
  // The issuing warp: a stage's products into the accumulator whose turn it is.  lead, step: an operand's descriptor without its
  // address, and from sixteen products to the next.  Codes: of the accumulator's wait, and the next one of the slots'.
  __device__ __forceinline__ bool multiply_stage(Place& at, uint32_t& chunk, bool elected, uint32_t idesc, uint32_t a_lead, uint32_t a_step,
                                                 uint32_t b_lead, uint32_t b_step, int code) const {
    const int acc = chunk & 1;
    if (!wait(free_(acc), ((chunk >> 1) & 1u) ^ 1u, code)) return false;
    tc_fence_after();
    Place of[3];
    uint32_t from[3];
#pragma unroll
    for (int part = kLo; part <= kHi; part++) {
      of[part] = at;
      from[part] = slot_at(at.slot) >> 4;
      at.next();
    }
    auto times = [&](int pa, int pb, bool first) {
#pragma unroll
      for (int j = 0; j < kK / 16; j++) {
        const uint64_t da = ((uint64_t)kDescK << 32) | (uint64_t)(a_lead + from[pa] + a_step * j);
        const uint64_t db = ((uint64_t)kDescK << 32) | (uint64_t)(b_lead + from[pb] + (16384u >> 4) + b_step * j);
        if (elected) mma_f16_pair(tmem + acc * BN, da, db, idesc, !first || j > 0);
      }
    };
    auto release = [&](uint32_t bar) {
      if (elected) mma_commit_pair(bar, 3);
    };
    if (!wait(full(of[kLo].slot), of[kLo].phase, code + 1) || !wait(full(of[kMid].slot), of[kMid].phase, code + 1)) return false;
    times(kMid, kMid, true);
    if (!wait(full(of[kHi].slot), of[kHi].phase, code + 1)) return false;
    times(kLo, kHi, false);
    times(kHi, kLo, false);
    release(empty(of[kLo].slot));
    times(kHi, kMid, false);
    times(kMid, kHi, false);
    release(empty(of[kMid].slot));
    times(kHi, kHi, false);
    release(empty(of[kHi].slot));
    release(done(acc));
    chunk++;
    return true;
  }
  // A drain warp adds kCols columns from `column` on, of its 32 lanes, of `stages` accumulators to its sums.
  template <int kCols>
  __device__ __forceinline__ bool drain(uint32_t& chunk, int stages, int column, float (&sum)[kCols], int code) const {
    constexpr int kLoad = kCols < 32 ? kCols : 32;
#pragma unroll
    for (int j = 0; j < kCols; j++) sum[j] = 0.0f;
    for (int k = 0; k < stages; k++, chunk++) {
      const int acc = chunk & 1;
      if (!wait(done(acc), (chunk >> 1) & 1u, code)) return false;
      tc_fence_after();
      const uint32_t from = tmem + ((threadIdx.x >> 5 & 3) << 21) + (uint32_t)(acc * BN + column);
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
      if ((threadIdx.x & 31) == 0) mbar_arrive_leader(free_(acc), 0);
    }
    return true;
  }
};
// A copying warp that gave up: copies already issued land before the CTA leaves: they have had the wait's limit, and some more.
__device__ __forceinline__ void outlast_copies() {
  for (int i = 0; i < 1024; i++) __nanosleep(100);
}

template <int BN>
__global__ void __launch_bounds__(kThreads, 1) k_gated_tc(const __grid_constant__ GatedParams p) {
  using T = Tile<BN>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u, exchange = base + kRing;
  Machine<BN> m;
  m.start(base, exchange + kExchange, &tmem_slot, &abort_flag, p.status, p.spin_limit, p.maps, 9);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = (int)m.rank;
  const int splits = p.splits, items = p.tiles_m * p.tiles_n * splits, first = blockIdx.x >> 1, step = gridDim.x >> 1;
  const int k_iters = (p.K + kK - 1) / kK;
  auto of_split = [&](int s) { return (int)((long)k_iters * s / splits); };       // its first stage
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRestRegs));
    typename Machine<BN>::Place at;
    bool ok = true;
    if (warp == 0) {
      // lanes 0, 1: gate's and up's 64 rows, lane 2: this CTA's half of the cases
      for (int w = first; w < items && ok; w += step) {
        int tm, tn;
        tile_coords_g<8>(w / splits, p.tiles_m, p.tiles_n, tm, tn);
        const int row = lane < 2 ? tm * 128 + rank * 64 : tn * BN + rank * (BN / 2);
        const int last = of_split(w % splits + 1);
        for (int kb = of_split(w % splits); kb < last && ok; kb++)
          ok = m.copy_stage(at, p.slot_tx, 31, [&](int part, uint32_t to, uint32_t bar) {
            if (lane < 3) tma_load_2d_pair(to + (uint32_t)lane * 8192u, &p.maps[3 * part + lane], kb * kK, row, bar);
          });
      }
      if (!ok) outlast_copies();
    } else if (warp == 1 && rank == 0) {
      const bool elected = elect_one();
      // fp32 accumulator, bfloat16 operands, both K-major, BN wide, 256 rows
      const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BN >> 3) << 17) | ((256u >> 4) << 24);
      uint32_t chunk = 0;
      for (int w = first; w < items && ok; w += step) {
        const int last = of_split(w % splits + 1);
        for (int kb = of_split(w % splits); kb < last && ok; kb++)
          ok = m.multiply_stage(at, chunk, elected, idesc, 1u << 16, 2, 1u << 16, 2, 32);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kDrainRegs));
    // Warp: lanes 32 q .. of the accumulator (q 0, 1 gate, 2, 3 up of units 32 (q & 1) ..), half the columns.  The two warps that
    // hold a unit's sums stage sixteen columns of both, then each finishes eight of them.  The code of a column is there once,
    // not once a column: it runs seldom, and unrolled over the columns and the activations it would be fetched from memory each time.
    constexpr int kCols = T::kCols;
    const int q = warp & 3, half = (warp - 4) >> 2, which = q >> 1, pair = (q & 1) * 2 + half;
    const uint32_t stage_at = exchange + (uint32_t)(pair * 8192 + lane * 4);
    uint32_t chunk = 0;
    for (int w = first; w < items; w += step) {
      int tm, tn;
      tile_coords_g<8>(w / splits, p.tiles_m, p.tiles_n, tm, tn);
      const int unit = tm * 128 + rank * 64 + (q & 1) * 32 + lane, n0 = tn * BN + half * kCols;
      // (asked for here, wanted behind the sums)
      const float bg = unit < p.M && p.bg ? p.bg[unit] : 0.0f, bu = unit < p.M && p.bu ? p.bu[unit] : 0.0f;
      const int sp = w % splits;
      float sum[kCols];
      bool ok = m.drain(chunk, of_split(sp + 1) - of_split(sp), half * kCols, sum, 34);
      if (splits > 1) {
        if (!ok) break;
        float* to = p.part + ((long)(sp * 2 + which) * p.N + n0) * p.M + unit;
        const int live = unit < p.M ? p.N - n0 : 0;
#pragma unroll
        for (int j = 0; j < kCols; j++)
          if (j < live) to[(long)j * p.M] = sum[j];
        continue;
      }
      // All drain warps go on, or none: pairs wait for each other below, and have done with the last tile's columns here.
      ok = all_ok(5, kEpiThreads, ok);
      if (!ok) break;
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
        float gs[8], us[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
          asm volatile("ld.shared.f32 %0, [%1];" : "=f"(gs[i]) : "r"(buf + (uint32_t)(8 * which + i) * 128u));
          asm volatile("ld.shared.f32 %0, [%1];" : "=f"(us[i]) : "r"(buf + 2048u + (uint32_t)(8 * which + i) * 128u));
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
          gs[i] += bg;
          us[i] += bu;
        }
        const int live = unit < p.M ? min(8, p.N - first_n) : 0;
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
  m.end();
}

// The splits' sums in order, and what the epilogue does with them.
template <int kAct>
__global__ void __launch_bounds__(256) k_gated_finish(const __grid_constant__ GatedParams p) {
  grid_dependents_launch();
  grid_dependency_wait();
  const long all = (long)p.M * p.N;
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < all; i += (long)gridDim.x * blockDim.x) {
    const int unit = (int)(i % p.M);
    float g = 0.0f, u = 0.0f;
#pragma unroll 8
    for (int k = 0; k < p.splits; k++) {
      g += p.part[2 * all * k + i];
      u += p.part[2 * all * k + all + i];
    }
    if (p.bg) g += p.bg[unit];
    if (p.bu) u += p.bu[unit];
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

// ---- products of parts as they are stored ---------------------------------------------------
// The derivative's products: of the weights and the gradients (K runs over units), of the inputs and the gradients (K over cases).
// One operand's K is its columns, so its tiles arrive with M or N contiguous (boxes of 64 x 64) and tcgen05 reads them so.  Tiles of
// 256 rows by BN columns a pair of CTAs; the rest as above.
// Two products share a launch, so that few tiles of either leave fewer SMs without work.
struct ProductPart {
  int M, N, tiles_m, tiles_n, npairs, nout, trans, k_iters;
  int a_map, b_map;                          // first of its tensor maps: a0 lo, mid, hi, (a1 ..); b0 lo, mid, hi, (b1 ..)
  int splits;                                // > 1: each tile's stages are shared out; split s leaves its sums in part + s * nout * M * N
  int items;                                 // tiles times splits
  float* part;
  float* out[2];
};
struct ProductParams {
  CUtensorMap maps[21];                      // two pairs, and one operand for two
  ProductPart product[2];
  int nmaps, items;
  int* status;
  uint32_t spin_limit, slot_tx;
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

// The splits' sums in order.
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
      q.out[o][i - o * n] = s;
    }
  }
}

template <int BN>
__global__ void __launch_bounds__(kThreads, 1) k_plane_product(const __grid_constant__ ProductParams p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  Machine<BN> m;
  m.start(base, base + kRing, &tmem_slot, &abort_flag, p.status, p.spin_limit, p.maps, p.nmaps);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = (int)m.rank;
  const int items = p.items, first = blockIdx.x >> 1, step = gridDim.x >> 1;
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRestRegs));
    typename Machine<BN>::Place place;
    bool ok = true;
    if (warp == 0) {
      // lanes 0, 1: 64 of this CTA's 128 rows each, lanes 2 on: its half of the columns (64 at a time where they are contiguous)
      const bool is_a = lane < 2;
      const int box = is_a ? lane : lane - 2;
      const uint32_t offset = (is_a ? 0u : 16384u) + (uint32_t)box * 8192u;
      for (int w = first; w < items && ok; w += step) {
        const ProductItem at(p, w);
        const ProductPart& part = p.product[at.which];
        const int row = (is_a ? at.tm * 256 + rank * 128 : at.tn * BN + rank * (BN / 2)) + 64 * box;
        const int per = part.k_iters, trans = part.trans;
        const bool mine = is_a || box < (trans ? BN / 128 : 1), along = is_a || trans;       // along: rows are the contiguous dimension
        int q = at.first / per, kb = at.first - q * per;
        for (int it = at.first; it < at.last && ok; it++) {
          const CUtensorMap* maps = &p.maps[is_a ? part.a_map + 3 * q : part.b_map + 3 * (trans ? at.out : q)];
          ok = m.copy_stage(place, p.slot_tx, 35, [&](int k, uint32_t to, uint32_t bar) {
            if (mine) tma_load_2d_pair(to + offset, maps + k, along ? row : kb * kK, along ? kb * kK : row, bar);
          });
          if (++kb == per) {
            kb = 0;
            q++;
          }
        }
      }
      if (!ok) outlast_copies();
    } else if (warp == 1 && rank == 0) {
      const bool elected = elect_one();
      // M or N contiguous: blocks of 64 (a row of 128 bytes an element of K) 64 rows apart; sixteen rows a step.  K-major as above.
      constexpr uint32_t kMn = ((uint32_t)(kK * 128) >> 4) << 16, kStepMn = 2048u >> 4;
      uint32_t chunk = 0;
      for (int w = first; w < items && ok; w += step) {
        const ProductItem at(p, w);
        const uint32_t trans = (uint32_t)p.product[at.which].trans;
        const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 15) | (trans << 16) | ((uint32_t)(BN >> 3) << 17) | ((256u >> 4) << 24);
        for (int it = at.first; it < at.last && ok; it++)
          ok = m.multiply_stage(place, chunk, elected, idesc, kMn, kStepMn, trans ? kMn : 1u << 16, trans ? kStepMn : 2u, 36);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kDrainRegs));
    constexpr int kCols = Tile<BN>::kCols;
    const int q = warp & 3, half = (warp - 4) >> 2;
    uint32_t chunk = 0;
    for (int w = first; w < items; w += step) {
      const ProductItem at(p, w);
      const ProductPart& part = p.product[at.which];
      float sum[kCols];
      if (!m.drain(chunk, at.last - at.first, half * kCols, sum, 38)) break;
      const int n0 = at.tn * BN + half * kCols, row = at.tm * 256 + rank * 128 + q * 32 + lane;
      const long M = part.M;
      const int live = row < part.M ? part.N - n0 : 0;
      float* to = (part.splits > 1 ? part.part + ((long)at.split * part.nout + at.out) * M * part.N : part.out[at.out]) + n0 * M + row;
#pragma unroll
      for (int j = 0; j < kCols; j++)
        if (j < live) to[j * M] = sum[j];
    }
  }
  m.end();
}

// ---- matrices as parts ---------------------------------------------------------------------
struct SplitJobs {
  SplitJob job[3];
  int first[3];          // each one's first block: of eight columns
  int h;
};

// A warp a column, or a part of it (grid.y): kBatch groups of kVec values a lane on their way.  Bound by HBM: 10 bytes a value;
// two matrices of 2048 x 8192 53 us, 6.3 TB/s (79 with four values a lane and conversions in place of integer rounding).
template <int kVec>
__global__ void __launch_bounds__(256) k_split_columns(const __grid_constant__ SplitJobs a) {
  constexpr int kBatch = kVec == 8 ? 2 : kVec == 4 ? 4 : 8;
  grid_dependents_launch();
  grid_dependency_wait();
  const int which = blockIdx.x >= a.first[2] ? 2 : blockIdx.x >= a.first[1] ? 1 : 0;
  const float* src = which == 2 ? a.job[2].x : which ? a.job[1].x : a.job[0].x;
  const Planes to = which == 2 ? a.job[2].to : which ? a.job[1].to : a.job[0].to;
  const long c = (long)(blockIdx.x - (which == 2 ? a.first[2] : which ? a.first[1] : a.first[0])) * 8 + (threadIdx.x >> 5);
  if (c >= to.cols) return;
  const float* x = src + c * a.h;
  const int items = a.h / kVec;
  for (int base = (blockIdx.y * kBatch * 32) + (threadIdx.x & 31); base < items; base += gridDim.y * kBatch * 32) {
    float v[kBatch][kVec];
#pragma unroll
    for (int b = 0; b < kBatch; b++)
      if (base + 32 * b < items) load<kVec>(x + (long)(base + 32 * b) * kVec, v[b]);
#pragma unroll
    for (int b = 0; b < kBatch; b++)
      if (base + 32 * b < items) store_parts<kVec>(to, (base + 32 * b) * kVec, c, v[b]);
  }
}

}  // namespace

int split_columns(const SplitJob* jobs, int njobs, int rows) {
  SplitJobs a = {};
  a.h = rows;
  bool vec = rows % 4 == 0;
  for (int i = 0; i < njobs; i++) vec = vec && ((uintptr_t)jobs[i].x & 15) == 0;
  int at = 0;
  for (int i = 0; i < 3; i++) {
    a.first[i] = at;
    if (i >= njobs) continue;
    a.job[i] = jobs[i];
    at += (jobs[i].to.cols + 7) / 8;
  }
  if (at == 0) return 0;
  const bool eights = vec && rows % 8 == 0;
  const int per = 32 * (vec ? 16 : 8);                   // rows of a warp's batch
  int parts = (rows + per - 1) / per;
  if (parts > 65535) parts = 65535;
  if (eights) (void)launch_dependent(k_split_columns<8>, dim3(at, parts), dim3(256), 0, stream(), a);
  else if (vec) (void)launch_dependent(k_split_columns<4>, dim3(at, parts), dim3(256), 0, stream(), a);
  else (void)launch_dependent(k_split_columns<1>, dim3(at, parts), dim3(256), 0, stream(), a);
  return check_launch();
}

namespace {
// The three maps of a matrix's parts, lo first.
bool maps_of(CUtensorMap* maps, int stride, const Planes& m, uint32_t box) {
  const uint64_t lda = (uint64_t)aux_rows(m.rows);
  return plane_map(maps, m.low, (uint64_t)m.rows, (uint64_t)m.cols, (uint64_t)m.low_ld, kK, box) &&
         plane_map(maps + stride, m.p, (uint64_t)m.rows, (uint64_t)m.cols, 2 * lda, kK, box) &&
         plane_map(maps + 2 * stride, m.p + lda, (uint64_t)m.rows, (uint64_t)m.cols, 2 * lda, kK, box);
}
}  // namespace

int gated_tc(const GatedForward& f) {
  GatedParams p = {};
  p.M = f.wg.cols;
  p.N = f.x.cols;
  p.K = f.wg.rows;
  p.activation = f.activation;
  p.bg = f.bg;
  p.bu = f.bu;
  p.gate = f.gate;
  p.up = f.up;
  p.y = f.y;
  p.status = status_word();
  p.spin_limit = wait_limit();
  p.tiles_m = (p.M + 127) / 128;
  // The tile's width, and whether the sums are shared out: what the pairs of CTAs need for their share of the work, in cycles.  A
  // stage takes as long as its instructions (12 BN) or the rows its copies bring; sums that are shared out cost a launch and their way
  // through memory.  Constants fitted to 20 shapes from 64 x 64 x 2000 to 2048 x 8192 x 1024 at every width and split: what it chooses
  // takes 2 % longer than the best of them on average, 13 % at most (4096 x 512, 20 cases: 17.6 us, 15.5).
  const long pairs = sm_count() / 2 > 0 ? sm_count() / 2 : 1, stages = (p.K + kK - 1) / kK;
  int bn = 256;
  double best = 0;
  for (int w = 256; w >= 32; w /= 2) {
    const long tiles = (long)p.tiles_m * ((p.N + w - 1) / w);
    for (long s = 1; s <= 16 && s <= stages; s++) {
      const long turns = (tiles * s + pairs - 1) / pairs;
      if (s > 1 && turns > 1) break;
      const double stage = 12.0 * w > 3.6 * (256 + w) ? 12.0 * w : 3.6 * (256 + w);
      const double cost = turns * (stage * ((stages + s - 1) / s) + 400.0 + 13.0 * w) + (s > 1 ? 3500.0 + (double)s * p.M * p.N / 240.0 : 0.0);
      if (best == 0 || cost < best) {
        best = cost;
        bn = w;
        p.splits = (int)s;
      }
    }
  }
  p.tiles_n = (p.N + bn - 1) / bn;
  if (!maps_of(p.maps, 3, f.wg, 64) || !maps_of(p.maps + 1, 3, f.wu, 64) || !maps_of(p.maps + 2, 3, f.x, bn / 2))
    return set_error("cuTensorMapEncodeTiled failed for a plane");
  const long tiles = (long)p.tiles_m * p.tiles_n * p.splits;
  if (tiles > 0x7fffffffL) return ERROR_UNSUPPORTED;
  CallScratch room(2, p.splits > 1 ? (size_t)p.splits * 2 * p.M * p.N * sizeof(float) : 0);
  p.part = (float*)room.p;
  if (p.splits > 1 && !p.part) return CUDA_ERROR;
  p.slot_tx = 2 * (16 * 1024 + bn * 64) + (uint32_t)take_injected_bytes();
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

int plane_products(const PlaneProduct* f, int nproducts, int V, int H, int cases) {
  ProductParams p = {};
  p.status = status_word();
  p.spin_limit = wait_limit();
  const long pairs = sm_count() / 2 > 0 ? sm_count() / 2 : 1;
  // The tile's width and how many each product's sums are shared out to (a pair of CTAs walks the items pairs apart, the inputs' gradient
  // first): what the pair with most work needs, in cycles, as in gated_tc.  As if all gradients were wanted, so that none's bits depend on
  // the others.  Fitted to the same 20 shapes: 3 % above the best on average, 30 % at most (128 x 2000, 150 cases: 33 us, 26);
  // the way through memory at twice its fitted price, as what it evens out does not pay where the power cap sets the clock (2048 x 8192,
  // 4096 cases: shares of four 110 us in memory, the product no shorter).
  int bn = 256, splits[2] = {1, 1};
  double best = 0;
  for (int w = 256; w >= 128; w /= 2) {
    const double stage = 12.0 * w > 4.2 * (256 + w) ? 12.0 * w : 4.2 * (256 + w);
    const long tiles[2] = {(V + 255) / 256 * (((long)cases + w - 1) / w), (V + 255) / 256 * (((long)H + w - 1) / w) * 2};
    const long all[2] = {2 * (((long)H + kK - 1) / kK), ((long)cases + kK - 1) / kK}, size[2] = {(long)V * cases, 2L * V * H};
    constexpr int kChoices[] = {1, 2, 3, 4, 6, 8, 12, 16, 24};
    for (int s0 : kChoices) {
      if (s0 > all[0]) break;
      for (int s1 : kChoices) {
        if (s1 > all[1]) break;
        const long n = tiles[0] * s0, total = n + tiles[1] * s1;
        const double l0 = stage * ((all[0] + s0 - 1) / s0) + 17.0 * w, l1 = stage * ((all[1] + s1 - 1) / s1) + 17.0 * w;
        double cost = 0;
        for (long i : {0L, n % pairs, total % pairs}) {       // (pairs between these have the same items)
          const long c0 = n / pairs + (i < n % pairs), c = total / pairs + (i < total % pairs);
          const double t = c0 * l0 + (c - c0) * l1;
          if (t > cost) cost = t;
        }
        if (s0 > 1 || s1 > 1) cost += 4200.0 + ((s0 > 1 ? (double)s0 * size[0] : 0.0) + (s1 > 1 ? (double)s1 * size[1] : 0.0)) / 150.0;
        if (best == 0 || cost < best) {
          best = cost;
          bn = w;
          splits[0] = s0;
          splits[1] = s1;
        }
      }
    }
  }
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
    q.tiles_m = (q.M + 255) / 256;
    q.tiles_n = (q.N + bn - 1) / bn;
    q.splits = splits[f[i].trans];
    const long n = (long)q.tiles_m * q.tiles_n * q.nout * q.splits;
    items += n;
    if (items > 0x3fffffffL) return ERROR_UNSUPPORTED;
    q.items = (int)n;
    if (q.splits > 1) bytes += (size_t)q.splits * q.nout * q.M * q.N * sizeof(float);
    q.a_map = p.nmaps;
    for (int side = 0; side < 2; side++) {
      const int count = side == 0 ? q.npairs : f[i].trans ? q.nout : q.npairs;
      if (side) q.b_map = p.nmaps;
      for (int m = 0; m < count; m++, p.nmaps += 3)
        if (!maps_of(p.maps + p.nmaps, 1, side ? f[i].b[m] : f[i].a[m], side == 0 || f[i].trans ? kK : bn / 2))
          return set_error("cuTensorMapEncodeTiled failed for a plane");
    }
    for (int o = 0; o < q.nout; o++) q.out[o] = f[i].out[o];
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
  p.slot_tx = 2 * (16 * 1024 + bn * 64) + (uint32_t)take_injected_bytes();
  const int err = bn == 256 ? launch_pairs(k_plane_product<256>, p, items) : launch_pairs(k_plane_product<128>, p, items);
  if (err || !bytes) return err;
  long blocks = (finished + 255) / 256;
  if (blocks > 8L * sm_count()) blocks = 8L * sm_count();
  (void)launch_dependent(k_plane_finish, dim3((unsigned)blocks), dim3(256), 0, stream(), p);
  return check_launch();
}

}  // namespace b200
