// Log probabilities of given tokens under the softmax of each column of logits, the distribution's entropy and its
// likeliest tokens, and the gradient.  With m = max z, s = sum exp(z - m), d = z - m:
//   log p_t = d_t - log s,   H = log s - (sum exp(d) d) / s
//   dz_i = g (1[i = t] - p_i) - q p_i (log p_i + H)      for gradients g of log p_t and q of H
// The logits are read once: every thread carries m, s and sum exp(d) d of what it has seen, joined by warps, then by the
// block.  Bound by HBM (4 bytes a logit forward, 8 back): 10 000 x 4096 35 us (4.7 TB/s; the sums' instructions are a third of it)
// and 56 us (5.9 TB/s).  For the k likeliest (k <= 32, equal logits by the lower number) the threads' maxima give a bound that
// at least k logits reach and few others do; the chunks of 128 logits whose maximum reaches it are read again and what reaches it
// is ranked (50 021 words of normal logits, k 20: about 60; 56 us for 777 columns, 39 without).  Where more than 512 do (64 where
// eight columns share a block: from k 28 on the bound of one warp's lanes lets more through in nearly every longer column), or a mask
// leaves fewer than k, sorted lists across the lanes of each warp find them, slowly where many logits rise above all before them.
// A column whose logits are all -inf has no distribution: log p is -inf, H 0 and the gradient 0.  A NaN or +inf among a
// column's logits makes all its results NaN (its likeliest tokens are then 0, 1, ...).
#include "common.cuh"

using namespace b200;

namespace {

constexpr int kMostTop = 32;

// Sums of powers of two: t is in units of log 2, which is multiplied in at the end.  A power's argument is rounded once and its value is
// ex2.approx's: two units in the last place and |d| 2^-24 of a term, 1.1e-7 and 7e-8 of log p over 10 000 and 50 021 words (6e-8 with
// torch's exponential), for a third of the instructions.
struct Sums {
  float m, s, t;          // maximum, sum exp(z - m), sum exp(z - m) (z - m) / log 2
};
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f, kLowest = -3.4028234e38f;

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// exp(x) for x <= 0, to two units in the last place whatever x is: what the product with log2 e rounds off is put back.
__device__ __forceinline__ float exp_accurate(float x) {
  const float y = x * kLog2e;
  float r = fmaf(x, kLog2e, -y);
  r = fmaf(x, 1.9259629911e-8f, r);
  const float e = exp2_approx(y);
  return y > -126.0f ? fmaf(e, r * kLn2, e) : e;
}

// The sums under a maximum of `m` (not below theirs).
__device__ __forceinline__ void rescale(Sums& a, float m) {
  const float d = (a.m - m) * kLog2e, f = exp2_approx(d);      // (a.m of -inf: 0, and its sums are 0 or NaN)
  a.t = f > 0.0f ? (a.t + d * a.s) * f : 0.0f * a.s;
  a.s *= f;
  a.m = m;
}
__device__ __forceinline__ Sums join(Sums a, Sums b) {
  const float m = fmaxf(a.m, b.m);
  if (m == -INFINITY) return a.s != a.s ? a : b;             // (nothing but -inf, or NaN)
  rescale(a, m);
  rescale(b, m);
  return Sums{m, a.s + b.s, a.t + b.t};
}

// The list a warp keeps: lane i holds the i-th likeliest so far.
struct Top {
  float v;
  int i;
};
__device__ __forceinline__ bool beats(float v, int i, float w, int j) { return v > w || (v == w && i < j); }

// Puts (v, i) of lane `from` where it belongs (it beats the k-th).
__device__ __forceinline__ void insert(Top& top, float v, int i, int from) {
  const int lane = threadIdx.x & 31;
  v = __shfl_sync(0xffffffffu, v, from);
  i = __shfl_sync(0xffffffffu, i, from);
  const float pv = __shfl_up_sync(0xffffffffu, top.v, 1);
  const int pi = __shfl_up_sync(0xffffffffu, top.i, 1);
  if (beats(v, i, top.v, top.i)) {
    const bool here = lane == 0 || !beats(v, i, pv, pi);
    top.v = here ? v : pv;
    top.i = here ? i : pi;
  }
}
// Offers one value a lane.
__device__ __forceinline__ void offer(Top& top, int k, float v, int i, float& kv, int& ki) {
  unsigned who = __ballot_sync(0xffffffffu, beats(v, i, kv, ki));
  while (who) {
    const int from = __ffs(who) - 1;
    insert(top, v, i, from);
    kv = __shfl_sync(0xffffffffu, top.v, k - 1);
    ki = __shfl_sync(0xffffffffu, top.i, k - 1);
    who &= who - 1;
    who &= __ballot_sync(0xffffffffu, beats(v, i, kv, ki));
  }
}

struct LogProbArgs {
  const float *z, *tokens;
  float *logp, *entropy, *stats, *top, *top_tokens;
  int h, w, k;
};

__device__ __forceinline__ int token_of(float f, int n) {
  if (!(fabsf(f) < 2147483648.0f)) return -1;
  int i = (int)f;
  if (i < 0) i += n;
  return i < 0 || i >= n ? -1 : i;
}

// A column in groups of four values on 16 bytes, wherever it starts: group q holds rows 4 q - o .. of a column that starts o floats
// behind a 16-byte boundary; only the first and the last may be partial.  (Value by value 9999 x 4096 takes 44 us, so 35.)
__device__ __forceinline__ int offset_in(const float* column) { return (int)((uintptr_t)column >> 2 & 3); }
__device__ __forceinline__ void load_group(const float* column, int r, int h, float none, float (&v)[4]) {
  if (r >= 0 && r + 4 <= h) {
    const float4 x = *reinterpret_cast<const float4*>(column + r);
    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = r + j >= 0 && r + j < h ? column[r + j] : none;
  }
}
__device__ __forceinline__ void store_group(float* column, int r, int h, const float (&v)[4]) {
  if (r >= 0 && r + 4 <= h) {
    *reinterpret_cast<float4*>(column + r) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (r + j >= 0 && r + j < h) column[r + j] = v[j];
  }
}

// A float's bits in the floats' order, both zeros alike, and back (0: below all).
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

constexpr int kCandidates = 512;       // of a block's columns together
constexpr int kChunks = 2048;          // chunks (a warp's 128 logits) whose maxima a block keeps
static_assert(kChunks * sizeof(uint32_t) == 32 * kMostTop * sizeof(Top), "a column's share of the maxima is its lists'");

// A column is read by `warps` of the block's warps (a power of two), the next kBatch groups of a thread on their way while it works
// on some.
template <bool kTop>
__global__ void __launch_bounds__(1024) k_log_prob(const LogProbArgs a, int warps) {
  constexpr int kBatch = 4;
  __shared__ Sums sums[32];
  __shared__ uint32_t bounds[32];
  // A column's own share of it, whether maxima or lists: the lists come after its maxima's last use, but other columns of the block
  // may still be at theirs.
  __shared__ union {
    uint32_t maxima[kTop ? kChunks : 1];
    Top lists[kTop ? 32 * kMostTop : 1];
  } shared;
  __shared__ Top candidates[kTop ? kCandidates : 1];
  __shared__ int counts[32];
  grid_dependents_launch();
  grid_dependency_wait();
  const int threads = 32 * warps, group = threadIdx.x / threads, groups = blockDim.x / threads, t = threadIdx.x % threads;
  const int lane = threadIdx.x & 31, wid = t >> 5, first_warp = group * warps;
  const long c = (long)blockIdx.x * groups + group;
  if (c >= a.w) return;                                // (a column's threads together: nobody waits for them)
  const float* col = a.z + c * a.h;
  const int o = offset_in(col), items = (a.h + o + 3) >> 2;
  auto meet = [&]() {
    if (warps == 1) __syncwarp();
    else if (groups == 1) __syncthreads();
    else if (group == 0) asm volatile("bar.sync 1, %0;" ::"r"(threads) : "memory");
    else if (group == 1) asm volatile("bar.sync 2, %0;" ::"r"(threads) : "memory");
    else if (group == 2) asm volatile("bar.sync 3, %0;" ::"r"(threads) : "memory");
    else asm volatile("bar.sync 4, %0;" ::"r"(threads) : "memory");      // (at most four columns of two warps or more)
  };
  // before(values of a batch), then f(value, its number) for each if it wants them; -inf beyond the last
  auto each = [&](auto before, auto f) {
    float next[kBatch][4];
    auto fetch = [&](int base) {
#pragma unroll
      for (int b = 0; b < kBatch; b++) {
        const int i = base + b * threads + t;
        if (i < items) {
          load_group(col, 4 * i - o, a.h, -INFINITY, next[b]);
        } else {
#pragma unroll
          for (int j = 0; j < 4; j++) next[b][j] = -INFINITY;
        }
      }
    };
    fetch(0);
    for (int base = 0; base < items; base += kBatch * threads) {
      float v[kBatch][4];
#pragma unroll
      for (int b = 0; b < kBatch; b++)
#pragma unroll
        for (int j = 0; j < 4; j++) v[b][j] = next[b][j];
      fetch(base + kBatch * threads);                  // on its way while this batch is worked on
      float m = -INFINITY;
#pragma unroll
      for (int b = 0; b < kBatch; b++)
#pragma unroll
        for (int j = 0; j < 4; j++) m = fmaxf(m, v[b][j]);
      if (!before(m, v, base)) continue;
#pragma unroll
      for (int b = 0; b < kBatch; b++)
#pragma unroll
        for (int j = 0; j < 4; j++) f(v[b][j], 4 * (base + b * threads + t) + j - o);
    }
  };
  // this warp's chunks' maxima: chunk b of its round i at maxima[(i * kBatch + b) * warps + wid]
  const int most = kChunks / groups;
  uint32_t* const maxima = shared.maxima + (kTop ? group * most : 0);
  Top* const lists = shared.lists + (kTop ? group * (32 * kMostTop / groups) : 0);       // one a warp: warps x groups is 32 at most
  const bool kept = ((items + kBatch * threads - 1) / (kBatch * threads)) * kBatch * warps <= most;
  Sums s = {-INFINITY, 0.0f, 0.0f};
  float m = kLowest;                                   // s.m, finite where nothing but -inf was seen
  each(
      [&](float best, const float (&v)[kBatch][4], int base) {
        if (best > s.m) {
          rescale(s, best);
          m = fmaxf(best, kLowest);
        }
        if (kTop && kept)
#pragma unroll
          for (int b = 0; b < kBatch; b++) {
            const uint32_t of_chunk = __reduce_max_sync(0xffffffffu, ordered(fmaxf(fmaxf(v[b][0], v[b][1]), fmaxf(v[b][2], v[b][3]))));
            if (lane == 0) maxima[base / 32 + b * warps + wid] = of_chunk;
          }
        return true;
      },
      [&](float v, int) {
        const float d = (v - m) * kLog2e, e = exp2_approx(d);
        s.s += e;
        s.t = fmaf(e, fmaxf(d, -200.0f), s.t);         // (2^-200 is 0 here: no 0 x inf)
      });
  if (kTop) {
    // the c-th largest of this warp's lanes' maxima: warps c >= k of them, so at least k logits are not below the smallest of the
    // warps' c-th
    uint32_t key = ordered(s.m), cth = 0;
    for (int i = (a.k + warps - 1) / warps; i > 0; i--) {
      cth = __reduce_max_sync(0xffffffffu, key);
      const unsigned who = __ballot_sync(0xffffffffu, key == cth);
      if (lane == __ffs(who) - 1) key = 0;
    }
    if (lane == 0) bounds[first_warp + wid] = cth;
    if (t == 0) counts[group] = 0;
  }
  auto joined = [&](Sums s) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      Sums x;
      x.m = __shfl_xor_sync(0xffffffffu, s.m, o);
      x.s = __shfl_xor_sync(0xffffffffu, s.s, o);
      x.t = __shfl_xor_sync(0xffffffffu, s.t, o);
      s = (lane & o) ? join(x, s) : join(s, x);              // (the same order in both lanes: the same bits)
    }
    return s;
  };
  s = joined(s);
  if (warps > 1) {
    if (lane == 0) sums[first_warp + wid] = s;
    meet();
    if (!kTop && wid) return;
    s = joined(lane < warps ? sums[first_warp + lane] : Sums{-INFINITY, 0.0f, 0.0f});
  } else if (kTop) {
    meet();
  }
  const bool none = s.m == -INFINITY && s.s == s.s, bad = s.s != s.s;
  const float ls = none ? 0.0f : logf(s.s);
  const float nan = __int_as_float(0x7fc00000);
  if (t == 0) {
    if (a.logp) {
      const int w = token_of(a.tokens[c], a.h);
      a.logp[c] = w < 0 || bad ? nan : none ? -INFINITY : (col[w] - s.m) - ls;
    }
    if (a.entropy) a.entropy[c] = bad ? nan : none ? 0.0f : ls - s.t * kLn2 / s.s;
    if (a.stats) {
      a.stats[2 * c] = bad ? nan : s.m;
      a.stats[2 * c + 1] = bad ? nan : ls;
    }
  }
  if constexpr (kTop) {
    float *top = a.top + c * a.k, *number = a.top_tokens + c * a.k;
    auto put = [&](int rank, const Top& x) {
      top[rank] = none ? -INFINITY : (x.v - s.m) - ls;
      number[rank] = (float)x.i;
    };
    if (bad) {
      if (t < a.k) {
        top[t] = nan;
        number[t] = (float)t;
      }
      return;
    }
    // The column again (from L1 or L2), where a chunk's maximum says so: what is not below the bound; all words that are left where the
    // bound is -inf.
    const float bound = fmaxf(unordered(__reduce_min_sync(0xffffffffu, lane < warps ? bounds[first_warp + lane] : 0xffffffffu)), kLowest);
    const int room = kCandidates / groups;
    Top* found = candidates + group * room;
    auto offer_found = [&](float v, int i) {
      if (v >= bound) {
        const int at = atomicAdd(&counts[group], 1);
        if (at < room) found[at] = Top{v, i};
      }
    };
    if (kept) {
      __syncwarp();                                    // (this warp's own maxima)
      const uint32_t least = ordered(bound);
      const int rounds = (items + threads - 1) / threads;
      for (int first = 0; first < rounds; first += 32) {       // 32 of the warp's chunks at a time, those wanted one by one
        unsigned wanted = __ballot_sync(0xffffffffu, first + lane < rounds && maxima[(first + lane) * warps + wid] >= least);
        while (wanted) {
          const int i = (first + __ffs(wanted) - 1) * threads + t;
          wanted &= wanted - 1;
          if (i < items) {
            float v[4];
            load_group(col, 4 * i - o, a.h, -INFINITY, v);
#pragma unroll
            for (int j = 0; j < 4; j++) offer_found(v[j], 4 * i + j - o);
          }
        }
      }
    } else {
      each([&](float best, const float (&)[kBatch][4], int) { return best >= bound; }, offer_found);
    }
    meet();
    const int n = counts[group];
    if (n >= a.k && n <= room) {
      for (int x = t; x < n; x += threads) {
        const Top mine = found[x];
        int rank = 0;
        for (int y = 0; y < n; y++) rank += beats(found[y].v, found[y].i, mine.v, mine.i);
        if (rank < a.k) put(rank, mine);
      }
      return;
    }
    // Too many (equal logits, a column in order) or too few: sorted lists.  (An item beyond the last beats nothing.)
    Top list = {-INFINITY, 0x7fffffff};
    float kv = -INFINITY;
    int ki = 0x7fffffff;
    each([](float, const float (&)[kBatch][4], int) { return true; }, [&](float v, int i) { offer(list, a.k, v, i >= 0 && i < a.h ? i : 0x7fffffff, kv, ki); });
    if (warps > 1) {
      if (lane < a.k) lists[wid * kMostTop + lane] = list;
      meet();
      if (wid) return;
    }
    for (int x = 1; x < warps; x++) {
      const Top other = lane < a.k ? lists[x * kMostTop + lane] : Top{-INFINITY, 0x7fffffff};
      offer(list, a.k, other.v, other.i, kv, ki);
    }
    if (lane < a.k) put(lane, list);
  }
}

// `warps` of a block's eight warps a column, grid.y parts of it.  A column without weight is not read.  kAlike: logits and gradient
// lie the same way to 16 bytes.
template <bool kAlike>
__global__ void __launch_bounds__(256) k_log_prob_deriv(const float* z, const float* tokens, const float* stats, const float* grad,
                                                        const float* entropy, const float* grad_entropy, float* dz, int h, int w, int warps) {
  constexpr int kBatch = kAlike ? 2 : 8, kValues = kAlike ? 4 : 1;
  grid_dependents_launch();
  grid_dependency_wait();
  const int threads = 32 * warps;
  const long c = (long)blockIdx.x * (8 / warps) + threadIdx.x / threads;
  if (c >= w) return;
  const float g = grad ? grad[c] : 0.0f, q = grad_entropy ? grad_entropy[c] : 0.0f, H = grad_entropy ? entropy[c] : 0.0f;
  const float m = stats[2 * c], ls = stats[2 * c + 1];
  const int t = g != 0.0f ? token_of(tokens[c], h) : -1;
  const bool zero = (g == 0.0f && q == 0.0f) || m == -INFINITY, bad = g != 0.0f && t < 0;
  const float* col = z + c * h;
  float* out = dz + c * h;
  const int o = kAlike ? offset_in(col) : 0, items = kAlike ? (h + o + 3) >> 2 : h, step = gridDim.y * threads;
  for (int base = blockIdx.y * threads + threadIdx.x % threads; base < items; base += kBatch * step) {
    float v[kBatch][kValues];
#pragma unroll
    for (int b = 0; b < kBatch; b++) {
      const int i = base + b * step;
      if (zero || i >= items) continue;
      if constexpr (kAlike) load_group(col, 4 * i - o, h, 0.0f, v[b]);
      else v[b][0] = col[i];
    }
#pragma unroll
    for (int b = 0; b < kBatch; b++) {
      const int i = base + b * step;
      if (i >= items) continue;
#pragma unroll
      for (int j = 0; j < kValues; j++) {
        float r = 0.0f;
        if (!zero) {
          const float lp = (v[b][j] - m) - ls, p = exp_accurate(lp);
          // -p (g + q (log p + H)), and 0 where p is: log p may be -inf there
          r = p > 0.0f ? -p * (g + q * (lp + H)) : 0.0f * p;
          if (kValues * i + j - o == t) r += g;
          if (bad) r = __int_as_float(0x7fc00000);
        }
        v[b][j] = r;
      }
      if constexpr (kAlike) store_group(out, 4 * i - o, h, v[b]);
      else out[i] = v[b][0];
    }
  }
}

// A row of w values.
int row_ok(const cudamat* v, int w) {
  if (!v) return 0;
  if (!v->on_device) return ERROR_NOT_ON_DEVICE;
  return v->size[0] == 1 && v->size[1] == w ? 0 : ERROR_INCOMPATIBLE_DIMENSIONS;
}

}  // namespace

extern "C" {

int log_prob(cudamat* logits, cudamat* tokens, cudamat* target, cudamat* entropy, cudamat* stats, cudamat* top, cudamat* top_tokens) {
  if (!logits->on_device || (stats && !stats->on_device) || (top && !top->on_device) || (top_tokens && !top_tokens->on_device))
    return ERROR_NOT_ON_DEVICE;
  if (logits->is_trans || (stats && stats->is_trans) || (top && top->is_trans) || (top_tokens && top_tokens->is_trans))
    return ERROR_TRANSPOSED;
  const int h = logits->size[0], w = logits->size[1];
  int err = row_ok(tokens, w);
  if (!err) err = row_ok(target, w);
  if (!err) err = row_ok(entropy, w);
  if (err) return err;
  if ((stats && (stats->size[0] != 2 || stats->size[1] != w)) || !top != !top_tokens ||
      (top && (!same_shape(top, top_tokens) || top->size[1] != w || top->size[0] > h)) || !tokens != !target)
    return ERROR_INCOMPATIBLE_DIMENSIONS;
  if (overlapping({target, entropy, stats, top, top_tokens, logits, unless_in_place(tokens, target)}, 5)) return ERROR_UNSUPPORTED;
  if (w == 0) return 0;
  if (h == 0 || h > (1 << 24) || (top && top->size[0] > kMostTop)) {
    set_error(h == 0 ? "columns without a logit have no distribution"
                     : h > (1 << 24) ? "a float32 does not hold every token of a column" : "at most 32 top tokens a column");
    return ERROR_UNSUPPORTED;
  }
  LogProbArgs a;
  auto at = [](cudamat* v) { return v ? v->data_device : nullptr; };
  a.z = logits->data_device;
  a.tokens = at(tokens);
  a.logp = at(target);
  a.entropy = at(entropy);
  a.stats = at(stats);
  a.top = at(top);
  a.top_tokens = at(top_tokens);
  a.h = h;
  a.w = w;
  a.k = top ? top->size[0] : 0;
  // as many warps a column as fill the device, with sixteen logits a thread or more
  int warps = 1;
  while (warps < 32 && (long)w * warps < 32L * sm_count() && (long)warps * 32 * 16 < h) warps *= 2;
  const int groups = warps < 8 ? 8 / warps : 1;          // columns of a block
  (void)launch_dependent(a.k ? k_log_prob<true> : k_log_prob<false>, dim3((w + groups - 1) / groups), dim3(32 * warps * groups), 0, stream(),
                         a, warps);
  return check_launch();
}

int log_prob_deriv(cudamat* logits, cudamat* tokens, cudamat* stats, cudamat* grad, cudamat* entropy, cudamat* grad_entropy,
                   cudamat* target) {
  if (!logits->on_device || !stats->on_device || !target->on_device) return ERROR_NOT_ON_DEVICE;
  if (logits->is_trans || stats->is_trans || target->is_trans) return ERROR_TRANSPOSED;
  const int h = logits->size[0], w = logits->size[1];
  int err = row_ok(tokens, w);
  if (!err) err = row_ok(grad, w);
  if (!err) err = row_ok(entropy, w);
  if (!err) err = row_ok(grad_entropy, w);
  if (err) return err;
  if (!same_shape(logits, target) || stats->size[0] != 2 || stats->size[1] != w || (grad && !tokens) || (grad_entropy && !entropy))
    return ERROR_INCOMPATIBLE_DIMENSIONS;
  if (overlapping({target, unless_in_place(logits, target), tokens, stats, grad, entropy, grad_entropy}, 1)) return ERROR_UNSUPPORTED;
  if (h == 0 || w == 0) return 0;
  if (h > (1 << 24)) {
    set_error("a float32 does not hold every token of a column");
    return ERROR_UNSUPPORTED;
  }
  auto at = [](cudamat* v) { return v ? v->data_device : nullptr; };
  const float* z = logits->data_device;
  float* dz = target->data_device;
  // a warp a column up to 256 logits, a block from 1024 on, and parts of a column where there are few
  int warps = 1;
  while (warps < 8 && warps * 256 < h) warps *= 2;
  const int per_block = 256 * 8;                         // logits of a block's batch
  int parts = (h + per_block - 1) / per_block;
  while (parts > 1 && (long)w * parts > 16L * sm_count()) parts = (parts + 1) / 2;
  const dim3 grid((w + 8 / warps - 1) / (8 / warps), parts);
  (void)launch_dependent(((uintptr_t)z & 15) == ((uintptr_t)dz & 15) ? k_log_prob_deriv<true> : k_log_prob_deriv<false>, grid, dim3(256), 0,
                         stream(), z, at(tokens), stats->data_device, at(grad), at(entropy), at(grad_entropy), dz, h, w, warps);
  return check_launch();
}

}  // extern "C"
