// Next-token sampling: temperature, top-k, top-p, min-p and the choice by a given
// uniform number, without a sort, with one read of the logits from memory.
//
// Tokens are ordered by (logit, lowest index first); top-k, top-p and min-p each
// keep a prefix of that order, so the kept set is "at or before one token", found
// as follows, and the choice walks the vocabulary in index order:
//   1. the row goes to shared memory (one block, or a cluster whose blocks each hold
//      a slice; wide rows that would take several waves of blocks so are read again from
//      L2 instead); maximum and minimum;
//   2. top-k of at most kShortK: the k-th largest of the threads' own maxima bounds the
//      k-th logit from below, so one pass lists little more than k tokens, and one block
//      goes on over the list;
//   3. top-k: a histogram of 1024 equal steps of the logit finds the step that holds
//      the k-th token, whose tokens are then compared with one another; top-p: the
//      same with the sum of weights in place of the count;
//   4. the choice: over the list, the same again with 1024 parts of the vocabulary as
//      steps; else sums per warp (a contiguous part of the row each), and the warp that
//      holds u * total has its part summed again in pieces.
// A step that holds more tokens than the compare list (equal logits in long runs) is
// cut by 8 bits of the 64-bit order key at a time until the rest fits.
//
// Weights 2^((l - max) log2(e) / T) are 64-bit integers in units of 2^-44: sums do
// not depend on the order of atomics, blocks or warps, and a token on the border of
// top-p or of u is decided alike however the row was split.  A weight is right to
// 2^-29 of itself and one unit (fp32 pairs for the exponent, a table of 64 powers, a short series;
// tests/test_sampling.py restates the steps), so that a sum over n tokens of like
// weight is right to about 2^-29 / sqrt(n) and the choice is that of exact arithmetic
// but for u or top-p in a few parts in 10^8.  (With the weights in 64-bit floating point 256 x 32000 of
// mixed settings took 58 us where these took 46.)  For top-p's border they are rounded to
// 2^-31 (see coarse()), so that a histogram holds its sums as two 32-bit words of 16 bits of the weights
// each: 32-bit adds are what shared memory does fast, and they bound a flat row's pass.
//
// Measured: 1 x 32000 bf16 with top-p 17 us (bound by the barriers of the cluster, about 2 K
// cycles each), 256 x 32000 bf16 of mixed settings 45, 64 x 131072 fp32 with top-p 69 (0.5 TB/s:
// bound by the instructions of the weights and the histogram's atomics, with 32 warps an SM).
#include <cfloat>
#include <stdexcept>
#include <string>

#include "common.cuh"
#include "kernels.h"
#include "vec.cuh"

namespace uhfs {

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 1024;   // two per thread
constexpr int kCap = 512;     // tokens compared with one another at the border
constexpr int kShortK = 256;  // top-k up to which one gathered list does
typedef unsigned long long u64;

constexpr int kMaxSplits = 8;
constexpr int kPowers = 64;   // entries of the table of 2^(i / 64)

// shared memory in front of the row's slice
struct alignas(16) Shared {
  uint32_t part[2][kBins];  // the block's histogram: the weights' lower and upper 16 bits
  uint32_t low[kBins];      // the choice over a list: 13 bits below them
  u64 hist[kBins];          // the same as sums; later the weights of the compared tokens
  u64 list[kCap];           // this block's tokens to compare (order keys)
  u64 warp_sum[kWarps];
  u64 sums[kMaxSplits * kWarps];  // warp_sum of every block
  uint32_t powers[kPowers];
  u64 border;               // order key of the last kept token
  u64 excl, goal;           // sum before the chosen bin; the sum that is looked for
  int bin;
  int count;                // entries of list (may exceed kCap: then not all are stored)
  int n_long;               // the same for the long list
  float mx, mn;             // this block's extremes
  int first;                // lowest index of the maximum in this block
  float warp_mx[kWarps], warp_mn[kWarps];
  int warp_first[kWarps];
};
static_assert(kCap <= kBins, "the compared tokens' weights reuse the histogram");
// behind it: the long list (long_cap order keys); in a cluster, the cluster's tokens to
// compare; the slice, whose place the cluster's long list takes once it is there

// The order: larger keys first.  Equal logits (-0 and 0 too) share the upper half.
__device__ __forceinline__ u64 order_key(float l, int idx) {
  uint32_t k = __float_as_uint(l + 0.f);
  k = (k & 0x80000000u) ? ~k : (k | 0x80000000u);
  return ((u64)k << 32) | (0xffffffffu - (uint32_t)idx);
}
__device__ __forceinline__ int key_index(u64 key) { return (int)(0xffffffffu - (uint32_t)key); }
__device__ __forceinline__ float key_logit(u64 key) {
  uint32_t k = (uint32_t)(key >> 32);
  k = (k & 0x80000000u) ? (k & 0x7fffffffu) : ~k;
  return __uint_as_float(k);
}

// 2^(i / 64) in units of 2^-30, from the series of exp
struct Powers {
  uint32_t v[kPowers];
};
constexpr Powers make_powers() {
  Powers p{};
  for (int i = 0; i < kPowers; ++i) {
    const double y = 0.69314718055994530942 * i / kPowers;
    double e = 1.0, term = 1.0;
    for (int k = 1; k < 24; ++k) {
      term *= y / k;
      e += term;
    }
    p.v[i] = (uint32_t)(e * 1073741824.0 + 0.5);
  }
  return p;
}
__constant__ Powers kPowerTable = make_powers();

struct Row {
  float mx;        // largest logit, finite
  float ch, cl;    // log2(e) / temperature as a sum of two fp32 numbers
  float dmin;      // -44.9 / ch: from there down a weight is 0
};

// 2^44 * 2^((l - max) c): 2^(k / 64) from the table times 1 + (2^r - 1), |r| <= 1/128, the
// latter from its series.  kExact: l - max with its rounding error; without, for 16-bit
// logits, whose difference is exact unless one is 2^15 times the other.
// Two at a time: the fp32 steps as packed f32x2 instructions.
struct Weights {
  u64 a, b;
};
// In units of 2^-31, rounded up or down by the token's place: the multiples of the golden ratio spread the
// thresholds so evenly that a run of equal weights sums to within some units of the truth, however small they are.
// (Rounded to the nearest, 131071 weights of 0.44 units were nothing, and of 1.6 two units each.)
__device__ __forceinline__ uint32_t coarse(u64 w, int idx) {
  return (uint32_t)((w + ((uint32_t)idx * 0x9E3779B1u >> 19)) >> 13);
}
template <bool kExact>
__device__ __forceinline__ Weights weights(const Row& row, const uint32_t* powers, float la, float lb) {
  auto both = [](float x) { return make_float2(x, x); };
  const float2 l = make_float2(la, lb), ch = both(row.ch);
  const float2 d0 = f2_add(l, both(-row.mx)), d = make_float2(fmaxf(d0.x, row.dmin), fmaxf(d0.y, row.dmin));
  const float2 p = f2_mul(d, ch);                            // x = p + q = (l - max) c
  float2 q = f2_fma(d, both(row.cl), f2_fma(d, ch, make_float2(-p.x, -p.y)));
  if constexpr (kExact) {
    const float2 bb = f2_sub(d0, l);
    const float2 e = f2_add(f2_sub(l, f2_sub(d0, bb)), f2_sub(both(-row.mx), bb));
    q = f2_fma(make_float2(d0.x < row.dmin ? 0.f : e.x, d0.y < row.dmin ? 0.f : e.y), ch, q);
  }
  constexpr float kMagic = 12582912.f;                       // 1.5 * 2^23: z's low bits are round(64 p)
  const float2 z = f2_fma(p, both((float)kPowers), both(kMagic));
  const float2 r = f2_add(f2_fma(f2_add(z, both(-kMagic)), both(-1.f / kPowers), p), q);
  // ln2, ln2^2 / 2, ln2^3 / 6
  const float2 em1 = f2_mul(r, f2_fma(r, f2_fma(r, both(0.055504109f), both(0.24022651f)), both(0.69314718f)));
  auto finish = [&](float zk, float e) {
    const int k = __float_as_int(zk);
    const uint32_t m0 = powers[k & (kPowers - 1)];
    const uint32_t m = m0 + (uint32_t)__float2int_rn((float)m0 * e);
    return ((u64)m << 32) >> (18 + (__float_as_int(kMagic) >> 6) - (k >> 6));
  };
  return Weights{finish(z.x, em1.x), finish(z.y, em1.y)};
}

// (no memory clobber: the barriers around them order these loads, and several are in flight at once)
__device__ __forceinline__ u64 peer_u64(const u64* p, int rank) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(smem_cluster_addr(p, rank)));
  return v;
}
__device__ __forceinline__ int peer_int(const int* p, int rank) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(smem_cluster_addr(p, rank)));
  return v;
}
__device__ __forceinline__ float peer_float(const float* p, int rank) {
  return __int_as_float(peer_int(reinterpret_cast<const int*>(p), rank));
}

__device__ __forceinline__ u64 warp_sum_u64(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// kSlice: the block's part of the row is in shared memory; else it is read again from memory (L2)
template <typename T, bool kSlice>
struct Sampler {
  Shared& sh;
  const T* slice;       // this block's part of the row
  int vocab;
  bool vec;             // whether the row can be read in 16-byte pieces
  bool infinite;        // some logits are infinite (only without a slice, whose values are replaced)
  int base;             // index of its first token
  int w_len;            // tokens per warp, a multiple of 8
  int splits;           // blocks that hold the tokens: 1 once they are listed
  u64* all;             // the cluster's tokens to compare
  Row row;
  float step;           // histogram steps per unit of the logit
  const u64* listed;    // the long list (null: the tokens are the slices')
  int n_listed;

  __device__ __forceinline__ void sync() const {
    if (splits > 1) cluster_sync_all();
    else __syncthreads();
  }

  // eight logits of the block's part, -inf for NaN and past the end
  __device__ __forceinline__ void fetch(const T* at, float* l) const {
    if constexpr (kSlice) {
      load8<T>(at, l);
    } else {
      const int left = vocab - (base + (int)(at - slice));
      if (vec && left >= 8) {
        load8<T>(at, l);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) l[i] = i < left ? to_float<T>(at[i]) : -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) l[i] = fmaxf(l[i], -INFINITY);  // (drops NaN)
      if (infinite) {
#pragma unroll
        for (int i = 0; i < 8; ++i) l[i] = l[i] == INFINITY ? 0.f : -INFINITY;
      }
    }
  }
  // one of those within the vocabulary that is not NaN
  __device__ __forceinline__ float fetch_one(const T* at) const {
    const float l = to_float<T>(*at);
    return !kSlice && infinite ? (l == INFINITY ? 0.f : -INFINITY) : l;
  }

  // f(logit, index) for the listed tokens, or this warp's and, as -inf, the padding behind them
  template <class Fn>
  __device__ __forceinline__ void each(Fn&& f) const {
    if (listed != nullptr) {
      for (int i = threadIdx.x; i < n_listed; i += kThreads) f(key_logit(listed[i]), key_index(listed[i]));
      return;
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const T* part = slice + warp * w_len;
    for (int v = lane * 8; v < w_len; v += 256) {
      float l[8];
      fetch(part + v, l);
#pragma unroll
      for (int i = 0; i < 8; ++i) f(l[i], base + warp * w_len + v + i);
    }
  }

  // f(two logits, index of the first) for this warp's tokens
  template <class Fn>
  __device__ __forceinline__ void each_pair(Fn&& f) const {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const T* part = slice + warp * w_len;
    for (int v = lane * 8; v < w_len; v += 256) {
      float l[8];
      fetch(part + v, l);
#pragma unroll
      for (int i = 0; i < 8; i += 2) f(l[i], l[i + 1], base + warp * w_len + v + i);
    }
  }

  __device__ __forceinline__ Weights weigh(float la, float lb) const {
    return weights<sizeof(T) == 4>(row, sh.powers, la, lb);
  }
  __device__ __forceinline__ u64 weigh(float l) const { return weigh(l, l).a; }

  // equal steps of the logit; the last takes everything 2^64 below the largest weight, and -inf
  __device__ __forceinline__ int bin_of(float l) const {
    return (int)fminf((row.mx - l) * step, (float)(kBins - 1));  // (NaN, from a step of 0: the last)
  }

  // The sum of v, which is a warp's own, over all warps of the cluster; *before: over those ahead
  __device__ __forceinline__ u64 sum_all(u64 v, int rank, u64* before) const {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) sh.warp_sum[warp] = v;
    sync();
    const int n = splits * kWarps;
    if (threadIdx.x < n)
      sh.sums[threadIdx.x] = splits > 1 ? peer_u64(&sh.warp_sum[threadIdx.x % kWarps], threadIdx.x / kWarps)
                                        : sh.warp_sum[threadIdx.x];
    __syncthreads();
    u64 total = 0, ahead = 0;
    for (int i = lane; i < n; i += 32) {
      const u64 x = sh.sums[i];
      if (i < rank * kWarps + warp) ahead += x;
      total += x;
    }
    *before = warp_sum_u64(ahead);
    return warp_sum_u64(total);
  }

  __device__ __forceinline__ void clear(int words, int bins) {
    for (int k = 0; k < words; ++k)
      for (int i = threadIdx.x; i < bins; i += kThreads) sh.part[k][i] = 0;
    __syncthreads();
  }
  // adds to the block's histogram (at most 2^16 tokens); w: at most 2^31, or a count of 1
  template <bool kWeights>
  __device__ __forceinline__ void add(int bin, uint32_t w) {
    if constexpr (!kWeights) {
      atomicAdd(&sh.part[0][bin], 1u);
    } else if (w != 0) {
      atomicAdd(&sh.part[0][bin], w & 0xffffu);
      if (w > 0xffffu) atomicAdd(&sh.part[1][bin], w >> 16);
    }
  }

  // First bin whose inclusive sum over the cluster reaches the goal, a whole number
  // from 1 to the sum of all bins that goal_of(sum) gives; sets sh.bin and sh.excl.
  template <class Fn>
  __device__ __forceinline__ u64 find_bin(int words, int bins, Fn&& goal_of) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    __syncthreads();
    u64 v[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int bin = threadIdx.x * 2 + i;
      if (bin < bins) {
        v[i] = sh.part[0][bin];
        if (words > 1) v[i] += (u64)sh.part[1][bin] << 16;
        if (words > 2) v[i] = (v[i] << 13) + sh.low[bin];
        if (splits > 1) sh.hist[bin] = v[i];
      }
    }
    // in a cluster the first block adds the blocks' sums and decides (all of them doing so
    // took four times as long: 64 KB of peers' shared memory each)
    const bool decide = splits == 1 || cluster_ctarank() == 0;
    if (splits > 1) {
      cluster_sync_all();
      if (decide) {
        u64 x[2][kMaxSplits];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int r = 0; r < kMaxSplits; ++r) {
            const int bin = threadIdx.x * 2 + i;
            x[i][r] = r < splits && bin < bins ? peer_u64(&sh.hist[bin], r) : 0;
          }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          v[i] = 0;
#pragma unroll
          for (int r = 0; r < kMaxSplits; ++r) v[i] += x[i][r];
        }
      }
    }
    if (decide) {
      u64 incl = v[0] + v[1];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
      }
      if (lane == 31) sh.warp_sum[warp] = incl;
      __syncthreads();
      u64 before = 0, total = 0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += sh.warp_sum[w];
        total += sh.warp_sum[w];
      }
      const u64 goal = goal_of(total);
      u64 excl = before + incl - v[0] - v[1];
      if (threadIdx.x == 0) sh.goal = goal;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (excl < goal && excl + v[i] >= goal) {
          sh.bin = threadIdx.x * 2 + i;
          sh.excl = excl;
        }
        excl += v[i];
      }
    }
    if (splits == 1) {
      __syncthreads();
      return sh.goal;
    }
    cluster_sync_all();
    if (!decide) {
      if (threadIdx.x == 0) sh.bin = peer_int(&sh.bin, 0);
      if (threadIdx.x == 32) sh.excl = peer_u64(&sh.excl, 0);
      if (threadIdx.x == 64) sh.goal = peer_u64(&sh.goal, 0);
    }
    __syncthreads();
    return sh.goal;
  }

  // Copies the blocks' lists (counts at `count`, order keys at `from`) to `to` unless they
  // are more than cap; returns how many.
  __device__ __forceinline__ int collect(const int* count, const u64* from, u64* to, int cap) const {
    const int lane = threadIdx.x & 31;
    const int mine = lane < splits ? peer_int(count, lane) : 0;
    int incl = mine;
#pragma unroll
    for (int o = 1; o < kMaxSplits; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    const int n = __shfl_sync(0xffffffffu, incl, splits - 1);
    if (n > cap) return n;
    // two warps for the list of each block
    for (int w = threadIdx.x >> 5; w < 2 * splits; w += kWarps) {
      const int r = w >> 1;
      const int m = __shfl_sync(0xffffffffu, mine, r), at = __shfl_sync(0xffffffffu, incl, r) - m;
      for (int i = lane + 32 * (w & 1); i < m; i += 64) to[at + i] = peer_u64(&from[i], r);
    }
    __syncthreads();
    return n;
  }

  // Appends the order keys of the tokens for which open(logit, index) holds to a list of
  // `cap`; *count counts on beyond it.  Only logits in [lo, hi] are asked about.
  template <class Open>
  __device__ __forceinline__ void push(float lo, float hi, Open&& open, u64* list, int* count, int cap) const {
    auto append = [&](float l, int idx) {
      if (open(l, idx)) {
        const int n = atomicAdd(count, 1);
        if (n < cap) list[n] = order_key(l, idx);
      }
    };
    if (listed != nullptr) {
      each(append);
      return;
    }
    // eight comparisons, then the few tokens that pass, read again
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const T* part = slice + warp * w_len;
    for (int v = lane * 8; v < w_len; v += 256) {
      float l[8];
      fetch(part + v, l);
      const int idx = base + warp * w_len + v;
      uint32_t mask = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) mask |= l[i] >= lo && l[i] <= hi ? 1u << i : 0u;
      // (a list that has run over is not used: no need to go on)
      if (mask != 0 && *(volatile int*)count > cap) return;
      while (mask != 0) {
        const int i = __ffs(mask) - 1;
        mask &= mask - 1;
        append(fetch_one(part + v + i), idx + i);
      }
    }
  }

  // Logits that can fall into steps first..last, with room for the roundings (and no -inf)
  __device__ __forceinline__ float step_low(int last) const {
    if (last >= kBins - 1 || !(step > 0.f)) return -FLT_MAX;
    const float d = (float)(last + 1) / step;
    return row.mx - d - (fabsf(row.mx) + d) * 1e-6f;
  }
  __device__ __forceinline__ float step_high(int first) const {
    if (first <= 0 || !(step > 0.f)) return FLT_MAX;
    const float d = (float)first / step;
    return row.mx - d + (fabsf(row.mx) + d) * 1e-6f;
  }

  // Lists the tokens for which open(logit, index) holds.  Returns how many; up to kCap
  // of them, `keys` (sh.list or `all`) holds their order keys, unordered.
  template <class Open>
  __device__ __forceinline__ int gather(float lo, float hi, Open&& open, const u64*& keys) {
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    push(lo, hi, open, sh.list, &sh.count, kCap);
    sync();
    keys = splits == 1 ? sh.list : all;
    return splits == 1 ? sh.count : collect(&sh.count, sh.list, all, kCap);
  }

  // Order key of the token at which the running sum, in order, of the counts or weights
  // of the tokens at or before `border` reaches its goal.
  template <bool kWeights, class Goal>
  __device__ __forceinline__ u64 select(u64 border, Goal&& goal_of) {
    constexpr int kWords = kWeights ? 2 : 1;
    auto val = [&](float l, int idx) -> uint32_t { return kWeights ? coarse(weigh(l), idx) : 1; };
    clear(kWords, kBins);
    if (listed != nullptr || !kWeights || border != 0) {
      each([&](float l, int idx) {
        if (l > -INFINITY && order_key(l, idx) >= border) add<kWeights>(bin_of(l), val(l, idx));
      });
    } else {
      each_pair([&](float la, float lb, int idx) {
        const Weights w = weigh(la, lb);
        add<kWeights>(bin_of(la), coarse(w.a, idx));
        add<kWeights>(bin_of(lb), coarse(w.b, idx + 1));
      });
    }
    const u64 goal = find_bin(kWords, kBins, goal_of);
    const int bin = sh.bin;
    u64 sum = sh.excl;   // of the tokens before those still in question
    int shift = 64;      // the upper 64 - shift bits of their keys are `prefix`
    u64 prefix = 0;
    while (true) {
      const u64* list;
      const int n = gather(
          step_low(bin), step_high(bin),
          [&](float l, int idx) {
            if (bin_of(l) != bin) return false;
            const u64 key = order_key(l, idx);
            return key >= border && (shift == 64 || (key >> shift) == prefix);
          },
          list);
      if (n <= kCap) {
        u64* w = sh.hist;  // (every block has passed the gather's barrier: the histogram has been read)
        for (int i = threadIdx.x; i < n; i += kThreads) w[i] = val(key_logit(list[i]), key_index(list[i]));
        if (threadIdx.x == 0) sh.border = 0;
        __syncthreads();
        // the blocks share the tokens out; eight lanes compare one with all others
        const int sub = threadIdx.x % 8, rank = splits > 1 ? (int)cluster_ctarank() : 0;
        for (int i0 = rank * (kThreads / 8); i0 < n; i0 += splits * (kThreads / 8)) {
          const int i = i0 + threadIdx.x / 8;
          const u64 key = i < n ? list[i] : 0;
          u64 before = 0;
          if (i < n)
#pragma unroll 4
            for (int j = sub; j < n; j += 8) {
              const u64 other = list[j], v = w[j];  // (both loads, then the choice: they overlap)
              before += other > key ? v : 0;
            }
#pragma unroll
          for (int o = 1; o < 8; o <<= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
          before += sum;
          if (i < n && sub == 0 && before < goal && before + w[i] >= goal) sh.border = key;
        }
        sync();  // one block has the border; the peers have read this block's list
        if (splits == 1) return sh.border;
        const int lane = threadIdx.x & 31;
        u64 found = lane < splits ? peer_u64(&sh.border, lane) : 0;
#pragma unroll
        for (int o = 1; o < kMaxSplits; o <<= 1) found = max(found, __shfl_xor_sync(0xffffffffu, found, o));
        sync();  // every block has read it
        return __shfl_sync(0xffffffffu, found, 0);
      }
      // too many: the next 8 bits of the key, largest first
      shift -= 8;
      clear(kWords, 256);
      each([&](float l, int idx) {
        const u64 key = order_key(l, idx);
        if (l > -INFINITY && key >= border && bin_of(l) == bin && (shift == 56 || (key >> (shift + 8)) == prefix))
          add<kWeights>(255 - (int)((key >> shift) & 255), val(l, idx));
      });
      const u64 left = sum;
      find_bin(kWords, 256, [&](u64) { return goal - left; });
      sum = left + sh.excl;
      prefix = (prefix << 8) | (u64)(255 - sh.bin);
      sync();  // the histogram and the counts have been read
    }
  }
};

// The running sum that the chosen token is the first to pass (0 <= goal < total)
__device__ __forceinline__ u64 choice(float u, u64 total) {
  const double want = fmin(fmax((double)u, 0.0), 1.0) * (double)total;  // NaN: 0
  const u64 goal = want >= (double)total ? total - 1 : (u64)want;
  return goal < total ? goal : total - 1;
}

template <typename T, bool kSlice>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const SampleArgs a) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  Shared& sh = *reinterpret_cast<Shared*>(smem_raw);
  const int splits = a.splits, long_cap = a.long_cap;
  u64* long_list = reinterpret_cast<u64*>(smem_raw + sizeof(Shared));
  u64* compare = long_list + long_cap;  // (with more than one block)
  u64* cluster_list = splits > 1 ? compare + kCap : compare;
  T* slice = reinterpret_cast<T*>(cluster_list);  // (kSlice)
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x % splits;
  const long long r = blockIdx.x / splits;
  const int w_len = a.warp_len, len = w_len * kWarps, base = rank * len;
  const T* src = static_cast<const T*>(a.logits) + r * a.ld;

  if (threadIdx.x < kPowers) sh.powers[threadIdx.x] = kPowerTable.v[threadIdx.x];

  // 1. the slice; tokens that cannot be chosen (NaN, past the end) become -inf
  float mx = -INFINITY, mn = INFINITY;
  auto take = [&](int v, float* l) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (!(l[i] > -INFINITY)) l[i] = -INFINITY;
      else {
        mx = fmaxf(mx, l[i]);
        mn = fminf(mn, l[i]);
      }
    }
    if constexpr (kSlice) store8<T>(slice + v, l);
  };
  int v = threadIdx.x * 8;
  constexpr int kStep = kThreads * 8;
  if (a.vec) {
    const int whole = min(len, a.vocab - base);  // (may be negative)
    for (; v + 3 * kStep + 8 <= whole; v += 4 * kStep) {  // four loads in flight
      float l[4][8];
#pragma unroll
      for (int k = 0; k < 4; ++k) load8<T>(src + base + v + k * kStep, l[k]);
#pragma unroll
      for (int k = 0; k < 4; ++k) take(v + k * kStep, l[k]);
    }
    for (; v + 8 <= whole; v += kStep) {
      float l[8];
      load8<T>(src + base + v, l);
      take(v, l);
    }
  }
  for (; v < len; v += kStep) {
    float l[8];
    const int left = a.vocab - (base + v);
#pragma unroll
    for (int i = 0; i < 8; ++i) l[i] = i < left ? to_float<T>(src[base + v + i]) : -INFINITY;
    take(v, l);
  }
  const float own = mx;  // this thread's maximum
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
  }
  if (lane == 0) {
    sh.warp_mx[warp] = mx;
    sh.warp_mn[warp] = mn;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    mx = fmaxf(mx, sh.warp_mx[w]);
    mn = fminf(mn, sh.warp_mn[w]);
  }
  if (splits > 1) {
    if (threadIdx.x == 0) {
      sh.mx = mx;
      sh.mn = mn;
    }
    cluster_sync_all();
    if (lane < splits) {
      mx = peer_float(&sh.mx, lane);
      mn = peer_float(&sh.mn, lane);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    }
  }
  Sampler<T, kSlice> s{sh,    kSlice ? slice : src + base, a.vocab, a.vec != 0, false, base, w_len, splits, compare,
                       Row{}, 0.f, nullptr, 0};

  const double temp = a.temperature_rows != nullptr ? (double)a.temperature_rows[r] : a.temperature;
  const int top_k = a.top_k_rows != nullptr ? a.top_k_rows[r] : a.top_k;
  const double top_p = a.top_p_rows != nullptr ? (double)a.top_p_rows[r] : a.top_p;
  const double min_p = a.min_p_rows != nullptr ? (double)a.min_p_rows[r] : a.min_p;
  const float u = a.uniform[r];

  if (mx == -INFINITY || !(temp > 0.0)) {
    // nothing to choose from, or the largest logit's first token
    int first = 0x7fffffff;
    if (mx > -INFINITY) s.each([&](float l, int idx) {
      if (l == mx) first = min(first, idx);
    });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) first = min(first, __shfl_xor_sync(0xffffffffu, first, o));
    if (lane == 0) sh.warp_first[warp] = first;
    __syncthreads();
    for (int w = 0; w < kWarps; ++w) first = min(first, sh.warp_first[w]);
    if (threadIdx.x == 0) sh.first = first;
    s.sync();
    if (rank == 0 && threadIdx.x == 0) {
      for (int k = 1; k < splits; ++k) first = min(first, peer_int(&sh.first, k));
      a.tokens[r] = mx > -INFINITY ? first : -1;
    }
    if (splits > 1) cluster_sync_all();  // no block leaves while it is read
    return;
  }

  float largest = own;
  if (mx == INFINITY) {
    // infinite logits have all the weight, alike: 0 in their place, -inf in the others'
    if constexpr (kSlice) {
      __syncthreads();
      T* part = slice + warp * w_len;
      for (int i = lane; i < w_len; i += 32)
        part[i] = from_float<T>(to_float<T>(part[i]) == INFINITY ? 0.f : -INFINITY);
      __syncthreads();
    } else {
      s.infinite = true;
    }
    largest = own == INFINITY ? 0.f : -INFINITY;
    mx = mn = 0.f;
  }
  // between 1e-30 (below, only the largest logit has a weight) and 1e30 the products stay finite
  const double c = 1.4426950408889634 / fmin(fmax(temp, 1e-30), 1e30);
  s.row.mx = mx;
  s.row.ch = (float)c;
  s.row.cl = (float)(c - (double)s.row.ch);
  s.row.dmin = -44.9f / s.row.ch;
  // min-p as the least weight; the largest weight, 2^44, always passes
  const u64 least = min_p > 0.0 ? (u64)(fmin(min_p, 1.0) * 17592186044416.0) : 0;
  const float range = fminf(mx - mn, 64.f / s.row.ch);
  s.step = range > 0.f ? (kBins - 1) / range : 0.f;

  u64 border = 0;  // every token
  const bool cut_k = top_k > 0 && top_k < a.vocab, short_k = cut_k && top_k <= kShortK;
  if (short_k) {
    // 2. the long list
    if (threadIdx.x == 0) sh.n_long = 0;
    // the step of the k-th of the threads' maxima: k of this block's tokens at least lie at or above it
    s.clear(1, kBins);
    if (largest > -INFINITY) s.template add<false>(s.bin_of(largest), 1);
    s.splits = 1;
    u64 maxima = 0;
    s.find_bin(1, kBins, [&](u64 t) {
      maxima = t;
      return min((u64)top_k, t);
    });
    s.splits = splits;
    const int last_bin = maxima < (u64)top_k ? kBins - 1 : sh.bin;  // too few threads have tokens: all of them
    s.push(s.step_low(last_bin), FLT_MAX, [&](float l, int) { return s.bin_of(l) <= last_bin; }, long_list,
           &sh.n_long, long_cap);
    s.sync();
    int n = sh.n_long;
    const u64* list = long_list;
    if (splits > 1) {
      n = s.collect(&sh.n_long, long_list, cluster_list, long_cap);
      list = cluster_list;
    }
    if (n <= long_cap) {
      if (splits > 1) cluster_arrive();  // (the lists have been read)
      if (rank != 0) {
        cluster_wait();  // no block leaves while its list is read
        return;
      }
      // one block goes on over the list
      s.splits = 1;
      s.listed = list;
      s.n_listed = n;
    } else {
      s.sync();  // the counts have been read
    }
  }
  // 3. the last token that is kept
  if (cut_k) border = s.template select<false>(border, [&](u64 t) { return min((u64)top_k, t); });
  if (top_p < 1.0)
    border = s.template select<true>(border, [&](u64 t) {
      // the fewest whose sum is at least top_p of the whole; at least one unit, which keeps the first
      return min((u64)fmax(ceil(top_p * (double)t), 1.0), t);
    });
  const float last = border != 0 ? key_logit(border) : -INFINITY;
  const int last_idx = border != 0 ? key_index(border) : 0x7fffffff;
  auto is_kept = [&](float l, int idx) { return l > last || (l == last && idx <= last_idx); };
  auto kept = [&](float l, int idx) -> u64 {
    if (!is_kept(l, idx)) return 0;
    const u64 w = s.weigh(l);
    return w >= least ? w : 0;
  };

  if (s.listed != nullptr) {
    // 4. the part of the vocabulary that passes u times the sum, and the token in it
    const int width = (a.vocab + kBins - 1) / kBins;
    s.clear(2, kBins);
    for (int i = threadIdx.x; i < kBins; i += kThreads) sh.low[i] = 0;
    __syncthreads();
    s.each([&](float l, int idx) {
      if (!is_kept(l, idx)) return;
      // 2^44 as 13 low bits and 32 more
      const u64 w = kept(l, idx);
      s.template add<true>(idx / width, (uint32_t)(w >> 13));
      if (w & 0x1fffu) atomicAdd(&sh.low[idx / width], (uint32_t)w & 0x1fffu);
    });
    const u64 goal = s.find_bin(3, kBins, [&](u64 t) { return choice(u, t) + 1; });
    const int part = sh.bin;
    const u64 before = sh.excl;
    const u64* keys;
    const int m = s.gather(-FLT_MAX, FLT_MAX, [&](float l, int idx) { return is_kept(l, idx) && idx / width == part; }, keys);
    u64* w = sh.hist;
    for (int i = threadIdx.x; i < m; i += kThreads) w[i] = kept(key_logit(keys[i]), key_index(keys[i]));
    __syncthreads();
    for (int i = threadIdx.x; i < m; i += kThreads) {
      const int idx = key_index(keys[i]);
      u64 at = before;
      for (int j = 0; j < m; ++j)
        if (key_index(keys[j]) < idx) at += w[j];
      if (at < goal && goal <= at + w[i]) a.tokens[r] = idx;
    }
    if (splits > 1) cluster_wait();
    return;
  }

  // 4. sums per warp, in the order of the vocabulary; the warp's part that holds u times the whole
  u64 sum = 0;
  s.each_pair([&](float la, float lb, int idx) {
    const bool ka = is_kept(la, idx), kb = is_kept(lb, idx + 1);
    if (ka || kb) {
      const Weights w = s.weigh(la, lb);
      if (ka && w.a >= least) sum += w.a;
      if (kb && w.b >= least) sum += w.b;
    }
  });
  sum = warp_sum_u64(sum);
  u64 before = 0;  // of the warps ahead of this one
  const u64 total = s.sum_all(sum, rank, &before);
  // first token whose running sum passes u * total (the largest weight is 2^44 units: total > 0)
  const u64 goal = choice(u, total);
  if (threadIdx.x == 0) sh.bin = -1;
  __syncthreads();
  if (lane == 0 && before <= goal && goal < before + sum) {
    sh.bin = warp;
    sh.excl = before;
  }
  __syncthreads();
  if (sh.bin >= 0) {
    // this block has the token: its warps take 256 tokens each of that warp's part
    const T* part = s.slice + sh.bin * w_len;
    const int v = (int)threadIdx.x * 8, idx = base + sh.bin * w_len + v;
    u64 w[8], mine = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = 0;
    if (v < w_len) {
      float l[8];
      s.fetch(part + v, l);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        w[i] = kept(l[i], idx + i);
        mine += w[i];
      }
    }
    u64 incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    if (lane == 31) sh.sums[warp] = incl;
    __syncthreads();
    u64 at = sh.excl + incl - mine;
    for (int k = 0; k < warp; ++k) at += sh.sums[k];
    if (at <= goal && goal < at + mine) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (at <= goal && goal < at + w[i]) a.tokens[r] = idx + i;
        at += w[i];
      }
    }
  }
  if (splits > 1) cluster_sync_all();  // no block leaves while its sums are read
}

template <typename T, bool kSlice>
void launch_splits(SampleArgs a, int splits, cudaStream_t s) {
  const int tile = kWarps * 8;
  a.splits = splits;
  a.warp_len = (int)(((long long)a.vocab + (long long)splits * tile - 1) / ((long long)splits * tile)) * 8;
  if (a.warp_len > kThreads * 8) throw std::runtime_error("sample: the vocabulary is too large");
  constexpr size_t kMaxSmem = 227 * 1024;
  a.long_cap = 2048;
  size_t smem;
  while (true) {  // a large vocabulary leaves less room (none is right too: the slices are used)
    const size_t own = kSlice ? (size_t)a.warp_len * kWarps * sizeof(T) : 0, list = (size_t)a.long_cap * sizeof(u64);
    smem = sizeof(Shared) + list + (splits > 1 ? kCap * sizeof(u64) + (own > list ? own : list) : own);
    if (smem <= kMaxSmem || a.long_cap == 0) break;
    a.long_cap = a.long_cap > 256 ? a.long_cap / 2 : 0;
  }
  if (smem > kMaxSmem) throw std::runtime_error("sample: the vocabulary does not fit the shared memory of 8 blocks");
  static PerDeviceOnce once;
  once([] {
    UHFS_CUDA_CHECK(
        cudaFuncSetAttribute(sample_kernel<T, kSlice>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMaxSmem));
  });
  if ((long long)a.rows * splits > 0x7fffffffll) throw std::runtime_error("sample: too many rows");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(a.rows * splits));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)splits;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = splits > 1 ? 1 : 0;
  UHFS_CUDA_CHECK(cudaLaunchKernelEx(&cfg, sample_kernel<T, kSlice>, (const SampleArgs)a));
  note_launch();
}

template <typename T>
void launch_sample(const SampleArgs& a, cudaStream_t s) {
  // Blocks per row: while they fit the GPU, one on each SM, when rows are few, and as many as
  // it takes to hold the row in 64 KB of each (then two blocks fit an SM).  Eight only for
  // up to 8 rows (clusters of eight wait for room: 16 x 32000 took 21 us, with four 18; one row 15.5
  // and 16.6), two on each SM no more (128 x 32000: 31 us, with one block a row 29), and at least
  // 4096 tokens to a block (1 x 4000: 14.5 us with two, 11 with one).
  const long long rows = a.rows, vocab = a.vocab;
  int splits = 1;
  while (splits < kMaxSplits &&
         (rows * splits * 2 <= (splits < 4 ? 148 : 64) || vocab * (int)sizeof(T) > splits * 65536ll) &&
         vocab > (long long)splits * kThreads * 8)
    splits *= 2;
  if (rows * splits > 2 * 148) {
    // More blocks than run at once: fewer that read the row again from L2 instead of keeping it (2^16
    // tokens to a block at most), where these are three quarters of what runs at once.  Rows that are in
    // L2: 64 x 131072 fp32 69 us, 85 with slices; 256 x 50000 fp32 85 and 129; 512 x 32000 fp32, top-k 50,
    // 37 and 60 (rows from memory: 90 and 91, 90 and 131, 42 and 67).  100 x 131072 bf16, whose 200
    // blocks leave half the SMs one: 104 and 87.
    int few = 1;
    while (few < kMaxSplits && (rows * few * 2 <= 2 * 148 || vocab > few * 65536ll)) few *= 2;
    if (few < splits && rows * few * 4 >= 2 * 148 * 3) return launch_splits<T, false>(a, few, s);
  }
  launch_splits<T, true>(a, splits, s);
}

}  // namespace

void sample_tokens(const SampleArgs& p, int dtype, cudaStream_t s) {
  if (p.rows <= 0) return;
  if (p.vocab <= 0) throw std::runtime_error("sample: empty vocabulary");
  SampleArgs a = p;
  const int elem = dtype == DT_F32 ? 4 : 2;
  a.vec = reinterpret_cast<uintptr_t>(p.logits) % 16 == 0 && (p.ld * elem) % 16 == 0;
  switch (dtype) {
    case DT_F32: launch_sample<float>(a, s); break;
    case DT_F16: launch_sample<__half>(a, s); break;
    case DT_BF16: launch_sample<__nv_bfloat16>(a, s); break;
    default: throw std::runtime_error("unsupported dtype");
  }
}

}  // namespace uhfs
