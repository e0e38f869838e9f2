// Next-token sampling: temperature, top-k, top-p, min-p and the choice by a given
// uniform number, without a sort, with one read of the logits.
//
// Tokens are ordered by (logit, lowest index first); top-k, top-p and min-p each
// keep a prefix of that order, so the kept set is "at or before one token", found
// as follows, and the choice walks the vocabulary in index order:
//   1. the row goes to shared memory (one block, or a cluster whose blocks each hold
//      a slice); maximum and minimum;
//   2. top-k of at most kShortK: the k-th largest of the threads' own maxima bounds
//      the k-th logit from below, so one pass gathers little more than k tokens and
//      the rest, top-p and the choice included, is done on that list;
//   3. otherwise, for top-k: a histogram of 1024 equal steps of the logit finds the
//      step that holds the k-th token, whose tokens are then compared with one
//      another; for top-p: the same with the sum of weights in place of the count;
//   4. sums of the kept weights per warp (a contiguous part of the row each); the warp
//      that holds u * total walks its part again.
// A step that holds more tokens than the list (equal logits in long runs) is cut by
// 8 bits of the 64-bit order key at a time until the rest fits.
//
// Weights 2^((l - max) log2(e) / T) are 64-bit integers in units of 2^-44: sums do
// not depend on the order of atomics, blocks or warps, and a token on the border of
// top-p or of u is decided alike however the row was split.  A weight is right to
// 2^-29 of itself (fp32 pairs for the exponent, a table of 64 powers, a short series;
// tests/test_sampling.py restates the steps), so that a sum over n tokens of like
// weight is right to about 2^-29 / sqrt(n) and the choice is that of exact arithmetic
// but for u in a few parts in 10^8.  In 64-bit floating point the same choice took
// 1.5 to 2 times the kernel's time.  A histogram holds its sums as three 32-bit words
// of 15 bits of the weights each (shared memory adds 32-bit words at full rate).
//
// Bound by latency for a few rows (a cluster joins its blocks four or five times), by
// the passes over shared memory for many.
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
constexpr int kCap = 1024;    // tokens compared with one another at the border
constexpr int kShortK = 256;  // top-k up to which one gathered list does
typedef unsigned long long u64;

constexpr int kMaxSplits = 8;
constexpr int kPowers = 64;   // entries of the table of 2^(i / 64)

// shared memory in front of the row's slice
struct alignas(16) Shared {
  uint32_t part[3][kBins];  // the block's histogram: bits 0..14, 15..29, 30..44 of the weights
  u64 hist[kBins];          // the same as sums; later the weights of the listed tokens
  u64 list[kCap];           // this block's listed tokens (order keys)
  u64 all[kCap];            // the cluster's
  u64 warp_sum[kWarps];
  u64 sums[kMaxSplits * kWarps];  // warp_sum of every block
  uint32_t powers[kPowers];
  u64 border;               // order key of the last kept token
  u64 excl;                 // sum before the chosen bin
  int bin;
  int count;                // entries of list (may exceed kCap: then not all are stored)
  float mx, mn;             // this block's extremes
  int first;                // lowest index of the maximum in this block
  float warp_mx[kWarps], warp_mn[kWarps];
  int warp_first[kWarps];
};
static_assert(kCap <= kBins, "the listed tokens' weights reuse the histogram");

// The order: larger keys first.  Equal logits (-0 and 0 too) share the upper half.
__device__ __forceinline__ u64 order_key(float l, int idx) {
  uint32_t k = __float_as_uint(l + 0.f);
  k = (k & 0x80000000u) ? ~k : (k | 0x80000000u);
  return ((u64)k << 32) | (0xffffffffu - (uint32_t)idx);
}
__device__ __forceinline__ float key_logit(u64 key) {
  uint32_t k = (uint32_t)(key >> 32);
  k = (k & 0x80000000u) ? (k & 0x7fffffffu) : ~k;
  return __uint_as_float(k);
}

// 2^(i / 64) in units of 2^-31, from the series of exp
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
    p.v[i] = (uint32_t)(e * 2147483648.0 + 0.5);
  }
  return p;
}
__constant__ Powers kPowerTable = make_powers();

struct Row {
  float mx;        // largest logit
  float ch, cl;    // log2(e) / temperature as a sum of two fp32 numbers
};

// 2^44 * 2^((l - max) c): 2^(k / 64) from the table and 2^r - 1 from its series, |r| <= 1/128
__device__ __forceinline__ u64 weight(const Row& row, const uint32_t* powers, float l) {
  // x = p + q = (l - max) * c to about 2^-46 of itself
  const float d = l == row.mx ? 0.f : l - row.mx, bb = d - l;
  const float e = (l - (d - bb)) + (-row.mx - bb);
  const float p = d * row.ch;
  const float q = fmaf(d, row.cl, fmaf(l == row.mx ? 0.f : e, row.ch, fmaf(d, row.ch, -p)));
  if (!(p > -46.f)) return 0;
  const float kf = rintf(p * (float)kPowers);
  const float t = (fmaf(kf, -1.f / kPowers, p) + q) * 0.69314718f;
  const float em1 = fmaf(fmaf(fmaf(t, 1.f / 24, 1.f / 6), t, 0.5f), t * t, t);
  const int k = (int)kf;
  const uint32_t m = powers[k & (kPowers - 1)];
  const u64 w = (u64)m + (u64)(int64_t)__float2int_rn((float)m * em1);
  return (w << 13) >> (-(k >> 6));
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

template <typename T>
struct Sampler {
  Shared& sh;
  const T* slice;       // this block's part of the row in shared memory
  int base;             // index of its first token
  int w_len;            // tokens per warp, a multiple of 8
  int splits;
  Row row;
  float step;           // histogram steps per unit of the logit

  __device__ __forceinline__ void sync() const {
    if (splits > 1) cluster_sync_all();
    else __syncthreads();
  }

  // f(logit, index) for this warp's tokens (-inf ones, padding among them, left out)
  template <class Fn>
  __device__ __forceinline__ void each(Fn&& f) const {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const T* part = slice + warp * w_len;
    for (int v = lane * 8; v < w_len; v += 256) {
      float l[8];
      load8<T>(part + v, l);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (l[i] > -INFINITY) f(l[i], base + warp * w_len + v + i);
    }
  }

  __device__ __forceinline__ u64 weigh(float l) const { return weight(row, sh.powers, l); }

  // equal steps of the logit; the last takes everything 2^64 below the largest weight
  __device__ __forceinline__ int bin_of(float l) const {
    return l == row.mx ? 0 : (int)fminf((row.mx - l) * step, (float)(kBins - 1));
  }

  __device__ __forceinline__ void clear(int words, int bins) {
    for (int k = 0; k < words; ++k)
      for (int i = threadIdx.x; i < bins; i += kThreads) sh.part[k][i] = 0;
    __syncthreads();
  }
  // adds to the block's histogram; kWeights: a weight below 2^45, else a count
  template <bool kWeights>
  __device__ __forceinline__ void add(int bin, u64 w) {
    if constexpr (!kWeights) {
      atomicAdd(&sh.part[0][bin], 1u);
    } else {
      const uint32_t a = (uint32_t)w & 0x7fffu, b = (uint32_t)(w >> 15) & 0x7fffu, c = (uint32_t)(w >> 30);
      if (a) atomicAdd(&sh.part[0][bin], a);
      if (b) atomicAdd(&sh.part[1][bin], b);
      if (c) atomicAdd(&sh.part[2][bin], c);
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
        if (words == 3) v[i] += ((u64)sh.part[1][bin] << 15) + ((u64)sh.part[2][bin] << 30);
        if (splits > 1) sh.hist[bin] = v[i];
      }
    }
    if (splits > 1) {
      cluster_sync_all();
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
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (excl < goal && excl + v[i] >= goal) {
        sh.bin = threadIdx.x * 2 + i;
        sh.excl = excl;
      }
      excl += v[i];
    }
    __syncthreads();
    return goal;
  }

  // Lists the cluster's tokens for which open(logit, index) holds.  Returns how many;
  // up to kCap of them, `keys` (sh.list or sh.all) holds their order keys, unordered.
  template <class Open>
  __device__ __forceinline__ int gather(Open&& open, const u64*& keys) {
    const int lane = threadIdx.x & 31;
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    each([&](float l, int idx) {
      if (open(l, idx)) {
        const int n = atomicAdd(&sh.count, 1);
        if (n < kCap) sh.list[n] = order_key(l, idx);
      }
    });
    sync();
    keys = sh.list;
    if (splits == 1) return sh.count;
    const int mine = lane < splits ? peer_int(&sh.count, lane) : 0;
    int incl = mine;
#pragma unroll
    for (int o = 1; o < kMaxSplits; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    const int n = __shfl_sync(0xffffffffu, incl, splits - 1);
    if (n > kCap) return n;
    keys = sh.all;
    // warp w copies the lists of blocks w, w + kWarps, ...
    for (int r = threadIdx.x >> 5; r < splits; r += kWarps) {
      const int m = __shfl_sync(0xffffffffu, mine, r), at = __shfl_sync(0xffffffffu, incl, r) - m;
      for (int i = lane; i < m; i += 32) sh.all[at + i] = peer_u64(&sh.list[i], r);
    }
    __syncthreads();
    return n;
  }

  // Order key of the token at which the running sum, in order, of the counts or weights
  // of the tokens at or before `border` reaches its goal.
  template <bool kWeights, class Goal>
  __device__ u64 select(u64 border, Goal&& goal_of) {
    constexpr int kWords = kWeights ? 3 : 1;
    auto val = [&](float l) -> u64 { return kWeights ? weigh(l) : 1; };
    clear(kWords, kBins);
    each([&](float l, int idx) {
      if (border == 0 || order_key(l, idx) >= border) add<kWeights>(bin_of(l), val(l));
    });
    const u64 goal = find_bin(kWords, kBins, goal_of);
    const int bin = sh.bin;
    u64 sum = sh.excl;   // of the tokens before those still in question
    int shift = 64;      // the upper 64 - shift bits of their keys are `prefix`
    u64 prefix = 0;
    while (true) {
      const u64* list;
      const int n = gather(
          [&](float l, int idx) {
            if (bin_of(l) != bin) return false;
            const u64 key = order_key(l, idx);
            return key >= border && (shift == 64 || (key >> shift) == prefix);
          },
          list);
      if (n <= kCap) {
        u64* w = sh.hist;  // (every block has passed the gather's barrier: the histogram has been read)
        for (int i = threadIdx.x; i < n; i += kThreads) w[i] = val(key_logit(list[i]));
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += kThreads) {
          const u64 key = list[i];
          u64 before = sum;
          for (int j = 0; j < n; ++j)
            if (list[j] > key) before += w[j];
          if (before < goal && before + w[i] >= goal) sh.border = key;
        }
        sync();  // border is set; the peers have read this block's list
        return sh.border;
      }
      // too many: the next 8 bits of the key, largest first
      shift -= 8;
      clear(kWords, 256);
      each([&](float l, int idx) {
        const u64 key = order_key(l, idx);
        if (key >= border && bin_of(l) == bin && (shift == 56 || (key >> (shift + 8)) == prefix))
          add<kWeights>(255 - (int)((key >> shift) & 255), val(l));
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

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const SampleArgs a) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  Shared& sh = *reinterpret_cast<Shared*>(smem_raw);
  T* slice = reinterpret_cast<T*>(smem_raw + sizeof(Shared));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int splits = a.splits, rank = blockIdx.x % splits;
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
    store8<T>(slice + v, l);
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
  Sampler<T> s{sh, slice, base, w_len, splits, Row{}, 0.f};

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

  // between 1e-30 (below, only the largest logit has a weight) and 1e30 the products stay finite
  const double c = 1.4426950408889634 / fmin(fmax(temp, 1e-30), 1e30);
  s.row.mx = mx;
  s.row.ch = (float)c;
  s.row.cl = (float)(c - (double)s.row.ch);
  // min-p as the least weight; the largest weight, 2^44, always passes
  const u64 least = min_p > 0.0 ? (u64)(fmin(min_p, 1.0) * 17592186044416.0) : 0;
  const float range = fminf(mx - mn, 64.f / s.row.ch);
  s.step = range > 0.f ? (kBins - 1) / range : 0.f;

  u64 border = 0;  // every token
  const bool cut_k = top_k > 0 && top_k < a.vocab;
  if (cut_k && top_k <= kShortK) {
    // 2. step that the k-th of the threads' maxima falls into: k tokens at least lie at or above it
    s.clear(1, kBins);
    if (own > -INFINITY) s.template add<false>(s.bin_of(own), 1);
    u64 maxima = 0;
    s.find_bin(1, kBins, [&](u64 total) {
      maxima = total;
      return min((u64)top_k, total);
    });
    const int bin = maxima < (u64)top_k ? kBins - 1 : sh.bin;  // too few threads have tokens: all of them
    const u64* list;
    const int n = s.gather([&](float l, int) { return s.bin_of(l) <= bin; }, list);
    if (n <= kCap) {
      if (rank == 0) {
        u64* w = sh.hist;
        for (int i = threadIdx.x; i < n; i += kThreads) w[i] = s.weigh(key_logit(list[i]));
        __syncthreads();
        // entries i = thread, thread + kThreads: place in the order and sum before it
        int place[kCap / kThreads];
        u64 before[kCap / kThreads];
        u64 sum = 0;
#pragma unroll
        for (int e = 0; e < kCap / kThreads; ++e) {
          const int i = threadIdx.x + e * kThreads;
          place[e] = 0;
          before[e] = 0;
          if (i < n) {
            const u64 key = list[i];
            for (int j = 0; j < n; ++j)
              if (list[j] > key) {
                ++place[e];
                before[e] += w[j];
              }
            if (place[e] < top_k) sum += w[i];
          }
        }
        sum = warp_sum_u64(sum);
        if (lane == 0) sh.warp_sum[warp] = sum;
        __syncthreads();
        u64 total = 0;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) total += sh.warp_sum[k];
        const u64 p_goal = top_p < 1.0 ? (u64)fmax(ceil(top_p * (double)total), 1.0) : ~0ull;
        __syncthreads();
        sum = 0;
#pragma unroll
        for (int e = 0; e < kCap / kThreads; ++e) {
          const int i = threadIdx.x + e * kThreads;
          if (i < n) {
            if (place[e] >= top_k || before[e] >= p_goal || w[i] < least) w[i] = 0;
            sum += w[i];
          }
        }
        sum = warp_sum_u64(sum);
        if (lane == 0) sh.warp_sum[warp] = sum;
        __syncthreads();
        total = 0;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) total += sh.warp_sum[k];
        const u64 goal = choice(u, total);
        for (int i = threadIdx.x; i < n; i += kThreads) {
          const uint32_t back = (uint32_t)list[i];  // larger for lower indices
          u64 at = 0;
          for (int j = 0; j < n; ++j)
            if ((uint32_t)list[j] > back) at += w[j];
          if (at <= goal && goal < at + w[i]) a.tokens[r] = (int64_t)(0xffffffffu - back);
        }
      }
      if (splits > 1) cluster_sync_all();  // no block leaves while its list is read
      return;
    }
  }
  if (cut_k) {
    // the k-th token of those that are not -inf, or the last of them
    s.sync();
    border = s.template select<false>(border, [&](u64 total) { return min((u64)top_k, total); });
  }
  if (top_p < 1.0) {
    // the fewest whose sum is at least top_p of the whole; at least one unit, which keeps the first
    border = s.template select<true>(
        border, [&](u64 total) { return min((u64)fmax(ceil(top_p * (double)total), 1.0), total); });
  }
  auto kept = [&](float l, int idx) -> u64 {
    if (border != 0 && order_key(l, idx) < border) return 0;
    const u64 w = s.weigh(l);
    return w >= least ? w : 0;
  };

  // 4. sums per warp, in the order of the vocabulary
  u64 sum = 0;
  s.each([&](float l, int idx) { sum += kept(l, idx); });
  sum = warp_sum_u64(sum);
  if (lane == 0) sh.warp_sum[warp] = sum;
  s.sync();
  const int n_sums = splits * kWarps;
  if (threadIdx.x < n_sums)
    sh.sums[threadIdx.x] = splits > 1 ? peer_u64(&sh.warp_sum[threadIdx.x % kWarps], threadIdx.x / kWarps)
                                      : sh.warp_sum[threadIdx.x];
  __syncthreads();
  u64 before = 0, total = 0;  // before: of the warps ahead of this one
  for (int i = lane; i < n_sums; i += 32) {
    const u64 x = sh.sums[i];
    if (i < rank * kWarps + warp) before += x;
    total += x;
  }
  before = warp_sum_u64(before);
  total = warp_sum_u64(total);
  // first token whose running sum passes u * total (the largest weight is 2^44 units: total > 0)
  const u64 goal = choice(u, total);
  if (before <= goal && goal < before + sum) {
    const T* part = slice + warp * w_len;
    for (int v0 = 0; v0 < w_len; v0 += 256) {
      const int v = v0 + lane * 8;
      u64 w[8], mine = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = 0;
      if (v < w_len) {
        float l[8];
        load8<T>(part + v, l);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (l[i] > -INFINITY) w[i] = kept(l[i], base + warp * w_len + v + i);
          mine += w[i];
        }
      }
      u64 incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
      }
      u64 at = before + incl - mine;
      if (at <= goal && goal < at + mine) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (at <= goal && goal < at + w[i]) a.tokens[r] = base + warp * w_len + v + i;
          at += w[i];
        }
      }
      before += __shfl_sync(0xffffffffu, incl, 31);
      if (goal < before) break;
    }
  }
  if (splits > 1) cluster_sync_all();  // no block leaves while its sums are read
}

template <typename T>
void launch_sample(SampleArgs a, cudaStream_t s) {
  // Blocks per row: enough for two on each SM when rows are few, and as many as it
  // takes to hold the row in 96 KB of each (two blocks on an SM).
  const int tile = kWarps * 8;
  int splits = 1;
  while (splits < kMaxSplits && ((long long)a.rows * splits < 2 * 148 || (long long)a.vocab * (int)sizeof(T) > splits * 98304ll) &&
         (long long)a.vocab > (long long)splits * kThreads * 4)
    splits *= 2;
  a.splits = splits;
  a.warp_len = (int)(((long long)a.vocab + (long long)splits * tile - 1) / ((long long)splits * tile)) * 8;
  const size_t smem = sizeof(Shared) + (size_t)a.warp_len * kWarps * sizeof(T);
  constexpr size_t kMaxSmem = 227 * 1024;
  if (smem > kMaxSmem) throw std::runtime_error("sample: the vocabulary does not fit the shared memory of 8 blocks");
  static PerDeviceOnce once;
  once([] {
    UHFS_CUDA_CHECK(cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMaxSmem));
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
  UHFS_CUDA_CHECK(cudaLaunchKernelEx(&cfg, sample_kernel<T>, (const SampleArgs)a));
  note_launch();
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
