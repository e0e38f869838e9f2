// Next-token sampling: temperature, top-k, top-p, min-p and the choice by a given
// uniform number, without a sort, with one read of the logits.
//
// Tokens are ordered by (logit, lowest index first); top-k, top-p and min-p each
// keep a prefix of that order, so the kept set is "at or before one token", found
// as follows, and the choice walks the vocabulary in index order:
//   1. the row goes to shared memory (one block, or a cluster whose blocks each hold
//      a slice); maximum and minimum;
//   2. top-k: a histogram of 1024 equal steps of the logit finds the step that holds
//      the k-th token, whose few tokens are then compared with one another;
//   3. top-p: the same with the sum of weights in place of the count;
//   4. sums of the kept weights per warp (a contiguous part of the row each); the warp
//      that holds u * total walks its part again.
// A step that holds more tokens than the list (equal logits in long runs) is cut by
// 8 bits of the 64-bit order key at a time until the rest fits.
//
// Weights 2^((l - max) log2(e) / T) are 64-bit integers in units of 2^-44: sums do
// not depend on the order of atomics, blocks or warps, and a token on the border of
// top-p or of u is decided alike however the row was split.  Within 2^16 of the
// largest a weight is computed in 64 bits (relative error below 2^-36, from the
// Taylor series of exp), below that in 32 bits, where its error is below 2^-35 of
// the largest weight.
//
// Bound by latency for a few rows, by HBM for many (one read of the logits).
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
static_assert(kCap <= kBins, "the border tokens' weights reuse the histogram");
constexpr float kFine = -16.f;  // log2 of the weight from which 64 bits are used
typedef unsigned long long u64;

// shared memory in front of the row's slice
struct alignas(16) Shared {
  u64 hist[kBins];      // later the weights of the border tokens
  u64 list[kCap];       // this block's border tokens
  u64 all[kCap];        // the cluster's
  u64 warp_sum[kWarps];
  u64 border;           // order key of the last kept token
  u64 excl;             // sum before the chosen bin
  int bin;
  int count;            // entries of list (may exceed kCap: then not all are stored)
  float mx, mn;         // this block's extremes, then the row's
  int first;            // lowest index of the maximum in this block
  float warp_mx[kWarps], warp_mn[kWarps];
  int warp_first[kWarps];
  int token;
};

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

struct Row {
  float mx;       // largest logit
  double mxd, c;  // the same; log2(e) / temperature
  float cf;
};

// log2 of the weight in 32 bits: 0 for the maximum itself (also where it is infinite)
__device__ __forceinline__ float log2_weight(const Row& r, float l) {
  return l == r.mx ? 0.f : (l - r.mx) * r.cf;
}

// round(2^44 * 2^((l - max) c))
__device__ __forceinline__ u64 weight(const Row& r, float l) {
  const float xf = log2_weight(r, l);
  if (xf < kFine) return __float2ull_rn(ex2_approx(xf) * 17592186044416.f);
  const double x = l == r.mx ? 0.0 : ((double)l - r.mxd) * r.c;
  const float nf = rintf(xf);
  const double y = (x - (double)nf) * 0.69314718055994530942;  // |y| < 0.35: y^10 / 10! < 2^-36
  double e = 1.0 / 362880;
  e = fma(e, y, 1.0 / 40320);
  e = fma(e, y, 1.0 / 5040);
  e = fma(e, y, 1.0 / 720);
  e = fma(e, y, 1.0 / 120);
  e = fma(e, y, 1.0 / 24);
  e = fma(e, y, 1.0 / 6);
  e = fma(e, y, 0.5);
  e = fma(e, y, 1.0);
  e = fma(e, y, 1.0);
  return __double2ull_rn(e * __hiloint2double((1023 + 44 + (int)nf) << 20, 0));
}

__device__ __forceinline__ u64 peer_u64(const u64* p, int rank) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(smem_cluster_addr(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ int peer_int(const int* p, int rank) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(smem_cluster_addr(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ float peer_float(const float* p, int rank) {
  return __int_as_float(peer_int(reinterpret_cast<const int*>(p), rank));
}

template <typename T>
struct Sampler {
  Shared& sh;
  const T* slice;       // this block's part of the row in shared memory
  int base;             // index of its first token
  int w_len;            // tokens per warp, a multiple of 8
  int splits;
  Row row;

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

  // First bin whose inclusive sum over the cluster reaches the goal, a whole number
  // from 1 to the sum of all bins that goal_of(sum) gives; sets sh.bin and sh.excl.
  template <class Fn>
  __device__ __forceinline__ u64 find_bin(int bins, Fn&& goal_of) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    u64 v[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int bin = threadIdx.x * 2 + i;
      if (bin < bins) {
        if (splits == 1) v[i] = sh.hist[bin];
        else
          for (int r = 0; r < splits; ++r) v[i] += peer_u64(&sh.hist[bin], r);
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

  // Order key of the token at which the running sum, in order, of val(logit) over the
  // tokens at or before `border` reaches its goal.
  template <class Val, class Goal>
  __device__ u64 select(float mn, u64 border, Val&& val, Goal&& goal_of) {
    // equal steps of the logit; the last takes everything 2^64 below the largest weight
    const float range = fminf(row.mx - mn, 64.f / row.cf);
    const float step = range > 0.f ? (kBins - 1) / range : 0.f;
    auto bin_of = [&](float l) {
      return l == row.mx ? 0 : (int)fminf((row.mx - l) * step, (float)(kBins - 1));
    };
    for (int i = threadIdx.x; i < kBins; i += kThreads) sh.hist[i] = 0;
    __syncthreads();
    each([&](float l, int idx) {
      if (order_key(l, idx) >= border) {
        const u64 w = val(l);
        if (w) atomicAdd(&sh.hist[bin_of(l)], w);
      }
    });
    sync();
    const u64 goal = find_bin(kBins, goal_of);
    const int bin = sh.bin;
    u64 sum = sh.excl;   // of the tokens before those still in question
    int shift = 64;      // the upper 64 - shift bits of their keys are `prefix`
    u64 prefix = 0;
    while (true) {
      auto open = [&](float l, u64 key) {
        return key >= border && bin_of(l) == bin && (shift == 64 || (key >> shift) == prefix);
      };
      if (threadIdx.x == 0) sh.count = 0;
      __syncthreads();
      each([&](float l, int idx) {
        const u64 key = order_key(l, idx);
        if (open(l, key)) {
          const int n = atomicAdd(&sh.count, 1);
          if (n < kCap) sh.list[n] = key;
        }
      });
      sync();
      int n = 0;
      for (int r = 0; r < splits; ++r) n += splits > 1 ? peer_int(&sh.count, r) : sh.count;
      if (n <= kCap) {
        const u64* list = sh.list;
        if (splits > 1) {
          int at = 0;
          for (int r = 0; r < splits; ++r) {
            const int m = peer_int(&sh.count, r);
            for (int i = threadIdx.x; i < m; i += kThreads) sh.all[at + i] = peer_u64(&sh.list[i], r);
            at += m;
          }
          list = sh.all;
          __syncthreads();
        }
        u64* w = sh.hist;
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
      for (int i = threadIdx.x; i < 256; i += kThreads) sh.hist[i] = 0;
      sync();  // (the peers have read sh.count)
      each([&](float l, int idx) {
        const u64 key = order_key(l, idx);
        if (key >= border && bin_of(l) == bin && (shift == 56 || (key >> (shift + 8)) == prefix)) {
          const u64 w = val(l);
          if (w) atomicAdd(&sh.hist[255 - (int)((key >> shift) & 255)], w);
        }
      });
      sync();
      const u64 left = sum;
      find_bin(256, [&](u64) { return goal - left; });
      sum = left + sh.excl;
      prefix = (prefix << 8) | (u64)(255 - sh.bin);
      sync();  // the histogram has been read
    }
  }
};

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

  // 1. the slice; tokens that cannot be chosen (NaN, past the end) become -inf
  float mx = -INFINITY, mn = INFINITY;
  for (int v = threadIdx.x * 8; v < len; v += kThreads * 8) {
    float l[8];
    const int left = a.vocab - (base + v);
    if (a.vec && left >= 8) {
      load8<T>(src + base + v, l);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) l[i] = i < left ? to_float<T>(src[base + v + i]) : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (!(l[i] > -INFINITY)) l[i] = -INFINITY;
      else {
        mx = fmaxf(mx, l[i]);
        mn = fminf(mn, l[i]);
      }
    }
    store8<T>(slice + v, l);
  }
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
  for (int w = 0; w < kWarps; ++w) {
    mx = fmaxf(mx, sh.warp_mx[w]);
    mn = fminf(mn, sh.warp_mn[w]);
  }
  if (threadIdx.x == 0) {
    sh.mx = mx;
    sh.mn = mn;
  }
  Sampler<T> s{sh, slice, base, w_len, splits, Row{}};
  s.sync();
  if (splits > 1)
    for (int k = 0; k < splits; ++k) {
      mx = fmaxf(mx, peer_float(&sh.mx, k));
      mn = fminf(mn, peer_float(&sh.mn, k));
    }

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
  s.row.mx = mx;
  s.row.mxd = (double)mx;
  s.row.c = 1.4426950408889634 / fmin(fmax(temp, 1e-30), 1e30);
  s.row.cf = (float)s.row.c;
  const Row row = s.row;
  u64 border = 0;  // every token
  if (top_k > 0 && top_k < a.vocab) {
    // the k-th token of those that are not -inf, or the last of them
    border = s.select(mn, border, [](float) { return (u64)1; },
                      [&](u64 total) { return min((u64)top_k, total); });
  }
  if (top_p < 1.0) {
    // the fewest whose sum is at least top_p of the whole; at least one unit, which keeps the first
    border = s.select(mn, border, [&](float l) { return weight(row, l); },
                      [&](u64 total) { return min((u64)fmax(ceil(top_p * (double)total), 1.0), total); });
  }
  const float min_lw = min_p > 0.0 ? (float)fmin(log2(min_p), 0.0) : -INFINITY;
  const double min_lwd = min_p > 0.0 ? fmin(log2(min_p), 0.0) : -INFINITY;
  auto kept = [&](float l, int idx) -> u64 {
    if (order_key(l, idx) < border) return 0;
    if (min_p > 0.0) {
      // 64 bits where 32 cannot tell the sides apart
      const float xf = log2_weight(row, l), slack = 1e-5f * (1.f - min_lw);
      if (xf < min_lw - slack) return 0;
      if (xf < min_lw + slack && l != row.mx && ((double)l - row.mxd) * row.c < min_lwd) return 0;
    }
    return weight(row, l);
  };

  // 4. sums per warp, in the order of the vocabulary
  u64 sum = 0;
  s.each([&](float l, int idx) { sum += kept(l, idx); });
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) sh.warp_sum[warp] = sum;
  s.sync();
  u64 before = 0, total = 0;  // before: of the warps ahead of this one
  for (int k = 0; k < splits; ++k)
    for (int w = 0; w < kWarps; ++w) {
      const u64 x = splits > 1 ? peer_u64(&sh.warp_sum[w], k) : sh.warp_sum[w];
      if (k < rank || (k == rank && w < warp)) before += x;
      total += x;
    }
  // first token whose running sum passes u * total (the largest weight is 2^44 units: total > 0)
  const double want = fmin(fmax((double)u, 0.0), 1.0) * (double)total;  // NaN: 0
  u64 goal = want >= (double)total ? total - 1 : (u64)want;
  if (goal >= total) goal = total - 1;
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
  while (splits < 8 && ((long long)a.rows * splits < 2 * 148 || (long long)a.vocab * (int)sizeof(T) > splits * 98304ll) &&
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
