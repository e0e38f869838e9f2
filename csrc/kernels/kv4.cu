// Key / value cache held in 4 bits: write, read back, and attention over it.
//
// Format.  The channels of one token and head are quantised in groups of 32:
//   lo = fp16(min),  s = fp16((max - lo) * fp32(1 / 15)),  code = rhe((x - lo) / s) in 0..15
// and a code stands for lo + s * code: 5 bits a value with its group's s and lo.
// Values are held to the range +-61440 (so that every lo + s * code is a finite
// fp16 number: a masked token then adds exactly 0, whatever was written), NaN
// becomes the group's minimum.
//
// Layout.  A page holds 32 tokens of one head, contiguous (D * 40 bytes), so a
// warp fetches it with one bulk copy:
//   K codes [32 tokens][D / 2 bytes], K s [32][NG], K lo [32][NG],
//   V codes [32 tokens][D / 2 bytes], V s [16 pairs][NG][2], V lo [16 pairs][NG][2]
// with NG = D / 32 groups.  Word (8 codes) w of a K row holds channels
// 32 * (w % NG) + 8 * (w / NG) ..+7: the quarter-warp lane that owns w / NG reads its words
// of all groups with one load.  Half word (4 codes) e of a V row holds channels
// 32 * (2 * (w % NW) + (e & 1)) + 4 * (w / NW) ..+3, w = e / 2, NW = D / 64: lane w / NW reads
// 4 channels of every group with one load.  Tokens t and t + 4 of 8 are a pair: the two
// tokens of an MMA operand register.
#include <stdexcept>
#include <string>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "vec.cuh"

namespace uhfs {

namespace {

constexpr int kPage = 32;     // tokens per page
constexpr int kGroup = 32;    // channels per (s, lo)
constexpr float kRange = 61440.f;

template <int D>
struct Kv4 {
  static constexpr int NG = D / kGroup;
  static constexpr int kCodes = kPage * D / 2;    // bytes of K (or V) codes
  static constexpr int kMeta = kPage * NG * 4;    // bytes of K (or V) s / lo
  static constexpr int kKS = kCodes, kKL = kKS + kMeta / 2, kVC = kCodes + kMeta, kVS = 2 * kCodes + kMeta,
                       kVL = kVS + kMeta / 2;
  static constexpr int kBytes = 2 * (kCodes + kMeta);
  static_assert(kBytes == D * 40 && kBytes % 16 == 0, "page size");
};

// place of a token's V s (or lo) of group gi in its plane
template <int D>
__device__ __forceinline__ int vslot(int tok, int gi) {
  const int pair = (tok >> 4) * 8 + (tok & 8 ? 4 : 0) + (tok & 3);
  return (pair * Kv4<D>::NG + gi) * 2 + ((tok >> 2) & 1);
}
// place of the half word that holds channels 4 c .. 4 c + 3 in a V row
template <int D>
__device__ __forceinline__ int vhalf(int c) {
  const int gi = c / 8;
  return ((c % 8) * (D / 64) + gi / 2) * 2 + (gi & 1);
}

// ------------------------------------------------------------ write / read
// A thread takes 8 channels of K and the same of V of kRows consecutive tokens: 4 threads
// share a group, D / 8 a row.  Both kernels move about 2.6 bytes a value, so a value may
// cost some 12 instructions before they bound them: the threads of a block span the heads
// (and, where those are few, several runs of tokens), so that a place costs no division by
// the number of heads and is worked out once for kRows tokens, whose loads overlap (four for
// 16-bit types: prompt write and read back of 8 x 2048, 16 x 128 take 62 and 38 us, 73 and 41 with one; two
// of 32-bit ones, which need the registers of four).  Measured at that size: write 62 us, 2.8
// TB/s (fp32 52 in a graph, bf16 59), bound by its instructions (184 for 8 values, min and max, quotients and places
// included), read back 38 us, 4.7 TB/s.
template <int D>
struct Place {
  int h, lw, t0;  // head, 8 channels of it, first token
  bool on;
};
template <int D, int kRows>
__device__ __forceinline__ Place<D> place(int H, int t_begin) {
  constexpr int LPR = D / 8;
  const int span = H * LPR, per_block = span < 256 ? 256 / span : 1;  // runs of tokens per block
  int u = blockIdx.x * 256 + threadIdx.x, run = 0;
  if (span < 256) {
    run = (int)threadIdx.x / span;
    u = (int)threadIdx.x - run * span;
  }
  return Place<D>{u / LPR, u % LPR, t_begin + ((int)blockIdx.y * per_block + run) * kRows, u < span && run < per_block};
}

// y + kMagic has round(y) in its low bits, for |y| < 2^22
constexpr float kMagic = 12582912.f;

// The codes of x[8], code i in bits 4 i .. 4 i + 3: round-half-even((x - lo) / s) in 0..15.
// kSure: at least 2^-17 away from a half, (x - lo) * (1 / s), which is off by less than 2^-17.2,
// rounds to the code.
constexpr float kSure = 0.5f - 1.f / 131072;
__device__ __noinline__ uint32_t quantize8_exact(float4 x0, float4 x1, float lo, float s) {
  const float x[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
  const float inv = s > 0.f ? __fdividef(1.f, s) : 0.f, half_s = 0.5f * s;
  uint32_t word = 0;
#pragma unroll
  for (int i = 7; i >= 0; --i) {
    const float d = x[i] - lo;
    const float y = fminf(fmaxf(d * inv, 0.f), 15.f), z = y + kMagic;  // (NaN: 0)
    int k = (int)(__float_as_uint(z) - __float_as_uint(kMagic));
    if (!(fabsf(y - (z - kMagic)) < kSure)) {
      // the remainder, which an FMA gives exactly, and the rounding error of x - lo = d + e
      const float bb = d - x[i], e = (x[i] - (d - bb)) + (-lo - bb);
      const float r = fmaf(-(float)k, s, d), up = (r - half_s) + e, dn = (r + half_s) + e;
      const int odd = k & 1;
      if (up > 0.f || (up == 0.f && odd)) ++k;
      if (dn < 0.f || (dn == 0.f && odd)) --k;
      k = s > 0.f ? min(max(k, 0), 15) : 0;
    }
    word = word * 16u + (uint32_t)k;
  }
  return word;
}

// the largest of |a|, |b| and |c|, NaN if one is NaN
__device__ __forceinline__ float max3_abs_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// A group's lo and s (its values are those of four neighbouring threads) and this thread's codes.
// Where every value is sure, within the codes' range and finite, the rounded product is the
// code; about one in 2^11 values of a bf16 tensor is not (mostly ties), and its thread's eight go
// the exact way.
__device__ __forceinline__ uint32_t quantize8(const float* x, float mn, float mx, __half* lo_h, __half* s_h) {
#pragma unroll
  for (int o = 1; o <= 2; o <<= 1) {  // (fminf and fmaxf pass over NaN)
    mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  }
  if (mn > mx) mn = mx = 0.f;  // nothing but NaN
  const float lo0 = fminf(fmaxf(mn, -kRange), kRange), hi = fminf(fmaxf(mx, -kRange), kRange);
  *lo_h = __float2half_rn(lo0);
  const float lo = __half2float(*lo_h);
  *s_h = __float2half_rn(fmaxf((hi - lo) * (1.f / 15.f), 0.f));
  const float s = __half2float(*s_h), inv = __fdividef(1.f, s);  // (s = 0: infinite, and nothing is sure)
  bool sure = (mn - lo) * inv > -kSure && (mx - lo) * inv < 15.f + kSure;
  // pairs of codes i and i + 4, as packed fp32
  auto both = [](float y) { return make_float2(y, y); };
  float2 n[4];  // minus the codes
  float off = 0.f;  // the farthest of the quotients from its code
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 d = f2_add(make_float2(x[i], x[i + 4]), both(-lo));
    n[i] = f2_fma(f2_fma(d, both(inv), both(kMagic)), both(-1.f), both(kMagic));
    const float2 e = f2_fma(d, both(inv), n[i]);
    off = max3_abs_nan(off, e.x, e.y);  // (NaN and infinities are not sure)
  }
  sure = sure && off < kSure;
  // the sums of four codes times powers of 16 are exact
  const float2 m = f2_fma(f2_fma(f2_fma(n[3], both(16.f), n[2]), both(16.f), n[1]), both(16.f), n[0]);
  const float2 z = f2_fma(m, both(-1.f), both(kMagic));
  uint32_t word = __byte_perm(__float_as_uint(z.x), __float_as_uint(z.y), 0x5410);
  if (!sure)
    word = quantize8_exact(make_float4(x[0], x[1], x[2], x[3]), make_float4(x[4], x[5], x[6], x[7]), lo, s);
  return word;
}

// 8 values as loaded
template <typename T>
struct Raw8 {
  uint4 v[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  // the values, their least and their largest (NaN passed over), 16-bit types two at a time
  __device__ __forceinline__ void range(float* x, float* mn, float* mx) const {
    const T* h = reinterpret_cast<const T*>(v);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_float<T>(h[i]);
    if constexpr (sizeof(T) == 2) {
      using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
      const T2* w = reinterpret_cast<const T2*>(v);
      const T2 lo = __hmin2(__hmin2(w[0], w[1]), __hmin2(w[2], w[3]));
      const T2 hi = __hmax2(__hmax2(w[0], w[1]), __hmax2(w[2], w[3]));
      // (all NaN: fminf and fmaxf drop one at a time, the last is dropped by the neighbours')
      *mn = fminf(fminf(to_float<T>(lo.x), to_float<T>(lo.y)), INFINITY);
      *mx = fmaxf(fmaxf(to_float<T>(hi.x), to_float<T>(hi.y)), -INFINITY);
    } else {
      *mn = INFINITY;
      *mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        *mn = fminf(*mn, x[i]);
        *mx = fmaxf(*mx, x[i]);
      }
    }
  }
};

template <int D, typename T, int kRows>
__global__ void __launch_bounds__(256, 4) kv4_append_kernel(const Kv4Append a) {
  using F = Kv4<D>;
  constexpr int LPR = D / 8;  // threads per row
  const Place<D> pl = place<D, kRows>(a.H, a.t_begin);
  const int lw = pl.lw, gi = lw / 4, b = blockIdx.z;  // channels [8 lw, 8 lw + 8)
  const int count = a.counts != nullptr ? min(a.counts[b], a.T) : a.T;
  const long long start = a.lengths[b];
  Raw8<T> k[kRows], v[kRows];
  bool live[kRows];
  const T* src_k = static_cast<const T*>(a.k) + b * a.k_stride_b + (long long)pl.h * (int)a.k_stride_h + lw * 8;
  const T* src_v = static_cast<const T*>(a.v) + b * a.v_stride_b + (long long)pl.h * (int)a.v_stride_h + lw * 8;
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int t = pl.t0 + i;
    live[i] = pl.on && t < count;
    if (live[i] && (start + t < 0 || start + t >= a.capacity)) {
      if (lw == 0) report_error(a.status, kErrBounds, 60);
      live[i] = false;
    }
    k[i] = v[i] = Raw8<T>{};
    if (live[i]) {
      k[i].load(src_k + (long long)t * (int)a.k_stride_t);
      v[i].load(src_v + (long long)t * (int)a.v_stride_t);
    }
  }
  unsigned char* head = a.pages + ((long long)b * a.H + pl.h) * a.pages_per_head * F::kBytes;
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    if (!__any_sync(0xffffffffu, live[i])) continue;  // (a row's threads agree)
    float x[8], mn, mx;
    __half klo, ks, vlo, vs;
    k[i].range(x, &mn, &mx);
    const uint32_t kw = quantize8(x, mn, mx, &klo, &ks);
    v[i].range(x, &mn, &mx);
    const uint32_t vw = quantize8(x, mn, mx, &vlo, &vs);
    // V words hold 4 channels of an even group and 4 of the next: the threads of the two exchange
    // halves, the even one takes the word of its first 4 channels
    const uint32_t other = __shfl_xor_sync(0xffffffffu, vw, 4);
    const uint32_t vword = gi & 1 ? __byte_perm(other, vw, 0x7632) : __byte_perm(vw, other, 0x5410);
    if (!live[i]) continue;
    const uint32_t pos = (uint32_t)(start + pl.t0 + i), tok = pos % kPage;
    unsigned char* page = head + (long long)(pos / kPage) * F::kBytes;
    reinterpret_cast<uint32_t*>(page)[tok * LPR + (lw % 4) * F::NG + gi] = kw;
    reinterpret_cast<uint32_t*>(page + F::kVC)[tok * LPR + vhalf<D>(2 * lw + (gi & 1)) / 2] = vword;
    if (lw % 4 == 0) {
      reinterpret_cast<__half*>(page + F::kKS)[tok * F::NG + gi] = ks;
      reinterpret_cast<__half*>(page + F::kKL)[tok * F::NG + gi] = klo;
      reinterpret_cast<__half*>(page + F::kVS)[vslot<D>(tok, gi)] = vs;
      reinterpret_cast<__half*>(page + F::kVL)[vslot<D>(tok, gi)] = vlo;
    }
  }
}

template <typename T>
__device__ __forceinline__ void store_values(T* dst, uint32_t w, __half s, __half lo) {
  const float sf = __half2float(s), lf = __half2float(lo);
  float f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)  // the code as 2^23 + code without a conversion
    f[i] = fmaf(sf, __uint_as_float(((w >> (4 * i)) & 15u) | 0x4B000000u) - 8388608.f, lf);
  store8<T>(dst, f);
}

// out[b][t][h][:] = token start + t
template <int D, typename T, int kRows>
__global__ void __launch_bounds__(256) kv4_read_kernel(const Kv4Read a) {
  using F = Kv4<D>;
  constexpr int LPR = D / 8;
  const Place<D> pl = place<D, kRows>(a.H, a.t_begin);
  if (!pl.on) return;
  const int lw = pl.lw, gi = lw / 4, b = blockIdx.z;
  const unsigned char* head = a.pages + ((long long)b * a.H + pl.h) * a.pages_per_head * F::kBytes;
  uint32_t kw[kRows], vw[kRows];
  __half ks[kRows], kl[kRows], vs[kRows], vl[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    if (pl.t0 + i >= a.n) break;
    const uint32_t pos = (uint32_t)(a.start + pl.t0 + i), tok = pos % kPage;
    const unsigned char* page = head + (long long)(pos / kPage) * F::kBytes;
    kw[i] = reinterpret_cast<const uint32_t*>(page)[tok * LPR + (lw % 4) * F::NG + gi];
    const uint16_t* vrow = reinterpret_cast<const uint16_t*>(page + F::kVC + tok * (D / 2));
    vw[i] = vrow[vhalf<D>(2 * lw)] | ((uint32_t)vrow[vhalf<D>(2 * lw + 1)] << 16);
    ks[i] = reinterpret_cast<const __half*>(page + F::kKS)[tok * F::NG + gi];
    kl[i] = reinterpret_cast<const __half*>(page + F::kKL)[tok * F::NG + gi];
    vs[i] = reinterpret_cast<const __half*>(page + F::kVS)[vslot<D>(tok, gi)];
    vl[i] = reinterpret_cast<const __half*>(page + F::kVL)[vslot<D>(tok, gi)];
  }
  const long long step = (long long)a.H * D;
  long long at = ((long long)b * a.n + pl.t0) * step + pl.h * D + lw * 8;
#pragma unroll
  for (int i = 0; i < kRows; ++i, at += step) {
    if (pl.t0 + i >= a.n) break;
    store_values<T>(static_cast<T*>(a.k) + at, kw[i], ks[i], kl[i]);
    store_values<T>(static_cast<T*>(a.v) + at, vw[i], vs[i], vl[i]);
  }
}

// --------------------------------------------------------------- attention
// The new tokens' queries of one key / value head (Tq tokens x group heads) are
// taken eight at a time as the N = 8 side of m16n8k16 products (fp16 in, fp32
// out); the 16 side is 16 tokens for S^T = K Q^T and 16 channels for O^T = V^T P^T,
// so the codes, the operand that costs instructions, are read with no padding.
//
// The kernel is bound by HBM (0.625 bytes a value) as long as unpacking stays under about
// 3 instructions a value, so the codes go to the tensor core as they are: w & 0x000f000f is a
// pair of fp16 subnormals, code * 2^-24 exactly, and w & 0x00f000f0 one of 16 code * 2^-24:
// one instruction for two codes, and no scale on this side.
//   K  s and lo are per token, a row of the 16 x 8 products: S = sum over groups of
//      s (q . code) + lo sum(q), s in fp32 on the product of each group, the lo term as
//      one more product for all groups (sum(q) as two fp16 numbers).  q / 16 stands in the
//      places of the odd codes.  q is only scaled, by a power of two per query that
//      brings it to [1, 2): a bf16 or fp16 q goes in without a rounding.
//   V  s and lo are per token, the products' inner dimension: O = sum over tokens of
//      r (code - 8) + P (lo + 8 s) with r = P s rounded to fp16 (P itself goes in as two
//      fp16 numbers); -8 r is one more product on the codes' rows (a constant operand: a row per
//      group in the lo product cost an operand each time), the lo term one row per group.  The 8 makes
//      the rounding's share that of code - 8, not of code: without it its error was twice as
//      large.
// So K is not rounded, and for V only P s and lo + 8 s are.
// Every warp works alone: it owns a ring of pages filled by bulk copies and takes
// every n-th page of the block's share (n warps), with its own running maximum (raised
// only when a score exceeds it by 2^2) and sum.  The warps of a block are joined in
// shared memory and the blocks of a cluster, which share one head's tokens, through
// distributed shared memory: one launch, no workspace, no atomics, and a sum order
// that depends on sizes only.
//
// Measured: 32 sequences of 2 to 4 K keys, 32 x 128: 122 us, 4.2 TB/s (the loads alone 96, the
// arithmetic alone 113: 630 instructions a page at 16 warps an SM, waiting on one another
// and on the integer pipe); 1 x 1000 keys, 12 x 64: 10 us; 5 new tokens over windows of 8192 of
// 4 sequences, 32 / 8 x 128: 41 us (three query tiles read each page).
constexpr int kMaxWarps = 8;  // per block
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescale = 2.0f;
// P goes in as 2^kRaise P, so that P s, an fp16 number, stays a normal one for small P and s (V of
// about 1e-4 over 32768 keys, scores of standard deviation 2.5: error 4e-2 of the output without, the
// result's own rounding with).  P <= 2^kRescale, so that s < kRaiseS leaves it within fp16's range; where
// a query sees a token of larger s (at most 2 * kRange / 15 = 8192), its power is lowered.
constexpr int kRaise = 10;
constexpr int kRaiseS = 18;  // exponent field of 8, the first s that is too large

__device__ __forceinline__ void mma_f16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_zero(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                             uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// codes 0 and 4 (even) or 1 and 5 (odd, times 16) of a word as fp16 subnormals; >> 8: the next two
__device__ __forceinline__ uint32_t even_codes(uint32_t w) { return w & 0x000f000fu; }
__device__ __forceinline__ uint32_t odd_codes(uint32_t w) { return w & 0x00f000f0u; }
constexpr float kCodeUnit = 16777216.f;  // 2^24
__device__ __forceinline__ __half2 as_half2(uint32_t x) { return *reinterpret_cast<__half2*>(&x); }
__device__ __forceinline__ uint32_t as_u32(__half2 x) { return *reinterpret_cast<uint32_t*>(&x); }

// N consecutive 32-bit words of shared memory (N = 1, 2, 4)
template <int N>
__device__ __forceinline__ void load_words(uint32_t* dst, const uint8_t* src) {
  if constexpr (N == 4) *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src);
  else if constexpr (N == 2) *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(src);
  else *dst = *reinterpret_cast<const uint32_t*>(src);
}

__device__ __forceinline__ float dsmem_load(const float* p, uint32_t rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(smem_cluster_addr(p, rank)) : "memory");
  return v;
}

template <int D>
struct Kv4Attn {
  static constexpr int kStages = D == 128 ? 2 : 4;  // pages in flight per warp
  // a block of `warps`: their pages, then in the same place the warps' sums [warps][8][D], their
  // m and l, and the block's result
  static __host__ __device__ constexpr int body(int warps) {
    const int ring = warps * kStages * Kv4<D>::kBytes, join = (warps * 8 * D + 2 * warps * 8 + 8 * D + 2 * 8) * 4;
    return ring > join ? ring : join;
  }
  static __host__ __device__ constexpr int smem(int warps) { return 128 + body(warps) + warps * kStages * 8; }
};

template <int D, typename T>
__global__ void __launch_bounds__(kMaxWarps * 32, 2) kv4_attend_kernel(const Kv4Attend a) {
  using F = Kv4<D>;
  using C = Kv4Attn<D>;
  constexpr int NG = F::NG, NS = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((128u - (smem_u32(smem_raw) & 127u)) & 127u);
  const int n_warps = blockDim.x >> 5;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::body(n_warps));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int splits = a.splits;                  // blocks of a cluster
  const int rank = blockIdx.x % splits;
  long long unit = blockIdx.x / splits;         // (batch, head, query tile)
  const int qt = (int)(unit % a.q_tiles);
  unit /= a.q_tiles;
  const int h = (int)(unit % a.Hkv), b = (int)(unit / a.Hkv);
  const int G = a.Hq / a.Hkv;

  const int count = a.counts != nullptr ? min(max(a.counts[b], 0), a.Tq) : a.Tq;
  const long long len = a.lengths[b];
  const int row0 = qt * 8, rows = min(8, count * G - row0);  // live queries of this tile (may be <= 0)
  if (threadIdx.x == 0 && rows > 0 && (len < 0 || len + count > a.capacity)) report_error(a.status, kErrBounds, 61);

  // this tile's tokens: [0, hi) for its last query, from `first` on for its first, and the sinks
  long long hi = 0, first = 0;
  if (rows > 0) {
    hi = min(max(len + (row0 + rows - 1) / G + 1, 0ll), (long long)a.capacity);
    if (a.window > 0) first = max(0ll, len + row0 / G + 1 - a.window);
  }
  const int p_hi = (int)((hi + kPage - 1) / kPage), p_first = (int)min(first / kPage, (long long)p_hi);
  const int p_sink = min((a.sinks + kPage - 1) / kPage, p_first);
  const int n_pages = p_sink + p_hi - p_first;
  const int share = (n_pages + splits - 1) / splits;
  const int i_end = min(n_pages, (rank + 1) * share);
  const int i_begin = rank * share + warp;  // this warp: i_begin, i_begin + n_warps, ...
  auto page_of = [&](int i) { return i < p_sink ? i : p_first + i - p_sink; };

  uint8_t* ring = smem + warp * (NS * F::kBytes);
  uint64_t* full = bars + warp * NS;
  const unsigned char* head = a.pages + ((long long)b * a.Hkv + h) * a.pages_per_head * F::kBytes;
  auto issue = [&](int i, int slot) {
    mbar_arrive_expect_tx(&full[slot], F::kBytes);
    bulk_load(ring + slot * F::kBytes, head + (long long)page_of(i) * F::kBytes, F::kBytes, &full[slot]);
  };
  if (lane == 0) {
    for (int s = 0; s < NS; ++s) mbar_init(&full[s], 1);
    fence_barrier_init();
    fence_proxy_async_smem();
    for (int s = 0; s < NS; ++s)
      if (i_begin + s * n_warps < i_end) issue(i_begin + s * n_warps, s);
  }
  __syncwarp();

  // ---- queries: column g of the tile, channels 32 gi + 8 t .. + 7 of each group
  uint32_t qf[NG][4];
  uint32_t qs_hi, qs_lo;  // sum(q) of groups 2 t, 2 t + 1 (second operand of the lo product)
  float scale2[2];
  {
    const int m = row0 + g;
    float q[NG][8];
    float mx = 0.f;
#pragma unroll
    for (int gi = 0; gi < NG; ++gi) {
#pragma unroll
      for (int i = 0; i < 8; ++i) q[gi][i] = 0.f;
      if (g < rows) {
        const T* src = static_cast<const T*>(a.q) + b * a.q_stride_b + (m / G) * a.q_stride_t +
                       (h * G + m % G) * a.q_stride_h + gi * kGroup + t * 8;
        load8<T>(src, q[gi]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) mx = fmaxf(mx, fabsf(q[gi][i]));
    }
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    // a power of two within (mx / 2, mx], of at most 2^100
    const uint32_t eb = min(__float_as_uint(mx) & 0x7f800000u, 227u << 23);
    const float up = mx > 1e-30f ? __uint_as_float(eb) : 1.f;
    const float dn = mx > 1e-30f ? __uint_as_float((254u << 23) - eb) : 1.f;
    float sums[NG];
#pragma unroll
    for (int gi = 0; gi < NG; ++gi) {
      float sum = 0.f;
      __half hq[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool odd = i & 1;  // odd codes come times 16
        hq[i] = __float2half_rn(q[gi][i] * (odd ? dn * 0.0625f : dn));
        sum += odd ? 16.f * __half2float(hq[i]) : __half2float(hq[i]);
      }
      // register k of a word holds codes k and k + 4
#pragma unroll
      for (int k = 0; k < 4; ++k) qf[gi][k] = as_u32(__halves2half2(hq[k], hq[k + 4]));
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      sums[gi] = sum;
    }
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int gi = 0; gi < NG; gi += 2)
      if (2 * t == gi) {
        s0 = sums[gi];
        s1 = sums[gi + 1];
      }
    const __half h0 = __float2half_rn(s0), h1 = __float2half_rn(s1);
    qs_hi = as_u32(__halves2half2(h0, h1));
    qs_lo = as_u32(__floats2half2_rn(s0 - __half2float(h0), s1 - __half2float(h1)));
#pragma unroll
    for (int c = 0; c < 2; ++c)  // columns 2 t and 2 t + 1 of the products
      scale2[c] = __shfl_sync(0xffffffffu, up, (2 * t + c) * 4) * (a.scale * kLog2e);
  }
  const int lim_all = (int)max(0ll, min(len + row0 / G + 1, (long long)a.capacity));  // visible to every live query
  const int low_all = rows > 0 && a.window > 0 ? (int)max(0ll, hi - a.window) : 0;

  float o[NG][2][4], o_lo[4] = {0.f, 0.f, 0.f, 0.f};  // code part by group; lo part: row = group
#pragma unroll
  for (int i = 0; i < NG; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) o[i][j >> 2][j & 3] = 0.f;
  // per query: maximum so far, what is subtracted from the scores (0 while there is none), log2 of P's factor
  float m_run[2] = {-INFINITY, -INFINITY}, base[2] = {0.f, 0.f}, l_run[2] = {0.f, 0.f};
  int raise[2] = {kRaise, kRaise};
  uint32_t headroom = (32 - kRaiseS) * 0x04000400u;  // brings the first s that some query has to lower its power for to 2^16
  const int prow = (g & 1) ? (g >> 1) + 4 : (g >> 1);  // token of product row g within 8

  int n_done = 0;
  for (int i = i_begin; i < i_end; i += n_warps, ++n_done) {
    const int slot = n_done % NS;
    if (!mbar_wait_warp(&full[slot], (uint32_t)(n_done / NS) & 1u, a.status, kErrWaitTimeoutFull, 62)) break;
    const uint8_t* pg = ring + slot * F::kBytes;
    const int key0 = page_of(i) * kPage;

    // S^T: 2 x (16 tokens x 8 queries)
    float s[2][4];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      const int ra = mt * 16 + prow, rb = ra + 8;
      uint32_t wa[NG], wb[NG], sa[NG / 2], sb[NG / 2], la, lb;
      load_words<NG>(wa, pg + ra * (D / 2) + t * (4 * NG));
      load_words<NG>(wb, pg + rb * (D / 2) + t * (4 * NG));
      load_words<NG / 2>(sa, pg + F::kKS + ra * (2 * NG));
      load_words<NG / 2>(sb, pg + F::kKS + rb * (2 * NG));
      load_words<1>(&la, pg + F::kKL + ra * (2 * NG) + (t % (NG / 2)) * 4);
      load_words<1>(&lb, pg + F::kKL + rb * (2 * NG) + (t % (NG / 2)) * 4);
      float lo_part[4];
      mma_f16_zero(lo_part, la, lb, la, lb, qs_hi, qs_lo);
      float sc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int gi = 0; gi < NG; ++gi) {
        float c[4];
        mma_f16_zero(c, even_codes(wa[gi]), even_codes(wb[gi]), odd_codes(wa[gi]), odd_codes(wb[gi]), qf[gi][0],
                     qf[gi][1]);
        const uint32_t xa = wa[gi] >> 8, xb = wb[gi] >> 8;
        mma_f16(c, even_codes(xa), even_codes(xb), odd_codes(xa), odd_codes(xb), qf[gi][2], qf[gi][3]);
        const __half2 ha = as_half2(sa[gi / 2]), hb = as_half2(sb[gi / 2]);
        const float fa = gi & 1 ? __high2float(ha) : __low2float(ha), fb = gi & 1 ? __high2float(hb) : __low2float(hb);
        sc[0] = fmaf(fa, c[0], sc[0]);
        sc[1] = fmaf(fa, c[1], sc[1]);
        sc[2] = fmaf(fb, c[2], sc[2]);
        sc[3] = fmaf(fb, c[3], sc[3]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) s[mt][e] = fmaf(sc[e], kCodeUnit, lo_part[e]) * scale2[e & 1];
    }
    if (key0 + kPage > lim_all || key0 < low_all) {
      // tokens visible to columns 2 t, 2 t + 1: [low, lim) and [0, sinks)
      int lim[2], low[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int col = 2 * t + c;
        lim[c] = low[c] = 0;
        if (col < rows) {
          const long long end = len + (row0 + col) / G + 1;
          lim[c] = (int)min(max(end, 0ll), (long long)a.capacity);
          low[c] = a.window > 0 ? (int)max(0ll, min(end - a.window, (long long)a.capacity)) : 0;
        }
      }
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = key0 + mt * 16 + (e >> 1) * 8 + prow;
          if (key >= lim[e & 1] || (key < low[e & 1] && key >= a.sinks)) s[mt][e] = -INFINITY;
        }
    }
    // running maximum per query: over this lane's tokens, then over the lanes of its columns
    float mx[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      mx[c] = fmaxf(fmaxf(s[0][c], s[0][2 + c]), fmaxf(s[1][c], s[1][2 + c]));
#pragma unroll
      for (int w = 4; w <= 16; w <<= 1) mx[c] = fmaxf(mx[c], __shfl_xor_sync(0xffffffffu, mx[c], w));
    }
    bool rescale = mx[0] > m_run[0] + kRescale || mx[1] > m_run[1] + kRescale;
    // some s of the page too large for a query (the sum's sign bits)?
    uint32_t vs[NG / 2], large = 0;
    load_words<NG / 2>(vs, pg + F::kVS + lane * (2 * NG));
#pragma unroll
    for (int n = 0; n < NG / 2; ++n) large |= vs[n] + headroom;
    if (__any_sync(0xffffffffu, (large & 0x80008000u) != 0)) {
      // the largest exponent of s among the tokens that each query sees
      uint32_t top[2] = {0, 0};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint16_t* sv = reinterpret_cast<const uint16_t*>(pg + F::kVS);
        uint32_t x = 0;
#pragma unroll
        for (int gi = 0; gi < NG; ++gi) x = max(x, (uint32_t)sv[vslot<D>(e * 8 + prow, gi)] >> 10);
#pragma unroll
        for (int c = 0; c < 2; ++c)
          if (s[e >> 1][(e & 1) * 2 + c] > -INFINITY) top[c] = max(top[c], x);
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int w = 4; w <= 16; w <<= 1) top[c] = max(top[c], __shfl_xor_sync(0xffffffffu, top[c], w));
        const int room = kRaise + kRaiseS - 1 - (int)top[c];
        rescale |= room < raise[c];
        raise[c] = min(raise[c], room);
      }
      // (pages of like scales do not come here again)
      headroom = (32 - kRaiseS - kRaise + __reduce_max_sync(0xffffffffu, max(raise[0], raise[1]))) * 0x04000400u;
    }
    if (__any_sync(0xffffffffu, rescale)) {
      float alpha[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float m_new = fmaxf(m_run[c], mx[c]);
        const float b_new = m_new == -INFINITY ? 0.f : m_new - (float)raise[c];
        alpha[c] = m_run[c] == -INFINITY ? 1.f : ex2_approx(base[c] - b_new);  // (no maximum: the sums are 0)
        m_run[c] = m_new;
        base[c] = b_new;
        l_run[c] *= alpha[c];
      }
#pragma unroll
      for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int j = 0; j < 8; ++j) o[n][j >> 2][j & 3] *= alpha[j & 1];
#pragma unroll
      for (int j = 0; j < 4; ++j) o_lo[j] *= alpha[j & 1];
    }
    // O^T += (s V)^T P^T: lane's tokens t, t + 4, t + 8, t + 12 of 16, channels 4 g .. + 3 of each group
    constexpr int NW = D / 64;  // words per lane and token
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[mt][e] = ex2_approx(s[mt][e] - base[e & 1]);
        l_run[e & 1] += s[mt][e];
      }
      // P as the products' second operand [16 tokens][8 queries], in two fp16 parts
      uint32_t ph[2], pl[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const __half2 hi2 = __floats2half2_rn(s[mt][2 * i], s[mt][2 * i + 1]);
        const float2 back = __half22float2(hi2);
        ph[i] = transpose8x8(as_u32(hi2));
        pl[i] = transpose8x8(as_u32(__floats2half2_rn(s[mt][2 * i] - back.x, s[mt][2 * i + 1] - back.y)));
      }
      uint32_t w[4][NW], s0[NG], s1[NG], l0, l1;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        load_words<NW>(w[k], pg + F::kVC + (mt * 16 + 4 * k + t) * (D / 2) + g * (4 * NW));
      const int pair0 = mt * 8 + t, pair1 = pair0 + 4;
      load_words<NG>(s0, pg + F::kVS + pair0 * (4 * NG));
      load_words<NG>(s1, pg + F::kVS + pair1 * (4 * NG));
      load_words<1>(&l0, pg + F::kVL + (pair0 * NG + g % NG) * 4);
      load_words<1>(&l1, pg + F::kVL + (pair1 * NG + g % NG) * 4);
      uint32_t c0, c1;  // s of the lo product's row
      load_words<1>(&c0, pg + F::kVS + (pair0 * NG + g % NG) * 4);
      load_words<1>(&c1, pg + F::kVS + (pair1 * NG + g % NG) * 4);
      l0 = as_u32(__hfma2(as_half2(c0), __float2half2_rn(8.f), as_half2(l0)));
      l1 = as_u32(__hfma2(as_half2(c1), __float2half2_rn(8.f), as_half2(l1)));
      mma_f16(o_lo, l0, 0u, l1, 0u, ph[0], ph[1]);
      mma_f16(o_lo, l0, 0u, l1, 0u, pl[0], pl[1]);
#pragma unroll
      for (int gi = 0; gi < NG; ++gi) {
        const __half2 a0 = as_half2(s0[gi]), a1 = as_half2(s1[gi]);
        const uint32_t b0 = as_u32(__hfma2(as_half2(ph[0]), a0, __hmul2(as_half2(pl[0]), a0)));
        const uint32_t b1 = as_u32(__hfma2(as_half2(ph[1]), a1, __hmul2(as_half2(pl[1]), a1)));
        const int nw = gi / 2;
        const uint32_t x = __byte_perm(w[0][nw], w[1][nw], gi & 1 ? 0x7632 : 0x5410);
        const uint32_t y = __byte_perm(w[2][nw], w[3][nw], gi & 1 ? 0x7632 : 0x5410);
        mma_f16(o[gi][0], even_codes(x), odd_codes(x), even_codes(y), odd_codes(y), b0, b1);
        const uint32_t x2 = x >> 8, y2 = y >> 8;
        mma_f16(o[gi][1], even_codes(x2), odd_codes(x2), even_codes(y2), odd_codes(y2), b0, b1);
        // -8 for every code (rows of the odd ones, times 16, are the upper eight)
        mma_f16(o[gi][0], 0x80088008u, 0x80808080u, 0x80088008u, 0x80808080u, b0, b1);
        mma_f16(o[gi][1], 0x80088008u, 0x80808080u, 0x80088008u, 0x80808080u, b0, b1);
      }
    }
    __syncwarp();  // every lane has read the page
    if (lane == 0 && i + NS * n_warps < i_end) issue(i + NS * n_warps, slot);
  }
  // copies still in flight (only after a wait that gave up): they land before the memory is used again
  if (i_begin + n_done * n_warps < i_end) {
    for (int s = 0; s < NS; ++s) {
      const int k = n_done + s;
      if (i_begin + k * n_warps < i_end)
        mbar_wait_warp(&full[k % NS], (uint32_t)(k / NS) & 1u, a.status, kErrWaitTimeoutFull, 63);
    }
  }
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int w = 4; w <= 16; w <<= 1) l_run[c] += __shfl_xor_sync(0xffffffffu, l_run[c], w);

  float lo_sum[NG][2];  // the lo part of this lane's channels and columns: lane (group, t) has it
#pragma unroll
  for (int gi = 0; gi < NG; ++gi)
#pragma unroll
    for (int c = 0; c < 2; ++c) lo_sum[gi][c] = __shfl_sync(0xffffffffu, o_lo[c], gi * 4 + t);

  // ---- join the block's warps
  float* wo = reinterpret_cast<float*>(smem);   // [warps][8][D]
  float* wm = wo + n_warps * 8 * D;              // [warps][8]
  float* wl = wm + n_warps * 8;
  float* bo = wl + n_warps * 8;                  // the block: [8][D], m, l
  float* bm = bo + 8 * D;
  float* bl = bm + 8;
  __syncthreads();  // the pages are done with
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int col = 2 * t + c;
    if (col >= rows) continue;
    float* dst = wo + (warp * 8 + col) * D + 4 * g;
#pragma unroll
    for (int gi = 0; gi < NG; ++gi)
      *reinterpret_cast<float4*>(dst + gi * kGroup) =
          make_float4(fmaf(o[gi][0][c], kCodeUnit, lo_sum[gi][c]), fmaf(o[gi][0][2 + c], kCodeUnit / 16, lo_sum[gi][c]),
                      fmaf(o[gi][1][c], kCodeUnit, lo_sum[gi][c]), fmaf(o[gi][1][2 + c], kCodeUnit / 16, lo_sum[gi][c]));
    if (g == 0) {
      wm[warp * 8 + col] = m_run[c] == -INFINITY ? -INFINITY : base[c];
      wl[warp * 8 + col] = l_run[c];
    }
  }
  __syncthreads();
  const int live = max(rows, 0) * D;
  for (int e = threadIdx.x; e < live; e += n_warps * 32) {
    const int col = e / D;
    float m = -INFINITY;
    for (int w = 0; w < n_warps; ++w) m = fmaxf(m, wm[w * 8 + col]);
    float l = 0.f, v = 0.f;
    for (int w = 0; w < n_warps; ++w) {
      // no maximum: nothing was visible (all sums are 0) or every score was NaN (so is the sum)
      const float f = m == -INFINITY ? 1.f : ex2_approx(wm[w * 8 + col] - m);
      l = fmaf(f, wl[w * 8 + col], l);
      v = fmaf(f, wo[w * 8 * D + e], v);
    }
    bo[e] = v;
    if (e % D == 0) {
      bm[col] = m;
      bl[col] = l;
    }
  }
  // ---- join the cluster's blocks: each writes its share of the outputs
  if (splits > 1) cluster_sync_all();
  else __syncthreads();
  T* out = static_cast<T*>(a.o);
  for (int e = threadIdx.x + rank * (n_warps * 32); e < live; e += splits * (n_warps * 32)) {
    const int col = e / D, mrow = row0 + col;
    float m = -INFINITY, l = 0.f, v = 0.f;
    if (splits == 1) {
      l = bl[col];
      v = bo[e];
    } else {
      for (int r = 0; r < splits; ++r) m = fmaxf(m, dsmem_load(bm + col, r));
      for (int r = 0; r < splits; ++r) {
        const float f = m == -INFINITY ? 1.f : ex2_approx(dsmem_load(bm + col, r) - m);
        l = fmaf(f, dsmem_load(bl + col, r), l);
        v = fmaf(f, dsmem_load(bo + e, r), v);
      }
    }
    out[(((long long)b * a.Tq + mrow / G) * a.Hq + h * G + mrow % G) * D + e % D] =
        from_float<T>(l > 0.f || l != l ? v / l : 0.f);
  }
  // queries past the sequence's own tokens: zeros
  if (rank == 0) {
    const int total = min(8, a.Tq * G - row0);
    for (int e = live + threadIdx.x; e < total * D; e += n_warps * 32) {
      const int mrow = row0 + e / D;
      out[(((long long)b * a.Tq + mrow / G) * a.Hq + h * G + mrow % G) * D + e % D] = from_float<T>(0.f);
    }
  }
  if (splits > 1) cluster_sync_all();  // no block leaves while another reads its sums
}

template <int D, typename T>
void launch_attend(const Kv4Attend& a, cudaStream_t s) {
  using C = Kv4Attn<D>;
  static PerDeviceOnce once;
  once([] {
    UHFS_CUDA_CHECK(
        cudaFuncSetAttribute(kv4_attend_kernel<D, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::smem(kMaxWarps)));
  });
  const long long units = (long long)a.B * a.Hkv * a.q_tiles;
  if (units * a.splits > 0x7fffffffll) throw std::runtime_error("kv4 attention: too many blocks");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(units * a.splits));
  cfg.blockDim = dim3(a.warps * 32);
  cfg.dynamicSmemBytes = C::smem(a.warps);
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)a.splits;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = a.splits > 1 ? 1 : 0;
  UHFS_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kv4_attend_kernel<D, T>, a));
  note_launch();
}

void check_shape(int D, const void* pages, const char* what) {
  if (D != 64 && D != 128) throw std::runtime_error(std::string(what) + ": head_dim must be 64 or 128");
  if (reinterpret_cast<uintptr_t>(pages) % 16 != 0) throw std::runtime_error(std::string(what) + ": pages must be 16-byte aligned");
}

// rows of 8 channels are moved in 16-byte pieces
void check_rows(const void* p, int elem, long long sb, long long st, long long sh, const char* what) {
  if (reinterpret_cast<uintptr_t>(p) % 16 != 0 || (sb * elem) % 16 != 0 || (st * elem) % 16 != 0 ||
      (sh * elem) % 16 != 0)
    throw std::runtime_error(std::string(what) + ": rows must be 16-byte aligned");
}

// Calls launch(grid of place<D, rows>, first sequence, its number, first token) for all tokens of
// all sequences: x over heads, y over runs of tokens, z over sequences.  One launch, unless there are more runs or
// sequences than the 65535 of y and z (262140 tokens of 16-bit type).
template <class Launch>
void for_row_grids(int B, int tokens, int H, int D, int rows, const char* what, Launch&& launch) {
  constexpr int kMaxGrid = 65535;
  if (H > (1 << 24)) throw std::runtime_error(std::string(what) + ": too many heads");
  const int span = H * (D / 8), per_run = (span < 256 ? 256 / span : 1) * rows;  // tokens
  const int step = kMaxGrid * per_run;
  for (int b = 0; b < B; b += kMaxGrid) {
    const int nb = B - b < kMaxGrid ? B - b : kMaxGrid;
    for (long long t = 0; t < tokens; t += step) {
      const int n = tokens - t < step ? (int)(tokens - t) : step;
      launch(dim3((unsigned)((span + 255) / 256), (unsigned)((n + per_run - 1) / per_run), (unsigned)nb), b, nb, (int)t);
    }
  }
}

}  // namespace

#define UHFS_KV4_TYPES(dtype, ...)                                  \
  switch (dtype) {                                                  \
    case DT_F32: { using T = float; __VA_ARGS__; break; }           \
    case DT_F16: { using T = __half; __VA_ARGS__; break; }          \
    case DT_BF16: { using T = __nv_bfloat16; __VA_ARGS__; break; }  \
    default: throw std::runtime_error("unsupported dtype");         \
  }

void kv4_append(const Kv4Append& p, int dtype, int D, cudaStream_t s) {
  if (p.B <= 0 || p.T <= 0 || p.H <= 0) return;
  check_shape(D, p.pages, "kv4 append");
  const int elem = dtype == DT_F32 ? 4 : 2;
  check_rows(p.k, elem, p.k_stride_b, p.k_stride_t, p.k_stride_h, "kv4 append");
  check_rows(p.v, elem, p.v_stride_b, p.v_stride_t, p.v_stride_h, "kv4 append");
  Kv4Append a = p;
  a.status = device_status_ptr();
  for (long long x : {p.k_stride_t, p.k_stride_h, p.v_stride_t, p.v_stride_h})
    if (x < 0 || x > 0x7fffffffll) throw std::runtime_error("kv4 append: strides of tokens and heads must fit 32 bits");
  UHFS_KV4_TYPES(dtype, {
    constexpr int kRows = sizeof(T) == 2 ? 4 : 2;
    for_row_grids(p.B, p.T, p.H, D, kRows, "kv4 append", [&](dim3 grid, int b, int nb, int t) {
      a.B = nb;
      a.t_begin = t;
      a.k = static_cast<const T*>(p.k) + b * p.k_stride_b;
      a.v = static_cast<const T*>(p.v) + b * p.v_stride_b;
      a.pages = p.pages + (long long)b * p.H * p.pages_per_head * (40 * D);
      a.lengths = p.lengths + b;
      if (p.counts != nullptr) a.counts = p.counts + b;
      if (D == 64) kv4_append_kernel<64, T, kRows><<<grid, 256, 0, s>>>(a);
      else kv4_append_kernel<128, T, kRows><<<grid, 256, 0, s>>>(a);
      note_launch();
      UHFS_CUDA_CHECK(cudaGetLastError());
    });
  });
}

void kv4_read(const Kv4Read& p, int dtype, int D, cudaStream_t s) {
  if (p.B <= 0 || p.n <= 0 || p.H <= 0) return;
  check_shape(D, p.pages, "kv4 read");
  if (p.start < 0 || (long long)p.start + p.n > (long long)p.pages_per_head * kPage)
    throw std::runtime_error("kv4 read: tokens outside the cache");
  check_rows(p.k, 4, 0, 0, 0, "kv4 read");
  check_rows(p.v, 4, 0, 0, 0, "kv4 read");
  constexpr int kRows = 4;
  Kv4Read a = p;
  UHFS_KV4_TYPES(dtype, {
    for_row_grids(p.B, p.n, p.H, D, kRows, "kv4 read", [&](dim3 grid, int b, int nb, int t) {
      a.B = nb;
      a.t_begin = t;
      a.pages = p.pages + (long long)b * p.H * p.pages_per_head * (40 * D);
      a.k = static_cast<T*>(p.k) + (long long)b * p.n * p.H * D;
      a.v = static_cast<T*>(p.v) + (long long)b * p.n * p.H * D;
      if (D == 64) kv4_read_kernel<64, T, kRows><<<grid, 256, 0, s>>>(a);
      else kv4_read_kernel<128, T, kRows><<<grid, 256, 0, s>>>(a);
      note_launch();
      UHFS_CUDA_CHECK(cudaGetLastError());
    });
  });
}

void kv4_attend(const Kv4Attend& p, int dtype, int D, cudaStream_t s) {
  if (p.B <= 0 || p.Tq <= 0 || p.Hq <= 0) return;
  check_shape(D, p.pages, "kv4 attention");
  if (dtype != DT_BF16 && dtype != DT_F16) throw std::runtime_error("kv4 attention: q must be bf16 or fp16");
  if (p.Hkv <= 0 || p.Hq % p.Hkv != 0) throw std::runtime_error("kv4 attention: query heads must be a multiple of key / value heads");
  if (p.window < 0 || p.sinks < 0 || p.window > (1 << 30) || p.sinks > (1 << 30))
    throw std::runtime_error("kv4 attention: window or sinks out of range");
  check_rows(p.q, 2, p.q_stride_b, p.q_stride_t, p.q_stride_h, "kv4 attention");
  Kv4Attend a = p;
  a.status = device_status_ptr();
  const long long rows = (long long)p.Tq * (p.Hq / p.Hkv);
  if (rows > (1 << 28)) throw std::runtime_error("kv4 attention: too many new tokens");
  a.q_tiles = (int)((rows + 7) / 8);
  const long long units = (long long)p.B * p.Hkv * a.q_tiles;
  int seen = p.pages_per_head;
  if (p.window > 0) {
    const long long w = (long long)(p.window + p.Tq) / kPage + 2 + (p.sinks + kPage - 1) / kPage;
    if (w < seen) seen = (int)w;
  }
  // An SM holds 16 warps.  Units are split, over as many blocks as fit at once and have a page
  // for every warp; a second wave of blocks costs more than the shorter first one saves (16 x
  // 8192 tokens, 8 heads: 57 us with 4 blocks of 8 warps, 47 with 2; 8 is the largest portable
  // cluster).  Blocks of 4 warps where there are enough of them to fill the SMs: they
  // leave less over (64 x 1024 tokens, 8 heads: 33 us, 39 with 8 warps); over several waves of
  // blocks 8 (32 x 4096 tokens, 32 heads: 125 us, 131 with 4).
  constexpr int kSmWarps = 16 * 148;
  a.warps = units * 8 * 4 > kSmWarps && units * 4 <= kSmWarps ? 4 : 8;
  a.splits = 1;
  while (a.splits < 8 && units * a.splits * 2 * a.warps <= kSmWarps && a.splits * 2 * a.warps <= seen + a.warps - 1)
    a.splits *= 2;
  if (dtype == DT_BF16) {
    if (D == 64) launch_attend<64, __nv_bfloat16>(a, s);
    else launch_attend<128, __nv_bfloat16>(a, s);
  } else {
    if (D == 64) launch_attend<64, __half>(a, s);
    else launch_attend<128, __half>(a, s);
  }
}

}  // namespace uhfs
