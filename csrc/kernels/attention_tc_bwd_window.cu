// Backward of causal attention with a sliding window and sinks on the tcgen05 tensor core.
//
// Key j is seen by query i >= j when i - j < window or j < sinks.  A work item is a block
// of 128 keys of one (batch, head); it loops over the 128-query blocks that see it: from
// the diagonal to (n0 + 127 + window - 1) / 128, or to the end for a block with sinks.  With a
// window an item has few steps (three for a window of 256), so what an item costs besides
// its steps -- loading K and V, filling the pipeline, storing dK and dV -- is as
// large as they are.  The kernel is therefore persistent, one CTA per SM, and with D = 64 an
// item's loads and first products run while the item before is finished and stored (D = 128 has
// shared memory for one K / V pair only).  Items are handed out from a counter, those with sinks,
// the longest, first: dealt out in turn, 16 heads of 2 x 4096 tokens gave CTAs 45 to 84 steps
// of a mean of 59, and the kernel 540 K cycles instead of 423 K.
//
// Measured with the sums before and the conversion after it (28 us of 16 x 1024), against
// 175 and 484 us of a CTA per item with every product waiting for the one before:
//   16 x 1024 tokens, 12 x 64, window 256, 4 sinks     155 us, about 6 K cycles a step
//   2 x 4096 tokens, 16 x 128, window 1024, 4 sinks    268 us, about 6 K cycles a step
// A step's five products are 1.3 K (D = 64) and 2.6 K cycles of the tensor core; what bounds
// it is the chain S -> P -> dS -> dQ of a step, of which two steps do not fit in TMEM (D = 128:
// dV, then S^T in P^T's place, then its exponentials: 1.3, 1.2 and 2 K cycles), and the
// shared memory that the products, dS^T and the dQ boxes share.  Measured without gain for
// D = 128: dK before dQ, which frees Q earlier and dP^T later, and the next tiles brought to L2.
//
// Per step i (S^T etc. are 128 keys x 128 queries):
//   MMA      S^T = K Q_i^T; dP^T = V dO_i^T; dV += P^T dO_i; dQ_i = dS K; dK += dS^T Q_i
//   compute  P^T = exp2(S^T * scale * log2e - lse) as soon as S^T is there, stored to TMEM (the
//            A operand of dV), then dS^T = P^T (dP^T - delta), stored to shared memory.
//            Warp w holds keys 32 (w % 4).. and queries 64 (w / 4).. of the block; of its two
//            32-query pieces, one that no key of the warp sees costs nothing, one that
//            all see no comparisons.
//   read-out dQ_i from TMEM through shared fp32 boxes with TMA reduce-add
// so dV runs while dS is computed, and S^T of the next step before this step's dK and dQ.
//
// TMEM (512 columns).  D = 64: S^T, dP^T, dV, dK, dQ and P^T side by side.  D = 128: P^T
// takes S^T's place once both warps of a lane quarter hold S^T, and dQ takes dP^T's; S^T of
// the next step then waits for dV, and dP^T for the read-out of dQ.
//
// P and dS enter their products as bf16 (each value off by at most 2^-8 of itself, which a sum over
// many keys or queries averages; the gradients come out 0.0024 from 64 bits, of which their own
// rounding to bf16 is 0.0017); S, dP, the softmax, delta and all sums are fp32.
//
// q / k / v / dO are read and dQ is added through [B][T][..] maps: rows past T read as
// zeros and are not written, so ragged sequences never meet.
// Warps: 0..7 compute, 8 items and K / V / Q / lse / delta loads, 9 MMA issuer, 10 dO loads,
// 12..15 dQ read-out.  512 threads launch
// with 128 registers; the compute warpgroups take kComputeRegs of the total.
// Every wait is bounded.
#include <cudaTypedefs.h>

#include <stdexcept>
#include <string>

#include "common.cuh"
#include "kernels.h"

namespace uhfs {

CUtensorMap make_tmap_bf16_3d(const void* base, uint64_t inner, uint64_t rows, uint64_t batch,
                              uint64_t row_stride_elems, uint64_t batch_stride_elems, uint32_t box_inner,
                              uint32_t box_rows);
CUtensorMap make_tmap_f32_3d(const void* base, uint64_t inner, uint64_t rows, uint64_t batch,
                             uint64_t row_stride_elems, uint64_t batch_stride_elems, uint32_t box_inner,
                             uint32_t box_rows);

namespace {

constexpr int BK = 128;  // keys per item
constexpr int BQ = 128;  // queries per step
constexpr int kCompute = 256;
constexpr int kReadout = 128;
constexpr int kThreads = 512;
constexpr int kLaunchRegs = 128;
constexpr float kLog2e = 1.4426950408889634f;

template <int D>
struct WinCfg {
  static constexpr bool kAlias = D == 128;   // P^T in S^T's columns, dQ in dP^T's
  static constexpr int kTile = 128 * D * 2;  // one [128][D] bf16 tile (D / 64 swizzled sub-tiles)
  static constexpr int kKV = kAlias ? 1 : 2;  // K / V buffers
  static constexpr int kNQ = kAlias ? 2 : 3, kNDO = kAlias ? 1 : 2;  // Q (with lse and delta) and dO stages
  static constexpr int kRing = 4;  // items handed out ahead
  static constexpr int kComputeRegs = kAlias ? 160 : 184, kServiceRegs = kAlias ? 96 : 72;
  static_assert(2 * 128 * kComputeRegs + 2 * 128 * kServiceRegs <= kThreads * kLaunchRegs, "register split");
  static constexpr int kDST = BK * BQ * 2;
  static constexpr int kBox = 128 * 32 * 4;  // fp32 dQ box: 128 rows x 32 columns
  static constexpr int kVec = 2 * kNQ * BQ * 4;
  static constexpr int kBars = 2 * kKV + 2 * kNQ + 2 * kNDO + 12 + 2 * kRing;
  static constexpr int kSmem =
      kKV * 2 * kTile + (kNQ + kNDO) * kTile + kDST + 2 * kBox + kVec + kBars * 8 + (kRing + 4) * 16 + 16;
  static_assert(kSmem <= 227 * 1024, "attention backward shared memory");
  static_assert(kBars % 2 == 0, "the items behind the barriers are 16-byte aligned");
  static constexpr uint32_t kST = 0, kDPT = 128, kDV = 256, kDK = 256 + D;
  static constexpr uint32_t kDQ = kAlias ? kDPT : 384, kPT = kAlias ? kST : 448;
};

struct WinArgs {
  int B, H, T, BH;
  long long F;
  float sl2, scale;
  int window, sinks;
  const float* lse;    // [B, H, T] log2 domain
  const float* delta;  // [B, H, T]
  int* counter;        // items taken, zero at the start
  DeviceStatus* status;
};

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
    fa_bwd_window_kernel(const __grid_constant__ CUtensorMap tm_qkv, const __grid_constant__ CUtensorMap tm_do,
                         const __grid_constant__ CUtensorMap tm_dq, const __grid_constant__ CUtensorMap tm_dqkv,
                         const WinArgs a) {
  using Cfg = WinCfg<D>;
  constexpr int KD = D / 64;
  constexpr uint32_t KV = Cfg::kKV, NQ = Cfg::kNQ, ND = Cfg::kNDO;
  extern __shared__ __align__(1024) uint8_t smem[];
  if ((smem_u32(smem) & 1023u) != 0) {  // the swizzled tiles need it, and there is no room to round up
    if (threadIdx.x == 0) report_error(a.status, kErrBounds, 429);
    return;
  }
  uint8_t* sKV = smem;                          // [KV][K | V]
  uint8_t* sQ = sKV + KV * 2 * Cfg::kTile;      // [NQ]
  uint8_t* sDO = sQ + NQ * Cfg::kTile;          // [ND]
  uint8_t* sDST = sDO + ND * Cfg::kTile;        // dS^T
  uint8_t* sBox = sDST + Cfg::kDST;             // [2]
  float* sLse = reinterpret_cast<float*>(sBox + 2 * Cfg::kBox);  // [NQ][128]
  float* sDelta = sLse + NQ * BQ;                                // [NQ][128]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sDelta + NQ * BQ);
  uint64_t* kv_full = bars;
  uint64_t* kv_empty = kv_full + KV;   // an item's products are done with K / V
  uint64_t* q_full = kv_empty + KV;
  uint64_t* q_empty = q_full + NQ;     // dK of the step is done
  uint64_t* do_full = q_empty + NQ;
  uint64_t* do_empty = do_full + ND;   // dV of the step is done
  uint64_t* s_full = do_empty + ND;
  uint64_t* dp_full = s_full + 1;
  uint64_t* p_full = s_full + 2;       // P^T stored, S^T read
  uint64_t* ds_full = s_full + 3;      // dS^T stored, dP^T read
  uint64_t* dv_done = s_full + 4;      // dV of the step is done: P^T may be overwritten
  uint64_t* ds_free = s_full + 5;      // dQ and dK of the step are done: dS^T may be overwritten
  uint64_t* dq_full = s_full + 6;
  uint64_t* dq_free = s_full + 7;      // dQ of the step read out
  uint64_t* dkv_free = s_full + 8;     // an item's dK / dV read out
  uint64_t* staged = s_full + 9;       // dK / dV is in the dS^T tile
  uint64_t* stored = s_full + 10;      // the stores have read it
  uint64_t* done = s_full + 11;
  uint64_t* item_full = s_full + 12;   // [kRing]
  uint64_t* item_empty = item_full + Cfg::kRing;
  int* sItem = reinterpret_cast<int*>(item_empty + Cfg::kRing);  // [kRing][4]
  int* sGroup = sItem + 4 * Cfg::kRing;                           // [2][2][4] items of the compute / read-out warps
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sGroup + 16);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int T = a.T;
  const int n_blocks = (T + BK - 1) / BK, n_qblocks = (T + BQ - 1) / BQ;
  const int n_sink = min(n_blocks, (a.sinks + BK - 1) / BK);  // key blocks with sinks
  const int n_items = n_blocks * a.BH;
  struct Item {  // steps == 0: no more items
    int b, h, n0, steps;
    __device__ int i_start() const { return n0 / BQ; }  // BQ == BK: the diagonal block
  };
  // items with sinks first; the others head by head, so that CTAs share a head's Q and dO in L2
  auto decode = [&](int it) {
    if (it >= n_items) return Item{0, 0, 0, 0};
    int bh, n_block;
    if (it < n_sink * a.BH) {
      bh = it % a.BH;
      n_block = it / a.BH;
    } else {
      const int r = it - n_sink * a.BH, rest = n_blocks - n_sink;
      bh = r / rest;
      n_block = n_sink + r % rest;
    }
    const int n0 = n_block * BK;
    const int end = n0 < a.sinks ? n_qblocks : min(n_qblocks, (n0 + BK - 1 + a.window - 1) / BQ + 1);
    return Item{bh / a.H, bh % a.H, n0, end - n_block};
  };
  auto warp_arrive = [&](uint64_t* bar) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
  };
  // item k of this CTA; after a failed wait as if there were none
  auto take = [&](uint32_t k, int where) {
    const uint32_t st = k % Cfg::kRing;
    if (!mbar_wait_bounded(&item_full[st], (k / Cfg::kRing) & 1u, a.status, kErrWaitTimeoutFull, where))
      return Item{0, 0, 0, 0};
    const int4 v = *reinterpret_cast<const int4*>(sItem + st * 4);
    return Item{v.x, v.y, v.z, v.w};
  };
  auto uniform = [](int v) { return __shfl_sync(0xffffffffu, v, 0); };
  // the same for a whole warp, which also gives the slot back
  auto take_warp = [&](uint32_t k, int where) {
    Item w = take(k, where);
    w = Item{uniform(w.b), uniform(w.h), uniform(w.n0), uniform(w.steps)};
    if (lane == 0) mbar_arrive(&item_empty[k % Cfg::kRing]);
    return w;
  };
  // the same for all warps of a group, which go on together after a failed wait too: they meet at
  // named barriers
  auto take_group = [&](uint32_t k, int where, bool first, int* shared, int barrier, int threads) {
    int4* slot = reinterpret_cast<int4*>(shared + (k & 1) * 4);
    if (first) {
      const Item w = take_warp(k, where);
      if (lane == 0) *slot = make_int4(w.b, w.h, w.n0, w.steps);
    }
    named_barrier_sync(barrier, threads);
    const int4 v = *slot;
    return Item{uniform(v.x), uniform(v.y), uniform(v.z), uniform(v.w)};
  };
  static_assert(BQ == BK, "the diagonal block of key block n is query block n");
  constexpr int kProducerWarp = 8, kMmaWarp = 9, kProducerWarp2 = 10;

  if (warp == kProducerWarp && lane == 0) {
    tma_prefetch_desc(&tm_qkv);
    tma_prefetch_desc(&tm_do);
    tma_prefetch_desc(&tm_dq);
    tma_prefetch_desc(&tm_dqkv);
    for (uint32_t i = 0; i < KV; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
    }
    for (uint32_t i = 0; i < NQ; ++i) {
      mbar_init(&q_full[i], 2);  // TMA bytes + the producer's lse and delta stores
      mbar_init(&q_empty[i], 1);
    }
    for (uint32_t i = 0; i < ND; ++i) {
      mbar_init(&do_full[i], 1);
      mbar_init(&do_empty[i], 1);
    }
    mbar_init(s_full, 1);
    mbar_init(dp_full, 1);
    mbar_init(p_full, kCompute / 32);
    mbar_init(ds_full, kCompute / 32);
    mbar_init(dv_done, 1);
    mbar_init(ds_free, 1);
    mbar_init(dq_full, 1);
    mbar_init(dq_free, kReadout / 32);
    mbar_init(dkv_free, kCompute / 32);
    mbar_init(staged, kCompute / 32);
    mbar_init(stored, 1);
    mbar_init(done, 1);
    for (int i = 0; i < Cfg::kRing; ++i) {
      mbar_init(&item_full[i], 1);
      mbar_init(&item_empty[i], 4);  // compute, read-out, MMA, second producer
    }
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp >= 8) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Cfg::kServiceRegs));
  if (warp == kProducerWarp || warp == kProducerWarp2) {
    // ------------------------------------------------------------ producers: K, V, Q, lse, delta; dO
    uint32_t k = 0;  // items of this CTA so far
    bool ok = true;
    // waits in lane 0; the same answer in every lane
    auto wait = [&](uint64_t* bar, uint32_t phase, int where) {
      int good = 1;
      if (lane == 0) good = mbar_wait_bounded(bar, phase, a.status, kErrWaitTimeoutEmpty, where);
      return __shfl_sync(0xffffffffu, good, 0) != 0;
    };
    uint32_t gq = 0, gd = 0;  // Q and dO tiles issued
    auto load_q = [&](const Item& w, int t) {
      const uint32_t st = gq % NQ;
      const int q0 = (w.i_start() + t) * BQ;
      // lse and delta share Q's stage: it is given back after dK, for which every warp has used both
      // (dV, which frees the dO stage, does not wait for delta's readers).  They are read before
      // the stage is free.
      float v[BQ / 32], u[BQ / 32];
#pragma unroll
      for (int i = 0; i < BQ / 32; ++i) {
        const int qq = q0 + i * 32 + lane;
        const long long at = ((long long)w.b * a.H + w.h) * T + qq;
        v[i] = qq < T ? __ldg(a.lse + at) : INFINITY;
        u[i] = qq < T ? __ldg(a.delta + at) : 0.f;
      }
      if (!wait(&q_empty[st], ((gq / NQ) & 1u) ^ 1u, 400)) return false;
      if (lane == 0) {
        mbar_arrive_expect_tx(&q_full[st], Cfg::kTile);
        for (int kd = 0; kd < KD; ++kd)
          tma_load_3d(sQ + st * Cfg::kTile + kd * (BQ * 128), &tm_qkv, &q_full[st], w.h * D + kd * 64, q0, w.b);
      }
#pragma unroll
      for (int i = 0; i < BQ / 32; ++i) {
        sLse[st * BQ + i * 32 + lane] = v[i];
        sDelta[st * BQ + i * 32 + lane] = u[i];
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full[st]);
      ++gq;
      return true;
    };
    auto load_do = [&](const Item& w, int t) {
      const uint32_t st = gd % ND;
      if (!wait(&do_empty[st], ((gd / ND) & 1u) ^ 1u, 401)) return false;
      const int q0 = (w.i_start() + t) * BQ;
      if (lane == 0) {
        mbar_arrive_expect_tx(&do_full[st], Cfg::kTile);
        for (int kd = 0; kd < KD; ++kd)
          tma_load_3d(sDO + st * Cfg::kTile + kd * (BQ * 128), &tm_do, &do_full[st], w.h * D + kd * 64, q0, w.b);
      }
      ++gd;
      return true;
    };
    // the first producer takes the items, one ahead, and hands them out
    auto publish = [&](uint32_t n, const Item& w) {
      if (!wait(&item_empty[n % Cfg::kRing], ((n / Cfg::kRing) & 1u) ^ 1u, 406)) return false;
      if (lane == 0) {
        *reinterpret_cast<int4*>(sItem + n % Cfg::kRing * 4) = make_int4(w.b, w.h, w.n0, w.steps);
        mbar_arrive(&item_full[n % Cfg::kRing]);
      }
      return true;
    };
    if (warp == kProducerWarp2) {
      for (uint32_t n = 0; ok; ++n) {
        const Item w = take_warp(n, 407);
        if (w.steps == 0) break;
        for (int t = 0; t < w.steps && ok; ++t) ok = load_do(w, t);
      }
    }
    int taken = 0;
    Item w = decode(blockIdx.x);
    if (warp == kProducerWarp) {
      if (lane == 0) taken = atomicAdd(a.counter, 1);
      ok = publish(0, w);
    }
    for (; ok && warp == kProducerWarp && w.steps > 0; ++k) {
      const uint32_t kb = k % KV;
      // Q before K and V: with one K / V buffer those wait for the item before
      if (!load_q(w, 0) || !wait(&kv_empty[kb], ((k / KV) & 1u) ^ 1u, 402)) {
        ok = false;
        break;
      }
      if (lane == 0) {
        uint8_t* sK = sKV + kb * 2 * Cfg::kTile;
        mbar_arrive_expect_tx(&kv_full[kb], 2 * Cfg::kTile);
        for (int kd = 0; kd < KD; ++kd) {
          tma_load_3d(sK + kd * (BK * 128), &tm_qkv, &kv_full[kb], (int)a.F + w.h * D + kd * 64, w.n0, w.b);
          tma_load_3d(sK + Cfg::kTile + kd * (BK * 128), &tm_qkv, &kv_full[kb], (int)(2 * a.F) + w.h * D + kd * 64,
                      w.n0, w.b);
        }
      }
      const Item next = decode((int)gridDim.x + uniform(taken));
      ok = publish(k + 1, next);
      if (lane == 0 && next.steps > 0) taken = atomicAdd(a.counter, 1);  // used an item later
      for (int t = 1; t < w.steps && ok; ++t) ok = load_q(w, t);
      w = next;
    }
    // every issued copy lands before the CTA exits
    if (lane == 0) {
      if (warp == kProducerWarp)
        for (uint32_t i = k > KV ? k - KV : 0; i < k; ++i)
          mbar_wait_bounded(&kv_full[i % KV], (i / KV) & 1u, a.status, kErrWaitTimeoutFull, 403);
      for (uint32_t i = gq > NQ ? gq - NQ : 0; i < gq; ++i)
        mbar_wait_bounded(&q_full[i % NQ], (i / NQ) & 1u, a.status, kErrWaitTimeoutFull, 404);
      for (uint32_t i = gd > ND ? gd - ND : 0; i < gd; ++i)
        mbar_wait_bounded(&do_full[i % ND], (i / ND) & 1u, a.status, kErrWaitTimeoutFull, 405);
    }
  } else if (warp == kMmaWarp) {
    // ------------------------------------------------------------ MMA issuer
    if (elect_one_sync()) {
      constexpr uint32_t id_s = make_idesc(1, 0, 0, BK, BQ);  // K / V K-major, Q / dO K-major
      constexpr uint32_t id_kv = make_idesc(1, 0, 1, BK, D);  // P^T / dS^T K-major, dO / Q MN-major
      constexpr uint32_t id_q = make_idesc(1, 1, 1, BQ, D);   // dS MN-major, K MN-major
      const uint64_t kmaj = make_smem_desc(0, 16, 1024, kSwizzle128B);
      const uint64_t mnmaj = make_smem_desc(0, 128 * 128, 1024, kSwizzle128B);
      const uint32_t kv16 = smem_u32(sKV) >> 4, q16 = smem_u32(sQ) >> 4, do16 = smem_u32(sDO) >> 4,
                     ds16 = smem_u32(sDST) >> 4;
      constexpr uint32_t tile16 = Cfg::kTile >> 4;
      uint32_t g = 0, k = 0;  // steps and items before the current ones
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t phase, int where) {
        return mbar_wait_bounded(bar, phase & 1u, a.status, kErrWaitTimeoutAccum, where);
      };
      Item w = take(0, 422), next{};
      for (; w.steps > 0 && ok; w = next, ++k) {
        next.steps = 0;
        const uint32_t k16 = kv16 + (k % KV) * 2 * tile16, v16 = k16 + tile16;
        auto issue_s = [&](uint32_t gs, uint32_t key16) {  // S^T of step gs; its columns are free
          if (!wait(&q_full[gs % NQ], gs / NQ, 410)) return false;
          tc_fence_after();
          const uint32_t b16 = q16 + (gs % NQ) * tile16;
#pragma unroll 1
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t off = ((kk >> 2) * (128 * 128) + (kk & 3) * 32) >> 4;
            tc_mma_f16(tmem + Cfg::kST, kmaj + key16 + off, kmaj + b16 + off, id_s, kk > 0 ? 1u : 0u);
          }
          tc_commit(s_full);
          return true;
        };
        auto issue_dp = [&](uint32_t gs, uint32_t value16) {  // dP^T of step gs; its columns are free
          if (!wait(&do_full[gs % ND], gs / ND, 411)) return false;
          tc_fence_after();
          const uint32_t b16 = do16 + (gs % ND) * tile16;
#pragma unroll 1
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t off = ((kk >> 2) * (128 * 128) + (kk & 3) * 32) >> 4;
            tc_mma_f16(tmem + Cfg::kDPT, kmaj + value16 + off, kmaj + b16 + off, id_s, kk > 0 ? 1u : 0u);
          }
          tc_commit(dp_full);
          return true;
        };
        // The item's first products, unless the item before issued them.  S^T's columns are free
        // (p_full and, aliased, dv_done of the last step were waited for below), dP^T's too (ds_full
        // and, aliased, dq_free)
        if ((KV == 1 || k == 0) &&
            (!wait(&kv_full[k % KV], k / KV, 412) || !issue_s(g, k16) ||
             (Cfg::kAlias && g > 0 && !wait(dq_free, g - 1, 413)) || !issue_dp(g, v16))) {
          ok = false;
          break;
        }
        for (int t = 0; t < w.steps; ++t, ++g) {
          // whether, and with which K / V, the step after this one is begun from here
          const bool more = t + 1 < w.steps;
          if (!more) {
            mbar_arrive(&item_empty[k % Cfg::kRing]);
            next = take(k + 1, 422);
          }
          const bool ahead = more || (KV == 2 && next.steps > 0);
          const uint32_t next16 = more ? k16 : kv16 + ((k + 1) % KV) * 2 * tile16;
          if (!wait(p_full, g, 414)) {
            ok = false;
            break;
          }
          // S^T of the next step, before dV where P^T has columns of its own
          if (!Cfg::kAlias && ahead &&
              ((!more && !wait(&kv_full[(k + 1) % KV], (k + 1) / KV, 421)) || !issue_s(g + 1, next16))) {
            ok = false;
            break;
          }
          // dV += P^T dO
          if (t == 0 && k > 0 && !wait(dkv_free, k - 1, 415)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t d16 = do16 + (g % ND) * tile16, qq16 = q16 + (g % NQ) * tile16;
#pragma unroll 1
          for (int kk = 0; kk < BQ / 16; ++kk)
            tc_mma_f16_ts(tmem + Cfg::kDV, tmem + Cfg::kPT + (uint32_t)(kk * 8), mnmaj + d16 + ((kk * 16 * 128) >> 4),
                          id_kv, (t > 0 || kk > 0) ? 1u : 0u);
          tc_commit(dv_done);
          tc_commit(&do_empty[g % ND]);
          if (Cfg::kAlias && (!wait(dv_done, g, 416) || (more && !issue_s(g + 1, k16)))) {
            ok = false;
            break;
          }
          // dQ = dS K, dK += dS^T Q
          if (!wait(ds_full, g, 417) || (!Cfg::kAlias && g > 0 && !wait(dq_free, g - 1, 418))) {
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll 1
          for (int kk = 0; kk < BK / 16; ++kk) {
            const uint32_t off = (kk * 16 * 128) >> 4;
            tc_mma_f16(tmem + Cfg::kDQ, mnmaj + ds16 + off, mnmaj + k16 + off, id_q, kk > 0 ? 1u : 0u);
          }
          tc_commit(dq_full);
          if (!Cfg::kAlias && ahead && !issue_dp(g + 1, next16 + tile16)) {
            ok = false;
            break;
          }
#pragma unroll 1
          for (int kk = 0; kk < BQ / 16; ++kk) {
            const uint32_t aoff = ((kk >> 2) * (128 * 128) + (kk & 3) * 32) >> 4;
            tc_mma_f16(tmem + Cfg::kDK, kmaj + ds16 + aoff, mnmaj + qq16 + ((kk * 16 * 128) >> 4), id_kv,
                       (t > 0 || kk > 0) ? 1u : 0u);
          }
          tc_commit(ds_free);
          tc_commit(&q_empty[g % NQ]);
          if (!more) tc_commit(&kv_empty[k % KV]);
          if (Cfg::kAlias && more && (!wait(dq_free, g, 419) || !issue_dp(g + 1, v16))) {
            ok = false;
            break;
          }
        }
      }
      tc_commit(done);
      mbar_wait_bounded(done, 0, a.status, kErrWaitTimeoutAccum, 420);
    }
  } else if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Cfg::kComputeRegs));
    // ------------------------------------------------------------ compute
    const int quarter = warp & 3, half = warp >> 2;
    const int r = quarter * 32 + lane;  // key row
    const uint32_t lb = tmem + ((uint32_t)(quarter * 32) << 16);
    const bool storer = warp == 0 && lane == 0;  // issues the dK / dV stores
    uint8_t* dst_row = sDST + half * (128 * 128) + r * 128;
    uint32_t g = 0, k = 0;
    // warp-uniform; after a failed wait a warp does no more work and waits no more, but still meets
    // the named barriers
    bool ok = true;
    uint32_t n_staged = 0, n_read = 0;
    // the stores so far have read the dS^T tile
    auto tile_read = [&]() {
      if (storer) {
        bulk_wait_group_read0();
        mbar_arrive(stored);
      }
      __syncwarp();
      return mbar_wait_warp(stored, n_read++ & 1u, a.status, kErrWaitTimeoutAccum, 437);
    };
    // dK (scaled) and dV of item w, whose last step was end - 1: every product is done with the
    // last dK.  They leave through the dS^T tile with TMA stores.
    auto store_item = [&](const Item& w, uint32_t end) {
      if (ok && !mbar_wait_warp(ds_free, (end - 1) & 1u, a.status, kErrWaitTimeoutAccum, 436)) ok = false;
      // 32 columns from `col`, as the 16-byte chunks ch0.. of this key's row
      auto put = [&](uint32_t col, float scale, uint8_t* row, int ch0) {
        uint32_t v[32];
        tmem_ld_32x32b_x32_async(lb + col, v);
        tmem_wait_ld_regs<32>(v);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t h4[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int i = q * 8 + e * 2;
            h4[e] = pack_bf16x2(__uint_as_float(v[i]) * scale, __uint_as_float(v[i + 1]) * scale);
          }
          *reinterpret_cast<uint4*>(row + (((ch0 + q) ^ (r & 7)) << 4)) = make_uint4(h4[0], h4[1], h4[2], h4[3]);
        }
      };
      uint8_t* row0 = sDST + r * 128;
      // the tile holds dK and dV for D = 64, one of them at a time for D = 128
#pragma unroll 1
      for (int i = 0; i < KD && ok; ++i) {
        if (i == 1 && !tile_read()) {
          ok = false;
          break;
        }
        tc_fence_after();
        if constexpr (D == 64) {
          put(Cfg::kDK + half * 32, a.scale, row0, 4 * half);
          put(Cfg::kDV + half * 32, 1.f, row0 + 128 * 128, 4 * half);
        } else {
#pragma unroll 1
          for (int c = 0; c < 2; ++c)
            put((i == 0 ? Cfg::kDK : Cfg::kDV) + half * 64 + c * 32, i == 0 ? a.scale : 1.f,
                row0 + half * (128 * 128), 4 * c);
        }
        if (i == KD - 1) {
          tc_fence_before();
          warp_arrive(dkv_free);  // the next item may accumulate
        }
        fence_proxy_async_smem();
        warp_arrive(staged);
        if (warp == 0) {
          ok = mbar_wait_warp(staged, n_staged & 1u, a.status, kErrWaitTimeoutAccum, 438);
          if (storer && ok) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const int part = D == 64 ? c : i, col = D == 64 ? 0 : c * 64;  // dK or dV, first column
              tma_store_3d(&tm_dqkv, sDST + c * (128 * 128), (int)((part + 1) * a.F) + w.h * D + col, w.n0, w.b);
            }
            bulk_commit_group();
          }
          __syncwarp();
        }
        ++n_staged;
      }
    };
    Item last{};
    for (;; ++k) {
      const Item w = take_group(k, 439, warp == 0, sGroup, 6, kCompute);
      if (w.steps == 0) break;
      const int key = w.n0 + r, key_lo = w.n0 + quarter * 32;
      for (int t = 0; t < w.steps; ++t, ++g) {
        const int qh = (w.i_start() + t) * BQ + half * 64;  // first query of this half
        // queries [qmin, qmax] of the half are visible to this key
        const int qmin = key < T ? key - qh : 64;
        const int qmax = key < a.sinks ? 64 : key + a.window - 1 - qh;
        // per 32-query piece: 0 none visible to the warp's keys, 1 some, 2 all
        int piece[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int lo = qh + 32 * c, hi = lo + 31;
          const bool none = key_lo >= T || hi < key_lo || (key_lo >= a.sinks && lo > key_lo + 31 + a.window - 1);
          const bool all = key_lo + 31 < T && lo >= key_lo + 31 &&
                           (key_lo + 31 < a.sinks || hi <= key_lo + a.window - 1);
          piece[c] = none ? 0 : all ? 2 : 1;
        }
        // ---- P^T
        if (ok && (!mbar_wait_warp(&q_full[g % NQ], (g / NQ) & 1u, a.status, kErrWaitTimeoutFull, 430) ||
                   !mbar_wait_warp(s_full, g & 1u, a.status, kErrWaitTimeoutAccum, 431)))
          ok = false;
        uint32_t sv[64];
        if (ok) {
          tc_fence_after();
          tmem_ld_32x32b_x32_async(lb + Cfg::kST + half * 64, sv);
          tmem_ld_32x32b_x32_async(lb + Cfg::kST + half * 64 + 32, sv + 32);
          tmem_wait_ld_regs<64>(sv);
        }
        if constexpr (Cfg::kAlias) {
          // P^T overwrites S^T: the other warp of these lanes has its part too
          tc_fence_before();
          named_barrier_sync(2 + quarter, 64);
          tc_fence_after();
        }
        if (!ok) continue;
        const float4* lse4 = reinterpret_cast<const float4*>(sLse + (g % NQ) * BQ + half * 64);
        uint32_t hp[32];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (piece[c] == 0) {
#pragma unroll
            for (int i = 0; i < 16; ++i) hp[c * 16 + i] = 0u;
#pragma unroll
            for (int i = 0; i < 32; ++i) sv[c * 32 + i] = 0u;
            continue;
          }
#pragma unroll
          for (int q4 = 0; q4 < 8; ++q4) {
            const float4 l = lse4[c * 8 + q4];
            const float lv[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int i = c * 32 + q4 * 4 + e;
              sv[i] = __float_as_uint(ex2_approx(fmaf(__uint_as_float(sv[i]), a.sl2, -lv[e])));
            }
          }
          if (piece[c] == 1) {
            // bits [qmin, qmax] of the piece
            const int b0 = max(qmin - c * 32, 0), b1 = min(qmax - c * 32, 31);
            const uint32_t vis = b0 > b1 ? 0u : (0xffffffffu >> (31 - (b1 - b0))) << b0;
#pragma unroll
            for (int i = 0; i < 32; ++i) sv[c * 32 + i] = (vis >> i) & 1u ? sv[c * 32 + i] : 0u;
          }
#pragma unroll
          for (int i = 0; i < 16; ++i)
            hp[c * 16 + i] =
                pack_bf16x2(__uint_as_float(sv[c * 32 + 2 * i]), __uint_as_float(sv[c * 32 + 2 * i + 1]));
        }
        // P^T of the step before has been read (aliased: S^T was issued after that)
        if (!Cfg::kAlias && g > 0 && !mbar_wait_warp(dv_done, (g - 1) & 1u, a.status, kErrWaitTimeoutAccum, 432)) {
          ok = false;
          continue;
        }
        tmem_st_32x32b_x32(lb + Cfg::kPT + half * 32, hp);
        tmem_wait_st();
        tc_fence_before();
        warp_arrive(p_full);
        // the item before is stored here where its successor's first S^T did not have to wait for it
        if (KV == 2 && t == 0 && k > 0) store_item(last, g);
        // ---- dS^T
        if (!mbar_wait_warp(dp_full, g & 1u, a.status, kErrWaitTimeoutAccum, 434)) {
          ok = false;
          continue;
        }
        tc_fence_after();
        uint32_t pv[64];
        tmem_ld_32x32b_x32_async(lb + Cfg::kDPT + half * 64, pv);
        tmem_ld_32x32b_x32_async(lb + Cfg::kDPT + half * 64 + 32, pv + 32);
        tmem_wait_ld_regs<64>(pv);
        const float4* dlt4 = reinterpret_cast<const float4*>(sDelta + (g % NQ) * BQ + half * 64);
        uint32_t hd[32];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (piece[c] == 0) {
#pragma unroll
            for (int i = 0; i < 16; ++i) hd[c * 16 + i] = 0u;
            continue;
          }
#pragma unroll
          for (int q4 = 0; q4 < 8; ++q4) {
            const float4 d = dlt4[c * 8 + q4];
            const int i = c * 32 + q4 * 4;
            hd[i / 2] = pack_bf16x2(__uint_as_float(sv[i]) * (__uint_as_float(pv[i]) - d.x),
                                    __uint_as_float(sv[i + 1]) * (__uint_as_float(pv[i + 1]) - d.y));
            hd[i / 2 + 1] = pack_bf16x2(__uint_as_float(sv[i + 2]) * (__uint_as_float(pv[i + 2]) - d.z),
                                        __uint_as_float(sv[i + 3]) * (__uint_as_float(pv[i + 3]) - d.w));
          }
        }
        if (g > 0 && !mbar_wait_warp(ds_free, (g - 1) & 1u, a.status, kErrWaitTimeoutAccum, 435)) {
          ok = false;
          continue;
        }
        if (t == 0 && k > 0 && !tile_read()) {  // the stores of the item before
          ok = false;
          continue;
        }
#pragma unroll
        for (int ch = 0; ch < 8; ++ch)
          *reinterpret_cast<uint4*>(dst_row + ((ch ^ (r & 7)) << 4)) =
              make_uint4(hd[ch * 4], hd[ch * 4 + 1], hd[ch * 4 + 2], hd[ch * 4 + 3]);
        tc_fence_before();
        fence_proxy_async_smem();
        warp_arrive(ds_full);
      }
      if (KV == 1) store_item(w, g);
      last = w;
    }
    if (KV == 2 && ok) store_item(last, g);  // every CTA has an item
    if (storer) bulk_wait_group0();
  } else if (warp >= 12) {
    // ------------------------------------------------------------ dQ read-out
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;  // query row within the block
    const uint32_t lb = tmem + ((uint32_t)(quarter * 32) << 16);
    const bool leader = warp == 12 && lane == 0;  // issues the TMA reductions
    uint32_t g = 0, chunk = 0;
    // Columns held in registers at once, in 32s.  Aliased, dP^T of the next step waits until dQ has left
    // TMEM, which then does not wait for the first half's boxes (280 -> 268 us of 2 x 4096,
    // 16 x 128); with D = 64 nothing waits for it, and the compute warps can use the registers.
    constexpr int kHeld = Cfg::kAlias ? 2 : 1;
    bool ok = true;  // per warp; the named barriers are met in any case
    for (uint32_t k = 0;; ++k) {
      const Item w = take_group(k, 443, warp == 12, sGroup + 8, 1, kReadout);
      if (w.steps == 0) break;
      for (int t = 0; t < w.steps; ++t, ++g) {
        if (ok && !mbar_wait_warp(dq_full, g & 1u, a.status, kErrWaitTimeoutAccum, 440)) ok = false;
#pragma unroll 1
        for (int c = 0; c < D / (32 * kHeld); ++c, ++chunk) {
          uint32_t v[kHeld][32];
#pragma unroll
          for (int u = 0; u < kHeld; ++u)
#pragma unroll
            for (int i = 0; i < 32; ++i) v[u][i] = 0u;
          if (ok) {
            tc_fence_after();
#pragma unroll
            for (int u = 0; u < kHeld; ++u) tmem_ld_32x32b_x32_async(lb + Cfg::kDQ + (c * kHeld + u) * 32, v[u]);
#pragma unroll
            for (int u = 0; u < kHeld; ++u) tmem_wait_ld_regs<32>(v[u]);
            if (c == D / (32 * kHeld) - 1) {
              tc_fence_before();
              warp_arrive(dq_free);
            }
          }
          uint8_t* box = sBox + (kHeld == 1 ? (chunk & 1) * Cfg::kBox : 0);
          if (leader) {  // the reductions that last used the box(es) have read them
            if constexpr (kHeld == 1) bulk_wait_group_read1();
            else bulk_wait_group_read0();
          }
          named_barrier_sync(1, kReadout);
          if (ok) {
#pragma unroll
            for (int u = 0; u < kHeld; ++u)
#pragma unroll
              for (int ch = 0; ch < 8; ++ch)
                *reinterpret_cast<uint4*>(box + u * Cfg::kBox + r * 128 + ((ch ^ (r & 7)) << 4)) =
                    make_uint4(v[u][ch * 4], v[u][ch * 4 + 1], v[u][ch * 4 + 2], v[u][ch * 4 + 3]);
            fence_proxy_async_smem();
          }
          named_barrier_sync(1, kReadout);
          if (leader && ok) {
#pragma unroll
            for (int u = 0; u < kHeld; ++u)
              tma_reduce_add_3d(&tm_dq, box + u * Cfg::kBox, w.h * D + (c * kHeld + u) * 32, (w.i_start() + t) * BQ, w.b);
            bulk_commit_group();
          }
        }
      }
    }
    if (leader) bulk_wait_group0();
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int D>
void launch(const AttnBwdParams& p, cudaStream_t s) {
  using Cfg = WinCfg<D>;
  static PerDeviceOnce once;
  once([] {
    UHFS_CUDA_CHECK(
        cudaFuncSetAttribute(fa_bwd_window_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmem));
    // setmaxnreg redistributes the launch allocation; a different launch count
    // could make the increase wait for registers that never come
    cudaFuncAttributes fa{};
    UHFS_CUDA_CHECK(cudaFuncGetAttributes(&fa, fa_bwd_window_kernel<D>));
    if (fa.numRegs != kLaunchRegs)
      throw std::runtime_error("fa_bwd_window_kernel: compiled with " + std::to_string(fa.numRegs) +
                               " registers per thread, the register split needs " + std::to_string(kLaunchRegs));
  });
  const uint64_t F = (uint64_t)p.f.H * D, T = (uint64_t)p.f.T, B = (uint64_t)p.f.B;
  CUtensorMap tq = make_tmap_bf16_3d(p.f.q, 3 * F, T, B, 3 * F, T * 3 * F, 64, 128);
  CUtensorMap td = make_tmap_bf16_3d(p.dout, F, T, B, (uint64_t)p.do_stride_t, T * (uint64_t)p.do_stride_t, 64, 128);
  CUtensorMap tdq = make_tmap_f32_3d(p.dq_accum, F, T, B, F, T * F, 32, 128);
  CUtensorMap tdqkv = make_tmap_bf16_3d(p.dq, 3 * F, T, B, 3 * F, T * 3 * F, 64, 128);
  WinArgs a{};
  a.B = p.f.B;
  a.H = p.f.H;
  a.T = p.f.T;
  a.BH = p.f.B * p.f.H;
  a.F = (long long)F;
  a.sl2 = p.f.scale * kLog2e;
  a.scale = p.f.scale;
  a.window = p.f.window;
  a.sinks = p.f.sinks;
  a.lse = p.f.lse;
  a.delta = p.delta;
  a.counter = reinterpret_cast<int*>(p.delta + (long long)p.f.B * p.f.H * p.f.T);
  a.status = device_status_ptr();
  const long long items = (long long)((p.f.T + BK - 1) / BK) * a.BH;
  int dev = 0, sms = 0;
  UHFS_CUDA_CHECK(cudaGetDevice(&dev));
  UHFS_CUDA_CHECK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  if (items > 0x7fff0000ll) throw std::runtime_error("flash attention backward: too many key blocks");
  fa_bwd_window_kernel<D><<<(int)(items < sms ? items : sms), kThreads, Cfg::kSmem, s>>>(tq, td, tdq, tdqkv, a);
  note_launch();
  UHFS_CUDA_CHECK(cudaGetLastError());
}

}  // namespace

void flash_attn_bwd_window(const AttnBwdParams& p, cudaStream_t s) {
  if (p.f.D == 64) launch<64>(p, s);
  else launch<128>(p, s);
}

}  // namespace uhfs
