// linear_ce.cu - softmax cross entropy of a projection onto the vocabulary, with both gradients, without
// keeping the logits.  x [N, K], w [V, K], targets [N]:
//   l = scale x w^T,  lse_i = log sum_v exp(l_iv),  loss_i = lse_i - l_{i,t_i} + z lse_i^2
//   dl_iv = r_i (p_iv (1 + 2 z lse_i) - [v = t_i]),  p_iv = exp(l_iv - lse_i)
//   dx = scale dl w,  dw = scale dl^T x
// r_i is the gradient of loss_i (0 for an ignored row).  2 N V K flops for the loss; dx and dw take 4 more.
//
// Rows are worked on in chunks (of at most 2^28 logits with gradients).  For a chunk:
//   1. ce_target_kernel (once for all rows): the target's logit l_t from x and its row of w.
//   2. ce_logits_kernel: a tcgen05 GEMM over tiles of 256 rows x 256 vocabulary entries on CTA pairs,
//      whose epilogue turns each logit into e = exp(l - l_t) while it is in registers, sums e per row and
//      tile (the target left out), and stores e in 16 bits for the gradients.
//   3. ce_join_kernel: S = the row's sum, loss = log1p(S), p_t = 1 / (1 + S): no cancellation however
//      close p_t is to 1.  It also writes the row's factors and x' = r p_t (1 + 2 z lse) x in 16 bits.
//   4. ce_grads_kernel: one tcgen05 launch for both gradient products of the chunk, with the row factors
//      pulled out of the sums: dx_i = f_i sum_v e_iv w_v and dw_v = sum_i e_iv x'_i.
//   The target's own term of dl is not in e (it is 0 there): -r (1 - p_t (1 + 2 z lse)) is known in fp32,
//   so dx takes coef_i w_{t_i} in the GEMM's epilogue and dw the weighted sum of x by token
//   (token_rows.cuh).  It is the largest term of most rows, and never passes through 16 bits.
// So a training step costs 6 N V K: the logits are computed once and their exponentials are the operand
// of the gradient products.  Where the gradients are asked for later (krsi_linear_ce_grad: the upstream
// gradient differs from row to row, or there are few rows), the logits are computed again, with the rows'
// log-sum-exps from the forward as reference (ce_rows_kernel in place of 1 to 3): 8 N V K.
//
// The loss alone of few rows needs no ce_target_kernel: the logits' epilogue keeps a running maximum per
// half tile as reference, and the tile that holds a row's target writes l_t (22.1 us became 20.8 for 16 rows
// of 768 over 32768).
//
// The reference l_t is known before the GEMM, so no tile waits for another.  It is a poor one only where
// some logit is far above the target's: past 2^kMaxLift the tile's sum is taken relative to the tile's
// maximum instead, and the row is marked; marked rows' blocks are computed once more by the same kernel
// with lse as reference ("second pass", skipped tile by tile elsewhere).  bf16 holds e over fp32's whole
// range.  f16 does not, so for f16 the second pass writes e = 2^10 p for every row and the first stores
// none: 8 N V K, the price of f16's range. x' in f16 is divided by a power of two above the largest row
// factor, which the products' fp32 sums are multiplied by again: with a z-loss the factors 1 + 2 z lse are known
// after the join only, and ce_rows_kernel then writes x' in the forward too.
//
// Rounding: e and x' are rounded to the operands' 16 bits (x' costs a second rounding in the softmax part
// of dw; the alternative is to compute the logits twice); everything else is fp32 until the result.  In dw's
// rows of tokens that are no row's target, which are these sums alone, that comes to 2.1e-3 to 2.3e-3 of their
// norm (2.8e-3 where another entry than the target leads) against 1.5e-3 to 1.7e-3 for the result's own rounding
// to bf16; where targets are, their fp32 term dominates.
//
// What bounds it (B200, 32768 x 1152 over 32768 entries, bf16, loss and gradients: 7.42 TFLOP): the tensor
// cores under the power cap.  Each GEMM below runs at 1.5 GHz by itself; the step takes 6.15 to 6.55 ms, of
// which 0.2 ms are the other kernels.  cuBLAS takes 5.84 ms for the three bare products in the same loop.
#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "gemm_common.cuh"
#include "token_rows.cuh"
#include "watchdog.cuh"

KRSI_DEFINE_WATCHDOG(ce)

namespace krsi {
namespace {

using namespace sm100;
using gemm::kmajor_sw128;
using gemm::make_map;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kMaxLift = 64.f;                    // log2: e <= 2^64 in bf16, sums far below fp32's range
constexpr float kHalfScale = 1024.f;                // f16: e = 2^10 p
constexpr int kIgnored = -2, kInvalid = -1;         // targets: ignored, outside [0, V)
// Fewer rows than this without gradients take the running reference. (From as many rows on "mean" and "sum"
// form gradients in the forward, with l_t as reference; the loss is to have the same bits either way.)
constexpr int64_t kRunningRows = 1024;

// ---------------------------------------------------------------- CTA-pair GEMM pipeline
constexpr int kBM = 128;                            // rows of A per CTA (256 per pair)
constexpr int kBN = 256;                            // columns of one MMA (at most)
constexpr int kBK = 64;
constexpr int kMaxStages = 6;
constexpr int kEpiWarp0 = 4;                        // the epilogue's first warp
constexpr int kLogitsEpi = 8, kGradsEpi = 12;       // epilogue warps
constexpr int kLogitsThreads = 32 * (kEpiWarp0 + kLogitsEpi), kGradsThreads = 32 * (kEpiWarp0 + kGradsEpi);
constexpr uint32_t kATile = kBM * kBK * 2;          // 16 KB
constexpr uint32_t kMnBox = 64 * kBK * 2;           // one [64 K-rows x 64 columns] MN-major box: 8 KB
// Shared memory: the epilogue warps' staged boxes, the barriers, then the operand ring.
constexpr uint32_t kLogitsBox = 4096;               // [32 rows x 64 columns] of 16 bits
constexpr uint32_t kGradsBox = 2048;                // [32 rows x 16 columns] of fp32
constexpr int kNumBars = 2 * kMaxStages + 2 + 2 + 1;   // full, empty, acc_full, acc_empty, drain
constexpr uint32_t kSmem = 232448;
constexpr uint32_t kUsable = kSmem - 1024 - 1024;   // less the 1024-byte alignment and the barriers' KB
static_assert(kNumBars * 8 + 16 <= 1024, "barriers");
constexpr uint32_t kTmemCols = 512;
// What an item's epilogue costs in K blocks where a single accumulator leaves it exposed, for dealing the items
// out: 10 as read from the launch's ends, which spread over 83 of 395 us when it was left out (2001 x 1152 over
// 50021: 857 us a step without it, 830 with 10, 833 to 841 with 14 and 20).  Elsewhere it gives 2% (3000 x 1024 over
// 50021: 983 us without, 946 to 964 with 5 to 20) or nothing (1100 x 512, 1500 x 768, 2001 x 2048; long sums).
constexpr int kEpilogueBlocks = 10;

// MN-major operand in the 128-byte swizzle: 64-column atoms of 8 K-rows x 128 B (SBO = 1024 B), the next
// 64 columns one box further; the K step of 16 rows advances the start by 2 KB.
__device__ __forceinline__ uint64_t mnmajor_sw128(uint32_t addr) { return smem_desc(addr, kMnBox, 1024, kSw128); }

// Shape of a kernel's pipeline.  An item's accumulator has `cols` columns, a multiple of 128 up to 512:
// one MMA of up to 256 columns, or two per K step; up to 256 columns two accumulators are used in turn,
// above there is room for one.  A stage holds the CTA's 128 rows of A and its half of each MMA's columns
// of B (8 KB per 64 columns), the second MMA's 16 KB after the first's.
struct Pipe {
  int cols;
  int epi_warps;
  uint32_t box_bytes;   // one epilogue warp's staged box
  __device__ __forceinline__ uint32_t bars_at() const { return epi_warps * box_bytes; }
  __device__ __forceinline__ uint32_t ring_at() const { return bars_at() + 1024; }
  __device__ __forceinline__ uint32_t stage_bytes() const { return kATile + (cols / 128) * kMnBox; }
  __device__ __forceinline__ int stages() const {
    return min((int)((kUsable - epi_warps * box_bytes) / stage_bytes()), kMaxStages);
  }
  __device__ __forceinline__ int accs() const { return cols <= kBN ? 2 : 1; }
};

struct MmaShape {
  uint64_t a, b;              // descriptors of stage 0
  uint32_t a_step, b_step;    // per 16 of K
  uint32_t idesc, idesc2;     // of the first and the second MMA of a K step
};

// The roles of one CTA of a pair over `n_items` items (the same list in both CTAs): warp 0 loads the K
// blocks of each item into the ring, the even CTA's warp 1 issues the MMAs, the warps from 4 on of both
// CTAs run the epilogue on their CTA's 128 rows.
//   item(i)                      item i of the list; its n_kb is the number of K blocks (at least 1)
//   load(item, kb, stage, bar)   issues this CTA's TMA loads of a K block (stage_bytes() in all)
//   shape(item)                  the descriptors of its MMAs
//   prepare(item)                what an epilogue warp can do before the accumulator is there
//   epilogue(item, prepared, taddr, release)  one epilogue warp; taddr is its lane quarter's accumulator
//                                address, and release() hands it back (once, after the last TMEM read)
// Every wait is bounded; a stalled pipeline ends the CTA with an error word.
template <typename ItemOf, typename Load, typename Shape, typename Prepare, typename Epilogue>
__device__ __forceinline__ void pair_gemm(uint8_t* smem, const Pipe pipe, int n_items, uint32_t limit, ItemOf item_of,
                                          Load load, Shape shape, Prepare prepare, Epilogue epilogue) {
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + pipe.bars_at());
  uint64_t* empty = full + kMaxStages;
  uint64_t* acc_full = empty + kMaxStages;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* drain = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint8_t* ring = smem + pipe.ring_at();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const bool even = cluster_ctarank() == 0;
  const uint32_t stage_bytes = pipe.stage_bytes();
  const int stages = pipe.stages(), accs = pipe.accs();

  if (threadIdx.x == 0) {
    for (int s = 0; s < kMaxStages; ++s) {
      mbar_init(&full[s], 1);      // the even CTA's expect_tx arrival + both CTAs' TMA bytes
      mbar_init(&empty[s], 1);     // the even CTA's tcgen05.commit
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);                // the even CTA's tcgen05.commit
      mbar_init(&acc_empty[b], 2 * pipe.epi_warps);   // one arrival per epilogue warp of both CTAs
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, kTmemCols);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync();   // both CTAs' barriers initialised and TMEM allocated before either signals the other
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  auto wait = [&](uint64_t* bar, uint32_t parity) {
    return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, abort_flag, limit)) != 0;
  };
  if (warp == 0) {
    bool ok = true;
    int s = 0, round = 0;          // ring position: stage, and how often the ring has wrapped
    for (int i = 0; i < n_items && ok; ++i) {
      const auto item = item_of(i);
      for (int kb = 0; kb < item.n_kb; ++kb) {
        if (round > 0 && !wait(&empty[s], (round - 1) & 1)) {
          ok = false;
          break;
        }
        if (lane == 0) {
          if (even) mbar_arrive_expect_tx(&full[s], 2 * stage_bytes);
          load(item, kb, ring + s * stage_bytes, mapa_shared(&full[s], 0));
        }
        __syncwarp();
        if (++s == stages) s = 0, ++round;
      }
    }
    if (!ok) {
      watchdog_fire(kWdCeLoad);
      // the K blocks in flight (both CTAs' loads count on the even CTA's barriers) land before the CTA exits
      if (even) {
        for (int k = 0; k < stages; ++k) {
          const int r = k < s ? round : round - 1;   // the round in which stage k was filled last
          for (uint32_t n = 0; r >= 0 && n < limit && !mbar_try_wait(&full[k], r & 1); ++n) {
          }
        }
      }
    }
  } else if (warp == 1 && even) {
    const uint64_t stage_step = stage_bytes >> 4;
    constexpr uint64_t kSecondB = (2 * kMnBox) >> 4;
    bool ok = true;
    int s = 0, round = 0;
    for (int i = 0; i < n_items && ok; ++i) {
      const int acc = i % accs, use = i / accs;
      const auto item = item_of(i);
      if (use >= 1 && !wait(&acc_empty[acc], (use - 1) & 1)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const MmaShape m = shape(item);
      const uint32_t d = tmem + acc * kBN;
      for (int kb = 0; kb < item.n_kb; ++kb) {
        if (!wait(&full[s], round & 1)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint64_t ad = m.a + s * stage_step, bd = m.b + s * stage_step;
#pragma unroll
        for (int kk = 0; kk < kBK / 16; ++kk) {
          const uint32_t add = (kb > 0 || kk > 0) ? 1u : 0u;
          mma_ss_pair_e(d, ad + kk * m.a_step, bd + kk * m.b_step, m.idesc, add);
          if (pipe.cols > kBN) mma_ss_pair_e(d + kBN, ad + kk * m.a_step, bd + kSecondB + kk * m.b_step, m.idesc2, add);
        }
        mma_commit_pair_e(mapa_shared(&empty[s], 0));   // stage s free in both CTAs
        mma_commit_pair_e(mapa_shared(&empty[s], 1));
        if (++s == stages) s = 0, ++round;
      }
      if (!ok) break;
      mma_commit_pair_e(mapa_shared(&acc_full[acc], 0));
      mma_commit_pair_e(mapa_shared(&acc_full[acc], 1));
    }
    if (!ok) watchdog_fire(kWdCeMma);
    mma_commit_pair_e(mapa_shared(drain, 0));
    for (uint32_t i = 0; i < limit && !mbar_try_wait(drain, 0); ++i) {
    }
  } else if (warp >= kEpiWarp0) {
    const uint32_t lane_addr = (uint32_t)((warp % 4) * 32) << 16;
    bool ok = true;
    for (int i = 0; i < n_items; ++i) {
      const int acc = i % accs;
      const auto item = item_of(i);
      const auto prepared = prepare(item);
      if (!wait(&acc_full[acc], (i / accs) & 1)) {
        ok = false;
        break;
      }
      tc_fence_after();
      epilogue(item, prepared, tmem + lane_addr + acc * kBN, [&]() {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (even) mbar_arrive(&acc_empty[acc]);
          else mbar_arrive_cluster(mapa_shared(&acc_empty[acc], 0));
        }
      });
    }
    if (!ok) watchdog_fire(kWdCeEpilogue);
    if (lane == 0) bulk_wait_all();   // staged stores have completed before the CTA exits
  }

  tc_fence_before();
  cluster_sync();   // the even CTA's MMAs (which read this CTA's shared memory and TMEM) are done
  tc_fence_after();
  if (warp == 1) tmem_dealloc_pair(tmem, kTmemCols);
}

__device__ __forceinline__ uint8_t* aligned_smem(uint8_t* raw) {
  return reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
}

template <typename I>
__device__ __forceinline__ int target_code(I t, long long ignore, int V) {
  return (long long)t == ignore ? kIgnored : (t >= 0 && t < (I)V) ? (int)t : kInvalid;
}
__device__ __forceinline__ int target_of(const void* targets, int bits, int row, long long ignore, int V) {
  return bits == 64 ? target_code(reinterpret_cast<const long long*>(targets)[row], ignore, V)
                    : target_code(reinterpret_cast<const int*>(targets)[row], ignore, V);
}

// ---------------------------------------------------------------- 1: targets
// One warp per row: t_i (kIgnored, kInvalid or the token) and the target's logit in log2 units.  An
// invalid target makes the row's loss and gradients NaN (an error that cannot be raised without a
// synchronisation is at least not silent).
template <int DT, typename I>
__global__ void __launch_bounds__(256)
ce_target_kernel(const typename Elem<DT>::T* __restrict__ x, const typename Elem<DT>::T* __restrict__ w,
                 const I* __restrict__ targets, int* __restrict__ tgt, float* __restrict__ l2t,
                 float* __restrict__ l2t_low, int* __restrict__ marked, int* __restrict__ ticket, int n, int V, int K,
                 long long ignore, float c) {
  pdl_enter();
  using E = Elem<DT>;
  using T = typename E::T;
  const int row = (int)(blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32), lane = threadIdx.x % 32;
  if (row >= n) return;
  if (row % (2 * kBM) == 0 && lane == 0) marked[row / (2 * kBM)] = 0;
  if (row == 0 && lane == 0) *ticket = 0;
  const long long t = (long long)targets[row];
  const int code = target_code(t, ignore, V);
  float dot = 0.f;
  if (code >= 0) {
    const T* xr = x + (int64_t)row * K;
    const T* wr = w + (int64_t)code * K;
#pragma unroll 4
    for (int k = lane * 8; k < K; k += 256) {
      const auto a = ldg16(xr + k), b = ldg16(wr + k);
#pragma unroll
      for (int e = 0; e < 8; ++e) dot = fmaf(E::load(a.v[e]), E::load(b.v[e]), dot);
    }
    dot = warp_sum(dot);
  }
  if (lane == 0) {
    tgt[row] = code;
    const float l = c * dot;
    l2t[row] = code >= 0 ? l : code == kIgnored ? 0.f : __int_as_float(0x7fffffff);
    l2t_low[row] = code >= 0 ? fmaf(c, dot, -l) : 0.f;   // what rounding took from it
  }
}

// ---------------------------------------------------------------- 2: logits
struct LogitsArgs {
  const int* tgt;          // of the chunk's first row
  const float* ref;        // per row: the log2 reference (l2t, or what ce_join_kernel chose)
  float2* part;            // [rows][2 * n_vt]: (reference, sum) of each half tile; null in the second pass
  const int* marked;       // second pass: the 256-row blocks to compute; null: all
  int rows, V;
  int n_rt, n_vt, n_kb;
  float c;                 // scale * log2(e)
  float e_scale;           // second pass: e is multiplied by it
  int store;               // e goes to memory
  // the loss alone, few rows: the targets themselves, and where the targets' logits go (else null)
  const void* targets;
  int target_bits;
  long long ignore;
  float *l2t_out, *l2t_low_out;
  int* ticket;
  uint32_t limit;
};

// Measured at 8192 x 32768 x 1152 (bf16, e stored): 420 us, 1,474 TFLOP/s, tensor pipe 81% active at 1.51 GHz;
// at 768 columns 300 us (1,370): the tiles' operands and e together come to 50 bytes a cycle and SM through
// L2, which is what it gives.  An epilogue of 8 warps (exponential, sum, store) stays behind the MMAs.
// RUNNING: the loss alone of few rows (see the top); a variant of its own, because its epilogue's few more
// instructions cost the others 0.8%.
template <bool F16, bool RUNNING>
__global__ void __launch_bounds__(kLogitsThreads, 1)
ce_logits_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap,
                 const __grid_constant__ CUtensorMap emap, const LogitsArgs a) {
  pdl_enter();   // before any global access and before claiming TMEM
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = aligned_smem(smem_raw);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rank = (int)cluster_ctarank();
  const int pair = (int)blockIdx.x / 2, n_pairs = (int)gridDim.x / 2;
  const bool second = a.part == nullptr;

  // Row tiles run fastest, so that the pairs at work share a few vocabulary tiles of w while x stays in
  // L2.  With a list of marked row tiles only those are computed.
  int n_rt = a.n_rt;
  if (a.marked != nullptr) {
    n_rt = 0;
    for (int r = 0; r < a.n_rt; ++r) n_rt += a.marked[r] != 0;
  }
  const int n_tiles = n_rt * a.n_vt;
  if (n_tiles == 0) return;   // nothing is marked (the same for every CTA)
  struct Tile {
    int rt, vt, n_kb;
  };

  const Pipe pipe{kBN, kLogitsEpi, kLogitsBox};
  pair_gemm(
      smem, pipe, pair < n_tiles ? (n_tiles - 1 - pair) / n_pairs + 1 : 0, a.limit,
      [&](int i) {
        const int t = pair + i * n_pairs;
        int rt = t % n_rt;
        if (a.marked != nullptr) {   // the rt-th marked one
          int r = 0;
          for (int k = rt;; ++r)
            if (a.marked[r] != 0 && k-- == 0) break;
          rt = r;
        }
        return Tile{rt, t / n_rt, a.n_kb};
      },
      [&](const Tile& m, int kb, uint8_t* st, uint32_t bar) {
        tma_load_2d_pair(st, &xmap, bar, kb * kBK, m.rt * (2 * kBM) + rank * kBM);
        tma_load_2d_pair(st + kATile, &wmap, bar, kb * kBK, m.vt * kBN + rank * kBM);
      },
      [&](const Tile&) {
        const uint32_t s0 = smem_u32(smem + pipe.ring_at());
        return MmaShape{kmajor_sw128(s0), kmajor_sw128(s0 + kATile), 32 >> 4, 32 >> 4,
                        idesc_f16(2 * kBM, kBN, F16 ? 0u : 1u, false, false), 0u};
      },
      [&](const Tile&) { return 0; },
      [&](const Tile& m, int, uint32_t taddr, auto release) {
        const int ew = warp - kEpiWarp0, half = ew / 4;
        const int row0 = m.rt * (2 * kBM) + rank * kBM + (warp % 4) * 32;
        const int row = row0 + lane;
        const int col0 = m.vt * kBN + half * 128;
        const bool in = row < a.rows;
        const int t = !in ? kIgnored : RUNNING ? target_of(a.targets, a.target_bits, row, a.ignore, a.V) : a.tgt[row];
        float ref = RUNNING ? -INFINITY : in ? a.ref[row] : 0.f;   // RUNNING: the largest logit so far
        if (RUNNING && pair == 0 && rank == 0 && threadIdx.x == 32 * kEpiWarp0) *a.ticket = 0;
        const bool live = t != kIgnored;
        const uint32_t keep = live ? 0xffffffffu : 0u;   // an ignored row's e is 0 whatever its logits are
        uint8_t* box = smem + ew * kLogitsBox;
        const uint32_t acc = taddr + half * 128;
        // One pass over the 128 columns, 32 at a time: y = l - ref in log2 units, -inf at the target and
        // past the vocabulary; sum += 2^y, top = max y, and (store) e in 16 bits through the staged box.
        // Where a row has a logit far above its target's, a pass more takes its sum relative to its
        // maximum instead.
        float sum;
        bool store = a.store != 0;
        for (bool again = false;; again = true) {
          float top = -INFINITY;
          sum = 0.f;
#pragma unroll 1
          for (int j = 0; j < 4; ++j) {
            uint32_t r[32];
            __syncwarp();
            tmem_ld32(acc + j * 32, r);
            tmem_wait_ld();
            const int c0 = col0 + j * 32;
            float y[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) y[e] = fmaf(__uint_as_float(r[e]), a.c, RUNNING ? 0.f : -ref);
            // what is left out: y, and for RUNNING the accumulator that it is made of again below
            auto leave_out = [&](int e) {
              y[e] = -INFINITY;
              if (RUNNING) r[e] = a.c < 0.f ? 0x7f800000u : 0xff800000u;
            };
            if (c0 + 32 > a.V) {
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (c0 + e >= a.V) leave_out(e);
            }
            if ((unsigned)(t - c0) < 32u) {
              float lt = 0.f;
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (t == c0 + e) {
                  lt = __uint_as_float(r[e]);
                  leave_out(e);
                }
              if (RUNNING) {
                a.l2t_out[row] = a.c * lt;
                a.l2t_low_out[row] = fmaf(a.c, lt, -(a.c * lt));
              }
            }
#pragma unroll
            for (int e = 0; e < 32; e += 2) top = max3(top, y[e], y[e + 1]);
            if (RUNNING && top > ref) {   // (while every logit so far is -inf the reference stays, and e is 0)
              sum *= ex2_approx(ref - top);
              ref = top;
            }
            if (RUNNING && ref != -INFINITY && a.c != 0.f) {   // l - ref in one rounding (of 0 there is none)
#pragma unroll
              for (int e = 0; e < 32; ++e) y[e] = fmaf(__uint_as_float(r[e]), a.c, -ref);
            }
#pragma unroll
            for (int e = 0; e < 32; ++e) y[e] = ex2_approx(y[e]);
#pragma unroll
            for (int e = 0; e < 32; ++e) sum += y[e];
            if (store) {
              if ((j & 1) == 0) {   // the box's previous content has been read
                if (lane == 0) bulk_wait_read_all();
                __syncwarp();
              }
#pragma unroll
              for (int p = 0; p < 4; ++p) {
                uint32_t o[4];
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                  const float lo = y[p * 8 + h * 2] * a.e_scale, hi = y[p * 8 + h * 2 + 1] * a.e_scale;
                  o[h] = (F16 ? pack_f16x2(lo, hi) : pack_bf16x2(lo, hi)) & keep;
                }
                // 128-byte rows, 16-byte packet index xor row (the 128-byte swizzle)
                const int packet = (j & 1) * 4 + p;
                *reinterpret_cast<uint4*>(box + lane * 128 + ((packet ^ (lane & 7)) << 4)) =
                    make_uint4(o[0], o[1], o[2], o[3]);
              }
              if ((j & 1) == 1) {
                fence_async_shared();
                __syncwarp();
                const int panel = (c0 - 32) / 64;   // stored whole: zeros past the vocabulary
                if (lane == 0 && panel * 64 < a.V && row0 < a.rows) {   // the map clips rows
                  tma_store_3d(&emap, box, 0, row0, panel);
                  bulk_commit_group();
                }
              }
            }
          }
          if (RUNNING || second || again || !__any_sync(0xffffffffu, live && top > kMaxLift)) break;
          if (live && top > kMaxLift) ref += top;
          store = false;
        }
        release();
        if (!second && in)
          a.part[(int64_t)row * (2 * a.n_vt) + m.vt * 2 + half] = make_float2(ref, live ? sum : 0.f);
      });
}

// ---------------------------------------------------------------- 3: rows
// The reduced loss and the weight of each row in it, by one block, in a fixed order.
template <int NT>
__device__ __forceinline__ void reduce_rows(const float* loss, const int* tgt, float* total, float* weight, int n,
                                            int mean) {
  __shared__ double sums[NT / 32];
  __shared__ int counts[NT / 32];
  double s = 0.0;
  int c = 0;
#pragma unroll 8
  for (int i = threadIdx.x; i < n; i += NT) {
    s += (double)__ldcg(loss + i);
    c += __ldcg(tgt + i) != kIgnored;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    c += __shfl_xor_sync(0xffffffffu, c, o);
  }
  if (threadIdx.x % 32 == 0) {
    sums[threadIdx.x / 32] = s;
    counts[threadIdx.x / 32] = c;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.0;
    c = 0;
    for (int w = 0; w < NT / 32; ++w) {
      s += sums[w];
      c += counts[w];
    }
    const int m = mean ? (c > 1 ? c : 1) : 1;
    *total = (float)(s / m);
    *weight = (float)(1.0 / m);
  }
}
template <int NT>
__global__ void __launch_bounds__(NT)
ce_reduce_kernel(const float* __restrict__ loss, const int* __restrict__ tgt, float* __restrict__ total,
                 float* __restrict__ weight, int n, int mean) {
  pdl_enter();
  reduce_rows<NT>(loss, tgt, total, weight, n, mean);
}
// Rows up to which 256 threads reduce (32 rows a thread; the join's last block where one join has all rows), above
// 1024: by the rows alone, since the loss is to have the same bits whatever the chunks.
constexpr int64_t kJoinReduceRows = 8192;

struct JoinArgs {
  float *total, *weight;   // with few rows the last block to finish reduces the losses itself; or null
  int* ticket;             // blocks that have finished (zeroed by ce_target_kernel)
  int mean;
  const float2* part;      // [rows][n_part]
  int n_part;
  int* tgt;                // of ce_target_kernel, or to be written from `targets`
  const void* targets;
  int target_bits, V;
  long long ignore;
  const float* l2t;
  const float* l2t_low;    // the exact target's logit less l2t
  float* loss;             // [rows]
  float2* stats;           // [rows]: (log2-sum-exp, 1 - p_t) for ce_rows_kernel, or null
  float* coef;             // [rows]: the target's term of dl; null: no gradients
  float* factor;           // [rows]: of the row's softmax part of dx
  float* ref;              // [rows]: the second pass's reference
  int* marked;
  void* xs;                // [rows, K]: x times the row's factor
  const void* x;
  int rows, K;
  int all_second;          // f16: every row takes the second pass
  float e_scale, z;
};

// The upstream gradient of the rows' losses.
struct Upstream {
  const float* g;          // per row (stride 1) or one (stride 0); null: 1
  int64_t stride;
  const float* weight;     // a factor of g for all rows, or null
  const float* top;        // f16, where row factors differ (g, or z's): their largest magnitude
  int scaled;              // f16: row factors are divided by unit() before they meet 16 bits
  __device__ __forceinline__ float of(int64_t row) const { return g ? g[row * stride] * (weight ? *weight : 1.f) : 1.f; }
  // The power of two above the largest |g weight (1 + 2 z lse)|.
  __device__ __forceinline__ float unit() const {
    if (!scaled || (top == nullptr && g == nullptr)) return 1.f;
    const uint32_t e = __float_as_uint(top ? *top : of(0)) & 0x7f800000u;
    return e == 0u || e >= 0x7f000000u ? 1.f : 2.f * __uint_as_float(e);
  }
};

// A row's x times a factor, in 16 bits (zeros where `dead`): `ahead` holds the first packets, 1280 columns of the
// row under way at once (3 and 8 packets take the same time at 512 to 4096 columns).
constexpr int kAhead = 5;
template <int DT>
struct RowCopy {
  using T = typename Elem<DT>::T;
  Vec16<T> ahead[kAhead];
  __device__ __forceinline__ void fetch(const T* x, int K, int lane) {
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (lane * 8 + j * 256 < K) ahead[j] = ldg16(x + lane * 8 + j * 256);
  }
  __device__ __forceinline__ void write(const T* x, T* out, int K, int lane, float f, bool dead) const {
    auto put = [&](int k, Vec16<T> v) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v.v[e] = Elem<DT>::store(dead ? 0.f : f * Elem<DT>::load(v.v[e]));
      stg16(out + k, v);
    };
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (lane * 8 + j * 256 < K) put(lane * 8 + j * 256, ahead[j]);
    for (int k = lane * 8 + kAhead * 256; k < K; k += 256) put(k, ldg16(x + k));
  }
};

// What the gradients need of each row where its log-sum-exp is known from the forward (one warp per row):
// the target, the factors and x'; e will be e_scale p.
struct RowsArgs {
  const void* targets;
  const float2* stats;     // (log2-sum-exp, 1 - p_t)
  Upstream up;
  int64_t row0;            // of the chunk, for g
  int* tgt;
  float *coef, *factor, *ref;
  const void* x;
  void* xs;
  int rows, V, K;
  long long ignore;
  float e_scale, z;
};
template <int DT, typename I>
__global__ void __launch_bounds__(256)
ce_rows_kernel(const RowsArgs a) {
  pdl_enter();
  using T = typename Elem<DT>::T;
  const int row = (int)(blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32), lane = threadIdx.x % 32;
  if (row >= a.rows) return;
  RowCopy<DT> copy;
  const T* xr = reinterpret_cast<const T*>(a.x) + (int64_t)row * a.K;
  copy.fetch(xr, a.K, lane);
  const int t = target_code(reinterpret_cast<const I*>(a.targets)[row], a.ignore, a.V);
  const bool dead = t == kIgnored;
  const float2 st = a.stats[row];
  const float r = a.up.of(a.row0 + row), zl = 2.f * a.z * st.x * kLn2, soft = r * (1.f + zl);
  if (lane == 0) {
    a.tgt[row] = t;
    a.coef[row] = dead ? 0.f : r * (zl * (1.f - st.y) - st.y);
    a.factor[row] = dead ? 0.f : soft / a.e_scale;
    a.ref[row] = st.x;
  }
  copy.write(xr, reinterpret_cast<T*>(a.xs) + (int64_t)row * a.K, a.K, lane, soft / a.up.unit(), dead);
}

template <int DT>
__device__ __forceinline__ void join_row(const JoinArgs& a, int row, int lane) {
  using T = typename Elem<DT>::T;
  const int t = a.targets ? target_of(a.targets, a.target_bits, row, a.ignore, a.V) : a.tgt[row];
  if (a.targets != nullptr && lane == 0) a.tgt[row] = t;
  const float l2t = t == kInvalid ? __int_as_float(0x7fffffff) : a.l2t[row], l2t_low = a.l2t_low[row];
  const float2* pr = a.part + (int64_t)row * a.n_part;
  const T* xr = reinterpret_cast<const T*>(a.x) + (int64_t)row * a.K;
  RowCopy<DT> copy;        // on its way while the sums are added
  if (a.coef != nullptr) copy.fetch(xr, a.K, lane);
  // The parts' sums relative to l_t, which most parts' already are, unless some part's reference is too far
  // above it for that.
  float s = 0.f, top = l2t;
  bool moved = false;
#pragma unroll 8
  for (int k = lane; k < a.n_part; k += 32) {
    const float2 p = pr[k];
    moved |= p.x != l2t;
    top = fmaxf(top, p.x);
    s += p.y;
  }
  bool lifted = false;
  if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    lifted = !(top - l2t <= kMaxLift);   // or NaN
    const float from = lifted ? top : l2t;
    s = 0.f;
#pragma unroll 8
    for (int k = lane; k < a.n_part; k += 32) {
      const float2 p = pr[k];
      if (p.y != 0.f) s += p.y * exp2f(p.x - from);   // (an empty part's reference may be -inf)
    }
  } else {
    lifted = !(l2t == l2t);              // no part at all: NaN
  }
  s = warp_sum(s);
  float lse2, rest, pt;        // log2-sum-exp; 1 - p_t; p_t
  if (t == kIgnored) {
    lse2 = rest = pt = 0.f;
    lifted = false;
  } else if (!lifted) {
    s *= exp2f(-l2t_low);      // relative to the logit itself: a large one's rounding shows in s
    pt = 1.f / (1.f + s);
    rest = s * pt;
    lse2 = l2t + kLog2e * log1pf(s);
  } else {
    s += exp2f(l2t - top);
    lse2 = top + log2f(s);
    pt = exp2f(l2t - lse2);
    rest = 1.f - pt;
  }
  const float lse = lse2 * kLn2;
  if (lane == 0) {
    const float nll = t == kIgnored ? 0.f : lifted ? (lse2 - l2t) * kLn2 : log1pf(s);
    a.loss[row] = t == kIgnored ? 0.f : nll + a.z * lse * lse;
    if (a.stats != nullptr) a.stats[row] = make_float2(lse2, rest);
  }
  if (a.coef == nullptr) return;
  const bool second = a.all_second != 0 || lifted, dead = t == kIgnored;
  const float soft = (1.f + 2.f * a.z * lse) * (second ? 1.f : pt);
  if (lane == 0) {
    a.coef[row] = dead ? 0.f : 2.f * a.z * lse * pt - rest;
    a.factor[row] = dead ? 0.f : soft / a.e_scale;
    a.ref[row] = second ? lse2 : l2t;
    if (lifted && !dead) a.marked[row / (2 * kBM)] = 1;   // every writer writes the same
  }
  copy.write(xr, reinterpret_cast<T*>(a.xs) + (int64_t)row * a.K, a.K, lane, soft, dead);
}
template <int DT>
__global__ void __launch_bounds__(256)
ce_join_kernel(const JoinArgs a) {
  pdl_enter();
  const int row = (int)(blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32);
  if (row < a.rows) join_row<DT>(a, row, threadIdx.x % 32);
  if (a.total == nullptr) return;
  __shared__ bool last;
  __threadfence();    // this block's losses before its ticket
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(a.ticket, 1) == (int)gridDim.x - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  reduce_rows<256>(a.loss, a.tgt, a.total, a.weight, a.rows, a.mean);
}

// The largest |g weight (1 + 2 z lse)| over the rows that are not ignored (a fixed result whatever the order);
// g: one per row, or null for what all rows have in common (`common`, or 1); stats: null where z is 0.
template <typename I>
__global__ void __launch_bounds__(1024)
ce_top_kernel(const float* __restrict__ g, const float* __restrict__ common, const float* __restrict__ weight,
              const float2* __restrict__ stats, const I* __restrict__ targets, long long ignore, float z,
              float* __restrict__ out, int n) {
  pdl_enter();
  __shared__ float tops[32];
  float m = 0.f;
#pragma unroll 8
  for (int i = threadIdx.x; i < n; i += 1024)
    if ((long long)targets[i] != ignore)
      m = fmaxf(m, fabsf((g ? g[i] : 1.f) * (stats ? 1.f + 2.f * z * stats[i].x * kLn2 : 1.f)));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (threadIdx.x % 32 == 0) tops[threadIdx.x / 32] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 32; ++w) m = fmaxf(m, tops[w]);
    if (common) m *= fabsf(*common);
    *out = weight ? m * fabsf(*weight) : m;
  }
}

// ---------------------------------------------------------------- 4: gradients
struct GradArgs {
  int rows, V, K;
  int cols, n_ct;          // columns per tile (a multiple of 128) and column tiles (of K)
  int n_rt, splits;        // dx: row tiles, shares of the vocabulary
  int kb_voc, kb_share;    // dx: K blocks in the vocabulary, and per share
  int n_vt, kb_rows;       // dw: vocabulary tiles, K blocks in the chunk's rows
  int n_dx, n_dw;          // items
  int low_first;           // dw items that the pairs with fewer dx items take first
  // dx: splits > 1: plain sums, fp32 [splits][256 n_rt][K]; else factor (e w) + coef w_t, fp32, or
  // scaled and rounded
  int dx32, dx_part;
  const int* tgt;
  const float* factor;
  const float* coef;
  const void* w;
  // dw: fp32 sums, stored or added; or scaled and rounded, and for the tokens that occur (by token_rows.cuh's
  // start, or with few rows by tgt itself) the fp32 sums as well: rows of `sums`, by token, or (by_entry) by the
  // token's first entry
  int dw32, accumulate, few, by_entry;
  float* sums;
  const int* start;
  tokens::Order order;
  Upstream up;
  float alpha;             // of the dw sums, times up.unit()
  float scale;
  uint32_t limit;
};

// Item i of a pair: its dx items first (each a longer sum), then its dw items; the pairs that have one dx
// item less take `low_first` dw items before the rest is dealt out evenly.
struct GradItem {
  int is_dx, tile, ct, split, n_kb;
};
// One epilogue thread's row of an item.
struct GradRow {
  float mul, coef;
  bool zero;
  int64_t w_at;     // dx: w_t's first element, which coef times is added; or -1
  float* sums;      // dw in 16 bits: where the token's row of fp32 sums goes; or null
};
__device__ __forceinline__ int pair_dx(const GradArgs& a, int pair, int P) {
  return a.n_dx / P + (pair < a.n_dx % P ? 1 : 0);
}
__device__ __forceinline__ int pair_low(const GradArgs& a, int pair, int P) {
  return pair >= a.n_dx % P ? a.low_first : 0;
}
__device__ __forceinline__ int pair_items(const GradArgs& a, int pair, int P) {
  const int rest = a.n_dw - a.low_first * (P - a.n_dx % P);
  const int q = P - 1 - pair;   // the rest is dealt from the last pair down
  return pair_dx(a, pair, P) + pair_low(a, pair, P) + rest / P + (q < rest % P ? 1 : 0);
}
__device__ __forceinline__ GradItem pair_item(const GradArgs& a, int pair, int P, int i) {
  const int nd = pair_dx(a, pair, P), nl = pair_low(a, pair, P), h = a.n_dx % P;
  if (i < nd) {
    const int d = pair + i * P, rest = d / a.n_ct;
    const int split = rest / a.n_rt;
    return {1, rest % a.n_rt, d % a.n_ct, split, min(a.kb_share, a.kb_voc - split * a.kb_share)};
  }
  i -= nd;
  const int w = i < nl ? i * (P - h) + (pair - h) : a.low_first * (P - h) + (i - nl) * P + (P - 1 - pair);
  return {0, w / a.n_ct, w % a.n_ct, 0, a.kb_rows};
}

// Measured at 8192 x 32768 x 1152 (both products, fp32 out): 890 to 904 us, 1,370 to 1,390 TFLOP/s, tensor pipe
// 75% active at 1.50 GHz, 1.5 GB read (e twice is 1.07 GB).  What it was before: 192-column tiles with two
// accumulators 1,206 us (12.3 TB/s of operands out of L2: bound there), 384 columns with e in rows 925 us, in
// panels 886.  With 256-column tiles and two accumulators the whole step takes 7.27 ms instead of 6.35.
// Twelve epilogue warps instead of eight: 3% on short sums (32 K blocks), where the single accumulator of wide
// tiles shows.
template <bool F16>
__global__ void __launch_bounds__(kGradsThreads, 1)
ce_grads_kernel(const __grid_constant__ CUtensorMap ekmap, const __grid_constant__ CUtensorMap wmap,
                const __grid_constant__ CUtensorMap emmap, const __grid_constant__ CUtensorMap xsmap,
                const __grid_constant__ CUtensorMap dxmap, const __grid_constant__ CUtensorMap dwmap,
                const GradArgs a) {
  pdl_enter();   // before any global access and before claiming TMEM
  constexpr int DT = F16 ? KRSI_F16 : KRSI_BF16;
  using E = Elem<DT>;
  using T = typename E::T;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = aligned_smem(smem_raw);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rank = (int)cluster_ctarank();
  const int pair = (int)blockIdx.x / 2, P = (int)gridDim.x / 2;
  const int cols1 = min(a.cols, kBN), cols2 = a.cols - cols1;   // of the two MMAs

  const Pipe pipe{a.cols, kGradsEpi, kGradsBox};
  pair_gemm(
      smem, pipe, pair_items(a, pair, P), a.limit,
      [&](int i) { return pair_item(a, pair, P, i); },
      [&](const GradItem& m, int kb, uint8_t* st, uint32_t bar) {
        const int k = ((m.is_dx ? m.split * a.kb_share : 0) + kb) * kBK;
        const CUtensorMap* b = m.is_dx ? &wmap : &xsmap;
        if (m.is_dx) tma_load_3d_pair(st, &ekmap, bar, 0, m.tile * (2 * kBM) + rank * kBM, k / 64);
        else tma_load_3d_pair(st, &emmap, bar, 0, k, (m.tile * 2 + rank) * 2);   // two panels
        const int c1 = m.ct * a.cols + rank * (cols1 / 2), c2 = m.ct * a.cols + cols1 + rank * (cols2 / 2);
        uint8_t* bs = st + kATile;
        for (int c = 0; c < cols1 / 2; c += 64, bs += kMnBox) tma_load_2d_pair(bs, b, bar, c1 + c, k);
        for (int c = 0; c < cols2 / 2; c += 64, bs += kMnBox) tma_load_2d_pair(bs, b, bar, c2 + c, k);
      },
      [&](const GradItem& m) {
        const uint32_t s0 = smem_u32(smem + pipe.ring_at());
        return MmaShape{m.is_dx ? kmajor_sw128(s0) : mnmajor_sw128(s0), mnmajor_sw128(s0 + kATile),
                        m.is_dx ? 32u >> 4 : (16u * 128u) >> 4, (16u * 128u) >> 4,
                        idesc_f16(2 * kBM, cols1, F16 ? 0u : 1u, !m.is_dx, true),
                        idesc_f16(2 * kBM, cols2, F16 ? 0u : 1u, !m.is_dx, true)};
      },
      [&](const GradItem& m) {
        const int row = m.tile * (2 * kBM) + rank * kBM + (warp % 4) * 32 + lane;   // of dx, or the token of dw
        GradRow r{1.f, 0.f, false, -1, nullptr};
        const bool few = !m.is_dx && a.sums && a.few;
        int first = -1;
        if (few) {
          if (a.by_entry) first = tokens::first_near(a.tgt, a.rows, row - lane);
          else if (tokens::tokens_near(a.tgt, a.rows, row - lane) >> lane & 1) first = row;
        }
        if (row >= (m.is_dx ? a.rows : a.V)) return r;
        if (!m.is_dx) {
          r.mul = a.alpha * a.up.unit();
          if (few) {
            if (first >= 0) r.sums = a.sums + (int64_t)first * a.K;
          } else if (a.sums) {
            const int k = a.order.key(row), at = a.start[k];
            if (at < a.start[k + 1]) r.sums = a.sums + (int64_t)(a.by_entry ? at : row) * a.K;
          }
        } else if (!a.dx_part) {
          const int t = a.tgt[row];
          r.mul = a.factor[row];
          r.coef = a.coef[row];
          r.zero = t == kIgnored;
          if (t >= 0) r.w_at = (int64_t)t * a.K;
        }
        return r;
      },
      [&](const GradItem& m, const GradRow& r, uint32_t taddr, auto release) {
        const int ew = warp - kEpiWarp0, third = ew / 4;
        const int row0 = m.tile * (2 * kBM) + rank * kBM + (warp % 4) * 32;
        const bool wide = m.is_dx ? a.dx32 : a.dw32;      // fp32 out
        const bool any = row0 < (m.is_dx ? a.rows : a.V);
        const CUtensorMap* map = m.is_dx ? &dxmap : &dwmap;
        const int out_row = m.is_dx ? m.split * (a.n_rt * 2 * kBM) + row0 : row0;
        // 16 columns at a time (every third 16 of the tile) through the staged box: [32 rows x 16 columns]
        // of fp32 in the 64-byte swizzle, or of 16 bits in the 32-byte swizzle, two such boxes in turn; the
        // maps clip rows and columns.  The target's row of w for the next columns is on its way while these
        // are worked on.
        Vec16<T> wt[2];
        auto fetch = [&](int col) {
          if (r.w_at >= 0)
#pragma unroll
            for (int p = 0; p < 2; ++p)
              if (col + 8 * p < a.K) wt[p] = ldg16(reinterpret_cast<const T*>(a.w) + r.w_at + col + 8 * p);
        };
        fetch(m.ct * a.cols + third * 16);
        constexpr int kStep = 16 * (kGradsEpi / 4);
        int turn = 0;
#pragma unroll 1
        for (int j = third * 16; j < a.cols; j += kStep, ++turn) {
          const int col = m.ct * a.cols + j;
          uint32_t q[16];
          __syncwarp();
          tmem_ld16(taddr + j, q);
          tmem_wait_ld();
          if (j + kStep >= a.cols) release();
          float v[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) v[e] = r.zero ? 0.f : r.mul * __uint_as_float(q[e]);
          if (r.w_at >= 0) {
#pragma unroll
            for (int p = 0; p < 2; ++p)
              if (col + 8 * p < a.K)
#pragma unroll
                for (int e = 0; e < 8; ++e) v[8 * p + e] = fmaf(r.coef, E::load(wt[p].v[e]), v[8 * p + e]);
            if (j + kStep < a.cols) fetch(col + kStep);
          }
          if (r.sums != nullptr) {   // (the 16-bit row is written again from these)
#pragma unroll
            for (int p = 0; p < 4; ++p)
              if (col + 4 * p < a.K)
                *reinterpret_cast<float4*>(r.sums + col + 4 * p) =
                    make_float4(v[4 * p], v[4 * p + 1], v[4 * p + 2], v[4 * p + 3]);
          }
          uint8_t* box = smem + ew * kGradsBox + (!wide && (turn & 1) ? kGradsBox / 2 : 0);
          if (lane == 0) {   // the box's previous content has been read
            if (wide || turn < 2) bulk_wait_read_all();
            else bulk_wait_read_but_one();
          }
          __syncwarp();
          if (wide) {   // 64-byte rows: the packet index xor bits 1-2 of the row
#pragma unroll
            for (int p = 0; p < 4; ++p)
              *reinterpret_cast<float4*>(box + lane * 64 + ((p ^ ((lane >> 1) & 3)) << 4)) =
                  make_float4(v[4 * p], v[4 * p + 1], v[4 * p + 2], v[4 * p + 3]);
          } else {      // 32-byte rows: xor bit 2 of the row
#pragma unroll
            for (int p = 0; p < 2; ++p) {
              uint32_t o[4];
#pragma unroll
              for (int h = 0; h < 4; ++h) {
                const float lo = a.scale * v[8 * p + 2 * h], hi = a.scale * v[8 * p + 2 * h + 1];
                o[h] = F16 ? pack_f16x2(lo, hi) : pack_bf16x2(lo, hi);
              }
              *reinterpret_cast<uint4*>(box + lane * 32 + ((p ^ ((lane >> 2) & 1)) << 4)) =
                  make_uint4(o[0], o[1], o[2], o[3]);
            }
          }
          fence_async_shared();
          __syncwarp();
          if (lane == 0 && any && col < a.K) {
            if (!m.is_dx && a.accumulate) tma_reduce_add_2d(map, box, col, out_row);
            else tma_store_2d(map, box, col, out_row);
          }
          if (lane == 0) bulk_commit_group();   // one group a step, empty where nothing is stored
        }
      });
}

// dx from the shares of the vocabulary (`share` values apart, added in order): 4 columns of kJoinRows rows
// per thread, their loads in flight together.
constexpr int kJoinRows = 4;
template <int DT>
__global__ void __launch_bounds__(128)
ce_dx_join_kernel(const float* __restrict__ part, int splits, int64_t share, const int* __restrict__ tgt,
                  const float* __restrict__ factor, const float* __restrict__ coef,
                  const typename Elem<DT>::T* __restrict__ w, void* __restrict__ dx, int rows, int K, float scale,
                  int dx32) {
  pdl_enter();
  using E = Elem<DT>;
  using T = typename E::T;
  const int col = (int)(blockIdx.x * blockDim.x + threadIdx.x) * 4;
  if (col >= K) return;
  const int row0 = blockIdx.y * kJoinRows;
  int t[kJoinRows];
  float v[kJoinRows][4] = {};
#pragma unroll
  for (int r = 0; r < kJoinRows; ++r) t[r] = row0 + r < rows ? tgt[row0 + r] : kIgnored;
#pragma unroll 2
  for (int s = 0; s < splits; ++s) {
#pragma unroll
    for (int r = 0; r < kJoinRows; ++r) {
      if (t[r] == kIgnored) continue;
      const float4 b = __ldg(reinterpret_cast<const float4*>(part + s * share + (int64_t)(row0 + r) * K + col));
      v[r][0] += b.x; v[r][1] += b.y; v[r][2] += b.z; v[r][3] += b.w;
    }
  }
#pragma unroll
  for (int r = 0; r < kJoinRows; ++r) {
    const int row = row0 + r;
    if (row >= rows) break;
    const int64_t at = (int64_t)row * K + col;
    const float f = t[r] == kIgnored ? 0.f : factor[row];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[r][e] *= f;
    if (t[r] >= 0) {
      const auto q = *reinterpret_cast<const tokens::Pack<T, 4>*>(w + (int64_t)t[r] * K + col);
      const float c = coef[row];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[r][e] = fmaf(c, E::load(q.v[e]), v[r][e]);
    }
    if (dx32) {
      *reinterpret_cast<float4*>(reinterpret_cast<float*>(dx) + at) = make_float4(v[r][0], v[r][1], v[r][2], v[r][3]);
    } else {
      tokens::Pack<T, 4> o;
#pragma unroll
      for (int e = 0; e < 4; ++e) o.v[e] = E::store(scale * v[r][e]);
      *reinterpret_cast<tokens::Pack<T, 4>*>(reinterpret_cast<T*>(dx) + at) = o;
    }
  }
}

// out = round(scale (g weight) a), 8 values per thread (n a multiple of 8).
template <int DT>
__global__ void __launch_bounds__(256)
ce_finish_kernel(const float* __restrict__ a, typename Elem<DT>::T* __restrict__ out, int64_t n, float scale,
                 const float* __restrict__ g, const float* __restrict__ weight) {
  pdl_enter();
  float s = scale;
  if (g) s *= *g;
  if (weight) s *= *weight;
  const int64_t stride = (int64_t)gridDim.x * blockDim.x * 8;
  for (int64_t i = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) * 8; i < n; i += stride) {
    const float4 b0 = *reinterpret_cast<const float4*>(a + i), b1 = *reinterpret_cast<const float4*>(a + i + 4);
    const float v[8] = {b0.x, b0.y, b0.z, b0.w, b1.x, b1.y, b1.z, b1.w};
    Vec16<typename Elem<DT>::T> o;
#pragma unroll
    for (int e = 0; e < 8; ++e) o.v[e] = Elem<DT>::store(s * v[e]);
    stg16(out + i, o);
  }
}

// The weighted sums of x by target token, added to rows of fp32 sums: in place, or (16-bit dw) into the
// finished rows.
struct DwSums {
  float* dw32;
  int64_t K;
  // One addition per element and call, so a reduction in L2 (no read to wait for) gives the same bits
  // every time.
  static constexpr bool kUsesFirst = false;
  using Base = tokens::NoBase;
  __device__ __forceinline__ Base fetch(int, int, uint32_t) const { return {}; }
  __device__ __forceinline__ void packet(int v, uint32_t c, const float* s, Base) const {
    float* p = dw32 + v * K + c * 8;
#pragma unroll
    for (int h = 0; h < 8; h += 4)
      asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(p + h), "f"(s[h]), "f"(s[h + 1]),
                   "f"(s[h + 2]), "f"(s[h + 3])
                   : "memory");
  }
  __device__ __forceinline__ void zero(int, uint32_t) const {}
  __device__ __forceinline__ void column(int v, int, int col, float s) const { dw32[v * K + col] += s; }
};
template <int DT>
struct DwRows {
  using T = typename Elem<DT>::T;
  const float* sums;       // rows by token, or by the token's first entry
  T* dw;
  int64_t K;
  float scale;
  bool by_entry;
  static constexpr bool kUsesFirst = true;
  struct Base {
    Vec16<float> a, b;
  };
  __device__ __forceinline__ Base fetch(int v, int first, uint32_t c) const {
    const float* p = sums + (by_entry ? first : v) * K + c * 8;
    return {ldg16(p), ldg16(p + 4)};
  }
  __device__ __forceinline__ void packet(int v, uint32_t c, const float* s, const Base& base) const {
    Vec16<T> o;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o.v[e] = Elem<DT>::store(scale * (base.a.v[e] + s[e]));
      o.v[4 + e] = Elem<DT>::store(scale * (base.b.v[e] + s[4 + e]));
    }
    stg16(dw + v * K + c * 8, o);
  }
  __device__ __forceinline__ void zero(int, uint32_t) const {}
  __device__ __forceinline__ void column(int v, int first, int col, float s) const {
    dw[v * K + col] = Elem<DT>::store(scale * (sums[(by_entry ? first : v) * K + col] + s));
  }
};

// ---------------------------------------------------------------- host
// 2-D view of fp32 rows, copied in boxes of 32 rows x 16 columns with the 64-byte swizzle; stores skip
// what is outside.
inline bool make_map_f32(CUtensorMap* map, const void* base, int64_t rows, int64_t cols) {
  attn::EncodeTiledFn enc = attn::encode_fn();
  if (!enc) return false;
  memset(map, 0, sizeof(*map));
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)cols * 4};
  cuuint32_t box[2] = {16, 32};
  cuuint32_t estr[2] = {1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, const_cast<void*>(base), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename Kern>
int max_pairs(Kern kern, int threads) {   // clusters of two of `kern` that fit on the device at once; 0: none
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * (device_sm_count() / 2));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = kSmem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) n = 0;
  cudaGetLastError();   // a refused query leaves no sticky error behind
  return n;
}

// Pairs that the device runs at once, asked once per device (both kernels, both types: the same shared
// memory and TMEM).
inline int device_pairs() {
  static std::atomic<int> cached[64];   // pairs + 1 once asked; races only repeat the question
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  int v = cached[dev].load(std::memory_order_relaxed);
  if (v == 0) {
    v = std::min(std::min(std::min(max_pairs(ce_logits_kernel<false, false>, kLogitsThreads),
                                   max_pairs(ce_logits_kernel<true, false>, kLogitsThreads)),
                          std::min(max_pairs(ce_logits_kernel<false, true>, kLogitsThreads),
                                   max_pairs(ce_logits_kernel<true, true>, kLogitsThreads))),
                 std::min(max_pairs(ce_grads_kernel<false>, kGradsThreads),
                          max_pairs(ce_grads_kernel<true>, kGradsThreads))) + 1;
    cached[dev].store(v, std::memory_order_relaxed);
  }
  return v - 1;
}

template <typename... KArgs, typename... Args>
cudaError_t launch_pairs(void (*kern)(KArgs...), int threads, int pairs, cudaStream_t stream, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * pairs);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...);
}

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// e, in panels of 64 vocabulary entries, each [rows][64]: what one TMA box takes (64 columns of some
// rows) is contiguous, where rows of V elements would scatter it over as many DRAM pages as it has rows.
inline bool make_panel_map(CUtensorMap* map, const void* base, int64_t rows, int64_t panels, bool f16,
                           uint32_t box_rows, uint32_t box_panels) {
  attn::EncodeTiledFn enc = attn::encode_fn();
  if (!enc) return false;
  memset(map, 0, sizeof(*map));
  cuuint64_t dims[3] = {64, (cuuint64_t)rows, (cuuint64_t)panels};
  cuuint64_t strides[2] = {128, (cuuint64_t)rows * 128};
  cuuint32_t box[3] = {64, box_rows, box_panels};
  cuuint32_t estr[3] = {1, 1, 1};
  return enc(map, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base),
             dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Sizes of one call.
struct Plan {
  int64_t N, V, K;
  bool dx, dw, known;      // gradients wanted; from known log-sum-exps (krsi_linear_ce_grad)
  bool grads;              // either
  bool direct;             // dw leaves the GEMM in 16 bits
  bool by_entry;           // then the fp32 sums of the tokens that occur stand by first entry, not by token
  int64_t n_vt, panels;    // vocabulary tiles; panels of e
  int64_t chunk, chunks;   // rows per chunk (a multiple of 256)
  int cols, n_ct;
  int64_t splits;          // of dx over the vocabulary
};

// (The tiles and shares do not depend on which gradients are wanted: one alone has the bits that it has with the
// other.)
inline Plan make_plan(int64_t N, int64_t V, int64_t K, bool dx, bool dw, bool known, int pairs) {
  const bool grads = dx || dw;
  Plan p{N, V, K, dx, dw, known, grads};
  p.n_vt = ceil_div(V, kBN);
  p.panels = ceil_div(V, 64);
  // Chunks of equal size, of at least 256 rows: with gradients of at most 2^28 logits (512 MB of e); the loss alone
  // keeps the half tiles' sums only, at most 256 MB of them (2^17 rows of up to 32768 entries).
  const int64_t kept = grads ? ((int64_t)1 << 28) / (p.panels * 64) : ((int64_t)1 << 28) / (2 * p.n_vt * 8);
  const int64_t most = std::max<int64_t>(256, std::min<int64_t>(1 << 17, kept / 256 * 256));
  p.chunks = std::max<int64_t>(1, ceil_div(N, most));
  p.chunk = std::max<int64_t>(256, ceil_div(ceil_div(N, p.chunks), 256) * 256);
  p.chunks = std::max<int64_t>(1, ceil_div(N, p.chunk));
  p.direct = known && p.chunks == 1;
  // V K floats of sums would be mostly empty with few rows: 604 MB for one row over 131072 x 1152.  By entry, N K
  // do, but a tile's epilogue then looks up first positions and not presence: 72.4 us against 71.6 for 257 rows of
  // 512 over 10007 (20 MB), which is taken from 32 MB on only.
  p.by_entry = p.direct && N < V && V * K > ((int64_t)1 << 23);
  // Column tiles of K.  Per K block of 64 a pair's tensor cores take 2 cycles a column, and its operands
  // (16 KB of A and 64 B a column of B for each CTA) come from L2 at about 50 bytes a cycle and SM, as
  // measured on the logits' tiles, so wider tiles feed the tensor cores better.  Up to 256 columns two
  // accumulators alternate and the epilogue is hidden: with short sums (few rows) that counts more.
  int64_t best = INT64_MAX;
  for (int m = 1; m <= (p.chunk <= 1024 ? 2 : 4); ++m) {
    const int64_t n = ceil_div(K, 128 * m);
    const int64_t cost = n * std::max<int64_t>(256 * m, (16384 + 8192 * m) / 50);
    if (cost <= best) {
      best = cost;
      p.cols = 128 * m;
      p.n_ct = (int)n;
    }
  }
  // dx has few, long sums: shares of the vocabulary where one sum is longer than a pair's part of all the
  // work (at least 8 K blocks each).
  const int64_t tiles = p.chunk / 256 * p.n_ct, kb = ceil_div(V, kBK);
  const int64_t work = tiles * kb + p.n_vt * p.n_ct * ceil_div(std::min(N, p.chunk), kBK);
  p.splits = std::max<int64_t>(1, std::min(ceil_div(kb * pairs, work), kb / 8));
  p.splits = ceil_div(kb, ceil_div(kb, p.splits));   // no empty share
  return p;
}

struct Space {
  void* e;
  void* xs;
  float2 *part, *stats;
  float *dw32, *dx_part;
  int* tgt;
  float *l2t, *l2t_low, *coef, *factor, *ref, *top;
  int *marked, *ticket;
  tokens::Space sorted;
  size_t bytes;
};
inline Space space_at(void* base, const Plan& p) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(base);
  Space s{};
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const uintptr_t r = at + off;
    off += (bytes + 255) / 256 * 256;
    return r;
  };
  const int64_t rows = std::min(p.chunk, p.N);
  s.tgt = reinterpret_cast<int*>(take((size_t)p.N * 4));
  s.l2t = reinterpret_cast<float*>(take((size_t)p.N * 4));
  s.l2t_low = reinterpret_cast<float*>(take((size_t)p.N * 4));
  s.marked = reinterpret_cast<int*>(take((size_t)(p.N / 256 + 1) * 4));
  s.ticket = reinterpret_cast<int*>(take(4));
  s.part = reinterpret_cast<float2*>(p.known ? 0 : take((size_t)rows * 2 * p.n_vt * 8));
  if (p.grads) {
    s.coef = reinterpret_cast<float*>(take((size_t)p.N * 4));
    s.factor = reinterpret_cast<float*>(take((size_t)p.N * 4));
    s.ref = reinterpret_cast<float*>(take((size_t)p.N * 4));
    s.top = reinterpret_cast<float*>(take(4));
    s.stats = reinterpret_cast<float2*>(p.known ? 0 : take((size_t)p.N * 8));
    s.e = reinterpret_cast<void*>(take((size_t)rows * p.panels * 128));
    s.xs = reinterpret_cast<void*>(take((size_t)rows * p.K * 2));
    s.dx_part = reinterpret_cast<float*>(p.dx && p.splits > 1 ? take((size_t)p.splits * p.chunk * p.K * 4) : 0);
    if (p.dw) {
      const int64_t sum_rows = p.by_entry ? p.N : p.V;
      s.dw32 = reinterpret_cast<float*>(p.known ? take((size_t)sum_rows * p.K * 4) : 0);
      if (p.N > tokens::kFewRows) {
        const size_t sort_off = off;
        s.sorted = tokens::space_at(reinterpret_cast<void*>(at + sort_off), p.N, p.V, p.K);
        off += s.sorted.bytes;
      }
    }
  }
  s.bytes = off;
  return s;
}

struct Call {
  const void *x, *w, *targets;
  int target_bits;
  float* loss;             // [N] rows: the forward; null: gradients from stats
  float *total, *row_weight;   // the reduced loss and the weight of a row in it, or null
  int mean;
  float2* stats;           // [N]: written by the forward (or null), read by the gradients
  const float* g;
  int64_t g_stride;
  const float* weight;
  void* dx;                // null: no gradients
  void* dw;
  float scale, z;
  int64_t ignore;
};

template <bool F16>
int run(const Call& c, const Plan& p, const Space& s, int pairs, cudaStream_t stream) {
  constexpr int DT = F16 ? KRSI_F16 : KRSI_BF16;
  using T = typename Elem<DT>::T;
  const float c2 = c.scale * kLog2e;
  const T* x = static_cast<const T*>(c.x);
  const T* w = static_cast<const T*>(c.w);
  const int N = (int)p.N, V = (int)p.V, K = (int)p.K;
  const bool known = c.loss == nullptr;   // the rows' log-sum-exps
  const bool wide = c.target_bits == 64;
  const dim3 row_grid((unsigned)ceil_div(N, 8));
  Upstream up{c.g, c.g_stride, c.weight, nullptr, F16};
  const bool running = !known && !p.grads && p.N < kRunningRows;
  if (!known && !running) {
    auto kern = [&](auto k, auto* t) {
      return launch_pdl(k, row_grid, dim3(256), 0, stream, x, w, t, s.tgt, s.l2t, s.l2t_low, s.marked, s.ticket, N, V, K,
                        (long long)c.ignore, c2);
    };
    KRSI_CUDA_TRY(wide ? kern(ce_target_kernel<DT, long long>, (const long long*)c.targets)
                       : kern(ce_target_kernel<DT, int>, (const int*)c.targets));
  }
  // f16 holds x' only where the row factors leave its magnitude near x's, so they are divided by a power of two
  // above the largest.  The factors differ between rows with one g per row, and with a z-loss: its 1 + 2 z lse is
  // known after the join, so the forward then forms x' as the gradients from known log-sum-exps do.
  const bool tops = F16 && p.grads && (c.z != 0.f || c.g_stride == 1);
  const bool rows_after_join = tops && !known;
  float2* stats = c.stats ? c.stats : s.stats;
  if (tops) up.top = s.top;
  auto find_top = [&](int64_t r0, int64_t rows) -> cudaError_t {
    auto kern = [&](auto k, auto* t) {
      return launch_pdl(k, dim3(1), dim3(1024), 0, stream, c.g_stride == 1 ? c.g + r0 : nullptr,
                        c.g_stride == 1 ? nullptr : c.g, c.weight, c.z != 0.f ? (const float2*)stats + r0 : nullptr, t + r0,
                        (long long)c.ignore, c.z, s.top, (int)rows);
    };
    return wide ? kern(ce_top_kernel<long long>, (const long long*)c.targets)
                : kern(ce_top_kernel<int>, (const int*)c.targets);
  };
  const float e_scale = F16 ? kHalfScale : 1.f;
  const bool few = p.N <= tokens::kFewRows;
  const bool joined = p.chunks == 1 && p.N <= kJoinReduceRows;
  if (p.grads && c.dw && !few)
    KRSI_CUDA_TRY(tokens::token_sort(c.targets, c.target_bits, N, V, c.ignore, s.sorted.start, s.sorted.pos,
                                     s.sorted.tok, stream));

  CUtensorMap wk, wm;
  const auto sw128 = CU_TENSOR_MAP_SWIZZLE_128B;
  if (!make_map(&wk, w, V, K, K, F16, kBK, kBM, sw128) || !make_map(&wm, w, V, K, K, F16, 64, kBK, sw128))
    return KRSI_ERR_CUDA;
  float* dw32 = known ? s.dw32 : static_cast<float*>(c.dw);
  CUtensorMap dwm = wm;
  if (c.dw && !(p.direct ? make_map(&dwm, c.dw, V, K, K, F16, 16, 32, CU_TENSOR_MAP_SWIZZLE_32B)
                         : make_map_f32(&dwm, dw32, V, K)))
    return KRSI_ERR_CUDA;
  for (int64_t r0 = 0; r0 < p.N; r0 += p.chunk) {
    const int64_t rows = std::min(p.chunk, p.N - r0);
    const void* targets = static_cast<const char*>(c.targets) + r0 * (c.target_bits / 8);
    const T* xc = x + r0 * K;
    CUtensorMap xm, es, ek, em, xs;
    if (!make_map(&xm, xc, rows, K, K, F16, kBK, kBM, sw128)) return KRSI_ERR_CUDA;
    es = xm;
    if (p.grads && (!make_panel_map(&es, s.e, rows, p.panels, F16, 32, 1) ||
                    !make_panel_map(&ek, s.e, rows, p.panels, F16, kBM, 1) ||
                    !make_panel_map(&em, s.e, rows, p.panels, F16, kBK, 2) ||
                    !make_map(&xs, s.xs, rows, K, K, F16, 64, kBK, sw128)))
      return KRSI_ERR_CUDA;
    LogitsArgs la{};
    la.tgt = s.tgt + r0;
    la.ref = s.l2t + r0;
    la.part = s.part;
    la.rows = (int)rows;
    la.V = V;
    la.n_rt = (int)ceil_div(rows, 256);
    la.n_vt = (int)p.n_vt;
    la.n_kb = (int)ceil_div(K, kBK);
    la.c = c2;
    la.e_scale = 1.f;
    la.store = p.grads && !F16;
    la.limit = kSpinLimit;
    if (running) {
      la.targets = targets;
      la.target_bits = c.target_bits;
      la.ignore = (long long)c.ignore;
      la.l2t_out = s.l2t + r0;
      la.l2t_low_out = s.l2t_low + r0;
      la.ticket = s.ticket;
    }
    const int logit_pairs = (int)std::min<int64_t>(pairs, (int64_t)la.n_rt * la.n_vt);
    if (!known) {
      KRSI_CUDA_TRY(launch_pairs(running ? ce_logits_kernel<F16, true> : ce_logits_kernel<F16, false>,
                                 kLogitsThreads, logit_pairs, stream, xm, wk, es, la));
      JoinArgs ja{};
      ja.total = joined ? c.total : nullptr;
      ja.weight = c.row_weight;
      ja.ticket = s.ticket;
      ja.mean = c.mean;
      ja.part = s.part;
      ja.n_part = 2 * (int)p.n_vt;
      ja.tgt = s.tgt + r0;
      ja.targets = running ? targets : nullptr;
      ja.target_bits = c.target_bits;
      ja.V = V;
      ja.ignore = (long long)c.ignore;
      ja.l2t = s.l2t + r0;
      ja.l2t_low = s.l2t_low + r0;
      ja.loss = c.loss + r0;
      ja.stats = stats ? stats + r0 : nullptr;
      ja.rows = (int)rows;
      ja.K = K;
      ja.all_second = F16;
      ja.e_scale = e_scale;
      ja.z = c.z;
      if (p.grads && !rows_after_join) {
        ja.coef = s.coef + r0;
        ja.factor = s.factor + r0;
        ja.ref = s.ref + r0;
        ja.marked = s.marked + r0 / 256;
        ja.xs = s.xs;
        ja.x = xc;
      }
      KRSI_CUDA_TRY(launch_pdl(ce_join_kernel<DT>, dim3((unsigned)ceil_div(rows, 8)), dim3(256), 0, stream, ja));
      if (!p.grads) continue;
    }
    if (known || rows_after_join) {
      if (tops) KRSI_CUDA_TRY(find_top(r0, rows));
      RowsArgs ra{};
      ra.targets = targets;
      ra.stats = stats + r0;
      ra.up = up;
      ra.row0 = r0;
      ra.tgt = s.tgt + r0;
      ra.coef = s.coef + r0;
      ra.factor = s.factor + r0;
      ra.ref = s.ref + r0;
      ra.x = xc;
      ra.xs = s.xs;
      ra.rows = (int)rows;
      ra.V = V;
      ra.K = K;
      ra.ignore = (long long)c.ignore;
      ra.e_scale = e_scale;
      ra.z = c.z;
      KRSI_CUDA_TRY(launch_pdl(wide ? ce_rows_kernel<DT, long long> : ce_rows_kernel<DT, int>,
                               dim3((unsigned)ceil_div(rows, 8)), dim3(256), 0, stream, ra));
    }

    la.ref = s.ref + r0;
    la.part = nullptr;
    la.marked = F16 || known ? nullptr : s.marked + r0 / 256;
    la.e_scale = e_scale;
    la.store = 1;
    KRSI_CUDA_TRY(launch_pairs(ce_logits_kernel<F16, false>, kLogitsThreads, logit_pairs, stream, xm, wk, es, la));

    GradArgs ga{};
    ga.rows = (int)rows;
    ga.V = V;
    ga.K = K;
    ga.cols = p.cols;
    ga.n_ct = p.n_ct;
    ga.n_rt = la.n_rt;
    ga.splits = (int)p.splits;
    ga.kb_voc = (int)ceil_div(V, kBK);
    ga.kb_share = (int)ceil_div(ga.kb_voc, p.splits);
    ga.n_vt = (int)p.n_vt;
    ga.kb_rows = (int)ceil_div(rows, kBK);
    ga.n_dx = c.dx ? ga.n_rt * ga.n_ct * ga.splits : 0;
    ga.n_dw = c.dw ? ga.n_vt * ga.n_ct : 0;
    const int P = (int)std::min<int64_t>(pairs, (int64_t)ga.n_dx + ga.n_dw);
    // Pairs with one dx item less than the others take dw items for it, as many as fit into its time. In K
    // blocks an item costs its own and, with one accumulator, its epilogue's.
    const int epilogue = p.cols > kBN ? kEpilogueBlocks : 0;
    if (ga.n_dx % P != 0)
      ga.low_first = std::min((ga.kb_share + epilogue) / (ga.kb_rows + epilogue), ga.n_dw / (P - ga.n_dx % P));
    ga.dx_part = ga.splits > 1;
    ga.dx32 = ga.dx_part || !known;
    ga.tgt = s.tgt + r0;
    ga.factor = s.factor + r0;
    ga.coef = s.coef + r0;
    ga.w = w;
    ga.dw32 = !p.direct;
    ga.accumulate = r0 > 0;
    ga.sums = p.direct ? dw32 : nullptr;
    ga.few = few;
    ga.by_entry = p.by_entry;
    ga.start = s.sorted.start;
    ga.order = s.sorted.order;
    ga.up = up;
    ga.alpha = 1.f / e_scale;
    ga.scale = c.scale;
    ga.limit = kSpinLimit;
    void* dxc = c.dx ? static_cast<char*>(c.dx) + (size_t)r0 * K * (known ? 2 : 4) : nullptr;
    CUtensorMap dxm = wm;
    const int64_t part_rows = (int64_t)ga.n_rt * 256;
    if (c.dx && !(ga.dx_part  ? make_map_f32(&dxm, s.dx_part, ga.splits * part_rows, K)
                  : !known ? make_map_f32(&dxm, dxc, rows, K)
                            : make_map(&dxm, dxc, rows, K, K, F16, 16, 32, CU_TENSOR_MAP_SWIZZLE_32B)))
      return KRSI_ERR_CUDA;
    KRSI_CUDA_TRY(launch_pairs(ce_grads_kernel<F16>, kGradsThreads, P, stream, ek, wm, em, xs, dxm, dwm, ga));
    if (ga.dx_part && c.dx)
      KRSI_CUDA_TRY(launch_pdl(ce_dx_join_kernel<DT>,
                               dim3((unsigned)ceil_div(K / 4, 128), (unsigned)ceil_div(rows, kJoinRows)), dim3(128), 0,
                               stream, (const float*)s.dx_part, ga.splits, part_rows * K, ga.tgt, ga.factor, ga.coef, w,
                               dxc, (int)rows, K, c.scale, known ? 0 : 1));
  }
  if (p.grads && c.dw) {   // the targets' part of dw
    if (p.direct) {
      const DwRows<DT> out{dw32, (T*)c.dw, p.K, c.scale, p.by_entry};
      KRSI_CUDA_TRY(few ? (tokens::sum_few<DT, 8, true>(x, s.coef, (const int*)s.tgt, out, false, N, V, -1, K, stream))
                        : (tokens::sum_by_token<DT, 8, true>(x, s.coef, s.sorted, out, false, N, V, K, stream)));
    } else {
      const DwSums out{dw32, p.K};
      KRSI_CUDA_TRY(few ? (tokens::sum_few<DT, 8, true>(x, s.coef, (const int*)s.tgt, out, false, N, V, -1, K, stream))
                        : (tokens::sum_by_token<DT, 8, true>(x, s.coef, s.sorted, out, false, N, V, K, stream)));
      if (known) {
        const int64_t n = p.V * p.K;
        KRSI_CUDA_TRY(launch_pdl(ce_finish_kernel<DT>, dim3((unsigned)std::min<int64_t>(ceil_div(n, 2048), 148 * 64)),
                                 dim3(256), 0, stream, (const float*)dw32, (T*)c.dw, n, c.scale, (const float*)nullptr,
                                 (const float*)nullptr));
      }
    }
  }
  if (c.total && !joined) {
    const bool small = p.N <= kJoinReduceRows;
    KRSI_CUDA_TRY(launch_pdl(small ? ce_reduce_kernel<256> : ce_reduce_kernel<1024>, dim3(1), dim3(small ? 256 : 1024), 0,
                             stream, (const float*)c.loss, (const int*)s.tgt, c.total, c.row_weight, N, c.mean));
  }
  return KRSI_OK;
}

inline int check(int64_t N, int64_t V, int64_t K, int target_bits, int dtype) {
  KRSI_CHECK_ARG(N >= 0 && V > 0 && K > 0);
  KRSI_CHECK_ARG(target_bits == 32 || target_bits == 64);
  if (dtype != KRSI_BF16 && dtype != KRSI_F16) return KRSI_ERR_UNSUPPORTED;
  // TMA row strides and 16-byte packets (K % 8); 32-bit tile and row indices (a chunk has at most 2^22 tiles)
  if (K % 8 != 0 || N > (1 << 30) || V > (1 << 30) || K > (1 << 20)) return KRSI_ERR_UNSUPPORTED;
  return KRSI_OK;
}

inline int run_checked(const Call& c, int64_t N, int64_t V, int64_t K, void* workspace, size_t workspace_bytes,
                       int dtype, cudaStream_t stream) {
  if (!aligned16(c.x) || !aligned16(c.w) || !aligned16(c.dx) || !aligned16(c.dw)) return KRSI_ERR_MISALIGNED;
  const int pairs = device_pairs();
  if (pairs <= 0) return KRSI_ERR_UNSUPPORTED;   // a device partition without clusters of two
  const Plan p = make_plan(N, V, K, c.dx != nullptr, c.dw != nullptr, c.loss == nullptr, pairs);
  const Space s = space_at(workspace, p);
  if (!workspace || workspace_bytes < s.bytes) return KRSI_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) % 256 != 0) return KRSI_ERR_MISALIGNED;
  KRSI_CUDA_TRY(gemm::bind_context());
  return dtype == KRSI_F16 ? run<true>(c, p, s, pairs, stream) : run<false>(c, p, s, pairs, stream);
}

}  // namespace
}  // namespace krsi

using namespace krsi;

extern "C" int krsi_linear_ce_workspace_size(int64_t N, int64_t V, int64_t K, int mode, size_t* bytes) {
  const int kind = mode & 3;
  KRSI_CHECK_ARG(bytes && N >= 0 && V > 0 && K > 0 && mode >= 0 && kind <= 2);
  KRSI_CHECK_ARG(mode == kind || (kind > 0 && (mode == kind + KRSI_CE_NO_DX || mode == kind + KRSI_CE_NO_DW)));
  const int pairs = device_pairs();
  if (pairs <= 0) return KRSI_ERR_UNSUPPORTED;
  *bytes = space_at(nullptr, make_plan(N, V, K, kind > 0 && !(mode & KRSI_CE_NO_DX),
                                          kind > 0 && !(mode & KRSI_CE_NO_DW), kind == 2, pairs)).bytes;
  return KRSI_OK;
}

extern "C" int krsi_linear_ce_fwd(const void* x, const void* w, const void* targets, int target_bits, float* loss,
                                  float* total, float* weight, float* stats, float* dx, float* dw,
                                  void* workspace, size_t workspace_bytes, int64_t N, int64_t V, int64_t K,
                                  float scale, int64_t ignore_index, float z_loss, int mean, int dtype,
                                  cudaStream_t stream) {
  const int rc = check(N, V, K, target_bits, dtype);
  if (rc != KRSI_OK) return rc;
  KRSI_CHECK_ARG((total != nullptr) == (weight != nullptr));
  if (N == 0) {
    if (dw) KRSI_CUDA_TRY(cudaMemsetAsync(dw, 0, (size_t)V * K * 4, stream));
    if (total) KRSI_CUDA_TRY(launch_pdl(ce_reduce_kernel<256>, dim3(1), dim3(256), 0, stream, (const float*)nullptr,
                                        (const int*)nullptr, total, weight, 0, mean));
    return KRSI_OK;
  }
  KRSI_CHECK_ARG(x && w && targets && loss);
  if (reinterpret_cast<uintptr_t>(stats) % 8 != 0) return KRSI_ERR_MISALIGNED;
  const Call c{x, w, targets, target_bits, loss, total, weight, mean, reinterpret_cast<float2*>(stats), nullptr, 0,
               nullptr, dx, dw, scale, z_loss, ignore_index};
  return run_checked(c, N, V, K, workspace, workspace_bytes, dtype, stream);
}

extern "C" int krsi_linear_ce_grad(const void* x, const void* w, const void* targets, int target_bits, const float* g,
                                   int64_t g_stride, const float* weight, const float* stats, void* dx, void* dw,
                                   void* workspace, size_t workspace_bytes, int64_t N, int64_t V, int64_t K,
                                   float scale, int64_t ignore_index, float z_loss, int dtype, cudaStream_t stream) {
  const int rc = check(N, V, K, target_bits, dtype);
  if (rc != KRSI_OK) return rc;
  KRSI_CHECK_ARG((g_stride == 0 || g_stride == 1) && (dx || dw));
  if (N == 0) {
    if (dw) KRSI_CUDA_TRY(cudaMemsetAsync(dw, 0, (size_t)V * K * 2, stream));
    return KRSI_OK;
  }
  KRSI_CHECK_ARG(x && w && targets && g && stats);
  if (reinterpret_cast<uintptr_t>(stats) % 8 != 0) return KRSI_ERR_MISALIGNED;
  const Call c{x, w, targets, target_bits, nullptr, nullptr, nullptr, 0,
               const_cast<float2*>(reinterpret_cast<const float2*>(stats)), g, g_stride, weight, dx, dw, scale, z_loss,
               ignore_index};
  return run_checked(c, N, V, K, workspace, workspace_bytes, dtype, stream);
}

extern "C" int krsi_linear_ce_finish(const float* grad, const float* g, const float* weight, void* out, int64_t n,
                                     float scale, int dtype, cudaStream_t stream) {
  KRSI_CHECK_ARG(n >= 0);
  if (dtype != KRSI_BF16 && dtype != KRSI_F16) return KRSI_ERR_UNSUPPORTED;
  if (n % 8 != 0) return KRSI_ERR_UNSUPPORTED;
  if (n == 0) return KRSI_OK;
  KRSI_CHECK_ARG(grad && out);
  if (!aligned16(grad) || !aligned16(out)) return KRSI_ERR_MISALIGNED;
  const dim3 grid((unsigned)std::min<int64_t>(ceil_div(n, 2048), 148 * 64));
  if (dtype == KRSI_F16)
    KRSI_CUDA_TRY(launch_pdl(ce_finish_kernel<KRSI_F16>, grid, dim3(256), 0, stream, grad, (__half*)out, n, scale, g,
                             weight));
  else
    KRSI_CUDA_TRY(launch_pdl(ce_finish_kernel<KRSI_BF16>, grid, dim3(256), 0, stream, grad, (__nv_bfloat16*)out, n,
                             scale, g, weight));
  return KRSI_OK;
}
