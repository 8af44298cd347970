// linear_q8.cu - the product of rows and a weight in 8 bits, for B200 (sm_100a):
//   out[i, j] = (sum_k q[i, k] * wq[j, k]) * scale[i] * wscale[j]
// q [rows, K] and wq [M, K] in e4m3 (nn.Linear's layout), one fp32 scale for each row of both, out [rows, M] in
// bf16, f16 or fp32.  The products of two e4m3 are exact in fp32; the sums are the tensor cores' fp32, the scales
// are applied to them in fp32 and the result is rounded once.
//
// Structure (as linear_geglu.cu): a persistent grid, 12 warps a CTA: warp 0 the TMA producer (128-byte swizzled
// K-major tiles of 128 values), warp 1 the TMEM owner and issuer of tcgen05.mma kind::f8f6f4 (32 values of K an
// instruction), one lane of each, warps 4-11 the epilogue.  Two accumulators alternate, so a tile's epilogue runs beside
// the next tile's MMAs.
//   up to 128 rows    linear_q8_kernel: one CTA on tiles of 128 rows x 64 columns (the weight's read bounds it:
//                     narrow tiles spread it over the SMs)
//   more              linear_q8_pair_kernel: CTA pairs (cta_group::2) on tiles of 256 rows x up to 256 columns, all
//                     columns of the same rows at the same time, so that out is written in whole rows
//
// What bounds it (32768 x 1152 x 9216 to bf16, 696 GFLOP and 604 MB of output: 332 to 339 us in a long loop, 2.1 PFLOP/s at
// 1.46 GHz under the power cap; 299 in short runs, 2.33, as are all figures from here): the output's way out and the power
// cap.  Without stores the same kernel takes 234 us; writing 604 MB alone takes 156 (3.9 TB/s), and the two do not hide
// each other wholly.  Measured on the way: boxes of 64 bytes a row, one a warp, in place of
// two of 128: 312; ordinary stores of the same boxes: 317; the weight's K blocks kept in shared memory while a pair
// walks down the rows (a third of the L2's reads): 301, and 130 against 116 for 3456 columns, for the shorter ring that
// leaves; pairs walking along the columns of rows of their own: 355.
// Every wait is bounded (watchdog.cuh); a stalled pipeline ends the CTA with an error word.
#include <atomic>

#include "common.cuh"
#include "gemm_common.cuh"
#include "watchdog.cuh"

KRSI_DEFINE_WATCHDOG(q8)

namespace krsi {
namespace {

using namespace sm100;
using gemm::drain_loads;
using gemm::kmajor_sw128;

constexpr int kBM = 128;                    // rows of q per CTA
constexpr int kBK = 128;                    // values of K per stage: one 128-byte swizzle row
constexpr int kThreads = 384;
constexpr int kEpiWarp0 = 4, kEpiWarps = 8;
constexpr uint32_t kATile = kBM * kBK;      // 16 KB

struct Q8Args {
  CUtensorMap omap;   // out, in an epilogue warp's boxes, where its rows start on 16 bytes
  const float* scale;
  const float* wscale;
  void* out;
  int rows, M;
  int bn;             // columns of a tile
  int n_ctiles;       // column tiles
  int n_tiles;        // row tiles x column tiles
  int n_kb;           // K blocks
  int q_rows, stages; // one CTA: rows of q in a stage, stages
  int unit;           // bytes that every row of out starts on: 8, 4 or less (16: TMA stores); of 16-bit types
  bool vec_scale;     // wscale starts on 16 bytes
  uint32_t spin_limit;
};

// The tiles of one CTA or pair: every `stride`th, columns first.
struct Tiles {
  const Q8Args& a;
  const int stride;
  int tile, row = 0, col = 0;
  __device__ __forceinline__ Tiles(const Q8Args& args, int first, int step) : a(args), stride(step), tile(first - step) {}
  __device__ __forceinline__ bool next() {   // to the next tile (at first: to the first one)
    tile += stride;
    if (tile >= a.n_tiles) return false;
    row = tile / a.n_ctiles;
    col = tile % a.n_ctiles;
    return true;
  }
};

// kind::f8f6f4, both operands e4m3 (format 0), K-major, fp32 sums: the bit layout is idesc_f16's.
__host__ __device__ constexpr uint32_t idesc_e4m3(uint32_t M, uint32_t N) { return idesc_f16(M, N, 0, false, false); }

// One lane of a converged warp.  It alone runs the producer's or the issuer's loop: where all 32 lanes waited, voted and
// elected for each instruction a K block took 430 cycles to issue (2048 x 4608 x 1152 to bf16: 16.7 us, 12.7 by one lane).
__device__ __forceinline__ bool elect_one() {
  uint32_t e;
  asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\tselp.u32 %0, 1, 0, e;\n\t}" : "=r"(e));
  return e != 0;
}
// Whether `bar` has reached the phase, without waiting.  With up to 128 rows the issuer asks for the next stage before it
// issues this one's MMAs, which hide the 220 cycles of an answer (16 x 4608 x 1152: 10.9 us became 9.95).  The pair kernel,
// which waits for its operands, does not: 700 x 1152 x 4608 to fp32 took 11.6 us instead of 9.3.
__device__ __forceinline__ uint32_t mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok;
}
template <int CTAS>
__device__ __forceinline__ void mma_q8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                       uint32_t accumulate) {
  if constexpr (CTAS == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Arrive on `bar` (an address in the cluster) when every MMA that this thread issued so far has completed.
__device__ __forceinline__ void mma_commit_pair(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// A box of rows of 16-bit values that start on a U but not on 16 bytes: consecutive lanes on consecutive U.  `at(r, byte)`:
// the box in shared memory; out: its first value, rows M values apart; `cols`, `rows`: what is left of the matrix from
// there.  (17261 x 965 to M bf16, indexed value by value it took 96 to 99 us: 76 for M 3436 by 8 bytes, 80 for 3438 by 4, 87
// for 3439 by 2; 71 for 3440 by TMA.  As LooseRows: 86, 93 and 98, for the shifts by half a word and longer ends.)
template <typename T, typename U, int ROWB, typename At>
__device__ __forceinline__ void store_box(At at, T* out, int M, int cols, int rows, int lane) {
  constexpr int kUnits = ROWB / (int)sizeof(U), kLanes = kUnits < 32 ? kUnits : 32;
  constexpr int kRowsAtOnce = 32 / kLanes, kTurns = 32 / kRowsAtOnce, kPer = sizeof(U) / sizeof(T);
  const int r0 = lane / kLanes;
#pragma unroll
  for (int h = 0; h < kUnits; h += kLanes) {
    const int u = h + lane % kLanes;
    const int left = u * kPer < cols ? rows - r0 : 0;
    U val[kTurns];
#pragma unroll
    for (int k = 0; k < kTurns; ++k) val[k] = *reinterpret_cast<const U*>(at(r0 + k * kRowsAtOnce, u * (int)sizeof(U)));
#pragma unroll
    for (int k = 0; k < kTurns; ++k)
      if (k * kRowsAtOnce < left)
        *reinterpret_cast<U*>(out + (int64_t)(r0 + k * kRowsAtOnce) * M + u * kPer) = val[k];
  }
}

// 32 rows of fp32 that do not start on 16 bytes: each lane writes its own row to shared memory where the values lie in
// the 32-byte sectors of memory, and the row's packets are read and stored whole.  What passes the end of a box comes
// first in the next one; only the packets at both ends of a row leave value by value.  (17261 x 965 to 3439 fp32: 99 us;
// as words of a box, lane by lane, 115; 3440 by TMA: 85.  An even M, whose lanes share banks: 108 either way for 3438.)
template <int ROWB>
struct LooseRows {
  static constexpr int kBox = ROWB / 4;   // values of a row in a box
  // Where row r starts in a box: between two rows is room for what passes the end (which nothing reads there); 8 values
  // more every 8 rows put lanes of different shift or row / 8 on different banks.
  static __device__ __forceinline__ int at(int r) { return 8 + r * (kBox + 8) + (r >> 3) * 8; }

  float* box;
  float* out;            // the first value of the rows
  int M, n, rows, lane;  // values between two rows; of each row; rows that are left
  int own;               // the values of a sector before this lane's row
  float carry[8];        // the last values of the box before

  __device__ __forceinline__ LooseRows(uint8_t* box_, float* out_, int M_, int n_, int rows_, int lane_)
      : box(reinterpret_cast<float*>(box_)), out(out_), M(M_), n(n_), rows(rows_), lane(lane_), own(shift(lane_)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) carry[i] = 0.f;
  }
  __device__ __forceinline__ int shift(int r) const {
    return (int)(((uint32_t)(reinterpret_cast<uintptr_t>(out) / 4) + (uint32_t)r * (uint32_t)M) % 8);
  }
  __device__ __forceinline__ void begin() {
#pragma unroll
    for (int i = 0; i < 8; ++i) box[at(lane) + own + i - 8] = carry[i];
  }
  __device__ __forceinline__ void put(int k, float v) {   // value k of this lane's row in the box
    box[at(lane) + own + k] = v;
    if (k >= kBox - 8) carry[k - (kBox - 8)] = v;
  }
  // PACKETS of each row of box b, and the ends of this lane's row.
  template <int PACKETS>
  __device__ __forceinline__ void leave(int b) {
    constexpr int kRows = 32 / PACKETS, kTurns = 32 / kRows;
    const int e0 = b * kBox + lane % PACKETS * 4;
    __syncwarp();
    float4 val[kTurns];
#pragma unroll
    for (int k = 0; k < kTurns; ++k)
      val[k] = *reinterpret_cast<const float4*>(box + at(k * kRows + lane / PACKETS) + lane % PACKETS * 4);
#pragma unroll
    for (int k = 0; k < kTurns; ++k) {
      const int r = k * kRows + lane / PACKETS, e = e0 - shift(r);   // from the row's first value
      if (r < rows && e >= 0 && e + 4 <= n) *reinterpret_cast<float4*>(out + (int64_t)r * M + e) = val[k];
    }
    if (lane < rows && n > 0) {
      const float* row = box + at(lane);
      float* to = out + (int64_t)lane * M - own;
      const int end = own + n, last = end / 4 * 4;   // (`last`: the packet that the row ends in)
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        if (b == 0 && own + k < end && own + k < (own + 3) / 4 * 4) to[own + k] = row[own + k];
        if (last >= b * kBox && last < b * kBox + PACKETS * 4 && last + k < end && last + k >= own)
          to[last + k] = row[last + k - b * kBox];
      }
    }
    __syncwarp();
  }
  __device__ __forceinline__ void finish(int b) {   // what passed the end of the last box, b - 1
    begin();
    leave<2>(b);
  }
};

// The epilogue of one warp: 32 rows (TMEM lanes) x the first `first` columns of each of the CTA's tiles, or the others,
// ROWB bytes of each row at a time (both parts are whole boxes, one at least).  A lane has a row of the accumulator, and
// writes its packets to one of the warp's two boxes in shared memory (rows of ROWB bytes, swizzled).  VEC, rows of out that
// start on 16 bytes: boxes leave by TMA stores; else by LooseRows (fp32) or store_box.  `row_of(t)`: the first row of a tile
// for this CTA.
template <int DT, bool VEC, int ROWB, typename RowOf, typename Release>
__device__ __forceinline__ bool q8_epilogue(uint8_t* boxes, uint32_t tmem, int acc_cols, int first, int warp, int lane,
                                            Tiles tiles, uint64_t* acc_full, volatile int* abort_flag, const Q8Args& a,
                                            RowOf row_of, Release release) {
  using T = typename Elem<DT>::T;
  constexpr bool kLoose = !VEC && DT == KRSI_F32;
  constexpr int kPer = 16 / (int)sizeof(T);          // values of a packet
  constexpr int kStep = ROWB / (int)sizeof(T);       // columns of a box
  constexpr int kLoad = kStep < 32 ? kStep : 32;     // columns read from TMEM at a time
  const int ew = warp - kEpiWarp0;
  const int quarter = ew % 4, part = ew / 4;  // TMEM lane quarter; which of the tile's columns
  const int base = part * first, cols = part ? a.bn - first : first;
  const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
  uint8_t* box = boxes + ew * 2 * (32 * ROWB);
  // packet p of row r: the 128- or 64-byte swizzle
  auto packet = [&](uint8_t* b, int r, int p) {
    return b + r * ROWB + ((ROWB == 128 ? p ^ (r & 7) : p ^ ((r >> 1) & 3)) << 4);
  };
  int turn = 0;
  bool ok = true;
  for (int i = 0; tiles.next(); ++i) {
    const int acc = i & 1;
    const int row0 = row_of(tiles) + quarter * 32;
    const int c_base = tiles.col * a.bn + base;
    const float s = row0 + lane < a.rows ? __ldg(a.scale + row0 + lane) : 0.f;
    const uint64_t s2 = f2_pack(s, s);
    if (!__all_sync(0xffffffffu, mbar_wait_bounded(&acc_full[acc], (i >> 1) & 1, abort_flag, a.spin_limit))) {
      ok = false;
      break;
    }
    tc_fence_after();
    const uint32_t acc_addr = tmem + lane_addr + acc * acc_cols + base;
    LooseRows<ROWB> loose(box, static_cast<float*>(a.out) + (int64_t)row0 * a.M + c_base, a.M,
                          a.M - c_base < cols ? a.M - c_base : cols, a.rows - row0, lane);   // (kLoose alone)
#pragma unroll 1
    for (int c0 = 0; c0 < cols; c0 += kStep, turn ^= 1) {
      uint8_t* out_box = box + turn * (32 * ROWB);
#pragma unroll
      for (int h = 0; h < kStep; h += kLoad) {
        const int col = c_base + c0 + h;
        uint32_t v[kLoad];
        if constexpr (kLoad == 32) tmem_ld32(acc_addr + c0 + h, v);
        else tmem_ld16(acc_addr + c0 + h, v);
        float ws[kLoad];
        if (a.vec_scale && col + kLoad <= a.M) {
#pragma unroll
          for (int e = 0; e < kLoad; e += 4) {
            const float4 w4 = __ldg(reinterpret_cast<const float4*>(a.wscale + col + e));
            ws[e] = w4.x; ws[e + 1] = w4.y; ws[e + 2] = w4.z; ws[e + 3] = w4.w;
          }
        } else {
#pragma unroll
          for (int e = 0; e < kLoad; ++e) ws[e] = col + e < a.M ? __ldg(a.wscale + col + e) : 0.f;
        }
        tmem_wait_ld();
        if (c0 + h + kLoad >= cols) {              // the accumulator has been read: the MMA may reuse it
          tc_fence_before();
          __syncwarp();
          if (lane == 0) release(acc);
        }
        if (kLoose && h == 0) loose.begin();
        if (VEC && h == 0) {
          if (lane == 0) bulk_wait_read_but_one();   // the box before the last one has been read
          __syncwarp();
        }
#pragma unroll
        for (int p = 0; p < kLoad / kPer; ++p) {
          uint32_t u[4];
#pragma unroll
          for (int k = 0; k < kPer / 2; ++k) {
            const int e = p * kPer + 2 * k;
            float lo, hi;
            f2_unpack(f2_mul(f2_mul(f2_pack(__uint_as_float(v[e]), __uint_as_float(v[e + 1])), s2),
                             f2_pack(ws[e], ws[e + 1])), lo, hi);
            if constexpr (DT == KRSI_F32) {
              u[2 * k] = __float_as_uint(lo);
              u[2 * k + 1] = __float_as_uint(hi);
            } else {
              u[k] = DT == KRSI_F16 ? pack_f16x2(lo, hi) : pack_bf16x2(lo, hi);
            }
          }
          if constexpr (kLoose) {
#pragma unroll
            for (int k = 0; k < 4; ++k) loose.put(h + p * 4 + k, __uint_as_float(u[k]));
          } else {
            *reinterpret_cast<uint4*>(packet(out_box, lane, h / kPer + p)) = make_uint4(u[0], u[1], u[2], u[3]);
          }
        }
      }
      const int col = c_base + c0;
      if constexpr (VEC) {
        fence_async_shared();
        __syncwarp();
        if (lane == 0) {
          if (col < a.M && row0 < a.rows) tma_store_2d(&a.omap, out_box, col, row0);   // (the map clips the box)
          bulk_commit_group();   // of a box that stays too: the wait above counts groups
        }
      } else if constexpr (kLoose) {
        loose.template leave<ROWB / 16>(c0 / kStep);
      } else {
        __syncwarp();
        const int left = a.rows - row0;
        T* out = static_cast<T*>(a.out) + (int64_t)row0 * a.M + col;
        auto at = [&](int r, int byte) { return packet(out_box, r, byte >> 4) + (byte & 15); };
        if (a.unit == 8) store_box<T, uint64_t, ROWB>(at, out, a.M, a.M - col, left, lane);
        else if (a.unit == 4) store_box<T, uint32_t, ROWB>(at, out, a.M, a.M - col, left, lane);
        else store_box<T, uint16_t, ROWB>(at, out, a.M, a.M - col, left, lane);
        __syncwarp();
      }
    }
    if constexpr (kLoose) loose.finish(cols / kStep);
  }
  if (VEC && lane == 0) bulk_wait_all();   // every store has completed before the CTA exits
  return ok;
}

// ---------------------------------------------------------------- up to 128 rows: one CTA, narrow tiles
// The weight comes from memory, so its K blocks in flight are what counts: a stage's tile of q has only as many rows as
// there are, up to eight more (a.q_rows), which leaves room for up to 20 K blocks of the weight's 8 KB instead of 8.  An
// MMA nevertheless reads 128 rows: what follows in shared memory, whatever it is, makes rows of the accumulator that
// nothing reads.  (4 rows of 2792 over 7843: 17.3 us with 8 blocks became 9.8.)  A stage has two K blocks, for half the
// waits and commits: 16 x 4608 x 1152 9.95 us became 9.3.
constexpr int kOneBN = 64;
constexpr int kOneMaxStages = 10;   // of two K blocks
constexpr uint32_t kOneWTile = kOneBN * kBK;                         // 8 KB
constexpr int kOneRowB = 64;                                         // bytes of a row in an output box
constexpr uint32_t kOneRing = 8 * (kATile + kOneWTile);              // 192 KB
constexpr uint32_t kOneBoxOff = kOneRing;
constexpr uint32_t kOneBarOff = kOneBoxOff + kEpiWarps * 2 * 32 * kOneRowB;
constexpr uint32_t kOneMiscOff = kOneBarOff + (2 * kOneMaxStages + 2 + 2 + 1) * 8;
constexpr uint32_t kOneSmem = kOneMiscOff + 16 + 1024;               // + slack for the 1024-byte alignment
constexpr uint32_t kOneTmemCols = 2 * kOneBN;
static_assert(kOneSmem <= 232448, "shared memory budget");

// A ring's position: slot, and the parity of its current use.  (A division of the K block's number by a.stages, in its
// place, took 3 us of 36 K blocks.)
struct Ring {
  int slot = 0;
  uint32_t parity = 0;
  __device__ __forceinline__ void next(int stages) {
    if (++slot == stages) {
      slot = 0;
      parity ^= 1;
    }
  }
};

// Stages for a.q_rows rows.  The tiles of q come first, so an MMA on the last one reads on into the weight's.
inline int one_stages(int q_rows) {
  const int n = (int)(kOneRing / (2 * (q_rows * kBK + kOneWTile)));
  return n < kOneMaxStages ? n : kOneMaxStages;
}

template <int DT, bool VEC>
__global__ void __launch_bounds__(kThreads, 1)
linear_q8_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap wmap,
                 const __grid_constant__ Q8Args a) {
  pdl_enter();   // before any global access and before claiming TMEM
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kOneBarOff);
  uint64_t* empty = full + kOneMaxStages;
  uint64_t* acc_full = empty + kOneMaxStages;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* drain = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + kOneMiscOff);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + kOneMiscOff + 4);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  Tiles tiles(a, blockIdx.x, gridDim.x);
  const uint32_t q_bytes = (uint32_t)a.q_rows * kBK, w_off = 2 * a.stages * q_bytes;

  if (threadIdx.x == 0) {
    for (int s = 0; s < a.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], kEpiWarps);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tensormap(&qmap);
    prefetch_tensormap(&wmap);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, kOneTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  auto wait = [&](uint64_t* bar, uint32_t parity) { return mbar_wait_bounded(bar, parity, abort_flag, a.spin_limit); };

  if (warp == 0 && elect_one()) {
    // ------------------------------------------------------------ TMA producer
    bool ok = true;
    Ring ring;
    int it = 0;
    while (ok && tiles.next()) {
      const int m0 = tiles.row * kBM, n0 = tiles.col * kOneBN;
      for (int kb = 0; kb < a.n_kb; kb += 2, ++it) {
        const int s = ring.slot, blocks = kb + 1 < a.n_kb ? 2 : 1;
        if (it >= a.stages && !wait(&empty[s], ring.parity ^ 1)) {
          ok = false;
          break;
        }
        ring.next(a.stages);
        mbar_arrive_expect_tx(&full[s], blocks * (q_bytes + kOneWTile));
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          if (b >= blocks) break;
          tma_load_2d(smem + w_off + (2 * s + b) * kOneWTile, &wmap, &full[s], (kb + b) * kBK, n0);
          tma_load_2d(smem + (2 * s + b) * q_bytes, &qmap, &full[s], (kb + b) * kBK, m0);
        }
      }
    }
    if (!ok) {   // every load issued has landed before this CTA exits
      watchdog_fire(kWdQ8Load);
      for (int j = it > a.stages ? it - a.stages : 0; j < it; ++j)
        for (uint32_t n = 0; n < a.spin_limit && !mbar_try_wait(&full[j % a.stages], (j / a.stages) & 1); ++n) {
        }
    }
  } else if (warp == 1 && elect_one()) {
    // ------------------------------------------------------------ MMA issuer
    constexpr uint32_t idesc = idesc_e4m3(kBM, kOneBN);
    const uint64_t q0 = kmajor_sw128(smem_u32(smem)), w0 = kmajor_sw128(smem_u32(smem + w_off));
    bool ok = true;
    Ring ring;
    uint32_t ready = 0;
    for (int i = 0; ok && tiles.next(); ++i) {
      const int acc = i & 1;
      if (i >= 2 && !wait(&acc_empty[acc], ((i >> 1) - 1) & 1)) {
        ok = false;
        break;
      }
      tc_fence_after();
      for (int kb = 0; kb < a.n_kb; kb += 2) {
        const int s = ring.slot;
        if (!ready && !wait(&full[s], ring.parity)) {
          ok = false;
          break;
        }
        ring.next(a.stages);
        ready = mbar_test(&full[ring.slot], ring.parity);
        tc_fence_after();
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          if (kb + b >= a.n_kb) break;
          const uint64_t ad = q0 + (uint64_t)(2 * s + b) * (q_bytes >> 4), bd = w0 + (uint64_t)(2 * s + b) * (kOneWTile >> 4);
#pragma unroll
          for (int kk = 0; kk < kBK / 32; ++kk)
            mma_q8<1>(tmem + acc * kOneBN, ad + kk * 2, bd + kk * 2, idesc, (kb + b > 0 || kk > 0) ? 1u : 0u);
        }
        mma_commit(&empty[s]);
      }
      if (!ok) break;
      mma_commit(&acc_full[acc]);
    }
    if (!ok) watchdog_fire(kWdQ8Mma);
    mma_commit(drain);   // every MMA issued above has completed before TMEM is released
    for (uint32_t i = 0; i < a.spin_limit && !mbar_try_wait(drain, 0); ++i) {
    }
  } else if (warp >= kEpiWarp0) {
    // ------------------------------------------------------------ epilogue
    const bool ok = q8_epilogue<DT, VEC, kOneRowB>(
        smem + kOneBoxOff, tmem, kOneBN, kOneBN / 2, warp, lane, tiles, acc_full, abort_flag, a,
        [&](const Tiles& t) { return t.row * kBM; }, [&](int acc) { mbar_arrive(&acc_empty[acc]); });
    if (!ok) watchdog_fire(kWdQ8Epilogue);
  }

  __syncwarp();   // (the lanes that were not elected)
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, kOneTmemCols);
}

// ---------------------------------------------------------------- CTA pairs (cta_group::2)
// Each CTA loads its own 128 rows of q and half of the tile's rows of wq; the even CTA issues M256 K32 MMAs that read
// both CTAs' shared memory and accumulate into both CTAs' TMEM.
constexpr int kPairBN = 256;
constexpr int kPairStages = 5;
constexpr uint32_t kPairStageBytes = 2 * kATile;                     // 32 KB
constexpr int kPairRowB = 128;                                       // bytes of a row in an output box
constexpr uint32_t kPairBoxOff = kPairStages * kPairStageBytes;
constexpr uint32_t kPairBarOff = kPairBoxOff + kEpiWarps * 2 * 32 * kPairRowB;
constexpr uint32_t kPairMiscOff = kPairBarOff + (2 * kPairStages + 2 + 2 + 1) * 8;
constexpr uint32_t kPairSmem = kPairMiscOff + 16 + 1024;
constexpr uint32_t kPairTmemCols = 2 * kPairBN;
static_assert(kPairSmem <= 232448, "shared memory budget");

template <int DT, bool VEC>
__global__ void __launch_bounds__(kThreads, 1)
linear_q8_pair_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap wmap,
                      const __grid_constant__ Q8Args a) {
  pdl_enter();   // before any global access and before claiming TMEM
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kPairBarOff);   // (used in the even CTA)
  uint64_t* empty = full + kPairStages;
  uint64_t* acc_full = empty + kPairStages;
  uint64_t* acc_empty = acc_full + 2;                                 // (used in the even CTA)
  uint64_t* drain = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + kPairMiscOff);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + kPairMiscOff + 4);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t rank = cluster_ctarank();
  const bool even = rank == 0;
  Tiles tiles(a, blockIdx.x / 2, gridDim.x / 2);
  const uint32_t w_bytes = (uint32_t)(a.bn / 2) * kBK;   // one CTA's half of the weight's K block

  if (threadIdx.x == 0) {
    for (int s = 0; s < kPairStages; ++s) {
      mbar_init(&full[s], 1);      // the even CTA's expect_tx arrival + both CTAs' TMA bytes
      mbar_init(&empty[s], 1);     // the even CTA's tcgen05.commit
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 2 * kEpiWarps);   // one arrival per epilogue warp of both CTAs
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tensormap(&qmap);
    prefetch_tensormap(&wmap);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, kPairTmemCols);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync();   // both CTAs' barriers initialised and TMEM allocated before either signals the other
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto wait = [&](uint64_t* bar, uint32_t parity) { return mbar_wait_bounded(bar, parity, abort_flag, a.spin_limit); };

  if (warp == 0 && elect_one()) {
    // ------------------------------------------------------------ TMA producer (both CTAs)
    bool ok = true;
    int it = 0;
    while (ok && tiles.next()) {
      const int m0 = tiles.row * (2 * kBM) + (int)rank * kBM;
      const int n0 = tiles.col * a.bn + (int)rank * (a.bn / 2);
      for (int kb = 0; kb < a.n_kb; ++kb, ++it) {
        const int s = it % kPairStages;
        if (it >= kPairStages && !wait(&empty[s], ((it / kPairStages) - 1) & 1)) {
          ok = false;
          break;
        }
        uint8_t* st = smem + s * kPairStageBytes;
        const uint32_t bar = mapa_shared(&full[s], 0);
        if (even) mbar_arrive_expect_tx(&full[s], 2 * (kATile + w_bytes));
        tma_load_2d_pair(st, &qmap, bar, kb * kBK, m0);
        tma_load_2d_pair(st + kATile, &wmap, bar, kb * kBK, n0);
      }
    }
    if (!ok) {
      watchdog_fire(kWdQ8Load);
      if (even) drain_loads<kPairStages>(full, it, a.spin_limit);   // covers both CTAs' loads of each stage
    }
  } else if (warp == 1 && even && elect_one()) {
    // ------------------------------------------------------------ MMA issuer (even CTA)
    const uint32_t idesc = idesc_e4m3(2 * kBM, (uint32_t)a.bn);
    const uint64_t desc0 = kmajor_sw128(smem_u32(smem));
    bool ok = true;
    int it = 0;
    for (int i = 0; ok && tiles.next(); ++i) {
      const int acc = i & 1;
      if (i >= 2 && !wait(&acc_empty[acc], ((i >> 1) - 1) & 1)) {
        ok = false;
        break;
      }
      tc_fence_after();
      for (int kb = 0; kb < a.n_kb; ++kb, ++it) {
        const int s = it % kPairStages;
        if (!wait(&full[s], (it / kPairStages) & 1)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint64_t ad = desc0 + (uint64_t)s * (kPairStageBytes >> 4), bd = ad + (kATile >> 4);
#pragma unroll
        for (int kk = 0; kk < kBK / 32; ++kk)
          mma_q8<2>(tmem + acc * kPairBN, ad + kk * 2, bd + kk * 2, idesc, (kb > 0 || kk > 0) ? 1u : 0u);
        mma_commit_pair(mapa_shared(&empty[s], 0));   // stage s free in both CTAs
        mma_commit_pair(mapa_shared(&empty[s], 1));
      }
      if (!ok) break;
      mma_commit_pair(mapa_shared(&acc_full[acc], 0));
      mma_commit_pair(mapa_shared(&acc_full[acc], 1));
    }
    if (!ok) watchdog_fire(kWdQ8Mma);
    mma_commit_pair(mapa_shared(drain, 0));
    for (uint32_t i = 0; i < a.spin_limit && !mbar_try_wait(drain, 0); ++i) {
    }
  } else if (warp >= kEpiWarp0) {
    // ------------------------------------------------------------ epilogue (both CTAs, own rows)
    constexpr int kStep = kPairRowB / (int)sizeof(typename Elem<DT>::T);   // columns of a box
    const bool ok = q8_epilogue<DT, VEC, kPairRowB>(
        smem + kPairBoxOff, tmem, kPairBN, (a.bn / kStep + 1) / 2 * kStep, warp, lane, tiles, acc_full, abort_flag, a,
        [&](const Tiles& t) { return t.row * (2 * kBM) + (int)rank * kBM; },
        [&](int acc) {
          if (even) mbar_arrive(&acc_empty[acc]);
          else mbar_arrive_cluster(mapa_shared(&acc_empty[acc], 0));
        });
    if (!ok) watchdog_fire(kWdQ8Epilogue);
  }

  __syncwarp();   // (the lanes that were not elected)
  tc_fence_before();
  cluster_sync();   // the even CTA's MMAs (which read this CTA's shared memory and TMEM) are done
  tc_fence_after();
  if (warp == 1) tmem_dealloc_pair(tmem, kPairTmemCols);
}

// ---------------------------------------------------------------- host side
// 2-D map (cols, rows) of a row-major matrix, `pitch` bytes between rows.
bool map_2d(CUtensorMap* map, CUtensorMapDataType type, const void* base, int64_t rows, int64_t cols, int64_t pitch,
            uint32_t box_cols, uint32_t box_rows, CUtensorMapSwizzle swizzle) {
  attn::EncodeTiledFn enc = attn::encode_fn();
  if (!enc) return false;
  memset(map, 0, sizeof(*map));
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)pitch};
  cuuint32_t box[2] = {box_cols, box_rows};
  cuuint32_t estr[2] = {1, 1};
  return enc(map, type, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

cudaLaunchConfig_t pair_config(cudaLaunchAttribute* attr, int clusters, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * clusters);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kPairSmem;
  cfg.stream = stream;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cfg;
}

// Clusters of two that fit on the device at once (0: none can be launched), per device, queried once.
template <int DT, bool VEC>
int pair_clusters() {
  static std::atomic<int> cached[64];   // clusters + 1 once queried; races only repeat the query
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  int v = cached[dev].load(std::memory_order_relaxed);
  if (v == 0) {
    auto kern = linear_q8_pair_kernel<DT, VEC>;
    int n = 0;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kPairSmem) == cudaSuccess) {
      cudaLaunchAttribute attr[2];
      cudaLaunchConfig_t cfg = pair_config(attr, device_sm_count() / 2, nullptr);
      cfg.numAttrs = 1;
      if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) n = 0;
    }
    cudaGetLastError();   // a refused query leaves no sticky error behind
    v = n + 1;
    cached[dev].store(v, std::memory_order_relaxed);
  }
  return v - 1;
}

bool output_map(Q8Args& a, int dt, int row_bytes) {
  const int es = dt == KRSI_F32 ? 4 : 2;
  const CUtensorMapDataType type = dt == KRSI_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : dt == KRSI_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                     : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return map_2d(&a.omap, type, a.out, a.rows, a.M, (int64_t)a.M * es, row_bytes / es, 32,
                row_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
}

// Columns of a pair's tile: the width that takes least by this count of cycles.  A K block costs its MMAs (2 cycles a
// column) or its operands' way from the L2 (some 48 bytes a cycle), whichever is longer; a tile 400 cycles more, and the
// last one's epilogue (its longer part) is not hidden.  Widths are whole output boxes (`step` columns: 64 of 16 bits, 32 of
// fp32).  (2001 x 1000 x 2743 to fp32: 160 columns 16.1 us, 192 17.6, 256 19.4, all in two rounds of tiles, 128 in three
// 19.1; 700 x 1152 x 4608 to bf16: 192 columns 8.8 us, 256 9.7, 128 11.0.)
int tile_columns(int64_t row_tiles, int64_t M, int n_kb, int pairs, int step) {
  int best = kPairBN;
  int64_t least = INT64_MAX;
  for (int bn = kPairBN; bn >= 2 * step; bn -= step) {
    const int64_t rounds = (row_tiles * ((M + bn - 1) / bn) + pairs - 1) / pairs;
    const int64_t block = 2 * bn > (16384 + 64 * bn) / 48 ? 2 * bn : (16384 + 64 * bn) / 48;
    const int64_t cycles = rounds * (n_kb * block + 400) + 20 * ((bn / step + 1) / 2 * step);
    if (cycles < least) {
      least = cycles;
      best = bn;
    }
  }
  return best;
}

template <int DT, bool VEC>
int launch(const void* q, int64_t q_pitch, const void* wq, int64_t w_pitch, int64_t K, Q8Args a, cudaStream_t stream) {
  const int clusters = a.rows > kBM ? pair_clusters<DT, VEC>() : 0;
  const int64_t bm = clusters > 0 ? 2 * kBM : kBM, rt = ((int64_t)a.rows + bm - 1) / bm;
  a.bn = clusters > 0 ? tile_columns(rt, a.M, a.n_kb, clusters, kPairRowB / (int)sizeof(typename Elem<DT>::T)) : kOneBN;
  const int64_t ct = ((int64_t)a.M + a.bn - 1) / a.bn;
  if (rt * ct > INT32_MAX / 2) return KRSI_ERR_UNSUPPORTED;
  a.n_ctiles = (int)ct;
  a.n_tiles = (int)(rt * ct);
  a.q_rows = a.rows < kBM ? (a.rows + 7) / 8 * 8 : kBM;
  a.stages = one_stages(a.q_rows);
  CUtensorMap qm, wm;
  // (a box of the weight: each CTA's half of a pair's columns, or the one CTA's)
  if (!map_2d(&qm, CU_TENSOR_MAP_DATA_TYPE_UINT8, q, a.rows, K, q_pitch, kBK, a.q_rows, CU_TENSOR_MAP_SWIZZLE_128B) ||
      !map_2d(&wm, CU_TENSOR_MAP_DATA_TYPE_UINT8, wq, a.M, K, w_pitch, kBK, clusters > 0 ? a.bn / 2 : a.bn,
              CU_TENSOR_MAP_SWIZZLE_128B) ||
      (VEC && !output_map(a, DT, clusters > 0 ? kPairRowB : kOneRowB)))
    return KRSI_ERR_CUDA;
  if (clusters > 0) {
    cudaLaunchAttribute attr[2];
    const cudaLaunchConfig_t cfg = pair_config(attr, a.n_tiles < clusters ? a.n_tiles : clusters, stream);
    KRSI_CUDA_TRY(cudaLaunchKernelEx(&cfg, linear_q8_pair_kernel<DT, VEC>, qm, wm, a));
    return KRSI_OK;
  }
  KRSI_CUDA_TRY((allow_smem<linear_q8_kernel<DT, VEC>>((int)kOneSmem)));
  const int sms = device_sm_count();
  KRSI_CUDA_TRY(launch_pdl(linear_q8_kernel<DT, VEC>, dim3(a.n_tiles < sms ? a.n_tiles : sms), dim3(kThreads), kOneSmem,
                           stream, qm, wm, a));
  return KRSI_OK;
}

}  // namespace
}  // namespace krsi

using namespace krsi;

extern "C" int krsi_linear_q8(const void* q, int64_t q_stride, const float* scale, const void* wq, int64_t w_stride,
                              const float* wscale, void* out, int64_t rows, int64_t K, int64_t M, int out_dtype,
                              cudaStream_t stream) {
  KRSI_CHECK_ARG(rows >= 0 && K > 0 && M > 0);
  if (out_dtype != KRSI_F32 && out_dtype != KRSI_BF16 && out_dtype != KRSI_F16) return KRSI_ERR_INVALID_ARGUMENT;
  if (rows == 0) return KRSI_OK;
  KRSI_CHECK_ARG(q && scale && wq && wscale && out && q_stride >= K && w_stride >= K);
  if (!aligned16(q) || !aligned16(wq) || q_stride % 16 != 0 || w_stride % 16 != 0) return KRSI_ERR_MISALIGNED;
  if (rows > INT32_MAX - 2 * kBM || K > INT32_MAX - kBK || M > INT32_MAX - kPairBN) return KRSI_ERR_UNSUPPORTED;
  const int es = out_dtype == KRSI_F32 ? 4 : 2;
  const bool vec = aligned16(out) && M * es % 16 == 0;
  KRSI_CUDA_TRY(gemm::bind_context());
  Q8Args a{};
  a.scale = scale;
  a.wscale = wscale;
  a.out = out;
  a.rows = (int)rows;
  a.M = (int)M;
  a.n_kb = (int)((K + kBK - 1) / kBK);
  for (a.unit = 8; (reinterpret_cast<uintptr_t>(out) | (uintptr_t)(M * es)) & (a.unit - 1); a.unit /= 2) {
  }
  a.vec_scale = aligned16(wscale);
  a.spin_limit = kSpinLimit;
#define KRSI_OUT(DT)                                                            \
  if (out_dtype == DT)                                                          \
    return vec ? launch<DT, true>(q, q_stride, wq, w_stride, K, a, stream) : launch<DT, false>(q, q_stride, wq, w_stride, K, a, stream)
  KRSI_OUT(KRSI_F32);
  KRSI_OUT(KRSI_BF16);
  KRSI_OUT(KRSI_F16);
#undef KRSI_OUT
  return KRSI_ERR_INVALID_ARGUMENT;
}
