// add_rmsnorm_bwd.cu - the backward of the residual norm (add_rmsnorm.cu), for B200.  From z, r and the gradients gy
// of y and gz of z, in fp32 with one rounding at the end:
//   dz = r * (gy * w - n * mean(gy * w * n)) + gz with n = z * r,   dw = sum over the rows of gy * n
// (x and res both have the gradient dz).  In this order nothing leaves fp32's range where dz does not: r^3, which the
// product taken apart has, is subnormal for rows of 5e12 and infinite for those of 1e-13.  dw: each block adds up its rows, a second kernel the blocks, in a fixed
// order.
#include "add_rmsnorm.cuh"
#include "sm100.cuh"

namespace krsi {
namespace {

using namespace norm;

struct BwdArgs {
  const void* gy; const void* gz; const void* z; const void* w; const float* rstd; void* dz;
  float* part;   // [blocks][n]
  int64_t rows;
  int n;
  bool w_f32;
};

// Rows of whole 16-byte packets of 16-bit values, up to 5 packets a lane (1280 values): a warp a row, 12 warps an SM.
// The next row's gy, z and gz are copied to shared memory (cp.async, each lane its own packets) while the current one
// is worked on: 83 KB an SM stay in flight.  The row stays as it is in memory, the column sums in 40 registers, the
// weight in shared memory; the arithmetic is in pairs (f32x2).
constexpr int kStageWarps = 12;
template <int DT>
__device__ __forceinline__ uint64_t widen2(uint32_t u) {
  if constexpr (DT == KRSI_BF16) {
    return sm100::f2_pack(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
    return sm100::f2_pack(f.x, f.y);
  }
}
template <int DT>
__device__ __forceinline__ uint32_t narrow2(uint64_t v) {
  float lo, hi;
  sm100::f2_unpack(v, lo, hi);
  return DT == KRSI_BF16 ? sm100::pack_bf16x2(lo, hi) : sm100::pack_f16x2(lo, hi);
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

template <int XT, int WT, int NCH>
__global__ void __launch_bounds__(kStageWarps * 32, 1)
add_rmsnorm_bwd_staged_kernel(const BwdArgs a) {
  pdl_enter();
  using namespace sm100;
  extern __shared__ __align__(16) uint8_t smem[];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, n = a.n;
  constexpr int kPart = NCH * 512;   // bytes of one operand's row: [NCH][32 lanes][16]
  const int parts = a.gz != nullptr ? 3 : 2;
  uint8_t* stage = smem + warp * 3 * kPart + lane * 16;
  const uint32_t stage_addr = smem_u32(stage);
  const int64_t stride = (int64_t)gridDim.x * kStageWarps;
  int64_t row = (int64_t)blockIdx.x * kStageWarps + warp;
  auto copy = [&](int part, const void* base, int64_t r) {
    const uint16_t* src = static_cast<const uint16_t*>(base) + r * n;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int col = (c * 32 + lane) * 8;
      if (col < n) copy16(stage_addr + part * kPart + c * 512, src + col);
    }
  };
  // the weight's packets: [NCH][32 lanes][16 bytes], twice that in fp32
  constexpr int kWeightPackets = WT == KRSI_F32 ? 2 : 1;
  uint4* weights = reinterpret_cast<uint4*>(smem + kStageWarps * 3 * kPart);
  for (int i = threadIdx.x; i < NCH * 32; i += kStageWarps * 32) {
#pragma unroll
    for (int k = 0; k < kWeightPackets; ++k) {
      uint4 u = make_uint4(0, 0, 0, 0);
      if (i * 8 < n) u = __ldg(reinterpret_cast<const uint4*>(a.w) + i * kWeightPackets + k);
      weights[k * NCH * 32 + i] = u;
    }
  }
  uint64_t acc[NCH][4];
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[c][k] = 0;
    // (the packets past the row are never copied: they hold zeros)
    if ((c * 32 + lane) * 8 >= n)
      for (int part = 0; part < 3; ++part)
        *reinterpret_cast<uint4*>(stage + part * kPart + c * 512) = make_uint4(0, 0, 0, 0);
  }
  __syncthreads();
  auto weight = [&](int c, uint64_t* o) {
    const uint4 u = weights[c * 32 + lane];
    if constexpr (WT == KRSI_F32) {
      const uint4 v = weights[(NCH + c) * 32 + lane];
      o[0] = f2_pack(__uint_as_float(u.x), __uint_as_float(u.y));
      o[1] = f2_pack(__uint_as_float(u.z), __uint_as_float(u.w));
      o[2] = f2_pack(__uint_as_float(v.x), __uint_as_float(v.y));
      o[3] = f2_pack(__uint_as_float(v.z), __uint_as_float(v.w));
    } else {
      o[0] = widen2<WT>(u.x); o[1] = widen2<WT>(u.y); o[2] = widen2<WT>(u.z); o[3] = widen2<WT>(u.w);
    }
  };
  if (row < a.rows) {
    copy(0, a.gy, row);
    copy(1, a.z, row);
    if (parts == 3) copy(2, a.gz, row);
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
  for (; row < a.rows; row += stride) {
    const float r = __ldg(a.rstd + row);
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    uint4 g[NCH], z[NCH];
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      g[c] = *reinterpret_cast<const uint4*>(stage + c * 512);
      z[c] = *reinterpret_cast<const uint4*>(stage + kPart + c * 512);
    }
    const int64_t next = row + stride;
    if (next < a.rows) {   // each lane refills the packets that it has just read itself
      copy(0, a.gy, next);
      copy(1, a.z, next);
    }
    const uint64_t r2 = f2_pack(r, r);
    uint64_t dot2 = 0;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const uint32_t gu[4] = {g[c].x, g[c].y, g[c].z, g[c].w}, zu[4] = {z[c].x, z[c].y, z[c].z, z[c].w};
      uint64_t w[4];
      weight(c, w);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint64_t gk = widen2<XT>(gu[k]), zk = widen2<XT>(zu[k]);
        const uint64_t nk = f2_mul(zk, r2);
        acc[c][k] = f2_fma(gk, nk, acc[c][k]);
        dot2 = f2_fma(f2_mul(gk, w[k]), nk, dot2);
      }
    }
    float lo, hi;
    f2_unpack(dot2, lo, hi);
    const float m = -(warp_sum(lo + hi) / (float)n);
    const uint64_t m2 = f2_pack(m, m);
    uint4* out = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.dz) + row * n);
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const uint32_t gu[4] = {g[c].x, g[c].y, g[c].z, g[c].w}, zu[4] = {z[c].x, z[c].y, z[c].z, z[c].w};
      uint4 add = make_uint4(0, 0, 0, 0);
      if (parts == 3) add = *reinterpret_cast<const uint4*>(stage + 2 * kPart + c * 512);
      const uint32_t au[4] = {add.x, add.y, add.z, add.w};
      uint32_t o[4];
      uint64_t w[4];
      weight(c, w);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint64_t gw = f2_mul(widen2<XT>(gu[k]), w[k]), nk = f2_mul(widen2<XT>(zu[k]), r2);
        o[k] = narrow2<XT>(f2_fma(f2_fma(nk, m2, gw), r2, widen2<XT>(au[k])));
      }
      if ((c * 32 + lane) * 8 < n) out[c * 32 + lane] = make_uint4(o[0], o[1], o[2], o[3]);
    }
    if (parts == 3 && next < a.rows) copy(2, a.gz, next);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // the block's column sums: warp by warp through shared memory, in order
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  float* sums = reinterpret_cast<float*>(smem);   // [warps][NCH * 256]: no more than the stages take
  static_assert(NCH * 256 * 4 <= 3 * kPart, "the sums fit the stages");
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    float4* dst = reinterpret_cast<float4*>(sums + warp * (NCH * 256) + (c * 32 + lane) * 8);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float4 v;
      f2_unpack(acc[c][2 * k], v.x, v.y);
      f2_unpack(acc[c][2 * k + 1], v.z, v.w);
      dst[k] = v;
    }
  }
  __syncthreads();
  for (int col = threadIdx.x; col < n; col += kStageWarps * 32) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < kStageWarps; ++i) t += sums[i * (NCH * 256) + col];
    a.part[(int64_t)blockIdx.x * n + col] = t;
  }
}

// Any other row: a block (or for short rows a warp) a row, straight from memory; what hides the latency is that
// several small blocks are on an SM.
template <int XT, int TPR, int VEC, int NCH>
__global__ void __launch_bounds__(TPR)
add_rmsnorm_bwd_kernel(const BwdArgs a) {
  pdl_enter();
  using T = typename Elem<XT>::T;
  __shared__ float red[2][32];
  const int t = threadIdx.x, n = a.n;
  float wv[NCH][VEC], acc[NCH][VEC];
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int col = (c * TPR + t) * VEC;
#pragma unroll
    for (int e = 0; e < VEC; ++e) wv[c][e] = acc[c][e] = 0.f;
    if (col < n) load_weight<XT, VEC>(a.w, a.w_f32, col, wv[c]);
  }
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
    const T* gy = static_cast<const T*>(a.gy) + row * n;
    const T* gz = static_cast<const T*>(a.gz) + row * n;
    const T* z = static_cast<const T*>(a.z) + row * n;
    float g[NCH][VEC], zv[NCH][VEC], add[NCH][VEC];
    const float r = __ldg(a.rstd + row);
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int col = (c * TPR + t) * VEC;
#pragma unroll
      for (int e = 0; e < VEC; ++e) g[c][e] = zv[c][e] = add[c][e] = 0.f;
      if (col < n) {
        load_row<XT, VEC>(gy + col, g[c], true);
        load_row<XT, VEC>(z + col, zv[c], true);
        if (a.gz != nullptr) load_row<XT, VEC>(gz + col, add[c], true);
      }
    }
    float dot = 0.f;
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        zv[c][e] *= r;
        acc[c][e] = fmaf(g[c][e], zv[c][e], acc[c][e]);
        g[c][e] *= wv[c][e];
        dot = fmaf(g[c][e], zv[c][e], dot);
      }
    dot = warp_sum(dot);
    if constexpr (TPR > 32) {   // (two buffers: one barrier a row)
      if (t % 32 == 0) red[turn][t / 32] = dot;
      __syncthreads();
      dot = 0.f;
#pragma unroll
      for (int i = 0; i < TPR / 32; ++i) dot += red[turn][i];
    }
    const float m = -(dot / (float)n);
    T* dz = static_cast<T*>(a.dz) + row * n;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int col = (c * TPR + t) * VEC;
      if (col < n) {
        float o[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) o[e] = fmaf(fmaf(zv[c][e], m, g[c][e]), r, add[c][e]);
        store_row<XT, VEC>(dz + col, o);
      }
    }
  }
  float* part = a.part + (int64_t)blockIdx.x * n;
#pragma unroll
  for (int c = 0; c < NCH; ++c)
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      if ((c * TPR + t) * VEC + e < n) part[(c * TPR + t) * VEC + e] = acc[c][e];
}

// dw: the blocks' sums in a fixed order.  32 columns a block (one a lane), warp i takes the rows i, i + 32, ..., its
// loads 16 at a time (1184 blocks' sums of 1149: 16.5 us with 16 warps and 8 loads, which is three times the round
// trips); then the warps' sums in order.
constexpr int kSumWarps = 32, kSumAhead = 16;
template <int WT>
__global__ void __launch_bounds__(kSumWarps * 32)
add_rmsnorm_dw_kernel(const float* __restrict__ part, void* __restrict__ dw, int blocks, int n) {
  pdl_enter();
  __shared__ float red[kSumWarps][32];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, col = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (col < n) {
    for (int p0 = warp; p0 < blocks; p0 += kSumWarps * kSumAhead) {
      float v[kSumAhead];
#pragma unroll
      for (int k = 0; k < kSumAhead; ++k) {
        const int p = p0 + k * kSumWarps;
        v[k] = p < blocks ? __ldg(part + (int64_t)p * n + col) : 0.f;
      }
#pragma unroll
      for (int k = 0; k < kSumAhead; ++k) s += v[k];
    }
  }
  red[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && col < n) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < kSumWarps; ++i) t += red[i][lane];
    static_cast<typename Elem<WT>::T*>(dw)[col] = Elem<WT>::store(t);
  }
}

// ---------------------------------------------------------------- host side
constexpr int kMaxBlocks = 1184;   // eight an SM: a fixed cap, so that the sums' order does not depend on the GPU
constexpr int kStagedBlocks = 148;

// (threads a row, packets a thread) for packets of 8, 4 and 1 values: the first that holds the row.  Five values are
// held for each of the row's, so 16 a thread at most but in the widest rows.
#define KRSI_PLANS8(X) \
  X(128, 2) X(256, 2) X(512, 2) X(1024, 2) X(1024, 4)
#define KRSI_PLANS4(X) \
  X(32, 1) X(32, 2) X(32, 4) X(64, 3) X(64, 4) X(128, 3) X(128, 4) X(256, 3) X(256, 4) X(512, 3) X(512, 4) X(1024, 3) \
  X(1024, 4)
#define KRSI_PLANS1(X) \
  X(32, 2) X(32, 4) X(32, 8) X(32, 12) X(64, 9) X(64, 12) X(128, 9) X(128, 12) X(256, 9) X(256, 12) X(512, 9) X(512, 12) \
  X(1024, 9) X(1024, 16)

template <int XT, int TPR, int VEC, int NCH>
int run(const BwdArgs& a, int64_t blocks, cudaStream_t s) {
  KRSI_CUDA_TRY(launch_pdl(add_rmsnorm_bwd_kernel<XT, TPR, VEC, NCH>, dim3((unsigned)blocks), dim3(TPR), 0, s, a));
  return KRSI_OK;
}
template <int XT, int WT, int NCH>
int run_staged(const BwdArgs& a, int64_t blocks, cudaStream_t s) {
  constexpr int smem = kStageWarps * 3 * NCH * 512 + (WT == KRSI_F32 ? 2 : 1) * NCH * 512;   // stages, weight
  KRSI_CUDA_TRY((allow_smem<add_rmsnorm_bwd_staged_kernel<XT, WT, NCH>>(smem)));
  KRSI_CUDA_TRY(launch_pdl(add_rmsnorm_bwd_staged_kernel<XT, WT, NCH>, dim3((unsigned)blocks), dim3(kStageWarps * 32),
                           smem, s, a));
  return KRSI_OK;
}
template <int XT, int WT>
int run_staged(int chunks, const BwdArgs& a, int64_t blocks, cudaStream_t s) {
  switch (chunks) {
    case 1: return run_staged<XT, WT, 1>(a, blocks, s);
    case 2: return run_staged<XT, WT, 2>(a, blocks, s);
    case 3: return run_staged<XT, WT, 3>(a, blocks, s);
    case 4: return run_staged<XT, WT, 4>(a, blocks, s);
    default: return run_staged<XT, WT, 5>(a, blocks, s);
  }
}
template <int XT>
int run_packets(int vec, const BwdArgs& a, int64_t* blocks, cudaStream_t s) {
  const int64_t packets = ((int64_t)a.n + vec - 1) / vec;
  if constexpr (XT != KRSI_F32) {
    if (vec == 8 && packets <= 32 * 5) {
      const int64_t need = (a.rows + kStageWarps - 1) / kStageWarps;
      *blocks = need < kStagedBlocks ? need : kStagedBlocks;
      const int chunks = (int)((packets + 31) / 32);
      return a.w_f32 ? run_staged<XT, KRSI_F32>(chunks, a, *blocks, s) : run_staged<XT, XT>(chunks, a, *blocks, s);
    }
  }
  *blocks = a.rows < kMaxBlocks ? a.rows : kMaxBlocks;
#define KRSI_RUN8(TPR, NCH) if (packets <= TPR * NCH) return run<XT, TPR, 8, NCH>(a, *blocks, s);
#define KRSI_RUN4(TPR, NCH) if (packets <= TPR * NCH) return run<XT, TPR, 4, NCH>(a, *blocks, s);
#define KRSI_RUN1(TPR, NCH) if (packets <= TPR * NCH) return run<XT, TPR, 1, NCH>(a, *blocks, s);
  if (vec == 8) {
    if constexpr (XT != KRSI_F32) { KRSI_PLANS8(KRSI_RUN8) }
  } else if (a.n > 16384) {
    return KRSI_ERR_UNSUPPORTED;
  } else if (vec == 4) {
    KRSI_PLANS4(KRSI_RUN4)
  } else {
    KRSI_PLANS1(KRSI_RUN1)
  }
#undef KRSI_RUN8
#undef KRSI_RUN4
#undef KRSI_RUN1
  return KRSI_ERR_UNSUPPORTED;
}

}  // namespace
}  // namespace krsi

using namespace krsi;

extern "C" int krsi_add_rmsnorm_bwd_workspace_size(int64_t rows, int64_t n, size_t* bytes) {
  KRSI_CHECK_ARG(rows >= 0 && n >= 0 && bytes);
  if (n > 0x7fffffff) return KRSI_ERR_UNSUPPORTED;
  *bytes = (size_t)(rows < kMaxBlocks ? rows : kMaxBlocks) * (size_t)n * sizeof(float);
  return KRSI_OK;
}

extern "C" int krsi_add_rmsnorm_bwd(const void* gy, const void* gz, const void* z, const void* w, const float* rstd,
                                    void* dz, void* dw, void* workspace, size_t workspace_bytes, int64_t rows,
                                    int64_t n, int x_dtype, int w_dtype, cudaStream_t stream) {
  KRSI_CHECK_ARG(rows >= 0 && n >= 0 && dtype_ok(x_dtype) && dtype_ok(w_dtype));
  if (n == 0) return KRSI_OK;
  KRSI_CHECK_ARG(w && dw);
  if (n > 0x7fffffff) return KRSI_ERR_UNSUPPORTED;
  if (rows == 0) {   // no rows: dw is zero
    KRSI_CUDA_TRY(cudaMemsetAsync(dw, 0, (size_t)n * (w_dtype == KRSI_F32 ? 4 : 2), stream));
    return KRSI_OK;
  }
  KRSI_CHECK_ARG(gy && z && rstd && dz);
  if (!types_ok(x_dtype, w_dtype)) return KRSI_ERR_UNSUPPORTED;
  size_t need = 0;
  krsi_add_rmsnorm_bwd_workspace_size(rows, n, &need);
  if (!workspace || workspace_bytes < need) return KRSI_ERR_WORKSPACE;
  const BwdArgs a{gy, gz, z, w, rstd, dz, static_cast<float*>(workspace), rows, (int)n, w_dtype == KRSI_F32};
  const int vec = packet_of(x_dtype, w_dtype, n, w, {gy, gz, z, dz});
  int64_t blocks = 0;
  const int rc = x_dtype == KRSI_F32    ? run_packets<KRSI_F32>(vec, a, &blocks, stream)
                 : x_dtype == KRSI_BF16 ? run_packets<KRSI_BF16>(vec, a, &blocks, stream)
                                        : run_packets<KRSI_F16>(vec, a, &blocks, stream);
  if (rc != KRSI_OK) return rc;
  const dim3 grid((unsigned)((n + 31) / 32)), block(kSumWarps * 32);
  const float* part = a.part;
  if (w_dtype == KRSI_F32)
    KRSI_CUDA_TRY(launch_pdl(add_rmsnorm_dw_kernel<KRSI_F32>, grid, block, 0, stream, part, dw, (int)blocks, (int)n));
  else if (w_dtype == KRSI_BF16)
    KRSI_CUDA_TRY(launch_pdl(add_rmsnorm_dw_kernel<KRSI_BF16>, grid, block, 0, stream, part, dw, (int)blocks, (int)n));
  else
    KRSI_CUDA_TRY(launch_pdl(add_rmsnorm_dw_kernel<KRSI_F16>, grid, block, 0, stream, part, dw, (int)blocks, (int)n));
  return KRSI_OK;
}
