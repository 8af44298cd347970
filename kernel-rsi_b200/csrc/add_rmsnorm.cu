// add_rmsnorm.cu - the residual's addition and RMSNorm in one pass, its output in the input's type or in 8 bits,
// for B200:
//   z = (x + res) rounded to x's type;   r = 1 / sqrt(mean(z^2) + eps)
//   y = w * (z * r) in fp32, rounded once to x's type (rmsnorm.cu rounds z * r to w's type first), or
//   q = e4m3(t * (448 / max|t|)), scale = max|t| * r / 448, with t = z * w in fp32: y is q * scale.
//   (448 / max is 448 times the rounded reciprocal, as torch divides a number by a tensor.)
// The codes do not depend on r (it cancels), so neither on the order of the sum of squares: the same row gives
// the same bits in any plan.  Without res, z is x and is not written.
// (The backward is in add_rmsnorm_bwd.cu.)
// Layout as in rmsnorm.cu: TPR threads hold a row in registers, thread t the packets at columns (c*TPR + t)*VEC.

#include <cuda_fp8.h>

#include "add_rmsnorm.cuh"

namespace krsi {
namespace {

using namespace norm;

constexpr float kE4m3Max = 448.0f;
// Rows whose largest |t| is below this are scaled as if it were that: 448 / max stays finite.
constexpr float kTinyTop = 7.888609052210118e-31f;   // 2^-100

enum Out : int { kOutRow = 0, kOutQ8 = 1 };   // (8 bits without w: the rows themselves)

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// (sum of a, max of b) over the TPR threads that share a row.
template <int TPR>
__device__ __forceinline__ void row_sum_max(float& a, float& b, float2* red) {
  a = warp_sum(a);
  b = warp_max(b);
  if constexpr (TPR > 32) {
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    if (lane == 0) red[wid] = make_float2(a, b);
    __syncthreads();
    a = 0.f;
    b = 0.f;
#pragma unroll
    for (int i = 0; i < TPR / 32; ++i) {
      const float2 v = red[i];
      a += v.x;
      b = fmaxf(b, v.y);
    }
  }
}

template <int TPR> struct NormCfg {
  static constexpr int kThreads = TPR == 32 ? 64 : TPR;
  static constexpr int kRowsPerBlock = kThreads / TPR;
};

__device__ __forceinline__ uint16_t e4m3x2(float lo, float hi) {
  return (uint16_t)__nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
template <int VEC>
__device__ __forceinline__ void store_q8(uint8_t* p, const float* in) {
  if constexpr (VEC == 1) {
    *p = (uint8_t)__nv_cvt_float_to_fp8(in[0], __NV_SATFINITE, __NV_E4M3);
  } else {
    uint32_t u[VEC / 4];
#pragma unroll
    for (int k = 0; k < VEC / 4; ++k)
      u[k] = (uint32_t)e4m3x2(in[4 * k], in[4 * k + 1]) | ((uint32_t)e4m3x2(in[4 * k + 2], in[4 * k + 3]) << 16);
    if constexpr (VEC == 4) *reinterpret_cast<uint32_t*>(p) = u[0];
    else *reinterpret_cast<uint2*>(p) = make_uint2(u[0], u[1]);
  }
}

struct NormArgs {
  const void* x; const void* res; const void* w; void* z; void* y;
  float* stat;           // kOutRow: rstd; else the scale
  int64_t rows, q_stride;
  int n;
  float eps;
};

template <int XT, bool WF32, int TPR, int VEC, int NCH, int OUT>
__global__ void __launch_bounds__(NormCfg<TPR>::kThreads)
add_rmsnorm_kernel(const NormArgs a) {
  pdl_enter();
  using T = typename Elem<XT>::T;
  using XE = Elem<XT>;
  __shared__ float2 red[32];
  const int t = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * NormCfg<TPR>::kRowsPerBlock + threadIdx.x / TPR;
  const bool live = row < a.rows;   // a block-per-row group is always live
  const int n = a.n;
  const T* xr = static_cast<const T*>(a.x) + row * n;
  const T* rr = static_cast<const T*>(a.res) + row * n;
  const bool add = a.res != nullptr;
  float v[NCH][VEC];
  float ss = 0.f, top = 0.f;
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int col = (c * TPR + t) * VEC;
    if (live && col < n) {
      load_row<XT, VEC>(xr + col, v[c], true);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[c][e] = 0.f;
    }
  }
  if (add) {
    T* zr = static_cast<T*>(a.z) + row * n;
    float b[NCH][VEC];
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int col = (c * TPR + t) * VEC;
      if (live && col < n) load_row<XT, VEC>(rr + col, b[c], true);
    }
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int col = (c * TPR + t) * VEC;
      if (live && col < n) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[c][e] = XE::round(v[c][e] + b[c][e]);
        store_row<XT, VEC>(zr + col, v[c]);
      }
    }
  }
#pragma unroll
  for (int c = 0; c < NCH; ++c)
#pragma unroll
    for (int e = 0; e < VEC; ++e) ss = fmaf(v[c][e], v[c][e], ss);
  if constexpr (OUT == kOutQ8) {   // v becomes t = z * w
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int col = (c * TPR + t) * VEC;
      if (a.w != nullptr && col < n) {
        float wv[VEC];
        load_weight<XT, VEC>(a.w, WF32, col, wv);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[c][e] *= wv[e];
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) top = fmaxf(top, fabsf(v[c][e]));
    }
  }
  row_sum_max<TPR>(ss, top, red);
  if (!live) return;
  if constexpr (OUT == kOutRow) {
    const float r = 1.0f / sqrtf(ss / (float)n + a.eps);
    if (t == 0) a.stat[row] = r;
    T* yr = static_cast<T*>(a.y) + row * n;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int col = (c * TPR + t) * VEC;
      if (col < n) {
        float wv[VEC], o[VEC];
        load_weight<XT, VEC>(a.w, WF32, col, wv);
#pragma unroll
        for (int e = 0; e < VEC; ++e) o[e] = wv[e] * (v[c][e] * r);
        store_row<XT, VEC>(yr + col, o);
      }
    }
  } else {
    top = fmaxf(top, kTinyTop);
    const float inv = __fmul_rn(kE4m3Max, __frcp_rn(top));
    if (t == 0) {
      // fmaxf drops NaN: the sum of squares brings it into the scale (0 * ss is 0 or NaN)
      const float r = 1.0f / sqrtf(ss / (float)n + a.eps);
      a.stat[row] = a.w != nullptr ? top * r / kE4m3Max : isnan(ss) ? ss : top / kE4m3Max;
    }
    uint8_t* qr = static_cast<uint8_t*>(a.y) + row * a.q_stride;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int col = (c * TPR + t) * VEC;
      if (col < n) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[c][e] = __fmul_rn(v[c][e], inv);
        store_q8<VEC>(qr + col, v[c]);
      }
    }
  }
}

// ---------------------------------------------------------------- host-side planning
// (threads a row, packets a thread) for packets of 8, 4 and 1 values: the first that holds the row.  A warp a row up to
// 40 values a thread (16 one by one), then blocks, as small as can be: several small blocks an SM keep more rows in
// flight between their barriers.
#define KRSI_PLANS8(X) \
  X(32, 1) X(32, 2) X(32, 3) X(32, 4) X(32, 5) X(64, 3) X(64, 5) X(128, 3) X(128, 5) X(256, 3) X(256, 5) X(512, 3) \
  X(512, 5) X(1024, 4)
#define KRSI_PLANS4(X) \
  X(32, 1) X(32, 2) X(32, 4) X(32, 6) X(32, 8) X(32, 10) X(64, 6) X(64, 10) X(128, 6) X(128, 10) X(256, 6) X(256, 10) \
  X(512, 6) X(512, 10)
#define KRSI_PLANS1(X) \
  X(32, 2) X(32, 4) X(32, 8) X(32, 12) X(32, 16) X(64, 9) X(64, 12) X(64, 16) X(128, 9) X(128, 12) X(128, 16) \
  X(256, 9) X(256, 12) X(256, 16) X(512, 9) X(512, 12) X(512, 16) X(1024, 9) X(1024, 12) X(1024, 16)

template <int XT, bool WF32, int TPR, int VEC, int NCH, int OUT>
int run(const NormArgs& a, cudaStream_t s) {
  using Cfg = NormCfg<TPR>;
  const int64_t grid = (a.rows + Cfg::kRowsPerBlock - 1) / Cfg::kRowsPerBlock;
  if (grid > 0x7fffffff) return KRSI_ERR_UNSUPPORTED;
  KRSI_CUDA_TRY(launch_pdl(add_rmsnorm_kernel<XT, WF32, TPR, VEC, NCH, OUT>, dim3((unsigned)grid), dim3(Cfg::kThreads), 0, s, a));
  return KRSI_OK;
}

template <int XT, bool WF32, int OUT>
int run_packets(int vec, const NormArgs& a, cudaStream_t s) {
  const int64_t packets = ((int64_t)a.n + vec - 1) / vec;
#define KRSI_RUN8(TPR, NCH) if (packets <= TPR * NCH) return run<XT, WF32, TPR, 8, NCH, OUT>(a, s);
#define KRSI_RUN4(TPR, NCH) if (packets <= TPR * NCH) return run<XT, WF32, TPR, 4, NCH, OUT>(a, s);
#define KRSI_RUN1(TPR, NCH) if (packets <= TPR * NCH) return run<XT, WF32, TPR, 1, NCH, OUT>(a, s);
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

template <int OUT>
int dispatch(int x_dtype, int w_dtype, int vec, const NormArgs& a, cudaStream_t s) {
  const bool f32 = w_dtype == KRSI_F32;
  switch (x_dtype) {
    case KRSI_F32: return run_packets<KRSI_F32, true, OUT>(vec, a, s);
    case KRSI_BF16: return f32 ? run_packets<KRSI_BF16, true, OUT>(vec, a, s) : run_packets<KRSI_BF16, false, OUT>(vec, a, s);
    default: return f32 ? run_packets<KRSI_F16, true, OUT>(vec, a, s) : run_packets<KRSI_F16, false, OUT>(vec, a, s);
  }
}

}  // namespace
}  // namespace krsi

using namespace krsi;

extern "C" int krsi_add_rmsnorm_fwd(const void* x, const void* res, const void* w, void* z, void* y, float* rstd,
                                    int64_t rows, int64_t n, float eps, int x_dtype, int w_dtype,
                                    cudaStream_t stream) {
  KRSI_CHECK_ARG(rows >= 0 && n >= 0 && dtype_ok(x_dtype) && dtype_ok(w_dtype));
  if (rows == 0) return KRSI_OK;
  KRSI_CHECK_ARG(n > 0 && x && w && y && rstd && (!res || z));
  if (n > 0x7fffffff) return KRSI_ERR_UNSUPPORTED;
  if (!types_ok(x_dtype, w_dtype)) return KRSI_ERR_UNSUPPORTED;
  return dispatch<kOutRow>(x_dtype, w_dtype, packet_of(x_dtype, w_dtype, n, w, {x, y, res, res ? z : nullptr}),
                           NormArgs{x, res, w, z, y, rstd, rows, 0, (int)n, eps}, stream);
}

extern "C" int krsi_add_rmsnorm_q8_fwd(const void* x, const void* res, const void* w, void* z, void* q,
                                       int64_t q_stride, float* scale, int64_t rows, int64_t n, float eps, int x_dtype,
                                       int w_dtype, cudaStream_t stream) {
  KRSI_CHECK_ARG(rows >= 0 && n >= 0 && dtype_ok(x_dtype) && dtype_ok(w_dtype));
  if (rows == 0) return KRSI_OK;
  KRSI_CHECK_ARG(n > 0 && x && w && q && scale && (!res || z) && q_stride >= n);
  if (n > 0x7fffffff) return KRSI_ERR_UNSUPPORTED;
  const bool q_ok = aligned16(q) && q_stride % 16 == 0;
  if (!types_ok(x_dtype, w_dtype)) return KRSI_ERR_UNSUPPORTED;
  return dispatch<kOutQ8>(x_dtype, w_dtype, q_ok ? packet_of(x_dtype, w_dtype, n, w, {x, res, res ? z : nullptr}) : 1,
                          NormArgs{x, res, w, z, q, scale, rows, q_stride, (int)n, eps}, stream);
}

extern "C" int krsi_quantise_rows(const void* x, void* q, int64_t q_stride, float* scale, int64_t rows, int64_t n,
                                  int x_dtype, cudaStream_t stream) {
  KRSI_CHECK_ARG(rows >= 0 && n >= 0 && dtype_ok(x_dtype));
  if (rows == 0) return KRSI_OK;
  KRSI_CHECK_ARG(n > 0 && x && q && scale && q_stride >= n);
  if (n > 0x7fffffff) return KRSI_ERR_UNSUPPORTED;
  const bool q_ok = aligned16(q) && q_stride % 16 == 0;
  return dispatch<kOutQ8>(x_dtype, x_dtype, q_ok ? packet_of(x_dtype, x_dtype, n, nullptr, {x}) : 1,
                          NormArgs{x, nullptr, nullptr, nullptr, q, scale, rows, q_stride, (int)n, 0.f}, stream);
}
