// add_rmsnorm.cu - the residual's addition and RMSNorm in one pass, its output in the input's type or in 8 bits,
// for B200:
//   z = (x + res) rounded to x's type;   r = 1 / sqrt(mean(z^2) + eps)
//   y = w * (z * r).to(w.dtype), stored in x's type (rmsnorm.cu's rounding points), or
//   q = e4m3(t * (448 / max|t|)), scale = max|t| * r / 448, with t = z * w in fp32: y is q * scale.
//   (448 / max is 448 times the rounded reciprocal, as torch divides a number by a tensor.)
// The codes do not depend on r (it cancels), so neither on the order of the sum of squares: the same row gives
// the same bits in any plan.  Without res, z is x and is not written.
// The backward is rmsnorm.cu's with the gradient of z added (krsi_rmsnorm_bwd_add).
// Layout as in rmsnorm.cu: TPR threads hold a row in registers, thread t the packets at columns (c*TPR + t)*VEC.

#include <cuda_fp8.h>

#include "common.cuh"

namespace krsi {
namespace {

constexpr float kE4m3Max = 448.0f;
// Rows whose largest |t| is below this are scaled as if it were that: 448 / max stays finite.
constexpr float kTinyTop = 7.888609052210118e-31f;   // 2^-100

enum Out : int { kOutRow = 0, kOutQ8 = 1, kOutQuantise = 2 };

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

template <int DT, int VEC>
__device__ __forceinline__ void load_row(const typename Elem<DT>::T* p, float* out, bool stream) {
  using E = Elem<DT>;
  if constexpr (VEC == 1) {
    out[0] = E::load(*p);
  } else {
    constexpr int PK = Vec16<typename E::T>::N;
#pragma unroll
    for (int e = 0; e < VEC; e += PK) {
      const auto v = stream ? ldg16_stream(p + e) : ldg16(p + e);
#pragma unroll
      for (int k = 0; k < PK; ++k) out[e + k] = E::load(v.v[k]);
    }
  }
}
template <int DT, int VEC>
__device__ __forceinline__ void store_row(typename Elem<DT>::T* p, const float* in) {
  using E = Elem<DT>;
  if constexpr (VEC == 1) {
    *p = E::store(in[0]);
  } else {
    Vec16<typename E::T> o;
#pragma unroll
    for (int k = 0; k < VEC; ++k) o.v[k] = E::store(in[k]);
    stg16(p, o);
  }
}
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

template <int XT, int WT, int TPR, int VEC, int NCH, int OUT>
__global__ void __launch_bounds__(NormCfg<TPR>::kThreads)
add_rmsnorm_kernel(const NormArgs a) {
  pdl_enter();
  using T = typename Elem<XT>::T;
  using XE = Elem<XT>;
  using WE = Elem<WT>;
  __shared__ float2 red[32];
  const int t = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * NormCfg<TPR>::kRowsPerBlock + threadIdx.x / TPR;
  const bool live = row < a.rows;   // a block-per-row group is always live
  const int n = a.n;
  const T* xr = static_cast<const T*>(a.x) + row * n;
  const T* rr = static_cast<const T*>(a.res) + row * n;
  const auto* w = static_cast<const typename WE::T*>(a.w);
  const bool add = OUT != kOutQuantise && a.res != nullptr;
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
  if constexpr (OUT != kOutRow) {   // v becomes t = z * w
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int col = (c * TPR + t) * VEC;
      if constexpr (OUT == kOutQ8) {
        if (col < n) {
          float wv[VEC];
          load_row<WT, VEC>(w + col, wv, false);
#pragma unroll
          for (int e = 0; e < VEC; ++e) v[c][e] *= wv[e];
        }
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
        load_row<WT, VEC>(w + col, wv, false);
#pragma unroll
        for (int e = 0; e < VEC; ++e) o[e] = WE::round(wv[e] * WE::round(v[c][e] * r));
        store_row<XT, VEC>(yr + col, o);
      }
    }
  } else {
    top = fmaxf(top, kTinyTop);
    const float inv = __fmul_rn(kE4m3Max, __frcp_rn(top));
    if (t == 0) {
      // fmaxf drops NaN: the sum of squares brings it into the scale (0 * ss is 0 or NaN)
      const float r = OUT == kOutQ8 ? 1.0f / sqrtf(ss / (float)n + a.eps) : 1.0f;
      a.stat[row] = OUT == kOutQ8 ? top * r / kE4m3Max : isnan(ss) ? ss : top / kE4m3Max;
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
struct NormPlan { int tpr, vec, nch; };

constexpr int kWarpChunks[] = {1, 2, 3, 4, 5, 6, 8};
constexpr int kBlock128Chunks[] = {3, 4, 6, 8};
constexpr int kBlock512Chunks[] = {4, 8};

bool plan(int64_t n, int vec, NormPlan* p) {
  p->vec = vec;
  const int64_t packets = (n + vec - 1) / vec;
  for (int c : kWarpChunks)
    if (packets <= 32 * c) { p->tpr = 32; p->nch = c; return true; }
  for (int c : kBlock128Chunks)
    if (packets <= 128 * c) { p->tpr = 128; p->nch = c; return true; }
  for (int c : kBlock512Chunks)
    if (packets <= 512 * c) { p->tpr = 512; p->nch = c; return true; }
  if (vec == 1 && packets <= 1024 * 16) { p->tpr = 1024; p->nch = 16; return true; }
  return false;
}

template <int XT, int WT, int TPR, int VEC, int NCH, int OUT>
int run(const NormArgs& a, cudaStream_t s) {
  using Cfg = NormCfg<TPR>;
  const int64_t grid = (a.rows + Cfg::kRowsPerBlock - 1) / Cfg::kRowsPerBlock;
  if (grid > 0x7fffffff) return KRSI_ERR_UNSUPPORTED;
  KRSI_CUDA_TRY(launch_pdl(add_rmsnorm_kernel<XT, WT, TPR, VEC, NCH, OUT>, dim3((unsigned)grid), dim3(Cfg::kThreads),
                           0, s, a));
  return KRSI_OK;
}

template <int XT, int WT, int VEC, int OUT>
int run_plan(const NormPlan& p, const NormArgs& a, cudaStream_t s) {
#define KRSI_RUN(TPR, NCH) if (p.tpr == TPR && p.nch == NCH) return run<XT, WT, TPR, VEC, NCH, OUT>(a, s)
  KRSI_RUN(32, 1); KRSI_RUN(32, 2); KRSI_RUN(32, 3); KRSI_RUN(32, 4); KRSI_RUN(32, 5); KRSI_RUN(32, 6);
  KRSI_RUN(32, 8); KRSI_RUN(128, 3); KRSI_RUN(128, 4); KRSI_RUN(128, 6); KRSI_RUN(128, 8); KRSI_RUN(512, 4);
  KRSI_RUN(512, 8);
  if constexpr (VEC == 1) { KRSI_RUN(1024, 16); }
#undef KRSI_RUN
  return KRSI_ERR_UNSUPPORTED;
}

template <int OUT>
int dispatch(int x_dtype, int w_dtype, const NormPlan& p, const NormArgs& a, cudaStream_t s) {
#define KRSI_DT(XT, WT, VW)            \
  if (x_dtype == XT && w_dtype == WT)  \
    return p.vec == 1 ? run_plan<XT, WT, 1, OUT>(p, a, s) : run_plan<XT, WT, VW, OUT>(p, a, s)
  KRSI_DT(KRSI_F32, KRSI_F32, 4);
  KRSI_DT(KRSI_BF16, KRSI_BF16, 8);
  KRSI_DT(KRSI_F16, KRSI_F16, 8);
  if constexpr (OUT != kOutQuantise) {
    KRSI_DT(KRSI_BF16, KRSI_F32, 8);
    KRSI_DT(KRSI_F16, KRSI_F32, 8);
  }
#undef KRSI_DT
  return KRSI_ERR_UNSUPPORTED;
}

bool dtype_ok(int d) { return d == KRSI_F32 || d == KRSI_BF16 || d == KRSI_F16; }

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
  const int vw = x_dtype == KRSI_F32 ? 4 : 8;
  const bool vec_ok = n % vw == 0 && aligned16(x) && aligned16(y) && aligned16(w) &&
                      (!res || (aligned16(res) && aligned16(z)));
  NormPlan p;
  if (!plan(n, vec_ok ? vw : 1, &p)) return KRSI_ERR_UNSUPPORTED;
  return dispatch<kOutRow>(x_dtype, w_dtype, p, NormArgs{x, res, w, z, y, rstd, rows, 0, (int)n, eps}, stream);
}

extern "C" int krsi_add_rmsnorm_q8_fwd(const void* x, const void* res, const void* w, void* z, void* q,
                                       int64_t q_stride, float* scale, int64_t rows, int64_t n, float eps, int x_dtype,
                                       int w_dtype, cudaStream_t stream) {
  KRSI_CHECK_ARG(rows >= 0 && n >= 0 && dtype_ok(x_dtype) && dtype_ok(w_dtype));
  if (rows == 0) return KRSI_OK;
  KRSI_CHECK_ARG(n > 0 && x && w && q && scale && (!res || z) && q_stride >= n);
  if (n > 0x7fffffff) return KRSI_ERR_UNSUPPORTED;
  const int vw = x_dtype == KRSI_F32 ? 4 : 8;
  const bool vec_ok = n % vw == 0 && aligned16(x) && aligned16(w) && aligned16(q) && q_stride % 16 == 0 &&
                      (!res || (aligned16(res) && aligned16(z)));
  NormPlan p;
  if (!plan(n, vec_ok ? vw : 1, &p)) return KRSI_ERR_UNSUPPORTED;
  return dispatch<kOutQ8>(x_dtype, w_dtype, p, NormArgs{x, res, w, z, q, scale, rows, q_stride, (int)n, eps}, stream);
}

extern "C" int krsi_quantise_rows(const void* x, void* q, int64_t q_stride, float* scale, int64_t rows, int64_t n,
                                  int x_dtype, cudaStream_t stream) {
  KRSI_CHECK_ARG(rows >= 0 && n >= 0 && dtype_ok(x_dtype));
  if (rows == 0) return KRSI_OK;
  KRSI_CHECK_ARG(n > 0 && x && q && scale && q_stride >= n);
  if (n > 0x7fffffff) return KRSI_ERR_UNSUPPORTED;
  const int vw = x_dtype == KRSI_F32 ? 4 : 8;
  const bool vec_ok = n % vw == 0 && aligned16(x) && aligned16(q) && q_stride % 16 == 0;
  NormPlan p;
  if (!plan(n, vec_ok ? vw : 1, &p)) return KRSI_ERR_UNSUPPORTED;
  return dispatch<kOutQuantise>(x_dtype, x_dtype, p,
                                NormArgs{x, nullptr, nullptr, nullptr, q, scale, rows, q_stride, (int)n, 0.f}, stream);
}
