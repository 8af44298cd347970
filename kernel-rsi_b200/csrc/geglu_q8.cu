// geglu_q8.cu - GEGLU with an 8-bit checkpoint of its input: the forward writes the output and an
// 8-bit copy of u, the backward reads that copy in place of u.
//   forward:  out = gelu_tanh(a) * b                  a = u[:, :F], b = u[:, F:]
//             (q, e) = the checkpoint: in each group of 32 columns of a half-row, a step 2^(e - 127)
//             and q = round(u / step) in [-127, 127]
//   backward: from a', b' = q * step:  db = g * gelu_tanh(a'),  da = g * b' * gelu_tanh'(a')
//             and, where asked for, out' = gelu_tanh(a') * b' again (the down projection's operand)
// The step is 2^-6 of the power of two below the group's largest magnitude, so that one lands in
// [64, 127]: u / step is exact (a power of two), its rounding is the only error, and it is at most half
// a step (one step where 127.5 and more round down to 127).  A power of two costs up to one bit against
// the exact maximum / 127, and in return the bits do not depend on how the quotient is computed.  A
// group with a value that is not finite keeps the exponent 255 and reads back as NaN.
//
// gelu_tanh(a) = a * s with s = 1 / (1 + exp(-2 z)), z = sqrt(2/pi) (a + 0.044715 a^3), and
// gelu_tanh'(a) = s + a s (1 - s) 2 dz/da.  Everything is fp32 and each output is rounded once.
//
// Bound by memory: 2F values read, F values and 2F bytes written per row forward; F values and 2F bytes
// read, 2F values written backward.  A thread holds 8 columns of both halves; a group is 4 lanes.
#include <algorithm>

#include "common.cuh"

namespace krsi {
namespace {

constexpr int kGroup = 32;        // columns that share a step
constexpr int kCols = 8;          // columns of each half per thread
constexpr int kSlots = kGroup / kCols;
constexpr float kTwoC = 1.5957691216057308f;                       // 2 sqrt(2 / pi)
constexpr float kA = 0.044715f;
constexpr float kLog2e = 1.4426950408889634f;

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};

// s = 1 / (1 + exp(-2 z)); exp overflows to inf for a very negative z, and s is then 0.
__device__ __forceinline__ float gate_sigmoid(float a) {
  const float z2 = kTwoC * (a + kA * a * a * a);
  return rcp_approx(1.0f + ex2_approx(-kLog2e * z2));
}
__device__ __forceinline__ float gate_slope(float a, float s) {
  const float dz2 = kTwoC * (1.0f + 3.0f * kA * a * a);
  return s + a * s * (1.0f - s) * dz2;
}

// Up to kCols columns from p (the columns from `left` on are zero), VEC at a time: VEC divides F, so an
// access is inside the row or outside it.
template <int DT, int VEC>
__device__ __forceinline__ void load_cols(const typename Elem<DT>::T* p, int left, float* v) {
  using P = Pack<typename Elem<DT>::T, VEC>;
#pragma unroll
  for (int k = 0; k < kCols; k += VEC) {
    if (k < left) {
      const P r = *reinterpret_cast<const P*>(p + k);
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[k + e] = Elem<DT>::load(r.v[e]);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[k + e] = 0.f;
    }
  }
}
template <int DT, int VEC>
__device__ __forceinline__ void store_cols(typename Elem<DT>::T* p, int left, const float* v) {
  using P = Pack<typename Elem<DT>::T, VEC>;
#pragma unroll
  for (int k = 0; k < kCols; k += VEC)
    if (k < left) {
      P r;
#pragma unroll
      for (int e = 0; e < VEC; ++e) r.v[e] = Elem<DT>::store(v[k + e]);
      *reinterpret_cast<P*>(p + k) = r;
    }
}

// The group's exponent byte from the magnitudes of its 4 lanes' columns (float bits order as integers;
// NaN above infinity above every finite value).
__device__ __forceinline__ uint32_t group_exponent(const float* v) {
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < kCols; ++k) top = max(top, __float_as_uint(v[k]) & 0x7fffffffu);
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
  return top >= 0x7f800000u ? 255u : max(top >> 23, 7u) - 6u;   // at least 1: a step of 2^-126
}
__device__ __forceinline__ float step_of(uint32_t e) { return __uint_as_float(e == 255u ? 0x7fffffffu : e << 23); }

template <int VEC>
__device__ __forceinline__ void store_q(int8_t* p, int left, const float* v, uint32_t e) {
  const float inv = __uint_as_float((254u - min(e, 253u)) << 23);   // 1 / step
  using P = Pack<int8_t, VEC>;
#pragma unroll
  for (int k = 0; k < kCols; k += VEC)
    if (k < left) {
      P r;
#pragma unroll
      for (int i = 0; i < VEC; ++i) r.v[i] = (int8_t)max(-127, min(127, __float2int_rn(v[k + i] * inv)));
      *reinterpret_cast<P*>(p + k) = r;
    }
}
template <int VEC>
__device__ __forceinline__ void load_q(const int8_t* p, int left, uint32_t e, float* v) {
  const float step = step_of(e);
  using P = Pack<int8_t, VEC>;
#pragma unroll
  for (int k = 0; k < kCols; k += VEC) {
    if (k < left) {
      const P r = *reinterpret_cast<const P*>(p + k);
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[k + i] = (float)r.v[i] * step;
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[k + i] = 0.f;
    }
  }
}

template <int DT, int VEC>
__global__ void __launch_bounds__(256)
geglu_q8_fwd_kernel(const typename Elem<DT>::T* __restrict__ u, typename Elem<DT>::T* __restrict__ out,
                    int8_t* __restrict__ q, uint8_t* __restrict__ ex, int64_t items, int F, uint32_t slots) {
  pdl_enter();
  const int64_t stride = (int64_t)gridDim.x * blockDim.x;
  const int64_t base = (int64_t)blockIdx.x * blockDim.x;
  for (int64_t b0 = base; b0 < items; b0 += stride) {   // uniform per block: every lane meets the shuffles
    const int64_t i = b0 + threadIdx.x;
    const bool live = i < items;
    const int64_t row = live ? i / slots : 0;
    const int slot = live ? (int)(i - row * slots) : 0, c = slot * kCols;
    const int left = live ? F - c : 0;
    const int64_t at = row * 2 * F + c;
    float a[kCols], b[kCols], o[kCols];
    load_cols<DT, VEC>(u + at, left, a);
    load_cols<DT, VEC>(u + at + F, left, b);
    const uint32_t ea = group_exponent(a), eb = group_exponent(b);
#pragma unroll
    for (int k = 0; k < kCols; ++k) o[k] = a[k] * gate_sigmoid(a[k]) * b[k];
    store_cols<DT, VEC>(out + row * F + c, left, o);
    if (q == nullptr) continue;
    store_q<VEC>(q + at, left, a, ea);
    store_q<VEC>(q + at + F, left, b, eb);
    if (live && slot % kSlots == 0) {
      uint8_t* er = ex + (row * slots + slot) / kSlots * 2;   // [row][group][gate, value]
      er[0] = (uint8_t)ea;
      er[1] = (uint8_t)eb;
    }
  }
}

template <int DT, int VEC, bool OUT>
__global__ void __launch_bounds__(256)
geglu_q8_bwd_kernel(const typename Elem<DT>::T* __restrict__ g, const int8_t* __restrict__ q,
                    const uint8_t* __restrict__ ex, typename Elem<DT>::T* __restrict__ du,
                    typename Elem<DT>::T* __restrict__ out, int64_t items, int F, uint32_t slots) {
  pdl_enter();
  const int64_t stride = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < items; i += stride) {
    const int64_t row = i / slots;
    const int slot = (int)(i - row * slots), c = slot * kCols, left = F - c;
    const int64_t at = row * 2 * F + c;
    const uint8_t* er = ex + (row * slots + slot) / kSlots * 2;
    float a[kCols], b[kCols], gv[kCols], o[kCols];
    load_q<VEC>(q + at, left, er[0], a);
    load_q<VEC>(q + at + F, left, er[1], b);
    load_cols<DT, VEC>(g + row * F + c, left, gv);
#pragma unroll
    for (int k = 0; k < kCols; ++k) {
      const float s = gate_sigmoid(a[k]), gel = a[k] * s;
      const float slope = gate_slope(a[k], s);
      if (OUT) o[k] = gel * b[k];
      a[k] = gv[k] * b[k] * slope;
      b[k] = gv[k] * gel;
    }
    store_cols<DT, VEC>(du + at, left, a);
    store_cols<DT, VEC>(du + at + F, left, b);
    if (OUT) store_cols<DT, VEC>(out + row * F + c, left, o);
  }
}

inline uint32_t slots_of(int64_t F) { return (uint32_t)((F + kGroup - 1) / kGroup * kSlots); }

inline dim3 grid_of(int64_t items) { return dim3((unsigned)std::min<int64_t>((items + 255) / 256, 1 << 22)); }

template <int DT, int VEC>
int fwd(const void* u, void* out, void* q, void* ex, int64_t rows, int64_t F, cudaStream_t stream) {
  using T = typename Elem<DT>::T;
  const int64_t items = rows * slots_of(F);
  KRSI_CUDA_TRY(launch_pdl(geglu_q8_fwd_kernel<DT, VEC>, grid_of(items), dim3(256), 0, stream, (const T*)u, (T*)out,
                           (int8_t*)q, (uint8_t*)ex, items, (int)F, slots_of(F)));
  return KRSI_OK;
}
template <int DT, int VEC>
int bwd(const void* g, const void* q, const void* ex, void* du, void* out, int64_t rows, int64_t F,
        cudaStream_t stream) {
  using T = typename Elem<DT>::T;
  const int64_t items = rows * slots_of(F);
  auto kern = out ? geglu_q8_bwd_kernel<DT, VEC, true> : geglu_q8_bwd_kernel<DT, VEC, false>;
  KRSI_CUDA_TRY(launch_pdl(kern, grid_of(items), dim3(256), 0, stream, (const T*)g, (const int8_t*)q,
                           (const uint8_t*)ex, (T*)du, (T*)out, items, (int)F, slots_of(F)));
  return KRSI_OK;
}

// Columns per access: the widest that divides F and suits the buffers (16-bit and fp32 buffers aligned
// to the access, q to as many bytes).
inline int access_cols(int64_t F, int es, uintptr_t wide, uintptr_t bytes) {
  int vec = 16 / es;
  while (vec > 1 && (F % vec != 0 || wide % (vec * es) != 0 || bytes % vec != 0)) vec /= 2;
  return vec;
}

#define KRSI_Q8_VEC(FN, DT, vec, ...)                                                     \
  switch (vec) {                                                                          \
    case 8: if constexpr (DT != KRSI_F32) return FN<DT, 8>(__VA_ARGS__); [[fallthrough]]; \
    case 4: return FN<DT, 4>(__VA_ARGS__);                                                \
    case 2: return FN<DT, 2>(__VA_ARGS__);                                                \
    default: return FN<DT, 1>(__VA_ARGS__);                                               \
  }
#define KRSI_Q8_DISPATCH(FN, vec, ...)                      \
  switch (dtype) {                                          \
    case KRSI_F32: KRSI_Q8_VEC(FN, KRSI_F32, vec, __VA_ARGS__)   \
    case KRSI_BF16: KRSI_Q8_VEC(FN, KRSI_BF16, vec, __VA_ARGS__) \
    default: KRSI_Q8_VEC(FN, KRSI_F16, vec, __VA_ARGS__)         \
  }

inline uintptr_t bits_of(const void* p) { return reinterpret_cast<uintptr_t>(p); }

inline int check(int64_t rows, int64_t F, int dtype) {
  KRSI_CHECK_ARG(rows >= 0 && F >= 0);
  KRSI_CHECK_ARG(dtype == KRSI_F32 || dtype == KRSI_BF16 || dtype == KRSI_F16);
  if (F > (1 << 30)) return KRSI_ERR_UNSUPPORTED;
  return KRSI_OK;
}

}  // namespace
}  // namespace krsi

using namespace krsi;

extern "C" int krsi_geglu_q8_fwd(const void* u, void* out, void* q, void* exponents, int64_t rows, int64_t F,
                                 int dtype, cudaStream_t stream) {
  const int rc = check(rows, F, dtype);
  if (rc != KRSI_OK) return rc;
  if (rows == 0 || F == 0) return KRSI_OK;
  KRSI_CHECK_ARG(u && out && (q != nullptr) == (exponents != nullptr));
  const int es = dtype == KRSI_F32 ? 4 : 2;
  const int vec = access_cols(F, es, bits_of(u) | bits_of(out), bits_of(q));
  KRSI_Q8_DISPATCH(fwd, vec, u, out, q, exponents, rows, F, stream)
}

extern "C" int krsi_geglu_q8_bwd(const void* g, const void* q, const void* exponents, void* du, void* out,
                                 int64_t rows, int64_t F, int dtype, cudaStream_t stream) {
  const int rc = check(rows, F, dtype);
  if (rc != KRSI_OK) return rc;
  if (rows == 0 || F == 0) return KRSI_OK;
  KRSI_CHECK_ARG(g && q && exponents && du);
  const int es = dtype == KRSI_F32 ? 4 : 2;
  const int vec = access_cols(F, es, bits_of(g) | bits_of(du) | bits_of(out), bits_of(q));
  KRSI_Q8_DISPATCH(bwd, vec, g, q, exponents, du, out, rows, F, stream)
}
